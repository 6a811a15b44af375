// Torch-tensor face of the serving operators (include/actune_b200_serving.h) as a
// CPython module: argument checks, output allocation, device and stream, one C-ABI call.
//
// It is C++ because a call for one token costs the host more than the GPU: the same
// checks, allocations and struct in Python (ctypes) measured 22-28 us a call against 3 us
// for the C entry itself.  Functions take positional arguments only (the Python functions
// of actune_b200/serving_ops.py name them), return the outputs, or an int: the non-zero
// status of the C entry.  Operands that do not fit raise RuntimeError; no C++ exception
// leaves the module.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "actune_b200.h"
#include "actune_b200_serving.h"

namespace {

using at::Tensor;

std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::ScalarType t) { return c10::toString(t); }
template <typename... Args>
[[noreturn]] void refuse(const Args&... args) {
  throw std::runtime_error((text(args) + ...));
}
#define REQUIRE(cond, ...) \
  do {                     \
    if (!(cond)) [[unlikely]] refuse(__VA_ARGS__); \
  } while (0)

// Tensor argument; None gives an undefined tensor where `optional`.
const Tensor& tensor(PyObject* o, const char* name, bool optional = false) {
  static const Tensor none;
  if (THPVariable_Check(o)) return THPVariable_Unpack(o);
  REQUIRE(optional && o == Py_None, name, optional ? " must be a tensor or None" : " must be a tensor");
  return none;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  REQUIRE(v >= 0, "a truth value is required");
  return v != 0;
}
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  REQUIRE(!(v == -1.0 && PyErr_Occurred()), name, " must be a number");
  return v;
}
int64_t whole(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  REQUIRE(!(v == -1 && PyErr_Occurred()), name, " must be a whole number");
  return v;
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? ACTUNE_DTYPE_F32 : t == at::kHalf ? ACTUNE_DTYPE_F16 : t == at::kBFloat16 ? ACTUNE_DTYPE_BF16
                                                                                                  : ACTUNE_DTYPE_NONE;
}
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

struct Named {
  const char* name;
  const Tensor* t;
};
c10::Device one_device(const Tensor& first, std::initializer_list<Named> others) {
  REQUIRE(first.is_cuda(), "CUDA required");
  for (const Named& o : others)
    REQUIRE(!o.t->defined() || o.t->device() == first.device(), "device mismatch: ", o.name, " is on ",
            o.t->device().str());
  return first.device();
}
Tensor empty(at::IntArrayRef size, at::ScalarType dtype, c10::Device device) {
  return at::empty(size, at::TensorOptions().dtype(dtype).device(device));
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* stream(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

// `out` given by the caller is written behind autograd's back.  Refused where a gradient
// would be taken through it; otherwise its version tells a backward pass that saved it.
void check_written(const Tensor& out) {
  REQUIRE(!(c10::GradMode::is_enabled() && out.requires_grad()),
          "out requires a gradient, and the serving operators have no backward: run them under torch.no_grad()");
}
void mark_written(const Tensor& out) {
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

PyObject* outputs(std::initializer_list<Tensor> list) {
  PyObject* tuple = PyTuple_New((Py_ssize_t)list.size());
  if (tuple == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : list) {
    PyObject* o = THPVariable_Wrap(t);
    if (o == nullptr) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// ------------------------------------------------------------------- gated norm
// Rows of the batch that share a row of modulation t ([width] or [groups, width]).
int64_t rows_of(const Tensor& t, int64_t width, int64_t rows, at::ScalarType dtype, const char* name) {
  if (!t.defined()) return 0;
  REQUIRE(t.scalar_type() == dtype, name, " must have the activations' dtype");
  REQUIRE(t.is_contiguous(), name, " must be contiguous");
  REQUIRE((t.dim() == 1 || t.dim() == 2) && t.size(-1) == width, name, " must be [", width, "] or [groups, ", width, "]");
  if (t.dim() == 1) return 0;
  const int64_t groups = t.size(0);
  REQUIRE(groups > 0 && rows % groups == 0, name, " has ", groups, " rows, which do not divide ", rows);
  return rows / groups;
}

// x, residual, pre_weight, post_weight, gate, shift, residual_scale, eps, gemma, quant_bits, codes8
PyObject* gated_norm(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "x");
  const Tensor& residual = tensor(a[1], "residual");
  REQUIRE(a[2] != Py_None, "pre_weight is required");
  const Tensor& pre = tensor(a[2], "pre_weight");
  const Tensor& post = tensor(a[3], "post_weight", true);
  const Tensor& gate = tensor(a[4], "gate", true);
  const Tensor& shift = tensor(a[5], "shift", true);
  REQUIRE(x.dim() == 2 && residual.sizes() == x.sizes(), "x and residual must be [T, D] of one shape");
  const at::ScalarType dtype = x.scalar_type();
  REQUIRE(dtype_code(dtype) != ACTUNE_DTYPE_NONE, "unsupported dtype ", dtype,
          " (float32, float16 or bfloat16 required)");
  REQUIRE(residual.scalar_type() == dtype, "x and residual must have one dtype");
  const int64_t rows = x.size(0), width = x.size(1);
  REQUIRE(width > 0 && (width == 1 || (x.stride(1) == 1 && residual.stride(1) == 1)),
          "the last dimension must be contiguous");
  const int64_t bits = a[9] == Py_None ? 0 : whole(a[9], "quant_bits");
  REQUIRE(bits == 0 || bits == 2 || bits == 4 || bits == 8, "Unsupported integer width");
  REQUIRE(bits == 0 || width % 64 == 0, "D must be a multiple of 64 to be quantized");
  const bool codes8 = truth(a[10]);
  actune_gated_norm_args g = {};
  g.struct_bytes = sizeof(g);
  g.post_rows = rows_of(post, width, rows, dtype, "post_weight");
  g.pre_rows = rows_of(pre, width, rows, dtype, "pre_weight");
  g.gate_rows = rows_of(gate, width, rows, dtype, "gate");
  g.shift_rows = rows_of(shift, width, rows, dtype, "shift");
  const c10::Device device = one_device(x, {{"residual", &residual}, {"pre_weight", &pre}, {"post_weight", &post},
                                            {"gate", &gate}, {"shift", &shift}});
  const c10::cuda::CUDAGuard guard(device);
  const Tensor out = empty({rows, width}, dtype, device), stream_out = empty({rows, width}, dtype, device);
  Tensor packed, scales;
  if (bits != 0) {
    packed = empty({rows, width * (codes8 ? 8 : bits) / 8}, at::kByte, device);
    scales = empty({rows, width / 64}, at::kFloat, device);
    g.packed = static_cast<uint8_t*>(packed.data_ptr());
    g.scales = static_cast<float*>(scales.data_ptr());
  }
  g.x = ptr(x), g.residual = ptr(residual), g.post_weight = ptr(post), g.pre_weight = ptr(pre), g.gate = ptr(gate);
  g.shift = ptr(shift), g.out = out.data_ptr(), g.residual_out = stream_out.data_ptr();
  g.T = rows, g.D = width, g.x_stride = row_stride(x), g.residual_stride = row_stride(residual);
  g.residual_scale = (float)number(a[6], "residual_scale"), g.eps = (float)number(a[7], "eps");
  g.dtype = dtype_code(dtype), g.gemma = truth(a[8]), g.quant_bits = (int32_t)bits, g.codes8 = codes8;
  const int status = actune_gated_norm(&g, stream(device));
  if (status != ACTUNE_OK) return PyLong_FromLong(status);
  return bits != 0 ? outputs({out, stream_out, packed, scales}) : outputs({out, stream_out});
}

// ------------------------------------------------------------------- adapters
// y, x, down, up, scale, plan buffer, plan rows, plan adapters, plan tile, out
PyObject* adapter_add(PyObject* const* a) {
  const Tensor& y = tensor(a[0], "y");
  const Tensor& x = tensor(a[1], "x");
  const Tensor& down = tensor(a[2], "down");
  const Tensor& up = tensor(a[3], "up");
  const Tensor& scale = tensor(a[4], "scale");
  const Tensor& plan = tensor(a[5], "plan");
  const int64_t plan_rows = whole(a[6], "rows"), plan_slots = whole(a[7], "adapters"), tile = whole(a[8], "tile");
  Tensor out = tensor(a[9], "out", true);
  REQUIRE(x.dim() == 2 && y.dim() == 2 && x.size(0) == y.size(0), "x and y must be [M, K] and [M, N]");
  const int64_t rows = x.size(0), k = x.size(1), n = y.size(1);
  REQUIRE(down.dim() == 3 && up.dim() == 3, "down must be [S, R, K] and up [S, N, R]");
  const int64_t slots = down.size(0), rank = down.size(1);
  REQUIRE(down.size(2) == k && up.size(0) == slots && up.size(1) == n && up.size(2) == rank, "down must be [S, R, ", k,
          "] and up [S, ", n, ", R]");
  REQUIRE(rank >= 1 && rank <= 128, "the adapters' rank must be between 1 and 128");
  const at::ScalarType dtype = x.scalar_type();
  REQUIRE(dtype == at::kHalf || dtype == at::kBFloat16, "unsupported dtype ", dtype,
          " (float16 or bfloat16 required)");
  REQUIRE(y.scalar_type() == dtype && down.scalar_type() == dtype && up.scalar_type() == dtype,
          "x, y, down and up must have one dtype");
  REQUIRE(scale.scalar_type() == at::kFloat && scale.numel() == slots, "scale must be float32 [S]");
  REQUIRE(down.is_contiguous() && up.is_contiguous() && scale.is_contiguous(), "contiguous adapters required");
  REQUIRE(plan_rows == rows && plan_slots == slots, "the plan is for ", plan_rows, " rows and ", plan_slots,
          " adapters, got ", rows, " and ", slots);
  REQUIRE(plan.scalar_type() == at::kInt && plan.is_contiguous() &&
              plan.numel() * 4 >= (int64_t)actune_adapter_plan_size(rows, slots, (int)tile),
          "the plan's buffer is too small");
  if (out.defined()) {
    REQUIRE(out.dim() == 2 && out.sizes() == y.sizes() && out.scalar_type() == dtype, "out must match y");
    // Rows of `out` that overlap would be written while others read them.
    REQUIRE(rows <= 1 || out.stride(0) >= n, "the rows of out must not overlap");
    REQUIRE(n <= 1 || out.stride(1) == 1, "the last dimension must be contiguous");
    check_written(out);
  }
  REQUIRE((k <= 1 || x.stride(1) == 1) && (n <= 1 || y.stride(1) == 1), "the last dimension must be contiguous");
  const c10::Device device =
      one_device(x, {{"y", &y}, {"down", &down}, {"up", &up}, {"scale", &scale}, {"plan", &plan}, {"out", &out}});
  const c10::cuda::CUDAGuard guard(device);
  if (!out.defined()) out = empty({rows, n}, dtype, device);
  actune_adapter_args g = {};
  g.struct_bytes = sizeof(g);
  g.workspace_bytes = actune_adapter_workspace_size(rows, k, slots, rank, (int)tile);
  Tensor workspace;
  if (g.workspace_bytes > 0) {
    workspace = empty({(int64_t)g.workspace_bytes}, at::kByte, device);
    g.workspace = workspace.data_ptr();
  }
  g.x = ptr(x), g.y = ptr(y), g.down = ptr(down), g.up = ptr(up), g.scale = static_cast<const float*>(ptr(scale));
  g.plan = static_cast<const int32_t*>(ptr(plan)), g.out = out.data_ptr();
  g.M = rows, g.N = n, g.K = k, g.S = slots, g.R = rank;
  g.x_stride = row_stride(x), g.y_stride = row_stride(y), g.out_stride = row_stride(out);
  g.tile = (int32_t)tile, g.dtype = dtype_code(dtype);
  const int status = actune_adapter_add(&g, stream(device));
  mark_written(out);
  return status != ACTUNE_OK ? PyLong_FromLong(status) : THPVariable_Wrap(out);
}

// ------------------------------------------------------------------- attention
const int32_t* lengths(const Tensor& t, int64_t count, const char* name) {
  if (!t.defined()) return nullptr;
  REQUIRE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == count && t.is_contiguous(), name,
          " must be a contiguous int32 vector of ", count);
  return static_cast<const int32_t*>(t.const_data_ptr());
}

// q, prefix_k, prefix_v, k, v, starts, prefix_lens, lens, causal, scale, out
PyObject* shared_prefix_attention(PyObject* const* a) {
  const Tensor& q = tensor(a[0], "q");
  const Tensor& pk = tensor(a[1], "prefix_k");
  const Tensor& pv = tensor(a[2], "prefix_v");
  const Tensor& k = tensor(a[3], "k");
  const Tensor& v = tensor(a[4], "v");
  const Tensor& starts = tensor(a[5], "starts", true);
  const Tensor& plens = tensor(a[6], "prefix_lens", true);
  const Tensor& lens = tensor(a[7], "lens", true);
  Tensor out = tensor(a[10], "out", true);
  REQUIRE(q.dim() == 4 && pk.dim() == 4 && pv.dim() == 4 && k.dim() == 4 && v.dim() == 4,
          "q, prefix_k, prefix_v, k and v must be 4-D");
  const at::ScalarType dtype = q.scalar_type();
  REQUIRE(dtype == at::kHalf || dtype == at::kBFloat16, "unsupported dtype ", dtype,
          " (float16 or bfloat16 required)");
  actune_prefix_attention_args g = {};
  g.struct_bytes = sizeof(g);
  g.B = q.size(0), g.T = q.size(1), g.H = q.size(2), g.D = q.size(3);
  g.G = pk.size(0), g.P = pk.size(1), g.KV = pk.size(2), g.S = k.size(1);
  REQUIRE(g.G > 0 && g.KV > 0 && g.H > 0 && g.H % g.KV == 0,
          "the query heads must be a multiple of the key/value heads");
  REQUIRE(g.D >= 1 && g.D <= 256, "the head size must be between 1 and 256");
  REQUIRE(pk.size(3) == g.D && pv.sizes() == pk.sizes(), "prefix_k and prefix_v must be [G, P, KV, ", g.D, "]");
  REQUIRE(k.size(0) == g.B && k.size(2) == g.KV && k.size(3) == g.D && v.sizes() == k.sizes(), "k and v must be [",
          g.B, ", S, ", g.KV, ", ", g.D, "]");
  REQUIRE(pk.scalar_type() == dtype && pv.scalar_type() == dtype && k.scalar_type() == dtype &&
              v.scalar_type() == dtype,
          "q, keys and values must have one dtype");
  REQUIRE(g.D == 1 || (q.stride(3) == 1 && pk.stride(3) == 1 && pv.stride(3) == 1 && k.stride(3) == 1 &&
                       v.stride(3) == 1),
          "the last dimension must be contiguous");
  if (out.defined()) check_written(out);
  const c10::Device device =
      one_device(q, {{"prefix_k", &pk}, {"prefix_v", &pv}, {"k", &k}, {"v", &v}, {"starts", &starts},
                     {"prefix_lens", &plens}, {"lens", &lens}, {"out", &out}});
  g.starts = lengths(starts, g.G + 1, "starts");
  g.prefix_lens = lengths(plens, g.G, "prefix_lens");
  g.lens = lengths(lens, g.B, "lens");
  const double scale = a[9] == Py_None ? 1.0 / std::sqrt((double)g.D) : number(a[9], "scale");
  REQUIRE(scale > 0.0 && scale < 3e38, "scale must be positive and finite");
  const c10::cuda::CUDAGuard guard(device);
  if (out.defined())
    REQUIRE(out.sizes() == q.sizes() && out.scalar_type() == dtype && out.is_contiguous(),
            "out must be contiguous and match q");
  else
    out = empty(q.sizes(), dtype, device);
  g.workspace_bytes = actune_prefix_attention_workspace_size(g.B, g.T, g.H, g.KV, g.D, g.G, g.P, g.S, g.starts != nullptr);
  Tensor workspace;
  if (g.workspace_bytes > 0) {
    workspace = empty({(int64_t)g.workspace_bytes}, at::kByte, device);
    g.workspace = workspace.data_ptr();
  }
  g.q = ptr(q), g.prefix_k = ptr(pk), g.prefix_v = ptr(pv), g.k = ptr(k), g.v = ptr(v), g.out = out.data_ptr();
  g.q_b = q.stride(0), g.q_t = q.stride(1), g.q_h = q.stride(2);
  g.pk_g = pk.stride(0), g.pk_p = pk.stride(1), g.pk_h = pk.stride(2);
  g.pv_g = pv.stride(0), g.pv_p = pv.stride(1), g.pv_h = pv.stride(2);
  g.k_b = k.stride(0), g.k_s = k.stride(1), g.k_h = k.stride(2);
  g.v_b = v.stride(0), g.v_s = v.stride(1), g.v_h = v.stride(2);
  g.scale = (float)scale, g.dtype = dtype_code(dtype), g.causal = truth(a[8]);
  const int status = actune_prefix_attention(&g, stream(device));
  mark_written(out);
  return status != ACTUNE_OK ? PyLong_FromLong(status) : THPVariable_Wrap(out);
}

// ------------------------------------------------------------------- module
template <PyObject* (*F)(PyObject* const*), Py_ssize_t COUNT>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  try {
    REQUIRE(count == COUNT, (int64_t)COUNT, " arguments required, got ", (int64_t)count);
    return F(args);
  } catch (const c10::OutOfMemoryError& e) {  // keeps its Python type
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t COUNT>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, COUNT>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<gated_norm, 11>("gated_norm"), method<adapter_add, 10>("adapter_add"),
                         method<shared_prefix_attention, 11>("shared_prefix_attention"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
