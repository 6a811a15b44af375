// Norm after a block, gate, residual scale and the norm before the next block, in one
// pass (sm_100a):
//   u = N(x; post)   s = alpha * residual + gate * u   h = N(s; pre) + shift
// Bound by HBM: a row is read once (x, residual) and written once (h, s), 4 * D values
// for about 12 flops each, so a row's values stay in registers between the two norms
// and the modulation rows come from L1/L2.  The second mean square needs s, which needs
// the first: two reductions over the row that cannot be merged.
//
// TPR threads share a row and hold CPT chunks of 8 values each.  Rows of up to 2048
// values belong to one warp when there are many of them (no block barrier between load
// and store, and the warps of an SM are in different phases); few rows are spread over
// more threads, since one row then has the SM's load latency to itself.
#include "serving.cuh"

namespace actune {
namespace {

struct NormParams {
  const void *x, *residual, *post, *pre, *gate, *shift;
  void *out, *residual_out;
  uint8_t* packed;
  float* scales;
  int64_t T, x_stride, residual_stride, post_rows, pre_rows, gate_rows, shift_rows;
  int D;
  float alpha, eps, one;  // one: what the weights are relative to (gemma 1, else 0)
  int bits, codes8;
};

template <typename T>
__device__ __forceinline__ const T* modulation(const void* base, int64_t rows, int64_t row, int D) {
  return reinterpret_cast<const T*>(base) + (rows ? row / rows : 0) * (int64_t)D;
}

// Sum over the threads of a row (TPR of them, consecutive).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += red[i];
  }
  return v;
}

// The group-64 codes of a lane's 8 rounded values; all 32 lanes call together.
__device__ __forceinline__ void emit_codes(const NormParams& p, const float (&v)[8], int64_t element, bool live) {
  uint32_t word[2];
  float scale;
  int width = p.bits;
  if (p.bits == 8) {
    scale = quantize_lane8<8>(v, word);
  } else if (p.codes8) {
    width = 8;
    scale = p.bits == 4 ? quantize_lane8<4, 8>(v, word) : quantize_lane8<2, 8>(v, word);
  } else {
    scale = p.bits == 4 ? quantize_lane8<4>(v, word) : quantize_lane8<2>(v, word);
  }
  if (!live) return;
  uint8_t* dst = p.packed + element / 8 * width;
  if (width == 8) store_lane_codes<8>(dst, word);
  else if (width == 4) store_lane_codes<4>(dst, word);
  else store_lane_codes<2>(dst, word);
  if ((threadIdx.x & 7) == 0) p.scales[element / 64] = scale;
}

template <typename T, int TPR, int CPT>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128) gated_norm_kernel(const NormParams p) {
  constexpr int ROWS = TPR > 128 ? 1 : 128 / TPR;
  __shared__ float red[2][32];
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  griddep_enter();  // dependent launch: x is the previous kernel's output
  if (row >= p.T) return;  // ROWS > 1 only with one warp per row: no barrier follows
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
  const T* res = reinterpret_cast<const T*>(p.residual) + row * p.residual_stride;
  Raw8<T> xr[CPT], rr[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + lane) * 8;
    if (i < p.D) {
      xr[c].load(x + i);
      rr[c].load(res + i);
    }
  }
  float v[CPT][8];
  float inv = 1.f;
  if (p.post) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      if ((c * TPR + lane) * 8 >= p.D) continue;
      xr[c].get(v[c]);
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(v[c][k], v[c][k], ss);
    }
    inv = rsqrtf(row_sum<TPR>(ss, red[0]) / (float)p.D + p.eps);
  }
  const T* post = p.post ? modulation<T>(p.post, p.post_rows, row, p.D) : nullptr;
  const T* gate = p.gate ? modulation<T>(p.gate, p.gate_rows, row, p.D) : nullptr;
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + lane) * 8;
    if (i >= p.D) continue;
    float w[8];
    xr[c].get(v[c]);
    Raw8<T> m;
    if (post) {
      m.load(post + i);
      m.get(w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = v[c][k] * inv * (p.one + w[k]);
    }
    if (gate) {
      m.load(gate + i);
      m.get(w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] *= w[k];
    }
    rr[c].get(w);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[c][k] = fmaf(p.alpha, w[k], v[c][k]);
      ss = fmaf(v[c][k], v[c][k], ss);
    }
    m.set(v[c]);
    m.store(reinterpret_cast<T*>(p.residual_out) + row * p.D + i);
  }
  inv = rsqrtf(row_sum<TPR>(ss, red[1]) / (float)p.D + p.eps);
  const T* pre = modulation<T>(p.pre, p.pre_rows, row, p.D);
  const T* shift = p.shift ? modulation<T>(p.shift, p.shift_rows, row, p.D) : nullptr;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + lane) * 8;
    const bool live = i < p.D;
    float w[8];
    if (live) {
      Raw8<T> m;
      m.load(pre + i);
      m.get(w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = v[c][k] * inv * (p.one + w[k]);
      if (shift) {
        m.load(shift + i);
        m.get(w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c][k] += w[k];
      }
      m.set(v[c]);
      m.store(reinterpret_cast<T*>(p.out) + row * p.D + i);
      m.get(v[c]);  // the codes are those of the rounded values
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = 0.f;
    }
    if (p.bits) emit_codes(p, v[c], row * p.D + i, live);
  }
}

// Any width, alignment and stride: one CTA per row, values read again for each pass.
template <typename T>
__global__ void __launch_bounds__(256) gated_norm_any_kernel(const NormParams p) {
  __shared__ float red[2][32];
  griddep_enter();
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
  const T* res = reinterpret_cast<const T*>(p.residual) + row * p.residual_stride;
  const T* post = p.post ? modulation<T>(p.post, p.post_rows, row, p.D) : nullptr;
  const T* gate = p.gate ? modulation<T>(p.gate, p.gate_rows, row, p.D) : nullptr;
  const T* pre = modulation<T>(p.pre, p.pre_rows, row, p.D);
  const T* shift = p.shift ? modulation<T>(p.shift, p.shift_rows, row, p.D) : nullptr;
  float inv = 1.f, ss = 0.f;
  if (post) {
    for (int i = threadIdx.x; i < p.D; i += 256) {
      const float a = widen<T>(x[i]);
      ss = fmaf(a, a, ss);
    }
    inv = rsqrtf(row_sum<256>(ss, red[0]) / (float)p.D + p.eps);
  }
  const auto stream_value = [&](int i) {
    float a = widen<T>(x[i]);
    if (post) a = a * inv * (p.one + widen<T>(post[i]));
    if (gate) a *= widen<T>(gate[i]);
    return fmaf(p.alpha, widen<T>(res[i]), a);
  };
  ss = 0.f;
  for (int i = threadIdx.x; i < p.D; i += 256) {
    const float s = stream_value(i);
    ss = fmaf(s, s, ss);
    reinterpret_cast<T*>(p.residual_out)[row * p.D + i] = narrow<T>(s);
  }
  const float inv2 = rsqrtf(row_sum<256>(ss, red[1]) / (float)p.D + p.eps);
  for (int i = threadIdx.x; i < p.D; i += 256) {
    float h = stream_value(i) * inv2 * (p.one + widen<T>(pre[i]));
    if (shift) h += widen<T>(shift[i]);
    reinterpret_cast<T*>(p.out)[row * p.D + i] = narrow<T>(h);
  }
}

template <typename T, int TPR, int CPT>
cudaError_t launch_rows(const NormParams& p, cudaStream_t stream) {
  constexpr int THREADS = TPR > 128 ? TPR : 128;
  return launch_pdl(gated_norm_kernel<T, TPR, CPT>, dim3((unsigned)ceil_div(p.T, THREADS / TPR)), THREADS, 0, stream,
                    p);
}

template <typename T>
cudaError_t launch_norm(const NormParams& p, bool vec, int num_sms, cudaStream_t stream) {
  if (!vec) return launch_pdl(gated_norm_any_kernel<T>, dim3((unsigned)p.T), 256, 0, stream, p);
  const int chunks = (p.D + 7) / 8;
  if (p.T >= (int64_t)num_sms * 8) {
    if (chunks <= 32) return launch_rows<T, 32, 1>(p, stream);
    if (chunks <= 64) return launch_rows<T, 32, 2>(p, stream);
    if (chunks <= 128) return launch_rows<T, 32, 4>(p, stream);
    if (chunks <= 256) return launch_rows<T, 32, 8>(p, stream);
  }
  if (chunks <= 128) return launch_rows<T, 128, 1>(p, stream);
  if (chunks <= 256) return launch_rows<T, 128, 2>(p, stream);
  if (chunks <= 512) return launch_rows<T, 512, 1>(p, stream);
  if (chunks <= 1024) return launch_rows<T, 512, 2>(p, stream);
  return launch_rows<T, 512, 4>(p, stream);
}

}  // namespace
}  // namespace actune

extern "C" int actune_gated_norm(const actune_gated_norm_args* a, void* stream) {
  using namespace actune;
  if (a == nullptr || a->struct_bytes != sizeof(actune_gated_norm_args)) return ACTUNE_ERR_INVALID_VALUE;
  if (a->T < 0 || a->T > 0x7fffffff || a->D <= 0 || a->D > (1 << 24) || a->post_rows < 0 || a->pre_rows < 0 ||
      a->gate_rows < 0 || a->shift_rows < 0 || a->x_stride < 0 || a->residual_stride < 0 || !(a->eps >= 0.f) ||
      (a->dtype != ACTUNE_DTYPE_F32 && a->dtype != ACTUNE_DTYPE_F16 && a->dtype != ACTUNE_DTYPE_BF16) ||
      (a->quant_bits != 0 && a->quant_bits != 2 && a->quant_bits != 4 && a->quant_bits != 8) ||
      (a->quant_bits != 0 && a->D % 64 != 0))
    return ACTUNE_ERR_INVALID_VALUE;
  if (a->T > 0 && (a->x == nullptr || a->residual == nullptr || a->pre_weight == nullptr || a->out == nullptr ||
                   a->residual_out == nullptr || (a->quant_bits != 0 && (a->packed == nullptr || a->scales == nullptr))))
    return ACTUNE_ERR_INVALID_VALUE;
  int num_sms = 0;
  const int rc = serving_device(&num_sms);
  if (rc != ACTUNE_OK || a->T == 0) return rc;
  const uintptr_t size = a->dtype == ACTUNE_DTYPE_F32 ? 4 : 2;
  for (const void* q : {a->x, a->residual, a->post_weight, a->pre_weight, a->gate, a->shift,
                        (const void*)a->out, (const void*)a->residual_out})
    if (!is_aligned(q, size)) return ACTUNE_ERR_MISALIGNED;
  if (a->quant_bits != 0 && (!is_aligned(a->packed, 8) || !is_aligned(a->scales, 4) || !is_aligned(a->out, 16)))
    return ACTUNE_ERR_MISALIGNED;
  bool vec = a->D % 8 == 0 && a->D <= 512 * 4 * 8 && a->x_stride % 8 == 0 && a->residual_stride % 8 == 0;
  for (const void* q : {a->x, a->residual, a->post_weight, a->pre_weight, a->gate, a->shift,
                        (const void*)a->out, (const void*)a->residual_out})
    vec = vec && is_aligned(q, 16);
  NormParams p = {a->x, a->residual, a->post_weight, a->pre_weight, a->gate, a->shift, a->out, a->residual_out,
                  a->packed, a->scales, a->T, a->x_stride, a->residual_stride, a->post_rows, a->pre_rows,
                  a->gate_rows, a->shift_rows, (int)a->D, a->residual_scale, a->eps, a->gemma ? 1.f : 0.f,
                  vec ? a->quant_bits : 0, a->codes8};
  auto* cs = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = a->dtype == ACTUNE_DTYPE_F32   ? launch_norm<float>(p, vec, num_sms, cs)
                  : a->dtype == ACTUNE_DTYPE_F16 ? launch_norm<__half>(p, vec, num_sms, cs)
                                                 : launch_norm<__nv_bfloat16>(p, vec, num_sms, cs);
  if (e == cudaSuccess && a->quant_bits != 0 && !vec)
    e = launch_quantize_group64(a->out, a->dtype, a->T * (a->D / 64), a->quant_bits, a->codes8 != 0, a->packed,
                                a->scales, num_sms, cs);
  return serving_status(e);
}
