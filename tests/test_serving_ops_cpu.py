"""Serving operators without a GPU: the C ABI's symbols and struct layouts, sizes, and
what the Python calls and the entry points refuse before any device is touched."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

from actune_b200 import _lib, ops

ROOT = Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "actune_b200_serving.h").read_text()


def struct_of(name):
    """The header's struct as a ctypes class."""
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, flags=re.S).group(1)
    fields = []
    for line in filter(None, (part.strip() for part in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"))):
        kind = ctypes.c_void_p if "*" in line else {"size_t": ctypes.c_size_t, "int64_t": ctypes.c_int64,
                                                    "int32_t": ctypes.c_int32, "float": ctypes.c_float}[line.split()[0]]
        fields += [(n.strip(" *"), kind) for n in re.sub(r"^(const )?\w+\s*\**", "", line).split(",")]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


GatedNormArgs, AdapterArgs, PrefixAttentionArgs = (struct_of(f"actune_{n}_args") for n in (
    "gated_norm", "adapter", "prefix_attention"))


def test_every_declared_symbol_is_exported_and_bound():
    declared = set(re.findall(r"^\s*(?:int|size_t)\s+(actune_[a-z0-9_]+)\s*\(", HEADER, flags=re.M))
    assert declared == set(_lib.SERVING_EXPORTS)
    library = ctypes.CDLL(str(_lib.LIB_PATH))
    for name in declared:
        assert hasattr(library, name)


def test_entry_points_refuse_before_touching_a_device():
    L = _lib.lib()
    for entry, struct in ((L.actune_gated_norm, GatedNormArgs), (L.actune_adapter_add, AdapterArgs),
                          (L.actune_prefix_attention, PrefixAttentionArgs)):
        assert entry(None, None) == _lib.ERR_INVALID_VALUE
        assert entry(ctypes.byref(struct()), None) == _lib.ERR_INVALID_VALUE  # struct_bytes missing
    size = ctypes.sizeof(GatedNormArgs)
    good = dict(struct_bytes=size, T=2, D=64, eps=1e-6, dtype=_lib.DTYPE_BF16, x_stride=64, residual_stride=64)
    for bad in (dict(T=-1), dict(D=0), dict(dtype=7), dict(quant_bits=3), dict(D=60, quant_bits=8), dict(eps=-1.0),
                dict(eps=float("nan")), dict(gate_rows=-1), {}):  # the last: null pointers
        assert L.actune_gated_norm(ctypes.byref(GatedNormArgs(**{**good, **bad})), None) == _lib.ERR_INVALID_VALUE
    size = ctypes.sizeof(AdapterArgs)
    good = dict(struct_bytes=size, M=4, N=8, K=8, S=2, R=4, x_stride=8, y_stride=8, out_stride=8, tile=16,
                dtype=_lib.DTYPE_BF16)
    for bad in (dict(tile=17), dict(R=0), dict(R=129), dict(S=0), dict(S=9000), dict(M=-1), dict(K=0), dict(N=-1),
                dict(dtype=_lib.DTYPE_F32), dict(out_stride=7)):
        assert L.actune_adapter_add(ctypes.byref(AdapterArgs(**{**good, **bad})), None) == _lib.ERR_INVALID_VALUE
    assert L.actune_adapter_plan(None, 4, 2, 16, None, None) == _lib.ERR_INVALID_VALUE


def test_attention_entry_refuses_before_touching_a_device():
    L = _lib.lib()
    good = dict(struct_bytes=ctypes.sizeof(PrefixAttentionArgs), B=2, T=1, H=4, KV=2, D=64, G=1, P=8, S=4,
                scale=0.125, dtype=_lib.DTYPE_BF16)
    for bad in (dict(H=3), dict(KV=0), dict(D=0), dict(D=257), dict(G=0), dict(P=-1), dict(S=-1), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(dtype=_lib.DTYPE_F32),
                dict(pk_p=-64), dict(B=1 << 21), dict(T=1 << 25)):
        args = PrefixAttentionArgs(**{**good, **bad})
        assert L.actune_prefix_attention(ctypes.byref(args), None) == _lib.ERR_INVALID_VALUE, bad


def test_attention_refuses_operands_that_do_not_fit():
    q, pk, k = torch.zeros(4, 2, 4, 64).half(), torch.zeros(2, 9, 2, 64).half(), torch.zeros(4, 5, 2, 64).half()

    def call(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.shared_prefix_attention(*args, **kw)

    call("CUDA required", q, pk, pk, k, k)
    call("4-D", q[0], pk, pk, k, k)
    call("unsupported dtype", q.float(), pk, pk, k, k)
    call("multiple of the key/value heads", q[:, :, :3], pk, pk, k, k)
    call("head size", torch.zeros(4, 2, 4, 264).half(), torch.zeros(2, 9, 2, 264).half(), pk, k, k)
    call("prefix_k and prefix_v", q, pk, pk[:, :8], k, k)
    call("prefix_k and prefix_v", q, pk[..., :32], pk[..., :32], k, k)
    call("k and v must be", q, pk, pk, k[:3], k[:3])
    call("k and v must be", q, pk, pk, k[:, :, :1], k[:, :, :1])
    call("one dtype", q, pk.bfloat16(), pk, k, k)
    call("last dimension", q, pk.transpose(1, 3).contiguous().transpose(1, 3), pk, k, k)


def test_adapter_sizes():
    L = _lib.lib()
    # tiles: 100 / 16 full ones and one more for each of 3 adapters and "none"
    assert L.actune_adapter_plan_size(100, 3, 16) == 4 * (4 + 4 * (6 + 4) + 100)
    assert L.actune_adapter_plan_size(0, 3, 16) == 16
    assert L.actune_adapter_plan_size(100, 3, 8) == 0 and L.actune_adapter_plan_size(-1, 3, 16) == 0
    assert L.actune_adapter_workspace_size(1, 4096, 1, 8, 16) == 32 * 16 * 4  # 32 slices of K, rank padded to 16
    assert L.actune_adapter_workspace_size(100000, 4096, 1, 100, 128) == 100000 * (128 + 1) * 4
    assert L.actune_adapter_workspace_size(1, 4096, 1, 129, 16) == 0


def test_gated_norm_refuses_operands_that_do_not_fit():
    x, w = torch.zeros(6, 64).bfloat16(), torch.zeros(64).bfloat16()

    def call(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.gated_norm(*args, **kw)

    call("CUDA required", x, x, w)
    call(r"\[T, D\]", x[0], x[0], w)
    call("one shape", x, x[:4], w)
    call("one dtype", x, x.half(), w)
    call("unsupported dtype", x.double(), x.double(), w)
    call("pre_weight is required", x, x, None)
    call("last dimension", x.t(), x.t(), w)
    call("integer width", x, x, w, quant_bits=3)
    call("multiple of 64", x[:, :60], x[:, :60], w[:60], quant_bits=8)


def test_adapter_add_refuses_operands_that_do_not_fit():
    y, x, s = torch.zeros(6, 32).half(), torch.zeros(6, 16).half(), torch.ones(2)
    down, up = torch.zeros(2, 4, 16).half(), torch.zeros(2, 32, 4).half()
    plan = ops.AdapterPlan(torch.zeros(64, dtype=torch.int32), 6, 2, 16)

    def call(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.adapter_add(*args, **kw)

    call("CUDA required", y, x, down, up, s, plan)
    call("x and y must be", y[0], x[0], down, up, s, plan)
    call("x and y must be", y, x[:5], down, up, s, plan)
    call("down must be", y, x, down[:, :, :8], up, s, plan)
    call("down must be", y, x, down, up[:, :, :2], s, plan)
    call("rank", y, x, torch.zeros(2, 129, 16).half(), torch.zeros(2, 32, 129).half(), s, plan)
    call("unsupported dtype", y.float(), x.float(), down, up, s, plan)
    call("one dtype", y, x.bfloat16(), down, up, s, plan)
    call("scale", y, x, down, up, s.half(), plan)
    call("contiguous adapters", y, x, torch.zeros(2, 16, 4).half().transpose(1, 2), up, s, plan)
    call("the plan is for", y[:5], x[:5], down, up, s, plan)
    call("out must match", y, x, down, up, s, plan, out=y[:5])
    call("must not overlap", y, x, down, up, s, plan, out=y[:1].expand(6, 32))
    with pytest.raises(RuntimeError, match="int32"):
        ops.adapter_plan(torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="CUDA required"):
        ops.adapter_plan(torch.zeros(4, dtype=torch.int32), 2)


def test_outputs_that_require_a_gradient_are_refused():
    y, x, s = torch.zeros(6, 32).half(), torch.zeros(6, 16).half(), torch.ones(2)
    down, up = torch.zeros(2, 4, 16).half(), torch.zeros(2, 32, 4).half()
    plan = ops.AdapterPlan(torch.zeros(64, dtype=torch.int32), 6, 2, 16)
    q, pk, k = torch.zeros(4, 2, 4, 64).half(), torch.zeros(2, 9, 2, 64).half(), torch.zeros(4, 5, 2, 64).half()
    for call in (lambda out: ops.adapter_add(y, x, down, up, s, plan, out=out(y)),
                 lambda out: ops.shared_prefix_attention(q, pk, pk, k, k, out=out(q))):
        with pytest.raises(RuntimeError, match="no backward"):
            call(lambda t: t.clone().requires_grad_())
        with pytest.raises(RuntimeError, match="no backward"):
            call(lambda t: t.clone().requires_grad_() * 2)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA required"):
            call(lambda t: t.clone().requires_grad_())


def test_adapter_sizes_whose_last_step_would_pass_31_bits_are_refused():
    """A block walks up to 16 steps of 128 columns or 8 of 256, and a slice of K is rounded up to
    128 elements for each of 32: the indexes behind the last one are 32-bit too."""
    L = _lib.lib()
    good = dict(struct_bytes=ctypes.sizeof(AdapterArgs), M=1, N=8, K=8, S=1, R=8, x_stride=8, y_stride=8,
                out_stride=0x7fffff00, tile=4, dtype=_lib.DTYPE_BF16)
    for bad in (dict(N=0x7fffff00), dict(N=0x7ffff000), dict(K=0x7fffff00), dict(K=0x7ffff800)):
        args = AdapterArgs(**{**good, **bad})
        assert L.actune_adapter_add(ctypes.byref(args), None) == _lib.ERR_INVALID_VALUE, bad
    assert L.actune_adapter_workspace_size(1, 0x7fffff00, 1, 8, 4) == 0
    assert L.actune_adapter_workspace_size(1, 0x7fff0000, 1, 8, 4) > 0


@pytest.mark.parametrize("source", ["prefix_attention.cu", "adapters.cu"])
def test_dependents_are_let_in_behind_the_tensor_memory_allocation(source):
    """A dependent launch may take an SM's tensor memory as soon as every block has signalled,
    and then waits for this launch to end: a block that has not allocated by then never does."""
    text = (ROOT / "actune_b200" / "csrc" / source).read_text()
    kernels = [part for part in text.split("__global__")[1:] if "tmem_alloc(" in part]
    assert kernels
    for kernel in kernels:
        kernel = re.sub(r"//.*", "", kernel)
        signal = re.search(r"griddep_(enter|launch_dependents)\(", kernel).start()
        allocated = kernel.index("tmem_alloc(")
        assert allocated < signal and "__syncthreads();" in kernel[allocated:signal]
