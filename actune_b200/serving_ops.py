"""Tensor-level calls of the serving operators (include/actune_b200_serving.h),
re-exported by ``actune_b200.ops``.

* ``shared_prefix_attention``: attention of a batch whose sequences share prefixes.
* ``adapter_plan`` / ``adapter_add``: low-rank adapters of many requests added to the
  output of the projection they share.
* ``gated_norm``: norm after a block, gate, residual scale and the norm before the
  next block in one launch, optionally with the group-64 activations of the result.

Conventions of ``ops``: tensors on one CUDA device, that device's current stream,
RuntimeError for operands that do not fit, outputs and scratch from torch's allocator
(so they belong to the stream the call runs on).  Nothing here synchronises.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def _require(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _same_device(first, **others):
    """The CUDA device of `first`; every other tensor given has to be there too."""
    _require(first.is_cuda, "CUDA required")
    device = first.device
    for name, t in others.items():
        _require(t is None or t.device == device, f"device mismatch: {name} is on {None if t is None else t.device}")
    return device


def _call(entry, what, device, *args):
    """One C-ABI call on `device` and its current stream."""
    if torch.cuda.current_device() == device.index:
        status = entry(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            status = entry(*args, torch.cuda.current_stream(device).cuda_stream)
    if status != _lib.OK:
        _lib.check(status, what)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _row_stride(t):
    """Elements between rows of t [M, width] (a single row has none of its own)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


# ------------------------------------------------------------------------- gated norm
def _rows_of(t, width, rows, dtype, name):
    """Rows of the batch that share a row of modulation `t` ([width] or [groups, width])."""
    if t is None:
        return 0
    _require(t.dtype == dtype, f"{name} must have the activations' dtype {dtype}")
    _require(t.is_contiguous(), f"{name} must be contiguous")
    if t.dim() == 1:
        _require(t.shape[0] == width, f"{name} must be [{width}] or [groups, {width}]")
        return 0
    _require(t.dim() == 2 and t.shape[1] == width, f"{name} must be [{width}] or [groups, {width}]")
    _require(t.shape[0] > 0 and rows % t.shape[0] == 0, f"{name} has {t.shape[0]} rows, which do not divide {rows}")
    return rows // t.shape[0] if rows else 0


def gated_norm(x, residual, pre_weight, *, post_weight=None, gate=None, shift=None, residual_scale=1.0, eps=1e-6,
               gemma=False, quant_bits=None, codes8=False):
    """The glue between two blocks of a decoder layer in one pass over each row:

        u = N(x; post_weight)                     (x itself without post_weight)
        s = residual_scale * residual + gate * u  (no gate: u)
        h = N(s; pre_weight) + shift

    with N(a; w) = a * rsqrt(mean(a^2) + eps) * w (``gemma``: 1 + w).  x and residual
    are [T, D] (float32, float16 or bfloat16; rows may be strided).  Each of
    post_weight, pre_weight, gate and shift is [D] or [groups, D], where consecutive
    T / groups rows share one of its rows (a modulation per environment; groups = T:
    per token).  Returns (h, s) contiguous; s is rounded once, and h is computed from
    the unrounded s.

    ``quant_bits`` (2, 4 or 8; D a multiple of 64) also returns the group-64
    activations of h, (h, s, packed, scales), bit-identical to
    ``quantize_group64(h, quant_bits, codes8=codes8)``."""
    _require(x.dim() == 2 and residual.shape == x.shape, "x and residual must be [T, D] of one shape")
    dtype = x.dtype
    code = _DTYPES.get(dtype)
    _require(code is not None, f"unsupported dtype {dtype} (float32, float16 or bfloat16 required)")
    _require(residual.dtype == dtype, "x and residual must have one dtype")
    rows, width = x.shape
    _require(pre_weight is not None, "pre_weight is required")
    _require(width > 0 and (width == 1 or (x.stride(1) == 1 and residual.stride(1) == 1)),
             "the last dimension must be contiguous")
    _require(quant_bits in (None, 2, 4, 8), "Unsupported integer width")
    _require(not quant_bits or width % 64 == 0, "D must be a multiple of 64 to be quantized")
    device = _same_device(x, residual=residual, pre_weight=pre_weight, post_weight=post_weight, gate=gate, shift=shift)
    out = torch.empty((rows, width), device=device, dtype=dtype)
    new_residual = torch.empty((rows, width), device=device, dtype=dtype)
    packed = scales = None
    if quant_bits:
        stored = 8 if codes8 else quant_bits
        packed = torch.empty((rows, width * stored // 8), device=device, dtype=torch.uint8)
        scales = torch.empty((rows, width // 64), device=device, dtype=torch.float32)
    args = _lib.GatedNormArgs(
        ctypes.sizeof(_lib.GatedNormArgs), _ptr(x), _ptr(residual), _ptr(post_weight), _ptr(pre_weight), _ptr(gate),
        _ptr(shift), _ptr(out), _ptr(new_residual), _ptr(packed), _ptr(scales), rows, width, _row_stride(x),
        _row_stride(residual), _rows_of(post_weight, width, rows, dtype, "post_weight"),
        _rows_of(pre_weight, width, rows, dtype, "pre_weight"), _rows_of(gate, width, rows, dtype, "gate"),
        _rows_of(shift, width, rows, dtype, "shift"), residual_scale, eps, code, bool(gemma), quant_bits or 0,
        bool(codes8))
    _call(_lib.lib().actune_gated_norm, "gated_norm", device, args)
    return (out, new_residual, packed, scales) if quant_bits else (out, new_residual)


# ------------------------------------------------------------------------- adapters
@dataclass(frozen=True)
class AdapterPlan:
    """The rows of a batch sorted by adapter slot (made by ``adapter_plan``; read by
    every ``adapter_add`` the batch passes through).  ``update`` routes the same number
    of rows anew into the same buffer, so a captured graph follows it."""

    buffer: torch.Tensor
    rows: int
    adapters: int
    tile: int

    def update(self, slots):
        _check_slots(slots, self.buffer.device)
        _require(slots.shape[0] == self.rows, f"the plan was made for {self.rows} rows, got {slots.shape[0]}")
        _call(_lib.lib().actune_adapter_plan, "adapter_plan", slots.device, _ptr(slots), self.rows, self.adapters,
              self.tile, _ptr(self.buffer))
        return self


def _check_slots(slots, device):
    _require(slots.dim() == 1 and slots.dtype == torch.int32 and slots.is_contiguous(),
             "slots must be a contiguous int32 vector")
    _require(slots.is_cuda, "CUDA required")
    _require(slots.device == device, "device mismatch: slots")


def adapter_plan(slots, adapters):
    """Sort a batch's rows by adapter: slots int32 [M] on the GPU (row m runs adapter
    slots[m]; anything outside 0 .. adapters - 1 means none) -> AdapterPlan.

    Tiles of rows that share an adapter have 16, 32 or 64 rows, by the mean number of
    rows per adapter that the sizes allow."""
    _check_slots(slots, slots.device)
    rows = slots.shape[0]
    _require(1 <= adapters <= 8191, "between 1 and 8191 adapters")
    mean = rows / min(adapters, rows) if rows else 0
    tile = 16 if mean <= 16 else 32 if mean <= 32 else 64
    size = _lib.lib().actune_adapter_plan_size(rows, adapters, tile)
    _require(size > 0, f"too many rows for one plan: {rows}")
    buffer = torch.empty(size // 4, device=slots.device, dtype=torch.int32)
    return AdapterPlan(buffer, rows, adapters, tile).update(slots)


def adapter_add(y, x, down, up, scale, plan, *, out=None):
    """out[m] = y[m] + scale[s] * up[s] @ (down[s] @ x[m]) for the adapter s of row m
    (rows without one keep y[m]): the low-rank adapters of a batch of requests, added to
    the output y [M, N] of the projection of x [M, K] that they share.

    down [S, R, K], up [S, N, R] (1 <= R <= 128) and x, y in one dtype, float16 or
    bfloat16; scale float32 [S]; ``plan`` from ``adapter_plan``.  Rows of x, y and out
    may be strided; ``out=y`` adds in place.  Sums are kept in 32 bits from x to the one
    rounding of out."""
    _require(x.dim() == 2 and y.dim() == 2 and x.shape[0] == y.shape[0], "x and y must be [M, K] and [M, N]")
    (rows, k), n = x.shape, y.shape[1]
    _require(down.dim() == 3 and up.dim() == 3, "down must be [S, R, K] and up [S, N, R]")
    slots, rank = down.shape[0], down.shape[1]
    _require(tuple(down.shape) == (slots, rank, k) and tuple(up.shape) == (slots, n, rank),
             f"down must be [S, R, {k}] and up [S, {n}, R]")
    _require(1 <= rank <= 128, "the adapters' rank must be between 1 and 128")
    _require(x.dtype in (torch.float16, torch.bfloat16), f"unsupported dtype {x.dtype} (float16 or bfloat16 required)")
    _require(y.dtype == x.dtype and down.dtype == x.dtype and up.dtype == x.dtype, "x, y, down and up must have one dtype")
    _require(scale.dtype == torch.float32 and scale.numel() == slots, "scale must be float32 [S]")
    _require(down.is_contiguous() and up.is_contiguous() and scale.is_contiguous(), "contiguous adapters required")
    _require(plan.rows == rows and plan.adapters == slots,
             f"the plan is for {plan.rows} rows and {plan.adapters} adapters, got {rows} and {slots}")
    if out is None:
        out = torch.empty((rows, n), device=x.device, dtype=x.dtype)
    _require(tuple(out.shape) == (rows, n) and out.dtype == x.dtype, "out must match y")
    for t in (x, y, out):
        _require(t.shape[1] <= 1 or t.stride(1) == 1, "the last dimension must be contiguous")
    # A row of `out` that another row overlaps, or an `out` laid over y in another way,
    # would be written while it is read.
    _require(rows <= 1 or out.stride(0) >= n, "the rows of out must not overlap")
    device = _same_device(x, y=y, down=down, up=up, scale=scale, out=out, plan=plan.buffer)
    L = _lib.lib()
    size = L.actune_adapter_workspace_size(rows, k, slots, rank, plan.tile)
    workspace = torch.empty(size, device=device, dtype=torch.uint8)
    args = _lib.AdapterArgs(
        ctypes.sizeof(_lib.AdapterArgs), _ptr(x), _ptr(y), _ptr(down), _ptr(up), _ptr(scale), _ptr(plan.buffer),
        _ptr(out), _ptr(workspace), size, rows, n, k, slots, rank, _row_stride(x), _row_stride(y), _row_stride(out),
        plan.tile, _DTYPES[x.dtype])
    _call(L.actune_adapter_add, "adapter_add", device, args)
    return out


# ------------------------------------------------------------------------- attention
def _lengths(t, count, device, name):
    if t is not None:
        _require(t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == count and t.is_contiguous(),
                 f"{name} must be a contiguous int32 vector of {count}")
        _require(t.device == device, f"device mismatch: {name}")


def shared_prefix_attention(q, prefix_k, prefix_v, k, v, *, starts=None, prefix_lens=None, lens=None, causal=False,
                            scale=None, out=None):
    """Attention of a batch whose sequences share prefixes, each prefix's keys and values
    held (and, for few query rows, read) once for all the sequences behind it.

    q [B, T, H, D]: T query tokens of each of B sequences; prefix_k / prefix_v
    [G, P, KV, D]: G prefixes; k / v [B, S, KV, D]: the sequences' own keys and values
    (S may be 0).  Query head h reads key/value head h // (H // KV).  Sequences
    starts[g] .. starts[g + 1] - 1 share prefix g (int32 [G + 1], non-decreasing from 0
    to B; by default the B sequences are dealt evenly, sequence b to prefix b * G // B).
    The first prefix_lens[g] rows of a prefix and the first lens[b] of a sequence's own
    count (int32; all by default); what lies behind them is never used, whatever it
    holds.  Every query sees its whole prefix; with ``causal`` query t sees own key j for
    j <= lens[b] - T + t, without it all of them.  A query that sees nothing gets zeros.
    ``scale`` (positive) defaults to D ** -0.5.

    float16 or bfloat16, D <= 256 contiguous, any other strides: cache views such as
    cache[:, :, 0].unsqueeze(2) and slices of a fused projection need no copy.  With D a
    multiple of 8 and 16-byte aligned rows it runs on the tensor cores, otherwise on a
    scalar kernel many times slower.  Returns [B, T, H, D], contiguous."""
    for t in (q, prefix_k, prefix_v, k, v):
        _require(t.dim() == 4, "q, prefix_k, prefix_v, k and v must be 4-D")
    B, T, H, D = q.shape
    G, P, KV, _ = prefix_k.shape
    S = k.shape[1]
    code = _DTYPES.get(q.dtype)
    _require(code in (_lib.DTYPE_F16, _lib.DTYPE_BF16), f"unsupported dtype {q.dtype} (float16 or bfloat16 required)")
    _require(G > 0 and KV > 0 and H % KV == 0, "the query heads must be a multiple of the key/value heads")
    _require(1 <= D <= 256, "the head size must be between 1 and 256")
    _require(tuple(prefix_k.shape) == (G, P, KV, D) and prefix_v.shape == prefix_k.shape,
             f"prefix_k and prefix_v must be [G, P, KV, {D}]")
    _require(tuple(k.shape) == (B, S, KV, D) and v.shape == k.shape, f"k and v must be [{B}, S, {KV}, {D}]")
    for t in (prefix_k, prefix_v, k, v):
        _require(t.dtype == q.dtype, "q, keys and values must have one dtype")
    for t in (q, prefix_k, prefix_v, k, v):
        _require(D == 1 or t.stride(3) == 1, "the last dimension must be contiguous")
    device = _same_device(q, prefix_k=prefix_k, prefix_v=prefix_v, k=k, v=v, out=out)
    _lengths(starts, G + 1, device, "starts")
    _lengths(prefix_lens, G, device, "prefix_lens")
    _lengths(lens, B, device, "lens")
    scale = D ** -0.5 if scale is None else float(scale)
    _require(0.0 < scale < 3e38, "scale must be positive and finite")
    if out is None:
        out = torch.empty((B, T, H, D), device=device, dtype=q.dtype)
    _require(out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous(),
             "out must be contiguous and match q")
    L = _lib.lib()
    size = L.actune_prefix_attention_workspace_size(B, T, H, KV, D, G, P, S)
    workspace = torch.empty(size, device=device, dtype=torch.uint8) if size else None
    args = _lib.PrefixAttentionArgs(
        ctypes.sizeof(_lib.PrefixAttentionArgs), _ptr(q), _ptr(prefix_k), _ptr(prefix_v), _ptr(k), _ptr(v),
        _ptr(starts), _ptr(prefix_lens), _ptr(lens), _ptr(out), _ptr(workspace), size, B, T, H, KV, D, G, P, S,
        *q.stride()[:3], *prefix_k.stride()[:3], *prefix_v.stride()[:3], *k.stride()[:3], *v.stride()[:3], scale, code,
        bool(causal))
    _call(L.actune_prefix_attention, "shared_prefix_attention", device, args)
    return out
