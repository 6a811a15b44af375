"""Tensor-level calls of the serving operators (include/actune_b200_serving.h),
re-exported by ``actune_b200.ops``.

* ``shared_prefix_attention``: attention of a batch whose sequences share prefixes.
* ``adapter_plan`` / ``adapter_add``: low-rank adapters of many requests added to the
  output of the projection they share.
* ``gated_norm``: norm after a block, gate, residual scale and the norm before the
  next block in one launch, optionally with the group-64 activations of the result.

Conventions of ``ops``: tensors on one CUDA device, that device's current stream,
RuntimeError for operands that do not fit, outputs and scratch from torch's allocator
(so they belong to the stream the call runs on).  Nothing here synchronises, and nothing
has a backward: outputs carry no gradient, and an ``out`` that requires one is refused
(RuntimeError) while gradients are enabled.  The checks
and the C-ABI call are in the compiled module ``_serving`` (csrc/torch/serving.cpp).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.utils import _pytree as pytree

from . import _lib

_MODULE = None


def _serving():
    """The compiled module; raises if it was not built."""
    global _MODULE
    if _MODULE is None:
        _lib.lib()  # loads (or names) the library the module links
        try:
            from . import _serving as module
        except ImportError as e:
            raise RuntimeError(f"actune_b200/_serving.so cannot be loaded ({e}); run `python -m actune_b200.build` "
                               "(the serving operators have no fallback implementation)") from e
        _MODULE = module
    return _MODULE


def _checked(result, what):
    if type(result) is int:
        _lib.check(result, what)
    return result


# ------------------------------------------------------------------------- gated norm
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
    return _checked(_serving().gated_norm(x, residual, pre_weight, post_weight, gate, shift, residual_scale, eps, gemma,
                                          quant_bits, codes8), "gated_norm")


# ------------------------------------------------------------------------- adapters
@dataclass(frozen=True)
class AdapterPlan:
    """The rows of a batch sorted by adapter slot (made by ``adapter_plan``; read by
    every ``adapter_add`` the batch passes through).  ``update`` routes the same number
    of rows anew into the same buffer, so a captured graph that reads it follows; the plan
    has to live as long as such a graph."""

    buffer: torch.Tensor
    rows: int
    adapters: int
    tile: int

    def update(self, slots):
        _check_slots(slots)
        if slots.device != self.buffer.device:
            raise RuntimeError(f"device mismatch: slots is on {slots.device}")
        if slots.shape[0] != self.rows:
            raise RuntimeError(f"the plan was made for {self.rows} rows, got {slots.shape[0]}")
        with torch.cuda.device(slots.device):
            _lib.check(_lib.lib().actune_adapter_plan(slots.data_ptr(), self.rows, self.adapters, self.tile,
                                                      self.buffer.data_ptr(),
                                                      torch.cuda.current_stream(slots.device).cuda_stream),
                       "adapter_plan")
        return self


# Among the arguments of a GraphReplay call a plan is its buffer, copied like any tensor,
# and its sizes, which are part of the call's identity.
pytree.register_pytree_node(AdapterPlan, lambda p: ([p.buffer], (p.rows, p.adapters, p.tile)),
                            lambda leaves, sizes: AdapterPlan(*leaves, *sizes),
                            serialized_type_name="actune_b200.AdapterPlan")


def _check_slots(slots):
    if slots.dim() != 1 or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise RuntimeError("slots must be a contiguous int32 vector")
    if not slots.is_cuda:
        raise RuntimeError("CUDA required")


def adapter_plan(slots, adapters):
    """Sort a batch's rows by adapter: slots int32 [M] on the GPU (row m runs adapter
    slots[m]; anything outside 0 .. adapters - 1 means none) -> AdapterPlan.

    Tiles of rows that share an adapter have 4, 16 or 128 rows, by the mean number of
    rows per adapter that the sizes allow; a row's result depends on its own operands and
    these sizes, not on the rows beside it."""
    _check_slots(slots)
    rows = slots.shape[0]
    if not 1 <= adapters <= 8191:
        raise RuntimeError("between 1 and 8191 adapters")
    mean = rows / min(adapters, rows) if rows else 0
    # The plan serves projections of every width, so its tiles are chosen by rows alone
    # (operands from memory, rank 16 where not said).  4 against 16 rows: 32 adapters of 1
    # row, 4096 -> 22016, 15.4 and 22.0 us; of 3 rows, 1024 -> 2560, 7.5 and 7.3 us.  16
    # against 128: 16 adapters of 20 rows, 4096 -> 12288, 18.4 and 21.4 us; of 40 rows, 2048
    # -> 32768 at rank 64, 92 and 55 us; of 50 rows, 1024 -> 2560, 11.4 and 10.7 us.
    tile = 4 if mean <= 2 else 16 if mean <= 32 else 128
    size = _lib.lib().actune_adapter_plan_size(rows, adapters, tile)
    if size == 0:
        raise RuntimeError(f"too many rows for one plan: {rows}")
    buffer = torch.empty(size // 4, device=slots.device, dtype=torch.int32)
    return AdapterPlan(buffer, rows, adapters, tile).update(slots)


def adapter_add(y, x, down, up, scale, plan, *, out=None):
    """out[m] = y[m] + scale[s] * up[s] @ (down[s] @ x[m]) for the adapter s of row m
    (rows without one keep y[m]): the low-rank adapters of a batch of requests, added to
    the output y [M, N] of the projection of x [M, K] that they share.

    down [S, R, K], up [S, N, R] (1 <= R <= 128) and x, y in one dtype, float16 or
    bfloat16; scale float32 [S]; ``plan`` from ``adapter_plan``.  Rows of x, y and out
    may be strided; ``out=y`` adds in place, and ``out`` overlaps no other operand.  Both
    products are summed in 32 bits and out is rounded once; between them ``down x`` is held
    in 32 bits in tiles of 4 rows, and in two 16-bit parts (16 bits of significand in
    bfloat16, 22 in float16) where matrix instructions take it."""
    return _checked(_serving().adapter_add(y, x, down, up, scale, plan.buffer, plan.rows, plan.adapters, plan.tile,
                                           out), "adapter_add")


# ------------------------------------------------------------------------- attention
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

    Scores, softmax and sums are held in 32 bits; the probabilities are rounded to the
    operands' type for their product with the values, which adds about as much error as the
    rounding of the output (the scalar kernel keeps them in 32 bits).  A value that is not
    finite may reach queries of its own sequence that ``causal`` keeps from it, and reaches
    no other sequence.

    float16 or bfloat16, D <= 256 contiguous, any other strides: cache views such as
    cache[:, :, 0].unsqueeze(2) and slices of a fused projection need no copy.  With D a
    multiple of 8 and 16-byte aligned rows it runs on the tensor cores, otherwise on a
    scalar kernel many times slower (4 x 50 tokens, 8 heads of 64: 11 and 123 us).  Returns
    [B, T, H, D], contiguous; ``out`` gives the room for it and overlaps no input."""
    return _checked(_serving().shared_prefix_attention(q, prefix_k, prefix_v, k, v, starts, prefix_lens, lens, causal,
                                                       scale, out), "shared_prefix_attention")
