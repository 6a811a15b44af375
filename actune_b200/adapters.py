"""Low-rank adapters of many requests beside the resident projections they share.

A served batch mixes requests that were fine-tuned apart: the packed (or any other)
projection is one for all of them, and each request adds its own adapter,
y = W x + scale * up (down x).  ``install_adapters`` gives projections of a model a set of
adapter slots, ``AdaptedLinear.load`` fills a slot, and ``adapter_scope(plan)`` says which
row of the batch runs which slot, the way ``precision_profile`` says which precision it
runs in:

    adapters = install_adapters(model, names, slots=16, rank=16)
    adapters["layers.0.qkv_proj"].load(3, down, up, scale=0.5)
    plan = ops.adapter_plan(slots_of_rows, 16)      # int32 [rows] on the GPU; -1: none
    with adapter_scope(plan):
        model(x)

Outside a scope the projections run alone.  ``GraphReplay`` takes the active plan (and
one among its arguments) as an input: calls under plans of the same sizes replay one
graph, each with its own routing, and a call outside a scope replays another.  A CUDA
graph captured by other means reads the buffer of the plan it was captured under: keep
that plan as long as the graph; ``plan.update(slots)`` before a replay routes the same
number of rows anew.
"""
from __future__ import annotations

from contextlib import contextmanager
from contextvars import ContextVar

import torch

from . import ops

_ACTIVE = ContextVar("actune_adapter_plan", default=None)


def active_adapter_plan():
    return _ACTIVE.get()


@contextmanager
def adapter_scope(plan):
    """Run the adapters of the enclosed calls' rows as ``plan`` (an ``ops.AdapterPlan``, or
    None for no adapters) says, in the current thread / async task."""
    token = _ACTIVE.set(plan)
    try:
        yield
    finally:
        _ACTIVE.reset(token)


class AdaptedLinear(torch.nn.Module):
    """A projection with ``slots`` adapters of up to ``rank``; empty slots add zero.

    ``projection`` is any module from [..., in_features] to [..., out_features] (a bank's
    ResidentLinear, an nn.Linear) whose output nobody else holds: the adapters are added
    to it in place.  They have no backward: in a scope, an output that requires a gradient
    is refused (RuntimeError), so such a projection is run under ``torch.no_grad()``."""

    def __init__(self, projection, slots, rank, dtype=torch.bfloat16, device=None):
        super().__init__()
        if not 1 <= slots <= 8191 or not 1 <= rank <= 128:
            raise ValueError("between 1 and 8191 slots of rank 1 to 128")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("adapters are float16 or bfloat16")
        device = projection.weight.device if device is None else device
        # Rows of `up` a multiple of 16 bytes: what the tensor-core form reads.
        held = (rank + 7) // 8 * 8
        self.projection = projection
        self.in_features, self.out_features, self.slots, self.rank = (projection.in_features, projection.out_features,
                                                                      slots, rank)
        self.register_buffer("down", torch.zeros(slots, held, self.in_features, device=device, dtype=dtype))
        self.register_buffer("up", torch.zeros(slots, self.out_features, held, device=device, dtype=dtype))
        self.register_buffer("scale", torch.zeros(slots, device=device, dtype=torch.float32))

    @torch.no_grad()
    def load(self, slot, down, up, scale=1.0):
        """Fill a slot with down [r, in_features], up [out_features, r], r <= rank."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        r = down.shape[0]
        if not 1 <= r <= self.rank or tuple(down.shape) != (r, self.in_features) or tuple(up.shape) != (
                self.out_features, r):
            raise ValueError(f"an adapter here is [r, {self.in_features}] and [{self.out_features}, r], r <= {self.rank}")
        self.clear(slot)
        self.down[slot, :r].copy_(down)
        self.up[slot, :, :r].copy_(up)
        self.scale[slot] = float(scale)

    @torch.no_grad()
    def clear(self, slot):
        self.down[slot].zero_()
        self.up[slot].zero_()
        self.scale[slot] = 0.0

    # What the model's glue asks a resident projection (harness.input_format).
    @property
    def padding(self):
        return getattr(self.projection, "padding", 0)

    @property
    def input_scale(self):
        return getattr(self.projection, "input_scale", None)

    @property
    def weight(self):
        return self.projection.weight

    def __getattr__(self, name):
        if name == "active_backend":  # only where the projection has precisions
            return getattr(super().__getattr__("projection"), name)
        return super().__getattr__(name)

    def forward(self, x):
        y = self.projection(x)
        plan = _ACTIVE.get()
        if plan is None:
            return y
        flat = y.reshape(-1, self.out_features)
        ops.adapter_add(flat, x.reshape(-1, self.in_features), self.down, self.up, self.scale, plan, out=flat)
        return flat.view(y.shape)


def install_adapters(model, names, slots, rank, dtype=torch.bfloat16):
    """Wrap the named projections of ``model`` in AdaptedLinear; {name: AdaptedLinear}.
    Everything is checked before the model is touched."""
    projections = {name: model.get_submodule(name) for name in names}
    for name, module in projections.items():
        if isinstance(module, AdaptedLinear) or not hasattr(module, "in_features") or not hasattr(module, "out_features"):
            raise ValueError(f"not a projection that adapters can be added to: {name}")
    adapted = {name: AdaptedLinear(module, slots, rank, dtype) for name, module in projections.items()}
    for name, module in adapted.items():
        parent, _, child = name.rpartition(".")
        setattr(model.get_submodule(parent), child, module)
    return adapted
