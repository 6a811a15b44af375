"""Adapter slots and scopes on the CPU: installing, loading, refusals, pass-through."""
import types

import pytest
import torch

from actune_b200 import ops
from actune_b200.adapters import AdaptedLinear, active_adapter_plan, adapter_scope, install_adapters
from actune_b200.graph import GraphReplay, _Capture


def model():
    m = torch.nn.Module()
    m.block = torch.nn.Module()
    m.block.up = torch.nn.Linear(12, 20, dtype=torch.bfloat16)
    m.block.down = torch.nn.Linear(20, 12, bias=False, dtype=torch.bfloat16)
    return m


def test_install_wraps_the_named_projections_and_passes_through_without_a_scope():
    m = model()
    before = m.block.up
    x = torch.randn(3, 12).bfloat16()
    want = before(x)
    adapted = install_adapters(m, ["block.up", "block.down"], slots=4, rank=6)
    assert m.block.up is adapted["block.up"] and m.block.up.projection is before
    assert torch.equal(m.block.up(x), want)
    assert m.block.up.in_features == 12 and m.block.up.out_features == 20 and m.block.up.weight is before.weight
    # the rank is held in whole 16-byte rows
    assert m.block.up.down.shape == (4, 8, 12) and m.block.up.up.shape == (4, 20, 8)
    assert m.block.up.padding == 0 and m.block.up.input_scale is None and not hasattr(m.block.up, "active_backend")


def test_install_checks_everything_before_touching_the_model():
    m = model()
    m.block.act = torch.nn.ReLU()
    with pytest.raises(ValueError, match="block.act"):
        install_adapters(m, ["block.up", "block.act"], 4, 8)
    assert isinstance(m.block.up, torch.nn.Linear)
    install_adapters(m, ["block.up"], 4, 8)
    with pytest.raises(ValueError, match="block.up"):
        install_adapters(m, ["block.up"], 4, 8)
    for slots, rank in ((0, 8), (9000, 8), (4, 0), (4, 129)):
        with pytest.raises(ValueError, match="slots"):
            install_adapters(m, ["block.down"], slots, rank)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        install_adapters(m, ["block.down"], 4, 8, dtype=torch.float32)


def test_load_and_clear_a_slot():
    a = AdaptedLinear(torch.nn.Linear(12, 20), slots=2, rank=6)
    down, up = torch.randn(4, 12), torch.randn(20, 4)
    a.load(1, torch.ones(6, 12), torch.ones(20, 6), 3.0)
    a.load(1, down, up, 0.5)  # replaces all of the earlier one
    assert torch.equal(a.down[1, :4], down.bfloat16()) and not a.down[1, 4:].any()
    assert torch.equal(a.up[1, :, :4], up.bfloat16()) and not a.up[1, :, 4:].any()
    assert a.scale.tolist() == [0.0, 0.5] and not a.down[0].any()
    a.clear(1)
    assert not a.down.any() and not a.up.any() and not a.scale.any()
    for slot, d, u in ((2, down, up), (-1, down, up), (0, torch.zeros(7, 12), torch.zeros(20, 7)),
                       (0, down[:, :11], up), (0, down, up[:19]), (0, down[:0], up[:, :0])):
        with pytest.raises(ValueError):
            a.load(slot, d, u)


def test_scope_is_nested_and_restored():
    plan, other = object(), object()
    assert active_adapter_plan() is None
    with adapter_scope(plan):
        with adapter_scope(other):
            assert active_adapter_plan() is other
        with adapter_scope(None):
            assert active_adapter_plan() is None
        assert active_adapter_plan() is plan
    assert active_adapter_plan() is None


def test_a_bank_projection_keeps_its_format():
    class Resident(torch.nn.Linear):
        padding, input_scale = 4, None

        def active_backend(self):
            return "backend"

    a = AdaptedLinear(Resident(12, 20), slots=1, rank=8)
    assert a.padding == 4 and hasattr(a, "active_backend") and a.active_backend() == "backend"


def plan_of(slots, adapters=4, tile=16):
    """A plan as far as a host test needs one: its buffer holds the slots."""
    return ops.AdapterPlan(torch.tensor(slots, dtype=torch.int32), len(slots), adapters, tile)


class HostReplay(GraphReplay):
    """Captures as a CUDA graph does, on the host: what was active while recording is
    what every replay reads, by the buffer it had then."""

    def _record(self, slot, tree):
        plan = active_adapter_plan()
        output = []
        graph = types.SimpleNamespace(
            plan=plan, replay=lambda: output.__setitem__(slice(None), [None if plan is None else plan.buffer.tolist()]))
        return _Capture(graph, output, {})


def test_graph_key_holds_the_sizes_of_the_active_plan():
    replay = GraphReplay(lambda x: x, {})
    leaves, tree = torch.utils._pytree.tree_flatten(((torch.zeros(2, 3),), {}))
    keys = [replay.key(leaves, tree)]
    for plan in (plan_of([0, 1]), plan_of([0, 1, 2]), plan_of([0, 1], adapters=5), plan_of([0, 1], tile=4)):
        with adapter_scope(plan):
            keys.append(replay.key(leaves, tree))
            with adapter_scope(None):
                assert replay.key(leaves, tree) == keys[0]
    assert len(set(keys)) == 5
    with adapter_scope(plan_of([1, 0])):  # another routing of the same sizes replays the same graph
        assert replay.key(leaves, tree) == keys[1]


@pytest.mark.parametrize("first", ["scope", "none"])
def test_a_replay_runs_the_active_plan_and_none_outside_a_scope(first):
    replay = HostReplay(lambda x: x, {})
    replay.enabled = True
    x = torch.zeros(2, 3)
    a, b = plan_of([0, 1]), plan_of([3, -1])
    if first == "none":
        assert replay(x) == [None]
    for plan in (a, b, a):
        with adapter_scope(plan):
            assert replay(x) == [plan.buffer.tolist()]
            with adapter_scope(None):
                assert replay(x) == [None]
        assert replay(x) == [None]
    a.buffer.copy_(torch.tensor([2, 2]))  # as AdapterPlan.update does
    with adapter_scope(a):
        assert replay(x) == [[2, 2]]
    assert len(replay.graphs) == 2 and replay.fallbacks == 0


def test_a_capture_reads_a_plan_of_its_own():
    """Whatever becomes of the plan it was captured under."""
    replay = HostReplay(lambda x: x, {})
    replay.enabled = True
    plan = plan_of([0, 1])
    with adapter_scope(plan):
        replay(torch.zeros(2, 3))
    (capture,) = replay.graphs.values()
    assert capture.graph.plan.buffer.data_ptr() != plan.buffer.data_ptr()


def test_adapters_are_refused_where_a_gradient_would_pass_them_by():
    """They are added behind autograd's back, whose gradient would lack their term."""
    layer = AdaptedLinear(torch.nn.Linear(12, 20, dtype=torch.bfloat16), slots=4, rank=8)
    x = torch.zeros(2, 12).bfloat16()
    with adapter_scope(ops.AdapterPlan(torch.zeros(64, dtype=torch.int32), 2, 4, 16)):
        with pytest.raises(RuntimeError, match="no backward"):
            layer(x)  # the projection's weight requires a gradient
        for context in (torch.no_grad, torch.inference_mode):
            with context(), pytest.raises(RuntimeError, match="CUDA required"):
                layer(x)
        with adapter_scope(None):
            assert layer(x).requires_grad
        layer.requires_grad_(False)
        with pytest.raises(RuntimeError, match="no backward"):
            layer(x.clone().requires_grad_())
        with pytest.raises(RuntimeError, match="CUDA required"):
            layer(x)


def test_a_plan_among_the_arguments_is_an_input_too():
    class ArgumentReplay(GraphReplay):
        def _record(self, slot, tree):
            (_, plan), _ = torch.utils._pytree.tree_unflatten(slot.statics, tree)
            output = []
            graph = types.SimpleNamespace(replay=lambda: output.__setitem__(slice(None), plan.buffer.tolist()))
            return _Capture(graph, output, {})

    replay = ArgumentReplay(lambda x, plan: x, {})
    replay.enabled = True
    x, slots = torch.zeros(2, 3), list(range(2000))  # longer than a tensor's repr shows
    for first in (0, 5, 7):
        slots[1000] = first
        assert replay(x, plan_of(slots)) == slots
    assert len(replay.graphs) == 1
    replay(x, plan_of(slots, tile=128))
    assert len(replay.graphs) == 2
