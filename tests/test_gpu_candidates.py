"""The serving operators together: action candidates behind shared prefixes, with adapters
per environment (actune_b200.candidates, small shapes).

One denoise step is compared with the same model whose three operators are replaced by
plain torch in 64 bits.  Both run the packed projections on 8-bit activations of bf16
values: where the two streams differ by a bf16 unit a code may step, so the outputs agree
to bf16 precision through the layers (2^-8 per rounded intermediate, about ten of them a
layer, adding in quadrature over two layers: 2^-8 * sqrt(20) < 2%).
"""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPE = dict(layers=2, hidden=256, heads=4, head_dim=64, mlp=512, prefix_tokens=24, horizon=6, action_dim=8,
             state_dim=5, steps=3, adapter_slots=4, rank=8)


def plain_attention(q, pk, pv, k, v):
    B, H, rep = q.shape[0], q.shape[2], q.shape[2] // pk.shape[2]
    of = torch.arange(B, device=q.device) * pk.shape[0] // B
    keys = torch.cat([pk[of], k], 1).double().repeat_interleave(rep, 2)
    values = torch.cat([pv[of], v], 1).double().repeat_interleave(rep, 2)
    s = torch.einsum("bthd,bnhd->bhtn", q.double(), keys) * q.shape[3] ** -0.5
    return torch.einsum("bhtn,bnhd->bthd", s.softmax(-1), values).to(q.dtype).contiguous()


def plain_norm(x, residual, pre, *, post_weight=None, gate=None, shift=None, gemma=False, quant_bits=None,
               codes8=False):
    from actune_b200 import ops
    rows = x.shape[0]

    def wide(t):
        return t.double() if t.dim() == 1 else t.double().repeat_interleave(rows // t.shape[0], 0)

    def norm(a, w):
        return a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + wide(w))

    u = x.double() if post_weight is None else norm(x.double(), post_weight)
    s = residual.double() + (u if gate is None else u * wide(gate))
    h = norm(s, pre) + (0 if shift is None else wide(shift))
    h, s = h.to(x.dtype), s.to(x.dtype)
    return (h, s, *ops.quantize_group64(h, quant_bits, codes8=codes8)) if quant_bits else (h, s)


def plain_adapter(slots):
    def add(y, x, down, up, scale, plan, out=None):
        delta = torch.zeros(y.shape, dtype=torch.float64, device=y.device)
        for s in range(down.shape[0]):
            rows = (slots == s).nonzero()[:, 0]
            delta[rows] = float(scale[s]) * (x[rows].double() @ down[s].double().T @ up[s].double().T)
        out.copy_((y.double() + delta).to(y.dtype))
        return out
    return add


@pytest.fixture(scope="module")
def policy():
    from actune_b200.candidates import CandidatePolicy
    p = CandidatePolicy(envs=3, candidates=2, seed=5, **SHAPE)
    g = torch.Generator(device="cuda").manual_seed(6)
    for module in p.adapters.values():
        for slot in range(3):  # the last slot stays empty
            r = 8 if slot else 5
            module.load(slot, torch.randn(r, module.in_features, device="cuda", generator=g) * 0.1,
                        torch.randn(module.out_features, r, device="cuda", generator=g) * 0.1, scale=0.5)
    yield p
    p.release()


def inputs(envs=3, candidates=2, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(envs, candidates, 6, 8, device="cuda", generator=g),
            torch.randn(envs, 5, device="cuda", generator=g),
            torch.randn(2, envs, 30, 2, 64, device="cuda", generator=g).bfloat16())


def route(p, *slots):
    p.route(torch.tensor(slots, dtype=torch.int32, device="cuda"))


def near(a, b, rel=0.02):
    assert float((a - b).norm() / b.norm()) < rel


def test_step_matches_plain_operators(policy, monkeypatch):
    from actune_b200 import adapters, candidates
    from actune_b200.adapters import adapter_scope
    noise, state, prefix = inputs()
    route(policy, 1, -1, 0)
    one = torch.ones((), device="cuda")
    with torch.inference_mode(), adapter_scope(policy.plan):
        got, _ = policy.denoise_step(noise, one, -one, state, prefix)
        rows = torch.tensor([1, -1, 0], device="cuda").repeat_interleave(12)
        monkeypatch.setattr(candidates, "ops", types.SimpleNamespace(shared_prefix_attention=plain_attention,
                                                                     gated_norm=plain_norm))
        monkeypatch.setattr(adapters, "ops", types.SimpleNamespace(adapter_add=plain_adapter(rows)))
        want, _ = policy.denoise_step(noise, one, -one, state, prefix)
    near(got - noise, want - noise)


def test_adapters_change_their_own_environment_only(policy):
    noise, state, prefix = inputs(seed=2)
    route(policy, -1, -1, -1)
    none = policy.sample(noise, state, prefix)
    route(policy, 3, 3, 3)  # an empty slot adds zero
    assert torch.equal(policy.sample(noise, state, prefix), none)
    route(policy, -1, 2, -1)
    some = policy.sample(noise, state, prefix)
    assert torch.equal(some[0], none[0]) and torch.equal(some[2], none[2])
    assert float((some[1] - none[1]).norm() / none[1].norm()) > 1e-3


def test_graph_replays_follow_the_routing(policy):
    noise, state, prefix = inputs(seed=3)
    for slots in ((0, 1, 2), (2, -1, 0), (1, 1, 1)):
        route(policy, *slots)
        eager = policy.sample(noise, state, prefix)
        assert torch.equal(policy.sample(noise, state, prefix, graph=True), eager)
    assert policy.step_graph.replays > 0 and policy.step_graph.fallbacks == 0


def test_candidates_are_those_drawn_alone(policy):
    from actune_b200.candidates import CandidatePolicy
    alone = CandidatePolicy(envs=3, candidates=1, seed=5, **SHAPE)
    with torch.no_grad():
        for name, module in policy.adapters.items():
            for buffer in ("down", "up", "scale"):
                getattr(alone.adapters[name], buffer).copy_(getattr(module, buffer))
    noise, state, prefix = inputs(seed=4)
    route(policy, 2, 0, -1)
    route(alone, 2, 0, -1)
    both = policy.sample(noise, state, prefix)
    for c in range(2):
        near(alone.sample(noise[:, c:c + 1].contiguous(), state, prefix)[:, 0] - noise[:, c], both[:, c] - noise[:, c])
    alone.release()


def test_bank_audit_sees_the_adapted_projections(policy):
    policy.runtime.before()
    noise, state, prefix = inputs(seed=5)
    policy.sample(noise, state, prefix)
    policy.runtime.audit("q11")
    assert all(m.calls == SHAPE["steps"] for m in policy.runtime.modules.values())
