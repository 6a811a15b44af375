"""Several action candidates per observation, from requests with adapters of their own.

The serving operators together, as a policy runs them.  A prefix pass (the VLM of
``harness.Pi05Backbone``) leaves each environment's keys and values; the action expert
then draws ``candidates`` chunks per environment from different noise:

* the candidates of an environment are sequences that share its prefix
  (``ops.shared_prefix_attention``: the cache holds it once, not once per candidate);
* every projection is a bank's packed projection plus the low-rank adapter of the
  environment's fine-tune (``adapters.AdaptedLinear``);
* blocks are joined by a norm after the block, a gate and shift per environment from the
  flow time and the state, and the norm before the next block, which also writes the next
  projection's group-64 activations (``ops.gated_norm``).

    python -m actune_b200.candidates [--envs 16] [--candidates 8]
"""
from __future__ import annotations

import argparse

import torch
import torch.nn.functional as F

from . import ops
from .adapters import adapter_scope, install_adapters
from .graph import GraphReplay
from .harness import build_bank, gated_act, input_format, projection_names, rope_cache_, rope_tables
from .kernels.grouped import share_quantized, shared_activation_scope
from .layers import install_bank


class CandidateLayer(torch.nn.Module):
    """Decoder layer between two normed streams: (h, residual) -> (h', residual'), where h'
    is normed for the layer that follows (``next_norm``)."""

    def __init__(self, hidden, heads, head_dim, mlp, device, dtype):
        super().__init__()
        self.heads, self.head_dim = heads, head_dim
        kw = dict(device=device, dtype=dtype)
        for name in ("input_norm", "attn_post_norm", "mlp_norm", "mlp_post_norm"):
            setattr(self, name, torch.nn.Parameter(torch.zeros(hidden, **kw)))
        self.qkv_proj = torch.nn.Linear(hidden, (heads + 2) * head_dim, bias=False, **kw)
        self.o_proj = torch.nn.Linear(heads * head_dim, hidden, bias=False, **kw)
        self.gate_up_proj = torch.nn.Linear(hidden, 2 * mlp, bias=False, **kw)
        self.down_proj = torch.nn.Linear(mlp, hidden, bias=False, **kw)

    def forward(self, h, residual, gates, next_norm, next_format, prefix, own, cos, sin):
        """h, residual: [B * T, hidden]; gates: (attention gate, MLP gate, shift), each
        [envs, hidden]; prefix: [envs, P, 2, head_dim] of this layer; own: [B, T, 2,
        head_dim], overwritten with this call's keys and values."""
        rows, (B, T), H, dh = h.shape[0], own.shape[:2], self.heads, self.head_dim
        qkv = self.qkv_proj(h)
        rope_cache_(qkv, cos, sin, H, dh, own, T, 0)
        attn = ops.shared_prefix_attention(qkv[:, :H * dh].view(B, T, H, dh), prefix[:, :, 0].unsqueeze(2),
                                           prefix[:, :, 1].unsqueeze(2), own[:, :, 0].unsqueeze(2),
                                           own[:, :, 1].unsqueeze(2))
        x = self.o_proj(attn.view(rows, H * dh))
        attn_gate, mlp_gate, shift = gates
        h, residual = join(x, residual, self.mlp_norm, self.attn_post_norm, attn_gate, None,
                           **input_format(self.gate_up_proj, rows))
        x = self.down_proj(gated_act(self.gate_up_proj(h), gelu=True, **input_format(self.down_proj, rows)))
        return join(x, residual, next_norm, self.mlp_post_norm, mlp_gate, shift, **next_format)


def join(x, residual, pre_weight, post_weight, gate, shift, quant_bits=None, codes8=False):
    """gated_norm between two blocks; activations it quantizes are offered to the active
    shared activation scope, so the next projection does not launch its own quantizer."""
    if not quant_bits or x.shape[1] % 64:
        return ops.gated_norm(x, residual, pre_weight, post_weight=post_weight, gate=gate, shift=shift, gemma=True)
    h, residual, packed, scales = ops.gated_norm(x, residual, pre_weight, post_weight=post_weight, gate=gate,
                                                 shift=shift, gemma=True, quant_bits=quant_bits, codes8=codes8)
    share_quantized(h, quant_bits, packed, scales, codes8)
    return h, residual


class CandidatePolicy(torch.nn.Module):
    """An action expert with the cache layout of ``harness.Pi05Backbone`` (one key/value
    head, [layers, envs, positions, 2, head_dim]) that draws several chunks per prefix."""

    def __init__(self, layers=18, hidden=1024, heads=8, head_dim=256, mlp=4096, prefix_tokens=304, horizon=50,
                 action_dim=32, state_dim=14, steps=10, envs=16, candidates=8, adapter_slots=16, rank=16, mode="w4a8",
                 alternate="w2a8", device="cuda", dtype=torch.bfloat16, seed=0):
        super().__init__()
        g = torch.Generator(device=device).manual_seed(seed)
        kw = dict(device=device, dtype=dtype)
        self.prefix_tokens, self.horizon, self.action_dim, self.steps = prefix_tokens, horizon, action_dim, steps
        self.envs, self.candidates = envs, candidates
        self.expert = torch.nn.ModuleList([CandidateLayer(hidden, heads, head_dim, mlp, device, dtype)
                                           for _ in range(layers)])
        self.action_in = torch.nn.Linear(action_dim, hidden, **kw)
        self.time_in = torch.nn.Linear(hidden, hidden, **kw)
        self.state_in = torch.nn.Linear(state_dim, hidden, **kw)
        self.modulate = torch.nn.Linear(hidden, 3 * hidden, **kw)
        self.action_out = torch.nn.Linear(hidden, action_dim, **kw)
        self.final_norm = torch.nn.Parameter(torch.zeros(hidden, **kw))
        with torch.no_grad():
            for p in self.parameters():
                if p.dim() == 2:
                    p.normal_(0.0, 0.02, generator=g)
                else:  # biases and (1 + w) norm weights
                    p.zero_()
        cos, sin = rope_tables(prefix_tokens + horizon, head_dim, 10000.0, device)
        B = envs * candidates
        self.register_buffer("rope_cos", cos[prefix_tokens:].repeat(B, 1).contiguous())
        self.register_buffer("rope_sin", sin[prefix_tokens:].repeat(B, 1).contiguous())
        half = hidden // 2
        self.register_buffer("time_freqs", torch.exp(-torch.arange(half, device=device) * (9.210340371976184 / half)))
        # One layer's own keys and values at a time.
        self.register_buffer("own_cache", torch.zeros(B, horizon, 2, head_dim, **kw))
        bank, clips = build_bank(self, {"expert": B * horizon * steps}, mode, alternate,
                                 ("expert.0.down_proj", f"expert.{layers - 1}.down_proj"), stacks=("expert",))
        self.runtime = install_bank(self, bank, clips)
        self.runtime.decode_weights()
        self.adapters = install_adapters(self, projection_names(self, ("expert",)), adapter_slots, rank, dtype)
        # Rows of one environment are consecutive: candidate, then action token.
        self.rows_of_env = candidates * horizon
        self.plan = ops.adapter_plan(torch.full((envs * self.rows_of_env,), -1, device=device, dtype=torch.int32),
                                     adapter_slots)
        self.step_graph = GraphReplay(self.denoise_step, self.runtime.modules, shared_a8=True)

    def route(self, slots):
        """Environment e runs adapter slots[e] (int32 [envs]; -1: none) from the next call on."""
        self.plan.update(slots.repeat_interleave(self.rows_of_env))

    def denoise_step(self, x_t, time, dt, state, prefix_cache):
        """One Euler step for x_t [envs, candidates, horizon, action_dim] (fp32) given state
        [envs, state_dim] and prefix_cache [layers, envs, >= prefix_tokens, 2, head_dim]."""
        dtype = self.action_in.weight.dtype
        ang = time * self.time_freqs
        temb = torch.cat([ang.sin(), ang.cos()]).to(dtype)
        cond = F.silu(self.time_in(temb)[None] + self.state_in(state.to(dtype)))
        gates = [t.contiguous() for t in self.modulate(cond).chunk(3, dim=-1)]
        gates[0], gates[1] = 1 + gates[0], 1 + gates[1]
        x = self.action_in(x_t.reshape(-1, self.action_dim).to(dtype))
        rows = x.shape[0]
        formats = [input_format(layer.qkv_proj, rows) for layer in self.expert] + [{}]
        norms = [layer.input_norm for layer in self.expert] + [self.final_norm]
        # The first layer's input: no block before it, so the stream is x itself.
        h, residual = join(torch.zeros_like(x), x, norms[0], None, None, gates[2], **formats[0])
        for i, layer in enumerate(self.expert):
            h, residual = layer(h, residual, gates, norms[i + 1], formats[i + 1], prefix_cache[i, :, :self.prefix_tokens],
                                self.own_cache, self.rope_cos, self.rope_sin)
        v_t = self.action_out(h).float().view(x_t.shape)
        return x_t + dt * v_t, time + dt

    def sample(self, noise, state, prefix_cache, graph=False):
        """Action candidates [envs, candidates, horizon, action_dim] from noise of that
        shape.  ``graph``: replay a captured step (adapters may be routed anew between
        calls: the plan is an input of the graph)."""
        dt = torch.full((), -1.0 / self.steps, dtype=torch.float32, device=noise.device)
        time = torch.full((), 1.0, dtype=torch.float32, device=noise.device)
        self.step_graph.enabled = graph
        x_t = noise
        with torch.inference_mode(), adapter_scope(self.plan), shared_activation_scope(not graph):
            for _ in range(self.steps):
                x_t, time = self.step_graph(x_t, time, dt, state, prefix_cache)
        return x_t

    def release(self):
        self.step_graph.release()


def main():
    ap = argparse.ArgumentParser(description="Draw action candidates for a batch of environments with adapters.")
    ap.add_argument("--envs", type=int, default=16)
    ap.add_argument("--candidates", type=int, default=8)
    ap.add_argument("--layers", type=int, default=18)
    ap.add_argument("--calls", type=int, default=5)
    a = ap.parse_args()
    policy = CandidatePolicy(layers=a.layers, envs=a.envs, candidates=a.candidates)
    g = torch.Generator(device="cuda").manual_seed(1)
    for module in policy.adapters.values():
        for slot in range(module.slots):
            module.load(slot, torch.randn(module.rank, module.in_features, device="cuda", generator=g) * 0.02,
                        torch.randn(module.out_features, module.rank, device="cuda", generator=g) * 0.02)
    prefix = torch.randn(a.layers, a.envs, policy.prefix_tokens, 2, 256, device="cuda", generator=g).bfloat16()
    state = torch.randn(a.envs, 14, device="cuda", generator=g)
    noise = torch.randn(a.envs, a.candidates, policy.horizon, policy.action_dim, device="cuda", generator=g)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for call in range(a.calls):
        policy.route(torch.randint(-1, 16, (a.envs,), device="cuda", generator=g, dtype=torch.int32))
        start.record()
        actions = policy.sample(noise, state, prefix, graph=True)
        end.record()
        end.synchronize()
        print(f"call {call}: {a.envs} x {a.candidates} chunks {tuple(actions.shape[2:])} in "
              f"{start.elapsed_time(end):.2f} ms, mean |action| {actions.abs().mean().item():.3f}")
    policy.release()


if __name__ == "__main__":
    main()
