"""Cases for timing the serving operators: attention over shared prefixes, low-rank
adapters of many requests, and the gated norm between blocks.

``prepare(case, seed)`` makes a case's inputs on the GPU, ``run(state)`` makes one
pass: with ``own`` set through ``actune_b200.ops``, otherwise as elementary torch
operations in 32 bits, rounded once at the end.  ``exact(case, seed)`` is the same
answer from the operator's definition in 64 bits, and ``work(case)`` the bytes and
operations a pass cannot do without.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # pi0.5-shaped policy, one observation, four action candidates: 50 action tokens
        # each attend to the shared 304-token prefix and to one another.
        dict(name="attn_pi05_1x4", op="attention", dtype="bf16", groups=1, seqs=4, tokens=50, heads=8, kv_heads=1,
             dim=256, prefix=304, suffix=50, causal=False, ragged=False, cache=True),
        # The same for a full serving batch: 16 observations, eight candidates each.
        dict(name="attn_pi05_16x8", op="attention", dtype="bf16", groups=16, seqs=128, tokens=50, heads=8, kv_heads=1,
             dim=256, prefix=304, suffix=50, causal=False, ragged=False, cache=True),
        # Token-by-token decoding of 32 sequences behind one long instruction, each with
        # up to 512 tokens of its own; grouped-query heads.
        dict(name="attn_decode_32_long", op="attention", dtype="bf16", groups=1, seqs=32, tokens=1, heads=32,
             kv_heads=8, dim=128, prefix=32768, suffix=512, causal=True, ragged=True, cache=False),
        # OFT-shaped heads: 56 parallel action tokens of 16 sequences behind two long
        # histories of unequal length and unequal share.
        dict(name="attn_oft_16_history", op="attention", dtype="bf16", groups=2, seqs=16, tokens=56, heads=32,
             kv_heads=32, dim=128, prefix=8192, suffix=56, causal=False, ragged=True, cache=False),
        # Odd everything: a few tokens at once (fp16), three prefixes of odd length, one
        # of them possibly empty, causal among a sequence's own tokens.
        dict(name="attn_odd_f16", op="attention", dtype="f16", groups=3, seqs=13, tokens=5, heads=12, kv_heads=4,
             dim=64, prefix=1001, suffix=77, causal=True, ragged=True, cache=False),
        # One token through one adapted 4096 x 4096 projection: the latency case.
        dict(name="adapter_1_token", op="adapter", dtype="bf16", requests=1, tokens=1, slots=8, rank=16, k=4096,
             n=4096, idle=0),
        # 32 single-token requests, each its own adapter, OFT gate/up projection.
        dict(name="adapter_32_requests", op="adapter", dtype="bf16", requests=32, tokens=1, slots=32, rank=16, k=4096,
             n=22016, idle=0),
        # 16 environments x 50 action tokens through the action expert's fused QKV, some
        # of them without an adapter.
        dict(name="adapter_expert_qkv", op="adapter", dtype="f16", requests=16, tokens=50, slots=12, rank=16, k=1024,
             n=2560, idle=3),
        # 16 prefix passes of 304 tokens through the VLM's fused gate/up at rank 64.
        dict(name="adapter_vlm_gate_up", op="adapter", dtype="bf16", requests=16, tokens=304, slots=16, rank=64,
             k=2048, n=32768, idle=0),
        # One token between two blocks of a 4096-wide decoder.
        dict(name="norm_1_token", op="norm", dtype="bf16", rows=1, width=4096, groups=1, post=True, gate="width",
             shift=False, gemma=False, scale=0.5, bits=0),
        # 16 environments x 50 action tokens of the action expert, gate, weight and shift
        # per environment (a flow-time modulated layer), quantized for the next packed
        # projection.
        dict(name="norm_expert_q8", op="norm", dtype="bf16", rows=800, width=1024, groups=16, post=True,
             gate="group", shift=True, gemma=True, scale=1.0, bits=8),
        # The prefix tokens of 128 observations, an odd count of rows.
        dict(name="norm_vlm_large", op="norm", dtype="bf16", rows=38911, width=2048, groups=1, post=True,
             gate="width", shift=False, gemma=True, scale=1.0, bits=0),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["attention", "adapter", "norm"])
    if op == "attention":
        while True:
            kv, rep = rng.choice([1, 1, 2, 4, 8, 32]), rng.choice([1, 2, 3, 4, 8])
            groups = _log(rng, 1, 16)
            case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), groups=groups,
                        seqs=groups * _log(rng, 1, 16) + (rng.randrange(groups) if groups > 1 else 0),
                        tokens=rng.choice([1, 1, _log(rng, 1, 64)]), heads=kv * rep, kv_heads=kv,
                        dim=rng.choice([64, 128, 256, 80]), prefix=_log(rng, 1, 32768), suffix=0,
                        causal=rng.random() < 0.5, ragged=True, cache=kv == 1 and rng.random() < 0.5)
            case["suffix"] = case["tokens"] + _log(rng, 1, 512) - 1
            copies = case["seqs"] * (case["prefix"] + case["suffix"]) * kv * case["dim"] * 4
            scores = case["seqs"] * case["tokens"] * case["heads"] * (case["prefix"] + case["suffix"]) * 4
            if work(case)["flops"] <= 6e10 and max(copies, scores) <= 6e9:
                return case
    if op == "adapter":
        while True:
            requests = _log(rng, 1, 64)
            case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), requests=requests,
                        tokens=rng.choice([1, _log(rng, 1, 304)]), slots=_log(rng, 1, 64),
                        rank=rng.choice([8, 16, 16, 32, 64, 128]), k=8 * _log(rng, 32, 1376),
                        n=8 * _log(rng, 32, 2752), idle=rng.randrange(1 + requests // 3))
            if requests * case["tokens"] * (case["n"] + case["k"]) <= 1e8:
                return case
    while True:
        groups, per = _log(rng, 1, 64), _log(rng, 1, 1024)
        bits = rng.choice([0, 0, 8])
        case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=groups * per,
                    width=64 * _log(rng, 4, 128) if bits else rng.choice([8 * _log(rng, 8, 1024), _log(rng, 33, 8191)]),
                    groups=groups, post=rng.random() < 0.75, gate=rng.choice(["none", "width", "group"]),
                    shift=rng.random() < 0.5, gemma=rng.random() < 0.5, scale=rng.choice([1.0, 0.5, 0.7]), bits=bits)
        if case["rows"] * case["width"] <= 6e7:
            return case


def _lengths(case, seed):
    """(starts, prefix_lens, lens) as Python lists: the shape of the batch, from the seed."""
    r = random.Random(seed * 1000003 + 17)
    g, b, p, s = case["groups"], case["seqs"], case["prefix"], case["suffix"]
    if not case["ragged"]:
        return [i * b // g for i in range(g + 1)], [p] * g, [s] * b
    starts = [0] + sorted(r.randrange(b + 1) for _ in range(g - 1)) + [b]
    plens = [p] + [r.randint(p // 2, p) for _ in range(g - 1)]
    r.shuffle(plens)
    low = case["tokens"] if case["tokens"] <= s else s
    return starts, plens, [r.randint(low, s) for _ in range(b)]


def _mean_keys(case):
    """Keys that a query row sees, as far as the case fixes them (half the room for ragged lengths)."""
    p, s, t = case["prefix"], case["suffix"], case["tokens"]
    if case["ragged"]:
        p, s = (p * 0.75 if case["groups"] > 1 else p), (s + t) / 2
    return p, s


def work(case):
    if case["op"] == "attention":
        p, s = _mean_keys(case)
        rows = case["seqs"] * case["tokens"] * case["heads"]
        per_key = case["kv_heads"] * case["dim"] * 2 * 2
        seen = p + (s - (case["tokens"] - 1) / 2 if case["causal"] else s)
        return dict(bytes=2 * rows * case["dim"] * 2 + (case["groups"] * p + case["seqs"] * s) * per_key,
                    flops=4.0 * rows * seen * case["dim"])
    if case["op"] == "adapter":
        m, active = case["requests"] * case["tokens"], case["requests"] - case["idle"]
        used = min(active, case["slots"])
        return dict(bytes=2.0 * (active * case["tokens"] * case["k"] + 2 * m * case["n"]
                                 + used * case["rank"] * (case["k"] + case["n"])),
                    flops=2.0 * active * case["tokens"] * case["rank"] * (case["k"] + case["n"]))
    size = 4 if case["dtype"] == "f32" else 2
    elements = case["rows"] * case["width"]
    rows_of = {"none": 0, "width": 1, "group": case["groups"]}
    small = (case["post"] + case["shift"] * case["groups"] + rows_of[case["gate"]] + 1) * case["width"]
    coded = elements * case["bits"] / 8 + elements / 64 * 4 if case["bits"] else 0
    return dict(bytes=float(4 * elements * size + small * size + coded), flops=12.0 * elements)


# ------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale + mean).to(dt)

    if case["op"] == "attention":
        G, B, T, P, S = case["groups"], case["seqs"], case["tokens"], case["prefix"], case["suffix"]
        H, KV, D = case["heads"], case["kv_heads"], case["dim"]
        starts, plens, lens = _lengths(case, seed)
        # The queries are a slice of the fused projection's output.
        qkv = randn(B * T, (H + 2 * KV) * D)
        q = qkv[:, :H * D].view(B, T, H, D)

        def keys_values(n, length):
            if case["cache"]:  # rows [key | value] of one KV head
                rows = randn(n, length, 2, D)
                return rows[:, :, 0].unsqueeze(2), rows[:, :, 1].unsqueeze(2)
            return randn(n, length, KV, D), randn(n, length, KV, D)

        pk, pv = keys_values(G, P)
        k, v = keys_values(B, S)
        # A few keys that many queries look at, as attention sinks are.
        pk[:, :: max(1, P // 5)] *= 2.0
        state = dict(case=case, q=q, prefix_k=pk, prefix_v=pv, k=k, v=v, causal=case["causal"])
        if case["ragged"]:
            # What lies behind a sequence's end is stale memory: not numbers to rely on.
            for t, n in ((pk, plens), (pv, plens), (k, lens), (v, lens)):
                gone = torch.arange(t.shape[1], device=DEV)[None, :] >= torch.tensor(n, device=DEV)[:, None]
                t.masked_fill_(gone[:, :, None, None], float("nan"))
            state |= dict(starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
                          prefix_lens=torch.tensor(plens, dtype=torch.int32, device=DEV),
                          lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        return state
    if case["op"] == "adapter":
        r = random.Random(seed * 1000003 + 29)
        R, T, S = case["requests"], case["tokens"], case["slots"]
        of = list(range(min(R, S))) + [r.randrange(S) for _ in range(R - min(R, S))]
        r.shuffle(of)
        for i in r.sample(range(R), case["idle"]):
            of[i] = -1
        slots = torch.tensor(of, dtype=torch.int32, device=DEV).repeat_interleave(T)
        state = dict(case=case, slots=slots, longest=max([of.count(s) for s in range(S)] + [1]) * T,
                     x=randn(R * T, case["k"]), y=randn(R * T, case["n"]),
                     down=randn(S, case["rank"], case["k"], scale=case["k"] ** -0.5),
                     up=randn(S, case["n"], case["rank"], scale=case["rank"] ** -0.5),
                     scale=torch.rand(S, device=DEV, generator=g) + 0.5)
        if own:  # the routing of a batch, made once and used by every projection of every layer
            from actune_b200 import ops
            state["plan"] = ops.adapter_plan(slots, S)
        return state
    rows, width, groups = case["rows"], case["width"], case["groups"]
    mean = 0.0 if case["gemma"] else 1.0
    # A residual stream has a few channels much larger than the others.
    residual = randn(rows, width)
    residual[:, 3 % width::97] *= 12.0
    return dict(case=case, x=randn(rows, width, scale=0.7), residual=residual,
                post_weight=randn(width, scale=0.2, mean=mean) if case["post"] else None,
                pre_weight=randn(width, scale=0.2, mean=mean),
                gate={"none": None, "width": randn(width, scale=0.5),
                      "group": randn(groups, width, scale=0.5)}[case["gate"]],
                shift=randn(groups, width, scale=0.2) if case["shift"] else None)


# ------------------------------------------------------------------------------ one pass
def _attention_plain(st):
    q, pk, pv, k, v = (st[n].float() for n in ("q", "prefix_k", "prefix_v", "k", "v"))
    B, T, H, D = q.shape
    (G, P, KV, _), S = pk.shape, k.shape[1]
    seq = torch.arange(B, device=q.device)
    if "starts" in st:
        group = (seq[:, None] >= st["starts"][None, 1:]).sum(1).clamp(max=G - 1)
        plen, slen = st["prefix_lens"][group], st["lens"]
    else:
        group, plen, slen = seq * G // B, torch.full_like(seq, P), torch.full_like(seq, S)
    in_prefix = torch.arange(P, device=q.device)[None, :] < plen[:, None]
    in_own = torch.arange(S, device=q.device)[None, :] < slen[:, None]
    keys = torch.cat([pk[group], k], 1).permute(0, 2, 3, 1)                       # B, KV, D, P + S
    live = torch.cat([in_prefix, in_own], 1)
    values = torch.where(live[:, :, None, None], torch.cat([pv[group], v], 1), 0.0).transpose(1, 2)
    rows = q.view(B, T, KV, H // KV, D).transpose(1, 2).reshape(B, KV, T * (H // KV), D)
    scores = (rows @ keys * D ** -0.5).view(B, KV, T, H // KV, P + S)
    seen = live[:, None, :].expand(B, T, P + S)
    if st["causal"]:
        last = (slen[:, None] - T + torch.arange(T, device=q.device))[:, :, None]
        before = torch.arange(S, device=q.device)[None, None, :] <= last
        seen = seen & torch.cat([torch.ones(B, T, P, dtype=torch.bool, device=q.device), before], 2)
    seen = seen[:, None, :, None, :]
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = weights.view(B, KV, T * (H // KV), P + S) @ values
    out = out.view(B, KV, T, H // KV, D) / torch.where(total == 0, 1.0, total)
    return out.transpose(1, 2).reshape(B, T, H, D).to(st["q"].dtype)


def _adapter_plain(st):
    x, y, down, up = (st[n].float() for n in ("x", "y", "down", "up"))
    S = down.shape[0]
    slots = st["slots"].long()
    used = slots >= 0
    slot = torch.where(used, slots, S)  # the last, empty place takes the rows without an adapter
    mine = slot[:, None] == torch.arange(S, device=x.device)[None, :]
    place = torch.where(used, (mine.cumsum(0) * mine).sum(1) - 1, 0)
    padded = torch.zeros(S + 1, st["longest"], x.shape[1], device=x.device)
    padded[slot, place] = x
    delta = (padded[:S] @ down.transpose(1, 2)) @ up.transpose(1, 2) * st["scale"][:, None, None]
    delta = torch.where(used[:, None], delta[slot.clamp(max=S - 1), place], 0.0)
    return (y + delta).to(st["y"].dtype)


def _norm_plain(st):
    case = st["case"]
    x, residual = st["x"].float(), st["residual"].float()
    one = 1.0 if case["gemma"] else 0.0
    per = case["rows"] // case["groups"]

    def spread(t):
        t = t.float()
        return t if t.dim() == 1 else t.repeat_interleave(per, 0)

    def norm(a, w):
        return a * torch.rsqrt(a.square().mean(-1, keepdim=True) + 1e-6) * (one + w)

    u = norm(x, spread(st["post_weight"])) if case["post"] else x
    s = residual * case["scale"] + (u if st["gate"] is None else spread(st["gate"]) * u)
    h = norm(s, spread(st["pre_weight"]))
    if st["shift"] is not None:
        h = h + spread(st["shift"])
    h = h.to(st["x"].dtype)
    out = [h, s.to(st["x"].dtype)]
    if case["bits"]:
        top = float(2 ** (case["bits"] - 1) - 1)
        parts = h.float().view(case["rows"], -1, 64)
        step = parts.abs().amax(-1, keepdim=True).clamp(min=1e-8) / torch.tensor(top, device=x.device)
        codes = torch.round(parts / step).clamp(-top - 1, top)
        out.append((codes * step).view(h.shape).to(h.dtype))
    return out


def _codes_to_values(packed, scales, dtype):
    """The values that 8-bit group-64 codes stand for."""
    codes = packed.view(torch.int8).view(packed.shape[0], -1, 64)
    return (codes.float() * scales[:, :, None]).view(packed.shape).to(dtype)


def run(state):
    case = state["case"]
    if not own:
        return {"attention": _attention_plain, "adapter": _adapter_plain, "norm": _norm_plain}[case["op"]](state)
    from actune_b200 import ops
    if case["op"] == "attention":
        return ops.shared_prefix_attention(state["q"], state["prefix_k"], state["prefix_v"], state["k"], state["v"],
                                           starts=state.get("starts"), prefix_lens=state.get("prefix_lens"),
                                           lens=state.get("lens"), causal=state["causal"])
    if case["op"] == "adapter":
        return ops.adapter_add(state["y"], state["x"], state["down"], state["up"], state["scale"], state["plan"])
    out = ops.gated_norm(state["x"], state["residual"], state["pre_weight"], post_weight=state["post_weight"],
                         gate=state["gate"], shift=state["shift"], residual_scale=case["scale"], eps=1e-6,
                         gemma=case["gemma"], quant_bits=case["bits"] or None)
    if not case["bits"]:
        return list(out)
    h, s, packed, scales = out
    return [h, s, _codes_to_values(packed, scales, h.dtype)]


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        starts, plens, lens = _lengths(case, seed)
        T, H, KV, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        out = torch.zeros(case["seqs"], T, H, D, dtype=torch.float64, device=DEV)
        for g in range(case["groups"]):
            for b in range(starts[g], starts[g + 1]):
                for head in range(KV):
                    mine = slice(head * (H // KV), (head + 1) * (H // KV))
                    keys = torch.cat([st["prefix_k"][g, :plens[g], head], st["k"][b, :lens[b], head]]).double()
                    values = torch.cat([st["prefix_v"][g, :plens[g], head], st["v"][b, :lens[b], head]]).double()
                    s = torch.einsum("thd,nd->thn", st["q"][b, :, mine].double(), keys) / math.sqrt(D)
                    if case["causal"]:
                        t = torch.arange(T, device=DEV)[:, None, None]
                        j = torch.arange(len(keys), device=DEV)[None, None, :] - plens[g]
                        s = s.masked_fill(j > lens[b] - T + t, float("-inf"))
                    out[b, :, mine] = torch.einsum("thn,nd->thd", torch.softmax(s, -1), values)
        return out
    if case["op"] == "adapter":
        out = st["y"].double()
        for s in range(case["slots"]):
            rows = (st["slots"] == s).nonzero()[:, 0]
            low = st["x"][rows].double() @ st["down"][s].double().T
            out[rows] += float(st["scale"][s]) * (low @ st["up"][s].double().T)
        return out
    rows, groups = case["rows"], case["groups"]

    def spread(t):
        return t.double().expand(groups, -1)[:, None, :]

    def norm(a, w):
        w = spread(w) + 1 if case["gemma"] else spread(w)
        return w * a / torch.sqrt((a * a).sum(-1, keepdim=True) / case["width"] + 1e-6)

    u = st["x"].double().view(groups, rows // groups, -1)
    if case["post"]:
        u = norm(u, st["post_weight"])
    if st["gate"] is not None:
        u = u * spread(st["gate"])
    s = u + case["scale"] * st["residual"].double().view(u.shape)
    h = norm(s, st["pre_weight"])
    if st["shift"] is not None:
        h = h + spread(st["shift"])
    # The codes are those of the rounded h: no value of their own in 64 bits.
    return [h.reshape(rows, -1), s.reshape(rows, -1)] + ([None] if case["bits"] else [])
