"""shared_prefix_attention on the GPU against its formula in 64 bits.

Tolerance, per element of out = sum p v / sum p: the rounding of the output type; each p
rounded to that type, unit * sum p |v| / sum p; and for the scores, sums of D products in
fp32 (D / 16 accumulations of 2^-23 and the product with the scale) and the exponential
(2^-22 and 2^-23 of the exponent's magnitude): a relative error of each p of
e = scale * (D / 16 + 4) 2^-23 max sum |q||k| + 2^-21 (1 + range of the scores), which
enters twice (numerator and denominator); sums over n keys, (n / 16 + 64) 2^-23.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -24}


def operands(B, T, H, KV, D, G, P, S, dtype, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    return rand(B, T, H, D) * spread, rand(G, P, KV, D), rand(G, P, KV, D), rand(B, S, KV, D), rand(B, S, KV, D)


def groups_of(B, G, starts):
    if starts is None:
        return [b * G // B for b in range(B)]
    return [sum(1 for s in starts[1:G] if s <= b) for b in range(B)]


def check(out, q, pk, pv, k, v, *, starts=None, plens=None, lens=None, causal=False, scale=None):
    B, T, H, D = q.shape
    G, P, KV, _ = pk.shape
    S, rep = k.shape[1], H // KV
    scale = D ** -0.5 if scale is None else scale
    unit = UNIT[q.dtype]
    of = groups_of(B, G, starts)
    for b in range(B):
        g = of[b]
        pl, sl = P if plens is None else plens[g], S if lens is None else lens[b]
        keys = torch.cat([pk[g, :pl], k[b, :sl]]).double().repeat_interleave(rep, 1).transpose(0, 1)    # H, n, D
        vals = torch.cat([pv[g, :pl], v[b, :sl]]).double().repeat_interleave(rep, 1).transpose(0, 1)
        n = keys.shape[1]
        if n == 0:
            assert not out[b].any()
            continue
        qb = q[b].double().transpose(0, 1)                                                              # H, T, D
        s = scale * qb @ keys.transpose(1, 2)
        magnitude = (scale * qb.abs() @ keys.abs().transpose(1, 2)).amax(-1, keepdim=True)
        if causal:
            j = torch.arange(n, device=q.device)[None, :] - pl
            late = j > sl - T + torch.arange(T, device=q.device)[:, None]
            s = s.masked_fill(late & (j >= 0), float("-inf"))
        seen = ~torch.isinf(s)
        p = torch.where(seen.any(-1, keepdim=True), torch.softmax(s, -1), 0.0).nan_to_num(0.0)
        ref, mass = p @ vals, p @ vals.abs()
        span = torch.where(seen, s, 0.0).abs().amax(-1, keepdim=True)
        e = (D / 16 + 4) * 2.0 ** -23 * magnitude + 2.0 ** -21 * (1 + span)
        tol = (unit + 2 * e + (n / 16 + 64) * 2.0 ** -23) * mass
        got = out[b].double().transpose(0, 1)
        bad = ~((got - ref).abs() <= unit * ref.abs() + tol * (1 + unit) + TINY[q.dtype])
        assert not bad.any(), f"sequence {b}: {int(bad.sum())} of {bad.numel()}, worst {float((got - ref).abs().max())}"


def ints(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def run_and_check(q, pk, pv, k, v, *, starts=None, plens=None, lens=None, causal=False, scale=None):
    from actune_b200 import _lib, ops
    out = ops.shared_prefix_attention(q, pk, pv, k, v, starts=ints(starts), prefix_lens=ints(plens), lens=ints(lens),
                                      causal=causal, scale=scale)
    check(out, q, pk, pv, k, v, starts=starts, plens=plens, lens=lens, causal=causal, scale=scale)
    assert _lib.device_error() == (0, 0)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256, 8, 72, 136, 200])
@pytest.mark.parametrize("B,T,H,KV,G,P,S", [
    (1, 1, 1, 1, 1, 1, 0),        # the smallest call
    (4, 50, 8, 1, 1, 304, 50),    # several row tiles of one sequence
    (6, 1, 8, 2, 2, 700, 130),    # single tokens, stacked
    (5, 3, 6, 3, 1, 0, 40),       # no prefix
    (3, 70, 4, 4, 3, 129, 0),     # nothing of their own, a prefix each
])
def test_matches_the_formula(B, T, H, KV, G, P, S, D, dtype):
    ops_ = operands(B, T, H, KV, D, G, P, S, dtype, D + T)
    run_and_check(*ops_)
    run_and_check(*ops_, causal=True)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P,S", [(127, 1), (128, 128), (129, 127), (63, 65), (64, 64), (1000, 3), (2049, 300)])
def test_lengths_around_the_key_blocks(P, S, D):
    for B, T in ((9, 1), (2, 40)):
        run_and_check(*operands(B, T, 8, 2, D, 1, P, S, torch.bfloat16, P + S))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("T", [1, 4, 33])
@pytest.mark.parametrize("D", [64, 128, 256, 80])
def test_ragged_groups_and_lengths_over_stale_memory(D, T, causal):
    """Uneven and empty groups, lengths from zero on, NaN and infinities behind every end."""
    B, G, P, S = 11, 4, 400, 150
    q, pk, pv, k, v = operands(B, T, 8, 2, D, G, P, S, torch.bfloat16, T)
    starts, plens = [0, 3, 3, 10, 11], [400, 7, 129, 0]
    lens = [0, 1, T, 150, 64, 65, 127, 128, 129, 3, 0]   # the last sequence: no prefix, no key of its own
    for t, lengths in ((pk, plens), (pv, plens), (k, lens), (v, lens)):
        for i, n in enumerate(lengths):
            t[i, n:] = float("nan") if i % 2 else float("inf")
    out = run_and_check(q, pk, pv, k, v, starts=starts, plens=plens, lens=lens, causal=causal)
    assert not out[10].any()


# Tiles that hold rows of several sequences and their own keys too (chosen when there are
# tiles enough): 40 and 33 rows a sequence against tiles of 128 and 256.
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,T,H,KV", [(256, 5, 8, 1), (256, 50, 8, 1), (128, 10, 16, 4), (64, 33, 8, 8), (72, 11, 6, 2)])
def test_tiles_across_sequences(D, T, H, KV, causal):
    from actune_b200 import _lib
    B, G, P, S = 120, 3, 260, 90
    assert _lib.lib().actune_prefix_attention_workspace_size(B, T, H, KV, D, G, P, S, 1) == 0  # nothing to join
    q, pk, pv, k, v = operands(B, T, H, KV, D, G, P, S, torch.bfloat16, T)
    starts, plens = [0, 61, 61, 120], [259, 5, 130]
    lens = [(7 * b) % (S + 1) for b in range(B)]  # from zero on
    for t, lengths in ((pk, plens), (pv, plens), (k, lens), (v, lens)):
        for i, n in enumerate(lengths):
            t[i, n:] = float("nan") if i % 2 else float("inf")
    run_and_check(q, pk, pv, k, v, starts=starts, plens=plens, lens=lens, causal=causal)
    run_and_check(q, pk, pv, k, v, starts=starts, plens=[0, 0, 0], lens=lens, causal=causal)


@pytest.mark.parametrize("D,H,KV", [(256, 8, 1), (128, 8, 2)])
def test_one_request_does_not_reach_another_in_its_tile(D, H, KV):
    from actune_b200 import ops
    q, pk, pv, k, v = operands(100, 9, H, KV, D, 2, 200, 70, torch.bfloat16, 9)
    clean = ops.shared_prefix_attention(q, pk, pv, k, v)
    bad = [3, 4, 17, 51]
    v[3], k[4, 2], v[17, 69], q[51] = float("inf"), float("nan"), float("nan"), float("nan")
    dirty = ops.shared_prefix_attention(q, pk, pv, k, v)
    keep = [b for b in range(100) if b not in bad]
    assert torch.equal(clean[keep], dirty[keep])
    assert all(not dirty[b].isfinite().any() for b in bad)


def test_rows_that_see_nothing_are_zero():
    q, pk, pv, k, v = operands(3, 6, 4, 2, 64, 1, 16, 10, torch.bfloat16, 1)
    out = run_and_check(q, pk, pv, k, v, plens=[0], lens=[2, 6, 10], causal=True)
    assert not out[0, :4].any() and out[0, 4:].abs().sum() > 0 and out[1].abs().sum(-1).all()


@pytest.mark.parametrize("B,T,H,KV,G,P,S,D", [
    (40, 1, 8, 1, 1, 9000, 70, 128),     # stacked over more than two row tiles, split
    (300, 1, 4, 4, 5, 600, 20, 64),      # many sequences
    (2, 200, 8, 8, 1, 3000, 200, 128),   # many tiles by sequence
    (16, 5, 12, 4, 3, 1001, 77, 64),
    (1, 1, 8, 8, 1, 40000, 0, 128),      # one row, split as far as it goes
    (33, 2, 16, 1, 1, 2000, 33, 256),
])
@pytest.mark.parametrize("causal", [False, True])
def test_every_way_of_cutting_the_work(B, T, H, KV, G, P, S, D, causal):
    run_and_check(*operands(B, T, H, KV, D, G, P, S, torch.bfloat16, B), causal=causal)


def test_cache_views_slices_and_scale():
    g = torch.Generator(device="cuda").manual_seed(5)
    B, T, H, D, G, P, S = 8, 10, 8, 64, 2, 90, 12
    qkv = torch.randn(B * T, (H + 2) * D, device="cuda", generator=g).bfloat16()
    q = qkv[:, :H * D].view(B, T, H, D)
    prefix = torch.randn(G, P + 30, 2, D, device="cuda", generator=g).bfloat16()
    own = torch.randn(B, S, 2, D, device="cuda", generator=g).bfloat16()
    args = (q, prefix[:, :P, 0].unsqueeze(2), prefix[:, :P, 1].unsqueeze(2), own[:, :, 0].unsqueeze(2),
            own[:, :, 1].unsqueeze(2))
    run_and_check(*args)
    run_and_check(*args, scale=0.31)
    # heads before rows, as [n, heads, rows, D] caches have them
    t = torch.randn(G, 2, P, D, device="cuda", generator=g).bfloat16().transpose(1, 2)
    u = torch.randn(B, 2, S, D, device="cuda", generator=g).bfloat16().transpose(1, 2)
    run_and_check(q, t, t, u, u)


@pytest.mark.parametrize("D", [1, 20, 64, 250])
def test_any_alignment_and_stride(D):
    """What the tensor cores' copies cannot take goes through the scalar kernel: odd head
    sizes, odd offsets, expanded (stride 0) prefixes."""
    q, pk, pv, k, v = operands(4, 3, 4, 2, D, 2, 33, 9, torch.bfloat16, D)
    run_and_check(q, pk, pv, k, v, causal=True)
    odd = torch.randn(2, 33, 2, D + 3, device="cuda").bfloat16()[..., 1:D + 1]
    run_and_check(q, odd, pv, k, v, lens=[0, 3, 9, 1])
    run_and_check(q, pk[:1].expand(2, -1, -1, -1), pv[:1].expand(2, -1, -1, -1), k, v)


@pytest.mark.parametrize("spread", [0.0, 12.0, 60.0])
def test_sharp_and_flat_scores(spread):
    """Scores far apart (the running maximum grows often and by much) and all equal."""
    for B, T in ((5, 1), (2, 80)):
        run_and_check(*operands(B, T, 4, 2, 128, 1, 1500, 100, torch.bfloat16, 3, spread=spread))
    q, pk, pv, k, v = operands(2, 64, 2, 2, 64, 1, 1000, 64, torch.float16, 4)
    ramp = torch.arange(1000, device="cuda")[None, :, None, None] / 100
    run_and_check(q.abs(), (pk.abs() * ramp).half(), pv, k, v)  # every block holds a new maximum


def test_one_request_does_not_reach_another():
    from actune_b200 import ops
    q, pk, pv, k, v = operands(24, 2, 8, 2, 128, 3, 500, 40, torch.bfloat16, 8)
    clean = ops.shared_prefix_attention(q, pk, pv, k, v)
    k[5, 3], v[5], v[6, 0], pv[2, 100] = float("nan"), float("inf"), float("nan"), float("nan")
    dirty = ops.shared_prefix_attention(q, pk, pv, k, v)
    keep = [b for b in range(16) if b not in (5, 6)]
    assert torch.equal(clean[keep], dirty[keep])
    assert dirty[6].isnan().all() and dirty[16:].isnan().all() and not dirty[5].isfinite().any()


def test_long_cache_beyond_32_bit_offsets():
    """Rows whose element offset passes 2^31 (and bytes 2^32) in one prefix cache."""
    P, D = 70000, 128
    big = torch.empty(1, P, 256, D, device="cuda", dtype=torch.bfloat16)  # 2.29e9 elements, 4.6 GB
    big[:, :, 250:252].normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    pk, pv = big[:, :, 250:251], big[:, :, 251:252]
    q, _, _, k, v = operands(3, 1, 4, 1, D, 1, 1, 5, torch.bfloat16, 2)
    run_and_check(q, pk, pv, k, v)


def test_repeatable_and_on_another_stream_and_in_a_graph():
    from actune_b200 import ops
    args = operands(16, 1, 16, 4, 128, 2, 3000, 60, torch.bfloat16, 21)
    lens = ints([60] * 16)
    want = ops.shared_prefix_attention(*args, lens=lens, causal=True)
    assert torch.equal(want, ops.shared_prefix_attention(*args, lens=lens, causal=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        moved = [a * 1.0 for a in args]
        got = ops.shared_prefix_attention(*moved, lens=lens, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.shared_prefix_attention(*args, lens=lens, causal=True)
    for n in (60, 7):
        lens.fill_(n)
        graph.replay()
        check(out, *args, lens=[n] * 16, causal=True)


def test_empty_batch():
    from actune_b200 import ops
    q, pk, pv, k, v = operands(2, 3, 4, 2, 64, 1, 10, 4, torch.bfloat16, 1)
    assert ops.shared_prefix_attention(q[:0], pk, pv, k[:0], v[:0]).shape == (0, 3, 4, 64)
    assert ops.shared_prefix_attention(q[:, :0], pk, pv, k, v).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("below", [16.0, 21.5, 23.4, 25.1, 27.0])
@pytest.mark.parametrize("B,T,H,KV,G,P,S,D", [
    (1, 1, 4, 4, 1, 32768, 0, 64),     # by sequence, parts joined
    (24, 1, 8, 2, 1, 32768, 5, 128),   # stacked
    (120, 5, 8, 1, 3, 8192, 64, 256),  # mixed tiles
    (2, 200, 4, 4, 2, 8192, 64, 64),
])
def test_a_long_tail_of_keys_far_below_a_sink_in_fp16(B, T, H, KV, G, P, S, D, below):
    """One key with value 0 ahead of all others by `below` (log2): the output is what the
    tail weighs, and none of it may fall under fp16's range on the way.

    The tail's probabilities all are about 2^-below of the sink's.  Each is rounded to fp16
    relative to a maximum of 2^7, in steps of 2^-24 at least: by 2^-32 of the sink's at
    most, beside the relative error of `check`'s bound."""
    g = torch.Generator(device="cuda").manual_seed(int(10 * below))

    def near(*shape, mean):  # exact in fp16 and of 5 values only: products and sums of scores are exact
        return (torch.randint(-2, 3, shape, device="cuda", generator=g) * 2.0 ** -5 + mean).half()

    q = torch.zeros(B, T, H, D, device="cuda").half()
    q[..., 0] = 1.0
    pk, k = torch.zeros(G, P, KV, D, device="cuda").half(), torch.zeros(B, S, KV, D, device="cuda").half()
    pk[..., 0], k[..., 0] = near(G, P, KV, mean=-below), near(B, S, KV, mean=-below)
    pk[:, 0] = 0.0  # the sink
    pv, v = near(G, P, KV, D, mean=1.0), near(B, S, KV, D, mean=1.0)
    pv[:, 0] = 0.0
    scale = 0.6931471805599453  # scores in log2
    from actune_b200 import _lib, ops
    out = ops.shared_prefix_attention(q, pk, pv, k, v, scale=scale)
    assert _lib.device_error() == (0, 0)
    for b in range(B):
        keys, values = torch.cat([pk[b * G // B], k[b]]).double(), torch.cat([pv[b * G // B], v[b]]).double()
        w = torch.exp2(keys[..., 0]).t()                       # KV, n
        p = w / w.sum(1, keepdim=True)
        ref = torch.einsum("kn,nkd->kd", p, values)
        mass = torch.einsum("kn,nkd->kd", p, values.abs())
        n = keys.shape[0]
        e = (D / 16 + 4) * 2.0 ** -23 * below + 2.0 ** -21 * (1 + below)
        tol = (UNIT[torch.float16] + 2 * e + (n / 16 + 64) * 2.0 ** -23) * mass \
            + 2.0 ** -32 / w.sum(1)[:, None] * torch.einsum("nkd->kd", values.abs())
        got = out[b].double().view(T, KV, H // KV, D)
        bad = (got - ref[None, :, None]).abs() > (UNIT[torch.float16] * ref.abs() + tol * (1 + UNIT[torch.float16])
                                                  + TINY[torch.float16])[None, :, None]
        assert not bad.any(), f"sequence {b}: {float((got - ref[None, :, None]).abs().max())} of {float(ref.abs().max())}"


@pytest.mark.parametrize("B,T,D", [(4, 50, 128), (24, 1, 64), (100, 9, 256), (3, 2, 20)])
def test_out_is_written_and_returned(B, T, D):
    from actune_b200 import ops
    args = operands(B, T, 8, 2, D, 1, 700, 30, torch.bfloat16, 31)
    want = ops.shared_prefix_attention(*args)
    room = torch.full((B + 2, T, 8, D), 7.0, device="cuda", dtype=torch.bfloat16)
    out = room[1:-1]
    assert ops.shared_prefix_attention(*args, out=out) is out and torch.equal(out, want)
    assert (room[0] == 7).all() and (room[-1] == 7).all()
    w = torch.ones(D, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    loss = (w * out).sum()
    ops.shared_prefix_attention(*args, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    for wrong in (room, out.transpose(2, 3).contiguous().transpose(2, 3), out.half()):
        with pytest.raises(RuntimeError, match="out must be contiguous and match q"):
            ops.shared_prefix_attention(*args, out=wrong)
