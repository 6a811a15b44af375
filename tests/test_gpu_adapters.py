"""Per-request low-rank adapters on the GPU against their formula in 64 bits.

Tolerance, per element of out = y + scale * up (down x): the rounding of the output
type; for down x, a chain of K / 16 accumulations of at most 2^-23 each (plus 64 for the
sums across warps and slices) of sum |down x|; the two-part split of it, 2^-16 of the
row's largest; for up v, 2 * R / 16 + 8 accumulations of 2^-23.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def operands(rows, k, n, slots, rank, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    return (rand(rows, n), rand(rows, k), rand(slots, rank, k, scale=k ** -0.5), rand(slots, n, rank),
            torch.rand(slots, device="cuda", generator=g) + 0.5)


def check(out, y, x, down, up, scale, slots):
    k, rank, unit = x.shape[1], down.shape[1], UNIT[out.dtype]
    for s in range(-1, down.shape[0]):
        rows = ((slots < 0) | (slots >= down.shape[0]) if s < 0 else slots == s).nonzero()[:, 0]
        if not len(rows):
            continue
        if s < 0:
            assert torch.equal(out[rows], y[rows])
            continue
        xs, d, u, f = x[rows].double(), down[s].double(), up[s].double(), float(scale[s])
        v = xs @ d.T
        dv = (k / 16 + 64) * 2.0 ** -23 * (xs.abs() @ d.abs().T) + 2.0 ** -16 * v.abs().amax(1, keepdim=True)
        ref = y[rows].double() + f * (v @ u.T)
        tol = f * (dv @ u.abs().T + (rank / 8 + 8) * 2.0 ** -23 * (v.abs() @ u.abs().T)) + 2.0 ** -22 * ref.abs()
        bad = (out[rows].double() - ref).abs() > unit * ref.abs() + tol * (1 + unit) + 2.0 ** -24
        assert not bad.any(), f"slot {s}: {int(bad.sum())} of {bad.numel()} out of tolerance"


def random_slots(rows, slots, seed, low=-1):
    return torch.randint(low, slots, (rows,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()


@pytest.mark.parametrize("rows,slots", [(1, 1), (1, 7), (16, 1), (17, 40), (33, 2), (100, 3), (65, 1), (300, 5),
                                        (1500, 700)])
def test_plan_covers_every_row_once_and_in_order(rows, slots):
    from actune_b200 import ops
    index = random_slots(rows, slots + 1, rows + slots, low=-2)  # below and above the range: no adapter
    plan = ops.adapter_plan(index, slots)
    words = plan.buffer.cpu()
    count = int(words[0])
    capacity = (len(words) - 4 - rows) // 4
    assert count <= capacity
    tiles = words[4:4 + 4 * count].view(-1, 4).tolist()
    order = words[4 + 4 * capacity:].tolist()
    assert sorted(order) == list(range(rows))
    seen = 0
    for slot, first, size, _ in tiles:
        assert first == seen and 1 <= size <= plan.tile
        seen += size
        mine = order[first:first + size]
        assert mine == sorted(mine)
        for m in mine:
            s = int(index[m])
            assert slot == (s if 0 <= s < slots else -1)
    assert seen == rows


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [1, 4, 7, 8, 16, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("rows,slots", [(1, 3), (40, 2), (200, 3)])
def test_matches_the_formula_at_every_rank(rows, slots, rank, dtype):
    from actune_b200 import ops
    y, x, down, up, scale = operands(rows, 520, 328, slots, rank, dtype, rank + rows)
    index = random_slots(rows, slots, rank)
    out = ops.adapter_add(y, x, down, up, scale, ops.adapter_plan(index, slots))
    check(out, y, x, down, up, scale, index)


@pytest.mark.parametrize("rows,k,n,slots", [(1, 8, 8, 1), (1, 4096, 4096, 8), (5, 1, 1, 2), (3, 33, 65, 2),
                                            (31, 1000, 1003, 31), (64, 2048, 640, 64), (129, 136, 72, 2),
                                            (70, 4104, 264, 1), (450, 260, 514, 9)])
def test_odd_sizes(rows, k, n, slots):
    from actune_b200 import ops
    y, x, down, up, scale = operands(rows, k, n, slots, 16, torch.bfloat16, k + n)
    index = random_slots(rows, slots, n)
    out = ops.adapter_add(y, x, down, up, scale, ops.adapter_plan(index, slots))
    check(out, y, x, down, up, scale, index)


@pytest.mark.parametrize("rows", [2, 37, 150])
def test_strided_unaligned_and_in_place(rows):
    from actune_b200 import ops
    for offset, pitch in ((8, 400), (3, 400), (0, 401)):
        y, x, down, up, scale = operands(rows, 264, 320, 4, 16, torch.bfloat16, offset)
        index = random_slots(rows, 4, 1)
        plan = ops.adapter_plan(index, 4)
        wide = torch.randn(rows, pitch, device="cuda").bfloat16()
        view = wide[:, offset:offset + 320]
        view.copy_(y)
        xs = torch.cat([x, x], 1)[:, 264:]
        want = ops.adapter_add(y, x, down, up, scale, plan)
        check(want, y, x, down, up, scale, index)
        around = wide.clone()
        assert ops.adapter_add(view, xs, down, up, scale, plan, out=view) is view
        check(view, y, x, down, up, scale, index)  # another alignment may run another kernel form
        around[:, offset:offset + 320] = view
        assert torch.equal(around, wide)  # nothing beside the rows was written


def test_non_finite_rows_stay_alone_and_no_adapter_reads_nothing():
    from actune_b200 import ops
    y, x, down, up, scale = operands(90, 256, 256, 3, 16, torch.bfloat16, 2)
    index = random_slots(90, 3, 4)
    clean = ops.adapter_add(y, x, down, up, scale, ops.adapter_plan(index, 3))
    x[5], x[6, 0], down[2] = float("nan"), float("inf"), float("nan")
    index[5], index[6], index[7] = 0, -1, 2
    out = ops.adapter_add(y, x, down, up, scale, ops.adapter_plan(index, 3))
    assert out[5].isnan().all() and torch.equal(out[6], y[6]) and out[7].isnan().all()
    keep = [i for i in range(90) if i not in (5, 6, 7) and int(index[i]) != 2]
    assert torch.equal(out[keep], clean[keep])


def test_large_and_small_magnitudes_in_fp16():
    """down x may leave fp16's range, or its precision, on the way: it is held in 32 bits."""
    from actune_b200 import ops
    for factor in (2.0 ** 9, 2.0 ** -12):
        y, x, down, up, scale = operands(20, 512, 128, 2, 8, torch.float16, 6)
        x, up = (x * factor).half(), (up / (factor * 16)).half()
        down = (down * 64).half() if factor > 1 else down
        index = random_slots(20, 2, 6, low=0)
        out = ops.adapter_add(y, x, down, up, scale, ops.adapter_plan(index, 2))
        check(out, y, x, down, up, scale, index)


def test_rows_are_independent_of_their_company():
    """A row alone and in a batch: the same bits (same sizes of slices) whatever sits beside it."""
    from actune_b200 import ops
    y, x, down, up, scale = operands(64, 512, 256, 4, 16, torch.bfloat16, 3)
    index = random_slots(64, 4, 8, low=0)
    out = ops.adapter_add(y, x, down, up, scale, ops.adapter_plan(index, 4))
    perm = torch.randperm(64, generator=torch.Generator().manual_seed(1)).cuda()
    again = ops.adapter_add(y[perm], x[perm], down, up, scale, ops.adapter_plan(index[perm].contiguous(), 4))
    assert torch.equal(again, out[perm])


def test_empty_batch_and_update_in_a_graph():
    from actune_b200 import ops
    y, x, down, up, scale = operands(48, 256, 256, 5, 16, torch.bfloat16, 12)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert ops.adapter_add(y[:0], x[:0], down, up, scale, ops.adapter_plan(none, 5)).shape == (0, 256)
    slots = random_slots(48, 5, 1)
    plan = ops.adapter_plan(slots, 5)
    ops.adapter_add(y, x, down, up, scale, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(slots)
        out = ops.adapter_add(y, x, down, up, scale, plan)
    for seed in (2, 3):
        slots.copy_(random_slots(48, 5, seed))
        graph.replay()
        check(out, y, x, down, up, scale, slots)


def test_graph_replay_follows_the_scope():
    """Captured under a plan or under none, then called under others and with the first gone."""
    from actune_b200 import ops
    from actune_b200.adapters import AdaptedLinear, adapter_scope
    from actune_b200.graph import GraphReplay
    linear = torch.nn.Linear(64, 96, bias=False, device="cuda", dtype=torch.bfloat16)
    layer = AdaptedLinear(linear, slots=3, rank=8)
    g = torch.Generator(device="cuda").manual_seed(1)
    for slot in range(3):
        layer.load(slot, torch.randn(8, 64, device="cuda", generator=g), torch.randn(96, 8, device="cuda", generator=g))
    x = torch.randn(40, 64, device="cuda", generator=g).bfloat16()
    with torch.inference_mode():
        y = linear(x)
        for captured in (0, None):
            replay = GraphReplay(layer, {})
            replay.enabled = True
            slots = [random_slots(40, 3, seed) for seed in range(3)]
            plans = [ops.adapter_plan(s, 3) for s in slots]

            def call(of):
                with adapter_scope(None if of is None else plans[of]):
                    out = replay(x)
                if of is None:
                    assert torch.equal(out, y)
                else:
                    check(out, y, x, layer.down, layer.up, layer.scale, slots[of])

            for of in (captured, 1, None, 0, 2, None):
                call(of)
            assert torch.equal(replay(x), y)  # outside any scope
            # The first plan goes, and its memory is something else's.
            plans[0] = slots[0] = None
            others = [torch.full_like(plans[1].buffer, -1) for _ in range(64)]
            for of in (1, None, 2):
                call(of)
            plans[2].update(slots[1])
            slots[2] = slots[1]
            call(2)
            assert len(replay.graphs) == 2 and replay.fallbacks == 0 and len(others) == 64
            replay.release()


def test_autograd_sees_what_out_overwrites():
    """A value saved for a backward pass and then written to is refused by that pass."""
    from actune_b200 import ops
    y, x, down, up, scale = operands(20, 64, 64, 2, 8, torch.bfloat16, 3)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    plan = ops.adapter_plan(random_slots(20, 2, 1), 2)
    for out in (None, y):
        loss = (w * y).sum()
        ops.adapter_add(y, x, down, up, scale, plan, out=out)
        if out is None:
            loss.backward()
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
    with torch.inference_mode():
        z = y * 1.0
        ops.adapter_add(z, x, down, up, scale, plan, out=z)
    ops.adapter_add(z, x, down, up, scale, plan, out=z)  # outside too: an inference tensor has no version


# The form of long prompts: tiles of 128 rows, y and out as boxes of 32 consecutive rows.
# Requests of every remainder of a box and of a tile, some without an adapter, over enough
# columns (the last step's 8 of 128) for a block to go through its rings several times.
RUNS = (304, 81, 50, 128, 16, 33, 700, 1, 31, 352, 15, 97, 304, 112)


def run_slots(rows, slots, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    while len(out) < rows:
        for n in RUNS:
            out += [int(torch.randint(-1, slots, (1,), generator=g))] * n
    return torch.tensor(out[:rows], dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 104, 128])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_prompts(in_place, rank, dtype):
    from actune_b200 import _lib, ops
    rows, n = 4864, 8200
    y, x, down, up, scale = operands(rows, 136, n, 16, rank, dtype, rank)
    index = run_slots(rows, 16, rank)
    plan = ops.adapter_plan(index, 16)
    assert plan.tile == 128
    out = y.clone() if in_place else None
    got = ops.adapter_add(y if out is None else out, x, down, up, scale, plan, out=out)
    assert _lib.device_error() == (0, 0)
    check(got, y, x, down, up, scale, index)


@pytest.mark.parametrize("rank", [16, 64, 128])
@pytest.mark.parametrize("columns", [72, 1024, 2056])
def test_long_prompts_strided_and_in_place(columns, rank):
    from actune_b200 import ops
    rows = 4200
    y, x, down, up, scale = operands(rows, 264, columns, 7, rank, torch.bfloat16, columns)
    index = run_slots(rows, 7, 5)
    plan = ops.adapter_plan(index, 7)
    wide = torch.randn(rows, columns + 64, device="cuda").bfloat16()
    view = wide[:, 8:columns + 8]
    view.copy_(y)
    around = wide.clone()
    ops.adapter_add(view, torch.cat([x, x], 1)[:, 264:], down, up, scale, plan, out=view)
    check(view, y, x, down, up, scale, index)
    around[:, 8:columns + 8] = view
    assert torch.equal(around, wide)
    one = y[:1].expand(rows, -1)  # one row of y for all
    check(ops.adapter_add(one, x, down, up, scale, plan), one, x, down, up, scale, index)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rank", [16, 64])
def test_long_prompts_keep_non_finite_rows_alone(rank, in_place):
    from actune_b200 import ops
    rows = 4864
    y, x, down, up, scale = operands(rows, 128, 2048, 16, rank, torch.bfloat16, 9)
    index = run_slots(rows, 16, 4)
    plan = ops.adapter_plan(index, 16)
    clean = ops.adapter_add(y, x, down, up, scale, plan)
    x[5], y[700, 9], x[2000, 3], down[3] = float("nan"), float("inf"), float("inf"), float("nan")
    index[[5, 2000]] = 1
    index[700] = -1
    plan.update(index)
    out = y.clone()
    out = ops.adapter_add(out if in_place else y, x, down, up, scale, plan, out=out if in_place else None)
    assert out[5].isnan().all() and torch.equal(out[700], y[700]) and not out[2000].isfinite().any()
    assert out[index == 3].isnan().all()
    keep = (index != 3)
    keep[[5, 700, 2000]] = False
    assert torch.equal(out[keep], clean[keep])


def test_long_prompts_of_large_and_small_magnitudes_in_fp16():
    from actune_b200 import ops
    for factor in (2.0 ** 9, 2.0 ** -12):
        for rank, n in ((16, 21000), (64, 328)):
            y, x, down, up, scale = operands(200, 512, n, 2, rank, torch.float16, 6)
            x, up = (x * factor).half(), (up / (factor * 16)).half()
            down = (down * 64).half() if factor > 1 else down
            index = run_slots(200, 2, 6)
            plan = ops.adapter_plan(index, 2)
            assert plan.tile == 128
            check(ops.adapter_add(y, x, down, up, scale, plan), y, x, down, up, scale, index)
