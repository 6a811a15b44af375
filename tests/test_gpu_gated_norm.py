"""gated_norm on the GPU against its formula in 64 bits.

Tolerance, per element: the one rounding of the output type, and 64 roundings of
2^-24 (sums of up to 8192 squares over a tree of threads, the reciprocal square root,
the products) of the magnitudes that enter it -- for h through the norm of
s = alpha r + gate u, whose terms may cancel, so the bound takes |alpha r| + |gate u|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
FP32 = 64 * 2.0 ** -24


def operands(rows, width, dtype, seed, *, post="width", gate="width", pre="width", shift=None, groups=1):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) + mean).to(dtype)

    def mod(kind, mean):
        return None if kind is None else rand(width, mean=mean) if kind == "width" else rand(groups, width, mean=mean)

    x, residual = rand(rows, width), rand(rows, width)
    residual[:, ::53] *= 20
    return x, residual, dict(post_weight=mod(post, 1.0), gate=mod(gate, 0.0), pre_weight=mod(pre, 1.0),
                             shift=mod(shift, 0.0))


def expected(x, residual, m, scale, eps, gemma):
    """(h, s, tolerance of h, tolerance of s) in 64 bits, without the output rounding."""
    rows = x.shape[0]

    def wide(t):
        t = t.double()
        return t if t.dim() == 1 else t.repeat_interleave(rows // t.shape[0], 0)

    def inverse(a):
        return 1 / (a.square().mean(-1, keepdim=True) + eps).sqrt()

    u = x.double()
    if m["post_weight"] is not None:
        u = u * inverse(u) * (wide(m["post_weight"]) + (1 if gemma else 0))
    if m["gate"] is not None:
        u = u * wide(m["gate"])
    r = scale * residual.double()
    s = r + u
    w = wide(m["pre_weight"]) + (1 if gemma else 0)
    shift = 0 if m["shift"] is None else wide(m["shift"])
    parts = r.abs() + u.abs()
    return s * inverse(s) * w + shift, s, FP32 * (parts * inverse(s) * w.abs() + abs(shift)), FP32 * parts


def check(got, ref, tol, dtype, what):
    bad = (got.double() - ref).abs() > UNIT[dtype] * ref.abs() + tol * (1 + UNIT[dtype]) + TINY[dtype]
    assert not bad.any(), f"{what}: {int(bad.sum())} values out of tolerance"


def run_and_check(x, residual, m, scale=1.0, eps=1e-6, gemma=False):
    from actune_b200 import ops
    m = dict(m)
    pre = m["pre_weight"]
    h, s = ops.gated_norm(x, residual, pre, post_weight=m["post_weight"], gate=m["gate"], shift=m["shift"],
                          residual_scale=scale, eps=eps, gemma=gemma)
    ref_h, ref_s, tol_h, tol_s = expected(x, residual, m, scale, eps, gemma)
    check(s, ref_s, tol_s, x.dtype, "residual")
    check(h, ref_h, tol_h, x.dtype, "norm")
    return h, s


# Widths around the kernel's row splits (8 values a thread; 32, 128 or 512 threads a row;
# the scalar form beyond 16384 and for widths that are no multiple of 8), and row counts on
# both sides of the many-rows rule.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 8), (1, 4096), (3, 1), (5, 7), (2, 264), (9, 1023), (4, 1024), (7, 2056),
                                        (3, 4104), (2, 8200), (1, 16384), (2, 16392), (1300, 64), (1301, 512),
                                        (1217, 1000), (1200, 2048), (1190, 2050)])
def test_matches_the_formula(rows, width, dtype):
    x, residual, m = operands(rows, width, dtype, rows * 7 + width)
    run_and_check(x, residual, m, scale=0.7)


# Enough rows for the kernel that streams them (16 per SM).
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width", [(2400, 520), (2501, 1000), (2600, 2048), (2387, 2056), (3001, 4096),
                                        (2400, 8192), (2400, 264), (5000, 776)])
def test_many_rows(rows, width, dtype):
    x, residual, m = operands(rows, width, dtype, rows + width)
    run_and_check(x, residual, m, scale=0.7)


@pytest.mark.parametrize("width", [640, 1536, 4096])
@pytest.mark.parametrize("post,gate,shift,groups", [(None, "group", "group", 1250), ("group", None, None, 5),
                                                    ("width", "group", "group", 2500), (None, None, "group", 100)])
def test_many_rows_with_modulations(width, post, gate, shift, groups):
    from actune_b200 import ops
    x, residual, m = operands(2500, width, torch.bfloat16, groups, post=post, gate=gate, shift=shift, pre="group",
                              groups=groups)
    wide = torch.cat([x, residual], 1)
    h, _ = run_and_check(wide[:, :width], wide[:, width:], m, gemma=True)
    got = ops.gated_norm(wide[:, :width], wide[:, width:], m["pre_weight"], post_weight=m["post_weight"],
                         gate=m["gate"], shift=m["shift"], gemma=True, quant_bits=4)
    want, scales = ops.quantize_group64(h, 4)
    assert torch.equal(got[0], h) and torch.equal(got[2], want) and torch.equal(got[3], scales)


@pytest.mark.parametrize("gemma", [False, True])
@pytest.mark.parametrize("post", [None, "width", "group"])
@pytest.mark.parametrize("gate", [None, "width", "group"])
@pytest.mark.parametrize("shift", [None, "group"])
def test_modulations_per_group(gemma, post, gate, shift):
    for rows, groups, width in ((30, 5, 192), (6, 6, 200), (1240, 40, 129), (1240, 1, 256)):
        x, residual, m = operands(rows, width, torch.bfloat16, 3 + groups, post=post, gate=gate, shift=shift,
                                  pre="group", groups=groups)
        run_and_check(x, residual, m, scale=1.3, gemma=gemma)


def test_strided_and_unaligned_rows():
    for width, pitch, offset in ((256, 520, 8), (256, 521, 0), (256, 520, 3), (320, 640, 320)):
        base = torch.randn(12, pitch + 16, device="cuda").bfloat16()
        x = base[:, offset:offset + width]
        _, residual, m = operands(12, width, torch.bfloat16, 5)
        wide = torch.cat([residual, residual], 1)
        h, s = run_and_check(x, wide[:, width:], m)
        assert h.is_contiguous() and s.is_contiguous()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bits,codes8", [(2, False), (2, True), (4, False), (4, True), (8, False)])
def test_codes_are_those_of_the_returned_norm(bits, codes8, dtype):
    """Bit for bit what quantize_group64 gives for h, on every row split and on the scalar form."""
    from actune_b200 import ops
    for rows, width, offset in ((1, 64, 0), (5, 1088, 0), (3, 4160, 0), (2, 8256, 0), (1250, 128, 0), (1210, 2048, 0),
                                (1200, 320, 0), (4, 128, 1)):
        x, residual, m = operands(rows, width + 8, dtype, rows + width)
        x, residual = x[:, offset:offset + width], residual[:, :width]
        m = {k: None if v is None else v[:width].contiguous() for k, v in m.items()}
        h, s, packed, scales = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"],
                                              gate=m["gate"], quant_bits=bits, codes8=codes8)
        plain, plain_s = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"], gate=m["gate"])
        want, want_scales = ops.quantize_group64(h, bits, codes8=codes8)
        assert torch.equal(h, plain) and torch.equal(s, plain_s)
        assert torch.equal(packed, want) and torch.equal(scales, want_scales), (rows, width)


def test_zero_rows_and_zero_values():
    from actune_b200 import ops
    x, residual, m = operands(4, 256, torch.bfloat16, 9)
    h, s = ops.gated_norm(x[:0], residual[:0], m["pre_weight"], gate=m["gate"])
    assert h.shape == s.shape == (0, 256)
    zeros = torch.zeros_like(x)
    h, s = ops.gated_norm(zeros, zeros, m["pre_weight"], post_weight=m["post_weight"])
    assert not h.any() and not s.any()
    h, _ = run_and_check(x * 0, residual, m, eps=0.0 + 1e-30)
    assert torch.isfinite(h).all()


def test_a_row_of_nan_stays_alone():
    x, residual, m = operands(1300, 256, torch.bfloat16, 11)
    from actune_b200 import ops
    clean, _ = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"])
    x[7] = float("nan")
    x[9, 0] = float("inf")
    dirty, _ = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"])
    keep = [i for i in range(1300) if i not in (7, 9)]
    assert torch.equal(clean[keep], dirty[keep]) and dirty[7].isnan().all()


def test_runs_on_the_current_stream_and_in_a_graph():
    from actune_b200 import ops
    x, residual, m = operands(48, 1024, torch.bfloat16, 13)
    want = ops.gated_norm(x, residual, m["pre_weight"], gate=m["gate"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        x2 = x * 1.0
        got = ops.gated_norm(x2, residual, m["pre_weight"], gate=m["gate"])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    static = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        out = ops.gated_norm(static, residual, m["pre_weight"], gate=m["gate"])
    static.copy_(x)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


# From 16 rows per SM on (2368 on 148 SMs) short rows take a warp each, long 16-bit ones
# the kernel that streams them; the cases above of up to 1301 rows are below that.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bits,codes8", [(2, False), (2, True), (4, False), (4, True), (8, False)])
def test_codes_of_many_rows(bits, codes8, dtype):
    from actune_b200 import ops
    for rows, width, groups in ((2400, 64, 1), (2500, 128, 5), (2400, 512, 2400), (2401, 576, 7), (2400, 1024, 16),
                                (2600, 1088, 1), (2400, 2048, 100), (2400, 4096, 3), (2369, 8192, 1)):
        x, residual, m = operands(rows, width, dtype, rows + width, gate="group", shift="group", groups=groups)
        h, s, packed, scales = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"],
                                              gate=m["gate"], shift=m["shift"], quant_bits=bits, codes8=codes8)
        plain, plain_s = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"], gate=m["gate"],
                                        shift=m["shift"])
        want, want_scales = ops.quantize_group64(h, bits, codes8=codes8)
        assert torch.equal(h, plain) and torch.equal(s, plain_s)
        assert torch.equal(packed, want) and torch.equal(scales, want_scales), (rows, width)
        ref_h, ref_s, tol_h, tol_s = expected(x, residual, m, 1.0, 1e-6, False)
        check(s, ref_s, tol_s, dtype, "residual")
        check(h, ref_h, tol_h, dtype, "norm")


@pytest.mark.parametrize("gemma", [False, True])
@pytest.mark.parametrize("post", [None, "width", "group"])
@pytest.mark.parametrize("gate", [None, "width", "group"])
@pytest.mark.parametrize("shift", [None, "group"])
def test_modulations_of_many_rows(gemma, post, gate, shift):
    for rows, groups, width, dtype in ((2480, 40, 129, torch.bfloat16), (2480, 1, 256, torch.bfloat16),
                                       (2480, 62, 1024, torch.bfloat16), (2480, 2480, 2056, torch.float16),
                                       (2480, 10, 640, torch.float32), (2480, 5, 4096, torch.float32)):
        x, residual, m = operands(rows, width, dtype, 3 + groups, post=post, gate=gate, shift=shift, pre="group",
                                  groups=groups)
        run_and_check(x, residual, m, scale=1.3, gemma=gemma)


@pytest.mark.parametrize("width", [256, 512, 1024, 2048, 4096])
def test_a_row_of_nan_stays_alone_among_many(width):
    from actune_b200 import ops
    x, residual, m = operands(2600, width, torch.bfloat16, 11)
    clean, clean_s = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"])
    x[7], x[9, 0], residual[1500, width - 1] = float("nan"), float("inf"), float("nan")
    dirty, dirty_s = ops.gated_norm(x, residual, m["pre_weight"], post_weight=m["post_weight"])
    keep = [i for i in range(2600) if i not in (7, 9, 1500)]
    assert torch.equal(clean[keep], dirty[keep]) and torch.equal(clean_s[keep], dirty_s[keep])
    assert dirty[7].isnan().all() and dirty[1500].isnan().all() and dirty_s[1500, 0].isfinite()
