"""The int8 activation operators against their plain 64-bit forms: every type, one token to many, odd widths, tensors off
the 16-byte grid and out of order, rows that are empty, zero, not finite or at the ends of the type's range; then the
layers made of them, their gradients, their runs with the optimizers, in graphs and on other streams."""

import copy

import pytest
import torch
from torch import nn

import int8_ref as R
import optimi_amd as optimi

pytestmark = pytest.mark.gpu


def rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen, dtype=torch.float64) * scale
    if len(shape) > 1 and x.numel():
        x *= torch.exp(torch.randn(shape[:-1] + (1,), generator=gen, dtype=torch.float64))
    return x.to(dtype)


def misaligned(t, device):
    """The same values one element behind an aligned address."""
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device=device)
    view = room[1:].view(t.shape)
    view.copy_(t)
    return view


# ---------------------------------------------------------------------------------- quantize

WIDTHS = [0, 1, 2, 7, 8, 9, 63, 64, 65, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 4095, 4096, 5504, 6144, 8192, 11008, 12289, 16384, 16385, 20003]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("cols", WIDTHS)
def test_quantize_and_back(hip_device, cols, dtype):
    x = rand((5, cols), dtype, cols)
    values, scales = optimi.int8_quantize(x.to(hip_device))
    q, s = R.quantize(x)
    assert values.dtype == torch.int8 and scales.dtype == torch.float32
    assert torch.equal(scales.cpu().double(), s)
    assert torch.equal(values.cpu().double(), q)
    for out in R.DTYPES:
        back = optimi.int8_dequantize(values, scales, out)
        assert back.dtype == out and torch.equal(back.cpu(), (q * s[:, None]).to(out))
    assert bool(((q * s[:, None] - x.double()).abs() <= s[:, None] / 2).all())


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("rows", [0, 1, 3, 4, 5, 257])
@pytest.mark.parametrize("cols", [3, 300, 1500])
def test_quantize_rows_and_alignment(hip_device, rows, cols, dtype):
    x = rand((rows, cols), dtype, rows + cols)
    q, s = R.quantize(x)
    for view in (misaligned(x, hip_device), x.to(hip_device).t().contiguous().t(), torch.stack([x, x], 1).to(hip_device)[:, 1]):
        values, scales = optimi.int8_quantize(view)
        assert torch.equal(values.cpu().double(), q) and torch.equal(scales.cpu().double(), s)
    back = optimi.int8_dequantize(misaligned(values, hip_device), scales, dtype)
    assert torch.equal(back.cpu(), (q * s[:, None]).to(dtype))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
def test_quantize_at_the_ends_of_the_range(hip_device, dtype):
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps
    rows = [[0.0] * 6, [-0.0] * 6, [info.max] * 6, [-info.max, info.max / 2, 1.0, 0.0, tiny, -tiny], [tiny] * 6, [info.smallest_normal] * 6,
            [float("inf"), 1, 2, 3, 4, 5], [1, float("-inf"), 2, 3, 4, 5], [1, 2, float("nan"), 3, 4, 5], [float("nan"), float("inf")] * 3]
    # the largest value just at, below and above 127 steps, ties to both sides
    for e in (-4, 0, 3):
        rows += [[127 * 2.0**e, 0.5 * 2.0**e, 1.5 * 2.0**e, 2.5 * 2.0**e, -0.5 * 2.0**e, -1.5 * 2.0**e], [126.5 * 2.0**e] * 6, [127.5 * 2.0**e] * 6, [128 * 2.0**e] * 6]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    values, scales = optimi.int8_quantize(x.to(hip_device))
    q, s = R.quantize(x)
    assert torch.equal(torch.nan_to_num(scales.cpu().double(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
    assert torch.equal(values.cpu().double(), q)
    back = optimi.int8_dequantize(values, scales, dtype).cpu()
    fine = torch.isfinite(x.double()).all(1)
    assert bool(torch.isfinite(back[fine].double()).all()), "a finite activation came back infinite"
    assert bool(torch.isnan(back[~fine].double()).all())


# ---------------------------------------------------------------------------------- matmul

SHAPES = [(1, 1, 1), (1, 16, 64), (1, 4096, 1024), (1, 77, 333), (2, 100, 129), (5, 33, 17), (15, 64, 256), (16, 65, 255), (17, 64, 256), (31, 130, 1000),
          (33, 200, 4096), (63, 255, 640), (64, 256, 128), (65, 257, 129), (127, 128, 127), (128, 512, 384), (129, 300, 70), (255, 256, 2048), (256, 256, 256),
          (257, 513, 1025), (300, 1000, 272), (512, 768, 1040), (700, 40, 3000), (1030, 770, 528), (40, 700, 16), (200, 300, 0), (3, 300, 0), (0, 5, 7), (5, 0, 7), (300, 300, 11008)]


def int8_inputs(m, n, k, seed, pow2=True):
    gen = torch.Generator().manual_seed(seed)
    a = torch.randint(-127, 128, (m, k), generator=gen, dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=gen, dtype=torch.int8)
    sa, sb = torch.rand(m, generator=gen) * 0.02 + 1e-3, torch.rand(n, generator=gen) * 1e-3 + 1e-4
    if pow2:
        sa, sb = torch.exp2(torch.round(torch.log2(sa))), torch.exp2(torch.round(torch.log2(sb)))
    return a, sa, b, sb


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_matmul(hip_device, shape, dtype):
    m, n, k = shape
    for bias, pow2 in ((None, True), (rand((n,), dtype, 5), False)):
        a, sa, b, sb = int8_inputs(m, n, k, m + n + k, pow2)
        y = optimi.int8_matmul(a.to(hip_device), sa.to(hip_device), b.to(hip_device), sb.to(hip_device),
                               bias=None if bias is None else bias.to(hip_device), dtype=dtype)
        want, allowed = R.matmul(a, sa, b, sb, bias, dtype)
        assert y.dtype == dtype
        R.close(y, want, allowed, f"{shape} bias={bias is not None}")


# products of so many tiles that the largest ones are used: even and odd widths, sums that end inside a step, one step alone
LARGE = [(2900, 2830, 272), (2817, 3000, 1111), (3000, 2900, 100), (5000, 1700, 128), (2600, 3400, 1), (4096, 4097, 640)]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", LARGE, ids=lambda s: "x".join(map(str, s)))
def test_large_matmul(hip_device, shape, dtype):
    m, n, k = shape
    a, sa, b, sb = (t.to(hip_device) for t in int8_inputs(m, n, k, 11, False))
    bias = rand((n,), dtype, 5).to(hip_device)
    y = optimi.int8_matmul(a, sa, b, sb, bias=bias, dtype=dtype)
    want, allowed = R.matmul(a, sa, b, sb, bias, dtype)
    R.close(y, want.cpu(), allowed.cpu(), str(shape))
    if k > 1:
        y = optimi.int8_matmul(misaligned(a, hip_device), sa, misaligned(b, hip_device), sb, bias=bias, dtype=dtype)
        R.close(y, want.cpu(), allowed.cpu(), f"{shape} off the grid")


@pytest.mark.parametrize("shape", [(1, 40, 512), (20, 70, 96), (130, 300, 256), (300, 260, 1024)], ids=lambda s: "x".join(map(str, s)))
def test_matmul_takes_views_and_any_alignment(hip_device, shape):
    m, n, k = shape
    a, sa, b, sb = int8_inputs(m, n, k, 3)
    want, allowed = R.matmul(a, sa, b, sb, None, torch.float32)
    dev = [t.to(hip_device) for t in (a, sa, b, sb)]
    for args in ([misaligned(a, hip_device), dev[1], misaligned(b, hip_device), dev[3]],
                 [dev[0].t().contiguous().t(), misaligned(sa, hip_device), torch.stack([b, b], 1).to(hip_device)[:, 0], torch.stack([sb, sb], 1).to(hip_device)[:, 0]]):
        R.close(optimi.int8_matmul(*args, dtype=torch.float32), want, allowed, str(shape))
    y = optimi.int8_matmul(dev[0].view(1, m, 1, k), dev[1].view(1, m, 1), dev[2], dev[3], dtype=torch.float32)
    assert y.shape == (1, m, 1, n)
    R.close(y.view(m, n), want, allowed, str(shape))


def test_matmul_is_exact_at_the_largest_sums(hip_device):
    """-128 times -128 in every place of the longest allowed sum is the largest whole number there can be."""
    k = 131071
    for m in (1, 40, 260):
        a = torch.full((m, k), -128, dtype=torch.int8, device=hip_device)
        b = torch.full((3, k), -128, dtype=torch.int8, device=hip_device)
        y = optimi.int8_matmul(a, torch.ones(m, device=hip_device), b, torch.tensor([1.0, 0.5, 2.0], device=hip_device), dtype=torch.float32)
        assert torch.equal(y.cpu(), torch.tensor([[2147467264.0, 1073733632.0, 4294934528.0]]).expand(m, 3))


def test_matmul_keeps_bad_rows_to_themselves(hip_device):
    m, n, k = 70, 300, 200
    a, sa, b, sb = int8_inputs(m, n, k, 9)
    sa[3], sb[7], sb[9] = float("nan"), float("inf"), 0.0
    y = optimi.int8_matmul(a.to(hip_device), sa.to(hip_device), b.to(hip_device), sb.to(hip_device), dtype=torch.bfloat16).cpu()
    assert bool(torch.isnan(y[3]).all()) and bool((y[:3, 9] == 0).all())
    rest = torch.ones(m, n, dtype=torch.bool)
    rest[3] = False
    rest[:, 7] = False
    assert bool(torch.isfinite(y[rest].double()).all())


# ---------------------------------------------------------------------------------- weight gradient

GRADS = [(1, 1, 1), (1, 300, 70), (2, 64, 64), (7, 65, 33), (31, 100, 200), (32, 64, 128), (33, 128, 64), (63, 255, 257), (64, 256, 256), (65, 257, 255), (127, 300, 513),
         (128, 256, 512), (200, 1000, 16), (257, 17, 1000), (512, 512, 256), (1000, 264, 520), (2000, 260, 300), (4096, 128, 128), (0, 40, 50), (5, 0, 7), (5, 7, 0)]


def checkpoint(rows, cols, seed, pow2=True):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (rows, cols), generator=gen, dtype=torch.int8)
    s = torch.exp2(torch.randint(-9, -3, (rows,), generator=gen).float())
    return q, s if pow2 else s * (1 + torch.rand(rows, generator=gen))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", GRADS, ids=lambda s: "x".join(map(str, s)))
def test_weight_grad(hip_device, shape, dtype):
    rows, outs, cols = shape
    g = rand((rows, outs), dtype, rows + outs, 1e-2)
    for pow2 in (True, False):
        q, s = checkpoint(rows, cols, sum(shape), pow2)
        dw, db = optimi.int8_weight_grad(g.to(hip_device), q.to(hip_device), s.to(hip_device), bias=True)
        R.close(dw, *R.weight_grad(g, q, s, dtype), f"weight {shape} pow2={pow2}")
        R.close(db, *R.column_sum(g, dtype), f"bias {shape}")
        alone = optimi.int8_weight_grad(g.to(hip_device), q.to(hip_device), s.to(hip_device))
        assert alone.dtype == dtype and torch.equal(alone, dw), "the same bits on every run"


LARGE_GRADS = [(1, 3000, 2900), (64, 2904, 2831), (65, 3000, 2800), (129, 2817, 3000), (200, 2896, 2817), (257, 5000, 1700), (1000, 33000, 16), (70, 33000, 3), (500, 16, 33001), (5, 7, 50000)]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", LARGE_GRADS, ids=lambda s: "x".join(map(str, s)))
def test_large_weight_grad(hip_device, shape, dtype):
    rows, outs, cols = shape
    g = rand((rows, outs), dtype, 3, 1e-2).to(hip_device)
    q, s = (t.to(hip_device) for t in checkpoint(rows, cols, 4))
    want, allowed = R.weight_grad(g, q, s, dtype)
    R.close(optimi.int8_weight_grad(g, q, s), want.cpu(), allowed.cpu(), str(shape))
    R.close(optimi.int8_weight_grad(misaligned(g, hip_device), misaligned(q, hip_device), s), want.cpu(), allowed.cpu(), f"{shape} off the grid")


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", [(65, 3000, 2800), (130, 2904, 2831)], ids=lambda s: "x".join(map(str, s)))
def test_large_weight_grad_of_gradients_that_are_not_finite(hip_device, shape, dtype):
    rows, outs, cols = shape
    g = rand((rows, outs), dtype, 4, 1e-2).to(hip_device)
    q, s = (t.to(hip_device) for t in checkpoint(rows, cols, 5))
    q[q == 0] = 1
    g[rows - 1, 5], g[0, 9], g[rows // 2, outs - 1] = float("inf"), float("-inf"), float("nan")
    for _ in range(2):  # the second time LDS holds the first's infinities
        got, want = optimi.int8_weight_grad(g, q, s).double(), R.weight_grad(g, q, s, dtype)[0]
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        inf = torch.isinf(want)
        assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf])


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", [(40, 64, 96), (130, 300, 264), (600, 256, 512)], ids=lambda s: "x".join(map(str, s)))
def test_weight_grad_takes_views_and_any_alignment(hip_device, shape, dtype):
    rows, outs, cols = shape
    g = rand((rows, outs), dtype, 1, 1e-2)
    q, s = checkpoint(rows, cols, 2)
    want = R.weight_grad(g, q, s, dtype)
    for args in ((misaligned(g, hip_device), misaligned(q, hip_device), misaligned(s, hip_device)),
                 (g.to(hip_device).t().contiguous().t(), torch.stack([q, q], 1).to(hip_device)[:, 1], s.to(hip_device))):
        R.close(optimi.int8_weight_grad(*args), *want, str(shape))
    dw = optimi.int8_weight_grad(g.to(hip_device).view(2, rows // 2, outs), q.to(hip_device).view(2, rows // 2, cols), s.to(hip_device).view(2, rows // 2))
    R.close(dw, *want, str(shape))
    same = g[:1].expand(rows, outs)  # what sum().backward() hands over
    R.close(optimi.int8_weight_grad(g[:1].to(hip_device).expand(rows, outs), q.to(hip_device), s.to(hip_device)), *R.weight_grad(same, q, s, dtype), "expanded")


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("rows", [3, 70, 300])
def test_weight_grad_of_gradients_that_are_not_finite(hip_device, rows, dtype):
    """Infinities and NaN reach their own outputs and no others; a row whose scale is NaN reaches all."""
    outs, cols = 300, 270
    g = rand((rows, outs), dtype, 4, 1e-2)
    q, s = checkpoint(rows, cols, 5)
    q[q == 0] = 1
    g[rows - 1, 5], g[0, 9], g[rows // 2, 11] = float("inf"), float("-inf"), float("nan")
    dw, db = (t.cpu().double() for t in optimi.int8_weight_grad(g.to(hip_device), q.to(hip_device), s.to(hip_device), bias=True))
    want, wb = R.weight_grad(g, q, s, dtype)[0], R.column_sum(g, dtype)[0]
    for got, ref in ((dw, want), (db, wb)):
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        inf = torch.isinf(ref)
        assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], ref[inf])
    s[rows - 1] = float("nan")
    assert bool(torch.isnan(optimi.int8_weight_grad(g.to(hip_device), q.to(hip_device), s.to(hip_device))).all())


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
def test_weight_grad_of_gradients_over_the_whole_range(hip_device, dtype):
    """Small gradients are not lost beside large ones: every output has gradients of one size, subnormal ones in fp16."""
    rows, outs, cols = 96, 64, 40
    low, high = {torch.float16: (-24, 10), torch.bfloat16: (-100, 100), torch.float32: (-100, 90)}[dtype]
    size = torch.exp2(torch.linspace(low, high, outs).round())
    g = (torch.randint(1, 4, (rows, outs), generator=torch.Generator().manual_seed(6)) * size).to(dtype)
    q, s = checkpoint(rows, cols, 7)
    s = torch.ones_like(s) if dtype == torch.float16 else s
    q = q.abs() // 8 if dtype == torch.float16 else q  # sums within fp16
    q, s = q.to(torch.int8), s
    if dtype == torch.float16:
        g = torch.where(g.double() > 1, g.double() / 64, g.double()).to(dtype)
    R.close(optimi.int8_weight_grad(g.to(hip_device), q.to(hip_device), s.to(hip_device)), *R.weight_grad(g, q, s, dtype), "range")


# ---------------------------------------------------------------------------------- the norm

NORM_WIDTHS = [1, 2, 7, 8, 9, 64, 300, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096, 5504, 8192, 11008, 16384, 16385, 18001]


@pytest.mark.parametrize("weight32", [False, True], ids=["weight_own", "weight_fp32"])
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("cols", NORM_WIDTHS)
def test_norm_forward(hip_device, cols, dtype, weight32):
    rows, eps = 6, 1e-5
    x, r = rand((rows, cols), dtype, cols), rand((rows, cols), dtype, cols + 1)
    x[2], r[2] = 0, 0  # a row of padding
    w = (1 + 0.2 * rand((cols,), torch.float64, 3)).to(torch.float32 if weight32 else dtype)
    for residual in (None, r):
        h = x if residual is None else (x.double() + residual.double()).to(dtype)
        d = x.to(hip_device)
        values, scales, hh, rstd = optimi.add_rms_norm_int8(d, w.to(hip_device), residual=None if residual is None else residual.to(hip_device), eps=eps)
        assert hh is d if residual is None else torch.equal(hh.cpu(), h)
        y, rr, rel_r, rel_y = R.norm(h, w, eps)
        R.close(rstd, rr, rel_r * rr, "rstd")
        q, s = values.cpu().double(), scales.cpu().double()
        absmax = y.abs().amax(1)
        want_s = R.step_of(absmax, 3e38)[0]
        near = (absmax / (127 * want_s) > 1 - 2 * rel_y) | (absmax / (63.5 * want_s) < 1 + 2 * rel_y)
        assert bool(((s == want_s) | (near & ((s == 2 * want_s) | (s == want_s / 2)))).all())
        assert bool((q.abs() <= 127).all())
        R.close(q * s[:, None], y, s[:, None] / 2 + rel_y * y.abs(), "y")
        assert bool((q[2] == 0).all()) and float(s[2]) == 1.0


@pytest.mark.parametrize("rows", [0, 1, 4, 5, 260])
@pytest.mark.parametrize("cols", [24, 1500])
def test_norm_rows_views_and_dimensions(hip_device, rows, cols):
    x, r = rand((rows, cols), torch.bfloat16, 1), rand((rows, cols), torch.bfloat16, 2)
    w = rand((cols,), torch.bfloat16, 3)
    first = optimi.add_rms_norm_int8(x.to(hip_device), w.to(hip_device), residual=r.to(hip_device))
    other = optimi.add_rms_norm_int8(misaligned(x, hip_device), misaligned(w, hip_device), residual=r.to(hip_device).t().contiguous().t())
    lead = optimi.add_rms_norm_int8(x.to(hip_device)[None, :, None], w.to(hip_device), residual=r.to(hip_device)[None, :, None])
    assert lead[0].shape == (1, rows, 1, cols) and lead[1].shape == (1, rows, 1) and lead[2].shape == (1, rows, 1, cols)
    for a, b, c in zip(first, other, lead):
        assert torch.equal(a, b) and torch.equal(a, c.reshape(a.shape))


def test_norm_marks_rows_that_are_not_finite(hip_device):
    x = rand((6, 500), torch.bfloat16, 1)
    x[1, 3], x[4, 7] = float("inf"), float("nan")
    values, scales, h, rstd = optimi.add_rms_norm_int8(x.to(hip_device), torch.ones(500, dtype=torch.bfloat16, device=hip_device))
    bad = torch.tensor([False, True, False, False, True, False])
    assert torch.equal(torch.isnan(scales.cpu()), bad)
    assert bool((values[bad.to(hip_device)] == 0).all())


@pytest.mark.parametrize("weight32", [False, True], ids=["weight_own", "weight_fp32"])
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("cols", NORM_WIDTHS)
def test_norm_backward(hip_device, cols, dtype, weight32):
    for rows in (1, 9, 70):
        h, g, gh = rand((rows, cols), dtype, 1), rand((rows, cols), dtype, 2, 1e-2), rand((rows, cols), dtype, 3, 1e-2)
        w = (1 + 0.2 * rand((cols,), torch.float64, 4)).to(torch.float32 if weight32 else dtype)
        rstd = R.norm(h, w, 1e-6)[1].float()
        for more in (None, gh):
            dx, dw = optimi.add_rms_norm_int8_backward(g.to(hip_device), h.to(hip_device), rstd.to(hip_device), w.to(hip_device),
                                                       grad_h=None if more is None else more.to(hip_device))
            want_dx, allow_dx, want_dw, allow_dw = R.norm_backward(g, h, rstd, w, more, dtype, w.dtype)
            R.close(dx, want_dx, allow_dx, f"dx {rows}")
            R.close(dw, want_dw, allow_dw, f"dweight {rows}")


@pytest.mark.parametrize("rows,cols", [(0, 40), (3000, 40), (5000, 130), (2100, 1100), (700, 17000)])
def test_norm_backward_of_many_rows(hip_device, rows, cols):
    dtype = torch.bfloat16
    h, g = rand((rows, cols), dtype, 1), rand((rows, cols), dtype, 2, 1e-2)
    w = rand((cols,), dtype, 4)
    rstd = R.norm(h, w, 1e-6)[1].float()
    args = (misaligned(g, hip_device), misaligned(h, hip_device), rstd.to(hip_device), w.to(hip_device))
    dx, dw = optimi.add_rms_norm_int8_backward(*args)
    want_dx, allow_dx, want_dw, allow_dw = R.norm_backward(g, h, rstd, w, None, dtype, dtype)
    R.close(dx, want_dx, allow_dx, "dx")
    R.close(dw, want_dw, allow_dw, "dweight")
    again = optimi.add_rms_norm_int8_backward(*args)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw), "the same bits on every run"


def test_norm_gradient_against_differences(hip_device):
    rows, cols, eps = 4, 37, 1e-5
    x, w = rand((rows, cols), torch.float32, 1), 1 + 0.3 * rand((cols,), torch.float32, 2)
    g, gh = rand((rows, cols), torch.float32, 3), rand((rows, cols), torch.float32, 4)

    def loss(x, w):
        return float((R.norm(x, w, eps)[0] * g.double()).sum() + (x.double() * gh.double()).sum())

    rstd = R.norm(x, w, eps)[1].float()
    dx, dw = optimi.add_rms_norm_int8_backward(*(t.to(hip_device) for t in (g, x, rstd, w)), grad_h=gh.to(hip_device))
    step = 1e-5
    for wrt, grad in ((x, dx.cpu().double()), (w, dw.cpu().double())):
        other = wrt.double()
        for i in range(0, wrt.numel(), 5):
            ends = []
            for sign in (1, -1):
                moved = other.clone()
                moved.view(-1)[i] += sign * step
                ends.append(loss(moved, w) if wrt is x else loss(x, moved))
            # step^2 times a third derivative of order 10, cancellation of two sums of order 1e3, float32 results
            assert abs((ends[0] - ends[1]) / (2 * step) - float(grad.view(-1)[i])) < 1e-6 * (1 + float(grad.abs().max()))


# ---------------------------------------------------------------------------------- layers

def restored(t):
    q, s = R.quantize(t)
    return q * s[..., None]


@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", [(1, 16, 40), (6, 48, 130), (70, 300, 264)], ids=lambda s: "x".join(map(str, s)))
def test_linear_and_its_gradients(hip_device, shape, dtype, bias):
    m, n, k = shape
    x, w, b, g = rand((2, m, k), dtype, 1), rand((n, k), dtype, 2, k**-0.5), rand((n,), dtype, 3), rand((2, m, n), dtype, 4, 1e-2)
    leaves = [t.to(hip_device).requires_grad_() for t in ((x, w, b) if bias else (x, w))]
    y = optimi.int8_linear(*leaves)
    y.backward(g.to(hip_device))
    q, s = R.quantize(x.view(-1, k))
    wq, ws = R.quantize(w)
    R.close(y.view(-1, n), *R.matmul(q, s, wq, ws, b if bias else None, dtype), "y")
    g2 = g.view(-1, n)
    R.close(leaves[1].grad, *R.weight_grad(g2, q, s, dtype), "dw")
    if bias:
        R.close(leaves[2].grad, *R.column_sum(g2, dtype), "db")
    dx, mass = g2.double() @ w.double(), g2.double().abs() @ w.double().abs()
    slack = 2 * (n + 8) * R.U * mass
    R.close(leaves[0].grad.view(-1, k), dx, slack + R.half(dtype) * (dx.abs() + slack) + 1.01 * R.least(dtype), "dx")


def test_linear_of_a_single_vector_and_of_no_rows(hip_device):
    w, b = rand((40, 24), torch.float32, 1).to(hip_device).requires_grad_(), rand((40,), torch.float32, 2).to(hip_device).requires_grad_()
    x = rand((1, 24), torch.float32, 3).to(hip_device)
    flat = x[0].clone().requires_grad_()
    y = optimi.int8_linear(flat, w, b)
    assert y.shape == (40,) and torch.equal(y, optimi.int8_linear(x, w, b)[0])
    y.sum().backward()
    assert flat.grad.shape == (24,) and w.grad.shape == (40, 24) and torch.equal(b.grad, torch.ones_like(b))
    (y,), h = optimi.add_rms_norm_int8_linear(flat, torch.ones(24, device=hip_device), [w], residual=x[0])
    assert y.shape == (40,) and h.shape == (24,)
    (y.sum() + h.sum()).backward()
    w.grad = b.grad = None
    none = torch.zeros(0, 24, device=hip_device, requires_grad=True)
    optimi.int8_linear(none, w, b).sum().backward()
    assert none.grad.shape == (0, 24) and not w.grad.any() and not b.grad.any()


def test_linear_under_autocast(hip_device):
    layer = optimi.Int8Linear(64, 32).to(hip_device)
    x = torch.randn(9, 64, device=hip_device, requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x)
        (z,), h = optimi.add_rms_norm_int8_linear(x, torch.ones(64, device=hip_device), [layer.weight], [layer.bias], residual=x)
    assert y.dtype == z.dtype == h.dtype == torch.bfloat16
    want = optimi.int8_linear(x.bfloat16(), layer.weight.bfloat16(), layer.bias.bfloat16())
    assert torch.equal(y, want)
    (y.float().sum() + z.float().sum() + h.float().sum()).backward()
    assert x.grad.dtype == layer.weight.grad.dtype == layer.bias.grad.dtype == torch.float32


def test_linear_keeps_only_what_it_needs(hip_device):
    x, w = torch.randn(64, 256, device=hip_device), torch.randn(128, 256, device=hip_device)
    y = optimi.int8_linear(x.clone().requires_grad_(), w)  # a frozen weight needs no checkpoint
    assert [t for t in y.grad_fn.saved_tensors if t is not None and t.dtype == torch.int8] == []
    y.sum().backward()
    y = optimi.int8_linear(x, w.clone().requires_grad_())
    kept = [t for t in y.grad_fn.saved_tensors if t is not None and t.shape == x.shape]
    assert [t.dtype for t in kept] == [torch.int8], "the activation is kept in 8 bits and in nothing else"
    y.sum().backward()
    with torch.no_grad():
        assert torch.equal(optimi.int8_linear(x, w), y.detach())


def norm_layers(dtype, m, k, outs, seed=0):
    x, r = rand((m, k), dtype, seed + 1), rand((m, k), dtype, seed + 2)
    nw = (1 + 0.2 * rand((k,), torch.float64, seed + 3)).to(dtype)
    ws = [rand((n, k), dtype, seed + 4 + i, k**-0.5) for i, n in enumerate(outs)]
    bs = [rand((n,), dtype, seed + 9 + i) if i else None for i, n in enumerate(outs)]
    return x, r, nw, ws, bs


@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
def test_norm_linear_and_its_gradients(hip_device, dtype, residual):
    """The fused node against the same operators called one by one, bit for bit, each of which is held to its formula above."""
    m, k, outs, eps = 37, 130, (48, 64, 80), 1e-5
    x, r, nw, ws, bs = norm_layers(dtype, m, k, outs)
    leaf = lambda t: None if t is None else t.to(hip_device).requires_grad_()  # noqa: E731
    lx, lr, ln, lw, lb = leaf(x), leaf(r) if residual else None, leaf(nw), [leaf(w) for w in ws], [leaf(b) for b in bs]
    ys, h = optimi.add_rms_norm_int8_linear(lx, ln, lw, biases=lb, residual=lr, eps=eps)
    gs, gh = [rand((m, n), dtype, 30 + n, 1e-2).to(hip_device) for n in outs], rand((m, k), dtype, 40, 1e-2).to(hip_device)
    if residual:
        torch.autograd.backward([*ys, h], [*gs, gh])
    else:
        assert h is lx
        torch.autograd.backward(list(ys), gs)
    with torch.no_grad():
        values, scales, hh, rstd = optimi.add_rms_norm_int8(lx, ln, residual=lr, eps=eps)
        assert torch.equal(h, hh)
        dy = None
        for y, g, w, b in zip(ys, gs, lw, lb):
            wv, wsc = optimi.int8_quantize(w)
            assert torch.equal(y, optimi.int8_matmul(values, scales, wv, wsc, bias=b, dtype=dtype))
            dw, db = optimi.int8_weight_grad(g, values, scales, bias=True)
            assert torch.equal(w.grad, dw) and (b is None or torch.equal(b.grad, db))
            dy = g @ w if dy is None else torch.addmm(dy, g, w)
        dx, dn = optimi.add_rms_norm_int8_backward(dy, hh, rstd, ln, grad_h=gh if residual else None)
        assert torch.equal(lx.grad, dx) and torch.equal(ln.grad, dn)
        assert lr is None or torch.equal(lr.grad, dx)


def test_norm_linear_with_outputs_that_nobody_uses(hip_device):
    x, r, nw, ws, bs = norm_layers(torch.float32, 20, 64, (32, 48))
    lx, ln = x.to(hip_device).requires_grad_(), nw.to(hip_device).requires_grad_()
    lr, lw = r.to(hip_device).requires_grad_(), [w.to(hip_device).requires_grad_() for w in ws]
    (y0, y1), h = optimi.add_rms_norm_int8_linear(lx, ln, lw, residual=lr)
    y1.sum().backward(retain_graph=True)
    assert lw[0].grad is None and lw[1].grad is not None and lx.grad is not None and torch.equal(lx.grad, lr.grad)
    lx.grad = lr.grad = ln.grad = lw[1].grad = None
    h.sum().backward()
    assert ln.grad is None and torch.equal(lx.grad, torch.ones_like(lx)) and torch.equal(lr.grad, torch.ones_like(lr))
    lx.grad.add_(1)
    assert torch.equal(lr.grad, torch.ones_like(lr)), "the two gradients share no memory"


def test_norm_linear_gradient_against_differences(hip_device):
    """dx and the norm's dweight are the derivatives of the layer as if nothing had been rounded."""
    m, k, eps = 3, 24, 1e-5
    x, r, nw, ws, _ = norm_layers(torch.float32, m, k, (10,))
    g, gh = rand((m, 10), torch.float32, 50), rand((m, k), torch.float32, 51)

    def loss(x, nw):
        h = x.double() + r.double()
        return float(((R.norm(h, nw, eps)[0] @ ws[0].double().T) * g.double()).sum() + (h * gh.double()).sum())

    lx, ln = x.to(hip_device).requires_grad_(), nw.to(hip_device).requires_grad_()
    (y,), h = optimi.add_rms_norm_int8_linear(lx, ln, [ws[0].to(hip_device)], residual=r.to(hip_device), eps=eps)
    torch.autograd.backward([y, h], [g.to(hip_device), gh.to(hip_device)])
    step = 1e-5
    for wrt, grad in ((x, lx.grad.cpu().double()), (nw, ln.grad.cpu().double())):
        for i in range(0, wrt.numel(), 3):
            ends = []
            for sign in (1, -1):
                moved = wrt.double().clone()
                moved.view(-1)[i] += sign * step
                ends.append(loss(moved, nw) if wrt is x else loss(x, moved))
            # h is rounded to float32 before the norm, the rest is as in the norm's own test
            assert abs((ends[0] - ends[1]) / (2 * step) - float(grad.view(-1)[i])) < 3e-6 * (1 + float(grad.abs().max()))


# ---------------------------------------------------------------------------------- models and optimizers

class Block(nn.Module):
    """A gated MLP behind a norm on a residual stream."""

    def __init__(self, width, inner):
        super().__init__()
        self.norm = nn.RMSNorm(width, eps=1e-5)
        self.gate, self.up, self.down = nn.Linear(width, inner, bias=False), nn.Linear(width, inner, bias=False), nn.Linear(inner, width)

    def forward(self, x, residual):
        (gate, up), h = optimi.add_rms_norm_int8_linear(x, self.norm.weight, [self.gate.weight, self.up.weight], residual=residual, eps=1e-5)
        return self.down(nn.functional.silu(gate) * up), h


class Stack(nn.Module):
    def __init__(self, width=96, inner=160, depth=2):
        super().__init__()
        self.blocks = nn.ModuleList(Block(width, inner) for _ in range(depth))
        self.head = nn.Sequential(nn.RMSNorm(width), nn.Linear(width, 50))

    def forward(self, x):
        h = torch.zeros_like(x)
        for block in self.blocks:
            x, h = block(x, h)
        return self.head(x + h)


def stack(device, dtype, seed=0):
    torch.manual_seed(seed)
    return optimi.prepare_for_int8_linear(Stack().to(dtype).to(device))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
def test_a_model_trains_with_gradient_release_as_with_whole_steps(hip_device, dtype):
    """The layers' gradients through the native release hook: the same parameters, bit for bit, as step() gives."""
    batches = [rand((3, 7, 96), dtype, 60 + i).to(hip_device) for i in range(3)]
    ends = []
    for release in (False, True):
        model = stack(hip_device, dtype)
        opt = optimi.StableAdamW(model.parameters(), lr=1e-3, gradient_release=release)
        if release:
            optimi.prepare_for_gradient_release(model, opt)
        for x in batches:
            model(x).float().square().mean().backward()
            if release:
                assert all(p.grad is None for p in model.parameters())
            opt.step()
            opt.zero_grad()
        torch.cuda.synchronize()
        ends.append([p.detach().clone() for p in model.parameters()])
    before = [p.detach() for p in stack(hip_device, dtype).parameters()]
    assert all(torch.equal(a, b) for a, b in zip(*ends))
    assert all(not torch.equal(a, b) for a, b in zip(before, ends[0]))


def test_the_prepared_model_is_near_the_plain_one(hip_device):
    torch.manual_seed(0)
    plain = nn.Sequential(nn.Linear(64, 128), nn.GELU(), nn.RMSNorm(128), nn.Linear(128, 64), nn.Linear(64, 32, bias=False)).to(hip_device)
    model = copy.deepcopy(plain)
    names = [n for n, _ in model.named_parameters()]
    params = list(model.parameters())
    optimi.prepare_for_int8_linear(model, skip=("4",))
    assert type(model[0]) is optimi.Int8Linear and type(model[4]) is nn.Linear
    assert [n for n, _ in model.named_parameters()] == names and all(a is b for a, b in zip(model.parameters(), params))
    x = torch.randn(33, 64, device=hip_device)
    want, got = plain(x), model(x)
    # two layers, each with two operands at most 2^-7 of their largest value off (about 1/100 of it in the mean)
    assert float((want - got).norm() / want.norm()) < 0.05
    calls = []
    handle = model[2].register_forward_hook(lambda *a: calls.append(1))  # a hook keeps the norm a module of its own
    with_hook = model(x)
    handle.remove()
    assert calls == [1] and float((with_hook - want).norm() / want.norm()) < 0.05
    other = copy.deepcopy(model)
    assert torch.equal(other(x), got)
    optimi.remove_int8_linear(model)
    assert type(model) is nn.Sequential and torch.equal(model(x), want)
    assert torch.equal(other(x), got)


def test_the_norm_in_a_sequence_hands_over_int8(hip_device):
    for eps in (None, 1e-3):
        model = nn.Sequential(nn.RMSNorm(80, eps=eps), nn.Linear(80, 48)).to(torch.bfloat16).to(hip_device)
        optimi.prepare_for_int8_linear(model)
        x = rand((9, 80), torch.bfloat16, 1, 0.05).to(hip_device)
        e = torch.finfo(torch.float32).eps if eps is None else eps
        (want,), _ = optimi.add_rms_norm_int8_linear(x, model[0].weight, [model[1].weight], [model[1].bias], eps=e)
        assert torch.equal(model(x), want)
        # the same eps as the module's own: its result, rounded to bf16, is half a step of either rounding away
        values, scales, _, _ = optimi.add_rms_norm_int8(x, model[0].weight, eps=e)
        plain = model[0](x).double()
        assert bool(((values.double() * scales.double()[:, None] - plain).abs() <= scales.double()[:, None] / 2 + 2.1 * R.half(torch.bfloat16) * plain.abs()).all())


# ---------------------------------------------------------------------------------- graphs, streams

def operators(x, r, g, nw, w, b):
    """A run of all operators as a layer makes it."""
    values, scales, h, rstd = optimi.add_rms_norm_int8(x, nw, residual=r)
    wv, ws = optimi.int8_quantize(w)
    y = optimi.int8_matmul(values, scales, wv, ws, bias=b, dtype=x.dtype)
    dw, db = optimi.int8_weight_grad(g, values, scales, bias=True)
    dx, dn = optimi.add_rms_norm_int8_backward(optimi.int8_dequantize(values, scales, x.dtype), h, rstd, nw, grad_h=r)
    return y, dw, db, dx, dn


def inputs(device, m, n, k, dtype, seed):
    shapes = [(m, k), (m, k), (m, n), (k,), (n, k), (n,)]
    return [rand(s, dtype, seed + i).to(device) for i, s in enumerate(shapes)]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("m", [1, 5, 40, 300, 700])
def test_two_captured_runs_replayed_in_turn(hip_device, m, dtype):
    runs = []
    for seed in (1, 100):
        args = inputs(hip_device, m, 520, 1040, dtype, seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            operators(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = operators(*args)
        runs.append((args, graph, outs))
    for turn in range(4):
        for args, _, _ in runs:
            for i, t in enumerate(args):
                t.copy_(rand(tuple(t.shape), dtype, 1000 + 10 * turn + i))
        for _, graph, _ in runs:
            graph.replay()
        for args, _, outs in runs:
            eager = operators(*args)  # the program's own work between replays
            torch.cuda.synchronize()
            for a, b in zip(outs, eager):
                assert torch.equal(a, b), f"replay {turn}"


def test_a_captured_training_step(hip_device):
    """Forward and backward of the prepared model in one graph, replayed on new batches."""
    model = stack(hip_device, torch.bfloat16)
    x = rand((5, 9, 96), torch.bfloat16, 1).to(hip_device)

    def passes():
        return torch.autograd.grad((model(x).float() ** 2).mean(dim=-1).mean(dim=-1).mean(), list(model.parameters()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = passes()
    for turn in range(4):
        x.copy_(rand((5, 9, 96), torch.bfloat16, 10 + turn))
        graph.replay()
        eager = passes()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, eager)), turn


def test_on_another_stream(hip_device):
    args = inputs(hip_device, 200, 300, 512, torch.bfloat16, 7)
    want = operators(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for stream in streams:  # all at once
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            outs.append(operators(*args))
    for stream in streams:
        torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------------- the C boundary

class Guarded:
    """Device buffers with a margin of a known pattern on both sides."""

    def __init__(self, device):
        self.device, self.made = device, []

    def __call__(self, like=None, shape=None, dtype=None, offset=0):
        shape, dtype = (tuple(like.shape), like.dtype) if like is not None else (shape, dtype)
        size = torch.empty((), dtype=dtype).element_size()
        n = size
        for d in shape:
            n *= d
        room = torch.full((n + 1024 + offset * size,), 0x5A, dtype=torch.uint8, device=self.device)
        inner = room[512 + offset * size: 512 + offset * size + n]
        view = inner.view(dtype).view(shape) if n else torch.empty(shape, dtype=dtype, device=self.device)
        if like is not None:
            view.copy_(like)
        self.made.append((room, 512 + offset * size, n, like))
        return view

    def check(self):
        for room, first, n, like in self.made:
            assert bool((room[:first] == 0x5A).all()) and bool((room[first + n:] == 0x5A).all()), "wrote outside of a buffer"
            if like is not None:
                assert torch.equal(room[first:first + n].cpu(), like.contiguous().view(-1).view(torch.uint8)), "wrote an input"


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", [(1, 5, 3), (3, 40, 7), (9, 33, 17), (65, 100, 1000), (130, 257, 129), (70, 1001, 515), (2600, 2700, 131), (40, 20, 17001)],
                         ids=lambda s: "x".join(map(str, s)))
def test_nothing_outside_of_the_outputs_is_written(hip_device, shape, dtype):
    """Every operator through the C ABI, into buffers one element off the grid with margins around them."""
    from optimi_amd import cabi
    L, code = cabi.lib(), {torch.float32: cabi.F32, torch.bfloat16: cabi.BF16, torch.float16: cabi.F16}[dtype]
    m, n, k = shape
    x, r, g, w, bias = rand((m, k), dtype, 1), rand((m, k), dtype, 2), rand((m, n), dtype, 3), rand((n, k), dtype, 4), rand((n,), dtype, 5)
    nw = rand((k,), dtype, 6)
    stream = torch.cuda.current_stream().cuda_stream

    def run(name, *args):
        cabi.check(getattr(L, "optimi_hip_" + name)(*(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args), stream), name)

    def work(name, *args):
        size = getattr(L, "optimi_hip_" + name + "_workspace")(*args)
        assert size >= 0
        return buf(shape=(size,), dtype=torch.uint8) if size else None

    for offset in (0, 1):
        buf = Guarded(hip_device)
        out = lambda *s, t=dtype: buf(shape=s, dtype=t, offset=offset)  # noqa: E731
        dx, dr, dg, dw, db, dn = (buf(t, offset=offset) for t in (x, r, g, w, bias, nw))
        q, s, wq, ws = out(m, k, t=torch.int8), out(m, t=torch.float32), out(n, k, t=torch.int8), out(n, t=torch.float32)
        run("int8_quantize", dx, m, k, code, q, s)
        run("int8_quantize", dw, n, k, code, wq, ws)
        back = out(m, k)
        run("int8_dequantize", q, s, m, k, code, back)
        y = out(m, n)
        run("int8_matmul", q, s, wq, ws, db, m, n, k, code, y, work("int8_matmul", m, n, k))
        gw, gb = out(n, k), out(n)
        run("int8_weight_grad", dg, q, s, m, n, k, code, gw, gb, work("int8_weight_grad", m, n, k, code, 1))
        h, q2, s2, rstd = out(m, k), out(m, k, t=torch.int8), out(m, t=torch.float32), out(m, t=torch.float32)
        run("add_rms_norm_int8", dx, dr, dn, m, k, code, code, 1e-6, h, q2, s2, rstd)
        gx, gn = out(m, k), out(k)
        run("add_rms_norm_int8_backward", back, dr, h, rstd, dn, m, k, code, code, gx, gn, work("add_rms_norm_int8_backward", m, k))
        torch.cuda.synchronize()
        buf.check()
        wq64, ws64 = R.quantize(w)
        x64, s64 = R.quantize(x)
        assert torch.equal(q.cpu().double(), x64) and torch.equal(s.cpu().double(), s64)
        R.close(y, *R.matmul(x64, s64, wq64, ws64, bias, dtype), "y")
        R.close(gw, *R.weight_grad(g, x64, s64, dtype), "gw")
        R.close(gb, *R.column_sum(g, dtype), "gb")
        assert torch.equal(h.cpu(), (x.double() + r.double()).to(dtype))


def test_offsets_beyond_32_bits(hip_device):
    """Rows behind the 2^32nd element give what they give alone."""
    rows, cols, outs, last = (1 << 20) + 100, 4100, 24, 300
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=hip_device)
    tail = rand((last, cols), torch.bfloat16, 1).to(hip_device)
    x[-last:] = tail
    values, scales = optimi.int8_quantize(x)
    q, s = optimi.int8_quantize(tail)
    assert torch.equal(values[-last:], q) and torch.equal(scales[-last:], s) and not values[:-last].any()
    assert torch.equal(optimi.int8_dequantize(values, scales)[-last:], optimi.int8_dequantize(q, s))
    w, ws = optimi.int8_quantize(rand((outs, cols), torch.bfloat16, 2).to(hip_device))
    assert torch.equal(optimi.int8_matmul(values, scales, w, ws)[-last:], optimi.int8_matmul(q, s, w, ws))
    g = torch.zeros(rows, outs, dtype=torch.bfloat16, device=hip_device)
    g[-last:] = rand((last, outs), torch.bfloat16, 3, 1e-2).to(hip_device)
    dw, db = optimi.int8_weight_grad(g, values, scales, bias=True)
    want, allowed = R.weight_grad(g[-last:], q, s, torch.bfloat16)
    R.close(dw, want.cpu(), allowed.cpu(), "weight gradient")
    nw = torch.ones(cols, dtype=torch.bfloat16, device=hip_device)
    del values
    nv, ns, h, rstd = optimi.add_rms_norm_int8(x, nw, residual=x)
    nv2, ns2, h2, rstd2 = optimi.add_rms_norm_int8(tail, nw, residual=tail)
    assert torch.equal(nv[-last:], nv2) and torch.equal(ns[-last:], ns2) and torch.equal(h[-last:], h2) and torch.equal(rstd[-last:], rstd2)
    del nv
    dx, _ = optimi.add_rms_norm_int8_backward(x, h, rstd, nw)
    assert torch.equal(dx[-last:], optimi.add_rms_norm_int8_backward(tail, h2, rstd2, nw)[0])


# ---------------------------------------------------------------------------------- refusals

def test_refusals(hip_device):
    d = dict(device=hip_device)
    q, s = torch.zeros(4, 8, dtype=torch.int8, **d), torch.ones(4, **d)
    w, ws = torch.zeros(6, 8, dtype=torch.int8, **d), torch.ones(6, **d)
    cases = [
        (lambda: optimi.int8_quantize(torch.zeros(4, 8)), "HIP device"),
        (lambda: optimi.int8_quantize(torch.zeros(4, 8, dtype=torch.float64, **d)), "unsupported dtype"),
        (lambda: optimi.int8_quantize(torch.zeros((), **d)), "at least one dimension"),
        (lambda: optimi.int8_dequantize(q, s[:3], torch.float32), "scales of size"),
        (lambda: optimi.int8_dequantize(q, s.double(), torch.float32), "must be float32"),
        (lambda: optimi.int8_dequantize(q.float(), s, torch.float32), "int8 values"),
        (lambda: optimi.int8_dequantize(q, s, torch.int32), "unsupported dtype"),
        (lambda: optimi.int8_dequantize(q, s.cpu(), torch.float32), "HIP device"),
        (lambda: optimi.int8_matmul(q, s, w[:, :7], ws), "inputs"),
        (lambda: optimi.int8_matmul(q, s, w[None], ws[None]), "matrix"),
        (lambda: optimi.int8_matmul(q, s, w, ws[:5]), "scales of size"),
        (lambda: optimi.int8_matmul(q, s, w, ws, bias=torch.zeros(6, **d), dtype=torch.bfloat16), "bias has dtype"),
        (lambda: optimi.int8_matmul(q, s, w, ws, bias=torch.zeros(5, **d), dtype=torch.float32), "6 elements"),
        (lambda: optimi.int8_matmul(torch.zeros(1, 131072, dtype=torch.int8, **d), s[:1], torch.zeros(1, 131072, dtype=torch.int8, **d), ws[:1]), "too large"),
        (lambda: optimi.int8_weight_grad(torch.zeros(5, 6, **d), q, s), "different rows"),
        (lambda: optimi.int8_weight_grad(torch.zeros(4, 6, dtype=torch.int8, **d), q, s), "unsupported dtype"),
        (lambda: optimi.add_rms_norm_int8(torch.zeros(4, 8, **d), torch.ones(7, **d)), "8 elements"),
        (lambda: optimi.add_rms_norm_int8(torch.zeros(4, 8, **d), torch.ones(8, dtype=torch.bfloat16, **d)), "dtype"),
        (lambda: optimi.add_rms_norm_int8(torch.zeros(4, 8, **d), torch.ones(8, **d), residual=torch.zeros(3, 8, **d)), "size"),
        (lambda: optimi.add_rms_norm_int8(torch.zeros(4, 8, **d), torch.ones(8, **d), residual=torch.zeros(4, 8, dtype=torch.float16, **d)), "dtype"),
        (lambda: optimi.add_rms_norm_int8(torch.zeros(4, 8, **d), torch.ones(8, **d), eps=-1.0), "scalar"),
        (lambda: optimi.add_rms_norm_int8(torch.zeros(4, 8, **d), torch.ones(8, **d), eps=float("nan")), "scalar"),
        (lambda: optimi.add_rms_norm_int8(torch.zeros(4, 0, **d), torch.ones(0, **d)), "count"),
        (lambda: optimi.add_rms_norm_int8_backward(torch.zeros(4, 8, **d), torch.zeros(4, 8, **d), torch.ones(3, **d), torch.ones(8, **d)), "rstd"),
        (lambda: optimi.add_rms_norm_int8_backward(torch.zeros(4, 8, **d), torch.zeros(4, 8, **d), torch.ones(4, **d), torch.ones(8, **d), grad_h=torch.zeros(4, 7, **d)), "size"),
    ]
    for i, (call, match) in enumerate(cases):
        with pytest.raises(RuntimeError, match=match):
            call()
            raise AssertionError(f"case {i} was not refused")
    with pytest.raises(TypeError, match="one dtype"):
        optimi.int8_linear(torch.zeros(4, 8, dtype=torch.bfloat16, **d), torch.zeros(6, 8, **d))
    with pytest.raises(ValueError, match="weights"):
        optimi.add_rms_norm_int8_linear(torch.zeros(4, 8, **d), torch.ones(8, **d), [])
    y = optimi.int8_linear(torch.ones(4, 8, requires_grad=True, **d), torch.ones(6, 8, requires_grad=True, **d))
    (gx,) = torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[0][0].variable], create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()  # no second derivatives
