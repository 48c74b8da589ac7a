"""The int8 operators and layers at the edges of what they allow, each against the operators' 64-bit forms or against the same
operators called one by one."""

import pytest
import torch
from torch import nn

import int8_ref as R
import optimi_amd as optimi
from optimi_amd import backend
from test_hip_int8 import Guarded, checkpoint, int8_inputs, misaligned, norm_layers, rand

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------- the lazy negative bit

def turned(t):
    """The same numbers, stored with the opposite sign under the negative bit; contiguous."""
    view = torch._neg_view(-t)
    assert view.is_neg() and view.is_contiguous() and torch.equal(view, t)
    return view


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
def test_tensors_with_the_negative_bit(hip_device, dtype):
    m, n, k = 9, 24, 40
    x, r, g, w, b, nw = (rand(s, dtype, i).to(hip_device) for i, s in enumerate([(m, k), (m, k), (m, n), (n, k), (n,), (k,)]))
    q, s = optimi.int8_quantize(x)
    wq, ws = optimi.int8_quantize(w)
    _, _, h, rstd = optimi.add_rms_norm_int8(x, nw, residual=r)
    calls = {
        "quantize": (lambda f: optimi.int8_quantize(f(x))),
        "dequantize": (lambda f: (optimi.int8_dequantize(f(q), f(s), dtype),)),
        "matmul": (lambda f: (optimi.int8_matmul(f(q), f(s), f(wq), f(ws), bias=f(b), dtype=dtype),)),
        "weight gradient": (lambda f: optimi.int8_weight_grad(f(g), f(q), f(s), bias=True)),
        "norm": (lambda f: optimi.add_rms_norm_int8(f(x), f(nw), residual=f(r))),
        "norm alone": (lambda f: optimi.add_rms_norm_int8(f(x), f(nw))),
        "norm backward": (lambda f: optimi.add_rms_norm_int8_backward(f(x), f(h), f(rstd), f(nw), grad_h=f(r))),
    }
    for name, call in calls.items():
        for got, want in zip(call(turned), call(lambda t: t)):
            assert torch.equal(got, want), name


# ---------------------------------------------------------------------------------- autocast around the backward pass

@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
def test_backward_inside_autocast_is_that_outside(hip_device, dtype, cast):
    """Layers that ran outside of autocast (or in a region where it is off) give the same gradients wherever backward() is called."""
    m, k, outs = 11, 48, (24, 40)
    x, r, nw, ws, bs = norm_layers(dtype, m, k, outs)
    gs = [rand((m, n), dtype, 60 + n, 1e-2).to(hip_device) for n in outs]
    results = []
    for inside in (False, True):
        leaf = lambda t: t.to(hip_device).requires_grad_()  # noqa: E731
        lx, lr, ln, lw, lb = leaf(x), leaf(r), leaf(nw), [leaf(w) for w in ws], leaf(bs[1])
        y = optimi.int8_linear(lx, lw[0])
        ys, h = optimi.add_rms_norm_int8_linear(lx, ln, lw, biases=[None, lb], residual=lr)
        with torch.autocast("cuda", dtype=cast, enabled=inside):
            torch.autograd.backward([y, *ys, h], [gs[0], *gs, h.detach()])
        results.append([t.grad for t in (lx, lr, ln, *lw, lb)])
    for a, b in zip(*results):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_a_whole_step_inside_autocast(hip_device, cast):
    m, k, outs = 11, 48, (24, 40)
    x, r, nw, ws, _ = norm_layers(torch.float32, m, k, outs)
    results = []
    for inside in (False, True):
        leaf = lambda t: t.to(hip_device).requires_grad_()  # noqa: E731
        lx, lr, ln, lw = leaf(x), leaf(r), leaf(nw), [leaf(w) for w in ws]
        with torch.autocast("cuda", dtype=cast):
            y = optimi.int8_linear(lx, lw[0])
            (a, b), h = optimi.add_rms_norm_int8_linear(lx, ln, lw, residual=lr)
            loss = y.float().square().mean() + a.float().square().mean() + b.float().square().mean() + h.float().square().mean()
            if inside:
                loss.backward()
        if not inside:
            loss.backward()
        results.append([t.grad for t in (lx, lr, ln, *lw)])
    for a, b in zip(*results):
        assert a.dtype == torch.float32 and torch.equal(a, b)


# ---------------------------------------------------------------------------------- sequences

def test_a_sequence_of_mixed_types_runs_as_it_did(hip_device):
    """A bf16 norm in front of an fp32 layer on fp32 input: torch takes it, so the prepared sequence has to."""
    plain = nn.Sequential(nn.RMSNorm(48, eps=1e-5).to(torch.bfloat16), nn.Linear(48, 24)).to(hip_device)
    x = rand((7, 48), torch.float32, 1).to(hip_device)
    normed = plain[0](x)
    assert plain(x).dtype == torch.float32
    optimi.prepare_for_int8_linear(plain)
    assert torch.equal(plain(x), optimi.int8_linear(normed, plain[1].weight, plain[1].bias))


# ---------------------------------------------------------------------------------- a sequence under autocast

@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_the_norm_of_a_sequence_sees_all_bits_under_autocast(hip_device, cast):
    """The residual stream stays in float32 up to the norm; only the layer runs in the autocast type."""
    m, k, n = 13, 96, 40
    model = nn.Sequential(nn.RMSNorm(k, eps=1e-5), nn.Linear(k, n)).to(hip_device)
    optimi.prepare_for_int8_linear(model)
    x = rand((m, k), torch.float32, 2).to(hip_device).requires_grad_()
    with torch.autocast("cuda", dtype=cast):
        y = model(x)
    g = rand((m, n), cast, 3, 1e-2).to(hip_device)
    y.backward(g)
    with torch.no_grad():
        w, b = model[1].weight.to(cast), model[1].bias.to(cast)
        values, scales, h, rstd = optimi.add_rms_norm_int8(x, model[0].weight, eps=1e-5)
        want = optimi.int8_matmul(values, scales, *optimi.int8_quantize(w), bias=b, dtype=cast)
        assert y.dtype == cast and torch.equal(y, want)
        dx, dn = optimi.add_rms_norm_int8_backward((g @ w).float(), h, rstd, model[0].weight)
        assert torch.equal(x.grad, dx) and torch.equal(model[0].weight.grad, dn)
        dw, db = optimi.int8_weight_grad(g, values, scales, bias=True)
        assert torch.equal(model[1].weight.grad, dw.float()) and torch.equal(model[1].bias.grad, db.float())


# ---------------------------------------------------------------------------------- layers that are frozen in part

@pytest.fixture
def no_weight_grad(monkeypatch):
    def refuse(*args):
        raise AssertionError("a weight gradient that nobody asked for")

    monkeypatch.setattr(backend.ext(), "int8_weight_grad", refuse)


def kept_int8(y):
    return [t for t in y.grad_fn.saved_tensors if t is not None and t.dtype == torch.int8]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", [(0, 40), (1, 5), (5, 1000), (127, 300), (128, 2048), (129, 2049), (1000, 40), (300, 9001)], ids=lambda s: "x".join(map(str, s)))
def test_a_bias_alone(hip_device, shape, dtype, no_weight_grad):
    m, n = shape
    x, w, g = rand((m, 24), dtype, 1).to(hip_device), rand((n, 24), dtype, 2).to(hip_device), rand((m, n), dtype, 3, 1e-2)
    b = torch.zeros(n, dtype=dtype, device=hip_device, requires_grad=True)
    y = optimi.int8_linear(x, w, b)
    assert kept_int8(y) == [], "a bias gradient needs no checkpoint"
    y.backward(g.to(hip_device))
    R.close(b.grad, *R.column_sum(g, dtype), "bias")
    grad, b.grad = b.grad, None
    optimi.int8_linear(x, w, b).backward(g.to(hip_device).t().contiguous().t())
    assert torch.equal(b.grad, grad)
    b.grad = None
    (y,), _ = optimi.add_rms_norm_int8_linear(x, torch.ones(24, dtype=dtype, device=hip_device), [w], biases=[b])
    y.backward(g.to(hip_device))
    assert torch.equal(b.grad, grad)


def test_a_bias_alone_of_one_vector_and_of_a_sum(hip_device, no_weight_grad):
    w, b = rand((40, 24), torch.float32, 1).to(hip_device), torch.zeros(40, device=hip_device, requires_grad=True)
    optimi.int8_linear(rand((24,), torch.float32, 2).to(hip_device), w, b).sum().backward()
    assert torch.equal(b.grad, torch.ones_like(b))
    optimi.int8_linear(rand((3, 5, 24), torch.float32, 2).to(hip_device), w, b).sum().backward()
    assert torch.equal(b.grad, torch.full_like(b, 16.0))


# ---------------------------------------------------------------------------------- frozen layers behind a norm

def test_frozen_layers_behind_a_trained_norm(hip_device, no_weight_grad):
    x, r, nw, ws, _ = norm_layers(torch.bfloat16, 20, 64, (32, 48))
    lx, ln = x.to(hip_device).requires_grad_(), nw.to(hip_device).requires_grad_()
    ws = [w.to(hip_device) for w in ws]
    (y0, y1), h = optimi.add_rms_norm_int8_linear(lx, ln, ws, residual=r.to(hip_device))
    assert kept_int8(y0) == [], "without a weight gradient the checkpoint is not needed"
    g0, g1 = torch.randn_like(y0), torch.randn_like(y1)
    torch.autograd.backward([y0, y1], [g0, g1])
    with torch.no_grad():
        _, _, h, rstd = optimi.add_rms_norm_int8(lx, ln, residual=r.to(hip_device))
        dx, dn = optimi.add_rms_norm_int8_backward(torch.addmm(g0 @ ws[0], g1, ws[1]), h, rstd, ln)
    assert torch.equal(lx.grad, dx) and torch.equal(ln.grad, dn)


def test_a_bias_alone_behind_a_norm(hip_device, no_weight_grad):
    x, _, nw, ws, bs = norm_layers(torch.bfloat16, 20, 64, (32, 48))
    lb = bs[1].to(hip_device).requires_grad_()
    (y,), _ = optimi.add_rms_norm_int8_linear(x.to(hip_device), nw.to(hip_device), [ws[1].to(hip_device)], biases=[lb])
    assert kept_int8(y) == []
    g = torch.randn_like(y)
    y.backward(g)
    R.close(lb.grad, *R.column_sum(g.cpu(), torch.bfloat16), "bias")


def test_one_of_two_layers_is_trained(hip_device):
    x, _, nw, ws, bs = norm_layers(torch.bfloat16, 20, 64, (32, 48))
    ln, lw, lb = nw.to(hip_device), [w.to(hip_device) for w in ws], bs[1].to(hip_device).requires_grad_()
    lw[0].requires_grad_()
    ys, _ = optimi.add_rms_norm_int8_linear(x.to(hip_device), ln, lw, biases=[None, lb])
    assert len(kept_int8(ys[0])) == 1
    assert [t.dtype for t in ys[0].grad_fn.saved_tensors if t is not None and t.shape == x.shape] == [torch.int8], "no gradient flows into the norm"
    gs = [torch.randn_like(y) for y in ys]
    torch.autograd.backward(ys, gs)
    values, scales, _, _ = optimi.add_rms_norm_int8(x.to(hip_device), ln)
    assert torch.equal(lw[0].grad, optimi.int8_weight_grad(gs[0], values, scales))
    R.close(lb.grad, *R.column_sum(gs[1].cpu(), torch.bfloat16), "bias")


# ---------------------------------------------------------------------------------- rows whose squares leave float32's range

ROW_WIDTHS = [1, 5, 8, 100, 513, 1001, 1500, 4100, 6000, 8200, 9000, 13000, 16385, 18001]


def extreme_rows(cols, dtype, sizes, seed):
    gen = torch.Generator().manual_seed(seed)
    x = (1 + torch.rand(len(sizes), cols, generator=gen, dtype=torch.float64)) * torch.where(torch.rand(len(sizes), cols, generator=gen) < 0.5, -1, 1)
    return (x * torch.tensor(sizes, dtype=torch.float64)[:, None]).to(dtype)


def check_extreme_norm(device, x, w, eps, residual=None):
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    values, scales, _, rstd = optimi.add_rms_norm_int8(x.to(device), w.to(device), residual=None if residual is None else residual.to(device), eps=eps)
    y, r, rel_r, rel_y = R.norm(h, w, eps)
    # 1/rms of the largest rows is below float32's normal range: two roundings to its smallest step
    coarse = 2.02 * R.least(torch.float32)
    R.close(rstd, r, rel_r * r + coarse, "rstd")
    q, s = values.cpu().double(), scales.cpu().double()
    assert bool((q.abs() <= 127).all())
    absmax = y.abs().amax(1, keepdim=True)
    assert bool((s[:, None] <= 2 * absmax / 63).all()), "a scale that does not fit its row"
    R.close(q * s[:, None], y, s[:, None] / 2 + (rel_y + coarse / r[:, None]) * y.abs(), "y")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cols", ROW_WIDTHS)
def test_norm_of_large_rows(hip_device, cols, dtype):
    """Finite rows whose squares have no place in float32 have an ordinary norm."""
    sizes = [2.0**e for e in (50, 57, 60, 63, 64, 80, 100, 120, 126)] + [1.0]
    x = extreme_rows(cols, dtype, sizes, cols)
    w = (1 + 0.2 * torch.rand(cols, generator=torch.Generator().manual_seed(1), dtype=torch.float64)).to(dtype)
    check_extreme_norm(hip_device, x, w, 1e-6)
    check_extreme_norm(hip_device, x / 2, w, 1e-6, residual=(x / 4).flip(0).contiguous())


@pytest.mark.parametrize("eps", [0.0, 1e-50, 1e-38, 1e-30])
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("cols", ROW_WIDTHS)
def test_norm_of_small_rows(hip_device, cols, dtype, eps):
    """With an eps below it, a row of tiny numbers has a norm as good as another's."""
    low = -22 if dtype == torch.float16 else -100
    x = extreme_rows(cols, dtype, [2.0**e for e in (low, low / 2, -20, -1)], cols + 1)
    if dtype != torch.float16:  # numbers of unlike size, the small ones below the range of squares altogether
        x = torch.cat([x, extreme_rows(cols, dtype, [2.0**-40, 2.0**-55, 2.0**-60, 2.0**-75], cols + 2)])
        x[-1, : cols // 2] *= 2.0**-40
    w = (1 + 0.2 * torch.rand(cols, generator=torch.Generator().manual_seed(1), dtype=torch.float64)).to(dtype)
    check_extreme_norm(hip_device, x, w, eps)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cols", [3, 40, 1500, 17000])
def test_norm_of_rows_whose_inverse_rms_is_too_large(hip_device, cols, dtype):
    """Subnormal rows without an eps: 1/rms has no place in float32, the normed row has."""
    x = extreme_rows(cols, dtype, [2.0**-130, 2.0**-131], cols)
    values, scales, _, rstd = optimi.add_rms_norm_int8(x.to(hip_device), torch.ones(cols, dtype=dtype, device=hip_device), eps=0.0)
    y, _, _, rel_y = R.norm(x, torch.ones(cols), 0.0)
    s = scales.cpu().double()[:, None]
    R.close(values.cpu().double() * s, y, s / 2 + rel_y * y.abs(), "y")
    assert bool(torch.isinf(rstd).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cols", [1, 40, 1500, 4100, 9000, 17000])
def test_norm_backward_of_extreme_rows(hip_device, cols, dtype):
    sizes = [2.0**e for e in (-100, -80, -64, -50, 50, 64, 80, 100, 126)]
    h, w = extreme_rows(cols, dtype, sizes, cols), torch.ones(cols, dtype=dtype)
    g, gh = rand((len(sizes), cols), dtype, 2, 1e-2), rand((len(sizes), cols), dtype, 3, 1e-2)
    rstd = R.norm(h, w, 0.0)[1].float()
    for more in (None, gh):
        dx, dw = optimi.add_rms_norm_int8_backward(*(t.to(hip_device) for t in (g, h, rstd, w)), grad_h=None if more is None else more.to(hip_device))
        want_dx, allow_dx, want_dw, allow_dw = R.norm_backward(g, h, rstd, w, more, dtype, dtype)
        R.close(dx, want_dx, allow_dx, "dx")
        R.close(dw, want_dw, allow_dw, "dweight")


@pytest.mark.parametrize("cols", [40, 1500, 17000])
def test_norm_of_extreme_rows_that_are_empty_or_not_finite(hip_device, cols):
    x = extreme_rows(cols, torch.bfloat16, [2.0**100] * 4, 1)
    x[0], x[1, 3], x[2, 5] = 0, float("inf"), float("nan")
    w = torch.ones(cols, dtype=torch.bfloat16)
    for eps in (1e-6, 1e-50):
        values, scales, _, rstd = (t.cpu() for t in optimi.add_rms_norm_int8(x.to(hip_device), w.to(hip_device), eps=eps))
        assert torch.equal(torch.isnan(scales), torch.tensor([False, True, True, False]))
        assert float(scales[0]) == 1.0 and not values[:3].any() and bool(values[3].any())
        assert abs(float(rstd[0]) * eps**0.5 - 1) < 4 * R.U


# ---------------------------------------------------------------------------------- scales at the ends of the range

@pytest.mark.parametrize("shape", [(1, 100, 2000), (4, 40, 64), (40, 70, 96), (100, 100, 16384), (130, 300, 1111), (2600, 2700, 131), (4096, 4096, 64)], ids=lambda s: "x".join(map(str, s)))
def test_matmul_of_scales_whose_product_is_ordinary(hip_device, shape):
    """A row of huge numbers against small weights, and the other way round: only the result has to fit the type."""
    m, n, k = shape
    a, _, b, _ = int8_inputs(m, n, k, 5)
    bias = rand((n,), torch.float32, 6)
    big, small = torch.full((m,), 2.0**110), torch.full((n,), 2.0**-115)
    big[m // 2] = 2.0**121
    small[n // 2] = 2.0**-126
    for sa, sb in ((big, small), (torch.full((m,), 2.0**-126), torch.full((n,), 2.0**121))):
        y = optimi.int8_matmul(a.to(hip_device), sa.to(hip_device), b.to(hip_device), sb.to(hip_device), bias=bias.to(hip_device), dtype=torch.float32)
        if m * n * k < 1 << 29:
            want, allowed = R.matmul(a, sa, b, sb, bias, torch.float32)
        else:
            want, allowed = (t.cpu() for t in R.matmul(*(t.to(hip_device) for t in (a, sa, b, sb, bias)), torch.float32))
        R.close(y, want, allowed, str(shape))


# ---------------------------------------------------------------------------------- bias gradients of large layers

# the wide kernel's sizes (in 16 bits): the bias gradient is a sum of columns beside it, one to three stripes of 2048
# columns, with and without a padded copy in front of its workspace, rows above and below the 128 partial sums
WIDE = [(1, 3000, 2900), (65, 3000, 2800), (127, 2904, 2831), (129, 2817, 3000), (200, 2896, 2817), (257, 5000, 1700), (1000, 2817, 2820), (300, 1000, 8300)]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", WIDE, ids=lambda s: "x".join(map(str, s)))
def test_bias_gradient_of_large_layers(hip_device, shape, dtype):
    rows, outs, cols = shape
    g, (q, s) = rand((rows, outs), dtype, 3, 1e-2).to(hip_device), (t.to(hip_device) for t in checkpoint(rows, cols, 4))
    want, allowed = R.weight_grad(g, q, s, dtype)
    bias, bias_allowed = R.column_sum(g.cpu(), dtype)
    for grad, values in ((g, q), (misaligned(g, hip_device), misaligned(q, hip_device))):
        dw, db = optimi.int8_weight_grad(grad, values, s, bias=True)
        R.close(dw, want.cpu(), allowed.cpu(), f"weight {shape}")
        R.close(db, bias, bias_allowed, f"bias {shape}")
        again = optimi.int8_weight_grad(grad, values, s, bias=True)
        assert torch.equal(again[0], dw) and torch.equal(again[1], db), "the same bits on every run"


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", [(65, 3000, 2800), (130, 2904, 2831), (129, 2817, 3000)], ids=lambda s: "x".join(map(str, s)))
def test_bias_gradient_of_large_layers_that_is_not_finite(hip_device, shape, dtype):
    rows, outs, cols = shape
    g, (q, s) = rand((rows, outs), dtype, 4, 1e-2).to(hip_device), (t.to(hip_device) for t in checkpoint(rows, cols, 5))
    g[rows - 1, 5], g[0, 9], g[rows // 2, outs - 1] = float("inf"), float("-inf"), float("nan")
    _, db = optimi.int8_weight_grad(g, q, s, bias=True)
    R.close(db, *R.column_sum(g.cpu(), dtype), "bias")


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("shape", [(129, 2817, 3000), (257, 5000, 1700)], ids=lambda s: "x".join(map(str, s)))
def test_a_large_weight_gradient_stays_in_its_buffers(hip_device, shape, dtype):
    """Through the C ABI, into buffers and a workspace of exactly the stated size with margins around them."""
    from optimi_amd import cabi
    L, code = cabi.lib(), {torch.float32: cabi.F32, torch.bfloat16: cabi.BF16, torch.float16: cabi.F16}[dtype]
    rows, outs, cols = shape
    g, (q, s) = rand((rows, outs), dtype, 3, 1e-2), checkpoint(rows, cols, 4)
    want, allowed = R.weight_grad(*(t.to(hip_device) for t in (g, q, s)), dtype)
    for offset in (0, 1):
        buf = Guarded(hip_device)
        dg, dq, ds = (buf(t, offset=offset) for t in (g, q, s))
        dw, db = buf(shape=(outs, cols), dtype=dtype, offset=offset), buf(shape=(outs,), dtype=dtype, offset=offset)
        size = L.optimi_hip_int8_weight_grad_workspace(rows, outs, cols, code, 1)
        assert size >= 0
        work = buf(shape=(size,), dtype=torch.uint8) if size else None
        pointers = [t.data_ptr() for t in (dg, dq, ds)], [t.data_ptr() for t in (dw, db)]
        cabi.check(L.optimi_hip_int8_weight_grad(*pointers[0], rows, outs, cols, code, *pointers[1], None if work is None else work.data_ptr(),
                                                 torch.cuda.current_stream().cuda_stream), "weight_grad")
        torch.cuda.synchronize()
        buf.check()
        R.close(dw, want.cpu(), allowed.cpu(), "weight")
        R.close(db, *R.column_sum(g, dtype), "bias")


# ---------------------------------------------------------------------------------- rows that end inside a vector

@pytest.mark.parametrize("weight32", [False, True], ids=["weight_own", "weight_fp32"])
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("cols", R.RAGGED)
def test_every_element_counts_once(hip_device, cols, dtype, weight32):
    """One loud element in the columns that the last vector shares with its neighbour, or beside them: counted twice or not at
    all, it changes everything by a factor (the oracle with that mistake is held against the allowances on the CPU)."""
    for at in R.loud_places(cols):
        h, g, w = R.loud_row(cols, at, dtype, torch.float32 if weight32 else dtype)
        values, scales, _, rstd = optimi.add_rms_norm_int8(h.to(hip_device), w.to(hip_device), eps=1e-6)
        y, r, rel_r, rel_y = R.norm(h, w, 1e-6)
        R.close(rstd, r, rel_r * r, f"rstd {at}")
        s = scales.cpu().double()[:, None]
        R.close(values.cpu().double() * s, y, s / 2 + rel_y * y.abs(), f"y {at}")
        r = r.float()
        dx, dw = optimi.add_rms_norm_int8_backward(g.to(hip_device), h.to(hip_device), r.to(hip_device), w.to(hip_device))
        want_dx, allow_dx, want_dw, allow_dw = R.norm_backward(g, h, r, w, None, dtype, w.dtype)
        R.close(dx, want_dx, allow_dx, f"dx {at}")
        R.close(dw, want_dw, allow_dw, f"dweight {at}")


# ---------------------------------------------------------------------------------- the most outputs

@pytest.mark.parametrize("m", [1, 4, 70])
def test_products_of_very_many_outputs(hip_device, m):
    """Launches of nearly 2^32 lanes and, off the 16-byte grid, of 2^23 tiles."""
    n, k = (1 << 28) - 16 if m < 5 else 1 << 28, 16
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    a, sa, _, _ = (t.to(hip_device) for t in int8_inputs(m, 1, k, 1))
    b, sb = torch.zeros(n, k, dtype=torch.int8, device=hip_device), torch.ones(n, device=hip_device)
    places = [slice(0, 300), slice((1 << 27) - 100, (1 << 27) + 200), slice(n - 300, n)]
    for i, at in enumerate(places):
        b[at] = torch.randint(-127, 128, (300, k), generator=torch.Generator().manual_seed(i), dtype=torch.int8).to(hip_device)
    if m > 4:
        b = misaligned(b, hip_device)
    y = optimi.int8_matmul(a, sa, b, sb)
    for at in places:
        assert torch.equal(y[:, at], optimi.int8_matmul(a, sa, b[at], sb[at]))
    assert not y[:, 300:1000].any() and not y[:, 1 << 26:(1 << 26) + 5000].any() and not y[:, n - 5000:n - 300].any()
