"""Plain 64-bit forms of the int8 activation operators, on the CPU, and the error that each kernel may make.

The allowances count roundings: `half(dtype)` is half a step of the result's type relative to the value, U is half a step of
float32, and a float32 sum of n terms is at most n U off the sum of the terms' absolute values, in whatever order
it is formed (matrix instructions may cut instead of rounding, which doubles it)."""

import torch

U = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the smallest number of the type: the absolute error of a result below its normal range."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def step_of(absmax, top):
    """(scale, most steps) for rows with these largest absolute values (float64), by trying exponents."""
    scale = torch.full_like(absmax, 2.0**-126)
    for e in range(-126, 123):
        scale = torch.where(absmax > 127 * scale, torch.full_like(scale, 2.0 ** (e + 1)), scale)
    scale = torch.where(absmax == 0, torch.ones_like(scale), scale)
    most = torch.where(scale * 64 > top, 63.0, 127.0).double()
    return scale, most


def quantize(x, top=None):
    """(values, scales) of the rows of x in float64, as float64."""
    top = float(torch.finfo(x.dtype).max) if top is None else top
    x = x.double()
    if x.shape[-1] == 0:
        return torch.zeros_like(x), torch.ones(x.shape[:-1], dtype=torch.float64)
    absmax = x.abs().amax(dim=-1)
    fine = torch.isfinite(absmax)
    scale, most = step_of(torch.where(fine, absmax, torch.zeros_like(absmax)), top)
    q = torch.clamp(torch.round(torch.where(fine[..., None], x, torch.zeros_like(x)) / scale[..., None]), -most[..., None], most[..., None])
    return q, torch.where(fine, scale, torch.full_like(scale, float("nan")))


def matmul(a, sa, b, sb, bias, dtype):
    """(result, allowance): whole-number sums; rounded once to float32, twice more by scales that are no powers
    of two (once each) and with the bias, then to the result's type."""
    s = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    y = s if bias is None else s + bias.double()
    return y, 4 * U * s.abs() + 2 * U * y.abs() + (half(dtype) * (1 + 8 * U)) * y.abs() + 1.01 * least(dtype)


def weight_grad(g, q, s, dtype):
    x = q.double() * s.double()[:, None]
    dw = g.double().T @ x
    total = g.double().abs().T @ x.abs()
    slack = 2 * (g.shape[0] + 8) * U * total
    if dtype != torch.float32 and bool((torch.frexp(s.double()).mantissa != 0.5).any()):
        slack = slack + half(dtype) * total  # values * scales rounded to the type
    return dw, slack + half(dtype) * (dw.abs() + slack) + 1.01 * least(dtype)


def column_sum(g, dtype):
    d, total = g.double().sum(0), g.double().abs().sum(0)
    slack = (g.shape[0] + 8) * U * total
    return d, slack + half(dtype) * (d.abs() + slack) + 1.01 * least(dtype)


def norm(h, w, eps):
    """(y, rstd, relative allowance of rstd, of y) for h as it is kept."""
    h = h.double()
    r = 1 / torch.sqrt(h.square().mean(dim=-1) + eps)
    # the sum of squares has only positive terms: n U relative, halved by the root; then the mean, eps, root and inverse
    rel = (h.shape[-1] + 8) * U / 2 + 4 * U
    return h * r[..., None] * w.double(), r, rel, rel + 3 * U


def norm_backward(g, h, r, w, gh, dtype, wdtype):
    """(dx, allowance, dw, allowance); r is the float32 rstd that the kernel is given."""
    g, h, r, w = g.double(), h.double(), r.double()[:, None], w.double()
    n = h.shape[1]
    xhat = h * r
    gw = g * w
    mean, mass = (gw * xhat).mean(1, keepdim=True), (gw * xhat).abs().mean(1, keepdim=True)
    dx = r * (gw - xhat * mean)
    more = torch.zeros_like(dx) if gh is None else gh.double()
    slack = r * (3 * U * gw.abs() + xhat.abs() * ((n + 12) * U * mass + 4 * U * mean.abs())) + 3 * U * (dx.abs() + more.abs())
    dx = dx + more
    dw, total = (g * xhat).sum(0), (g * xhat).abs().sum(0)
    wslack = (g.shape[0] + 12) * U * total
    return (dx, slack + half(dtype) * (dx.abs() + slack) + 1.01 * least(dtype),
            dw, wslack + half(wdtype) * (dw.abs() + wslack) + 1.01 * least(wdtype))


def close(got, want, allowed, what=""):
    """Elementwise |got - want| <= allowed; NaN where NaN is wanted, infinities equal."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    special = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    both = special & ~torch.isnan(want)
    assert torch.equal(got[both], want[both]), f"{what}: infinities differ"
    over = ((got - want).abs() > allowed) & ~special
    if bool(over.any()):
        at = int(((got - want).abs() / allowed.clamp(min=1e-300)).where(~special, torch.zeros_like(got)).flatten().argmax())
        raise AssertionError(f"{what}: {int(over.sum())} of {over.numel()} off, worst at {at}: got {got.flatten()[at]}, "
                             f"want {want.flatten()[at]}, allowed {allowed.flatten()[at]}")


# Rows that end inside a vector of eight: the kernels read the row's last eight elements there, some of which are the
# neighbour's too.
RAGGED = [9, 13, 65, 511, 513, 1023, 1025, 2047, 2049, 4097, 6145, 8193, 12289, 16385, 18001, 20003]


def loud_places(cols):
    """Columns to put a loud element at: first and last of those that two vectors share, before them, and the row's last."""
    shared = range(cols - 8, cols - cols % 8)
    return sorted({shared[0], shared[-1], max(0, shared[0] - 1), cols - 1})


def loud_row(cols, at, dtype, wdtype):
    """(h, g, w): three rows of small numbers with one large one in column `at` of the activation and of its gradient."""
    gen = torch.Generator().manual_seed(cols + at)
    h = torch.randn(3, cols, generator=gen, dtype=torch.float64) * 2.0**-9
    g = torch.randn(3, cols, generator=gen, dtype=torch.float64) * 2.0**-9
    h[:, at], g[:, at] = 24.0, 4.0
    w = 1 + 0.2 * torch.rand(cols, generator=gen, dtype=torch.float64)
    return h.to(dtype), g.to(dtype), w.to(wdtype)
