"""Cases that time training with activations held in 8 bits: the residual add and RMS norm with an int8 output,
the int8 checkpoint of an activation, the int8 matrix product and the weight gradient taken from a checkpoint.

``run`` computes each case in elementary torch operations, or, with ``own`` set, through the package's
operators.  An int8 activation is a matrix of whole numbers in [-127, 127] with one scale per row (token), the
smallest power of two that keeps the row inside that range.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one token of a decoding loop or of a tiny probe batch: launch latency is all there is
        {"name": "norm_forward_1x4096", "op": "norm_forward", "rows": 1, "cols": 4096, "dtype": "bf16", "residual": True},
        # a pre-norm of the 7B list on 8192 tokens: the block's sum, its norm and the int8 operand in one go
        {"name": "norm_forward_8192x4096", "op": "norm_forward", "rows": 8192, "cols": 4096, "dtype": "bf16", "residual": True},
        # the way back through the same norm, with the gradient that arrives on the residual path
        {"name": "norm_backward_8192x4096", "op": "norm_backward", "rows": 8192, "cols": 4096, "dtype": "bf16", "residual": True},
        # ragged batch and width, fp16, a norm without a residual path
        {"name": "norm_backward_1237x2047", "op": "norm_backward", "rows": 1237, "cols": 2047, "dtype": "fp16", "residual": False},
        # the widest activation of the 7B list (the down projection's input) kept in 8 bits and restored
        {"name": "checkpoint_16384x11008", "op": "checkpoint", "rows": 16384, "cols": 11008, "dtype": "bf16"},
        # a small odd fp32 activation
        {"name": "checkpoint_777x1001", "op": "checkpoint", "rows": 777, "cols": 1001, "dtype": "fp32"},
        # one token through the 7B list's up projection: the weight has to be read and nothing else counts
        {"name": "matmul_1x11008x4096", "op": "matmul", "rows": 1, "outs": 11008, "cols": 4096, "dtype": "bf16", "bias": False},
        # a short prompt through the down projection: few rows, a long sum
        {"name": "matmul_200x4096x11008", "op": "matmul", "rows": 200, "outs": 4096, "cols": 11008, "dtype": "bf16", "bias": False},
        # odd everything, with a bias
        {"name": "matmul_517x1001x1111", "op": "matmul", "rows": 517, "outs": 1001, "cols": 1111, "dtype": "fp16", "bias": True},
        # a training batch through the up projection
        {"name": "matmul_8192x11008x4096", "op": "matmul", "rows": 8192, "outs": 11008, "cols": 4096, "dtype": "bf16", "bias": False},
        # a ragged batch of fp32 gradients on a small layer of the MLP list
        {"name": "weight_grad_1000x4096x1023", "op": "weight_grad", "rows": 1000, "outs": 4096, "cols": 1023, "dtype": "fp32", "bias": True},
        # the weight gradient of the up projection over a training batch
        {"name": "weight_grad_8192x11008x4096", "op": "weight_grad", "rows": 8192, "outs": 11008, "cols": 4096, "dtype": "bf16", "bias": False},
    ]


MOST_VALUES = 16384 * 11008          # of one activation
MOST_PRODUCTS = 8192 * 11008 * 4096  # of one matrix product


def _log_size(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["norm_forward", "norm_backward", "checkpoint", "matmul", "weight_grad"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    rows = _log_size(rng, 1, 16384)
    cols = _log_size(rng, 16, 16384)
    if rng.random() < 0.5:  # widths of real layers are whole vectors, half of the time
        cols = max(16, cols // 64 * 64)
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
    if op in ("matmul", "weight_grad"):
        outs = _log_size(rng, 16, 16384)
        # fp32 gradients cost several products each
        most = MOST_PRODUCTS // (4 if dtype == "fp32" and op == "weight_grad" else 1)
        while case["rows"] * case["cols"] * outs > most:
            case["rows"] = max(1, case["rows"] // 2)
        case["outs"] = outs
        case["bias"] = rng.random() < 0.5
    else:
        while case["rows"] * case["cols"] > MOST_VALUES:
            case["rows"] //= 2
        if op != "checkpoint":
            case["residual"] = rng.random() < 0.7
    return case


# --------------------------------------------------------------------------------------------------
# The plain form


def _quantize(x, dtype):
    """(values, scales) of the rows of x (float32 values that a tensor of `dtype` held or led to)."""
    absmax = x.abs().amax(dim=1)
    bits = absmax.view(torch.int32)
    # absmax = m * 2^e with 1 <= m < 2, and 127 = 1.984375 * 2^6
    exponent = (bits >> 23) - 127 - 6 + ((bits & 0x7FFFFF) > 0x7E0000).int()
    exponent = exponent.clamp(min=-126)
    scale = ((exponent + 127) << 23).view(torch.float32)
    scale = torch.where(absmax == 0, torch.ones_like(scale), scale)
    # 64 steps have to stay a number of the activation's own type
    limit = torch.where(torch.isfinite((scale * 64).to(dtype)), 127.0, 63.0)
    finite = torch.isfinite(absmax)
    values = torch.round(x / scale[:, None])
    values = torch.minimum(torch.maximum(values, -limit[:, None]), limit[:, None])
    values = torch.where(finite[:, None], values, torch.zeros_like(values)).to(torch.int8)
    return values, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def _run_plain(s):
    dtype = s["dtype"]
    if s["op"] == "norm_forward":
        h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(dtype)
        hf = h.float()
        rstd = torch.rsqrt((hf * hf).mean(dim=1) + EPS)
        values, scales = _quantize(hf * rstd[:, None] * s["weight"].float(), torch.float32)
        restored = (values.float() * scales[:, None]).to(torch.bfloat16)
        return (restored, rstd) if s["residual"] is None else (restored, rstd, h)
    if s["op"] == "norm_backward":
        g, h, rstd, w = s["grad"].float(), s["h"].float(), s["rstd"], s["weight"].float()
        xhat = h * rstd[:, None]
        gw = g * w
        dx = rstd[:, None] * (gw - xhat * (gw * xhat).mean(dim=1, keepdim=True))
        if s["grad_h"] is not None:
            dx = dx + s["grad_h"].float()
        return dx.to(dtype), (g * xhat).sum(dim=0).to(s["weight"].dtype)
    if s["op"] == "checkpoint":
        values, scales = _quantize(s["x"].float(), dtype)
        return (values.float() * scales[:, None]).to(dtype), scales
    if s["op"] == "matmul":
        y = (s["values"].float() @ s["weight"].float().t()) * s["scales"][:, None] * s["weight_scales"]
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(dtype)
    g = s["grad"].float()
    dw = (g.t() @ (s["values"].float() * s["scales"][:, None])).to(dtype)
    return (dw, g.sum(dim=0).to(dtype)) if s["bias"] else dw


# --------------------------------------------------------------------------------------------------
# The package's operators


def _run_own(s):
    import optimi_amd as optimi

    dtype = s["dtype"]
    if s["op"] == "norm_forward":
        values, scales, h, rstd = optimi.add_rms_norm_int8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        restored = optimi.int8_dequantize(values, scales, torch.bfloat16)
        return (restored, rstd) if s["residual"] is None else (restored, rstd, h)
    if s["op"] == "norm_backward":
        return optimi.add_rms_norm_int8_backward(s["grad"], s["h"], s["rstd"], s["weight"], grad_h=s["grad_h"])
    if s["op"] == "checkpoint":
        values, scales = optimi.int8_quantize(s["x"])
        return optimi.int8_dequantize(values, scales, dtype), scales
    if s["op"] == "matmul":
        return optimi.int8_matmul(s["values"], s["scales"], s["weight"], s["weight_scales"], bias=s["bias"], dtype=dtype)
    return optimi.int8_weight_grad(s["grad"], s["values"], s["scales"], bias=s["bias"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------------------------------
# Inputs


def _activation(gen, rows, cols, dtype):
    """Token vectors of unlike lengths, with a few loud channels, as transformer activations have them."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.002
    x *= torch.where(loud, 6.0, 1.0)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, cols, op = DTYPES[case["dtype"]], case["rows"], case["cols"], case["op"]
    state = {"op": op, "dtype": dtype}
    if op in ("norm_forward", "norm_backward"):
        state["weight"] = (1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(dtype)
        x = _activation(gen, rows, cols, dtype)
        if op == "norm_forward":
            state["x"] = x
            state["residual"] = _activation(gen, rows, cols, dtype) if case["residual"] else None
        else:
            state["h"] = x
            state["rstd"] = torch.rsqrt((x.float() * x.float()).mean(dim=1) + EPS)
            state["grad"] = (1e-2 * torch.randn(rows, cols, generator=gen, device="cuda")).to(dtype)
            state["grad_h"] = (1e-2 * torch.randn(rows, cols, generator=gen, device="cuda")).to(dtype) if case["residual"] else None
    elif op == "checkpoint":
        state["x"] = _activation(gen, rows, cols, dtype)
    else:
        outs = case["outs"]
        state["values"], state["scales"] = _quantize(_activation(gen, rows, cols, dtype).float(), dtype)
        if op == "matmul":
            w = (torch.randn(outs, cols, generator=gen, device="cuda") / math.sqrt(cols)).to(dtype)
            state["weight"], state["weight_scales"] = _quantize(w.float(), dtype)
            state["bias"] = (0.1 * torch.randn(outs, generator=gen, device="cuda")).to(dtype) if case["bias"] else None
        else:
            state["grad"] = (1e-2 * torch.randn(rows, outs, generator=gen, device="cuda")).to(dtype)
            state["bias"] = case["bias"]
    return state


# --------------------------------------------------------------------------------------------------
# What a case cannot do without


def work(case):
    rows, cols, size = case["rows"], case["cols"], 4 if case["dtype"] == "fp32" else 2
    n = rows * cols
    if case["op"] == "norm_forward":  # the sum in and out, the int8 values written and read once, the bf16 restored
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 1 + 1 + 2) + cols * size + rows * 12, "flops": 8 * n}
    if case["op"] == "norm_backward":
        return {"bytes": n * size * (4 if case["residual"] else 3) + 2 * cols * size + rows * 4, "flops": 12 * n}
    if case["op"] == "checkpoint":
        return {"bytes": n * (size + 1 + 1 + size) + rows * 8, "flops": 4 * n}
    outs = case["outs"]
    if case["op"] == "matmul":
        return {"bytes": n + outs * cols + rows * outs * size + 4 * (rows + outs), "flops": 2 * n * outs}
    return {"bytes": n + rows * outs * size + outs * cols * size + 4 * rows, "flops": 2 * n * outs}


# --------------------------------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_rows(y, top):
    """The values that int8 rows stand for: steps of the smallest power of two >= absmax / 127."""
    absmax = y.abs().max(dim=1, keepdim=True).values
    mantissa, exponent = torch.frexp(absmax / 127)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(min=-126)
    power = ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)  # exactly 2^exponent, which pow() need not give
    step = torch.where(absmax == 0, torch.ones_like(absmax), power)
    most = torch.where(step * 64 > top, 63.0, 127.0).double()
    return torch.clamp(torch.round(y / step), -most, most) * step, step.squeeze(1)


def exact(case, seed):
    s = prepare(case, seed)
    op, dtype = s["op"], s["dtype"]
    top = float(torch.finfo(dtype).max)
    if op == "norm_forward":
        h64 = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        stored = h64.to(dtype).double()  # the norm is that of the sum as it is kept
        rstd = 1 / torch.sqrt(stored.pow(2).sum(dim=1) / case["cols"] + EPS)
        restored, _ = _exact_rows(stored * rstd.unsqueeze(1) * s["weight"].double(), float(torch.finfo(torch.float32).max))
        return (restored, rstd) if s["residual"] is None else (restored, rstd, h64)
    if op == "norm_backward":
        g, w, r = s["grad"].double(), s["weight"].double(), s["rstd"].double().unsqueeze(1)
        h = s["h"].double()
        # d(h_j r) / dh_i = r (delta_ij - r^2 h_i h_j / n)
        inner = torch.einsum("ij,ij->i", g * w, h).unsqueeze(1)
        dx = r * g * w - r.pow(3) / case["cols"] * h * inner
        if s["grad_h"] is not None:
            dx = dx + s["grad_h"].double()
        return dx, torch.einsum("ij,ij->j", g, h * r)
    if op == "checkpoint":
        return _exact_rows(s["x"].double(), top)
    if op == "matmul":
        y = torch.mm(s["values"].double() * s["scales"].double().unsqueeze(1), (s["weight"].double() * s["weight_scales"].double().unsqueeze(1)).t())
        return y if s["bias"] is None else y + s["bias"].double()
    restored = s["values"].double() * s["scales"].double().unsqueeze(1)
    dw = torch.mm(s["grad"].double().t(), restored)
    return (dw, s["grad"].double().sum(dim=0)) if s["bias"] else dw
