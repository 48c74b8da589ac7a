"""What the int8 operators refuse and what a prepared model runs as before, at the edges; no GPU is touched."""

import ctypes

import pytest
import torch
from torch import nn

import optimi_amd as optimi
from optimi_amd import cabi, int8

P = ctypes.c_void_p(256)  # never dereferenced: every call below is refused
UNALIGNED = ctypes.c_void_p(264)


# ---------------------------------------------------------------------------------- sizes

@pytest.mark.parametrize("m,n,k", [(1 << 30, 1 << 28, 8), (1 << 30, 1 << 28, 7), (5, 4, 131072), (-1, 4, 8), (4, 1 << 29, 8), (1 << 31, 4, 8)])
def test_matmul_and_its_workspace_refuse_the_same_sizes(m, n, k):
    L = cabi.lib()
    for dtype in (cabi.F32, cabi.BF16, cabi.F16):
        assert L.optimi_hip_int8_matmul(P, P, P, P, None, m, n, k, dtype, P, P, None) == -2
    assert L.optimi_hip_int8_matmul_workspace(m, n, k) == -2


def test_the_widest_weight_is_taken_for_any_number_of_rows():
    for m in (1, 4, 5, 64):
        assert cabi.lib().optimi_hip_int8_matmul_workspace(m, 1 << 28, 16) == 0


@pytest.mark.parametrize("rows,outs,cols", [(64, 1 << 24, 1 << 24), (8, (1 << 24) + 1, 4), (8, 4, (1 << 24) + 1), (1 << 31, 4, 4), (8, -1, 4), (8, 4, -1)])
def test_weight_grad_and_its_workspace_refuse_the_same_sizes(rows, outs, cols):
    L = cabi.lib()
    for dtype in (cabi.F32, cabi.BF16, cabi.F16):
        for bias in (None, P):
            assert L.optimi_hip_int8_weight_grad(P, P, P, rows, outs, cols, dtype, P, bias, P, None) == -2
            assert L.optimi_hip_int8_weight_grad_workspace(rows, outs, cols, dtype, bias is not None) == -2


def test_the_norm_and_its_workspace_refuse_the_same_sizes():
    L = cabi.lib()
    for rows, cols in ((5, 0), (0, 0), (-1, 8), (5, -8), (1 << 31, 8), (5, 1 << 29)):
        assert L.optimi_hip_add_rms_norm_int8_backward(P, None, P, P, P, rows, cols, cabi.BF16, cabi.BF16, P, P, P, None) == -2
        assert L.optimi_hip_add_rms_norm_int8_backward_workspace(rows, cols) == -2


def test_a_product_too_large_for_small_tiles_asks_for_alignment():
    """Operands off the 16-byte grid go through 64 x 64 tiles; where a launch cannot hold so many, that is said."""
    L = cabi.lib()
    m, n, k = 1 << 20, 1 << 17, 64
    assert L.optimi_hip_int8_matmul_workspace(m, n, k) == 0
    assert L.optimi_hip_int8_matmul(UNALIGNED, P, P, P, None, m, n, k, cabi.BF16, P, None, None) == -4


# ---------------------------------------------------------------------------------- which modules run as one node

@pytest.fixture
def ran(monkeypatch):
    """Torch operations in the operators' place; records whether a prepared sequence ran a layer by itself or with its norm."""
    calls = []

    def linear(x, weight, bias=None):
        calls.append("linear")
        return nn.functional.linear(x, weight, bias)

    def norm(x, weight, residual=None, eps=1e-6):
        calls.append("fused")
        return nn.functional.rms_norm(x, weight.shape, weight, eps), torch.ones(len(x)), x, torch.ones(len(x))

    monkeypatch.setattr(int8, "int8_linear", linear)
    monkeypatch.setattr(int8, "add_rms_norm_int8", norm)
    monkeypatch.setattr(int8, "int8_quantize", lambda x: (x, None))
    monkeypatch.setattr(int8, "int8_matmul", lambda x, sx, w, sw, bias, dtype: nn.functional.linear(x, w, bias))
    monkeypatch.setattr(int8.backend, "check_supported", lambda t: None)
    return calls


def sequence(norm_dtype=torch.float32, layer_dtype=torch.float32):
    torch.manual_seed(0)
    plain = nn.Sequential(nn.RMSNorm(8, eps=1e-5).to(norm_dtype), nn.Linear(8, 4).to(layer_dtype))
    return optimi.prepare_for_int8_linear(plain)


@pytest.mark.parametrize("x,norm,layer,want", [
    (torch.float32, torch.float32, torch.float32, "fused"),
    (torch.bfloat16, torch.bfloat16, torch.bfloat16, "fused"),
    (torch.float32, torch.bfloat16, torch.float32, "linear"),
    (torch.float32, torch.float16, torch.float32, "linear"),
])
def test_the_types_decide_whether_a_norm_and_its_layer_are_one(ran, x, norm, layer, want):
    model = sequence(norm, layer)
    plain = nn.Sequential(*(optimi.remove_int8_linear(sequence(norm, layer))))
    t = torch.randn(3, 8).to(x)
    y, y0 = model(t), plain(t)
    assert ran == [want]
    assert y.dtype == y0.dtype and torch.allclose(y.float(), y0.float(), rtol=0.02, atol=0.02)


def test_types_that_torch_refuses_are_refused(ran):
    model = sequence(torch.float32, torch.bfloat16)
    with pytest.raises(RuntimeError):
        model(torch.randn(3, 8))
    assert "fused" not in ran


# ---------------------------------------------------------------------------------- modules that someone else has to see called

@pytest.mark.parametrize("at", [0, 1])
def test_a_forward_of_its_own_is_called(ran, at):
    """Libraries that offload or move modules replace the instance's forward."""
    model = sequence()
    inner, seen = model[at].forward, []

    def wrapped(x):
        seen.append(at)
        return inner(x)

    model[at].forward = wrapped
    x = torch.randn(3, 8)
    model(x)
    assert seen == [at] and ran == ["linear"]
    del model[at].forward
    model(x)
    assert ran == ["linear", "fused"]


def test_a_compiled_module_is_called(ran):
    model, seen = sequence(), []
    model[0]._compiled_call_impl = lambda x: seen.append(1) or x
    model(torch.randn(3, 8))
    assert seen == [1] and ran == ["linear"]


@pytest.mark.parametrize("register", [nn.modules.module.register_module_forward_hook, nn.modules.module.register_module_forward_pre_hook,
                                      nn.modules.module.register_module_full_backward_hook, nn.modules.module.register_module_full_backward_pre_hook])
def test_hooks_on_all_modules_see_every_module(ran, register):
    model, seen = sequence(), []
    handle = register(lambda module, *args: seen.append(type(module).__name__))
    try:
        model(torch.randn(3, 8, requires_grad=True)).sum().backward()
    finally:
        handle.remove()
    assert "RMSNorm" in seen and "Int8Linear" in seen and ran == ["linear"]
    model(torch.randn(3, 8))
    assert ran == ["linear", "fused"]


# ---------------------------------------------------------------------------------- layers that the product cannot take

def test_preparation_leaves_layers_alone_that_are_too_wide():
    """The product's sums hold 131071 inputs; a layer of more goes on as it was."""
    with torch.device("meta"):
        model = nn.Sequential(nn.RMSNorm(131072), nn.Linear(131072, 2), nn.Linear(2, 131072), nn.Linear(131071, 2))
    optimi.prepare_for_int8_linear(model)
    assert [type(m) for m in model] == [nn.RMSNorm, nn.Linear, optimi.Int8Linear, optimi.Int8Linear]
    with torch.device("meta"):
        wide = nn.Sequential(nn.Linear(131072, 2))
    with pytest.raises(ValueError, match="no `nn.Linear`"):
        optimi.prepare_for_int8_linear(wide)
