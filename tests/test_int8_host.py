"""What the int8 operators refuse before any device work, at the C boundary and in Python, and the model preparation's
bookkeeping; no GPU is touched."""

import copy
import ctypes
import pickle
import warnings

import pytest
import torch
from torch import nn

import optimi_amd as optimi
from optimi_amd import cabi

P = ctypes.c_void_p(256)  # never dereferenced: every call below is refused or has nothing to do
ODD = ctypes.c_void_p(257)
HUGE = 1 << 31


def test_quantize_and_dequantize_check_their_arguments():
    L = cabi.lib()
    assert L.optimi_hip_int8_quantize(P, 4, 8, 7, P, P, None) == -3
    assert L.optimi_hip_int8_quantize(P, -1, 8, cabi.F32, P, P, None) == -2
    assert L.optimi_hip_int8_quantize(P, 4, HUGE, cabi.F32, P, P, None) == -2
    assert L.optimi_hip_int8_quantize(P, HUGE, 4, cabi.F32, P, P, None) == -2
    assert L.optimi_hip_int8_quantize(None, 4, 8, cabi.F32, P, P, None) == -1
    assert L.optimi_hip_int8_quantize(P, 4, 8, cabi.F32, P, None, None) == -1
    assert L.optimi_hip_int8_quantize(ODD, 4, 8, cabi.BF16, P, P, None) == -4
    assert L.optimi_hip_int8_quantize(None, 0, 8, cabi.F32, None, None, None) == 0
    assert L.optimi_hip_int8_dequantize(P, P, 4, 8, 3, P, None) == -3
    assert L.optimi_hip_int8_dequantize(P, P, 4, -8, cabi.F32, P, None) == -2
    assert L.optimi_hip_int8_dequantize(P, None, 4, 8, cabi.F32, P, None) == -1
    assert L.optimi_hip_int8_dequantize(P, P, 4, 8, cabi.F32, ODD, None) == -4
    assert L.optimi_hip_int8_dequantize(None, None, 4, 0, cabi.F32, None, None) == 0


def test_products_check_their_arguments():
    L = cabi.lib()
    mm = L.optimi_hip_int8_matmul
    assert mm(P, P, P, P, None, 4, 4, 8, 9, P, P, None) == -3
    assert mm(P, P, P, P, None, -4, 4, 8, cabi.F32, P, P, None) == -2
    assert mm(P, P, P, P, None, 4, 4, 131072, cabi.F32, P, P, None) == -2
    assert mm(P, P, P, P, None, 4, HUGE, 8, cabi.F32, P, P, None) == -2
    assert mm(None, P, P, P, None, 4, 4, 8, cabi.F32, P, P, None) == -1
    assert mm(P, P, P, P, ODD, 4, 4, 8, cabi.F32, P, P, None) == -4
    assert mm(P, P, P, P, None, 4, 4, 8, cabi.BF16, ODD, P, None) == -4
    assert mm(None, None, None, None, None, 0, 4, 8, cabi.F32, None, None, None) == 0
    assert L.optimi_hip_int8_matmul_workspace(4, 4, 131072) == -2
    assert L.optimi_hip_int8_matmul_workspace(-1, 4, 8) == -2
    assert L.optimi_hip_int8_matmul_workspace(4096, 4096, 4096) >= 0
    wg = L.optimi_hip_int8_weight_grad
    assert wg(P, P, P, 4, 4, 8, 5, P, None, P, None) == -3
    assert wg(P, P, P, 4, -4, 8, cabi.F32, P, None, P, None) == -2
    assert wg(None, P, P, 4, 4, 8, cabi.F32, P, None, P, None) == -1
    assert wg(P, P, P, 4, 4, 8, cabi.F32, None, None, P, None) == -1
    assert wg(P, P, P, 4096, 512, 512, cabi.F32, P, P, None, None) == -1  # a sum that is split needs the workspace
    assert wg(P, P, P, 4, 4, 8, cabi.F32, ODD, None, P, None) == -4
    assert wg(None, None, None, 4, 0, 8, cabi.F32, None, None, None, None) == 0
    assert L.optimi_hip_int8_weight_grad_workspace(4, 4, 8, 5, 0) == -3
    assert L.optimi_hip_int8_weight_grad_workspace(4, 4, HUGE, cabi.F32, 0) == -2
    assert L.optimi_hip_int8_weight_grad_workspace(4096, 512, 512, cabi.F32, 1) >= 512 * 4


def test_the_norm_checks_its_arguments():
    L = cabi.lib()
    f, b = L.optimi_hip_add_rms_norm_int8, L.optimi_hip_add_rms_norm_int8_backward
    assert f(P, P, P, 4, 8, cabi.BF16, cabi.F16, 1e-6, P, P, P, P, None) == -3
    assert f(P, P, P, 4, -8, cabi.BF16, cabi.F32, 1e-6, P, P, P, P, None) == -2
    assert f(P, P, P, 4, 0, cabi.BF16, cabi.F32, 1e-6, P, P, P, P, None) == -2
    assert f(P, P, P, 4, 8, cabi.BF16, cabi.BF16, -1e-6, P, P, P, P, None) == -7
    assert f(P, P, P, 4, 8, cabi.BF16, cabi.BF16, float("nan"), P, P, P, P, None) == -7
    assert f(P, P, P, 4, 8, cabi.BF16, cabi.BF16, 1e-6, None, P, P, P, None) == -1  # a residual needs h
    assert f(P, ODD, P, 4, 8, cabi.BF16, cabi.BF16, 1e-6, P, P, P, P, None) == -4
    assert f(None, None, None, 0, 8, cabi.BF16, cabi.BF16, 1e-6, None, None, None, None, None) == 0
    assert b(P, None, P, P, P, 4, 8, cabi.F16, cabi.BF16, P, P, P, None) == -3
    assert b(P, None, P, P, P, 4, 0, cabi.F16, cabi.F16, P, P, P, None) == -2
    assert b(P, None, P, P, P, 4, 8, cabi.F16, cabi.F16, P, None, P, None) == -1
    assert b(P, None, P, P, P, 4, 8, cabi.F16, cabi.F16, P, P, None, None) == -1
    assert b(P, ODD, P, P, P, 4, 8, cabi.F16, cabi.F16, P, P, P, None) == -4
    assert L.optimi_hip_add_rms_norm_int8_backward_workspace(-1, 8) == -2
    assert L.optimi_hip_add_rms_norm_int8_backward_workspace(100, 8) >= 8 * 4


def test_tensors_on_the_cpu_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    for call in (lambda: optimi.int8_quantize(x), lambda: optimi.int8_dequantize(q, s), lambda: optimi.int8_matmul(q, s, q, s),
                 lambda: optimi.int8_weight_grad(w[:4], q, s), lambda: optimi.add_rms_norm_int8(x, torch.ones(8)),
                 lambda: optimi.add_rms_norm_int8_backward(x, x, s, torch.ones(8)), lambda: optimi.int8_linear(x, w),
                 lambda: optimi.Int8Linear(8, 6)(x)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def model():
    return nn.Sequential(nn.RMSNorm(8), nn.Linear(8, 16), nn.ModuleDict({"proj": nn.Linear(16, 4), "lm_head": nn.Linear(4, 4, bias=False)}))


def test_preparation_changes_linear_layers_and_nothing_else():
    m = model()
    state, params = {k: v.clone() for k, v in m.state_dict().items()}, list(m.parameters())
    assert optimi.prepare_for_int8_linear(m, skip="lm_head") is m
    assert type(m[1]) is optimi.Int8Linear and type(m[2]["proj"]) is optimi.Int8Linear and type(m[2]["lm_head"]) is nn.Linear
    assert isinstance(m, nn.Sequential) and isinstance(m[1], nn.Linear) and type(m[0]) is nn.RMSNorm
    assert all(a is b for a, b in zip(params, m.parameters()))
    assert list(m.state_dict()) == list(state) and all(torch.equal(state[k], v) for k, v in m.state_dict().items())
    with pytest.raises(ValueError, match="already"):
        optimi.prepare_for_int8_linear(m)
    twin, sent = copy.deepcopy(m), pickle.loads(pickle.dumps(m))
    optimi.remove_int8_linear(m)
    assert type(m) is nn.Sequential and type(m[1]) is nn.Linear and not hasattr(m, "_int8_linear_modules")
    for other in (twin, sent):  # copies stand on their own
        assert type(other[1]) is optimi.Int8Linear
        optimi.remove_int8_linear(other)
        assert type(other) is nn.Sequential and type(other[1]) is nn.Linear
    with pytest.warns(UserWarning, match="no int8 linear"):
        optimi.remove_int8_linear(m)


def test_preparation_leaves_subclasses_alone_and_refuses_models_without_layers():
    class Special(nn.Linear):
        pass

    m = nn.ModuleList([Special(4, 4), nn.Linear(4, 4)])
    optimi.prepare_for_int8_linear(m)
    assert type(m[0]) is Special and type(m[1]) is optimi.Int8Linear
    with pytest.raises(ValueError, match="no `nn.Linear`"):
        optimi.prepare_for_int8_linear(nn.Sequential(nn.RMSNorm(4)))
    one = nn.Linear(3, 3)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        optimi.prepare_for_int8_linear(one)
        assert type(one) is optimi.Int8Linear
        optimi.remove_int8_linear(one)
    assert type(one) is nn.Linear
