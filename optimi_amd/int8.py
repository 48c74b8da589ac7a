"""Training with activations held in 8 bits: the operators, the linear layer made of them, and the
model preparation beside ``prepare_for_gradient_release``.

A linear layer keeps its input for the backward pass; here it keeps it as int8 with one scale per
row (token), half of what 16 bits take, multiplies the same int8 values with the weight's in the
forward pass, and forms the weight gradient from them in 16 bits.  The gradient of the input
is a plain product of the incoming gradient and the weight in their own type: gradients are not
quantized.  The optimizers, gradient release and ``state_dict`` see ordinary parameters and
gradients.  (No counterpart in the reference.)

All functions run HIP kernels on the current stream, take float32, bfloat16 or float16 tensors of
any number of leading dimensions (a non-contiguous one is copied first), raise ``RuntimeError`` for
tensors they cannot take, and may be captured into HIP graphs.  The layers raise ``TypeError`` for tensors of
different types and ``NotImplementedError`` for a weight of any other type than these three.  Tensors that a caller
brings from another stream are the caller's to synchronize, as everywhere in PyTorch.

Gradients flow through ``int8_linear``, ``add_rms_norm_int8_linear`` and the modules, once and in reverse mode: second
derivatives, forward-mode derivatives and ``torch.func`` transforms are refused.  The operators below them (``int8_quantize``
to ``add_rms_norm_int8_backward``) take no part in autograd: what they return has no history, whatever their inputs require.
"""

from __future__ import annotations

import math
import warnings
from contextlib import nullcontext
from typing import Iterable, Sequence

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable
from torch.nn.modules import module as nn_module

from . import backend

__all__ = [
    "int8_quantize", "int8_dequantize", "int8_matmul", "int8_weight_grad", "add_rms_norm_int8", "add_rms_norm_int8_backward",
    "int8_linear", "add_rms_norm_int8_linear", "Int8Linear", "prepare_for_int8_linear", "remove_int8_linear",
]


def int8_quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    """``(values, scales)`` of the rows (last dimension) of ``x``: int8 values in [-127, 127] and one float32
    scale per row, the smallest power of two that holds the row; ``values * scales`` stands for ``x``, at
    most half a scale away.  (Under scales whose 64th multiple x's type does not hold, those of its largest numbers, values stay
    within 63 and less than one scale away.)  Rows of zeros get the scale 1.  A row with an infinity or a NaN gets the scale
    NaN, so that an overflow stays visible.  Not differentiable."""
    return backend.ext().int8_quantize(x)


def int8_dequantize(values: Tensor, scales: Tensor, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``values * scales[..., None]`` in ``dtype``.  Not differentiable."""
    return backend.ext().int8_dequantize(values, scales, dtype)


def int8_matmul(values: Tensor, scales: Tensor, weight_values: Tensor, weight_scales: Tensor, bias: Tensor | None = None,
                dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``(values * scales[..., None]) @ (weight_values * weight_scales[:, None]).T + bias`` in ``dtype``, from int8
    ``values [..., K]`` and ``weight_values [N, K]``; the sums are exact in int32 (K <= 131071).  Not differentiable, the
    bias included."""
    return backend.ext().int8_matmul(values, scales, weight_values, weight_scales, bias, dtype)


def int8_weight_grad(grad: Tensor, values: Tensor, scales: Tensor, bias: bool = False):
    """The weight gradient ``grad.T @ (values * scales[..., None])`` (``[N, K]``, grad's dtype) of a linear layer
    from its incoming gradient ``grad [..., N]`` and the int8 checkpoint of its input ``[..., K]``, summed in
    float32; with ``bias`` also the bias gradient, as ``(weight_grad, bias_grad)``.  Not differentiable.

    Products are those of ``grad`` and ``values * scales`` rounded to grad's type.  bfloat16 holds the latter exactly under scales
    that are powers of two; float16 as long as they are multiples of 2^-24 and within 65504, which those of a float16 tensor are.  Products of
    float32 gradients are exact where ``grad * scales`` lies between 2^-110 and the largest float, but for one rounding under scales
    that are no powers of two."""
    dw, db = backend.ext().int8_weight_grad(grad, values, scales, bias)
    return (dw, db) if bias else dw


def add_rms_norm_int8(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-6) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """``(values, scales, h, rstd)``: the sum ``h = x + residual`` (``x`` itself without a residual), its
    ``rstd = 1 / sqrt(mean(h**2) + eps)`` per row, and the int8 form of ``h * rstd * weight``, which is
    never written in more bits.  ``weight`` has x's dtype or float32.  Finite rows of any size have their norm, also where squares
    leave float32's range.  Not differentiable by itself: see ``add_rms_norm_int8_linear`` and ``add_rms_norm_int8_backward``."""
    return backend.ext().add_rms_norm_int8(x, weight, residual, eps)


def add_rms_norm_int8_backward(grad: Tensor, h: Tensor, rstd: Tensor, weight: Tensor, grad_h: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """``(dx, dweight)`` of the norm for the gradient ``grad`` of its output; ``dx`` is the gradient of ``x`` and of
    ``residual`` alike and contains ``grad_h``, what arrives at ``h`` itself.  Not differentiable."""
    return backend.ext().add_rms_norm_int8_backward(grad, h, rstd, weight, grad_h)


def _check_linear(x: Tensor, weight: Tensor, bias: Tensor | None):
    backend.check_supported(weight)
    if x.dtype != weight.dtype or (bias is not None and bias.dtype != weight.dtype):
        raise TypeError(f"optimi_amd: an int8 linear layer needs input, weight and bias of one dtype, got {x.dtype}, {weight.dtype}"
                        + (f" and {bias.dtype}" if bias is not None else ""))


def _product(values, scales, weight, bias, dtype):
    weight_values, weight_scales = int8_quantize(weight)
    return int8_matmul(values, scales, weight_values, weight_scales, bias, dtype)


def _times_weight(grad: Tensor, weight: Tensor, plus: Tensor | None = None) -> Tensor:
    """``grad @ weight (+ plus)`` as one product of two matrices, whatever grad's dimensions and strides, in their own
    type: a backward pass may be called inside ``torch.autocast``, which would turn them into another one."""
    shape, (n, k) = grad.shape[:-1], weight.shape
    grad = grad.reshape(math.prod(shape), n)
    with torch.autocast("cuda", enabled=False) if torch.is_autocast_enabled("cuda") else nullcontext():
        out = grad.mm(weight) if plus is None else torch.addmm(plus.view(grad.shape[0], k), grad, weight)
    return out.view(*shape, k)


def _parameter_grads(grad, values, scales, need_weight, need_bias):
    if need_weight:
        return backend.ext().int8_weight_grad(grad, values, scales, need_bias)
    return None, backend.ext().int8_bias_grad(grad) if need_bias else None


class _Int8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        values, scales = int8_quantize(x)
        # the checkpoint is for the weight's gradient alone
        ctx.save_for_backward(weight, *((values, scales) if ctx.needs_input_grad[1] else (None, None)))
        return _product(values, scales, weight, bias, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weight, values, scales = ctx.saved_tensors
        dx = _times_weight(grad, weight) if ctx.needs_input_grad[0] else None
        return dx, *_parameter_grads(grad, values, scales, *ctx.needs_input_grad[1:3])


def _autocast(*tensors):
    """Under ``torch.autocast`` a linear layer runs in the autocast dtype, as ``nn.Linear`` does."""
    if not torch.is_autocast_enabled("cuda"):
        return tensors
    dtype = torch.get_autocast_dtype("cuda")
    return tuple(None if t is None else t.to(dtype) for t in tensors)


def int8_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None) -> Tensor:
    """``x @ weight.T + bias`` with x and weight quantized to int8 by rows, differentiable.  The backward pass
    keeps x in 8 bits; quantization passes gradients straight through.  Input, weight and bias are of one dtype;
    under ``torch.autocast`` they are cast to its dtype first."""
    x, weight, bias = _autocast(x, weight, bias)
    _check_linear(x, weight, bias)
    return _Int8Linear.apply(x, weight, bias)


class _AddRmsNormInt8Linear(torch.autograd.Function):
    """The norm in x's type and the layers in theirs, which need not be the same."""

    @staticmethod
    def forward(ctx, x, residual, norm_weight, eps, *layers):
        weights, biases = layers[: len(layers) // 2], layers[len(layers) // 2:]
        values, scales, h, rstd = add_rms_norm_int8(x, norm_weight, residual, eps)
        ctx.set_materialize_grads(False)
        ctx.with_residual = residual is not None
        # the checkpoint is for the weights' gradients alone, the sum for the norm's
        checkpoint = (values, scales) if any(ctx.needs_input_grad[4:4 + len(weights)]) else (None, None)
        kept = (h, rstd, norm_weight) if any(ctx.needs_input_grad[:3]) else (None, None, None)
        ctx.save_for_backward(*checkpoint, *kept, *weights)
        outs = tuple(_product(values, scales, w, b, w.dtype) for w, b in zip(weights, biases))
        return (h, *outs) if ctx.with_residual else outs

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        values, scales, h, rstd, norm_weight, *weights = ctx.saved_tensors
        grad_h, grads = (grads[0], grads[1:]) if ctx.with_residual else (None, grads)
        n = len(weights)
        need_x, need_residual, need_norm = ctx.needs_input_grad[:3]
        dws, dbs, dy = [None] * n, [None] * n, None
        for i, (grad, weight) in enumerate(zip(grads, weights)):
            if grad is None:
                continue
            if need_x or need_residual or need_norm:
                dy = _times_weight(grad, weight, plus=dy)
            dws[i], dbs[i] = _parameter_grads(grad, values, scales, ctx.needs_input_grad[4 + i], ctx.needs_input_grad[4 + n + i])
        dx, dnorm = grad_h, None
        if dy is not None:
            dx, dnorm = add_rms_norm_int8_backward(dy.to(h.dtype), h, rstd, norm_weight, grad_h)
        return (dx if need_x else None, dx if need_residual else None, dnorm if need_norm else None, None, *dws, *dbs)


def add_rms_norm_int8_linear(x: Tensor, norm_weight: Tensor, weights: Sequence[Tensor], biases: Sequence[Tensor | None] | None = None,
                             residual: Tensor | None = None, eps: float = 1e-6) -> tuple[tuple[Tensor, ...], Tensor]:
    """``(outputs, h)``: ``h = x + residual`` (``x`` itself without a residual) and, for every weight, the int8 linear
    layer of ``rms_norm(h) * norm_weight``, differentiable.  The normed activation exists as int8 only: one checkpoint
    that all the layers (query, key and value, or gate and up) multiply and all their weight gradients read.  ``norm_weight`` has
    x's dtype or float32; ``torch.autocast`` casts as in ``int8_linear`` (and ``h`` is of the autocast dtype then)."""
    weights = tuple(weights)
    biases = (None,) * len(weights) if biases is None else tuple(biases)
    if not weights or len(biases) != len(weights):
        raise ValueError(f"optimi_amd: got {len(weights)} weights and {len(biases)} biases")
    x, residual = _autocast(x, residual)
    weights, biases = _autocast(*weights), _autocast(*biases)
    for w, b in zip(weights, biases):
        _check_linear(x, w, b)
    outs = _AddRmsNormInt8Linear.apply(x, residual, norm_weight, eps, *weights, *biases)
    return (outs, x) if residual is None else (outs[1:], outs[0])


class Int8Linear(nn.Linear):
    """``nn.Linear`` computed by ``int8_linear``; parameters and ``state_dict`` are nn.Linear's."""

    def forward(self, x: Tensor) -> Tensor:
        return int8_linear(x, self.weight, self.bias)


def _only_forward(module: nn.Module) -> bool:
    """Whether a call of the module is its class's forward() and nothing else: no hooks of its own or on all modules, no
    forward() of the instance, not compiled."""
    return not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks
                or nn_module._global_forward_hooks or nn_module._global_forward_pre_hooks or nn_module._global_backward_hooks
                or nn_module._global_backward_pre_hooks or "forward" in module.__dict__ or module._compiled_call_impl is not None)


def _is_norm_of(norm: nn.Module, layer: nn.Module) -> bool:
    return (type(norm) is nn.RMSNorm and type(layer) is Int8Linear and norm.elementwise_affine
            and tuple(norm.normalized_shape) == (layer.in_features,) and _only_forward(norm) and _only_forward(layer))


def _types_fit(x: Tensor, norm: nn.Module, layer: nn.Module) -> bool:
    """Whether the operators take these types together; torch's own modules take more of them."""
    return (x.dtype in backend.SUPPORTED_DTYPES and norm.weight.dtype in (x.dtype, torch.float32)
            and (layer.weight.dtype == x.dtype or torch.is_autocast_enabled("cuda")))


def _norm_layer(x: Tensor, norm: nn.Module, layer: nn.Module) -> Tensor:
    """Under ``torch.autocast`` the layer is cast and the norm is not: its input may be a residual stream of more bits."""
    weight, bias = _autocast(layer.weight, layer.bias)
    _check_linear(weight, weight, bias)
    # nn.RMSNorm without an eps adds that of the type it computes in
    eps = torch.finfo(torch.float32).eps if norm.eps is None else norm.eps
    (y,) = _AddRmsNormInt8Linear.apply(x, None, norm.weight, eps, weight, bias)
    return y


class _Int8Sequential(nn.Sequential):
    """Runs an RMSNorm that is directly followed by an Int8Linear as one node, where their types allow it."""

    def forward(self, x):
        modules = list(self)
        i = 0
        while i < len(modules):
            if i + 1 < len(modules) and _is_norm_of(modules[i], modules[i + 1]) and _types_fit(x, modules[i], modules[i + 1]):
                x = _norm_layer(x, modules[i], modules[i + 1])
                i += 2
            else:
                x = modules[i](x)
                i += 1
        return x


_PREPARED = {nn.Linear: Int8Linear, nn.Sequential: _Int8Sequential}
_MODULES_ATTR = "_int8_linear_modules"
_MOST_INPUTS = 131071  # that a sum of int8 products in 32 bits holds


def prepare_for_int8_linear(model: nn.Module, skip: Iterable[str] = ()) -> nn.Module:
    """Makes every ``nn.Linear`` of ``model`` (in place; itself included) an ``Int8Linear``, except those whose qualified
    name contains one of the strings in ``skip``, and lets an ``nn.RMSNorm`` directly before one in an ``nn.Sequential``
    hand it int8 values, where their types go together and nothing hooks or replaces their calls (under ``torch.autocast`` the
    norm takes its input as it comes, the layer runs in the autocast type).  Subclasses of these modules and layers of more
    than 131071 inputs are left alone.  Parameters stay the same objects: optimizers built before or after, gradient release
    and checkpoints work as they did.  ``ValueError`` if the model is prepared already or holds no such layer.  Undo with
    ``remove_int8_linear``.

    The layers run on a HIP device only.  Every forward pass quantizes the weight again, so there is little to win with few rows:
    forward and backward of a bfloat16 layer take 0.84 to 0.95 of nn.Linear's time at 8192 rows (4096 to 11008 inputs and outputs;
    0.79 to 0.96 at 4096) and about the same up to 1024.  A serving loop quantizes its weights once and calls ``int8_matmul``."""
    if isinstance(skip, str):
        skip = (skip,)
    skip = tuple(skip)
    if hasattr(model, _MODULES_ATTR):
        raise ValueError("`model` is prepared for int8 linear layers already.")
    layers = [m for name, m in model.named_modules()
              if type(m) is nn.Linear and m.in_features <= _MOST_INPUTS and not any(s in name for s in skip)]
    if not layers:
        raise ValueError("`model` has no `nn.Linear` to compute in int8.")
    changed = layers + [m for m in model.modules() if type(m) is nn.Sequential]
    for module in changed:
        module.__class__ = _PREPARED[type(module)]
    object.__setattr__(model, _MODULES_ATTR, changed)
    return model


def remove_int8_linear(model: nn.Module) -> nn.Module:
    """Gives the layers that ``prepare_for_int8_linear`` changed their former classes; warns if there are none."""
    changed = getattr(model, _MODULES_ATTR, None)
    if changed is None:
        warnings.warn("`model` has no int8 linear layers to remove.")
        return model
    back = {new: old for old, new in _PREPARED.items()}
    for module in changed:
        if type(module) in back:
            module.__class__ = back[type(module)]
    object.__delattr__(model, _MODULES_ATTR)
    return model
