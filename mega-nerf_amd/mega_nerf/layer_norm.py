"""Layer norm over the last dimension, forward and backward (csrc/layer_norm.hip): what a trunk or a gate wider than the reference's
plain ReLU layers (nerf.py:62-113) is normalised with, beside the layer-by-layer kernels of csrc/layerwise.hip.

``layer_norm`` is the differentiable call.  ``layer_norm_forward`` / ``layer_norm_backward`` are its two passes for callers that keep
their own tape (as models.layerwise does): they record nothing for autograd, whatever their inputs require, and may be recorded into a
HIP graph, which the autograd node refuses: a graph's backward pass is recorded from the explicit call."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from mega_nerf import _native as N


def _check(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]) -> Tuple[int, int]:
    code = N.element_type(x, 'x')
    if x.dim() == 0 or x.shape[-1] == 0:
        raise N.NativeError('layer_norm needs a last dimension of one element at least (got shape {})'.format(tuple(x.shape)))
    wcode = 0
    for t, name in ((weight, 'weight'), (bias, 'bias')):
        if t is None:
            continue
        wcode = N.element_type(t, name)
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise N.NativeError('{} must have shape {} (got {})'.format(name, tuple(x.shape[-1:]), tuple(t.shape)))
        N.on_device_of(x, t, name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise N.NativeError('weight and bias must be of one type (got {} and {})'.format(weight.dtype, bias.dtype))
    return code, wcode


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): y like ``x`` [..., C]; mean and rstd fp32 [rows], what :func:`layer_norm_backward` reads.  float32, float16 or
    bfloat16; ``weight`` / ``bias`` [C] of any of them."""
    code, wcode = _check(x, weight, bias)
    shape = x.shape
    x, rows, cols, ldx = N.matrix(x)
    w = weight.contiguous() if weight is not None else None
    b = bias.contiguous() if bias is not None else None
    y = x.new_empty(shape)
    mean = x.new_empty(rows, dtype=torch.float32)
    rstd = x.new_empty(rows, dtype=torch.float32)
    N.launch(x, N.lib().mnr_layer_norm_forward, y.data_ptr(), cols, mean.data_ptr(), rstd.data_ptr(), x.data_ptr(), ldx, N.ptr(w), N.ptr(b), rows, cols,
             eps, code, wcode)
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor,
                        need: Tuple[bool, bool, bool] = (True, True, True)) -> Tuple[Optional[torch.Tensor], ...]:
    """(dx, dweight, dbias) for d(loss)/dy = ``dy``; ``need`` says which are wanted (None in the others' places).  Without a weight
    the column sums are fp32.  The same inputs give the same bits."""
    code, wcode = _check(x, weight, None)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise N.NativeError('dy must be like x: {} {} (got {} {})'.format(tuple(x.shape), x.dtype, tuple(dy.shape), dy.dtype))
    N.on_device_of(x, dy, 'dy')
    x, rows, cols, ldx = N.matrix(x)
    g, _, _, ldg = N.matrix(dy)
    for t, name in ((mean, 'mean'), (rstd, 'rstd')):
        if t.dtype != torch.float32 or t.numel() != rows:
            raise N.NativeError('{} must be float32 with {} elements, as layer_norm_forward returned it'.format(name, rows))
        N.on_device_of(x, t, name)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    w = weight.contiguous() if weight is not None else None
    dx = x.new_empty(dy.shape) if need[0] else None
    wtype = weight.dtype if weight is not None else torch.float32
    dw = x.new_empty(cols, dtype=wtype) if need[1] else None
    db = x.new_empty(cols, dtype=wtype) if need[2] else None
    lib = N.lib()
    size = lib.mnr_layer_norm_backward_workspace_bytes(rows, cols, code) if need[1] or need[2] else 0
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    N.launch(x, lib.mnr_layer_norm_backward, N.ptr(dx), cols, N.ptr(dw), N.ptr(db), g.data_ptr(), ldg, x.data_ptr(), ldx, N.ptr(w), mean.data_ptr(),
             rstd.data_ptr(), rows, cols, code, wcode, N.ptr(ws), size)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_type = bias.dtype if bias is not None else None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        N.refuse_captured_backward('layer_norm')
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy, x, weight, mean, rstd, ctx.needs_input_grad[:3])
        if db is not None and db.dtype != ctx.bias_type:
            db = db.to(ctx.bias_type)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, differentiable in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps)
