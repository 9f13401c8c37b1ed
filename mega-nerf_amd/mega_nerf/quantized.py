"""Matrix product in 8-bit integers with a scale for every row of the input and every output channel (csrc/int8_product.hip): the dense
layers of a wide model served at a quarter of the bytes and on the 8-bit matrix pipe, beside the fp32 products of csrc/tgemm.hip and
csrc/layerwise.hip.  Inference only: quantisation has no gradient here.  A parameter counts as a constant; what a recorded computation
has produced is refused, since its gradient would end here without a word."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from mega_nerf import _native as N

_PITCH = 128                 # rows of quantised values start at multiples of this many bytes


class QuantizedRows(NamedTuple):
    """``values`` int8 [rows, cols] and ``scale`` float32 [rows]: row r stands for scale[r] * values[r]."""
    values: torch.Tensor
    scale: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        return self.values.float() * self.scale[:, None]


def _refuse_recorded(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.grad_fn is not None for t in tensors):
        raise NotImplementedError('{} is inference-only (use torch.no_grad())'.format(what))


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """``x`` [rows, cols] (float32, float16, bfloat16) with the scale max|row| / 127 for each row; values are rounded to the nearest,
    ties to even.  A row of zeros gets scale 0; a row that holds an inf or NaN gets scale NaN.  A weight [out, in] is quantised the
    same way, once: its rows are the output channels.  The values' rows start 128 bytes apart or a multiple of it, zeros in between
    (what the product reads fastest)."""
    _refuse_recorded('quantize_rows', x)
    code = N.element_type(x, 'x')
    if x.dim() != 2 or x.shape[1] == 0:
        raise N.NativeError('quantize_rows expects [rows, cols] with a column at least (got {})'.format(tuple(x.shape)))
    x, rows, cols, ldx = N.matrix(x)
    pitch = (cols + _PITCH - 1) // _PITCH * _PITCH
    values = x.new_empty((rows, pitch), dtype=torch.int8)
    scale = x.new_empty(rows, dtype=torch.float32)
    N.launch(x, N.lib().mnr_quantize_rows, values.data_ptr(), pitch, scale.data_ptr(), x.data_ptr(), ldx, rows, cols, code)
    return QuantizedRows(values[:, :cols] if pitch > cols else values, scale)


def _operand(q: QuantizedRows, name: str, zero_tail: bool):
    """(tensor, scale, rows, cols, pitch) of values that the kernel can read as they lie, else of a copy: 16-byte aligned rows, readable
    up to the next multiple of 16 columns, and for the left operand zeros there (its tail cannot be known, so it is copied)."""
    v, s = q
    if v.dtype != torch.int8 or v.dim() != 2 or v.shape[1] == 0:
        raise N.NativeError('{}.values must be int8 [rows, cols] with a column at least (got {} {})'.format(name, v.dtype, tuple(v.shape)))
    if not v.is_cuda:
        N.require_device(v, name + '.values')
    rows, cols = v.shape
    if s.dtype != torch.float32 or s.dim() != 1 or s.shape[0] != rows:
        raise N.NativeError('{}.scale must be float32 [{}] (got {} {})'.format(name, rows, s.dtype, tuple(s.shape)))
    N.on_device_of(v, s, name + '.scale')
    up = (cols + 15) // 16 * 16
    pitch = v.stride(0) if rows > 1 else up
    if not (v.stride(1) == 1 and pitch % 16 == 0 and pitch >= up and pitch < 1 << 22 and v.data_ptr() % 16 == 0 and not (zero_tail and up > cols) and
            v.storage_offset() + max(rows - 1, 0) * pitch + up <= v.untyped_storage().nbytes()):
        pitch = (cols + _PITCH - 1) // _PITCH * _PITCH
        held = v.new_zeros((rows, pitch))
        held[:, :cols] = v
        v = held
    return v, s.contiguous(), rows, cols, pitch


def _epilogue(x: torch.Tensor, n: int, bias: Optional[torch.Tensor], out_dtype: torch.dtype):
    if bias is not None:
        if bias.dtype != torch.float32 or bias.dim() != 1 or bias.shape[0] != n:
            raise N.NativeError('bias must be float32 [{}] (got {} {})'.format(n, bias.dtype, tuple(bias.shape)))
        N.on_device_of(x, bias, 'bias')
        bias = bias.contiguous()
    code = N.ELEMENT_TYPES.get(out_dtype)
    if code is None:
        raise N.NativeError('the output is float32, float16 or bfloat16 (got {})'.format(out_dtype))
    return bias, code


def int8_product(a: QuantizedRows, b: QuantizedRows, bias: Optional[torch.Tensor] = None, relu: bool = False,
                 out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[M, N] = a [M, K] times the transpose of b [N, K] (+ bias float32 [N], ReLU): the integer sums are exact (K <= 131071), scaled in
    fp32 and rounded once to ``out_dtype``."""
    _refuse_recorded('int8_product', a[1], b[1], bias)
    av, sa, m, k, lda = _operand(a, 'a', True)
    bv, sb, n, kb, ldb = _operand(b, 'weight', False)
    N.on_device_of(av, bv, 'weight')
    if kb != k:
        raise N.NativeError('the input has {} columns, the weight {}'.format(k, kb))
    bias, code = _epilogue(av, n, bias, out_dtype)
    y = av.new_empty((m, n), dtype=out_dtype)
    N.launch(av, N.lib().mnr_int8_product, y.data_ptr(), n, av.data_ptr(), lda, sa.data_ptr(), bv.data_ptr(), ldb, sb.data_ptr(), N.ptr(bias), m, n, k,
             1 if relu else 0, code)
    return y


def int8_linear(x: torch.Tensor, weight: QuantizedRows, bias: Optional[torch.Tensor] = None, relu: bool = False,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A dense layer served in 8 bits: x [..., K] is quantised row by row (as :func:`quantize_rows`), multiplied with ``weight`` =
    ``quantize_rows(w)`` of an nn.Linear weight [N, K], scaled, ``bias`` added, ReLU if ``relu``; [..., N] of x's type, or
    ``out_dtype``."""
    if x.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError('int8_linear is inference-only (use torch.no_grad())')
    _refuse_recorded('int8_linear', weight[1], bias)
    xcode = N.element_type(x, 'x')
    shape = x.shape
    if x.dim() == 0 or shape[-1] == 0:
        raise N.NativeError('int8_linear expects [..., K] with a column at least (got {})'.format(tuple(shape)))
    x, m, k, ldx = N.matrix(x)
    bv, sb, n, kb, ldb = _operand(weight, 'weight', False)
    N.on_device_of(x, bv, 'weight')
    if kb != k:
        raise N.NativeError('the input has {} columns, the weight {}'.format(k, kb))
    out_dtype = x.dtype if out_dtype is None else out_dtype
    bias, code = _epilogue(x, n, bias, out_dtype)
    y = x.new_empty(shape[:-1] + (n,), dtype=out_dtype)
    lib = N.lib()
    size = lib.mnr_int8_linear_workspace_bytes(m, k)
    ws = x.new_empty(size, dtype=torch.uint8)
    N.launch(x, lib.mnr_int8_linear, y.data_ptr(), n, x.data_ptr(), ldx, xcode, bv.data_ptr(), ldb, sb.data_ptr(), N.ptr(bias), m, n, k, 1 if relu else 0,
             code, ws.data_ptr(), size)
    return y
