"""Table lookup with a scale, and the table's gradient by sorted indices (csrc/embedding.hip): the per-image appearance vectors of
nerf.py:84-85,149 outside the fused kernels, in any width and type.  Sums are free of atomics and in a fixed order: the same inputs give
the same bits (``mnr_scatter_rows`` of the layer-by-layer path adds with atomics: its last bits change from run to run).

``embedding`` is the differentiable call; ``embedding_forward`` / ``embedding_backward`` are its passes for callers with a tape of their
own: they record nothing for autograd, and may be recorded into a HIP graph."""
from __future__ import annotations

from typing import Optional

import torch

from mega_nerf import _native as N


def _index(idx: torch.Tensor, like: torch.Tensor):
    code = N.INDEX_TYPES.get(idx.dtype)
    if code is None:
        raise N.NativeError('indices must be int32, int64 or float32 (got {})'.format(idx.dtype))
    N.on_device_of(like, idx, 'idx')
    return idx.contiguous(), code


def embedding_forward(idx: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[idx]``: [*idx.shape, width] of the table's type.  Indices outside the table are clamped (as the lookup of the
    layer-by-layer path does); a float32 index is truncated."""
    code = N.element_type(table, 'table')
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise N.NativeError('table must be [count, width] with a row and a column at least (got {})'.format(tuple(table.shape)))
    idx, icode = _index(idx, table)
    out = table.new_empty(idx.shape + table.shape[1:])
    table, count, width, ldt = N.matrix(table)
    N.launch(table, N.lib().mnr_embedding_forward, out.data_ptr(), width, table.data_ptr(), ldt, count, width, idx.data_ptr(), icode, scale,
             idx.numel(), code)
    return out


def embedding_backward(dy: torch.Tensor, idx: torch.Tensor, count: int, scale: float = 1.0, padding_idx: Optional[int] = None,
                       dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The gradient of a [count, width] table: row v = scale * the sum of dy over the places where idx is v (0 where it never is, and
    for ``padding_idx``).  ``dtype``: dy's (default) or float32; sums are fp32 and rounded once."""
    code = N.element_type(dy, 'dy')
    if dy.dim() < 1 or dy.shape[:-1] != idx.shape or dy.shape[-1] == 0:
        raise N.NativeError('dy must be [*idx.shape, width] = {} + [width] (got {})'.format(tuple(idx.shape), tuple(dy.shape)))
    if count < 1:
        raise N.NativeError('count must be 1 at least (got {})'.format(count))
    dtype = dy.dtype if dtype is None else dtype
    if dtype not in (dy.dtype, torch.float32):
        raise N.NativeError('the gradient is float32 or of dy\'s type (got {})'.format(dtype))
    pad = -1 if padding_idx is None else int(padding_idx)
    if padding_idx is not None and not 0 <= pad < count:
        raise N.NativeError('padding_idx must be a row of the table (got {} of {})'.format(padding_idx, count))
    idx, icode = _index(idx, dy)
    g, rows, width, ldg = N.matrix(dy)
    grad = dy.new_empty((count, width), dtype=dtype)
    lib = N.lib()
    size = lib.mnr_embedding_backward_workspace_bytes(rows, count, width)
    ws = dy.new_empty(size, dtype=torch.uint8)
    N.launch(g, lib.mnr_embedding_backward, grad.data_ptr(), N.ELEMENT_TYPES[dtype], g.data_ptr(), ldg, idx.data_ptr(), icode, rows, count, width, pad,
             float(scale), code, ws.data_ptr(), size)
    return grad


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, idx, table, scale, padding_idx):
        ctx.save_for_backward(idx)
        ctx.args = (table.shape[0], scale, padding_idx)
        return embedding_forward(idx, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        N.refuse_captured_backward('embedding')
        (idx,) = ctx.saved_tensors
        return None, embedding_backward(dy, idx, *ctx.args), None, None


def embedding(idx: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[idx]``, differentiable in the table; ``padding_idx``: a row that gets no gradient."""
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise N.NativeError('padding_idx must be a row of the table (got {} of {})'.format(padding_idx, table.shape[0]))
    return _Embedding.apply(idx, table, scale, padding_idx)
