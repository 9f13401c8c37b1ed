"""A learned gate over the cells (csrc/gate.hip): which k cells a row goes to and with what weights, the gradient of the weights, and
the rows of every cell in one stable order.  The container's own router (models.mega_nerf.MegaNeRF, mega_nerf.py:19-49) goes by the
distance to the cells' centroids; this one goes by scores that a layer has computed, and gives its choice in the same terms: per row
the cells and blend weights, per cell the list of its rows.

``route_topk`` is the differentiable call; ``route_topk_forward`` / ``route_topk_backward`` are its passes for callers with a tape of
their own: they record nothing for autograd, and may be recorded into a HIP graph."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from mega_nerf import _native as N

_SCORES = {'softmax': 0, 'sigmoid': 1}
_MAX_K, _MAX_DISPATCH = 32, (1 << 24) - 1


def _score(score: str) -> int:
    if score not in _SCORES:
        raise N.NativeError('score must be softmax or sigmoid (got {!r})'.format(score))
    return _SCORES[score]


def _logits(logits: torch.Tensor):
    code = N.element_type(logits, 'logits')
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise N.NativeError('logits must be [..., cells] with a cell at least (got {})'.format(tuple(logits.shape)))
    return (code,) + tuple(N.matrix(logits))


def _choice(logits: torch.Tensor, k: int, n_groups: int, k_groups: int, group_top: int) -> None:
    """Before anything is allocated, and before ctypes takes numbers of 2^32 and more for their low 32 bits."""
    n = logits.shape[-1]
    if not 1 <= k <= min(n, _MAX_K):
        raise N.NativeError('route_topk chooses 1 to {} cells, at most as many as there are (got {} of {})'.format(_MAX_K, k, n))
    if not 1 <= n_groups <= n or n % n_groups:
        raise N.NativeError('n_groups must divide the cells evenly (got {} for {} cells)'.format(n_groups, n))
    if not 1 <= k_groups <= n_groups or k > k_groups * (n // n_groups):
        raise N.NativeError('k_groups must be 1 to n_groups and its groups hold k cells (got {} of {} groups, k {})'.format(k_groups, n_groups, k))
    if group_top not in (1, 2):
        raise N.NativeError('group_top must be 1 or 2 (got {})'.format(group_top))


def _mask(mask: Optional[torch.Tensor], logits: torch.Tensor):
    """(tensor, row pitch): bool, like the logits or one row [cells] for all of them."""
    if mask is None:
        return None, 0
    if mask.dtype != torch.bool:
        raise N.NativeError('mask must be bool (got {})'.format(mask.dtype))
    N.on_device_of(logits, mask, 'mask')
    if mask.shape == logits.shape[-1:]:
        return mask.contiguous(), 0
    if mask.shape != logits.shape:
        raise N.NativeError('mask must be {} or {} (got {})'.format(tuple(logits.shape), tuple(logits.shape[-1:]), tuple(mask.shape)))
    mask, _, _, ldm = N.matrix(mask)
    return mask, ldm


def route_topk_forward(logits: torch.Tensor, k: int, score: str = 'softmax', bias: Optional[torch.Tensor] = None,
                       mask: Optional[torch.Tensor] = None, n_groups: int = 1, k_groups: int = 1, group_top: int = 1,
                       renormalise: bool = True, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(weights float32 [..., k], cells int32 [..., k]) of ``logits`` [..., n_cells].

    A cell is open where ``mask`` (bool, [..., n_cells] or [n_cells]) is set and its logit is above -inf.  s = softmax over the open
    cells, or sigmoid.  The k cells with the largest s + ``bias`` are chosen (without a bias: the largest logits), largest first, the
    lowest number among equals; the bias [n_cells] float32 moves the choice only, never the weights.  With ``n_groups`` > 1 the cells
    lie in groups of neighbours, and only the ``k_groups`` groups stay open whose ``group_top`` (1 or 2) best s + bias sum highest.
    weights = scale * s, over the sum of the chosen s if ``renormalise``.

    k is 1 to 32, of up to 1024 cells.  Fewer than k open cells: the slots left over hold cell -1 with weight 0.  A NaN among a row's
    open logits (softmax: or +inf) gives that row cells -1 and weights NaN."""
    sc = _score(score)
    if logits.dim() and logits.shape[-1]:
        _choice(logits, k, n_groups, k_groups, group_top)
    code, x, rows, n, ldl = _logits(logits)
    m, ldm = _mask(mask, logits)
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (n,):
            raise N.NativeError('bias must be float32 [{}] (got {} {})'.format(n, bias.dtype, tuple(bias.shape)))
        N.on_device_of(logits, bias, 'bias')
        bias = bias.contiguous()
    shape = logits.shape[:-1] + (int(k),)
    weights = x.new_empty(shape, dtype=torch.float32)
    cells = x.new_empty(shape, dtype=torch.int32)
    N.launch(x, N.lib().mnr_gate_forward, weights.data_ptr(), cells.data_ptr(), x.data_ptr(), ldl, N.ptr(bias), N.ptr(m), ldm, rows, n, k, sc, n_groups,
             k_groups, group_top, 1 if renormalise else 0, float(scale), code)
    return weights, cells


def route_topk_backward(dweights: torch.Tensor, logits: torch.Tensor, cells: torch.Tensor, score: str = 'softmax',
                        mask: Optional[torch.Tensor] = None, renormalise: bool = True, scale: float = 1.0) -> torch.Tensor:
    """d(loss)/d(logits) for d(loss)/d(weights) = ``dweights``, the choice ``cells`` of :func:`route_topk_forward` being fixed (score,
    mask, renormalise and scale as there).  A row without cells gets zeros."""
    sc = _score(score)
    code, x, rows, n, ldl = _logits(logits)
    m, ldm = _mask(mask, logits)
    if cells.dtype != torch.int32 or cells.dim() != logits.dim() or cells.shape[:-1] != logits.shape[:-1]:
        raise N.NativeError('cells must be int32 {} + [k] (got {} {})'.format(tuple(logits.shape[:-1]), cells.dtype, tuple(cells.shape)))
    if dweights.shape != cells.shape or dweights.dtype != torch.float32:
        raise N.NativeError('dweights must be float32 {} (got {} {})'.format(tuple(cells.shape), dweights.dtype, tuple(dweights.shape)))
    N.on_device_of(logits, cells, 'cells')
    N.on_device_of(logits, dweights, 'dweights')
    cells = cells.contiguous()
    g, _, k, ldg = N.matrix(dweights)
    dx = x.new_empty(logits.shape)
    N.launch(x, N.lib().mnr_gate_backward, dx.data_ptr(), n, g.data_ptr(), ldg, x.data_ptr(), ldl, cells.data_ptr(), N.ptr(m), ldm, rows, n, k, sc,
             1 if renormalise else 0, float(scale), code)
    return dx


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, score, bias, mask, n_groups, k_groups, group_top, renormalise, scale):
        weights, cells = route_topk_forward(logits, k, score, bias, mask, n_groups, k_groups, group_top, renormalise, scale)
        ctx.save_for_backward(logits, cells, mask)
        ctx.how = (score, renormalise, scale)
        ctx.mark_non_differentiable(cells)
        return weights, cells

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, _):
        N.refuse_captured_backward('route_topk')
        logits, cells, mask = ctx.saved_tensors
        score, renormalise, scale = ctx.how
        return (route_topk_backward(dweights, logits, cells, score, mask, renormalise, scale),) + (None,) * 9


def route_topk(logits: torch.Tensor, k: int, score: str = 'softmax', bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
               n_groups: int = 1, k_groups: int = 1, group_top: int = 1, renormalise: bool = True,
               scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`route_topk_forward`, its weights differentiable in the logits."""
    return _RouteTopk.apply(logits, k, score, bias, mask, n_groups, k_groups, group_top, renormalise, scale)


def dispatch(cells: torch.Tensor, n_cells: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(order int32 [cells.numel()], offsets int32 [n_cells + 1]): the slots of ``cells`` (int32, flattened) sorted by cell and, inside a
    cell, by slot; cell c's are ``order[offsets[c]:offsets[c + 1]]``, slots without a cell come last.  A slot's row is slot // k.  No
    host synchronisation."""
    if cells.dtype != torch.int32:
        raise N.NativeError('cells must be int32 (got {})'.format(cells.dtype))
    if not 1 <= n_cells <= _MAX_DISPATCH:
        raise N.NativeError('dispatch needs 1 to {} cells (got {})'.format(_MAX_DISPATCH, n_cells))
    N.require_device(cells, 'cells')
    cells = cells.contiguous()
    slots = cells.numel()
    order = cells.new_empty(slots)
    offsets = cells.new_empty(int(n_cells) + 1)
    lib = N.lib()
    size = lib.mnr_gate_dispatch_workspace_bytes(slots, n_cells)
    ws = cells.new_empty(size, dtype=torch.uint8)
    N.launch(cells, lib.mnr_gate_dispatch, order.data_ptr(), offsets.data_ptr(), cells.data_ptr(), slots, n_cells, ws.data_ptr(), size)
    return order, offsets
