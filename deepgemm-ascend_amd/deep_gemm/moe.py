"""Tokens sorted by expert, moved into the rows of an M-grouped contiguous layout and back, with the gradients.

A mixture-of-experts layer runs between these calls:

    topk_idx, topk_weights = moe_route(logits, topk)          # [T, E] router logits -> a token's experts and their weights
    layout = moe_sort(topk_idx, num_experts)                  # [T, K] expert ids -> rows of an M-grouped layout
    rows = moe_dispatch(x, layout)                            # [M, H] tokens in their rows (bf16, fp8, packed fp4, ...)
    m_grouped_bf16_gemm_nt_contiguous(rows, w, y, layout.psum)
    out = moe_combine(y, layout, topk_weights)                # [T, N] weighted sums of a token's rows

and its gradient between ``moe_combine_backward`` and ``moe_dispatch_backward``, the router's from ``moe_route_backward``.  No autograd
graph is recorded: results of inputs that require gradients have none, and a program chains the backward calls itself.  Nothing
synchronises with the host: the number of rows M is a bound over every routing (``moe_num_rows``), and the rows past the last group are
padding.
"""
import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .gemm import _call, _operators, _stream
from .layout import _assert, _align
from .runtime import cu_cap, get_dry_run, get_mk_alignment_for_contiguous_layout

MAX_GROUPS = 1024


class MoELayout(NamedTuple):
    """Where the pairs (token t, choice c) of a batch lie.  ``psum`` is the grouped layout of the M-grouped GEMMs (and of
    the K-grouped ones over the same rows), ``m_indices`` its form with ``use_psum_layout=False``."""
    slots: torch.Tensor       # [T, K] int32: row of the pair, -1 for a dropped one
    source: torch.Tensor      # [M] int32: t * K + c of the row's pair, -1 for padding
    psum: torch.Tensor        # [G] int32: end of a group's rows (it starts at the next multiple of the alignment)
    m_indices: torch.Tensor   # [M] int32: group of the row, -1 for padding


def moe_num_rows(num_pairs: int, num_groups: int) -> int:
    """Rows that hold ``num_pairs`` pairs over ``num_groups`` groups whatever the routing, at the current M-grouped
    alignment (set_mk_alignment_for_contiguous_layout)."""
    a = get_mk_alignment_for_contiguous_layout()
    return (num_pairs + min(num_groups, num_pairs) * (a - 1)) // a * a


_SCORES = {'softmax': _lib.DG_SCORES_SOFTMAX, 'sigmoid': _lib.DG_SCORES_SIGMOID}
MAX_EXPERTS, MAX_TOPK, MAX_EXPERT_GROUPS = 1024, 16, 64


def _route_args(logits: torch.Tensor, topk: int, scores: str, renormalize: bool, scale: float) -> Tuple[torch.Tensor, _lib.MoERouteArgs]:
    _assert(logits.dim() == 2 and logits.is_cuda, 'logits must be a [T, E] device tensor')
    _assert(logits.dtype in _DTYPES, 'logits must be bf16 or fp32')
    _assert(1 <= logits.size(1) <= MAX_EXPERTS, f'between 1 and {MAX_EXPERTS} experts')
    _assert(logits.size(0) <= 2 ** 30, 'at most 2^30 tokens')
    _assert(0 <= topk <= min(MAX_TOPK, logits.size(1)), f'topk must be at most {MAX_TOPK} and at most the experts')
    logits = _plain(logits)
    a = _lib.MoERouteArgs()
    a.tokens, a.experts, a.topk = logits.size(0), logits.size(1), topk
    a.scores, a.renormalize, a.scale, a.dtype = _SCORES[scores], int(renormalize), scale, _DTYPES[logits.dtype]
    a.logits, a.logits_ld, a.num_cus = logits.data_ptr(), logits.stride(0) if logits.size(0) > 1 else logits.size(1), cu_cap()
    return logits, a


def moe_route(logits: torch.Tensor, topk: int, scores: str = 'softmax', bias: Optional[torch.Tensor] = None, num_groups: int = 1,
              topk_groups: int = 1, group_top: int = 2, renormalize: bool = True, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ids [T, topk] int32, weights [T, topk] fp32): the experts of each token, as ``moe_sort`` and ``moe_combine`` take them, from the
    router's ``logits`` [T, E] (bf16 or fp32, E at most 1024, topk at most 16).

    Scores s are the ``softmax`` of a row or the ``sigmoid`` of each logit.  ``bias`` [E] (fp32; for balance) is added for the choice
    alone.  With ``num_groups`` > 1 (at most 64) the experts lie in that many groups of equal size, and the ``topk_groups`` groups whose
    ``group_top`` (1 or 2) best biased scores have the largest sum stay.  The topk best biased scores there are chosen, best first, equal
    ones by the lowest index, compared as 64 bits give them (without a bias, and with one group or ``group_top`` 1, as the logits are).
    ``renormalize``: weights s / (sum of the chosen s + 1e-20) instead of s; both times ``scale``.

    An expert whose logit or bias is -inf is never chosen; where fewer than topk are left, ids are -1 (dropped pairs for ``moe_sort``)
    and weights 0.  NaN counts as the largest number."""
    _assert(scores in _SCORES, f'unknown scores {scores}: softmax or sigmoid')
    ext = _operators(logits)
    if ext is not None:
        made = ext.moe_route(logits, topk, scores == 'sigmoid', bias, num_groups, topk_groups, group_top, renormalize, scale, cu_cap(),
                             _stream(logits))
        if made:
            return made[0], made[1]
    logits, a = _route_args(logits, topk, scores, renormalize, scale)
    e = logits.size(1)
    _assert(num_groups <= MAX_EXPERT_GROUPS, f'at most {MAX_EXPERT_GROUPS} groups of experts')
    _assert(num_groups >= 1 and e % num_groups == 0, f'{num_groups} groups do not divide {e} experts')
    _assert(1 <= topk_groups <= num_groups, 'topk_groups must be between 1 and num_groups')
    _assert(group_top in (1, 2), 'group_top must be 1 or 2')
    _assert(topk <= topk_groups * (e // num_groups), "topk must be at most the kept groups' experts")
    if bias is not None:
        _assert(bias.dtype == torch.float32 and bias.shape == (e,) and bias.device == logits.device, 'bias must be a [E] fp32 tensor')
        bias = bias.contiguous()
    ids = torch.empty((logits.size(0), topk), dtype=torch.int32, device=logits.device)
    weights = torch.empty((logits.size(0), topk), dtype=torch.float32, device=logits.device)
    if not get_dry_run():
        a.num_groups, a.topk_groups, a.group_top = num_groups, topk_groups, group_top
        a.bias, a.ids, a.weights = bias.data_ptr() if bias is not None else None, ids.data_ptr(), weights.data_ptr()
        _call('dg_moe_route', a, logits)
    return ids, weights


def moe_route_backward(d_weights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, scores: str = 'softmax', renormalize: bool = True,
                       scale: float = 1.0) -> torch.Tensor:
    """Gradient [T, E] of ``moe_route``'s logits, in their type, from that of its weights (fp32) and its ids; the bias has none.
    Negative ids have no gradient; nor have ids past the last expert, which are reported (``check_errors``)."""
    _assert(scores in _SCORES, f'unknown scores {scores}: softmax or sigmoid')
    ext = _operators(logits)
    if ext is not None:
        made = ext.moe_route_backward(d_weights, logits, ids, scores == 'sigmoid', renormalize, scale, cu_cap(), _stream(logits))
        if made:
            return made[0]
    _assert(ids.dim() == 2 and ids.dtype == torch.int32 and ids.size(0) == logits.size(0) and ids.device == logits.device,
            'ids must be a [T, topk] int32 tensor')
    logits, a = _route_args(logits, ids.size(1), scores, renormalize, scale)
    _assert(d_weights.dtype == torch.float32 and d_weights.shape == ids.shape and d_weights.device == logits.device,
            'd_weights must be a [T, topk] fp32 tensor')
    ids, d_weights = ids.contiguous(), d_weights.contiguous()
    d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if not get_dry_run():
        a.ids, a.d_weights = ids.data_ptr(), d_weights.data_ptr()
        a.d_logits, a.d_logits_ld = d_logits.data_ptr(), d_logits.size(1)
        _call('dg_moe_route_backward', a, logits)
    return d_logits


def _args(layout: MoELayout, num_groups: int = 0, alignment: int = 1) -> _lib.MoELayoutArgs:
    t, k = layout.slots.shape
    return _lib.MoELayoutArgs(t, k, num_groups, layout.source.numel(), alignment, layout.slots.data_ptr(),
                              layout.source.data_ptr(), layout.psum.data_ptr(), layout.m_indices.data_ptr())


def _check_layout(layout: MoELayout, device) -> Tuple[int, int, int]:
    """(T, K, M)"""
    for name, t, dim in zip(MoELayout._fields, layout, (2, 1, 1, 1)):
        _assert(t.dtype == torch.int32 and t.dim() == dim and t.is_contiguous(), f'layout.{name} must be a contiguous int32 tensor')
        _assert(t.device == device, f'layout.{name} must be on the same device as the rows')
    _assert(max(layout.slots.numel(), layout.source.numel()) <= 2 ** 30, 'a layout has at most 2^30 pairs and rows')
    _assert(layout.m_indices.numel() == layout.source.numel(), 'layout.source and layout.m_indices must have one entry per row')
    return layout.slots.size(0), layout.slots.size(1), layout.source.numel()


def moe_sort(topk_idx: torch.Tensor, num_groups: int, num_rows: Optional[int] = None) -> MoELayout:
    """The layout of the pairs of ``topk_idx`` [T, K] (int32 or int64 expert ids; a negative id drops its pair).

    Pairs of an expert keep their order.  ``num_rows`` (a multiple of the M-grouped alignment) is the extent of the
    layout, by default the bound of ``moe_num_rows``; pairs that do not fit a smaller one are dropped and reported, as
    ids past the last group are (``check_errors``)."""
    _assert(topk_idx.dim() == 2 and topk_idx.dtype in (torch.int32, torch.int64), 'topk_idx must be a [T, K] int32 or int64 tensor')
    _assert(topk_idx.is_cuda, 'topk_idx must be a device tensor')
    _assert(1 <= num_groups <= MAX_GROUPS, f'num_groups must be in [1, {MAX_GROUPS}]')
    alignment = get_mk_alignment_for_contiguous_layout()
    t, k = topk_idx.shape
    rows = moe_num_rows(t * k, num_groups) if num_rows is None else int(num_rows)
    ext = _operators(topk_idx)
    if ext is not None:
        made = ext.moe_sort(topk_idx, num_groups, rows, alignment, cu_cap(), _stream(topk_idx))
        if made:
            return MoELayout(*made)
    _assert(rows >= 0 and rows % alignment == 0, f'num_rows must be a multiple of the alignment {alignment}')
    _assert(max(t * k, rows) <= 2 ** 30, 'a layout has at most 2^30 pairs and rows')
    topk_idx = topk_idx.contiguous()
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=topk_idx.device)
    layout = MoELayout(new(t, k), new(rows), new(num_groups), new(rows))
    if get_dry_run():
        return layout
    _lib.raise_pending()
    lib = _lib.load()
    need = ctypes.c_int64()
    _lib.check(lib.dg_moe_sort_workspace_size(t * k, num_groups, ctypes.byref(need)), lib)
    ws = torch.empty(need.value, dtype=torch.uint8, device=topk_idx.device) if need.value else None
    _lib.check(lib.dg_moe_sort(topk_idx.data_ptr(), topk_idx.element_size(), _args(layout, num_groups, alignment),
                               ws.data_ptr() if ws is not None else None, need.value, cu_cap(), _stream(topk_idx)), lib)
    return layout


def moe_dispatch(x, layout: MoELayout, zero_padding: bool = True):
    """Rows [M, H] of the layout from the tokens' rows ``x`` [T, H], of any type of 1, 2 or 4 bytes: row ``slots[t, c]`` is
    token t's.  ``x`` may be a pair (codes, sf) of quantised rows and scale factors in the required layout (as ``mx_quantize``
    or ``transform_sf_into_required_layout`` give them); so is the result then.

    Padding rows are zeros; with ``zero_padding=False`` they are left unwritten, which M-grouped GEMMs allow (their output
    rows are zeros all the same) and K-grouped ones do not."""
    sf = None
    if isinstance(x, tuple):
        x, sf = x
    ext = _operators(x)
    if ext is not None:
        made = ext.moe_dispatch(x, sf, layout, zero_padding, cu_cap(), _stream(x))
        if made:
            return made[0] if sf is None else (made[0], made[1])
    _assert(x.dim() == 2 and x.is_cuda, 'x must be a [T, H] device tensor')
    _assert(x.element_size() in (1, 2, 4), 'x must have elements of 1, 2 or 4 bytes')
    t, _, m = _check_layout(layout, x.device)
    _assert(x.size(0) == t, f'x has {x.size(0)} rows, the layout {t} tokens')
    x = _plain(x)
    h, esize = x.size(1), x.element_size()
    out = torch.empty((m, h), dtype=x.dtype, device=x.device)
    sf_out, k64, sf_ld, out_ld = None, 0, 0, _align(m, 2)
    if sf is not None:
        _assert(sf.dtype == torch.int16 and sf.dim() == 2 and sf.size(0) == t and sf.device == x.device,
                'sf must be an int16 [T, ceil(K / 64)] tensor')
        _assert(t <= 1 or sf.stride(0) == 1, 'sf must be in the required layout (rows contiguous)')
        k64, sf_ld = sf.size(1), sf.stride(1) if sf.size(1) > 1 else t
        sf_out = torch.empty((k64, out_ld), dtype=torch.int16, device=x.device)[:, :m].transpose(0, 1)
    if not get_dry_run():
        _lib.raise_pending()
        lib = _lib.load()
        _lib.check(lib.dg_moe_dispatch(
            x.data_ptr(), x.stride(0) * esize, h * esize, _args(layout), out.data_ptr(), h * esize,
            sf.data_ptr() if sf is not None else None, sf_ld, k64, sf_out.data_ptr() if sf is not None else None, out_ld,
            int(zero_padding), cu_cap(), _stream(x)), lib)
    return out if sf is None else (out, sf_out)


_DTYPES = {torch.bfloat16: _lib.DG_DTYPE_BF16, torch.float32: _lib.DG_DTYPE_F32}


def _plain(t: torch.Tensor) -> torch.Tensor:
    """t with rows of contiguous values that do not overlap (an expanded row is written out)."""
    return t if (t.size(1) <= 1 or t.stride(1) == 1) and (t.size(0) <= 1 or t.stride(0) >= t.size(1)) else t.contiguous()


def _check_rows(name: str, t: torch.Tensor, size: int, what: str) -> torch.Tensor:
    _assert(t.dim() == 2 and t.is_cuda, f'{name} must be a 2D device tensor')
    _assert(t.dtype in _DTYPES, f'{name} must be bf16 or fp32')
    _assert(t.size(0) == size, f'{name} has {t.size(0)} rows, the layout {size} {what}')
    return _plain(t)


def _check_weights(weights: torch.Tensor, layout: MoELayout) -> torch.Tensor:
    _assert(weights.dtype == torch.float32 and weights.shape == layout.slots.shape, 'weights must be a [T, K] fp32 tensor')
    _assert(weights.device == layout.slots.device, 'weights must be on the same device as the layout')
    return weights.contiguous()


def moe_combine(rows: torch.Tensor, layout: MoELayout, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[T, H] sums over a token's choices of ``weights[t, c] * rows[slots[t, c]]`` (no weights: 1), in fp32 in order, rounded
    once to the type of ``rows`` (bf16 or fp32).  Dropped pairs add nothing, whatever their weight."""
    ext = _operators(rows)
    if ext is not None:
        made = ext.moe_combine(rows, layout, weights, cu_cap(), _stream(rows))
        if made:
            return made[0]
    t, _, m = _check_layout(layout, rows.device)
    rows = _check_rows('rows', rows, m, 'rows')
    if weights is not None:
        weights = _check_weights(weights, layout)
    out = torch.empty((t, rows.size(1)), dtype=rows.dtype, device=rows.device)
    if not get_dry_run():
        _lib.raise_pending()
        lib = _lib.load()
        _lib.check(lib.dg_moe_combine(
            rows.data_ptr(), rows.stride(0), _DTYPES[rows.dtype], rows.size(1), _args(layout),
            weights.data_ptr() if weights is not None else None, out.data_ptr(), rows.size(1), cu_cap(), _stream(rows)), lib)
    return out


def moe_dispatch_backward(d_rows: torch.Tensor, layout: MoELayout) -> torch.Tensor:
    """Gradient [T, H] of ``moe_dispatch``'s x: the sums of the gradients of a token's rows."""
    return moe_combine(d_rows, layout)


def moe_combine_backward(d_out: torch.Tensor, rows: torch.Tensor, layout: MoELayout,
                         weights: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``moe_combine``: (d_rows [M, H] = weights[t, c] * d_out[t] in the pairs' rows, zeros in padding rows;
    d_weights [T, K] fp32 = <d_out[t], rows[slots[t, c]]>, 0 for dropped pairs)."""
    ext = _operators(rows)
    if ext is not None:
        made = ext.moe_combine_backward(d_out, rows, layout, weights, cu_cap(), _stream(rows))
        if made:
            return made[0], made[1]
    t, k, m = _check_layout(layout, rows.device)
    rows = _check_rows('rows', rows, m, 'rows')
    d_out = _check_rows('d_out', d_out, t, 'tokens')
    _assert(d_out.dtype == rows.dtype and d_out.size(1) == rows.size(1) and d_out.device == rows.device,
            'd_out must have the type, width and device of rows')
    weights = _check_weights(weights, layout)
    d_rows = torch.empty((m, rows.size(1)), dtype=rows.dtype, device=rows.device)
    d_weights = torch.empty((t, k), dtype=torch.float32, device=rows.device)
    if not get_dry_run():
        _lib.raise_pending()
        lib = _lib.load()
        _lib.check(lib.dg_moe_combine_backward(
            d_out.data_ptr(), d_out.stride(0), rows.data_ptr(), rows.stride(0), _DTYPES[rows.dtype], rows.size(1), _args(layout),
            weights.data_ptr(), d_rows.data_ptr(), rows.size(1), d_weights.data_ptr(), cu_cap(), _stream(rows)), lib)
    return d_rows, d_weights
