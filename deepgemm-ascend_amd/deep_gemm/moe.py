"""Tokens sorted by expert, moved into the rows of an M-grouped contiguous layout and back, with the gradients.

A mixture-of-experts layer runs between two of these calls:

    layout = moe_sort(topk_idx, num_experts)                  # [T, K] expert ids -> rows of an M-grouped layout
    rows = moe_dispatch(x, layout)                            # [M, H] tokens in their rows (bf16, fp8, packed fp4, ...)
    m_grouped_bf16_gemm_nt_contiguous(rows, w, y, layout.psum)
    out = moe_combine(y, layout, topk_weights)                # [T, N] weighted sums of a token's rows

and its gradient between ``moe_combine_backward`` and ``moe_dispatch_backward``.  No autograd graph is recorded: results of inputs
that require gradients have none, and a program chains the backward calls itself.  Nothing synchronises with the host: the
number of rows M is a bound over every routing (``moe_num_rows``), and the rows past the last group are padding.
"""
import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .gemm import _operators, _stream
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
