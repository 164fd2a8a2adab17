"""The gated activation between two products, with an 8-bit checkpoint of its input for the backward pass.

    act, saved = swiglu(h, checkpoint=True)                       # saved: e4m3 codes and scales of h, which may be freed
    d_h, act = swiglu_backward(d_act, saved, with_act=True)       # act once more, for the gradient of the weights behind it

Rows may be those of an M-grouped layout: with ``m_indices`` its padding rows are not read.  No autograd graph is recorded.
"""
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .gemm import _call, _operators, _stream
from .layout import _assert
from .moe import _plain
from .mx import _DTYPES, _FORMATS
from .norm import _ld, _new_codes, _sf_ld
from .runtime import cu_cap, get_dry_run

Saved = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _args(rows: int, width: int, values: torch.Tensor, m_indices: Optional[torch.Tensor], zero_padding: bool):
    _assert(values.dtype in _DTYPES, 'values must be bf16 or fp32')
    _assert(rows <= 2 ** 30 and width <= 2 ** 29, 'every extent must be at most 2^30')
    if m_indices is not None:
        _assert(m_indices.dtype == torch.int32 and m_indices.shape == (rows,) and m_indices.device == values.device,
                'm_indices must be a [M] int32 tensor beside the rows')
        m_indices = m_indices.contiguous()
    a = _lib.SwigluArgs()
    a.rows, a.width, a.dtype, a.format = rows, width, _DTYPES[values.dtype], -1
    a.m_indices, a.zero_padding = m_indices.data_ptr() if m_indices is not None else None, int(zero_padding)
    a.num_cus = cu_cap()
    return m_indices, a


def swiglu(h: torch.Tensor, fmt: Optional[str] = None, checkpoint: bool = False, m_indices: Optional[torch.Tensor] = None,
           zero_padding: bool = True):
    """act [M, F] = gate / (1 + exp(-gate)) * up of the rows ``h`` = (gate | up) [M, 2 F] (bf16 or fp32), in fp32, rounded once to their
    type; with ``fmt`` 'e4m3' or 'e2m1' the pair (codes, sf) that ``mx_quantize`` would give of the fp32 values (F a multiple of 32).
    The fp32 values are off by up to |gate| + 4 units of 2^-24 for negative gates, and by 4 for others.

    ``checkpoint``: (act, saved), where saved is what ``mx_quantize(h, 'e4m3')`` gives, from the same read (F a multiple of 32).
    ``m_indices`` [M] int32 (as ``moe_sort`` gives it): rows with a negative entry are padding; they are not read, and are zeros in the
    results, or with ``zero_padding=False`` unwritten (scale factors are zeros all the same)."""
    _assert(fmt is None or fmt in _FORMATS, f'unknown format {fmt}: e2m1 or e4m3')
    ext = _operators(h)
    if ext is not None:
        made = ext.swiglu(h, -1 if fmt is None else _FORMATS[fmt], checkpoint, m_indices, zero_padding, cu_cap(), _stream(h))
        if made:
            act = made[0] if fmt is None else (made[0], made[1])
            return (act, (made[-2], made[-1])) if checkpoint else act
    _assert(h.dim() == 2 and h.is_cuda and h.size(1) % 2 == 0, 'h must be a [M, 2 F] device tensor')
    m, f = h.size(0), h.size(1) // 2
    m_indices, a = _args(m, f, h, m_indices, zero_padding)
    _assert(f % 32 == 0 or (fmt is None and not checkpoint), f'F must be a multiple of the block of 32 values, got {f}')
    h = _plain(h)
    a.h, a.h_ld = h.data_ptr(), _ld(h)
    if fmt is None:
        act = torch.empty((m, f), dtype=h.dtype, device=h.device)
        a.act, a.act_ld = act.data_ptr(), f
    else:
        act = _new_codes(h, fmt, m, f)
        a.format, a.act, a.act_ld, a.act_sf, a.act_sf_ld = _FORMATS[fmt], act[0].data_ptr(), act[0].size(1), act[1].data_ptr(), _sf_ld(act[1])
    saved = None
    if checkpoint:
        saved = _new_codes(h, 'e4m3', m, 2 * f)
        a.saved, a.saved_ld, a.saved_sf, a.saved_sf_ld = saved[0].data_ptr(), 2 * f, saved[1].data_ptr(), _sf_ld(saved[1])
    if m and f and not get_dry_run():
        _call('dg_swiglu_forward', a, h)
    return (act, saved) if checkpoint else act


def swiglu_backward(d_act: torch.Tensor, saved: Saved, with_act: bool = False, m_indices: Optional[torch.Tensor] = None,
                    zero_padding: bool = True):
    """d_h [M, 2 F] of the rows that ``saved`` holds, in the type of ``d_act`` [M, F]: h itself (of that type), or the checkpoint (codes,
    sf) that ``swiglu`` gave.  ``with_act``: (d_h, act), the activation of the same values again.  ``m_indices`` and ``zero_padding`` as in
    ``swiglu``."""
    codes, sf = saved if isinstance(saved, tuple) else (saved, None)
    ext = _operators(d_act)
    if ext is not None:
        made = ext.swiglu_backward(d_act, codes, sf, with_act, m_indices, zero_padding, cu_cap(), _stream(d_act))
        if made:
            return (made[0], made[1]) if with_act else made[0]
    _assert(d_act.dim() == 2 and d_act.is_cuda, 'd_act must be a [M, F] device tensor')
    m, f = d_act.shape
    m_indices, a = _args(m, f, d_act, m_indices, zero_padding)
    _assert(codes.shape == (m, 2 * f) and codes.device == d_act.device, 'saved must hold [M, 2 F] values beside d_act')
    if sf is None:
        _assert(codes.dtype == d_act.dtype, 'h must have the type of d_act')
        codes = _plain(codes)
        a.h, a.h_ld = codes.data_ptr(), _ld(codes)
    else:
        _assert(codes.dtype == torch.float8_e4m3fn, 'the codes of a checkpoint are float8_e4m3fn')
        _assert(f % 32 == 0, f'F must be a multiple of the block of 32 values, got {f}')
        _assert(sf.dtype == torch.int16 and sf.shape == (m, f // 32) and sf.device == d_act.device, 'sf must be int16 [M, 2 F / 64]')
        # (copies whose rows lie as the kernel reads them)
        if codes.numel() and (codes.stride(1) != 1 or _ld(codes) % 8 or _ld(codes) < 2 * f or codes.data_ptr() % 8):
            codes = codes.clone(memory_format=torch.contiguous_format)
        if sf.numel() and ((m > 1 and sf.stride(0) != 1) or sf.data_ptr() % 4 or _sf_ld(sf) % 2 or _sf_ld(sf) < m):
            sf = _new_codes(d_act, 'e4m3', m, 2 * f)[1].copy_(sf)
        a.saved, a.saved_ld, a.saved_sf, a.saved_sf_ld = codes.data_ptr(), _ld(codes), sf.data_ptr(), _sf_ld(sf)
    d_act = _plain(d_act)
    d_h = torch.empty((m, 2 * f), dtype=d_act.dtype, device=d_act.device)
    act = torch.empty((m, f), dtype=d_act.dtype, device=d_act.device) if with_act else None
    if m and f and not get_dry_run():
        a.d_act, a.d_act_ld, a.d_h, a.d_h_ld = d_act.data_ptr(), _ld(d_act), d_h.data_ptr(), 2 * f
        if with_act:
            a.act, a.act_ld = act.data_ptr(), f
        _call('dg_swiglu_backward', a, d_act)
    return (d_h, act) if with_act else d_h
