"""Root-mean-square norm with the residual's addition before it and, on demand, quantised rows behind it.

    y, h, rstd = rms_norm(x, weight, residual)
    d_x, d_weight = rms_norm_backward(d_y, h, weight, rstd, d_h)

``y`` may leave as codes and scale factors, which the GEMMs take as an operand with recipe (1, 32).  No autograd graph is recorded: the
results of inputs that require gradients have none, and a program makes the second call itself.
"""
import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .gemm import _call, _operators, _stream
from .layout import _align, _assert, _ceil_div
from .moe import _plain
from .mx import _DTYPES, _FORMATS
from .runtime import cu_cap, get_dry_run

MAX_WIDTH = 32768


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _new_codes(like: torch.Tensor, fmt: str, rows: int, k: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes of rows x k values and their scale factors in the required layout, unwritten."""
    codes = torch.empty((rows, k // 2), dtype=torch.int8, device=like.device) if fmt == 'e2m1' else \
        torch.empty((rows, k), dtype=torch.float8_e4m3fn, device=like.device)
    return codes, torch.empty((_ceil_div(k, 64), _align(rows, 2)), dtype=torch.int16, device=like.device)[:, :rows].transpose(0, 1)


def _sf_ld(sf: torch.Tensor) -> int:
    return sf.stride(1) if sf.size(1) > 1 else _align(sf.size(0), 2)


def _args(x: torch.Tensor, weight: torch.Tensor) -> Tuple[torch.Tensor, _lib.RmsNormArgs]:
    _assert(x.dim() == 2 and x.is_cuda, 'the rows must be a [T, H] device tensor')
    _assert(x.dtype in _DTYPES and weight.dtype in _DTYPES, 'values and weight must be bf16 or fp32')
    _assert(1 <= x.size(1) <= MAX_WIDTH, f'H must be between 1 and {MAX_WIDTH}')
    _assert(x.size(0) <= 2 ** 30, 'at most 2^30 tokens')
    _assert(weight.shape == (x.size(1),) and weight.device == x.device, 'weight must be a [H] tensor beside the rows')
    weight = weight.contiguous()
    a = _lib.RmsNormArgs()
    a.tokens, a.width, a.dtype, a.weight_dtype, a.format = x.size(0), x.size(1), _DTYPES[x.dtype], _DTYPES[weight.dtype], -1
    a.weight, a.num_cus = weight.data_ptr(), cu_cap()
    return weight, a


def _beside(name: str, t: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    _assert(t.shape == x.shape and t.dtype == x.dtype and t.device == x.device, f'{name} must have the shape, type and device of the rows')
    return _plain(t)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6, fmt: Optional[str] = None):
    """(y, h, rstd) of the rows ``x`` [T, H] (bf16 or fp32, H at most 32768): h = x + ``residual`` rounded to their type (x itself without a
    residual), rstd [T] = 1 / sqrt(mean(h^2) + eps) in fp32, y = h * rstd * ``weight`` [H] (bf16 or fp32) rounded once.

    With ``fmt`` 'e4m3' or 'e2m1' (H a multiple of 32), y is the pair (codes, sf) that ``mx_quantize`` would give of the fp32 values."""
    _assert(fmt is None or fmt in _FORMATS, f'unknown format {fmt}: e2m1 or e4m3')
    ext = _operators(x)
    if ext is not None:
        made = ext.rms_norm(x, weight, residual, eps, -1 if fmt is None else _FORMATS[fmt], cu_cap(), _stream(x))
        if made:
            h = x if residual is None else made[-1]
            return (made[0], h, made[1]) if fmt is None else ((made[0], made[1]), h, made[2])
    weight, a = _args(x, weight)
    _assert(fmt is None or x.size(1) % 32 == 0, f'H must be a multiple of the block of 32 values, got {x.size(1)}')
    rows = _plain(x)
    h = x
    if residual is not None:
        residual = _beside('residual', residual, x)
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.residual, a.residual_ld, a.h, a.h_ld = residual.data_ptr(), _ld(residual), h.data_ptr(), x.size(1)
    rstd = torch.empty(x.size(0), dtype=torch.float32, device=x.device)
    if fmt is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.y, a.y_ld = y.data_ptr(), x.size(1)
    else:
        y = _new_codes(x, fmt, x.size(0), x.size(1))
        a.format, a.y, a.y_ld, a.sf, a.sf_ld = _FORMATS[fmt], y[0].data_ptr(), y[0].size(1), y[1].data_ptr(), _sf_ld(y[1])
    if x.size(0) and not get_dry_run():
        a.eps, a.x, a.x_ld, a.rstd = eps, rows.data_ptr(), _ld(rows), rstd.data_ptr()
        _call('dg_rms_norm_forward', a, x)
    return y, h, rstd


def rms_norm_backward(d_y: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      d_h: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(d_x [T, H], d_weight [H] fp32) from the gradient of y, with ``h`` and ``rstd`` as ``rms_norm`` gave them; d_x, in the type of the
    rows, is the gradient of x and of the residual.  ``d_h`` is what reaches h past the norm (the residual stream's), added to d_x."""
    ext = _operators(h)
    if ext is not None:
        made = ext.rms_norm_backward(d_y, h, weight, rstd, d_h, cu_cap(), _stream(h))
        if made:
            return made[0], made[1]
    weight, a = _args(h, weight)
    d_y = _beside('d_y', d_y, h)
    d_h = None if d_h is None else _beside('d_h', d_h, h)
    _assert(rstd.dtype == torch.float32 and rstd.shape == h.shape[:1] and rstd.device == h.device, 'rstd must be a [T] fp32 tensor')
    h, rstd = _plain(h), rstd.contiguous()
    d_x = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    if h.size(0) == 0:
        return d_x, torch.zeros(h.size(1), dtype=torch.float32, device=h.device)
    d_weight = torch.empty(h.size(1), dtype=torch.float32, device=h.device)
    if get_dry_run():
        return d_x, d_weight
    need = ctypes.c_int64()
    lib = _lib.load()
    _lib.check(lib.dg_rms_norm_workspace_size(a, ctypes.byref(need)), lib)
    ws = torch.empty(need.value, dtype=torch.uint8, device=h.device)
    a.h, a.h_ld, a.rstd, a.d_y, a.d_y_ld = h.data_ptr(), _ld(h), rstd.data_ptr(), d_y.data_ptr(), _ld(d_y)
    if d_h is not None:
        a.d_h, a.d_h_ld = d_h.data_ptr(), _ld(d_h)
    a.d_x, a.d_x_ld, a.d_weight = d_x.data_ptr(), d_x.size(1), d_weight.data_ptr()
    a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    _call('dg_rms_norm_backward', a, h)
    return d_x, d_weight
