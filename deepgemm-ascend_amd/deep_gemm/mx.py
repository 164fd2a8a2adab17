"""Microscaled quantisation (blocks of 32 values of a row under a power of two) to e2m1 and e4m3, back, and the product
of activations quantised on the way.

``mx_quantize`` returns what the GEMMs take as an operand with recipe (1, 32): codes (e4m3, or e2m1 packed two to an int8
byte) and UE8M0 scale factors in the required layout.  No autograd graph is recorded.
"""
from typing import Optional, Tuple

import torch

from . import _lib
from .gemm import _is_fp4, _operators, _stream, fp8_fp4_gemm_nt
from .layout import _align, _assert, _ceil_div
from . import runtime as _rt
from .runtime import cu_cap, get_dry_run, get_jit

_FORMATS = {'e2m1': _lib.DG_MX_E2M1, 'e4m3': _lib.DG_MX_E4M3}
_DTYPES = {torch.bfloat16: _lib.DG_DTYPE_BF16, torch.float32: _lib.DG_DTYPE_F32}


def _run(fn: str, x: torch.Tensor, codes: torch.Tensor, sf: torch.Tensor, fmt: str) -> None:
    if x.numel() == 0 or get_dry_run():
        return
    _lib.raise_pending()
    lib = _lib.load()
    a = _lib.MxArgs()
    batched = x.dim() == 3
    a.format, a.x_dtype = _FORMATS[fmt], _DTYPES[x.dtype]
    a.batches, a.rows, a.k = x.size(0) if batched else 1, x.size(-2), x.size(-1)
    a.x, a.x_ld = x.data_ptr(), x.stride(-2) if x.size(-2) > 1 else x.size(-1)
    a.codes, a.codes_ld = codes.data_ptr(), codes.stride(-2) if codes.size(-2) > 1 else codes.size(-1)
    # (a single k64 column of scale factors has no stride that matters)
    a.sf, a.sf_ld = sf.data_ptr(), sf.stride(-1) if sf.size(-1) > 1 else _align(x.size(-2), 2)
    if batched:
        a.x_batch_stride, a.codes_batch_stride, a.sf_batch_stride = x.stride(0), codes.stride(0), sf.stride(0)
    a.num_cus = cu_cap()
    _lib.check(getattr(lib, fn)(a, _stream(x)), lib)


def mx_quantize(x: torch.Tensor, fmt: str = 'e2m1') -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, sf) of ``x`` [.., M, K] (bf16 or fp32, two or three dimensions, K a multiple of 32).

    A block's scale is the smallest power of two, at least 2^-126, that keeps it within the format (6 or 448), so nothing
    saturates; values round to nearest, ties to even.  A block that holds an infinity or a NaN becomes NaN (scale byte 255)
    and so does every product that reads it."""
    _assert(fmt in _FORMATS, f'unknown format {fmt}: e2m1 or e4m3')
    ext = _operators(x)
    if ext is not None:
        made = ext.mx_quantize(x, fmt == 'e2m1', cu_cap(), _stream(x))
        if made:
            return made[0], made[1]
    _assert(x.dim() in (2, 3) and x.is_cuda, 'x must be a [M, K] or [B, M, K] device tensor')
    _assert(x.dtype in _DTYPES, 'x must be bf16 or fp32')
    m, k = x.size(-2), x.size(-1)
    _assert(max(x.shape) <= 2 ** 30, 'every extent must be at most 2^30')
    _assert(k % 32 == 0, f'K must be a multiple of the block of 32 values, got {k}')
    if k > 1 and (x.stride(-1) != 1 or (m > 1 and x.stride(-2) < k)):   # (an expanded row is written out)
        x = x.contiguous()
    lead = x.shape[:-2]
    codes = torch.empty((*lead, m, k // 2), dtype=torch.int8, device=x.device) if fmt == 'e2m1' else \
        torch.empty((*lead, m, k), dtype=torch.float8_e4m3fn, device=x.device)
    sf = torch.empty((*lead, _ceil_div(k, 64), _align(m, 2)), dtype=torch.int16, device=x.device)[..., :m].transpose(-1, -2)
    _run('dg_mx_quantize', x, codes, sf, fmt)
    return codes, sf


def mx_dequantize(q: Tuple[torch.Tensor, torch.Tensor], dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [.., M, K] of (codes, sf) as ``mx_quantize`` gives them, exact in bf16 and fp32 down to the type's
    smallest numbers."""
    codes, sf = q
    ext = _operators(codes)
    if ext is not None and dtype in _DTYPES:
        made = ext.mx_dequantize(codes, sf, dtype == torch.float32, cu_cap(), _stream(codes))
        if made:
            return made[0]
    fmt = 'e2m1' if _is_fp4(codes) else 'e4m3'
    _assert(fmt == 'e2m1' or codes.dtype == torch.float8_e4m3fn, 'codes must be packed e2m1 (int8) or float8_e4m3fn')
    _assert(codes.dim() in (2, 3) and codes.is_cuda and sf.device == codes.device, 'codes and sf must be device tensors')
    _assert(dtype in _DTYPES, 'dtype must be bf16 or fp32')
    m, k = codes.size(-2), codes.size(-1) * (2 if fmt == 'e2m1' else 1)
    _assert(k % 32 == 0, f'K must be a multiple of the block of 32 values, got {k}')
    _assert(sf.dtype == torch.int16 and sf.shape == (*codes.shape[:-1], _ceil_div(k, 64)), 'sf must be int16 [.., M, ceil(K / 64)]')
    _assert(m <= 1 or sf.stride(-2) == 1, 'sf must be in the required layout (rows contiguous)')
    # (copies whose rows lie as the kernel reads them, also of tensors that are contiguous but start anywhere)
    if codes.size(-1) > 1 and (codes.stride(-1) != 1 or any(s % 8 for s in codes.stride()[:-1]) or codes.data_ptr() % 8 or
                               (m > 1 and codes.stride(-2) < codes.size(-1))):
        codes = codes.clone(memory_format=torch.contiguous_format)
    if sf.data_ptr() % 4 or (sf.size(-1) > 1 and (sf.stride(-1) % 2 or sf.stride(-1) < m)) or (sf.dim() == 3 and sf.stride(0) % 2):
        sf = torch.empty((*sf.shape[:-2], sf.size(-1), _align(m, 2)), dtype=torch.int16, device=sf.device)[..., :m].transpose(-1, -2).copy_(sf)
    out = torch.empty((*codes.shape[:-1], k), dtype=dtype, device=codes.device)
    _run('dg_mx_dequantize', out, codes, sf, fmt)
    return out


def mx_gemm_nt(x: torch.Tensor, w: Tuple[torch.Tensor, torch.Tensor], d: torch.Tensor, fmt: str = 'e2m1',
               c: Optional[torch.Tensor] = None) -> None:
    """D = quantised(x) @ w^T (+ C): ``x`` [M, K] bf16 or fp32 is quantised to ``fmt`` on the way, ``w`` = (codes, sf) holds [N, K]
    weights in e2m1 as ``mx_quantize`` gives them; ``d`` [M, N] bf16 or fp32 and ``c`` as in ``fp8_fp4_gemm_nt``."""
    _assert(_is_fp4(w[0]), 'mx_gemm_nt takes e2m1 weights (for e4m3 ones: mx_quantize, then fp8_gemm_nt)')
    _assert(fmt in _FORMATS, f'unknown format {fmt}: e2m1 or e4m3')
    ext = _operators(x)
    if ext is not None and not get_jit() and \
            ext.mx_gemm(x, w[0], w[1], d, c, fmt == 'e2m1', _rt._num_sms, cu_cap(), _rt._mk_alignment, _stream(x)):
        return
    fp8_fp4_gemm_nt(mx_quantize(x, fmt), w, d, c, recipe_a=(1, 32), recipe_b=(1, 32))
