"""Low-rank adapters of many requests at once, beside a shared projection.

    layout = moe_sort(adapter_ids.view(-1, 1), num_adapters)      # once a step: tokens sorted by adapter, negative ids have none
    bf16_gemm_nt(x, w, d)                                         # any projection that all share
    lora_gemm_nt(x, a, b, d, layout, scales, c=d)                 # and each token's own adapter on top
"""
import ctypes
from typing import Optional

import torch

from . import _lib
from .gemm import _call, _operators, _stream
from .layout import _assert
from .moe import MoELayout, _args as _layout_args, _check_layout, _plain
from .mx import _DTYPES
from .norm import _ld
from .runtime import cu_cap, get_dry_run

MAX_RANK = 256


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous, 16-byte aligned rows."""
    lead = all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)
    if t.stride(-1) == 1 and lead and t.data_ptr() % 16 == 0 and (t.size(-2) <= 1 or t.stride(-2) >= t.size(-1)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def lora_gemm_nt(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, layout: MoELayout,
                 scales: Optional[torch.Tensor] = None, c: Optional[torch.Tensor] = None) -> None:
    """D[t] = C[t] + scales[i] * (x[t] @ a[i]^T) @ b[i]^T, i the adapter of token t; a token without one has D[t] = C[t].

    ``x`` [T, K], ``a`` [L, R, K] and ``b`` [L, N, R] are bf16, K and R multiples of 8, R at most 256 (adapters of lower rank have zeros);
    ``d`` [T, N] is bf16 or fp32, ``c`` (of its type) is d itself, a tensor that does not overlap it, or None for 0; ``scales`` [L] fp32 (None:
    1).  ``layout`` is ``moe_sort``'s of the tokens' adapter ids [T, 1], sorted once for every projection of a step; a small alignment
    (32) suits few tokens.  The inner products are held in fp32 and enter the second product whole for an fp32 d, to 2^-17 for a bf16 one."""
    ext = _operators(x)
    if ext is not None and ext.lora_gemm(x, a, b, d, layout, scales, c, cu_cap(), _stream(x)):
        return
    _assert(x.dim() == 2 and a.dim() == 3 and b.dim() == 3 and d.dim() == 2 and x.is_cuda, 'x [T, K], a [L, R, K], b [L, N, R] and d [T, N] must be device tensors')
    _assert(all(t.dtype == torch.bfloat16 for t in (x, a, b)), 'x, a and b must be bf16')
    _assert(d.dtype in _DTYPES, 'd must be bf16 or fp32')
    t, k = x.shape
    adapters, rank, n = a.size(0), a.size(1), b.size(1)
    _assert(a.size(2) == k, f"Conflicting shape dimension 'k': x gives {k}, a gives {a.size(2)}")
    _assert(b.size(0) == adapters and b.size(2) == rank, f'a holds {adapters} adapters of rank {rank}, b {b.size(0)} of rank {b.size(2)}')
    _assert(d.shape == (t, n), f'd must be [{t}, {n}]')
    _assert(8 <= rank <= MAX_RANK and rank % 8 == 0, f'the rank must be a multiple of 8, at most {MAX_RANK}')
    _assert(k >= 8 and k % 8 == 0, f'K must be a multiple of 8, got {k}')
    _assert(max(t, k, n, adapters) <= 2 ** 30, 'every extent must be at most 2^30')
    _assert(all(o.device == x.device for o in (a, b, d)), 'x, a, b and d must be on the same device')
    tokens, choices, rows = _check_layout(layout, x.device)
    _assert(tokens == t and choices == 1, f'the layout must be of one choice for each of {t} tokens')
    _assert(rows % 32 == 0, "the layout's rows must be a multiple of 32")
    _assert((n <= 1 or d.stride(1) == 1) and (t <= 1 or d.stride(0) >= n), 'd must have contiguous rows that do not overlap')
    if scales is not None:
        _assert(scales.dtype == torch.float32 and scales.shape == (adapters,) and scales.device == x.device, 'scales must be a [L] fp32 tensor')
        scales = scales.contiguous()
    if c is not None:
        _assert(c.shape == d.shape and c.dtype == d.dtype and c.device == d.device, 'c must have the shape, type and device of d')
        _assert(c.data_ptr() != d.data_ptr() or c.stride() == d.stride(), 'c in place of d must have its strides')
        c = _plain(c)
    if t == 0 or n == 0 or get_dry_run():
        return
    x, a, b = _rows(x), _rows(a), _rows(b)
    p = _lib.LoraArgs()
    p.tokens, p.adapters, p.rank, p.n, p.k = t, adapters, rank, n, k
    p.x, p.x_ld = x.data_ptr(), _ld(x)
    p.a, p.a_ld, p.a_stride = a.data_ptr(), a.stride(1) if rank > 1 else k, a.stride(0) if adapters > 1 else 0
    p.b, p.b_ld, p.b_stride = b.data_ptr(), b.stride(1) if n > 1 else rank, b.stride(0) if adapters > 1 else 0
    p.scales = scales.data_ptr() if scales is not None else None
    p.c, p.c_ld = (c.data_ptr(), _ld(c)) if c is not None else (None, 0)
    p.d, p.d_ld, p.d_dtype = d.data_ptr(), _ld(d), _DTYPES[d.dtype]
    held = _layout_args(layout, alignment=32)   # (every alignment that can be set is a multiple of it)
    p.layout, p.num_cus = ctypes.pointer(held), cu_cap()
    lib, need = _lib.load(), ctypes.c_int64()
    _lib.check(lib.dg_lora_workspace_size(p, ctypes.byref(need)), lib)
    ws = torch.empty(need.value, dtype=torch.uint8, device=x.device)
    p.workspace, p.workspace_bytes = ws.data_ptr() if need.value else None, need.value
    _call('dg_lora_gemm', p, x)
