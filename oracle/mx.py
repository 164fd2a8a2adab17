"""Oracle of the microscaled quantisation (test infrastructure only; see ``oracle/__init__.py``): every value is compared
with the whole table of the format's values, in 64 bits."""
import math

import numpy as np
import torch

from . import quant

E2M1 = [float(v) for v in quant.FP4_VALUES[:8]]
E4M3 = [float(v) for v in quant.e4m3_decode_table()[:0x7f]]   # (positive, finite; ascending)


def scale_bytes_of(amax: np.ndarray, fmt: str) -> np.ndarray:
    """Exponent bytes of the smallest powers of two, at least 2^-126, under which amax stays inside the format (255: no
    finite number).  With amax = m 2^e and the largest value l 2^p, m and l in [0.5, 1): e - p, and one more where m > l."""
    l, p = math.frexp(6.0 if fmt == 'e2m1' else 448.0)
    m, e = np.frexp(amax)
    e = np.where(amax == 0, -1000, e)
    return np.where(np.isfinite(amax), np.maximum(e - p + (m > l), -126) + 127, 255).astype(np.int64)


def quantize(x: torch.Tensor, fmt: str):
    """(codes [M, K] uint8 as whole codes, bytes [M, K / 32]) of x [M, K]."""
    table = np.array(E2M1 if fmt == 'e2m1' else E4M3)
    m, k = x.shape
    v = x.double().numpy().reshape(m, k // 32, 32)
    with np.errstate(invalid='ignore'):
        amax = np.abs(v).max(-1)   # (NaN where a value is)
    scales = scale_bytes_of(amax, fmt)
    nan = (scales == 255)[..., None]
    a = np.where(nan, 0.0, np.abs(v)) / np.exp2((np.where(scales == 255, 127, scales) - 127).astype(np.float64))[..., None]
    hi = np.searchsorted(table, a).clip(max=len(table) - 1)          # first table value >= a
    lo = (hi - 1).clip(min=0)
    up = (table[hi] - a < a - table[lo]) | ((table[hi] - a == a - table[lo]) & (hi % 2 == 0))
    codes = np.where(up | (hi == 0), hi, lo)
    sign = np.signbit(v) & ~nan
    codes = np.where(nan, 0, codes) + np.where(sign, 8 if fmt == 'e2m1' else 128, 0)
    return torch.from_numpy(codes.reshape(m, k).astype(np.uint8)), torch.from_numpy(scales)


def values(codes: torch.Tensor, scales: torch.Tensor, fmt: str) -> torch.Tensor:
    """fp64 values of whole codes under their exponent bytes."""
    table = quant.FP4_VALUES if fmt == 'e2m1' else quant.e4m3_decode_table()
    v = torch.tensor(np.array(table, dtype=np.float64))[codes.long()]
    s = torch.exp2(scales.double() - 127)
    s[scales == 255] = float('nan')
    return v * s.repeat_interleave(32, dim=-1)


def unpack(codes: torch.Tensor) -> torch.Tensor:
    """Whole codes of packed e2m1 or e4m3 tensors."""
    if codes.dtype == torch.int8:
        c = codes.contiguous().view(torch.uint8)
        return torch.stack((c & 15, c >> 4), dim=-1).flatten(-2)
    return codes.contiguous().view(torch.uint8)


def scale_bytes(sf: torch.Tensor, blocks: int) -> torch.Tensor:
    """Exponent bytes [.., M, blocks] of required-layout scale factors."""
    p = sf.to(torch.int64) & 0xffff
    return torch.stack((p & 255, p >> 8), dim=-1).flatten(-2)[..., :blocks]
