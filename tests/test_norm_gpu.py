"""The norm with the residual's addition and quantised output against the oracle, with its gradient."""
import pytest
import torch

import deep_gemm
from helpers import gen
from oracle import blocks as ob

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
ROUND = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}
# A row's sum of squares: at most 64 steps a thread and 20 to join them, halved by the root; some operations more.
SUM = 64 * U32


def _inputs(t, h, dtype, seed=0, weight=None):
    g = gen(seed + t + h)
    x, r, d_y, d_h = (torch.randn(t, h, generator=g).to(dtype) for _ in range(4))
    return x, r * 3, (1 + 0.2 * torch.randn(h, generator=g)).to(weight or dtype), d_y, d_h


@pytest.mark.parametrize('t,h', [(1, 1), (1, 7168), (3, 8), (5, 31), (2, 512), (17, 513), (33, 1024), (7, 1407), (600, 2048), (9, 2049),
                                 (513, 4100), (4, 8192), (3, 16384), (515, 9000), (2, 20001), (514, 32768), (1, 32768), (1025, 77)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('residual', [True, False])
def test_forward_and_gradient(t, h, dtype, residual):
    x, r, w, d_y, d_h = _inputs(t, h, dtype, weight=torch.float32 if t % 2 else torch.bfloat16)
    r, d_h = (r, d_h) if residual else (None, None)
    dev = [None if v is None else v.cuda() for v in (x, r, w, d_y, d_h)]
    y, got_h, rstd = deep_gemm.rms_norm(dev[0], dev[2], dev[1], 1e-5)
    want, want_h, want_rstd = ob.rms_norm(x, w, r, 1e-5)
    assert y.dtype == dtype and rstd.dtype == torch.float32
    assert torch.equal(got_h.cpu(), want_h)
    assert ((rstd.cpu().double() - want_rstd).abs() <= SUM * want_rstd).all()
    assert ((y.cpu().double() - want).abs() <= (ROUND[dtype] + SUM + 4 * U32) * want.abs()).all()

    d_x, d_w = deep_gemm.rms_norm_backward(dev[3], got_h, dev[2], rstd, dev[4])
    want, mag, want_w, mag_w = ob.rms_norm_backward(d_y, want_h, w, want_rstd, d_h)
    assert d_x.dtype == dtype and d_w.dtype == torch.float32
    # (a row's inner product in the same steps, rstd three times)
    assert ((d_x.cpu().double() - want).abs() <= ROUND[dtype] * want.abs() + 5 * SUM * mag).all()
    # a team's rows one after another, the workgroups' and 32 at the end
    steps = -(-t // 256) + 64
    assert ((d_w.cpu().double() - want_w).abs() <= (steps * U32 + SUM) * mag_w).all()


@pytest.mark.parametrize('t,h', [(1, 32), (1, 7168), (3, 64), (16, 96), (513, 96), (17, 1440), (600, 2048), (1001, 4128), (515, 8192), (5, 8224), (2, 32768)])
@pytest.mark.parametrize('fmt', ['e4m3', 'e2m1'])
def test_quantised_output_is_the_quantisers(t, h, fmt):
    """Codes and scale factors are what mx_quantize gives of the fp32 rows, bit for bit."""
    for dtype in (torch.float32, torch.bfloat16):
        x, _, w, _, _ = (v.cuda() for v in _inputs(t, h, dtype))
        (codes, sf), same, rstd = deep_gemm.rms_norm(x, w, None, 1e-6, fmt)
        y, _, rstd2 = deep_gemm.rms_norm(x.float(), w.float(), None, 1e-6)
        want, want_sf = deep_gemm.mx_quantize(y, fmt)
        assert same is x and torch.equal(rstd, rstd2)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(sf, want_sf)
        if t % 2:   # (the partner of an odd last row)
            assert (torch.as_strided(sf, (sf.size(1),), (sf.stride(1),), sf.storage_offset() + t) == 0).all()


def test_quantised_output_with_residual():
    x, r, w, _, _ = (v.cuda() for v in _inputs(37, 512, torch.bfloat16))
    q, h, rstd = deep_gemm.rms_norm(x, w, r, fmt='e4m3')
    again, _, rstd2 = deep_gemm.rms_norm(h, w, fmt='e4m3')
    assert torch.equal(rstd, rstd2) and torch.equal(q[1], again[1]) and torch.equal(q[0].view(torch.uint8), again[0].view(torch.uint8))


def test_infinities_and_nan_stay_in_their_rows():
    x, _, w, d_y, _ = (v.cuda() for v in _inputs(700, 160, torch.float32))
    clean = deep_gemm.rms_norm(x, w, fmt='e4m3')[0]
    bad = x.clone()
    bad[3, 5], bad[9, 1] = float('nan'), float('inf')
    y, _, rstd = deep_gemm.rms_norm(bad, w)
    keep = torch.ones(700, dtype=torch.bool)
    keep[[3, 9]] = False
    assert torch.isnan(y[3]).all() and torch.isnan(y[9, 1]) and torch.equal(y[keep], deep_gemm.rms_norm(x, w)[0][keep])
    q = deep_gemm.rms_norm(bad, w, fmt='e4m3')[0]
    assert torch.equal(q[1][keep], clean[1][keep])
    assert torch.isnan(deep_gemm.mx_dequantize(q, torch.float32)[3]).all()
    zero = torch.zeros(4, 96, device='cuda')
    assert (deep_gemm.rms_norm(zero, w[:96])[0] == 0).all()


def test_strides_and_odd_addresses():
    for dtype in (torch.float32, torch.bfloat16):
        whole = torch.randn(70, 403, generator=gen(1)).to(dtype).cuda()
        part, w = whole[:, 1:353], torch.randn(352, generator=gen(2)).to(dtype).cuda()
        res = whole.t()[:352, :70].t()
        for fmt in (None, 'e4m3'):
            a, b = deep_gemm.rms_norm(part, w, res, fmt=fmt), deep_gemm.rms_norm(part.contiguous(), w, res.contiguous(), fmt=fmt)
            assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
            for u, v in zip(a[0] if fmt else (a[0],), b[0] if fmt else (b[0],)):
                assert torch.equal(u.view(torch.int8) if fmt and u.dtype != torch.int16 else u, v.view(torch.int8) if fmt and v.dtype != torch.int16 else v)
        rstd = deep_gemm.rms_norm(part, w)[2]
        ones = torch.ones((), dtype=dtype, device='cuda').expand(70, 352)
        for a, b in zip(deep_gemm.rms_norm_backward(ones, part, w, rstd, res),
                        deep_gemm.rms_norm_backward(ones.contiguous(), part.contiguous(), w, rstd, res.contiguous())):
            assert torch.equal(a, b)


def test_nothing_to_do():
    w = torch.ones(64, device='cuda')
    x = torch.empty(0, 64, device='cuda')
    y, h, rstd = deep_gemm.rms_norm(x, w, x)
    assert y.shape == h.shape == (0, 64) and rstd.shape == (0,)
    (codes, sf), _, _ = deep_gemm.rms_norm(x, w, fmt='e2m1')
    assert codes.shape == (0, 32) and sf.shape == (0, 1)
    d_x, d_w = deep_gemm.rms_norm_backward(x, x, w, rstd)
    assert d_x.shape == (0, 64) and (d_w == 0).all()


def test_rows_past_4_gib():
    t, h = 140001, 16384
    x = torch.empty(t, h, dtype=torch.bfloat16, device='cuda').normal_()
    w = torch.ones(h, dtype=torch.bfloat16, device='cuda')
    y, _, rstd = deep_gemm.rms_norm(x, w)
    d_x, _ = deep_gemm.rms_norm_backward(y, x, w, rstd)
    for part in (slice(0, 3), slice(t - 3, t)):
        assert torch.equal(y[part], deep_gemm.rms_norm(x[part].repeat(300, 1), w)[0][:3])
        want = ob.rms_norm_backward(y[part].cpu(), x[part].cpu(), w.cpu(), rstd[part].cpu())
        assert ((d_x[part].cpu().double() - want[0]).abs() <= 2.0 ** -8 * want[0].abs() + 5 * SUM * want[1]).all()
