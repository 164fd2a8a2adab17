"""The gated activation, its 8-bit checkpoint and its gradient against the oracle and the quantiser."""
import pytest
import torch

import deep_gemm
from helpers import gen
from oracle import blocks as ob

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
ROUND = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}
# An exponent's rounding (twice its size) and some operations.
EDGE = lambda gate: (3 * gate.abs().clamp(max=110) + 24) * U32
# The sigmoid is held in fp32, and its values below 2^-126 (gates below -87.3) are 0.  Times the gate, with gate * exp(gate) falling
# past there (at -110 it is below 2^-150): act off by at most 110 * 2^-126, the gradients by 111 * 2^-126, less than 2^-119, times the
# other half and d_act, below 2^5 in these inputs.
TINY = 2.0 ** -114


def _inputs(m, f, dtype, seed=0, spread=1.0):
    g = gen(seed + m + f)
    return (spread * torch.randn(m, 2 * f, generator=g)).to(dtype), torch.randn(m, f, generator=g).to(dtype)


def _bits(q):
    return q[0].view(torch.uint8), q[1]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(_bits(a), _bits(b)))


@pytest.mark.parametrize('m,f', [(1, 1), (1, 2048), (3, 7), (8, 512), (9, 513), (65, 1411), (777, 96), (1030, 4096), (20000, 64), (70000, 520)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_values_and_gradient(m, f, dtype):
    h, d = _inputs(m, f, dtype, spread=4.0)
    rows = slice(0, m) if m * f < 1 << 22 else torch.randint(0, m, (500,), generator=gen(1))
    act = deep_gemm.swiglu(h.cuda())
    d_h, again = deep_gemm.swiglu_backward(d.cuda(), h.cuda(), with_act=True)
    assert act.dtype == d_h.dtype == dtype and torch.equal(act, again)
    assert torch.equal(deep_gemm.swiglu_backward(d.cuda(), h.cuda()), d_h)
    h, d = h[rows], d[rows]
    gate = h[:, :f].double()
    want = ob.swiglu(h)
    assert ((act.cpu()[rows].double() - want).abs() <= (ROUND[dtype] + EDGE(gate)) * want.abs() + TINY).all()
    want, mag = ob.swiglu_backward(d, h)
    off = EDGE(gate).repeat(1, 2)
    assert ((d_h.cpu()[rows].double() - want).abs() <= ROUND[dtype] * want.abs() + off * mag + TINY).all()


@pytest.mark.parametrize('m,f', [(1, 32), (1, 2048), (5, 96), (8, 544), (33, 1024), (777, 160), (1031, 4096), (30001, 480), (66000, 544)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_quantised_output_and_checkpoint_are_the_quantisers(m, f, dtype):
    h, d = (v.cuda() for v in _inputs(m, f, dtype))
    want = deep_gemm.mx_quantize(h, 'e4m3')
    wide = deep_gemm.swiglu(h.float())
    for fmt in (None, 'e4m3', 'e2m1'):
        act, saved = deep_gemm.swiglu(h, fmt, checkpoint=True)
        assert _same(saved, want)
        if fmt is None:
            assert torch.equal(act, deep_gemm.swiglu(h)) and torch.equal(act, wide.to(dtype))
        else:
            assert _same(act, deep_gemm.mx_quantize(wide, fmt)) and _same(act, deep_gemm.swiglu(h, fmt))
    if m % 2:   # (the partner of an odd last row)
        sf = want[1]
        for s in (saved[1], act[1]):
            assert (torch.as_strided(s, (s.size(1),), (s.stride(1),), s.storage_offset() + m) == 0).all()
    # the gradient from the checkpoint is that of the values it stands for
    values = deep_gemm.mx_dequantize(want, torch.float32)
    d_h, again = deep_gemm.swiglu_backward(d, saved, with_act=True)
    ref_d, ref_act = deep_gemm.swiglu_backward(d.float(), values, with_act=True)
    assert torch.equal(d_h, ref_d.to(dtype)) and torch.equal(again, ref_act.to(dtype))


def test_gradient_against_differences():
    h, d = (v.double() for v in _inputs(6, 5, torch.float32))
    got = deep_gemm.swiglu_backward(d.float().cuda(), h.float().cuda()).cpu().double()
    for e in range(10):
        step = torch.zeros(6, 10).double()
        step[:, e] = 1e-4
        want = ((ob.swiglu(h + step) - ob.swiglu(h - step)) * d).sum(1) / 2e-4
        # (the rounding of the inputs to fp32, and the third order of the differences)
        assert ((got[:, e] - want).abs() < 1e-6 + 1e-6 * want.abs()).all()


def test_far_values():
    gate = torch.tensor([-3e38, -1e4, -200., -104., -90., -88., -0., 0., 88., 200., 3e38, float('inf')])
    h = torch.stack((gate, torch.ones_like(gate)), 1)
    act = deep_gemm.swiglu(h.cuda()).cpu().double()[:, 0]
    want = ob.swiglu(h)[:, 0]
    assert torch.equal(torch.isfinite(act), torch.isfinite(want))
    fine = torch.isfinite(want)
    assert ((act - want)[fine].abs() <= EDGE(gate.double())[fine] * want[fine].abs() + TINY).all()
    d_h = deep_gemm.swiglu_backward(torch.ones(12, 1, device='cuda'), h.cuda()).cpu().double()[:-1]
    want, mag = ob.swiglu_backward(torch.ones(11, 1), h[:-1])
    assert ((d_h - want).abs() <= EDGE(gate.double())[:-1].unsqueeze(1) * mag + TINY).all()


@pytest.mark.parametrize('m,f', [(64, 96), (1248, 544), (70016, 64)])
def test_padding_rows(m, f):
    g = gen(m)
    h, d = (v.cuda() for v in _inputs(m, f, torch.bfloat16))
    idx = torch.where(torch.rand(m, generator=g) < 0.4, 3, -1).int().cuda()
    live = idx >= 0
    h[~live], d[~live] = float('nan'), float('inf')      # (never read)
    clean_h, clean_d = torch.where(live.unsqueeze(1), h, 0.0), torch.where(live.unsqueeze(1), d, 0.0)
    act, saved = deep_gemm.swiglu(h, None, True, idx)
    q = deep_gemm.swiglu(h, 'e4m3', m_indices=idx)
    want, want_saved = deep_gemm.swiglu(clean_h, None, True)
    assert torch.equal(act, want) and torch.equal(saved[0].view(torch.uint8), want_saved[0].view(torch.uint8))
    assert torch.equal(saved[1][live], want_saved[1][live]) and (saved[1][~live] == 0).all() and (q[1][~live] == 0).all()
    assert (deep_gemm.mx_dequantize(saved)[~live] == 0).all()
    assert torch.equal(deep_gemm.mx_dequantize(q), deep_gemm.mx_dequantize(deep_gemm.swiglu(clean_h, 'e4m3')))
    for s, ref in ((saved, want_saved), (h, clean_h)):
        a, b = deep_gemm.swiglu_backward(d, s, True, idx), deep_gemm.swiglu_backward(clean_d, ref, True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # unwritten: live rows alone are defined
    part = deep_gemm.swiglu(h, None, False, idx, zero_padding=False)
    assert torch.equal(part[live], want[live])
    back = deep_gemm.swiglu_backward(d, saved, False, idx, zero_padding=False)
    assert torch.equal(back[live], deep_gemm.swiglu_backward(clean_d, want_saved)[live])


def test_unwritten_padding_is_left_as_it_was():
    """Through the C ABI, on buffers of a known content."""
    from deep_gemm import _lib
    m, f = 40, 64
    h = torch.randn(m, 2 * f, device='cuda')
    idx = torch.where(torch.arange(m) % 3 == 0, 0, -1).int().cuda()
    act, d_h = torch.full((m, f), 7.0, device='cuda'), torch.full((m, 2 * f), 7.0, device='cuda')
    a = _lib.SwigluArgs()
    a.rows, a.width, a.dtype, a.format = m, f, _lib.DG_DTYPE_F32, -1
    a.h, a.h_ld, a.act, a.act_ld, a.m_indices = h.data_ptr(), 2 * f, act.data_ptr(), f, idx.data_ptr()
    a.d_act, a.d_act_ld, a.d_h, a.d_h_ld = h.data_ptr(), 2 * f, d_h.data_ptr(), 2 * f
    lib = _lib.load()
    _lib.check(lib.dg_swiglu_forward(a, torch.cuda.current_stream().cuda_stream), lib)
    a.act = None
    _lib.check(lib.dg_swiglu_backward(a, torch.cuda.current_stream().cuda_stream), lib)
    for t in (act, d_h):
        assert (t[idx < 0] == 7.0).all() and (t[idx >= 0] != 7.0).all()


def test_strides_and_odd_addresses():
    for dtype in (torch.float32, torch.bfloat16):
        whole = torch.randn(90, 403, generator=gen(1)).to(dtype).cuda()
        h, d = whole[:, 1:385], whole.t()[:192, :90].t()
        assert torch.equal(deep_gemm.swiglu(h), deep_gemm.swiglu(h.contiguous()))
        a, s = deep_gemm.swiglu(h, 'e4m3', True)
        b, r = deep_gemm.swiglu(h.contiguous(), 'e4m3', True)
        assert _same(a, b) and _same(s, r)
        assert torch.equal(deep_gemm.swiglu_backward(d, h), deep_gemm.swiglu_backward(d.contiguous(), h.contiguous()))
        # a checkpoint whose codes and scale factors lie otherwise
        codes = torch.empty(90, 399, dtype=torch.uint8, device='cuda')[:, 5:389].copy_(s[0].view(torch.uint8)).view(torch.float8_e4m3fn)
        want = deep_gemm.swiglu_backward(d, s)
        assert torch.equal(deep_gemm.swiglu_backward(d, (codes, s[1].contiguous())), want)


def test_nothing_to_do():
    for m, f in ((0, 64), (4, 0)):
        h = torch.empty(m, 2 * f, device='cuda')
        assert deep_gemm.swiglu(h).shape == (m, f)
        act, saved = deep_gemm.swiglu(h, 'e2m1', True)
        assert act[0].shape == (m, f // 2) and saved[0].shape == (m, 2 * f)
        assert deep_gemm.swiglu_backward(h[:, :f], saved).shape == (m, 2 * f)


def test_rows_past_4_gib():
    m, f = 150001, 8192
    h = torch.empty(m, 2 * f, dtype=torch.bfloat16, device='cuda').normal_()
    act, saved = deep_gemm.swiglu(h, None, True)
    d_h = deep_gemm.swiglu_backward(act, saved)
    for part in (slice(0, 3), slice(m - 3, m)):
        a, s = deep_gemm.swiglu(h[part], None, True)
        assert torch.equal(act[part], a) and torch.equal(saved[0][part].view(torch.uint8), s[0].view(torch.uint8))
        assert torch.equal(d_h[part], deep_gemm.swiglu_backward(act[part], s))
