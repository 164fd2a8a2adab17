"""Microscaled quantisation and its product against the oracle: codes and scale factors bit for bit, values bit for bit,
products within their rounding."""
import pytest
import torch

import deep_gemm
from helpers import gen
from oracle import mx as ox

pytestmark = pytest.mark.gpu

U32, UBF16 = 2.0 ** -24, 2.0 ** -8


def _check(x, fmt, dev=None):
    """mx_quantize of x (two dimensions) against the oracle; (codes, sf) on the device."""
    codes, sf = deep_gemm.mx_quantize(x.cuda() if dev is None else dev, fmt)
    m, k = x.shape
    want, scales = ox.quantize(x, fmt)
    assert torch.equal(ox.scale_bytes(sf.cpu(), k // 32), scales)
    assert torch.equal(ox.unpack(codes.cpu()), want)
    if k % 64:   # the half of the last pair that holds no block
        assert (sf.cpu()[:, -1].to(torch.int32) >> 8 & 255 == 0).all()
    return codes, sf


@pytest.mark.parametrize('fmt', ['e2m1', 'e4m3'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,k', [(1, 32), (1, 4096), (2, 64), (7, 96), (9, 512), (65, 544), (130, 1440), (33, 7168)])
def test_quantize(fmt, dtype, m, k):
    x = (torch.randn(m, k, generator=gen(m + k)) * torch.exp(3 * torch.randn(m, 1, generator=gen(k)))).to(dtype)
    codes, sf = _check(x, fmt)
    assert codes.stride(-1) == 1 and (sf.stride(0) == 1 or m == 1)
    for out in (torch.float32, torch.bfloat16):
        got = deep_gemm.mx_dequantize((codes, sf), out).cpu()
        assert torch.equal(got.double(), ox.values(*ox.quantize(x, fmt), fmt).to(out).double())


@pytest.mark.parametrize('fmt', ['e2m1', 'e4m3'])
def test_quantize_many_rows(fmt):
    """The tall tiles (64 rows)."""
    x = torch.randn(16400, 2080, generator=gen(1)).bfloat16().cuda()
    codes, sf = deep_gemm.mx_quantize(x, fmt)
    for part in (slice(0, 40), slice(8180, 8220), slice(16380, 16400)):
        want, scales = ox.quantize(x[part].cpu(), fmt)
        assert torch.equal(ox.unpack(codes[part].cpu()), want) and torch.equal(ox.scale_bytes(sf[part].cpu(), 65), scales)
    small = deep_gemm.mx_quantize(x[:100], fmt)
    assert torch.equal(codes[:100].view(torch.int8), small[0].view(torch.int8)) and torch.equal(sf[:100], small[1])
    back = deep_gemm.mx_dequantize((codes, sf))
    assert torch.equal(back[:100], deep_gemm.mx_dequantize(small))
    assert torch.equal(back[-20:].cpu().double(), ox.values(want, scales, fmt))


@pytest.mark.parametrize('fmt', ['e2m1', 'e4m3'])
@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
def test_dequantize_rows_that_start_anywhere(fmt, out):
    """Rows from an odd one on, single rows, scale factors of other strides and codes at an odd address give what the whole gives."""
    x = torch.randn(2, 21, 160, generator=gen(6)).cuda()
    codes, sf = deep_gemm.mx_quantize(x, fmt)
    whole = deep_gemm.mx_dequantize((codes, sf), out)
    for rows in (slice(1, 21), slice(3, 4), slice(20, 21), slice(2, 9)):
        assert torch.equal(deep_gemm.mx_dequantize((codes[1, rows], sf[1, rows]), out), whole[1, rows])
        assert torch.equal(deep_gemm.mx_dequantize((codes[:, rows], sf[:, rows]), out), whole[:, rows])
    assert torch.equal(deep_gemm.mx_dequantize((codes[0, 5:6], sf[0, 5:6].contiguous()), out), whole[0, 5:6])
    for held in (codes, codes[0]):
        at = torch.empty(held.numel() + 1, dtype=torch.uint8, device='cuda')[1:].view(held.dtype).view(held.shape)
        at.copy_(held)
        assert at.is_contiguous() and at.data_ptr() % 8
        assert torch.equal(deep_gemm.mx_dequantize((at, sf if held is codes else sf[0]), out), whole if held is codes else whole[0])
    odd = torch.empty(2, 3, 23, dtype=torch.int16, device='cuda')[:, :, 1:22].transpose(1, 2)   # (rows 23 apart)
    odd.copy_(sf)
    assert torch.equal(deep_gemm.mx_dequantize((codes, odd), out), whole)
    assert torch.equal(deep_gemm.mx_dequantize((codes[0], odd[0]), out), whole[0])


@pytest.mark.parametrize('fmt', ['e2m1', 'e4m3'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_edges(fmt, dtype):
    """Ties, block maxima on either side of the format's largest value, zeros of both signs, numbers near the ends of the
    type's range, and numbers below the smallest normal one."""
    top = 6.0 if fmt == 'e2m1' else 448.0
    table = torch.tensor(ox.E2M1 if fmt == 'e2m1' else ox.E4M3[::5])
    mids = (table[1:] + table[:-1]) / 2
    rows = []
    for block in torch.cat((table, mids, -mids, -table)).split(30):
        rows.append(torch.cat((torch.tensor([top, -top]), torch.nn.functional.pad(block, (0, 30 - block.numel())))))
    for amax in (top, top * (1 + 2.0 ** -7), top * (1 - 2.0 ** -7), 1.0, 2.0 ** -126, 1.5 * 2.0 ** -125, 2.0 ** -130, 0.0, 3e38, 2.0 ** 127):
        rows.append(torch.linspace(-amax, amax, 32, dtype=torch.float64).float())
    x = torch.stack(rows).to(dtype)
    x = torch.cat((x, -x, torch.zeros_like(x[:1]), -torch.zeros_like(x[:1])))
    _check(x, fmt)


@pytest.mark.parametrize('fmt', ['e2m1', 'e4m3'])
def test_infinities_and_nan(fmt):
    """A block with an infinity or a NaN is NaN, its neighbours are not; so is what a product makes of it."""
    x = torch.randn(5, 128, generator=gen(2))
    x[1, 40], x[2, 127], x[3, 0] = float('inf'), float('nan'), float('-inf')
    codes, sf = _check(x, fmt)
    back = deep_gemm.mx_dequantize((codes, sf), torch.float32).cpu()
    bad = torch.zeros(5, 4, dtype=torch.bool)
    bad[1, 1] = bad[2, 3] = bad[3, 0] = True
    assert torch.equal(back.isnan(), bad.repeat_interleave(32, dim=1))
    w = deep_gemm.mx_quantize(torch.randn(48, 128, generator=gen(3)).cuda(), 'e2m1')
    d = torch.empty(5, 48, dtype=torch.float32, device='cuda')
    deep_gemm.mx_gemm_nt(x.cuda(), w, d, fmt)
    assert torch.equal(d.cpu().isnan().all(dim=1), bad.any(dim=1)) and not d.cpu()[[0, 4]].isnan().any()


@pytest.mark.parametrize('fmt', ['e2m1', 'e4m3'])
def test_python_path_matches_the_extension(monkeypatch, fmt):
    x = torch.randn(77, 160, generator=gen(6)).cuda()
    run = lambda: (*deep_gemm.mx_quantize(x, fmt), deep_gemm.mx_dequantize(deep_gemm.mx_quantize(x, fmt)))
    fast = run()
    monkeypatch.setattr('deep_gemm.mx._operators', lambda t: None)
    for a, b in zip(run(), fast):
        assert a.dtype == b.dtype and a.stride() == b.stride()
        assert torch.equal(a.view(torch.int8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.int8) if a.dtype == torch.float8_e4m3fn else b)


def test_strides_and_batches():
    x = torch.randn(3, 21, 160, generator=gen(4)).bfloat16()
    for fmt in ('e2m1', 'e4m3'):
        codes, sf = deep_gemm.mx_quantize(x.cuda(), fmt)
        for i in range(3):
            want, scales = ox.quantize(x[i], fmt)
            assert torch.equal(ox.unpack(codes[i].cpu()), want) and torch.equal(ox.scale_bytes(sf[i].cpu(), 5), scales)
        assert torch.equal(deep_gemm.mx_dequantize((codes, sf))[1], deep_gemm.mx_dequantize((codes[1], sf[1])))
        wide = torch.zeros(21, 171, dtype=torch.bfloat16, device='cuda')
        wide[:, 3:163] = x[0].cuda()
        _check(x[0], fmt, wide[:, 3:163])
        _check(x[0], fmt, x[0].t().contiguous().t().cuda())
        _check(x[0, ::2], fmt, x[0].cuda()[::2])
        _check(x[0, :, :96], fmt, x[0].cuda()[:, :96])


@pytest.mark.parametrize('fmt', ['e2m1', 'e4m3'])
@pytest.mark.parametrize('m,n,k', [(1, 64, 32), (1, 1000, 4096), (3, 129, 96), (16, 2112, 1440), (17, 300, 7168), (129, 257, 544),
                                   (300, 512, 2048)])
def test_product(fmt, m, n, k):
    x, w = torch.randn(m, k, generator=gen(m)).bfloat16(), torch.randn(n, k, generator=gen(n)) * k ** -0.5
    q = deep_gemm.mx_quantize(w.cuda(), 'e2m1')
    a = ox.values(*ox.quantize(x, fmt), fmt)
    b = ox.values(*ox.quantize(w, 'e2m1'), 'e2m1')
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    for dtype in (torch.bfloat16, torch.float32):
        d = torch.full((m, n), float('nan'), dtype=dtype, device='cuda')
        deep_gemm.mx_gemm_nt(x.cuda(), q, d, fmt)
        bound = k * U32 * mag
        if dtype == torch.bfloat16:
            bound = bound * (1 + UBF16) + UBF16 * ref.abs()
        assert ((d.cpu().double() - ref).abs() <= bound).all()
    c = d.clone()
    deep_gemm.mx_gemm_nt(x.cuda(), q, c, fmt, c=c)
    assert ((c.cpu().double() - 2 * ref).abs() <= 2 * (k + 1) * U32 * mag).all()


def test_quantize_under_a_cu_cap_and_in_a_graph():
    x = torch.randn(500, 1056, generator=gen(5)).bfloat16().cuda()
    want = deep_gemm.mx_quantize(x)
    full = deep_gemm.get_num_sms()
    try:
        deep_gemm.set_num_sms(24)
        got = deep_gemm.mx_quantize(x)
    finally:
        deep_gemm.set_num_sms(full)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    stream = torch.cuda.Stream()
    buf = x.clone()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            back = deep_gemm.mx_dequantize(deep_gemm.mx_quantize(buf))
    for scale in (1.0, 3.0, 0.25):
        buf.copy_(x * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(back, deep_gemm.mx_dequantize(deep_gemm.mx_quantize(buf)))


def _layout(counts, alignment):
    """psum and extent of groups of these sizes, with a spare block of padding rows at the end."""
    psum, at = [], 0
    for c in counts:
        psum.append(at + c)
        at += -(-c // alignment) * alignment
    return torch.tensor(psum, dtype=torch.int32), at + alignment


@pytest.mark.parametrize('counts,alignment', [
    ([1], 32), ([0, 1, 0, 0, 5], 32), ([16, 17, 0, 33, 3], 32), ([32, 64, 100, 1, 1, 1, 1], 32), ([0, 0, 0], 64), ([2] * 40, 32), ([40, 1, 1], 128),
])
@pytest.mark.parametrize('n,k', [(32, 32), (100, 96), (257, 544), (512, 4096)])
def test_experts_of_few_rows(counts, alignment, n, k):
    """M-grouped products of e2m1 rows, few to a group: each group's rows with its weights, zeros in padding rows, whatever
    the padding rows of A and its scales hold."""
    g, groups = gen(n + k + len(counts)), len(counts)
    psum, m = _layout(counts, alignment)
    x, w = torch.randn(m, k, generator=g).bfloat16(), torch.randn(groups, n, k, generator=g) * k ** -0.5
    codes, sf = deep_gemm.mx_quantize(x.cuda(), 'e2m1')
    starts = [0] + [-(-int(p) // alignment) * alignment for p in psum[:-1]]
    live = torch.zeros(m, dtype=torch.bool)
    for s, p in zip(starts, psum.tolist()):
        live[s:p] = True
    dead = (~live).cuda()
    codes[dead] = -1
    held = torch.full((sf.size(1), m + m % 2), -1, dtype=torch.int16, device='cuda')[:, :m].transpose(0, 1)
    held.copy_(sf)
    held[dead] = -1                       # (scale bytes 255: NaN)
    q = deep_gemm.mx_quantize(w.cuda(), 'e2m1')
    a = ox.values(*ox.quantize(x, 'e2m1'), 'e2m1')
    ref, mag = torch.zeros(m, n, dtype=torch.float64), torch.zeros(m, n, dtype=torch.float64)
    for e, (s, p) in enumerate(zip(starts, psum.tolist())):
        b = ox.values(*ox.quantize(w[e], 'e2m1'), 'e2m1')
        ref[s:p], mag[s:p] = a[s:p] @ b.t(), a[s:p].abs() @ b.abs().t()
    deep_gemm.set_mk_alignment_for_contiguous_layout(alignment)
    try:
        for dtype in (torch.bfloat16, torch.float32):
            d = torch.full((m, n), float('nan'), dtype=dtype, device='cuda')
            deep_gemm.m_grouped_fp8_fp4_gemm_nt_contiguous((codes, held), q, d, psum.cuda())
            bound = k * U32 * mag
            if dtype == torch.bfloat16:
                bound = bound * (1 + UBF16) + UBF16 * ref.abs()
            assert ((d.cpu().double() - ref).abs() <= bound).all()
            wide = torch.full((m, n + 3), 7.0, dtype=dtype, device='cuda')
            deep_gemm.m_grouped_fp8_fp4_gemm_nt_contiguous((codes, held), q, wide[:, 1:n + 1], psum.cuda())
            assert torch.equal(wide[:, 1:n + 1], d) and (wide[:, 0] == 7).all() and (wide[:, n + 1:] == 7).all()
    finally:
        deep_gemm.set_mk_alignment_for_contiguous_layout(256)


@pytest.mark.parametrize('counts,n,k', [
    ([300] + [0] * 9, 70, 160), ([64, 65, 128, 129, 0, 1, 192], 100, 96), ([70] + [0] * 257 + [130, 1, 66] + [0] * 3 + [64], 33, 64),
    ([65] * 5 + [1] * 7, 257, 2048), ([0] * 255 + [200] + [0] * 20 + [90], 32, 32),
])
def test_groups_of_more_rows_than_one_pass(counts, n, k):
    """Groups of more than 64 rows among few: the later rows are work of their own, found by scanning the layout."""
    test_experts_of_few_rows(counts, 32, n, k)


@pytest.mark.parametrize('counts,alignment', [
    ([1, 64, 0, 65], 64), ([0, 3, 40, 128, 1], 64), ([0] * 3 + [5], 64), ([1, 128, 0, 129, 7], 128), ([2] * 70, 128), ([100, 192, 30], 192),
])
@pytest.mark.parametrize('n,k', [(100, 96), (257, 544), (512, 2048)])
def test_experts_on_small_tiles(counts, alignment, n, k):
    """Layouts of a small tile to a group or little more."""
    test_experts_of_few_rows(counts, alignment, n, k)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,n,k', [(1, 1, 32), (1, 64, 8192), (2, 33, 160), (15, 500, 1056), (16, 2112, 2048), (16, 2112, 7168), (16, 16, 64),
                                   (1, 10000, 512), (1, 129, 32768)])
def test_few_rows_quantised_inside(dtype, m, n, k):
    """The product that quantises its rows itself against the quantiser followed by the GEMM's oracle."""
    x, w = torch.randn(m, k, generator=gen(m)).to(dtype), torch.randn(n, k, generator=gen(n)) * k ** -0.5
    x[0, :32] = 0
    if k > 64:
        x[m - 1, 40:50] *= 1e-6
    q = deep_gemm.mx_quantize(w.cuda(), 'e2m1')
    a, b = ox.values(*ox.quantize(x, 'e2m1'), 'e2m1'), ox.values(*ox.quantize(w, 'e2m1'), 'e2m1')
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    wide = torch.full((m, k + 8), float('nan'), dtype=dtype, device='cuda')
    wide[:, 4:k + 4] = x.cuda()
    for inp in (x.cuda(), wide[:, 4:k + 4]):
        d = torch.full((m, n), float('nan'), device='cuda')
        deep_gemm.mx_gemm_nt(inp, q, d)
        assert ((d.cpu().double() - ref).abs() <= k * U32 * mag).all()
        deep_gemm.mx_gemm_nt(inp, q, d, c=d)
        assert ((d.cpu().double() - 2 * ref).abs() <= 2 * (k + 1) * U32 * mag).all()


def test_few_rows_matches_the_general_path(monkeypatch):
    x, w = torch.randn(5, 256, generator=gen(7)).bfloat16().cuda(), deep_gemm.mx_quantize(torch.randn(96, 256, generator=gen(8)).cuda())
    fast, general = (torch.empty(5, 96, dtype=torch.bfloat16, device='cuda') for _ in range(2))
    deep_gemm.mx_gemm_nt(x, w, fast)
    monkeypatch.setattr('deep_gemm.mx._operators', lambda t: None)
    deep_gemm.mx_gemm_nt(x, w, general)
    assert (fast.float() - general.float()).abs().max() <= 2 * UBF16 * general.float().abs().max()
