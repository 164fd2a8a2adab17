"""Token sorting and movement (moe_sort, moe_dispatch, moe_combine and their gradients) against the oracle: layouts bit for
bit, copies bit for bit, sums within their rounding."""
import pytest
import torch

import deep_gemm
from deep_gemm import _lib
from helpers import gen
from oracle import moe as om

pytestmark = pytest.mark.gpu

U32, UBF16 = 2.0 ** -24, 2.0 ** -8   # unit roundoffs


@pytest.fixture(autouse=True)
def _restore():
    yield
    deep_gemm.set_mk_alignment_for_contiguous_layout(256)
    torch.cuda.synchronize()
    _lib.load().dg_take_errors()


def _ids(t, k, n, g, kind='spread', dtype=torch.int32):
    if kind == 'spread':
        ids = torch.randint(0, n, (t, k), generator=g)
    elif kind == 'one':          # every pair to one expert
        ids = torch.full((t, k), n - 1)
    elif kind == 'none':         # nothing but dropped pairs
        ids = torch.full((t, k), -1)
    else:                        # dropped pairs among few experts
        ids = torch.randint(-n, max(1, n // 4), (t, k), generator=g)
    return ids.to(dtype)


def _sort(ids, n, alignment, num_rows=None):
    deep_gemm.set_mk_alignment_for_contiguous_layout(alignment)
    layout = deep_gemm.moe_sort(ids.cuda(), n, num_rows)
    want = om.sort(ids, n, alignment, layout.source.numel())
    for name, got, ref in zip(layout._fields, layout, want):
        assert torch.equal(got.cpu(), ref), name
    return layout, want


@pytest.mark.parametrize('t,k,n,alignment', [
    (0, 8, 4, 32), (1, 1, 1, 32), (1, 8, 256, 32), (3, 0, 5, 32), (16, 8, 256, 32), (63, 1, 7, 64), (65, 3, 64, 256),
    (1000, 8, 65, 128), (1024, 8, 1024, 32), (1025, 8, 33, 64), (4099, 6, 513, 128), (20011, 5, 300, 32), (2, 9, 1000, 96),
])
@pytest.mark.parametrize('kind', ['spread', 'one', 'none', 'dropped'])
def test_sort(t, k, n, alignment, kind):
    ids = _ids(t, k, n, gen(t + n), kind, torch.int64 if t % 2 else torch.int32)
    _sort(ids, n, alignment)


@pytest.mark.parametrize('t,k,n,alignment', [(400000, 8, 7, 64), (262145, 8, 1000, 32), (1500001, 3, 65, 128), (2800000, 6, 256, 128)])
def test_sort_of_millions_of_pairs(t, k, n, alignment):
    """More blocks of pairs than each workgroup reads the counts of (2^21 pairs), against a stable sort; a third is dropped."""
    ids = torch.randint(-n // 2, n, (t, k), generator=gen(t)).to(torch.int32)
    ids[t // 2:t // 2 + 9000] = n - 1
    deep_gemm.set_mk_alignment_for_contiguous_layout(alignment)
    layout = deep_gemm.moe_sort(ids.cuda(), n)
    key = torch.where(ids < 0, n, ids).reshape(-1)
    counts = torch.bincount(key, minlength=n + 1)[:n]
    padded = (counts + alignment - 1) // alignment * alignment
    start = torch.cumsum(padded, 0) - padded
    order = torch.sort(key, stable=True).indices[:int(counts.sum())]
    group = key[order].long()
    row = start[group] + torch.arange(len(order)) - (torch.cumsum(counts, 0) - counts)[group]
    slots = torch.full((t * k,), -1, dtype=torch.int32)
    slots[order] = row.int()
    source = torch.full((layout.source.numel(),), -1, dtype=torch.int32)
    m_indices = source.clone()
    source[row], m_indices[row] = order.int(), group.int()
    for got, ref in zip(layout, (slots.view(t, k), source, (start + counts).int(), m_indices)):
        assert torch.equal(got.cpu(), ref)


def test_sort_takes_time_in_proportion():
    """2^26 pairs are eight times as many as 2^23: where every workgroup reads every block's counts they take 64 times as long."""
    times = []
    for t in (1 << 20, 1 << 23):
        ids = torch.randint(0, 256, (t, 8), device='cuda', dtype=torch.int32)
        best = float('inf')
        for _ in range(4):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            deep_gemm.moe_sort(ids, 256)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        times.append(best)
    print('2^23 and 2^26 pairs:', times)
    assert times[1] < 16 * times[0]


def test_sort_reports_ids_past_the_last_group():
    ids = torch.tensor([[0, 5], [3, -7], [2, 1]], dtype=torch.int32)
    _sort(ids, 4, 32)
    with pytest.raises(RuntimeError, match='expert id'):
        deep_gemm.check_errors()
    deep_gemm.check_errors()


@pytest.mark.parametrize('t', [100, 3000])
def test_sort_into_too_few_rows_drops_and_reports(t):
    _sort(_ids(t, 4, 9, gen(t)), 9, 32, 128)
    with pytest.raises(RuntimeError, match='more rows'):
        deep_gemm.check_errors()


def test_sort_in_a_graph_and_on_another_stream():
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    for t in (50, 2000):
        ids = [_ids(t, 8, 40, gen(s)) for s in range(3)]
        buf = ids[0].cuda()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            deep_gemm.moe_sort(buf, 40)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                layout = deep_gemm.moe_sort(buf, 40)
        for i in (1, 2, 0, 1):
            buf.copy_(ids[i])
            graph.replay()
            torch.cuda.synchronize()
            for got, ref in zip(layout, om.sort(ids[i], 40, 32, layout.source.numel())):
                assert torch.equal(got.cpu(), ref)


WIDTHS = [1, 2, 7, 32, 129, 512, 1408, 4104]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize('h', WIDTHS)
def test_dispatch(dtype, h):
    g = gen(h)
    layout, (slots, source, _, _) = _sort(_ids(45, 5, 11, g, 'dropped' if h % 2 else 'spread'), 11, 32)
    x = torch.randint(-128, 128, (45, h * dtype.itemsize), dtype=torch.int8, generator=g).view(dtype)
    # (a row stride that is not the width)
    wide = torch.empty(45, h + 3, dtype=dtype, device='cuda')
    wide[:, :h] = x.cuda()
    for inp in (x.cuda(), wide[:, :h]):
        rows = deep_gemm.moe_dispatch(inp, layout)
        assert torch.equal(rows.cpu().view(torch.int8), om.dispatch(x.view(torch.int8).view(45, -1), source, 5).view(torch.int8))
        part = deep_gemm.moe_dispatch(inp, layout, zero_padding=False)
        live = source >= 0
        assert torch.equal(part.cpu().view(torch.int8)[live], rows.cpu().view(torch.int8)[live])


@pytest.mark.parametrize('t,k64', [(1, 1), (33, 5), (700, 3)])
def test_dispatch_moves_scale_factors(t, k64):
    g = gen(t)
    layout, (slots, source, _, _) = _sort(_ids(t, 3, 6, g), 6, 32)
    codes = torch.randint(-128, 128, (t, 32 * k64), dtype=torch.int8, generator=g)
    sf = torch.randint(-32768, 32768, (t, k64), dtype=torch.int16, generator=g)
    held = torch.zeros(k64, t + t % 2, dtype=torch.int16, device='cuda')[:, :t].transpose(0, 1)
    held.copy_(sf)
    rows, out = deep_gemm.moe_dispatch((codes.cuda(), held), layout, zero_padding=False)
    live = source >= 0
    assert torch.equal(out.cpu(), om.dispatch(sf, source, 3))
    assert torch.equal(rows.cpu()[live], om.dispatch(codes, source, 3)[live])
    assert out.size(0) <= 1 or (out.stride(0) == 1 and out.stride(1) % 2 == 0)


def test_layouts_of_no_choices():
    """No row has a token: rows are padding, also where a layout's sources name pairs all the same."""
    full = lambda *shape, v=0: torch.full(shape, v, dtype=torch.int32, device='cuda')
    layout = deep_gemm.MoELayout(full(4, 0), full(64, v=3), full(2), full(64))
    x, sf = torch.ones(4, 64, dtype=torch.int8, device='cuda'), full(2, 4, v=5).to(torch.int16).t()
    rows, out = deep_gemm.moe_dispatch((x, sf), layout)
    assert rows.shape == (64, 64) and out.shape == (64, 2) and (out == 0).all()
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    layout = deep_gemm.moe_sort(full(4, 0), 2, num_rows=64)
    for a in deep_gemm.moe_dispatch((x, sf), layout):
        assert a.size(0) == 64 and (a == 0).all()
    rows = torch.ones(64, 32, device='cuda')
    assert (deep_gemm.moe_combine(rows, layout) == 0).all()
    d_rows, d_weights = deep_gemm.moe_combine_backward(rows[:4], rows, layout, torch.ones(4, 0, device='cuda'))
    assert (d_rows == 0).all() and d_weights.shape == (4, 0)


def _close(got, ref, mag, n, dtype):
    """A sum of n products in fp32, in order, then rounded to dtype."""
    err = (got.double() - ref).abs()
    bound = (n + 1) * U32 * mag
    if dtype == torch.bfloat16:
        bound = bound * (1 + UBF16) + UBF16 * ref.abs()
    return bool((err <= bound).all())


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('h', WIDTHS)
@pytest.mark.parametrize('k', [1, 6, 19])
def test_combine_and_gradients(dtype, h, k):
    g = gen(h + k)
    t = 23
    layout, (slots, source, _, _) = _sort(_ids(t, k, 13, g, 'dropped' if k == 6 else 'spread'), 13, 32)
    m = source.numel()
    rows, d_out = torch.randn(m, h, generator=g).to(dtype), torch.randn(t, h, generator=g).to(dtype)
    # what dropped pairs and padding rows hold is used nowhere
    rows[source < 0] = float('nan')
    w = torch.randn(t, k, generator=g)
    w_in = torch.where(slots < 0, torch.tensor(float('inf')), w)
    dev = rows.cuda()
    ref, mag = om.combine(rows, slots, w)
    assert _close(deep_gemm.moe_combine(dev, layout, w_in.cuda()).cpu(), ref, mag, k, dtype)
    ref, mag = om.combine(rows, slots)
    assert _close(deep_gemm.moe_combine(dev, layout).cpu(), ref, mag, k, dtype)
    assert _close(deep_gemm.moe_dispatch_backward(dev, layout).cpu(), ref, mag, k, dtype)
    d_rows, d_w = deep_gemm.moe_combine_backward(d_out.cuda(), dev, layout, w_in.cuda())
    ref_rows, ref_w, mag_w = om.combine_backward(d_out, rows, slots, w)
    assert _close(d_rows.cpu(), ref_rows, ref_rows.abs(), 1, dtype)
    assert (d_rows.cpu()[source < 0] == 0).all()
    # (a thread adds its values in order, then at most 8 steps join the threads)
    assert ((d_w.cpu().double() - ref_w).abs() <= (h + 8) * U32 * mag_w).all()
    # strided rows, off 16-byte boundaries
    wide = torch.zeros(m, h + 5, dtype=dtype, device='cuda')
    wide[:, 1:h + 1] = dev
    assert torch.equal(deep_gemm.moe_combine(wide[:, 1:h + 1], layout, w_in.cuda()), deep_gemm.moe_combine(dev, layout, w_in.cuda()))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('t,k,h', [(1, 8, 7168), (3, 2, 16001), (70, 3, 5003), (130, 9, 4100), (600, 2, 2050), (1030, 1, 2048), (1100, 3, 700)])
def test_wide_rows_of_few_tokens_and_short_ones_of_many(dtype, t, k, h):
    """Rows that several workgroups share, and gradients that fewer threads than a workgroup take."""
    g = gen(h + k)
    layout, (slots, source, _, _) = _sort(_ids(t, k, 13, g), 13, 32)
    m = source.numel()
    x, rows, d_out = (torch.randn(n, h, generator=g).to(dtype) for n in (t, m, t))
    moved = deep_gemm.moe_dispatch(x.cuda(), layout).cpu()
    live = source >= 0
    assert torch.equal(moved[live], x[(source[live] // k).long()]) and (moved[~live] == 0).all()
    rows[~live] = float('nan')
    w = torch.randn(t, k, generator=g)
    ref, mag = om.combine(rows, slots, w)
    assert _close(deep_gemm.moe_combine(rows.cuda(), layout, w.cuda()).cpu(), ref, mag, k, dtype)
    d_rows, d_w = deep_gemm.moe_combine_backward(d_out.cuda(), rows.cuda(), layout, w.cuda())
    ref_rows, ref_w, mag_w = om.combine_backward(d_out, rows, slots, w)
    assert _close(d_rows.cpu(), ref_rows, ref_rows.abs(), 1, dtype)
    assert ((d_w.cpu().double() - ref_w).abs() <= (h + 8) * U32 * mag_w).all()


def test_gradients_against_differences():
    """<d/ds loss(s), direction> of a weighted there-and-back movement against central differences in 64 bits."""
    g = gen(7)
    t, k, h = 9, 3, 40
    layout, (slots, source, _, _) = _sort(_ids(t, k, 5, g, 'dropped'), 5, 32)
    x, w, d_out = torch.randn(t, h, generator=g), torch.randn(t, k, generator=g), torch.randn(t, h, generator=g)
    scale = torch.randn(source.numel(), 1, generator=g)          # the "experts": a factor for each row

    def loss(x, w):
        rows = om.dispatch(x.double(), source, k) * scale.double()
        return float((om.combine(rows, slots, w)[0] * d_out.double()).sum())

    rows = deep_gemm.moe_dispatch(x.cuda(), layout) * scale.cuda()
    d_rows, d_w = deep_gemm.moe_combine_backward(d_out.cuda(), rows, layout, w.cuda())
    d_x = deep_gemm.moe_dispatch_backward(d_rows * scale.cuda(), layout)
    dx, dw = torch.randn(t, h, generator=g), torch.randn(t, k, generator=g)
    step = 2.0 ** -10
    by_x = (loss(x.double() + step * dx.double(), w) - loss(x.double() - step * dx.double(), w)) / (2 * step)
    by_w = (loss(x, w.double() + step * dw.double()) - loss(x, w.double() - step * dw.double())) / (2 * step)
    got_x, got_w = float((d_x.cpu().double() * dx.double()).sum()), float((d_w.cpu().double() * dw.double()).sum())
    terms = t * k * h
    assert abs(got_x - by_x) < 8 * U32 * terms * 8 and abs(got_w - by_w) < 8 * U32 * terms * 8


def test_under_a_cu_cap():
    g = gen(3)
    ids, x, w = _ids(3000, 4, 17, g), torch.randn(3000, 64, generator=g), torch.randn(3000, 4, generator=g)
    full = deep_gemm.get_num_sms()
    _, _ = _sort(ids, 17, 32)
    layout = deep_gemm.moe_sort(ids.cuda(), 17)
    rows = deep_gemm.moe_dispatch(x.cuda(), layout)
    want = (*layout, rows, deep_gemm.moe_combine(rows, layout, w.cuda()), *deep_gemm.moe_combine_backward(x.cuda(), rows, layout, w.cuda()))
    try:
        deep_gemm.set_num_sms(24)
        layout = deep_gemm.moe_sort(ids.cuda(), 17)
        rows = deep_gemm.moe_dispatch(x.cuda(), layout)
        got = (*layout, rows, deep_gemm.moe_combine(rows, layout, w.cuda()), *deep_gemm.moe_combine_backward(x.cuda(), rows, layout, w.cuda()))
    finally:
        deep_gemm.set_num_sms(full)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_python_path_matches_the_extension(monkeypatch, dtype):
    assert _lib.ext() is not None
    g = gen(5)
    ids, x, w = _ids(200, 4, 9, g, 'dropped').cuda(), torch.randn(200, 72, generator=g).to(dtype).cuda(), torch.rand(200, 4, generator=g).cuda()
    q = deep_gemm.mx_quantize(torch.randn(200, 160, generator=g).to(dtype).cuda())
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)

    def everything():
        layout = deep_gemm.moe_sort(ids, 9)
        rows = deep_gemm.moe_dispatch(x, layout)
        return (*layout, rows, *deep_gemm.moe_dispatch(q, layout), deep_gemm.moe_combine(rows, layout, w),
                deep_gemm.moe_dispatch_backward(rows, layout), *deep_gemm.moe_combine_backward(x, rows, layout, w))
    fast = everything()
    monkeypatch.setattr('deep_gemm.moe._operators', lambda t: None)
    for a, b in zip(everything(), fast):
        assert a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)


def test_rows_feed_the_grouped_gemms():
    """moe_sort's layouts are what the M-grouped and K-grouped GEMMs take."""
    g = gen(11)
    t, k, n, h, f, alignment = 70, 3, 6, 128, 192, 64
    layout, (slots, source, _, _) = _sort(_ids(t, k, n, g, 'dropped'), n, alignment)
    x, w = torch.randn(t, h, generator=g).bfloat16(), torch.randn(n, f, h, generator=g).bfloat16()
    ids = layout.m_indices.cpu()
    rows = deep_gemm.moe_dispatch(x.cuda(), layout)
    for psum in (True, False):
        d = torch.empty(rows.size(0), f, dtype=torch.float32, device='cuda')
        deep_gemm.m_grouped_bf16_gemm_nt_contiguous(rows, w.cuda(), d, layout.psum if psum else layout.m_indices, use_psum_layout=psum)
        for r in range(rows.size(0)):
            if ids[r] >= 0:
                a, b = rows[r].cpu().double(), w[ids[r]].double()
                assert ((d[r].cpu().double() - b @ a).abs() <= h * U32 * (b.abs() @ a.abs())).all()
    deep_gemm.check_errors()
    d_y = torch.randn(rows.size(0), f, generator=g).bfloat16()
    d_y[ids < 0] = 0
    d_w = torch.empty(n, f, h, dtype=torch.float32, device='cuda')
    deep_gemm.k_grouped_bf16_gemm_tn_contiguous(d_y.cuda(), rows, d_w, None, layout.psum)
    for e in range(n):
        a, b = d_y[ids == e].double(), rows.cpu()[ids == e].double()
        assert ((d_w[e].cpu().double() - a.t() @ b).abs() <= (rows.size(0) + 1) * U32 * (a.abs().t() @ b.abs())).all()
