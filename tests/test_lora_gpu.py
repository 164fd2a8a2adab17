"""Adapters of many requests against the oracle."""
import pytest
import torch

import deep_gemm
from deep_gemm import _lib
from helpers import gen
from oracle import blocks as ob

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
ROUND = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _restore():
    yield
    deep_gemm.set_mk_alignment_for_contiguous_layout(256)
    torch.cuda.synchronize()
    _lib.load().dg_take_errors()


def _inputs(t, adapters, rank, k, n, seed=0, without=0.2, out=torch.bfloat16):
    g = gen(seed + t + k)
    x = torch.randn(t, k, generator=g).bfloat16()
    a = (torch.randn(adapters, rank, k, generator=g) * k ** -0.5).bfloat16()
    b = (torch.randn(adapters, n, rank, generator=g) * rank ** -0.5).bfloat16()
    ids = torch.randint(0, adapters, (t,), generator=g)
    ids[torch.rand(t, generator=g) < without] = -1
    return x, a, b, ids, 0.5 + torch.rand(adapters, generator=g), torch.randn(t, n, generator=g).to(out)


def _layout(ids, adapters, alignment=32):
    deep_gemm.set_mk_alignment_for_contiguous_layout(alignment)
    return deep_gemm.moe_sort(ids.view(-1, 1).cuda(), adapters)


def _check(d, x, a, b, ids, scales, c, some=None):
    """Sums of k and then of the rank in fp32, the inner ones taken to 2^-17, one rounding."""
    rows = torch.arange(x.size(0)) if some is None else some
    want, mag = ob.lora(x[rows], a, b, ids[rows], scales, None if c is None else c[rows])
    off = ((x.size(1) + a.size(1) + 8) * U32 + 2.0 ** -17) * mag
    assert ((d.cpu()[rows].double() - want).abs() <= ROUND[d.dtype] * want.abs() + off).all()


@pytest.mark.parametrize('t,adapters,rank,k,n', [
    (1, 1, 8, 8, 1), (1, 8, 16, 4096, 7168), (2, 3, 24, 72, 33), (16, 16, 16, 2048, 512), (48, 20, 16, 7168, 300), (17, 5, 40, 264, 515),
    (65, 4, 64, 1024, 1031), (31, 2, 128, 512, 96), (5, 3, 256, 136, 77), (40, 3, 200, 4096, 260), (600, 2, 32, 512, 519), (700, 9, 16, 776, 256),
    (1030, 40, 8, 128, 1000), (515, 1, 64, 256, 2056), (2000, 100, 16, 64, 128), (520, 3, 128, 264, 300), (900, 2, 256, 328, 513), (1500, 64, 48, 96, 40),
])
@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
def test_products(t, adapters, rank, k, n, out):
    x, a, b, ids, scales, c = _inputs(t, adapters, rank, k, n, out=out)
    some = torch.arange(t) if t < 300 else torch.randint(0, t, (200,), generator=gen(1))
    dev = [v.cuda() for v in (x, a, b)]
    for alignment in (32, 256) if t < 700 else (64, 96):
        layout = _layout(ids, adapters, alignment)
        d = torch.full((t, n), float('nan'), dtype=out, device='cuda')
        deep_gemm.lora_gemm_nt(*dev, d, layout, scales.cuda(), c.cuda())
        _check(d, x, a, b, ids, scales, c, some)
        assert torch.equal(d.cpu()[ids < 0], c[ids < 0])
        in_place = c.cuda()
        deep_gemm.lora_gemm_nt(*dev, in_place, layout, scales.cuda(), in_place)
        assert torch.equal(in_place, d)
        deep_gemm.lora_gemm_nt(*dev, d, layout)
        _check(d, x, a, b, ids, None, None, some)
        assert (d.cpu()[ids < 0] == 0).all()


@pytest.mark.parametrize('t', [3, 70, 800])
def test_no_token_has_an_adapter_or_all_have_one(t):
    x, a, b, _, scales, c = _inputs(t, 4, 16, 256, 200)
    for one in (-1, 2):
        ids = torch.full((t,), one)
        d = torch.empty(t, 200, dtype=torch.bfloat16, device='cuda')
        deep_gemm.lora_gemm_nt(x.cuda(), a.cuda(), b.cuda(), d, _layout(ids, 4), scales.cuda(), c.cuda())
        _check(d, x, a, b, ids, scales, c)


@pytest.mark.parametrize('t', [9, 600])
def test_other_tokens_numbers_stay_theirs(t):
    """Infinities and NaN of one token, one adapter and the rows behind c touch nobody else's."""
    x, a, b, ids, scales, c = _inputs(t, 3, 24, 256, 100, without=0.3)
    ids[:3] = torch.tensor([0, 0, 1])
    layout = _layout(ids, 3)
    d, e = (torch.empty(t, 100, dtype=torch.bfloat16, device='cuda') for _ in range(2))
    deep_gemm.lora_gemm_nt(x.cuda(), a.cuda(), b.cuda(), d, layout, scales.cuda(), c.cuda())
    x[0, 3], a[1, 2, 5], b[1, 7, 1] = float('nan'), float('inf'), float('nan')
    deep_gemm.lora_gemm_nt(x.cuda(), a.cuda(), b.cuda(), e, layout, scales.cuda(), c.cuda())
    same = (ids != 1) & (torch.arange(t) != 0)
    assert torch.equal(d.cpu()[same], e.cpu()[same]) and torch.isnan(e[0]).all()


def test_groups_past_the_last_adapter_are_reported():
    for t in (20, 700):
        x, a, b, ids, scales, c = _inputs(t, 6, 16, 128, 96)
        layout = _layout(ids, 6)
        d = torch.empty(t, 96, dtype=torch.bfloat16, device='cuda')
        deep_gemm.lora_gemm_nt(x.cuda(), a[:4].cuda(), b[:4].cuda(), d, layout, scales[:4].cuda(), c.cuda())
        with pytest.raises(RuntimeError, match='past the last adapter'):
            deep_gemm.check_errors()
        known = torch.where(ids < 4, ids, -1)
        _check(d, x, a[:4], b[:4], known, scales[:4], c)


def test_strides_and_odd_addresses():
    x, a, b, ids, scales, c = _inputs(70, 4, 16, 128, 101)
    layout = _layout(ids, 4)
    want = torch.empty(70, 101, dtype=torch.bfloat16, device='cuda')
    deep_gemm.lora_gemm_nt(x.cuda(), a.cuda(), b.cuda(), want, layout, scales.cuda(), c.cuda())
    off = lambda t: torch.cat((torch.zeros(*t.shape[:-1], 3, dtype=t.dtype), t, torch.zeros(*t.shape[:-1], 2, dtype=t.dtype)), -1).cuda()[..., 3:3 + t.size(-1)]
    wide = torch.empty(70, 207, dtype=torch.bfloat16, device='cuda')[:, 5:106]
    for xs, As, bs in ((off(x), off(a), off(b)), (x.t().contiguous().t().cuda(), a.transpose(1, 2).contiguous().transpose(1, 2).cuda(), b.cuda())):
        deep_gemm.lora_gemm_nt(xs, As, bs, wide, layout, scales.cuda(), off(c))
        assert torch.equal(wide, want)
    shared = a[:1].cuda().expand(4, 16, 128)   # one matrix for all
    deep_gemm.lora_gemm_nt(x.cuda(), shared, b.cuda(), wide, layout)
    _check(wide.contiguous(), x, a[:1].expand(4, 16, 128), b, ids, None, None)


def test_nothing_to_do():
    a, b = torch.zeros(2, 8, 64, dtype=torch.bfloat16, device='cuda'), torch.zeros(2, 5, 8, dtype=torch.bfloat16, device='cuda')
    layout = _layout(torch.zeros(0, dtype=torch.int32), 2)
    deep_gemm.lora_gemm_nt(torch.zeros(0, 64, dtype=torch.bfloat16, device='cuda'), a, b, torch.zeros(0, 5, device='cuda'), layout)
    layout = _layout(torch.zeros(3, dtype=torch.int32), 2)
    x = torch.ones(3, 64, dtype=torch.bfloat16, device='cuda')
    deep_gemm.lora_gemm_nt(x, a, b[:, :0], torch.zeros(3, 0, device='cuda'), layout)
    # no adapters at all: every token keeps c
    c, d = torch.ones(3, 5, device='cuda'), torch.zeros(3, 5, device='cuda')
    none = _layout(torch.full((3,), -1), 1)
    deep_gemm.lora_gemm_nt(x, a[:0], b[:0], d, none, None, c)
    assert torch.equal(c, d)


def test_outputs_past_4_gib():
    t, n = 70000, 32768
    x, a, b, ids, scales, _ = _inputs(t, 5, 16, 64, n)
    d = torch.ones(t, n, dtype=torch.bfloat16, device='cuda')
    deep_gemm.lora_gemm_nt(x.cuda(), a.cuda(), b.cuda(), d, _layout(ids, 5, 128), scales.cuda(), d)
    for part in (torch.arange(3), torch.arange(t - 3, t)):
        want, mag = ob.lora(x[part], a, b, ids[part], scales, torch.ones(3, n))
        assert ((d[part].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + (90 * U32 + 2.0 ** -17) * mag).all()


@pytest.mark.parametrize('t,adapters,rank,k,n', [(3, 3, 8, 64, 40), (40, 4, 24, 128, 300), (60, 20, 16, 8192, 256), (600, 3, 40, 96, 260),
                                                 (520, 2, 128, 64, 300), (700, 40, 16, 64, 64), (12, 2, 256, 64, 72)])
def test_fp32_outputs_hold_the_inner_products_in_full(t, adapters, rank, k, n):
    """Two products of bf16 to an inner product, and one of the rank to a column: no sum hides what is cut on the way."""
    g = gen(t + n)
    x, a, b = torch.zeros(t, k), torch.randn(adapters, rank, k, generator=g), torch.zeros(adapters, n, rank)
    x[:, 1], x[:, k - 3] = torch.randn(t, generator=g), torch.randn(t, generator=g)
    b[:, torch.arange(n), torch.arange(n) % rank] = torch.randn(adapters, n, generator=g)
    x, a, b = x.bfloat16(), a.bfloat16(), b.bfloat16()
    ids, scales = torch.randint(0, adapters, (t,), generator=g), 0.5 + torch.rand(adapters, generator=g)
    d = torch.empty(t, n, device='cuda')
    deep_gemm.lora_gemm_nt(x.cuda(), a.cuda(), b.cuda(), d, _layout(ids, adapters), scales.cuda())
    want, mag = ob.lora(x, a, b, ids, scales)
    # The sum of two and its scale; the products of the inner product's parts (exact) in as many additions: at most eight steps of at
    # most an unit in the last place each.
    assert ((d.cpu().double() - want).abs() <= 16 * U32 * mag).all()
