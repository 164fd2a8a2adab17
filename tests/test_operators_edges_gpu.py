"""Sizes of zero, broadcast inputs, tensors of more than 4 GiB and other streams, for the operators around the GEMMs."""
import pytest
import torch

import deep_gemm
from helpers import gen
from oracle import moe as om, mx as ox

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _restore():
    yield
    deep_gemm.set_mk_alignment_for_contiguous_layout(256)


def test_nothing_to_do():
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    for t, k in ((0, 4), (5, 0)):
        layout = deep_gemm.moe_sort(torch.zeros(t, k, dtype=torch.int32, device='cuda'), 6)
        assert layout.source.numel() == 0 and (layout.psum == 0).all()
        x = torch.ones(t, 64, dtype=torch.bfloat16, device='cuda')
        rows = deep_gemm.moe_dispatch(x, layout)
        assert rows.shape == (0, 64)
        w = torch.ones(t, k, device='cuda')
        out = deep_gemm.moe_combine(rows, layout, w)
        assert out.shape == (t, 64) and (out == 0).all()
        d_rows, d_w = deep_gemm.moe_combine_backward(out, rows, layout, w)
        assert d_rows.shape == (0, 64) and d_w.shape == (t, k)
    layout = deep_gemm.moe_sort(torch.zeros(3, 2, dtype=torch.int32, device='cuda'), 4)
    assert deep_gemm.moe_dispatch(torch.ones(3, 0, device='cuda'), layout).shape == (layout.source.numel(), 0)
    assert deep_gemm.moe_combine(torch.ones(layout.source.numel(), 0, device='cuda'), layout).shape == (3, 0)
    for shape in ((0, 64), (4, 0), (0, 4, 64), (2, 0, 32)):
        codes, sf = deep_gemm.mx_quantize(torch.ones(shape, device='cuda'))
        assert codes.shape == (*shape[:-1], shape[-1] // 2) and sf.shape == (*shape[:-1], -(-shape[-1] // 64))
        assert deep_gemm.mx_dequantize((codes, sf)).shape == shape
    q = deep_gemm.mx_quantize(torch.ones(8, 64, device='cuda'))
    d = torch.empty(0, 8, device='cuda')
    deep_gemm.mx_gemm_nt(torch.ones(0, 64, device='cuda'), q, d)


def test_broadcast_inputs():
    """Expanded tensors (a gradient of ones, one row for all tokens) give what their copies give."""
    g = gen(1)
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    layout = deep_gemm.moe_sort(torch.randint(0, 5, (20, 3), generator=g).cuda(), 5)
    m = layout.source.numel()
    rows = torch.randn(m, 48, generator=g).cuda()
    w = torch.rand(20, 1, generator=g).cuda().expand(20, 3)
    for d_out in (torch.ones((), device='cuda').expand(20, 48), torch.randn(48, generator=g).cuda().expand(20, 48)):
        for a, b in zip(deep_gemm.moe_combine_backward(d_out, rows, layout, w),
                        deep_gemm.moe_combine_backward(d_out.contiguous(), rows, layout, w.contiguous())):
            assert torch.equal(a, b)
        assert torch.equal(deep_gemm.moe_dispatch(d_out, layout), deep_gemm.moe_dispatch(d_out.contiguous(), layout))
    one = torch.randn(96, generator=g).cuda().expand(7, 96)
    for a, b in zip(deep_gemm.mx_quantize(one), deep_gemm.mx_quantize(one.contiguous())):
        assert torch.equal(a, b)
    x, v = torch.randn(64, generator=g).bfloat16().cuda().expand(9, 64), torch.randn(100, 64, generator=g).bfloat16().cuda()
    target = torch.full((), 7, device='cuda').expand(9)
    loss, lse = deep_gemm.linear_cross_entropy(x, v, target)
    assert torch.equal(loss, deep_gemm.linear_cross_entropy(x.contiguous(), v, target.contiguous())[0])
    ones = torch.ones((), device='cuda').expand(9)
    for a, b in zip(deep_gemm.linear_cross_entropy_backward(ones, x, v, target, lse),
                    deep_gemm.linear_cross_entropy_backward(ones.contiguous(), x.contiguous(), v, target.contiguous(), lse)):
        assert torch.equal(a, b)


def test_rows_past_4_gib():
    t, n, h = 300000, 3, 8192
    deep_gemm.set_mk_alignment_for_contiguous_layout(64)
    ids = torch.randint(0, n, (t, 1), generator=gen(2)).cuda()
    layout = deep_gemm.moe_sort(ids, n)
    x = torch.randn(t, h, dtype=torch.bfloat16, device='cuda')
    rows = deep_gemm.moe_dispatch(x, layout)
    assert rows.numel() * 2 > 1 << 32
    at = layout.slots[:, 0].long()
    assert torch.equal(ids[:, 0], layout.m_indices[at].long()) and torch.equal(layout.source[at], torch.arange(t, device='cuda', dtype=torch.int32))
    for part in (slice(0, 500), slice(t // 2, t // 2 + 500), slice(t - 500, t)):
        assert torch.equal(rows[at[part]], x[part])
    assert (rows[layout.source < 0] == 0).all()
    assert torch.equal(deep_gemm.moe_combine(rows, layout), x)
    w = torch.full((t, 1), 2.0, device='cuda')
    d_rows, d_w = deep_gemm.moe_combine_backward(x, rows, layout, w)
    for part in (slice(0, 500), slice(t - 500, t)):
        assert torch.equal(d_rows[at[part]], 2 * x[part])
        ref = x[part].double().square().sum(1, keepdim=True)
        assert ((d_w[part].double() - ref).abs() <= h * 2.0 ** -24 * ref).all()


def test_quantisation_past_4_gib():
    m, k = 70000, 32768
    x = torch.empty(m, k, dtype=torch.bfloat16, device='cuda').normal_()
    codes, sf = deep_gemm.mx_quantize(x)
    back = deep_gemm.mx_dequantize((codes, sf))
    for part in (slice(0, 3), slice(m // 2, m // 2 + 3), slice(m - 3, m)):
        want = ox.values(*ox.quantize(x[part].cpu(), 'e2m1'), 'e2m1')
        assert torch.equal(back[part].cpu().double(), want)


def test_vocabulary_past_4_gib():
    t, h, v = 24, 4096, 600001
    x = torch.randn(t, h, dtype=torch.bfloat16, device='cuda')
    w = torch.empty(v, h, dtype=torch.bfloat16, device='cuda').normal_().mul_(h ** -0.5)
    assert w.numel() * 2 > 1 << 32
    target = torch.randint(0, v, (t,), generator=gen(3)).cuda()
    target[0] = v - 1
    d_loss = torch.full((t,), 1.0 / t, device='cuda')
    loss, lse = deep_gemm.linear_cross_entropy(x, w, target)
    d_x, d_w = deep_gemm.linear_cross_entropy_backward(d_loss, x, w, target, lse)
    z = torch.cat([x.float() @ part.float().t() for part in w.split(100000)], dim=1)
    ref = torch.logsumexp(z.double(), 1)
    # (logits of 4096 products in fp32)
    assert (lse.double() - ref).abs().max() < 1e-4
    assert (loss.double() - (ref - z.double().gather(1, target.unsqueeze(1)).squeeze(1))).abs().max() < 2e-4
    p = torch.exp(z - ref.float().unsqueeze(1))
    p[torch.arange(t, device='cuda'), target] -= 1
    p /= t
    ref_x = sum(a @ b.float() for a, b in zip(p.split(100000, dim=1), w.split(100000)))
    assert (d_x.float() - ref_x).norm() < 2 * 2.0 ** -8 / 3 ** 0.5 * ref_x.norm()
    for part in (slice(0, 2000), slice(300000, 302000), slice(v - 2000, v)):
        ref_w = p[:, part].t() @ x.float()
        assert (d_w[part].float() - ref_w).norm() < 2 * 2.0 ** -8 / 3 ** 0.5 * ref_w.norm()


def test_on_another_stream():
    """Everything of a step on a stream of its own, behind work that takes a while on it."""
    g = gen(4)
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    ids, x = torch.randint(0, 9, (200, 4), generator=g).cuda(), torch.randn(200, 96, generator=g).cuda()
    w = torch.rand(200, 4, generator=g).cuda()

    def step(x):
        layout = deep_gemm.moe_sort(ids, 9)
        rows = deep_gemm.moe_dispatch(x, layout)
        q = deep_gemm.mx_dequantize(deep_gemm.mx_quantize(x), torch.float32)
        return rows, deep_gemm.moe_combine(rows, layout, w), *deep_gemm.moe_combine_backward(x, rows, layout, w), q
    want = step(x * 3)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    big = torch.ones(1 << 28, device='cuda')
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        for _ in range(10):
            big.mul_(1.0)
        got = step(x * 3)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
