"""Routing of tokens to experts against the oracle: ids exactly, weights and gradients within their rounding."""
import pytest
import torch

import deep_gemm
from deep_gemm import _lib
from helpers import gen
from oracle import blocks as ob

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
INF = float('inf')
ROUND = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _restore():
    yield
    torch.cuda.synchronize()
    _lib.load().dg_take_errors()


def _logits(t, n, dtype=torch.float32, seed=0):
    return (1.5 * torch.randn(t, n, generator=gen(seed + n))).to(dtype)


def _check(logits, topk, kind='softmax', bias=None, **kw):
    ids, w = deep_gemm.moe_route(logits.cuda(), topk, kind, None if bias is None else bias.cuda(), **kw)
    want, want_w = ob.route(logits, topk, kind, bias, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids.cpu(), want)
    # an exponent's rounding (twice its size in units) and, for softmax, a sum of at most 16 + 6 steps and some operations
    biggest = logits.float().clamp(-100, 100).abs().max()
    assert ((w.cpu().double() - want_w).abs() <= (4 * biggest + 64) * U32 * want_w.abs() + 1e-37).all()
    return ids, w


@pytest.mark.parametrize('t,n,topk,groups,keep', [
    (1, 1, 1, 1, 1), (1, 8, 8, 1, 1), (3, 7, 2, 1, 1), (16, 64, 6, 8, 3), (17, 65, 5, 1, 1), (31, 96, 4, 3, 2), (64, 128, 16, 4, 2),
    (5, 160, 6, 8, 3), (100, 256, 8, 8, 4), (33, 257, 1, 1, 1), (9, 384, 9, 6, 4), (40, 512, 8, 64, 5), (7, 513, 16, 1, 1), (20, 1000, 7, 10, 3),
    (11, 1024, 8, 16, 4),
])
@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('biased', [False, True])
def test_choice(t, n, topk, groups, keep, kind, dtype, biased):
    bias = 0.1 * torch.randn(n, generator=gen(n + 1)) if biased else None
    _check(_logits(t, n, dtype, t), topk, kind, bias, num_groups=groups, topk_groups=keep, renormalize=bool(t % 2), scale=2.5)


@pytest.mark.parametrize('group_top', [1, 2])
@pytest.mark.parametrize('groups', [4, 32, 64])
def test_group_scores(group_top, groups):
    bias = 0.1 * torch.randn(128, generator=gen(3))
    for b in (None, bias):
        _check(_logits(50, 128, seed=5), 4, 'sigmoid', b, num_groups=groups, topk_groups=groups // 2, group_top=group_top)


def test_equal_numbers_go_to_the_lowest_index():
    g = gen(2)
    for kind in ('softmax', 'sigmoid'):
        logits = torch.randint(-2, 3, (60, 256), generator=g).float()
        bias = torch.randint(0, 2, (256,), generator=g) * 0.25
        _check(logits, 8, kind)
        _check(logits.bfloat16(), 8, kind, bias, num_groups=8, topk_groups=3)
        _check(torch.zeros(5, 64), 6, kind, torch.zeros(64), num_groups=4, topk_groups=2)


def test_numbers_that_32_bits_do_not_tell_apart():
    """Logits that differ in their last bits, so that scores and groups' sums are equal in fp32."""
    base = torch.randn(40, 256, generator=gen(4))
    bits = base.view(torch.int32) // 4096 * 4096 + torch.randint(0, 3, (40, 256), generator=gen(5)).int()
    near = bits.view(torch.float32)
    near[:, 1::2] = (bits[:, 0::2] + torch.randint(-1, 2, (40, 128), generator=gen(6)).int()).view(torch.float32)
    bias = torch.full((256,), 0.125)
    for kind in ('softmax', 'sigmoid'):
        _check(near, 8, kind)
        _check(near, 8, kind, bias)
        _check(near, 8, kind, bias, num_groups=8, topk_groups=4)


def test_masks():
    logits = _logits(12, 64)
    logits[0] = -INF                     # nothing left
    logits[1, :] = -INF
    logits[1, 5] = 0.5                   # one expert left
    logits[2, 3:] = -INF                 # three left
    logits[3] = torch.finfo(torch.float32).min
    logits[4, ::2] = torch.finfo(torch.float32).min
    logits[5, 8:16] = -INF               # a whole group out
    for kind in ('softmax', 'sigmoid'):
        for bias in (None, torch.randn(64, generator=gen(7)) * 0.1):
            for groups, keep in ((1, 1), (8, 4)):
                ids, w = _check(logits, 6, kind, bias, num_groups=groups, topk_groups=keep)
                assert (ids[0] == -1).all() and (w[0] == 0).all()
                assert ids[1].tolist()[:2] == [5, -1] and (ids[2] == -1).sum() >= 3
    closed = torch.zeros(64)
    closed[10:50] = -INF                 # experts that are closed for all
    ids, _ = _check(logits[6:], 6, 'sigmoid', closed)
    assert ((ids < 10) | (ids >= 50)).all()


def test_masks_of_the_types_lowest_value():
    low = torch.finfo(torch.bfloat16).min
    logits = _logits(6, 100, torch.bfloat16)
    logits[:, 4:] = low
    _check(logits, 8, 'softmax')
    _check(logits, 8, 'sigmoid', torch.randn(100, generator=gen(1)))


def test_nan_and_infinity_come_first():
    for kind in ('softmax', 'sigmoid'):
        logits = _logits(4, 40)
        logits[1, 7] = float('nan')
        logits[2, 9] = INF
        clean, _ = deep_gemm.moe_route(_logits(4, 40).cuda(), 4, kind)
        ids, w = deep_gemm.moe_route(logits.cuda(), 4, kind)
        assert ids[1, 0] == 7 and ids[2, 0] == 9
        assert torch.isnan(w[1]).any() and torch.equal(ids[[0, 3]], clean[[0, 3]]) and torch.isfinite(w[[0, 3]]).all()


def test_strides_and_odd_addresses():
    whole = torch.randn(50, 203, generator=gen(9))
    for dtype in (torch.float32, torch.bfloat16):
        part = whole.to(dtype).cuda()[:, 1:162]
        a, b = deep_gemm.moe_route(part, 5, 'sigmoid'), deep_gemm.moe_route(part.contiguous(), 5, 'sigmoid')
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        t = whole.to(dtype).cuda().t()   # columns
        a, b = deep_gemm.moe_route(t, 5), deep_gemm.moe_route(t.contiguous(), 5)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        one = part[:1].expand(9, 161)
        assert (deep_gemm.moe_route(one, 5)[0] == deep_gemm.moe_route(part[:1], 5)[0]).all()


@pytest.mark.parametrize('t,n,topk', [(1, 3, 3), (5, 64, 4), (17, 130, 6), (40, 256, 8), (9, 300, 16), (6, 1024, 7)])
@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('renormalize', [True, False])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gradient(t, n, topk, kind, renormalize, dtype):
    logits = _logits(t, n, dtype, 3)
    ids, _ = deep_gemm.moe_route(logits.cuda(), topk, kind)
    if t > 4:
        ids[2, 0] = -1           # a dropped choice
        ids[3, 1] = ids[3, 0]    # an expert that repeats
        ids[4] = -1
    d = torch.randn(t, topk, generator=gen(t))
    got = deep_gemm.moe_route_backward(d.cuda(), logits.cuda(), ids, kind, renormalize, 1.5)
    want, mag = ob.route_backward(d, logits, ids.cpu(), kind, renormalize, 1.5)
    assert got.dtype == dtype
    assert ((got.cpu().double() - want).abs() <= ROUND[dtype] * want.abs() + 100 * U32 * mag).all()


@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
def test_gradient_against_differences(kind):
    logits, d = _logits(4, 20).double(), torch.randn(4, 3, generator=gen(1)).double()
    ids = ob.route(logits, 3, kind)[0]
    weights = lambda l: (lambda w: w / w.sum(1, keepdim=True))(ob.scores(l, kind).gather(1, ids.long()))
    got = deep_gemm.moe_route_backward(d.float().cuda(), logits.float().cuda(), ids.cuda(), kind).cpu().double()
    for e in range(20):
        step = torch.zeros(4, 20).double()
        step[:, e] = 1e-4
        want = ((weights(logits + step) - weights(logits - step)) * d).sum(1) / 2e-4
        # (the rounding of logits to fp32, and the second order of the differences)
        assert ((got[:, e] - want).abs() < 1e-6 + 1e-5 * want.abs()).all()


def test_gradient_reports_ids_past_the_last_expert():
    logits = _logits(3, 10).cuda()
    ids = torch.tensor([[1, 2], [3, 10], [4, 5]], dtype=torch.int32, device='cuda')
    d = torch.ones(3, 2, device='cuda')
    got = deep_gemm.moe_route_backward(d, logits, ids, 'sigmoid', renormalize=False)
    with pytest.raises(RuntimeError, match='expert id'):
        deep_gemm.check_errors()
    ids[1, 1] = -1
    assert torch.equal(got, deep_gemm.moe_route_backward(d, logits, ids, 'sigmoid', renormalize=False))


def test_nothing_to_do_and_dropped_rows():
    for dtype in (torch.float32, torch.bfloat16):
        ids, w = deep_gemm.moe_route(torch.empty(0, 8, device='cuda', dtype=dtype), 3)
        assert ids.shape == w.shape == (0, 3)
        assert deep_gemm.moe_route_backward(w, torch.empty(0, 8, device='cuda', dtype=dtype), ids).shape == (0, 8)
    ids, w = deep_gemm.moe_route(torch.zeros(4, 8, device='cuda'), 0)
    assert ids.shape == (4, 0)
    assert (deep_gemm.moe_route_backward(w, torch.zeros(4, 8, device='cuda'), ids) == 0).all()
    out = torch.full((4, 8), -INF, device='cuda')
    ids, w = deep_gemm.moe_route(out, 2)
    for kind in ('softmax', 'sigmoid'):
        assert (deep_gemm.moe_route_backward(torch.ones(4, 2, device='cuda'), out, ids, kind) == 0).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
def test_zeros_of_either_sign_are_equal(dtype, kind):
    """As logits that were multiplied by a mask hold them: the lowest index among them, of experts and of groups."""
    g = gen(11)
    zero = torch.where(torch.rand(40, 96, generator=g) < 0.5, -0.0, 0.0)
    logits = torch.where(torch.rand(40, 96, generator=g) < 0.3, zero, -torch.rand(40, 96, generator=g) - 0.1).to(dtype)
    logits[0], logits[1] = -1, -1
    logits[0, [3, 10]], logits[1, [3, 10]] = torch.tensor([-0.0, 0.0]).to(dtype), torch.tensor([0.0, -0.0]).to(dtype)
    logits[2] = zero[2]
    for topk in (1, 8):
        _check(logits, topk, kind)
        for groups in (8, 12, 16):   # (12: groups that are a run of lanes; 8 and 16: that are none)
            for group_top in (1, 2):
                _check(logits, min(topk, 3 * (96 // groups)), kind, num_groups=groups, topk_groups=3, group_top=group_top)
    ids, _ = deep_gemm.moe_route(logits[:2].cuda(), 2, kind)
    assert ids.tolist() == [[3, 10], [3, 10]]


@pytest.mark.parametrize('experts,groups', [(4, 2), (64, 8), (256, 8), (60, 10), (96, 16)])
@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
def test_sums_of_groups_that_cancel(experts, groups, kind):
    """The two best of a group lie far from each other and from zero: their sum is small, its rounding in fp32 is not."""
    per = experts // groups
    logits = _logits(600, experts, seed=21)
    for big in (2.0 ** 12, 2.0 ** 16, 1e6, 2.0 ** 20):
        bias = torch.full((experts,), -big)
        bias[torch.arange(groups) * per + torch.arange(groups) % per] = big
        _check(logits, 1, kind, bias, num_groups=groups, topk_groups=1)


@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
def test_closed_experts_beside_nan_stay_closed(kind):
    closed = torch.randn(64, generator=gen(8)) * 0.1
    closed[:20] = -INF
    closed[40:48] = -INF                 # (a whole group of eight among them)
    logits = _logits(6, 64)
    logits[1, 3] = float('nan')          # a closed expert's own logit
    logits[2, [3, 30]] = float('nan')
    logits[3, [5, 33]] = INF
    logits[4] = float('nan')
    logits[5, 21:] = float('nan')
    logits[5, 25] = -INF
    for groups, keep in ((1, 1), (8, 3), (16, 6)):
        ids, _ = deep_gemm.moe_route(logits.cuda(), 6, kind, closed.cuda(), groups, keep)
        want, _ = ob.route(logits, 6, kind, closed, groups, keep)
        assert torch.equal(ids.cpu(), want)
        assert (closed[ids[ids >= 0].long().cpu()] > -INF).all()


def test_numbers_in_64_bits_to_their_last():
    """Scores that differ by a few of a double's last bits, or in none: sigmoids near 1, alone and under a bias."""
    g = gen(31)
    logits = 28 + 12 * torch.rand(60, 128, generator=g)
    logits[::2] = logits[::2].round()
    for bias in (torch.zeros(128), torch.randint(0, 3, (128,), generator=g) * 0.5):
        _check(logits, 8, 'sigmoid', bias)
        _check(logits, 16, 'sigmoid', bias)
        _check(logits, 3, 'sigmoid', bias, num_groups=8, topk_groups=2)
        _check(logits, 3, 'sigmoid', bias, num_groups=32, topk_groups=5)
    far = torch.cat((logits, -logits), 1)   # (and among others far below)
    _check(far, 16, 'sigmoid', torch.zeros(256), num_groups=4, topk_groups=3)
    _check(torch.cat((far, far, far), 1), 16, 'sigmoid', torch.zeros(768))


@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
def test_small_weights_are_as_exact_as_large_ones(kind):
    logits = -80 * torch.rand(200, 16, generator=gen(41))
    logits[:, 3] = torch.rand(200, generator=gen(42))
    ids, w = deep_gemm.moe_route(logits.cuda(), 16, kind, renormalize=False)
    want = ob.scores(logits, kind).gather(1, ids.cpu().long())
    # The exponential (2 units), softmax's sum of 16 (20 units at most, its largest terms exact to 4), a quotient and a product.  Softmax's
    # exponent is a difference in fp32, off by half a step, 2^-24 |l - top| at most; exp(x + e) = exp(x) (1 + e), so by |l - top| units.
    units = torch.tensor(8.0)
    if kind == 'softmax':
        units = 28 + (logits.max(1, keepdim=True).values - logits).double().gather(1, ids.cpu().long())
    assert ((w.cpu().double() - want).abs() <= units * U32 * want).all()
