"""Linear cross entropy and its gradient against the 64-bit oracle and against differences."""
import pytest
import torch

import deep_gemm
from deep_gemm import _lib
from helpers import gen
from oracle import loss as ol

pytestmark = pytest.mark.gpu

U32, UBF16 = 2.0 ** -24, 2.0 ** -8
# relative error of an fp32 exponential of an argument that is itself rounded: its own (1 ulp, 2 u) and the argument's
EXP = 2 * U32


def _inputs(t, h, v, seed=0, scale=2.0, ignored=0.2, dtype=torch.int64):
    g = gen(seed + t + h + v)
    x = torch.randn(t, h, generator=g).bfloat16()
    w = (torch.randn(v, h, generator=g) * scale * h ** -0.5).bfloat16()
    target = torch.randint(0, v, (t,), generator=g)
    target[torch.rand(t, generator=g) < ignored] = -100
    return x, w, target.to(dtype), torch.rand(t, generator=g) / max(t, 1)


def _logit_error(x, w):
    """Bound of the error of an fp32 logit: h products added in fp32."""
    return x.shape[1] * U32 * (x.double().abs() @ w.double().abs().t())


def _check(x, w, target, d_loss, dev=None):
    dx, dw, dt, dl = dev or (x.cuda(), w.cuda(), target.cuda(), d_loss.cuda() if d_loss is not None else None)
    loss, lse = deep_gemm.linear_cross_entropy(dx, dw, dt)
    want, want_lse, z = ol.forward(x, w, target)
    e = _logit_error(x, w)
    span = (z.amax(1) - z.amin(1)).unsqueeze(1)
    # lse: the largest error of a logit, the exponentials' (their arguments are differences of logits in units of log 2),
    # the additions of v terms and the roundings of the result
    v = w.shape[0]
    bound = e.amax(1) + EXP + (4 + span.squeeze(1)) * U32 + min(v, 2048) * U32 + 4 * U32 * (want_lse.abs() + z.abs().amax(1) + 1)
    assert ((lse.cpu().double() - want_lse).abs() <= bound).all()
    live = target >= 0
    assert (loss.cpu()[~live] == 0).all()
    assert ((loss.cpu().double() - want).abs()[live] <= (2 * bound)[live]).all()
    if d_loss is None:
        return
    got_x, got_w = deep_gemm.linear_cross_entropy_backward(dl, dx, dw, dt, lse)
    d = ol.d_logits(x, w, target, d_loss)
    # d: the errors of logit and lse in the exponent, the exponential's, the subtraction's, then bf16
    p = torch.exp(z - want_lse.unsqueeze(1)) * torch.where(live, d_loss.double(), 0.0).unsqueeze(1)
    err = p * (e + bound.unsqueeze(1) + EXP + (4 + span) * U32) + 4 * U32 * d.abs()
    err = err * (1 + UBF16) + UBF16 * d.abs()
    for got, ref, other, er, dd in ((got_x, d @ w.double(), w.double(), err, d), (got_w, d.t() @ x.double(), x.double(), err.t(), d.t())):
        n = other.shape[0]
        bound_g = er @ other.abs() + (n + 8) * U32 * (dd.abs() @ other.abs()) * 2
        bound_g = bound_g * (1 + UBF16) + UBF16 * ref.abs()
        assert ((got.cpu().double() - ref).abs() <= bound_g + 1e-40).all()


@pytest.mark.parametrize('t,h,v', [
    (1, 8, 1), (1, 64, 1000), (2, 128, 255), (5, 72, 257), (8, 64, 300), (63, 200, 999), (129, 136, 1025), (130, 512, 129),
    (257, 64, 2049), (300, 256, 3000), (520, 1024, 700), (1, 2048, 5003), (17, 1536, 4001),
])
@pytest.mark.parametrize('dtype', [torch.int64, torch.int32])
def test_loss_and_gradient(t, h, v, dtype):
    _check(*_inputs(t, h, v, dtype=dtype))


@pytest.mark.parametrize('t', [16, 31, 32, 33, 64, 65, 96, 255, 256])
@pytest.mark.parametrize('h,v', [(8, 130), (136, 127), (392, 300), (1024, 2049)])
def test_gradients_of_few_tokens(t, h, v):
    """Up to 256 tokens the gradient of w is a kernel of short K: whole and cut stages of 32 tokens, tiles of 128 words and values."""
    _check(*_inputs(t, h, v, seed=1))


@pytest.mark.parametrize('t', [5, 40, 300])
@pytest.mark.parametrize('h,v', [(72, 257), (136, 128)])
def test_gradients_stay_within_their_rows(t, h, v):
    """Leading dimensions past the width: nothing but the rows' values is written, and nothing behind the inputs is read."""
    x, w, target, d_loss = _inputs(t, h, v, seed=2)
    wide = [torch.full((n + 2, h + 24), float('nan'), dtype=torch.bfloat16, device='cuda') for n in (t, v)]
    for buf, rows in zip(wide, (x, w)):
        buf[1:-1, 8:8 + h] = rows.cuda()
    dx, dw, dt, dl = wide[0][1:-1, 8:8 + h], wide[1][1:-1, 8:8 + h], target.cuda(), d_loss.cuda()
    _check(x, w, target, d_loss, (dx, dw, dt, dl))
    _, lse = deep_gemm.linear_cross_entropy(dx, dw, dt)
    want = deep_gemm.linear_cross_entropy_backward(dl, dx, dw, dt, lse)
    keep, a = deep_gemm.loss._args(dx, dw, dt, -100)
    assert a.x_ld == a.w_ld == h + 24
    out = [torch.full((n + 2, h + 24), 7.0, dtype=torch.bfloat16, device='cuda') for n in (t, v)]
    a.lse, a.d_loss, a.d_x_ld, a.d_w_ld = lse.data_ptr(), dl.data_ptr(), h + 24, h + 24
    a.d_x, a.d_w = out[0][1:, 8:].data_ptr(), out[1][1:, 8:].data_ptr()
    deep_gemm.loss._run('dg_linear_xent_backward', a, 1, dx)
    for buf, ref in zip(out, want):
        assert torch.equal(buf[1:-1, 8:8 + h], ref)
        buf[1:-1, 8:8 + h] = 7.0
        assert (buf == 7.0).all()


def test_large_logits_and_sharp_rows():
    """Logits of several hundred: exponentials of anything but the largest vanish, and nothing overflows.  (The gradient's
    entries below the smallest normal fp32 number, which the matrix unit flushes, have no relative bound: gradients are
    compared at logits of tens.)"""
    for scale in (10.0, 200.0):
        x, w, target, d_loss = _inputs(40, 128, 600, scale=scale, ignored=0.0)
        target[:20] = (x.double() @ w.double().t()).argmax(1)[:20]
        _check(x, w, target, d_loss if scale == 10.0 else None)
    loss, lse = deep_gemm.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda())
    for got in deep_gemm.linear_cross_entropy_backward(d_loss.cuda(), x.cuda(), w.cuda(), target.cuda(), lse):
        assert torch.isfinite(got).all()


def test_all_tokens_ignored():
    x, w, _, d_loss = _inputs(33, 64, 500)
    target = torch.full((33,), -100)
    loss, lse = deep_gemm.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda())
    got_x, got_w = deep_gemm.linear_cross_entropy_backward(d_loss.cuda(), x.cuda(), w.cuda(), target.cuda(), lse)
    assert (loss == 0).all() and (got_x == 0).all() and (got_w == 0).all()


def test_nan_stays_in_its_token():
    """A token of NaN: its loss is NaN, the other tokens' losses and d_x are not; ignored, its d_x is 0."""
    x, w, target, d_loss = _inputs(20, 64, 300, ignored=0.0)
    x[3] = float('nan')
    loss, lse = deep_gemm.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda())
    assert torch.equal(loss.isnan().cpu(), torch.arange(20) == 3)
    got_x, _ = deep_gemm.linear_cross_entropy_backward(d_loss.cuda(), x.cuda(), w.cuda(), target.cuda(), lse)
    assert torch.equal(got_x.isnan().any(1).cpu(), torch.arange(20) == 3)
    target[3] = -100
    d_loss[3] = float('inf')
    loss, lse = deep_gemm.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda())
    got_x, _ = deep_gemm.linear_cross_entropy_backward(d_loss.cuda(), x.cuda(), w.cuda(), target.cuda(), lse)
    assert not loss.isnan().any() and (got_x[3] == 0).all() and not got_x.isnan().any()


def test_ignore_index_and_targets_outside_the_vocabulary():
    x, w, target, d_loss = _inputs(50, 64, 300, ignored=0.0)
    target[:10] = 7
    loss, _ = deep_gemm.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda(), ignore_index=7)
    want = ol.forward(x, w, target, 7)[0]
    assert (loss[:10] == 0).all() and torch.allclose(loss.cpu().double(), want, atol=1e-4)
    deep_gemm.check_errors()
    target[:2] = torch.tensor([300, -5])
    loss, lse = deep_gemm.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda())
    assert (loss[:2] == 0).all() and (loss[2:] != 0).all()
    with pytest.raises(RuntimeError, match='outside the vocabulary'):
        deep_gemm.check_errors()
    got_x, _ = deep_gemm.linear_cross_entropy_backward(d_loss.cuda(), x.cuda(), w.cuda(), target.cuda(), lse)
    assert (got_x[:2] == 0).all() and (got_x[2:] != 0).any(1).all()


def test_strided_rows_and_what_lies_beside_them():
    """Rows with a stride; NaN around x and w is read by nothing (9 tokens, 331 words: no whole pieces)."""
    x, w, target, d_loss = _inputs(9, 72, 331)
    held = []
    for t in (x, w):
        wide = torch.full((t.shape[0] + 16, 96), float('nan'), dtype=torch.bfloat16, device='cuda')
        wide[8:-8, 8:80] = t.cuda()
        held.append(wide[8:-8, 8:80])
    _check(x, w, target, d_loss, (held[0], held[1], target.cuda(), d_loss.cuda()))
    _check(x, w, target, d_loss, (x.t().contiguous().t().cuda(), held[1], target.cuda(), d_loss.cuda()))


def test_python_path_matches_the_extension(monkeypatch):
    x, w, target, d_loss = (a.cuda() for a in _inputs(70, 64, 400))
    def both():
        loss, lse = deep_gemm.linear_cross_entropy(x, w, target)
        return loss, lse, *deep_gemm.linear_cross_entropy_backward(d_loss, x, w, target, lse)
    fast = both()
    monkeypatch.setattr('deep_gemm.loss._operators', lambda t: None)
    for a, b in zip(both(), fast):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_no_tokens():
    w = torch.ones(30, 64, dtype=torch.bfloat16, device='cuda')
    x, target, d_loss = w[:0], torch.zeros(0, dtype=torch.int64, device='cuda'), torch.zeros(0, device='cuda')
    loss, lse = deep_gemm.linear_cross_entropy(x, w, target)
    assert loss.shape == lse.shape == (0,)
    d_x, d_w = deep_gemm.linear_cross_entropy_backward(d_loss, x, w, target, lse)
    assert d_x.shape == (0, 64) and (d_w == 0).all() and d_w.shape == w.shape


def test_pieces_of_the_vocabulary():
    """More words than one piece holds: d_x is summed over the pieces (against fp32 products on this device)."""
    t, h, v = 8200, 128, 70001
    x, w, target, d_loss = (a.cuda() for a in _inputs(t, h, v))
    a = _lib.LinearXentArgs()
    a.tokens, a.width, a.vocab, a.x_ld, a.w_ld, a.x, a.w, a.target_bytes = t, h, v, h, h, x.data_ptr(), w.data_ptr(), 8
    import ctypes
    need = ctypes.c_int64()
    assert _lib.load().dg_linear_xent_workspace_size(a, 1, ctypes.byref(need)) == 0
    assert need.value < 2 * t * v   # (it holds a part of the words)
    loss, lse = deep_gemm.linear_cross_entropy(x, w, target)
    got_x, got_w = deep_gemm.linear_cross_entropy_backward(d_loss, x, w, target, lse)
    z = x.float() @ w.float().t()
    ref = torch.logsumexp(z, 1)
    assert (lse - ref).abs().max() < 1e-4
    p = torch.exp(z - ref.unsqueeze(1))
    p[torch.arange(t, device='cuda'), target.clamp(min=0)] -= 1
    p *= torch.where(target >= 0, d_loss, 0.0).unsqueeze(1)
    # (bf16 in d and in the result: each within 2^-8 of a value, 2^-8 / sqrt(3) at random)
    for got, want in ((got_x, p @ w.float()), (got_w, p.t() @ x.float())):
        assert (got.float() - want).norm() < 2 * UBF16 / 3 ** 0.5 * want.norm()
        assert torch.isfinite(got).all()


@pytest.mark.parametrize('t', [1, 40, 256, 257])
def test_gradients_follow_the_weights_of_the_losses(t):
    """d is held in units of the largest |d_loss|: a power of two times all of them is that times the gradients, to the last bit, and
    an ignored token's d_loss has no part in it.  (Another sign is not: the matrix unit's sums round differently for it.)"""
    x, w, target, d_loss = (a.cuda() for a in _inputs(t, 72, 1025, seed=3))
    target[0] = 1024
    lse = deep_gemm.linear_cross_entropy(x, w, target)[1]
    want = deep_gemm.linear_cross_entropy_backward(d_loss, x, w, target, lse)
    for times in (2.0 ** 20, 2.0 ** -20):
        got = deep_gemm.linear_cross_entropy_backward(d_loss * times, x, w, target, lse)
        for a, b in zip(got, want):
            assert torch.equal(a.float(), b.float() * times)
    for loud in (1e30, float('inf'), float('nan')):
        got = deep_gemm.linear_cross_entropy_backward(torch.where(target < 0, loud, d_loss), x, w, target, lse)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for d in deep_gemm.linear_cross_entropy_backward(torch.zeros_like(d_loss), x, w, target, lse):
        assert (d == 0).all()


@pytest.mark.parametrize('t', [5, 256, 257])
def test_pieces_of_strided_words(t):
    """Rows of w so far apart that 9000 of them are two pieces: d_x is complete, and rounded once, behind the second."""
    x, w, target, d_loss = _inputs(t, 64, 9000, seed=4)
    target[0], target[1] = 8999, 0
    held = torch.empty((9000, 1 << 16), dtype=torch.bfloat16, device='cuda')[:, :64]
    held.copy_(w)
    _check(x, w, target, d_loss, (x.cuda(), held, target.cuda(), d_loss.cuda()))


@pytest.mark.parametrize('t', [1020, 1030, 1100, 2200])
def test_gradient_of_rows_past_2_and_4_gib(t):
    """Rows of x 2 MiB apart, 1024 of them to 2 GiB: every token takes part in d_w, and with its own row."""
    x, w, target, d_loss = _inputs(t, 72, 300, seed=5)
    target[-1], target[1024 % t] = 299, 7
    held = torch.empty((t, 1 << 20), dtype=torch.bfloat16, device='cuda')[:, :72]
    held.copy_(x)
    _check(x, w, target, d_loss, (held, w.cuda(), target.cuda(), d_loss.cuda()))


def test_gradient_of_the_most_tokens():
    """2^20 whole rows of width 1032 (2.16 GB), against fp32 products on this device."""
    t, h, v = 1 << 20, 1032, 40
    x = torch.empty(t, h, dtype=torch.bfloat16, device='cuda').normal_()
    w = torch.empty(v, h, dtype=torch.bfloat16, device='cuda').normal_().mul_(h ** -0.5)
    target = torch.randint(0, v, (t,), generator=gen(6)).cuda()
    d_loss = (torch.rand(t, generator=gen(7)) / t).cuda()
    lse = deep_gemm.linear_cross_entropy(x, w, target)[1]
    got_x, got_w = deep_gemm.linear_cross_entropy_backward(d_loss, x, w, target, lse)
    ref_w = torch.zeros(v, h, dtype=torch.float64, device='cuda')
    wf = w.float()
    for i in range(0, t, 1 << 16):
        part = slice(i, i + (1 << 16))
        xf = x[part].float()
        p = torch.softmax(xf @ wf.t(), dim=1)
        p[torch.arange(1 << 16, device='cuda'), target[part]] -= 1
        p *= d_loss[part].unsqueeze(1)
        ref_w += (p.t().contiguous() @ xf).double()
        ref_x = p @ wf
        # (bf16 in d and in the result: each within 2^-8 of a value, 2^-8 / sqrt(3) at random)
        assert (got_x[part].float() - ref_x).norm() < 2 * UBF16 / 3 ** 0.5 * ref_x.norm()
    assert (got_w.double() - ref_w).norm() < 2 * UBF16 / 3 ** 0.5 * ref_w.norm()


@pytest.mark.parametrize('t', [1, 5, 255, 257, 600])
@pytest.mark.parametrize('v,ld', [(1000, 72), (9000, 1 << 16)])
def test_targets_count_in_full_whatever_the_weights(t, v, ld):
    """d_x where the words that are targets are 32 times as large as the others (in columns that x does not have, so that they are as
    likely as any): the target's term is all but alone in its sum, and nothing but the result's rounding may be left of it."""
    x, w, target, d_loss = _inputs(t, 72, v, seed=8)
    x[:, 36:] = 0
    words = torch.tensor([0, 3, 130, 255, 256, 511, v // 2, v - 1])
    w[words, 36:] = torch.randn(8, 36, generator=gen(t)).bfloat16() * 32
    target = torch.where(target >= 0, words[target % 8], target)
    target[0] = v - 1
    held = torch.empty((v, ld), dtype=torch.bfloat16, device='cuda')[:, :72]
    held.copy_(w)
    args = x.cuda(), held, target.cuda()
    lse = deep_gemm.linear_cross_entropy(*args)[1]
    got = deep_gemm.linear_cross_entropy_backward(d_loss.cuda(), *args, lse)[0].cpu().double()
    d = ol.d_logits(x, w, target, d_loss)
    _, want_lse, z = ol.forward(x, w, target)
    live, at, u = target >= 0, torch.where(target >= 0, target, 0), UBF16   # (u: a rounding to bf16, eight bits)
    e = _logit_error(x, w)
    span = (z.amax(1) - z.amin(1)).unsqueeze(1)
    lse_error = e.amax(1) + EXP + (4 + span.squeeze(1)) * U32 + v * U32 + 4 * U32 * (want_lse.abs() + z.abs().amax(1) + 1)
    p = torch.exp(z - want_lse.unsqueeze(1)) * torch.where(live, d_loss.double(), 0.0).unsqueeze(1)
    err = p * (e + lse_error.unsqueeze(1) + EXP + (4 + span) * U32) + 8 * U32 * d.abs()
    rounded = u * d.abs() * (1 + u)
    rounded[torch.arange(t), at] = 0
    ref = d @ w.double()
    # (products and sums in fp32, in pieces and ranges: as many additions as words)
    bound = (err + rounded) @ w.double().abs() + (v + 16) * U32 * (d.abs() @ w.double().abs())
    bound = bound * (1 + u) + u * ref.abs()
    assert ((got - ref).abs() <= bound + 1e-40).all()


def test_gradient_against_differences():
    g = gen(9)
    t, h, v = 24, 64, 200
    x, w, target, d_loss = _inputs(t, h, v, ignored=0.1)
    loss, lse = deep_gemm.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda())
    got_x, got_w = deep_gemm.linear_cross_entropy_backward(d_loss.cuda(), x.cuda(), w.cuda(), target.cuda(), lse)
    dx, dw = torch.randn(t, h, generator=g).double(), torch.randn(v, h, generator=g).double() * h ** -0.5
    f = lambda x, w: float((ol.forward(x, w, target)[0] * d_loss.double()).sum())
    step = 1e-4
    by_x = (f(x.double() + step * dx, w) - f(x.double() - step * dx, w)) / (2 * step)
    by_w = (f(x, w.double() + step * dw) - f(x, w.double() - step * dw)) / (2 * step)
    # (bf16 gradients: 2^-8 of every term twice, once in d and once in the result; differences: a third derivative's share)
    for got, d, want in ((got_x, dx, by_x), (got_w, dw, by_w)):
        terms = (got.cpu().double() * d).abs().sum()
        assert abs(float((got.cpu().double() * d).sum()) - want) < 2 * UBF16 * float(terms) + 1e-6


def test_under_a_cu_cap_and_in_a_graph():
    x, w, target, d_loss = (a.cuda() for a in _inputs(300, 128, 3000))
    def both():
        loss, lse = deep_gemm.linear_cross_entropy(x, w, target)
        return loss, lse, *deep_gemm.linear_cross_entropy_backward(d_loss, x, w, target, lse)
    want = both()
    full = deep_gemm.get_num_sms()
    try:
        deep_gemm.set_num_sms(24)
        capped = both()
    finally:
        deep_gemm.set_num_sms(full)
    # (fewer CUs may take other tiles: sums in another order)
    for a, b in zip(capped, want):
        assert (a.float() - b.float()).norm() <= UBF16 * b.float().norm()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = both()
    for s in (1.0, 2.0, 0.5, 1.0):
        x.mul_(s)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, both()):
            assert torch.equal(a, b)
