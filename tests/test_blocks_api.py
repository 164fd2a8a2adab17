"""Argument checks of the operators between the products, through the C ABI and the Python layer (nothing is launched), and their
oracle against other ways to the same numbers."""
import ctypes

import pytest
import torch

import deep_gemm
from deep_gemm import _lib
from helpers import gen
from oracle import blocks as ob


@pytest.fixture(scope='module')
def lib():
    return _lib.load()


def _refused(lib, rc, text):
    assert rc == -1 and text in lib.dg_last_error().decode(), lib.dg_last_error()


def _with(args, kw):
    for name, v in kw.items():
        setattr(args, name, v)
    return args


def test_route_refusals(lib):
    def run(fn='dg_moe_route', **kw):
        a = _lib.MoERouteArgs(4, 64, 6, 0, 8, 4, 2, 1, 1.0, 1, 4096, 64, None, 4096, 4096, 4096, 4096, 64, 0)
        return getattr(lib, fn)(_with(a, kw), None)
    for fn in ('dg_moe_route', 'dg_moe_route_backward'):
        assert getattr(lib, fn)(None, None) == -1
        _refused(lib, run(fn, scores=2), 'unknown scores')
        _refused(lib, run(fn, dtype=2), 'bf16 or fp32')
        _refused(lib, run(fn, tokens=-1), '2^30 tokens')
        _refused(lib, run(fn, experts=0), '1024 experts')
        _refused(lib, run(fn, experts=1025), '1024 experts')
        _refused(lib, run(fn, topk=17), 'at most 16')
        _refused(lib, run(fn, experts=4, num_groups=1, topk_groups=1), 'at most the experts')
        _refused(lib, run(fn, logits_ld=63), 'leading dimension')
        _refused(lib, run(fn, logits=None), 'null tensor')
        _refused(lib, run(fn, ids=None), 'null tensor')
        _refused(lib, run(fn, logits=4098), 'aligned')
        assert run(fn, tokens=0) == 0
    _refused(lib, run(num_groups=7), 'divide the experts')
    _refused(lib, run(num_groups=0), 'divide the experts')
    _refused(lib, run(experts=256, logits_ld=256, num_groups=128), '64 groups')
    _refused(lib, run(topk_groups=9), 'topk_groups')
    _refused(lib, run(topk_groups=0), 'topk_groups')
    _refused(lib, run(group_top=3), 'group_top')
    _refused(lib, run(topk=9, topk_groups=1), "kept groups' experts")
    _refused(lib, run(weights=None), 'null tensor')
    _refused(lib, run('dg_moe_route_backward', d_weights=None), 'null tensor')
    _refused(lib, run('dg_moe_route_backward', d_logits_ld=8), 'leading dimension')


def test_norm_refusals(lib):
    def args(**kw):
        a = _lib.RmsNormArgs()
        for name in ('x', 'weight', 'rstd', 'y', 'h', 'd_y', 'd_x', 'd_weight', 'workspace'):
            setattr(a, name, 4096)
        for name in ('x_ld', 'residual_ld', 'h_ld', 'y_ld', 'd_y_ld', 'd_h_ld', 'd_x_ld'):
            setattr(a, name, 64)
        a.tokens, a.width, a.format, a.workspace_bytes = 4, 64, -1, 1 << 20
        return _with(a, kw)
    f = lambda **kw: lib.dg_rms_norm_forward(args(**kw), None)
    b = lambda **kw: lib.dg_rms_norm_backward(args(**kw), None)
    for run in (f, b):
        _refused(lib, run(dtype=2), 'bf16 or fp32')
        _refused(lib, run(weight_dtype=2), 'bf16 or fp32')
        _refused(lib, run(tokens=-1), '2^30 tokens')
        _refused(lib, run(width=0), '32768')
        _refused(lib, run(width=32769), '32768')
        _refused(lib, run(weight=None), 'null tensor')
        _refused(lib, run(rstd=None), 'null tensor')
        _refused(lib, run(weight=4097), 'aligned')
    _refused(lib, f(format=2), 'unknown format')
    _refused(lib, f(format=1, width=48), 'block of 32')
    _refused(lib, f(format=1), 'null tensor')
    _refused(lib, f(format=1, sf=4096, sf_ld=3), 'leading dimension')
    _refused(lib, f(format=1, sf=4096, sf_ld=5), 'even')
    _refused(lib, f(format=1, sf=4098, sf_ld=4), '4-byte')
    _refused(lib, f(format=1, sf=4096, sf_ld=4, y_ld=68), '8-byte aligned')
    _refused(lib, f(x_ld=63), 'leading dimension')
    _refused(lib, f(residual=4096, residual_ld=8), 'leading dimension')
    _refused(lib, f(residual=4096, h=None), 'null tensor')
    _refused(lib, b(d_y=None), 'null tensor')
    _refused(lib, b(d_x_ld=8), 'leading dimension')
    _refused(lib, b(workspace_bytes=16), 'workspace')
    _refused(lib, b(workspace=None), 'workspace')
    assert f(tokens=0) == 0
    need = ctypes.c_int64()
    assert lib.dg_rms_norm_workspace_size(args(), ctypes.byref(need)) == 0 and need.value > 0
    assert lib.dg_rms_norm_workspace_size(args(), None) == -1 and lib.dg_rms_norm_forward(None, None) == -1 and lib.dg_rms_norm_backward(None, None) == -1


def test_swiglu_refusals(lib):
    def args(**kw):
        a = _lib.SwigluArgs()
        for name in ('h', 'act', 'd_act', 'd_h'):
            setattr(a, name, 4096)
        a.rows, a.width, a.format = 4, 64, -1
        a.h_ld, a.act_ld, a.saved_ld, a.saved_sf_ld, a.act_sf_ld, a.d_act_ld, a.d_h_ld = 128, 64, 128, 4, 4, 64, 128
        return _with(a, kw)
    f = lambda **kw: lib.dg_swiglu_forward(args(**kw), None)
    b = lambda **kw: lib.dg_swiglu_backward(args(**kw), None)
    for run in (f, b):
        _refused(lib, run(dtype=2), 'bf16 or fp32')
        _refused(lib, run(format=2), 'unknown format')
        _refused(lib, run(rows=-1), 'negative size')
        _refused(lib, run(width=1 << 30), 'at most 2^30')
        _refused(lib, run(h_ld=127), 'leading dimension')
        _refused(lib, run(h=4097), 'aligned')
        assert run(rows=0) == 0 and run(width=0) == 0
    _refused(lib, f(format=0, width=48), 'block of 32')
    _refused(lib, f(format=1), 'null tensor')
    _refused(lib, f(format=1, act_sf=4096, act_sf_ld=5), 'even')
    _refused(lib, f(format=1, act_sf=4096, act_ld=68), '8-byte')
    _refused(lib, f(act=None), 'null tensor')
    _refused(lib, f(saved=4096), 'null tensor')
    _refused(lib, f(saved=4096, saved_sf=4096, saved_ld=120), 'leading dimension')
    _refused(lib, f(saved=4096, saved_sf=4096, saved_ld=132), '8-byte')
    _refused(lib, f(saved=4096, saved_sf=4096, width=48), 'block of 32')
    _refused(lib, b(format=1), 'unknown format')
    _refused(lib, b(h=None), 'null tensor')
    _refused(lib, b(d_act=None), 'null tensor')
    _refused(lib, b(d_h_ld=64), 'leading dimension')
    assert lib.dg_swiglu_forward(None, None) == -1 and lib.dg_swiglu_backward(None, None) == -1


def test_lora_refusals(lib):
    layout = _lib.MoELayoutArgs(4, 1, 3, 96, 32, 4096, 4096, 4096, 4096)

    def args(held=layout, **kw):
        a = _lib.LoraArgs()
        for name in ('x', 'a', 'b', 'd', 'workspace'):
            setattr(a, name, 4096)
        a.tokens, a.adapters, a.rank, a.n, a.k = 4, 3, 16, 64, 128
        a.x_ld, a.a_ld, a.a_stride, a.b_ld, a.b_stride, a.c_ld, a.d_ld = 128, 128, 2048, 16, 1024, 64, 64
        a.workspace_bytes = 1 << 30
        if held is not None:
            a.layout = ctypes.pointer(held)
        return _with(a, kw)
    run = lambda held=layout, **kw: lib.dg_lora_gemm(args(held, **kw), None)
    _refused(lib, run(None), 'null args')
    _refused(lib, run(n=-1), 'negative size')
    _refused(lib, run(rank=0), 'multiple of 8')
    _refused(lib, run(rank=12), 'multiple of 8')
    _refused(lib, run(rank=264), 'at most 256')
    _refused(lib, run(k=0), 'multiple of 8')
    _refused(lib, run(k=100), 'multiple of 8')
    _refused(lib, run(d_dtype=2), 'bf16 or fp32')
    _refused(lib, run(tokens=5), 'one choice')
    _refused(lib, run(_lib.MoELayoutArgs(2, 2, 3, 96, 32, 4096, 4096, 4096, 4096), tokens=2), 'one choice')
    _refused(lib, run(_lib.MoELayoutArgs(4, 1, 3, 80, 16, 4096, 4096, 4096, 4096)), 'multiple of 32')
    _refused(lib, run(x=None), 'null tensor')
    _refused(lib, run(b=None), 'null tensor')
    _refused(lib, run(x_ld=120), 'leading dimension')
    _refused(lib, run(d_ld=63), 'leading dimension')
    _refused(lib, run(c=8192, c_ld=63), 'leading dimension')
    _refused(lib, run(x=4104), '16-byte')
    _refused(lib, run(b_ld=20), '16-byte')
    _refused(lib, run(c=4096, c_ld=72), 'leading dimension')
    assert run(n=0) == 0
    need = ctypes.c_int64()
    assert lib.dg_lora_workspace_size(args(), ctypes.byref(need)) == 0 and need.value == 0   # (one launch)
    big = args(k=8192, x_ld=8192, a_ld=8192, a_stride=16 * 8192)
    assert lib.dg_lora_workspace_size(big, ctypes.byref(need)) == 0 and need.value > 0
    big.workspace_bytes = need.value - 1
    _refused(lib, lib.dg_lora_gemm(big, None), 'workspace')


def test_python_refusals():
    x = torch.zeros(4, 64)
    for call in (lambda: deep_gemm.moe_route(x, 2), lambda: deep_gemm.rms_norm(x, x[0]), lambda: deep_gemm.swiglu(x),
                 lambda: deep_gemm.swiglu_backward(x, x), lambda: deep_gemm.rms_norm_backward(x, x, x[0], x[:, 0])):
        with pytest.raises(RuntimeError, match='device tensor'):
            call()
    with pytest.raises(RuntimeError, match='unknown scores'):
        deep_gemm.moe_route(x, 2, 'relu')
    with pytest.raises(RuntimeError, match='unknown scores'):
        deep_gemm.moe_route_backward(x, x, x, 'relu')
    with pytest.raises(RuntimeError, match='unknown format'):
        deep_gemm.rms_norm(x, x[0], fmt='e5m2')
    with pytest.raises(RuntimeError, match='unknown format'):
        deep_gemm.swiglu(x, 'fp8')


# ------------------------------------------------------------------------------------------------ the oracle
@pytest.mark.parametrize('kind', ['softmax', 'sigmoid'])
def test_oracle_route(kind):
    logits, bias = torch.randn(30, 24, generator=gen(1)), 0.1 * torch.randn(24, generator=gen(2))
    s = torch.softmax(logits.double(), 1) if kind == 'softmax' else torch.sigmoid(logits.double())
    ids, w = ob.route(logits, 5, kind, bias, renormalize=False)
    want = (s + bias.double()).topk(5, 1).indices
    assert torch.equal(ids.long(), want) and torch.allclose(w, s.gather(1, want), rtol=1e-12)
    ids, w = ob.route(logits, 5, kind, None, 6, 2, 2, scale=3.0)
    assert torch.allclose(w.sum(1), torch.full((30,), 3.0).double()) and ((ids // 4).sort(1).values.diff(dim=1) != 0).sum(1).max() <= 1
    l = logits.double().requires_grad_()
    p = (torch.softmax(l, 1) if kind == 'softmax' else torch.sigmoid(l)).gather(1, ids.long())
    d = torch.randn(30, 5, generator=gen(3)).double()
    (p / (p.sum(1, keepdim=True) + 1e-20) * 3.0).backward(d)
    assert torch.allclose(ob.route_backward(d, logits, ids, kind, scale=3.0)[0], l.grad, rtol=1e-9, atol=1e-12)


def test_oracle_gradients():
    g = gen(4)
    x, w, d = (torch.randn(7, 12, generator=g).double().requires_grad_(), torch.randn(12, generator=g).double().requires_grad_(),
               torch.randn(7, 12, generator=g).double())
    y = torch.nn.functional.rms_norm(x, (12,), w, 1e-6)
    y.backward(d)
    want, h, rstd = ob.rms_norm(x.detach(), w.detach())
    assert torch.allclose(want, y) and h is not None
    d_x, _, d_w, _ = ob.rms_norm_backward(d, x.detach(), w.detach(), rstd)
    assert torch.allclose(d_x, x.grad) and torch.allclose(d_w, w.grad)
    h = torch.randn(6, 10, generator=g).double().requires_grad_()
    act = torch.nn.functional.silu(h[:, :5]) * h[:, 5:]
    act.backward(d[:6, :5])
    assert torch.allclose(ob.swiglu(h.detach()), act) and torch.allclose(ob.swiglu_backward(d[:6, :5], h.detach())[0], h.grad)


def test_oracle_lora():
    g = gen(5)
    x, a, b = torch.randn(6, 16, generator=g), torch.randn(3, 8, 16, generator=g), torch.randn(3, 5, 8, generator=g)
    ids, s, c = torch.tensor([0, 2, -1, 1, 2, 0]), torch.rand(3, generator=g), torch.randn(6, 5, generator=g)
    want = c.double()
    for e in range(3):
        want = want + torch.where(ids == e, s[e], 0.0).double().unsqueeze(1) * (x.double() @ a[e].double().t() @ b[e].double().t())
    assert torch.allclose(ob.lora(x, a, b, ids, s, c)[0], want)


def test_lora_refuses_layouts_whose_groups_start_anywhere(lib):
    """A tile of 16 or 32 rows belongs to one adapter only where groups start at multiples of 32."""
    a = _lib.LoraArgs()
    for name in ('x', 'a', 'b', 'd', 'workspace'):
        setattr(a, name, 4096)
    a.tokens, a.adapters, a.rank, a.n, a.k = 64, 3, 16, 64, 128
    a.x_ld, a.a_ld, a.a_stride, a.b_ld, a.b_stride, a.c_ld, a.d_ld = 128, 128, 2048, 16, 1024, 64, 64
    for alignment in (1, 8, 16, 48):
        held = _lib.MoELayoutArgs(64, 1, 3, 96, alignment, 4096, 4096, 4096, 4096)
        a.layout = ctypes.pointer(held)
        _refused(lib, lib.dg_lora_gemm(a, None), 'alignment')
        _refused(lib, lib.dg_lora_workspace_size(a, ctypes.byref(ctypes.c_int64())), 'alignment')
