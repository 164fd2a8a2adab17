"""The operators between the products under a CU cap, on other streams, from several calls at once, in captured graphs beside eager
work, and together in a layer."""
import importlib.util
from pathlib import Path

import pytest
import torch

import deep_gemm
from helpers import gen

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _restore():
    yield
    deep_gemm.set_mk_alignment_for_contiguous_layout(256)


def _layer(s):
    """Every operator once, on the inputs s; flat outputs."""
    ids, w = deep_gemm.moe_route(s['logits'], 4, 'sigmoid', s['bias'], 8, 3)
    d_logits = deep_gemm.moe_route_backward(s['dw'], s['logits'], ids, 'sigmoid')
    q, h, rstd = deep_gemm.rms_norm(s['x'], s['weight'], s['res'], fmt='e4m3')
    d_x, d_weight = deep_gemm.rms_norm_backward(s['dy'], h, s['weight'], rstd, s['dh'])
    act, saved = deep_gemm.swiglu(s['x'], 'e4m3', True, s['idx'])
    d_h, again = deep_gemm.swiglu_backward(s['dy'][:, :256].contiguous(), saved, True, s['idx'])
    d = torch.empty_like(s['c'])
    deep_gemm.lora_gemm_nt(s['x'], s['a'], s['b'], d, s['layout'], s['scales'], s['c'])
    return [ids, w, d_logits, q[0].view(torch.uint8), q[1], h, rstd, d_x, d_weight, act[0].view(torch.uint8), act[1], saved[0].view(torch.uint8),
            saved[1], d_h, again, d]


def _inputs(t, seed=0):
    g = gen(seed)
    n = lambda *shape: torch.randn(*shape, generator=g).cuda()
    ids = torch.randint(-1, 6, (t, 1), generator=g).cuda()
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    return {'logits': n(t, 64), 'bias': 0.1 * n(64), 'dw': n(t, 4), 'x': n(t, 512).bfloat16(), 'res': n(t, 512).bfloat16(), 'weight': n(512).bfloat16(),
            'dy': n(t, 512).bfloat16(), 'dh': n(t, 512).bfloat16(), 'idx': torch.where(torch.rand(t, generator=g) < 0.3, -1, 1).int().cuda(),
            'a': n(6, 32, 512).bfloat16(), 'b': n(6, 300, 32).bfloat16(), 'scales': n(6), 'c': n(t, 300).bfloat16(), 'layout': deep_gemm.moe_sort(ids, 6)}


def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('t', [1, 33, 2500])
def test_the_same_every_time_and_under_a_cu_cap(t):
    s = _inputs(t)
    want = _layer(s)
    assert _equal(_layer(s), want)
    whole = deep_gemm.get_num_sms()
    try:
        for n in (1, 24):
            deep_gemm.set_num_sms(n)
            assert _equal(_layer(s), want)
    finally:
        deep_gemm.set_num_sms(whole)


def test_the_python_path_gives_the_same(monkeypatch):
    from deep_gemm import _lib
    s = _inputs(300)
    want = _layer(s)
    monkeypatch.setattr(_lib, '_ext', None)
    monkeypatch.setattr(_lib, '_ext_tried', True)
    assert _equal(_layer(s), want)


def test_on_other_streams_at_once():
    """Two streams, each behind work of its own, with calls that alternate."""
    states = [_inputs(700, i) for i in range(2)]
    want = [_layer(s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    big = [torch.ones(1 << 26, device='cuda') for _ in states]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                big[i].mul_(1.0)
                got[i].append(_layer(states[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(_equal(g, want[i]) for g in got[i])


def test_captured_and_replayed_beside_eager_calls():
    s, other = _inputs(600), _inputs(600, 5)
    want, want_other = [v.clone() for v in _layer(s)], [v.clone() for v in _layer(other)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            _layer(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):   # (two graphs, with memory of their own)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(_layer(s))
        graphs.append(graph)
    names = ('logits', 'x', 'res', 'dy', 'c')
    first = {n: s[n].clone() for n in names}
    for turn in range(4):
        for n in names:
            s[n].copy_(first[n] if turn % 2 == 0 else other[n])
        for graph, out in zip(graphs, outs):
            graph.replay()
            eager = _layer(s)
            torch.cuda.synchronize()
            assert _equal(out, eager)
            if turn % 2 == 0:
                assert _equal(out, want)
    assert _equal(_layer(other), want_other)


spec = importlib.util.spec_from_file_location('moe_layer', Path(__file__).resolve().parents[1] / 'examples' / 'moe_layer.py')
ex = importlib.util.module_from_spec(spec)
spec.loader.exec_module(ex)


@pytest.mark.parametrize('tokens', [65, 700])
def test_the_layers_training_step(tokens):
    """Gradients of the example's layer against autograd in fp32 on the experts that the router chose."""
    layer = ex.Layer(hidden=256, inner=128, experts=16, topk=3, groups=4, topk_groups=2)
    g = torch.Generator(device='cuda')
    g.manual_seed(3)
    x, res, d_out = (torch.randn(tokens, 256, generator=g, device='cuda').bfloat16() for _ in range(3))
    deep_gemm.set_mk_alignment_for_contiguous_layout(128)
    out, kept = ex.forward(layer, x, res)
    d_x, grads = ex.backward(layer, kept, d_out)
    ids = kept['ids']
    xf, rf, *ws = (t.float().requires_grad_() for t in (x, res, *layer.parameters()))
    weight, router, up, down = ws
    h = xf + rf
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * weight
    p = torch.sigmoid(y @ router.t()).gather(1, ids.long())
    w = 2.5 * p / p.sum(1, keepdim=True)
    ref = h
    for e in range(16):
        gate, lin = (y @ up[e].t()).chunk(2, dim=1)
        ref = ref + torch.where(ids == e, w, 0.0).sum(1, keepdim=True) * ((torch.nn.functional.silu(gate) * lin) @ down[e].t())
    ref.backward(d_out.float())
    assert (out.float() - ref).norm() < 10 * 2.0 ** -8 / 3 ** 0.5 * ref.norm()
    # Activations in 8 bits for the gradient: values off by up to 2^-4 (2^-4 / sqrt(3) / 2 on average over a step's range, in the gate
    # and in the other half), beside about ten roundings to bf16.
    for got, want in zip((d_x, *grads), (xf.grad, *(w.grad for w in ws))):
        assert (got.float() - want).norm() < (2 * 2.0 ** -4 / 3 ** 0.5 + 10 * 2.0 ** -8 / 3 ** 0.5) * want.norm()


@pytest.mark.parametrize('tokens', [1, 9, 40])
def test_the_layers_decoding_step(tokens):
    layer = ex.Layer(hidden=256, inner=128, experts=16, topk=3, groups=4, topk_groups=2)
    g = torch.Generator(device='cuda')
    g.manual_seed(4)
    x, res = (torch.randn(tokens, 256, generator=g, device='cuda').bfloat16() for _ in range(2))
    deep_gemm.set_mk_alignment_for_contiguous_layout(128)
    want, _ = ex.forward(layer, x, res)
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    served = ex.Served(layer, adapters=3, rank=8)
    none = deep_gemm.moe_sort(torch.full((tokens, 1), -1, device='cuda'), 3)
    out = ex.decode(served, x, res, none)
    # e4m3 rows and weights through two products, each off by up to 2^-4 of a value
    assert (out.float() - want.float()).norm() < 4 * 2.0 ** -4 / 3 ** 0.5 * want.float().norm()
    some = deep_gemm.moe_sort((torch.arange(tokens, device='cuda') % 3).view(-1, 1), 3)
    with_adapters = ex.decode(served, x, res, some)
    h = (x.float() + res.float()).bfloat16()
    for t in range(tokens):
        e = t % 3
        delta = (h[t].float() @ served.a[e].float().t()) @ served.b[e].float().t()
        ref = out[t].float() + delta
        assert (with_adapters[t].float() - ref).norm() < 4 * 2.0 ** -8 * ref.norm()


def test_example_runs():
    ex.main(tokens=100)


def _ends(n, k=5):
    """The first rows, those around the end of a first launch of 2^32 threads, and the last."""
    return [slice(0, k), slice(n // 2, n // 2 + k), slice(n - 40, n)]


def test_routes_of_more_threads_than_one_launch_has():
    t = (1 << 28) + 37                     # (16 threads to a token)
    logits = torch.empty(t, 2, dtype=torch.bfloat16, device='cuda').normal_()
    ids, w = deep_gemm.moe_route(logits, 1)
    assert torch.equal(ids[:, 0] == 1, logits[:, 1] > logits[:, 0]) and (w == 1).all()
    d = torch.ones(t, 1, device='cuda')
    d_logits = deep_gemm.moe_route_backward(d, logits, ids, renormalize=False)
    for part in _ends(t):
        assert torch.equal(d_logits[part], deep_gemm.moe_route_backward(d[part], logits[part], ids[part], renormalize=False))


def test_norms_of_more_threads_than_one_launch_has():
    t, h = (1 << 22) + 41, 4104            # (1024 threads to a row)
    x = torch.ones(t, h, dtype=torch.bfloat16, device='cuda')
    for part in _ends(t):
        x[part].normal_()
    w = torch.ones(h, dtype=torch.bfloat16, device='cuda')
    y, _, rstd = deep_gemm.rms_norm(x, w)
    for part in _ends(t):
        want = deep_gemm.rms_norm(x[part], w)
        assert torch.equal(y[part], want[0]) and torch.equal(rstd[part], want[2])


def test_activations_of_more_threads_than_one_launch_has():
    m = 1 << 30                            # (four threads to a row)
    h = torch.empty(m, 2, dtype=torch.bfloat16, device='cuda').normal_()
    act = deep_gemm.swiglu(h)
    for part in _ends(m):
        assert torch.equal(act[part], deep_gemm.swiglu(h[part]))
