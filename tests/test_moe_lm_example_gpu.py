"""The example's training step against plain torch's gradients in fp32, and its 4-bit decoding against the bf16 weights."""
import importlib.util
from pathlib import Path

import pytest
import torch

import deep_gemm
from oracle import mx as ox

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location('moe_lm_step', Path(__file__).resolve().parents[1] / 'examples' / 'moe_lm_step.py')
ex = importlib.util.module_from_spec(spec)
spec.loader.exec_module(ex)


@pytest.fixture(autouse=True)
def _restore():
    yield
    deep_gemm.set_mk_alignment_for_contiguous_layout(256)


def _plain(block, x, target):
    """Loss and gradients by autograd in fp32, on the experts that the bf16 router chooses."""
    ids = ex.route(block, x)[0]
    xf, *ws = (t.float().requires_grad_() for t in (x, *block.parameters()))
    router, up, down, head = ws
    probs = torch.softmax(xf @ router.t(), dim=1)
    top = probs.gather(1, ids)
    w = top / top.sum(1, keepdim=True)
    out = xf
    for e in range(block.experts):
        gate = torch.where(ids == e, w, 0.0).sum(1, keepdim=True)
        out = out + gate * (ex.swiglu(xf @ up[e].t()) @ down[e].t())
    loss = torch.nn.functional.cross_entropy(out @ head.t(), target)
    loss.backward()
    return loss.detach(), [w.grad for w in ws], xf.grad


@pytest.mark.parametrize('tokens,alignment', [(700, 128), (65, 64)])
def test_training_step(tokens, alignment):
    deep_gemm.set_mk_alignment_for_contiguous_layout(alignment)
    block = ex.Block(hidden=256, inner=128, experts=8, topk=3, vocab=1500)
    g = torch.Generator(device='cuda')
    g.manual_seed(3)
    x = torch.randn(tokens, 256, generator=g, device='cuda').bfloat16()
    target = torch.randint(0, 1500, (tokens,), generator=g, device='cuda')
    loss, grads, d_x = ex.train_step(block, x, target)
    ref, ref_grads, ref_x = _plain(block, x, target)
    # bf16 activations and gradients: about ten roundings of 2^-8 / sqrt(3) on the way
    assert abs(float(loss) - float(ref)) < 0.02
    for got, want in zip((*grads, d_x), (*ref_grads, ref_x)):
        assert (got.float() - want).norm() < 10 * 2.0 ** -8 / 3 ** 0.5 * want.norm()


def _quantised(x):
    """fp32 values of x after the oracle's e2m1 quantisation."""
    flat = x.reshape(-1, x.size(-1)).cpu()
    return ox.values(*ox.quantize(flat, 'e2m1'), 'e2m1').float().view(x.shape).to(x.device)


@pytest.mark.parametrize('tokens,alignment', [(1, 32), (8, 32), (40, 32), (9, 64), (40, 256)])
def test_decoding_step(tokens, alignment):
    """The logits of the 4-bit step against fp32 products of dequantised weights and activations, token by token and expert by expert,
    rounded to bf16 where the step holds bf16."""
    deep_gemm.set_mk_alignment_for_contiguous_layout(alignment)
    block = ex.Block(hidden=256, inner=128, experts=8, topk=3, vocab=1500)
    g = torch.Generator(device='cuda')
    g.manual_seed(4)
    x = torch.randn(tokens, 256, generator=g, device='cuda').bfloat16()
    got = ex.decode_step(ex.Quantised(block), x)
    up, down, head = (_quantised(w) for w in (block.up, block.down, block.head))
    ids, weights, _ = ex.route(block, x)
    xq, out = _quantised(x), torch.zeros(tokens, 256, device='cuda')
    for t in range(tokens):
        for c in range(block.topk):
            e = int(ids[t, c])
            h = (xq[t:t + 1] @ up[e].t()).bfloat16()
            out[t] += weights[t, c] * (_quantised(ex.swiglu(h)) @ down[e].t()).bfloat16().float()[0]
    want = _quantised(x + out.bfloat16()) @ head.t()
    # (what is left are sums in another order, and the few values that another last bit takes to the next 4-bit code)
    assert (got - want).norm() < 10 * 2.0 ** -8 / 3 ** 0.5 * want.norm()


def test_training_lowers_the_loss_and_decoding_follows():
    losses, logits = ex.main(steps=10)
    assert losses[-1] < 0.9 * losses[0]
    assert torch.isfinite(logits).all()
