"""One mixture-of-experts block under a language-model head: training steps in bf16, then decoding with 4-bit weights.

    python examples/moe_lm_step.py

Training: route, sort the tokens by expert, move them into the rows of an M-grouped layout, the experts' two products, weighted
sums back, and the loss over the vocabulary without its logits; then the gradient of all of it, weights' gradients by K-grouped
products over the same rows.  Decoding: the trained weights in e2m1, tokens quantised and moved with their scale factors, the
head as a product that quantises its rows itself.
"""
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'deepgemm-ascend_amd'))

import torch  # noqa: E402
import torch.nn.functional as F  # noqa: E402

import deep_gemm  # noqa: E402


class Block:
    """Weights of the block: router [E, H], experts' gate and up [E, 2 F, H] and down [E, H, F], head [V, H]."""

    def __init__(self, hidden=512, inner=256, experts=16, topk=4, vocab=5000, seed=0, device='cuda'):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        def make(*shape):
            return (torch.randn(*shape, generator=g, device=device) * shape[-1] ** -0.5).bfloat16()
        self.topk, self.experts = topk, experts
        self.router, self.up, self.down = make(experts, hidden), make(experts, 2 * inner, hidden), make(experts, hidden, inner)
        self.head = make(vocab, hidden)

    def parameters(self):
        return self.router, self.up, self.down, self.head


def route(block: Block, x: torch.Tensor):
    """(expert ids [T, K], their weights [T, K] fp32, probabilities [T, E])."""
    probs = torch.softmax((x @ block.router.t()).float(), dim=1)
    top, ids = probs.topk(block.topk, dim=1)
    return ids, top / top.sum(dim=1, keepdim=True), probs


def route_backward(block: Block, x, ids, weights, probs, d_weights):
    """Gradients of x and the router through the chosen experts' normalised probabilities."""
    total = probs.gather(1, ids).sum(dim=1, keepdim=True)
    d_top = (d_weights - (d_weights * weights).sum(dim=1, keepdim=True)) / total
    d_probs = torch.zeros_like(probs).scatter_(1, ids, d_top)
    d_logits = (probs * (d_probs - (d_probs * probs).sum(dim=1, keepdim=True))).bfloat16()
    return d_logits @ block.router, d_logits.t() @ x


def swiglu(h: torch.Tensor) -> torch.Tensor:
    gate, up = h.chunk(2, dim=1)
    return F.silu(gate) * up


def swiglu_backward(h: torch.Tensor, d: torch.Tensor) -> torch.Tensor:
    gate, up = h.float().chunk(2, dim=1)
    s = torch.sigmoid(gate)
    return torch.cat((d.float() * up * s * (1 + gate * (1 - s)), d.float() * gate * s), dim=1).bfloat16()


def train_step(block: Block, x: torch.Tensor, target: torch.Tensor):
    """(mean loss, gradients of router, up, down and head) of the tokens x [T, H]."""
    t, hidden = x.shape
    ids, weights, probs = route(block, x)
    layout = deep_gemm.moe_sort(ids, block.experts)
    rows = deep_gemm.moe_dispatch(x, layout)
    m = rows.size(0)
    empty = lambda width: torch.empty(m, width, dtype=torch.bfloat16, device=x.device)
    h, y = empty(block.up.size(1)), empty(hidden)
    deep_gemm.m_grouped_bf16_gemm_nt_contiguous(rows, block.up, h, layout.psum)
    act = swiglu(h)
    deep_gemm.m_grouped_bf16_gemm_nt_contiguous(act, block.down, y, layout.psum)
    out = x + deep_gemm.moe_combine(y, layout, weights)
    loss, lse = deep_gemm.linear_cross_entropy(out, block.head, target)

    d_out, d_head = deep_gemm.linear_cross_entropy_backward(torch.full_like(loss, 1.0 / t), out, block.head, target, lse)
    d_y, d_weights = deep_gemm.moe_combine_backward(d_out, y, layout, weights)
    d_act, d_rows = empty(act.size(1)), empty(hidden)
    deep_gemm.m_grouped_bf16_gemm_nn_contiguous(d_y, block.down, d_act, layout.psum)
    d_h = swiglu_backward(h, d_act)
    deep_gemm.m_grouped_bf16_gemm_nn_contiguous(d_h, block.up, d_rows, layout.psum)
    d_up, d_down = torch.empty_like(block.up), torch.empty_like(block.down)
    deep_gemm.k_grouped_bf16_gemm_tn_contiguous(d_h, rows, d_up, None, layout.psum)
    deep_gemm.k_grouped_bf16_gemm_tn_contiguous(d_y, act, d_down, None, layout.psum)
    d_x_routed, d_router = route_backward(block, x, ids, weights, probs, d_weights)
    d_x = d_out + deep_gemm.moe_dispatch_backward(d_rows, layout) + d_x_routed
    return loss.mean(), (d_router, d_up, d_down, d_head), d_x


class Quantised:
    """The block's experts and head in e2m1 under scales of 32 values."""

    def __init__(self, block: Block):
        self.block = block
        self.up, self.down, self.head = (deep_gemm.mx_quantize(w) for w in (block.up, block.down, block.head))


def decode_step(q: Quantised, x: torch.Tensor) -> torch.Tensor:
    """Logits [T, V] of a few tokens x [T, H]."""
    block, hidden = q.block, x.size(1)
    ids, weights, _ = route(block, x)
    layout = deep_gemm.moe_sort(ids, block.experts)
    rows = deep_gemm.moe_dispatch(deep_gemm.mx_quantize(x), layout, zero_padding=False)
    m = rows[0].size(0)
    h = torch.empty(m, block.up.size(1), dtype=torch.bfloat16, device=x.device)
    y = torch.empty(m, hidden, dtype=torch.bfloat16, device=x.device)
    deep_gemm.m_grouped_fp8_fp4_gemm_nt_contiguous(rows, q.up, h, layout.psum)
    deep_gemm.m_grouped_fp8_fp4_gemm_nt_contiguous(deep_gemm.mx_quantize(swiglu(h)), q.down, y, layout.psum)
    out = x + deep_gemm.moe_combine(y, layout, weights)
    logits = torch.empty(x.size(0), block.head.size(0), dtype=torch.float32, device=x.device)
    deep_gemm.mx_gemm_nt(out, q.head, logits)
    return logits


def main(steps: int = 10, tokens: int = 2000, lr: float = 8.0):
    block = Block()
    g = torch.Generator(device='cuda')
    g.manual_seed(1)
    x = torch.randn(tokens, block.head.size(1), generator=g, device='cuda').bfloat16()
    target = torch.randint(0, block.head.size(0), (tokens,), generator=g, device='cuda')
    deep_gemm.set_mk_alignment_for_contiguous_layout(128)
    losses = []
    for step in range(steps):
        loss, grads, _ = train_step(block, x, target)
        losses.append(float(loss))
        print(f'step {step}: loss {losses[-1]:.4f}', flush=True)
        for p, d in zip(block.parameters(), grads):
            p.sub_((lr * d.float()).to(p.dtype))
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    logits = decode_step(Quantised(block), x[:8])
    right = float((logits.argmax(1) == target[:8]).float().mean())
    print(f'decoding 8 tokens with 4-bit weights: logits {tuple(logits.shape)}, {right:.0%} of the trained targets on top', flush=True)
    deep_gemm.set_mk_alignment_for_contiguous_layout(256)
    return losses, logits


if __name__ == '__main__':
    main()
