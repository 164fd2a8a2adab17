"""One mixture-of-experts layer with its norm: a training step that keeps the experts' activations in 8 bits, and decoding in 8 bits
with an adapter of its own for each request.

    python examples/moe_layer.py

Training: residual addition and norm, routing by groups with a bias for balance, the experts' two products with the gated activation
between them, weighted sums back; then the gradient of all of it, from the 8-bit checkpoint.  Decoding: the norm leaves its rows in
e4m3 (and again in bf16 for the router), the activation leaves its rows in e4m3, the adapters add to the layer's output.
"""
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'deepgemm-ascend_amd'))

import torch  # noqa: E402

import deep_gemm  # noqa: E402

SCALE = 2.5


class Layer:
    """Norm weight [H], router [E, H], experts' gate and up [E, 2 F, H] and down [E, H, F], and the router's bias [E]."""

    def __init__(self, hidden=512, inner=256, experts=32, topk=4, groups=4, topk_groups=2, seed=0, device='cuda'):
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def make(*shape):
            return (torch.randn(*shape, generator=g, device=device) * shape[-1] ** -0.5).bfloat16()
        self.topk, self.experts, self.groups, self.topk_groups = topk, experts, groups, topk_groups
        self.weight = torch.ones(hidden, dtype=torch.bfloat16, device=device)
        self.router, self.up, self.down = make(experts, hidden), make(experts, 2 * inner, hidden), make(experts, hidden, inner)
        self.bias = torch.zeros(experts, device=device)

    def parameters(self):
        return self.weight, self.router, self.up, self.down


def choose(layer: Layer, y: torch.Tensor):
    """(logits, ids, weights) of the normed tokens."""
    logits = torch.empty(y.size(0), layer.experts, dtype=torch.float32, device=y.device)
    deep_gemm.bf16_gemm_nt(y, layer.router, logits)
    return logits, *deep_gemm.moe_route(logits, layer.topk, 'sigmoid', layer.bias, layer.groups, layer.topk_groups, scale=SCALE)


def balance(layer: Layer, ids: torch.Tensor, step: float = 0.001):
    """The bias moves against the experts that had more than their share."""
    load = torch.zeros(layer.experts + 1, device=ids.device).index_add_(0, (ids.reshape(-1).long() + 1), torch.ones(ids.numel(), device=ids.device))[1:]
    layer.bias -= step * torch.sign(load - load.mean())


def forward(layer: Layer, x: torch.Tensor, residual: torch.Tensor):
    """(the residual stream after the layer, what the gradient needs): of the experts' rows it keeps codes and scales."""
    y, h, rstd = deep_gemm.rms_norm(x, layer.weight, residual)
    logits, ids, weights = choose(layer, y)
    layout = deep_gemm.moe_sort(ids, layer.experts)
    rows = deep_gemm.moe_dispatch(y, layout)
    m = rows.size(0)
    inner = torch.empty(m, layer.up.size(1), dtype=torch.bfloat16, device=x.device)
    outer = torch.empty(m, x.size(1), dtype=torch.bfloat16, device=x.device)
    deep_gemm.m_grouped_bf16_gemm_nt_contiguous(rows, layer.up, inner, layout.psum)
    act, saved = deep_gemm.swiglu(inner, checkpoint=True, m_indices=layout.m_indices)
    deep_gemm.m_grouped_bf16_gemm_nt_contiguous(act, layer.down, outer, layout.psum)
    out = h + deep_gemm.moe_combine(outer, layout, weights)
    return out, {'y': y, 'h': h, 'rstd': rstd, 'logits': logits, 'ids': ids, 'weights': weights, 'layout': layout, 'saved': saved, 'outer': outer}


def backward(layer: Layer, kept, d_out: torch.Tensor):
    """(gradient of x and of the residual, gradients of the parameters)"""
    layout, y = kept['layout'], kept['y']
    d_outer, d_weights = deep_gemm.moe_combine_backward(d_out, kept['outer'], layout, kept['weights'])
    d_act = torch.empty(d_outer.size(0), layer.down.size(2), dtype=torch.bfloat16, device=y.device)
    deep_gemm.m_grouped_bf16_gemm_nn_contiguous(d_outer, layer.down, d_act, layout.psum)
    d_inner, act = deep_gemm.swiglu_backward(d_act, kept['saved'], with_act=True, m_indices=layout.m_indices)
    d_rows = torch.empty(d_outer.size(0), y.size(1), dtype=torch.bfloat16, device=y.device)
    deep_gemm.m_grouped_bf16_gemm_nn_contiguous(d_inner, layer.up, d_rows, layout.psum)
    d_up, d_down = torch.empty_like(layer.up), torch.empty_like(layer.down)
    deep_gemm.k_grouped_bf16_gemm_tn_contiguous(d_inner, deep_gemm.moe_dispatch(y, layout), d_up, None, layout.psum)
    deep_gemm.k_grouped_bf16_gemm_tn_contiguous(d_outer, act, d_down, None, layout.psum)
    d_logits = deep_gemm.moe_route_backward(d_weights, kept['logits'], kept['ids'], 'sigmoid', scale=SCALE).bfloat16()
    d_y = deep_gemm.moe_dispatch_backward(d_rows, layout) + d_logits @ layer.router
    d_x, d_norm = deep_gemm.rms_norm_backward(d_y, kept['h'], layer.weight, kept['rstd'], d_out)
    return d_x, (d_norm, d_logits.t() @ y, d_up, d_down)


class Served:
    """The layer with experts in e4m3 and adapters of its output (a [L, R, H], b [L, H, R])."""

    def __init__(self, layer: Layer, adapters: int = 4, rank: int = 16, seed: int = 1):
        hidden, device = layer.weight.numel(), layer.weight.device
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.layer = layer
        self.up, self.down = (deep_gemm.mx_quantize(w, 'e4m3') for w in (layer.up, layer.down))
        self.a = (torch.randn(adapters, rank, hidden, generator=g, device=device) * hidden ** -0.5).bfloat16()
        self.b = (0.1 * torch.randn(adapters, hidden, rank, generator=g, device=device)).bfloat16()


def decode(served: Served, x: torch.Tensor, residual: torch.Tensor, adapters) -> torch.Tensor:
    """The residual stream after the layer for a few tokens; `adapters`: the tokens sorted by adapter."""
    layer = served.layer
    y, h, _ = deep_gemm.rms_norm(x, layer.weight, residual)
    _, ids, weights = choose(layer, y)
    layout = deep_gemm.moe_sort(ids, layer.experts)
    rows = deep_gemm.moe_dispatch(deep_gemm.rms_norm(h, layer.weight, fmt='e4m3')[0], layout, zero_padding=False)
    m = rows[0].size(0)
    inner = torch.empty(m, layer.up.size(1), dtype=torch.bfloat16, device=x.device)
    outer = torch.empty(m, x.size(1), dtype=torch.bfloat16, device=x.device)
    recipe = dict(recipe_a=(1, 32), recipe_b=(1, 32))
    deep_gemm.m_grouped_fp8_gemm_nt_contiguous(rows, served.up, inner, layout.psum, **recipe)
    act = deep_gemm.swiglu(inner, 'e4m3', m_indices=layout.m_indices, zero_padding=False)
    deep_gemm.m_grouped_fp8_gemm_nt_contiguous(act, served.down, outer, layout.psum, **recipe)
    out = h + deep_gemm.moe_combine(outer, layout, weights)
    deep_gemm.lora_gemm_nt(h, served.a, served.b, out, adapters, c=out)
    return out


def main(tokens: int = 2000):
    layer = Layer()
    g = torch.Generator(device='cuda')
    g.manual_seed(2)
    x, residual, d_out = (torch.randn(tokens, layer.weight.numel(), generator=g, device='cuda').bfloat16() for _ in range(3))
    deep_gemm.set_mk_alignment_for_contiguous_layout(128)
    out, kept = forward(layer, x, residual)
    d_x, grads = backward(layer, kept, d_out)
    balance(layer, kept['ids'])
    print(f'training: out {tuple(out.shape)}, gradients {[tuple(d.shape) for d in (d_x, *grads)]}', flush=True)
    deep_gemm.set_mk_alignment_for_contiguous_layout(32)
    served = Served(layer)
    adapters = deep_gemm.moe_sort(torch.arange(8, device='cuda').view(-1, 1) % 5 - 1, 4)   # (some requests have none)
    out = decode(served, x[:8], residual[:8], adapters)
    print(f'decoding 8 tokens in 8 bits with adapters: {tuple(out.shape)}', flush=True)
    deep_gemm.check_errors()
    deep_gemm.set_mk_alignment_for_contiguous_layout(256)
    return out


if __name__ == '__main__':
    main()
