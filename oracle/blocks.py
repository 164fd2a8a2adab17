"""Oracle of what stands between the products: routing, the norm, the gated activation and adapters, from their definitions in 64
bits (test infrastructure only; see ``oracle/__init__.py``).  Gradients come as (values, magnitudes of what was summed for them)."""
import torch

INF = float('inf')


def scores(logits: torch.Tensor, kind: str) -> torch.Tensor:
    l = logits.double()
    if kind == 'sigmoid':
        return 1 / (1 + torch.exp(-l))
    top = l.amax(1, keepdim=True)
    e = torch.exp(l - torch.where(top == -INF, 0.0, top))
    return e / e.sum(1, keepdim=True)


def route(logits, topk, kind='softmax', bias=None, num_groups=1, topk_groups=1, group_top=2, renormalize=True, scale=1.0):
    """(ids [T, K], weights [T, K]), a token and a choice at a time."""
    s = scores(logits, kind)
    b = s if bias is None else s + bias.double()
    t, n = s.shape
    out = (logits == -INF) | (torch.zeros_like(s, dtype=torch.bool) if bias is None else (bias == -INF).expand(t, n))
    if bias is None and (num_groups == 1 or group_top == 1 or topk_groups == num_groups):
        b = logits.double()   # (the same order, also where scores round to one number)
    ids = torch.full((t, topk), -1, dtype=torch.int32)
    weights = torch.zeros(t, topk, dtype=torch.float64)
    order = lambda v: INF if v != v else v   # (NaN is the largest)
    for i in range(t):
        live = [e for e in range(n) if not out[i, e]]
        if num_groups > 1:
            per, found = n // num_groups, []
            for g in range(num_groups):
                best = sorted((order(float(b[i, e])) for e in live if e // per == g), reverse=True)[:group_top]
                found.append((-sum(best) if best else INF, g))
            kept = {g for _, g in sorted(found)[:topk_groups]}
            live = [e for e in live if e // per in kept]
        chosen = sorted(live, key=lambda e: (0 if b[i, e] != b[i, e] else 1, -order(float(b[i, e])), e))[:topk]
        for c, e in enumerate(chosen):
            ids[i, c], weights[i, c] = e, s[i, e]
    if renormalize:
        weights = weights / (weights.sum(1, keepdim=True) + 1e-20)
    return ids, weights * scale


def route_backward(d_weights, logits, ids, kind='softmax', renormalize=True, scale=1.0):
    s = scores(logits, kind)
    t, n = s.shape
    live = (ids >= 0) & (ids < n)
    at = torch.where(live, ids, 0).long()
    w = torch.where(live, s.gather(1, at), 0.0)
    d = torch.where(live, d_weights.double(), 0.0) * scale
    mag = d.abs()
    if renormalize:
        total = w.sum(1, keepdim=True) + 1e-20
        mag = (mag + (mag * w).sum(1, keepdim=True) / total) / total
        d = (d - (d * w).sum(1, keepdim=True) / total) / total
    d, mag = torch.where(live, d, 0.0), torch.where(live, mag, 0.0)
    g = torch.zeros_like(s).scatter_add_(1, at, d)
    m = torch.zeros_like(s).scatter_add_(1, at, mag)
    if kind == 'softmax':
        return s * (g - (d * w).sum(1, keepdim=True)), s * (m + (mag * w).sum(1, keepdim=True))
    slope = s * (1 / (1 + torch.exp(logits.double())))
    return g * slope, m * slope


def rms_norm(x, weight, residual=None, eps=1e-6):
    """(y, h, rstd)"""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = h.double()
    rstd = 1 / torch.sqrt((v * v).mean(1) + eps)
    return v * rstd.unsqueeze(1) * weight.double(), h, rstd


def rms_norm_backward(d_y, h, weight, rstd, d_h=None):
    """(d_x, magnitudes, d_weight, magnitudes)"""
    d, v, w, r = d_y.double(), h.double(), weight.double(), rstd.double().unsqueeze(1)
    inner = w * d * v
    d_x = r * (w * d - v * r * r * inner.mean(1, keepdim=True))
    m_x = r * ((w * d).abs() + v.abs() * r * r * inner.abs().mean(1, keepdim=True))
    if d_h is not None:
        d_x, m_x = d_x + d_h.double(), m_x + d_h.double().abs()
    return d_x, m_x, (d * v * r).sum(0), (d * v * r).abs().sum(0)


def swiglu(h):
    gate, up = h.double().chunk(2, dim=1)
    return gate / (1 + torch.exp(-gate)) * up


def swiglu_backward(d_act, h):
    """(d_h, magnitudes)"""
    gate, up = h.double().chunk(2, dim=1)
    d, s = d_act.double(), 1 / (1 + torch.exp(-gate))
    back = 1 / (1 + torch.exp(gate))   # 1 - s
    d_g, m_g = d * up * s * (1 + gate * back), (d * up).abs() * s * (1 + gate.abs() * back)
    return torch.cat((d_g, d * gate * s), 1), torch.cat((m_g, (d * gate).abs() * s), 1)


def lora(x, a, b, ids, scales=None, c=None):
    """(d, magnitudes of its sums)"""
    t, n = x.shape[0], b.shape[1]
    d = torch.zeros(t, n, dtype=torch.float64) if c is None else c.double()
    mag = d.abs()
    for i in range(t):
        e = int(ids[i])
        if 0 <= e < a.shape[0]:
            f = 1.0 if scales is None else float(scales[e])
            d[i] += f * (a[e].double() @ x[i].double()) @ b[e].double().t()
            mag[i] += abs(f) * (a[e].double().abs() @ x[i].double().abs()) @ b[e].double().abs().t()
    return d, mag
