"""Cases that measure what stands between and beside the matrix products of a mixture-of-experts language model: routing to
experts, the norm with the residual's addition and 8-bit output, the gated activation with an 8-bit checkpoint, and the low-rank
adapters of many requests.

``run`` computes a case in plain torch operations (``own`` false) or with this repository's operators (``own`` true);
``exact`` computes the same outputs in 64 bits.
"""
import os
import sys

import torch

own = False

EPS = 1e-6      # of the norm
TINY = 1e-20    # of the routers' sums


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the router of a decode step of 16 requests, groups of experts and a bias for balance: latency
        {'name': 'route_decode', 'op': 'route', 'tokens': 16, 'experts': 256, 'topk': 8, 'groups': 8, 'topk_groups': 4,
         'scores': 'sigmoid', 'bias': True, 'dtype': 'f32', 'grad': False},
        # the same router over a long prefill
        {'name': 'route_prefill', 'op': 'route', 'tokens': 32768, 'experts': 256, 'topk': 8, 'groups': 8, 'topk_groups': 4,
         'scores': 'sigmoid', 'bias': True, 'dtype': 'f32', 'grad': False},
        # a training step's router: softmax, an odd number of tokens, with gradient
        {'name': 'route_train', 'op': 'route', 'tokens': 8191, 'experts': 160, 'topk': 6, 'groups': 1, 'topk_groups': 1,
         'scores': 'softmax', 'bias': False, 'dtype': 'bf16', 'grad': True},
        # the norm before a decode step's 8-bit products
        {'name': 'norm_decode', 'op': 'norm', 'tokens': 16, 'width': 7168, 'dtype': 'bf16', 'residual': True, 'format': 'e4m3', 'grad': False},
        # a training step's norm, there and back
        {'name': 'norm_train', 'op': 'norm', 'tokens': 8192, 'width': 4096, 'dtype': 'bf16', 'residual': True, 'format': 'none', 'grad': True},
        # fp32 at odd sizes, no residual
        {'name': 'norm_odd', 'op': 'norm', 'tokens': 1021, 'width': 1407, 'dtype': 'f32', 'residual': False, 'format': 'none', 'grad': True},
        # the rows between two products of experts in a decode step, most of them padding, to 8 bits
        {'name': 'gate_decode', 'op': 'gate', 'rows': 1248, 'width': 2048, 'dtype': 'bf16', 'format': 'e4m3', 'checkpoint': False,
         'padding': 0.8, 'grad': False},
        # a training step's activation: kept in 8 bits, used in the backward pass
        {'name': 'gate_train', 'op': 'gate', 'rows': 32768, 'width': 2048, 'dtype': 'bf16', 'format': 'none', 'checkpoint': True,
         'padding': 0.0, 'grad': True},
        # a chunk of odd rows and width, nothing quantised
        {'name': 'gate_odd', 'op': 'gate', 'rows': 777, 'width': 1411, 'dtype': 'bf16', 'format': 'none', 'checkpoint': False,
         'padding': 0.0, 'grad': True},
        # one request's token through its adapter
        {'name': 'lora_single', 'op': 'lora', 'tokens': 1, 'adapters': 8, 'rank': 16, 'width': 4096, 'cols': 7168, 'out': 'bf16', 'without': 0.0},
        # a decode step of 48 requests over 20 adapters
        {'name': 'lora_decode', 'op': 'lora', 'tokens': 48, 'adapters': 20, 'rank': 16, 'width': 7168, 'cols': 4096, 'out': 'bf16', 'without': 0.1},
        # a prefill of several requests
        {'name': 'lora_prefill', 'op': 'lora', 'tokens': 4099, 'adapters': 8, 'rank': 32, 'width': 2048, 'cols': 7168, 'out': 'bf16', 'without': 0.1},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even in its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(('route', 'norm', 'gate', 'lora'))
    case = {'op': op}
    if op == 'route':
        groups = rng.choice((1, 1, 4, 8))
        experts = groups * _log(rng, 2, 64) if groups > 1 else _log(rng, 8, 512)
        keep = 1 if groups == 1 else rng.randint(max(1, groups // 4), groups)
        case.update(tokens=_log(rng, 1, 32768), experts=experts, topk=rng.randint(1, min(8, keep * (experts // groups))), groups=groups,
                    topk_groups=keep, scores=rng.choice(('softmax', 'sigmoid')), bias=rng.random() < 0.5,
                    dtype=rng.choice(('f32', 'f32', 'bf16')), grad=rng.random() < 0.4)
        case['tokens'] = min(case['tokens'], (1 << 23) // experts)
    elif op == 'norm':
        case.update(tokens=_log(rng, 1, 8192), dtype=rng.choice(('bf16', 'bf16', 'f32')), residual=rng.random() < 0.7,
                    format=rng.choice(('none', 'e4m3')), grad=rng.random() < 0.5)
        case['width'] = 32 * _log(rng, 2, 256) if case['format'] != 'none' else _log(rng, 64, 8192)
        case['tokens'] = min(case['tokens'], (1 << 24) // case['width'])
    elif op == 'gate':
        case.update(rows=_log(rng, 1, 32768), dtype=rng.choice(('bf16', 'bf16', 'f32')), format=rng.choice(('none', 'e4m3')),
                    checkpoint=rng.random() < 0.5, padding=rng.choice((0.0, 0.0, 0.5)), grad=rng.random() < 0.5)
        small = case['checkpoint'] or case['format'] != 'none'
        case['width'] = 32 * _log(rng, 1, 128) if small else _log(rng, 16, 4096)
        case['rows'] = min(case['rows'], (1 << 25) // case['width'])
    else:
        case.update(tokens=_log(rng, 1, 4096), adapters=_log(rng, 1, 64), rank=8 * _log(rng, 1, 16), width=8 * _log(rng, 32, 896),
                    cols=_log(rng, 64, 7168), out=rng.choice(('bf16', 'bf16', 'f32')), without=rng.choice((0.0, 0.1, 0.5)))
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _dtype(name):
    return torch.bfloat16 if name == 'bf16' else torch.float32


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device='cuda', dtype=torch.float32).mul_(scale).to(dtype)


def _layout(ids, groups, alignment):
    """(slots, source, psum, m_indices) of one choice a token: the rows of an M-grouped layout, -1 for padding and for tokens
    without a group."""
    t = ids.numel()
    rows = (t + min(groups, t) * (alignment - 1)) // alignment * alignment
    key = torch.where(ids < 0, groups, ids.long())
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=groups + 1)[:groups]
    aligned = (counts + alignment - 1) // alignment * alignment
    start, before = torch.cumsum(aligned, 0) - aligned, torch.cumsum(counts, 0) - counts
    sorted_key = key[order]
    live = sorted_key < groups
    at = sorted_key.clamp(max=groups - 1)
    row = torch.where(live, start[at] + torch.arange(t, device=ids.device) - before[at], rows)
    slots = torch.empty(t, dtype=torch.int32, device=ids.device)
    slots[order] = torch.where(live, row, -1).to(torch.int32)
    source, indices = (torch.full((rows + 1,), -1, dtype=torch.int32, device=ids.device) for _ in range(2))
    source[row], indices[row] = order.to(torch.int32), sorted_key.to(torch.int32)
    return slots.view(t, 1), source[:rows].clone(), (start + counts).to(torch.int32), indices[:rows].clone()


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    op, s = case['op'], {'case': case}
    if op == 'route':
        t, n = case['tokens'], case['experts']
        # some experts are more popular than others; the bias works against that
        popular = _randn(g, n, scale=0.5)
        s['logits'] = (_randn(g, t, n) + popular).to(_dtype(case['dtype']))
        s['bias'] = (-0.1 * popular + _randn(g, n, scale=0.02)) if case['bias'] else None
        s['d_weights'] = _randn(g, t, case['topk'])
    elif op == 'norm':
        t, h, dt = case['tokens'], case['width'], _dtype(case['dtype'])
        # tokens of different size, as a residual stream has
        s['x'] = _randn(g, t, h, dtype=dt)
        s['residual'] = (_randn(g, t, h) * torch.exp(_randn(g, t, 1))).to(dt) if case['residual'] else None
        s['weight'] = (1 + _randn(g, h, scale=0.1)).to(dt)
        s['d_y'] = _randn(g, t, h, dtype=dt)
        s['d_h'] = _randn(g, t, h, dtype=dt) if case['residual'] else None
    elif op == 'gate':
        m, f, dt = case['rows'], case['width'], _dtype(case['dtype'])
        s['h'], s['d_act'] = _randn(g, m, 2 * f, dtype=dt), _randn(g, m, f, dtype=dt)
        s['m_indices'] = None
        if case['padding']:   # runs of 32 rows of one group, each with padding behind
            row = torch.arange(m, device='cuda')
            s['m_indices'] = torch.where(row % 32 < round(32 * (1 - case['padding'])), row // 32, -1).to(torch.int32)
            live = (s['m_indices'] >= 0).unsqueeze(1)
            s['h'], s['d_act'] = s['h'] * live, s['d_act'] * live   # (as the products leave padding rows)
    else:
        t, n, r, k, cols = case['tokens'], case['adapters'], case['rank'], case['width'], case['cols']
        s['x'] = _randn(g, t, k, dtype=torch.bfloat16)
        s['a'] = _randn(g, n, r, k, dtype=torch.bfloat16, scale=k ** -0.5)
        s['b'] = _randn(g, n, cols, r, dtype=torch.bfloat16, scale=r ** -0.5)
        s['scales'] = 0.5 + torch.rand(n, generator=g, device='cuda')
        s['c'] = _randn(g, t, cols, dtype=_dtype(case['out']))   # what the shared projection gave
        ids = torch.randint(0, n, (t,), generator=g, device='cuda')
        s['ids'] = torch.where(torch.rand(t, generator=g, device='cuda') < case['without'], -1, ids).to(torch.int32)
        # sorted once a step, for every projection of every layer
        s['layout'] = _layout(s['ids'], n, 32 if t <= 256 else 128)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _e4m3(x):
    """fp32 values of x in e4m3 under the smallest power of two per 32 values that keeps them within the format."""
    b = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bits = b.abs().amax(dim=-1).view(torch.int32)
    e = ((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000).to(torch.int32)).clamp(1, 254)
    scale = (e << 23).view(torch.float32).unsqueeze(-1)
    return ((b / scale).to(torch.float8_e4m3fn).float() * scale).reshape(x.shape)


def _output(y, case):
    """fp32 results in the type of the case; what is held in 8 bits as the values it stands for."""
    return _e4m3(y).to(torch.bfloat16) if case['format'] == 'e4m3' else y.to(_dtype(case['dtype']))


def _plain_route(s):
    case = s['case']
    # (64 bits: scores next to each other decide)
    l = s['logits'].double()
    t, n = l.shape
    if case['scores'] == 'softmax':
        e = (l - l.amax(dim=1, keepdim=True)).exp()
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1 / (1 + (-l).exp())
    key = score if s['bias'] is None else score + s['bias'].double()
    if case['groups'] > 1:
        best = key.view(t, case['groups'], -1).sort(dim=2, descending=True).values[:, :, :2].sum(dim=2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :case['topk_groups']]
        keep = torch.zeros_like(best).scatter(1, kept, 1.0) > 0
        key = torch.where(keep.repeat_interleave(n // case['groups'], dim=1), key, -torch.inf)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :case['topk']]
    w = score.gather(1, ids)
    total = w.sum(dim=1, keepdim=True) + TINY
    out = {'ids': ids.to(torch.int32), 'weights': (2.5 * w / total).float()}
    if case['grad']:
        d = 2.5 * s['d_weights'].double()
        d = torch.zeros_like(score).scatter(1, ids, (d - (d * w).sum(dim=1, keepdim=True) / total) / total)
        if case['scores'] == 'softmax':
            d = score * (d - (d * score).sum(dim=1, keepdim=True))
        else:
            d = d * score * (1 - score)
        out['d_logits'] = d.to(s['logits'].dtype)
    return out


def _plain_norm(s):
    case, dt = s['case'], _dtype(s['case']['dtype'])
    h = s['x'] if s['residual'] is None else (s['x'].float() + s['residual'].float()).to(dt)
    v, w = h.float(), s['weight'].float()
    rstd = ((v * v).mean(dim=1) + EPS) ** -0.5
    r = rstd.unsqueeze(1)
    out = {'y': _output(v * r * w, case), 'h': h, 'rstd': rstd}
    if case['grad']:
        d = s['d_y'].float()
        wd = w * d
        d_x = r * (wd - v * (r * r * (wd * v).mean(dim=1, keepdim=True)))
        out['d_x'] = (d_x if s['d_h'] is None else d_x + s['d_h'].float()).to(dt)
        out['d_weight'] = (d * v * r).sum(dim=0)
    return out


def _plain_gate(s):
    case, dt = s['case'], _dtype(s['case']['dtype'])
    h = s['h'].float()
    gate, up = h.chunk(2, dim=1)
    out = {'act': _output(gate / (1 + (-gate).exp()) * up, case)}
    if case['checkpoint']:
        h = _e4m3(h)
        out['saved'] = h.to(torch.bfloat16)
        gate, up = h.chunk(2, dim=1)
    if case['grad']:
        d, sig = s['d_act'].float(), 1 / (1 + (-gate).exp())
        out['d_h'] = torch.cat((d * up * sig * (1 + gate * (1 - sig)), d * gate * sig), dim=1).to(dt)
        out['again'] = (gate * sig * up).to(dt)
    return out


def _plain_lora(s):
    t, (n, r, k), cols = s['x'].shape[0], s['a'].shape, s['b'].shape[1]
    at, live = s['ids'].clamp(min=0).long(), (s['ids'] >= 0).view(t, 1)
    # every adapter's inner products, those of a token's own kept
    inner = (s['x'].float() @ s['a'].float().view(n * r, k).t()).view(t, n, r)
    own_one = (torch.arange(n, device='cuda') == at.unsqueeze(1)).unsqueeze(2)
    inner = torch.where(own_one, inner, 0.0).view(t, n * r)
    delta = s['scales'][at].unsqueeze(1) * (inner @ s['b'].float().transpose(1, 2).reshape(n * r, cols))
    return (s['c'].float() + torch.where(live, delta, 0.0)).to(s['c'].dtype)


# ------------------------------------------------------------------------------------------------ this repository's operators
def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'deepgemm-ascend_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    import deep_gemm
    return deep_gemm


def _own(s):
    dg = _package()
    case = s['case']
    op = case['op']
    if op == 'route':
        ids, weights = dg.moe_route(s['logits'], case['topk'], case['scores'], bias=s['bias'], num_groups=case['groups'],
                                    topk_groups=case['topk_groups'], scale=2.5)
        if not case['grad']:
            return {'ids': ids, 'weights': weights}
        d_logits = dg.moe_route_backward(s['d_weights'], s['logits'], ids, case['scores'], scale=2.5)
        return {'ids': ids, 'weights': weights, 'd_logits': d_logits}
    if op in ('norm', 'gate'):
        fmt = None if case['format'] == 'none' else case['format']
    if op == 'norm':
        y, h, rstd = dg.rms_norm(s['x'], s['weight'], s['residual'], EPS, fmt)
        out = {'y': y if fmt is None else dg.mx_dequantize(y), 'h': h, 'rstd': rstd}
        if case['grad']:
            out['d_x'], out['d_weight'] = dg.rms_norm_backward(s['d_y'], h, s['weight'], rstd, s['d_h'])
        return out
    if op == 'gate':
        saved = s['h']
        act = dg.swiglu(s['h'], fmt, case['checkpoint'], s['m_indices'])
        if case['checkpoint']:
            act, saved = act
        out = {'act': act if fmt is None else dg.mx_dequantize(act)}
        if case['checkpoint']:
            out['saved'] = dg.mx_dequantize(saved)
        if case['grad']:
            out['d_h'], out['again'] = dg.swiglu_backward(s['d_act'], saved, True, s['m_indices'])
        return out
    d = torch.empty_like(s['c'])
    dg.lora_gemm_nt(s['x'], s['a'], s['b'], d, dg.MoELayout(*s['layout']), s['scales'], s['c'])
    return d


def run(state):
    if own:
        return _own(state)
    return {'route': _plain_route, 'norm': _plain_norm, 'gate': _plain_gate, 'lora': _plain_lora}[state['case']['op']](state)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    op = case['op']
    if op == 'route':
        t, n, k, e = case['tokens'], case['experts'], case['topk'], 2 if case['dtype'] == 'bf16' else 4
        # the logits; ids and weights; and for the gradient the logits, ids and weights' gradient again, the logits' gradient
        moved = t * (n * e + 8 * k) + (t * (2 * n * e + 8 * k) if case['grad'] else 0)
        return {'bytes': moved, 'flops': (20.0 if case['grad'] else 10.0) * t * n}
    if op == 'norm':
        t, h, e = case['tokens'], case['width'], 2 if case['dtype'] == 'bf16' else 4
        quant = case['format'] != 'none'
        # x (and the residual, the sum); y, and where it is quantised its values back
        moved = t * h * e * (3 if case['residual'] else 1) + t * h * (2 * (1 + 1 / 32) + 2 if quant else e)
        if case['grad']:   # d_y, h, d_x (and the residual's gradient)
            moved += t * h * e * (4 if case['residual'] else 3)
        return {'bytes': moved, 'flops': (12.0 if case['grad'] else 4.0) * t * h}
    if op == 'gate':
        live = case['rows'] * (1 - case['padding'])
        f, e = case['width'], 2 if case['dtype'] == 'bf16' else 4
        code = 1 + 1 / 32
        # the two halves of a row in; the activation out (and where it is quantised its values), every row's
        moved = live * 2 * f * e + case['rows'] * f * (2 * code + 2 if case['format'] != 'none' else e)
        if case['checkpoint']:   # codes written, and read for their values
            moved += case['rows'] * 2 * f * (2 * code + 2)
        if case['grad']:
            moved += live * f * (e + 2 * (code if case['checkpoint'] else e)) + case['rows'] * 3 * f * e
        return {'bytes': moved, 'flops': (20.0 if case['grad'] else 6.0) * live * f}
    t, r, k, n = case['tokens'], case['rank'], case['width'], case['cols']
    live = t * (1 - case['without'])
    used = min(case['adapters'], live)
    e = 2 if case['out'] == 'bf16' else 4
    return {'bytes': 2 * live * k + 2 * used * r * (k + n) + 2 * t * n * e, 'flops': 2.0 * live * r * (k + n)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_e4m3(x):
    """The quantised values from the definition: the smallest power of two that keeps a block inside the format, then the
    nearest multiple of the local step, ties to even."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2((amax / 448.0).clamp(min=2.0 ** -126))).clamp(min=-126))
    scale = torch.where(amax / scale > 448.0, scale * 2, scale)
    scale = torch.where((amax / (scale / 2) <= 448.0) & (scale > 2.0 ** -126), scale / 2, scale)
    v = b / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6.0) - 3)
    return (torch.round(v / step) * step * scale).reshape(x.shape)


def exact(case, seed):
    s, op = prepare(case, seed), case['op']
    if op == 'route':
        l = s['logits'].double().requires_grad_()
        p = torch.softmax(l, dim=1) if case['scores'] == 'softmax' else torch.sigmoid(l)
        with torch.no_grad():
            key = p if s['bias'] is None else p + s['bias'].double()
            t, n = key.shape
            if case['groups'] > 1:
                per = n // case['groups']
                score = torch.stack([part.topk(min(2, per), dim=1).values.sum(1) for part in key.split(per, dim=1)], dim=1)
                for _ in range(case['groups'] - case['topk_groups']):   # (the worst group leaves, the last of equal ones)
                    last = case['groups'] - 1 - score.flip(1).argmin(dim=1)
                    score[torch.arange(t), last] = torch.inf
                    gone = torch.arange(n, device='cuda') // per == last.unsqueeze(1)
                    key = key.masked_fill(gone, -torch.inf)
            key, chosen = key.clone(), []
            for _ in range(case['topk']):   # (argmax: the first of equal ones)
                chosen.append(key.argmax(dim=1))
                key[torch.arange(t), chosen[-1]] = -torch.inf
            ids = torch.stack(chosen, dim=1)
        w = p.gather(1, ids)
        w = 2.5 * w / (w.sum(dim=1, keepdim=True) + TINY)
        found = {'ids': None, 'weights': w.detach()}
        if case['grad']:
            w.backward(s['d_weights'].double())
            found['d_logits'] = l.grad
        return found
    if op == 'norm':
        h = s['x'] if s['residual'] is None else (s['x'].double() + s['residual'].double()).to(s['x'].dtype)
        v, w = h.double().requires_grad_(), s['weight'].double().requires_grad_()
        rstd = 1 / torch.sqrt(v.square().mean(dim=1) + EPS)
        y = v * rstd.unsqueeze(1) * w
        found = {'y': _exact_e4m3(y.detach()) if case['format'] == 'e4m3' else y.detach(), 'h': h.double(), 'rstd': rstd.detach()}
        if case['grad']:
            y.backward(s['d_y'].double())
            found['d_x'] = v.grad if s['d_h'] is None else v.grad + s['d_h'].double()
            found['d_weight'] = w.grad
        return found
    if op == 'gate':
        h = s['h'].double()
        act = torch.nn.functional.silu(h[:, :case['width']]) * h[:, case['width']:]
        found = {'act': _exact_e4m3(act) if case['format'] == 'e4m3' else act}
        if case['checkpoint']:
            h = _exact_e4m3(h)
            found['saved'] = h
        if case['grad']:
            h = h.clone().requires_grad_()
            again = torch.nn.functional.silu(h[:, :case['width']]) * h[:, case['width']:]
            again.backward(s['d_act'].double())
            found['d_h'], found['again'] = h.grad, again.detach()
        return found
    d = s['c'].double()
    for i in range(case['adapters']):
        mine = (s['ids'] == i).nonzero().squeeze(1)
        d[mine] += s['scales'][i].double() * (s['x'][mine].double() @ s['a'][i].double().t() @ s['b'][i].double().t())
    return d
