"""Cases that measure the operators around the matrix products: tokens sorted by expert and moved there and back with
their gradients, microscaled quantisation with its product, and the cross entropy of a linear layer over a large
vocabulary with its gradient.

``run`` computes a case in plain torch operations in 32 bits (``own`` false) or with this repository's operators
(``own`` true); ``exact`` computes the same outputs in 64 bits.
"""
import os
import sys

import torch

own = False

IGNORE = -100


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the router's result of a decode step of 16 requests: latency
        {'name': 'sort_decode', 'op': 'sort', 'tokens': 16, 'topk': 8, 'groups': 256, 'alignment': 32, 'dropped': 0.0},
        # a long prefill on a rank that holds half of the experts (the other pairs are dropped)
        {'name': 'sort_prefill', 'op': 'sort', 'tokens': 32768, 'topk': 8, 'groups': 256, 'alignment': 128, 'dropped': 0.5},
        # one training step's movement: there, back with weights, and both gradients
        {'name': 'permute_train', 'op': 'permute', 'tokens': 8192, 'topk': 8, 'groups': 64, 'alignment': 128, 'width': 4096,
         'dtype': 'bf16', 'dropped': 0.0},
        # the same in fp32 at odd sizes, with dropped pairs
        {'name': 'permute_odd', 'op': 'permute', 'tokens': 1021, 'topk': 6, 'groups': 40, 'alignment': 64, 'width': 1407,
         'dtype': 'f32', 'dropped': 0.1},
        # a layer's weights to 4 bits and back (training with quantised weights, or loading)
        {'name': 'quant_weights', 'op': 'quant', 'rows': 7168, 'width': 16384, 'format': 'e2m1', 'dtype': 'bf16'},
        # a chunk of activations to 8 bits, odd rows, a width that ends inside a pair of blocks
        {'name': 'quant_chunk', 'op': 'quant', 'rows': 777, 'width': 1440, 'format': 'e4m3', 'dtype': 'f32'},
        # one token through a 4-bit layer
        {'name': 'product_decode', 'op': 'product', 'rows': 1, 'cols': 7168, 'width': 4096, 'format': 'e2m1'},
        # a prefill through the same kind of layer
        {'name': 'product_prefill', 'op': 'product', 'rows': 4096, 'cols': 7168, 'width': 2048, 'format': 'e2m1'},
        # a decode step through a layer of 4-bit experts: sort, quantise, move, product, back with weights
        {'name': 'experts_decode', 'op': 'experts', 'tokens': 32, 'topk': 8, 'groups': 32, 'alignment': 32, 'cols': 2048,
         'width': 4096, 'dropped': 0.0},
        # the log probability of a prompt's tokens (no gradient)
        {'name': 'loss_score', 'op': 'loss', 'tokens': 131, 'width': 2048, 'vocab': 32000, 'grad': False},
        # a short step: odd numbers of tokens and of words
        {'name': 'loss_odd', 'op': 'loss', 'tokens': 777, 'width': 1536, 'vocab': 32003, 'grad': True},
        # a training step's last layer
        {'name': 'loss_train', 'op': 'loss', 'tokens': 8192, 'width': 4096, 'vocab': 131072, 'grad': True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even in its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(('sort', 'permute', 'quant', 'product', 'experts', 'loss'))
    case = {'op': op}
    if op in ('sort', 'permute', 'experts'):
        case['topk'] = rng.randint(1, 8)
        case['groups'] = _log(rng, 8, 256)
        case['alignment'] = rng.choice((32, 64, 128, 256))
        case['dropped'] = rng.choice((0.0, 0.0, 0.1, 0.5))
    if op == 'sort':
        case['tokens'] = _log(rng, 1, 32768)
    elif op == 'permute':
        case.update(tokens=_log(rng, 1, 8192), width=_log(rng, 64, 7168), dtype=rng.choice(('bf16', 'bf16', 'f32')))
        if case['tokens'] * case['topk'] * case['width'] > 1 << 28:   # (about the largest listed)
            case['tokens'] = max(1, (1 << 28) // (case['topk'] * case['width']))
    elif op == 'quant':
        case.update(rows=_log(rng, 1, 7168), width=32 * _log(rng, 2, 512), format=rng.choice(('e2m1', 'e2m1', 'e4m3')),
                    dtype=rng.choice(('bf16', 'bf16', 'f32')))
    elif op == 'product':
        case.update(rows=_log(rng, 1, 4096), cols=_log(rng, 64, 7168), width=32 * _log(rng, 2, 224),
                    format=rng.choice(('e2m1', 'e2m1', 'e4m3')))
    elif op == 'experts':
        case.update(tokens=_log(rng, 1, 1024), groups=_log(rng, 4, 64), cols=8 * _log(rng, 8, 256), width=32 * _log(rng, 4, 128))
    else:
        case.update(tokens=_log(rng, 1, 8192), width=8 * _log(rng, 16, 512), vocab=_log(rng, 1000, 131072),
                    grad=rng.random() < 0.7)
    return case


def num_rows(case):
    """Rows that hold every pair whatever the routing: each group that has any starts at a multiple of the alignment."""
    pairs, a = case['tokens'] * case['topk'], case['alignment']
    return (pairs + min(case['groups'], pairs) * (a - 1)) // a * a


# ------------------------------------------------------------------------------------------------ inputs
def _dtype(name):
    return torch.bfloat16 if name == 'bf16' else torch.float32


def _ids(case, g):
    """[tokens, topk] distinct experts a token, some more popular than others; -1 marks a dropped pair."""
    t, k, n = case['tokens'], case['topk'], case['groups']
    score = torch.rand(t, n, generator=g, device='cuda') + 0.5 * torch.rand(n, generator=g, device='cuda')
    score = torch.cat((score, torch.rand(t, max(0, k - n), generator=g, device='cuda') - 1), dim=1)
    ids = score.topk(k, dim=1).indices
    ids = torch.where(ids < n, ids, -1)
    if case['dropped']:
        ids = torch.where(torch.rand(t, k, generator=g, device='cuda') < case['dropped'], -1, ids)
    return ids.to(torch.int32)


def _weights(case, g):
    return torch.softmax(torch.randn(case['tokens'], case['topk'], generator=g, device='cuda'), dim=1)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device='cuda', dtype=torch.float32).mul_(scale).to(dtype)


def _packed(codes):
    """4-bit codes, two to a byte along the last axis, the even one low."""
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).view(torch.int8)


def _scale_pairs(exps):
    """[..., rows, blocks] exponent bytes as the products take them: pairs in int16, rows contiguous, an even number."""
    *lead, rows, blocks = exps.shape
    padded = torch.zeros(*lead, rows + rows % 2, blocks + blocks % 2, dtype=torch.int32, device=exps.device)
    padded[..., :rows, :blocks] = exps
    pairs = (padded[..., 0::2] | (padded[..., 1::2] << 8)).to(torch.int16)
    return pairs.transpose(-1, -2).contiguous()[..., :rows].transpose(-1, -2)


def _quantised_weights(g, *shape):
    """Normal weights in 4 bits: (codes, scale pairs), made a group at a time."""
    made = []
    for _ in range(shape[0] if len(shape) == 3 else 1):
        exps, codes = _e2m1(_randn(g, *shape[-2:], scale=shape[-1] ** -0.5))
        made.append((_packed(codes), _scale_pairs(exps).transpose(-1, -2)))
    if len(shape) == 2:
        return made[0][0], made[0][1].transpose(-1, -2)
    k64, ld = -(-shape[2] // 64), shape[1] + shape[1] % 2
    sf = torch.zeros(shape[0], k64, ld, dtype=torch.int16, device='cuda')[..., :shape[1]]
    for i, (_, s) in enumerate(made):
        sf[i] = s
    return torch.stack([c for c, _ in made]), sf.transpose(-1, -2)


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    op, s = case['op'], {'case': case}
    if op in ('sort', 'permute', 'experts'):
        s['ids'] = _ids(case, g)
    if op in ('permute', 'experts'):
        s['weights'] = _weights(case, g)
    if op == 'permute':
        dt, h, m = _dtype(case['dtype']), case['width'], num_rows(case)
        s['x'] = _randn(g, case['tokens'], h, dtype=dt)
        s['y'] = _randn(g, m, h, dtype=dt)                      # the experts' outputs
        s['d_out'] = _randn(g, case['tokens'], h, dtype=dt)     # the gradient of what came back
        s['d_rows'] = _randn(g, m, h, dtype=dt)                 # the gradient of the experts' inputs
    elif op == 'quant':
        # rows of different size, as weights and activations have
        x = _randn(g, case['rows'], case['width']) * torch.exp(_randn(g, case['rows'], 1))
        s['x'] = x.to(_dtype(case['dtype']))
    elif op == 'product':
        s['x'] = _randn(g, case['rows'], case['width'], dtype=torch.bfloat16)
        s['w'] = _quantised_weights(g, case['cols'], case['width'])
    elif op == 'experts':
        s['x'] = _randn(g, case['tokens'], case['width'], dtype=torch.bfloat16)
        s['w'] = _quantised_weights(g, case['groups'], case['cols'], case['width'])
    elif op == 'loss':
        t = case['tokens']
        s['x'] = _randn(g, t, case['width'], dtype=torch.bfloat16)
        s['w'] = _randn(g, case['vocab'], case['width'], dtype=torch.bfloat16, scale=2.0 * case['width'] ** -0.5)
        target = torch.randint(0, case['vocab'], (t,), generator=g, device='cuda')
        if t > 1:   # (prompt and padding tokens)
            target = torch.where(torch.rand(t, generator=g, device='cuda') < 0.1, IGNORE, target)
        s['target'] = target
        s['d_loss'] = torch.full((t,), 1.0 / t, device='cuda')   # a mean over the tokens
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _sort(ids, groups, alignment, rows):
    t, k = ids.shape
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, groups, flat)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=groups + 1)[:groups]
    aligned = (counts + alignment - 1) // alignment * alignment
    start = torch.cumsum(aligned, 0) - aligned
    before = torch.cumsum(counts, 0) - counts
    sorted_key = key[order]
    live = sorted_key < groups
    group = sorted_key.clamp(max=max(groups - 1, 0))
    row = start[group] + torch.arange(t * k, device=ids.device) - before[group]
    slots = torch.full((t * k,), -1, dtype=torch.int32, device=ids.device)
    slots[order] = torch.where(live, row, -1).to(torch.int32)
    source = torch.full((rows + 1,), -1, dtype=torch.int32, device=ids.device)
    indices = source.clone()
    at = torch.where(live, row, rows)                            # (dropped pairs: a row past the last)
    source[at] = order.to(torch.int32)
    indices[at] = sorted_key.to(torch.int32)
    return slots.view(t, k), source[:rows], (start + counts).to(torch.int32), indices[:rows]


def _gathered(rows, slots):
    """[tokens, topk, width] fp32 rows of the pairs, zeros for dropped ones."""
    live = (slots >= 0).unsqueeze(-1)
    return torch.where(live, rows[slots.clamp(min=0).long()].float(), 0.0)


def _spread(x, source, topk):
    """fp32 [rows, width]: the token of each row, zeros for padding rows."""
    return torch.where((source >= 0).unsqueeze(-1), x[(source.clamp(min=0) // topk).long()].float(), 0.0)


def _blocks(x):
    """fp32 blocks of 32 values and their largest magnitudes."""
    b = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    return b, b.abs().amax(dim=-1)


def _exponents(amax, top_exponent, top_mantissa):
    """Exponent byte of the smallest power of two that takes no value of a block past the largest number of the format,
    top_mantissa * 2^top_exponent."""
    bits = amax.view(torch.int32)
    e = (bits >> 23) - top_exponent + ((bits & 0x7fffff) > round((top_mantissa - 1) * (1 << 23))).to(torch.int32)
    return e.clamp(1, 254)


def _e2m1(x):
    """(exponent bytes, 4-bit codes) of x in blocks of 32, to nearest, ties to even."""
    b, amax = _blocks(x)
    exps = _exponents(amax, 2, 1.5)
    v = b / (exps << 23).view(torch.float32).unsqueeze(-1)
    a = v.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code | ((v < 0).to(torch.uint8) << 3)).to(torch.uint8)
    return exps, code.reshape(x.shape)


def _values(exps, codes):
    """fp32 values of 4-bit codes under their exponent bytes."""
    table = torch.tensor((0., .5, 1., 1.5, 2., 3., 4., 6., -0., -.5, -1., -1.5, -2., -3., -4., -6.), device=codes.device)
    v = table[codes.long()].reshape(*exps.shape, 32) * (exps << 23).view(torch.float32).unsqueeze(-1)
    return v.reshape(codes.shape)


def _rounded(x, fmt):
    """fp32 values of x after quantisation."""
    if fmt == 'e2m1':
        return _values(*_e2m1(x))
    b, amax = _blocks(x)
    scale = (_exponents(amax, 8, 1.75) << 23).view(torch.float32).unsqueeze(-1)
    return ((b / scale).to(torch.float8_e4m3fn).float() * scale).reshape(x.shape)


def _weight_values(codes, sf):
    """fp32 values of packed 4-bit weights under their scale pairs."""
    c = codes.view(torch.uint8)
    c = torch.stack((c & 15, c >> 4), dim=-1).reshape(*c.shape[:-1], c.shape[-1] * 2)
    pairs = sf.to(torch.int32) & 0xffff
    exps = torch.stack((pairs & 255, pairs >> 8), dim=-1).reshape(*sf.shape[:-1], sf.shape[-1] * 2)
    return _values(exps[..., :c.shape[-1] // 32].contiguous(), c)


def _plain(s):
    case = s['case']
    op = case['op']
    if op in ('sort', 'permute', 'experts'):
        slots, source, psum, indices = _sort(s['ids'], case['groups'], case['alignment'], num_rows(case))
    if op == 'sort':
        return {'slots': slots, 'source': source, 'psum': psum, 'm_indices': indices}
    if op == 'permute':
        dt, w = _dtype(case['dtype']), s['weights']
        rows = _spread(s['x'], source, case['topk'])
        y = _gathered(s['y'], slots)
        out = (w.unsqueeze(-1) * y).sum(dim=1)
        d_weights = torch.where(slots >= 0, (s['d_out'].float().unsqueeze(1) * y).sum(dim=-1), 0.0)
        row_weights = torch.where(source >= 0, w.reshape(-1)[source.clamp(min=0).long()], 0.0)
        d_y = _spread(s['d_out'], source, case['topk']) * row_weights.unsqueeze(-1)
        d_x = _gathered(s['d_rows'], slots).sum(dim=1)
        return {'rows': rows.to(dt), 'out': out.to(dt), 'd_y': d_y.to(dt), 'd_weights': d_weights, 'd_x': d_x.to(dt)}
    if op == 'quant':
        return _rounded(s['x'], case['format']).to(s['x'].dtype)
    if op == 'product':
        return (_rounded(s['x'], case['format']) @ _weight_values(*s['w']).t()).to(torch.bfloat16)
    if op == 'experts':
        t, k, n = case['tokens'], case['topk'], case['groups']
        w = _weight_values(*s['w']).reshape(n * case['cols'], case['width'])
        every = (_rounded(s['x'], 'e2m1') @ w.t()).view(t, n, case['cols'])
        live = s['ids'] >= 0
        chosen = every[torch.arange(t, device='cuda').unsqueeze(1), s['ids'].clamp(min=0).long()]
        return (torch.where(live, s['weights'], 0.0).unsqueeze(-1) * chosen).sum(dim=1).to(torch.bfloat16)
    x, w, target = s['x'].float(), s['w'].float(), s['target']
    logits = x @ w.t()
    top = logits.amax(dim=1, keepdim=True)
    lse = (top + (logits - top).exp().sum(dim=1, keepdim=True).log()).squeeze(1)
    live, at = target != IGNORE, target.clamp(min=0).unsqueeze(1)
    loss = torch.where(live, lse - logits.gather(1, at).squeeze(1), 0.0)
    if not case['grad']:
        return {'loss': loss, 'lse': lse}
    d = (logits - lse.unsqueeze(1)).exp()
    d.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    d = d * torch.where(live, s['d_loss'], 0.0).unsqueeze(1)
    return {'loss': loss, 'lse': lse, 'd_x': (d @ w).to(torch.bfloat16), 'd_w': (d.t() @ x).to(torch.bfloat16)}


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
    if op in ('sort', 'permute', 'experts'):
        dg.set_mk_alignment_for_contiguous_layout(case['alignment'])
        layout = dg.moe_sort(s['ids'], case['groups'])
    if op == 'sort':
        return {'slots': layout.slots, 'source': layout.source, 'psum': layout.psum, 'm_indices': layout.m_indices}
    if op == 'permute':
        rows = dg.moe_dispatch(s['x'], layout)
        out = dg.moe_combine(s['y'], layout, s['weights'])
        d_y, d_weights = dg.moe_combine_backward(s['d_out'], s['y'], layout, s['weights'])
        d_x = dg.moe_dispatch_backward(s['d_rows'], layout)
        return {'rows': rows, 'out': out, 'd_y': d_y, 'd_weights': d_weights, 'd_x': d_x}
    if op == 'quant':
        return dg.mx_dequantize(dg.mx_quantize(s['x'], case['format']), s['x'].dtype)
    if op == 'product':
        d = torch.empty(case['rows'], case['cols'], dtype=torch.bfloat16, device='cuda')
        dg.mx_gemm_nt(s['x'], s['w'], d, case['format'])
        return d
    if op == 'experts':
        rows = dg.moe_dispatch(dg.mx_quantize(s['x'], 'e2m1'), layout, zero_padding=False)
        d = torch.empty(rows[0].size(0), case['cols'], dtype=torch.bfloat16, device='cuda')
        dg.m_grouped_fp8_fp4_gemm_nt_contiguous(rows, s['w'], d, layout.psum)
        return dg.moe_combine(d, layout, s['weights'])
    loss, lse = dg.linear_cross_entropy(s['x'], s['w'], s['target'], ignore_index=IGNORE)
    if not case['grad']:
        return {'loss': loss, 'lse': lse}
    d_x, d_w = dg.linear_cross_entropy_backward(s['d_loss'], s['x'], s['w'], s['target'], lse, ignore_index=IGNORE)
    return {'loss': loss, 'lse': lse, 'd_x': d_x, 'd_w': d_w}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    op = case['op']
    if op in ('sort', 'permute', 'experts'):
        t, k, m = case['tokens'], case['topk'], num_rows(case)
        pairs = t * k
        sort_bytes = 8 * pairs + 8 * m + 4 * case['groups']
    if op == 'sort':
        return {'bytes': sort_bytes, 'flops': 0}
    if op == 'permute':
        e, h = 2 if case['dtype'] == 'bf16' else 4, case['width']
        live = pairs * (1 - case['dropped'])
        # there: x, rows; back: the pairs' outputs, out; its gradient: d_out, the outputs, d_y; the first one's: d_rows, d_x
        elems = (t + m) + (live + t) + (t + live + m) + (live + t)
        return {'bytes': sort_bytes + e * h * elems + 12 * pairs, 'flops': 6.0 * live * h}
    code = {'e2m1': 0.5, 'e4m3': 1.0}
    if op == 'quant':
        n, e = case['rows'] * case['width'], 2 if case['dtype'] == 'bf16' else 4
        return {'bytes': n * (2 * e + 2 * code[case['format']] + 2 / 32), 'flops': 0}
    if op == 'product':
        m, n, k = case['rows'], case['cols'], case['width']
        return {'bytes': 2 * m * k + n * k * (0.5 + 1 / 32) + 2 * m * n, 'flops': 2.0 * m * n * k}
    if op == 'experts':
        n, h = case['cols'], case['width']
        live = pairs * (1 - case['dropped'])
        used = min(case['groups'], live)
        return {'bytes': 2 * t * h + used * n * h * (0.5 + 1 / 32) + 2 * t * n + 8 * pairs, 'flops': 2.0 * live * n * h}
    t, h, v = case['tokens'], case['width'], case['vocab']
    if not case['grad']:
        return {'bytes': 2 * (t * h + v * h) + 16 * t, 'flops': 2.0 * t * v * h}
    # the logits and the two products of the gradient
    return {'bytes': 4 * (t * h + v * h) + 20 * t, 'flops': 6.0 * t * v * h}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_blocks(x, fmt):
    """The quantised values from the definition: the smallest power of two that keeps a block inside the format, then the
    nearest multiple of the local step, ties to even."""
    x = x.double()
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    largest, low, bits = (6.0, 0.0, 1) if fmt == 'e2m1' else (448.0, -6.0, 3)
    scale = torch.exp2(torch.ceil(torch.log2((amax / largest).clamp(min=2.0 ** -126))).clamp(min=-126))
    scale = torch.where(amax / scale > largest, scale * 2, scale)
    scale = torch.where((amax / (scale / 2) <= largest) & (scale > 2.0 ** -126), scale / 2, scale)
    v = b / scale
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** low))).clamp(min=low)
    step = torch.exp2(exponent - bits)
    return (torch.round(v / step) * step * scale).reshape(x.shape)


def _exact_weights(codes, sf):
    """Packed 4-bit weights in 64 bits, from the bit fields of codes and exponents."""
    c = codes.view(torch.uint8).long()
    c = torch.stack((c % 16, c // 16), dim=-1).flatten(-2)
    sign, e, m = c // 8, c // 2 % 4, c % 2
    mag = torch.where(e == 0, 0.5 * m, torch.exp2(e.double() - 1) * (1 + 0.5 * m))
    pairs = sf.long() % 65536
    exps = torch.stack((pairs % 256, pairs // 256), dim=-1).flatten(-2)[..., :c.shape[-1] // 32]
    return torch.where(sign == 1, -mag, mag) * torch.exp2(exps.double() - 127).repeat_interleave(32, dim=-1)


def exact(case, seed):
    s, op = prepare(case, seed), case['op']
    if op == 'sort':
        return None   # (whole numbers)
    if op == 'quant':
        return _exact_blocks(s['x'], case['format'])
    if op == 'product':
        return _exact_blocks(s['x'], case['format']) @ _exact_weights(*s['w']).t()
    if op in ('permute', 'experts'):
        ids, w = s['ids'].long(), s['weights'].double()
        t, k = ids.shape
    if op == 'experts':
        x, out = _exact_blocks(s['x'], 'e2m1'), torch.zeros(t, case['cols'], dtype=torch.float64, device='cuda')
        for e in range(case['groups']):
            gate = torch.where(ids == e, w, 0.0).sum(dim=1, keepdim=True)
            out += gate * (x @ _exact_weights(s['w'][0][e], s['w'][1][e]).t())
        return out
    if op == 'permute':
        m, h, a = num_rows(case), case['width'], case['alignment']
        x, y, d_out, d_rows = (s[n].double() for n in ('x', 'y', 'd_out', 'd_rows'))
        rows = torch.zeros(m, h, dtype=torch.float64, device='cuda')
        d_y, out, d_x = rows.clone(), torch.zeros_like(x), torch.zeros_like(x)
        d_w = torch.zeros(t * k, dtype=torch.float64, device='cuda')
        first = 0
        for e in range(case['groups']):   # a group's pairs in order, one group after another
            pair = (ids.reshape(-1) == e).nonzero().squeeze(1)
            n, token = pair.numel(), pair // k
            mine = slice(first, first + n)
            gate = w.reshape(-1)[pair].unsqueeze(1)
            rows[mine] = x[token]
            d_y[mine] = gate * d_out[token]
            d_w[pair] = (d_out[token] * y[mine]).sum(1)
            out.index_add_(0, token, gate * y[mine])
            d_x.index_add_(0, token, d_rows[mine])
            first += -(-n // a) * a
        return {'rows': rows, 'out': out, 'd_y': d_y, 'd_weights': d_w.view(t, k), 'd_x': d_x}
    x, w, target = s['x'].double(), s['w'].double(), s['target']
    live = target != IGNORE
    loss, lse = [], []
    d_x, d_w = torch.zeros_like(x), torch.zeros_like(w)
    for i in range(0, x.shape[0], 1024):   # (a chunk of tokens at a time)
        part = slice(i, min(i + 1024, x.shape[0]))
        z = x[part] @ w.t()
        n = torch.arange(z.shape[0], device='cuda')
        l = torch.logsumexp(z, dim=1)
        at = torch.where(live[part], target[part], 0)
        loss.append(torch.where(live[part], l - z[n, at], 0.0))
        lse.append(l)
        if case['grad']:
            p = torch.exp(z - l.unsqueeze(1))
            p[n, at] -= 1
            p *= torch.where(live[part], s['d_loss'][part].double(), 0.0).unsqueeze(1)
            d_x[part] = p @ w
            d_w += p.t() @ x[part]
    found = {'loss': torch.cat(loss), 'lse': torch.cat(lse)}
    if case['grad']:
        found.update(d_x=d_x, d_w=d_w)
    return found
