"""Oracle of the token sorting and movement (test infrastructure only; see ``oracle/__init__.py``): a pair at a time, in
64 bits."""
import torch


def sort(ids: torch.Tensor, num_groups: int, alignment: int, num_rows: int):
    """(slots [T, K], source [M], psum [G], m_indices [M]); pairs that do not fit num_rows are dropped."""
    t, k = ids.shape
    groups = [[] for _ in range(num_groups)]
    for p, e in enumerate(ids.reshape(-1).tolist()):
        if 0 <= e < num_groups:
            groups[e].append(p)
    slots = torch.full((t * k,), -1, dtype=torch.int32)
    source = torch.full((num_rows,), -1, dtype=torch.int32)
    m_indices = source.clone()
    psum, first = [], 0
    for e, pairs in enumerate(groups):
        for i, p in enumerate(pairs):
            if first + i < num_rows:
                slots[p], source[first + i], m_indices[first + i] = first + i, p, e
        psum.append(min(num_rows, first + len(pairs)))
        first += -(-len(pairs) // alignment) * alignment
    return slots.view(t, k), source, torch.tensor(psum, dtype=torch.int32), m_indices


def dispatch(x: torch.Tensor, source: torch.Tensor, topk: int) -> torch.Tensor:
    """[M, H]: the tokens in their rows, zeros in padding rows."""
    out = torch.zeros(source.numel(), *x.shape[1:], dtype=x.dtype)
    live = source >= 0
    out[live] = x[(source[live] // max(topk, 1)).long()]
    return out


def combine(rows: torch.Tensor, slots: torch.Tensor, weights=None):
    """(out [T, H], sum of the terms' magnitudes [T, H]) in 64 bits."""
    t, k = slots.shape
    out = torch.zeros(t, rows.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for i in range(t):
        for c in range(k):
            s = int(slots[i, c])
            if s >= 0:
                v = rows[s].double() * (1.0 if weights is None else float(weights[i, c]))
                out[i] += v
                mag[i] += v.abs()
    return out, mag


def combine_backward(d_out: torch.Tensor, rows: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor):
    """(d_rows [M, H], d_weights [T, K], sum of the magnitudes of d_weights' terms [T, K]) in 64 bits."""
    t, k = slots.shape
    d_rows = torch.zeros(rows.shape, dtype=torch.float64)
    d_weights = torch.zeros(t, k, dtype=torch.float64)
    mag = torch.zeros_like(d_weights)
    for i in range(t):
        for c in range(k):
            s = int(slots[i, c])
            if s >= 0:
                d_rows[s] = d_out[i].double() * float(weights[i, c])
                terms = d_out[i].double() * rows[s].double()
                d_weights[i, c], mag[i, c] = terms.sum(), terms.abs().sum()
    return d_rows, d_weights, mag
