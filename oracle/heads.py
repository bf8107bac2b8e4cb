"""Float64 CPU statements of the operators on attention heads and the paged cache.

From their definitions, token by token and head by head; no kernel's order of
work is followed. Used by the tests alone.
"""

import math

import torch


def angles(positions, rotary, base=10000.0):
    """Angles [tokens, rotary / 2] of whole positions."""
    f = torch.tensor([base ** (-2.0 * i / rotary) for i in range(rotary // 2)], dtype=torch.float64)
    return positions.double()[:, None] * f


def pairs(rotary, interleaved):
    i = torch.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def turn(x, cos, sin, interleaved=False):
    """x [tokens, heads, dim] with its pairs turned; cos and sin [tokens, rotary / 2]."""
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = pairs(2 * cos.shape[-1], interleaved)
    y = x.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def from_table(table, positions):
    """(cos, sin) of the positions, NaN outside the table."""
    half = table.shape[1] // 2
    rows = table.double()[positions.long().clamp(0, table.shape[0] - 1)]
    bad = (positions < 0) | (positions >= table.shape[0])
    rows = torch.where(bad[:, None], math.nan, rows)
    return rows[:, :half], rows[:, half:]


def norm(x, weight, eps):
    """Each head over its root mean square, times the weight."""
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def norm_turn(x, weight, eps, table, positions, interleaved=False):
    """The forward of ``qk_norm_rotary`` for one tensor (weight or table may be None)."""
    y = x.double() if weight is None else norm(x, weight, eps)
    return y if table is None else turn(y, *from_table(table, positions), interleaved)


def norm_turn_grad(x, weight, eps, table, positions, g, interleaved=False):
    """(dx, dweight) for the upstream gradient g, from the Jacobian of the norm:
    d n_i / d x_j = (delta_ij - n_i n_j / dim) / rms."""
    x, g = x.double(), g.double()
    if table is not None:
        cos, sin = from_table(table, positions)
        g = turn(g, cos, -sin, interleaved)
    if weight is None:
        return g, None
    rms = torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x / rms
    gw = g * weight.double()
    return (gw - n * (n * gw).mean(-1, keepdim=True)) / rms, (g * n).sum((0, 1))


def sequences(lengths, starts, tokens):
    """(sequence, position) of each token; sequence -1 where it has none."""
    batch = len(lengths)
    if starts is None:
        per = tokens // batch if batch else 0
        starts = [b * per for b in range(batch + 1)]
    out = [(-1, -1)] * tokens
    for b in range(batch):
        first, end = int(starts[b]), int(starts[b + 1])
        for t in range(first, end):
            out[t] = (b, int(lengths[b]) - (end - first) + t - first)
    return out


def place(page_table, b, p, page_size, n_pages):
    """(page, slot) of position p of sequence b, or None."""
    if p < 0 or p // page_size >= page_table.shape[1]:
        return None
    page = int(page_table[b, p // page_size])
    return (page, p % page_size) if 0 <= page < n_pages else None


def append(q, k, v, k_cache, v_cache, page_table, lengths, starts, q_weight, k_weight, eps, table, interleaved):
    """(q', k_cache', v_cache') in float64; q' rows of no sequence are NaN."""
    tokens = k.shape[0]
    where = sequences(lengths.tolist(), None if starts is None else starts.tolist(), tokens)
    pos = torch.tensor([p for _, p in where], dtype=torch.int64)
    k_cache, v_cache = k_cache.double().clone(), v_cache.double().clone()
    kt = norm_turn(k, k_weight, eps, table, pos, interleaved)
    for t, (b, p) in enumerate(where):
        at = place(page_table, b, p, k_cache.shape[1], k_cache.shape[0]) if b >= 0 else None
        if at is not None:
            k_cache[at] = kt[t]
            v_cache[at] = v[t].double()
    if q is None:
        return None, k_cache, v_cache
    q = norm_turn(q, q_weight, eps, table, pos, interleaved)
    q[[b < 0 for b, _ in where]] = math.nan
    return q, k_cache, v_cache


def attend(q, k_cache, v_cache, page_table, lengths, starts, scale, softcap=0.0, window=0, bounds=False):
    """Attention of each token; with ``bounds`` also the largest |score - top score|,
    the largest sum of |q k| times scale, and sum softmax |v|, for error bounds."""
    tokens, heads, dim = q.shape
    group = heads // k_cache.shape[2]
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    spread, reach, mass = torch.zeros(tokens, heads), torch.zeros(tokens, heads), torch.zeros_like(out)
    for t, (b, p) in enumerate(sequences(lengths.tolist(), None if starts is None else starts.tolist(), tokens)):
        if b < 0:
            continue
        first = max(0, p - window + 1) if window else 0
        at = [place(page_table, b, j, k_cache.shape[1], k_cache.shape[0])
              for j in range(first, min(p + 1, int(lengths[b])))]
        at = [x for x in at if x is not None]
        if not at:
            continue
        page, slot = torch.tensor([x[0] for x in at]), torch.tensor([x[1] for x in at])
        keys, values = k_cache[page, slot].double(), v_cache[page, slot].double()  # [n, kv_heads, dim]
        keys, values = keys.repeat_interleave(group, 1), values.repeat_interleave(group, 1)
        x = q[t].double()
        s = (keys * x).sum(-1) * scale
        if softcap > 0:
            s = softcap * torch.tanh(s / softcap)
        top = s.amax(0)
        e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(0)
        pr = e / torch.where(total == 0, 1.0, total)
        out[t] = torch.where((total == 0)[:, None], 0.0, (pr[..., None] * values).sum(0))
        if bounds:
            spread[t] = (top - s.amin(0)).float()
            reach[t] = ((keys * x).abs().sum(-1).amax(0) * scale).float()
            mass[t] = (pr[..., None] * values.abs()).sum(0)
    return (out, spread, reach, mass) if bounds else out
