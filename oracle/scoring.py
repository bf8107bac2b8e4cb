"""Float64 CPU statements of the scoring and distillation operators.

From their definitions, entry by entry where that is plainest; no kernel's
order of work is followed. Used by the tests alone.
"""

import math

import torch


def scores(x, temperature=1.0, softcap=0.0):
    """The capped, tempered logits in float64."""
    x = x.double()
    if softcap > 0:
        x = softcap * torch.tanh(x / softcap)
    return x / temperature


def _log_softmax(z):
    """``ln softmax`` of each row; rows of -inf alone stay -inf."""
    # relative to the largest: beside scores of 1e38 the logarithm of the sum would be lost in 64 bits, too
    top = z.amax(-1, keepdim=True)
    d = z - torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    out = d - torch.logsumexp(d, -1, keepdim=True)
    empty = (z == -math.inf).all(-1, keepdim=True)
    out = torch.where(empty, z, out)
    return torch.where((torch.isnan(z) | (z == math.inf)).any(-1, keepdim=True), math.nan, out)


def _plogp(logp):
    p = logp.exp()
    return torch.where(p == 0, torch.zeros_like(p), p * logp)


def logprob_rows(x, tokens, temperature=1.0, softcap=0.0, ignore_index=-100):
    """``(logprobs, entropy)`` of ``[rows, vocab]``; tokens may be None."""
    logp = _log_softmax(scores(x, temperature, softcap))
    entropy = -_plogp(logp).sum(-1)
    if tokens is None:
        return None, entropy
    picked = torch.empty_like(entropy)
    for r, t in enumerate(tokens.tolist()):
        if t == ignore_index:
            picked[r] = entropy[r] = 0.0
        elif not 0 <= t < x.shape[1]:
            picked[r] = math.nan
        else:
            picked[r] = logp[r, t]
    return picked, entropy


def top_rows(x, k, temperature=1.0, softcap=0.0):
    """``(top_logprobs, top_ids)``: NaN first, then by value, then by column."""
    logp = _log_softmax(scores(x, temperature, softcap))
    v = x.double()
    rows = [sorted(range(len(r)), key=lambda i: (0 if r[i] != r[i] else 1, -r[i] if r[i] == r[i] else 0.0, i))[:k]
            for r in v.tolist()]
    ids = torch.tensor(rows, dtype=torch.int64).reshape(len(rows), k)
    return logp.gather(1, ids), ids


def logprob_grad_rows(x, tokens, g_logprobs, g_entropy, temperature=1.0, softcap=0.0, ignore_index=-100):
    """``(gradient, size)``: the gradient of ``sum(g_logprobs * logprobs +
    g_entropy * entropy)`` by each logit, and the sum of its terms' absolute
    values, which what an evaluation in fewer bits may be off by goes by."""
    z = scores(x, temperature, softcap)
    logp = _log_softmax(z)
    p = logp.exp()
    entropy = -_plogp(logp).sum(-1, keepdim=True)
    slope = torch.full_like(z, 1.0 / temperature)
    if softcap > 0:
        slope = slope * torch.cosh(x.double() / softcap) ** -2
    grad, size = torch.zeros_like(z), torch.zeros_like(z)
    for r in range(x.shape[0]):
        t = None if tokens is None else int(tokens[r])
        if t == ignore_index or bool((z[r] == -math.inf).all()):
            slope[r] = 0.0  # whatever the row holds (a NaN logit has a NaN slope)
            continue
        g = 0.0 if g_logprobs is None or t is None else float(g_logprobs[r])
        e = 0.0 if g_entropy is None else float(g_entropy[r])
        if t is not None and not 0 <= t < x.shape[1]:
            grad[r] = math.nan
            continue
        pl = torch.where(p[r] == 0, torch.zeros_like(p[r]), p[r] * (logp[r] + entropy[r]))
        pa = torch.where(p[r] == 0, torch.zeros_like(p[r]), p[r] * (logp[r].abs() + entropy[r]))
        grad[r] = -g * p[r] - e * pl
        size[r] = abs(g) * p[r] + abs(e) * pa
        if t is not None:
            grad[r, t] += g
            size[r, t] += abs(g)
    return grad * slope, size * slope


def distill_rows(x, teacher, ids, temperature=1.0, softcap=0.0, ignore_index=-100):
    """``(losses, q, counted)``: each row's loss, the teacher's probabilities
    by column ``[rows, vocab]`` and whether the row has entries."""
    logp = _log_softmax(scores(x, temperature, softcap))
    rows, vocab = x.shape
    losses, full = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, vocab, dtype=torch.float64)
    counted = torch.zeros(rows, dtype=torch.bool)
    for r in range(rows):
        entries = [(int(i), float(t)) for i, t in zip(ids[r], teacher[r].double()) if int(i) != ignore_index]
        if any(not 0 <= i < vocab or math.isnan(t) or t == math.inf for i, t in entries):
            losses[r], full[r], counted[r] = math.nan, math.nan, True
            continue
        entries = [(i, t / temperature) for i, t in entries if t != -math.inf]
        if not entries:
            continue
        counted[r] = True
        top = max(t for _, t in entries)
        norm = top + math.log(sum(math.exp(t - top) for _, t in entries))
        for i, t in entries:
            q = math.exp(t - norm)
            if q > 0:
                losses[r] += temperature ** 2 * q * ((t - norm) - float(logp[r, i]))
                full[r, i] += q
        if torch.isnan(losses[r]):
            full[r] = math.nan
    return losses, full, counted


def distill_grad_rows(x, teacher, ids, upstream, temperature=1.0, softcap=0.0, ignore_index=-100):
    """``(gradient, size)`` of ``sum(upstream * losses)``, as logprob_grad_rows."""
    z = scores(x, temperature, softcap)
    empty = (z == -math.inf).all(-1, keepdim=True)
    p = torch.where(empty, torch.zeros_like(z), _log_softmax(z).exp())
    _, q, counted = distill_rows(x, teacher, ids, temperature, softcap, ignore_index)
    slope = torch.full_like(z, temperature)
    if softcap > 0:
        slope = slope * torch.cosh(x.double() / softcap) ** -2
    by = upstream.double().reshape(-1, 1) * slope * counted[:, None]
    grad = torch.where(counted[:, None], (p - q) * by, torch.zeros_like(z))
    return grad, torch.where(counted[:, None], (p + q) * by.abs(), torch.zeros_like(z))
