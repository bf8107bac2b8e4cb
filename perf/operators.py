"""Scoring and distilling with a language model's head: the calls whose speed is measured.

Three operators of this framework, one dict per case:

* ``logprobs``: log probabilities of given tokens, the entropy and the top
  alternatives of each row of logits (``kernels.hip.token_logprobs``), forward,
  or forward and backward;
* ``distill``: the distillation loss against a teacher's top logits
  (``kernels.hip.topk_distillation``), forward and backward;
* ``lmhead``: log probabilities and entropies straight from hidden states and
  the head's weight, without logits in memory (``kernels.hip.lmhead_logprobs``),
  forward, or forward and backward.

``run`` computes each in elementary torch operations in 32 bits, or, where
``own`` is set, calls the framework. ``exact`` restates them in float64.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "autokernel-halo-strix_amd")
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_IGNORE = -100


def listed():
    return [
        # one decode step of a batch of 8 under a grammar's mask, with the 20 top alternatives an API returns
        {"name": "logprobs_decode", "op": "logprobs", "dtype": "bf16", "rows": 8, "vocab": 50257, "top": 20,
         "masked": True, "temperature": 0.7, "softcap": 0.0, "ignored": False, "train": False},
        # one step of one sequence over a large vocabulary, logits kept in fp32
        {"name": "logprobs_one_row", "op": "logprobs", "dtype": "f32", "rows": 1, "vocab": 262144, "top": 5,
         "masked": False, "temperature": 1.0, "softcap": 30.0, "ignored": False, "train": False},
        # scoring 8 x 1024 tokens of finished rollouts, prompt tokens ignored
        {"name": "logprobs_score", "op": "logprobs", "dtype": "bf16", "rows": 8192, "vocab": 50304, "top": 0,
         "masked": False, "temperature": 1.0, "softcap": 0.0, "ignored": True, "train": False},
        # a teacher's pass: the 64 top logits of each of 4096 tokens, kept for a student
        {"name": "logprobs_teacher", "op": "logprobs", "dtype": "bf16", "rows": 4096, "vocab": 32768, "top": 64,
         "masked": False, "temperature": 1.0, "softcap": 0.0, "ignored": False, "train": False},
        # a policy-gradient step with an entropy bonus over materialised logits, rows off the 16-byte grid
        {"name": "logprobs_train", "op": "logprobs", "dtype": "bf16", "rows": 4096, "vocab": 50257, "top": 0,
         "masked": False, "temperature": 0.9, "softcap": 0.0, "ignored": True, "train": True},
        # distillation of a short batch in fp16, 20 alternatives a token as an API gives them
        {"name": "distill_small", "op": "distill", "dtype": "f16", "rows": 200, "vocab": 50257, "top": 20,
         "temperature": 1.0, "softcap": 0.0},
        # a distillation step of 4 x 1024 tokens from 64 stored logits a token
        {"name": "distill_train", "op": "distill", "dtype": "bf16", "rows": 4096, "vocab": 32768, "top": 64,
         "temperature": 2.0, "softcap": 0.0},
        # fp32 logits of a capped head, an odd number of tokens, many alternatives
        {"name": "distill_f32", "op": "distill", "dtype": "f32", "rows": 1999, "vocab": 50257, "top": 128,
         "temperature": 2.0, "softcap": 30.0},
        # scoring one short completion
        {"name": "lmhead_short", "op": "lmhead", "dtype": "bf16", "rows": 37, "vocab": 50257, "d": 768,
         "temperature": 1.0, "softcap": 0.0, "train": False},
        # scoring 8 x 1024 tokens of rollouts with a GPT-2-sized head
        {"name": "lmhead_score", "op": "lmhead", "dtype": "bf16", "rows": 8192, "vocab": 50304, "d": 768,
         "temperature": 1.0, "softcap": 0.0, "train": False},
        # a policy-gradient step of the reference's small language model: 4 x 256 tokens, softcap 30
        {"name": "lmhead_train_1k", "op": "lmhead", "dtype": "bf16", "rows": 1024, "vocab": 32768, "d": 768,
         "temperature": 0.9, "softcap": 30.0, "train": True},
        # the same step of 8 x 1024 tokens
        {"name": "lmhead_train_8k", "op": "lmhead", "dtype": "bf16", "rows": 8192, "vocab": 50304, "d": 768,
         "temperature": 1.0, "softcap": 0.0, "train": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _rough(rng, n, unit):
    """n as it is one time in three, otherwise a multiple of ``unit``."""
    return n if rng.random() < 1 / 3 else max(unit, n // unit * unit)


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs", "distill", "distill", "lmhead", "lmhead"])
    temperature = round(rng.uniform(0.5, 2.0), 2)
    softcap = rng.choice([0.0, 0.0, 30.0])
    if op == "lmhead":
        train = rng.random() < 0.5
        vocab = _rough(rng, _spread(rng, 2000, 50304), 64)
        d = _rough(rng, _spread(rng, 128, 768), 64)
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16"]), "rows": _spread(rng, 16, 8192),
                "vocab": vocab, "d": d, "temperature": temperature, "softcap": softcap, "train": train}
    vocab = _rough(rng, _spread(rng, 2000, 262144), 64)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "distill":
        rows = min(_spread(rng, 8, 4096), 130_000_000 // vocab)
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "top": _spread(rng, 1, 128),
                "temperature": temperature, "softcap": softcap}
    rows = min(_spread(rng, 1, 8192), 130_000_000 // vocab)
    train = rows >= 64 and rng.random() < 0.4
    return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab,
            "top": 0 if train else rng.choice([0, 1, 5, 20, 64, 128]), "masked": rng.random() < 0.3,
            "temperature": temperature, "softcap": softcap, "ignored": rng.random() < 0.5, "train": train}


def prepare(case, seed):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, n, v = _DT[case["dtype"]], case["rows"], case["vocab"]

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def tokens():
        return torch.randint(0, v, (n,), generator=g, device="cuda")

    st = dict(case)
    if case["op"] == "lmhead":
        st["hidden"] = rnd(n, case["d"]).to(dt)
        st["weight"] = (rnd(v, case["d"]) * (2.0 / math.sqrt(case["d"]))).to(dt)
        st["tokens"] = tokens()
        st["tokens"][: n // 4] = _IGNORE  # the prompt
        if case["train"]:
            st["hidden"].requires_grad_()
            st["weight"].requires_grad_()
    else:
        # a few confident tokens over a wide base, as a trained head gives them
        x = rnd(n, v) * 2.0
        x += 6.0 * (torch.rand(n, v, generator=g, device="cuda") > 0.9995)
        if case["op"] == "distill":
            t = x + 0.7 * rnd(n, v)
            val, ids = t.topk(case["top"], dim=1)
            # a teacher that gave fewer alternatives for some tokens, and none for the prompt's
            count = torch.randint(1, case["top"] + 1, (n, 1), generator=g, device="cuda")
            count[torch.rand(n, 1, generator=g, device="cuda") < 0.7] = case["top"]
            count[: n // 8] = 0
            gone = torch.arange(case["top"], device="cuda")[None, :] >= count
            st["teacher"] = val.float().contiguous()
            st["ids"] = ids.masked_fill(gone, _IGNORE).contiguous()
        else:
            st["tokens"] = tokens()
            if case["masked"]:
                x.masked_fill_(torch.rand(n, v, generator=g, device="cuda") > 0.05, -math.inf)
                x.scatter_(1, st["tokens"][:, None], 3.0)
            if case["ignored"]:
                st["tokens"][: n // 4] = _IGNORE
        st["logits"] = x.to(dt)
        del x
        if case["op"] == "distill" or case["train"]:
            st["logits"].requires_grad_()
    # the upstream gradients; fp16 training multiplies its loss, here by 8 times the tokens
    scale = 8.0 * n if case["dtype"] == "f16" else 1.0
    if case["op"] == "distill":
        st["g_loss"] = torch.full((), 0.7 * scale, device="cuda")  # the loss's weight beside the data's own
    if case.get("train"):
        st["g_logprobs"] = rnd(n) * (scale / n)  # advantages over the batch
        st["g_entropy"] = torch.full((n,), 0.01 * scale / n, device="cuda")
    return st


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_scores(x, case):
    """(scores, d scores / d logits) in fp32: the softcap, then the temperature."""
    x = x.detach().float()
    if case["softcap"] > 0:
        th = torch.tanh(x / case["softcap"])
        return case["softcap"] * th / case["temperature"], (1 - th * th) / case["temperature"]
    return x / case["temperature"], 1.0 / case["temperature"]


def _plain_stats(z):
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    logp = d - torch.log(s)
    p = e / s
    plogp = torch.where(p > 0, p * logp, torch.zeros((), device=z.device))
    return p, logp, -plogp.sum(1)


def _plain_picked(logp, entropy, tok):
    counted = tok != _IGNORE
    picked = logp.gather(1, tok.clamp(min=0)[:, None])[:, 0]
    zero = torch.zeros((), device=tok.device)
    return torch.where(counted, picked, zero), torch.where(counted, entropy, zero), counted


def _plain_dscores(p, logp, entropy, counted, tok, g_logprobs, g_entropy):
    zero = torch.zeros((), device=tok.device)
    gl = torch.where(counted, g_logprobs, zero)[:, None]
    ge = torch.where(counted, g_entropy, zero)[:, None]
    dz = torch.where(p > 0, -p * (gl + ge * (logp + entropy[:, None])), zero)
    return dz.scatter_add_(1, tok.clamp(min=0)[:, None], gl)


def _plain_logprobs(st):
    x, tok = st["logits"], st["tokens"]
    z, dzdx = _plain_scores(x, st)
    p, logp, entropy = _plain_stats(z)
    lp, ent, counted = _plain_picked(logp, entropy, tok)
    if st["train"]:
        dz = _plain_dscores(p, logp, entropy, counted, tok, st["g_logprobs"], st["g_entropy"])
        return lp, ent, (dz * dzdx).to(x.dtype)
    if not st["top"]:
        return lp, ent
    # one whole number for each entry: its logit's place among the numbers, then the lower index first
    bits = (x.detach().float() + 0.0).view(torch.int32).to(torch.int64)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32
    key += (1 << 31) - 1 - torch.arange(x.shape[1], device=x.device)
    ids = (1 << 31) - 1 - (key.topk(st["top"], dim=1).values & 0xFFFFFFFF)
    return lp, ent, logp.gather(1, ids), ids


def _plain_distill(st):
    x, t, ids = st["logits"], st["teacher"].float() / st["temperature"], st["ids"]
    there = ids != _IGNORE
    counted = there.any(1)
    at = ids.clamp(min=0)
    t = t.masked_fill(~there, -math.inf)
    t = t - t.amax(1, keepdim=True)
    e = torch.exp(t)
    s = e.sum(1, keepdim=True)
    zero = torch.zeros((), device=x.device)
    q = torch.where(there, e / s, zero)
    logq = torch.where(there, t - torch.log(s), zero)
    z, dzdx = _plain_scores(x, st)
    p, logp, _ = _plain_stats(z)
    t2 = st["temperature"] ** 2
    rows = t2 * (q * (logq - logp.gather(1, at))).sum(1)
    n = counted.sum().clamp(min=1)
    dz = torch.where(counted[:, None], p, zero).scatter_add_(1, at, -q)
    return rows.masked_fill(~counted, 0.0).sum() / n, (dz * (st["g_loss"] * (t2 / n)) * dzdx).to(x.dtype)


def _plain_lmhead(st):
    h, w, tok = st["hidden"].detach().float(), st["weight"].detach().float(), st["tokens"]
    z, dzdx = _plain_scores(h @ w.t(), st)
    p, logp, entropy = _plain_stats(z)
    lp, ent, counted = _plain_picked(logp, entropy, tok)
    if not st["train"]:
        return lp, ent
    dz = _plain_dscores(p, logp, entropy, counted, tok, st["g_logprobs"], st["g_entropy"]) * dzdx
    return lp, ent, (dz @ w).to(st["hidden"].dtype), (dz.t() @ h).to(st["weight"].dtype)


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _own_logprobs(st):
    from kernels.hip.token_logprobs import kernel_fn
    r = kernel_fn(st["logits"], st["tokens"], temperature=st["temperature"], softcap=st["softcap"],
                  ignore_index=_IGNORE, top_k=st["top"])
    if st["train"]:
        (gx,) = torch.autograd.grad((r.logprobs, r.entropy), (st["logits"],), (st["g_logprobs"], st["g_entropy"]))
        return r.logprobs, r.entropy, gx
    if not st["top"]:
        return r.logprobs, r.entropy
    return r.logprobs, r.entropy, r.top_logprobs, r.top_ids


def _own_distill(st):
    from kernels.hip.topk_distillation import kernel_fn
    loss = kernel_fn(st["logits"], st["teacher"], st["ids"], temperature=st["temperature"], softcap=st["softcap"],
                     ignore_index=_IGNORE)
    (gx,) = torch.autograd.grad(loss, (st["logits"],), (st["g_loss"],))
    return loss, gx


def _own_lmhead(st):
    from kernels.hip.lmhead_logprobs import kernel_fn
    r = kernel_fn(st["hidden"], st["weight"], st["tokens"], temperature=st["temperature"], softcap=st["softcap"],
                  ignore_index=_IGNORE)
    if not st["train"]:
        return r.logprobs, r.entropy
    gh, gw = torch.autograd.grad((r.logprobs, r.entropy), (st["hidden"], st["weight"]),
                                 (st["g_logprobs"], st["g_entropy"]))
    return r.logprobs, r.entropy, gh, gw


def run(state):
    op = state["op"]
    if own:
        return {"logprobs": _own_logprobs, "distill": _own_distill, "lmhead": _own_lmhead}[op](state)
    return {"logprobs": _plain_logprobs, "distill": _plain_distill, "lmhead": _plain_lmhead}[op](state)


def work(case):
    n, v, e = case["rows"], case["vocab"], _SIZE[case["dtype"]]
    if case["op"] == "lmhead":
        d = case["d"]
        weights = (n + v) * d * e
        return {"bytes": weights * (2 if case["train"] else 1) + n * (32 if case["train"] else 16),
                "flops": 2 * n * v * d * (3 if case["train"] else 1)}
    if case["op"] == "distill":
        return {"bytes": 2 * n * v * e + n * case["top"] * 12, "flops": 8 * n * v}
    per_row = 16 + 12 * case["top"] + (8 if case["train"] else 0)
    return {"bytes": (2 if case["train"] else 1) * n * v * e + n * per_row,
            "flops": (12 if case["train"] else 6) * n * v}


# ---------------------------------------------------------------------------
# In 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_head(x, case):
    """A function of float64 logits that returns (scores, log probabilities)."""
    z = x if case["softcap"] == 0 else case["softcap"] * torch.tanh(x / case["softcap"])
    z = z / case["temperature"]
    return z, z - torch.logsumexp(z, 1, keepdim=True)


def _exact_grad_logits(x, case, logp, weight_of, entropy_of, tok):
    """d (sum of weight_of * logp[tok] + entropy_of * H) / d logits, through the
    Jacobian of the log softmax: J^T c = c - p sum(c), with c the derivative by
    each log probability."""
    p = logp.exp()
    c = -entropy_of[:, None] * p * torch.where(p > 0, logp + 1, 0.0)
    c[torch.arange(len(tok), device=x.device), tok] += weight_of
    dz = c - p * c.sum(1, keepdim=True)
    if case["softcap"] > 0:
        dz = dz / torch.cosh(x / case["softcap"]) ** 2
    return dz / case["temperature"]


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "distill":
            return _exact_distill(case, st)
        x = (st["logits"] if case["op"] == "logprobs" else None)
        x = x.double() if x is not None else st["hidden"].double() @ st["weight"].double().t()
        _, logp = _exact_head(x, case)
        tok = st["tokens"]
        here = (tok >= 0).double()
        row = torch.arange(len(tok), device=tok.device)
        ids = torch.where(tok >= 0, tok, 0)
        lp = torch.where(tok >= 0, logp[row, ids], 0.0)
        p = logp.exp()
        ent = -torch.xlogy(p, p).sum(1) * here
        if case["train"]:
            gx = _exact_grad_logits(x, case, logp, here * st["g_logprobs"].double(),
                                    here * st["g_entropy"].double(), ids)
            if case["op"] == "logprobs":
                return lp, ent, gx
            return lp, ent, gx @ st["weight"].double(), gx.t() @ st["hidden"].double()
        if case.get("top"):
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]].clone()
            return lp, ent, torch.gather(logp, 1, order), order
        return lp, ent


def _exact_distill(case, st):
    x, ids, t = st["logits"].double(), st["ids"], case["temperature"]
    _, logp = _exact_head(x, case)
    have = ids >= 0
    q = torch.softmax(torch.where(have, st["teacher"].double() / t, -1e300), 1) * have
    rows = have.any(1)
    n = max(1, int(rows.sum()))
    slot = torch.where(have, ids, 0)
    terms = torch.xlogy(q, q) - q * torch.gather(logp, 1, slot)
    loss = t * t * (terms * have).sum() / n
    full = torch.zeros_like(x).scatter_add_(1, slot, q)
    dz = logp.exp() * rows[:, None] - full
    if case["softcap"] > 0:
        dz = dz / torch.cosh(x / case["softcap"]) ** 2
    return loss, dz * (st["g_loss"].double() * (t / n))
