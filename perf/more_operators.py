"""Attention's operators around a paged cache: the calls whose speed is measured.

Four operators of this framework, one dict per case:

* ``rotary``: the rotation of positions on queries and keys
  (``kernels.hip.rotary``), forward, or forward and backward;
* ``norm``: an RMSNorm of each head of queries and keys with the rotation in the
  same pass (``kernels.hip.qk_norm_rotary``), forward, or forward and backward;
* ``append``: new keys and values into a paged cache, queries and keys rotated
  on the way (``kernels.hip.paged_append``);
* ``attend``: attention of each sequence's new tokens over its paged cache
  (``kernels.hip.paged_attention``), one token a sequence or many.

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
_EPS = 1e-6


def listed():
    return [
        # a training step's queries and keys, 8 x 1024 tokens, positions counted along the sequence
        {"name": "rotary_train", "op": "rotary", "dtype": "bf16", "batch": 8, "seq": 1024, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "factor": 1.0, "far": 0, "train": True},
        # scoring an odd number of tokens far into a long context, part of each head rotated, fp32
        {"name": "rotary_partial", "op": "rotary", "dtype": "f32", "batch": 1, "seq": 1999, "q_heads": 16, "kv_heads": 4,
         "dim": 80, "rotary": 48, "interleaved": True, "factor": 4.0, "far": 100000, "train": False},
        # one decode step of 8 sequences, heads of a GPT-2-sized model
        {"name": "norm_decode", "op": "norm", "dtype": "f16", "batch": 8, "seq": 1, "q_heads": 12, "kv_heads": 12,
         "dim": 64, "rotary": 64, "interleaved": False, "factor": 1.0, "far": 900, "train": False},
        # a training step of 8 x 1024 tokens with shared key heads, the weights' gradients too
        {"name": "norm_train", "op": "norm", "dtype": "bf16", "batch": 8, "seq": 1024, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "factor": 1.0, "far": 0, "train": True},
        # the same in fp32 for a small odd batch, part of a 96-wide head rotated in neighbouring pairs
        {"name": "norm_f32", "op": "norm", "dtype": "f32", "batch": 7, "seq": 143, "q_heads": 16, "kv_heads": 2,
         "dim": 96, "rotary": 64, "interleaved": True, "factor": 2.0, "far": 0, "train": True},
        # one decode step of 64 sequences
        {"name": "append_decode", "op": "append", "dtype": "bf16", "batch": 64, "context": 1024, "chunk": 1, "mixed": False,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "normed": False, "page": 16},
        # ragged prompts of up to 2048 tokens that arrive together, heads normed on the way
        {"name": "append_prompts", "op": "append", "dtype": "f16", "batch": 6, "context": 2048, "chunk": 2048, "mixed": False,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "normed": True, "page": 64},
        # one decode step of one short sequence, heads of a GPT-2-sized model
        {"name": "attend_one", "op": "attend", "dtype": "bf16", "batch": 1, "context": 777, "chunk": 1, "mixed": False,
         "q_heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "window": 0, "softcap": 0.0},
        # one decode step of 64 sequences of 2048 to 8192 tokens
        {"name": "attend_decode", "op": "attend", "dtype": "bf16", "batch": 64, "context": 8192, "chunk": 1, "mixed": False,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "softcap": 0.0},
        # one decode step of two very long sequences
        {"name": "attend_long", "op": "attend", "dtype": "f16", "batch": 2, "context": 130001, "chunk": 1, "mixed": False,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "softcap": 0.0},
        # decode steps together with chunks of up to 500 tokens of longer prompts, capped scores, a sliding window
        {"name": "attend_mixed", "op": "attend", "dtype": "f16", "batch": 16, "context": 7000, "chunk": 500, "mixed": True,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "window": 4096, "softcap": 30.0},
        # ragged prompts of up to 4096 tokens from their first token on
        {"name": "attend_prompts", "op": "attend", "dtype": "bf16", "batch": 4, "context": 4096, "chunk": 4096, "mixed": False,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "softcap": 0.0},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "append", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 64, 72, 80, 96, 128, 128, 192, 256])
    rotary = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
    interleaved = rng.random() < 0.4
    if op in ("rotary", "norm"):
        width = (q_heads + kv_heads) * dim
        tokens = _spread(rng, 1, 8192)
        tokens = max(1, min(tokens, 40_000_000 // width))
        batch = min(tokens, _spread(rng, 1, 32))
        return {"op": op, "dtype": dtype, "batch": batch, "seq": tokens // batch, "q_heads": q_heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": interleaved,
                "factor": rng.choice([1.0, 1.0, 4.0]), "far": rng.choice([0, 0, _spread(rng, 100, 500000)]),
                "train": rng.random() < 0.6}
    page = rng.choice([8, 16, 16, 32, 48, 64, 128])
    batch = _spread(rng, 1, 64)
    chunk = rng.choice([1, 1, _spread(rng, 2, 16), _spread(rng, 2, 2048)])
    chunk = max(1, min(chunk, 8192 // batch))
    mixed = chunk > 1 and rng.random() < 0.3
    if op == "append":
        context = min(chunk + _spread(rng, 1, 4096), max(chunk, 60_000_000 // (batch * kv_heads * dim)))
        return {"op": op, "dtype": dtype, "batch": batch, "context": context, "chunk": chunk, "mixed": mixed,
                "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": interleaved,
                "normed": rng.random() < 0.5, "page": page}
    # few tokens over the longest contexts, many over shorter ones; fp32 stays small
    keys = (20_000_000 if dtype == "f32" else 160_000_000) // (batch * kv_heads * dim)
    context = chunk + _spread(rng, 1, 100000)
    context = max(chunk, min(context, keys, (30_000_000 if dtype == "f32" else 500_000_000) // (batch * chunk * q_heads)))
    return {"op": op, "dtype": dtype, "batch": batch, "context": context, "chunk": chunk, "mixed": mixed,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": rng.choice([0, 0, 0, _spread(rng, 1, context)]), "softcap": rng.choice([0.0, 0.0, 30.0])}


def _layout(case):
    """([length], [new tokens]) of the sequences: lengths from the whole context down
    to a quarter of it, chunks down to a half; of mixed ones every other has one token."""
    b, context, chunk = case["batch"], case["context"], case["chunk"]
    counts = [max(1, chunk - (i * chunk) // (2 * b)) for i in range(b)]
    if case["mixed"]:
        counts = [c if i % 2 == 0 else 1 for i, c in enumerate(counts)]
    lengths = [max(c, context - (i * 3 * context) // (4 * b)) for i, c in enumerate(counts)]
    return lengths, counts


def prepare(case, seed):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, hq, hk, d = _DT[case["dtype"]], case["q_heads"], case["kv_heads"], case["dim"]

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    st = dict(case)
    if case["op"] in ("rotary", "norm"):
        b, s = case["batch"], case["seq"]
        if case["train"]:
            st["q"], st["k"] = (rnd(b, s, h, d).to(dt).requires_grad_() for h in (hq, hk))
            # fp16 training multiplies its loss
            scale = 8.0 if case["dtype"] == "f16" else 1e-3
            st["g_q"], st["g_k"] = ((scale * rnd(b, s, h, d)).to(dt) for h in (hq, hk))
        else:
            # one projection gives queries, keys and values side by side
            qkv = rnd(b, s, hq + 2 * hk, d).to(dt)
            st["q"], st["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
        st["positions"] = None  # 0, 1, ... along the sequence
        if case["far"]:
            first = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device="cuda")
            st["positions"] = first + torch.arange(s, device="cuda")
        st["table"] = _table(case, case["far"] + s)
    else:
        lengths, counts = _layout(case)
        page, need = case["page"], [-(-n // case["page"]) for n in lengths]
        total = sum(need) + 8
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["batch"], max(need) + 1), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        st.update(pages=table, lengths=whole(lengths), tokens=starts[-1], most=max(counts))
        st["starts"] = whole(starts) if max(counts) > 1 else None  # one token of each sequence
        st["k_cache"] = rnd(total, page, hk, d).to(dt)
        st["v_cache"] = rnd(total, page, hk, d).to(dt)
        if case["op"] == "append":
            qkv = rnd(starts[-1], hq + 2 * hk, d).to(dt)
            st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
            st["table"] = _table({**case, "factor": 1.0}, case["context"])
        else:
            st["q"] = (2.0 * rnd(starts[-1], hq, d)).to(dt)  # scores spread as a trained head's are
    if case["op"] == "norm" or case.get("normed"):
        st["q_weight"], st["k_weight"] = ((1.0 + 0.1 * rnd(d)).to(dt) for _ in range(2))
        if case.get("train"):
            st["q_weight"].requires_grad_()
            st["k_weight"].requires_grad_()
    return st


def _angles(case, positions):
    """[positions, rotary / 2] in float64; a longer context by a factor divides the positions."""
    r = case["rotary"]
    f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    return positions.double()[..., None] / case["factor"] * f


def _table(case, n):
    """The cosines and the sines of n positions, [n, rotary] in 32 bits, as a model keeps them."""
    a = _angles(case, torch.arange(n, device="cuda"))
    return torch.cat([torch.cos(a), torch.sin(a)], 1).float()


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_rotate(x, cos, sin, st):
    """x [..., heads, dim] in fp32; cos and sin [..., 1, rotary / 2]."""
    r = st["rotary"]
    if st["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return turned if r == x.shape[-1] else torch.cat([turned, x[..., r:]], -1)


def _plain_norm(x):
    x = x.detach().float()
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return x * inv, inv


def _plain_norm_back(dz, n, inv, w):
    dw = (dz * n).flatten(0, -2).sum(0)
    g = dz * w
    return (g - n * (g * n).mean(-1, keepdim=True)) * inv, dw


def _plain_heads(st):
    r = st["rotary"]
    q, k = st["q"], st["k"]
    rows = st["table"][:q.shape[1]] if st["positions"] is None else st["table"][st["positions"]]
    cos, sin = rows[..., None, :r // 2], rows[..., None, r // 2:]
    normed = st["op"] == "norm"
    out, grads, dws = [], [], []
    for x, up, w in ((q, "g_q", "q_weight"), (k, "g_k", "k_weight")):
        if normed:
            n, inv = _plain_norm(x)
            weight = st[w].detach().float()
            z = n * weight
        else:
            z = x.detach().float()
        out.append(_plain_rotate(z, cos, sin, st).to(x.dtype))
        if st["train"]:
            dz = _plain_rotate(st[up].float(), cos, -sin, st)
            if normed:
                dz, dw = _plain_norm_back(dz, n, inv, weight)
                dws.append(dw.to(x.dtype))
            grads.append(dz.to(x.dtype))
    return (*out, *grads, *dws)


def _plain_places(st):
    """(sequence, position) of each new token."""
    if st["starts"] is None:
        b = torch.arange(st["batch"], device="cuda")
        return b, st["lengths"].long() - 1
    t = torch.arange(st["tokens"], device="cuda")
    starts = st["starts"].long()
    b = torch.searchsorted(starts, t, right=True) - 1
    return b, st["lengths"].long()[b] - starts[b + 1] + t


def _plain_append(st):
    b, pos = _plain_places(st)
    r, dt = st["rotary"], st["q"].dtype
    rows = st["table"][pos]
    cos, sin = rows[:, None, :r // 2], rows[:, None, r // 2:]
    q, k = st["q"].float(), st["k"].float()
    if st["normed"]:
        q = _plain_norm(q)[0] * st["q_weight"].float()
        k = _plain_norm(k)[0] * st["k_weight"].float()
    page, slot = st["pages"].long()[b, pos // st["page"]], pos % st["page"]
    st["k_cache"][page, slot] = _plain_rotate(k, cos, sin, st).to(dt)
    st["v_cache"][page, slot] = st["v"]
    return _plain_rotate(q, cos, sin, st).to(dt), st["k_cache"], st["v_cache"]


def _plain_attend(st):
    hq, hk, d, most, n = st["q_heads"], st["kv_heads"], st["dim"], st["most"], st["context"]
    batch, group = st["batch"], hq // hk
    b, pos = _plain_places(st)
    starts = torch.arange(batch + 1, device="cuda") if st["starts"] is None else st["starts"].long()
    count, length = (starts[1:] - starts[:-1])[:, None], st["lengths"].long()[:, None]
    i = torch.arange(most, device="cuda")
    j = torch.arange(n, device="cuda")
    # the new tokens of each sequence, filled up to the longest chunk, the heads of a group together
    q = st["q"].float()[(starts[:-1, None] + i).clamp(max=st["tokens"] - 1)].view(batch, most, hk, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, d)
    page = st["pages"].long()[:, j // st["page"]].clamp(min=0)
    k = st["k_cache"][page, j % st["page"]].float().permute(0, 2, 3, 1).contiguous()
    v = st["v_cache"][page, j % st["page"]].float().permute(0, 2, 1, 3).contiguous()
    s = (q @ k) * (1.0 / math.sqrt(d))
    if st["softcap"] > 0:
        s = st["softcap"] * torch.tanh(s / st["softcap"])
    at = (length - count + i)[:, :, None]
    seen = (j <= at) & (j < length[:, :, None])
    if st["window"]:
        seen = seen & (j > at - st["window"])
    s = s.view(batch, hk, group, most, n).masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = (e.view(batch, hk, group * most, n) @ v).view(batch, hk, group, most, d) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, d)
    first = starts[:-1][b]
    return o[b, torch.arange(st["tokens"], device="cuda") - first].to(st["q"].dtype)


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _own_heads(st):
    if st["op"] == "rotary":
        from kernels.hip.rotary import kernel_fn
        q, k = kernel_fn(st["q"], st["k"], st["table"], st["positions"], interleaved=st["interleaved"])
        leaves = (st["q"], st["k"])
    else:
        from kernels.hip.qk_norm_rotary import kernel_fn
        q, k = kernel_fn(st["q"], st["k"], st["q_weight"], st["k_weight"], st["table"], st["positions"], eps=_EPS,
                         interleaved=st["interleaved"])
        leaves = (st["q"], st["k"], st["q_weight"], st["k_weight"])
    if not st["train"]:
        return q, k
    return (q, k, *torch.autograd.grad((q, k), leaves, (st["g_q"], st["g_k"])))


def _own_append(st):
    from kernels.hip.paged_append import kernel_fn
    q = kernel_fn(st["k"], st["v"], st["k_cache"], st["v_cache"], st["pages"], st["lengths"], st["starts"], q=st["q"],
                  q_weight=st.get("q_weight"), k_weight=st.get("k_weight"), eps=_EPS, table=st["table"],
                  interleaved=st["interleaved"])
    return q, st["k_cache"], st["v_cache"]


def _own_attend(st):
    from kernels.hip.paged_attention import kernel_fn
    return kernel_fn(st["q"], st["k_cache"], st["v_cache"], st["pages"], st["lengths"], st["starts"],
                     softcap=st["softcap"], window=st["window"], max_chunk=st["most"])


def run(state):
    op = state["op"]
    if own:
        return {"rotary": _own_heads, "norm": _own_heads, "append": _own_append, "attend": _own_attend}[op](state)
    return {"rotary": _plain_heads, "norm": _plain_heads, "append": _plain_append, "attend": _plain_attend}[op](state)


def work(case):
    e, hq, hk, d = _SIZE[case["dtype"]], case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("rotary", "norm"):
        tokens = case["batch"] * case["seq"]
        x = tokens * (hq + hk) * d * e
        table = (tokens if case["far"] else case["seq"]) * case["rotary"] * 4
        passes = 2 if not case["train"] else 4 if case["op"] == "rotary" else 5
        each = 3 if case["op"] == "rotary" else 8
        return {"bytes": passes * x + table, "flops": (3 if case["train"] else 1) * each * tokens * (hq + hk) * d}
    lengths, counts = _layout(case)
    tokens = sum(counts)
    if case["op"] == "append":
        return {"bytes": tokens * (2 * (hq + 2 * hk) * d * e + 4 * case["rotary"]),
                "flops": (11 if case["normed"] else 3) * tokens * (hq + hk) * d}
    window = case["window"] or case["context"]
    keys = pairs = 0
    for n, c in zip(lengths, counts):
        keys += n - max(0, n - c + 1 - window)  # from the first key that the first new token sees
        full = max(0, min(c, n - window))  # tokens that see a whole window
        pairs += full * window + sum(min(n - i, window) for i in range(full, c))
    return {"bytes": 2 * keys * hk * d * e + 2 * tokens * hq * d * e, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------
# In 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_pairs(case):
    """The indices of the two elements of each rotated pair."""
    i = torch.arange(case["rotary"] // 2, device="cuda")
    return (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + case["rotary"] // 2)


def _exact_turn(x, angle, case, back=False):
    """x [tokens, heads, dim] turned by the angles [tokens, rotary / 2]: products of complex numbers."""
    first, second = _exact_pairs(case)
    z = torch.complex(x[..., first], x[..., second])
    z = z * torch.polar(torch.ones_like(angle), -angle if back else angle)[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rms(x, w):
    return x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * w


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("rotary", "norm"):
            return _exact_heads(case, st)
        if case["op"] == "append":
            return _exact_append(case, st)
        return _exact_attend(case, st)


def _exact_heads(case, st):
    b, s = case["batch"], case["seq"]
    positions = st["positions"] if st["positions"] is not None else torch.arange(s, device="cuda").expand(b, s)
    angle = _angles(case, positions.reshape(-1))
    outs, grads, weights = [], [], []
    for x, up, w in (("q", "g_q", "q_weight"), ("k", "g_k", "k_weight")):
        shape = st[x].shape
        x = st[x].double().reshape(b * s, *shape[2:])
        wd = st[w].double() if case["op"] == "norm" else None
        z = x if wd is None else _exact_rms(x, wd)
        outs.append(_exact_turn(z, angle, case).view(shape))
        if case["train"]:
            dz = _exact_turn(st[up].double().reshape(x.shape), angle, case, back=True)
            if wd is not None:
                # d/dx of x / rms: the identity less the projection on x, over rms
                rms = torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + _EPS)
                weights.append((dz * x / rms).sum((0, 1)))
                g = dz * wd
                dz = g / rms - x * (g * x).sum(-1, keepdim=True) / (x.shape[-1] * rms ** 3)
            grads.append(dz.view(shape))
    return (*outs, *grads, *weights)


def _exact_append(case, st):
    lengths, counts = _layout(case)
    k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    if case["normed"]:
        q, k = _exact_rms(q, st["q_weight"].double()), _exact_rms(k, st["k_weight"].double())
    done, at = [], 0
    for i, (n, c) in enumerate(zip(lengths, counts)):
        pos = torch.arange(n - c, n, device="cuda")
        angle = _angles({**case, "factor": 1.0}, pos)
        flat = st["pages"][i].long()[pos // case["page"]] * case["page"] + pos % case["page"]
        k_cache.flatten(0, 1)[flat] = _exact_turn(k[at:at + c], angle, case)
        v_cache.flatten(0, 1)[flat] = v[at:at + c]
        done.append(_exact_turn(q[at:at + c], angle, case))
        at += c
    return torch.cat(done), k_cache, v_cache


def _exact_attend(case, st):
    lengths, counts = _layout(case)
    hk, d = case["kv_heads"], case["dim"]
    done, at = [], 0
    for i, (n, c) in enumerate(zip(lengths, counts)):
        pages = st["pages"][i, :-(-n // case["page"])].long()
        keys = st["k_cache"][pages].flatten(0, 1)[:n].double()
        values = st["v_cache"][pages].flatten(0, 1)[:n].double()
        p = torch.arange(n - c, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden |= j <= p - case["window"]
        heads = []
        for h in range(case["q_heads"]):
            own_kv = h * hk // case["q_heads"]
            s = st["q"][at:at + c, h].double() @ keys[:, own_kv].t().contiguous() / math.sqrt(d)
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            heads.append(torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ values[:, own_kv].contiguous())
        done.append(torch.stack(heads, 1))
        at += c
    return torch.cat(done)
