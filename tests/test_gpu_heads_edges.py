"""Edges of the operators on attention heads and the paged cache on the GPU."""

import math

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from heads_util import E, attend_bound, close, half_eps, make_batch, partner_abs, tiny, turn_bound
from oracle import heads as oracle

pytestmark = gpu
DEV = "cuda"


def serving_call(seed=21):
    """A small call of both cache operators: (append's arguments, attention's tensors)."""
    g = torch.Generator().manual_seed(seed)
    pages, lens, starts, total = make_batch([3, 2], [7, 2], 4, seed)
    k, v, q = (torch.randn(5, h, 64, generator=g) for h in (2, 2, 4))
    kc, vc = (torch.randn(total, 4, 2, 64, generator=g) for _ in range(2))
    return {n: t.to(DEV) for n, t in dict(k=k, v=v, k_cache=kc, v_cache=vc, page_table=pages, lengths=lens, starts=starts,
                                          q=q).items()}


@pytest.mark.parametrize("recorded", [True, False])
def test_serving_refuses_forward_mode(recorded):
    need_gpu()
    import torch.autograd.forward_ad as fw
    from kernels.hip import paged_append, paged_attention
    say("serving, forward mode", recorded)
    c = serving_call()
    attend = {n: t for n, t in c.items() if n not in ("k", "v")}
    for fn, args, names in ((paged_append.kernel_fn, c, ("k", "v", "k_cache", "v_cache", "q")),
                            (paged_attention.kernel_fn, attend, ("q", "k_cache", "v_cache"))):
        for name in names:
            with fw.dual_level(), torch.set_grad_enabled(recorded):
                dual = fw.make_dual(args[name], torch.ones_like(args[name]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(**{**args, name: dual})


# ---------------------------------------------------------------------------
# Attention at its edges
# ---------------------------------------------------------------------------
def one_hot_call(scores, dtype, dim, tokens=1, heads=(2, 1), page=16, seed=22):
    """A call of one sequence whose key j has the score scores[j] in every row, exactly: the
    queries are 1 in their first element alone, where the keys hold their score (scale 1).
    Returns (arguments, values [keys, kv heads, dim] that the caller may overwrite)."""
    g = torch.Generator().manual_seed(seed)
    n = len(scores)
    pages, lens, starts, total = make_batch([tokens], [n], page, seed)
    q = torch.zeros(tokens, heads[0], dim, dtype=dtype)
    q[..., 0] = 1.0
    kc = torch.zeros(total, page, heads[1], dim, dtype=dtype)
    vc = torch.randn(total, page, heads[1], dim, generator=g).to(dtype)
    j = torch.arange(n)
    at = pages[0, j // page].long(), j % page
    kc[..., 0][at] = scores.to(dtype)[:, None]
    return [q, kc, vc, pages, lens, starts], at


def attend_on_gpu(args, **kw):
    from kernels.hip.paged_attention import kernel_fn
    return kernel_fn(*(t.to(DEV) for t in args), **kw)


@pytest.mark.parametrize("tokens, hint", [(1, 1), (1, 100), (40, 40)])
@pytest.mark.parametrize("below", [12.0, 15.0, 17.5])
def test_small_weights_of_fp16(below, tokens, hint):
    """One key far above n equal ones: their weights e^-below keep their digits in the product.

    Bound: a weight is rounded once, u = 2^-11 of it while it is normal in fp16; with the row's
    top at 2^11 or more, one below 2^-14 is off by half of 2^-24, 2^-36 of the top, and the top
    is at most the row's sum: 2^-36 sum |v| in all. The rest as in attend_bound; the scores are
    exact, the exponential's argument is within E |s - top| log2(e), its result within 2 E."""
    need_gpu()
    n, dim, dtype = 8192, 64, torch.float16
    say("small weights", below, tokens, hint)
    scores = torch.full((n,), -below)
    scores[3] = 0.0
    args, at = one_hot_call(scores, dtype, dim, tokens)
    args[2][at] = 100.0 + torch.arange(dim, dtype=dtype)  # (one row: every key's value)
    args[2][at[0][3], at[1][3]] = 0.0                     # the top key's
    got = attend_on_gpu(args, scale=1.0, max_chunk=hint)
    for head in range(2):
        for t in range(tokens):
            seen = n - tokens + t + 1
            w = (seen - 1) * math.exp(-below)
            want = (100.0 + torch.arange(dim, dtype=torch.float64)) * (w / (1.0 + w))
            mass = want
            rest = 2.0 ** -36 * seen * (100.0 + dim)
            bound = (2 * half_eps(dtype) + 2 * (2 * below + 8) * E + 2 * (n / 32 + 64) * E) * mass + rest + 2.0 ** -25
            close(got[t, head], want, bound, f"{below} {t} {head}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dim", [64, 66])
@pytest.mark.parametrize("tokens", [1, 70])
def test_scores_near_the_ends_of_fp32(tokens, dim, dtype):
    """Finite scores that leave fp32 in base 2 (beyond 2.36e38) are scores like others: equal
    ones share the row, the larger win alone (they differ by far more than exp's range), in
    every kernel, in whichever order and part they come. The mean of n equal weights carries
    its sums' roundings, each weight being the same number: (n / 32 + 64 + 4) E, and u of the
    result and of the 16-bit weight."""
    need_gpu()
    n = 1500
    low = torch.finfo(dtype).min
    for name, pick in (("all lowest", lambda s: s.fill_(low)),
                       ("all highest", lambda s: s.fill_(-low)),
                       ("the last above the lowest", lambda s: s.fill_(low).__setitem__(slice(900, 950), low * 0.75)),
                       ("the first above the lowest", lambda s: s.fill_(low).__setitem__(slice(3, 9), low * 0.75)),
                       ("ordinary ones beside the lowest", lambda s: s.fill_(low).__setitem__(slice(1000, 1003), 1.0)),
                       ("the highest beside ordinary ones", lambda s: s.fill_(1.0).__setitem__(slice(700, 720), -low)),
                       ("higher and higher", lambda s: s.fill_(-1.0).__setitem__(slice(40, 44), -low * 0.75)
                        or s.__setitem__(slice(1300, 1330), -low))):
        say(name, tokens, dim, dtype)
        scores = torch.zeros(n)
        pick(scores)
        args, at = one_hot_call(scores, dtype, dim, tokens)
        scores = scores.to(dtype).float()
        values = args[2][at][:, 0].double()
        for hint in (1, tokens):
            got = attend_on_gpu(args, scale=1.0, max_chunk=hint)
            for t in (0, tokens - 1):
                seen = n - tokens + t + 1
                s = scores[:seen]
                win = s == s.max()
                want = values[:seen][win].mean(0)
                mass = values[:seen][win].abs().mean(0)
                u = half_eps(dtype) if dtype != torch.float32 else 0.0
                bound = half_eps(dtype) * want.abs() + (u + 2 * (n / 32 + 68) * E) * mass
                for head in range(2):
                    close(got[t, head], want, bound, f"{name}, hint {hint}, row {t}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("scale", [1e-3, 0.69, 0.7, 1.0, 3.0])
def test_scales(scale, dtype):
    """Ordinary scores at scales on both sides of 1 / log2(e), cut among workers."""
    need_gpu()
    for counts, lengths, heads, dim in (([1, 1], [2500, 70], (4, 2), 64), ([70, 1], [901, 1500], (4, 2), 128), ([3], [600], (2, 1), 66)):
        say("scale", scale, counts, dtype)
        g = torch.Generator().manual_seed(25)
        pages, lens, starts, total = make_batch(counts, lengths, 16, 25)
        q = torch.randn(sum(counts), heads[0], dim, generator=g).to(dtype)
        kc, vc = (torch.randn(total, 16, heads[1], dim, generator=g).to(dtype) for _ in range(2))
        want, spread, reach, mass = oracle.attend(q, kc, vc, pages, lens, starts, scale, bounds=True)
        bound = attend_bound(want, spread, reach, mass, max(lengths), dim, dtype)
        if dtype == torch.float16:  # (weights below 2^-25 of the top, as above)
            bound = bound + 2.0 ** -36 * max(lengths) * float(vc.abs().max())
        for hint in (1, max(counts)):
            close(attend_on_gpu([q, kc, vc, pages, lens, starts], scale=scale, max_chunk=hint), want, bound, f"{scale} {counts} {hint}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim", [64, 66])
def test_values_that_are_not_finite_by_their_weights(dim, dtype):
    """A value that is not finite takes part by its weight, wherever its unit's border falls:
    an infinity times 0 (a score of -inf) is NaN, times a weight above 0 itself; rows that
    do not see its key do not see it."""
    need_gpu()
    n, page = 300, 16
    for tokens in (3, 100):
        for key in (5, n - 2):            # in a unit that all rows see; in one that only some see
            for value in (math.inf, -math.inf, math.nan):
                for score in (-math.inf, 0.0):
                    say("not finite", dim, dtype, tokens, key, value, score)
                    scores = torch.zeros(n)
                    scores[key] = score
                    args, at = one_hot_call(scores, dtype, dim, tokens, page=page)
                    want_clean = attend_on_gpu(args, scale=1.0, max_chunk=tokens)
                    args[2][at[0][key], at[1][key], 0, 7] = value
                    for hint in (1, tokens):
                        got = attend_on_gpu(args, scale=1.0, max_chunk=hint)
                        for t in range(tokens):
                            x = got[t, :, 7]
                            if n - tokens + t < key:
                                assert torch.isfinite(x).all()
                            elif score == 0.0 and not math.isnan(value):
                                assert (x == value).all(), (t, x)
                            else:
                                assert torch.isnan(x).all(), (t, x)
                        rest = [d for d in range(dim) if d != 7]
                        assert torch.isfinite(got[..., rest]).all()
                        if hint == tokens:
                            assert torch.equal(got[..., rest], want_clean[..., rest])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim", [64, 66])
@pytest.mark.parametrize("cap", [1.0, 30.0, 256.0, 300.0, 1e4])
def test_caps_keep_the_digits_of_scores(cap, dim, dtype):
    """The cap's error is relative to the score: x = s / cap within 2 E, tanh within 8 E, its
    product with the cap within 2 E: rho = 12 E |s|, and for fp16 with caps up to 256 and bf16
    besides an absolute one, 4 cap 2^-24 (the dot product is exact here). Then the exponential: its argument
    within 2 E (|s| + spread), its result within 4 E; a weight's error rho moves the quotient by
    2 rho sum p |v| at most. The two sums are chains of at most as many terms as keys are seen,
    64 and a 32nd of them, and the 8 of joining and dividing."""
    need_gpu()
    g = torch.Generator().manual_seed(23)
    for n, tokens, spread in ((600, 3, 10.0), (600, 3, 1e-3), (600, 3, 100.0), (4, 2, 4.0), (5, 3, 1.0), (6, 1, 3.0)):
        say("cap", cap, dim, dtype, n, spread)
        scores = (spread * (2 * torch.rand(n, generator=g) - 1)).to(dtype).float()
        args, at = one_hot_call(scores, dtype, dim, tokens)
        values = args[2][at][:, 0].double()
        for hint in (1, 100):
            got = attend_on_gpu(args, scale=1.0, softcap=cap, max_chunk=hint)
            for t in range(tokens):
                seen = n - tokens + t + 1
                s = cap * torch.tanh(scores[:seen].double() / cap)
                p = torch.softmax(s, 0)[:, None]
                want, mass = (p * values[:seen]).sum(0), (p * values[:seen].abs()).sum(0)
                size = float(s.abs().max())
                rho = 12 * E * size + 6 * E * size + 8 * E
                quick = dtype == torch.bfloat16 or (dtype == torch.float16 and cap <= 256)
                rho += 4 * cap * E if quick else 0.0
                u = half_eps(dtype) if dtype != torch.float32 else 0.0
                bound = half_eps(dtype) * want.abs() + (u + 2 * math.expm1(rho) + 2 * (seen / 32 + min(seen, 64) + 8) * E) * mass
                for head in range(2):
                    close(got[t, head], want, bound, f"cap {cap}, {n} scores to {spread}, hint {hint}, row {t}")


# ---------------------------------------------------------------------------
# Head norms at far scales
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["vectors", "pairs", "offset"])
@pytest.mark.parametrize("size", [3e-20, 1e-10, 1e18])
def test_norm_gradients_at_far_scales(size, layout):
    """eps 0, heads of far sizes, in rows of whole vectors and off them: gradients as large as
    the inverse of the heads. Squares near 1e-39 are below fp32's normal range and carry half
    of 2^-149 each, which is 8e-7 of the smallest sum here (64 times 9e-40), 4e-7 = 7 E of its root; the
    rest as in the norm's bound, 48 E, twice over for the two products, of the terms' sizes."""
    need_gpu()
    from kernels.hip.qk_norm_rotary import kernel_fn
    from kernels.hip.rotary import rotary_table
    g = torch.Generator().manual_seed(24)
    dim, rotary = (66, 22) if layout == "pairs" else (64, 64)
    say("far scales", size, layout)
    sign = torch.where(torch.rand(9, 3, dim, generator=g) < 0.5, -1.0, 1.0)
    x = size * sign * (1.0 + 0.5 * torch.rand(9, 3, dim, generator=g))
    up = torch.randn(9, 3, dim, generator=g)
    w = 1 + 0.1 * torch.randn(dim, generator=g)
    table = rotary_table(rotary, 16)
    xd = x.to(DEV)
    if layout == "offset":
        xd = torch.empty(x.numel() + 1, device=DEV)[1:].view(x.shape).copy_(xd)
    xd, wd = xd.requires_grad_(), w.to(DEV).requires_grad_()
    y, _ = kernel_fn(xd, None, wd, None, table.to(DEV), eps=0.0)
    dx, dw = torch.autograd.grad(y, (xd, wd), up.to(DEV))
    want, want_w = oracle.norm_turn_grad(x, w, 0.0, table, torch.arange(9), up)
    turned = partner_abs(up, rotary, False) * w.double().abs()
    inv = 1.0 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True))
    n = (x.double() * inv).abs()
    terms = inv * (turned + n * (turned * n).mean(-1, keepdim=True))
    close(dx, want, 128 * E * terms, "dx")
    close(dw, want_w, 128 * E * (partner_abs(up, rotary, False) * n).sum((0, 1)) + 1e-37, "dweight")


# ---------------------------------------------------------------------------
# Bad pages, lengths and starts write where they should and nowhere else
# ---------------------------------------------------------------------------
GUARD = 77.0


def guarded(t, lead=1, heads=1):
    """(a view that holds t, what surrounds it): t [n, .., heads, dim] inside a larger tensor of
    guards, `lead` rows and `heads` heads more on either side."""
    shape = list(t.shape)
    shape[0] += 2 * lead
    shape[-2] += 2 * heads
    buf = torch.full(shape, GUARD, dtype=t.dtype, device=DEV)
    view = buf[lead:lead + t.shape[0]][..., heads:heads + t.shape[-2], :]
    view.copy_(t)

    def untouched():
        rest = buf.clone()
        rest[lead:lead + t.shape[0]][..., heads:heads + t.shape[-2], :] = GUARD
        return bool((rest == GUARD).all())

    return view, untouched


BAD_APPENDS = [  # lengths, starts as given, ordered starts that mean the same (None: one token each)
    ([3, 3, 7, 2], None, None),
    ([9, -5, 2 ** 31 - 1, -2 ** 31], None, None),
    ([1, 1, 1, 1], [5, 9, -3, 100, 2 ** 31 - 1], [0, 0, 0, 4, 4]),
    ([8, 8, 8, 8], [3, 2, 1, 0, -1], [0, 0, 0, 0, 0]),
    ([2, 4, 1, 8], [1, 2, 2, 2, 3], [1, 2, 2, 2, 3]),
    ([2, 4, 8, 8], [0, 1, 4, 2 ** 31 - 1, 2 ** 31 - 1], [0, 1, 4, 4, 4]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dim", [64, 66])
@pytest.mark.parametrize("case", BAD_APPENDS, ids=str)
def test_bad_appends_stay_inside(case, dim, dtype):
    need_gpu()
    from kernels.hip import paged_append
    from kernels.hip.rotary import rotary_table
    lengths, starts, ordered = case
    say("bad append", case, dim, dtype)
    g = torch.Generator().manual_seed(26)
    k, v, q = (torch.randn(4, h, dim, generator=g).to(dtype) for h in (2, 2, 3))
    pages = torch.tensor([[9, 1], [-1, 0], [0, 2 ** 31 - 1], [-2 ** 31, 1]], dtype=torch.int32)
    table = rotary_table(dim - 2, 8)
    lens = torch.tensor(lengths, dtype=torch.int32)
    kc, vc = (torch.randn(2, 4, 2, dim, generator=g).to(dtype) for _ in range(2))
    kd, k_kept = guarded(kc)
    vd, v_kept = guarded(vc)
    qd, q_kept = guarded(torch.full_like(q, 5.0))
    st = None if starts is None else torch.tensor(starts, dtype=torch.int32)
    got = paged_append.kernel_fn(k.to(DEV), v.to(DEV), kd, vd, pages.to(DEV), lens.to(DEV), None if st is None else st.to(DEV),
                                 q=q.to(DEV), table=table.to(DEV), q_out=qd)
    assert got is qd and k_kept() and v_kept() and q_kept()
    so = None if ordered is None else torch.tensor(ordered, dtype=torch.int32)
    # (lengths near the ends of int32 are places past the table's width or before the first)
    want_q, want_k, want_v = oracle.append(q, k, v, kc, vc, pages, lens, so, None, None, 0.0, table, False)
    where = oracle.sequences(lengths, None if so is None else ordered, 4)
    none = torch.tensor([b < 0 for b, _ in where])
    want_q[none] = 5.0
    close(qd, want_q, turn_bound(want_q.nan_to_num(), q, dim - 2, False, dtype), "q")
    # (a place's turned key came from elements of at most the largest key's size)
    off = half_eps(dtype) * want_k.abs() + 4 * E * 2 * float(k.abs().max()) + tiny(dtype)
    close(kd, want_k, torch.where(want_k == kc.double(), 0.0, off), "k_cache")
    assert torch.equal(vd.cpu().double(), want_v)
    # without q_out the rows of no sequence are 0
    fresh = paged_append.kernel_fn(k.to(DEV), v.to(DEV), kd, vd, pages.to(DEV), lens.to(DEV), None if st is None else st.to(DEV),
                                   q=q.to(DEV), table=table.to(DEV))
    assert not fresh[none.to(DEV)].any() and k_kept() and v_kept()


BAD_STARTS = [  # as given, ordered starts that mean the same
    ([0, 50, 43], [0, 43, 43]),
    ([-9, 2 ** 31 - 1, 3], [0, 43, 43]),
    ([43, 0, 0], [0, 0, 0]),
    ([7, 7, 7], [7, 7, 7]),
    ([20, 30, 25], [20, 30, 30]),
    ([5, 6, 40], [5, 6, 40]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dim", [64, 66])
@pytest.mark.parametrize("case", BAD_STARTS, ids=str)
def test_bad_starts_of_attention_stay_inside(case, dim, dtype):
    """Rows that have a sequence are its attention, the others stay as they were or are 0, and
    nothing around the output is written."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    given, ordered = case
    say("bad starts", case, dim, dtype)
    g = torch.Generator().manual_seed(27)
    pages, lens, _, total = make_batch([3, 40], [90, 100], 16, 27)
    pages[0, 2], pages[1, 3] = -7, 2 ** 31 - 1
    q = torch.randn(43, 4, dim, generator=g).to(dtype)
    kc, vc = (torch.randn(total, 16, 2, dim, generator=g).to(dtype) for _ in range(2))
    args = [t.to(DEV) for t in (q, kc, vc, pages, lens, torch.tensor(given, dtype=torch.int32))]
    want, spread, reach, mass = oracle.attend(q, kc, vc, pages, lens, torch.tensor(ordered), 1 / math.sqrt(dim), bounds=True)
    bound = attend_bound(want, spread, reach, mass, 100, dim, dtype)
    none = torch.tensor([b < 0 for b, _ in oracle.sequences(lens.tolist(), ordered, 43)])
    for hint in (1, 43):
        out, kept = guarded(torch.full_like(q, 5.0))
        assert kernel_fn(*args, max_chunk=hint, out=out) is out and kept()
        assert (out[none.to(DEV)] == 5).all()
        close(out.cpu()[~none], want[~none], bound[~none], f"hint {hint}")
        fresh = kernel_fn(*args, max_chunk=hint)
        assert not fresh[none.to(DEV)].any() and torch.equal(fresh.cpu()[~none], out.cpu()[~none])


def test_lengths_past_the_table_are_cut():
    """Lengths past the page table's width: the token sees the positions that the table has."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 66)):
        say("long lengths", dtype, dim)
        g = torch.Generator().manual_seed(28)
        pages = torch.tensor([[2, 0, 1], [3, 4, 5]], dtype=torch.int32)
        q = torch.randn(2, 4, dim, generator=g).to(dtype)
        kc, vc = (torch.randn(6, 16, 2, dim, generator=g).to(dtype) for _ in range(2))
        want, spread, reach, mass = oracle.attend(q, kc, vc, pages, torch.tensor([48, 48]), None, 0.2, bounds=True)
        bound = attend_bound(want, spread, reach, mass, 48, dim, dtype)
        for lengths in ([2 ** 31 - 1, 49], [10 ** 6, 2 ** 31 - 1]):
            out, kept = guarded(torch.full_like(q, 5.0))
            kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages, torch.tensor(lengths, dtype=torch.int32))), scale=0.2, out=out)
            assert kept()
            close(out, want, bound, str(lengths))


def test_outputs_in_place_of_the_queries():
    """q_out and out may be the queries themselves, parts of a fused projection too; nothing else
    that a call reads or writes."""
    need_gpu()
    from kernels.hip import paged_append, paged_attention
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 66), (torch.float16, 128)):
        for counts, lengths in (([1] * 9, [700, 3, 90, 1, 65, 300, 2000, 16, 17]), ([90, 1, 40], [500, 900, 40])):
            say("in place", dtype, dim, len(counts))
            g = torch.Generator().manual_seed(29)
            pages, lens, starts, total = make_batch(counts, lengths, 16, 29)
            pages, lens, starts = pages.to(DEV), lens.to(DEV), starts.to(DEV)
            fused = torch.randn(sum(counts), 8, dim, generator=g).to(dtype).to(DEV)
            kc, vc = (torch.randn(total, 16, 2, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
            w = torch.ones(dim, dtype=dtype, device=DEV)

            def append(f, **kw):
                caches = kc.clone(), vc.clone()
                return paged_append.kernel_fn(f[:, 4:6], f[:, 6:], *caches, pages, lens, starts, q=f[:, :4], q_weight=w, k_weight=w,
                                              **kw), *caches

            fresh = append(fused)
            own = fused.clone()
            got = append(own, q_out=own[:, :4])
            assert all(torch.equal(a, b) for a, b in zip(got, fresh)) and torch.equal(own[:, 4:], fused[:, 4:])
            with pytest.raises(ValueError, match="q_out shares memory with k"):
                append(own, q_out=own[:, 4:])
            with pytest.raises(ValueError, match="q_out shares memory with q"):
                append(own, q_out=own[:, 1:5])
            want = paged_attention.kernel_fn(fused[:, :4], kc, vc, pages, lens, starts, max_chunk=max(counts))
            got = paged_attention.kernel_fn(own.copy_(fused)[:, :4], kc, vc, pages, lens, starts, max_chunk=max(counts), out=own[:, :4])
            assert torch.equal(got, want) and torch.equal(own[:, 4:], fused[:, 4:])
            with pytest.raises(ValueError, match="out shares memory with q"):
                paged_attention.kernel_fn(own[:, :4], kc, vc, pages, lens, starts, out=own[:, 2:6])
