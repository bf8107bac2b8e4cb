"""GPU tests of the scoring operators where their rules at the edges decide:
ignored rows, saturated softcaps, masks of infinities and lowest values, log
probabilities at their bound, autocast, forward mode, torch.compile, many rows.

Tolerances are those of the row and head tests, whose derivation stands there;
what is added here is derived at its test.
"""

import math

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from oracle import scoring
from test_gpu_lmhead_logprobs import HALF, check, operands
from test_gpu_scoring import (DEV, DTYPES, ROW, TINY, U, check_distill, check_logprobs, close, grad_tol, logits_of,
                              special_rows, teacher_of)

pytestmark = gpu


# ---------------------------------------------------------------------------
# Autocast
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("inside", [True, False])
def test_head_in_fp32_under_autocast(inside):
    """fp32 operands keep their type under autocast: logits, and the gradient's
    logits formed again, are fp32 whether the backward runs inside or after."""
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn
    say("head fp32 autocast", inside)
    h, w, t = (a.to(DEV) for a in operands(70, 1001, 48, torch.float32, 4))
    h.requires_grad_()
    w.requires_grad_()

    def loss():
        r = kernel_fn(h, w, t, softcap=20.0)
        return r, r.logprobs.sum() + 0.3 * r.entropy.sum()

    r, total = loss()
    want = [*r, *torch.autograd.grad(total, (h, w))]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        r, total = loss()
        if inside:
            got = torch.autograd.grad(total, (h, w))
    if not inside:
        got = torch.autograd.grad(total, (h, w))
    assert all(torch.equal(a, b) for a, b in zip([*r, *got], want))


# ---------------------------------------------------------------------------
# Saturated softcaps
# ---------------------------------------------------------------------------
def saturated(n, dtype, sign):
    """Hidden states and weights whose logits are sign * (38, 38.25, ..., 53.75) on
    vocab rows 0..63 and small elsewhere: with a cap of 1, exp(2 z) leaves fp32."""
    h, w, t = operands(n, 300, 64, dtype, 17, scale=0.5)
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    w[:64] = 0.0
    w[:64, 0] = sign * (38.0 + 0.25 * torch.arange(64.0))
    t[:] = torch.arange(n) % 64
    return h, w, t


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("n", [5, 300])
@pytest.mark.parametrize("sign", [1, -1])
def test_head_gradients_of_saturated_caps(dtype, n, sign):
    """The cap's slope goes to e^-108 without passing an infinity on the way."""
    need_gpu()
    say("saturated", dtype, n, sign)
    check(*saturated(n, dtype, sign), 1.0, 1.0)


@pytest.mark.parametrize("n", [5, 300])
@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_loss_gradients_of_saturated_caps(dtype, n):
    """The same of the head's loss: dz = (p - [target]) / n (1 - tanh^2), within one
    rounding of the type and 2e-6 of the scale 1 / n, as its other tests."""
    need_gpu()
    from kernels.hip import _lib
    from kernels.hip.chunked_linear_cross_entropy import ChunkedLinearCrossEntropyLoss, lmhead_ce_forward
    say("saturated loss", dtype, n)
    for sign, size in ((1, 1.0), (-1, 1.0), (1, 16.0)):  # (and far past the range)
        h, w, t = saturated(n, dtype, sign)
        w[:64] *= size
        hd, wd, td = h.to(DEV), w.to(DEV), t.to(DEV)
        _, lse, nv = lmhead_ce_forward(hd, wd, td, softcap=1.0)
        dz = torch.empty(n, 300, dtype=dtype, device=DEV)
        _lib.lmhead_ce_bwd(hd, wd, td, lse, torch.ones(1, device=DEV), nv.float(), dz, -100, 1.0)
        x = h.double() @ w.double().t()
        p = torch.softmax(torch.tanh(x), 1)
        p[torch.arange(n), t] -= 1
        ref = p / torch.cosh(x.clamp(-300, 300)) ** 2 / n
        got = dz.double().cpu()
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2e-6 / n + TINY[dtype]
        assert bool(((got - ref).abs() <= tol).all())
        hl, wl = hd.clone().requires_grad_(), wd.clone().requires_grad_()
        gh, gw = torch.autograd.grad(ChunkedLinearCrossEntropyLoss(softcap=1.0)(hl, wl, td), (hl, wl))
        assert bool(torch.isfinite(gh).all()) and bool(torch.isfinite(gw).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_row_gradients_of_saturated_caps(dtype):
    """The slope keeps its relative accuracy down to the smallest normal number: with
    the given token beside the cap, dx = (1 - p) 4 e^-2a, a = x / cap up to 43; the
    exponent 2 a is rounded to u of it, 43 * 2 u < ROW."""
    need_gpu()
    from kernels.hip.token_logprobs import kernel_fn
    say("row slopes", dtype)
    a = torch.arange(30.0, 43.0, 0.25)
    x = torch.zeros(len(a), 700)
    x[:, 5] = a
    t = torch.full((len(a),), 5)
    leaf = x.to(dtype).to(DEV).requires_grad_()
    (g,) = torch.autograd.grad(kernel_fn(leaf, t.to(DEV), softcap=1.0).logprobs.sum(), leaf)
    ref, size = scoring.logprob_grad_rows(x.to(dtype), t, torch.ones(len(a)), None, 1.0, 1.0)
    close(g, ref, (2 * ROW + torch.finfo(dtype).eps / 2) * size * 1.001 + TINY[dtype] + 1e-45, "gradient")


# ---------------------------------------------------------------------------
# Ignored rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("every", [3, 1])
def test_head_ignored_rows_hold_anything(n, softcap, every):
    """Ignored rows of NaN, of infinities and of finite values whose logits pass
    fp32: results and hidden states' gradients 0, everything else as without them.
    ``every``: every third row, or a run of rows in front."""
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn
    say("head ignored", n, softcap, every)
    h, w, t = operands(n, 1153, 64, torch.bfloat16, 23)
    gone = torch.zeros(n, dtype=torch.bool)
    gone[::3] = every == 3
    gone[:n // 3] |= every == 1
    t[1:4] = 7
    t[gone] = -100
    at = gone.nonzero().flatten()
    up = torch.randn(2, n, generator=torch.Generator().manual_seed(2)).to(DEV)

    def run(h, need_w):
        hl, wl = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(need_w)
        r = kernel_fn(hl, wl, t.to(DEV), temperature=0.7, softcap=softcap)
        return [*r, *torch.autograd.grad([r.logprobs, r.entropy], [hl, wl][:1 + need_w], list(up))]

    calm = h.clone()
    calm[at] = 0.0
    want = run(calm, True)
    assert all(bool(torch.isfinite(a).all()) for a in want)
    past = h.clone()  # finite, with logits of either infinity and of both at once
    past[at] = 3e38 * h[at].sign().where(h[at] != 0, torch.ones((), dtype=h.dtype))
    wild = h.clone()
    wild[at[::2]] = math.nan
    wild[at[1::2]] = math.inf
    for x, need_w in ((past, True), (wild, False)):
        got = run(x, need_w)
        assert bool((got[0][at] == 0).all()) and bool((got[1][at] == 0).all()) and bool((got[2][at] == 0).all())
        # the other rows' tiles do not see them; the weight's gradient has zeros of them
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# Log probabilities are at most 0
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("n", [64, 512])
@pytest.mark.parametrize("temperature", [1e-3, 0.02, 1.0])
def test_head_log_probabilities_are_at_most_zero(dtype, n, temperature):
    """The given token holds all of the row: its own dot product and the tiles' logits
    differ by their roundings, divided by the temperature."""
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn
    say("head bound", dtype, n, temperature)
    h, w, _ = operands(n, 600, 832, dtype, 29, scale=12.0)
    t = (h.double() @ w.double().t()).argmax(1)
    lp = kernel_fn(h.to(DEV), w.to(DEV), t.to(DEV), temperature=temperature).logprobs
    assert bool((lp <= 0).all()), float(lp.max())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [40, 300])
def test_row_log_probabilities_are_at_most_zero(dtype, rows):
    """The same with a softcap, whose tanh the sums take in a shorter form."""
    need_gpu()
    from kernels.hip.token_logprobs import kernel_fn
    say("row bound", dtype, rows)
    x = logits_of(rows, 3001, dtype, 33)
    x[:, 11] = 20.0 + 0.125 * torch.arange(rows, device=DEV)
    t = torch.full((rows,), 11, device=DEV)
    for temperature in (0.01, 0.3):
        r = kernel_fn(x, t, temperature=temperature, softcap=30.0, top_k=2)
        assert bool((r.logprobs <= 0).all()) and bool((r.top_logprobs <= 0).all()), float(r.logprobs.max())
        assert bool((kernel_fn(x, t, temperature=temperature, softcap=30.0).logprobs <= 0).all())


# ---------------------------------------------------------------------------
# Infinities and lowest values
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,vocab,live", [(5, 700, 3), (300, 700, 3), (300, 1024, 200), (300, 1153, 600), (260, 600, 599)])
def test_head_softcap_of_infinite_logits(n, vocab, live):
    """A logit of -inf is -softcap, wherever its column is in a tile. The live tokens'
    logits are 0, so with k = V - live capped ones s = live + k e^(-cap / T)."""
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn
    say("head capped -inf", n, vocab, live)
    g = torch.Generator().manual_seed(8)
    w = torch.zeros(vocab, 64, dtype=torch.bfloat16)
    w[:, 0] = -1e30
    at = torch.randperm(vocab, generator=g)[:live]
    w[at, 0] = 0.0
    h = torch.zeros(n, 64, dtype=torch.bfloat16)
    h[:, 0] = 1e30
    t = at[torch.randint(0, live, (n,), generator=g)]
    t[::2] = (w[:, 0] != 0).nonzero().flatten()[torch.randint(0, vocab - live, (len(t[::2]),), generator=g)]
    x = torch.where(w[:, 0] == 0, 0.0, -math.inf).double().expand(n, vocab)
    lp, ent = scoring.logprob_rows(x, t, 2.0, 3.0)
    r = kernel_fn(h.to(DEV), w.to(DEV), t.to(DEV), temperature=2.0, softcap=3.0)
    tol = ROW + 2 * 8 * U * 3.0 / 2.0
    close(r.logprobs, lp, tol + 4 * U * lp.abs(), "logprobs")
    close(r.entropy, ent, tol * (1 + 2 * math.log(vocab)), "entropy")
    # saturated: no gradient but of the live tokens' columns
    wl = w.to(DEV).requires_grad_()
    (gw,) = torch.autograd.grad(kernel_fn(h.to(DEV), wl, t.to(DEV), temperature=2.0, softcap=3.0).entropy.sum(), wl)
    assert bool((gw[(w[:, 0] != 0).to(DEV)] == 0).all()) and bool(torch.isfinite(gw).all())


@pytest.mark.parametrize("n", [6, 70, 300])
@pytest.mark.parametrize("temperature", [0.25, 1.0])
def test_head_masks_of_the_lowest_value(n, temperature):
    """A constant hidden feature and a weight column of bf16's lowest value mask most of
    the vocabulary with finite logits of -3.39e38, whole tiles of it, as -inf does;
    a row of which every logit is that value is uniform."""
    need_gpu()
    from kernels.hip import _lib
    from kernels.hip.lmhead_logprobs import kernel_fn
    say("head lowest", n, temperature)
    h, w, t = operands(n, 1153, 64, torch.bfloat16, 31)
    low = torch.finfo(torch.bfloat16).min
    h[:, :2], w[:, :2] = 0.0, 0.0
    keep = torch.zeros(1153, dtype=torch.bool)
    keep[[3, 400, 401, 1150]] = True
    h[:, 0] = 1.0
    w[~keep, 0] = low
    w[:, 1] = low
    h[2] = 0.0
    h[2, 1] = 1.0  # nothing left: uniform
    t[:] = torch.tensor([3, 400, 401, 1150])[torch.arange(n) % 4]
    t[3] = 9       # masked
    x = h.double() @ w.double().t()
    lp, ent = scoring.logprob_rows(x, t, temperature)
    hd, wd, td = h.to(DEV), w.to(DEV), t.to(DEV)
    r = kernel_fn(hd, wd, td, temperature=temperature)
    terr = (72 * U * 40 + 2 * U * 40) / temperature  # (the kept logits are sums of |h w| below 40)
    assert float((h[:, 2:].double().abs() @ w[:, 2:].double().abs().t()).max()) < 40
    far = lp < -1e30
    assert far.tolist() == [i == 3 for i in range(n)] and float(r.logprobs[3]) < -1e37
    close(r.logprobs.cpu()[~far], lp[~far], ROW + 2 * terr + 4 * U * lp[~far].abs(), "logprobs")
    close(r.entropy, ent, (ROW + 2 * terr) * (1 + 2 * math.log(1153)), "entropy")
    # the logits' gradient
    f = lambda *s: torch.empty(*s, device=DEV)
    lp2, ent2, st, co = f(n), f(n), f(n, 4), f(n, 4)
    up = torch.randn(2, n, generator=torch.Generator().manual_seed(1))
    dz = torch.zeros(n, 1280, dtype=torch.bfloat16, device=DEV)[:, :1153]
    _lib.lmhead_logprobs(hd, wd, td, lp2, ent2, st, temperature, 0.0, -100)
    _lib.lmhead_logprobs_coefs(td, st, up[0].to(DEV), up[1].to(DEV), co, 1153, temperature, -100)
    _lib.lmhead_logprobs_bwd_range(hd, wd, td, co, dz, 0, temperature, 0.0, -100)
    assert torch.equal(lp2, r.logprobs) and torch.equal(ent2, r.entropy)
    ref, size = scoring.logprob_grad_rows(x, t, up[0], up[1], temperature)
    # ln p and H are off by absolute amounts too (as in the head's other tests)
    p = torch.softmax(scoring.scores(x, temperature), 1)
    tol = size * (4 * terr + 2 * ROW)
    tol = tol + p * up[1].abs()[:, None] * (ROW + 2 * terr) * (2 + 2 * math.log(1153)) / temperature
    tol = tol + 1.01 * torch.finfo(dz.dtype).eps / 2 * ref.abs() + 2.0 ** -120
    close(dz, ref, tol, "gradient")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [40, 3001, 40007])
def test_special_rows_with_a_softcap(dtype, vocab):
    """Under a softcap infinities are logits of +-softcap, a row of -inf alone is
    uniform; NaN stay NaN."""
    need_gpu()
    say("special capped", dtype, vocab)
    x = special_rows(vocab, dtype)
    tok = torch.randint(0, vocab, (14,), generator=torch.Generator().manual_seed(2))
    tok[1], tok[2], tok[5] = vocab // 2, vocab - 1, -100
    r = check_logprobs(x.to(DEV), tok.to(DEV), 0.8, 7.0, top_k=min(20, vocab))
    assert bool(torch.isfinite(r.entropy[[0, 1, 2, 3, 4, 6, 8, 9, 10, 11, 12]]).all())
    many = x.repeat(20, 1).to(DEV)
    from kernels.hip.token_logprobs import kernel_fn
    whole = kernel_fn(many, tok.repeat(20).to(DEV), temperature=0.8, softcap=7.0)
    lp, h = scoring.logprob_rows(x, tok, 0.8, 7.0)
    close(whole.logprobs[-14:], lp, 2 * ROW + 4 * U * torch.nan_to_num(lp.abs()), "logprobs")
    close(whole.entropy[-14:], h, 2 * ROW * (1 + 2 * math.log(vocab)), "entropy")
    ids = torch.stack([torch.randperm(vocab, generator=torch.Generator().manual_seed(4))[:6] for _ in range(14)])
    t = torch.randn(14, 6, generator=torch.Generator().manual_seed(5))
    ids[8, 2], t[9, 1], t[12] = vocab, math.nan, -math.inf
    check_distill(x.to(DEV), t.to(DEV), ids.to(DEV), 1.5, 7.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_softcaps_that_temperatures_leave_without_digits(dtype):
    """The cap's tanh is within 2^-22: up to 2^20 temperatures of it the scores keep
    digits, and past that the calls are refused."""
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn as head
    from kernels.hip.token_logprobs import kernel_fn as logprobs
    from kernels.hip.topk_distillation import kernel_fn as distill
    say("cap and temperature", dtype)
    x = logits_of(9, 1500, dtype, 31)
    t = torch.randint(0, 1500, (9,), generator=torch.Generator().manual_seed(5)).to(DEV)
    check_logprobs(x, t, 30 * 2.0 ** -20, 30.0, grads=False)
    tv, ti = teacher_of(x, 20, 6)
    h = torch.randn(9, 64, device=DEV).to(dtype)
    for cap, temperature in ((1e4, 1e-3), (30.0, 1e-18), (30.0, 2.0 ** -16)):
        with pytest.raises(ValueError, match="softcap"):
            logprobs(x, t, softcap=cap, temperature=temperature)
        with pytest.raises(ValueError, match="softcap"):
            distill(x, tv, ti, softcap=cap, temperature=temperature)
    with pytest.raises(ValueError, match="softcap"):
        head(h, torch.randn(1500, 64, device=DEV).to(dtype), t, softcap=1e4, temperature=1e-3)


# ---------------------------------------------------------------------------
# Forward mode, torch.compile, many rows
# ---------------------------------------------------------------------------
def entry_points():
    from kernels.hip import lmhead_logprobs, token_logprobs, topk_distillation
    g = torch.Generator().manual_seed(1)
    x = (3 * torch.randn(2, 5, 301, generator=g)).to(DEV)
    t = torch.randint(0, 301, (2, 5), generator=g).to(DEV)
    t[0, 1] = -100
    tv, ti = torch.randn(2, 5, 20, generator=g).to(DEV), torch.randint(0, 301, (2, 5, 20), generator=g).to(DEV)
    h, w = torch.randn(2, 5, 128, generator=g).to(DEV), (0.1 * torch.randn(301, 128, generator=g)).to(DEV)
    head = lambda h, w: lmhead_logprobs.kernel_fn(h, w, t, softcap=30.0)
    return {
        "logprobs": ((x,), lambda x: token_logprobs.kernel_fn(x, t, temperature=0.7, top_k=9)[:2]),
        "distill": ((x.bfloat16(),), lambda x: [topk_distillation.kernel_fn(x, tv, ti, temperature=2.0)]),
        "head": ((h.bfloat16(), w.bfloat16()), head),
        "head fp32": ((h, w), head),
    }


@pytest.mark.parametrize("name", ["logprobs", "distill", "head", "head fp32"])
def test_forward_mode_is_refused(name):
    need_gpu()
    import torch.autograd.forward_ad as fw
    leaves, fn = entry_points()[name]
    say("forward mode", name)
    for i in range(len(leaves)):
        for grad_mode in (True, False):
            with fw.dual_level(), torch.set_grad_enabled(grad_mode):
                args = list(leaves)
                args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(*args)
    out = fn(*[a.requires_grad_() for a in leaves])[0]
    with fw.dual_level():
        up = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            out.backward(up)


@pytest.mark.parametrize("name", ["logprobs", "distill", "head", "head fp32"])
def test_under_torch_compile(name):
    need_gpu()
    import torch._dynamo
    import torch._dynamo.compiled_autograd as compiled
    leaves, fn = entry_points()[name]
    say("compile", name)
    leaves = [a.requires_grad_() for a in leaves]
    outs = fn(*leaves)
    want = [*outs, *torch.autograd.grad(sum(o.sum() for o in outs), leaves)]
    torch._dynamo.reset()
    outs = torch.compile(fn, backend="eager")(*leaves)
    got = [*outs, *torch.autograd.grad(sum(o.sum() for o in outs), leaves)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    total = sum(o.sum() for o in fn(*leaves))
    with compiled._enable(torch.compile(backend="eager")):
        total.backward()
    torch._dynamo.reset()
    for a, b in zip(leaves, want[len(outs):]):
        assert torch.equal(a.grad, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_more_rows_than_workgroups(dtype):
    """2^20 + 3 rows of a small vocabulary, and the last ones checked."""
    need_gpu()
    from kernels.hip.token_logprobs import kernel_fn as logprobs
    from kernels.hip.topk_distillation import kernel_fn as distill
    say("many rows", dtype)
    n = (1 << 20) + 3
    g = torch.Generator(device=DEV).manual_seed(3)
    x = (2 * torch.randn(n, 8, generator=g, device=DEV)).to(dtype).requires_grad_()
    t = torch.randint(0, 8, (n,), generator=g, device=DEV)
    t[::5] = -100
    r = logprobs(x, t, top_k=3)
    part = slice(n - 9, n)
    xc, tc = x.detach()[part].cpu(), t[part].cpu()
    lp, h = scoring.logprob_rows(xc, tc)
    tv, ti = scoring.top_rows(xc, 3)
    close(r.logprobs[part], lp, ROW + 4 * U * lp.abs(), "logprobs")
    close(r.entropy[part], h, ROW * (1 + 2 * math.log(8)), "entropy")
    close(r.top_logprobs[part], tv, ROW + 4 * U * tv.abs(), "top_logprobs")
    assert torch.equal(r.top_ids[part].cpu(), ti)
    assert torch.equal(logprobs(x, t).logprobs, r.logprobs) and torch.equal(r.logprobs == 0, t == -100)
    (gx,) = torch.autograd.grad(r.logprobs.sum() + 0.5 * r.entropy.sum(), x)
    ref, size = scoring.logprob_grad_rows(xc, tc, torch.ones(9), 0.5 * torch.ones(9))
    close(gx[part], ref, grad_tol(ref, size, dtype, 1.0, 0.0), "gradient")
    ids, tl = torch.randint(0, 8, (n, 2), generator=g, device=DEV), torch.randn(n, 2, generator=g, device=DEV)
    losses = distill(x, tl, ids, reduction="none")
    want, _, _ = scoring.distill_rows(xc, tl[part].cpu(), ids[part].cpu())
    close(losses[part], want, 2 * ROW + 24 * U * (1 + math.log(8) + 2 * xc.double().abs().amax(1)), "losses")
    (gx,) = torch.autograd.grad(losses.sum(), x)
    ref, size = scoring.distill_grad_rows(xc, tl[part].cpu(), ids[part].cpu(), torch.ones(9))
    close(gx[part], ref, 2 * grad_tol(ref, size, dtype, 1.0, 0.0), "distillation gradient")


def test_head_fp32_beyond_one_chunk():
    need_gpu()
    say("head fp32 chunks")
    check(*operands(1100, 301, 40, torch.float32, 6), 1.2)
