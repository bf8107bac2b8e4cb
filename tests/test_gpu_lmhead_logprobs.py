"""GPU parity of the fused lm-head log probabilities against the float64 oracle.

Tolerances. A logit is an fp32 sum of d exact products of half-precision
values, of which Z below is the largest absolute partial sum's bound (sum of
|h w| over d): off by at most (d + 8) u Z, u = 2^-24 (the matrix cores' order is
not fixed, any order of d additions is within that). In the exponent the tile's
offset m c2 is rounded once: u |m| / T. Through the softmax a log probability
moves by at most twice the largest score's error, plus ROW as in the row
kernels (chains of at most 150 additions); entropies by that times 1 + 2 ln V.
The logits' gradient is rounded to the element type once, so a product's
entry is off by (eps / 2 + relative error of the terms) of the sum of its
terms' sizes, and once more by half a step of its own.
"""

import math

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from oracle import scoring
from test_gpu_scoring import ROW, U, close

pytestmark = gpu
DEV = "cuda"


def operands(n, vocab, d, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g).to(dtype)
    w = (torch.randn(vocab, d, generator=g) * (scale / math.sqrt(d))).to(dtype)
    t = torch.randint(0, vocab, (n,), generator=g)
    if n > 3:
        t[1], t[2], t[3] = -100, vocab - 1, 0
    return h, w, t


def check(h, w, t, temperature=1.0, softcap=0.0, grads=True):
    from kernels.hip.lmhead_logprobs import kernel_fn
    dtype, d = h.dtype, h.shape[1]
    x = h.double() @ w.double().t()
    z = float((h.double().abs() @ w.double().abs().t()).max())
    terr = ((d + 8) * U * z + 2 * U * float(x.abs().max()) + 8 * U * softcap) / temperature
    lnv = math.log(max(2, w.shape[0]))
    hd, wd = h.to(DEV), w.to(DEV)
    td = t.to(DEV) if t is not None else None
    kw = dict(temperature=temperature, softcap=softcap)
    r = kernel_fn(hd, wd, td, **kw)
    lp, ent = scoring.logprob_rows(x, t, temperature, softcap)
    if t is not None:
        close(r.logprobs, lp, ROW + 2 * terr + 4 * U * torch.nan_to_num(lp.abs()), "logprobs")
    close(r.entropy, ent, (ROW + 2 * terr) * (1 + 2 * lnv), "entropy")
    if not grads:
        return
    g = torch.Generator().manual_seed(1)
    gl = torch.randn(h.shape[0], generator=g) if t is not None else None
    ge = torch.randn(h.shape[0], generator=g)
    hl, wl = hd.clone().requires_grad_(), wd.clone().requires_grad_()
    r = kernel_fn(hl, wl, td, **kw)
    assert torch.equal(r.entropy, kernel_fn(hd, wd, td, **kw).entropy)
    for pair in ((gl, ge), (None, ge), (gl, None)):
        outs = [(o, u.to(DEV)) for o, u in zip(r, pair) if u is not None]
        if not outs:
            continue
        gh, gw = torch.autograd.grad([o for o, _ in outs], [hl, wl], [u for _, u in outs], retain_graph=True)
        dz, size = scoring.logprob_grad_rows(x, t, pair[0], pair[1], temperature, softcap)
        eps = torch.finfo(dtype).eps / 2
        # relative error of a term: its exponent's, and the chains' of lse and entropy; fp16 also steps of its subnormals
        rel = 4 * terr + 2 * ROW
        term = dz.abs() * eps + size * rel + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        # the hardware exponential is 0 below fp32's smallest normal number: a term
        # p (g + e (ln p + H)) / T with p < 2^-126 is lost whole; p |ln p| rises with p
        # there, so it is at most 2^-126 (|g| + |e| (88 + ln V)) / T, 88 > 126 ln 2. (At
        # T = 0.01 three rows of the vocab have their largest p at 2^-127, 2^-130, 2^-134.)
        gsum = sum(u.abs() * f for u, f in ((pair[0], 1.0), (pair[1], 88.0 + lnv)) if u is not None)
        term = term + (gsum * 2.0 ** -126 / temperature).double()[:, None]
        if pair[1] is not None:
            # -e p (ln p + H): ln p and H are off by absolute amounts (the tolerances above),
            # also where both are 0 and the term's size with them (one token holding all)
            counted = torch.ones(h.shape[0]) if t is None else (t != -100).double()
            p = torch.softmax(scoring.scores(x, temperature, softcap), 1)
            term = term + (counted * pair[1].abs())[:, None] * p * (ROW + 2 * terr) * (2 + 2 * lnv) / temperature
        for got, ref, err in ((gh, dz @ w.double(), term @ w.double().abs()),
                              (gw, dz.t() @ h.double(), term.t() @ h.double().abs())):
            acc = (dz.shape[0] + dz.shape[1]) * U
            tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
            close(got, ref, err * (1 + acc) + 1.01 * eps * ref.abs() + tiny + acc * err / eps, "gradient")


HALF = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("n,vocab,d", [(1, 1, 64), (1, 300, 64), (5, 255, 100), (37, 1000, 72), (256, 256, 64),
                                       (300, 1153, 192), (513, 2048, 128), (257, 5003, 7)])
def test_lmhead(dtype, n, vocab, d):
    need_gpu()
    say("lmhead logprobs", dtype, n, vocab, d)
    check(*operands(n, vocab, d, dtype, n + vocab))


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("temperature,softcap", [(0.3, 0.0), (2.5, 0.0), (0.7, 5.0), (1.0, 30.0), (0.05, 30.0)])
def test_lmhead_temperature_and_softcap(dtype, temperature, softcap):
    need_gpu()
    say("lmhead logprobs scale", dtype, temperature, softcap)
    check(*operands(300, 1000, 128, dtype, 3), temperature, softcap)


@pytest.mark.parametrize("temperature", [1e-3, 0.01, 50.0])
def test_lmhead_far_temperatures(temperature):
    """Scores in the thousands: each tile's offset is rounded, and its rest taken out again."""
    need_gpu()
    check(*operands(40, 700, 64, torch.bfloat16, 9, scale=8.0), temperature)


def test_lmhead_fp32():
    need_gpu()
    check(*operands(70, 1001, 48, torch.float32, 4), 0.8, 20.0)


def test_lmhead_without_tokens_and_special_tokens():
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn
    h, w, t = operands(40, 700, 64, torch.bfloat16, 5)
    check(h, w, None)
    t[4] = 700  # out of range: a NaN row, and with it the weight's gradient
    check(h, w, t, grads=False)
    hl = h.to(DEV).requires_grad_()
    r = kernel_fn(hl, w.to(DEV), t.to(DEV))
    (gh,) = torch.autograd.grad(r.logprobs.sum(), hl)
    rows = torch.isnan(gh).any(1).cpu()
    assert rows.tolist() == [i == 4 for i in range(40)] and bool((gh[1] == 0).all())
    t[:] = -100  # nothing counted
    check(h, w, t)


def test_lmhead_vocab_ranges(monkeypatch):
    """The backward over several vocab ranges."""
    need_gpu()
    from kernels.hip import chunked_linear_cross_entropy as clce
    monkeypatch.setattr(clce, "GRAD_LOGITS_BUDGET", 300 * 2 * 512)
    check(*operands(300, 2003, 128, torch.bfloat16, 6), 1.3)


def test_lmhead_agrees_with_the_row_kernels_and_the_loss():
    """The three forms of the head, on one model: the loss's per-row values are the
    negative log probabilities, and the row kernels see the same logits."""
    need_gpu()
    from kernels.hip.chunked_linear_cross_entropy import lmhead_ce_forward
    from kernels.hip.lmhead_logprobs import kernel_fn
    from kernels.hip.token_logprobs import kernel_fn as rows
    h, w, t = (a.to(DEV) for a in operands(700, 3001, 192, torch.bfloat16, 7))
    r = kernel_fn(h.view(7, 100, 192), w, t.view(7, 100), softcap=30.0)
    _, _, _, losses = lmhead_ce_forward(h, w, t, return_losses=True, softcap=30.0)
    assert torch.allclose(r.logprobs.reshape(-1), -losses, atol=2e-5, rtol=1e-6)
    full = rows(h.float() @ w.float().t(), t, softcap=30.0, top_k=3)
    assert torch.allclose(full.logprobs, r.logprobs.reshape(-1), atol=5e-5, rtol=1e-6)
    assert torch.allclose(full.entropy, r.entropy.reshape(-1), atol=5e-4)


def test_lmhead_graph_replays():
    need_gpu()
    from kernels.hip import _lib
    h, w, t = (a.to(DEV) for a in operands(300, 1001, 128, torch.bfloat16, 8))
    f = lambda *s: torch.empty(*s, device=DEV)
    lp, ent, st, co = f(300), f(300), f(300, 4), f(300, 4)
    up = torch.randn(300, generator=torch.Generator().manual_seed(1)).to(DEV)
    dz = torch.zeros(300, 1088, dtype=torch.bfloat16, device=DEV)[:, :1001]

    def run():
        _lib.lmhead_logprobs(h, w, t, lp, ent, st, 0.9, 0.0, -100)
        _lib.lmhead_logprobs_coefs(t, st, up, up, co, 1001, 0.9, -100)
        _lib.lmhead_logprobs_bwd_range(h, w, t, co, dz, 0, 0.9, 0.0, -100)

    run()
    torch.cuda.synchronize()
    ref = [o.clone() for o in (lp, ent, dz)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(4):
        for o in (lp, ent, dz):
            o.fill_(7)
        torch.cuda.synchronize()
        say("lmhead logprobs graph: replay", i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((lp, ent, dz), ref))
        run()


@pytest.mark.parametrize("n,vocab,live", [(5, 700, 3), (300, 1024, 200), (300, 1153, 300), (260, 600, 599)])
def test_lmhead_logits_past_fp32(n, vocab, live):
    """In bf16 (fp16's products stay in fp32's range). Weight rows whose products pass fp32 to -inf mask their tokens, tiles of
    them alone too; a hidden row for which all are such has no distribution.
    The live tokens' logits are 0, so ln p = -ln(live) and the entropy ln(live)."""
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn
    say("lmhead past fp32", n, vocab, live)
    g = torch.Generator().manual_seed(8)
    w = torch.zeros(vocab, 64, dtype=torch.bfloat16)
    w[:, 0] = -1e30
    at = torch.randperm(vocab, generator=g)[:live]
    w[at, 0] = 0.0
    w[:, 1] = -1e30
    h = torch.zeros(n, 64, dtype=torch.bfloat16)
    h[:, 0] = 1e30
    h[1] = 0.0
    h[1, 1] = 1e30  # all -inf
    t = at[torch.randint(0, live, (n,), generator=g)]
    masked = (w[:, 0] != 0).nonzero().flatten()
    t[2] = masked[0]
    hd, wd, td = h.to(DEV).requires_grad_(), w.to(DEV), t.to(DEV)
    r = kernel_fn(hd, wd, td)
    lp, ent = r.logprobs.double().cpu(), r.entropy.double().cpu()
    rows = torch.ones(n, dtype=torch.bool)
    rows[1] = False
    assert float((ent[rows] - math.log(live)).abs().max()) <= ROW * (1 + 2 * math.log(live)) and ent[1] == 0
    assert lp[1] == -math.inf and lp[2] == -math.inf
    rows[2] = False
    assert float((lp[rows] + math.log(live)).abs().max()) <= ROW + 4 * U * math.log(live)
    # the gradient's rows of the weight: sum over rows of dz h, 0 but in column 0 (and nothing from row 1)
    wl = w.to(DEV).requires_grad_()
    (gw,) = torch.autograd.grad(kernel_fn(h.to(DEV), wl, td).entropy.sum(), wl)
    assert bool((gw[:, 1:] == 0).all()) and bool((gw[masked.to(DEV)] == 0).all())
    (gh,) = torch.autograd.grad(r.entropy.sum(), hd)
    assert bool((gh[1] == 0).all()) and not bool(torch.isnan(gh).any())


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("n,vocab,d,softcap", [(32, 513, 320, 0.0), (33, 129, 64, 30.0), (64, 2000, 832, 0.0), (65, 777, 256, 0.0),
                                               (128, 1153, 576, 30.0), (129, 1153, 576, 30.0)])
def test_lmhead_few_tokens(dtype, n, vocab, d, softcap):
    """Both sides of the token blocks, last K chunks of one to four blocks, vocab rows left in the last group."""
    need_gpu()
    say("lmhead few", dtype, n, vocab, d, softcap)
    check(*operands(n, vocab, d, dtype, n + d), 0.9, softcap)
    check(*operands(n, vocab, d, dtype, n + d + 1)[:2], None, 1.0, softcap)
