"""GPU parity of the scoring operators over logits: token log probabilities with
entropy and alternatives, and distillation from a teacher's top logits, against
the float64 oracle.

Tolerances, from fp32 arithmetic (u = 2^-24):

* a row's sums are chains of at most 150 additions of non-negative (s) or
  non-positive (u) terms, each term off by at most 8 u of itself for every unit
  of ln V (the exponent's product and the hardware exponential): relative error
  150 u + 8 u ln V. ln s, u / s and a log probability then have absolute errors
  of at most that times 1, |u / s| and 1, plus 4 u of their own size. ROW below
  is 300 u = 1.8e-5: 150 u + 8 u ln V at V = 2^17;
* the softcap's tanh is within 4 u of 1, so scores are off by 4 u softcap / T;
* gradients: 2 ROW of the terms' size, plus half a step of the output type
  (finfo.eps / 2) of the value, plus half its smallest subnormal.
"""

import math

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from oracle import scoring

pytestmark = gpu
DEV = "cuda"
U = 2.0 ** -24
ROW = 300 * U
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def close(got, want, tol, what):
    """NaN and infinities in the same places, elsewhere within ``tol``. What
    passes the output type's range is an infinity of that type."""
    want = torch.where(want.abs() > torch.finfo(got.dtype).max, want.sign() * math.inf, want.double())
    got = got.detach().cpu().double()
    fine = torch.isfinite(want)
    same = torch.where(torch.isnan(want), torch.isnan(got), got == want)
    assert bool(same[~fine].all()), f"{what}: special values differ"
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    off = (got - want).abs()
    bad = fine & ~(off <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float((off / tol)[bad].max())} times the tolerance")


def score_tol(temperature, softcap):
    return 4 * U * softcap / temperature


def grad_tol(ref, size, dtype, temperature, softcap):
    return (2 * ROW + 8 * score_tol(temperature, softcap)) * size + torch.finfo(dtype).eps / 2 * ref.abs() * 1.001 \
        + TINY[dtype] + 1e-37


def logits_of(rows, vocab, dtype, seed, pitch=None, offset=0):
    """Rows of a trained head's kind: a wide base and a few confident tokens;
    ``pitch`` and ``offset`` put them off the 16-byte grid."""
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(rows, vocab, generator=g)
    x += 7 * (torch.rand(rows, vocab, generator=g) > 0.999)
    pitch = pitch or vocab
    buf = torch.zeros(rows * pitch + offset + 8, dtype=dtype, device=DEV)
    view = buf[offset:offset + rows * pitch].view(rows, pitch)[:, :vocab]
    view.copy_(x.to(dtype))
    return view


def check_logprobs(x, tokens, temperature=1.0, softcap=0.0, top_k=0, grads=True):
    from kernels.hip.token_logprobs import kernel_fn
    xc = x.detach().cpu()
    tc = tokens.cpu() if tokens is not None else None
    leaf = x.detach()
    r = kernel_fn(leaf, tokens, temperature=temperature, softcap=softcap, top_k=top_k)
    lp, h = scoring.logprob_rows(xc, tc, temperature, softcap)
    lnv = math.log(max(2, x.shape[1]))
    st = score_tol(temperature, softcap)
    if tokens is None:
        assert r.logprobs is None
    else:
        assert r.logprobs.dtype == torch.float32
        close(r.logprobs, lp, ROW + 2 * st + 4 * U * torch.nan_to_num(lp.abs(), 0, 0, 0), "logprobs")
    close(r.entropy, h, (ROW + 2 * st) * (1 + 2 * lnv), "entropy")
    if top_k:
        tv, ti = scoring.top_rows(xc, top_k, temperature, softcap)
        assert torch.equal(r.top_ids.cpu(), ti), "top_ids"
        close(r.top_logprobs, tv, ROW + 2 * st + 4 * U * torch.nan_to_num(tv.abs(), 0, 0, 0), "top_logprobs")
    if not grads:
        return r
    g = torch.Generator().manual_seed(9)
    gl = torch.randn(x.shape[0], generator=g) if tokens is not None else None
    ge = torch.randn(x.shape[0], generator=g)
    leaf = x.detach().requires_grad_()  # (a view with x's strides)
    r = kernel_fn(leaf, tokens, temperature=temperature, softcap=softcap, top_k=top_k)
    for pair in ((gl, ge), (gl, None), (None, ge)):
        outs = [(o, u.to(DEV)) for o, u in zip((r.logprobs, r.entropy), pair) if u is not None]
        if not outs:
            continue
        (gx,) = torch.autograd.grad([o for o, _ in outs], [leaf], [u for _, u in outs], retain_graph=True)
        assert gx.shape == x.shape and gx.dtype == x.dtype
        ref, size = scoring.logprob_grad_rows(xc, tc, pair[0], pair[1], temperature, softcap)
        close(gx, ref, grad_tol(torch.nan_to_num(ref), size, x.dtype, temperature, softcap), "gradient")
    return r


DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (3, 7, 7), (2, 8, 3), (5, 65, 20), (9, 1000, 256), (4, 2049, 0),
                                              (3, 8191, 64), (17, 16385, 5), (2, 50257, 128)])
def test_logprobs(dtype, rows, vocab, top_k):
    need_gpu()
    say("logprobs", dtype, rows, vocab, top_k)
    x = logits_of(rows, vocab, dtype, rows + vocab)
    t = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(5)).to(DEV)
    if rows > 2:
        t[1], t[2] = -100, vocab  # ignored; out of range
    check_logprobs(x, t, top_k=top_k)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("pitch,offset", [(5003, 0), (5003, 1), (5120, 3), (5008, 8)])
def test_logprobs_pitches_and_addresses(dtype, pitch, offset):
    need_gpu()
    say("logprobs strided", dtype, pitch, offset)
    x = logits_of(300, 5001, dtype, 3, pitch, offset)  # 300 rows: uncut; 3: cut
    t = torch.randint(0, 5001, (300,), generator=torch.Generator().manual_seed(6)).to(DEV)
    check_logprobs(x[:3], t[:3], top_k=20)
    check_logprobs(x, t, top_k=20)


@pytest.mark.parametrize("temperature,softcap", [(0.25, 0.0), (3.0, 0.0), (0.7, 30.0), (1.0, 5.0)])
@pytest.mark.parametrize("rows", [2, 260])
def test_logprobs_temperature_and_softcap(rows, temperature, softcap):
    need_gpu()
    say("logprobs scale", rows, temperature, softcap)
    x = logits_of(rows, 3001, torch.bfloat16, 11)
    t = torch.randint(0, 3001, (rows,), generator=torch.Generator().manual_seed(7)).to(DEV)
    check_logprobs(x, t, temperature, softcap, top_k=10)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab,top_k", [(2500, 7), (5003, 100), (9000, 256), (17001, 64), (33000, 5), (60000, 128), (70001, 256)])
def test_logprobs_top_of_many_rows(dtype, vocab, top_k):
    """Uncut rows of every width: each way a thread holds a row, and its groups' maxima."""
    need_gpu()
    say("logprobs many", dtype, vocab, top_k)
    from kernels.hip.token_logprobs import kernel_fn
    x = logits_of(600, vocab, dtype, vocab)
    x[1] = x[1].round()  # many ties
    t = torch.randint(0, vocab, (600,), generator=torch.Generator().manual_seed(7)).to(DEV)
    for rows in (600, 300):  # one wave a row, four
        r = kernel_fn(x[:rows], t[:rows], top_k=top_k)
        # exact ids of all rows: the logit's place among the numbers, then the column
        bits = (x[:rows].float() + 0.0).view(torch.int32).to(torch.int64)
        key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) - torch.arange(vocab, device=DEV)
        assert torch.equal(r.top_ids, key.topk(top_k, dim=1).indices)
        logp = torch.log_softmax(x[:rows].double(), 1)
        close(r.top_logprobs, logp.gather(1, r.top_ids).cpu(), 2 * ROW, "top_logprobs")
        close(r.logprobs, logp.gather(1, t[:rows, None])[:, 0].cpu(), 2 * ROW, "logprobs")


def test_logprobs_without_tokens():
    need_gpu()
    check_logprobs(logits_of(6, 3000, torch.float32, 1), None, top_k=4)
    check_logprobs(logits_of(300, 3000, torch.float16, 1), None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 262144), (2, 300001), (257, 140000)])
def test_logprobs_wide(dtype, rows, vocab):
    """Rows past one workgroup's registers are cut whatever their number."""
    need_gpu()
    say("logprobs wide", dtype, rows, vocab)
    x = logits_of(rows, vocab, dtype, 4)
    t = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(8)).to(DEV)
    if rows < 10:
        check_logprobs(x, t, top_k=256)
    else:
        r = check_logprobs(x[-3:], t[-3:], top_k=20, grads=False)
        from kernels.hip.token_logprobs import kernel_fn
        whole = kernel_fn(x, t, top_k=20)
        assert torch.equal(whole.top_ids[-3:], r.top_ids)
        assert torch.allclose(whole.logprobs[-3:], r.logprobs, rtol=0, atol=2 * ROW)
        assert torch.allclose(whole.entropy[-3:], r.entropy, rtol=0, atol=2 * ROW * 25)


def special_rows(vocab, dtype):
    g = torch.Generator().manual_seed(21)
    base = 2 * torch.randn(14, vocab, generator=g)
    low = torch.finfo(dtype).min
    base[0] = -math.inf                       # nothing left
    base[1] = -math.inf                       # one entry left
    base[1, vocab // 2] = 1.0
    base[2, vocab // 3:] = -math.inf          # a third left
    base[3] = low                             # every logit the lowest value
    base[4, 5:] = low                         # five left beside the lowest value
    base[5, vocab - 1] = math.nan
    base[6, 0] = math.inf
    base[7] = math.nan
    base[8] = 0.0                             # ties, of both zeros
    base[8, ::3] = -0.0
    base[9] = 1.0
    base[9, vocab - 3:] = 2.0
    base[10, 3] = torch.finfo(dtype).max
    base[11] = -math.inf                      # fewer left than alternatives asked for
    base[11, vocab - 7:] = torch.arange(7.0)
    base[12] = base[12].round()               # thousands of equal logits, among them the top's border
    base[13, :4] = math.nan
    return base.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [40, 3001, 40007])
@pytest.mark.parametrize("copies", [1, 20])
def test_logprobs_special_rows(dtype, vocab, copies):
    """Copies: 14 rows are cut into segments, 280 are not."""
    need_gpu()
    say("logprobs special", dtype, vocab, copies)
    x = special_rows(vocab, dtype)
    tok = torch.randint(0, vocab, (14,), generator=torch.Generator().manual_seed(2))
    tok[1], tok[2], tok[5] = vocab // 2, vocab - 1, -100
    if copies > 1:
        from kernels.hip.token_logprobs import kernel_fn
        xs, ts = x.repeat(copies, 1).to(DEV), tok.repeat(copies).to(DEV)
        small = kernel_fn(x.to(DEV), tok.to(DEV), top_k=20)
        r = kernel_fn(xs, ts, top_k=20)
        for a, b, tol in zip(r, small, (2 * ROW, 2 * ROW * 25, 2 * ROW, 0)):
            for c in range(copies):
                assert torch.allclose(a[14 * c:14 * c + 14].double(), b.double(), rtol=1e-6, atol=tol, equal_nan=True)
        x, tok = xs[-14:], ts[-14:]
    check_logprobs(x.to(DEV), tok.to(DEV), top_k=min(20, vocab))
    check_logprobs(x.to(DEV), tok.to(DEV), top_k=1, temperature=0.5, grads=False)


def teacher_of(x, k, seed, dtype=torch.float32, pad=True):
    """A teacher near the student: its top k, fewer for some rows, none for the first."""
    g = torch.Generator().manual_seed(seed)
    t = x.cpu().float() + 0.5 * torch.randn(x.shape, generator=g)
    val, ids = t.topk(k, dim=1)
    if pad:
        n = torch.randint(1, k + 1, (x.shape[0], 1), generator=g)
        n[0] = 0
        ids = ids.masked_fill(torch.arange(k)[None, :] >= n, -100)
        if x.shape[0] > 2 and k > 1:
            ids[1, 0], ids[1, 1] = x.shape[1] - 1, x.shape[1] - 1  # the same id twice
            ids[2, 0] = -100                                        # padding in front
    return val.to(dtype).to(DEV), ids.to(DEV)


def check_distill(x, teacher, ids, temperature=1.0, softcap=0.0):
    from kernels.hip.topk_distillation import kernel_fn
    xc, tc, ic = x.detach().cpu(), teacher.cpu(), ids.cpu()
    want, _, counted = scoring.distill_rows(xc, tc, ic, temperature, softcap)
    # each of a row's terms is q (ln q - ln p): their q sum to 1, both logarithms
    # within ROW and 4 u of their size; the teacher's own scaling adds 8 u |t| / T
    size = 1 + math.log(x.shape[1]) + 2 * torch.nan_to_num(xc.double(), 0, 0, 0).abs().amax(1) / temperature
    tol = temperature ** 2 * ((2 * ROW + 2 * score_tol(temperature, softcap)) + 24 * U * size)
    kw = dict(temperature=temperature, softcap=softcap)
    rows = kernel_fn(x.detach(), teacher, ids, reduction="none", **kw)
    close(rows, want, tol, "losses")
    n = max(1, int(counted.sum()))
    mean = kernel_fn(x.detach(), teacher, ids, **kw)
    assert mean.shape == () and mean.dtype == torch.float32
    close(mean.reshape(1), want.sum().reshape(1) / n, tol.max() + 200 * U * torch.nan_to_num(want).abs().mean(), "mean")
    leaf = x.detach().requires_grad_()
    up = torch.randn(x.shape[0], generator=torch.Generator().manual_seed(3))
    (gx,) = torch.autograd.grad(kernel_fn(leaf, teacher, ids, reduction="none", **kw), leaf, up.to(DEV))
    ref, size = scoring.distill_grad_rows(xc, tc, ic, up, temperature, softcap)
    close(gx, ref, 2 * grad_tol(torch.nan_to_num(ref), torch.nan_to_num(size), x.dtype, temperature, softcap), "gradient")
    (gx,) = torch.autograd.grad(kernel_fn(leaf, teacher, ids, **kw), leaf, torch.tensor(0.3, device=DEV))
    ref, size = scoring.distill_grad_rows(xc, tc, ic, torch.full((x.shape[0],), 0.3 / n), temperature, softcap)
    close(gx, ref, 2 * grad_tol(torch.nan_to_num(ref), torch.nan_to_num(size), x.dtype, temperature, softcap), "gradient of the mean")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 7, 2), (6, 300, 256), (5, 2049, 64), (270, 1031, 20),
                                          (3, 50257, 128), (2, 140000, 33)])
def test_distill(dtype, rows, vocab, k):
    need_gpu()
    say("distill", dtype, rows, vocab, k)
    x = logits_of(rows, vocab, dtype, rows + vocab)
    check_distill(x, *teacher_of(x, k, 1, pad=rows > 1), temperature=2.0)


@pytest.mark.parametrize("teacher_dtype", DTYPES, ids=str)
@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (0.5, 20.0), (4.0, 30.0)])
def test_distill_scales_and_teacher_types(teacher_dtype, temperature, softcap):
    need_gpu()
    say("distill scale", teacher_dtype, temperature, softcap)
    x = logits_of(5, 4003, torch.bfloat16, 2, 4099, 3)
    t, i = teacher_of(x, 40, 2, teacher_dtype)
    wide_t, wide_i = torch.zeros(5, 47, dtype=t.dtype, device=DEV), torch.zeros(5, 43, dtype=i.dtype, device=DEV)
    wide_t[:, :40], wide_i[:, :40] = t, i
    check_distill(x, wide_t[:, :40], wide_i[:, :40], temperature, softcap)  # rows at a pitch


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [40, 40007])
def test_distill_special_rows(dtype, vocab):
    need_gpu()
    say("distill special", dtype, vocab)
    x = special_rows(vocab, dtype).to(DEV)
    g = torch.Generator().manual_seed(4)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:6] for _ in range(14)])
    t = torch.randn(14, 6, generator=g)
    ids[1, 0] = vocab // 2
    ids[2] = torch.arange(6)     # all unmasked
    ids[4] = torch.arange(6)     # the last one has the lowest value
    t[4, 5] = -math.inf          # and no teacher
    ids[8, 2], t[9, 1], t[12] = vocab, math.nan, -math.inf  # out of range; NaN; no teacher at all
    keep = [r for r in range(14) if r not in (3, 10)]  # (a loss past fp32, where the scores are)
    check_distill(x[keep], t[keep].to(DEV), ids[keep].to(DEV))


def test_teacher_to_student():
    """The operators together: a teacher's top alternatives, and a student distilled from them."""
    need_gpu()
    from kernels.hip.token_logprobs import kernel_fn as logprobs
    from kernels.hip.topk_distillation import kernel_fn as distill
    teacher = logits_of(4 * 33, 5003, torch.bfloat16, 5).reshape(4, 33, 5003)
    student = logits_of(4 * 33, 5003, torch.float32, 6).reshape(4, 33, 5003).requires_grad_()
    tok = torch.randint(0, 5003, (4, 33), generator=torch.Generator().manual_seed(1)).to(DEV)
    tok[:, :5] = -100
    with torch.no_grad():
        t = logprobs(teacher, tok, top_k=50)
    assert t.logprobs.shape == t.entropy.shape == (4, 33) and t.top_ids.shape == t.top_logprobs.shape == (4, 33, 50)
    ids = t.top_ids.masked_fill((tok == -100)[..., None], -100)
    s = logprobs(student, tok)
    loss = distill(student, t.top_logprobs, ids, temperature=1.5) - (s.logprobs.sum() + 0.1 * s.entropy.sum()) / 112
    loss.backward()
    x = student.detach().cpu().reshape(-1, 5003)
    tc = tok.cpu().reshape(-1)
    a, sa = scoring.distill_grad_rows(x, t.top_logprobs.cpu().reshape(-1, 50), ids.cpu().reshape(-1, 50),
                                      torch.full((132,), 1 / 112), 1.5)
    b, sb = scoring.logprob_grad_rows(x, tc, torch.full((132,), -1 / 112), torch.full((132,), -0.1 / 112))
    close(student.grad.reshape(-1, 5003), a + b, 3 * ROW * (sa + sb) + 1e-30, "gradient")


def test_streams_devices_and_graphs():
    """Captured on a side stream and replayed, with eager work between the replays;
    every replay gives the eager results bit for bit."""
    need_gpu()
    from kernels.hip import _lib
    x = logits_of(6, 50257, torch.bfloat16, 5)
    many = logits_of(300, 5003, torch.float16, 5)
    t = torch.randint(0, 5003, (6,), generator=torch.Generator().manual_seed(1)).to(DEV)
    tm = torch.randint(0, 5003, (300,), generator=torch.Generator().manual_seed(1)).to(DEV)
    teacher, ids = teacher_of(x, 40, 3)
    up = torch.randn(6, generator=torch.Generator().manual_seed(1)).to(DEV)
    f = lambda *s: torch.empty(*s, device=DEV)
    lp, h, st, tv = f(6), f(6), f(6, 4), f(6, 20)
    ti = torch.empty(6, 20, dtype=torch.int64, device=DEV)
    lp2, h2, tv2 = f(300), f(300), f(300, 9)
    ti2 = torch.empty(300, 9, dtype=torch.int64, device=DEV)
    g, gd = torch.empty_like(x.contiguous()), torch.empty_like(x.contiguous())
    losses, sd, loss, scale = f(6), f(6, 4), f(()), f(1)

    def run():
        _lib.token_logprobs(x, t, lp, h, st, tv, ti, 0.8, 0.0, -100)
        _lib.token_logprobs(many, tm, lp2, h2, None, tv2, ti2, 1.0, 30.0, -100)
        _lib.token_logprobs_bwd(x, t, st, up, up, g, 0.8, 0.0, -100)
        _lib.topk_distill(x, teacher, ids, losses, sd, loss, scale, 2.0, 0.0, -100)
        _lib.topk_distill_bwd(x, teacher, ids, sd, up[:1], scale, gd, 2.0, 0.0, -100)

    outs = [lp, h, tv, ti, lp2, h2, tv2, ti2, g, losses, loss, scale, gd]
    run()
    torch.cuda.synchronize()
    ref = [o.clone() for o in outs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    torch.cuda.synchronize()
    for i in range(4):
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        say("scoring graph: replay", i)
        graph.replay()
        torch.cuda.synchronize()
        for k, (o, want) in enumerate(zip(outs, ref)):
            assert torch.equal(o.nan_to_num(5), want.nan_to_num(5)), (i, k)
        run()  # eager work between the replays


def test_runs_are_bitwise_the_same():
    need_gpu()
    from kernels.hip.token_logprobs import kernel_fn
    x = logits_of(5, 50257, torch.bfloat16, 5).clone().requires_grad_()
    t = torch.randint(0, 50257, (5,), generator=torch.Generator().manual_seed(1)).to(DEV)
    first = None
    for _ in range(3):
        r = kernel_fn(x, t, top_k=64)
        (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), x)
        got = [*r, g]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("softcap", [1e-3, 1.0, 2.0, 1e4])
def test_gradients_near_and_far_from_the_cap(dtype, softcap):
    """Logits beyond a small cap, whose slope 1 - tanh^2 goes down to e^-30 (its
    exponent 2 |x| / cap is rounded to 2 u of it, within ROW), and a cap beyond all logits."""
    need_gpu()
    say("softcap", dtype, softcap)
    x = logits_of(9, 1500, dtype, 31)
    if softcap < 1.0:
        x.mul_(softcap)  # (x / cap up to 15; of fp16's subnormals each is exact)
    else:
        x.clamp_(-15 * softcap, 15 * softcap)
    t = torch.randint(0, 1500, (9,), generator=torch.Generator().manual_seed(5)).to(DEV)
    check_logprobs(x, t, 1.0, softcap, top_k=4)
    check_distill(x, *teacher_of(x, 20, 6), softcap=softcap)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_ignored_rows_among_many(dtype):
    """Whole rows (256 and more), every third ignored and some of those NaN: nothing of them
    reaches their results, their gradients or their neighbours; all ignored; ignored with alternatives."""
    need_gpu()
    from kernels.hip.token_logprobs import kernel_fn
    say("ignored", dtype)
    x = logits_of(300, 1031, dtype, 41)
    t = torch.randint(0, 1031, (300,), generator=torch.Generator().manual_seed(4))
    t[::3] = -100
    check_logprobs(x, t.to(DEV))
    check_logprobs(x, t.to(DEV), top_k=3)
    y = x.clone()
    y[::6] = math.nan
    for a, b in zip(kernel_fn(x, t.to(DEV))[:2], kernel_fn(y, t.to(DEV))[:2]):
        assert torch.equal(a, b)
    leaf = y.requires_grad_()
    r = kernel_fn(leaf, t.to(DEV))
    (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), leaf)
    assert bool((g[::3] == 0).all()) and bool(torch.isfinite(g).all())
    r = kernel_fn(x, torch.full((300,), -100, device=DEV))
    assert bool((r.logprobs == 0).all()) and bool((r.entropy == 0).all())
    # rows of several segments
    x = logits_of(257, 70001, dtype, 42)
    t = torch.randint(0, 70001, (257,), generator=torch.Generator().manual_seed(4))
    t[::3] = -100
    x[::6] = math.nan
    leaf = x.requires_grad_()
    r = kernel_fn(leaf, t.to(DEV))
    lp, h = scoring.logprob_rows(x[1:5].detach().cpu(), t[1:5])
    close(r.logprobs[1:5], lp, ROW + 4 * U * lp.abs(), "logprobs")
    close(r.entropy[1:5], h, ROW * (1 + 2 * math.log(70001)), "entropy")
    assert bool((r.logprobs[::3] == 0).all()) and bool((r.entropy[::3] == 0).all()) and bool(torch.isfinite(r.logprobs).all())
    (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), leaf)
    assert bool((g[::3] == 0).all()) and bool(torch.isfinite(g).all())
