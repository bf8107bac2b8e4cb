"""Host logic of the scoring operators (CPU tier): the launchers are routed to
the float64 oracle, so these tests check shapes, types, autograd contracts and
refusals; the library's own refusals return before any HIP call."""

import math

import pytest
import torch

from kernels.hip import _lib
from kernels.hip import lmhead_logprobs as ll
from kernels.hip import token_logprobs as tl
from kernels.hip import topk_distillation as td
from oracle import scoring


@pytest.fixture
def scoring_backend(monkeypatch):
    def logprobs(x, tok, lp, h, stats, tv, ti, temperature, softcap, ignore):
        a, b = scoring.logprob_rows(x, tok, temperature, softcap, ignore)
        if lp is not None:
            lp.copy_(a)
        h.copy_(b)
        if stats is not None:
            stats.zero_()
        if ti is not None:
            v, i = scoring.top_rows(x, ti.shape[1], temperature, softcap)
            tv.copy_(v)
            ti.copy_(i)

    def logprobs_bwd(x, tok, stats, gl, ge, grad, temperature, softcap, ignore):
        for g in (gl, ge):
            assert g is None or (g.dtype == torch.float32 and g.is_contiguous() and g.dim() == 1)
        grad.copy_(scoring.logprob_grad_rows(x, tok, gl, ge, temperature, softcap, ignore)[0])

    def distill(x, t, ids, losses, stats, loss, scale, temperature, softcap, ignore):
        rows, _, counted = scoring.distill_rows(x, t, ids, temperature, softcap, ignore)
        losses.copy_(rows)
        stats.zero_()
        if loss is not None:
            n = max(1, int(counted.sum()))
            loss.copy_(rows.sum() / n)
            scale.fill_(1 / n)

    def distill_bwd(x, t, ids, stats, g, scale, grad, temperature, softcap, ignore):
        up = g * scale if scale is not None else g
        assert g.numel() == (1 if scale is not None else x.shape[0])
        grad.copy_(scoring.distill_grad_rows(x, t, ids, up.expand(x.shape[0]), temperature, softcap, ignore)[0])

    def lmhead(h, w, tok, lp, ent, stats, temperature, softcap, ignore):
        assert h.shape[1] % 64 == 0 and h.is_contiguous() and w.is_contiguous()
        logprobs(h.double() @ w.double().t(), tok, lp, ent, stats, None, None, temperature, softcap, ignore)

    saved = {}

    def coefs(tok, stats, gl, ge, out, vocab, temperature, ignore):
        saved.update(gl=gl, ge=ge)

    def lmhead_bwd(h, w, tok, co, grad, v0, temperature, softcap, ignore):
        full = scoring.logprob_grad_rows(h.double() @ w.double().t(), tok, saved["gl"], saved["ge"], temperature,
                                         softcap, ignore)[0]
        grad.copy_(full[:, v0:v0 + grad.shape[1]])

    def add(out, value, mode):
        out.copy_(value + (out.double() if mode == 2 else 0))

    for name, fn in (("token_logprobs", logprobs), ("token_logprobs_bwd", logprobs_bwd), ("topk_distill", distill),
                     ("topk_distill_bwd", distill_bwd), ("require_device", lambda *t: None),
                     ("lmhead_logprobs", lmhead), ("lmhead_logprobs_coefs", coefs),
                     ("lmhead_logprobs_bwd_range", lmhead_bwd), ("lmhead_grad_workspace_bytes", lambda n, v, d: 256),
                     ("lmhead_grad_hidden", lambda g, w, out, mode, ws: add(out, g.double() @ w.double(), mode)),
                     ("lmhead_grad_weight", lambda g, h, out, mode, ws: add(out, g.double().t() @ h.double(), mode))):
        monkeypatch.setattr(_lib, name, fn)


def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="GPU"):
        tl.kernel_fn(torch.randn(2, 5))
    with pytest.raises(RuntimeError, match="GPU"):
        td.kernel_fn(torch.randn(2, 5), torch.randn(2, 3), torch.zeros(2, 3, dtype=torch.int64))


def test_shapes_types_and_gradients(scoring_backend):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 17, generator=g).bfloat16().requires_grad_()
    tok = torch.randint(0, 17, (2, 3), generator=g, dtype=torch.int32)
    r = tl.kernel_fn(x, tok, top_k=4, temperature=0.5)
    assert r.logprobs.shape == r.entropy.shape == (2, 3) and r.top_ids.shape == r.top_logprobs.shape == (2, 3, 4)
    assert r.top_ids.dtype == torch.int64 and r.logprobs.dtype == torch.float32
    assert r.logprobs.requires_grad and not r.top_logprobs.requires_grad
    (r.logprobs.sum() + 2 * r.entropy.sum()).backward()
    ref, _ = scoring.logprob_grad_rows(x.detach().reshape(6, 17), tok.reshape(-1), torch.ones(6), 2 * torch.ones(6), 0.5)
    assert x.grad.dtype == x.dtype and torch.equal(x.grad.reshape(6, 17), ref.bfloat16())
    # one row without leading dimensions; no tokens; nothing to differentiate
    one = tl.kernel_fn(x[0, 0].detach(), torch.tensor(3), top_k=2)
    assert one.logprobs.shape == () and one.top_ids.shape == (2,) and not one.entropy.requires_grad
    none = tl.kernel_fn(x.detach())
    assert none.logprobs is None and none.top_ids is None and none.entropy.shape == (2, 3)
    # no rows
    empty = tl.kernel_fn(x[:0].detach(), tok[:0], top_k=2)
    assert empty.logprobs.shape == (0, 3) and empty.top_ids.shape == (0, 3, 2)
    x0 = torch.randn(0, 5, requires_grad=True)
    tl.kernel_fn(x0, torch.zeros(0, dtype=torch.int64)).logprobs.sum().backward()
    assert x0.grad.shape == (0, 5)


def test_gradients_of_one_output_and_broadcast_upstream(scoring_backend):
    x = torch.randn(4, 9, requires_grad=True)
    tok = torch.tensor([1, -100, 3, 8])
    r = tl.kernel_fn(x, tok)
    (g,) = torch.autograd.grad(r.entropy.sum(), x, retain_graph=True)  # an expanded upstream gradient
    assert torch.allclose(g.double(), scoring.logprob_grad_rows(x.detach(), tok, None, torch.ones(4))[0], atol=1e-6)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(r.logprobs.double().sum(), x, create_graph=True)


def test_distillation_contract(scoring_backend):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 11, generator=g, requires_grad=True)
    t = torch.randn(2, 3, 4, generator=g).half()
    ids = torch.randint(0, 11, (2, 3, 4), generator=g)
    ids[0, 0] = -100
    ids[1, 1, 2:] = -100
    loss = td.kernel_fn(x, t, ids, temperature=2.0)
    rows = td.kernel_fn(x, t, ids, temperature=2.0, reduction="none")
    assert loss.shape == () and rows.shape == (2, 3) and float(rows.detach()[0, 0]) == 0
    assert float(loss.detach()) == pytest.approx(float(rows.detach().sum()) / 5, rel=1e-6)
    (gx,) = torch.autograd.grad(loss, x, torch.tensor(0.5))
    (gr,) = torch.autograd.grad(rows, x, torch.full((2, 3), 0.1))
    assert torch.allclose(gx, gr, atol=1e-7)
    # every row without entries; no rows
    assert float(td.kernel_fn(x, t, torch.full_like(ids, -100))) == 0
    assert float(td.kernel_fn(x[:0], t[:0], ids[:0])) == 0
    assert td.kernel_fn(x[:0], t[:0], ids[:0], reduction="none").shape == (0, 3)
    # a teacher that requires a gradient is a constant
    assert not td.kernel_fn(x.detach(), t.clone().requires_grad_(), ids).requires_grad


@pytest.mark.parametrize("dtype,budget", [(torch.bfloat16, 4 << 30), (torch.float16, 6 * 256 * 2), (torch.float32, 0)])
def test_lmhead_contract(scoring_backend, monkeypatch, dtype, budget):
    """Padded hidden sizes, vocab ranges, fp32 row chunks, gradients of either operand."""
    from kernels.hip import chunked_linear_cross_entropy as clce
    from kernels.hip.lmhead_logprobs import kernel_fn
    monkeypatch.setattr(clce, "GRAD_LOGITS_BUDGET", budget)
    g = torch.Generator().manual_seed(3)
    h = torch.randn(2, 3, 70, generator=g).to(dtype).requires_grad_()
    w = (0.2 * torch.randn(600, 70, generator=g)).to(dtype).requires_grad_()
    tok = torch.tensor([[5, -100, 599], [0, 1, 300]])
    kw = dict(temperature=0.8, softcap=10.0, chunk_size=4)
    r = kernel_fn(h, w, tok, **kw)
    x = (h.double().reshape(6, 70) @ w.double().t()).detach()
    lp, ent = scoring.logprob_rows(x, tok.reshape(-1), 0.8, 10.0)
    assert r.logprobs.shape == r.entropy.shape == (2, 3)
    assert torch.allclose(r.logprobs.double().reshape(-1), lp, atol=1e-5)
    assert torch.allclose(r.entropy.double().reshape(-1), ent, atol=1e-5)
    gl, ge = torch.randn(2, 3, generator=g), torch.randn(2, 3, generator=g)
    gh, gw = torch.autograd.grad((r.logprobs, r.entropy), (h, w), (gl, ge), retain_graph=True)
    dz = scoring.logprob_grad_rows(x, tok.reshape(-1), gl.reshape(-1), ge.reshape(-1), 0.8, 10.0)[0]
    tol = 3e-2 if dtype != torch.float32 else 1e-5
    assert gh.dtype == gw.dtype == dtype and gh.shape == h.shape
    for got, want in ((gh.reshape(6, 70), dz @ w.double()), (gw, dz.t() @ h.double().reshape(6, 70))):
        assert float((got.double() - want).norm() / want.norm()) < tol
    (gh2,) = torch.autograd.grad(r.entropy, h, ge, retain_graph=True)
    assert gh2.shape == h.shape
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(r.logprobs.sum(), h, create_graph=True)
    # no tokens, no rows, a weight of another type, one row
    assert kernel_fn(h.detach(), w.detach()).logprobs is None
    assert kernel_fn(h.detach()[0, 0], w.detach().float(), torch.tensor(7)).logprobs.shape == ()
    e = kernel_fn(h[:0], w, tok[:0])
    assert e.logprobs.shape == (0, 3)
    assert torch.equal(torch.autograd.grad(e.entropy.sum(), w)[0], torch.zeros_like(w))


def test_lmhead_refusals(scoring_backend):
    from kernels.hip.lmhead_logprobs import kernel_fn
    h, w, tok = torch.randn(3, 64), torch.randn(9, 64), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="go with"):
        kernel_fn(h, w[:, :63], tok)
    with pytest.raises(ValueError, match="go with"):
        kernel_fn(h, w[0], tok)
    with pytest.raises(ValueError, match="empty"):
        kernel_fn(h, w[:0], tok)
    with pytest.raises(ValueError, match="tokens"):
        kernel_fn(h, w, tok[:2])
    with pytest.raises(TypeError, match="whole"):
        kernel_fn(h, w, tok.float())
    with pytest.raises(TypeError, match="dtype"):
        kernel_fn(h.double(), w, tok)
    for bad in (0, 1e-4, 1e20):
        with pytest.raises(ValueError, match="temperature"):
            kernel_fn(h, w, tok, temperature=bad)
    with pytest.raises(ValueError, match="softcap"):
        kernel_fn(h, w, tok, softcap=-1)
    with pytest.raises(ValueError, match="chunk_size"):
        kernel_fn(h, w, tok, chunk_size=0)


def test_refusals(scoring_backend):
    x, tok = torch.randn(3, 8), torch.zeros(3, dtype=torch.int64)
    t, ids = torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    for bad in (0.0, -1.0, math.nan, math.inf, 1e-20, 1e20):
        with pytest.raises(ValueError, match="temperature"):
            tl.kernel_fn(x, tok, temperature=bad)
        with pytest.raises(ValueError, match="temperature"):
            td.kernel_fn(x, t, ids, temperature=bad)
    for bad in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="softcap"):
            tl.kernel_fn(x, tok, softcap=bad)
    for bad in (-1, 9, 257):
        with pytest.raises(ValueError, match="top_k"):
            tl.kernel_fn(x, tok, top_k=bad)
    with pytest.raises(ValueError, match="top_k"):
        tl.kernel_fn(torch.randn(1, 300), top_k=257)
    with pytest.raises(ValueError, match="tokens"):
        tl.kernel_fn(x, tok[:2])
    with pytest.raises(ValueError, match="tokens"):
        tl.kernel_fn(x, tok[:, None])
    for wrong in (tok.float(), tok.bool()):
        with pytest.raises(TypeError, match="whole numbers"):
            tl.kernel_fn(x, wrong)
    with pytest.raises(TypeError, match="dtype"):
        tl.kernel_fn(x.double(), tok)
    with pytest.raises(ValueError, match="vocab"):
        tl.kernel_fn(torch.randn(3, 0), tok)
    with pytest.raises(ValueError, match="vocab"):
        tl.kernel_fn(torch.empty(1, (1 << 20) + 1), tok[:1])
    with pytest.raises(ValueError, match="vocab"):
        tl.kernel_fn(torch.tensor(1.0))
    with pytest.raises(ValueError, match="teacher_logits"):
        td.kernel_fn(x, t[:2], ids[:2])
    with pytest.raises(ValueError, match="teacher_ids"):
        td.kernel_fn(x, t, ids[:, :1])
    with pytest.raises(TypeError, match="whole numbers"):
        td.kernel_fn(x, t, ids.float())
    with pytest.raises(TypeError, match="dtype"):
        td.kernel_fn(x, t.double(), ids)
    with pytest.raises(ValueError, match="entries"):
        td.kernel_fn(x, t[:, :0], ids[:, :0])
    with pytest.raises(ValueError, match="entries"):
        td.kernel_fn(x, torch.randn(3, 257), torch.zeros(3, 257, dtype=torch.int64))
    with pytest.raises(ValueError, match="reduction"):
        td.kernel_fn(x, t, ids, reduction="sum")


@pytest.fixture(scope="module")
def lib():
    if not _lib.is_available():
        pytest.skip("libautokernel_gfx950.so not built")
    return _lib.load()


def test_library_refusals(lib):
    def fwd(logits=16, tokens=None, lp=None, h=None, stats=None, tv=None, ti=None, ws=None, nbytes=0, rows=600,
            vocab=8, ld=8, top=0, temperature=1.0, softcap=0.0, dtype=0):
        return lib.ak_token_logprobs_fwd(logits, tokens, lp, h, stats, tv, ti, ws, nbytes, rows, vocab, ld, top,
                                         temperature, softcap, -100, dtype, None)

    def says(word):
        return word in lib.ak_last_error()

    assert fwd(dtype=7) == -2 and says(b"dtype")
    assert fwd(rows=-1) == -1 and fwd(vocab=0) == -1
    assert fwd(vocab=(1 << 20) + 1, ld=1 << 21) == -2 and says(b"vocab")
    assert fwd(ld=7) == -1 and says(b"pitch")
    assert fwd(rows=1 << 62) == -1 and says(b"addressing")
    for t in (0.0, math.nan, math.inf, 1e20):
        assert fwd(temperature=t) == -1 and says(b"temperature")
    for c in (-1.0, math.nan, math.inf):
        assert fwd(softcap=c) == -1 and says(b"softcap")
    assert fwd(top=9) == -1 and fwd(top=-1) == -1 and says(b"top_k")
    assert fwd(logits=None) == -1 and says(b"null")
    assert fwd(tokens=16) == -1 and fwd(top=2) == -1 and says(b"null")
    assert fwd(stats=8) == -1 and says(b"aligned")
    need = lib.ak_token_logprobs_workspace_bytes(2, 50257, 20, 0)
    assert need > 0 and lib.ak_token_logprobs_workspace_bytes(4096, 50257, 0, 2) == 0
    plain = lib.ak_token_logprobs_workspace_bytes(2, 50257, 0, 0)
    assert fwd(rows=2, vocab=50257, ld=50257, nbytes=plain - 1, ws=256) == -4 and says(b"workspace")
    assert fwd(rows=2, vocab=50257, ld=50257, nbytes=plain) == -4 and 0 < plain < need
    assert fwd(rows=2, vocab=50257, ld=50257, top=20, tv=16, ti=16, nbytes=need, ws=8) == -4 and says(b"workspace")
    assert fwd(rows=0, logits=None) == 0

    def bwd(stats=16, grad=16, ld=8, ldg=8):
        return lib.ak_token_logprobs_bwd(16, None, stats, None, None, grad, 4, 8, ld, ldg, 1.0, 0.0, -100, 0, None)

    assert bwd(stats=None) == -1 and bwd(grad=None) == -1 and says(b"null")
    assert bwd(ldg=7) == -1 and bwd(ld=7) == -1 and says(b"pitch")
    assert bwd(stats=8) == -1 and says(b"aligned")

    def distill(teacher=16, ids=16, losses=16, stats=16, loss=None, scale=None, rows=600, top=2, ldt=2, ldi=2, tdt=0):
        return lib.ak_topk_distill_fwd(16, teacher, ids, losses, stats, loss, scale, None, 0, rows, 8, top, 8, ldt, ldi,
                                       1.0, 0.0, -100, 0, tdt, None)

    assert distill(tdt=9) == -2 and says(b"teacher")
    assert distill(top=0) == -1 and distill(top=257, ldt=300, ldi=300) == -1 and says(b"entries")
    assert distill(ldt=1) == -1 and distill(ldi=1) == -1 and says(b"pitch")
    assert distill(teacher=None) == -1 and distill(ids=None) == -1 and distill(losses=None) == -1
    assert distill(loss=16) == -1 and distill(scale=16) == -1 and says(b"null")
    assert distill(stats=8) == -1 and says(b"aligned")
    assert distill(rows=0, teacher=None, ids=None, losses=None, stats=None) == 0
    assert lib.ak_topk_distill_bwd(16, 16, 16, 16, 16, 2, None, 16, 4, 8, 2, 8, 2, 2, 8, 1.0, 0.0, -100, 0, 0, None) == -1
    assert says(b"grad_stride")


@pytest.mark.parametrize("ve", [4, 8])
def test_workspace_covers_every_shape(lib, ve):
    """The query grows with what the forward writes: one 16-byte partial and top keys a segment."""
    code = {4: 0, 8: 2}[ve]
    for rows in (1, 2, 7, 100, 255, 256, 5000):
        for vocab in (1, 100, 2048, 50257, 1 << 20):
            a = lib.ak_token_logprobs_workspace_bytes(rows, vocab, 0, code)
            b = lib.ak_token_logprobs_workspace_bytes(rows, vocab, min(256, vocab), code)
            segs_least = -(-max(1, vocab // ve) // 8192)
            if rows >= 256:
                assert (a > 0) == (segs_least > 1)
            assert a >= (rows * segs_least * 16 if segs_least > 1 else 0) and (b > 0 or segs_least == 1)


def test_library_refusals_of_the_head(lib):
    def says(word):
        return word in lib.ak_last_error()

    def fwd(h=16, w=16, tok=None, lp=None, stats=None, ws=None, nbytes=0, n=8, v=16, d=64, ldh=64, ldw=64, t=1.0,
            cap=0.0, dtype=2):
        return lib.ak_lmhead_logprobs_fwd(h, w, tok, lp, None, stats, ws, nbytes, n, v, d, ldh, ldw, t, cap, -100, dtype,
                                          None)

    assert fwd(dtype=0) == -2 and says(b"bf16")
    assert fwd(d=100, ldh=104, ldw=104) == -2 and says(b"multiple")
    assert fwd(n=0) == -1 and fwd(v=0) == -1 and fwd(n=1 << 31) == -1 and says(b"shape")
    assert fwd(ldh=63) == -1 and fwd(ldw=65) == -1 and fwd(ldh=1 << 23) == -1 and says(b"pitch")
    assert fwd(h=None) == -1 and fwd(tok=16) == -1 and says(b"null")
    assert fwd(h=8) == -1 and fwd(w=24) == -1 and says(b"aligned")
    assert fwd(stats=4) == -1 and says(b"aligned")
    assert fwd(t=1e-4) == -1 and fwd(t=math.nan) == -1 and says(b"temperature")
    assert fwd(cap=-1.0) == -1 and fwd(cap=math.inf) == -1 and says(b"softcap")
    need = lib.ak_lmhead_logprobs_workspace_bytes(8, 16)
    assert need >= 2 * 8 * 12 and fwd(nbytes=need - 1, ws=16) == -4 and fwd(nbytes=need) == -4
    assert fwd(nbytes=need, ws=24) == -4 and says(b"workspace")

    def bwd(co=16, gl=16, ldg=16, v0=0, vn=16):
        return lib.ak_lmhead_logprobs_bwd_range(16, 16, None, co, gl, ldg, 8, 16, v0, vn, 64, 64, 64, 1.0, 0.0, -100, 2,
                                                None)

    assert bwd(v0=-1) == -1 and bwd(v0=1) == -1 and bwd(vn=0) == -1 and says(b"range")
    assert bwd(co=None) == -1 and bwd(gl=None) == -1 and says(b"null")
    assert bwd(co=8) == -1 and bwd(gl=17) == -1 and says(b"aligned")
    assert bwd(ldg=15) == -1 and says(b"pitch")

    def coefs(stats=16, co=16, n=8, v=16, t=1.0):
        return lib.ak_lmhead_logprobs_coefs(None, stats, None, None, co, n, v, t, -100, None)

    assert coefs(stats=None) == -1 and coefs(co=None) == -1 and says(b"null")
    assert coefs(stats=4) == -1 and coefs(co=8) == -1 and says(b"aligned")
    assert coefs(n=-1) == -1 and coefs(v=0) == -1 and coefs(t=0.0) == -1 and coefs(n=0, stats=None) == 0


def test_softcaps_out_of_range(scoring_backend):
    """Caps whose tanh, within 2^-22 of 1, would say less than the logits (or nothing: 1e-50 is 0 in fp32)."""
    x, tok, ids = torch.randn(3, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int64)
    for bad in (1e-50, 9e-4, 2e4, 1e38):
        with pytest.raises(ValueError, match="softcap"):
            tl.kernel_fn(x, tok, softcap=bad)
        with pytest.raises(ValueError, match="softcap"):
            td.kernel_fn(x, x[:, :2], ids, softcap=bad)
        with pytest.raises(ValueError, match="softcap"):
            ll.kernel_fn(torch.randn(3, 64), torch.randn(8, 64), tok, softcap=bad)
    for good in (1e-3, 1e4):
        tl.kernel_fn(x, tok, softcap=good)


@pytest.mark.parametrize("cap", [1e-40, 9e-4, 2e4, 3e38])
def test_library_refuses_softcaps_out_of_range(lib, cap):
    for rc in (lib.ak_token_logprobs_fwd(16, None, None, None, None, None, None, None, 0, 600, 8, 8, 0, 1.0, cap, -100, 0, None),
               lib.ak_topk_distill_fwd(16, 16, 16, 16, 16, None, None, None, 0, 600, 8, 2, 8, 2, 2, 1.0, cap, -100, 0, 0, None),
               lib.ak_lmhead_logprobs_fwd(16, 16, None, None, None, None, None, 0, 8, 16, 64, 64, 64, 1.0, cap, -100, 2, None)):
        assert rc == -1 and b"softcap" in lib.ak_last_error()


@pytest.mark.parametrize("inside", [True, False])
def test_lmhead_fp32_keeps_its_type_under_autocast(scoring_backend, monkeypatch, inside):
    """The logits of the forward and those that the backward forms again are fp32, and
    results and gradients are those without autocast, inside the block and behind it."""
    seen = []
    for name in ("token_logprobs", "token_logprobs_bwd"):
        fn = getattr(_lib, name)
        monkeypatch.setattr(_lib, name, lambda x, *a, fn=fn: (seen.append(x.dtype), fn(x, *a))[1])
    g = torch.Generator().manual_seed(1)
    h, w = torch.randn(5, 40, generator=g, requires_grad=True), torch.randn(30, 40, generator=g, requires_grad=True)
    tok = torch.tensor([1, 29, -100, 3, 4])

    def call():
        r = ll.kernel_fn(h, w, tok, chunk_size=2)
        return list(r), r.logprobs.sum() + 0.5 * r.entropy.sum()

    outs, total = call()
    want = [*outs, *torch.autograd.grad(total, (h, w))]
    with torch.autocast("cpu", dtype=torch.bfloat16):
        outs, total = call()
        if inside:
            grads = torch.autograd.grad(total, (h, w))
    if not inside:
        grads = torch.autograd.grad(total, (h, w))
    assert set(seen) == {torch.float32} and len(seen) == 12
    assert all(torch.equal(a, b) for a, b in zip([*outs, *grads], want))


def test_forward_mode_is_refused(scoring_backend):
    """A tangent is not dropped, with gradients recorded or not; a teacher is a constant, its tangent too."""
    import torch.autograd.forward_ad as fw
    x, tok, ids = torch.randn(3, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int64)
    h, w = torch.randn(3, 64), torch.randn(8, 64)
    dual = lambda t: fw.make_dual(t, torch.ones_like(t))
    for record in (True, False):
        with fw.dual_level(), torch.set_grad_enabled(record):
            for call in (lambda: tl.kernel_fn(dual(x), tok), lambda: tl.kernel_fn(dual(x), top_k=2),
                         lambda: td.kernel_fn(dual(x), x[:, :2], ids), lambda: ll.kernel_fn(dual(h), w, tok),
                         lambda: ll.kernel_fn(h, dual(w)), lambda: ll.kernel_fn(h.bfloat16(), dual(w), tok)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
            assert fw.unpack_dual(td.kernel_fn(x, dual(x[:, :2]), ids)).tangent is None
            assert tl.kernel_fn(x, tok).logprobs.shape == (3,)  # others as ever
    # an upstream gradient's tangent
    leaf = x.clone().requires_grad_()
    outs = [tl.kernel_fn(leaf, tok).logprobs, td.kernel_fn(leaf, x[:, :2], ids, reduction="none"),
            ll.kernel_fn(h, w.clone().requires_grad_(), tok).entropy]
    for out in outs:
        with fw.dual_level():
            up = dual(torch.ones(3))
            with pytest.raises(RuntimeError, match="forward-mode"):
                out.backward(up)


@pytest.mark.parametrize("cap,temperature", [(1e4, 1e-3), (30.0, 1e-18), (30.0, 2e-5)])
def test_softcaps_that_the_temperature_leaves_without_digits(scoring_backend, cap, temperature):
    """Capped scores are exact to 2^-22 cap / T: a cap over 2^20 temperatures is refused."""
    x, tok, ids = torch.randn(3, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int64)
    kw = dict(softcap=cap, temperature=temperature)
    with pytest.raises(ValueError, match="softcap"):
        tl.kernel_fn(x, tok, **kw)
    with pytest.raises(ValueError, match="softcap"):
        td.kernel_fn(x, x[:, :2], ids, **kw)
    if temperature >= 1e-3:
        with pytest.raises(ValueError, match="softcap"):
            ll.kernel_fn(torch.randn(3, 64), torch.randn(8, 64), tok, **kw)
    tl.kernel_fn(x, tok, softcap=cap, temperature=cap / 2 ** 20)


@pytest.mark.parametrize("cap,t", [(1e4, 1e-3), (30.0, 2e-5)])
def test_library_refuses_softcaps_of_too_many_temperatures(lib, cap, t):
    calls = [lib.ak_token_logprobs_fwd(16, None, None, None, None, None, None, None, 0, 600, 8, 8, 0, t, cap, -100, 0, None),
             lib.ak_token_logprobs_bwd(16, None, 16, None, None, 16, 4, 8, 8, 8, t, cap, -100, 0, None),
             lib.ak_topk_distill_fwd(16, 16, 16, 16, 16, None, None, None, 0, 600, 8, 2, 8, 2, 2, t, cap, -100, 0, 0, None)]
    if t >= 1e-3:
        calls.append(lib.ak_lmhead_logprobs_fwd(16, 16, None, None, None, None, None, 0, 8, 16, 64, 64, 64, t, cap, -100, 2, None))
    assert all(rc == -1 for rc in calls) and b"softcap" in lib.ak_last_error()
