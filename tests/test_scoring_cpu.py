"""Host logic of the scoring operators (CPU tier): the launchers are routed to
the float64 oracle, so these tests check shapes, types, autograd contracts and
refusals; the library's own refusals return before any HIP call."""

import math

import pytest
import torch

from kernels.hip import _lib
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

    for name, fn in (("token_logprobs", logprobs), ("token_logprobs_bwd", logprobs_bwd), ("topk_distill", distill),
                     ("topk_distill_bwd", distill_bwd), ("require_device", lambda *t: None)):
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
    (g,) = torch.autograd.grad(r.logprobs.double().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_distillation_contract(scoring_backend):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 11, generator=g, requires_grad=True)
    t = torch.randn(2, 3, 4, generator=g).half()
    ids = torch.randint(0, 11, (2, 3, 4), generator=g)
    ids[0, 0] = -100
    ids[1, 1, 2:] = -100
    loss = td.kernel_fn(x, t, ids, temperature=2.0)
    rows = td.kernel_fn(x, t, ids, temperature=2.0, reduction="none")
    assert loss.shape == () and rows.shape == (2, 3) and float(rows[0, 0]) == 0
    assert float(loss) == pytest.approx(float(rows.sum()) / 5, rel=1e-6)
    (gx,) = torch.autograd.grad(loss, x, torch.tensor(0.5))
    (gr,) = torch.autograd.grad(rows, x, torch.full((2, 3), 0.1))
    assert torch.allclose(gx, gr, atol=1e-7)
    # every row without entries; no rows
    assert float(td.kernel_fn(x, t, torch.full_like(ids, -100))) == 0
    assert float(td.kernel_fn(x[:0], t[:0], ids[:0])) == 0
    assert td.kernel_fn(x[:0], t[:0], ids[:0], reduction="none").shape == (0, 3)
    # a teacher that requires a gradient is a constant
    assert not td.kernel_fn(x.detach(), t.clone().requires_grad_(), ids).requires_grad


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
    assert need > 0 and lib.ak_token_logprobs_workspace_bytes(4096, 50257, 20, 2) == 0
    assert fwd(rows=2, vocab=50257, ld=50257, nbytes=need - 1, ws=256) == -4 or need == 0
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
