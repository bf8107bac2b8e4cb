"""Host logic of the operators on attention heads and the paged cache (CPU tier):
the launchers are routed to the float64 oracle, so these tests check shapes, types,
autograd contracts and refusals; the library's own refusals return before any HIP call."""

import ctypes
import math

import pytest
import torch

from heads_util import make_batch
from kernels.hip import _heads, _lib, paged_append, paged_attention, qk_norm_rotary, rotary
from oracle import heads as oracle


def _positions(positions, n, tokens):
    p = torch.arange(n) if positions is None else positions.reshape(-1)
    return p[torch.arange(tokens) % n].long()


@pytest.fixture
def heads_backend(monkeypatch):
    def forward(q, k, wq, wk, table, positions, n, q_out, k_out, eps, interleaved, inverse):
        for h, w, out in ((q, wq, q_out), (k, wk, k_out)):
            if h is None:
                continue
            assert h.t.shape == (h.outer, h.inner, h.heads, h.dim) and out.is_contiguous()
            x = h.t.reshape(-1, h.heads, h.dim)
            t = table
            if inverse:
                t = table.clone()
                t[:, t.shape[1] // 2:] *= -1
            y = oracle.norm_turn(x, w, eps, t, _positions(positions, n, len(x)), interleaved)
            out.copy_(y.reshape(out.shape))

    def backward(q, k, wq, wk, table, positions, n, gq, gk, dq, dk, dwq, dwk, ws, eps, interleaved):
        for h, w, g, dx, dw in ((q, wq, gq, dq, dwq), (k, wk, gk, dk, dwk)):
            if h is None:
                continue
            x, up = h.t.reshape(-1, h.heads, h.dim), g.t.reshape(-1, h.heads, h.dim)
            a, b = oracle.norm_turn_grad(x, w, eps, table, _positions(positions, n, len(x)), up, interleaved)
            dx.copy_(a.reshape(dx.shape))
            if dw is not None:
                dw.copy_(b)

    def append(q, k, v, wq, wk, table, q_out, kc, vc, batch, eps, interleaved, zero):
        a, b, c = oracle.append(q, k, v, kc, vc, batch.pages, batch.lengths, batch.starts, wq, wk, eps, table, interleaved)
        kc.copy_(b)
        vc.copy_(c)
        if q is not None:
            q_out.copy_(torch.where(torch.isnan(a), 0.0 if zero else q_out.double(), a))

    def attend(q, kc, vc, batch, out, chunk, scale, softcap, window, zero):
        assert 1 <= chunk <= max(1, q.shape[0])
        out.copy_(oracle.attend(q, kc, vc, batch.pages, batch.lengths, batch.starts, scale, softcap, window))

    for name, fn in (("qk_norm_rotary", forward), ("qk_norm_rotary_bwd", backward), ("paged_append", append),
                     ("paged_attention", attend), ("require_device", lambda *t: None),
                     ("qk_norm_rotary_bwd_workspace_bytes", lambda *a: 256)):
        monkeypatch.setattr(_lib, name, fn)


# ---------------------------------------------------------------------------
# The oracle
# ---------------------------------------------------------------------------
def test_oracle_known_answers():
    # a quarter turn of the first pair, position 0 as it was
    cos, sin = torch.tensor([[1.0], [0.0]]), torch.tensor([[0.0], [1.0]])
    x = torch.tensor([[[3.0, 4.0, 7.0]], [[3.0, 4.0, 7.0]]])
    assert oracle.turn(x, cos, sin).tolist() == [[[3.0, 4.0, 7.0]], [[-4.0, 3.0, 7.0]]]
    # halves and neighbours pair the same elements once they are reordered
    g = torch.Generator().manual_seed(0)
    y = torch.randn(5, 2, 8, generator=g)
    a = oracle.angles(torch.arange(5), 8)
    shuffle = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7])
    assert torch.allclose(oracle.turn(y, a.cos(), a.sin())[..., shuffle], oracle.turn(y[..., shuffle], a.cos(), a.sin(), True))
    # scores of turned heads depend on the distance alone
    q, k = torch.randn(1, 1, 8, generator=g), torch.randn(1, 1, 8, generator=g)

    def score(p, j):
        t = [oracle.turn(x, a.cos(), a.sin()) for x, a in ((q, oracle.angles(torch.tensor([p]), 8)),
                                                            (k, oracle.angles(torch.tensor([j]), 8)))]
        return float((t[0] * t[1]).sum())

    assert score(9, 5) == pytest.approx(score(104, 100), rel=1e-12)


def test_oracle_gradient_is_autograd():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(4, 3, 6, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64)
    up = torch.randn(4, 3, 6, generator=g, dtype=torch.float64)
    table = torch.cat([oracle.angles(torch.arange(4), 4).cos(), oracle.angles(torch.arange(4), 4).sin()], 1)
    for inter in (False, True):
        lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = oracle.norm_turn(lx, lw, 1e-3, table, torch.arange(4), inter)
        want = torch.autograd.grad(y, (lx, lw), up)
        got = oracle.norm_turn_grad(x, w, 1e-3, table, torch.arange(4), up, inter)
        assert all(torch.allclose(a, b, rtol=1e-10, atol=1e-12) for a, b in zip(got, want))


def test_oracle_attention_is_causal_softmax():
    g = torch.Generator().manual_seed(2)
    n, page = 13, 4
    pages, lens, starts, total = make_batch([n], [n], page, 3)
    q = torch.randn(n, 4, 8, generator=g).double()
    k, v = torch.randn(n, 2, 8, generator=g).double(), torch.randn(n, 2, 8, generator=g).double()
    kc, vc = torch.full((total, page, 2, 8), math.nan), torch.full((total, page, 2, 8), math.nan)
    kc, vc = oracle.append(None, k, v, kc, vc, pages, lens, starts, None, None, 0.0, None, False)[1:]
    for window in (0, 5):
        got = oracle.attend(q, kc, vc, pages, lens, starts, 0.3, 0.0, window)
        i = torch.arange(n)
        hide = i[None, :] > i[:, None]
        if window:
            hide = hide | (i[None, :] <= i[:, None] - window)
        for h in range(4):
            s = (q[:, h] @ k[:, h // 2].t() * 0.3).masked_fill(hide, -math.inf)
            assert torch.allclose(got[:, h], torch.softmax(s, -1) @ v[:, h // 2])


# ---------------------------------------------------------------------------
# Tables
# ---------------------------------------------------------------------------
def test_rotary_table():
    t = rotary.rotary_table(8, 5)
    a = oracle.angles(torch.arange(5), 8)
    assert t.shape == (5, 8) and t.dtype == torch.float32 and t.is_contiguous()
    assert torch.equal(t, torch.cat([a.cos(), a.sin()], 1).float())
    far = rotary.rotary_table(2, (1 << 24) + 10)  # made in parts
    assert far[-1, 0] == torch.cos(torch.tensor(float((1 << 24) + 9), dtype=torch.float64)).float()
    f = rotary.rotary_frequencies(64)
    lin = rotary.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(lin, f / 4)
    ntk = rotary.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == f[0] and float(ntk[-1]) == pytest.approx(float(f[-1]) / 4, rel=1e-12)
    yarn = rotary.rotary_frequencies(64, scaling="yarn", factor=4.0, original_positions=2048)
    turns = 2048 * f / (2 * math.pi)
    fast, slow = turns >= 32 * 1.4, turns <= 1 / 1.4  # (a pair's index is rounded outward)
    assert torch.equal(yarn[fast], f[fast]) and torch.allclose(yarn[slow], f[slow] / 4) and fast.any() and slow.any()
    assert (yarn <= f).all() and (yarn >= f / 4 * (1 - 1e-12)).all()
    scaled = rotary.rotary_table(64, 3, scaling="yarn", factor=4.0, original_positions=2048)
    assert float(scaled[0, 0]) == pytest.approx(0.1 * math.log(4.0) + 1, rel=1e-6) and scaled[0, 32] == 0
    plain = rotary.rotary_table(64, 3, scaling="yarn", factor=4.0, original_positions=2048, attention_factor=1.0)
    assert plain[0, 0] == 1


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(positions=0), dict(scaling="other"),
                                dict(factor=2.0), dict(factor=0.5, scaling="linear"), dict(base=1.0), dict(base=math.inf),
                                dict(scaling="yarn", factor=2.0), dict(scaling="ntk", rotary_dim=2, factor=2.0),
                                dict(scaling="linear", factor=math.nan),
                                dict(scaling="yarn", factor=2.0, original_positions=10, beta_fast=0.5)], ids=str)
def test_rotary_table_refusals(kw):
    kw = {"rotary_dim": 8, "positions": 4, **kw}
    with pytest.raises(ValueError):
        rotary.rotary_table(kw.pop("rotary_dim"), kw.pop("positions"), **kw)


# ---------------------------------------------------------------------------
# Rotary positions and head norms
# ---------------------------------------------------------------------------
def test_no_cpu_fallback():
    x, w, t = torch.randn(2, 1, 4), torch.ones(4), rotary.rotary_table(4, 2)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary.kernel_fn(x, None, t)
    with pytest.raises(RuntimeError, match="GPU"):
        qk_norm_rotary.kernel_fn(x, None, w, None)
    c = torch.zeros(1, 4, 1, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_append.kernel_fn(x, x, c, c.clone(), i, i[0])
    with pytest.raises(RuntimeError, match="GPU"):
        paged_attention.kernel_fn(x, c, c, i, i[0])


def test_shapes_types_and_gradients(heads_backend):
    g = torch.Generator().manual_seed(3)
    table = rotary.rotary_table(4, 9)
    for lead in ((), (5,), (2, 5), (2, 2, 3)):
        q = torch.randn(*lead, 3, 6, generator=g).bfloat16().requires_grad_()
        k = torch.randn(*lead, 2, 6, generator=g).bfloat16().requires_grad_()
        a, b = rotary.kernel_fn(q, k, table)
        assert a.shape == q.shape and b.shape == k.shape and a.dtype == b.dtype == torch.bfloat16
        (a.sum() + 2 * b.sum()).backward()
        assert q.grad.shape == q.shape and k.grad.dtype == k.dtype
        assert rotary.kernel_fn(q.detach(), None, table)[1] is None
        assert not rotary.kernel_fn(q.detach(), k.detach(), table)[0].requires_grad
        with torch.no_grad():
            assert not rotary.kernel_fn(q, k, table)[0].requires_grad
        w = torch.ones(6, requires_grad=True)
        y, _ = qk_norm_rotary.kernel_fn(q, None, w, None, table)
        y.float().square().sum().backward()
        assert w.grad.shape == (6,) and w.grad.dtype == torch.float32
    q = torch.randn(0, 3, 6, requires_grad=True)
    rotary.kernel_fn(q, None, table)[0].sum().backward()
    assert q.grad.shape == (0, 3, 6)


def test_views_are_read_in_place(heads_backend):
    fused = torch.randn(2, 5, 7, 6)
    for x in (fused[:, :, 1:4], fused.transpose(1, 2).contiguous().transpose(1, 2), fused[:, ::2], fused[:1].expand(4, 5, 7, 6)):
        h = _heads.as_heads(x, "x")
        assert h.t.data_ptr() == x.data_ptr() and h.strides == x.stride()[:3]
    h = _heads.as_heads(fused.transpose(-1, -2), "x")  # not dense: copied
    assert h.t.stride(3) == 1 and torch.equal(h.t, fused.transpose(-1, -2))


@pytest.mark.parametrize("make, error, text", [
    (lambda q, k, t: (q, k.half(), t), TypeError, "q is"),
    (lambda q, k, t: (q.double(), None, t), TypeError, "dtype"),
    (lambda q, k, t: (q, k[:1], t), ValueError, "differ in heads"),
    (lambda q, k, t: (q, k[..., :4], t), ValueError, "differ in heads"),
    (lambda q, k, t: (q[0, 0, 0], None, t), ValueError, "heads, dim"),
    (lambda q, k, t: (q, k, t.double()), ValueError, "table"),
    (lambda q, k, t: (q, k, t[:, :3]), ValueError, "table"),
    (lambda q, k, t: (q, k, t.repeat(1, 2)), ValueError, "table"),
    (lambda q, k, t: (q, k, t[0]), ValueError, "table"),
    (lambda q, k, t: (q, k, t[:0]), ValueError, "table"),
    (lambda q, k, t: (q, k, t.clone().requires_grad_()), ValueError, "constants"),
    (lambda q, k, t: (q, k, t, torch.zeros(2, 5)), TypeError, "whole"),
    (lambda q, k, t: (q, k, t, torch.zeros(2, 5, dtype=torch.bool)), TypeError, "whole"),
    (lambda q, k, t: (q, k, t, torch.zeros(2, 4, dtype=torch.int64)), ValueError, "positions"),
    (lambda q, k, t: (q, k, t, torch.zeros(1, 2, 5, dtype=torch.int64)), ValueError, "positions"),
    (lambda q, k, t: (torch.zeros(2, 1, 2050), None, t), ValueError, "2048"),
], ids=str)
def test_rotary_refusals(heads_backend, make, error, text):
    q, k, t = torch.randn(2, 5, 3, 6), torch.randn(2, 5, 1, 6), rotary.rotary_table(6, 9)
    with pytest.raises(error, match=text):
        rotary.kernel_fn(*make(q, k, t))


def test_norm_refusals(heads_backend):
    q, k, w, t = torch.randn(5, 3, 6), torch.randn(5, 1, 6), torch.ones(6), rotary.rotary_table(6, 9)
    for args, error in (((q, k, w, None), "k_weight"), ((q, k, None, w), "q_weight"), ((q, None, w, w), "without k"),
                        ((q, k, w[:5], w), "does not match"), ((q, k, w, w, None, torch.arange(5)), "without a table")):
        with pytest.raises(ValueError, match=error):
            qk_norm_rotary.kernel_fn(*args)
    for eps in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            qk_norm_rotary.kernel_fn(q, k, w, w, t, eps=eps)
    x = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(qk_norm_rotary.kernel_fn(x, None, w, None)[0].square().sum(), x, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: rotary.kernel_fn(d, None, t), lambda: qk_norm_rotary.kernel_fn(d, None, w, None)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_rotary_second_derivative(heads_backend):
    x = torch.randn(3, 2, 6, dtype=torch.float32, requires_grad=True)
    t = rotary.rotary_table(6, 3)
    (g,) = torch.autograd.grad((rotary.kernel_fn(x, None, t)[0] ** 2).sum() / 2, x, create_graph=True)
    assert torch.allclose(g, x, atol=1e-6)
    (h,) = torch.autograd.grad((g * torch.ones_like(g)).sum(), x)
    assert torch.allclose(h, torch.ones_like(h), atol=1e-6)


# ---------------------------------------------------------------------------
# The paged cache
# ---------------------------------------------------------------------------
def _cache_call():
    pages, lens, starts, total = make_batch([3, 2], [7, 2], 4, 5)
    k, v, q = torch.randn(5, 2, 6), torch.randn(5, 2, 6), torch.randn(5, 4, 6)
    return dict(k=k, v=v, k_cache=torch.zeros(total, 4, 2, 6), v_cache=torch.zeros(total, 4, 2, 6), page_table=pages,
                lengths=lens, starts=starts, q=q)


def test_append_and_attend(heads_backend):
    c = _cache_call()
    t = rotary.rotary_table(6, 9)
    version = c["k_cache"]._version
    q = paged_append.kernel_fn(**c, table=t)
    assert q.shape == c["q"].shape and c["k_cache"]._version > version and c["v_cache"]._version > 0
    out = paged_attention.kernel_fn(q, c["k_cache"], c["v_cache"], c["page_table"], c["lengths"], c["starts"])
    assert out.shape == q.shape
    same = torch.empty_like(q)
    assert paged_attention.kernel_fn(q, c["k_cache"], c["v_cache"], c["page_table"], c["lengths"], c["starts"], out=same,
                                     max_chunk=1000) is same
    assert torch.equal(same, out)
    c.pop("q")
    assert paged_append.kernel_fn(**c) is None
    with torch.inference_mode():
        i = {k: v.clone() for k, v in c.items()}
        assert paged_append.kernel_fn(**i) is None
    w = torch.ones(6, requires_grad=True)
    with torch.no_grad():
        paged_append.kernel_fn(**c, k_weight=w)


@pytest.mark.parametrize("change, error, text", [
    (lambda c: c.update(k=c["k"][0]), ValueError, "k and v"),
    (lambda c: c.update(v=c["v"][:, :1]), ValueError, "k and v"),
    (lambda c: c.update(v=c["v"].half()), TypeError, "v is"),
    (lambda c: c.update(k=c["k"].double(), v=c["v"].double()), TypeError, "dtype"),
    (lambda c: c.update(k_cache=c["k_cache"].half()), TypeError, "k_cache"),
    (lambda c: c.update(k_cache=c["k_cache"][:, :, :1]), ValueError, "k_cache"),
    (lambda c: c.update(k_cache=c["k_cache"][:, :0]), ValueError, "k_cache"),
    (lambda c: c.update(v_cache=c["v_cache"][1:]), ValueError, "differ"),
    (lambda c: c.update(v_cache=c["v_cache"][:1].expand_as(c["v_cache"])), ValueError, "share"),
    (lambda c: c.update(v_cache=c["k_cache"]), ValueError, "same place"),
    (lambda c: c.update(k_cache=torch.zeros(*c["k_cache"].shape[:3], 12)[..., ::2]), ValueError, "dense"),
    (lambda c: c.update(page_table=c["page_table"].long()), TypeError, "int32"),
    (lambda c: c.update(page_table=c["page_table"][0]), ValueError, "page_table"),
    (lambda c: c.update(lengths=c["lengths"].long()), TypeError, "int32"),
    (lambda c: c.update(lengths=c["lengths"][:1]), ValueError, "batches"),
    (lambda c: c.update(starts=c["starts"].long()), TypeError, "int32"),
    (lambda c: c.update(starts=c["starts"][:2]), ValueError, "batch \\+ 1"),
    (lambda c: c.update(starts=None), ValueError, "same number"),
    (lambda c: c.update(q=c["q"][:4]), ValueError, "q must"),
    (lambda c: c.update(q=c["q"].half()), TypeError, "q is"),
    (lambda c: c.update(q=None, q_weight=torch.ones(6)), ValueError, "without q"),
    (lambda c: c.update(q=None, q_out=torch.ones(5, 4, 6)), ValueError, "without q"),
    (lambda c: c.update(q_out=torch.ones(5, 4, 7)), ValueError, "q_out"),
    (lambda c: c.update(q_out=torch.ones(1, 4, 6).expand(5, 4, 6)), ValueError, "q_out"),
    (lambda c: c.update(k_weight=torch.ones(5)), ValueError, "k_weight"),
    (lambda c: c.update(eps=-1.0), ValueError, "eps"),
    (lambda c: c.update(table=torch.zeros(4, 8)), ValueError, "table"),
    (lambda c: c.update(k=c["k"].requires_grad_()), RuntimeError, "no gradient"),
    (lambda c: c.update(k_weight=torch.ones(6, requires_grad=True)), RuntimeError, "no gradient"),
    (lambda c: c.update(v_cache=c["v_cache"].requires_grad_()), RuntimeError, "no gradient"),
], ids=str)
def test_append_refusals(heads_backend, change, error, text):
    c = _cache_call()
    change(c)
    with pytest.raises(error, match=text):
        paged_append.kernel_fn(**c)


@pytest.mark.parametrize("change, error, text", [
    (lambda c: c.update(q=c["q"][0]), ValueError, "q must"),
    (lambda c: c.update(q=c["q"][:, :3]), ValueError, "evenly"),
    (lambda c: c.update(q=c["q"][:, :0]), ValueError, "evenly"),
    (lambda c: c.update(q=torch.zeros(5, 4, 1030)), ValueError, "1024"),
    (lambda c: c.update(q=c["q"].half()), TypeError, "k_cache"),
    (lambda c: c.update(q=c["q"].double()), TypeError, "dtype"),
    (lambda c: c.update(q=c["q"][..., :4]), ValueError, "k_cache"),
    (lambda c: c.update(v_cache=c["v_cache"][1:]), ValueError, "differ"),
    (lambda c: c.update(scale=0.0), ValueError, "scale"),
    (lambda c: c.update(scale=-1.0), ValueError, "scale"),
    (lambda c: c.update(scale=math.nan), ValueError, "scale"),
    (lambda c: c.update(scale=math.inf), ValueError, "scale"),
    (lambda c: c.update(softcap=-1.0), ValueError, "softcap"),
    (lambda c: c.update(softcap=1e-9), ValueError, "softcap"),
    (lambda c: c.update(softcap=math.nan), ValueError, "softcap"),
    (lambda c: c.update(window=-1), ValueError, "window"),
    (lambda c: c.update(max_chunk=0), ValueError, "max_chunk"),
    (lambda c: c.update(starts=c["starts"].long()), TypeError, "int32"),
    (lambda c: c.update(starts=None), ValueError, "same number"),
    (lambda c: c.update(out=torch.zeros(5, 4, 7)), ValueError, "out"),
    (lambda c: c.update(out=torch.zeros(5, 4, 6).half()), ValueError, "out"),
    (lambda c: c.update(out=torch.zeros(5, 1, 6).expand(5, 4, 6)), ValueError, "out"),
    (lambda c: c.update(q=c["q"].requires_grad_()), RuntimeError, "no gradient"),
    (lambda c: c.update(k_cache=c["k_cache"].requires_grad_()), RuntimeError, "no gradient"),
], ids=str)
def test_attention_refusals(heads_backend, change, error, text):
    c = _cache_call()
    del c["k"], c["v"]
    change(c)
    with pytest.raises(error, match=text):
        paged_attention.kernel_fn(**c)


def test_places_that_share_memory():
    x = torch.zeros(4, 3, 2, 5)
    for good in (x, x.transpose(1, 2), x[::2], x[:, :1], x.permute(3, 1, 0, 2), x[:0], torch.zeros(())):
        assert _heads.dense_places(good)
    for bad in (x[:1].expand(4, 3, 2, 5), torch.zeros(20).as_strided((4, 6), (3, 1))):
        assert not _heads.dense_places(bad)


# ---------------------------------------------------------------------------
# The library's refusals (no HIP call is made)
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    if not _lib.is_available():
        pytest.skip("libautokernel_gfx950.so not built")
    return _lib.load()


P = 4096  # stands for a pointer; never followed


def norm_args(**kw):
    d = dict(q=P, k=P, q_weight=P, k_weight=P, table=P, positions=None, q_out=P, k_out=P, outer=1, inner=2, q_heads=2, k_heads=1,
             dim=8, rotary=8, table_rows=4, n_positions=2, q_so=32, q_si=16, q_sh=8, k_so=16, k_si=8, k_sh=8, eps=1e-6, flags=0,
             dtype=2, stream=None)
    d.update(kw)
    return list(d.values())


@pytest.mark.parametrize("kw, code", [
    (dict(dtype=3), -2), (dict(dim=0), -2), (dict(dim=2049), -2), (dict(rotary=7), -1), (dict(rotary=10), -1), (dict(table=None), -1),
    (dict(table_rows=0), -1), (dict(eps=-1.0), -1), (dict(eps=math.nan), -1), (dict(eps=math.inf), -1), (dict(q_heads=-1), -1),
    (dict(outer=-1), -1), (dict(q_si=-16), -1), (dict(inner=2 ** 62), -1), (dict(q_si=2 ** 62), -1), (dict(n_positions=0), -1),
    (dict(q=None), -1), (dict(k_out=None), -1), (dict(k_weight=None), -1)], ids=str)
def test_norm_entry_refusals(lib, kw, code):
    assert lib.ak_qk_norm_rotary_fwd(*norm_args(**kw)) == code and lib.ak_last_error()


def test_norm_entry_empty(lib):
    assert lib.ak_qk_norm_rotary_fwd(*norm_args(inner=0)) == 0
    assert lib.ak_qk_norm_rotary_fwd(*norm_args(q_heads=0, k_heads=0)) == 0
    size = lib.ak_qk_norm_rotary_bwd_workspace_bytes
    assert size(0, 4, 2, 64) == 0 and size(10, 4, 2, 64) % 16 == 0 and size(10 ** 9, 4, 2, 64) <= 2048 * 64 * 4


def test_norm_backward_entry_refusals(lib):
    size = lib.ak_qk_norm_rotary_bwd_workspace_bytes(2, 2, 1, 8)
    a = dict(zip("qkwvtpabcdefW", [P] * 13))
    good = list(a.values()) + [size] + [1, 2, 2, 1, 8, 8, 4, 2] + [32, 16, 8, 16, 8, 8] * 2 + [1e-6, 0, 2, None]
    for i, bad, code in ((13, size - 1, -4), (12, None, -4), (0, None, -1), (9, None, -1), (8, None, -1), (18, 4096, -2),
                         (19, 5, -1), (21, 0, -1), (28, -1, -1), (34, -1.0, -1), (36, 9, -2)):
        args = list(good)
        args[i] = bad
        assert lib.ak_qk_norm_rotary_bwd(*args) == code, (i, bad)


def paged_args(entry, **kw):
    if entry == "append":
        d = dict(q=P, k=P, v=P, q_weight=None, k_weight=None, table=P, q_out=P, k_cache=P, v_cache=P, page_table=P, lengths=P,
                 starts=P, tokens=3, batch=2, q_heads=4, kv_heads=2, dim=64, rotary=64, table_rows=9, n_pages=5, page_size=16,
                 max_pages=3, ld_pages=3, q_st=256, q_sh=64, k_st=128, k_sh=64, v_st=128, v_sh=64, qo_st=256, qo_sh=64,
                 kc_sp=2048, kc_ss=128, kc_sh=64, vc_sp=2048, vc_ss=128, vc_sh=64, eps=1e-6, flags=0, dtype=2, stream=None)
    else:
        d = dict(q=P, k_cache=P, v_cache=P, page_table=P, lengths=P, starts=P, out=P, workspace=P, workspace_bytes=1 << 40, tokens=3,
                 batch=2, q_heads=4, kv_heads=2, dim=64, n_pages=5, page_size=16, max_pages=3, ld_pages=3, max_chunk=3, q_st=256,
                 q_sh=64, o_st=256, o_sh=64, kc_sp=2048, kc_ss=128, kc_sh=64, vc_sp=2048, vc_ss=128, vc_sh=64, scale=0.1,
                 softcap=0.0, window=0, flags=0, dtype=2, stream=None)
    assert set(kw) <= set(d), kw
    d.update(kw)
    return list(d.values())


COMMON = [(dict(dtype=7), -2), (dict(dim=0), -2), (dict(dim=5000), -2), (dict(tokens=-1), -1), (dict(batch=-1), -1),
          (dict(page_size=0), -1), (dict(n_pages=-1), -1), (dict(max_pages=-1), -1), (dict(ld_pages=2), -1), (dict(lengths=None), -1),
          (dict(page_table=None), -1), (dict(starts=None), -1), (dict(starts=None, batch=0), -1), (dict(kv_heads=0), -1),
          (dict(kc_ss=-1), -1), (dict(vc_sp=2 ** 62), -1), (dict(q=None), -1), (dict(k_cache=None), -1), (dict(tokens=2 ** 31), -1)]


@pytest.mark.parametrize("kw, code", COMMON + [(dict(rotary=65), -1), (dict(table=None), -1), (dict(eps=-1.0), -1),
                                               (dict(q_out=None), -1), (dict(k=None), -1), (dict(v=None), -1),
                                               (dict(q_heads=-1), -1)], ids=str)
def test_append_entry_refusals(lib, kw, code):
    assert lib.ak_paged_append(*paged_args("append", **kw)) == code and lib.ak_last_error()
    assert lib.ak_paged_append(*paged_args("append", tokens=0)) == 0


@pytest.mark.parametrize("kw, code", COMMON + [(dict(q_heads=3), -1), (dict(scale=0.0), -1), (dict(scale=math.nan), -1),
                                               (dict(softcap=-1.0), -1), (dict(window=-1), -1), (dict(out=None), -1),
                                               (dict(max_pages=2 ** 30, ld_pages=2 ** 30), -1)], ids=str)
def test_attention_entry_refusals(lib, kw, code):
    assert lib.ak_paged_attention(*paged_args("attend", **kw)) == code and lib.ak_last_error()
    assert lib.ak_paged_attention(*paged_args("attend", tokens=0)) == 0


def test_attention_workspace(lib):
    size = lib.ak_paged_attention_workspace_bytes
    need = size(2, 2, 32, 8, 128, 100000, 1, 2)
    assert need > 0
    args = paged_args("attend", tokens=2, starts=None, q_heads=32, kv_heads=8, dim=128, max_pages=6250, ld_pages=6250, max_chunk=1,
                      workspace_bytes=need - 1)
    assert lib.ak_paged_attention(*args) == -4
    args[args.index(need - 1)] = need
    args[7] = P + 8  # not aligned
    assert lib.ak_paged_attention(*args) == -4
    assert size(0, 2, 32, 8, 128, 100000, 1, 2) == 0 and size(5, 0, 32, 8, 128, 100000, 1, 2) == 0
    assert isinstance(need, int) and ctypes.sizeof(ctypes.c_size_t) == 8
