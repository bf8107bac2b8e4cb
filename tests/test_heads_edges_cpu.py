"""Host-side edges of the operators on attention heads and the paged cache (CPU tier)."""

import pytest
import torch

from kernels.hip import _heads, _lib, paged_append, paged_attention, qk_norm_rotary, rotary
from test_heads_cpu import _cache_call, heads_backend  # noqa: F401 (a fixture)


@pytest.mark.parametrize("mode", ["recorded", "no_grad"])
@pytest.mark.parametrize("name", ["k", "v", "k_cache", "v_cache", "q", "q_weight", "k_weight", "table", "q_out"])
def test_append_refuses_tangents(heads_backend, name, mode):  # noqa: F811
    """A dual tensor's requires_grad is False: the cache operators would drop its tangent."""
    c = dict(_cache_call(), q_weight=torch.ones(6), k_weight=torch.ones(6), table=rotary.rotary_table(6, 9))
    c["q_out"] = torch.zeros_like(c["q"])
    before = c["k_cache"].clone()
    with torch.set_grad_enabled(mode == "recorded"), torch.autograd.forward_ad.dual_level():
        c[name] = torch.autograd.forward_ad.make_dual(c[name], torch.ones_like(c[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged_append.kernel_fn(**c)
    assert torch.equal(c["k_cache"], before)


@pytest.mark.parametrize("mode", ["recorded", "no_grad"])
@pytest.mark.parametrize("name", ["q", "k_cache", "v_cache", "out"])
def test_attention_refuses_tangents(heads_backend, name, mode):  # noqa: F811
    c = _cache_call()
    del c["k"], c["v"]
    c["out"] = torch.zeros_like(c["q"])
    with torch.set_grad_enabled(mode == "recorded"), torch.autograd.forward_ad.dual_level():
        c[name] = torch.autograd.forward_ad.make_dual(c[name], torch.ones_like(c[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged_attention.kernel_fn(**c)


def test_training_operators_refuse_a_tables_tangents(heads_backend):  # noqa: F811
    x, w, t = torch.randn(3, 1, 6), torch.ones(6), rotary.rotary_table(6, 3)
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: rotary.kernel_fn(x, None, t), lambda: qk_norm_rotary.kernel_fn(x, None, w, None, t)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.skipif(not _lib.is_available(), reason="libautokernel_gfx950.so not built")
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_attention_workspace_keeps_its_parts_aligned(dtype):
    """Behind the line and the jobs stand parts that are read and written 16 bytes at a time: with
    an odd number of workers, of many rows, their base has to be a multiple of 16 all the same.
    (Parts of many rows are whole multiples of 16 bytes, so the total tells the base.)"""
    size = _lib.load().ak_paged_attention_workspace_bytes
    for tokens, batch, heads, dim, keys in ((150, 1, 2, 64, 192), (150, 1, 2, 128, 192), (150, 1, 1, 64, 192), (130, 1, 3, 64, 130),
                                            (77, 1, 1, 64, 200), (333, 3, 5, 64, 64), (999, 2, 7, 256, 250)):
        need = size(tokens, batch, heads, heads, dim, keys, tokens, dtype)
        assert need > 0 and need % 16 == 0, (tokens, batch, heads, dim, keys, need)


def test_shared_memory_is_told():
    """Against the sets of places, over random views of one buffer; what it cannot tell is False."""
    import random
    rng = random.Random(1)

    def view(base):
        kind = rng.randrange(4)
        if kind == 0:
            n = rng.randint(1, 40)
            return base[rng.randint(0, 200):][:n]
        rows, pitch = rng.randint(1, 6), rng.randint(6, 30)
        heads, dim = rng.randint(1, 3), rng.randint(1, 3)
        if kind == 1:
            pitch = 20
        dims = (rows, heads, dim), (pitch, dim, 1)
        if kind == 3:
            dims = (heads, rows, dim), (dim, pitch, 1)
        return base.as_strided(*dims, rng.randint(0, 150))

    base, places = torch.zeros(600), torch.arange(600.0)
    told = 0
    for _ in range(3000):
        state = rng.getstate()
        a, b = view(base), view(base)
        rng.setstate(state)
        pa, pb = view(places), view(places)
        meet = bool(set(pa.reshape(-1).tolist()) & set(pb.reshape(-1).tolist()))
        got = _heads.share_memory(a, b)
        assert got == _heads.share_memory(b, a) and (meet or not got)
        x, y = _heads._spans(a), _heads._spans(b)
        if x is not None and y is not None and (x[0] == 1 or y[0] == 1 or x[1] == y[1]):
            assert got == meet, (a.shape, a.stride(), b.shape, b.stride())
            told += meet
    assert told > 300
    assert not _heads.share_memory(base[:0], base)


def test_outputs_that_share_memory(heads_backend):  # noqa: F811
    """A kernel's rows are read and written in no order: an output is apart from what is read
    beside it, or the queries themselves."""
    fused = torch.randn(5, 8, 6)
    c = dict(_cache_call(), q=fused[:, :4], k=fused[:, 4:6], v=fused[:, 6:])
    paged_append.kernel_fn(**c, q_out=c["q"])
    for q_out, text in ((fused[:, 1:5], "q"), (fused[:, 4:], "k"), (fused[:, 2:6], "q")):
        with pytest.raises(ValueError, match=f"q_out shares memory with {text}"):
            paged_append.kernel_fn(**c, q_out=q_out)
    both = torch.zeros(c["k_cache"].shape[0] + 1, 4, 2, 6)
    with pytest.raises(ValueError, match="k_cache shares memory with v_cache"):
        paged_append.kernel_fn(**dict(c, k_cache=both[1:], v_cache=both[:-1]))
    pair = torch.zeros(c["k_cache"].shape[0], 2, 4, 2, 6)
    paged_append.kernel_fn(**dict(c, k_cache=pair[:, 0], v_cache=pair[:, 1]))
    long = torch.randn(7, 4, 6)
    a = dict(q=long[1:6], k_cache=c["k_cache"], v_cache=c["v_cache"], page_table=c["page_table"], lengths=c["lengths"],
             starts=c["starts"])
    for out, text in ((long[:5], "q"), (long[2:], "q"), (c["k_cache"].view(-1, 4, 6)[:5], "k_cache")):
        with pytest.raises(ValueError, match=f"out shares memory with {text}"):
            paged_attention.kernel_fn(**a, out=out)
    assert paged_attention.kernel_fn(**a, out=a["q"]) is a["q"]
