"""Host-side edges of the operators on attention heads and the paged cache (CPU tier)."""

import pytest
import torch

from kernels.hip import _lib, paged_append, paged_attention, qk_norm_rotary, rotary
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
