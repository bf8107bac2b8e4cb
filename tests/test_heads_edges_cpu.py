"""Host-side edges of the operators on attention heads and the paged cache (CPU tier)."""

import pytest
import torch

from kernels.hip import paged_append, paged_attention, qk_norm_rotary, rotary
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
