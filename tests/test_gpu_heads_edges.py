"""Edges of the operators on attention heads and the paged cache on the GPU."""

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from heads_util import make_batch

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
