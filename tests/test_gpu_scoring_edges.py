"""GPU tests of the scoring operators where their rules at the edges decide:
ignored rows, saturated softcaps, masks of infinities and lowest values, log
probabilities at their bound, autocast, forward mode, torch.compile, many rows.

Tolerances are those of the row and head tests, whose derivation stands there;
what is added here is derived at its test.
"""

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from test_gpu_lmhead_logprobs import operands
from test_gpu_scoring import DEV

pytestmark = gpu


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
