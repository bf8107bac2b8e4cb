"""The scoring oracle against known answers, differences and torch autograd (CPU tier)."""

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import scoring


def test_known_answers():
    x = torch.tensor([[0.0, math.log(2.0), math.log(3.0)]])
    lp, h = scoring.logprob_rows(x, torch.tensor([1]))
    p = [1 / 6, 1 / 3, 1 / 2]
    assert float(lp) == pytest.approx(math.log(1 / 3), rel=1e-6)  # (the inputs are rounded)
    assert float(h) == pytest.approx(-sum(q * math.log(q) for q in p), rel=1e-6)
    top, ids = scoring.top_rows(x, 2)
    assert ids.tolist() == [[2, 1]] and float(top[0, 0]) == pytest.approx(math.log(1 / 2), rel=1e-6)
    # uniform rows: entropy ln V, ties by column; an empty row; NaN first
    x = torch.tensor([[0.0, -0.0, 0.0], [-math.inf] * 3, [1.0, math.nan, 2.0]])
    lp, h = scoring.logprob_rows(x, torch.tensor([2, 0, -100]))
    assert float(h[0]) == pytest.approx(math.log(3)) and lp[1] == -math.inf and h[1] == 0
    assert lp[2] == 0 and h[2] == 0
    assert scoring.top_rows(x, 3)[1].tolist() == [[0, 1, 2], [0, 1, 2], [1, 2, 0]]
    # equal scores of any size are uniform
    lp, h = scoring.logprob_rows(torch.full((1, 4), torch.finfo(torch.float32).min), torch.tensor([3]))
    assert float(lp) == pytest.approx(-math.log(4)) and float(h) == pytest.approx(math.log(4))


@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (0.6, 0.0), (2.0, 5.0)])
def test_logprob_gradient_is_autograd_and_differences(temperature, softcap):
    g = torch.Generator().manual_seed(1)
    x = (3 * torch.randn(4, 11, generator=g, dtype=torch.float64)).requires_grad_()
    t = torch.tensor([3, -100, 0, 10])
    gl, ge = torch.randn(4, generator=g, dtype=torch.float64), torch.randn(4, generator=g, dtype=torch.float64)

    def value(x):
        logp = F.log_softmax(scoring.scores(x, temperature, softcap), -1)
        here = t >= 0
        lp = logp.gather(1, t.clamp(min=0)[:, None])[:, 0]
        h = -(logp.exp() * logp).sum(-1)
        return (here * (gl * lp + ge * h)).sum()

    value(x).backward()
    grad, size = scoring.logprob_grad_rows(x.detach(), t, gl, ge, temperature, softcap)
    assert torch.allclose(grad, x.grad, rtol=1e-10, atol=1e-12)
    assert bool((size + 1e-12 >= grad.abs()).all())
    lp, h = scoring.logprob_rows(x.detach(), t, temperature, softcap)
    assert torch.allclose((gl * lp + ge * h).sum(), value(x.detach()), rtol=1e-12)
    d = 1e-6 * torch.randn(4, 11, generator=g, dtype=torch.float64)
    change = value(x.detach() + d) - value(x.detach() - d)
    assert torch.allclose(change, 2 * (grad * d).sum(), rtol=1e-5, atol=1e-14)


@pytest.mark.parametrize("temperature,softcap", [(1.0, 0.0), (2.0, 0.0), (1.5, 4.0)])
def test_distillation_is_kl_div_and_differences(temperature, softcap):
    g = torch.Generator().manual_seed(2)
    x = (2 * torch.randn(5, 9, generator=g, dtype=torch.float64)).requires_grad_()
    teacher = torch.randn(5, 3, generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(9, generator=g)[:3] for _ in range(5)])
    ids[1, 2] = -100
    ids[3] = -100
    ids[4, 1] = ids[4, 0]  # the same id twice
    up = torch.randn(5, generator=g, dtype=torch.float64)
    there = ids != -100
    q = torch.softmax((teacher / temperature).masked_fill(~there, -1e9), -1) * there

    def value(x):
        logp = F.log_softmax(scoring.scores(x, temperature, softcap), -1).gather(1, ids.clamp(min=0))
        kl = F.kl_div(logp, q, reduction="none") * there
        return (up * temperature ** 2 * kl.sum(-1)).sum()

    value(x).backward()
    grad, _ = scoring.distill_grad_rows(x.detach(), teacher, ids, up, temperature, softcap)
    assert torch.allclose(grad, x.grad, rtol=1e-10, atol=1e-12)
    losses, _, counted = scoring.distill_rows(x.detach(), teacher, ids, temperature, softcap)
    assert counted.tolist() == [True, True, True, False, True] and losses[3] == 0
    assert torch.allclose((up * losses).sum(), value(x.detach()), rtol=1e-10)
    d = 1e-6 * torch.randn(5, 9, generator=g, dtype=torch.float64)
    change = value(x.detach() + d) - value(x.detach() - d)
    assert torch.allclose(change, 2 * (grad * d).sum(), rtol=1e-5, atol=1e-14)


def test_ignored_rows_have_no_gradient_whatever_they_hold():
    x = torch.tensor([[1.0, math.nan, 2.0], [math.inf, -math.inf, math.nan], [0.5, 1.0, -1.0]])
    t = torch.tensor([-100, -100, 1])
    for softcap in (0.0, 4.0):
        grad, size = scoring.logprob_grad_rows(x, t, torch.ones(3), torch.ones(3), 0.7, softcap)
        assert bool((grad[:2] == 0).all()) and bool((size[:2] == 0).all()) and bool(torch.isfinite(grad[2]).all())
