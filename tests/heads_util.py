"""Inputs and error bounds of the tests of the operators on attention heads.

The bounds, with u = half an eps of the result's type and e = 2^-24 (half an eps
of fp32, in which the kernels compute):

* a turned element is x0 c - x1 s: the table's c and s carry e each, the products
  and their difference e each: 3 e (|x0| + |x1|), u |y| for the last rounding;
* a norm: the sum of squares of a head adds at most dim / 64 + 2 vectors of 8 + 6
  levels of lanes < 56 terms one after the other for dim <= 2048 (56 e, halved by the
  root), the mean, eps, root, reciprocal and two products 2 e each: below 48 e;
* a sum over many rows: e times the longest chain of additions;
* attention: a score adds dim products (dim e reach, with reach = scale sum |q k|),
  and the exponential of s - top gets its argument within 4 e (|s| + spread) and
  returns it within 4 e; the cap's tanh adds 2^-21 cap. A probability of a relative
  error r moves the quotient by at most 2 r sum(p |v|); its rounding to 16 bits (u) only
  the numerator. The sums over keys add at most keys / 32 + 64 terms in a chain.
"""

import math

import torch

E = 2.0 ** -24


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Below the type's normal range a rounding is off by half the smallest step
    (and the kernels may flush: the whole range)."""
    return torch.finfo(dtype).tiny


def partner_abs(x, rotary, interleaved):
    """|x0| + |x1| at both elements of each pair, |x| past the pairs."""
    from oracle import heads
    y = x.double().abs()
    if rotary:
        a, b = heads.pairs(rotary, interleaved)
        both = y[..., a] + y[..., b]
        y = y.clone()
        y[..., a], y[..., b] = both, both
    return y


def close(got, want, bound, what=""):
    got, want, bound = got.double().cpu(), want.double(), bound.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN where there should be none, or the other way"
    off = torch.where(nan | (got == want), 0.0, (got - want).abs())
    worst = float((off - bound.nan_to_num()).max()) if off.numel() else 0.0
    assert worst <= 0.0, f"{what}: off by {float(off.max()):.3g}, {worst:.3g} over the bound"


def turn_bound(y, z, rotary, interleaved, dtype, units=4.0, factor=1.0):
    """Of a turned y = rot(z) whose z carries (units - 3) e already."""
    return half_eps(dtype) * y.abs() + units * E * factor * partner_abs(z, rotary, interleaved) + tiny(dtype)


def make_batch(counts, lengths, page_size, seed, spare=3, extra_columns=2):
    """(page_table, lengths, starts, pages): pages in a shuffled order, -1 past the need."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page_size) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(counts), max(need + [0]) + extra_columns), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32)
    return table, torch.tensor(lengths, dtype=torch.int32), starts, total


def attend_bound(out, spread, reach, mass, keys, dim, dtype, softcap=0.0):
    rho = (dim + 8) * E * reach + 8 * E * (reach + spread) + 8 * E + (2.0 ** -21 * softcap)
    chain = (keys / 32 + 64) * E
    probability = half_eps(dtype) if dtype != torch.float32 else 0.0
    rho = rho.double()[..., None]
    return half_eps(dtype) * out.abs() + (probability + 2 * torch.expm1(rho) + 2 * chain + 4 * E) * mass + tiny(dtype)
