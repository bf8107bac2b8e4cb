"""Rotary positions of queries and keys on gfx950 (MI355X).

The pairs of a head's first ``rotary_dim`` elements are turned by the angles of
the token's position ``p``: with ``(x0, x1)`` = elements ``(i, i + rotary_dim / 2)``,
or ``(2 i, 2 i + 1)`` where ``interleaved``,

    y0 = x0 cos[p, i] - x1 sin[p, i],   y1 = x1 cos[p, i] + x0 sin[p, i]

in fp32 with one rounding; the other elements pass through. The angles come from
a table of cosines and sines that :func:`rotary_table` makes in float64 (an angle
of a far position in fp32 has lost its digits), plain or scaled for contexts
longer than those of training. One launch turns queries and keys
(``csrc/heads.hip``: each element is read and written once); the gradient turns
the upstream gradients back, and can itself be differentiated.

A position outside the table gives NaN in the turned elements.

No counterpart among the reference's kernels that this package covers: its
registry's ``rotary_embedding`` pattern (``autokernel/_patterns.py``) keeps its
name only.
"""

import math
import os
from typing import Optional, Tuple

import torch

from kernels.hip import _heads, _lib
from kernels.hip.token_logprobs import refuse_tangents

KERNEL_TYPE = "rotary"
BACKEND = "hip"

HIP_SRC = os.path.join(_lib.CSRC_DIR, "heads.hip")

SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_positions: Optional[int] = None, beta_fast: float = 32.0,
                       beta_slow: float = 1.0) -> torch.Tensor:
    """Angle per position of each pair, float64 ``[rotary_dim / 2]`` on the CPU:
    ``f_i = base^(-2 i / rotary_dim)``, for a context ``factor`` times the trained one

    * ``"linear"``: divided by ``factor`` (positions interpolated);
    * ``"ntk"``: of the base ``base * factor^(rotary_dim / (rotary_dim - 2))``, which
      leaves the fastest pair as it was and divides the slowest by ``factor``;
    * ``"yarn"``: pairs that turn ``beta_fast`` times or more within
      ``original_positions`` stay, those that turn ``beta_slow`` times or less are
      divided by ``factor``, those between are blended linearly in their index (Peng
      et al., "YaRN", 2023).
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (math.isfinite(base) and base > 1.0 and math.isfinite(factor) and factor >= 1.0):
        raise ValueError(f"base must be above 1 and factor at least 1, got {base} and {factor}")
    if scaling is None and factor != 1.0:
        raise ValueError(f"factor {factor} without a scaling")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-i / rotary_dim)
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        if original_positions is None or original_positions < 1:
            raise ValueError("yarn scaling needs original_positions, the context of training")
        if not 0.0 < beta_slow <= beta_fast:
            raise ValueError(f"beta_slow must be positive and at most beta_fast, got {beta_slow} and {beta_fast}")

        def index(turns):  # the pair that turns so often within the trained context
            return rotary_dim * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(index(beta_fast)), 0)
        high = min(math.ceil(index(beta_slow)), rotary_dim - 1)
        slow = ((i / 2 - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f * (1.0 - slow) + f / factor * slow
    return f


def rotary_table(rotary_dim: int, positions: int, *, base: float = 10000.0, scaling: Optional[str] = None,
                 factor: float = 1.0, original_positions: Optional[int] = None, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attention_factor: Optional[float] = None, device=None) -> torch.Tensor:
    """The table that the rotary kernels take: float32 ``[positions, rotary_dim]``,
    the cosines of a position's ``rotary_dim / 2`` angles, then their sines. Made in
    float64, once for a model; see :func:`rotary_frequencies` for the scalings.

    ``attention_factor`` multiplies both (None: 1, with yarn ``0.1 ln(factor) + 1``).
    """
    if positions < 1:
        raise ValueError(f"positions must be positive, got {positions}")
    f = rotary_frequencies(rotary_dim, base=base, scaling=scaling, factor=factor, original_positions=original_positions,
                           beta_fast=beta_fast, beta_slow=beta_slow)
    if attention_factor is None:
        attention_factor = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
    f = f.to(device)
    table = torch.empty((positions, rotary_dim), dtype=torch.float32, device=f.device)
    half = rotary_dim // 2
    step = max(1, (1 << 24) // rotary_dim)  # bounds the float64 temporaries
    for p in range(0, positions, step):
        q = min(positions, p + step)
        a = torch.arange(p, q, dtype=torch.float64, device=f.device)[:, None] * f
        table[p:q, :half] = torch.cos(a) * attention_factor
        table[p:q, half:] = torch.sin(a) * attention_factor
    return table


def check_pair(q: torch.Tensor, k: Optional[torch.Tensor]) -> None:
    _lib.dtype_code(q.dtype)
    if k is None:
        return
    if k.dtype != q.dtype:
        raise TypeError(f"q is {q.dtype}, k is {k.dtype}")
    if q.dim() < 2 or k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [..., heads, dim] and differ in heads only")


def _turn(q, k, table, positions, n_positions, interleaved, inverse):
    hq = _heads.as_heads(q, "q")
    hk = None if k is None else _heads.as_heads(k, "k")
    out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    out_k = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _lib.qk_norm_rotary(hq, hk, None, None, table, positions, n_positions, out_q, out_k, 0.0, interleaved, inverse)
    return out_q, out_k


class _Rotary(torch.autograd.Function):
    """Linear in q and k: its backward is itself, turned the other way."""

    @staticmethod
    def forward(ctx, q, k, table, positions, n_positions, interleaved, inverse):
        ctx.save_for_backward(table, positions)
        ctx.params = (n_positions, interleaved, inverse)
        return _turn(q, k, table, positions, n_positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, g_q, g_k):
        refuse_tangents(KERNEL_TYPE, g_q, g_k)
        table, positions = ctx.saved_tensors
        n_positions, interleaved, inverse = ctx.params
        g_q, g_k = rotate(g_q, g_k, table, positions, n_positions, interleaved, not inverse)
        return (g_q, g_k) + (None,) * 5


def rotate(q, k, table, positions, n_positions, interleaved, inverse):
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, table, positions, n_positions, interleaved, inverse)
    return _turn(q, k, table, positions, n_positions, interleaved, inverse)


def kernel_fn(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: Optional[torch.Tensor] = None,
              *, interleaved: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(q, k)`` with their positions turned in, contiguous.

    Args:
        q: ``[..., heads, dim]`` fp32, fp16 or bf16, dim at most 2048; views (of a
            fused projection, of ``[batch, heads, seq, dim]`` transposed) are read in place.
        k: the same with its own number of heads, or None.
        table: from :func:`rotary_table`; its width is the turned part of a head.
        positions: whole numbers, of q's leading shape or broadcast to it; None: 0,
            1, ... along the last leading dimension.
        interleaved: pairs of neighbours instead of halves.
    """
    interleaved = bool(interleaved)
    host = _lib.native(q, *_lib.given(k, table, positions))
    if host is not None:
        out = host.rotary(q, k, table, positions, interleaved)
        if out is not None:
            return out
    _lib.require_device(q, k, table, positions)
    refuse_tangents(KERNEL_TYPE, q, k)
    check_pair(q, k)
    _heads.as_heads(q, "q")
    _heads.check_table(table, q.shape[-1])
    positions, n_positions = _heads.check_positions(positions, q.shape[:-2])
    return rotate(q, k, table, positions, n_positions, interleaved, False)
