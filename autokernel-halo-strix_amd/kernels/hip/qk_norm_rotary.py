"""RMSNorm of each head of queries and keys with their rotary positions, in one
pass, on gfx950 (MI355X).

    n = x / sqrt(mean(x^2) + eps) * weight        over a head's elements
    y = n with its pairs turned (``kernels.hip.rotary``), or n without a table

in fp32 with one rounding (the sum of squares too: heads whose squares leave
fp32's range, past 1e18 or, with eps 0, below 1e-20, have no norm there). The
forward reads and writes each element once (``csrc/heads.hip``); so does the
backward with the upstream gradient beside it, which it turns back, and from
which it sums the weights' gradients over tokens and heads in fp32, in a fixed
order. Differentiable once.

No counterpart in the reference, whose RMSNorm (``kernels/hip/rmsnorm.py:156-177``)
takes whole rows and whose registry keeps the rotary pattern's name only.
"""

import os
from typing import Optional, Tuple

import torch

from kernels.hip import _heads, _lib
from kernels.hip.rotary import check_pair
from kernels.hip.token_logprobs import differentiable_once, refuse_tangents

KERNEL_TYPE = "qk_norm_rotary"
BACKEND = "hip"

HIP_SRC = os.path.join(_lib.CSRC_DIR, "heads.hip")

DEFAULT_EPS = 1e-6


def check_weight(w: Optional[torch.Tensor], name: str, x: torch.Tensor) -> torch.Tensor:
    if w is None:
        raise ValueError(f"{name} is missing")
    if w.dim() != 1 or w.numel() != x.shape[-1]:
        raise ValueError(f"{name} shape {tuple(w.shape)} does not match the head dimension {x.shape[-1]}")
    return w.to(x.dtype).contiguous()


def check_eps(eps: float) -> float:
    eps = float(eps)
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    return eps


def _forward(q, k, q_weight, k_weight, table, positions, n_positions, eps, interleaved):
    hq = _heads.as_heads(q, "q")
    hk = None if k is None else _heads.as_heads(k, "k")
    out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    out_k = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _lib.qk_norm_rotary(hq, hk, q_weight, k_weight, table, positions, n_positions, out_q, out_k, eps, interleaved, False)
    return out_q, out_k


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, n_positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
        ctx.params = (n_positions, eps, interleaved)
        return _forward(q, k, q_weight, k_weight, table, positions, n_positions, eps, interleaved)

    @staticmethod
    def backward(ctx, g_q, g_k):
        differentiable_once(KERNEL_TYPE, g_q, g_k)
        q, k, q_weight, k_weight, table, positions = ctx.saved_tensors
        n_positions, eps, interleaved = ctx.params
        hq, hgq = _heads.as_heads(q, "q"), _heads.as_heads(g_q.to(q.dtype), "q's gradient")
        dq, dk, dqw, dkw = torch.empty(q.shape, dtype=q.dtype, device=q.device), None, None, None
        hk = hgk = None
        if k is not None:
            hk, hgk = _heads.as_heads(k, "k"), _heads.as_heads(g_k.to(q.dtype), "k's gradient")
            dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        if ctx.needs_input_grad[2]:
            dqw = torch.empty(q.shape[-1], dtype=q.dtype, device=q.device)
        if k is not None and ctx.needs_input_grad[3]:
            dkw = torch.empty(q.shape[-1], dtype=q.dtype, device=q.device)
        bytes_ = _lib.qk_norm_rotary_bwd_workspace_bytes(hq.outer * hq.inner, hq.heads, hk.heads if hk else 0, hq.dim)
        ws = torch.empty(bytes_, dtype=torch.uint8, device=q.device)
        _lib.qk_norm_rotary_bwd(hq, hk, q_weight.contiguous(), None if k is None else k_weight.contiguous(), table, positions,
                                n_positions, hgq, hgk, dq, dk, dqw, dkw, ws, eps, interleaved)
        return (dq, dk, dqw, dkw) + (None,) * 5


def kernel_fn(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: torch.Tensor, k_weight: Optional[torch.Tensor],
              table: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *, eps: float = DEFAULT_EPS,
              interleaved: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(q, k)`` normed head by head and with their positions turned in, contiguous.

    Args:
        q: ``[..., heads, dim]`` fp32, fp16 or bf16, dim at most 2048; views are read in place.
        k: the same with its own number of heads, or None (with ``k_weight`` None).
        q_weight, k_weight: ``[dim]``, cast to q's type.
        table: from ``kernels.hip.rotary.rotary_table``, or None: no rotation.
        positions, interleaved: as in ``kernels.hip.rotary.kernel_fn``.
        eps: added to the mean square.
    """
    eps, interleaved = check_eps(eps), bool(interleaved)
    host = _lib.native(q, *_lib.given(k, q_weight, k_weight, table, positions))
    if host is not None and q_weight is not None:
        out = host.qk_norm_rotary(q, k, q_weight, k_weight, table, positions, eps, interleaved)
        if out is not None:
            return out
    _lib.require_device(q, k, q_weight, k_weight, table, positions)
    refuse_tangents(KERNEL_TYPE, q, k, q_weight, k_weight)
    check_pair(q, k)
    _heads.as_heads(q, "q")
    q_weight = check_weight(q_weight, "q_weight", q)
    if k is None and k_weight is not None:
        raise ValueError("k_weight without k")
    if k is not None:
        k_weight = check_weight(k_weight, "k_weight", k)
    if table is None:
        if positions is not None:
            raise ValueError("positions without a table")
        n_positions = 1
    else:
        _heads.check_table(table, q.shape[-1])
        positions, n_positions = _heads.check_positions(positions, q.shape[:-2])
    args = (q, k, q_weight, k_weight, table, positions, n_positions, eps, interleaved)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRotary.apply(*args)
    return _forward(*args)
