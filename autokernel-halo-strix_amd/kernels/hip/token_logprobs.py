"""Token log probabilities, entropy and top alternatives on gfx950 (MI355X).

For each row of logits ``x``, with ``y = softcap * tanh(x / softcap)`` (or
``x``) and ``p = softmax(y / temperature)``:

* ``logprobs = ln p[token]`` of the given token;
* ``entropy = -sum_v p_v ln p_v``;
* ``top_logprobs``, ``top_ids``: the ``top_k`` largest ``ln p`` and their
  columns, in descending order, equal logits by column.

The forward reads the logits once (``csrc/token_logprobs.hip``); few or very
wide rows, as a decode step has them, are cut over the whole GPU. Gradients
reach the logits through ``logprobs`` and ``entropy``; the backward reads the
logits once and writes their gradient once, from the rows' saved statistics.
The alternatives have no gradient. The backward is differentiable once.

Rules at the edges:

* a row whose token is ``ignore_index`` has logprob 0, entropy 0 and a zero
  gradient, whatever it holds (its alternatives are its own);
* a token outside ``[0, vocab)`` that is not ``ignore_index`` gives a NaN
  logprob, and a NaN gradient row;
* -inf masks a logit. A row of -inf alone has logprobs of -inf, entropy 0, a zero
  gradient. (With a softcap -inf is ``-softcap``, which masks nothing, and such
  a row uniform.)
* a row that holds a NaN, or without a softcap +inf (with one it becomes
  ``softcap``), has NaN results, NaN first among its alternatives.

No counterpart in the reference, whose cross-entropy
(``kernels/ce_fused.py:557-785``) gives the loss of given tokens only.
"""

import os
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from kernels.hip import _lib

KERNEL_TYPE = "token_logprobs"
BACKEND = "hip"

HIP_SRC = os.path.join(_lib.CSRC_DIR, "token_logprobs.hip")


class TokenLogprobs(NamedTuple):
    """fp32 ``logprobs`` and ``entropy`` of the rows' shape, ``top_logprobs``
    (fp32) and ``top_ids`` (int64) with a last dimension of ``top_k``; None
    where not asked for."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def check_scale(temperature: float, softcap: float, least: float = 1e-18) -> None:
    """The temperature and softcap that the scoring kernels take."""
    if not least <= temperature <= 1e18:
        raise ValueError(f"temperature must be between {least:g} and 1e18, got {temperature}")
    if softcap != 0.0 and not 1e-3 <= softcap <= 1e4:
        raise ValueError(f"softcap must be 0 (off) or between 1e-3 and 1e4, got {softcap}")
    # the capped scores are exact to 2^-22 softcap / temperature: a quarter there
    if softcap > temperature * 2 ** 20:
        raise ValueError(f"softcap must be at most 2^20 temperatures, got {softcap} and {temperature}")


def whole_numbers(t: torch.Tensor, name: str, shape) -> torch.Tensor:
    """``t`` of the given shape as contiguous int64."""
    if t.dtype == torch.bool or t.is_floating_point() or t.is_complex():
        raise TypeError(f"{name} must be whole numbers, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} shape {tuple(t.shape)} != {tuple(shape)}")
    return t.to(torch.int64).contiguous()


def refuse_tangents(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuse forward mode: the kernels would drop a tangent without a word."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative: its backward is the derivative there is")


def differentiable_once(name: str, *upstream: Optional[torch.Tensor]) -> None:
    """Refuse a backward that is itself to be differentiated (its kernels' results
    carry no graph: what should have a gradient would pass as a constant)."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name} is differentiable once: its backward takes no create_graph=True")
    refuse_tangents(name, *upstream)


def row_gradient(g: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """An upstream gradient of a row each as contiguous fp32."""
    return None if g is None else g.detach().to(torch.float32).reshape(-1).contiguous()


def check_vocab(logits: torch.Tensor) -> int:
    """The logits' last dimension, as the row kernels take it."""
    _lib.dtype_code(logits.dtype)
    if logits.dim() == 0 or not 0 < logits.shape[-1] <= _lib.MAX_SCORE_VOCAB:
        raise ValueError(f"logits must be [..., vocab] with a vocab of 1 to {_lib.MAX_SCORE_VOCAB}, "
                         f"got shape {tuple(logits.shape)}")
    return logits.shape[-1]


def _forward(rows2d, tokens, temperature, softcap, ignore_index, top_k, keep):
    """``(logprobs, entropy, top_logprobs, top_ids, stats)`` of ``[rows, vocab]``."""
    n = rows2d.shape[0]
    f32 = dict(dtype=torch.float32, device=rows2d.device)
    logprobs = torch.empty(n, **f32) if tokens is not None else None
    entropy = torch.empty(n, **f32)
    stats = torch.empty((n, 4), **f32) if keep else None
    top_logprobs = torch.empty((n, top_k), **f32) if top_k else None
    top_ids = torch.empty((n, top_k), dtype=torch.int64, device=rows2d.device) if top_k else None
    if n:
        _lib.token_logprobs(rows2d, tokens, logprobs, entropy, stats, top_logprobs, top_ids, temperature,
                            softcap, ignore_index)
    return logprobs, entropy, top_logprobs, top_ids, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, softcap, ignore_index, top_k):
        rows2d = _lib.as_rows(logits, logits.shape[-1])
        *out, stats = _forward(rows2d, tokens, temperature, softcap, ignore_index, top_k, True)
        ctx.save_for_backward(rows2d, tokens, stats)
        ctx.params = (temperature, softcap, ignore_index)
        ctx.shape = logits.shape
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in out[2:] if t is not None))
        return tuple(out)

    @staticmethod
    def backward(ctx, g_logprobs, g_entropy, *unused):
        differentiable_once(KERNEL_TYPE, g_logprobs, g_entropy)
        rows2d, tokens, stats = ctx.saved_tensors
        grad = torch.empty(ctx.shape, dtype=rows2d.dtype, device=rows2d.device)
        if grad.numel():
            v = ctx.shape[-1]
            _lib.token_logprobs_bwd(_lib.as_rows(rows2d, v), tokens, stats.contiguous(), row_gradient(g_logprobs),
                                    row_gradient(g_entropy), grad.view(-1, v), *ctx.params)
        return (grad,) + (None,) * 5


def kernel_fn(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
              softcap: float = 0.0, ignore_index: int = -100, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` under ``logits``, with the rows' entropies
    and their ``top_k`` top alternatives.

    Args:
        logits: ``[..., vocab]`` fp32, fp16 or bf16, vocab at most 2^20.
        tokens: whole numbers of the leading shape, or None (no ``logprobs``).
        temperature: divides the (capped) logits.
        softcap: logit softcap, 1e-3 to 1e4 (0 = off) and at most ``2^20
            temperature``; scores are exact to ``2^-22 softcap / temperature``
            under it.
        ignore_index: token value of rows to leave out.
        top_k: alternatives of each row, 0 to min(256, vocab).
    """
    temperature, softcap, ignore_index, top_k = float(temperature), float(softcap), int(ignore_index), int(top_k)
    host = _lib.native(logits) if tokens is None else _lib.native(logits, tokens)
    if host is not None:
        out = host.token_logprobs(logits, tokens, temperature, softcap, ignore_index, top_k)
        if out is not None:
            return TokenLogprobs(*out)
    _lib.require_device(logits, tokens)
    refuse_tangents(KERNEL_TYPE, logits)
    vocab = check_vocab(logits)
    lead = logits.shape[:-1]
    check_scale(temperature, softcap)
    if not 0 <= top_k <= min(_lib.MAX_TOP, vocab):
        raise ValueError(f"top_k must be 0 to min({_lib.MAX_TOP}, vocab), got {top_k}")
    if tokens is not None:
        tokens = whole_numbers(tokens, "tokens", lead).view(-1)
    if logits.requires_grad and torch.is_grad_enabled():
        out = _TokenLogprobs.apply(logits, tokens, temperature, softcap, ignore_index, top_k)
    else:
        out = _forward(_lib.as_rows(logits, vocab), tokens, temperature, softcap, ignore_index, top_k, False)[:4]
    logprobs, entropy, top_logprobs, top_ids = out
    if len(lead) != 1:
        logprobs = logprobs.view(lead) if logprobs is not None else None
        entropy = entropy.view(lead)
        if top_k:
            top_logprobs, top_ids = top_logprobs.view(*lead, top_k), top_ids.view(*lead, top_k)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)
