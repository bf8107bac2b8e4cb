"""Token log probabilities and entropy from hidden states, without logits, gfx950.

:mod:`kernels.hip.token_logprobs` over the logits ``hidden @ weight^T``, fused
with the head's product as :mod:`kernels.hip.chunked_linear_cross_entropy` fuses
the loss: what scoring finished text, and a policy-gradient step with an
entropy bonus, need of a language model's head. Rules at the edges are those of
``token_logprobs``.

fp16 and bf16, any hidden size (``csrc/lmhead_ce.hip``): the tile kernel forms
the logits on the matrix cores and folds each tile into a maximum, ``sum e^t``
and ``sum e^t t`` of each token in registers; a row kernel joins them and adds
the given tokens' scores as their own dot products. The backward forms the
tiles again, writes the logits' gradient in the input type (one rounding, as
both products after it take that type; fp16 loses entries below 6e-8 unless the
caller scales its loss) for as much of the vocabulary at a time
as ``GRAD_LOGITS_BUDGET`` of the loss allows, and runs the loss's two gradient
GEMMs on it. For fp32 the logits of ``chunk_size`` rows at a time come from a
GEMM and go through the row kernels (under autocast too: operands keep their
type). The backward is differentiable once.

No counterpart in the reference, whose chunked loss
(``kernels/hip/chunked_linear_cross_entropy.py:50-175``) returns the mean only.
"""

import os
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from kernels.hip import _lib
from kernels.hip import chunked_linear_cross_entropy as clce
from kernels.hip.chunked_linear_cross_entropy import _fused_ok, _kernel_operands, gradients_by_ranges, own_types
from kernels.hip.token_logprobs import (check_scale, differentiable_once, refuse_tangents, row_gradient,
                                        whole_numbers)

KERNEL_TYPE = "lmhead_logprobs"
BACKEND = "hip"

HIP_SRC = os.path.join(_lib.CSRC_DIR, "lmhead_ce.hip")


class LmheadLogprobs(NamedTuple):
    """fp32, of the rows' shape; ``logprobs`` is None without tokens."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor


def _rows(t, start, end):
    return t[start:end] if t is not None else None



def _forward(hidden, weight, tokens, temperature, softcap, ignore_index, chunk_size, keep):
    """``(logprobs, entropy, stats)``."""
    n = hidden.shape[0]
    fused = _fused_ok(hidden, weight, softcap, 0.0)
    f32 = dict(dtype=torch.float32, device=hidden.device)
    logprobs = torch.empty(n, **f32) if tokens is not None else None
    entropy = torch.empty(n, **f32)
    stats = torch.empty((n, 4), **f32) if keep else None
    if n and fused:
        h, w = _kernel_operands(hidden, weight)
        _lib.lmhead_logprobs(h, w, tokens, logprobs, entropy, stats, temperature, softcap, ignore_index)
    elif n:
        with own_types(hidden):
            for start in range(0, n, chunk_size):
                end = min(start + chunk_size, n)
                _lib.token_logprobs(F.linear(hidden[start:end], weight), _rows(tokens, start, end),
                                    _rows(logprobs, start, end), entropy[start:end], _rows(stats, start, end), None,
                                    None, temperature, softcap, ignore_index)
    return logprobs, entropy, stats


class _LmheadLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, tokens, temperature, softcap, ignore_index, chunk_size):
        logprobs, entropy, stats = _forward(hidden, weight, tokens, temperature, softcap, ignore_index, chunk_size,
                                            True)
        ctx.save_for_backward(hidden, weight, tokens, stats)
        ctx.params = (temperature, softcap, ignore_index)
        ctx.chunk_size = chunk_size
        ctx.set_materialize_grads(False)
        return logprobs, entropy

    @staticmethod
    def backward(ctx, g_logprobs, g_entropy):
        differentiable_once(KERNEL_TYPE, g_logprobs, g_entropy)
        hidden, weight, tokens, stats = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        gl, ge = row_gradient(g_logprobs), row_gradient(g_entropy)
        n, d = hidden.shape
        vocab = weight.shape[0]
        if n == 0:
            gh = torch.empty_like(hidden) if need_h else None
            gw = torch.zeros_like(weight) if need_w else None
        elif _fused_ok(hidden, weight, ctx.params[1], 0.0):
            temperature, softcap, ignore_index = ctx.params
            coefs = torch.empty((n, 4), dtype=torch.float32, device=hidden.device)
            _lib.lmhead_logprobs_coefs(tokens, stats.contiguous(), gl, ge, coefs, vocab, temperature, ignore_index)
            h, w = _kernel_operands(hidden, weight)

            def write_range(g, v0):
                _lib.lmhead_logprobs_bwd_range(h, w, tokens, coefs, g, v0, temperature, softcap, ignore_index)

            gh, gw = gradients_by_ranges(h, w, write_range, d, need_h, need_w)
        else:
            h, w = hidden.contiguous(), weight.contiguous()
            stats = stats.contiguous()
            gh = torch.empty_like(h) if need_h else None
            gw = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device) if need_w else None
            with own_types(h):
                for start in range(0, n, ctx.chunk_size):
                    end = min(start + ctx.chunk_size, n)
                    logits = F.linear(h[start:end], w)
                    grad = torch.empty_like(logits)  # (the row kernel reads the logits again behind its stores)
                    _lib.token_logprobs_bwd(logits, _rows(tokens, start, end), stats[start:end],
                                            _rows(gl, start, end), _rows(ge, start, end), grad, *ctx.params)
                    if need_h:
                        gh[start:end] = grad @ w
                    if need_w:
                        gw.addmm_(grad.t(), h[start:end])
        return gh, gw, None, None, None, None, None


def kernel_fn(hidden: torch.Tensor, weight: torch.Tensor, tokens: Optional[torch.Tensor] = None, *,
              temperature: float = 1.0, softcap: float = 0.0, ignore_index: int = -100,
              chunk_size: int = 512) -> LmheadLogprobs:
    """Log probabilities of ``tokens`` under ``softmax(hidden @ weight^T)``, and its entropy.

    Args:
        hidden: ``[..., d]`` fp16, bf16 or fp32.
        weight: ``[vocab, d]``; another type is converted to hidden's.
        tokens: whole numbers of the leading shape, or None (no ``logprobs``).
        temperature: divides the (capped) logits; at least 1e-3.
        softcap: logit softcap, 1e-3 to 1e4 (0 = off), as in ``token_logprobs``.
        ignore_index: token value of rows to leave out, whatever they and
            their logits hold; but ``weight``'s gradient sums 0 times their
            hidden states, which have to be finite where it is asked for.
        chunk_size: rows per chunk of the fp32 path's GEMMs.
    """
    temperature, softcap, ignore_index, chunk_size = float(temperature), float(softcap), int(ignore_index), int(chunk_size)
    host = _lib.native(hidden, weight) if tokens is None else _lib.native(hidden, weight, tokens)
    if host is not None and chunk_size > 0:
        out = host.lmhead_logprobs(hidden, weight, tokens, temperature, softcap, ignore_index,
                                   float(clce.GRAD_LOGITS_BUDGET))
        if out is not None:
            return LmheadLogprobs(*out)
    _lib.require_device(hidden, weight, tokens)
    refuse_tangents(KERNEL_TYPE, hidden, weight)
    _lib.dtype_code(hidden.dtype)
    if hidden.dim() == 0 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1]:
        raise ValueError(f"hidden shape {tuple(hidden.shape)} does not go with weight {tuple(weight.shape)}")
    vocab, d = weight.shape
    if not vocab or not d:
        raise ValueError(f"weight must not be empty, got shape {tuple(weight.shape)}")
    if hidden.dtype == torch.float32 and vocab > _lib.MAX_SCORE_VOCAB:
        raise ValueError(f"fp32 takes a vocab of at most {_lib.MAX_SCORE_VOCAB}, got {vocab}")
    check_scale(temperature, softcap, least=1e-3)
    if chunk_size < 1:
        raise ValueError(f"chunk_size must be at least 1, got {chunk_size}")
    lead = hidden.shape[:-1]
    if tokens is not None:
        tokens = whole_numbers(tokens, "tokens", lead).view(-1)
    if weight.dtype != hidden.dtype:
        _lib.dtype_code(weight.dtype)
        weight = weight.to(hidden.dtype)
    h2d = hidden.reshape(-1, d)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        logprobs, entropy = _LmheadLogprobs.apply(h2d, weight, tokens, temperature, softcap, ignore_index, chunk_size)
    else:
        logprobs, entropy, _ = _forward(h2d, weight, tokens, temperature, softcap, ignore_index, chunk_size, False)
    if len(lead) != 1:
        logprobs, entropy = (t.view(lead) if t is not None else None for t in (logprobs, entropy))
    return LmheadLogprobs(logprobs, entropy)
