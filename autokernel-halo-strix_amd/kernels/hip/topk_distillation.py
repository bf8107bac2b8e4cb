"""Distillation from a teacher's top logits on gfx950 (MI355X).

A teacher is kept as its ``k`` top logits of each row and their columns
(:mod:`kernels.hip.token_logprobs` gives both; log probabilities serve as
logits). With the student's ``p = softmax(y / T)`` over the whole vocabulary
(``y`` its logits, capped where ``softcap`` says so) and the teacher's ``q =
softmax(teacher / T)`` over the row's entries,

    loss = T^2 sum_k q_k (ln q_k - ln p[id_k])
    d loss / d y_v = T (p_v - sum of q_k with id_k == v)

``T^2`` keeps the gradient's size as the temperature ``T`` changes. The
forward reads the student's logits once; the backward reads them once more and
writes the gradient once, rounded once whatever the upstream gradient
(``csrc/topk_distill.hip``). The teacher is a constant. The backward is
differentiable once.

Rules at the edges:

* an entry whose id is ``ignore_index`` is not there (teachers that kept fewer
  alternatives are padded with it), nor is one whose logit is -inf; the same id
  twice counts twice;
* a row without entries has loss 0, a zero gradient and no part in the mean;
* an id outside ``[0, vocab)`` that is not ``ignore_index``, a NaN or +inf on
  either side give a NaN loss and a NaN gradient row;
* an entry that the student masks (-inf) while the teacher has it makes the
  row's loss +inf;
* with a softcap the student's infinities are ``softcap`` and ``-softcap``.

No counterpart in the reference.
"""

import os

import torch

from kernels.hip import _lib
from kernels.hip.token_logprobs import (check_scale, check_vocab, differentiable_once, refuse_tangents,
                                        row_gradient, whole_numbers)

KERNEL_TYPE = "topk_distillation"
BACKEND = "hip"

HIP_SRC = os.path.join(_lib.CSRC_DIR, "topk_distill.hip")


def _forward(rows2d, teacher, ids, temperature, softcap, ignore_index, mean):
    """``(loss or losses, stats, scale)``."""
    n = rows2d.shape[0]
    f32 = dict(dtype=torch.float32, device=rows2d.device)
    losses, stats = torch.empty(n, **f32), torch.empty((n, 4), **f32)
    loss = torch.empty((), **f32) if mean else None
    scale = torch.empty(1, **f32) if mean else None
    if n or mean:
        _lib.topk_distill(rows2d, teacher, ids, losses, stats, loss, scale, temperature, softcap, ignore_index)
    return (loss if mean else losses), stats, scale


class _TopkDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, ids, temperature, softcap, ignore_index, mean):
        rows2d = _lib.as_rows(logits, logits.shape[-1])
        loss, stats, scale = _forward(rows2d, teacher, ids, temperature, softcap, ignore_index, mean)
        ctx.save_for_backward(rows2d, teacher, ids, stats, scale)
        ctx.params = (temperature, softcap, ignore_index)
        ctx.shape = logits.shape
        return loss

    @staticmethod
    def backward(ctx, g_loss):
        differentiable_once(KERNEL_TYPE, g_loss)
        rows2d, teacher, ids, stats, scale = ctx.saved_tensors
        grad = torch.empty(ctx.shape, dtype=rows2d.dtype, device=rows2d.device)
        if grad.numel():
            v, k = ctx.shape[-1], ids.shape[-1]
            _lib.topk_distill_bwd(_lib.as_rows(rows2d, v), _lib.as_rows(teacher, k), _lib.as_rows(ids, k),
                                  stats.contiguous(), row_gradient(g_loss), scale, grad.view(-1, v), *ctx.params)
        return (grad,) + (None,) * 6


def kernel_fn(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, *,
              temperature: float = 1.0, softcap: float = 0.0, ignore_index: int = -100,
              reduction: str = "mean") -> torch.Tensor:
    """Distillation loss of a student's logits against a teacher's top logits.

    Args:
        logits: the student's, ``[..., vocab]`` fp32, fp16 or bf16, vocab at most 2^20.
        teacher_logits: ``[..., k]`` of any of these types, ``k`` from 1 to 256.
        teacher_ids: whole numbers ``[..., k]``, the columns of ``teacher_logits``.
        temperature: divides both sides' logits.
        softcap: the student's logit softcap, as in ``token_logprobs``.
        ignore_index: id of entries that are not there.
        reduction: ``"mean"`` over the rows that have entries (a 0-d tensor),
            or ``"none"`` (one loss a row).
    """
    temperature, softcap, ignore_index = float(temperature), float(softcap), int(ignore_index)
    host = _lib.native(logits, teacher_logits, teacher_ids)
    if host is not None and reduction in ("mean", "none"):
        loss = host.topk_distillation(logits, teacher_logits, teacher_ids, temperature, softcap, ignore_index,
                                      reduction == "mean")
        if loss is not None:
            return loss
    _lib.require_device(logits, teacher_logits, teacher_ids)
    refuse_tangents(KERNEL_TYPE, logits)
    vocab = check_vocab(logits)
    if reduction not in ("mean", "none"):
        raise ValueError(f"reduction must be 'mean' or 'none', got {reduction!r}")
    lead = logits.shape[:-1]
    _lib.dtype_code(teacher_logits.dtype)
    if teacher_logits.dim() != logits.dim() or teacher_logits.shape[:-1] != lead:
        raise ValueError(f"teacher_logits shape {tuple(teacher_logits.shape)} does not go with logits "
                         f"{tuple(logits.shape)}")
    k = teacher_logits.shape[-1]
    if not 1 <= k <= _lib.MAX_TOP:
        raise ValueError(f"1 to {_lib.MAX_TOP} teacher entries a row are taken, got {k}")
    check_scale(temperature, softcap)
    ids = whole_numbers(teacher_ids, "teacher_ids", teacher_logits.shape).view(-1, k)
    teacher = _lib.as_rows(teacher_logits.detach(), k)
    mean = reduction == "mean"
    if logits.requires_grad and torch.is_grad_enabled():
        loss = _TopkDistillation.apply(logits, teacher, ids, temperature, softcap, ignore_index, mean)
    else:
        loss = _forward(_lib.as_rows(logits, vocab), teacher, ids, temperature, softcap, ignore_index, mean)[0]
    return loss if mean else loss.view(lead)
