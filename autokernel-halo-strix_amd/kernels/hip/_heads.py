"""What the operators on attention heads share: views of heads as the kernels take
them, checks of positions, tables, pages and sequences."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from kernels.hip import _lib
from kernels.hip.token_logprobs import refuse_tangents

MAX_HEAD_DIM = 2048


class Heads(NamedTuple):
    """``[outer, inner, heads, dim]`` with a dense last dimension."""
    t: torch.Tensor
    outer: int
    inner: int
    heads: int
    dim: int

    @property
    def strides(self) -> Tuple[int, int, int]:
        return self.t.stride()[:3]


def as_heads(x: torch.Tensor, name: str) -> Heads:
    """``[..., heads, dim]`` as the kernels take it: without a copy where the last
    dimension is dense and the leading ones but the last fold into one."""
    if x.dim() < 2:
        raise ValueError(f"{name} must be [..., heads, dim], got shape {tuple(x.shape)}")
    *lead, heads, dim = x.shape
    if not 0 < dim <= MAX_HEAD_DIM:
        raise ValueError(f"{name}'s head dimension must be 1 to {MAX_HEAD_DIM}, got {dim}")
    inner = lead[-1] if lead else 1
    outer = 1
    for n in lead[:-1]:
        outer *= n
    t = x.reshape(outer, inner, heads, dim)
    if dim > 1 and t.stride(3) != 1:
        t = t.contiguous()
    return Heads(t, outer, inner, heads, dim)


def check_table(table: torch.Tensor, dim: int) -> int:
    """The rotated part of a head, from a table of angles ``[positions, rotary]``."""
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("table must be contiguous float32 [positions, rotary_dim] "
                         f"(see rotary_table), got {table.dtype} {tuple(table.shape)}")
    rotary = table.shape[1]
    if rotary < 2 or rotary % 2 or rotary > dim or table.shape[0] < 1:
        raise ValueError(f"table {tuple(table.shape)} does not turn an even part of a head of {dim}")
    if table.requires_grad:
        raise ValueError("the angles are constants: table must not require a gradient")
    refuse_tangents("the table of angles", table)
    return rotary


def check_positions(positions: Optional[torch.Tensor], lead) -> Tuple[Optional[torch.Tensor], int]:
    """``(positions as the kernels take them, their number)``: token t has the
    (t mod number)-th; None counts along the last leading dimension."""
    lead = tuple(lead)
    if positions is None:
        return None, max(1, lead[-1] if lead else 1)
    if positions.dtype == torch.bool or positions.is_floating_point() or positions.is_complex():
        raise TypeError(f"positions must be whole numbers, got {positions.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        positions = positions.to(torch.int64)
    if positions.dim() > len(lead):
        raise ValueError(f"positions {tuple(positions.shape)} do not match the leading shape {lead}")
    if tuple(positions.shape) != lead[len(lead) - positions.dim():]:
        try:
            positions = positions.expand(lead)
        except RuntimeError:
            raise ValueError(f"positions {tuple(positions.shape)} do not match the leading shape {lead}") from None
    return positions.contiguous(), max(1, positions.numel())


def no_gradient(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuse a call that autograd would have to record, or that brings tangents (a dual
    tensor's requires_grad is False)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or on detached tensors")
    refuse_tangents(name, *tensors)


def dense_places(t: torch.Tensor) -> bool:
    """Whether no two elements share a place (as far as strides nest)."""
    reach = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < reach:
            return False
        reach = stride * (size - 1) + reach
    return True


def _spans(t: torch.Tensor) -> Optional[Tuple[int, int, int]]:
    """``(n, pitch, length)``: t fills n spans of `length` elements, `pitch` apart; None where
    its strides are of another kind."""
    length, rest = 1, []
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if not rest and stride == length:
            length *= size
        else:
            rest.append((size, stride, length))
    return None if len(rest) > 1 else rest[0] if rest else (1, length, length)


def share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one type are sure to share a place: as far as each is one run of
    elements, or rows at one pitch (the parts of a fused projection)."""
    if a.numel() == 0 or b.numel() == 0 or a.device != b.device:
        return False
    x, y = _spans(a), _spans(b)
    if x is None or y is None or (x[0] > 1 and y[0] > 1 and x[1] != y[1]):
        return False
    pitch = x[1] if x[0] > 1 else y[1]
    apart = (b.data_ptr() - a.data_ptr()) // a.element_size()
    # spans i and j meet where apart - x's length < (i - j) pitch < apart + y's length
    least = max((apart - x[2]) // pitch + 1, 1 - y[0])
    most = min(-((-apart - y[2]) // pitch) - 1, x[0] - 1)
    return least <= most


def check_apart(out: torch.Tensor, name: str, may_be: Optional[torch.Tensor], **others: torch.Tensor) -> None:
    """Refuse an output that shares memory with what is read (or written) beside it; it may be
    `may_be` itself, whose rows are read before they are written."""
    for other, t in others.items():
        itself = t is may_be and out.data_ptr() == t.data_ptr() and out.shape == t.shape and out.stride() == t.stride()
        if not itself and share_memory(out, t):
            raise ValueError(f"{name} shares memory with {other}")


def check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int, dim: int, dtype: torch.dtype) -> None:
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dim() != 4 or t.shape[1] < 1 or tuple(t.shape[2:]) != (heads, dim):
            raise ValueError(f"{name} must be [pages, page_size, {heads}, {dim}], got {tuple(t.shape)}")
        if t.dtype != dtype:
            raise TypeError(f"{name} is {t.dtype}, the new tokens are {dtype}")
        if dim > 1 and t.stride(3) != 1:
            raise ValueError(f"{name} must have a dense last dimension")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} differ")


class Batch(NamedTuple):
    """The sequences of a call, as the kernels take them."""
    pages: torch.Tensor
    lengths: torch.Tensor
    starts: Optional[torch.Tensor]


def check_batch(page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor], tokens: int) -> Batch:
    for t, name, dims in ((page_table, "page_table", 2), (lengths, "lengths", 1), (starts, "starts", 1)):
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimension{'s' * (dims > 1)}, got shape {tuple(t.shape)}")
    batch = page_table.shape[0]
    if lengths.shape[0] != batch:
        raise ValueError(f"lengths {tuple(lengths.shape)} and page_table {tuple(page_table.shape)} are of different batches")
    if starts is not None:
        if starts.shape[0] != batch + 1:
            raise ValueError(f"starts must have batch + 1 = {batch + 1} entries, got {starts.shape[0]}")
        starts = starts.contiguous()
    elif tokens and (batch == 0 or tokens % batch):
        raise ValueError(f"without starts every sequence has the same number of tokens: {tokens} tokens, {batch} sequences")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1 or batch > 1 and page_table.stride(0) < page_table.shape[1]:
        page_table = page_table.contiguous()
    return Batch(page_table, lengths.contiguous(), starts)


def check_out(out: torch.Tensor, name: str, like: torch.Tensor) -> None:
    if out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"{name} must be {like.dtype} {tuple(like.shape)}, got {out.dtype} {tuple(out.shape)}")
    if (out.shape[-1] > 1 and out.stride(-1) != 1) or not dense_places(out):
        raise ValueError(f"{name} must have a dense last dimension and no two elements in one place")


def wrote(*tensors: torch.Tensor) -> None:
    """Tell autograd that these were written in place."""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


__all__ = ["Heads", "as_heads", "check_table", "check_positions", "no_gradient", "check_cache", "check_batch", "Batch",
           "check_out", "check_apart", "share_memory", "dense_places", "wrote", "MAX_HEAD_DIM", "_lib"]
