"""New keys and values into a paged cache, keys and queries normed and turned on
the way, on gfx950 (MI355X).

The cache is ``[pages, page_size, kv_heads, dim]``, for keys and for values (any
strides with a dense last dimension: a ``[pages, kv_heads, page_size, dim]`` cache is
passed transposed). Position ``p`` of sequence ``b`` lives in slot ``p % page_size``
of page ``page_table[b, p // page_size]``. A call brings every sequence's new
tokens, one after the other: sequence ``b``'s are rows ``starts[b]`` to
``starts[b + 1]`` and are the last of its ``lengths[b]`` positions (lengths count the
new tokens). The same ``page_table``, ``lengths`` and ``starts`` then go to
``kernels.hip.paged_attention``.

One launch (``csrc/heads.hip``) reads queries, keys and values once, applies what
``kernels.hip.qk_norm_rotary`` does at each token's position, and writes keys and
values into their slots. Nothing is written for a token of no sequence, at a
negative position, past ``page_table``'s width or on a page outside the cache. Two
new tokens must not share a slot: pages that sequences share are for positions
before the new ones.

For serving: it has no gradient. No counterpart in the reference.
"""

import os
from typing import Optional

import torch

from kernels.hip import _heads, _lib
from kernels.hip.qk_norm_rotary import DEFAULT_EPS, check_eps, check_weight

KERNEL_TYPE = "paged_append"
BACKEND = "hip"

HIP_SRC = os.path.join(_lib.CSRC_DIR, "heads.hip")


def kernel_fn(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *, q: Optional[torch.Tensor] = None,
              q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = DEFAULT_EPS,
              table: Optional[torch.Tensor] = None, interleaved: bool = False,
              q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes k and v into the caches; returns q normed and turned (None without q).

    Args:
        k, v: ``[tokens, kv_heads, dim]``, of the caches' type.
        k_cache, v_cache: ``[pages, page_size, kv_heads, dim]`` fp32, fp16 or bf16, written in place.
        page_table: int32 ``[batch, most pages of a sequence]``; entries past a
            sequence's length are not read.
        lengths: int32 ``[batch]``, with the new tokens.
        starts: int32 ``[batch + 1]``, ascending from 0, or None: the same number of
            tokens for each sequence (one, in a decode step).
        q: ``[tokens, q_heads, dim]``, or None.
        q_weight, k_weight: ``[dim]`` of the head norms, or None.
        table, interleaved: as in ``kernels.hip.rotary``; None: no rotation. A
            position past the table is written as NaN.
        q_out: where q's result goes (rows of no sequence stay as they are), may be
            q itself and shares no memory with the other tensors; None: a new tensor
            (with zeros there).
    """
    eps, interleaved = check_eps(eps), bool(interleaved)
    host = _lib.native(k, v, k_cache, v_cache, page_table, lengths, *_lib.given(starts, q, q_weight, k_weight, table, q_out))
    if host is not None:
        done = host.paged_append(k, v, k_cache, v_cache, page_table, lengths, starts, q, q_weight, k_weight, eps, table,
                                 interleaved, q_out)
        if done is not None:
            return q_out if q_out is not None else done[1]
    _lib.require_device(k, v, k_cache, v_cache, page_table, lengths, starts, q, q_weight, k_weight, table, q_out)
    _heads.no_gradient(KERNEL_TYPE, k, v, k_cache, v_cache, q, q_weight, k_weight, q_out)
    _lib.dtype_code(k.dtype)
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"k and v must be [tokens, kv_heads, dim], got {tuple(k.shape)} and {tuple(v.shape)}")
    tokens, heads, dim = k.shape
    if heads < 1 or not 0 < dim <= _heads.MAX_HEAD_DIM:
        raise ValueError(f"k must have heads of 1 to {_heads.MAX_HEAD_DIM} elements, got shape {tuple(k.shape)}")
    if v.dtype != k.dtype:
        raise TypeError(f"k is {k.dtype}, v is {v.dtype}")
    _heads.check_cache(k_cache, v_cache, heads, dim, k.dtype)
    if not _heads.dense_places(k_cache) or not _heads.dense_places(v_cache):
        raise ValueError("two places of a cache share their memory")
    if k_cache.numel() and k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError("k_cache and v_cache begin at the same place")
    _heads.check_apart(k_cache, "k_cache", None, v_cache=v_cache)
    batch = _heads.check_batch(page_table, lengths, starts, tokens)
    if q is None:
        if q_weight is not None or q_out is not None:
            raise ValueError("q_weight or q_out without q")
    else:
        if q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != dim:
            raise ValueError(f"q must be [{tokens}, q_heads, {dim}], got {tuple(q.shape)}")
        if q.dtype != k.dtype:
            raise TypeError(f"q is {q.dtype}, k is {k.dtype}")
    if q_weight is not None:
        q_weight = check_weight(q_weight, "q_weight", q)
    if k_weight is not None:
        k_weight = check_weight(k_weight, "k_weight", k)
    if table is not None:
        _heads.check_table(table, dim)
    zero = q_out is None
    if q is not None:
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _heads.check_out(q_out, "q_out", q)
            _heads.check_apart(q_out, "q_out", q, q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache)
        q = q if dim == 1 or q.stride(2) == 1 else q.contiguous()
    k = k if dim == 1 or k.stride(2) == 1 else k.contiguous()
    v = v if dim == 1 or v.stride(2) == 1 else v.contiguous()
    _lib.paged_append(q, k, v, q_weight, k_weight, table, q_out, k_cache, v_cache, batch, eps, interleaved, zero)
    _heads.wrote(k_cache, v_cache)
    if not zero:
        _heads.wrote(q_out)
    return q_out
