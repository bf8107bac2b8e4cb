"""Attention of new tokens over a paged cache on gfx950 (MI355X).

Each sequence's new tokens (one in a decode step, a chunk of a prompt, or both in
one call) attend to all of the sequence's positions up to their own, which
``kernels.hip.paged_append`` put into the cache, the new ones among them: with
``p`` a token's position, over the keys ``j <= p`` (and ``j > p - window``)

    s_j = scale q . k_j       (softcap > 0: softcap tanh(s_j / softcap))
    out = sum_j softmax(s)_j v_j

Query heads share key heads in groups (head ``h`` reads ``h * kv_heads // q_heads``).
One pass over the keys with a running maximum and sum in fp32
(``csrc/paged_attention.hip``); the keys of few rows are cut over the whole GPU and
joined in a fixed order, so results are reproducible.

Rules at the edges: a key past the sequence's length, past the window or on a page
outside the cache takes no part, whatever it or its value holds. A key that is seen
with a score of -inf has the weight 0, and its value takes part with that (0 times
what is not finite is NaN). A token that sees no key gives 0, as does one that sees
only scores of -inf beside finite values; a NaN score gives a NaN row.

For serving: it has no gradient. No counterpart in the reference.
"""

import math
import os
from typing import Optional

import torch

from kernels.hip import _heads, _lib

KERNEL_TYPE = "paged_attention"
BACKEND = "hip"

HIP_SRC = os.path.join(_lib.CSRC_DIR, "paged_attention.hip")

MAX_DIM = 1024


def check_scores(scale: Optional[float], softcap: float, window: int, dim: int):
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    softcap, window = float(softcap), int(window)
    if not 1e-18 <= scale <= 1e18:
        raise ValueError(f"scale must be between 1e-18 and 1e18, got {scale}")
    if softcap != 0.0 and not 1e-3 <= softcap <= 1e4:
        raise ValueError(f"softcap must be 0 (off) or between 1e-3 and 1e4, got {softcap}")
    if window < 0:
        raise ValueError(f"window must be 0 (none) or positive, got {window}")
    return scale, softcap, window


def kernel_fn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
              softcap: float = 0.0, window: int = 0, max_chunk: Optional[int] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q`` over the cached keys and values of its sequences.

    Args:
        q: ``[tokens, q_heads, dim]`` of the caches' type, dim at most 1024; q_heads a
            multiple of the caches' heads.
        k_cache, v_cache: ``[pages, page_size, kv_heads, dim]`` fp32, fp16 or bf16, any
            strides with a dense last dimension.
        page_table, lengths, starts: as in ``kernels.hip.paged_append``.
        scale: of the scores; None: ``1 / sqrt(dim)``.
        softcap: cap of the scaled scores, 1e-3 to 1e4 (0 = off).
        window: the most keys that a token sees, its own the last (0 = all).
        max_chunk: the most new tokens of one sequence, where the caller knows: it
            chooses the kernel, results do not depend on its being right. None: all of
            the call's tokens (without starts: those of each sequence), which takes the
            kernel for many rows: a decode step of 64 sequences given by starts alone
            takes 298 us, with max_chunk=1 (or without starts) 265.
        out: where the result goes (rows of no sequence stay as they are), may be q
            itself and shares no memory with the caches; None: a new tensor (with zeros
            there).
    """
    host = _lib.native(q, k_cache, v_cache, page_table, lengths, *_lib.given(starts, out))
    if host is not None and q.dim() == 3 and q.shape[2]:
        numbers = check_scores(scale, softcap, window, q.shape[2])
        if max_chunk is not None and int(max_chunk) < 1:
            raise ValueError(f"max_chunk must be positive, got {max_chunk}")
        done = host.paged_attention(q, k_cache, v_cache, page_table, lengths, starts, *numbers,
                                    q.shape[0] if max_chunk is None else int(max_chunk), out)
        if done is not None:
            return done if out is None else out
    _lib.require_device(q, k_cache, v_cache, page_table, lengths, starts, out)
    _heads.no_gradient(KERNEL_TYPE, q, k_cache, v_cache, out)
    _lib.dtype_code(q.dtype)
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError(f"q must be [tokens, q_heads, dim] and the caches [pages, page_size, kv_heads, dim], "
                         f"got {tuple(q.shape)} and {tuple(k_cache.shape)}")
    tokens, heads, dim = q.shape
    kv_heads = k_cache.shape[2]
    if not 0 < dim <= MAX_DIM:
        raise ValueError(f"the head dimension must be 1 to {MAX_DIM}, got {dim}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads do not share {kv_heads} key heads evenly")
    _heads.check_cache(k_cache, v_cache, kv_heads, dim, q.dtype)
    scale, softcap, window = check_scores(scale, softcap, window, dim)
    batch = _heads.check_batch(page_table, lengths, starts, tokens)
    if max_chunk is not None and int(max_chunk) < 1:
        raise ValueError(f"max_chunk must be positive, got {max_chunk}")
    if starts is None:
        chunk = tokens // max(1, page_table.shape[0])
    else:
        chunk = tokens if max_chunk is None else min(int(max_chunk), tokens)
    zero = out is None
    if zero:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _heads.check_out(out, "out", q)
        _heads.check_apart(out, "out", q, q=q, k_cache=k_cache, v_cache=v_cache)
    q = q if dim == 1 or q.stride(2) == 1 else q.contiguous()
    size = q.element_size()
    if dim * size % 16 == 0 and (q.data_ptr() | q.stride(0) * size | q.stride(1) * size) % 16:
        q = q.clone(memory_format=torch.contiguous_format)  # off the alignment the whole cache goes through the slow kernel
    if tokens:
        _lib.paged_attention(q, k_cache, v_cache, batch, out, max(1, chunk), scale, softcap, window, zero)
    if not zero:
        _heads.wrote(out)
    return out
