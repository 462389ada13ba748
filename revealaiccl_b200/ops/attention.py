"""Attention next to the experts of a served layer.

``attention_prompt`` (csrc/kernels/attention_prompt.cu) is for whole prompts or
chunks of them, ``attention_cached`` (csrc/kernels/attention_cached.cu) for the
one new token of each sequence in a decode step, over the paged cache in 4 bits
of ``kv_cache.py``.  Both with grouped heads: query head h reads key head h //
(query heads / key heads).
"""

from __future__ import annotations

import torch

from . import status as _status
from ._native import kernels
from .kv_cache import KVCache4


def attention_cached(
    q: torch.Tensor,
    cache: KVCache4,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    return_lse: bool = False,
    check: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """out[b, h] = softmax(scale * q[b, h] K^T) V over the first lengths[b] tokens that the cache has of sequence b.

    q [B, heads, head_dim]: bf16 or fp32, rows contiguous, any other strides;
    heads a multiple (up to 128) of the cache's.  block_table int32 [B, n]:
    token i of sequence b lies in page block_table[b, i // page_size]; entries
    behind a sequence's last page are not read.  lengths int32 [B]; an empty
    sequence gets zeros.  scale: default head_dim ** -0.5.

    The query heads of a key head are worked on in equal chunks of up to 16, or 8
    where q or the result is fp32, and each chunk reads the cache again.  A row of
    the table has room for less than 2^31 tokens, and for less than 2^38 by key
    heads and chunks; all rows for less than 2^43 by them.

    Sums, maxima and the result are kept in fp32 and rounded once, to out_dtype
    (default: q's type; fp32 queries give fp32).  For bf16 results the
    probabilities enter their product as f16 numbers; for fp32 results queries
    and probabilities are two f16 numbers each, 22 bits (for a number 2^-14 or
    more below its row's largest, fewer).
    ``return_lse``: also log sum exp(scale * q K^T), fp32 [B, heads], -inf for
    empty sequences, to join results over parts of a context.

    A page that is not the cache's is left out, a length behind the table's row
    cut, and both are recorded: ``check=True`` waits and raises.  Enqueues two
    launches on the current stream without synchronising and can be captured in
    a CUDA graph.  Workspace, of torch's allocator: up to 20 MB.  There is no
    backward: tensors that require a gradient or carry a tangent are refused.
    """
    res, lse = kernels().attention_cached(q, *cache._parts(), block_table, lengths, scale, out, out_dtype, return_lse)
    if check:
        _status.check_serving(q.device)
    return (res, lse) if return_lse else res


def attention_prompt(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor | None = None,
    *,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    check: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """out[i, h] = softmax(scale * q[i, h] K^T) V over the keys of token i's sequence that it sees.

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim]: all bf16
    or all fp32, rows contiguous, any other strides; heads a multiple (up to
    128) of kv_heads.  Sequences are packed: tokens cu_seqlens_q[b] to
    cu_seqlens_q[b + 1] of q attend to tokens cu_seqlens_k[b] to
    cu_seqlens_k[b + 1] of k and v (int32, default: the same).  ``causal``: the
    last token of a sequence in q sees all its keys, every one before it one
    less, so k and v may begin with earlier tokens of a chunked prompt.  A token
    that sees nothing gets zeros, and rows of ``out`` before the first and behind
    the last sequence are left as they were.  What a token does not see does not
    enter its result, infinities and NaN included; of what it does see, an
    infinity whose weight is below 2^-75 may come out as NaN.  scale: default
    head_dim ** -0.5.  At most 2^16 sequences.

    Sums, maxima and the result are kept in fp32 and rounded once, to q's type.
    With bf16 inputs the probabilities enter their product as bf16 numbers, up to
    2^-8 off each; fp32 inputs and their probabilities are three bf16 numbers each,
    24 bits (an infinite logit may come out as NaN).  Values below 2^-100 lose bits
    (in bf16 below 2^-85 where logits rise by more than 15 after a token's first 128
    keys), as do fp32 queries and keys below 2^-110.  ``return_lse``: also log sum exp(scale * q K^T),
    fp32 [tokens, heads], -inf where a token sees nothing or logits of -inf alone,
    undefined outside of the sequences.

    Offsets that lie outside of the tensors or fall are cut and recorded:
    ``check=True`` waits and raises.  Enqueues one to three launches on the
    current stream without synchronising and can be captured in a CUDA graph;
    rows that do not start on 16 bytes are copied first.  Workspace, of torch's
    allocator: those copies, one and a half times the inputs in fp32, and with few
    tiles of many keys up to 32 times the result in fp32.  There is no backward:
    tensors that require a gradient or carry a tangent are refused.
    """
    res, lse = kernels().attention_prompt(q, k, v, cu_seqlens_q, cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k,
                                          causal, scale, out, return_lse)
    if check:
        _status.check_serving(q.device)
    return (res, lse) if return_lse else res


__all__ = ["attention_cached", "attention_prompt"]
