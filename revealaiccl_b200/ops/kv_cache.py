"""The paged cache of keys and values in 4 bits (csrc/kernels/kv_cache.cu).

What a served model keeps between a prompt and its decode steps.
``kv_cache_write`` quantises new keys and values into it, ``attention_cached``
reads it for a decode step, ``kv_cache_read`` brings earlier tokens back for the
next chunk of a prompt (``attention_prompt``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import status as _status
from ._native import kernels

GROUP = 16                 # numbers that share a scale
HEAD_DIMS = (64, 128)
PAGE_SIZES = tuple(1 << i for i in range(4, 17))


@dataclass(frozen=True, eq=False)   # equal to itself: tensors' comparisons have no one answer
class KVCache4:
    """Pages of ``page_size`` tokens for every key head, 4.5 bits a number.

    Sixteen consecutive numbers x of a head of a token have one scale: s =
    e4m3(max |x| / (6 unit)), and are held as c = e2m1(x / (s unit)), both
    rounded to nearest, ties to even, and saturating; c s unit is what is read
    back.  Where a scale rounds to 0 so do its numbers, and a NaN makes its
    sixteen NaN.  With a unit of 1 scales reach from 2^-9 to 448: numbers up to
    2688.  For others choose ``k_unit`` and ``v_unit``, powers of two.

    k_codes, v_codes: uint8 [pages, kv_heads, page_size, head_dim / 2], the even
    dimension in the low four bits.  k_scales, v_scales: float8_e4m3fn [pages,
    kv_heads, page_size, head_dim / 16].  Contiguous, on 16 bytes.  A token's
    place ("slot") is page * page_size + its row in the page.  page_size: a power
    of two from 16 to 65536, at most 2^24 / kv_heads; less than 2^31 places.
    """

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    k_unit: float = 1.0
    v_unit: float = 1.0

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *, k_unit: float = 1.0, v_unit: float = 1.0,
              device: torch.device | str = "cuda") -> "KVCache4":
        """A cache of zeros."""
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"KVCache4: head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"KVCache4: page_size must be a power of two from 16 to 65536, got {page_size}")

        def zeros(width, dtype):
            return torch.zeros(pages, kv_heads, page_size, width, dtype=torch.uint8, device=device).view(dtype)

        return cls(zeros(head_dim // 2, torch.uint8), zeros(head_dim // GROUP, torch.float8_e4m3fn),
                   zeros(head_dim // 2, torch.uint8), zeros(head_dim // GROUP, torch.float8_e4m3fn), k_unit, v_unit)

    @property
    def pages(self) -> int:
        return self.k_codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]

    def _parts(self):
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.k_unit, self.v_unit


def kv_cache_write(cache: KVCache4, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *, check: bool = False) -> None:
    """Quantise keys and values k, v [N, kv_heads, head_dim] into the cache's slots [N].

    k and v: both bf16 or both fp32, rows contiguous, any other strides.  slots:
    int32 or int64; a token with a slot below zero is left out.  Where several
    tokens of a call name one slot, the last of them is kept.  A slot behind the
    cache's end is left out too, and recorded: ``check=True`` waits and raises.

    Enqueues one launch (for every 2^20 tokens) on the current stream without
    synchronising and can be captured in a CUDA graph.  There is no backward.
    """
    kernels().kv_cache_write(*cache._parts(), k, v, slots)
    if check:
        _status.check_serving(k.device)


def kv_cache_read(
    cache: KVCache4,
    slots: torch.Tensor,
    *,
    dtype: torch.dtype | None = None,
    k_out: torch.Tensor | None = None,
    v_out: torch.Tensor | None = None,
    check: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [N, kv_heads, head_dim] of the cache's slots [N], in order.

    dtype: bf16 (default) or fp32, or by ``k_out`` and ``v_out``, which may have
    any strides with contiguous rows but may not share memory with the cache or
    each other; they may lie between each other's rows by the same strides, as the
    two halves of a joint buffer do.  Nothing is rounded: a code times its scale has at most 6 bits.
    slots: int32 or int64, the same one any number of times; zeros come back for
    a slot below zero, and for one behind the cache's end, which is recorded:
    ``check=True`` waits and raises.

    Enqueues one launch on the current stream without synchronising and can be
    captured in a CUDA graph.
    """
    res = kernels().kv_cache_read(*cache._parts(), slots, dtype, k_out, v_out)
    if check:
        _status.check_serving(slots.device)
    return res


__all__ = ["GROUP", "HEAD_DIMS", "PAGE_SIZES", "KVCache4", "kv_cache_read", "kv_cache_write"]
