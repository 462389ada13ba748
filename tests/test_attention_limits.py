"""Where numbers of a call would not hold in the kernels: tables too wide for their counts, scales too large.  Refused before any GPU is needed."""

import pytest
import torch

from revealaiccl_b200.ops import _native

if not _native.has_kernels():  # pragma: no cover
    pytest.skip("kernel library not built", allow_module_level=True)

from revealaiccl_b200.ops.attention import attention_cached, attention_prompt
from revealaiccl_b200.ops.kv_cache import KVCache4

BF16, FP32 = torch.bfloat16, torch.float32
NO_GPU = "must be on a CUDA device"     # what the CPU's tensors meet behind all other checks


@pytest.mark.parametrize("seqs,heads,group,dtype,out_dtype,words", [
    (1, 127, 1, BF16, BF16, NO_GPU), (1, 129, 1, BF16, BF16, "2\\^32 or more"), (1, 256, 2, BF16, BF16, "2\\^32 or more"),
    (1, 16, 128, BF16, BF16, NO_GPU), (1, 16, 128, BF16, FP32, "2\\^32 or more"), (1, 16, 128, FP32, FP32, "2\\^32 or more"),
    (4096, 1, 1, BF16, BF16, NO_GPU), (4097, 1, 1, BF16, BF16, "2\\^37 or more"), (2049, 1, 17, BF16, BF16, "2\\^37 or more"),
    (2049, 1, 16, BF16, BF16, NO_GPU), (0, 1, 1, BF16, BF16, NO_GPU),
])
def test_widest_tables(seqs, heads, group, dtype, out_dtype, words):
    cache = KVCache4.empty(0, 65536, heads, 64, device="cpu")
    table = torch.zeros(1, 32767, dtype=torch.int32).expand(seqs, -1)     # 2^31 - 65536 tokens to a sequence
    q = torch.zeros(1, heads * group, 64, dtype=dtype).expand(seqs, -1, -1)
    with pytest.raises(ValueError, match=words):
        attention_cached(q, cache, table, torch.zeros(seqs, dtype=torch.int32), out_dtype=out_dtype)


@pytest.mark.parametrize("scale,words", [(2.3e38, NO_GPU), (-2.3e38, NO_GPU), (2.4e38, "scale must be"), (-3.4e38, "scale must be"), (1e300, "scale must be"),
                                         (float("nan"), "scale must be"), (float("inf"), "scale must be"), (0.0, NO_GPU)])
def test_scales(scale, words):
    """Exponentials are of base 2: a scale that overflows by log2(e) would turn logits of 0 into NaN."""
    cache = KVCache4.empty(1, 16, 1, 64, device="cpu")
    q, lens, table = torch.zeros(1, 1, 64, dtype=BF16), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match=words):
        attention_cached(q, cache, table, lens, scale=scale)
    with pytest.raises(ValueError, match=words):
        attention_prompt(q, q, q, torch.zeros(2, dtype=torch.int32), scale=scale)


def test_caches_are_told_apart_and_found():
    one, other = (KVCache4.empty(1, 16, 1, 64, device="cpu") for _ in range(2))
    assert one == one and one != other and [other, one].index(one) == 1 and {one: 1, other: 2}[other] == 2


@pytest.mark.parametrize("q_heads,kv_heads", [(2, 0), (0, 1), (1, 2), (129, 1)])
def test_plans_of_no_call(q_heads, kv_heads):
    """A quotient of zero heads would end the process."""
    q, k = torch.zeros(3, q_heads, 64, dtype=BF16), torch.zeros(3, kv_heads, 64, dtype=BF16)
    with pytest.raises(ValueError, match="heads"):
        _native.kernels().attention_prompt_plan(q, k, k, 1, 148)
    with pytest.raises(ValueError, match="heads"):
        attention_prompt(q, k, k, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        _native.kernels().attention_prompt_plan(q[0], k, k, 1, 148)
