"""attention_cached where what several warps and CTAs have of a sequence hardly counts, and over rows of pages of any width."""

import pytest
import torch

from test_attention_cached_gpu import BF16, DEV, FP32, NAN, _attend, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [100, 128, 500, 20000])
@pytest.mark.parametrize("below", [1.0, 100.0, 200.0])
def test_nan_of_a_part_that_hardly_counts(below, tokens, dim, dtype):
    """The first 64 tokens lie `below` under the others; a NaN among them is seen whichever warps and CTAs have the rest."""
    from revealaiccl_b200.ops.kv_cache import KVCache4, kv_cache_write
    cache = KVCache4.empty(-(-tokens // 64), 64, 2, dim)
    k = torch.zeros(tokens, 2, dim, device=DEV)
    k[64:, :, 0] = 6.0                         # of a scale of 1: held as it is
    v = torch.randn(tokens, 2, dim, generator=_gen(1), device=DEV)
    q = torch.zeros(1, 6, dim, device=DEV, dtype=dtype)
    q[:, :, 0] = below / 6.0
    table = torch.arange(cache.pages, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([tokens], dtype=torch.int32, device=DEV)

    def out(values):
        kv_cache_write(cache, k, values, torch.arange(tokens, device=DEV), check=True)
        return _attend(q, cache, table, lens, scale=1.0, check=True)

    base = out(v)
    assert base.isfinite().all()
    v2 = v.clone()
    v2[5, 0, 20] = NAN                         # its sixteen too
    want = base.clone()
    want[:, :3, 16:32] = NAN
    got = out(v2)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
