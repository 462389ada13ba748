"""kv_cache_write of more tokens than one launch has: the last token of a slot is kept, and the time grows with the tokens."""

import pytest
import torch

from test_kv_cache_gpu import BF16, DEV, FP32, _cache, _gen, _write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,wide", [(BF16, True), (FP32, False)], ids=["bf16", "fp32"])
@pytest.mark.parametrize("pad", [0, 3], ids=["aligned", "strided"])
def test_slots_named_again_by_later_launches(pad, dtype, wide):
    n, dim = 2 ** 21 + 77, 64
    gen = _gen(1)
    got, want = (_cache(2 ** 19 // 64, 64, 1, dim) for _ in range(2))
    places = got.pages * 64
    slots = torch.randint(-places // 8, places, (n,), generator=gen, device=DEV)
    slots[2 ** 20 - 2:2 ** 20 + 2] = 5             # around the first border
    slots[-1] = slots[0] = 7
    k, v = (torch.randn(n, dim + pad, generator=gen, device=DEV).to(dtype)[:, None, :dim] for _ in range(2))
    _write(got, k, v, slots if wide else slots.int())
    last = torch.full((places,), -1, device=DEV).scatter_reduce(0, slots.clamp_min(0), torch.where(slots >= 0, torch.arange(n, device=DEV), -1), "amax")
    named = (last >= 0).nonzero()[:, 0]
    assert len(named) > 0.9 * places and last[5] >= 2 ** 20 + 1 and last[7] == n - 1
    for part in named.split(100000):               # every slot once
        _write(want, k[last[part]], v[last[part]], part)
    for a, b in ((got.k_codes, want.k_codes), (got.v_codes, want.v_codes), (got.k_scales.view(torch.uint8), want.k_scales.view(torch.uint8)),
                 (got.v_scales.view(torch.uint8), want.v_scales.view(torch.uint8))):
        assert torch.equal(a, b)


def test_time_grows_with_the_tokens():
    """A quarter of the tokens takes a quarter of the time, not a sixteenth: the ratio of 8 between both is their geometric mean."""
    from revealaiccl_b200.ops.kv_cache import kv_cache_write
    times = {}
    for n in (2 ** 21, 2 ** 23):
        cache = _cache(n // 64, 64, 1, 64)
        k = torch.randn(n, 1, 64, device=DEV, dtype=BF16)
        slots = torch.randperm(n, device=DEV)
        kv_cache_write(cache, k, k, slots)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        kv_cache_write(cache, k, k, slots)
        end.record()
        end.synchronize()
        times[n] = start.elapsed_time(end)
    assert times[2 ** 23] < 8 * times[2 ** 21], times
