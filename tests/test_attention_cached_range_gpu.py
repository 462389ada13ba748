"""attention_cached where what several warps and CTAs have of a sequence hardly counts, and over rows of pages of any width."""

import pytest
import torch

from test_attention_cached_gpu import BF16, DEV, FP32, NAN, _attend, _check, _filled, _gen, _q, _table

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


@pytest.mark.parametrize("page", [16, 32])
def test_longest_row_of_the_table(page):
    """2^31 tokens but a page's, of one page over and over; a length behind the row is cut to that and recorded."""
    from revealaiccl_b200.ops.kv_cache import KVCache4, kv_cache_write
    from revealaiccl_b200.ops.status import DeviceStatusError, check_serving
    cache = KVCache4.empty(1, page, 1, 64)
    v = torch.randint(-6, 7, (page, 1, 64), generator=_gen(3), device=DEV).float()
    v[v.abs() == 5] = 0.0                          # what 4 bits have, at a scale of 1
    v[:, :, ::16] = 6.0
    kv_cache_write(cache, torch.zeros_like(v), v, torch.arange(page, device=DEV), check=True)
    row = torch.zeros(1, 2 ** 31 // page - 1, dtype=torch.int32, device=DEV)
    most = 2 ** 31 - page
    for lengths in ([most, 5, 0, page], [5, 2 ** 31 - 1, 1, most]):
        q = torch.randn(4, 3, 64, generator=_gen(4), device=DEV).to(BF16)
        out, lse = _attend(q, cache, row.expand(4, -1), torch.tensor(lengths, dtype=torch.int32, device=DEV), return_lse=True)
        if max(lengths) > most:
            with pytest.raises(DeviceStatusError, match="bounds"):
                check_serving(DEV)
        check_serving(DEV)
        for b, n in enumerate(lengths):
            n = min(n, most)
            want = torch.zeros(64, dtype=torch.float64, device=DEV) if n == 0 else v[:min(n, page), 0].double().mean(0)
            # weights of 128 and small whole numbers add up exactly up to 2^24 times their unit, which a warp's share is below
            assert ((out[b].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()
            assert (lse[b].double() - (torch.tensor(float(n), dtype=torch.float64).log().item() if n else -float("inf"))).abs().nan_to_num(0.0).max() < 1e-5


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_tens_of_thousands_of_sequences(dtype):
    """Short ones, empty ones and some that several CTAs share; the time grows with their number, not with its square."""
    from revealaiccl_b200.ops.kv_cache import KVCache4, kv_cache_write
    n, heads, group, dim, page = 65536, 2, 3, 64, 16
    cache = KVCache4.empty(400, page, heads, dim)
    kv = torch.randn(2, 6400, heads, dim, generator=_gen(5), device=DEV)
    kv_cache_write(cache, kv[0], kv[1], torch.arange(6400, device=DEV), check=True)
    table = torch.arange(400, dtype=torch.int32, device=DEV).expand(n, -1)
    lens = torch.randint(0, 70, (n,), generator=_gen(6), device=DEV).int()
    lens[1000:3000] = 0
    long = torch.tensor([0, 17, 2999, 40000, n - 1], device=DEV)
    lens[long] = torch.tensor([6400, 6399, 3000, 6001, 5000], device=DEV).int()
    q = torch.randn(1, heads * group, dim, generator=_gen(7), device=DEV).to(dtype)
    out, lse = _attend(q.expand(n, -1, -1), cache, table, lens, return_lse=True, check=True)
    kinds = torch.cat([torch.arange(70, device=DEV), lens[long]]).int()     # one sequence of each length
    want, wlse = _attend(q.expand(len(kinds), -1, -1), cache, table[:len(kinds)], kinds, return_lse=True, check=True)
    kind = lens.long().clamp_max(69)
    kind[long] = torch.arange(70, 75, device=DEV)
    # both are within 2^-8 (bf16), 2^-18 of the values' mean size (fp32) of the formula; equal where a warp has all of a sequence
    bound = (2.0 ** -7 if dtype == BF16 else 2.0 ** -17) * 4
    assert ((out.float() - want[kind].float()).abs() <= bound).all()
    assert torch.equal(lse == -float("inf"), wlse[kind] == -float("inf")) and not out[lens == 0].any()
    assert ((lse - wlse[kind]).nan_to_num(0.0).abs() <= 1e-5).all()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    _attend(q.expand(n, -1, -1), cache, table, lens)
    end.record()
    end.synchronize()
    assert start.elapsed_time(end) < 10.0, "65536 sequences of 35 tokens: 0.4 ms of tiles"


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size,unit", [(1e30, 2.0 ** 40), (1e38, 2.0 ** 63), (1e-30, 2.0 ** 63), (1e-10, 2.0 ** -64), (1e30, 2.0 ** -64)])
def test_queries_and_units_that_meet_in_the_scale(size, unit, dtype):
    """Logits of ordinary size from queries, a unit of the keys and a scale whose products are not, two by two."""
    lengths = [500, 77]
    cache = _filled(40, 16, 2, 128, k_unit=unit, v_unit=0.25)
    table = _table(lengths, 16, cache.pages)
    q = (_q(2, 6, 128, FP32).clamp(-3, 3) * size).to(dtype)
    for sign in (1, -1):
        _check(q, cache, table, lengths, scale=sign * 0.05 / size / unit)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", [3e-38, 1e-39, 1e-40])
def test_queries_below_the_least_normal_number(size, dtype):
    """They keep the bits that they have."""
    lengths = [500, 77]
    cache = _filled(40, 16, 2, 128)
    table = _table(lengths, 16, cache.pages)
    q = _q(2, 6, 128, FP32)
    q[1, 2:4] = 0.0
    q = (q * size).to(dtype)
    assert q.any()                              # torch has not made zeros of them
    for sign in (1, -1):
        _check(q, cache, table, lengths, scale=sign * min(0.05 / size, 2e38))
