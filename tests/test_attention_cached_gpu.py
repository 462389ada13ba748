"""attention_cached against the formula in 64 bits over what the cache's bytes stand for."""

import pytest
import torch

from attention_reference import attention64, cache64, norm_bound, slots_of
from serving_reference import check_close, check_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")
WEIGHT = {BF16: 2.0 ** -10, FP32: 2.0 ** -20}   # two roundings of a weight: f16, or two f16 parts


def _attend(*a, **kw):
    from revealaiccl_b200.ops.attention import attention_cached
    return attention_cached(*a, **kw)


def _gen(seed=0):
    return torch.Generator(DEV).manual_seed(seed)


def _filled(pages, page, heads, dim, seed=0, **kw):
    """A cache of random bytes: every code, scales of 2^-6 to 16."""
    from revealaiccl_b200.ops.kv_cache import KVCache4
    gen = _gen(seed)
    cache = KVCache4.empty(pages, page, heads, dim, **kw)
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, device=DEV, dtype=torch.uint8))
        scales.view(torch.uint8).copy_(torch.randint(8, 89, scales.shape, generator=gen, device=DEV, dtype=torch.uint8))
    return cache


def _table(lengths, page, pages, seed=0, extra=1):
    """Random distinct pages for every sequence; entries behind a sequence's last page name none."""
    need = [-(-n // page) for n in lengths]
    assert sum(need) <= pages
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lengths), max(need, default=0) + extra), -7, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table.to(DEV)


def _spoil(cache, table, lengths):
    """What no sequence has: NaN scales and any codes."""
    used = torch.zeros(cache.pages * cache.page_size, dtype=torch.bool, device=DEV)
    for s in slots_of(table, lengths, cache.page_size):
        used[s.to(DEV)] = True
    spoil = ~used.view(cache.pages, 1, cache.page_size, 1)
    for scales in (cache.k_scales, cache.v_scales):
        b = scales.view(torch.uint8)
        b.copy_(torch.where(spoil, torch.tensor(0x7f, dtype=torch.uint8, device=DEV), b))


def _want(q, cache, table, lengths, scale=None, out_dtype=None):
    outs = []
    for i, s in enumerate(slots_of(table, lengths, cache.page_size)):
        k, v = cache64(cache, s.to(DEV))
        both = FP32 if q.dtype == FP32 or out_dtype == FP32 else BF16
        outs.append(attention64(q[i:i + 1], k, v, torch.tensor([len(s)], device=DEV), scale, WEIGHT[both], out_dtype))
    return [torch.cat(x) for x in zip(*outs)]


def _check(q, cache, table, lengths, *, scale=None, out_dtype=None, **kw):
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse = _attend(q, cache, table, lens, scale=scale, out_dtype=out_dtype, return_lse=True, check=True, **kw)
    want, wlse, bound, lbound, largest = _want(q, cache, table, lengths, scale, out_dtype)
    check_close(out, want, bound)
    empty = wlse == -INF
    assert torch.equal(lse.double() == -INF, empty)
    check_close(torch.where(empty, 0, lse.double()), torch.where(empty, 0, wlse), lbound)
    if want.abs().sum() > 0 and want.isfinite().all():
        check_norm(out, want, norm_bound(out.dtype, False, largest))
    return out, lse


def _q(n, heads, dim, dtype, seed=0, pad=0):
    t = torch.randn(n, heads * dim + pad, generator=_gen(seed + 100), device=DEV).to(dtype)
    return t[:, :heads * dim].unflatten(1, (heads, dim))


RAGGED = [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 257]


@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 4), (2, 7), (2, 12)])
def test_ragged(heads, group, dtype, out_dtype, dim, page):
    cache = _filled(90, page, heads, dim, seed=page + group)
    table = _table(RAGGED, page, cache.pages)
    _spoil(cache, table, RAGGED)
    _check(_q(len(RAGGED), heads * group, dim, dtype, pad=8), cache, table, RAGGED, out_dtype=out_dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads,group,page,lengths", [
    (1, 1, 64, [20011]), (1, 16, 16, [9000]), (2, 33, 256, [3001, 2]), (8, 4, 64, [1000]), (16, 1, 1024, [2000, 0, 1500]),
    (1, 128, 32, [700]), (2, 8, 64, [5000, 1, 4000, 63]),
])
def test_shared_by_many(heads, group, page, lengths, dtype):
    """Sequences that several warps, and several CTAs, have parts of."""
    cache = _filled(sum(-(-n // page) for n in lengths) + 1, page, heads, 128, seed=3)
    table = _table(lengths, page, cache.pages)
    _spoil(cache, table, lengths)
    _check(_q(len(lengths), heads * group, 128, dtype), cache, table, lengths)


@pytest.mark.parametrize("seqs", [1, 300, 1500])
def test_many_short(seqs):
    lengths = [(7 * i) % 40 for i in range(seqs)]
    cache = _filled(sum(-(-n // 16) for n in lengths) + 1, 16, 2, 64)
    table = _table(lengths, 16, cache.pages)
    _spoil(cache, table, lengths)
    _check(_q(seqs, 6, 64, BF16), cache, table, lengths)


def test_all_empty():
    cache = _filled(2, 16, 2, 64)
    table = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    out, lse = _check(_q(3, 4, 64, BF16), cache, table, [0, 0, 0])
    assert not out.any() and (lse == -INF).all()
    none = _attend(_q(0, 4, 64, BF16), cache, torch.zeros(0, 2, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV))
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e4, 1e30])
def test_queries_of_any_size(size, dtype):
    lengths = [500, 77]
    cache = _filled(40, 16, 2, 128)
    table = _table(lengths, 16, cache.pages)
    q = (_q(2, 6, 128, FP32) * size).to(dtype)
    _check(q, cache, table, lengths, scale=0.05 / size if size < 1e30 else 1e-32)
    _check(q, cache, table, lengths, scale=-0.05 / size if size < 1e30 else -1e-32)
    _check(q, cache, table, lengths, scale=0.0)


def test_peaked_and_growing():
    """Logits that grow along the sequence, so that maxima change in every tile, and one that outweighs all others."""
    from revealaiccl_b200.ops.kv_cache import KVCache4, kv_cache_write
    n = 900
    for order in (1, -1):
        cache = KVCache4.empty(60, 16, 1, 64)
        ramp = torch.linspace(-40, 40, n, device=DEV)[::order].contiguous() if order == 1 else torch.linspace(-40, 40, n, device=DEV).flip(0)
        k = torch.randn(n, 1, 64, generator=_gen(1), device=DEV) * 0.1
        k[:, 0, 0] = ramp
        v = torch.randn(n, 1, 64, generator=_gen(2), device=DEV)
        kv_cache_write(cache, k, v, torch.arange(n, device=DEV), check=True)
        q = _q(1, 4, 64, FP32)
        q[:, :, 0] = torch.tensor([1.0, 8.0, -3.0, 0.1], device=DEV)
        table = torch.arange(60, dtype=torch.int32, device=DEV)[None]
        _check(q, cache, table, [n], scale=1.0)
        _check(q.to(BF16), cache, table, [n], scale=1.0)


def test_values_of_any_size():
    from revealaiccl_b200.ops.kv_cache import KVCache4, kv_cache_write
    for dtype, size, unit in ((BF16, 1e-2, 1.0), (FP32, 400.0, 1.0), (FP32, 1e9, 2.0 ** 28), (BF16, 1e-9, 2.0 ** -32)):
        cache = KVCache4.empty(10, 16, 2, 64, v_unit=unit, k_unit=0.5)
        x = torch.randn(150, 2, 64, generator=_gen(4), device=DEV)
        kv_cache_write(cache, x, x * size, torch.arange(150, device=DEV), check=True)
        _check(_q(1, 4, 64, dtype), cache, torch.arange(10, dtype=torch.int32, device=DEV)[None], [150])


def test_nan_and_infinities_stay_where_they_are():
    lengths = [100, 200, 50]
    cache = _filled(30, 16, 2, 64)
    table = _table(lengths, 16, cache.pages)
    q = _q(3, 4, 64, BF16)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    base = _attend(q, cache, table, lens)
    page, row = int(table[1, 3]), 5
    cache.v_scales.view(torch.uint8)[page, 1, row, 2] = 0x7f     # sixteen values of head 1
    got = _attend(q, cache, table, lens, check=True)
    assert got[1, 2:, 32:48].isnan().all()
    got[1, 2:, 32:48] = base[1, 2:, 32:48]
    assert torch.equal(got, base)
    cache.v_scales.view(torch.uint8)[page, 1, row, 2] = 40
    base = _attend(q, cache, table, lens)
    cache.k_scales.view(torch.uint8)[page, 0, row, 0] = 0x7f
    got = _attend(q, cache, table, lens, check=True)
    assert got[1, :2].isnan().all()
    got[1, :2] = base[1, :2]
    assert torch.equal(got, base)
    cache.k_scales.view(torch.uint8)[page, 0, row, 0] = 40
    base = _attend(q, cache, table, lens)
    for odd in (NAN, INF):
        x = q.clone()
        x[2, 3, 7] = odd
        got = _attend(x, cache, table, lens, check=True)
        assert got[2, 3].isnan().all()
        got[2, 3] = base[2, 3]
        assert torch.equal(got, base)


def test_pages_and_lengths_outside_are_recorded():
    from revealaiccl_b200.ops.status import DeviceStatusError
    cache = _filled(10, 16, 1, 64)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
    q = _q(2, 2, 64, BF16)
    good = _attend(q, cache, table, torch.tensor([48, 32], dtype=torch.int32, device=DEV), check=True)
    for lengths, cut in (([48, 33 + 16], [48, 48]), ([-1, 32], [0, 32]), ([48, 2 ** 31 - 1], [48, 48])):
        with pytest.raises(DeviceStatusError, match="bounds"):
            _attend(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), check=True)
        got = _attend(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        with pytest.raises(DeviceStatusError):
            _attend(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), check=True)
        assert torch.equal(got, _attend(q, cache, table, torch.tensor(cut, dtype=torch.int32, device=DEV), check=True))
    for bad in (-1, 10, 2 ** 31 - 1):
        holes = table.clone()
        holes[1, 1] = bad
        with pytest.raises(DeviceStatusError, match="bounds"):
            _attend(q, cache, holes, torch.tensor([48, 48], dtype=torch.int32, device=DEV), check=True)
        got = _attend(q, cache, holes, torch.tensor([48, 48], dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        with pytest.raises(DeviceStatusError):
            _attend(q, cache, holes, torch.tensor([48, 48], dtype=torch.int32, device=DEV), check=True)
        assert torch.equal(got[0], good[0])
        # what is left: the other two pages
        two = torch.tensor([[3, 5]], dtype=torch.int32, device=DEV)
        want, _, bound, *_ = _want(q[1:], cache, two, [32])
        check_close(got[1:], want, bound)


def test_out_and_strides():
    lengths = [70, 9]
    cache = _filled(20, 16, 2, 64)
    table = _table(lengths, 16, cache.pages)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = _q(2, 4, 64, BF16)
    base = _attend(q, cache, table, lens)
    for q2 in (_window(q, 3), q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(_attend(q2, cache, table, lens), base)
    for out_dtype in (BF16, FP32):
        wide = torch.full((2, 5, 71), 7.0, device=DEV, dtype=out_dtype)
        out = wide[:, 1:, 3:67]
        version = out._version
        assert _attend(q, cache, table, lens, out=out).data_ptr() == out.data_ptr() and out._version > version
        want = _attend(q, cache, table, lens, out_dtype=out_dtype)
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert (wide == 7.0).all()
    skip = torch.full((2, 2 * table.shape[1]), -1, dtype=torch.int32, device=DEV)
    skip[:, :table.shape[1]] = table
    assert torch.equal(_attend(q, cache, skip[:, :table.shape[1]], lens), base)


def _window(t, off):
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + off + 2, dtype=t.dtype, device=DEV)
    wide[..., off:off + t.shape[-1]] = t
    return wide[..., off:off + t.shape[-1]]


def test_same_page_in_many_sequences():
    """A shared prefix: several sequences, and places of one, name the same pages."""
    cache = _filled(5, 16, 2, 64)
    table = torch.tensor([[1, 1, 2], [1, 1, 3], [1, 1, 1]], dtype=torch.int32, device=DEV)
    _check(_q(3, 4, 64, BF16), cache, table, [48, 40, 33])


def test_sums_go_in_a_fixed_order():
    lengths = [3000, 10, 1234]
    cache = _filled(300, 16, 2, 128)
    table = _table(lengths, 16, cache.pages)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = _q(3, 8, 128, FP32)
    base = _attend(q, cache, table, lens)
    for _ in range(5):
        assert torch.equal(_attend(q, cache, table, lens), base)


def test_captured():
    """A graph replayed with other lengths, pages and queries, while another graph of the same call runs next to it."""
    cache = _filled(300, 16, 2, 128)
    states = []
    for i in range(2):
        side = torch.cuda.Stream()
        q, lens = _q(3, 8, 128, BF16, seed=i), torch.ones(3, dtype=torch.int32, device=DEV)
        table = torch.zeros(3, 90, dtype=torch.int32, device=DEV)
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = _attend(q, cache, table, lens, return_lse=True)
        states.append((side, q, lens, table, graph, out, lse))
    torch.cuda.synchronize()
    for lengths in ([1, 0, 5], [1400, 3, 900], [16, 32, 33], [0, 0, 0]):
        for i, (side, q, lens, table, graph, out, lse) in enumerate(states):
            lens.copy_(torch.tensor(lengths, dtype=torch.int32))
            table[:, :] = _table(lengths, 16, 300, seed=i, extra=200)[:, :90]
            q.copy_(_q(3, 8, 128, BF16, seed=sum(lengths) + i))
        torch.cuda.synchronize()
        for side, *_, graph, _, _ in states:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for side, q, lens, table, graph, out, lse in states:
            want, wlse, bound, *_ = _want(q, cache, table, lengths)
            check_close(out, want, bound)
            assert torch.equal(lse == -INF, wlse == -INF)


def test_behind_32_bits():
    """Pages whose codes lie behind 2^32 bytes."""
    from revealaiccl_b200.ops.kv_cache import KVCache4
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 30 GB")
    pages = (2 ** 32 + 2 ** 22) // (8 * 128 * 64)
    cache = KVCache4.empty(pages, 128, 8, 128)
    part = _filled(3, 128, 8, 128)
    where = torch.tensor([pages - 1, 5, pages - 7], device=DEV)
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        getattr(cache, name).view(torch.uint8)[where] = getattr(part, name).view(torch.uint8)
    q = _q(1, 16, 128, BF16)
    n = torch.tensor([300], dtype=torch.int32, device=DEV)
    got = _attend(q, cache, where.int()[None], n, check=True)
    assert torch.equal(got, _attend(q, part, torch.arange(3, dtype=torch.int32, device=DEV)[None], n))
