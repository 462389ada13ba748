"""kv_cache_write and kv_cache_read against the definition in 64 bits: every number equal."""

import pytest
import torch

from attention_reference import cache64, quantise64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _cache(pages, page, heads, dim, **kw):
    from revealaiccl_b200.ops.kv_cache import KVCache4
    return KVCache4.empty(pages, page, heads, dim, **kw)


def _write(*a, **kw):
    from revealaiccl_b200.ops.kv_cache import kv_cache_write
    kv_cache_write(*a, check=True, **kw)


def _read(*a, **kw):
    from revealaiccl_b200.ops.kv_cache import kv_cache_read
    return kv_cache_read(*a, check=True, **kw)


def _gen(seed=0):
    return torch.Generator(DEV).manual_seed(seed)


def _randn(*shape, gen, dtype=FP32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def _same(got, want):
    """Equal numbers; NaN where the definition has it."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))


def _check(cache, k, v, slots):
    """Write, then compare what the bytes stand for, and what is read back, with the definition."""
    _write(cache, k, v, slots)
    used = (slots >= 0)[:, None, None]
    want = [torch.where(used, quantise64(x, u), 0.0) for x, u in ((k, cache.k_unit), (v, cache.v_unit))]
    for got, w in zip(cache64(cache, slots), want):
        _same(got, w)
    for dt in (BF16, FP32):
        for got, w in zip(_read(cache, slots, dtype=dt), want):
            assert got.dtype == dt
            _same(got, w)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n,heads,dim,page,wide", [(1, 1, 64, 16, True), (1, 8, 128, 64, False), (3, 5, 64, 32, True), (37, 3, 128, 16, True),
                                                   (297, 2, 64, 128, False), (1111, 1, 128, 256, True), (5000, 2, 64, 16, False)])
def test_random(n, heads, dim, page, wide, dtype):
    gen = _gen(n)
    cache = _cache(-(-n // page) + 2, page, heads, dim)
    slots = torch.randperm(cache.pages * page, generator=gen, device=DEV)[:n].to(torch.int64 if wide else torch.int32)
    if n > 2:
        slots[[0, n - 1]] = -1
        slots[n // 2] = -2 ** 31
    k, v = (_randn(n, heads, dim, gen=gen, dtype=dtype, scale=s) for s in (3.0, 0.2))
    _check(cache, k, v, slots)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_edges(dtype):
    """Every scale with every number next to an edge between two codes: ties and their neighbours, zeros of either sign."""
    scales = torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    x = torch.zeros(126, 64, dtype=torch.float64)
    for i in range(4):                       # four groups to a row of 64, with different neighbours of the edges
        x[:, 16 * i] = 6 * scales            # the group's scale, by its largest
        x[:, 16 * i + 1:16 * i + 8] = edges * scales[:, None]
        x[:, 16 * i + 8:16 * i + 15] = -edges * scales[:, None]
        x[:, 16 * i + 15] = -0.0
    x = x.to(dtype).to(DEV)
    tiny = torch.finfo(dtype).eps
    bits = torch.int16 if dtype == BF16 else torch.int32
    for i, step in ((1, 1), (2, -1)):        # the next number up, the next one down
        part = x[:, 16 * i + 1:16 * i + 15].contiguous()
        x[:, 16 * i + 1:16 * i + 15] = (part.view(bits) + step).view(dtype)
    x[:, 49:63] *= 1 + tiny                  # and a few roundings further
    cache = _cache(8, 16, 1, 64)
    slots = torch.arange(126, device=DEV)
    _check(cache, x[:, None], x.flip(0)[:, None], slots)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_scale_edges(dtype):
    """Largest numbers at, and next to, the edges between two scales, beyond the largest and below the smallest."""
    e4m3 = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    top = 6 * (e4m3[1:] + e4m3[:-1]) / 2
    bits = torch.int16 if dtype == BF16 else torch.int32
    base = top.to(dtype)
    rows = torch.cat([(base.view(bits) + d).view(dtype) for d in (-1, 0, 1)]
                     + [torch.tensor([2688.0, 2689.0, 1e5, 3e38, 1e-38, 1e-30, 0.0, 5e-3, 2.0 ** -10 * 6], dtype=dtype)])
    x = torch.zeros(len(rows), 1, 64, dtype=dtype)
    x[:, 0, ::16] = rows[:, None]
    x[:, 0, 1::16] = -rows[:, None] / 3
    x[:, 0, 2::16] = rows[:, None] / 17
    x = x.to(DEV)
    _check(_cache(len(rows) // 16 + 1, 16, 1, 64), x, -x, torch.arange(len(rows), device=DEV))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_infinities_and_nan(dtype):
    x = _randn(6, 2, 128, gen=_gen(1), dtype=dtype)
    x[0, 0, 3], x[1, 1, 20], x[2, 0, 127] = INF, -INF, NAN
    x[3, 1, 64], x[3, 1, 65] = INF, NAN
    x[4, 0, :] = INF
    _check(_cache(1, 16, 2, 128), x, x.flip(0).contiguous(), torch.arange(6, device=DEV))


def test_units():
    x = _randn(20, 2, 64, gen=_gen(2), scale=1e6)
    cache = _cache(2, 16, 2, 64, k_unit=2.0 ** 14, v_unit=2.0 ** -30)
    _check(cache, x, x * 1e-14, torch.arange(20, device=DEV))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("offset,token,order", [(0, 8 * 200, "thd"), (8, 3 * 128 * 2 + 8, "thd"), (3, 3 * 128 + 5, "thd"), (0, 0, "htd")])
def test_strides(offset, token, order, dtype):
    """Rows out of wider ones, on and off 16 bytes, heads before tokens; into outputs of other strides."""
    n, h, d = 19, 3, 128
    gen = _gen(3)
    cache = _cache(3, 16, h, d)
    slots = torch.randperm(48, generator=gen, device=DEV)[:n]

    def rows(fill=None):
        if order == "htd":
            t = _randn(h, n, d, gen=gen, dtype=dtype).transpose(0, 1)
        else:
            t = _randn(n * token + offset + 3 * d, gen=gen, dtype=dtype)[offset:].as_strided((n, h, d), (token, d, 1), offset)
        return t

    k, v = rows(), rows()
    _check(cache, k, v, slots)
    ko, vo = rows(), rows()
    kb = ko.as_strided((ko.untyped_storage().nbytes() // ko.element_size(),), (1,), 0)
    mark = torch.ones_like(kb, dtype=torch.bool)
    mark.as_strided(ko.shape, ko.stride(), ko.storage_offset()).fill_(False)
    before = kb.clone()
    version = ko._version
    _read(cache, slots, k_out=ko, v_out=vo)
    assert ko._version > version
    want = cache64(cache, slots)
    _same(ko, want[0])
    _same(vo, want[1])
    assert torch.equal(kb[mark], before[mark])


@pytest.mark.parametrize("n", [2, 50, 700, 3000])
@pytest.mark.parametrize("kinds", [1, 7, 400])
def test_last_of_a_slot_is_kept(n, kinds):
    """Many tokens for few places: whatever their CTAs are, the last one's keys and values are what is held, none mixed."""
    gen = _gen(n + kinds)
    cache = _cache(32, 16, 3, 64)
    slots = torch.randint(0, kinds, (n,), generator=gen, device=DEV) * (512 // 400 if kinds == 400 else 1)
    slots[::5] = -1
    k, v = _randn(n, 3, 64, gen=gen), _randn(n, 3, 64, gen=gen)
    _write(cache, k, v, slots)
    last = {}
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            last[s] = i
    if not last:
        return
    where, who = torch.tensor(list(last), device=DEV), torch.tensor(list(last.values()), device=DEV)
    got = cache64(cache, where)
    _same(got[0], quantise64(k[who]))
    _same(got[1], quantise64(v[who]))
    rest = torch.ones(512, dtype=torch.bool, device=DEV)
    rest[where] = False
    assert not any(x.any() for x in cache64(cache, rest.nonzero()[:, 0]))


def test_slots_outside_are_recorded():
    from revealaiccl_b200.ops.status import DeviceStatusError
    cache = _cache(2, 16, 1, 64)
    k = torch.ones(3, 1, 64, device=DEV)
    for bad in (32, 2 ** 31 - 1, 2 ** 40):
        slots = torch.tensor([4, bad, 5], device=DEV)
        with pytest.raises(DeviceStatusError, match="bounds"):
            _write(cache, k, k, slots)
        with pytest.raises(DeviceStatusError, match="bounds"):
            _read(cache, slots)
        got, _ = _read(cache, slots.clamp_max(31))
        _same(got[[0, 2]], quantise64(k[:2]))
        assert not got[1].any()


def test_read_same_slot_often():
    cache = _cache(1, 16, 2, 64)
    x = _randn(16, 2, 64, gen=_gen(5), dtype=BF16)
    _write(cache, x, x, torch.arange(16, device=DEV, dtype=torch.int32))
    slots = torch.tensor([3] * 40 + [-1, 15], device=DEV, dtype=torch.int32)
    k, v = _read(cache, slots)
    want = cache64(cache, slots)
    _same(k, want[0])
    _same(v, want[1])


def test_no_tokens():
    cache = _cache(1, 16, 2, 64)
    slots = torch.empty(0, dtype=torch.int64, device=DEV)
    k, v = _read(cache, slots)
    assert k.shape == v.shape == (0, 2, 64)
    _write(cache, k, v, slots)


def test_behind_32_bits():
    """A cache whose codes lie behind 2^32 bytes."""
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 30 GB")
    pages = (2 ** 32 + 2 ** 20) // (8 * 128 * 64)
    cache = _cache(pages, 128, 8, 128)
    n = 100
    slots = pages * 128 - 1 - torch.arange(n, device=DEV) * 3
    x = _randn(n, 8, 128, gen=_gen(6), dtype=BF16)
    _check(cache, x, x.flip(0).contiguous(), slots)
    low = torch.arange(0, 2 ** 20, 1009, device=DEV)
    assert not any(t.any() for t in _read(cache, low))


def test_captured_and_other_stream():
    """One graph, replayed with other inputs, on a stream of its own."""
    cache = _cache(4, 16, 2, 128)
    k, v = _randn(9, 2, 128, gen=_gen(7), dtype=BF16), _randn(9, 2, 128, gen=_gen(8), dtype=BF16)
    slots = torch.arange(9, device=DEV)
    from revealaiccl_b200.ops.kv_cache import kv_cache_read, kv_cache_write
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kv_cache_write(cache, k, v, slots)
        ko, vo = kv_cache_read(cache, slots)
    for i in range(3):
        k.copy_(_randn(9, 2, 128, gen=_gen(20 + i), dtype=BF16))
        slots.copy_(torch.randperm(64, generator=_gen(i), device=DEV)[:9])
        graph.replay()
        torch.cuda.synchronize()
        _same(ko, quantise64(k))
        _same(vo, quantise64(v))


def test_versions():
    cache = _cache(1, 16, 1, 64)
    before = [t._version for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    x = torch.ones(1, 1, 64, device=DEV)
    _write(cache, x, x, torch.zeros(1, dtype=torch.int64, device=DEV))
    assert all(t._version > b for t, b in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), before))
