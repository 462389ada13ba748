"""What the attention operators refuse: shapes, types and strides are checked before the device, so no GPU is needed."""

import pytest
import torch

from revealaiccl_b200.ops import _native

if not _native.has_kernels():  # pragma: no cover
    pytest.skip("kernel library not built", allow_module_level=True)

from revealaiccl_b200.ops.attention import attention_cached, attention_prompt
from revealaiccl_b200.ops.kv_cache import KVCache4, kv_cache_read, kv_cache_write

BF16, FP32, INT = torch.bfloat16, torch.float32, torch.int32


def _cache(pages=3, page=16, heads=2, dim=64, **kw):
    return KVCache4.empty(pages, page, heads, dim, device="cpu", **kw)


def _with(cache, **kw):
    return KVCache4(**{**{n: getattr(cache, n) for n in ("k_codes", "k_scales", "v_codes", "v_scales", "k_unit", "v_unit")}, **kw})


def _write(**kw):
    a = dict(cache=_cache(), k=torch.zeros(5, 2, 64, dtype=BF16), v=torch.zeros(5, 2, 64, dtype=BF16), slots=torch.zeros(5, dtype=INT))
    a.update(kw)
    return kv_cache_write(**a)


def _read(**kw):
    a = dict(cache=_cache(), slots=torch.zeros(5, dtype=INT))
    a.update(kw)
    return kv_cache_read(a.pop("cache"), a.pop("slots"), **a)


def _cached(**kw):
    a = dict(q=torch.zeros(4, 6, 64, dtype=BF16), cache=_cache(), block_table=torch.zeros(4, 3, dtype=INT), lengths=torch.zeros(4, dtype=INT))
    a.update(kw)
    return attention_cached(a.pop("q"), a.pop("cache"), a.pop("block_table"), a.pop("lengths"), **a)


def _prompt(**kw):
    a = dict(q=torch.zeros(9, 6, 64, dtype=BF16), k=torch.zeros(9, 2, 64, dtype=BF16), v=torch.zeros(9, 2, 64, dtype=BF16),
             cu_seqlens_q=torch.zeros(3, dtype=INT))
    a.update(kw)
    return attention_prompt(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("cu_seqlens_q"), a.pop("cu_seqlens_k", None), **a)


def _t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def _codes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


def test_empty_cache_refuses():
    with pytest.raises(ValueError, match="head_dim"):
        KVCache4.empty(1, 16, 1, 96, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        KVCache4.empty(1, 8, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        KVCache4.empty(1, 48, 1, 64, device="cpu")
    c = KVCache4.empty(3, 32, 5, 128, device="cpu")
    assert (c.pages, c.page_size, c.kv_heads, c.head_dim) == (3, 32, 5, 128)


CACHES = [
    (lambda: _with(_cache(), k_codes=_codes(3, 2, 16)), "codes must be"),
    (lambda: _with(_cache(), k_codes=_codes(3, 2, 16, 48)), "64 or 128 dimensions"),
    (lambda: _with(_cache(), v_codes=_codes(3, 2, 16, 64)), "v_codes must be a contiguous uint8"),
    (lambda: _with(_cache(), v_codes=torch.zeros(3, 2, 16, 32, dtype=torch.int8)), "v_codes must be a contiguous uint8"),
    (lambda: _with(_cache(), k_scales=_codes(3, 2, 16, 4)), "k_scales must be a contiguous float8"),
    (lambda: _with(_cache(), v_scales=_cache(dim=128).v_scales), "v_scales must be a contiguous float8"),
    (lambda: _with(_cache(), v_codes=_codes(3, 16, 2, 32).transpose(1, 2)), "v_codes must be a contiguous uint8"),
    (lambda: _with(_cache(), v_codes=_codes(3 * 2 * 16 * 32 + 8)[8:].view(3, 2, 16, 32)), "on 16 bytes"),
    (lambda: KVCache4(*[_codes(1, 1, 24, 32), _codes(1, 1, 24, 4).view(torch.float8_e4m3fn)] * 2), "page_size must be a power of two"),
    (lambda: KVCache4(*[_codes(1, 1, 8, 32), _codes(1, 1, 8, 4).view(torch.float8_e4m3fn)] * 2), "page_size must be a power of two"),
    (lambda: KVCache4(*[_codes(0, 1025, 16, 32), _codes(0, 1025, 16, 4).view(torch.float8_e4m3fn)] * 2), "1 to 1024 kv_heads"),
    (lambda: KVCache4(*[_codes(0, 512, 65536, 32), _codes(0, 512, 65536, 4).view(torch.float8_e4m3fn)] * 2), r"at most 2\^24"),
    (lambda: KVCache4(*[_codes(1).expand(2 ** 27, 1, 16, 32), _codes(1).expand(2 ** 27, 1, 16, 4).view(torch.float8_e4m3fn)] * 2), r"less than 2\^31"),
    (lambda: _with(_cache(), k_unit=3.0), "k_unit must be a power of two"),
    (lambda: _with(_cache(), v_unit=0.0), "v_unit must be a power of two"),
    (lambda: _with(_cache(), v_unit=-2.0), "v_unit must be a power of two"),
    (lambda: _with(_cache(), v_unit=2.0 ** 64), "v_unit must be a power of two"),
    (lambda: _with(_cache(), v_unit=float("inf")), "v_unit must be a power of two"),
]


@pytest.mark.parametrize("call", [_write, _read, _cached], ids=["write", "read", "cached"])
@pytest.mark.parametrize("make,words", CACHES)
def test_caches_are_refused(make, words, call):
    with pytest.raises(ValueError, match=words):
        call(cache=make())


def test_units():
    with pytest.raises(ValueError, match="CUDA device"):
        _write(cache=_cache(k_unit=2.0 ** -60, v_unit=2.0 ** 60))


@pytest.mark.parametrize("kw,words", [
    (dict(), "CUDA device"),
    (dict(k=_t(5, 128)), r"k must be \[tokens"),
    (dict(k=_t(64, 2, 5).transpose(0, 2)), "contiguous rows"),
    (dict(k=_t(5, 3, 64), v=_t(5, 3, 64)), "by the slots and the cache"),
    (dict(k=_t(6, 2, 64), v=_t(6, 2, 64)), "by the slots and the cache"),
    (dict(v=_t(5, 2, 128)), "by the slots and the cache"),
    (dict(v=_t(5, 2, 64, dtype=FP32)), "both be bf16 or both be fp32"),
    (dict(k=_t(5, 2, 64).half(), v=_t(5, 2, 64).half()), "both be bf16 or both be fp32"),
    (dict(slots=torch.zeros(5, dtype=torch.int16)), "slots must be"),
    (dict(slots=torch.zeros(5, 1, dtype=INT)), "slots must be"),
    (dict(slots=torch.zeros(10, dtype=INT)[::2]), "slots must be"),
    (dict(slots=torch.zeros(5, dtype=INT, device="meta")), "slots must be on cpu"),
])
def test_write_refuses(kw, words):
    with pytest.raises(ValueError, match=words):
        _write(**kw)


@pytest.mark.parametrize("kw,words", [
    (dict(), "CUDA device"),
    (dict(slots=torch.zeros(5)), "slots must be"),
    (dict(dtype=torch.float16), "bf16 or fp32"),
    (dict(k_out=_t(5, 2, 64)), "given together"),
    (dict(k_out=_t(5, 2, 64), v_out=_t(4, 2, 64)), "v_out must have shape"),
    (dict(k_out=_t(5, 2, 64), v_out=_t(5, 2, 64, dtype=FP32)), "v_out must have shape"),
    (dict(k_out=_t(5, 2, 64), v_out=_t(5, 2, 64), dtype=FP32), "k_out must have shape"),
    (dict(k_out=_t(5, 1, 64).expand(5, 2, 64), v_out=_t(5, 2, 64)), "elements of k_out share"),
])
def test_read_refuses(kw, words):
    with pytest.raises(ValueError, match=words):
        _read(**kw)


@pytest.mark.parametrize("kw,words", [
    (dict(), "CUDA device"),
    (dict(q=_t(4, 384)), r"q must be \[tokens"),
    (dict(q=_t(4, 6, 128)), "128 dimensions to a head"),
    (dict(q=_t(4, 5, 64)), "1 to 128 heads for each"),
    (dict(q=_t(4, 0, 64)), "1 to 128 heads for each"),
    (dict(q=_t(4, 258, 64)), "1 to 128 heads for each"),
    (dict(q=_t(4, 6, 64).half()), "bf16 or fp32"),
    (dict(block_table=_t(3, 3, dtype=INT)), "block_table must be"),
    (dict(block_table=_t(4, 3, dtype=torch.int64)), "block_table must be"),
    (dict(block_table=_t(3, 4, dtype=INT).t()), "block_table must be"),
    (dict(block_table=_t(1, dtype=INT).expand(4, 2 ** 27)), "contiguous rows|room for"),
    (dict(lengths=_t(3, dtype=INT)), "lengths must be"),
    (dict(lengths=_t(4, dtype=torch.int64)), "lengths must be"),
    (dict(lengths=_t(8, dtype=INT)[::2]), "lengths must be"),
    (dict(scale=float("nan")), "scale must be"),
    (dict(scale=1e300), "scale must be"),
    (dict(out=_t(4, 6, 128)), "out must have"),
    (dict(out=_t(4, 6, 64, dtype=FP32), out_dtype=BF16), "out must have"),
    (dict(out_dtype=torch.float16), "the output is fp32"),
    (dict(q=_t(4, 6, 64, dtype=FP32), out_dtype=BF16), "the output is fp32"),
    (dict(out=_t(4, 1, 64).expand(4, 6, 64)), "elements of out share"),
])
def test_cached_refuses(kw, words):
    with pytest.raises(ValueError, match=words):
        _cached(**kw)


@pytest.mark.parametrize("kw,words", [
    (dict(), "CUDA device"),
    (dict(q=_t(9, 384)), r"q must be \[tokens"),
    (dict(q=_t(9, 6, 96), k=_t(9, 2, 96), v=_t(9, 2, 96)), "64 or 128 dimensions"),
    (dict(k=_t(9, 2, 128)), "k and v must be"),
    (dict(v=_t(8, 2, 64)), "k and v must be"),
    (dict(q=_t(9, 5, 64)), "1 to 128 heads for each"),
    (dict(q=_t(9, 258, 64)), "1 to 128 heads for each"),
    (dict(k=_t(9, 0, 64), v=_t(9, 0, 64)), "1 to 128 heads for each"),
    (dict(q=_t(9, 6, 64, dtype=FP32)), "all be bf16 or all be fp32"),
    (dict(q=_t(9, 6, 64).half(), k=_t(9, 2, 64).half(), v=_t(9, 2, 64).half()), "all be bf16 or all be fp32"),
    (dict(k=_t(9, 64, 2).transpose(1, 2)), "contiguous rows"),
    (dict(q=_t(1, 65536, 64), k=_t(9, 1024, 64), v=_t(9, 1024, 64)), "less than 65536 in all"),
    (dict(cu_seqlens_q=_t(2 ** 16 + 2, dtype=INT)), r"at most 2\^16 sequences"),
    (dict(cu_seqlens_q=_t(0, dtype=INT)), "one entry more"),
    (dict(cu_seqlens_q=_t(3, dtype=torch.int64)), "cu_seqlens_q must be"),
    (dict(cu_seqlens_k=_t(2, dtype=INT)), "cu_seqlens_k must be"),
    (dict(scale=float("inf")), "scale must be"),
    (dict(out=_t(9, 6, 64, dtype=FP32)), "out must have"),
    (dict(out=_t(9, 5, 64)), "out must have"),
    (dict(out=_t(9, 1, 64).expand(9, 6, 64)), "elements of out share"),
])
def test_prompt_refuses(kw, words):
    with pytest.raises(ValueError, match=words):
        _prompt(**kw)


def test_shared_memory_is_refused():
    q = _t(9, 6, 64)
    with pytest.raises(ValueError, match="out shares memory with another"):
        _prompt(q=q, out=q)
    buf = _t(9, 10, 64)
    with pytest.raises(ValueError, match="out shares memory with another"):
        _prompt(q=buf[:, :6], k=buf[:, 6:8], v=buf[:, 8:], out=buf[:, 2:8])
    q = _t(4, 6, 64)
    with pytest.raises(ValueError, match="out shares memory with another"):
        _cached(q=q, out=q)
    kv = _t(5, 2, 64)
    with pytest.raises(ValueError, match="v_out shares memory with another"):
        _read(k_out=kv, v_out=kv)
    c = _cache()
    with pytest.raises(ValueError, match="the cache shares memory with another"):
        _write(cache=_with(c, v_codes=c.k_codes))
    with pytest.raises(ValueError, match="the cache shares memory with another"):
        _write(cache=c, k=c.k_codes.view(BF16).view(-1)[:640].view(5, 2, 64))
    with pytest.raises(ValueError, match="CUDA device"):   # keys and values may be the same, and lie apart or in one another
        _write(k=kv, v=kv)


def test_gradients_and_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    for call, name, shape in ((_prompt, "q", (9, 6, 64)), (_prompt, "v", (9, 2, 64)), (_cached, "q", (4, 6, 64)), (_write, "k", (5, 2, 64))):
        x = torch.zeros(*shape, dtype=BF16, requires_grad=True)
        with pytest.raises(RuntimeError, match="no backward"):
            call(**{name: x})
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call(**{name: x})
        with fwd.dual_level(), pytest.raises(RuntimeError, match="no derivative"):
            call(**{name: fwd.make_dual(torch.zeros(*shape, dtype=BF16), torch.ones(*shape, dtype=BF16))})


def test_freed_storages_are_refused():
    def freed(t):
        t = t.clone()
        t.untyped_storage().resize_(0)
        return t

    for call, name, t in ((_prompt, "k", _t(9, 2, 64)), (_prompt, "cu_seqlens_q", _t(3, dtype=INT)), (_prompt, "out", _t(9, 6, 64)),
                          (_cached, "q", _t(4, 6, 64)), (_cached, "block_table", _t(4, 3, dtype=INT)), (_cached, "lengths", _t(4, dtype=INT)),
                          (_write, "v", _t(5, 2, 64)), (_write, "slots", _t(5, dtype=INT)), (_read, "slots", _t(5, dtype=INT))):
        with pytest.raises(ValueError, match=f"{name} reaches behind its storage"):
            call(**{name: freed(t)})
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        with pytest.raises(ValueError, match=f"{name} reaches behind its storage"):
            _cached(cache=_with(_cache(), **{name: freed(getattr(_cache(), name))}))


def test_plans():
    """Which calls share a tile's keys between CTAs, and which tensors are copied to aligned rows first."""
    plan = _native.kernels().attention_prompt_plan
    q, k = _t(1, 8, 128), _t(20000, 2, 128)
    assert plan(q, k, k, 1, 148)["splits"] == 32
    assert plan(q, k[:1023], k[:1023], 1, 148)["splits"] == 1
    assert plan(q, k[:1024], k[:1024], 1, 148)["splits"] == 2
    assert plan(_t(20000, 8, 128), k, k, 1, 148)["splits"] == 1
    wide = _t(30, 2, 72)
    assert not any(plan(wide[..., :64], wide[..., 8:], wide[..., :64], 1, 148)[f"pack_{x}"] for x in "qkv")
    got = plan(wide[..., 1:65], wide[..., :64], wide[:, :1, :64].expand(30, 2, 64), 1, 148)
    assert got["pack_q"] and not got["pack_k"] and got["pack_v"]
    assert not any(plan(wide[..., 1:65].float(), wide.float()[..., :64], wide.float()[..., :64], 1, 148)[f"pack_{x}"] for x in "qkv")
