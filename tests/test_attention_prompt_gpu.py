"""attention_prompt against the formula in 64 bits."""

import pytest
import torch

from attention_reference import attention64, norm_bound
from serving_reference import check_close, check_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")
WEIGHT = {BF16: 2.0 ** -7, FP32: 2.0 ** -20}   # two roundings of a weight: bf16, or two parts


def _attend(*a, **kw):
    from revealaiccl_b200.ops.attention import attention_prompt
    return attention_prompt(*a, **kw)


def _gen(seed=0):
    return torch.Generator(DEV).manual_seed(seed)


def _rows(n, heads, dim, dtype, seed, pad=0, scale=1.0):
    t = (torch.randn(n, heads * dim + pad, generator=_gen(seed), device=DEV) * scale).to(dtype)
    return t[:, :heads * dim].unflatten(1, (heads, dim))


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().to(DEV)


def _make(q_lens, k_lens, hk, group, dim, dtype, seed=0, pad=0):
    return (_rows(sum(q_lens), hk * group, dim, dtype, seed, pad), _rows(sum(k_lens), hk, dim, dtype, seed + 1, pad),
            _rows(sum(k_lens), hk, dim, dtype, seed + 2, pad))


def _want(q, k, v, q_lens, k_lens, causal, scale=None):
    outs, a, b = [], 0, 0
    for n, m in zip(q_lens, k_lens):
        see = torch.arange(n, device=DEV) + (m - n + 1) if causal else torch.full((n,), m, device=DEV)
        outs.append(attention64(q[a:a + n], k[b:b + m], v[b:b + m], see.clamp_min(0), scale, WEIGHT[q.dtype]))
        a, b = a + n, b + m
    return [torch.cat(x) for x in zip(*outs)]


def _check(q, k, v, q_lens, k_lens, causal=True, scale=None, **kw):
    out, lse = _attend(q, k, v, _cu(q_lens), _cu(k_lens), causal=causal, scale=scale, return_lse=True, check=True, **kw)
    want, wlse, bound, lbound, largest = _want(q, k, v, q_lens, k_lens, causal, scale)
    n = sum(q_lens)
    check_close(out[:n], want, bound)
    empty = wlse == -INF
    assert torch.equal(lse[:n].double() == -INF, empty)
    check_close(torch.where(empty, 0, lse[:n].double()), torch.where(empty, 0, wlse), lbound)
    if want.abs().sum() > 0 and want.isfinite().all():
        check_norm(out[:n], want, norm_bound(out.dtype, True, largest))
    return out, lse


DTYPES = pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("hk,group", [(1, 1), (2, 4), (1, 7), (3, 2), (1, 16)])
@pytest.mark.parametrize("lens", [[1], [5, 0, 128, 1, 129], [300], [31, 32, 33, 63, 64, 65, 127]])
def test_packed(lens, hk, group, causal, dim, dtype):
    q, k, v = _make(lens, lens, hk, group, dim, dtype, seed=sum(lens) + group, pad=16)
    _check(q, k, v, lens, lens, causal)


@DTYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens", [([1], [1000]), ([3, 200, 7], [3, 777, 0]), ([100, 50], [20, 51]), ([257], [1025]),
                                           ([64, 1, 1], [192, 128, 129])])
def test_behind_earlier_tokens(q_lens, k_lens, causal, dim, dtype):
    """Chunks behind earlier tokens; more queries than keys, so that the first see nothing; sequences without keys."""
    q, k, v = _make(q_lens, k_lens, 2, 3, dim, dtype, seed=7)
    _check(q, k, v, q_lens, k_lens, causal)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hk,group,lens", [(2, 4, [2500]), (1, 1, [3000, 1100]), (4, 5, [900, 1800]), (1, 128, [70])])
def test_longer(hk, group, lens, dim):
    q, k, v = _make(lens, lens, hk, group, dim, BF16, seed=11)
    _check(q, k, v, lens, lens)
    if sum(lens) < 3000:
        q, k, v = _make(lens, lens, hk, group, dim, FP32, seed=12)
        _check(q, k, v, lens, lens)


def _plan(q, k, v, seqs):
    from revealaiccl_b200.ops._native import kernels
    return kernels().attention_prompt_plan(q, k, v, seqs, torch.cuda.get_device_properties(DEV).multi_processor_count)


@DTYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("hk,group,dim,q_lens,k_lens", [
    (1, 1, 64, [1], [9001]), (2, 4, 128, [3, 40], [5000, 4100]), (1, 8, 128, [130, 0, 2], [4000, 700, 0]), (2, 3, 64, [7, 5], [3, 8000]),
])
def test_keys_shared_by_ctas(hk, group, dim, q_lens, k_lens, causal, dtype):
    """Few queries of many keys: several CTAs to a tile.  What no token sees stays outside, and rows around are left alone."""
    q, k, v = _make(q_lens, k_lens, hk, group, dim, dtype, seed=27)
    assert _plan(q, k, v, len(q_lens))["splits"] > 1
    out, lse = _check(q, k, v, q_lens, k_lens, causal)
    n = sum(q_lens)
    big, wide = torch.zeros(n + 9, hk * group, dim, dtype=dtype, device=DEV), torch.full((n + 9, hk * group + 1, dim), 7.0, dtype=dtype, device=DEV)
    big[4:4 + n] = q
    k2, v2 = (torch.cat([x, torch.full_like(x[:50], NAN)]) for x in (k, v))
    got, glse = _attend(big, k2, v2, _cu(q_lens) + 4, _cu(k_lens), causal=causal, out=wide[:, 1:], return_lse=True, check=True)
    assert torch.equal(got[4:4 + n], out) and torch.equal(glse[4:4 + n], lse)
    got[4:4 + n] = 7.0
    assert (wide == 7.0).all()
    v2[k_lens[0] - 1, 0, 3] = INF                   # the last key of the first sequence
    if q_lens[0] <= k_lens[0]:
        got = _attend(q, k2, v2, _cu(q_lens), _cu(k_lens), causal=causal, check=True)
        last = q_lens[0] - 1 if causal else 0
        assert (got[last:q_lens[0], :group, 3] == INF).all()
        got[last:q_lens[0], :group, 3] = out[last:q_lens[0], :group, 3]
        assert torch.equal(got, out)


@DTYPES
@pytest.mark.parametrize("seqs", [33, 400, 2100])
def test_many_sequences(seqs, dtype):
    lens = [(5 * i) % 23 for i in range(seqs)]
    lens[seqs // 2] = 300                        # of many tiles, between others
    q, k, v = _make(lens, lens, 2, 2, 64, dtype, seed=13)
    _check(q, k, v, lens, lens)


@DTYPES
def test_scales_and_sizes(dtype):
    lens = [150, 90]
    q, k, v = _make(lens, lens, 2, 2, 64, dtype, seed=15)
    for scale in (0.0, 1.0, -0.3):
        _check(q, k, v, lens, lens, scale=scale)
    _check((q.float() * 1e10).to(dtype), (k.float() * 1e-8).to(dtype), v, lens, lens, scale=1e-3)
    _check(q, k, (v.float() * 1e20).to(dtype), lens, lens)
    # logits that grow along the keys, and that fall
    for order in (1, -1):
        ramp = k.clone()
        ramp[:, :, 0] = (torch.arange(len(k), device=DEV) * (0.5 * order)).to(dtype)[:, None]
        one = q.clone()
        one[:, :, 0] = 1.0
        _check(one, ramp, v, lens, lens, scale=1.0)


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_what_is_not_seen_does_not_enter(causal, dim, dtype):
    """NaN and infinities in keys and values of later tokens, of neighbours in the packing and behind the last sequence."""
    q_lens, k_lens = [100, 200, 30], [100, 260, 30]
    q, k, v = _make(q_lens, [100, 260, 130], 2, 2, dim, dtype, seed=17)
    base, base_lse = _check(q, k, v, q_lens, k_lens, causal)
    k2, v2 = k.clone(), v.clone()
    k2[390:], v2[390:] = NAN, INF              # behind the last sequence
    k2[100 + 250, 0], v2[100 + 250, 0] = NAN, NAN   # a late token of the second
    v2[100 + 255, 1, 5], v2[100 + 256, 1, 5], v2[100 + 254, 1, 6] = INF, -INF, INF
    out, lse = _attend(q, k2, v2, _cu(q_lens), _cu(k_lens), causal=causal, return_lse=True, check=True)
    other = torch.ones(330, dtype=torch.bool, device=DEV)
    other[100:300] = False
    assert torch.equal(out[other], base[other]) and torch.equal(lse[other], base_lse[other])
    want, wlse, bound, *_ = _want(q, k2, v2, q_lens, k_lens, causal)
    if causal:
        first = 100 + 250 - 60                 # the rows that see token 250 of the keys
        assert torch.equal(out[100:first, :2], base[100:first, :2]) and out[first:300, :2].isnan().all()
        assert torch.equal(lse[100:first], base_lse[100:first])
    else:
        assert out[100:300, :2].isnan().all()
    check_close(out[:330, 2:], want[:, 2:], bound[:, 2:])


@DTYPES
def test_infinite_and_nan_queries(dtype):
    lens = [140, 20]
    q, k, v = _make(lens, lens, 1, 2, 64, dtype, seed=19)
    base = _attend(q, k, v, _cu(lens))
    q2 = q.clone()
    q2[3, 1, 5], q2[130, 0, 0] = NAN, NAN
    out = _attend(q2, k, v, _cu(lens), check=True)
    assert out[3, 1].isnan().all() and out[130, 0].isnan().all()
    out[3, 1], out[130, 0] = base[3, 1], base[130, 0]
    assert torch.equal(out, base)


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
def test_strides_and_out(dim, dtype):
    lens = [90, 45]
    q, k, v = _make(lens, lens, 2, 3, dim, dtype, seed=21)
    base = _attend(q, k, v, _cu(lens))

    def window(t, off):
        wide = torch.full((len(t) + 1, t.shape[1], t.shape[2] + off + 5), NAN, dtype=dtype, device=DEV)
        wide[:len(t), :, off:off + t.shape[2]] = t
        return wide[:len(t), :, off:off + t.shape[2]]

    def heads_first(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    fused = torch.cat([q, k, v], 1)
    split = fused[:, :6], fused[:, 6:8], fused[:, 8:]
    for a, b, c in ((window(q, 1), window(k, 3), window(v, 0)), (heads_first(q), heads_first(k), heads_first(v)), split,
                    (q, window(k, 1), v), (window(q, 8), k, heads_first(v))):
        assert torch.equal(_attend(a, b, c, _cu(lens), check=True), base)
    one = k[:, :1].expand(-1, 2, -1)           # one key head, expanded
    assert torch.equal(_attend(q, one, one, _cu(lens)), _attend(q, one.contiguous(), one.contiguous(), _cu(lens)))
    for off in (0, 1, 8):
        wide = torch.full((150, 7, dim + 16), 7.0, dtype=dtype, device=DEV)
        out = wide[:135, :6, off:off + dim]
        version = out._version
        assert _attend(q, k, v, _cu(lens), out=out).data_ptr() == out.data_ptr() and out._version > version
        assert torch.equal(out, base)
        out.fill_(7.0)
        assert (wide == 7.0).all()
    # rows behind the last sequence, and before the first, stay as they were
    out = torch.full((200, 6, dim), 7.0, dtype=dtype, device=DEV)
    big = torch.zeros(200, 6, dim, dtype=dtype, device=DEV)
    big[10:145] = q
    got = _attend(big, k, v, _cu(lens) + torch.tensor(10, device=DEV, dtype=torch.int32), _cu(lens), out=out, check=True)
    assert torch.equal(got[10:145], base) and (got[:10] == 7.0).all() and (got[145:] == 7.0).all()


def test_offsets_outside_are_recorded():
    from revealaiccl_b200.ops.status import DeviceStatusError
    q, k, v = _make([40], [40], 1, 2, 64, BF16)
    for cu in ([0, 41], [-1, 40], [0, 30, 20], [0, 2 ** 31 - 1], [50, 60]):
        c = torch.tensor(cu, dtype=torch.int32, device=DEV)
        with pytest.raises(DeviceStatusError, match="bounds"):
            _attend(q, k, v, c, check=True)
        with pytest.raises(DeviceStatusError, match="bounds"):
            _attend(q, k, v, torch.tensor([0] * (len(cu) - 1) + [40], dtype=torch.int32, device=DEV), c, check=True)
    _check(q, k, v, [40], [40])


def test_nothing_to_do():
    q, k, v = _make([0], [0], 1, 2, 64, BF16)
    assert _attend(q, k, v, _cu([0])).shape == (0, 2, 64)
    q, k, v = _make([5], [0], 1, 2, 64, BF16)
    out, lse = _attend(q, k, v, _cu([5]), _cu([0]), return_lse=True, check=True)
    assert not out.any() and (lse == -INF).all()


def test_sums_go_in_a_fixed_order():
    lens = [700, 90]
    q, k, v = _make(lens, lens, 2, 4, 128, BF16, seed=23)
    base = _attend(q, k, v, _cu(lens))
    for _ in range(5):
        assert torch.equal(_attend(q, k, v, _cu(lens)), base)


@DTYPES
def test_captured(dtype):
    """A graph replayed with other offsets and inputs, next to another one of the same call."""
    states = []
    for i in range(2):
        side = torch.cuda.Stream()
        q, k, v = _make([300], [500], 2, 2, 64, dtype, seed=30 + i)
        cq, ck = _cu([0, 0, 0]), _cu([0, 0, 0])
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = _attend(q, k, v, cq, ck)
        states.append((side, q, k, v, cq, ck, graph, out))
    torch.cuda.synchronize()
    for q_lens, k_lens in (([100, 100, 100], [100, 300, 100]), ([1, 0, 299], [5, 7, 480]), ([0, 0, 1], [0, 0, 500])):
        for side, q, k, v, cq, ck, graph, out in states:
            cq.copy_(_cu(q_lens))
            ck.copy_(_cu(k_lens))
            v.mul_(1.5)
        torch.cuda.synchronize()
        for side, *_, graph, _ in states:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for side, q, k, v, cq, ck, graph, out in states:
            want, _, bound, *_ = _want(q, k, v, q_lens, k_lens, True)
            check_close(out[:sum(q_lens)], want, bound)


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("times", [4, 5], ids=["by_length", "in_order"])
def test_tiles_one_after_another(times, dim, dtype):
    """More tiles than SMs, of sequences long, short, empty and without keys: what one leaves behind does not reach the next."""
    q_lens, k_lens = [300, 17, 0, 260, 130, 1, 520] * times, [300, 17, 40, 261, 0, 700, 520] * times
    hk = 10
    q, k, v = _make(q_lens, k_lens, hk, 1, dim, dtype, seed=33)
    base, base_lse = _check(q, k, v, q_lens, k_lens)
    v2 = v.clone()
    rows, ends = [], _cu(k_lens).tolist()[1:]
    for i, (end, row) in enumerate(zip(ends, _cu(q_lens).tolist()[1:])):
        if i % 2 and k_lens[i] and q_lens[i]:       # the last key, which the last row alone sees
            v2[end - 1, :, i % dim] = (NAN, INF, -INF)[i % 3]
            rows.append((row - 1, i % dim, (NAN, INF, -INF)[i % 3]))
    out, lse = _attend(q, k, v2, _cu(q_lens), _cu(k_lens), return_lse=True, check=True)
    want = base.clone()
    for row, d, x in rows:
        want[row, :, d] = x
    assert len(rows) > 2 * times and torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0)) and torch.equal(lse, base_lse)
