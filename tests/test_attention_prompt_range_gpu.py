"""attention_prompt where logits grow along the keys, and where values are as large or as small as their type has them."""

import math

import pytest
import torch

from attention_reference import attention64
from serving_reference import check_close
from test_attention_prompt_gpu import BF16, DEV, DTYPES, FP32, NAN, WEIGHT, _attend, _check, _cu, _make, _plan, _want

pytestmark = pytest.mark.gpu
MOST = {BF16: torch.finfo(BF16).max, FP32: 3e38}


def _steered(q_lens, logits, hk, group, dim, dtype, seed=0):
    """q and k whose products are `logits` (one to a key), but for a row's factor 1, 0 or -1 and small random numbers."""
    q, k, v = _make(q_lens, [len(logits)], hk, group, dim, dtype, seed)
    q, k = q * 0.1, k * 0.1
    row = torch.arange(q.shape[0] * q.shape[1], device=DEV).view(q.shape[:2])
    q[:, :, 0] = (1 - row % 3).to(dtype)
    k[:, :, 0] = torch.as_tensor(logits, device=DEV, dtype=torch.float32).to(dtype)[:, None]
    return q, k, v


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("order", [1, -1], ids=["up", "down"])
@pytest.mark.parametrize("size", [1.0, 1e30])
def test_logits_that_grow_past_every_step(size, order, causal, dim, dtype):
    """By a nat with every key, 185 powers of two with every 128, in rows next to some whose logits stay or fall."""
    logits = [order * float(i) for i in range(900)]
    q, k, v = _steered([290], logits, 2, 2, dim, dtype, seed=40)
    v = (v.float() * size).to(dtype)
    assert _plan(q, k, v, 1)["splits"] == 1
    _check(q, k, v, [290], [900], causal, scale=1.0)


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("step", [0.05, 0.3, 1.0])
@pytest.mark.parametrize("size", [1.0, 1e30])
def test_logits_that_grow_in_shared_keys(size, step, dim, dtype):
    logits = [step * i for i in range(3000)]
    q, k, v = _steered([5], logits, 2, 3, dim, dtype, seed=42)
    v = (v.float() * size).to(dtype)
    assert _plan(q, k, v, 1)["splits"] > 1
    _check(q, k, v, [5], [3000], scale=1.0)


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rise", [5.5, 7.5, 31.0, 60.0, 127.0])
@pytest.mark.parametrize("value", [1e20, 1e22, 1e37, "most", "least"])
def test_large_values_behind_a_rise(value, rise, dim, dtype):
    """128 keys at 0, then 1000 that are `rise` powers of two above them: one value everywhere is the answer too."""
    value = {"most": MOST[dtype], "least": -MOST[dtype]}.get(value, value)
    v = torch.full((1128, 2, dim), value, device=DEV).to(dtype)
    value = float(v[0, 0, 0])
    q, k = torch.zeros(140, 4, dim, dtype=dtype, device=DEV), torch.zeros_like(v)
    q[:, :, 0], k[128:, :, 0] = 1.0, rise
    for causal in (False, True):
        out = _attend(q, k, v, _cu([140]), _cu([1128]), causal=causal, scale=math.log(2.0), check=True)
        check_close(out, torch.full_like(out, value).double(), torch.full_like(out, abs(value) * 2.0 ** (-7 if dtype == BF16 else -20)).double())


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
def test_largest_values_of_shared_keys(dim, dtype):
    """As many keys as it takes for several CTAs, all alike: their sums are thousands of the largest number."""
    v = torch.full((20000, 2, dim), MOST[dtype], dtype=dtype, device=DEV)
    v[:, 1] = -MOST[dtype]
    q, k = torch.ones(2, 2, dim, dtype=dtype, device=DEV), torch.zeros_like(v)
    assert _plan(q, k, v, 1)["splits"] > 1
    out, lse = _attend(q, k, v, _cu([2]), _cu([20000]), causal=False, return_lse=True, check=True)
    want = v[:1].double().expand_as(out)
    check_close(out, want, want.abs() * 2.0 ** (-7 if dtype == BF16 else -20))
    assert (lse - math.log(20000)).abs().max() < 1e-5   # of 9.9, whose last place is 2^-20, and 20000 additions' share


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
def test_many_equal_weights_of_one_cta(dim, dtype):
    """20000 keys that no other CTA shares: their sum has to be brought down on the way."""
    heads = 75
    q, k, v = _make([1], [20000], heads, 1, dim, dtype, seed=44)
    k = torch.zeros_like(k)
    v[:, 0], v[:, 1] = MOST[dtype], -MOST[dtype]
    assert _plan(q, k, v, 1)["splits"] == 1
    out, lse = _attend(q, k, v, _cu([1]), _cu([20000]), return_lse=True, check=True)
    want = v.double().mean(0)[None]
    assert out.isfinite().all()
    # weights are powers of two; the additions of 20000 numbers, in 160 sums of a step's
    assert ((out.double() - want).abs() <= 2.0 ** (-8 if dtype == BF16 else -20) * want.abs() + 20000 * 2.0 ** -24 * v.double().abs().mean(0)).all()
    assert (lse - math.log(20000)).abs().max() < 1e-5


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys,splits", [(1128, 1), (3000, 2)])
def test_rounded_weights_do_not_lift_the_largest_values(keys, splits, dim):
    """Weights of 1.0041 are rounded to 1.0078, all alike: a mean of bf16's largest number stays that number."""
    heads = 75 if splits == 1 else 2
    v = torch.full((keys, heads, dim), MOST[BF16], dtype=BF16, device=DEV)
    q, k = torch.zeros(1, heads, dim, dtype=BF16, device=DEV), torch.zeros_like(v)
    q[:, :, 0], k[128:, :, 0] = 1.0, 0.0041
    assert (_plan(q, k, v, 1)["splits"] > 1) == (splits > 1)
    out = _attend(q, k, v, _cu([1]), _cu([keys]), scale=1.0, check=True)
    assert (out == MOST[BF16]).all()


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("k_len", [300, 3000])
def test_small_values(k_len, dim, dtype):
    """Values of 2^-100 lose nothing that values of 1 keep."""
    q, k, v = _make([7], [k_len], 2, 2, dim, dtype, seed=46)
    out = _attend(q, k, v * 2.0 ** -100, _cu([7]), _cu([k_len]), check=True)
    want, _, bound, *_ = _want(q, k, v, [7], [k_len], True)
    check_close(out * 2.0 ** 100, want, bound)


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_and_infinities_behind_a_rise(dim, dtype):
    """What is not finite still reaches the rows that see it, and no others."""
    logits = [float(i) for i in range(600)]
    q, k, v = _steered([300], logits, 1, 2, dim, dtype, seed=48)
    base = _attend(q, k, v, _cu([300]), _cu([600]), scale=1.0, check=True)
    v2 = v.clone()
    v2[550, 0, 3], v2[560, 0, 7], v2[570, 0, 8] = NAN, math.inf, -math.inf
    out = _attend(q, k, v2, _cu([300]), _cu([600]), scale=1.0, check=True)
    want = base.clone()
    want[250:, :, 3], want[260:, :, 7], want[270:, :, 8] = NAN, math.inf, -math.inf
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("below", [1.0, 80.0, 200.0])
def test_nan_and_infinities_of_a_part_that_hardly_counts(below, dim, dtype):
    """Keys that several CTAs share, most of them `below` under the last ones: what they see is not lost in the joining."""
    logits = [0.0] * 2500 + [below] * 500
    q, k, v = _steered([5], logits, 2, 3, dim, dtype, seed=50)
    q[:, :, 0] = 1.0
    assert _plan(q, k, v, 1)["splits"] > 1
    base = _attend(q, k, v, _cu([5]), _cu([3000]), scale=1.0, check=True)
    v2 = v.clone()
    v2[10, 0, 3] = NAN
    v2[2400, 1, 5] = NAN
    v2[2998, 0, 9] = NAN                    # which rows 3 and 4 see
    out = _attend(q, k, v2, _cu([5]), _cu([3000]), scale=1.0, check=True)
    want = base.clone()
    want[:, :3, 3], want[:, 3:, 5], want[3:, :3, 9] = NAN, NAN, NAN
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    v2 = v.clone()
    v2[10, 0, 3], v2[2400, 1, 5] = math.inf, -math.inf
    out = _attend(q, k, v2, _cu([5]), _cu([3000]), scale=1.0, check=True)
    assert not out[:, :3, 3].isfinite().any() and not out[:, 3:, 5].isfinite().any()
    out[:, :3, 3], out[:, 3:, 5] = base[:, :3, 3], base[:, 3:, 5]
    assert torch.equal(out, base)


@DTYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("q_len,k_len", [(5, 3000), (290, 900)], ids=["shared", "one_cta"])
def test_keys_whose_logits_are_all_minus_infinity(q_len, k_len, causal, dim, dtype):
    """Keys shut out by a number that makes their logit -inf (in fp32 by overflow): whole tiles and whole CTAs' shares of them."""
    for shut in (slice(0, 2 * k_len // 3), slice(k_len // 3, k_len), slice(128, k_len - 1)):
        q, k, v = _make([q_len], [k_len], 2, 3, dim, dtype, seed=52)
        assert (_plan(q, k, v, 1)["splits"] > 1) == (q_len == 5)
        q[:, :, 0], k[:, :, 0] = 10.0, 0.0
        k[shut, :, 0] = -math.inf if dtype == BF16 else -3e38
        out, lse = _attend(q, k, v, _cu([q_len]), _cu([k_len]), causal=causal, return_lse=True, check=True)
        keep = torch.ones(k_len, dtype=torch.bool, device=DEV)
        keep[shut] = False
        see = torch.arange(q_len, device=DEV) + (k_len - q_len + 1) if causal else torch.full((q_len,), k_len, device=DEV)
        want, wlse, bound, lbound, _ = attention64(q, k[keep], v[keep], keep.cumsum(0)[see - 1], None, WEIGHT[dtype])
        check_close(out, want, bound)
        check_close(lse, wlse, lbound)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len,k_len", [(5, 3000), (290, 900)], ids=["shared", "one_cta"])
def test_no_key_but_at_minus_infinity(q_len, k_len, dim):
    q, k, v = _make([q_len], [k_len], 2, 3, dim, BF16, seed=54)
    q[:, :, 0], k[:, 0, 0] = 1.0, -math.inf
    out, lse = _attend(q, k, v, _cu([q_len]), _cu([k_len]), return_lse=True, check=True)
    assert out[:, :3].isnan().all() and (lse[:, :3] == -math.inf).all()
    want, wlse, bound, lbound, _ = _want(q[:, 3:], k[:, 1:], v[:, 1:], [q_len], [k_len], True)
    check_close(out[:, 3:], want, bound)
    check_close(lse[:, 3:], wlse, lbound)


def test_more_keys_than_two_seconds_of_steps():
    """One token behind 4 * 10^8 keys, all of one CTA's (80 tiles for all that the plan can tell): warps without work wait that long."""
    n, dim = 400_000_000, 64
    if torch.cuda.mem_get_info()[0] < 70e9:
        pytest.skip("needs 51 GB of device memory")
    x = torch.zeros(n + 1, 1, dim, dtype=BF16, device=DEV)
    x[:128] = 1.0
    x[-1, 0, 3] = math.inf                             # of the last key's value, which no key has
    q = torch.ones(1, 1, dim, dtype=BF16, device=DEV)
    cu_q, cu_k = _cu([1] + [0] * 79), _cu([n] + [0] * 79)
    assert _plan(q, x[:-1], x[1:], 80)["splits"] == 1
    out = _attend(q, x[:-1], x[1:], cu_q, cu_k, scale=0.5, check=True)
    # the first 128 keys lie 32 nats above the others, which all together are 4e8 exp(-32) / 128 = 4e-8 of them; 127 of their values are 1
    assert out[0, 0, 3] == math.inf
    out[0, 0, 3] = out[0, 0, 4]
    assert (out == 127 / 128).all()
