"""Results that lie between the elements of other tensors of the call, without sharing any."""

import random

import pytest
import torch

from revealaiccl_b200.ops import _native

if not _native.has_kernels():  # pragma: no cover
    pytest.skip("kernel library not built", allow_module_level=True)

from revealaiccl_b200.ops.attention import attention_cached, attention_prompt
from revealaiccl_b200.ops.kv_cache import KVCache4, kv_cache_read, kv_cache_write

BF16, INT = torch.bfloat16, torch.int32
NO_GPU = "must be on a CUDA device"     # what the CPU's tensors meet behind all other checks


def _joint(n, heads, dim, device, fill=0.0):
    """Pairs (k, v) [n, heads, dim] in one buffer each: behind one another in a row, by turns of heads, of dimensions, of tokens."""
    by_row = torch.full((n, 2 * heads, dim), fill, dtype=BF16, device=device)
    by_head = torch.full((n, heads, 2, dim), fill, dtype=BF16, device=device)
    by_dim = torch.full((n, heads, 2 * dim), fill, dtype=BF16, device=device)
    by_token = torch.full((n, 2, heads, dim), fill, dtype=BF16, device=device)
    heads_first = torch.full((heads, 2, n, dim), fill, dtype=BF16, device=device)
    return [(by_row[:, :heads], by_row[:, heads:]), (by_row[:, heads:], by_row[:, :heads]), (by_head[:, :, 0], by_head[:, :, 1]),
            (by_dim[:, :, dim:], by_dim[:, :, :dim]), (by_token[:, 0], by_token[:, 1]),
            (heads_first[:, 0].transpose(0, 1), heads_first[:, 1].transpose(0, 1))]


@pytest.mark.parametrize("heads", [1, 2, 3])
@pytest.mark.parametrize("n", [1, 2, 5])
def test_joint_buffers_are_taken(n, heads):
    cache = KVCache4.empty(3, 16, heads, 64, device="cpu")
    for k, v in _joint(n, heads, 64, "cpu"):
        with pytest.raises(ValueError, match=NO_GPU):
            kv_cache_read(cache, torch.zeros(n, dtype=INT), k_out=k, v_out=v)
    buf = torch.zeros(n, 12, 64, dtype=BF16)
    kv = torch.zeros(n, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match=NO_GPU):
        attention_prompt(buf[:, :6], kv, kv, torch.zeros(2, dtype=INT), out=buf[:, 6:])
    with pytest.raises(ValueError, match=NO_GPU):
        attention_cached(buf[:, 6:6 + 2 * heads], cache, torch.zeros(n, 2, dtype=INT), torch.zeros(n, dtype=INT), out=buf[:, :2 * heads])


def test_no_shared_element_is_taken():
    """Random strides over one buffer, against the elements' own places."""
    rng = random.Random(0)
    buf = torch.zeros(40000, dtype=BF16)
    taken = refused = 0
    for _ in range(4000):
        n, heads = rng.choice((1, 2, 3, 5)), rng.choice((1, 2, 3))
        token = rng.choice((64, 100, 128, 192, 256, 384, 512))
        places = []
        for _ in range(2):
            strides = (rng.choice((token, token, rng.randrange(64, 600))), rng.choice((64, 128, 64 * n, token * n, rng.randrange(64, 600))), 1)
            places.append(torch.as_strided(buf, (n, heads, 64), strides, rng.randrange(0, 1200)))
        at = [torch.arange(buf.numel()).as_strided(t.shape, t.stride(), t.storage_offset()).flatten() for t in places]
        if any(len(a.unique()) < a.numel() for a in at):
            continue
        meet = bool(torch.isin(at[0], at[1]).any())
        with pytest.raises(ValueError) as e:
            kv_cache_read(KVCache4.empty(1, 16, heads, 64, device="cpu"), torch.zeros(n, dtype=INT), k_out=places[0], v_out=places[1])
        if "v_out shares memory" in str(e.value):
            refused += not meet
        elif NO_GPU in str(e.value):
            assert not meet, [(t.shape, t.stride(), t.storage_offset()) for t in places]
            taken += 1
    assert taken > 500 and refused < taken


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_joint_buffers_hold_what_separate_ones_do(dtype):
    gen = torch.Generator("cuda").manual_seed(0)
    n, heads, dim = 100, 3, 64
    cache = KVCache4.empty(8, 16, heads, dim)
    new = torch.randn(2, n, heads, dim, generator=gen, device="cuda").to(dtype)
    slots = torch.randperm(128, device="cuda")[:n]
    kv_cache_write(cache, new[0], new[1], slots)
    k, v = kv_cache_read(cache, slots, check=True)
    for k_out, v_out in _joint(n, heads, dim, "cuda", 7.0):
        kv_cache_read(cache, slots, k_out=k_out, v_out=v_out, check=True)
        assert torch.equal(k_out, k) and torch.equal(v_out, v)
    cu = torch.tensor([0, 30, n], dtype=INT, device="cuda")
    q = torch.randn(n, 6, dim, generator=gen, device="cuda").to(dtype)
    want = attention_prompt(q, new[0], new[1], cu)
    buf = torch.full((n, 18, dim), 7.0, dtype=dtype, device="cuda")
    for q_at, out_at in ((0, 6), (6, 0), (1, 12)):
        buf.fill_(7.0)
        buf[:, q_at:q_at + 6] = q
        assert torch.equal(attention_prompt(buf[:, q_at:q_at + 6], new[0], new[1], cu, out=buf[:, out_at:out_at + 6], check=True), want)
        assert torch.equal(buf[:, q_at:q_at + 6], q)
        buf[:, q_at:q_at + 6], buf[:, out_at:out_at + 6] = 7.0, 7.0
        assert (buf == 7.0).all()
    lens, table = torch.tensor([0, 5, 30], dtype=INT, device="cuda"), torch.arange(2, dtype=INT, device="cuda").expand(3, -1)
    want = attention_cached(q[:3], cache, table, lens)
    buf = torch.full((3, 18, dim), 7.0, dtype=dtype, device="cuda")
    buf[:, 1:7] = q[:3]
    assert torch.equal(attention_cached(buf[:, 1:7], cache, table, lens, out=buf[:, 8:14], check=True), want)
    assert torch.equal(buf[:, 1:7], q[:3])
