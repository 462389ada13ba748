"""The attention operators together, as a served layer uses them: a prompt in two chunks, then decode steps, next to linear()
and moe_few_tokens().  Every attention is held to the formula over what was written before it."""

import pytest
import torch

from attention_reference import attention64, quantise64
from serving_reference import check_close
from test_attention_cached_gpu import WEIGHT as CACHED_WEIGHT
from test_attention_prompt_gpu import WEIGHT as PROMPT_WEIGHT

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32
HEADS, KV, DIM, HIDDEN, PAGE = 8, 2, 64, 512, 16


class _Layer:
    """Weights of one layer, its cache, and what the 64-bit side knows of every sequence's keys and values."""

    def __init__(self, dtype, seqs, most):
        from revealaiccl_b200.ops.kv_cache import KVCache4
        gen = torch.Generator(DEV).manual_seed(5)

        def weight(*shape):
            return (torch.randn(*shape, generator=gen, device=DEV) * shape[-1] ** -0.5).to(dtype)

        self.dtype = dtype
        self.w_qkv, self.w_out = weight((HEADS + 2 * KV) * DIM, HIDDEN), weight(HIDDEN, HEADS * DIM)
        self.router, self.w1, self.w2 = weight(8, HIDDEN), weight(8, 2 * 256, HIDDEN), weight(8, HIDDEN, 256)
        pages = seqs * -(-most // PAGE) + 5
        self.cache = KVCache4.empty(pages, PAGE, KV, DIM)
        for t in (self.cache.k_scales, self.cache.v_scales):   # what nobody wrote must not matter
            t.view(torch.uint8).fill_(0x7f)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(6))
        self.table = order[:seqs * -(-most // PAGE)].view(seqs, -1).int().to(DEV)
        self.k = [[] for _ in range(seqs)]
        self.v = [[] for _ in range(seqs)]

    def slots(self, b, pos):
        return self.table[b, pos // PAGE].long() * PAGE + pos % PAGE

    def qkv(self, x):
        from revealaiccl_b200.ops.linear import linear
        y = linear(x, self.w_qkv).unflatten(1, (HEADS + 2 * KV, DIM))
        return y[:, :HEADS], y[:, HEADS:HEADS + KV], y[:, HEADS + KV:]

    def keep(self, b, k, v):
        self.k[b].append(quantise64(k))
        self.v[b].append(quantise64(v))

    def held(self, b):
        return torch.cat(self.k[b]), torch.cat(self.v[b])


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_prompt_in_chunks_then_decode(dtype):
    from revealaiccl_b200.ops.attention import attention_cached, attention_prompt
    from revealaiccl_b200.ops.kv_cache import kv_cache_read, kv_cache_write
    from revealaiccl_b200.ops.linear import linear
    from revealaiccl_b200.ops.moe_few import moe_few_tokens
    from revealaiccl_b200.ops.status import check_serving

    chunks, steps = [[70, 1, 33], [19, 40, 0]], 4
    layer = _Layer(dtype, 3, 140)
    gen = torch.Generator(DEV).manual_seed(7)
    length = [0, 0, 0]
    for nth, lens in enumerate(chunks):
        x = torch.randn(sum(lens), HIDDEN, generator=gen, device=DEV).to(dtype)
        q, k, v = layer.qkv(x)
        slots = torch.cat([layer.slots(b, torch.arange(length[b], length[b] + n, device=DEV)) for b, n in enumerate(lens)])
        kv_cache_write(layer.cache, k, v, slots)
        at = 0
        for b, n in enumerate(lens):
            layer.keep(b, k[at:at + n], v[at:at + n])
            at += n
        full = [a + n for a, n in zip(length, lens)]
        cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
        if nth == 0:
            keys, values, cu_k = k, v, cu          # nothing came before
        else:
            context = torch.cat([layer.slots(b, torch.arange(n, device=DEV)) for b, n in enumerate(full)])
            keys, values = kv_cache_read(layer.cache, context, dtype=dtype)
            cu_k = torch.tensor([0] + full, device=DEV).cumsum(0).int()
        out = attention_prompt(q, keys, values, cu, cu_k)
        at = ak = 0
        for b, n in enumerate(lens):
            m = n if nth == 0 else full[b]
            kk, vv = (k[at:at + n].double(), v[at:at + n].double()) if nth == 0 else layer.held(b)
            seen = torch.arange(n, device=DEV) + (m - n + 1)
            want, _, bound, *_ = attention64(q[at:at + n], kk, vv, seen, None, PROMPT_WEIGHT[dtype])
            check_close(out[at:at + n], want, bound)
            at, ak = at + n, ak + m
        x = linear(out.flatten(1), layer.w_out, residual=x)
        assert x.isfinite().all()
        length = full
    # decode: one graph, replayed with each step's tokens
    x = torch.randn(3, HIDDEN, generator=gen, device=DEV).to(dtype)
    slots, lens = torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)

    def step():
        q, k, v = layer.qkv(x)
        kv_cache_write(layer.cache, k, v, slots)
        out, lse = attention_cached(q, layer.cache, layer.table, lens, return_lse=True)
        h = linear(out.flatten(1), layer.w_out, residual=x)
        y, _, _ = moe_few_tokens(h, layer.router, layer.w1, layer.w2, top_k=2, residual=h)
        return q, k, v, out, lse, y

    graph = torch.cuda.CUDAGraph()
    slots.fill_(-1)
    with torch.cuda.graph(graph):
        q, k, v, out, lse, y = step()
    for _ in range(steps):
        slots.copy_(torch.stack([layer.slots(b, torch.tensor(n, device=DEV)) for b, n in enumerate(length)]))
        length = [n + 1 for n in length]
        lens.copy_(torch.tensor(length, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(3):
            layer.keep(b, k[b:b + 1], v[b:b + 1])
            want, wlse, bound, lbound, _ = attention64(q[b:b + 1], *layer.held(b), torch.tensor([length[b]], device=DEV), None, CACHED_WEIGHT[dtype])
            check_close(out[b:b + 1], want, bound)
            check_close(lse[b:b + 1], wlse, lbound)
        assert y.isfinite().all()
        x.copy_(torch.nn.functional.normalize(y.float()).mul(HIDDEN ** 0.5).to(dtype))
    check_serving(DEV)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_parts_of_a_context_join_by_their_sums(dtype):
    """Keys in three parts, one of them empty: outputs weighted by exp(lse - joint lse) are the whole's."""
    from revealaiccl_b200.ops.attention import attention_prompt
    gen = torch.Generator(DEV).manual_seed(9)
    q, k, v = (torch.randn(n, h, DIM, generator=gen, device=DEV).to(dtype) for n, h in ((40, HEADS), (300, KV), (300, KV)))

    def cu(n):
        return torch.tensor([0, n], dtype=torch.int32, device=DEV)

    parts = [attention_prompt(q, k[a:b], v[a:b], cu(40), cu(b - a), causal=False, return_lse=True) for a, b in ((0, 170), (170, 170), (170, 300))]
    total = torch.logsumexp(torch.stack([lse.double() for _, lse in parts]), 0)
    got = sum(o.double() * torch.exp(lse.double() - total)[..., None] for o, lse in parts)
    want, wlse, bound, lbound, _ = attention64(q, k, v, torch.full((40,), 300, device=DEV), None, PROMPT_WEIGHT[dtype])
    check_close(got, want, 2 * bound)      # each part has its own roundings, and weights of at most 1 in all
    check_close(total, wlse, 2 * lbound)


def test_calls_at_once():
    """The same calls on two streams at a time, into memory of their own, with one cache to read from."""
    from test_attention_cached_gpu import _filled, _q, _table
    from revealaiccl_b200.ops.attention import attention_cached, attention_prompt
    lengths = [900, 40, 333]
    cache = _filled(100, 16, 2, 128)
    table = _table(lengths, 16, cache.pages)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    qs = [_q(3, 8, 128, BF16, seed=i) for i in range(4)]
    rows = torch.randn(600, 12, 128, generator=torch.Generator(DEV).manual_seed(2), device=DEV).to(BF16)
    cu = torch.tensor([0, 250, 600], dtype=torch.int32, device=DEV)

    def both(q, i):
        return attention_cached(q, cache, table, lens), attention_prompt(rows[:, :8], rows[:, 8:10], rows[:, 8 + i % 2:10 + i % 2], cu)

    want = [both(q, i) for i, q in enumerate(qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(10):
        got = []
        for i, (s, q) in enumerate(zip(streams, qs)):
            with torch.cuda.stream(s):
                got.append(both(q, i))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
