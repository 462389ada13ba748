"""moe_few_tokens(): the mixture-of-experts layer for a few tokens, against 64 bits."""

import pytest
import torch

from serving_reference import HALF, PARTS, U, check_close, check_norm, linear64, moe64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32
INF = float("inf")


def _moe(*a, **k):
    from revealaiccl_b200.ops.moe_few import moe_few_tokens
    return moe_few_tokens(*a, **k)


def _plan(a, k, act):
    from revealaiccl_b200.ops._native import kernels
    from revealaiccl_b200.ops.grouped_gemm import ACT_IDS
    return kernels().moe_few_plan(a["x"], a["w1"], a["w2"], k, ACT_IDS[act], torch.cuda.get_device_properties(DEV).multi_processor_count)


def _make(T, D, E, F, O, act, dtype, seed=0, bias=False):
    g = torch.Generator(DEV).manual_seed(seed)

    def n(*shape, s=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * s

    n1 = 2 * F if act == "swiglu" else F
    a = dict(x=n(T, D).to(dtype), router_w=n(E, D, s=D ** -0.5).to(dtype), w1=n(E, n1, D, s=D ** -0.5).to(dtype),
             w2=n(E, O, F, s=F ** -0.5).to(dtype))
    if bias:
        a.update(router_b=n(E, s=0.1), b1=n(E, n1, s=0.1), b2=n(E, O, s=0.1))
    return a


def _sizes(tensor, dtype, pairs, O=None):
    """(D, F, O): widths whose (token, choice) pairs read few bytes of weights (by rows, on CUDA cores) or many (on the tensor
    cores, from 30 MB in bf16 and 540 MB in fp32), as csrc/kernels/moe_few.cu chooses."""
    if not tensor:
        return 256, 96, O or 128
    D, F = (512, 1000) if dtype == BF16 else (1024, 1400)
    while pairs * (2 if dtype == BF16 else 4) * 3 * D * F < (32e6 if dtype == BF16 else 560e6):
        F += 1000
    return D, F, O or D


def _check(a, k, act, gate_mode, norm=True, **kw):
    out, ids, gates = _moe(**a, top_k=k, act=act, gate_mode=gate_mode, **kw)
    kw = {n: v for n, v in kw.items() if n != "out"}
    want, bound, rid, rg, grel, gap = moe64(**a, top_k=k, act=act, gate_mode=gate_mode, **kw)
    # The choices are the reference's where no two logits lie closer than their errors: a logit of order one is summed
    # by 32 lanes in D / 32 steps each and five additions, errors of 2^-24 and random sign; four times that, for two logits.
    assert gap > 4 * U * ((a["x"].shape[1] / 32) ** 0.5 + 8), "two logits too close to tell"
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu(), rid)
    check_close(gates.cpu(), rg, grel * rg.abs() + U * rg.abs() + 2.0 ** -126)  # fp32 has no normal number below 2^-126
    check_close(out, want, bound)
    dt, odt = a["x"].dtype, out.dtype
    if norm and want.numel() >= 64 and not want.isnan().any():
        hidden = HALF[dt] if dt == BF16 else 2 * PARTS
        check_norm(out, want, 2 * (HALF[odt] + hidden + U * (a["x"].shape[1] ** 0.5 + a["w2"].shape[2] ** 0.5 + 16)) + grel)
    return out, ids, gates


SIZES = [  # T, D, E, k, F, O
    (1, 1, 1, 1, 1, 1), (1, 64, 4, 1, 16, 16), (1, 2048, 4, 1, 32, 16), (2, 256, 64, 6, 176, 256), (3, 100, 5, 2, 77, 33),
    (4, 128, 8, 8, 128, 128), (7, 512, 16, 4, 200, 512), (8, 1024, 8, 2, 1792, 1024), (13, 264, 60, 4, 40, 136),
    (16, 384, 255, 8, 24, 384), (17, 520, 24, 3, 344, 72), (31, 65, 9, 3, 129, 250), (33, 256, 64, 6, 704, 256),
    (37, 512, 4, 2, 3000, 130), (48, 200, 128, 5, 56, 200), (63, 320, 3, 3, 320, 640), (64, 256, 8, 2, 1024, 256),
    (64, 128, 1, 1, 5000, 128), (64, 192, 32, 8, 96, 1000),
]


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,D,E,k,F,O", SIZES)
def test_sizes(T, D, E, k, F, O, dtype):
    act = ("swiglu", "relu", "gelu", "silu", "swiglu")[(T + D + F) % 5]
    mode = ("topk_softmax", "softmax", "none")[(T + E) % 3]
    _check(_make(T, D, E, F, O, act, dtype, seed=T + D, bias=(T + k) % 2 == 0), k, act, mode)


@pytest.mark.parametrize("tensor", [False, True], ids=["rows", "tensor"])
@pytest.mark.parametrize("act,mode", [("swiglu", "topk_softmax"), ("relu", "softmax"), ("gelu", "none"), ("silu", "topk_softmax"),
                                      ("none", "softmax"), ("swiglu", "none"), ("swiglu", "softmax")])
@pytest.mark.parametrize("dtype,out_dtype,res_dtype", [(BF16, BF16, BF16), (BF16, FP32, BF16), (BF16, BF16, FP32), (FP32, FP32, FP32),
                                                       (FP32, FP32, BF16)])
def test_acts_gates_types(act, mode, dtype, out_dtype, res_dtype, tensor):
    D, F, O = _sizes(tensor, dtype, 9 if act != "swiglu" else 18, 192)
    a = _make(9, D, 12, F, O, act, dtype, seed=3, bias=True)
    r = torch.randn(9, O, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(res_dtype)
    out, _, _ = _check(a, 3, act, mode, residual=r, out_dtype=out_dtype)
    assert out.dtype == out_dtype


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 6, 17, 33, 49, 64])
@pytest.mark.parametrize("tensor", [False, True], ids=["rows", "tensor"])
def test_every_token_on_one_expert(T, dtype, tensor):
    D, F, O = _sizes(tensor, dtype, T, 256)
    a = _make(T, D, 16 if T > 1 else 2, F, O, "swiglu", dtype, bias=True)
    if T == 1:
        a["router_b"][1] += 100.0
        _, ids, _ = _check(a, 1, "swiglu", "softmax")
        assert (ids == 1).all()
        return
    a["router_b"][11] += 100.0
    _, ids, _ = _check(a, 1, "swiglu", "softmax")
    assert (ids == 11).all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tensor", [False, True], ids=["rows", "tensor"])
def test_masks(dtype, tensor):
    """Blocked experts, tokens with fewer free experts than choices, tokens with none; what is blocked is not read."""
    T, E = 12, 8
    D, F, O = _sizes(tensor, dtype, T * 2, 128)
    a = _make(T, D, E, F, O, "swiglu", dtype, bias=True)
    g = torch.Generator(DEV).manual_seed(5)
    mask = torch.rand(T, E, generator=g, device=DEV) < 0.4
    mask[0] = True            # none left
    mask[1] = True
    mask[1, 3] = False        # one left
    mask[:, 6] = True         # blocked for every token: may hold anything
    for name in ("w1", "w2", "b1", "b2"):
        a[name][6] = float("nan")
    a["router_w"][6] = float("nan")
    r = torch.randn(T, 128, generator=g, device=DEV).to(dtype)
    clean = {n: v.clone() for n, v in a.items()}
    for name, v in clean.items():
        if name != "x":
            v[6] = 0
    out, ids, gates = _moe(**a, top_k=3, act="swiglu", gate_mode="topk_softmax", block_mask=mask, residual=r)
    want, wid, wgates = _check(clean, 3, "swiglu", "topk_softmax", block_mask=mask, residual=r)
    assert torch.equal(out, want) and torch.equal(ids, wid) and torch.equal(gates, wgates)
    assert (ids[0] == -1).all() and (gates[0] == 0).all() and torch.equal(out[0], r[0])
    assert ids[1].tolist() == [3, -1, -1] and gates[1].tolist() == [1, 0, 0]
    out, ids, _ = _moe(**clean, top_k=3, act="swiglu", gate_mode="softmax", block_mask=mask.to(torch.uint8))
    assert (out[0] == 0).all()
    # one mask for all tokens, all blocked
    out, ids, _ = _moe(**clean, top_k=2, act="swiglu", gate_mode="none", block_mask=torch.ones(E, device=DEV, dtype=torch.bool))
    assert (out == 0).all() and (ids == -1).all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D,E,k", [(2048, 4, 1), (77, 1, 1), (256, 8, 8), (2048, 16, 3), (1000, 16, 2), (256, 17, 2), (4096, 8, 2)])
def test_one_token(D, E, k, dtype):
    """One token, on both sides of where its few experts are routed by the experts' kernel: masks, no expert left, NaN, ties."""
    a = _make(1, D, E, 72, 40, "swiglu", dtype, seed=E, bias=True)
    r = torch.randn(1, 40, device=DEV).to(dtype)
    for mode in ("topk_softmax", "softmax", "none"):
        _, ids, _ = _check(a, k, "swiglu", mode, residual=r)
        mask = torch.zeros(E, device=DEV, dtype=torch.bool)
        mask[ids[0, 0]] = True
        _, ids, gates = _check(a, k, "swiglu", mode, residual=r, block_mask=mask)
        assert not (ids == int(mask.nonzero())).any() and (k < E or ids[0, -1] == -1 and gates[0, -1] == 0)
        out, ids, gates = _moe(**a, top_k=k, act="swiglu", gate_mode=mode, residual=r, block_mask=~torch.zeros_like(mask))
        assert (ids == -1).all() and (gates == 0).all() and torch.equal(out, r)
    b = dict(a, router_w=a["router_w"][:1].expand(E, D), router_b=a["router_b"][:1].expand(E).contiguous())
    _, ids, _ = _moe(**b, top_k=k, act="swiglu", gate_mode="softmax")
    assert ids[0].tolist() == list(range(k))
    b = dict(a, x=a["x"].clone())
    b["x"][0, D // 2] = float("nan")
    out, ids, _ = _moe(**b, top_k=k, act="swiglu", gate_mode="topk_softmax")
    assert out.isnan().all() and ids[0].tolist() == list(range(k))


@pytest.mark.parametrize("mode", ["topk_softmax", "softmax", "none"])
def test_bias_as_mask(mode):
    """A bias of -inf blocks; the type's lowest value is a number like any other and comes last."""
    a = _make(5, 128, 6, 64, 64, "silu", BF16, bias=True)
    a["router_b"][2] = -INF
    a["router_b"][4] = torch.finfo(FP32).min
    _, ids, gates = _check(a, 6, "silu", mode)
    assert (ids[:, 5] == -1).all() and (ids[:, 4] == 4).all() and (gates[:, 5] == 0).all()
    a["router_b"][:] = -INF
    out, ids, gates = _moe(**a, top_k=2, act="silu", gate_mode=mode)
    assert (ids == -1).all() and (gates == 0).all() and (out == 0).all()


def test_ties_go_to_the_lower_expert():
    a = _make(10, 256, 32, 32, 32, "relu", BF16)
    a["router_w"][:] = a["router_w"][:1]
    _, ids, _ = _moe(**a, top_k=8, act="relu", gate_mode="softmax")
    assert (ids.cpu() == torch.arange(8, dtype=torch.int32)).all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tensor", [False, True], ids=["rows", "tensor"])
def test_special_values_stay_where_they_are(dtype, tensor):
    """A NaN or infinite token, and weights of experts that nobody chose, leave the other tokens alone."""
    D, F, O = _sizes(tensor, dtype, 12, 96)
    a = _make(6, D, 16, F, O, "swiglu", dtype)
    base, ids, _ = _moe(**a, top_k=2, act="swiglu", gate_mode="topk_softmax")
    unused = [e for e in range(16) if not (ids == e).any()]
    b = {n: v.clone() for n, v in a.items()}
    for e in unused:
        b["w1"][e], b["w2"][e] = float("nan"), INF
    out, _, _ = _moe(**b, top_k=2, act="swiglu", gate_mode="topk_softmax")
    assert unused and torch.equal(out, base)
    a["x"][2, 7] = float("nan")
    a["x"][4, 9] = INF
    out, ids, _ = _moe(**a, top_k=2, act="swiglu", gate_mode="topk_softmax")
    assert out[2].isnan().all() and ids[2].tolist() == [0, 1]
    keep = [0, 1, 3, 5]
    assert torch.equal(out[keep], base[keep])


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 0), (8, 24)])
@pytest.mark.parametrize("tensor", [False, True], ids=["rows", "tensor"])
def test_strides(dtype, offset, pad, tensor):
    """Every tensor as a window of a wider buffer, every other expert of a larger bank; what lies around out stays."""
    T, E = 5, 6
    D, F, O = _sizes(tensor, dtype, T * 2, 72)
    g = torch.Generator(DEV).manual_seed(2)

    def window(*shape, s):
        wide = (torch.randn(*shape[:-1], shape[-1] + offset + pad, generator=g, device=DEV) * s).to(dtype)
        return wide[..., offset:offset + shape[-1]]

    a = dict(x=window(T, D, s=1.0), router_w=window(E, D, s=D ** -0.5), w1=window(2 * E, 2 * F, D, s=D ** -0.5)[::2],
             w2=window(2 * E, O, F, s=F ** -0.5)[1::2])
    ob = torch.full((T + 2, O + offset + pad), 7.0, device=DEV, dtype=dtype)
    r = window(T, O, s=1.0)
    mask = torch.zeros(T, E + 3, device=DEV, dtype=torch.bool)[:, 1:E + 1]
    _check(a, 2, "swiglu", "topk_softmax", residual=r, block_mask=mask, out=ob[1:T + 1, offset:offset + O])
    ob[1:T + 1, offset:offset + O] = 7.0
    assert torch.equal(ob, torch.full_like(ob, 7.0))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,D,E,k,F,O,act", [(33, 401, 4, 4, 2203, 302, "swiglu"), (64, 515, 8, 8, 1777, 131, "gelu"), (20, 1803, 4, 3, 1809, 1803, "swiglu"),
                                             (64, 2051, 1, 1, 1001, 77, "relu"), (40, 512, 3, 3, 2000, 520, "swiglu"), (12, 2050, 2, 2, 3001, 66, "silu")])
def test_many_tokens_on_odd_rows(T, D, E, k, F, O, act, dtype):
    """Weights off 16 bytes with enough tokens for a copy of the experts: odd widths, and windows at odd places."""
    a = _make(T, D, E, F, O, act, dtype, bias=True)
    if D % 8 == 0:
        for n in ("w1", "w2"):
            w = a[n]
            wide = torch.full((2 * w.shape[0], w.shape[1] + 1, w.shape[2] + 3), float("nan"), device=DEV, dtype=dtype)
            view = wide[1::2, 1:, 1:1 + w.shape[2]]
            view.copy_(w)
            a[n] = view
    _check(a, k, act, "topk_softmax", residual=torch.randn(T, O, device=DEV).to(dtype))


@pytest.mark.parametrize("T", [1, 4, 48])
def test_experts_that_share_their_weights(T):
    """Experts, or rows of an expert, that are one tensor expanded."""
    a = _make(T, 512, 4, 1000, 256, "swiglu", BF16)
    _check(dict(a, w1=a["w1"][:1].expand(4, -1, -1), w2=a["w2"][:1].expand(4, -1, -1)), 3, "swiglu", "softmax")
    _check(dict(a, w2=a["w2"][:, :1].expand(-1, 256, -1)), 3, "swiglu", "softmax")


def test_empty_batch_and_in_place():
    a = _make(4, 64, 4, 32, 64, "swiglu", BF16)
    e = dict(a, x=a["x"][:0])
    out, ids, gates = _moe(**e, top_k=2)
    assert out.shape == (0, 64) and ids.shape == (0, 2) and gates.shape == (0, 2)
    r = torch.randn(4, 64, device=DEV).bfloat16()
    want, _, _ = _moe(**a, top_k=2, residual=r)
    got, _, _ = _moe(**a, top_k=2, residual=r, out=r)
    assert got.data_ptr() == r.data_ptr() and torch.equal(got, want)


def test_far_experts():
    """Element offsets past 32 bits in the experts' weights: the last of 60 experts of a bank of 4.3 G elements."""
    D, F, E = 4096, 5888, 60
    bank = torch.zeros(E, 2 * F + F, D, device=DEV, dtype=BF16)
    w1, w2 = bank[:, :2 * F], bank.view(E, -1)[:, 2 * F * D:].view(E, D, F)
    g = torch.Generator(DEV).manual_seed(0)
    x = torch.randn(2, D, generator=g, device=DEV).bfloat16()
    for e in (0, E - 1):
        w1[e].normal_(0, D ** -0.5, generator=g)
        w2[e].normal_(0, F ** -0.5, generator=g)
    bias = torch.zeros(E, device=DEV)
    bias[[0, E - 1]] = 100.0
    rw = (torch.randn(E, D, generator=g, device=DEV) * D ** -0.5).bfloat16()
    out, ids, gates = _moe(x, rw, w1, w2, top_k=2, router_b=bias)
    assert (ids.sort(dim=1).values.cpu() == torch.tensor([0, E - 1])).all()
    pick = torch.tensor([0, E - 1], device=DEV)
    want, bound, _, _, _, _ = moe64(x, rw[pick], w1[pick], w2[pick], top_k=2, act="swiglu", gate_mode="topk_softmax",
                                    router_b=bias[pick])
    check_close(out, want, bound)


def test_repeats_and_streams():
    """The same bits every time, on side streams too and while another call runs."""
    sets = [_make(T, 512, E, F, 512, "swiglu", BF16, seed=T) for T, E, F in ((1, 64, 352), (30, 16, 512), (64, 8, 1000), (3, 4, 5000))]
    want = [_moe(**a, top_k=2) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(20):
        for a, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(_moe(**a, top_k=2))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(u, v) for u, v in zip(g, want[i % len(want)]))


@pytest.mark.parametrize("F", [96, 1000], ids=["rows", "tensor"])
def test_a_block_of_a_served_model(F):
    """Attention output projection, experts and a shared expert as one decode step, eager and as two captured graphs
    replayed in turn, with new inputs each time."""
    from revealaiccl_b200.ops.linear import linear
    T, D, E, S = 11, 256, 16, 160
    a = _make(T, D, E, F, D, "swiglu", BF16, seed=8)
    g = torch.Generator(DEV).manual_seed(9)
    attn = torch.randn(T, D, generator=g, device=DEV).bfloat16()
    wo = (torch.randn(D, D, generator=g, device=DEV) * D ** -0.5).bfloat16()
    su = (torch.randn(2 * S, D, generator=g, device=DEV) * D ** -0.5).bfloat16()
    sd = (torch.randn(D, S, generator=g, device=DEV) * S ** -0.5).bfloat16()
    x = a.pop("x")

    def step():
        h = linear(attn, wo, residual=x)
        y, ids, gates = _moe(h, **a, top_k=4, residual=h)
        return h, linear(linear(h, su, act="swiglu"), sd, residual=y, out=y), ids, gates

    def check(result):
        h, y, ids, gates = result
        want, bound = linear64(attn, wo, residual=x)
        check_close(h, want, bound)
        want, bound, rid, rg, _, gap = moe64(h, **a, top_k=4, act="swiglu", gate_mode="topk_softmax", residual=h)
        assert gap > 1e-6 and torch.equal(ids.cpu(), rid)
        u = linear(h, su, act="swiglu")
        s, sb = linear64(u, sd)
        # the routed sum was rounded once before the shared expert's product was added
        check_close(y, want + s, bound + sb + HALF[BF16] * (want + s).abs() + HALF[BF16] * bound)

    check(step())
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
        graphs.append((graph, result))
    for i in range(4):
        attn.normal_(generator=g), x.normal_(generator=g)
        want = [t.clone() for t in step()]
        graph, result = graphs[i % 2]
        graph.replay()
        assert all(torch.equal(u, v) for u, v in zip(result, want))
        check(result)


@pytest.mark.parametrize("dtype,act,k", [("bf16", "swiglu", 2), ("fp32", "gelu", 2), ("fp32", "relu", 1)])
def test_layer_few_tokens(dtype, act, k):
    """A layer's decode step beside its batches: same router, masks and experts, and the batch's results stay."""
    from revealaiccl_b200.moe.config import MoELayerConfig
    from revealaiccl_b200.moe.layer import ProgressiveMoELayer

    cfg = MoELayerConfig(
        name=f"few_{dtype}_{act}", tokens_per_rank=512, hidden=256, experts=8, top_k=k, chunk_sizes=(64,) * 8, ffn_hidden=128,
        out_dim=256, activation=act, dtype=dtype, placement="contiguous", gate_mode="topk_softmax" if k > 1 else "none",
        mask_mode="topology_source" if act == "relu" else "none", router_init="unit_logits", expert_init="normal002")
    layer = ProgressiveMoELayer(cfg, device=torch.device("cuda", 0), timeout_s=5.0)
    try:
        before = layer.forward("early").clone()
        w = layer.weights
        for T in (1, 5, 64):
            x = layer.inputs.tokens[:T].clone()
            res = torch.randn(T, cfg.out_dim, device=DEV).to(x.dtype)
            out, ids, gates = layer.few_tokens(x, residual=res)
            mask = None
            if cfg.mask_mode == "topology_source":
                mask = torch.zeros(T, cfg.experts, dtype=torch.bool, device=DEV)
                mask[torch.arange(T), torch.arange(T) % cfg.experts] = True
            want, bound, rid, rg, grel, gap = moe64(x, w.router_w, w.w1, w.w2, top_k=k, act=act, gate_mode=cfg.gate_mode,
                                                    router_b=w.router_b, b1=w.b1, b2=w.b2, block_mask=mask, residual=res)
            assert gap > 4 * U * ((cfg.hidden / 32) ** 0.5 + 8)
            assert torch.equal(ids.cpu(), rid) and torch.equal(ids, layer.expert_ids[:T])
            check_close(out, want, bound)
        assert torch.equal(layer.forward("early"), before)
        assert layer.verify()["pass"]
    finally:
        layer.close()


@pytest.mark.parametrize("where", ["x", "w1", "w2"])
@pytest.mark.parametrize("T", [1, 64])
def test_largest_numbers(T, where):
    """Finite fp32 numbers up to the type's largest in the tokens, the weights and the activations, by rows and on the
    tensor cores: what they are multiplied by keeps each result far below it."""
    E, D, F, O = 4, 512, 1200, 512
    top = torch.finfo(FP32).max
    a = _make(T, D, E, F, O, "relu", FP32, seed=4)
    a["router_w"].zero_()
    a["router_b"] = torch.randn(E, device=DEV, generator=torch.Generator(DEV).manual_seed(5))
    a["x"] = a["x"].sign() * (torch.arange(D, device=DEV) == 3)
    if where == "x":          # z = top * w1
        a["x"] *= top
        a["w1"] *= 2.0 ** -100
    elif where == "w1":       # z = +-top, and so are the activations
        a["w1"] = a["w1"].sign() * top
        a["w2"] *= 2.0 ** -100
    else:
        a["w1"] *= 2.0 ** -40
        a["w2"] = a["w2"].sign() * top
        a["w2"][:, :, F // 2:] = 0
        a["w2"][:, :, ::3] = 0
    out, ids, gates = _moe(**a, top_k=2, act="relu", gate_mode="topk_softmax")
    want, bound, rid, rg, _, _ = moe64(**a, top_k=2, act="relu", gate_mode="topk_softmax")
    assert torch.equal(ids.cpu(), rid) and out.isfinite().all()
    check_close(out, want, bound)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tensor", [False, True], ids=["rows", "tensor"])
def test_tokens_that_share_their_rows(dtype, tensor):
    """Tokens that are one row expanded, or windows that overlap."""
    E, D, O, T = 6, 512, 512, 9
    F = 10000 if tensor else 96
    a = _make(1, D, E, F, O, "swiglu", dtype, seed=6)
    path = _plan(dict(a, x=a["x"].expand(T, D)), 2, "swiglu")
    assert path["path"] == ("tensor" if tensor else "rows") and path["pack_x"] == tensor
    out, ids, _ = _check(dict(a, x=a["x"].expand(T, D)), 2, "swiglu", "softmax")
    assert (out == out[:1]).all() and (ids == ids[:1]).all()
    long = torch.randn(T * 64 + D, device=DEV, generator=torch.Generator(DEV).manual_seed(7)).to(dtype)
    _check(dict(a, x=long.as_strided((T, D), (64, 1))), 2, "swiglu", "softmax")
