"""Every path of linear() and moe_few_tokens() by name: each test asserts that its call takes the kernels that it is about."""

import pytest
import torch

from serving_reference import PARTS, U, check_close, check_norm, linear64, moe64
from test_linear_gpu import _linear, _make as _make_linear, _norm_bound
from test_moe_few_gpu import _check, _make, _moe, _plan

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32
INF = float("inf")


def _linear_plan(x, w, act, residual=None, out=None, out_dtype=None):
    from revealaiccl_b200.ops._native import kernels
    from revealaiccl_b200.ops.grouped_gemm import ACT_IDS
    dt = out.dtype if out is not None else out_dtype or x.dtype
    return kernels().linear_plan(x, w, ACT_IDS[act], residual, out, dt == BF16, torch.cuda.get_device_properties(DEV).multi_processor_count)


def _window(*shape, dtype, gen, scale=1.0, offset=1, pad=3):
    wide = (torch.randn(*shape[:-1], shape[-1] + offset + pad, generator=gen, device=DEV) * scale).to(dtype)
    return wide[..., offset:offset + shape[-1]]


# ---------------------------------------------------------------------------- linear

@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "swiglu"])
@pytest.mark.parametrize("out_dtype,res_dtype", [(BF16, BF16), (BF16, FP32), (FP32, BF16)])
def test_dense_256(act, out_dtype, res_dtype):
    """Tiles of 256 columns: several for each pair of SMs, ragged rows and columns, biases and residuals in every column."""
    m, k, n = 4300, 1096, 4616
    x, w, b, r = _make_linear(m, k, n, act, BF16, True, True, seed=1, res_dtype=res_dtype)
    assert _linear_plan(x, w, act, r, out_dtype=BF16)["tile"] == 256
    got = _linear(x, w, b, act=act, residual=r, out_dtype=out_dtype)
    want, bound = linear64(x, w, b, act, r, out_dtype)
    check_close(got, want, bound)


@pytest.mark.parametrize("m,k,n,act,dtype,tile", [
    (2100, 1096, 1200, "none", BF16, 256), (1100, 2056, 2600, "swiglu", BF16, 128), (700, 5000, 2600, "gelu", BF16, 128),
    (1500, 264, 3000, "swiglu", BF16, 128), (700, 1032, 900, "silu", FP32, 128), (900, 648, 1900, "swiglu", FP32, 128),
])
def test_dense_tiles(m, k, n, act, dtype, tile):
    x, w, b, r = _make_linear(m, k, n, act, dtype, True, True, seed=2)
    plan = _linear_plan(x, w, act, r)
    assert plan["kernel"] == "dense" and plan["tile"] == tile
    got = _linear(x, w, b, act=act, residual=r)
    want, bound = linear64(x, w, b, act, r)
    check_close(got, want, bound)
    check_norm(got, want, 2 * _norm_bound(k, dtype, dtype))


@pytest.mark.parametrize("m,k,n,act,dtype,tile", [
    (600, 8192, 2049, "none", BF16, 128), (600, 8192, 2049, "swiglu", BF16, 256), (1000, 4096, 2049, "swiglu", BF16, 128),
    (300, 2048, 1025, "swiglu", FP32, 128), (600, 2048, 1025, "gelu", FP32, 128),
])
def test_dense_tiles_off_16_bytes(m, k, n, act, dtype, tile):
    """out and residual as windows at odd places; what lies around out stays."""
    x, w, b, _ = _make_linear(m, k, n, act, dtype, True, False, seed=3)
    r = _window(m, n, dtype=dtype, gen=torch.Generator(DEV).manual_seed(4))
    ob = torch.full((m + 2, n + 4), 7.0, device=DEV, dtype=dtype)
    out = ob[1:m + 1, 1:n + 1]
    plan = _linear_plan(x, w, act, r, out)
    assert plan["kernel"] == "dense" and plan["tile"] == tile
    _linear(x, w, b, act=act, residual=r, out=out)
    want, bound = linear64(x, w, b, act, r)
    check_close(out, want, bound)
    check_norm(out, want, 2 * _norm_bound(k, dtype, dtype))
    out.fill_(7.0)
    assert torch.equal(ob, torch.full_like(ob, 7.0))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m,k,n,kernel,ranks", [(4, 512, 200, "vector", 0), (20, 2048, 512, "rows", 8), (700, 1024, 2000, "dense", 0),
                                                (3000, 64, 300, "rows", 1)])
def test_rows_apart(m, k, n, kernel, ranks, dtype):
    """A NaN or infinite row leaves the others' bits alone, whichever kernel runs."""
    x, w, b, r = _make_linear(m, k, n, "silu", dtype, True, True, seed=5)
    plan = _linear_plan(x, w, "silu", r)
    if not (dtype == FP32 and m == 3000):
        assert plan["kernel"] == kernel and plan["ranks"] == ranks
    base = _linear(x, w, b, act="silu", residual=r)
    x[1, 5], x[m - 2, k - 1] = float("nan"), INF
    got = _linear(x, w, b, act="silu", residual=r)
    keep = torch.ones(m, dtype=torch.bool, device=DEV)
    keep[[1, m - 2]] = False
    assert torch.equal(got[keep], base[keep]) and got[1].isnan().all() and not got[m - 2].isfinite().all()


# ---------------------------------------------------------------------------- layer

def _widths(T, k, dtype, act, D, O):
    """F from which the (token, choice) pairs read enough weights for the tensor cores."""
    F, eb = 200, 2 if dtype == BF16 else 4
    while T * k * eb * F * ((2 if act == "swiglu" else 1) * D + O) < (31e6 if dtype == BF16 else 550e6):
        F += 200
    return F


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_special_values_on_the_tensor_cores(dtype):
    """A NaN or infinite token, and weights of experts that nobody chose, leave the other tokens' bits alone."""
    T, D, O = 6, 512, 256
    F = _widths(T, 2, dtype, "swiglu", D, O)
    a = _make(T, D, 16, F, O, "swiglu", dtype)
    assert _plan(a, 2, "swiglu")["path"] == "tensor"
    base, ids, _ = _check(a, 2, "swiglu", "topk_softmax")
    unused = [e for e in range(16) if not (ids == e).any()]
    b = {n: v.clone() for n, v in a.items()}
    for e in unused:
        b["w1"][e], b["w2"][e] = float("nan"), INF
    out, _, _ = _moe(**b, top_k=2, act="swiglu", gate_mode="topk_softmax")
    assert unused and torch.equal(out, base)
    # The choices of the odd tokens change to others, and with the number of chosen experts the SMs' shares of their hidden
    # rows: a token's parts are then other sums, so the bits may differ and the 64-bit bound is what holds.
    a["router_b"] = torch.zeros(16, device=DEV)
    a["router_b"][[3, 9]] = 100.0
    kw = dict(top_k=2, act="swiglu", gate_mode="topk_softmax")
    _, ids, _ = _check(a, 2, "swiglu", "topk_softmax")
    assert (ids.sort().values.cpu() == torch.tensor([3, 9])).all()
    want, bound = moe64(**a, **kw)[:2]
    odd = dict(a, x=a["x"].clone())
    odd["x"][2, 7], odd["x"][4, 9] = INF, float("nan")
    out, ids, _ = _moe(**odd, **kw)
    assert out[4].isnan().all() and not out[2].isfinite().all()
    keep = [0, 1, 3, 5]
    check_close(out[keep], want[keep], bound[keep])
    # only these two experts for every token, so that the odd ones share all tiles with the others: the same sums
    mask = torch.ones(16, dtype=torch.bool, device=DEV)
    mask[[3, 9]] = False
    base, _, _ = _check(a, 2, "swiglu", "topk_softmax", block_mask=mask)
    out, ids, _ = _moe(**odd, **kw, block_mask=mask)
    assert (ids[keep + [4]].sort().values.cpu() == torch.tensor([3, 9])).all()   # infinite: a logit of -inf counts as blocked
    assert torch.equal(out[keep], base[keep]) and out[4].isnan().all() and not out[2].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 6, 17, 33, 64])
def test_one_expert_on_the_tensor_cores(T, dtype):
    D, O = 512, 256
    a = _make(T, D, 16, _widths(T, 1, dtype, "swiglu", D, O), O, "swiglu", dtype, bias=True)
    a["router_b"][11] += 100.0
    assert _plan(a, 1, "swiglu")["path"] == "tensor"
    _, ids, _ = _check(a, 1, "swiglu", "softmax")
    assert (ids == 11).all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 5, 40])
def test_no_expert_left_on_the_tensor_cores(T, dtype):
    """No token has an expert: residual or zeros, and nothing of the experts is read."""
    D, O, E, k = 512, 136, 8, 2
    a = _make(T, D, E, _widths(T, k, dtype, "gelu", D, O), O, "gelu", dtype, bias=True)
    assert _plan(a, k, "gelu")["path"] == "tensor"
    for n in ("w1", "w2", "b1", "b2"):
        a[n].fill_(float("nan"))
    r = torch.randn(T, O, device=DEV).to(dtype)
    blocked = torch.ones(T, E, dtype=torch.bool, device=DEV)
    out, ids, gates = _moe(**a, top_k=k, act="gelu", gate_mode="softmax", block_mask=blocked, residual=r)
    assert torch.equal(out, r) and (ids == -1).all() and (gates == 0).all()
    out, _, _ = _moe(**a, top_k=k, act="gelu", gate_mode="softmax", block_mask=blocked)
    assert (out == 0).all()
    # one token of them has one
    if T > 1:
        blocked[T - 1, 5] = False
        for n in ("w1", "w2", "b1", "b2"):
            a[n][5] = _make(1, D, 1, a["w2"].shape[2], O, "gelu", dtype, bias=True, seed=9)[n][0]
        clean = {n: v.nan_to_num(0.0) if n in ("w1", "w2", "b1", "b2") else v for n, v in a.items()}
        want, wid, _ = _check(clean, k, "gelu", "softmax", block_mask=blocked, residual=r)
        out, ids, _ = _moe(**a, top_k=k, act="gelu", gate_mode="softmax", block_mask=blocked, residual=r)
        assert torch.equal(out, want) and torch.equal(ids, wid) and torch.equal(out[:-1], r[:-1])


@pytest.mark.parametrize("dtype,offset,pad", [(BF16, 0, 8), (BF16, 8, 24), (FP32, 0, 8), (FP32, 8, 24), (FP32, 4, 0)])
def test_windows_on_the_tensor_cores(dtype, offset, pad):
    """Every tensor as a window of a wider buffer whose rows start on 16 bytes (out and residual: anywhere)."""
    T, E, D, O = 5, 6, 512, 72
    F = _widths(T, 2, dtype, "swiglu", D, O)
    g = torch.Generator(DEV).manual_seed(2)

    def window(*shape, s=1.0):
        return _window(*shape, dtype=dtype, gen=g, scale=s, offset=offset, pad=pad)

    a = dict(x=window(T, D), router_w=window(E, D, s=D ** -0.5), w1=window(2 * E, 2 * F, D, s=D ** -0.5)[::2],
             w2=window(2 * E, O, F, s=F ** -0.5)[1::2])
    assert _plan(a, 2, "swiglu")["path"] == "tensor"
    ob = torch.full((T + 2, O + 9), 7.0, device=DEV, dtype=dtype)
    _check(a, 2, "swiglu", "topk_softmax", residual=_window(T, O, dtype=dtype, gen=g), out=ob[1:T + 1, 5:5 + O])
    ob[1:T + 1, 5:5 + O] = 7.0
    assert torch.equal(ob, torch.full_like(ob, 7.0))


@pytest.mark.parametrize("T,D,E,k,act", [(64, 1088, 4, 1, "swiglu"), (64, 2048, 8, 2, "gelu"), (17, 2500, 4, 2, "swiglu"),
                                         (33, 1440, 6, 3, "silu"), (49, 4096, 3, 2, "swiglu"), (64, 5000, 2, 2, "relu"),
                                         (64, 4096, 4, 2, "swiglu")])
def test_wide_fp32_layers(T, D, E, k, act):
    """fp32 layers so wide that product 1 is a long sum: masks that differ by token, tokens without an expert, biases, a residual
    in place, an out that is a window."""
    O = 264
    a = _make(T, D, E, _widths(T, k, FP32, act, D, O), O, act, FP32, seed=T + D, bias=True)
    assert _plan(a, k, act)["path"] == "tensor"
    g = torch.Generator(DEV).manual_seed(D)
    mask = torch.rand(T, E, generator=g, device=DEV) < 0.3
    mask[0] = mask[T // 2] = mask[T - 1] = True
    _check(a, k, act, "topk_softmax", block_mask=mask)
    ob = torch.full((T + 2, O + 9), 7.0, device=DEV)
    r = torch.randn(T, O, generator=g, device=DEV)
    out = ob[1:T + 1, 5:5 + O]
    out.copy_(r)
    want, wid, wgates = _check(a, k, act, "softmax", block_mask=mask, residual=r)
    got, ids, gates = _moe(**a, top_k=k, act=act, gate_mode="softmax", block_mask=mask, residual=out, out=out)
    assert torch.equal(got, want) and torch.equal(ids, wid) and torch.equal(gates, wgates)
    assert torch.equal(out[0], r[0]) and torch.equal(out[T - 1], r[T - 1])
    out.fill_(7.0)
    assert torch.equal(ob, torch.full_like(ob, 7.0))
    # Errors of random sign: two products made of parts, the additions of two sums, and what the tensor core cuts in a chain
    # of at most 384 of D (48 instructions).
    want, _, _, _, _, _ = moe64(**a, top_k=k, act=act, gate_mode="none", block_mask=mask)
    got, _, _ = _moe(**a, top_k=k, act=act, gate_mode="none", block_mask=mask)
    check_norm(got, want, 4 * PARTS + U * (D ** 0.5 + a["w2"].shape[2] ** 0.5 + 16 + 48))


# ---------------------------------------------------------------------------- both

def test_writing_to_out_is_seen_by_autograd():
    """A tensor that an operation saved for its backward pass, then given as out: that pass has to fail, not use what was written."""
    x, w, _, _ = _make_linear(3, 64, 32, "none", FP32, False, False)
    a = _make(3, 64, 4, 32, 32, "relu", FP32)
    for write in (lambda out: _linear(x, w, out=out), lambda out: _moe(**a, top_k=2, act="relu", out=out)):
        scale = torch.ones(3, 32, device=DEV, requires_grad=True)
        saved = torch.randn(3, 32, device=DEV)
        before = saved._version
        (scale * saved).sum().backward()
        y = (scale * saved).sum()
        write(saved)
        assert saved._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with torch.inference_mode():
            out = torch.empty(3, 32, device=DEV)
            write(out)
        write(out)   # an inference tensor has no counter


def test_a_record_is_raised_once_and_leaves_other_calls_alone():
    """The record of a wait that ran out, written here by the host: the next check raises it with its fields, the one after
    passes, and calls made while it stands, with long waits in them, give the same bits as before."""
    from revealaiccl_b200.ops import status
    from revealaiccl_b200.ops._native import kernels
    from revealaiccl_b200.parallel.peer import device_view

    index = torch.cuda.current_device()
    record = device_view(kernels().serving_status_address(index), (status.STATUS_WORDS,), torch.int32, torch.device(DEV, index))
    fields = torch.tensor([1, 620, 17, 33, 5, 0, 2_000_000_000, 0], dtype=torch.int32, device=DEV)
    calls = []
    for m, k, n, act, dtype in ((64, 14336, 4096, "swiglu", BF16), (2048, 8192, 4096, "none", BF16), (64, 8192, 2048, "none", FP32),
                                (1024, 4096, 4096, "gelu", FP32)):
        x, w, b, r = _make_linear(m, k, n, act, dtype, True, True)
        calls.append(lambda x=x, w=w, b=b, r=r, act=act, **kw: _linear(x, w, b, act=act, residual=r, **kw))
    for dtype in (BF16, FP32):
        a = _make(40, 1024, 8, 6000, 1024, "swiglu", dtype)
        assert _plan(a, 2, "swiglu")["path"] == "tensor"
        calls.append(lambda a=a, **kw: _moe(**a, top_k=2, **kw)[0])
    want = [c() for c in calls]
    status.check_serving()
    for c, v in zip(calls, want):
        record.copy_(fields)
        assert torch.equal(c(), v)
        with pytest.raises(status.DeviceStatusError, match="pipeline mbarrier wait timed out") as e:
            c(check=True)
        assert e.value.record == {"code": 1, "kernel_id": 620, "block": 17, "thread": 33, "index": 5, "bound": 2_000_000_000}
        assert torch.equal(c(check=True), v) and (record == 0).all()
        record.copy_(fields)
        with pytest.raises(status.DeviceStatusError):
            status.check_serving(index)
        status.check_serving()


@pytest.mark.parametrize("T,k,E,act", [(1, 4, 16, "swiglu"), (9, 2, 8, "gelu"), (30, 1, 2, "silu"), (64, 2, 4, "swiglu"), (64, 1, 1, "relu")])
@pytest.mark.parametrize("tensor", [False, True], ids=["rows", "tensor"])
def test_bf16_activations_keep_their_bits(T, k, E, act, tensor):
    """A bf16 layer with an fp32 result: the activations between the products are not rounded to bf16, however the call runs.
    Two bf16 parts hold one to 2^-16.  The tensor core cuts what it adds, 2^-23 at most for each 16 of D and, with both parts,
    for each 8 of F."""
    D, O = 512, 384
    F = _widths(T, k, BF16, act, D, O) if tensor else 48
    a = _make(T, D, E, F, O, act, BF16, seed=T)
    assert _plan(a, k, act)["path"] == ("tensor" if tensor else "rows")
    out, _, _ = _check(a, k, act, "none", out_dtype=FP32)
    want = moe64(**a, top_k=k, act=act, gate_mode="none", out_dtype=FP32)[0]
    check_norm(out, want, 2.0 ** -16 + 2 * U * (D / 16 + F / 8 + 16))


def test_largest_bf16_activations():
    """Activations that bf16 cannot round without an infinity, and infinite ones, which stay with their token."""
    T, D, E, k, O = 8, 512, 4, 1, 256
    a = _make(T, D, E, _widths(T, k, BF16, "relu", D, O), O, "relu", BF16, seed=3)
    a["x"] = torch.zeros_like(a["x"])
    a["x"][:, 3] = 1.0 + 2.0 ** -6
    a["router_w"].zero_()
    a["w1"] = a["w1"].sign() * 3.35e38          # in bf16, times 1 + 2^-6: 3.402e38, between the largest numbers of bf16 and fp32
    a["b1"] = torch.zeros(E, a["w1"].shape[1], device=DEV)
    top = float(a["w1"].abs().max()) * (1 + 2.0 ** -6)
    assert torch.finfo(BF16).max < top < torch.finfo(FP32).max
    a["w2"] *= 2.0 ** -100
    assert _plan(a, k, "relu")["path"] == "tensor"
    out, _, _ = _moe(**a, top_k=k, act="relu", gate_mode="none", out_dtype=FP32)
    want, bound = moe64(**a, top_k=k, act="relu", gate_mode="none", out_dtype=FP32)[:2]
    check_close(out, want, bound)
    base = out
    a["x"][5, 3] = 2.0
    out, _, _ = _moe(**a, top_k=k, act="relu", gate_mode="none", out_dtype=FP32)
    keep = [i for i in range(T) if i != 5]
    assert torch.equal(out[keep], base[keep]) and not out[5].isfinite().any()


@pytest.mark.parametrize("m,k,n,act,kernel", [
    (1, 14336, 256, "none", "vector"), (20, 8192, 512, "none", "rows"), (40, 14336, 12288, "none", "rows"), (64, 8192, 9000, "swiglu", "rows"),
    (10, 520, 100, "none", "rows"), (300, 8192, 1032, "gelu", "rows"), (1100, 4104, 4096, "none", "dense"), (1100, 8192, 2600, "swiglu", "dense"),
    (2100, 8192, 1200, "none", "dense"), (700, 1000, 2049, "none", "rows"),
])
def test_bf16_products_to_fp32(m, k, n, act, kernel):
    """Exact products and 32-bit sums, over any K: errors of random sign, and the cuts of the tensor core in one chain of 512
    (32 instructions; dense tiles 64); a whole K of 8192 without chains would be 1.6e-5 off."""
    x, w, b, _ = _make_linear(m, k, n, act, BF16, True, False, seed=8)
    plan = _linear_plan(x, w, act, out_dtype=FP32)
    assert plan["kernel"] == kernel and plan["chained"] == (kernel != "vector")
    got = _linear(x, w, b, act=act, out_dtype=FP32)
    want, bound = linear64(x, w, b, act, None, FP32)
    check_close(got, want, bound)
    check_norm(got, want, (2 if act == "swiglu" else 1) * U * (k ** 0.5 / 2 + 8 + (64 if kernel == "dense" else 32)))


FIRST_IN_A_CAPTURE = """
import torch
from revealaiccl_b200.ops.linear import linear
from revealaiccl_b200.ops.moe_few import moe_few_tokens

def make(*shape, dtype):
    return (torch.randn(*shape, device="cuda") * 0.1).to(dtype)

for dtype in (torch.bfloat16, torch.float32):
    w, big = make(512, 256, dtype=dtype), make(2048, 1024, dtype=dtype)
    layer = dict(router_w=make(8, 256, dtype=dtype), w1=make(8, 20000, 256, dtype=dtype), w2=make(8, 256, 10000, dtype=dtype))
    small = dict(router_w=make(8, 256, dtype=dtype), w1=make(8, 64, 256, dtype=dtype), w2=make(8, 256, 32, dtype=dtype))
    x1, x20, x999, odd = (make(m, k, dtype=dtype) for m, k in ((1, 256), (20, 256), (999, 1024), (20, 257)))
    calls = (lambda: linear(x1, w), lambda: linear(x20, w, act="swiglu"), lambda: linear(x999, big), lambda: linear(odd[:, 1:], w),
             lambda: moe_few_tokens(x1, **small, top_k=2)[0], lambda: moe_few_tokens(x20, **small, top_k=2)[0],
             lambda: moe_few_tokens(x20, **layer, top_k=2)[0])
    for call in calls:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graph.replay()
        assert torch.equal(out, call())
print("all captured")
"""


def test_first_calls_inside_captures():
    """A process whose first call of each kernel is captured: nothing that a first call sets up breaks the capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "all captured" in p.stdout, p.stderr[-2000:]


@pytest.mark.parametrize("T,D,E,k,F,act", [(22, 1024, 16, 4, 5888, "swiglu"), (23, 1046, 24, 5, 4672, "swiglu"), (5, 1792, 8, 4, 8000, "swiglu"),
                                           (16, 2048, 8, 2, 4096, "gelu"), (40, 1440, 8, 3, 2500, "swiglu"), (64, 1120, 6, 2, 4000, "silu"),
                                           (64, 4096, 3, 2, 1500, "swiglu"), (12, 640, 2, 1, 9000, "swiglu"), (1, 4960, 8, 8, 2000, "swiglu")])
def test_fp32_layers_have_fp32_sums(T, D, E, k, F, act):
    """The tensor core cuts its sums, 2e-6 of them for each 1024 of K, which one chain of K may not show: no chain of either
    product is longer than 160.  SwiGLU multiplies two of them.  Beside that, numbers in parts are 2^-22 off, and a few dozen
    sums of chains, tokens and choices are rounded."""
    a = _make(T, D, E, F, D, act, FP32, seed=D)
    assert _plan(a, k, act)["path"] == ("rows" if k * T * 4 * F * (D + (2 if act == "swiglu" else 1) * D) <= 540e6 else "tensor")
    out, _, _ = _check(a, k, act, "none")
    want = moe64(**a, top_k=k, act=act, gate_mode="none")[0]
    once = 2.1 if act == "swiglu" else 1.1
    check_norm(out, want, 2e-6 / 1024 * 160 * (once + 1) + 2.0 ** -22 * (once + 1) + 8 * U)
