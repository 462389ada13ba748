"""linear(): dense product with bias, activation and residual, against 64 bits."""

import pytest
import torch

from serving_reference import HALF, PARTS, U, check_close, check_norm, linear64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def _linear(*a, **k):
    from revealaiccl_b200.ops.linear import linear
    return linear(*a, **k)


def _make(m, k, n, act, dtype, bias, residual, seed=0, res_dtype=None):
    g = torch.Generator(DEV).manual_seed(seed)
    rows = 2 * n if act == "swiglu" else n
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype)
    w = (torch.randn(rows, k, generator=g, device=DEV) / max(k, 1) ** 0.5).to(dtype)
    b = torch.randn(rows, generator=g, device=DEV) * 0.1 if bias else None
    r = torch.randn(m, n, generator=g, device=DEV).to(res_dtype or dtype) if residual else None
    return x, w, b, r


def _norm_bound(k, dtype, out_dtype):
    # the result's rounding, and errors of random sign in k additions
    return HALF[out_dtype] + U * (k ** 0.5 + 8) + (PARTS if dtype == FP32 else 0.0)


SIZES = [  # rows, K, N (the result's width)
    (1, 1, 1), (1, 64, 128), (1, 4096, 512), (2, 8, 16), (3, 100, 7), (5, 2048, 33), (7, 65, 129), (8, 128, 64),
    (15, 200, 250), (16, 256, 384), (17, 1000, 130), (31, 72, 1000), (33, 520, 257), (48, 2048, 704), (64, 1408, 640),
    (65, 320, 200), (100, 96, 100), (127, 513, 65), (128, 1024, 256), (129, 1408, 300), (200, 4096, 96), (255, 33, 255),
    (256, 512, 512), (257, 640, 520), (512, 64, 2048), (777, 1408, 392), (1000, 1000, 1000), (2048, 256, 1024),
    (4097, 136, 264),
]


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(m, k, n, dtype):
    act = ("none", "swiglu", "gelu", "silu", "relu")[(m + k + n) % 5]
    x, w, b, r = _make(m, k, n, act, dtype, (m + n) % 2 == 0, (m + k) % 2 == 0, seed=m)
    got = _linear(x, w, b, act=act, residual=r)
    want, bound = linear64(x, w, b, act, r)
    assert got.dtype == dtype
    check_close(got, want, bound)
    if m * n >= 256:
        check_norm(got, want, 2 * _norm_bound(k, dtype, dtype))


FEW = [  # on both sides of where very few rows go to CUDA cores: many weights, and odd widths
    (1, 4096, 4104), (1, 2048, 9000), (2, 4096, 2048), (3, 1000, 3001), (4, 1024, 2048), (5, 2048, 520), (6, 264, 4096),
    (7, 1408, 1000), (8, 2048, 2048), (8, 4097, 129), (9, 1024, 512),
]


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("m,k,n", FEW)
def test_few_rows(m, k, n, act, dtype):
    x, w, b, r = _make(m, k, n, act, dtype, True, n % 2 == 0, seed=n)
    got = _linear(x, w, b, act=act, residual=r)
    want, bound = linear64(x, w, b, act, r)
    check_close(got, want, bound)
    check_norm(got, want, 2 * _norm_bound(k, dtype, dtype))


@pytest.mark.parametrize("m", [1, 4, 40, 130, 600])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "swiglu"])
@pytest.mark.parametrize("dtype,out_dtype,res_dtype", [(BF16, BF16, FP32), (BF16, FP32, BF16), (BF16, FP32, FP32),
                                                       (FP32, FP32, BF16), (FP32, FP32, FP32)])
def test_types_and_epilogues(m, act, dtype, out_dtype, res_dtype):
    x, w, b, r = _make(m, 384, 272, act, dtype, True, True, seed=m, res_dtype=res_dtype)
    got = _linear(x, w, b, act=act, residual=r, out_dtype=out_dtype)
    want, bound = linear64(x, w, b, act, r, out_dtype)
    assert got.dtype == out_dtype
    check_close(got, want, bound)


@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_fp32_results_are_not_tf32(m, dtype):
    """Exact products, 32-bit sums: a tf32 product of fp32 inputs would be 1e-4 off."""
    x, w, _, _ = _make(m, 1024, 512, "none", dtype, False, False)
    got = _linear(x, w, out_dtype=FP32)
    want, _ = linear64(x, w, out_dtype=FP32)
    check_norm(got, want, U * (1024 ** 0.5 + 8) + PARTS)


@pytest.mark.parametrize("m,n,k", [(64, 12288, 4096), (1, 256, 14336), (20, 512, 8192), (300, 1024, 8192), (1100, 4096, 4096)])
def test_long_sums(m, n, k):
    """Chains of thousands of products, over several waves of tiles: the error of fp32 sums grows with the root of K."""
    x, w, _, _ = _make(m, k, n, "none", FP32, False, False)
    got = _linear(x, w)
    want, bound = linear64(x, w)
    check_close(got, want, bound)
    check_norm(got, want, U * (k ** 0.5 / 2 + 8) + PARTS)


@pytest.mark.parametrize("m", [1, 37, 300])
@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 0), (4, 3), (8, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_strides_and_alignment(m, offset, pad, dtype):
    """x, weight and residual as windows of wider buffers at any offset; what lies around out stays."""
    k, n = 264, 136
    g = torch.Generator(DEV).manual_seed(m)
    xb = torch.randn(m, k + offset + pad, generator=g, device=DEV).to(dtype)
    wb = torch.randn(n, k + offset + pad, generator=g, device=DEV).to(dtype)
    rb = torch.randn(m, n + offset + pad, generator=g, device=DEV).to(dtype)
    ob = torch.full((m + 2, n + offset + pad), 7.0, device=DEV, dtype=dtype)
    x, w = xb[:, offset:offset + k], wb[:, offset:offset + k] / k ** 0.5
    w = wb[:, offset:offset + k]
    r, out = rb[:, offset:offset + n], ob[1:m + 1, offset:offset + n]
    got = _linear(x, w, residual=r, out=out)
    assert got.data_ptr() == out.data_ptr()
    want, bound = linear64(x, w, residual=r)
    check_close(out, want, bound)
    ob[1:m + 1, offset:offset + n] = 7.0
    assert torch.equal(ob, torch.full_like(ob, 7.0))


def test_broadcast_rows():
    x = torch.randn(1, 320, device=DEV, dtype=BF16).expand(20, 320)
    w = torch.randn(96, 320, device=DEV, dtype=BF16)
    want, bound = linear64(x, w)
    check_close(_linear(x, w), want, bound)


@pytest.mark.parametrize("m", [1, 50, 400])
def test_in_place_residual(m):
    x, w, b, r = _make(m, 256, 320, "none", BF16, True, True)
    want = _linear(x, w, b, residual=r)
    out = r.clone()
    got = _linear(x, w, b, residual=out, out=out)
    assert torch.equal(got, want)


def test_empty():
    w = torch.randn(8, 16, device=DEV, dtype=BF16)
    assert _linear(torch.empty(0, 16, device=DEV, dtype=BF16), w).shape == (0, 8)
    assert _linear(torch.randn(3, 16, device=DEV, dtype=BF16), w[:0]).shape == (3, 0)
    b, r = torch.randn(8, device=DEV), torch.randn(3, 8, device=DEV)
    got = _linear(torch.empty(3, 0, device=DEV), torch.empty(8, 0, device=DEV), b, act="relu", residual=r)
    assert torch.equal(got, b.clamp_min(0) + r)
    r = torch.randn(20, 8, device=DEV)
    got = _linear(torch.empty(20, 0, device=DEV, dtype=BF16), torch.empty(8, 0, device=DEV, dtype=BF16), b, residual=r, out_dtype=FP32)
    assert torch.equal(got, b + r)


@pytest.mark.parametrize("m", [4, 200])
def test_special_values_stay_in_their_row(m):
    x, w, b, _ = _make(m, 128, 96, "relu", BF16, True, False)
    x[1, 5], x[2, 7], x[3, 0] = float("nan"), float("inf"), 3e38
    got = _linear(x, w, b, act="relu")
    assert got[1].isnan().all()
    keep = [i for i in range(m) if i not in (1, 2, 3)]
    clean = x.clone()
    clean[1:4] = 0
    assert torch.equal(got[keep], _linear(clean, w, b, act="relu")[keep])
    assert not got[2].isfinite().all()


def test_long_rows():
    """Element offsets past 32 bits: the last rows of a result of 2^31 elements and more."""
    m, k, n = 70000, 16, 31000
    x = torch.randn(m, k, device=DEV, dtype=BF16)
    w = torch.randn(n, k, device=DEV, dtype=BF16)
    got = _linear(x, w)
    for rows in (slice(0, 3), slice(m // 2, m // 2 + 3), slice(m - 3, m)):
        want, bound = linear64(x[rows], w)
        check_close(got[rows], want, bound)


def test_repeats_and_streams():
    """The same bits every time, on side streams too and while another call runs."""
    cases = [_make(m, 2048, n, act, BF16, True, True, seed=m) for m, n, act in ((3, 512, "none"), (48, 704, "swiglu"),
                                                                                (300, 520, "gelu"))]
    acts = ("none", "swiglu", "gelu")
    want = [_linear(x, w, b, act=a, residual=r) for (x, w, b, r), a in zip(cases, acts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(20):
        for (x, w, b, r), a, s in zip(cases, acts, streams):
            with torch.cuda.stream(s):
                got.append(_linear(x, w, b, act=a, residual=r))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % len(want)])


@pytest.mark.parametrize("m,k", [(2, 512), (2, 515), (300, 512), (300, 515)])
def test_graph_replay(m, k):
    x, w, b, r = _make(m, k, 384, "silu", BF16, True, True)
    _linear(x, w, b, act="silu", residual=r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _linear(x, w, b, act="silu", residual=r)
    for seed in (1, 2):
        x2, w2, _, r2 = _make(m, k, 384, "silu", BF16, True, True, seed=seed)
        x.copy_(x2), w.copy_(w2), r.copy_(r2)
        graph.replay()
        assert torch.equal(out, _linear(x, w, b, act="silu", residual=r))


def test_check_reads_and_clears_the_status():
    from revealaiccl_b200.ops import status
    x, w, b, r = _make(3, 256, 64, "silu", BF16, True, True)
    assert torch.equal(_linear(x, w, b, act="silu", residual=r, check=True), _linear(x, w, b, act="silu", residual=r))
    status.check_serving()
    status.check_serving(x.device)


LARGEST = torch.finfo(FP32).max


@pytest.mark.parametrize("m", [4, 20, 300])
def test_largest_numbers(m):
    """Finite fp32 numbers up to the type's largest, in x and in the weights: the products are at most half as large."""
    k, n = 100, 96
    top = torch.tensor([LARGEST, -LARGEST, 3.4020e38, -3.4020e38, 3.4019e38, 3.3e38, 1e38], device=DEV)
    i = torch.arange(m, device=DEV)
    x = torch.zeros(m, k, device=DEV)
    x[i, i % k] = top[i % len(top)]
    w = torch.tensor([0.5, -0.5, 2.0 ** -30, 1 / 3, -0.3], device=DEV)[torch.arange(n * k, device=DEV) % 5].view(n, k)
    want, bound = linear64(x, w)
    check_close(_linear(x, w), want, bound)
    x = torch.tensor([0.5, -0.25, 0.3], device=DEV)[torch.arange(m, device=DEV) % 3][:, None] * (torch.arange(k, device=DEV) == 7)
    w = top[torch.arange(n * k, device=DEV) % len(top)].view(n, k)
    want, bound = linear64(x, w)
    check_close(_linear(x, w), want, bound)
