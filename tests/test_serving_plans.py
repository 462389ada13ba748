"""Which kernels linear() and moe_few_tokens() choose, on a device of 148 SMs: a rule on shapes, types, addresses and strides
that needs no GPU (addresses of meta tensors are zero, so aligned)."""

import pytest
import torch

from revealaiccl_b200.ops import _native

if not _native.has_kernels():  # pragma: no cover
    pytest.skip("kernel library not built", allow_module_level=True)

BF16, FP32 = torch.bfloat16, torch.float32


def _few(x, w1, w2, top_k=2, act="swiglu"):
    from revealaiccl_b200.ops.grouped_gemm import ACT_IDS
    return _native.kernels().moe_few_plan(x, w1, w2, top_k, ACT_IDS[act], 148)


def _empty(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("F,path", [(96, "rows"), (8000, "tensor")])
def test_rows_that_overlap_are_no_operand_of_copies(F, path):
    """Tokens or weight rows that are one tensor expanded, or lie closer than their length, are read by address or copied."""
    E, D, O = 4, 512, 512
    w1, w2 = _empty(E, 2 * F, D), _empty(E, O, F)
    apart = _few(_empty(8, D), w1, w2)
    assert apart["path"] == path and not apart["pack_x"]
    for x in (_empty(1, D).expand(8, D), _empty(8 * D).as_strided((8, D), (64, 1))):
        p = _few(x, w1, w2)
        assert p["path"] == path and p["pack_x"] == (path == "tensor")
    assert not _few(_empty(1, D).expand(1, D), w1, w2)["pack_x"]
    # weights: by rows, element by element, or copied
    for a, b in ((_empty(E * 2 * F * D).as_strided((E, 2 * F, D), (2 * F * 64, 64, 1)), w2),
                 (w1, _empty(E * O * F).as_strided((E, O, F), (O * 16, 16, 1)))):
        p = _few(_empty(8, D), a, b)
        assert (p["path"] == "rows" and not p["vec"]) or p["pack_w"]


@pytest.mark.parametrize("stages", [2, 3, 4, 9, 12])
def test_last_fills_of_a_ring(stages):
    """What a loading thread waits for before its CTA leaves: the last fill of every stage that was filled."""
    stage, phase, fills = 0, 0, []
    for filled in range(5 * stages + 2):
        want = []
        for s, f in reversed(fills):
            if s not in [w[0] for w in want]:
                want.append((s, f))
        assert _native.kernels().serving_last_fills(stages, filled) == want
        fills.append((stage, phase))
        stage += 1
        if stage == stages:
            stage, phase = 0, phase ^ 1
