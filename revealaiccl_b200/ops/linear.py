"""Dense product with bias, activation and residual in its epilogue (csrc/kernels/linear.cu).

The projections next to the experts (a shared expert, an attention output):
``grouped_gemm`` multiplies row segments by per-expert weights and needs its
segments on the device; ``linear`` is one weight for all rows, any sizes, from
one decode row to a prefill batch.
"""

from __future__ import annotations

import torch

from . import status as _status
from ._native import kernels
from .grouped_gemm import ACT_IDS


def linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    act: str = "none",
    residual: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    check: bool = False,
) -> torch.Tensor:
    """act(x @ weight.T + bias) + residual.

    x [M, K], weight [N, K]: both bf16 or both fp32, rows contiguous, any row
    stride.  ``act="swiglu"``: weight holds N/2 gate rows, then N/2 up rows,
    and the result, silu(gate) * up, is [M, N/2].  bias: fp32 [N].  residual:
    fp32 or bf16 of the result's shape; ``out`` may be the same tensor, but its
    range of memory may not overlap another input's.

    Sums are kept in fp32 and rounded once, to out_dtype (default: x's type;
    fp32 inputs give fp32).  fp32 inputs are multiplied to fp32 accuracy, not
    to tf32's: an infinite result may come out as NaN, and numbers below 2^-113
    are taken to 2^-137 of absolute error only.

    Enqueues on the current stream without synchronising and can be captured in
    a CUDA graph.  Rows of x or weight that do not start on 16 bytes are copied
    first (not for up to 4 rows of x, 8 in fp32), which costs up to twice the
    product's own reads.  Workspace, of torch's allocator: those copies, and for
    many fp32 rows twice the size of x and weight.  At most 2^30 rows and 2^24
    columns and weight rows; 2^21 rows when there are no columns.
    ``check=True`` waits and raises on a recorded device status.  There is no
    backward: tensors that require a gradient or carry a tangent are refused.
    """
    if act not in ACT_IDS:
        raise ValueError(f"linear: act must be one of {sorted(ACT_IDS)}")
    res = kernels().linear(x, weight, bias, ACT_IDS[act], residual, out, out_dtype)
    if check:
        _status.check_serving(x.device)
    return res


__all__ = ["linear"]
