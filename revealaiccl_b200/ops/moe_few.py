"""A whole mixture-of-experts layer for a few tokens (csrc/kernels/moe_few.cu).

``ProgressiveMoELayer`` serves batches of thousands of tokens, revealed chunk
by chunk; ``moe_few_tokens`` is the same layer for a decode step of 1 to 64
tokens on one GPU, where reading the chosen experts' weights is all the time
there is.  Same routing contract (larger logit first, then the smaller expert;
NaN behind every number), gates and experts as the layer
(rlccl/transport/reference_router.py:15-25, reference_full_moe.py:249-300).
"""

from __future__ import annotations

import torch

from . import status as _status
from ._native import kernels
from .grouped_gemm import ACT_IDS

GATE_IDS = {"none": 0, "topk_softmax": 1, "softmax": 2}
MAX_TOKENS = 64
MAX_EXPERTS = 255
MAX_TOP_K = 8


def moe_few_tokens(
    x: torch.Tensor,
    router_w: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    *,
    top_k: int,
    act: str = "swiglu",
    gate_mode: str = "topk_softmax",
    router_b: torch.Tensor | None = None,
    b1: torch.Tensor | None = None,
    b2: torch.Tensor | None = None,
    block_mask: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    check: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """out[t] = sum_j gate[t, j] * (w2[e] @ act(w1[e] @ x[t] + b1[e]) + b2[e]) + residual[t], e = ids[t, j].

    x [T, D] (T <= 64), router_w [E, D], w1 [E, F, D] ([E, 2F, D], gate rows
    then up rows, for ``act="swiglu"``), w2 [E, O, F]: all bf16 or all fp32,
    rows contiguous, any other strides.  router_b [E], b1, b2: fp32.
    block_mask: bool or uint8 [E] or [T, E], true where an expert may not be
    chosen; a logit of -inf counts as blocked.  A choice that no expert is left
    for has id -1 and gate 0, and a token without any expert gets its residual
    (or zeros).  residual [T, O]: fp32 or bf16; ``out`` may be the same tensor,
    but its range of memory may not overlap another input's.

    Sums are kept in fp32, and the hidden activations in fp32 or as two bf16
    numbers (2^-16), whatever the size of the call; the result is rounded once.
    A result that is infinite may come out as NaN, and fp32 numbers below 2^-113
    are taken to 2^-137 of absolute error only.  bf16 layers leave the tensor
    core's own sums over D, which drift by up to 2e-6 of the activation for each
    1024 of it.
    Returns (out [T, O] in out_dtype or x's type, expert ids int32 [T, top_k],
    gates fp32 [T, top_k]).

    Enqueues two or three launches (wide fp32 layers: for each 16 or 32 tokens)
    on the current stream without synchronising and can be captured in a CUDA
    graph.  Outputs and workspace come from torch's allocator on that stream;
    the workspace is up to T (SMs + 2 top_k) rows of O fp32 numbers, 172 MB for
    64 tokens at an O of 4096 and top_k 8.  Expert rows that do not start on 16
    bytes are read element by element or, where many tokens share few experts,
    copied first, which takes as much memory as all experts.  ``check=True``
    waits and raises on a recorded device status.  There is no backward: tensors
    that require a gradient or carry a tangent are refused.
    """
    if act not in ACT_IDS:
        raise ValueError(f"moe_few_tokens: act must be one of {sorted(ACT_IDS)}")
    if gate_mode not in GATE_IDS:
        raise ValueError(f"moe_few_tokens: gate_mode must be one of {sorted(GATE_IDS)}")
    res = kernels().moe_few_tokens(x, router_w, w1, w2, top_k, ACT_IDS[act], GATE_IDS[gate_mode], router_b, b1, b2,
                                   block_mask, residual, out, out_dtype)
    if check:
        _status.check_serving(x.device)
    return res


__all__ = ["GATE_IDS", "MAX_EXPERTS", "MAX_TOKENS", "MAX_TOP_K", "moe_few_tokens"]
