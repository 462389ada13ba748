"""What the serving operators of the framework are measured on.

Two operators:

* ``moe``: a whole mixture-of-experts layer for a few tokens (router, top-k, gates, the chosen experts' MLPs, the
  weighted sum), as one decode step of a served model calls it;
* ``linear``: a matrix product with bias, activation and residual in its epilogue, from one row to a whole batch, as a
  shared expert or any projection next to the experts calls it.

``own`` false computes them with elementary torch operations; true calls ``revealaiccl_b200.ops``.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _moe(name, tokens, hidden, experts, top_k, ffn, out_dim, act, gate_mode, dtype, *, bias=False, zipf=0.0, masked=0.0,
         residual=False):
    case = {"op": "moe", "tokens": tokens, "hidden": hidden, "experts": experts, "top_k": top_k, "ffn": ffn,
            "out_dim": out_dim, "act": act, "gate_mode": gate_mode, "dtype": dtype, "bias": bias, "zipf": zipf,
            "masked": masked, "residual": residual}
    return {"name": name, **case} if name else case


def _linear(name, rows, k, n, act, dtype, *, bias=False, residual=False, pad=0):
    case = {"op": "linear", "rows": rows, "k": k, "n": n, "act": act, "dtype": dtype, "bias": bias, "residual": residual,
            "pad": pad}
    return {"name": name, **case} if name else case


def listed():
    return [
        # the R4 layer of the framework, one token: nothing but latency
        _moe("moe_r4_1tok", 1, 2048, 4, 1, 32, 16, "relu", "none", "fp32", bias=True),
        # one decoding stream through the fine-grained layer (64 experts, six of them read)
        _moe("moe_fine_1tok", 1, 2048, 64, 6, 1408, 2048, "swiglu", "softmax", "bf16"),
        # a ragged decode batch of it, some experts blocked for some tokens and a few tokens blocked whole (padding)
        _moe("moe_fine_37tok", 37, 2048, 64, 6, 1408, 2048, "swiglu", "softmax", "bf16", masked=0.1, residual=True),
        # a small decode batch through eight wide experts
        _moe("moe_wide_8tok", 8, 4096, 8, 2, 14336, 4096, "swiglu", "topk_softmax", "bf16", residual=True),
        # the largest decode batch, most tokens on a few of sixteen experts
        _moe("moe_skewed_64tok", 64, 2048, 16, 2, 8192, 2048, "swiglu", "topk_softmax", "bf16", zipf=1.2),
        # fp32 experts with GELU
        _moe("moe_fp32_16tok", 16, 1024, 8, 2, 4096, 1024, "gelu", "topk_softmax", "fp32", bias=True),
        # one token through a square projection with its residual
        _linear("linear_1row", 1, 4096, 4096, "none", "bf16", residual=True),
        # the shared expert's gate and up projections for a decode batch
        _linear("linear_swiglu_48rows", 48, 2048, 5632, "swiglu", "bf16"),
        # a ragged prefill chunk through a down projection, read out of a wider buffer
        _linear("linear_777rows", 777, 1408, 2048, "none", "bf16", bias=True, residual=True, pad=64),
        # the largest prefill batch through the widest gate and up projections
        _linear("linear_swiglu_16384rows", 16384, 4096, 28672, "swiglu", "bf16"),
        # an fp32 batch through an expert-sized projection with GELU
        _linear("linear_fp32_4096rows", 4096, 1024, 4096, "gelu", "fp32", bias=True),
        # a few fp32 rows into an odd number of outputs
        _linear("linear_fp32_7rows", 7, 2048, 33, "relu", "fp32", bias=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _width(rng, low, high):
    """A width of low to high: mostly a multiple of 64, sometimes of 8, now and then any number."""
    v = _log_int(rng, low, high)
    step = rng.choice((64, 64, 64, 64, 64, 8, 8, 1))
    return max(low, v // step * step)


def draw(rng):
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if rng.random() < 0.5:
        experts = rng.choice((4, 8, 16, 24, 60, 64, 128))
        top_k = rng.randint(1, min(8, experts))
        hidden, act = _width(rng, 256, 4096), rng.choice(("swiglu", "swiglu", "swiglu", "gelu", "silu", "relu"))
        most = 200_000_000 // (experts * hidden)  # weights of one projection, all experts
        ffn, out_dim = _width(rng, 32, max(64, min(14336, most))), rng.choice((hidden, hidden, hidden, _width(rng, 16, hidden)))
        return _moe("", _log_int(rng, 1, 64), hidden, experts, top_k, ffn, out_dim, act,
                    rng.choice(("topk_softmax", "topk_softmax", "softmax", "none")), dtype, bias=rng.random() < 0.3,
                    zipf=rng.choice((0.0, 0.0, round(rng.uniform(0.5, 1.5), 2))), masked=rng.choice((0.0, 0.0, 0.1)),
                    residual=rng.random() < 0.5)
    rows, k = _log_int(rng, 1, 16384), _width(rng, 64, 14336)
    most = (1 << 40) // (rows * k) if dtype == "bf16" else (1 << 37) // (rows * k)
    n, act = _width(rng, 16, max(32, min(28672, most))), rng.choice(("none", "none", "relu", "gelu", "silu", "swiglu", "swiglu"))
    return _linear("", rows, k, n + n % 2 if act == "swiglu" else n, act, dtype, bias=rng.random() < 0.5,
                   residual=rng.random() < 0.5, pad=rng.choice((0, 0, 64)))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        t = torch.empty(shape, dtype=dtype, device=dev)
        return t.normal_(0.0, scale, generator=gen)

    s = dict(case)
    if case["op"] == "moe":
        T, D, E, F, O = (case[k] for k in ("tokens", "hidden", "experts", "ffn", "out_dim"))
        n1 = 2 * F if case["act"] == "swiglu" else F
        s["x"] = normal(T, D)
        s["router_w"] = normal(E, D, scale=D ** -0.5)  # logits ~ N(0, 1) for unit tokens
        s["w1"] = normal(E, n1, D, scale=D ** -0.5)
        s["w2"] = normal(E, O, F, scale=F ** -0.5)
        s["b1"] = normal(E, n1, scale=0.1, dtype=torch.float32) if case["bias"] else None
        s["b2"] = normal(E, O, scale=0.1, dtype=torch.float32) if case["bias"] else None
        s["router_b"] = normal(E, scale=0.1, dtype=torch.float32) if case["bias"] else None
        if case["zipf"]:  # an additive Zipf preference for some experts
            order = torch.randperm(E, generator=gen, device=dev)
            skew = -case["zipf"] * torch.log1p(order.float())
            s["router_b"] = skew if s["router_b"] is None else s["router_b"] + skew
        s["block_mask"] = None
        if case["masked"]:
            mask = torch.rand(T, E, generator=gen, device=dev) < case["masked"]
            s["block_mask"] = mask | (torch.rand(T, 1, generator=gen, device=dev) < case["masked"])
        s["residual"] = normal(T, O) if case["residual"] else None
    else:
        M, K, N = case["rows"], case["k"], case["n"]
        s["x"] = normal(M, K + case["pad"])[:, :K]
        s["weight"] = normal(N, K, scale=K ** -0.5)
        s["b"] = normal(N, scale=0.1, dtype=torch.float32) if case["bias"] else None
        s["residual"] = normal(M, N // 2 if case["act"] == "swiglu" else N) if case["residual"] else None
    return s


def _act(z, act):
    if act == "swiglu":
        gate, up = z.chunk(2, dim=-1)
        return gate / (1 + torch.exp(-gate)) * up
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _route(s):
    """ids [T, k] (-1: no expert left), gates [T, k], in 64 bits: which expert comes k-th lies next to a border."""
    logits = s["x"].double() @ s["router_w"].double().t()
    if s["router_b"] is not None:
        logits = logits + s["router_b"].double()
    if s["block_mask"] is not None:
        logits = logits.masked_fill(s["block_mask"], -math.inf)
    values, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, ids = values[:, :s["top_k"]], order[:, :s["top_k"]]
    none = top == -math.inf
    peak = values[:, :1].masked_fill(values[:, :1] == -math.inf, 0)  # a token without any expert: sums of zero
    if s["gate_mode"] == "topk_softmax":
        total = torch.exp(top - peak).sum(dim=-1, keepdim=True)
    else:
        total = torch.exp(values - peak).sum(dim=-1, keepdim=True)
    gates = torch.ones_like(top) if s["gate_mode"] == "none" else torch.exp(top - peak) / total
    return ids.masked_fill(none, -1).int(), gates.masked_fill(none, 0)


def _plain_moe(s):
    ids, gates = _route(s)
    gates = gates.float()
    T, k = ids.shape
    E, x = s["experts"], s["x"].float()
    chosen = ids.clamp_min(0).long()
    if T * k < E:  # few choices: each one's weights on their own
        pick = chosen.reshape(-1)
        z = torch.matmul(s["w1"][pick].float(), x.repeat_interleave(k, 0)[:, :, None])[:, :, 0]
        h = _act(z if s["b1"] is None else z + s["b1"][pick], s["act"])
        y = torch.matmul(s["w2"][pick].float(), h[:, :, None])[:, :, 0]
        y = (y if s["b2"] is None else y + s["b2"][pick]).reshape(T, k, -1)
    else:  # every expert on every token, then the chosen ones
        z = torch.matmul(x, s["w1"].float().transpose(1, 2))
        h = _act(z if s["b1"] is None else z + s["b1"][:, None], s["act"])
        y = torch.matmul(h, s["w2"].float().transpose(1, 2))
        y = y if s["b2"] is None else y + s["b2"][:, None]
        y = y[chosen, torch.arange(T, device=x.device)[:, None]]
    out = (y * gates[:, :, None]).sum(dim=1)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return {"out": out.to(s["x"].dtype), "expert_ids": ids, "gates": gates}


def _plain_linear(s):
    z = s["x"].float() @ s["weight"].float().t()
    y = _act(z if s["b"] is None else z + s["b"], s["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def run(state):
    s = state
    if own:
        if s["op"] == "moe":
            from revealaiccl_b200.ops.moe_few import moe_few_tokens

            out, ids, gates = moe_few_tokens(
                s["x"], s["router_w"], s["w1"], s["w2"], top_k=s["top_k"], act=s["act"], gate_mode=s["gate_mode"],
                router_b=s["router_b"], b1=s["b1"], b2=s["b2"], block_mask=s["block_mask"], residual=s["residual"])
            return {"out": out, "expert_ids": ids, "gates": gates}
        from revealaiccl_b200.ops.linear import linear

        return linear(s["x"], s["weight"], s["b"], act=s["act"], residual=s["residual"])
    return _plain_moe(s) if s["op"] == "moe" else _plain_linear(s)


def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    glu = 2 if case["act"] == "swiglu" else 1
    if case["op"] == "moe":
        T, D, E, k, F, O = (case[n] for n in ("tokens", "hidden", "experts", "top_k", "ffn", "out_dim"))
        # experts that some token chooses: each chosen with probability k / E by each token (without a preference)
        used = E * (1 - (1 - k / E) ** T)
        each = glu * F * D + O * F
        extra = 4 * used * (glu * F + O) + 4 * E if case["bias"] else 0
        return {"bytes": b * (used * each + E * D + T * (D + O + (O if case["residual"] else 0))) + extra + 8 * T * k
                + (T * E if case["masked"] else 0),
                "flops": 2 * T * (k * each + E * D)}
    M, K, N = case["rows"], case["k"], case["n"]
    outs = M * N // glu
    return {"bytes": b * (M * K + N * K + outs * (2 if case["residual"] else 1)) + (4 * N if case["bias"] else 0),
            "flops": 2 * M * N * K}


def _act64(z, act):
    half = z.shape[-1] // 2
    if act == "swiglu":
        return torch.sigmoid(z[..., :half]) * z[..., :half] * z[..., half:]
    return {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu": lambda v: v * torch.special.ndtr(v)}[act](z)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "linear":
        z = x @ s["weight"].double().t()
        if s["b"] is not None:
            z += s["b"]
        y = _act64(z, case["act"])
        return y if s["residual"] is None else y + s["residual"]
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    logits = torch.einsum("td,ed->te", x, s["router_w"].double())
    logits = logits if s["router_b"] is None else logits + s["router_b"]
    allowed = torch.ones(T, E, dtype=torch.bool, device=x.device) if s["block_mask"] is None else ~s["block_mask"]
    out = torch.zeros(T, case["out_dim"], dtype=torch.float64, device=x.device)
    ids = torch.full((T, k), -1, dtype=torch.int32)
    gates = torch.zeros(T, k, dtype=torch.float64)
    host, ok = logits.tolist(), allowed.tolist()
    for t in range(T):  # every token by hand: its allowed experts by falling logit, ties to the lowest index
        order = sorted((e for e in range(E) if ok[t][e]), key=lambda e: (-host[t][e], e))
        pool = order if case["gate_mode"] == "softmax" else order[:k]
        for j, e in enumerate(order[:k]):
            ids[t, j] = e
            gates[t, j] = 1.0 if case["gate_mode"] == "none" else 1.0 / sum(math.exp(host[t][o] - host[t][e]) for o in pool)
    for e in range(E):
        rows, slot = (ids == e).nonzero(as_tuple=True)
        if not len(rows):
            continue
        rows, slot = rows.to(x.device), slot.to(x.device)
        z = x[rows] @ s["w1"][e].double().t()
        z = z if s["b1"] is None else z + s["b1"][e]
        y = _act64(z, case["act"]) @ s["w2"][e].double().t()
        y = y if s["b2"] is None else y + s["b2"][e]
        out[rows] += y * gates.to(x.device)[rows, slot][:, None]
    if s["residual"] is not None:
        out += s["residual"]
    return {"out": out, "expert_ids": ids, "gates": gates}
