"""What the attention operators of the framework are measured on.

Four operators, the attention half of a served layer next to ``linear`` and ``moe_few_tokens``:

* ``prompt``: attention over whole prompts or chunks of them, packed sequences of different lengths, causal, grouped heads;
* ``decode``: attention of one new token of each sequence over a paged cache held in 4 bits;
* ``write``: new keys and values go into that cache, quantised as they are written, and are read back;
* ``read``: keys and values of earlier tokens are read back out of it, as the next chunk of a prompt needs them.

The cache holds numbers of 4 bits (e2m1: a sign and 0, 0.5, 1, 1.5, 2, 3, 4 or 6), sixteen of a head's with one scale of 8
bits (e4m3).  The scale is the sixteen's largest magnitude by 6, rounded; a number is then x by the scale, rounded; both
to nearest, ties to even, and saturating.

``own`` false computes them with elementary torch operations; true calls ``revealaiccl_b200.ops``.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 16


def _prompt(name, seqs, tokens, kv_heads, group, dim, dtype, *, past=0, causal=True, lse=False, pad=0, shape=0):
    """``tokens`` new tokens over all sequences; ``past``: earlier tokens over all sequences, which come first in k and v."""
    case = {"op": "prompt", "seqs": seqs, "tokens": tokens, "kv_heads": kv_heads, "group": group, "dim": dim, "dtype": dtype,
            "past": past, "causal": causal, "lse": lse, "pad": pad, "shape": shape}
    return {"name": name, **case} if name else case


def _decode(name, seqs, longest, kv_heads, group, dim, page, dtype, *, ragged=True, empty=False, lse=False, pad=0, shape=0):
    case = {"op": "decode", "seqs": seqs, "longest": longest, "kv_heads": kv_heads, "group": group, "dim": dim, "page": page,
            "dtype": dtype, "ragged": ragged, "empty": empty, "lse": lse, "pad": pad, "shape": shape}
    return {"name": name, **case} if name else case


def _move(name, op, seqs, tokens, kv_heads, dim, page, dtype, *, padding=0, pad=0, shape=0):
    """``padding``: tokens without a place in the cache (slot -1)."""
    case = {"op": op, "seqs": seqs, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
            "padding": padding, "pad": pad, "shape": shape}
    return {"name": name, **case} if name else case


def listed():
    return [
        # a few short prompts of a chat, packed: latency counts
        _prompt("prompt_5short", 5, 300, 4, 4, 64, "bf16", shape=1),
        # chunks of eight prompts, each behind what is already in the cache (its log-sums too, to join other parts)
        _prompt("prompt_8chunks", 8, 4096, 8, 4, 128, "bf16", past=12000, lse=True, pad=128, shape=2),
        # one long document at once
        _prompt("prompt_16k", 1, 16384, 8, 4, 128, "bf16"),
        # an encoder's batch in fp32: every token sees its whole sequence, each head its own keys
        _prompt("prompt_fp32", 3, 2049, 16, 1, 64, "fp32", causal=False, shape=3),
        # one decoding stream, not far along
        _decode("decode_1x1000", 1, 1000, 8, 4, 128, 64, "bf16", ragged=False),
        # a ragged decode batch in small pages, one place of it not in use
        _decode("decode_37ragged", 37, 8192, 2, 8, 128, 16, "bf16", empty=True, lse=True, pad=256, shape=4),
        # a large batch of long contexts
        _decode("decode_64x16k", 64, 16384, 8, 4, 128, 64, "bf16", ragged=False),
        # odd head counts and lengths in fp32
        _decode("decode_fp32_7", 7, 4001, 5, 3, 64, 32, "fp32", shape=5),
        # one step's new tokens, out of the joint projection's rows
        _move("write_64tok", "write", 64, 64, 8, 128, 64, "bf16", pad=4096, padding=3, shape=6),
        # a whole prompt batch
        _move("write_16k", "write", 4, 16384, 8, 128, 64, "bf16", shape=7),
        # a short prefix in fp32
        _move("read_333", "read", 2, 333, 5, 64, 32, "fp32", shape=8),
        # the contexts in front of a batch of chunks
        _move("read_64k", "read", 16, 65536, 8, 128, 64, "bf16", padding=100, shape=9),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "decode", "decode", "write", "read"))
    dtype, dim, shape = rng.choice(("bf16", "bf16", "fp32")), rng.choice((64, 128, 128)), rng.randrange(1 << 30)
    kv_heads = rng.choice((1, 2, 3, 4, 5, 8, 8, 16))
    group, page = rng.choice((1, 2, 3, 4, 4, 5, 6, 7, 8, 12, 16)), rng.choice((16, 32, 64, 64, 128, 256))
    pad = rng.choice((0, 0, 64))
    if op == "prompt":
        heads = kv_heads * group
        flops = 2e12 if dtype == "bf16" else 1e11
        # tokens and past that cost at most so much with one sequence
        tokens = _log_int(rng, 1, max(8, min(16384, int(math.sqrt(flops / (4 * dim * heads))))))
        past = rng.choice((0, 0, _log_int(rng, 1, max(2, min(32768, int(flops / (4 * dim * heads * tokens)))))))
        return _prompt("", _log_int(rng, 1, min(64, tokens)), tokens, kv_heads, group, dim, dtype, past=past,
                       causal=rng.random() < 0.75, lse=rng.random() < 0.4, pad=pad, shape=shape)
    if op == "decode":
        seqs = _log_int(rng, 1, 128)
        most = int((1.1e9 if dtype == "bf16" else 4e8) / (seqs * kv_heads * dim * 9 / 8))
        return _decode("", seqs, _log_int(rng, 1, max(16, min(65536, most))), kv_heads, group, dim, page, dtype,
                       ragged=rng.random() < 0.7, empty=rng.random() < 0.3, lse=rng.random() < 0.4, pad=pad, shape=shape)
    tokens = _log_int(rng, 1, (16384 if op == "write" else 65536) * 8 // max(8, kv_heads) * 128 // dim // (2 if dtype == "fp32" else 1))
    return _move("", op, _log_int(rng, 1, min(64, tokens)), tokens, kv_heads, dim, page, dtype,
                 padding=rng.choice((0, min(tokens, 5))), pad=pad, shape=shape)


def _share(total, parts, rng, least=0):
    """``total`` dealt to ``parts`` unevenly, each at least ``least``."""
    weights = [rng.uniform(0.2, 1.0) ** 2 for _ in range(parts)]
    rest, scale = total - least * parts, sum(weights)
    out = [least + int(rest * w / scale) for w in weights]
    out[rng.randrange(parts)] += total - sum(out)
    return out


def _lengths(case):
    """Prompt: (new, past) of each sequence.  Decode: cached tokens of each.  Write and read: tokens of each."""
    rng = random.Random(case["shape"])
    if case["op"] == "prompt":
        new = _share(case["tokens"], case["seqs"], rng, 1)
        return new, _share(case["past"], case["seqs"], rng) if case["past"] else [0] * case["seqs"]
    if case["op"] == "decode":
        n, longest = case["seqs"], case["longest"]
        lens = [_log_int(rng, max(1, longest // 16), longest) if case["ragged"] else longest for _ in range(n)]
        lens[rng.randrange(n)] = longest
        if case["empty"] and n > 1:
            lens[lens.index(min(lens))] = 0
        return lens
    return _share(case["tokens"], case["seqs"], rng, 1)


def _quantise(x):
    """Codes uint8 [..., D] (one to a byte) and scales fp32 [..., D / 16]; by comparisons, in 64 bits."""
    x = x.double().unflatten(-1, (-1, GROUP))
    scale = (x.abs().amax(-1) / 6).clamp_max(448).to(torch.float8_e4m3fn).double()
    q = x.abs() / torch.where(scale > 0, scale, 1)[..., None]
    code = torch.zeros_like(q, dtype=torch.uint8)
    for edge in (0.25, 1.25, 2.5, 5.0):   # ties go down
        code += q > edge
    for edge in (0.75, 1.75, 3.5):        # ties go up
        code += q >= edge
    code = torch.where(scale[..., None] > 0, code, 0) + 8 * (x < 0).to(torch.uint8)
    return code.flatten(-2), scale.float()


def _pack(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def _values(codes, scales):
    """fp32 numbers of packed codes [..., D / 2] and e4m3 scales [..., D / 16]."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    one = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).long()
    return (grid[one].unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=gen)


def _rows(gen, n, heads, dim, pad, dtype, channels=None):
    """[n, heads, dim] out of rows that are ``pad`` numbers wider."""
    t = _normal(gen, n, heads * dim + pad, dtype=dtype)[:, :heads * dim].unflatten(1, (heads, dim))
    if channels is not None:
        t.mul_(channels)
    return t


def _pages(case, lens, gen):
    """A cache's tensors, filled, and the block table [seqs, most] and slots of the sequences' tokens, in order."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in lens]
    count = sum(need) + 3
    order = torch.randperm(count, generator=gen, device="cuda").int()
    most = max(1, max(need))
    table = torch.full((len(lens), most), -1, dtype=torch.int32)
    at = 0
    host = order.cpu()
    for i, n in enumerate(need):
        table[i, :n] = host[at:at + n]
        at += n
    table = table.cuda()
    c = {}
    for name in ("k", "v"):
        c[name + "_codes"] = torch.empty(count, heads, page, dim // 2, dtype=torch.uint8, device="cuda")
        c[name + "_scales"] = torch.empty(count, heads, page, dim // GROUP, dtype=torch.float8_e4m3fn, device="cuda")
        channels = torch.exp(_normal(gen, heads, 1, dim, scale=0.5)) if name == "k" else 1.0   # some channels of keys are larger
        step = max(1, (1 << 24) // (heads * page * dim))
        for i in range(0, count, step):
            n = min(step, count - i)
            code, scale = _quantise(_normal(gen, n, heads, page, dim) * channels)
            c[name + "_codes"][i:i + n], c[name + "_scales"][i:i + n] = _pack(code), scale.to(torch.float8_e4m3fn)
    return c, table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s, dt = dict(case), DTYPES[case["dtype"]]
    heads, dim, pad = case["kv_heads"], case["dim"], case["pad"]
    channels = torch.exp(_normal(gen, heads, dim, scale=0.5)).to(dt)
    if case["op"] == "prompt":
        new, past = _lengths(case)
        s["new"], s["all"] = new, [a + b for a, b in zip(new, past)]
        s["q"] = _rows(gen, sum(new), heads * case["group"], dim, pad, dt)
        s["k"] = _rows(gen, sum(s["all"]), heads, dim, pad, dt, channels)
        s["v"] = _rows(gen, sum(s["all"]), heads, dim, pad, dt)
        s["cu_q"] = torch.tensor([0] + new).cumsum(0).int().cuda()
        s["cu_k"] = torch.tensor([0] + s["all"]).cumsum(0).int().cuda()
        return s
    s["lens"] = _lengths(case)
    first = [0] * case["seqs"]
    if case["op"] != "decode":   # the tokens begin somewhere behind others
        where = random.Random(case["shape"] + 1)
        first = [where.randrange(2 * case["page"]) for _ in first]
    c, s["table"] = _pages(case, [a + n for a, n in zip(first, s["lens"])], gen)
    if own:
        from revealaiccl_b200.ops.kv_cache import KVCache4

        s["cache"] = KVCache4(**c)
    else:
        s["cache"] = c
    if case["op"] == "decode":
        s["lengths"] = torch.tensor(s["lens"], dtype=torch.int32, device="cuda")
        s["q"] = _rows(gen, case["seqs"], heads * case["group"], dim, pad, dt)
        return s
    slots, page, table = [], case["page"], s["table"].cpu()
    for i, n in enumerate(s["lens"]):
        pos = torch.arange(first[i], first[i] + n)
        slots.append(table[i].long()[pos // page] * page + pos % page)
    slots = torch.cat(slots)
    if case["padding"]:
        slots[torch.randperm(len(slots), generator=torch.Generator().manual_seed(seed))[:case["padding"]]] = -1
    s["slots"] = slots.cuda()
    if case["op"] == "write":
        s["k"] = _rows(gen, len(slots), heads, dim, pad, dt, channels)
        s["v"] = _rows(gen, len(slots), heads, dim, pad, dt)
    return s


def _attend(q, k, v, past, causal):
    """q [Tq, Hk, G, D], k and v [Tk, Hk, D], all fp32: outputs [Tq, Hk, G, D] and log-sums [Tq, Hk, G]."""
    Tq, Hk, G, D = q.shape
    out, lse = torch.empty_like(q), q.new_empty(Tq, Hk, G)
    kt, vt = k.permute(1, 2, 0), v.transpose(0, 1)           # [Hk, D, Tk], [Hk, Tk, D]
    step = max(1, (1 << 29) // (Hk * G * max(1, len(k))))
    for i in range(0, Tq, step):
        rows = q[i:i + step].permute(1, 0, 2, 3)             # [Hk, n, G, D]
        n = rows.shape[1]
        z = (rows.reshape(Hk, n * G, D) * D ** -0.5) @ kt
        if causal:
            last = torch.arange(i, i + n, device=q.device).repeat_interleave(G) + past
            z.masked_fill_(torch.arange(len(k), device=q.device)[None, :] > last[:, None], -math.inf)
        peak = z.amax(-1, keepdim=True)
        p = z.sub_(peak).exp_()
        total = p.sum(-1, keepdim=True)
        y = (p @ vt) / total
        out[i:i + n] = y.reshape(Hk, n, G, D).permute(1, 0, 2, 3)
        lse[i:i + n] = (peak + total.log())[..., 0].reshape(Hk, n, G).permute(1, 0, 2)
    return out, lse


def _plain_prompt(s):
    Hk, G = s["kv_heads"], s["group"]
    q = s["q"].float().unflatten(1, (Hk, G))
    k, v = s["k"].float(), s["v"].float()
    outs, sums, a, b = [], [], 0, 0
    for new, full in zip(s["new"], s["all"]):
        o, l = _attend(q[a:a + new], k[b:b + full], v[b:b + full], full - new, s["causal"])
        outs.append(o)
        sums.append(l)
        a, b = a + new, b + full
    return torch.cat(outs).flatten(1, 2).to(s["q"].dtype), torch.cat(sums).flatten(1, 2)


def _plain_decode(s):
    Hk, G, D, c = s["kv_heads"], s["group"], s["dim"], s["cache"]
    q = s["q"].float().unflatten(1, (Hk, G))
    out, lse = torch.zeros_like(q), torch.full(q.shape[:3], -math.inf, device=q.device)
    for i, n in enumerate(s["lens"]):
        if not n:
            continue
        pages = s["table"][i, :-(-n // s["page"])].long()
        k, v = (_values(c[x + "_codes"][pages], c[x + "_scales"][pages]).transpose(1, 2).flatten(0, 1)[:n] for x in "kv")
        out[i:i + 1], lse[i:i + 1] = _attend(q[i:i + 1], k, v, 0, False)
    return out.flatten(1, 2).to(s["q"].dtype), lse.flatten(1, 2)


def _place(s):
    used = s["slots"] >= 0
    at = s["slots"][used]
    return used, at // s["page"], at % s["page"]


def _plain_write(s):
    used, page, row = _place(s)
    for name in ("k", "v"):
        code, scale = _quantise(s[name][used])
        s["cache"][name + "_codes"][page, :, row] = _pack(code)
        s["cache"][name + "_scales"].view(torch.uint8)[page, :, row] = scale.to(torch.float8_e4m3fn).view(torch.uint8)
    return _plain_read(s)


def _plain_read(s):
    used, page, row = _place(s)
    outs = []
    for name in ("k", "v"):
        out = torch.zeros(len(used), s["kv_heads"], s["dim"], device="cuda")
        scales = s["cache"][name + "_scales"].view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn)
        out[used] = _values(s["cache"][name + "_codes"][page, :, row], scales)
        outs.append(out.to(DTYPES[s["dtype"]]))
    return tuple(outs)


def run(state):
    s = state
    if own:
        from revealaiccl_b200.ops.attention import attention_cached, attention_prompt
        from revealaiccl_b200.ops.kv_cache import kv_cache_read, kv_cache_write

        if s["op"] == "prompt":
            return attention_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"], return_lse=s["lse"])
        if s["op"] == "decode":
            return attention_cached(s["q"], s["cache"], s["table"], s["lengths"], return_lse=s["lse"])
        if s["op"] == "write":
            kv_cache_write(s["cache"], s["k"], s["v"], s["slots"])
        return kv_cache_read(s["cache"], s["slots"], dtype=DTYPES[s["dtype"]])
    if s["op"] == "write":
        return _plain_write(s)
    if s["op"] == "read":
        return _plain_read(s)
    out, lse = _plain_prompt(s) if s["op"] == "prompt" else _plain_decode(s)
    return (out, lse) if s["lse"] else out


def work(case):
    b, heads, dim, lens = (2 if case["dtype"] == "bf16" else 4), case["kv_heads"], case["dim"], _lengths(case)
    if case["op"] == "prompt":
        new, past = lens
        pairs = sum(n * p + n * (n + 1) // 2 if case["causal"] else n * (n + p) for n, p in zip(new, past))
        qs, ks = sum(new) * heads * case["group"], (sum(new) + sum(past)) * heads
        return {"bytes": b * dim * 2 * (qs + ks) + (4 * qs if case["lse"] else 0), "flops": 4 * dim * heads * case["group"] * pairs}
    row = dim // 2 + dim // GROUP    # of one head's key or value in the cache
    if case["op"] == "decode":
        qs = case["seqs"] * heads * case["group"]
        return {"bytes": sum(lens) * heads * 2 * row + b * dim * 2 * qs + (4 * qs if case["lse"] else 0),
                "flops": 4 * dim * heads * case["group"] * sum(lens)}
    n, used = case["tokens"], case["tokens"] - case["padding"]
    read = 2 * heads * (used * row + n * dim * b) + 8 * n
    # about a comparison and a product for each number that is written, and a product for each that is read
    if case["op"] == "write":
        return {"bytes": read + 2 * heads * used * (dim * b + row) + 8 * n, "flops": 6 * heads * used * dim}
    return {"bytes": read, "flops": 2 * heads * used * dim}


# --- in 64 bits, from the definition


def _exact_attention(q, k, v, visible, scale):
    """One head: q [n, D], k and v [m, D], the first visible[i] of them for row i."""
    z = torch.einsum("nd,md->nm", q, k) * scale
    z = torch.where(torch.arange(len(k), device=q.device) < visible[:, None], z, -math.inf)
    lse = torch.logsumexp(z, dim=1)
    weights = torch.exp(z - torch.where(lse > -math.inf, lse, 0)[:, None])
    return torch.einsum("nm,md->nd", weights, v), lse


def _exact_numbers(x):
    """Sixteen by sixteen: what the cache holds for x [..., D], by exponents."""
    x = x.double()
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    s = g.abs().max(dim=-1, keepdim=True).values / 6
    step = torch.exp2(torch.floor(torch.log2(s.clamp_min(2.0 ** -6))) - 3)   # e4m3: 3 bits behind the leading one, 2^-9 at least
    s = (torch.round(s / step) * step).clamp_max(448)
    a = g.abs() / torch.where(s == 0, 1, s)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(a)       # e2m1: 0.5 below 2, 1 below 4, 2 below 6
    return (torch.sign(g) * (torch.round(a / step) * step).clamp_max(6) * s).reshape(x.shape)


def _exact_cached(codes, scales):
    low, high = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    n = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    n[..., 0::2], n[..., 1::2] = low, high
    m = n % 8
    size = torch.where(m < 2, m / 2, (1 + m % 2 / 2) * torch.exp2(torch.floor(m / 2) - 1))
    return torch.where(n >= 8, -size, size) * scales.double().repeat_interleave(GROUP, dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    heads, dim = case["kv_heads"], case["dim"]
    cache = s.get("cache")
    if own and cache is not None:
        cache = {n: getattr(cache, n) for n in ("k_codes", "k_scales", "v_codes", "v_scales")}
    if case["op"] == "write":
        used = (s["slots"] >= 0)[:, None, None]
        return tuple(torch.where(used, _exact_numbers(s[n]), 0) for n in ("k", "v"))
    if case["op"] == "read":
        outs = []
        for n in ("k", "v"):
            codes, scales = (cache[f"{n}_{x}"].view(torch.uint8).transpose(1, 2).flatten(0, 1)[s["slots"].clamp_min(0)]
                             for x in ("codes", "scales"))
            outs.append(torch.where((s["slots"] >= 0)[:, None, None], _exact_cached(codes, scales.view(torch.float8_e4m3fn)), 0))
        return tuple(outs)
    G = case["group"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    a = b = 0
    for i in range(case["seqs"]):
        if case["op"] == "prompt":
            n, m = s["new"][i], s["all"][i]
            k, v = s["k"][b:b + m].double(), s["v"][b:b + m].double()
            visible = torch.arange(n, device="cuda") + (m - n + 1) if case["causal"] else torch.full((n,), m, device="cuda")
        else:
            n, m = 1, s["lens"][i]
            where = torch.arange(m, device="cuda")
            page = s["table"][i].long()[where // case["page"]]
            k, v = (_exact_cached(cache[x + "_codes"][page, :, where % case["page"]],
                                  cache[x + "_scales"].view(torch.uint8)[page, :, where % case["page"]].view(torch.float8_e4m3fn))
                    for x in "kv")
            visible = torch.tensor([m], device="cuda")
        if m:
            for h in range(heads * G):
                out[a:a + n, h], lse[a:a + n, h] = _exact_attention(s["q"][a:a + n, h].double(), k[:, h // G], v[:, h // G],
                                                                    visible, 1 / math.sqrt(dim))
        a, b = a + n, b + m
    return (out, lse) if case["lse"] else out
