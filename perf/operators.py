"""The decoder's compact serving operators, as cases that can be timed: attention over a key/value
cache held in 8 bits, the writes of that cache, and linears with 4-bit weights.

``listed`` gives fixed cases at large-v3 width (20 heads of 64, 448 text positions, 1500 encoder rows,
vocabulary 51866), ``draw`` random ones of the same ranges. With ``own`` false ``run`` is the plain
form (elementary torch operations in fp32), with ``own`` true the framework's entry points. ``exact``
is the definition in 64 bits.

The cache's definition: positions are held in blocks of 32 tokens. A block of one (slot, head) that is
complete is 8-bit codes (e4m3) with one power-of-two scale for its keys and one for its values; the
newest positions also stand as they came in a ring of 64 rows (position p in row p % 64), and the
block that is not complete yet is read from there.
"""
from __future__ import annotations

import math

import torch

own = False

D = 64
BLOCK = 32
RING = 64
E4M3_MAX = 448.0
SELF_LEN = 448
CROSS_LEN = 1500
VOCAB = 51866
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one live stream's token reads its window's 1500 encoder rows: latency, one workgroup a head is too few
        {"name": "cross_one", "kind": "cross", "dtype": "bf16", "streams": 1, "tokens": 1, "heads": 20, "length": 1500, "ragged": False},
        # the same for 52 streams, the default slot count: the largest stream of bytes of a decode step
        {"name": "cross_batch", "kind": "cross", "dtype": "fp16", "streams": 52, "tokens": 1, "heads": 20, "length": 1500, "ragged": False},
        # 16 streams verify 5-token drafts over windows of their own lengths
        {"name": "cross_verify", "kind": "cross", "dtype": "bf16", "streams": 16, "tokens": 5, "heads": 20, "length": 1500, "ragged": True},
        # 16 streams' prompts of 224 tokens: bound by the matrix cores
        {"name": "cross_prompt", "kind": "cross", "dtype": "bf16", "streams": 16, "tokens": 224, "heads": 20, "length": 1500, "ragged": False},
        # one live stream appends its token and attends: the smallest call
        {"name": "self_one", "kind": "self", "dtype": "bf16", "streams": 1, "tokens": 1, "heads": 20, "filled": 200},
        # 52 streams of ragged histories
        {"name": "self_batch", "kind": "self", "dtype": "fp16", "streams": 52, "tokens": 1, "heads": 20, "filled": 447},
        # 16 prompts of 224 tokens into empty slots, attended causally and appended
        {"name": "self_prompt", "kind": "self", "dtype": "bf16", "streams": 16, "tokens": 224, "heads": 20, "filled": 0},
        # the encoder output's keys and values of one window into the cache
        {"name": "fill_one", "kind": "fill", "dtype": "bf16", "streams": 1, "heads": 20, "length": 1500},
        # ... of 16 windows (the halves of one projection's output)
        {"name": "fill_batch", "kind": "fill", "dtype": "fp16", "streams": 16, "heads": 20, "length": 1500},
        # one stream's token through the MLP's first projection
        {"name": "linear_one", "kind": "linear", "dtype": "bf16", "rows": 1, "in": 1280, "out": 5120, "group": 64, "gelu": True},
        # 52 streams' tokens through the query, key and value projections
        {"name": "linear_batch", "kind": "linear", "dtype": "fp16", "rows": 52, "in": 1280, "out": 3840, "group": 32, "gelu": False},
        # 16 prompts of 224 tokens through the MLP's second projection: a full matrix product
        {"name": "linear_prompt", "kind": "linear", "dtype": "bf16", "rows": 3584, "in": 5120, "out": 1280, "group": 128, "gelu": False},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["cross", "self", "fill", "linear"])
    dtype = rng.choice(["bf16", "fp16"])
    heads = rng.choice([6, 8, 12, 16, 20])
    if kind == "cross":
        streams = _log(rng, 1, 52)
        return {"kind": kind, "dtype": dtype, "streams": streams, "heads": heads, "ragged": rng.random() < 0.5,
                "tokens": rng.choice([1, _log(rng, 1, 8), _log(rng, 1, min(224, 16 * 224 // streams))]),
                "length": rng.choice([CROSS_LEN, _log(rng, 1, CROSS_LEN)])}
    if kind == "self":
        streams = _log(rng, 1, 52)
        tokens = rng.choice([1, _log(rng, 1, 8), _log(rng, 1, min(224, 16 * 224 // streams))])
        return {"kind": kind, "dtype": dtype, "streams": streams, "heads": heads, "tokens": tokens,
                "filled": rng.choice([0, _log(rng, 1, SELF_LEN - tokens)])}
    if kind == "fill":
        return {"kind": kind, "dtype": dtype, "streams": _log(rng, 1, 16), "heads": heads,
                "length": rng.choice([CROSS_LEN, _log(rng, 1, CROSS_LEN)])}
    width = 64 * rng.randint(6, 20)
    n_in, n_out = rng.choice([(width, width), (width, 3 * width), (width, 4 * width), (4 * width, width),
                              (width, rng.randint(VOCAB - 2, VOCAB))])
    rows = _log(rng, 1, 64 if n_out > 5120 else 3584)
    return {"kind": kind, "dtype": dtype, "rows": rows, "in": n_in, "out": n_out,
            "group": rng.choice([g for g in (32, 64, 128) if n_in % g == 0]), "gelu": n_out == 4 * width}


# ---- inputs -----------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _perm(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _pow2(e):
    """fp32 2^e of whole e from -126 to 127 by its bits (exp2 and ldexp on the GPU may be an ulp off)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _keys(g, *shape, dtype):
    """Projected rows: a few of the 64 dimensions are much larger than the others."""
    x = torch.randn(shape, generator=g, device="cuda")
    big = 1.0 + 3.0 * (torch.rand(shape[-2:], generator=g, device="cuda") < 0.05)
    return (x * big).to(dtype)


def _random_cache(g, slots, heads, length, ring_dtype):
    """Buffers of a cache in use: codes of normal values over their range, a scale a block, a ring."""
    blocks = -(-length // BLOCK)
    st = {}
    for n in "kv":
        st[n + "_codes"] = _randn(g, slots, heads, blocks * BLOCK, D, std=110.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        st[n + "_scales"] = _pow2(torch.randint(-8, -5, (slots, heads, blocks), generator=g, device="cuda"))
        if ring_dtype is not None:
            st[n + "_ring"] = _randn(g, slots, heads, RING, D, dtype=ring_dtype)
    return st


def _linear_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    n, k, group = case["out"], case["in"], case["group"]
    return {
        "x": _randn(g, case["rows"], k, dtype=dt),
        "codes": _randn(g, n, k, std=2.6).round_().clamp_(-7, 7).to(torch.int8),
        "scales": (torch.rand(n, k // group, generator=g, device="cuda") * 0.004 + 0.012).to(dt),
        "bias": _randn(g, n, dtype=dt, std=0.1),
    }


def _fill_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    B, T, H = case["streams"], case["length"], case["heads"]
    kv = _keys(g, B, T, 2 * H, D, dtype=dt)  # one projection's output: keys, then values
    return {"k": kv[:, :, :H], "v": kv[:, :, H:], "slots": _perm(g, B + 2)[:B].contiguous(), "n_slots": B + 2}


def _cross_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    B, H, L = case["streams"], case["heads"], case["length"]
    st = _random_cache(g, B + 2, H, L, None)
    st["q"] = _randn(g, B, case["tokens"], H, D, dtype=dt)
    st["slots"] = _perm(g, B + 2)[:B].to(torch.int32)
    st["lens"] = torch.randint(-(-L // 2), L + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
    return st


def _self_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    B, H, T = case["streams"], case["heads"], case["tokens"]
    st = _random_cache(g, B + 2, H, SELF_LEN, dt)
    qkv = _keys(g, B, T, 3 * H, D, dtype=dt)  # one projection's output
    st["q"], st["k"], st["v"] = qkv[:, :, :H], qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]
    st["slots"] = _perm(g, B + 2)[:B].to(torch.int32)
    st["lens"] = torch.randint(case["filled"] // 2, case["filled"] + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    return st


_INPUTS = {"cross": _cross_inputs, "self": _self_inputs, "fill": _fill_inputs, "linear": _linear_inputs}


def prepare(case, seed):
    st = _INPUTS[case["kind"]](case, seed)
    st["kind"], st["case"] = case["kind"], dict(case)
    if case["kind"] == "fill":
        blocks = -(-case["length"] // BLOCK)
        for n in "kv":
            st[n + "_codes"] = torch.zeros(st["n_slots"], case["heads"], blocks * BLOCK, D, device="cuda").to(torch.float8_e4m3fn)
            st[n + "_scales"] = torch.ones(st["n_slots"], case["heads"], blocks, device="cuda")
    if own:  # the handles that a program keeps: the cache around its buffers, the packed weights
        import whisperdrz_amd as w

        if case["kind"] == "linear":
            st["layer"] = w.QuantLinear4.from_codes(st["codes"], st["scales"], st["bias"])
        else:
            length = SELF_LEN if case["kind"] == "self" else case["length"]
            st["cache"] = w.FlashKVCache8(int(st["k_codes"].shape[0]), length, case["heads"], D, dtype=DTYPES[case["dtype"]],
                                          ring=case["kind"] == "self", storage={n: st[n] for n in st if n[:2] in ("k_", "v_")})
    return st


def work(case):
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["in"], case["out"]
        return {"bytes": 2 * m * (k + n) + n * k // 2 + 2 * n * (k // case["group"]) + 2 * n, "flops": 2 * m * n * k}
    B, H = case["streams"], case["heads"]
    if case["kind"] == "fill":
        e = B * H * case["length"] * D
        return {"bytes": 2 * e * 3 + 2 * 4 * B * H * (-(-case["length"] // BLOCK)), "flops": 4 * e}
    T = case["tokens"]
    if case["kind"] == "cross":
        keys = 0.75 * case["length"] if case["ragged"] else case["length"]
        seen, new = keys, 0
    else:
        keys = 0.75 * case["filled"]
        seen, new = keys + (T + 1) / 2, T
    # codes and scales of the keys, the queries and outputs, the new rows read and written once
    nbytes = B * H * (2 * keys * (D + 4 / BLOCK) + 2 * 2 * T * D + 2 * new * (2 * D + D))
    return {"bytes": int(nbytes), "flops": int(4 * B * H * T * seen * D)}


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    return {"cross": _cross, "self": _self, "fill": _fill, "linear": _linear}[state["kind"]](state)


def _linear(st):
    case = st["case"]
    if own:
        import whisperdrz_amd as w

        return w.linear4(st["x"], st["layer"], gelu=case["gelu"])
    weight = (st["codes"].view(case["out"], -1, case["group"]).float() * st["scales"].float()[:, :, None]).view(case["out"], case["in"])
    y = st["x"].float() @ weight.T + st["bias"].float()
    if case["gelu"]:
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y.to(st["x"].dtype)


def _quantize(x):
    """Codes and scales of fp32 blocks [..., 32, 64]: the least power of two under which the largest
    finite value is at most 448, from 2^-100 to 2^100; what is not finite becomes NaN."""
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), torch.zeros_like(x)).amax((-2, -1))
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875)).clamp(-100, 100)
    e = torch.where(top == 0, torch.full_like(e, -100), e)
    y = (x * _pow2(-e)[..., None, None]).clamp(-E4M3_MAX, E4M3_MAX)
    y = torch.where(fine, y, torch.full_like(y, math.nan))
    return y.to(torch.float8_e4m3fn), _pow2(e)


def _dequantized(codes, scales):
    """fp32 [B, H, L, 64] of codes and their blocks' scales."""
    B, H, L, _ = codes.shape
    return (codes.float().view(B, H, -1, BLOCK, D) * scales[..., None, None]).view(B, H, L, D)


def _attend(q, k, v, limit):
    """softmax(q k / 8) v over the keys below limit[b, t]: q [B, T, H, 64], k and v fp32 [B, H, L, 64]."""
    s = (q.float().transpose(1, 2) @ k.transpose(2, 3)) * D ** -0.5
    seen = torch.arange(k.shape[2], device=q.device) < limit[:, :, None]
    s = s.masked_fill(~seen[:, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p @ v) / p.sum(-1, keepdim=True)
    return o.transpose(1, 2).to(q.dtype)


def _cross(st):
    case, lens = st["case"], st["lens"]
    if own:
        import whisperdrz_amd as w

        return w.flash_attn_with_kvcache8(st["q"], st["cache"], cache_seqlens=lens, cache_batch_idx=st["slots"])
    at = st["slots"].long()
    k, v = (_dequantized(st[n + "_codes"][at], st[n + "_scales"][at]) for n in "kv")
    B, T = case["streams"], case["tokens"]
    limit = (lens if lens is not None else torch.full((B,), case["length"], device=k.device))[:, None].expand(B, T)
    return _attend(st["q"], k, v, limit)


def _self(st):
    case = st["case"]
    if own:
        import whisperdrz_amd as w

        o = w.flash_attn_with_kvcache8(st["q"], st["cache"], st["k"], st["v"], cache_seqlens=st["lens"], cache_batch_idx=st["slots"])
    else:
        at, lens, T = st["slots"].long(), st["lens"].long(), case["tokens"]
        pos = torch.arange(SELF_LEN, device=at.device)
        done = (lens // BLOCK * BLOCK)[:, None]  # positions below it are codes
        end = lens + T
        row = (end[:, None] - 1) - (end[:, None] - 1 - torch.arange(RING, device=at.device)) % RING  # newest position of a ring row
        keep = (row < lens[:, None]) | (row < (end // BLOCK * BLOCK - BLOCK)[:, None])  # ... written before, or not at all
        block = torch.arange(SELF_LEN // BLOCK, device=at.device)
        closed = (block >= done // BLOCK) & (block < (end // BLOCK)[:, None])  # blocks that these rows complete
        whole = {}
        for n in "kv":
            new = st[n].float().transpose(1, 2)
            ring = st[n + "_ring"][at]
            x = _dequantized(st[n + "_codes"][at], st[n + "_scales"][at])
            x = torch.where((pos < done)[:, None, :, None], x, ring.float()[:, :, pos % RING])
            shift = (pos - lens[:, None])[:, None, :, None]
            x = torch.where(shift >= 0, new.gather(2, shift.clamp(0, T - 1).expand(-1, case["heads"], -1, D)), x)
            whole[n] = x
            codes, scales = _quantize(x.view(*x.shape[:2], -1, BLOCK, D))
            sel = closed[:, None, :, None, None]
            old = st[n + "_codes"][at].view(torch.uint8).view(*x.shape[:2], -1, BLOCK, D)
            codes = torch.where(sel, codes.view(torch.uint8), old).view(*x.shape)
            st[n + "_codes"].view(torch.uint8)[at] = codes
            st[n + "_scales"][at] = torch.where(closed[:, None], scales, st[n + "_scales"][at])
            fresh = st[n].transpose(1, 2).gather(2, (row - lens[:, None]).clamp(0, T - 1)[:, None, :, None].expand(-1, case["heads"], -1, D))
            st[n + "_ring"][at] = torch.where(keep[:, None, :, None], ring, fresh)
        limit = lens[:, None] + 1 + torch.arange(T, device=at.device)
        o = _attend(st["q"], whole["k"], whole["v"], limit)
    return [o] + [st[n + b] for b in ("_codes", "_scales", "_ring") for n in "kv"]


def _fill(st):
    case = st["case"]
    if own:
        st["cache"].set_cross_attention(st["k"], st["v"], st["slots"])
    else:
        B, T, H = case["streams"], case["length"], case["heads"]
        for n in "kv":
            x = torch.zeros(B, H, st[n + "_codes"].shape[2], D, device=st[n].device)
            x[:, :, :T] = st[n].float().transpose(1, 2)
            codes, scales = _quantize(x.view(B, H, -1, BLOCK, D))
            st[n + "_codes"].view(torch.uint8)[st["slots"]] = codes.view(torch.uint8).view(x.shape)
            st[n + "_scales"][st["slots"]] = scales
    return [st[n + b] for b in ("_codes", "_scales") for n in "kv"]


# ---- the definition in 64 bits ----------------------------------------------------------------


def _pow2_64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(x):
    """fp64 values rounded to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(x)
    step = _pow2_64((e - 4).clamp_min(-9))
    return (x / step).round() * step


def _block64(x):
    """One block's rounded values in units of its scale, and the scale (fp64, finite values)."""
    top = float(x.abs().max())
    e = -100
    while e < 100 and math.ldexp(E4M3_MAX, e) < top:
        e += 1
    scale = math.ldexp(1.0, e)
    return _e4m3((x / scale).clamp(-E4M3_MAX, E4M3_MAX)), scale


def _rows64(codes, scales):
    return codes.double() * scales.double().repeat_interleave(BLOCK, -1)[..., None]


def _softmax64(q, k, v, first):
    """q [H, T, 64], k and v [H, L, 64]: query t sees the first `first + t` keys, or all where None."""
    s = torch.matmul(q, k.mT.contiguous()) / 8.0
    if first is not None:
        s = s + torch.triu(torch.full(s.shape[1:], -math.inf, dtype=torch.float64, device=s.device), diagonal=first)
    return torch.matmul(torch.softmax(s, -1), v)


def exact(case, seed):
    kind, st = case["kind"], _INPUTS[case["kind"]](case, seed)
    if kind == "linear":
        w = st["codes"].double() * st["scales"].double().repeat_interleave(case["group"], 1)
        y = torch.addmm(st["bias"].double(), st["x"].double(), w.T.contiguous())
        return torch.nn.functional.gelu(y) if case["gelu"] else y
    if kind == "cross":
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        for b, slot in enumerate(st["slots"].tolist()):
            n = case["length"] if st["lens"] is None else int(st["lens"][b])
            k, v = (_rows64(st[x + "_codes"][slot], st[x + "_scales"][slot])[:, :n] for x in "kv")
            out[b] = _softmax64(st["q"][b].double().transpose(0, 1), k, v, None).transpose(0, 1)
        return out
    if kind == "fill":
        blocks = -(-case["length"] // BLOCK)
        res = []
        for n in "kv":
            codes = torch.zeros(st["n_slots"], case["heads"], blocks * BLOCK, D, dtype=torch.float64, device="cuda")
            scales = torch.ones(st["n_slots"], case["heads"], blocks, dtype=torch.float64, device="cuda")
            x = st[n].double().transpose(1, 2)
            for j in range(blocks):  # a block's largest value by comparison with every border
                part = x[:, :, j * BLOCK:(j + 1) * BLOCK]
                top = part.abs().amax((2, 3))
                e = torch.full_like(top, -100)
                for p in range(-100, 40):
                    e = torch.where(top > math.ldexp(E4M3_MAX, p), torch.full_like(e, p + 1), e)
                s = _pow2_64(e)
                codes[st["slots"], :, j * BLOCK:j * BLOCK + part.shape[2]] = _e4m3(part / s[:, :, None, None])
                scales[st["slots"], :, j] = s
            res.append((codes, scales))
        return [res[0][0], res[1][0], res[0][1], res[1][1]]
    T, out, state = case["tokens"], torch.empty(st["q"].shape, dtype=torch.float64, device="cuda"), {}
    for n in "kv":
        state[n] = [st[n + b].double() for b in ("_codes", "_scales", "_ring")]
    for b, (slot, cs) in enumerate(zip(st["slots"].tolist(), st["lens"].tolist())):
        rows = {}
        for n in "kv":
            codes, scales, ring = (t[slot] for t in state[n])
            c0, end = cs // BLOCK * BLOCK, cs + T
            new = st[n][b].double().transpose(0, 1)
            seq = torch.cat([_rows64(codes, scales)[:, :c0], ring[:, [p % RING for p in range(c0, cs)]], new], 1)
            rows[n] = seq
            for j in range(c0 // BLOCK, end // BLOCK):
                for h in range(case["heads"]):
                    codes[h, j * BLOCK:(j + 1) * BLOCK], scales[h, j] = _block64(seq[h, j * BLOCK:(j + 1) * BLOCK])
            for p in range(max(cs, (end // BLOCK - 1) * BLOCK), end):
                ring[:, p % RING] = seq[:, p]
        out[b] = _softmax64(st["q"][b].double().transpose(0, 1), rows["k"], rows["v"], cs + 1).transpose(0, 1)
    return [out] + [state[n][i] for i in range(3) for n in "kv"]
