"""The operators of paged serving, as cases that can be timed: page tables and slot maps built on the GPU,
attention of new tokens over a paged key-value cache, packed prompts' attention with the writes of their
pages, and the log probabilities of given tokens.

``listed`` gives fixed cases (large-v3 width, 20 heads of 64, 448 text positions, 1500 encoder rows, vocabulary
51866, and generic grouped heads over long contexts), ``draw`` random ones of the same ranges. With ``own`` false
``run`` is the plain form (elementary torch operations in fp32), with ``own`` true the framework's entry points.
``exact`` is the definition in 64 bits.

The cache's definition: a page holds ``page`` positions of every key/value head, ``[n_pages, kv_heads, page, dim]``.
A stream's table names its pages in order: position p of stream s is row ``p % page`` of page
``tables[s, p // page]``, and its slot is ``tables[s, p // page] * page + p % page``. Pages that nobody holds stand on
a stack (``free_pages``, the first ``n_free`` of them).
"""
from __future__ import annotations

import math

import torch

own = False

VOCAB = 51866
CROSS_LEN = 1500
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the next token of 8 live streams gets its place before the step: the smallest launch
        {"name": "plan_step", "kind": "plan", "streams": 8, "held": 447, "new": 1, "page": 16},
        # 1000 requests of up to 224 tokens arrive together behind histories of their own
        {"name": "plan_prompts", "kind": "plan", "streams": 1000, "held": 224, "new": 224, "page": 32},
        # one live stream's token appends and attends: latency
        {"name": "pages_one", "kind": "pages", "dtype": "bf16", "streams": 1, "tokens": 1, "heads": 20, "kv_heads": 20, "dim": 64, "page": 16, "length": 200, "append": True},
        # a decode step of 52 streams of ragged histories
        {"name": "pages_batch", "kind": "pages", "dtype": "bf16", "streams": 52, "tokens": 1, "heads": 20, "kv_heads": 20, "dim": 64, "page": 32, "length": 447, "append": True},
        # 16 streams verify 5-token drafts
        {"name": "pages_draft", "kind": "pages", "dtype": "fp16", "streams": 16, "tokens": 5, "heads": 20, "kv_heads": 20, "dim": 64, "page": 16, "length": 443, "append": True},
        # long contexts of a model with grouped heads: the bytes of the cache, split over its length
        {"name": "pages_long", "kind": "pages", "dtype": "bf16", "streams": 4, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "length": 32767, "append": True},
        # one short prompt into its pages: the smallest call
        {"name": "prompt_one", "kind": "prompt", "dtype": "bf16", "streams": 1, "heads": 20, "kv_heads": 20, "dim": 64, "length": 13, "keys": 0, "page": 16, "padded": 0},
        # 64 prompts and texts of up to 448 tokens, packed without padding, and written to their pages
        {"name": "prompt_batch", "kind": "prompt", "dtype": "fp16", "streams": 64, "heads": 20, "kv_heads": 20, "dim": 64, "length": 448, "keys": 0, "page": 32, "padded": 40},
        # 16 packed prompts over their windows' encoder rows (no mask)
        {"name": "prompt_cross", "kind": "prompt", "dtype": "bf16", "streams": 16, "heads": 20, "kv_heads": 20, "dim": 64, "length": 224, "keys": CROSS_LEN, "page": 0, "padded": 0},
        # two long prompts of a model with grouped heads: bound by the matrix cores
        {"name": "prompt_long", "kind": "prompt", "dtype": "bf16", "streams": 2, "heads": 32, "kv_heads": 8, "dim": 128, "length": 8192, "keys": 0, "page": 64, "padded": 0},
        # one stream's sampled token, its entropy and five alternatives
        {"name": "logprobs_one", "kind": "logprobs", "dtype": "fp32", "rows": 1, "vocab": VOCAB, "top": 5, "blocked": True},
        # the tokens of 16 texts scored at once (word confidences)
        {"name": "logprobs_texts", "kind": "logprobs", "dtype": "bf16", "rows": 3584, "vocab": VOCAB, "top": 3, "blocked": False},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "pages", "pages", "prompt", "prompt", "logprobs"])
    dtype = rng.choice(["bf16", "fp16"])
    page = rng.choice([16, 32, 64, 128])
    heads, kv_heads, dim = rng.choice([(20, 20, 64), (12, 12, 64), (6, 6, 64), (16, 4, 64), (32, 8, 128), (16, 2, 128), (8, 1, 128), (8, 8, 128)])
    if kind == "plan":
        return {"kind": kind, "streams": _log(rng, 1, 1000), "held": rng.choice([0, _log(rng, 1, 2000)]),
                "new": rng.choice([1, _log(rng, 1, 224)]), "page": page}
    if kind == "pages":
        streams = _log(rng, 1, 64)
        tokens = rng.choice([1, 1, rng.randint(2, 8)])
        most = min(32767, 131068 // streams * 8 // kv_heads)  # the longest case's cache at most
        return {"kind": kind, "dtype": dtype, "streams": streams, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "page": page, "length": rng.choice([_log(rng, 1, min(447, most)), _log(rng, 1, most)]), "append": rng.random() < 0.8}
    if kind == "prompt":
        cross = dim == 64 and rng.random() < 0.25
        streams = _log(rng, 1, 16 if cross else 64)
        length = _log(rng, 1, 448 if cross else min(8192, 16384 // streams))
        return {"kind": kind, "dtype": dtype, "streams": streams, "heads": heads, "kv_heads": kv_heads, "dim": dim, "length": length,
                "keys": rng.choice([CROSS_LEN, _log(rng, 1, CROSS_LEN)]) if cross else 0,
                "page": 0 if cross else rng.choice([0, page]), "padded": rng.choice([0, rng.randint(1, 100)])}
    return {"kind": kind, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": _log(rng, 1, 1792),
            "vocab": rng.choice([VOCAB, 51864, 51865, _log(rng, 1000, 150000) // 2 + 500]), "top": rng.choice([0, 1, rng.randint(2, 20)]),
            "blocked": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, *shape, dtype):
    """Projected rows: a few of the last dimension's channels are much larger than the others."""
    x = torch.randn(shape, generator=g, device="cuda")
    big = 1.0 + 3.0 * (torch.rand(shape[-2:], generator=g, device="cuda") < 0.05)
    return (x * big).to(dtype)


def _spread(n, hi, lo):
    """n whole numbers, evenly from lo to hi (one: hi): the lengths of a batch. Their order is the seed's."""
    return [hi - (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _shuffled(g, values, dtype=torch.int32):
    order = torch.randperm(len(values), generator=g, device="cuda")
    return torch.tensor(values, dtype=dtype, device="cuda")[order]


def _tables(g, streams, lens, page, max_len, spare):
    """Page tables of a pool in use: `streams` rows hold `lens` positions in pages of any order, two more streams
    hold nothing, and the other pages are free (at least `spare` of them)."""
    n, width = streams.numel() + 2, -(-max_len // page)
    held = torch.zeros(n, dtype=torch.int64, device="cuda")
    held[streams] = (lens.long() + page - 1) // page
    used = int(held.sum())
    pages = torch.randperm(used + spare, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(width, device="cuda")
    at = (held.cumsum(0) - held)[:, None] + col
    tables = torch.where(col < held[:, None], pages[at.clamp(max=used + spare - 1)], torch.full_like(pages[:1], -1))
    free = torch.full_like(pages, -1)
    free[:spare] = pages[used:]
    seq_lens = torch.zeros(n, dtype=torch.int32, device="cuda")
    seq_lens[streams] = lens.to(torch.int32)
    return {"tables": tables.contiguous(), "page_counts": held.to(torch.int32), "seq_lens": seq_lens, "free_pages": free,
            "n_free": torch.tensor([spare], dtype=torch.int32, device="cuda")}


def _plan_inputs(case, seed):
    g, B, page = _gen(seed), case["streams"], case["page"]
    streams = torch.randperm(B + 2, generator=g, device="cuda")[:B]
    lens = _shuffled(g, _spread(B, case["held"], case["held"] // 2))
    new = _shuffled(g, _spread(B, case["new"], (case["new"] + 1) // 2))
    st = _tables(g, streams, lens, page, case["held"] + case["new"], B * (case["new"] // page + 2))
    st.update(streams=streams.to(torch.int32), lens=lens, new=new, total=int(new.sum()))
    return st


def _pages_inputs(case, seed):
    g, dt, B, page, T = _gen(seed), DTYPES[case["dtype"]], case["streams"], case["page"], case["tokens"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    streams = torch.randperm(B + 2, generator=g, device="cuda")[:B]
    lens = _shuffled(g, _spread(B, case["length"], case["length"] // 2))
    after = lens + T if case["append"] else lens
    st = _tables(g, streams, after, page, case["length"] + T, 3)
    for n in "kv":
        st[n + "_pages"] = _rows(g, st["free_pages"].numel(), Hk, page, D, dtype=dt)
    qkv = _rows(g, B, T, H + 2 * Hk, D, dtype=dt)  # one projection's output
    st["q"], st["k"], st["v"] = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    st.update(streams=streams.to(torch.int32), lens=lens)
    return st


def _prompt_inputs(case, seed):
    g, dt, B, page = _gen(seed), DTYPES[case["dtype"]], case["streams"], case["page"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    lens = _shuffled(g, _spread(B, case["length"], (case["length"] + 1) // 2), torch.int64)
    zero = lens.new_zeros(1)
    st = {"cu": torch.cat([zero, lens.cumsum(0)]).to(torch.int32)}
    st["host"] = lens.tolist()
    total = sum(st["host"]) + case["padded"]
    if case["keys"]:  # the encoder rows' projections, windows of their own lengths
        klens = _shuffled(g, _spread(B, case["keys"], (case["keys"] + 1) // 2), torch.int64)
        st["cu_k"], st["host_k"] = torch.cat([zero, klens.cumsum(0)]).to(torch.int32), klens.tolist()
        st["q"] = _rows(g, total, H, D, dtype=dt)
        kv = _rows(g, sum(st["host_k"]), 2 * Hk, D, dtype=dt)
        st["k"], st["v"] = kv[:, :Hk], kv[:, Hk:]
    else:
        st["cu_k"], st["host_k"] = None, st["host"]
        qkv = _rows(g, total, H + 2 * Hk, D, dtype=dt)
        st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    if case["padded"]:
        st["out"] = torch.zeros(total, H, D, dtype=dt, device="cuda")
    if page:
        n_pages = -(-total // page) + 2
        slots = torch.randperm(n_pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        st["slots"] = slots.view(-1)[:total].contiguous()
        if case["padded"]:
            st["slots"][-case["padded"]:] = -1  # rows behind the last sequence are not kept
        for n in "kv":
            st[n + "_pages"] = torch.zeros(n_pages, Hk, page, D, dtype=dt, device="cuda")
    return st


def _logprobs_inputs(case, seed):
    g, rows, V = _gen(seed), case["rows"], case["vocab"]
    logits = (2.5 * torch.randn(rows, V, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
    tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
    peak = torch.rand(rows, generator=g, device="cuda") < 0.7  # mostly the row's own choice, clear of the others
    at = torch.arange(rows, device="cuda")
    logits[at, tokens] = torch.where(peak, torch.full_like(logits[:, 0], 14.0), logits[at, tokens])
    blocked = None
    if case["blocked"]:
        blocked = torch.rand(rows, V, generator=g, device="cuda") < 0.3
        blocked[at, tokens] = False
    return {"logits": logits, "tokens": tokens, "blocked": blocked}


_INPUTS = {"plan": _plan_inputs, "pages": _pages_inputs, "prompt": _prompt_inputs, "logprobs": _logprobs_inputs}
_STATE = ("tables", "page_counts", "seq_lens", "free_pages", "n_free")


def prepare(case, seed):
    st = _INPUTS[case["kind"]](case, seed)
    st["kind"], st["case"] = case["kind"], dict(case)
    if own:  # the handles that a program keeps: the tables and one layer's pages around their buffers
        import whisperdrz_amd as w

        page = case.get("page", 0)
        if case["kind"] in ("plan", "pages"):
            n, n_pages = int(st["seq_lens"].numel()), int(st["free_pages"].numel())
            most = case["held"] + case["new"] if case["kind"] == "plan" else case["length"] + case["tokens"]
            st["handle"] = w.PageTables(n, n_pages, page, most, storage={x: st[x] for x in _STATE})
        elif case["kind"] == "prompt" and page:
            st["handle"] = w.PageTables(case["streams"], int(st["k_pages"].shape[0]), page, page * int(st["k_pages"].shape[0]), device="cuda")
        if "k_pages" in st:
            st["cache"] = w.FlashKVPages(st["handle"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]],
                                         storage={x: st[x] for x in ("k_pages", "v_pages")})
    return st


def work(case):
    if case["kind"] == "logprobs":
        n, size = case["rows"] * case["vocab"], DTYPES[case["dtype"]].itemsize
        return {"bytes": n * (size + case["blocked"]) + case["rows"] * (16 + 12 * case["top"]), "flops": 4 * n}
    B = case["streams"]
    if case["kind"] == "plan":
        page, new = case["page"], sum(_spread(B, case["new"], (case["new"] + 1) // 2))
        got = new / page  # pages that are taken from the stack into the tables, and go back
        return {"bytes": int(B * 4 * 8 + new * 16 + got * 4 * 4), "flops": int(B * 4 + new * 4)}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "pages":
        T, held = case["tokens"], _spread(B, case["length"], case["length"] // 2)
        new = T if case["append"] else 0
        seen = sum(held) + B * ((T + 1) / 2 if new else 0)
        # the history's keys and values, the queries and outputs, the new rows read and written once
        return {"bytes": int(2 * D * (2 * Hk * sum(held) + B * (2 * H * T + 4 * Hk * new))), "flops": int(4 * H * T * seen * D)}
    lens = _spread(B, case["length"], (case["length"] + 1) // 2)
    keys = _spread(B, case["keys"], (case["keys"] + 1) // 2)
    # which keys meet which queries is the seed's: the mean
    pairs = sum(lens) * sum(keys) / B if case["keys"] else sum(n * (n + 1) / 2 for n in lens)
    rows = sum(keys) if case["keys"] else sum(lens)
    nbytes = 2 * D * (2 * H * sum(lens) + 2 * Hk * rows * (2 if case["page"] else 1))
    return {"bytes": int(nbytes), "flops": int(4 * H * pairs * D)}


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    return {"plan": _plan, "pages": _pages, "prompt": _prompt, "logprobs": _logprobs}[state["kind"]](state)


def _plan(st):
    """The step's tokens get their places, and are given back (as those of a draft that was rejected)."""
    page, total = st["case"]["page"], st["total"]
    if own:
        plan = st["handle"].plan(st["new"], total, st["streams"])
        st["handle"].truncate(st["lens"], st["streams"])
        res = [plan.cu_seqlens, plan.starts, plan.slots, plan.positions]
    else:
        tables, counts, seq_lens, free, n_free = (st[x] for x in _STATE)
        at, new, B, dev = st["streams"].long(), st["new"].long(), st["case"]["streams"], st["new"].device
        starts, held, top = seq_lens[at], counts[at].long(), n_free.long()
        need = ((starts + new + page - 1) // page - held).clamp(min=0)
        off = need.cumsum(0) - need
        j = torch.arange(st["case"]["new"] // page + 2, device=dev)
        take = j < need[:, None]
        where = (at[:, None] * tables.shape[1] + held[:, None] + j)[take]
        tables.view(-1)[where] = free[(top - 1 - off[:, None] - j)[take]]
        cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
        row = torch.repeat_interleave(torch.arange(B, device=dev), new, output_size=total)
        positions = starts.long()[row] + torch.arange(total, device=dev) - cu[row]
        slots = tables[at[row], positions // page].long() * page + positions % page
        counts[at] = (held + need).to(torch.int32)
        seq_lens[at] = (starts + new).to(torch.int32)
        n_free -= need.sum().to(torch.int32)
        # back to the lengths before
        keep = (st["lens"].long() + page - 1) // page
        gone = counts[at].long() - keep
        off, sum_gone = gone.cumsum(0) - gone, gone.sum()
        take = j < gone[:, None]
        where = (at[:, None] * tables.shape[1] + keep[:, None] + j)[take]
        free[(n_free.long() + sum_gone - 1 - off[:, None] - j)[take]] = tables.view(-1)[where]
        tables.view(-1)[where] = -1
        counts[at], seq_lens[at] = keep.to(torch.int32), st["lens"]
        n_free += sum_gone.to(torch.int32)
        res = [cu.to(torch.int32), starts, slots, positions]
    return res + [st[x] for x in _STATE]


def _softmax_rows(q, k, v, limit):
    """softmax(q k / sqrt(D)) v over the keys below limit (broadcast to [..., T, 1]): q [..., T, D], k and v
    [..., L, D], all fp32; rows without keys give zeros."""
    s = (q @ k.transpose(-1, -2)) * q.shape[-1] ** -0.5
    if limit is not None:
        s = s.masked_fill(torch.arange(k.shape[-2], device=q.device) >= limit, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, torch.ones_like(total), total)


def _pages(st):
    case = st["case"]
    if own:
        import whisperdrz_amd as w

        new = (st["k"], st["v"]) if case["append"] else (None, None)
        o = w.flash_attn_with_kvpages(st["q"], st["cache"], *new, cache_seqlens=st["lens"], cache_batch_idx=st["streams"])
    else:
        B, T, H, Hk, D, page = (case[x] for x in ("streams", "tokens", "heads", "kv_heads", "dim", "page"))
        tables, lens = st["tables"][st["streams"].long()].long(), st["lens"].long()[:, None]
        t = torch.arange(T, device=lens.device)
        if case["append"]:
            pos = lens + t
            at = tables.gather(1, pos // page)
            for n in "kv":
                st[n + "_pages"][at, :, pos % page] = st[n]
        rows = []
        for n in "kv":
            x = st[n + "_pages"][tables.clamp(min=0)]  # [B, pages, Hk, page, D]
            rows.append(x.transpose(1, 2).reshape(B, Hk, 1, -1, D).float())
        if not case["append"]:  # what nobody has written does not count
            rows[1] = rows[1] * (torch.arange(rows[1].shape[3], device=lens.device) < lens)[:, None, None, :, None]
        q = st["q"].float().view(B, T, Hk, H // Hk, D).permute(0, 2, 3, 1, 4)
        limit = (lens + 1 + t if case["append"] else lens.expand(B, T))[:, None, None, :, None]
        o = _softmax_rows(q, rows[0], rows[1], limit).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(st["q"].dtype)
    return [o, st["k_pages"], st["v_pages"]] if case["append"] else o


def _prompt(st):
    case, out = st["case"], st.get("out")
    if own:
        import whisperdrz_amd as w

        if case["page"]:
            st["cache"].write(st["k"], st["v"], st["slots"])
        o = w.packed_attention(st["q"], st["k"], st["v"], st["cu"], st["cu_k"], causal=not case["keys"], out=out)
    else:
        H, Hk, D, page = (case[x] for x in ("heads", "kv_heads", "dim", "page"))
        if page:
            kept = st["slots"][:st["slots"].numel() - case["padded"]]
            for n in "kv":
                st[n + "_pages"][kept // page, :, kept % page] = st[n][:kept.numel()]
        o = out if out is not None else torch.empty(st["q"].shape, dtype=st["q"].dtype, device="cuda")
        a = b = 0
        for n, nk in zip(st["host"], st["host_k"]):
            q = st["q"][a:a + n].float().view(n, Hk, H // Hk, D).permute(1, 2, 0, 3)
            k, v = (st[x][b:b + nk].float().transpose(0, 1)[:, None] for x in "kv")
            limit = None if case["keys"] else (torch.arange(n, device=q.device) + 1)[:, None]
            step = Hk if H * n * nk <= 1 << 28 else 1  # heads at once
            for h in range(0, Hk, step):
                r = _softmax_rows(q[h:h + step], k[h:h + step], v[h:h + step], limit)
                o[a:a + n].view(n, Hk, H // Hk, D)[:, h:h + step] = r.permute(2, 0, 1, 3).to(o.dtype)
            a, b = a + n, b + nk
    return [o, st["k_pages"], st["v_pages"]] if case["page"] else o


def _logprobs(st):
    top, tokens = st["case"]["top"], st["tokens"]
    if own:
        import whisperdrz_amd as w

        r = w.token_logprobs(st["logits"], tokens, top=top, blocked=st["blocked"])
        return [r.logprobs, r.entropy] + ([r.top_logprobs, r.top_ids] if top else [])
    x = st["logits"].float()
    if st["blocked"] is not None:
        x = x.masked_fill(st["blocked"], -math.inf)
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, dtype=torch.float64)  # long sums
    log_total = torch.log(total)
    entropy = log_total - (e * d.masked_fill(e == 0, 0.0)).sum(-1, dtype=torch.float64) / total
    res = [(d.gather(1, tokens[:, None])[:, 0].double() - log_total).float(), entropy.float()]
    if top:
        ids, values, index = [], [], torch.arange(x.shape[1], device=x.device)
        for _ in range(top):  # the largest value left, of equal ones the lowest index
            m = d.amax(-1, keepdim=True)
            i = torch.where(d == m, index, x.shape[1]).amin(-1, keepdim=True)
            values.append((m[:, 0].double() - log_total).float())
            ids.append(i[:, 0])
            d.scatter_(1, i, -math.inf)
        res += [torch.stack(values, 1), torch.stack(ids, 1)]
    return res


# ---- the definition in 64 bits ----------------------------------------------------------------


def _exact_plan(case, st):
    page, lens, new = case["page"], st["lens"].tolist(), st["new"].tolist()
    streams, table = st["streams"].tolist(), st["tables"].tolist()
    free = st["free_pages"].tolist()[:int(st["n_free"])]
    cu, slots, positions = [0], [], []
    for s, n, more in zip(streams, lens, new):
        row = [p for p in table[s] if p >= 0]
        for p in range(n, n + more):
            if p // page == len(row):
                row.append(free.pop())
            slots.append(row[p // page] * page + p % page)
            positions.append(p)
        cu.append(len(slots))
    whole = lambda x: torch.tensor(x, dtype=torch.int64, device="cuda")
    return [whole(cu).int(), st["lens"], whole(slots), whole(positions)] + [st[x] for x in _STATE]


def _attention64(q, k, v, first):
    """q [n, H, D], k and v [L, Hk, D]: query t sees the first `first + t` keys, all where None."""
    n, H, D = q.shape
    L, Hk = k.shape[:2]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    if L == 0:
        return out
    mask = None if first is None else torch.ones(n, L, dtype=torch.bool, device=q.device).tril(first - 1)
    for h in range(H):
        kh, vh = (x[:, h // (H // Hk)].double() for x in (k, v))
        s = torch.matmul(q[:, h].double(), kh.T.contiguous()) / math.sqrt(D)
        if mask is not None:
            s = torch.where(mask, s, torch.full_like(s, -math.inf))
        out[:, h] = torch.matmul(torch.softmax(s, -1), vh)
    return out


def exact(case, seed):
    kind, st = case["kind"], _INPUTS[case["kind"]](case, seed)
    if kind == "plan":
        return _exact_plan(case, st)
    if kind == "logprobs":
        logprobs, entropy, values, ids = [], [], [], []
        for i in range(0, case["rows"], 256):
            x = st["logits"][i:i + 256].double()
            if st["blocked"] is not None:
                x = torch.where(st["blocked"][i:i + 256], torch.full_like(x, -math.inf), x)
            lp = torch.log_softmax(x, -1)
            logprobs.append(lp.gather(1, st["tokens"][i:i + 256, None])[:, 0])
            entropy.append(torch.special.entr(lp.exp()).sum(-1))
            if case["top"]:
                order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
                values.append(lp.gather(1, order))
                ids.append(order)
        return [torch.cat(t) for t in (logprobs, entropy, values, ids) if t]
    if kind == "pages":
        page, T = case["page"], case["tokens"]
        pages = [st["k_pages"].double(), st["v_pages"].double()]
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        for b, (s, n) in enumerate(zip(st["streams"].tolist(), st["lens"].tolist())):
            table = st["tables"][s].long()
            if case["append"]:
                for t in range(T):
                    for x, y in zip(pages, (st["k"], st["v"])):
                        x[table[(n + t) // page], :, (n + t) % page] = y[b, t].double()
            end = n + T if case["append"] else n
            at = table[:-(-end // page)]
            k, v = (x[at].transpose(0, 1).flatten(1, 2)[:, :end].transpose(0, 1) for x in pages)
            out[b] = _attention64(st["q"][b], k, v, n + 1 if case["append"] else None)
        return [out] + pages if case["append"] else out
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    a = b = 0
    for n, nk in zip(st["host"], st["host_k"]):
        out[a:a + n] = _attention64(st["q"][a:a + n], st["k"][b:b + nk], st["v"][b:b + nk], None if case["keys"] else 1)
        a, b = a + n, b + nk
    if not case["page"]:
        return out
    pages = [st["k_pages"].double(), st["v_pages"].double()]
    for i, slot in enumerate(st["slots"].tolist()):
        if slot >= 0:
            for x, n in zip(pages, "kv"):
                x[slot // case["page"], :, slot % case["page"]] = st[n][i].double()
    return [out] + pages
