"""Serving several requests over one paged KV cache, as measurable cases.

Four operators, in the order a step of a serving program calls them:

  plan    request lengths -> pages from the free list, block tables, slots and
          positions of the step's packed rows (ifr_paged_plan)
  store   rotary embedding of the rows' q and k, k and v written to their
          slots of the cache (ifr_paged_rope_store)
  attn    attention of each request's new rows over its pages, one row or
          thousands per request (ifr_paged_attention)
  window  the same with a sliding window and a few first rows that stay
          visible

A cache holds [page][row of the page][KV head][dim]; a request's rows lie on
the pages its row of the block table names, in order.  The new rows of all
requests are packed one after another (row_start), the last of them at
position kv_len - 1 of its request.
"""

import math
import random

import numpy as np
import torch

DEV = "cuda:0"

# query heads, KV heads, head size, RoPE base, NeoX pairs
SHAPES = {
    "h896": (14, 2, 64, 1e6, True),
    "h1536": (12, 2, 128, 1e6, True),
    "h2048": (32, 4, 64, 1e4, False),
    "h4096": (32, 8, 128, 5e5, False),
}
# query and output type, cache type
TYPES = {"f16": (torch.float16, torch.float16), "mixed": (torch.float32, torch.float16),
         "f32": (torch.float32, torch.float32)}

own = False


def listed():
    return [
        # a decode step of a small batch: every request one row, few of them onto a new page
        {"name": "plan_decode_32", "kind": "plan", "page": 16, "requests": 32, "ctx_lo": 40, "ctx_hi": 4096,
         "new_lo": 1, "new_hi": 1, "mix": 1, "release": 0.0, "short": 0.0},
        # a busy server's step: prompt chunks among decodes, finished requests released, too few pages for the last ones
        {"name": "plan_mixed_1021", "kind": "plan", "page": 16, "requests": 1021, "ctx_lo": 1, "ctx_hi": 8192,
         "new_lo": 1, "new_hi": 512, "mix": 2, "release": 0.1, "short": 0.04},
        # a decode step's rows (8B widths)
        {"name": "store_decode_32", "kind": "store", "shape": "h4096", "type": "f16", "page": 16, "requests": 32,
         "ctx_lo": 40, "ctx_hi": 4096, "new_lo": 1, "new_hi": 1, "mix": 3},
        # two prompts' chunks, far into their contexts
        {"name": "store_chunks_8190", "kind": "store", "shape": "h4096", "type": "f16", "page": 64, "requests": 2,
         "ctx_lo": 4000, "ctx_hi": 120000, "new_lo": 4095, "new_hi": 4095, "mix": 4},
        # one request's decode step at a short context (1.1B widths, activations in f32 as the op API has them)
        {"name": "attn_decode_145", "kind": "attn", "shape": "h2048", "type": "mixed", "page": 16, "requests": 1,
         "ctx_lo": 144, "ctx_hi": 144, "new_lo": 1, "new_hi": 1, "mix": 5, "window": 0, "sinks": 0},
        # a batch of chats at very different lengths
        {"name": "attn_decode_64", "kind": "attn", "shape": "h4096", "type": "f16", "page": 16, "requests": 64,
         "ctx_lo": 200, "ctx_hi": 8191, "new_lo": 1, "new_hi": 1, "mix": 6, "window": 0, "sinks": 0},
        # the reference's f32 cache, a small model's heads
        {"name": "attn_decode_8_f32", "kind": "attn", "shape": "h896", "type": "f32", "page": 32, "requests": 8,
         "ctx_lo": 1000, "ctx_hi": 6000, "new_lo": 1, "new_hi": 1, "mix": 7, "window": 0, "sinks": 0},
        # two long documents being answered
        {"name": "attn_decode_long", "kind": "attn", "shape": "h4096", "type": "f16", "page": 64, "requests": 2,
         "ctx_lo": 100000, "ctx_hi": 131071, "new_lo": 1, "new_hi": 1, "mix": 8, "window": 0, "sinks": 0},
        # prompt chunks and decodes in one step
        {"name": "attn_chunks_9", "kind": "attn", "shape": "h4096", "type": "f16", "page": 16, "requests": 9,
         "ctx_lo": 300, "ctx_hi": 8000, "new_lo": 200, "new_hi": 2048, "mix": 9, "window": 0, "sinks": 0},
        # a follow-up prompt, f32 activations over an f16 cache
        {"name": "attn_chunk_517_mixed", "kind": "attn", "shape": "h2048", "type": "mixed", "page": 32, "requests": 1,
         "ctx_lo": 1021, "ctx_hi": 1021, "new_lo": 517, "new_hi": 517, "mix": 10, "window": 0, "sinks": 0},
        # decode steps of long chats under a window
        {"name": "window_decode_32", "kind": "window", "shape": "h4096", "type": "f16", "page": 16, "requests": 32,
         "ctx_lo": 3000, "ctx_hi": 32000, "new_lo": 1, "new_hi": 1, "mix": 11, "window": 4096, "sinks": 4},
        # a long prompt's last chunk under a window
        {"name": "window_chunk_4095", "kind": "window", "shape": "h4096", "type": "f16", "page": 64, "requests": 1,
         "ctx_lo": 12289, "ctx_hi": 12289, "new_lo": 4095, "new_hi": 4095, "mix": 12, "window": 1024, "sinks": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# what a drawn case may cost: below the largest listed ones
MOST_BYTES, MOST_FLOPS = 8.0e8, 4.0e11


def draw(rng):
    kind = rng.choice(["plan", "store", "attn", "attn", "attn", "attn", "window", "window"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    mix = rng.randrange(1 << 30)
    if kind == "plan":
        hi = _log(rng, 20, 20000)
        return {"kind": kind, "page": page, "requests": _log(rng, 1, 1000), "ctx_lo": rng.choice([0, 1, hi // 10]),
                "ctx_hi": hi, "new_lo": 1, "new_hi": rng.choice([1, 1, _log(rng, 2, 500)]), "mix": mix,
                "release": rng.choice([0.0, 0.05, 0.3]), "short": rng.choice([0.0, 0.0, 0.05, 0.5])}
    shape = rng.choice(sorted(SHAPES))
    case = {"kind": kind, "shape": shape, "type": rng.choice(["f16", "f16", "mixed", "f32"]), "page": page,
            "requests": _log(rng, 1, 96), "ctx_lo": 0, "ctx_hi": _log(rng, 30, 60000), "new_lo": 1,
            "new_hi": rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 3000)]), "mix": mix}
    case["ctx_lo"] = rng.choice([0, case["ctx_hi"] // 20, case["ctx_hi"]])
    if kind == "store":
        while work(case)["bytes"] > 2.8e8:
            case["requests"] = (case["requests"] + 1) // 2
            case["new_hi"] = (case["new_hi"] + 1) // 2
        return case
    case["window"] = _log(rng, 50, 8000) if kind == "window" else 0
    case["sinks"] = rng.choice([0, 1, 4, 4, 16, 70]) if kind == "window" else 0
    # an f32 product runs at a sixteenth of an f16 one's rate
    part = {"f16": 1.0, "mixed": 0.5, "f32": 1 / 16}[case["type"]]
    while work(case)["bytes"] > MOST_BYTES or work(case)["flops"] > MOST_FLOPS * part:
        if case["requests"] > 1:
            case["requests"] = case["requests"] * 3 // 4
        else:
            case["ctx_hi"] = case["ctx_hi"] * 3 // 4
            case["ctx_lo"] = min(case["ctx_lo"], case["ctx_hi"])
            case["new_hi"] = (case["new_hi"] * 3 + 3) // 4
    return case


def lengths(case):
    """(rows in the cache, new rows) of each request: spread over the logarithm, the first at the upper ends."""
    rng = random.Random(case["mix"])
    n = case["requests"]
    spread = lambda lo, hi: [hi] + [_log(rng, max(lo, 1), max(hi, 1)) if hi else 0 for _ in range(n - 1)]  # noqa: E731
    ctx, new = spread(case["ctx_lo"], case["ctx_hi"]), spread(case["new_lo"], case["new_hi"])
    if case["ctx_lo"] == 0:  # some requests begin
        ctx = [0 if i and rng.random() < 0.2 else c for i, c in enumerate(ctx)]
    if case["new_hi"] > 8:  # decodes among the chunks
        new = [1 if i and rng.random() < 0.3 else v for i, v in enumerate(new)]
    return ctx, new


def seen(case):
    """Pairs of a new row and a cache row that it sees, of all requests; and the cache rows that any row sees."""
    ctx, new = lengths(case)
    w, s = case.get("window", 0), case.get("sinks", 0)
    pairs = rows = 0
    for c, n in zip(ctx, new):
        if not w:
            pairs += n * c + n * (n + 1) // 2
            rows += c + n
            continue
        p = np.arange(c, c + n, dtype=np.int64)
        near = np.minimum(p + 1, w)
        pairs += int(near.sum() + np.minimum(s, p + 1 - near).sum())
        first = max(0, c - w + 1)
        rows += c + n - first + min(s, first)
    return pairs, rows


def work(case):
    k = case["kind"]
    ctx, new = lengths(case)
    rows = sum(new)
    if k == "plan":
        # lengths and new table entries in and out, a position and a slot per row
        pages = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in zip(ctx, new))
        return {"bytes": 4 * 6 * case["requests"] + 8 * pages + 12 * rows, "flops": 0}
    heads, kvh, hs, _, _ = SHAPES[case["shape"]]
    q, kv = (torch.finfo(t).bits // 8 for t in TYPES[case["type"]])
    if k == "store":
        return {"bytes": rows * ((heads + 2 * kvh) * hs * 4 + heads * hs * q + 2 * kvh * hs * kv + 12),
                "flops": rows * (heads + kvh) * hs * 3}
    pairs, kept = seen(case)
    return {"bytes": kept * kvh * hs * 2 * kv + rows * heads * hs * 2 * q, "flops": 4 * pairs * heads * hs}


# ---------------------------------------------------------------- inputs --

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + stream * 7919 + 12345) % (1 << 62))
    return g


def _randn(shape, g, std=1.0, dtype=torch.float32):
    x = torch.empty(shape, device=DEV, dtype=dtype)
    return x.normal_(0.0, std, generator=g)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, device=DEV, dtype=dtype)


def _tables(case, seed, ctx, new, spare):
    """Pages of the rows in the cache, drawn from a shuffled list; the pages left are the free list."""
    page = case["page"]
    held = [-(-c // page) for c in ctx]
    most = max(-(-(c + n) // page) for c, n in zip(ctx, new))
    n_pages = sum(-(-(c + n) // page) for c, n in zip(ctx, new)) + spare
    order = torch.randperm(n_pages, generator=_gen(seed, 90), device=DEV).to(torch.int32)
    filled = torch.arange(most, device=DEV)[None, :] < _ints(held)[:, None]
    table = torch.full((len(ctx), most), -1, device=DEV, dtype=torch.int32)
    table[filled] = order[:sum(held)]
    return table, order[sum(held):], n_pages


def prepare(case, seed):
    ctx, new = lengths(case)
    s = {"case": case, "rows": sum(new), "requests": len(ctx), "ctx": ctx, "new": new}
    if case["kind"] == "plan":
        table, free, n_pages = _tables(case, seed, ctx, new, 5)
        rng = np.random.default_rng(seed)
        gone = rng.random(len(ctx)) < case["release"]
        count = max(0, int(len(free) * (1.0 - case["short"])))
        s |= {"n_pages": n_pages, "table": table, "count": _ints([count]), "ctx_len": _ints(ctx),
              "new_len": _ints(np.where(gone, -1, new).tolist()),
              "free": torch.cat([free, torch.full((n_pages - len(free),), -1, device=DEV, dtype=torch.int32)])}
        s["out"] = {"count": torch.empty_like(s["count"]), "ctx_len": torch.empty_like(s["ctx_len"]),
                    "row_start": torch.empty(len(ctx) + 1, device=DEV, dtype=torch.int32),
                    "kv_len": torch.empty_like(s["ctx_len"]),
                    "positions": torch.empty(s["rows"], device=DEV, dtype=torch.int32),
                    "slots": torch.empty(s["rows"], device=DEV, dtype=torch.int64)}
        return s
    heads, kvh, hs, base, neox = SHAPES[case["shape"]]
    qt, kt = TYPES[case["type"]]
    page, rows = case["page"], s["rows"]
    total = [c + n for c, n in zip(ctx, new)]
    if case["kind"] == "store":
        # only the pages that the new rows lie on: the rows before them are not touched
        start = [c // page * page for c in ctx]
        table, _, n_pages = _tables(case, seed, [t - a for t, a in zip(total, start)], [0] * len(ctx), 3)
        local = np.concatenate([np.arange(c - a, c - a + n) for c, a, n in zip(ctx, start, new)])
        pos = np.concatenate([np.arange(c, c + n) for c, n in zip(ctx, new)])
        req = torch.from_numpy(np.repeat(np.arange(len(ctx)), new)).to(DEV)
        local = torch.from_numpy(local).to(DEV)
        g = _gen(seed, 1)
        s |= {"slots": table[req, local // page].long() * page + local % page,
              "positions": torch.from_numpy(pos).to(DEV).to(torch.int32), "n_pages": n_pages, "table": table,
              "qkv": _randn((rows, (heads + 2 * kvh) * hs), g),
              "key": _randn((n_pages, page, kvh, hs), g, dtype=kt), "value": _randn((n_pages, page, kvh, hs), g, dtype=kt),
              "q": torch.empty((rows, heads, hs), device=DEV, dtype=qt)}
        return s
    table, _, n_pages = _tables(case, seed, total, [0] * len(ctx), 3)
    g = _gen(seed, 2)
    s |= {"table": table, "n_pages": n_pages, "kv_len": _ints(total),
          "row_start": _ints(np.concatenate([[0], np.cumsum(new)]).tolist()),
          # scores of standard deviation 2: a few rows of the cache carry most of a row's weight
          "q": _randn((rows, heads, hs), g, 2.0).to(qt), "key": _randn((n_pages, page, kvh, hs), g, dtype=kt),
          "value": _randn((n_pages, page, kvh, hs), g, dtype=kt), "out": torch.empty((rows, heads, hs), device=DEV, dtype=qt)}
    return s


# ------------------------------------------------------- the plain forms --

def _plan_plain(s):
    page, rows, most = s["case"]["page"], s["rows"], s["table"].shape[1]
    ctx, new, free = s["ctx_len"].long(), s["new_len"].long(), s["free"].clone()
    gone = new < 0
    new = new.clamp(min=0)
    held = (ctx + page - 1) // page
    column = torch.arange(most, device=DEV)[None, :]
    # the pages of released requests go onto the free list, in the order of the requests and their tables
    back = s["table"][gone[:, None] & (column < held[:, None])]
    count = s["count"].long()
    top = count + back.numel()
    free[count + torch.arange(back.numel(), device=DEV)] = back
    end = torch.cumsum(new, 0)
    start = end - new
    fits = ((ctx + new) <= most * page) & (end <= rows) & ~gone
    need = torch.where(fits, (ctx + new + page - 1) // page - held, 0)
    off = torch.cumsum(need, 0) - need
    ok = fits & ((need == 0) | (off + need <= top))  # one that needs no page goes on
    taken = torch.where(ok, need, 0)
    fresh = (column >= held[:, None]) & (column < (held + taken)[:, None])
    at = top - 1 - (off[:, None] + column - held[:, None])
    table = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], s["table"])
    row = torch.arange(rows, device=DEV)
    req = torch.searchsorted(end, row, right=True)
    inside = req < end.numel()
    req = req.clamp(max=end.numel() - 1)
    pos = ctx[req] + row - start[req]
    live = inside & ok[req]
    slots = table[req, (pos // page).clamp(max=most - 1)].long() * page + pos % page
    kv = torch.where(ok, ctx + new, 0)
    return {"count": (top - taken.sum()).to(torch.int32), "free": free, "table": table,
            "ctx_len": torch.where(gone, 0, torch.where(ok, ctx + new, ctx)).to(torch.int32),
            "row_start": torch.cat([start, end[-1:]]).to(torch.int32), "kv_len": kv.to(torch.int32),
            "positions": torch.where(live, pos, -1).to(torch.int32), "slots": torch.where(live, slots, -1)}


def _store_plain(s):
    heads, kvh, hs, base, neox = SHAPES[s["case"]["shape"]]
    x = s["qkv"].view(s["rows"], heads + 2 * kvh, hs)
    # angles in 64 bits: at position 1e5 a 32-bit angle is off by 4e-3
    theta = base ** (-2.0 * torch.arange(hs // 2, device=DEV, dtype=torch.float64) / hs)
    angle = s["positions"].double()[:, None] * theta
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    r = x[:, :heads + kvh]
    if neox:
        a, b = r[..., :hs // 2], r[..., hs // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    s["q"].copy_(r[:, :heads])
    s["key"].view(-1, kvh, hs)[s["slots"]] = r[:, heads:].to(s["key"].dtype)
    s["value"].view(-1, kvh, hs)[s["slots"]] = x[:, heads + kvh:].to(s["value"].dtype)
    return {"q": s["q"], "key": s["key"], "value": s["value"]}


def _scores_softmax(q, k, v, visible):
    """q [.., heads, rows, dims] over k, v [.., KV heads, keys, dims], visible [.., 1, 1, rows, keys]."""
    kvh, hs, rows = k.shape[-3], k.shape[-1], q.shape[-2]
    group = q.shape[-3] // kvh
    q = q.unflatten(-3, (kvh, group)).flatten(-3, -2)  # the heads that share a KV head, as rows of one product
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hs))
    p.unflatten(-2, (group, rows)).masked_fill_(~visible, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    return torch.matmul(p.div_(p.sum(-1, keepdim=True)), v).unflatten(-2, (group, rows)).flatten(-4, -3)


def _visible(pos, key, w, sinks):
    m = key <= pos
    return m & ((key > pos - w) | (key < sinks)) if w else m


def _attn_plain(s):
    c, page = s["case"], s["case"]["page"]
    w, sinks = c["window"], c["sinks"]
    heads, kvh, hs, _, _ = SHAPES[c["shape"]]
    key, value = s["key"].view(-1, kvh, hs), s["value"].view(-1, kvh, hs)
    if c["new_hi"] == 1:
        # decode: the requests as one padded batch, over the rows that any of them sees
        last = s["kv_len"].long()[:, None] - 1
        n = min(max(s["ctx"]) + 1, w + sinks if w else 1 << 62)
        at = torch.arange(n, device=DEV)[None, :]
        if w:
            first = (last - w + 1).clamp(min=0)
            at = torch.where(at < first.clamp(max=sinks), at, at - first.clamp(max=sinks) + first)
        at, ok = at.expand(last.shape[0], n).clamp(max=s["table"].shape[1] * page - 1), at <= last
        slot = s["table"].gather(1, at // page).long().clamp(min=0) * page + at % page
        k, v = key[slot].float().transpose(1, 2), value[slot].float().transpose(1, 2)
        v = v * ok[:, None, :, None]
        out = _scores_softmax(s["q"].float()[:, :, None], k, v, (ok & _visible(last, at, w, sinks))[:, None, None, None])
        s["out"].copy_(out[:, :, 0])
        return s["out"]
    row = 0
    for r, (ctx, n) in enumerate(zip(s["ctx"], s["new"])):
        # a request's chunk over the rows that any of its rows sees, a few rows at a time where the scores are large
        step = max(1, min(n, (1 << 30) // (heads * (ctx + n))))
        for i in range(0, n, step):
            pos = torch.arange(ctx + i, ctx + min(i + step, n), device=DEV)
            first = max(0, ctx + i - w + 1) if w else 0
            last = ctx + min(i + step, n)
            at = torch.cat([torch.arange(min(sinks, first), device=DEV), torch.arange(first, last, device=DEV)])
            slot = s["table"][r, at // page].long() * page + at % page
            k, v = key[slot].float().transpose(0, 1), value[slot].float().transpose(0, 1)
            q = s["q"][row + i:row + i + pos.numel()].float().transpose(0, 1)
            out = _scores_softmax(q, k, v, _visible(pos[:, None], at[None, :], w, sinks)[None, None])
            s["out"][row + i:row + i + pos.numel()] = out.transpose(0, 1).to(s["out"].dtype)
        row += n
    return s["out"]


# ------------------------------------------------ the framework's kernels --

_CTX = None


def _context():
    global _CTX
    if _CTX is None:
        import inferi_amd

        torch.cuda.init()
        _CTX = inferi_amd.LlmContext(0)
    return _CTX


def _handles(s):
    """The argument structs that a program keeps beside its buffers."""
    if "args" in s:
        return s["args"]
    import inferi_amd as I

    c = s["case"]
    if c["kind"] == "plan":
        o = s["out"]
        s["args"] = I.PagedPlan(
            n_requests=s["requests"], n_rows=s["rows"], n_pages=s["n_pages"], page_size=c["page"],
            max_pages=s["table"].shape[1], ctx_len=s["ctx_len"].data_ptr(), new_len=s["new_len"].data_ptr(),
            free_pages=s["free"].data_ptr(), free_count=s["count"].data_ptr(), free_count_out=o["count"].data_ptr(),
            block_table=s["table"].data_ptr(), ctx_len_out=o["ctx_len"].data_ptr(),
            row_start=o["row_start"].data_ptr(), kv_len=o["kv_len"].data_ptr(), positions=o["positions"].data_ptr(),
            slots=o["slots"].data_ptr())
        return s["args"]
    heads, kvh, hs, base, neox = SHAPES[c["shape"]]
    qt, kt = (I.F16 if t == torch.float16 else I.F32 for t in TYPES[c["type"]])
    cache = I.PagedCache(key=s["key"].data_ptr(), value=s["value"].data_ptr(), block_table=s["table"].data_ptr(),
                         dtype=kt, n_pages=s["n_pages"], page_size=c["page"], max_pages=s["table"].shape[1],
                         n_kv_heads=kvh, head_size=hs)
    if c["kind"] == "store":
        wide = s["qkv"].shape[1]
        x = s["qkv"].data_ptr()
        args = I.PagedRope(
            n_rows=s["rows"], n_heads=heads, variant=I.ROPE_NEOX if neox else I.ROPE_ORIGINAL, base_freq=base,
            q=x, k=x + 4 * heads * hs, v=x + 4 * (heads + kvh) * hs, ld_q=wide, ld_k=wide, ld_v=wide,
            positions=s["positions"].data_ptr(), slots=s["slots"].data_ptr(), q_out=s["q"].data_ptr(), q_dtype=qt)
    else:
        args = I.PagedAttentionParams(
            n_requests=s["requests"], n_rows=s["rows"], n_heads=heads, q_dtype=qt, max_new=max(s["new"]),
            max_kv=max(a + b for a, b in zip(s["ctx"], s["new"])), window=c["window"], n_sinks=c["sinks"],
            row_start=s["row_start"].data_ptr(), kv_len=s["kv_len"].data_ptr(), q=s["q"].data_ptr(),
            out=s["out"].data_ptr())
    s["args"] = cache, args
    return s["args"]


def _run_own(s):
    ctx, kind = _context(), s["case"]["kind"]
    args = _handles(s)
    if kind == "plan":
        ctx.paged_plan(args)
        o = s["out"]
        return {"count": o["count"], "free": s["free"], "table": s["table"], "ctx_len": o["ctx_len"],
                "row_start": o["row_start"], "kv_len": o["kv_len"], "positions": o["positions"], "slots": o["slots"]}
    if kind == "store":
        ctx.paged_rope_store(*args)
        return {"q": s["q"], "key": s["key"], "value": s["value"]}
    import inferi_amd as I

    I.PagedAttention.launch(ctx, *args)
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return _plan_plain(state) if kind == "plan" else _store_plain(state) if kind == "store" else _attn_plain(state)


# ------------------------------------------------------ the exact results --

def exact(case, seed):
    """The definitions in 64 bits, request by request and head by head."""
    if case["kind"] == "plan":
        return None  # whole numbers only
    s = prepare(case, seed)
    heads, kvh, hs, base, neox = SHAPES[case["shape"]]
    if case["kind"] == "store":
        x = s["qkv"].double().view(s["rows"], heads + 2 * kvh, hs)
        pairs = torch.arange(hs // 2, device=DEV)
        i0, i1 = (pairs, pairs + hs // 2) if neox else (2 * pairs, 2 * pairs + 1)
        one = torch.ones((), device=DEV, dtype=torch.float64)
        turn = torch.polar(one, s["positions"].double()[:, None] / torch.pow(one * base, 2.0 * pairs.double() / hs))
        r = x.clone()
        z = torch.complex(x[:, :heads + kvh, i0], x[:, :heads + kvh, i1]) * turn[:, None]
        r[:, :heads + kvh, i0], r[:, :heads + kvh, i1] = z.real, z.imag
        key, value = s["key"].double(), s["value"].double()
        page, row = s["slots"] // case["page"], s["slots"] % case["page"]
        key[page, row], value[page, row] = r[:, heads:heads + kvh], r[:, heads + kvh:]
        return {"q": r[:, :heads], "key": key, "value": value}
    if work(case)["flops"] > 2.0e12:
        return None
    out = torch.empty((s["rows"], heads, hs), device=DEV, dtype=torch.float64)
    row = 0
    for r, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        j = torch.arange(c + n, device=DEV)
        p = torch.arange(c, c + n, device=DEV)[:, None]
        hidden = j[None, :] > p
        if case["window"]:
            hidden |= (j[None, :] <= p - case["window"]) & (j[None, :] >= case["sinks"])
        page, at = s["table"][r, j // case["page"]].long(), j % case["page"]
        for h in range(heads):
            k, v = s["key"][page, at, h * kvh // heads].double(), s["value"][page, at, h * kvh // heads].double()
            z = torch.mm(s["q"][row:row + n, h].double(), k.t().contiguous()) / math.sqrt(hs)
            z[hidden] = -math.inf
            out[row:row + n, h] = torch.mm(torch.softmax(z, -1), v)
        row += n
    return out
