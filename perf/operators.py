"""Cases of the paged key-value cache operators: plan (block tables and slot
maps from request lengths), append (new K/V rows into the pages) and decode
(attention of one new token per request over the pages).

A cache is a pair of tensors [pages, page_size, kv_heads, head_dim]; a slot is
page * page_size + offset.  `run` computes the plain form in elementary torch
operations, or, where `own` is true, calls the framework."""
import importlib
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0


def listed():
    return [
        # plan: the step of a serving loop in which every running request gets one token
        {"name": "plan step of 256", "op": "plan", "requests": 256, "held_lo": 1, "held_hi": 4096, "added_lo": 1,
         "added_hi": 1, "page": 16, "width": 512, "spare": 40},
        # plan: prompts of mixed lengths enter an empty cache together
        {"name": "plan prompts", "op": "plan", "requests": 48, "held_lo": 0, "held_hi": 0, "added_lo": 1,
         "added_hi": 4096, "page": 16, "width": 512, "spare": 0},
        # plan: a very wide batch of short continuations (drafts or chunks of a few tokens)
        {"name": "plan wide", "op": "plan", "requests": 8192, "held_lo": 0, "held_hi": 8000, "added_lo": 1,
         "added_hi": 7, "page": 32, "width": 256, "spare": 1000},
        # append: one new token of each of 32 requests, where only latency counts
        {"name": "append step of 32", "op": "append", "tokens": 32, "padding": 0, "kv_heads": 8, "dim": 128,
         "page": 16, "in": "bf16", "cache": "bf16", "run": 1, "heads_first": False},
        # append: the prompts of a batch, whole pages at a time
        {"name": "append prompts f16", "op": "append", "tokens": 32768, "padding": 100, "kv_heads": 8, "dim": 64,
         "page": 16, "in": "f16", "cache": "f16", "run": 512, "heads_first": False},
        # append: prompts into a cache held in 8 bits, pages with the heads outermost
        {"name": "append prompts e4m3", "op": "append", "tokens": 10007, "padding": 3, "kv_heads": 4, "dim": 128,
         "page": 64, "in": "bf16", "cache": "e4m3", "run": 333, "heads_first": True},
        # decode: one user's single request, where only latency counts
        {"name": "decode one", "op": "decode", "batch": 1, "empty": 0, "len_lo": 1000, "len_hi": 1000, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "in": "bf16", "cache": "bf16", "out": "bf16", "window": 0,
         "heads_first": False},
        # decode: as many slices as the forward's largest batch (1024 of up to 2048 keys, head_dim 64), O in f32
        {"name": "decode mha f16", "op": "decode", "batch": 64, "empty": 0, "len_lo": 1024, "len_hi": 2048,
         "q_heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "in": "f16", "cache": "f16", "out": "f32", "window": 0,
         "heads_first": False},
        # decode: a serving batch of very different lengths, shared KV heads, a few padded rows
        {"name": "decode gqa ragged", "op": "decode", "batch": 64, "empty": 3, "len_lo": 1, "len_hi": 8192,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "in": "bf16", "cache": "bf16", "out": "bf16",
         "window": 0, "heads_first": False},
        # decode: few requests over long documents, one KV head for all query heads
        {"name": "decode mqa long", "op": "decode", "batch": 3, "empty": 0, "len_lo": 50001, "len_hi": 131072,
         "q_heads": 32, "kv_heads": 1, "dim": 128, "page": 32, "in": "bf16", "cache": "bf16", "out": "bf16",
         "window": 0, "heads_first": False},
        # decode: a sliding window, the pages before it given back, an odd page size, the forward's head_dim 32
        {"name": "decode window", "op": "decode", "batch": 96, "empty": 0, "len_lo": 1, "len_hi": 8192, "q_heads": 16,
         "kv_heads": 8, "dim": 32, "page": 7, "in": "f16", "cache": "f16", "out": "f16", "window": 1023,
         "heads_first": False},
        # decode: a cache in 8 bits, twice the tokens in the same memory, pages with the heads outermost
        {"name": "decode e4m3", "op": "decode", "batch": 48, "empty": 0, "len_lo": 1, "len_hi": 16384, "q_heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "in": "bf16", "cache": "e4m3", "out": "bf16", "window": 0,
         "heads_first": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "decode", "decode"])
    page = rng.choice([1, 5, 7, 8, 16, 16, 32, 64, 100, 128])
    if op == "plan":
        requests = _log(rng, 1, 8192)
        added_hi = _log(rng, 1, max(1, min(4096, 98000 // requests)))
        held_hi = rng.choice([0, _log(rng, 1, min(8000, max(1, page * 2000000 // requests)))])  # tables of up to 2M entries
        return {"op": op, "requests": requests, "held_lo": 0, "held_hi": held_hi,
                "added_lo": rng.choice([0, 1, added_hi]), "added_hi": added_hi, "page": page,
                "width": (held_hi + added_hi) // page + rng.randrange(1, 40), "spare": rng.choice([-1, 0, 33])}
    dim = rng.choice([16, 32, 64, 64, 128, 128])
    kinds = [("f16", "f16"), ("bf16", "bf16")] + ([("f16", "e4m3"), ("bf16", "e4m3")] if dim >= 32 else [])
    given, cache = rng.choice(kinds)
    if op == "append":
        kv_heads = rng.choice([1, 2, 3, 8, 16])
        tokens = _log(rng, 1, 16000000 // (kv_heads * dim))
        # tokens of different requests lie in pages of their own: not so many that the pool outgrows the prompts' one
        small = tokens * page * kv_heads * dim < 32000000
        return {"op": op, "tokens": tokens, "padding": rng.choice([0, 1, 57]), "kv_heads": kv_heads, "dim": dim,
                "page": page, "in": given, "cache": cache, "run": rng.choice([1, 17, 700] if small else [350, 700]),
                "heads_first": rng.random() < 0.3}
    kv_heads = rng.choice([1, 2, 5, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8, 12, 16, 32, 40])
    batch = _log(rng, 1, 300)
    window = rng.choice([0, 0, 0, _log(rng, 1, 4000)])
    # the gathered f32 forms of K and V, and the products, stay under those of the largest listed cases
    most = 400000000 // (batch * kv_heads * dim) * 8 // max(8, group)
    len_hi = _log(rng, 1, max(1, min(200000, most)))
    return {"op": op, "batch": batch, "empty": rng.choice([0, 0, 1, 2]), "len_lo": rng.choice([1, len_hi, len_hi // 3 + 1]),
            "len_hi": len_hi, "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "in": given,
            "cache": cache, "out": rng.choice(["f32", given, given]), "window": window,
            "heads_first": rng.random() < 0.3}


def _spread(count, lo, hi):
    """`count` whole numbers from lo to hi, evenly spaced: the same for every seed."""
    return [hi if count == 1 else lo + (hi - lo) * i // (count - 1) for i in range(count)]


def _lens(case):
    """The requests' cached lengths; the last `empty` requests are padding."""
    empty = min(case["empty"], case["batch"] - 1)
    return _spread(case["batch"] - empty, case["len_lo"], case["len_hi"]) + [0] * empty


def _plan_need(case):
    """(held, added, new pages of each request) before the requests are shuffled."""
    n = case["requests"]
    held, added = _spread(n, case["held_lo"], case["held_hi"]), _spread(n, case["added_hi"], case["added_lo"])
    page = case["page"]
    return held, added, [-(-(h + a) // page) - -(-h // page) for h, a in zip(held, added)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _pages(case, pages, g, std):
    """K and V pages; one page more than the cache has stands behind them in memory (the plain form's place for padding)."""
    shape = (pages + 1, case["kv_heads"], case["page"], case["dim"]) if case["heads_first"] else (
        pages + 1, case["page"], case["kv_heads"], case["dim"])
    out = []
    for _ in range(2):
        x = torch.empty(shape, dtype=DTYPES[case["in"]], device="cuda").normal_(0.0, std, generator=g)
        x = (x * 24.0).to(DTYPES[case["cache"]]) if case["cache"] == "e4m3" else x
        out.append(x.transpose(1, 2) if case["heads_first"] else x)
    return out


def _scales(case, g):
    """A cache in 8 bits holds each head's values over a scale, here between 1/48 and 1/24."""
    if case["cache"] != "e4m3":
        return None, None
    return tuple((torch.rand(case["kv_heads"], generator=g, device="cuda") + 1.0) / 48.0 for _ in range(2))


def _prepare_plan(case, g):
    held, added, need = _plan_need(case)
    order = torch.randperm(case["requests"], generator=g, device="cuda")
    held = torch.tensor(held, dtype=torch.int32, device="cuda")[order].contiguous()
    added = torch.tensor(added, dtype=torch.int32, device="cuda")[order].contiguous()
    page, width = case["page"], case["width"]
    have = (held + page - 1) // page
    total, new = int(have.sum()), sum(need)
    free = max(0, new + case["spare"])
    ids = torch.randperm(total + free, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["requests"], width), -1, dtype=torch.int32, device="cuda")
    columns = torch.arange(width, device="cuda")
    table[columns[None, :] < have[:, None]] = ids[:total]
    tokens = int(added.sum())
    made = lambda n, dtype: torch.zeros(n, dtype=dtype, device="cuda")  # noqa: E731
    return {"held": held, "added": added, "table": table, "free_pages": ids[total:].contiguous(),
            "free_count": torch.tensor([free], dtype=torch.int32, device="cuda"), "page": page,
            "seq_lens": made(case["requests"], torch.int32), "starts": made(case["requests"] + 1, torch.int32),
            "slots": made(tokens + 5, torch.int64), "positions": made(tokens + 5, torch.int32),
            "left": made(1, torch.int32), "status": made(4, torch.int32)}


def _prepare_append(case, g):
    tokens, page, run_length = case["tokens"], case["page"], case["run"]
    runs = -(-tokens // run_length)
    per = -(-run_length // page)
    pages = runs * per + runs * per // 4 + 1
    k_pages, v_pages = _pages(case, pages, g, 0.5)
    k_scale, v_scale = _scales(case, g)
    ids = torch.randperm(pages, generator=g, device="cuda")[:runs * per].view(runs, per)
    t = torch.arange(tokens, device="cuda")
    at = t % run_length
    slots = ids[t // run_length, at // page] * page + at % page
    slots = torch.cat([slots, torch.full((case["padding"],), -1, dtype=torch.int64, device="cuda")])
    # K and V as a projection leaves them: rows of one matrix [tokens, 2 * kv_heads * dim]
    rows = torch.empty(tokens + case["padding"], 2, case["kv_heads"], case["dim"], dtype=DTYPES[case["in"]], device="cuda")
    rows.normal_(0.0, 1.0, generator=g)
    s = {"k": rows[:, 0], "v": rows[:, 1], "slots": slots.contiguous(), "k_pages": k_pages, "v_pages": v_pages,
         "k_scale": k_scale, "v_scale": v_scale, "pages": pages}
    if own:
        s["cache"] = _framework().paged.Cache(k_pages[:pages], v_pages[:pages], k_scale=k_scale, v_scale=v_scale)
    return s


def _prepare_decode(case, g):
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    empty = min(case["empty"], case["batch"] - 1)
    order = torch.randperm(case["batch"] - empty, generator=g, device="cuda")
    lens = torch.cat([lens[:case["batch"] - empty][order], lens[case["batch"] - empty:]])
    page, batch, heads, dim = case["page"], case["batch"], case["q_heads"], case["dim"]
    have = (lens.long() + page - 1) // page
    # pages wholly before the window were given back
    first = ((lens.long() - case["window"]).clamp_min(0) // page) if case["window"] else torch.zeros_like(have)
    width = max(1, -(-case["len_hi"] // page)) + 2
    columns = torch.arange(width, device="cuda")[None, :]
    used = (columns >= first[:, None]) & (columns < have[:, None])
    pages = max(1, int(used.sum()))
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    table[used] = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[:int(used.sum())]
    k_pages, v_pages = _pages(case, pages, g, 1.0)
    k_scale, v_scale = _scales(case, g)
    # the query heads as a projection leaves them, beside the new K and V of the same matrix
    q = torch.empty(batch, heads + 2 * case["kv_heads"], dim, dtype=DTYPES[case["in"]], device="cuda")
    q = q.normal_(0.0, 1.0, generator=g)[:, :heads]
    s = {"q": q, "table": table, "lens": lens, "scale": dim ** -0.5, "window": case["window"], "k_pages": k_pages,
         "v_pages": v_pages, "k_scale": k_scale, "v_scale": v_scale, "page": page, "kv_heads": case["kv_heads"],
         "out": DTYPES[case["out"]], "most": max(1, case["len_hi"])}
    if own:
        ncz = _framework()
        s["cache"] = ncz.paged.Cache(k_pages[:pages], v_pages[:pages], k_scale=k_scale, v_scale=v_scale)
        s["workspace"] = ncz.paged.decode_workspace(s["cache"], heads)
        s["o"] = torch.empty(batch, heads, dim, dtype=s["out"], device="cuda")
        s["lse"] = torch.empty(batch, heads, dtype=torch.float32, device="cuda")
    return s


def _framework():
    return importlib.import_module("not-cute-zig_b200")


def prepare(case, seed):
    g = _generator(seed)
    state = {"plan": _prepare_plan, "append": _prepare_append, "decode": _prepare_decode}[case["op"]](case, g)
    state["op"] = case["op"]
    return state


def _run_plan(s):
    if own:
        _framework().paged.plan(s["held"], s["added"], s["free_pages"], s["free_count"], s["table"], s["seq_lens"],
                                s["slots"], page_size=s["page"], positions=s["positions"], starts=s["starts"],
                                left=s["left"], status=s["status"])
        return {k: s[k] for k in ("table", "seq_lens", "slots", "positions", "starts", "left", "status")}
    page, table, width = s["page"], s["table"], s["table"].shape[1]
    held, added, capacity = s["held"].long(), s["added"].long(), s["slots"].numel()
    have, want = (held + page - 1) // page, (held + added + page - 1) // page
    fits = want <= width
    need = torch.where(fits, want - have, 0)
    end = need.cumsum(0)
    free = s["free_count"].long()
    served = fits & ((need == 0) | (end <= free))
    first = end - need
    stop = added.cumsum(0)
    start = stop - added
    columns = torch.arange(width, device=table.device)[None, :]
    new = served[:, None] & (columns >= have[:, None]) & (columns < want[:, None])
    take = (free - 1 - first[:, None] - (columns - have[:, None])).clamp(0, max(0, s["free_pages"].numel() - 1))
    pool = s["free_pages"] if s["free_pages"].numel() else table.new_zeros(1)
    table.copy_(torch.where(new, pool[take], table))
    t = torch.arange(capacity, device=table.device)
    r = torch.searchsorted(stop, t, right=True)
    inside = r < held.numel()
    r = r.clamp_max(held.numel() - 1)
    position = torch.where(inside, held[r] + t - start[r], 0)
    id_ = table[r, (position // page).clamp_max(width - 1)].long()
    slots = torch.where(inside & served[r] & (id_ >= 0), id_ * page + position % page, -1)
    taken = torch.where(served & (need > 0), end, 0).max()
    tokens = stop[-1:]
    status = torch.cat([tokens, taken[None], (~served).sum()[None], (tokens - capacity).clamp_min(0)])
    return {"table": table, "seq_lens": torch.where(served, held + added, held).int(), "slots": slots,
            "positions": position.int(), "starts": torch.cat([start, tokens]).clamp_max(capacity).int(),
            "left": (free - taken).int(), "status": status.int()}


def _run_append(s):
    pages = s["pages"]
    if own:
        _framework().paged.append(s["k"], s["v"], s["slots"], s["cache"])
        return s["k_pages"][:pages], s["v_pages"][:pages]
    page = s["k_pages"].shape[1]
    at = torch.where(s["slots"] < 0, pages * page, s["slots"])
    for rows, pool, scale in ((s["k"], s["k_pages"], s["k_scale"]), (s["v"], s["v_pages"], s["v_scale"])):
        if scale is not None:
            rows = (rows.float() / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(pool.dtype)
            # 8-bit values move as bytes: index_put takes no float8
            pool, rows = pool.view(torch.uint8), rows.view(torch.uint8)
        pool[at // page, at % page] = rows
    return s["k_pages"][:pages], s["v_pages"][:pages]


def _run_decode(s):
    if own:
        _framework().paged.decode(s["q"], s["cache"], s["table"], s["lens"], s["o"], scale=s["scale"],
                                  window=s["window"], lse=s["lse"], workspace=s["workspace"])
        return s["o"], s["lse"]
    batch, heads, dim = s["q"].shape
    page, kv = s["page"], s["kv_heads"]
    key = torch.arange(s["most"], device=s["q"].device)
    lens = s["lens"].long()[:, None]
    id_ = s["table"][:, key // page].long()
    seen = (key < lens) & (id_ >= 0)
    if s["window"]:
        seen &= key >= lens - s["window"]
    id_ = id_.clamp_min(0)
    at = (key % page).expand(batch, -1)

    def gathered(pool):  # [batch, kv_heads, keys, dim] in f32, rows outside the mask 0
        small = pool.dtype == torch.float8_e4m3fn
        rows = pool.view(torch.uint8)[id_, at].view(pool.dtype) if small else pool[id_, at]
        return torch.where(seen[:, :, None, None], rows.float(), 0.0).transpose(1, 2)

    q = s["q"].float().view(batch, kv, heads // kv, dim)
    scores = torch.matmul(q, gathered(s["k_pages"]).transpose(2, 3)) * s["scale"]
    if s["k_scale"] is not None:
        scores = scores * s["k_scale"][:, None, None]
    scores = torch.where(seen[:, None, None, :], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, gathered(s["v_pages"])) / torch.where(total == 0, 1.0, total)
    if s["v_scale"] is not None:
        o = o * s["v_scale"][:, None, None]
    lse = top + torch.log(total)
    return o.reshape(batch, heads, dim).to(s["out"]), lse.reshape(batch, heads)


def run(state):
    return {"plan": _run_plan, "append": _run_append, "decode": _run_decode}[state["op"]](state)


def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}
    if case["op"] == "plan":
        held, added, need = _plan_need(case)
        # lengths read and written, the new pages moved, one held page per request that goes on in it, slots and positions
        partial = sum(1 for h, a in zip(held, added) if h % case["page"] and a)
        return {"bytes": 16 * len(held) + 8 * sum(need) + 4 * partial + 12 * sum(added), "flops": 0}
    if case["op"] == "append":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": values * (size[case["in"]] + size[case["cache"]]) + 8 * (case["tokens"] + case["padding"]),
                "flops": values if case["cache"] == "e4m3" else 0}
    lens = [min(n, case["window"]) if case["window"] else n for n in _lens(case)]
    keys, rows = sum(lens), case["batch"] * case["q_heads"]
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size[case["cache"]]
            + rows * (case["dim"] * (size[case["in"]] + size[case["out"]]) + 4)
            + 4 * sum(-(-n // case["page"]) for n in lens),
            "flops": 4 * keys * case["q_heads"] * case["dim"]}


def _exact_append(case, seed):
    s = prepare(case, seed)
    keep = (s["slots"] >= 0).nonzero()[:, 0]
    slots, page = s["slots"][keep], case["page"]
    out = []
    for name in ("k", "v"):
        pool = s[name + "_pages"][:s["pages"]].double()
        rows = s[name][keep].double()
        if s[name + "_scale"] is not None:
            rows = torch.clamp(rows / s[name + "_scale"].double()[None, :, None], -E4M3_MAX, E4M3_MAX)
        pool[torch.div(slots, page, rounding_mode="floor"), torch.remainder(slots, page)] = rows
        out.append(pool)
    return tuple(out)


def _exact_decode(case, seed):
    """Request by request from the definition, every page of its keys looked up in its table."""
    s = prepare(case, seed)
    q, page, group = s["q"].double(), case["page"], case["q_heads"] // case["kv_heads"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    scales = [torch.ones(case["kv_heads"], device=q.device) if x is None else x for x in (s["k_scale"], s["v_scale"])]
    for b, n in enumerate(s["lens"].tolist()):
        lo = max(0, n - case["window"]) if case["window"] else 0
        key = torch.arange(lo, n, device=q.device)
        ids = s["table"][b, torch.div(key, page, rounding_mode="floor")]
        key, ids = key[ids >= 0], ids[ids >= 0].long()
        if not key.numel():
            continue
        for h in range(case["kv_heads"]):
            k, v = _head_rows(s["k_pages"], h, ids, key % page), _head_rows(s["v_pages"], h, ids, key % page)
            heads = slice(h * group, (h + 1) * group)
            score = q[b, heads] @ (k * scales[0][h].double()).T * s["scale"]
            lse[b, heads] = torch.logsumexp(score, -1)
            o[b, heads] = torch.softmax(score, -1) @ (v * scales[1][h].double())
    return o, lse


def _head_rows(pool, h, ids, at):
    if pool.dtype == torch.float8_e4m3fn:
        return pool.view(torch.uint8)[:, :, h][ids, at].view(torch.float8_e4m3fn).double()
    return pool[:, :, h][ids, at].double()


def exact(case, seed):
    if case["op"] == "plan":
        return None
    return (_exact_append if case["op"] == "append" else _exact_decode)(case, seed)
