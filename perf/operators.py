"""What the operators of a mixed serving batch cost, and what they compute.

One decode or prefill step over many requests does the following beside the shared weights:

* ``pages``   block tables and slot maps from the requests' lengths (reserve, and trim to hand pages back)
* ``append``  the step's keys and values into the paged cache, with the 8-bit key bounds of every page they touch
* ``sparse``  attention of each new token over the pages that those bounds score highest
* ``lora``    low-rank adapters, one per request, added to a shared projection's output
* ``logits``  repetition, frequency and presence penalties, biases and grammar masks before the sampler

``run`` computes each in elementary torch operations, or, where ``own`` is set, through zeroplatform_b200.ops.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one decode step of a full batch: every request adds one token, few of them a page
        {"name": "pages decode 64", "op": "pages", "batch": 64, "new_lo": 1, "new_hi": 1, "len_hi": 2047, "page": 16,
         "pad": 0},
        # prompts of very different lengths admitted together into a padded token buffer
        {"name": "pages prefill 256", "op": "pages", "batch": 256, "new_lo": 1, "new_hi": 511, "len_hi": 300,
         "page": 16, "pad": 37},
        # one new token of each request into its last page (grouped-query heads, half-precision pool)
        {"name": "append decode 64", "op": "append", "batch": 64, "new_lo": 1, "new_hi": 1, "hkv": 8, "hd": 128,
         "page": 16, "pool": "fp16"},
        # prompt chunks that begin and end inside pages, every head with its own keys
        {"name": "append prefill 4096", "op": "append", "batch": 16, "new_lo": 65, "new_hi": 447, "hkv": 32,
         "hd": 128, "page": 16, "pool": "fp16"},
        # a single long conversation, where latency is what counts
        {"name": "sparse 1x8k", "op": "sparse", "batch": 1, "hq": 32, "hkv": 8, "hd": 128, "page": 16,
         "ctx_lo": 8191, "ctx_hi": 8191, "budget": 64, "sink": 1, "recent": 2, "pool": "fp16"},
        # a small model's batch, head size 64, one key head per query head, single-precision pool
        {"name": "sparse 24x2k fp32", "op": "sparse", "batch": 24, "hq": 12, "hkv": 12, "hd": 64, "page": 16,
         "ctx_lo": 1, "ctx_hi": 2048, "budget": 32, "sink": 1, "recent": 1, "pool": "fp32"},
        # a batch of long documents
        {"name": "sparse 32x32k", "op": "sparse", "batch": 32, "hq": 32, "hkv": 8, "hd": 128, "page": 16,
         "ctx_lo": 4096, "ctx_hi": 32768, "budget": 128, "sink": 1, "recent": 4, "pool": "fp16"},
        # one request with one adapter
        {"name": "lora 1 row", "op": "lora", "rows": 1, "run": 1, "adapters": 4, "rank": 16, "k": 4096, "n": 4096,
         "w": "fp16"},
        # a decode batch whose requests use different adapters of different ranks, some of them none
        {"name": "lora 64 rows mixed", "op": "lora", "rows": 64, "run": 1, "adapters": 40, "rank": 32, "k": 4096,
         "n": 11008, "w": "bf16"},
        # prompts of eight requests, a few hundred tokens each
        {"name": "lora prefill 2048", "op": "lora", "rows": 2048, "run": 250, "adapters": 8, "rank": 64, "k": 4096,
         "n": 4096, "w": "fp16"},
        # one request's logits before sampling
        {"name": "logits 1x32000", "op": "logits", "rows": 1, "vocab": 32000, "past": 700, "biases": 0, "masks": 1,
         "x": "fp32"},
        # a batch under a large vocabulary, half of its rows in a grammar
        {"name": "logits 64x131072", "op": "logits", "rows": 64, "vocab": 131072, "past": 2000, "biases": 50,
         "masks": 8, "x": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "append", "sparse", "lora", "logits"])
    if op == "pages":
        lo = rng.choice([0, 1, 1])
        hi = rng.choice([1, 1, 4, _log(rng, 8, 400)])
        return {"op": op, "batch": _log(rng, 1, 256), "new_lo": lo, "new_hi": max(lo, hi),
                "len_hi": _log(rng, 16, 2040), "page": rng.choice([8, 16, 32, 64]), "pad": rng.randint(0, 40)}
    if op == "append":
        hi = rng.choice([1, 1, 5, _log(rng, 8, 400)])
        return {"op": op, "batch": _log(rng, 1, 16 if hi > 5 else 200), "new_lo": min(1, hi), "new_hi": hi,
                "hkv": rng.choice([1, 2, 5, 8, 12, 32]), "hd": rng.choice([64, 128, 256]),
                "page": rng.choice([8, 16, 32]), "pool": rng.choice(["fp16", "fp16", "fp32"])}
    if op == "sparse":
        hkv, group = rng.choice([(1, 7), (2, 4), (8, 4), (4, 8), (12, 1), (2, 16), (5, 3)])
        hd, pool = rng.choice([64, 128, 128, 256]), rng.choice(["fp16", "fp16", "fp32"])
        hi, budget = _log(rng, 200, 16000), _log(rng, 8, 128)
        # no more requests than the largest listed case's cache and reads allow
        most = min(32, int(2e9 / (hi * hkv * hd * 2 * SIZE[pool])), int(2.5e8 / (budget * 32 * hkv * hd * SIZE[pool])))
        return {"op": op, "batch": _log(rng, 1, max(1, most)), "hq": hkv * group, "hkv": hkv, "hd": hd,
                "page": rng.choice([8, 16, 32]), "ctx_lo": rng.choice([1, hi // 2, hi]), "ctx_hi": hi,
                "budget": budget, "sink": rng.randint(0, 2), "recent": rng.randint(1, 4), "pool": pool}
    if op == "lora":
        rows = _log(rng, 1, 2000)
        return {"op": op, "rows": rows, "run": rng.choice([1, 3, 100]) if rows > 64 else 1,
                "adapters": rng.randint(1, 12), "rank": rng.choice([8, 16, 24, 32, 64]),
                "k": 32 * _log(rng, 8, 128), "n": _log(rng, 200, 4096), "w": rng.choice(["fp16", "bf16", "fp32"])}
    return {"op": op, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 131072), "past": _log(rng, 1, 4000),
            "biases": rng.choice([0, 7, 300]), "masks": rng.choice([0, 1, 5]),
            "x": rng.choice(["fp32", "fp16", "bf16"])}


def _spread(n, lo, hi):
    """n whole numbers over [lo, hi], the last one hi: the ragged lengths of a case."""
    return [hi if i == n - 1 else lo + int((i * 0.6180339887 + 0.37) % 1.0 * (hi - lo + 1)) for i in range(n)]


def _up(a, b):
    return -(-a // b)


def _adapter_rows(case):
    """The adapter of each row: runs of `run` rows, every seventh run without one."""
    run, na = case["run"], case["adapters"]
    return [-1 if (r // run) % 7 == 6 else (r // run) * 5 % na for r in range(case["rows"])]


def _rank_of(case):
    """Ranks of the adapters: the full one, and smaller ones among them."""
    r = case["rank"]
    return [r if i % 3 != 1 else max(1, r // 2 - i % 2) for i in range(case["adapters"])]


def work(case):
    op = case["op"]
    if op == "pages":
        old, new = _spread(case["batch"], 0, case["len_hi"]), _spread(case["batch"], case["new_lo"], case["new_hi"])
        pages = sum(_up(a + b, case["page"]) - _up(a, case["page"]) for a, b in zip(old, new))
        tokens = sum(new) + case["pad"]
        # per request: row, count and length in, length, offset and grant out, then the new length in and out; a page
        # is read from the stack and written to the table, and back; slot, position, row and length of every token
        return {"bytes": 32 * case["batch"] + 16 * pages + 20 * tokens, "flops": 0}
    if op == "append":
        old, new = _append_lengths(case)
        row = case["hkv"] * case["hd"]
        held = sum(a % case["page"] for a in old)  # keys already in a page whose bounds change
        pages = sum(_up(a + b, case["page"]) - a // case["page"] for a, b in zip(old, new))
        return {"bytes": sum(new) * (row * (8 + 2 * SIZE[case["pool"]]) + 8) + held * row * SIZE[case["pool"]]
                + pages * (2 * row + 4 * case["hkv"]), "flops": 0}
    if op == "sparse":
        ctx = _spread(case["batch"], case["ctx_lo"], case["ctx_hi"])
        pages = [_up(c, case["page"]) for c in ctx]
        sel = sum(min(c, case["budget"] * case["page"]) for c in ctx)
        scored = sum(p for p in pages if p > case["budget"])
        hkv, hd, hq, b = case["hkv"], case["hd"], case["hq"], case["batch"]
        return {"bytes": scored * hkv * (2 * hd + 4) + sum(pages) * 4 + sel * hkv * hd * 2 * SIZE[case["pool"]]
                + b * hq * hd * 8 + b * hkv * case["budget"] * 4,
                "flops": 4.0 * scored * hq * hd + 4.0 * sel * hq * hd}
    if op == "lora":
        rows, ranks = [a for a in _adapter_rows(case) if a >= 0], _rank_of(case)
        k, n = case["k"], case["n"]
        return {"bytes": sum(ranks[a] for a in set(rows)) * (k + n) * SIZE[case["w"]] + len(rows) * k * 4
                + case["rows"] * (8 * n + 4), "flops": sum(2.0 * ranks[a] * (k + n) for a in rows)}
    rows, v = case["rows"], case["vocab"]
    return {"bytes": rows * (v * (SIZE[case["x"]] + 4) + 4 * case["past"] + 8 * case["biases"])
            + min(rows, case["masks"]) * v // 8, "flops": 2.0 * rows * (case["past"] + case["biases"])}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _append_lengths(case):
    new = _spread(case["batch"], case["new_lo"], case["new_hi"])
    old = _spread(case["batch"], 0, 3 * case["page"] - 1)
    return old, new


def _bounds_of(k):
    """8-bit bounds of keys k [..., tokens, hd]: s = max|k| / 127 in 32 bits, lo = floor(min / s), hi = ceil(max / s).
    Quotients in 64 bits, where none that is not a whole number rounds to one."""
    lo, hi = k.amin(-2).double(), k.amax(-2).double()
    s = (torch.maximum(lo.abs(), hi.abs()).amax(-1) / 127).float()
    d = torch.where(s > 0, s, torch.ones_like(s))[..., None].double()
    codes = torch.stack([torch.floor(lo / d), torch.ceil(hi / d)], -2).clamp(-127, 127)
    return codes.to(torch.int8), s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    op, s = case["op"], {"case": case}
    if op == "pages":
        page, batch = case["page"], case["batch"]
        old, new = _spread(batch, 0, case["len_hi"]), _spread(batch, case["new_lo"], case["new_hi"])
        max_pages = _up(max(a + b for a, b in zip(old, new)), page) + 3
        used = [_up(a, page) for a in old]
        need = sum(_up(a + b, page) for a, b in zip(old, new))
        num = need + 11
        perm = torch.randperm(num, generator=g, device=DEV).int()
        rows = torch.randperm(batch + 5, generator=g, device=DEV)[:batch]
        table = torch.full((batch + 5, max_pages), -1, dtype=torch.int32, device=DEV)
        cols = torch.arange(max_pages, device=DEV)
        mask = cols[None] < _int(used)[:, None]
        at = (_int(used).cumsum(0) - _int(used)).long()[:, None] + cols
        table[rows] = torch.where(mask, perm[at.clamp(max=num - 1)], table[rows])
        lens = torch.zeros(batch + 5, dtype=torch.int32, device=DEV)
        lens[rows] = _int(old)
        left = num - sum(used)
        free = torch.zeros(num, dtype=torch.int32, device=DEV)
        free[:left] = perm[sum(used):]
        tokens = sum(new) + case["pad"]
        empty = lambda n, t=torch.int32: torch.empty(n, dtype=t, device=DEV)  # noqa: E731
        s.update(table=table, lens=lens, free=free, count=_int([left]), rows=rows.int(), new=_int(new),
                 old=_int(old), tokens=tokens, page=page,
                 plan=(empty(batch + 1), empty(tokens, torch.int64), empty(tokens), empty(tokens), empty(tokens),
                       empty(batch)))
        return s
    if op == "append":
        page, hkv, hd, batch = case["page"], case["hkv"], case["hd"], case["batch"]
        old, new = _append_lengths(case)
        per = _up(max(a + b for a, b in zip(old, new)), page)
        pages = batch * per
        table = torch.randperm(pages, generator=g, device=DEV).view(batch, per)
        b = torch.repeat_interleave(torch.arange(batch, device=DEV), _int(new))
        first = (_int(new).cumsum(0) - _int(new)).long()
        pos = _int(old).long()[b] + torch.arange(sum(new), device=DEV) - first[b]
        s.update(k=rnd(sum(new), hkv, hd), v=rnd(sum(new), hkv, hd), slots=table[b, pos // page] * page + pos % page)
        t = DTYPES[case["pool"]]
        s.update(k_pool=rnd(pages, hkv, page, hd).to(t), v_pool=rnd(pages, hkv, page, hd).to(t),
                 bounds=torch.zeros((pages, hkv, 2, hd), dtype=torch.int8, device=DEV),
                 scales=torch.zeros((pages, hkv), device=DEV))
        return s
    if op == "sparse":
        page, hkv, hd, batch = case["page"], case["hkv"], case["hd"], case["batch"]
        ctx = _spread(batch, case["ctx_lo"], case["ctx_hi"])
        per = _up(max(ctx), page)
        pages, t = batch * per, DTYPES[case["pool"]]
        table = torch.randperm(pages, generator=g, device=DEV).int().view(batch, per)
        # keys share a direction per page, as neighbouring tokens do: some pages matter more than others
        k = torch.empty((pages, hkv, page, hd), dtype=t, device=DEV)
        v = torch.empty_like(k)
        bounds = torch.empty((pages, hkv, 2, hd), dtype=torch.int8, device=DEV)
        scales = torch.empty((pages, hkv), device=DEV)
        step = 4096
        for p in range(0, pages, step):
            m = min(step, pages - p)
            k[p:p + m] = (rnd(m, hkv, page, hd) + 1.5 * rnd(m, hkv, 1, hd)).to(t)
            v[p:p + m] = rnd(m, hkv, page, hd).to(t)
            bounds[p:p + m], scales[p:p + m] = _bounds_of(k[p:p + m])
        s.update(q=rnd(batch, case["hq"], hd), k_pool=k, v_pool=v, bounds=bounds, scales=scales, table=table,
                 ctx=_int(ctx), out=torch.empty((batch, case["hq"], hd), device=DEV),
                 sel=torch.empty((batch, hkv, case["budget"]), dtype=torch.int32, device=DEV))
        return s
    if op == "lora":
        k, n, r, na, t = case["k"], case["n"], case["rank"], case["adapters"], DTYPES[case["w"]]
        s.update(x=rnd(case["rows"], k), y=rnd(case["rows"], n), a=(rnd(na, r, k) / math.sqrt(k)).to(t),
                 b=(rnd(na, n, r) / math.sqrt(r)).to(t), adapter=_int(_adapter_rows(case)),
                 ranks=_int(_rank_of(case)), scales=0.5 + torch.rand(na, generator=g, device=DEV),
                 out=torch.empty((case["rows"], n), device=DEV))
        return s
    rows, v, past, nb, nm = case["rows"], case["vocab"], case["past"], case["biases"], case["masks"]
    ids = lambda *shape: torch.randint(0, v, shape, generator=g, device=DEV, dtype=torch.int32)  # noqa: E731
    # text repeats itself: most of a history comes from a few hundred tokens
    words = ids(rows, min(300, max(1, past // 2)))
    pick = (torch.rand((rows, past), generator=g, device=DEV) ** 2 * words.shape[1]).long()
    lens = _spread(rows, past // 2, past)
    s.update(x=(3 * rnd(rows, v)).to(DTYPES[case["x"]]), past=words.gather(1, pick), past_len=_int(lens),
             prompt_len=_int([n // 3 for n in lens]),
             repetition=1 + 0.5 * torch.rand(rows, generator=g, device=DEV),
             frequency=0.3 * torch.rand(rows, generator=g, device=DEV),
             presence=0.5 * torch.rand(rows, generator=g, device=DEV), out=torch.empty((rows, v), device=DEV),
             bias_start=None, bias_ids=None, bias=None, mask=None, mask_rows=None)
    if nb:
        order = torch.rand((rows, v), generator=g, device=DEV).topk(min(nb, v), 1).indices
        s.update(bias_start=_int([i * order.shape[1] for i in range(rows + 1)]),
                 bias_ids=order.reshape(-1).int(), bias=2 * rnd(order.numel()))
    if nm:
        # a grammar allows a few tokens in some states and nearly all of them in others
        share = torch.tensor([0.01 if i % 2 else 0.9 for i in range(nm)], device=DEV)[:, None]
        bits = torch.rand((nm, _up(v, 32) * 32), generator=g, device=DEV) < share
        words32 = (bits.view(nm, -1, 32).long() << torch.arange(32, device=DEV)).sum(-1)
        s.update(mask=torch.where(words32 >= 2 ** 31, words32 - 2 ** 32, words32).int(),
                 mask_rows=_int([i % nm if i % 2 == 0 else -1 for i in range(rows)]))
    return s


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        from zeroplatform_b200 import ops
        c = s["case"]
        if op == "pages":
            pool = (s["table"], s["lens"], s["free"], s["count"])
            plan = ops.reserve_pages(*pool, s["new"], s["page"], rows=s["rows"], out=s["plan"])
            ops.trim_pages(*pool, s["old"], s["page"], rows=s["rows"])
            return (*plan, *pool)
        if op == "append":
            ops.append_kv(s["k"], s["v"], s["slots"], s["k_pool"], s["v_pool"], s["bounds"], s["scales"])
            return s["k_pool"], s["v_pool"], s["bounds"] * s["scales"][:, :, None, None], s["scales"]
        if op == "sparse":
            return ops.sparse_paged_attention(s["q"], s["k_pool"], s["v_pool"], s["bounds"], s["scales"], s["table"],
                                              s["ctx"], c["budget"], sink=c["sink"], recent=c["recent"],
                                              out=s["out"], sel=s["sel"])
        if op == "lora":
            return ops.lora_add(s["y"], s["x"], s["a"], s["b"], s["adapter"], ranks=s["ranks"], scales=s["scales"],
                                out=s["out"])
        return ops.process_logits(s["x"], out=s["out"], past=s["past"], past_len=s["past_len"],
                                  prompt_len=s["prompt_len"], repetition=s["repetition"], frequency=s["frequency"],
                                  presence=s["presence"], bias_start=s["bias_start"], bias_ids=s["bias_ids"],
                                  bias=s["bias"], mask=s["mask"], mask_rows=s["mask_rows"])
    return {"pages": _pages, "append": _append, "sparse": _sparse, "lora": _lora, "logits": _logits}[op](s)


def _pages(s):
    table, lens, free, count, rows, page = s["table"], s["lens"], s["free"], s["count"], s["rows"].long(), s["page"]
    max_pages, tokens = table.shape[1], s["tokens"]
    new = s["new"].clamp(min=0).long()
    old = lens[rows].long()
    have = (old + page - 1) // page
    need = (old + new + page - 1) // page
    start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    fits = (old + new <= max_pages * page) & (start[1:] <= tokens)
    more = torch.where(fits, need - have, 0)
    upto = more.cumsum(0)
    granted = fits & (upto <= count.long())
    # the pages of each request, from the top of the stack
    col = torch.arange(max_pages, device=table.device)
    take = granted[:, None] & (col >= have[:, None]) & (col < need[:, None])
    at = count.long() - 1 - ((upto - more)[:, None] + col - have[:, None])
    mine = torch.where(take, free[at.clamp(0, free.numel() - 1)], table[rows])
    table[rows] = mine
    lens[rows] = torch.where(granted, old + new, old).int()
    count -= torch.where(granted, more, 0).sum().int()
    # slots, positions, rows and lengths of the tokens
    t = torch.arange(tokens, device=table.device)
    b = torch.searchsorted(start[1:], t, right=True)
    inside = b < rows.numel()
    b = b.clamp(max=rows.numel() - 1)
    live = inside & granted[b]
    pos = old[b] + t - start[b]
    col = (pos // page).clamp(0, max_pages - 1)
    slots = torch.where(live, mine[b, col].long() * page + pos % page, -1)
    plan = (start.int(), slots, torch.where(live, pos, 0).int(), torch.where(live, rows[b], -1).int(),
            torch.where(live, pos + 1, 0).int(), granted.int())
    # and back to the lengths before, the last request's last page first
    had = lens[rows].long()
    keep_len = torch.minimum(s["old"].clamp(min=0).long(), had)
    have, keep = (had + page - 1) // page, (keep_len + page - 1) // page
    gone = have - keep
    before = gone.flip(0).cumsum(0).flip(0) - gone
    col = torch.arange(max_pages, device=table.device)
    drop = (col >= keep[:, None]) & (col < have[:, None])
    at = count.long() + before[:, None] + have[:, None] - 1 - col
    at = torch.where(drop, at, free.numel())
    free.copy_(torch.cat([free, free.new_zeros(1)]).scatter(0, at.reshape(-1), mine.reshape(-1))[:-1])
    table[rows] = torch.where(drop, -1, mine)
    lens[rows] = keep_len.int()
    count += gone.sum().int()
    return (*plan, table, lens, free, count)


def _append(s):
    k_pool, v_pool, slots = s["k_pool"], s["v_pool"], s["slots"]
    page = k_pool.shape[2]
    p, t = slots // page, slots % page
    k_pool[p, :, t] = s["k"].to(k_pool.dtype)
    v_pool[p, :, t] = s["v"].to(v_pool.dtype)
    # a page holds keys up to the last slot written to it
    filled = torch.zeros(k_pool.shape[0], dtype=torch.int64, device=p.device).scatter_reduce(
        0, p, t + 1, "amax", include_self=True)
    out = (torch.arange(page, device=p.device) >= filled[:, None])[:, None, :, None]
    k = k_pool.float()
    lo, hi = k.masked_fill(out, math.inf).amin(2), k.masked_fill(out, -math.inf).amax(2)
    scale = (torch.maximum(lo.abs(), hi.abs()).amax(-1).double() / 127).float()
    d = torch.where(scale > 0, scale, torch.ones_like(scale))[..., None].double()
    codes = torch.stack([torch.floor(lo.double() / d), torch.ceil(hi.double() / d)], 2).clamp(-127, 127)
    touched = filled > 0
    s["bounds"].copy_(torch.where(touched[:, None, None, None], codes, s["bounds"].double()).to(torch.int8))
    s["scales"].copy_(torch.where(touched[:, None], scale, s["scales"]))
    return k_pool, v_pool, s["bounds"] * s["scales"][:, :, None, None], s["scales"]


def _sparse(s):
    c = s["case"]
    q, table, ctx = s["q"], s["table"].long(), s["ctx"].long()
    batch, hq, hd = q.shape
    hkv, page, budget = c["hkv"], c["page"], c["budget"]
    per = table.shape[1]
    pages = (ctx + page - 1) // page
    # queries in 16 bits (two signed bytes: 127 * 256 at most), bounds in 8: the score's products and sums are whole
    # numbers below 2^53
    sq = (q.abs().amax(-1).double() / 32512).float()
    qi = torch.round(q / torch.where(sq > 0, sq, torch.ones_like(sq))[..., None]).double()
    qi = qi.view(batch, hkv, hq // hkv, hd)
    bounds = s["bounds"][table].transpose(1, 2)  # [batch][hkv][pages][2][hd]
    dot = torch.matmul(qi.clamp(max=0), bounds[..., 0, :].double().transpose(-1, -2))
    dot = dot + torch.matmul(qi.clamp(min=0), bounds[..., 1, :].double().transpose(-1, -2))
    score = (dot.float() * sq.view(batch, hkv, -1, 1)).amax(2) * s["scales"][table].transpose(1, 2)
    col = torch.arange(per, device=q.device)
    forced = (col < c["sink"]) | (col >= pages[:, None] - c["recent"])
    score = torch.where(forced[:, None], math.inf, score)
    score = torch.where((col < pages[:, None])[:, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget]
    order = torch.where(order < pages[:, None, None], order, per)
    order = torch.cat([order, order.new_full((batch, hkv, max(0, budget - per)), per)], -1).sort(-1).values
    sel = torch.where(order < per, order, -1)
    # attention over the chosen pages
    phys = table.gather(1, order.clamp(max=per - 1).view(batch, -1)).view(batch, hkv, budget)
    head = torch.arange(hkv, device=q.device)[None, :, None]
    k = s["k_pool"][phys, head].float().view(batch, hkv, budget * page, hd)
    v = s["v_pool"][phys, head].float().view(batch, hkv, budget * page, hd)
    at = order[..., None] * page + torch.arange(page, device=q.device)
    live = ((sel >= 0)[..., None] & (at < ctx[:, None, None, None])).view(batch, hkv, 1, -1)
    z = torch.matmul(q.view(batch, hkv, -1, hd) * (1 / math.sqrt(hd)), k.transpose(-1, -2))
    z = z.masked_fill(~live, -math.inf)
    z = torch.exp(z - z.amax(-1, keepdim=True))
    out = torch.matmul(z, v) / z.sum(-1, keepdim=True)
    return out.view(batch, hq, hd), sel.int()


def _lora(s):
    x, a, b, adapter = s["x"], s["a"].float(), s["b"].float(), s["adapter"].long()
    na, r, k = a.shape
    # every adapter's rows at once, then each row keeps its own adapter's
    t = torch.matmul(x, a.view(na * r, k).t()).view(-1, na, r)
    mine = (adapter[:, None] == torch.arange(na, device=x.device))[:, :, None]
    mine = mine & (torch.arange(r, device=x.device) < s["ranks"][:, None])
    t = torch.where(mine, t * s["scales"][:, None], 0)
    return s["y"] + torch.matmul(t.view(-1, na * r), b.transpose(1, 2).reshape(na * r, -1))


def _logits(s):
    x = s["x"].float()
    rows, v = x.shape
    col = torch.arange(s["past"].shape[1], device=x.device)
    said = col < s["past_len"][:, None]
    ids = s["past"].long()
    written = (said & (col >= s["prompt_len"][:, None])).float()
    count = torch.zeros_like(x).scatter_add_(1, ids, written)
    seen = torch.zeros_like(x).scatter_add_(1, ids, said.float()) > 0
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        start = s["bias_start"].long()
        row = torch.searchsorted(start[1:], torch.arange(s["bias"].numel(), device=x.device), right=True)
        add = torch.zeros(rows * v, dtype=torch.float64, device=x.device)
        x = x + add.index_add_(0, row * v + s["bias_ids"].long(), s["bias"].double()).view(rows, v).float()
    if s["mask"] is not None:
        tok = torch.arange(v, device=x.device)
        ok = (s["mask"][:, tok // 32] >> (tok % 32).int()) & 1
        at = s["mask_rows"].long()
        x = torch.where((at[:, None] < 0) | (ok[at.clamp(min=0)] != 0), x, -math.inf)
    return x


# ---------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits, a request at a time
# ---------------------------------------------------------------------------------------------------------


def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None  # whole numbers throughout
    s = prepare(case, seed)
    if op == "append":
        page = case["page"]
        k, v = s["k_pool"].double(), s["v_pool"].double()
        slots = s["slots"].tolist()
        last = {}
        for i, at in enumerate(slots):
            k[at // page, :, at % page] = s["k"][i].double()
            v[at // page, :, at % page] = s["v"][i].double()
            last[at // page] = at % page + 1
        bounds = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=DEV)
        scales = torch.zeros(s["scales"].shape, dtype=torch.float64, device=DEV)
        stored = k.to(s["k_pool"].dtype).double()
        for p, n in last.items():
            lo, hi = stored[p, :, :n].min(1).values, stored[p, :, :n].max(1).values
            scales[p] = torch.maximum(lo.abs(), hi.abs()).max(-1).values / 127
            step = scales[p].float().double()[:, None]
            bounds[p] = torch.stack([(lo / step).floor().clamp(-127, 127) * step,
                                     (hi / step).ceil().clamp(-127, 127) * step], 1)
        return k, v, bounds, scales
    if op == "sparse":
        batch, hq, hkv, hd, page = case["batch"], case["hq"], case["hkv"], case["hd"], case["page"]
        out = torch.zeros((batch, hq, hd), dtype=torch.float64, device=DEV)
        for i, ctx in enumerate(_spread(batch, case["ctx_lo"], case["ctx_hi"])):
            n = _up(ctx, page)
            at = s["table"][i, :n].long()
            for h in range(hkv):
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                q = s["q"][i, heads]
                step = (q.abs().max(-1, keepdim=True).values.double() / 32512).float()
                qi = (q / step).round().double()
                b = s["bounds"][at, h].double()
                dot = torch.maximum(qi[:, None] * b[None, :, 0], qi[:, None] * b[None, :, 1]).sum(-1)
                score = (dot.float() * step).max(0).values * s["scales"][at, h]
                score[:case["sink"]] = math.inf
                score[max(0, n - case["recent"]):] = math.inf
                # the budget's largest, the lower page first among equals
                rank = sorted(range(n), key=list(zip((-score).tolist(), range(n))).__getitem__)
                pick = torch.tensor(sorted(rank[:case["budget"]]), device=DEV)
                k = s["k_pool"][at[pick], h].double().reshape(-1, hd)
                v = s["v_pool"][at[pick], h].double().reshape(-1, hd)
                live = (pick[:, None] * page + torch.arange(page, device=DEV)).reshape(-1) < ctx
                z = (q.double() @ k[live].t() / math.sqrt(hd)).softmax(-1)
                out[i, heads] = z @ v[live]
        return out, None
    if op == "lora":
        out = s["y"].double()
        rows = _adapter_rows(case)
        for a, r in enumerate(_rank_of(case)):
            at = torch.tensor([i for i, x in enumerate(rows) if x == a], dtype=torch.int64, device=DEV)
            t = s["x"][at].double() @ s["a"][a, :r].double().t()
            out[at] += s["scales"][a].double() * (t @ s["b"][a, :, :r].double().t())
        return out
    x = s["x"].double()
    for i in range(case["rows"]):
        n, m = int(s["past_len"][i]), int(s["prompt_len"][i])
        ids, times = s["past"][i, :n].long().unique(return_counts=True)
        rep = s["repetition"][i].double()
        x[i, ids] = torch.where(x[i, ids] > 0, x[i, ids] / rep, x[i, ids] * rep)
        ids, times = s["past"][i, m:n].long().unique(return_counts=True)
        x[i, ids] -= s["frequency"][i].double() * times + s["presence"][i].double()
        if s["bias"] is not None:
            at = slice(int(s["bias_start"][i]), int(s["bias_start"][i + 1]))
            x[i].index_add_(0, s["bias_ids"][at].long(), s["bias"][at].double())
        if s["mask"] is not None and int(s["mask_rows"][i]) >= 0:
            word = s["mask"][int(s["mask_rows"][i])].long() & 0xFFFFFFFF
            bits = (word[:, None] >> torch.arange(32, device=DEV)).reshape(-1)[:case["vocab"]] & 1
            x[i, bits == 0] = -math.inf
    return x
