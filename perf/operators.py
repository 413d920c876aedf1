"""The operators of a decode step over a key/value cache that is held in pages of 4-bit codes, and
the log probabilities at its end: their cases, their inputs, their plain forms and their exact values.

* ``plan``: block tables and slot maps from request lengths. A pool of pages, a table of the pages of
  every request; a call brings the tables in line with the requests' lengths (pages are taken from the
  free list or given back) and writes, for every new token, its position and the slot of its keys and values.
* ``append``: rotary embedding of the new tokens' query and key heads, the keys and values quantised
  to 4 bits (one scale and one minimum a token and head) into their slots.
* ``attention``: the new tokens' queries against the cached keys and values of their request.
* ``logprobs``: log probability of a given token, entropy of the row, the most likely tokens.

Layout of the cache, ``uint8 [pages, kv_heads, page_size * 136]``: granules of 16 tokens, 2176 bytes each:
key codes ``[16][64]``, key parameters ``[16][2]`` bf16 (scale, minimum), then the same for the values.
Byte ``i`` of a token's 64 holds dimensions ``2 i`` (low four bits) and ``2 i + 1``; of the four 16-byte
chunks of token ``r`` of a granule, chunk ``c`` is stored at place ``c ^ ((r >> 1) & 3)``. A code ``n`` stands
for ``scale * n + minimum``.
"""
import math

import torch

own = False

HD = 128                       # dimensions of a head
GRANULE, GRANULE_BYTES = 16, 2176
LOG2_MAX_TOKENS = 16           # largest prompt batch of a drawn case: 2^16 rows


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one user alone, one new token: nothing but latency
        {"name": "plan one request", "op": "plan", "requests": 1, "old_max": 300, "old_min": 300, "new_max": 1, "page": 64, "fixed": True},
        # the decode benchmark's batch at its cache length, every sequence one token on
        {"name": "plan decode 256", "op": "plan", "requests": 256, "old_max": 4096, "old_min": 3900, "new_max": 1, "page": 16, "fixed": True},
        # prompts of many lengths admitted at once, their rows back to back
        {"name": "plan prompts", "op": "plan", "requests": 61, "old_max": 0, "old_min": 0, "new_max": 2048, "page": 64, "fixed": False},
        # the decode benchmark's batch, all heads on one GPU
        {"name": "append decode 256", "op": "append", "rows": 256, "q_heads": 32, "kv_heads": 8, "page": 64, "padding": 0},
        # the prefill benchmark's prompts (8 x 2048 tokens) going into the cache
        {"name": "append prompts 16384", "op": "append", "rows": 16384, "q_heads": 32, "kv_heads": 8, "page": 64, "padding": 37},
        # one user alone, a short conversation, one rank's heads of an 8-way split
        {"name": "attention one short", "op": "attention", "requests": 1, "len_min": 333, "len_max": 333, "q_heads": 4, "kv_heads": 1, "page": 16, "new_max": 1},
        # one micro-batch of the decode benchmark on one rank of 8
        {"name": "attention decode 128x4096", "op": "attention", "requests": 128, "len_min": 4096, "len_max": 4096, "q_heads": 4, "kv_heads": 1, "page": 64, "new_max": 1},
        # a serving mix: lengths from one token to long ones, all heads
        {"name": "attention ragged", "op": "attention", "requests": 48, "len_min": 1, "len_max": 16384, "q_heads": 32, "kv_heads": 8, "page": 32, "new_max": 1},
        # drafted tokens checked at once: up to four rows a request, causal among themselves; long documents
        {"name": "attention drafts long", "op": "attention", "requests": 5, "len_min": 20000, "len_max": 65536, "q_heads": 32, "kv_heads": 8, "page": 64, "new_max": 4},
        # one row of the benchmark's vocabulary, five alternatives
        {"name": "logprobs one row", "op": "logprobs", "rows": 1, "vocab": 128256, "top": 5, "fp32": False, "pad": 0, "banned": 0.0},
        # the decode benchmark's batch
        {"name": "logprobs 256", "op": "logprobs", "rows": 256, "vocab": 128256, "top": 20, "fp32": False, "pad": 0, "banned": 0.0},
        # scoring given text: no alternatives; fp32 logits of an odd vocabulary, half of it forbidden
        {"name": "logprobs scoring fp32", "op": "logprobs", "rows": 1500, "vocab": 32003, "top": 0, "fp32": True, "pad": 5, "banned": 0.5},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "logprobs"])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "plan":
        requests = _spread(rng, 1, 1000)
        fixed = rng.random() < 0.5
        old = _spread(rng, 1, 8192)
        new = rng.choice([1, 1, 2, 5]) if fixed else _spread(rng, 1, max(1, min(4096, 2 ** LOG2_MAX_TOKENS // requests)))
        return {"op": op, "requests": requests, "old_max": old, "old_min": rng.choice([0, old // 2, old]), "new_max": new, "page": page, "fixed": fixed}
    if op == "append":
        kv = rng.choice([1, 2, 3, 8])
        return {"op": op, "rows": _spread(rng, 1, 16384), "q_heads": kv * rng.choice([1, 3, 4]), "kv_heads": kv, "page": page, "padding": rng.choice([0, 1, 9])}
    if op == "attention":
        kv = rng.choice([1, 2, 8])
        group = rng.choice([1, 3, 4, 5, 8, 16])
        longest = _spread(rng, 1, 65536)
        tokens = 1 << 21                              # key rows of all requests and heads together
        requests = _spread(rng, 1, max(1, min(256, tokens // (longest * kv))))
        return {"op": op, "requests": requests, "len_min": rng.choice([1, (longest + 1) // 2, longest]), "len_max": longest,
                "q_heads": kv * group, "kv_heads": kv, "page": page, "new_max": rng.choice([1, 1, 1, 2, 3, 7])}
    rows = _spread(rng, 1, 2000)
    vocab = _spread(rng, 100, max(100, min(160000, 32000000 // rows)))
    return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]), "fp32": rng.random() < 0.4,
            "pad": rng.choice([0, 0, 3, 8]), "banned": rng.choice([0.0, 0.0, 0.3])}


def _pages(length, page):
    return -(-length // page)


# ----------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case, lo, hi, g):
    """Lengths of [lo, hi], even over their logarithm; the longest one is there."""
    n = case["requests"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    v = torch.exp(math.log(max(lo, 1)) + u * (math.log(hi + 0.999) - math.log(max(lo, 1)))).floor().clamp(max(lo, 0), hi) if hi else torch.zeros(n, device="cuda")
    v[-1] = hi
    return v.to(torch.int32)


def _quantise(x):
    """Rows [..., 128] fp32 (values of bf16) -> codes (whole numbers in fp32), scale and minimum (fp32, values of bf16)."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = (high / 15 - low / 15).bfloat16().float()
    codes = torch.where(scale > 0, ((x - low) / scale).round().clamp(0, 15), torch.zeros_like(x))
    return codes, scale, low


def _places():
    r, c = torch.arange(GRANULE, device="cuda").view(16, 1), torch.arange(4, device="cuda").view(1, 4)
    return r.expand(16, 4), c ^ ((r >> 1) & 3)


def _pack(codes, scale, low):
    """Codes [..., 16, 128] with scale and minimum [..., 16, 1] -> the 1088 bytes of a granule's keys or values."""
    b = codes.to(torch.uint8)
    b = (b[..., 0::2] | (b[..., 1::2] << 4)).unflatten(-1, (4, 16))
    r, p = _places()
    b = b[..., r, p, :].flatten(-3)                    # the exchange of places is its own inverse
    params = torch.cat([scale, low], -1).bfloat16().contiguous().view(torch.uint8).flatten(-2)
    return torch.cat([b, params], -1)


def _unpack(half, dtype=torch.float32):
    """1088 bytes -> the values [..., 16, 128] they stand for."""
    r, p = _places()
    b = half[..., :1024].unflatten(-1, (16, 4, 16))[..., r, p, :].flatten(-2)
    codes = torch.stack([b & 15, b >> 4], -1).flatten(-2).to(dtype)
    params = half[..., 1024:].contiguous().view(torch.bfloat16).unflatten(-1, (16, 2)).to(dtype)
    return params[..., :1] * codes + params[..., 1:]


def _filled_cache(pages, heads, page, g):
    """A cache of quantised N(0, 1) keys and values."""
    cache = torch.empty(pages, heads, page // GRANULE, GRANULE_BYTES, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (heads * page * HD))
    for at in range(0, pages, step):
        part = cache[at:at + step]
        for half in (part[..., :1088], part[..., 1088:]):
            x = torch.randn(*part.shape[:3], GRANULE, HD, generator=g, device="cuda").bfloat16().float()
            half.copy_(_pack(*_quantise(x)))
    return cache.view(pages, heads, page * 136)


def _angles(positions):
    """cos and sin [positions, 128] fp32 of the rotary embedding, theta 10000, angles in 64 bits."""
    f = 10000.0 ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "plan":
        n, page = case["requests"], case["page"]
        old = _lengths(case, case["old_min"], case["old_max"], g)
        if case["old_max"]:
            old = torch.where(torch.rand(n, generator=g, device="cuda") < 0.05, 0, old).to(torch.int32)   # places of the batch that are free
        new = torch.randint(1, case["new_max"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        if case["fixed"]:
            new = torch.where(old > 0, new, 0).to(torch.int32)
            rows = n * case["new_max"]
        else:
            rows = n * case["new_max"] + 3
        width = _pages(case["old_max"] + case["new_max"], page) + 1
        total = n * width + 5
        order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
        held = (old + page - 1) // page
        mask = torch.arange(width, device="cuda")[None] < held[:, None]
        taken = order[:n * width].view(n, width)
        table = torch.where(mask, taken, -1).to(torch.int32)
        # the pages that no request holds, in a random order, and room behind them
        key = torch.cat([mask.flatten().to(torch.int32), torch.zeros(5, dtype=torch.int32, device="cuda")])
        at = torch.argsort(key, stable=True)
        free = order[at].contiguous()
        count = (total - held.sum()).to(torch.int32).reshape(1)
        i32 = dict(dtype=torch.int32, device="cuda")
        return {"case": dict(case), "old": old, "zero": torch.zeros_like(old), "new": new, "lens": old + new, "table": table, "held": held.to(torch.int32), "free": free,
                "count": count, "starts": torch.zeros(n + 1, **i32), "slots": torch.zeros(rows, **i32), "positions": torch.zeros(rows, **i32),
                "starts_back": torch.zeros(n + 1, **i32), "none": torch.zeros(0, **i32)}
    if op == "append":
        rows, page = case["rows"], case["page"]
        width = (case["q_heads"] + 2 * case["kv_heads"]) * HD
        qkv = torch.randn(rows + case["padding"], width, generator=g, device="cuda").bfloat16()
        pages = _pages(rows, page) + 2
        cache = torch.zeros(pages, case["kv_heads"], page * 136, dtype=torch.uint8, device="cuda")
        slots = torch.full((rows + case["padding"],), -1, dtype=torch.int32, device="cuda")
        if rows > 512:                                # prompts: runs of tokens, page after page
            order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
            i = torch.arange(rows, device="cuda")
            slots[:rows] = order[i // page] * page + (i % page).to(torch.int32)
        else:                                         # a decode step: every token in a page of its own request
            slots[:rows] = torch.randperm(pages * page, generator=g, device="cuda", dtype=torch.int32)[:rows]
        longest = 8192
        positions = torch.randint(0, longest, (rows + case["padding"],), generator=g, device="cuda", dtype=torch.int32)
        return {"case": dict(case), "qkv": qkv, "slots": slots, "positions": positions, "angles": _angles(longest), "cache": cache, "out": torch.zeros_like(qkv)}
    if op == "attention":
        page, n = case["page"], case["requests"]
        lens = _lengths(case, case["len_min"], case["len_max"], g)
        width = _pages(case["len_max"], page)
        held = (lens + page - 1) // page
        pages = int(held.sum()) + 1
        shuffle = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
        column = torch.arange(width, device="cuda")[None]
        dense = (held.cumsum(0) - held)[:, None] + column
        table = torch.where(column < held[:, None], shuffle[dense.clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
        cache = _filled_cache(pages, case["kv_heads"], page, g)
        many = case["new_max"]
        new = torch.minimum(torch.randint(1, many + 1, (n,), generator=g, device="cuda", dtype=torch.int32), lens)
        starts = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), new.cumsum(0).to(torch.int32)])
        rows = n * many
        q = torch.randn(rows, (case["q_heads"] + 2 * case["kv_heads"]) * HD, generator=g, device="cuda").bfloat16()[:, :case["q_heads"] * HD]
        return {"case": dict(case), "q": q, "cache": cache, "table": table, "lens": lens, "new": new, "starts": starts,
                "out": torch.zeros(rows, case["q_heads"] * HD, dtype=torch.bfloat16, device="cuda"), "scratch": None}
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn(rows, vocab + case["pad"], generator=g, device="cuda").mul_(2.5)
    if case["banned"]:
        logits = torch.where(torch.rand(rows, vocab + case["pad"], generator=g, device="cuda") < case["banned"], -math.inf, logits)
    logits[:, vocab // 3] = 6.0                       # no row without a token that is allowed
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    ids = torch.where(torch.isfinite(logits.gather(1, ids[:, None])[:, 0]), ids, vocab // 3)
    if not case["fp32"]:
        logits = logits.bfloat16()
    return {"case": dict(case), "logits": logits[:, :vocab], "ids": ids, "out": None, "scratch": None}


# ------------------------------------------------------------------- runs
def run(state):
    return {"plan": _plan, "append": _append, "attention": _attention, "logprobs": _logprobs}[state["case"]["op"]](state)


def _plan(s):
    """The step's pages are taken and its rows laid out; then the step is taken back, its pages returned."""
    c = s["case"]
    per_request = c["new_max"] if c["fixed"] else 0
    call = _own_plan if own else _plain_plan
    call(s["lens"], s["new"], s["table"], s["held"], s["free"], s["count"], s["starts"], s["slots"], s["positions"], c["page"], per_request)
    call(s["old"], s["zero"], s["table"], s["held"], s["free"], s["count"], s["starts_back"], s["none"], s["none"], c["page"], 0)
    return {"slots": s["slots"], "positions": s["positions"], "starts": s["starts"], "table": s["table"], "held": s["held"],
            "free": s["free"], "count": s["count"]}


def _own_plan(lens, new, table, held, free, count, starts, slots, positions, page, per_request):
    from dynaflow_b200 import ops

    ops.page_plan(lens, new, table, held, free, count, starts, slots, positions, page_size=page, rows_per_request=per_request)


def _plain_plan(lens, new, table, held, free, count, starts, slots, positions, page, per_request):
    n, width = table.shape
    dev = table.device
    column = torch.arange(width, device=dev)[None]
    need = (lens + page - 1) // page
    back, more = (held - need).clamp(min=0), (need - held).clamp(min=0)
    back_at, more_at = back.cumsum(0) - back, more.cumsum(0) - more
    returned = back.sum()
    # pages given back go on top of the free list, the first of them uppermost; a place past its end takes what is not written
    size = free.numel()
    leaving = (column >= need[:, None]) & (column < held[:, None])
    place = count + returned - 1 - (back_at[:, None] + column - need[:, None])
    grown = torch.cat([free, free.new_zeros(1)]).scatter(0, torch.where(leaving, place, size).flatten(), table.flatten())[:size]
    top = count + returned
    enough = more.sum() <= top
    coming = (column >= held[:, None]) & (column < need[:, None]) & enough
    from_ = (top - 1 - (more_at[:, None] + column - held[:, None])).clamp(0, size - 1)
    table.copy_(torch.where(coming, grown[from_.flatten()].view(n, width), torch.where(leaving, -1, table)))
    held.copy_(torch.where((need <= held) | enough, need, held))
    free.copy_(grown)
    count.copy_(top - torch.where(enough, more.sum(), 0))
    if per_request:
        starts.copy_(torch.arange(n + 1, device=dev) * per_request)
    else:
        starts.copy_(torch.cat([new.new_zeros(1), new.cumsum(0)]))
    row = torch.arange(slots.numel(), device=dev, dtype=torch.int32)
    if row.numel():
        request = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=n - 1)
        i = row - starts[request]
        fresh = i < new[request]
        position = torch.where(fresh, lens[request] - new[request] + i, 0)
        column_of = position // page
        known = fresh & (column_of < held[request])
        slots.copy_(torch.where(known, table[request, column_of.clamp(max=width - 1)] * page + position % page, -1))
        positions.copy_(position)


def _append(s):
    c = s["case"]
    hq, hkv, page = c["q_heads"], c["kv_heads"], c["page"]
    if own:
        from dynaflow_b200 import ops

        ops.rope_append_paged4(s["qkv"], s["positions"], s["slots"], s["angles"], hq, hkv, s["cache"], page_size=page, out=s["out"])
        return {"out": s["out"]}
    # every row that has a slot: rotated queries, and keys and values as the cache holds them from now on
    x = s["qkv"].float().view(-1, hq + 2 * hkv, HD)
    angle = s["angles"][s["positions"].long()][:, None]
    cos, sin = angle[..., :64], angle[..., 64:]
    turn, values = x[:, :hq + hkv], x[:, hq + hkv:]
    a, b = turn[..., :64], turn[..., 64:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).bfloat16().float()
    stored = torch.stack([turned[:, hq:], values], 2)                   # [rows, kv heads, key or value, 128]
    codes, scale, low = _quantise(stored)
    stands_for = scale * codes + low
    rows = torch.cat([turned[:, :hq], stands_for[:, :, 0], stands_for[:, :, 1]], 1).bfloat16().flatten(1)
    real = s["slots"] >= 0
    s["out"].copy_(torch.where(real[:, None], rows, s["out"]))
    # into the cache: a token's 64 bytes and its parameters, byte by byte at their places; padding goes to a page that is not kept
    cache = s["cache"]
    padded = torch.cat([cache.view(-1, hkv, page // 16, GRANULE_BYTES), cache.new_zeros(1, hkv, page // 16, GRANULE_BYTES)])
    slot = torch.where(real, s["slots"].long(), cache.shape[0] * page)
    where, r = (slot // page, slot % page // 16), slot % 16
    b = codes.to(torch.uint8)
    b = b[..., 0::2] | (b[..., 1::2] << 4)
    chunk = torch.arange(64, device=b.device) // 16 ^ ((r[:, None] >> 1) & 3)
    byte = r[:, None] * 64 + chunk * 16 + torch.arange(64, device=b.device) % 16                     # [rows, 64]
    params = torch.cat([scale, low], -1).bfloat16().contiguous().view(torch.uint8)
    byte = torch.cat([byte, 1024 + r[:, None] * 4 + torch.arange(4, device=b.device)], 1)
    byte = torch.cat([byte, 1088 + byte], 1)                                                         # [rows, 136]
    data = torch.cat([b, params], -1).flatten(2)                                                     # [rows, kv heads, 136]
    head = torch.arange(hkv, device=b.device)
    padded[where[0][:, None, None], head[None, :, None], where[1][:, None, None], byte[:, None]] = data
    cache.copy_(padded[:-1].view_as(cache))
    return {"out": s["out"]}


def _attention(s):
    c = s["case"]
    hq, hkv, page, many = c["q_heads"], c["kv_heads"], c["page"], c["new_max"]
    if own:
        from dynaflow_b200 import ops

        if s["scratch"] is None:
            s["scratch"] = ops.attention_paged4_workspace(c["requests"], hq, hkv, many, s["q"].device)
        if many == 1:
            ops.attention_paged4(s["q"], s["cache"], s["table"], s["lens"], s["out"], s["scratch"], page_size=page)
        else:
            ops.attention_paged4(s["q"], s["cache"], s["table"], s["lens"], s["out"], s["scratch"], page_size=page, row_starts=s["starts"], new_lens=s["new"], max_new=many)
        return {"out": s["out"]}
    n, width = s["table"].shape
    group = hq // hkv
    granules = s["cache"][s["table"].clamp(min=0)].view(n, width, hkv, page // 16, GRANULE_BYTES).transpose(1, 2)    # [n, kv heads, width, ...]
    keys = _unpack(granules[..., :1088]).flatten(2, 4)                                                              # [n, kv heads, width * page, 128]
    values = _unpack(granules[..., 1088:]).flatten(2, 4)
    i = torch.arange(many, device=keys.device)[None]
    row = torch.where(i < s["new"][:, None], s["starts"][:-1, None] + i, s["q"].shape[0])                            # [n, many]; absent: past the last row
    q = torch.cat([s["q"], s["q"].new_zeros(1, hq * HD)])[row].float().view(n, many, hkv, group, HD).transpose(1, 2)
    scores = (q.reshape(n, hkv, many * group, HD) @ keys.transpose(-1, -2)).view(n, hkv, many, group, -1) * HD ** -0.5
    limit = s["lens"][:, None] - s["new"][:, None] + i + 1
    seen = torch.arange(width * page, device=keys.device)[None, None] < limit[..., None]                             # [n, many, keys]
    scores = torch.where(seen[:, None, :, None], scores, -math.inf)
    weight = torch.exp(scores - scores.amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    got = (weight.view(n, hkv, many * group, -1) @ values).view(n, hkv, many, group, HD).transpose(1, 2).reshape(n * many, hq * HD).bfloat16()
    padded = torch.cat([s["out"], s["out"].new_zeros(1, hq * HD)])
    padded[row.flatten()] = got
    s["out"].copy_(padded[:-1])
    return {"out": s["out"]}


def _logprobs(s):
    c = s["case"]
    if own:
        from dynaflow_b200 import ops

        if s["out"] is None:
            s["out"] = ops.token_logprobs_out(c["rows"], c["top"], s["logits"].device)
            s["scratch"] = ops.token_logprobs_workspace(c["rows"], c["vocab"], c["top"], s["logits"].device)
        ops.token_logprobs(s["logits"], s["ids"], c["top"], out=s["out"], workspace=s["scratch"])
        logprob, entropy, top_ids, top_logprobs = s["out"]
    else:
        x = s["logits"].float()
        high = x.amax(-1, keepdim=True)
        e = torch.exp(x - high)
        total = e.sum(-1, keepdim=True, dtype=torch.float64)
        log_total = high + total.log()
        logprob = (x.gather(1, s["ids"][:, None]) - log_total)[:, 0].float()
        part = torch.where(e > 0, e * (x - high), 0).sum(-1, dtype=torch.float64)
        entropy = (total.log()[:, 0] - part / total[:, 0]).float()
        if c["top"]:
            value, at = torch.sort(x, dim=-1, descending=True, stable=True)
            top_ids = at[:, :c["top"]].to(torch.int32)
            top_logprobs = (value[:, :c["top"]] - log_total).float()
    if not c["top"]:
        return {"logprob": logprob, "entropy": entropy}
    return {"logprob": logprob, "entropy": entropy, "top_ids": top_ids, "top_logprobs": top_logprobs}


# ------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "plan":
        n, new = case["requests"], (1 + case["new_max"]) / 2
        rows = n * case["new_max"]
        pages = n * max(new / case["page"], min(1.0, new / case["page"]))
        return {"bytes": 2 * n * 16 + 4 * (n + 1) + rows * 8 + pages * 16, "flops": 0}
    if op == "append":
        row = (case["q_heads"] + 2 * case["kv_heads"]) * HD * 2
        return {"bytes": case["rows"] * (2 * row + 136 * case["kv_heads"] + 512 + 8), "flops": case["rows"] * (case["q_heads"] + 2 * case["kv_heads"]) * HD * 6}
    if op == "attention":
        lo, hi, n = case["len_min"], case["len_max"], case["requests"]
        mean = hi if lo == hi else (hi - lo) / (math.log(hi) - math.log(max(lo, 1)))
        keys = mean * (n - 1) + hi
        rows = n * (1 + case["new_max"]) / 2
        return {"bytes": keys * case["kv_heads"] * 136 + rows * case["q_heads"] * HD * 4 + keys / case["page"] * 4,
                "flops": keys * (1 + case["new_max"]) / 2 * case["q_heads"] * HD * 4}
    size = case["rows"] * case["vocab"]
    return {"bytes": size * (4 if case["fp32"] else 2) + case["rows"] * (16 + 8 * case["top"]), "flops": size * 5}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The same from the definitions, in 64 bits, a request, head or block of rows at a time."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None                                    # whole numbers only
    if op == "append":
        hq, hkv = case["q_heads"], case["kv_heads"]
        out = torch.zeros(s["qkv"].shape, dtype=torch.float64, device="cuda")
        rows = (s["slots"] >= 0).nonzero()[:, 0]
        angle = s["positions"][rows].double()[:, None] * torch.exp(torch.arange(64, device="cuda", dtype=torch.float64) * (-math.log(10000.0) / 64))
        for h in range(hq + 2 * hkv):
            x = s["qkv"][rows, h * HD:(h + 1) * HD].double()
            if h < hq + hkv:
                z = torch.complex(x[:, :64], x[:, 64:]) * torch.polar(torch.ones_like(angle), angle)
                x = torch.cat([z.real, z.imag], 1)
            if h >= hq:
                x = x.bfloat16().double()              # a key or value is a bf16 number before it is quantised
                low, high = x.min(1, keepdim=True).values, x.max(1, keepdim=True).values
                step = ((high - low) / 15).bfloat16().double()
                x = low + step * torch.clamp(torch.round((x - low) / step), 0, 15)
            out[rows, h * HD:(h + 1) * HD] = x
        return {"out": out}
    if op == "attention":
        hq, hkv, page = case["q_heads"], case["kv_heads"], case["page"]
        if case["requests"] * hkv > 3000 or s["lens"].sum().item() * hkv > 1 << 23:
            return None
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        chunk_of = torch.arange(64, device="cuda") // 16
        token = torch.arange(page, device="cuda")
        byte = (token % 16 * 64)[:, None] + ((chunk_of[None] ^ (token // 2 % 4)[:, None]) * 16) + torch.arange(64, device="cuda") % 16
        byte = byte + (token // 16 * GRANULE_BYTES)[:, None]
        param = (token // 16 * GRANULE_BYTES + 1024 + token % 16 * 4)[:, None] + torch.arange(4, device="cuda")
        lens, new, starts = s["lens"].tolist(), s["new"].tolist(), s["starts"].tolist()
        for b in range(case["requests"]):
            pages = s["cache"][s["table"][b, :_pages(lens[b], page)].long()]
            for k in range(hkv):
                sides = []
                for at in (0, 1088):
                    p = pages[:, k]
                    raw = p[:, (byte + at).flatten()].view(-1, 64)
                    two = p[:, (param + at).flatten()].contiguous().view(torch.bfloat16).view(-1, 2).double()
                    codes = torch.empty(raw.shape[0], HD, dtype=torch.float64, device="cuda")
                    codes[:, 0::2], codes[:, 1::2] = (raw % 16).double(), (raw // 16).double()
                    sides.append((codes * two[:, :1] + two[:, 1:])[:lens[b]])
                for j in range(new[b]):
                    last = lens[b] - new[b] + j + 1
                    r = starts[b] + j
                    heads = slice(k * (hq // hkv) * HD, (k + 1) * (hq // hkv) * HD)
                    q = s["q"][r, heads].double().view(-1, HD)
                    p = torch.softmax(q @ sides[0][:last].T / math.sqrt(HD), -1)
                    out[r, heads] = (p @ sides[1][:last]).flatten()
        return {"out": out}
    top = case["top"]
    found = {"logprob": [], "entropy": [], "top_logprobs": []}
    for at in range(0, case["rows"], 128):
        x = torch.log_softmax(s["logits"][at:at + 128].double(), -1)
        found["logprob"].append(x.gather(1, s["ids"][at:at + 128, None])[:, 0])
        found["entropy"].append(-torch.special.xlogy(x.exp(), x.exp()).sum(-1))
        if top:
            found["top_logprobs"].append(x.sort(-1, descending=True).values[:, :top])
    got = {k: torch.cat(v) for k, v in found.items() if v}
    if top:
        got["top_ids"] = None
    return got
