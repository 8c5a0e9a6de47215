"""What is measured of the chunked path over the paged cache: prompts (and whatever a request brings at once) enter the
cache in chunks of new tokens, many requests to a call, their tokens packed one request behind the other.

Four operators, in the order a step uses them:

* plan    block tables and slot maps from request lengths: the cache is cut back to the rows each request keeps, pages
          for the new tokens are taken from the free list (lowest first, requests in order), and every new token gets
          its slot (page * page_len + row), its position and its request.
* append  K and V rows of the packed tokens to their slots of one layer.
* chunk   attention of the packed tokens over their requests' cache rows, each token up to and including itself.
* window  the same with a sliding window, behind which only the first few rows (sinks) stay visible.

`own` false: elementary torch operations; `own` true: the calls a user makes of `subspec_b200`.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, batch, new, cached, *, page_len=16, heads=28, kv_heads=4, dim=128, dtype="bf16", long=0, window=0,
          sinks=0, mix=1):
    """`new`, `cached`: the most tokens a request brings and has; `long`: the tokens of the last request, which brings a
    chunk while the others bring `new`; `mix`: which ragged lengths (0: all of them the most)."""
    c = dict(op=op, batch=batch, new=new, cached=cached, page_len=page_len, heads=heads, kv_heads=kv_heads, dim=dim,
             dtype=dtype, long=long, window=window, sinks=sinks, mix=mix)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one step of a batch of 64: a token each, behind caches of up to 4k rows
        _case("plan_decode_64", "plan", 64, 1, 4031),
        # a full server takes in prompts: 128 requests, up to 2k new tokens each
        _case("plan_prompts_128", "plan", 128, 2048, 2048),
        # the K / V rows of one token for each of 64 requests
        _case("append_decode_64", "append", 64, 1, 4031),
        # prompts' rows: 16 requests, about 12k tokens, eight KV heads
        _case("append_prompts_16", "append", 16, 1024, 500, heads=32, kv_heads=8),
        # a lone request's next token behind 4k rows: latency
        _case("chunk_decode_1", "chunk", 1, 1, 4095, mix=0),
        # the next token of 64 requests with ragged caches of up to 8k rows: bandwidth
        _case("chunk_decode_64", "chunk", 64, 1, 8191),
        # three short odd chunks of a small model in fp16, pages that are no power of two
        _case("chunk_odd_3", "chunk", 3, 37, 1000, page_len=24, heads=14, kv_heads=2, dim=64, dtype="fp16", mix=3),
        # prompts from their first token on, ragged
        _case("chunk_prompts_6", "chunk", 6, 2500, 0, mix=5),
        # a chunk of a long document
        _case("chunk_long_1", "chunk", 1, 2048, 30720, mix=0),
        # one request's chunk among 32 requests that each bring a token
        _case("chunk_mixed_33", "chunk", 33, 1, 4000, heads=32, kv_heads=8, long=1024),
        # the next token of 48 requests, a window of 1024 rows and four sinks over long caches
        _case("window_decode_48", "window", 48, 1, 16000, heads=32, kv_heads=8, window=1024, sinks=4),
        # two long prompts under the same window
        _case("window_prompts_2", "window", 2, 6000, 0, dtype="fp16", window=1024, sinks=4, mix=7),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "chunk", "chunk", "chunk", "window", "window"])
    page_len = rng.choice([8, 16, 16, 16, 24, 32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    dim, dtype = rng.choice([64, 128, 128]), rng.choice(["bf16", "bf16", "fp16"])
    mix = rng.randrange(1, 1 << 20)
    shape = dict(page_len=page_len, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=dtype, mix=mix)
    if op == "plan":
        return _case(None, op, _between(rng, 1, 128), _between(rng, 1, 2048), _between(rng, 1, 4096), **shape)
    if op == "append":
        batch = _between(rng, 1, 64)
        return _case(None, op, batch, _between(rng, 1, max(1, 12000 // batch)), _between(rng, 1, 4096), **shape)
    more = {}
    if op == "window":
        more = dict(window=_between(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 4, 16, 64]))
    kind = rng.choice(["decode", "chunks", "mixed"])
    if kind == "decode":
        batch = _between(rng, 1, 64)
        return _case(None, op, batch, 1, _between(rng, 1, 8191), **shape, **more)
    if kind == "mixed":
        batch = _between(rng, 2, 33 * 32 // max(32, kv_heads * group))
        return _case(None, op, batch, 1, _between(rng, 1, 4000), long=_between(rng, 2, 1024), **shape, **more)
    most = 28 * 2048 * 30720 // (kv_heads * group)  # pairs of query and cache row a head
    new, cached = _between(rng, 1, 2500), rng.choice([0, _between(rng, 1, 16000)])
    new = max(1, min(new, most // (cached + 2500)))
    batch = min(_between(rng, 1, 8), max(1, most // (new * (cached + new))))
    return _case(None, op, batch, new, cached, **shape, **more)


def _lengths(case):
    """(new tokens, cached rows) of every request: they belong to the case."""
    rng, batch = random.Random(case["mix"]), case["batch"]
    if case["mix"] == 0:
        new, cached = [case["new"]] * batch, [case["cached"]] * batch
    else:
        new = [rng.randint((case["new"] + 1) // 2, case["new"]) for _ in range(batch)]
        cached = [rng.randint(case["cached"] // 4, case["cached"]) for _ in range(batch)]
    if case["long"]:
        new[-1], cached[-1] = case["long"], case["cached"] // 8
    return new, cached


def _ceil(a, b):
    return -(-a // b)


def prepare(case, seed):
    dev, gen = torch.device("cuda"), torch.Generator("cuda")
    gen.manual_seed(seed)
    new, cached = _lengths(case)
    batch, pl, dtype = case["batch"], case["page_len"], _TYPES[case["dtype"]]
    total = [n + c for n, c in zip(new, cached)]
    width = max(_ceil(t, pl) for t in total) + 1
    i32 = dict(dtype=torch.int32, device=dev)
    s = dict(op=case["op"], page_len=pl, n_new=torch.tensor(new, **i32), cached=torch.tensor(cached, **i32),
             kv_len=torch.tensor(total, **i32), tokens=sum(new), max_q=max(new), max_kv=max(total), layer=1,
             window=case["window"], sinks=case["sinks"])
    # physical pages in no order; a request's list holds what its rows need (before a plan: its cached rows')
    held = [_ceil(c if case["op"] == "plan" else t, pl) for c, t in zip(cached, total)]
    pages = sum(_ceil(t, pl) for t in total) + 32 + (sum(new) // pl) // 8
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    flat = torch.full((batch, width), -1, dtype=torch.int32)
    at = torch.arange(width)[None, :] < torch.tensor(held)[:, None]
    flat[at] = order[:sum(held)].cpu()
    s["page_table"], s["n_pages"], s["pages"] = flat.to(dev), torch.tensor(held, **i32), pages
    if case["op"] == "plan":
        free = torch.ones(_ceil(pages, 32) * 32, dtype=torch.int64)
        free[order[:sum(held)].cpu().long()] = 0
        word = (free.view(-1, 32) << torch.arange(32)).sum(1)
        s["free_mask"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).to(dev)
        s["kv_len"] = s["cached"].clone()
        if own:
            from subspec_b200.pages import DevicePagePool

            s["pool"] = DevicePagePool(batch, pages, pl, width, dev, max_append=sum(new))
            for name in ("free_mask", "page_table", "n_pages", "kv_len"):
                getattr(s["pool"], name).copy_(s[name])
        return s
    h, hq, d = case["kv_heads"], case["heads"], case["dim"]
    s["q_indptr"] = torch.tensor([sum(new[:b]) for b in range(batch + 1)], **i32)
    s["cache"] = torch.empty(2, pages, 2, pl, h, d, dtype=dtype, device=dev).normal_(generator=gen)
    # the rows of the fused q / k / v projection
    qkv = torch.empty(sum(new), hq + 2 * h, d, dtype=dtype, device=dev).normal_(generator=gen)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + h], qkv[:, hq + h:]
    if case["op"] == "append":
        b = torch.repeat_interleave(torch.arange(batch), torch.tensor(new))
        pos = torch.cat([torch.arange(c, c + n) for n, c in zip(new, cached)])
        s["slot_map"] = (flat[b, pos // pl].long() * pl + pos % pl).to(dev)
    return s


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "append": _plain_append, "chunk": _plain_attention, "window": _plain_attention}[state["op"]](state)


def _run_own(s):
    if s["op"] == "plan":
        pool = s["pool"]
        plan = pool.plan_chunks(s["n_new"], set_len=s["cached"])
        return dict(q_indptr=plan.q_indptr, slot_map=plan.slot_map, positions=plan.positions,
                    batch_indices=plan.batch_indices, page_table=pool.page_table, n_pages=pool.n_pages,
                    kv_len=pool.kv_len, free_mask=pool.free_mask)
    from subspec_b200 import attention

    if s["op"] == "append":
        attention.append_paged_kv_slots(s["cache"], s["layer"], s["k"], s["v"], slot_map=s["slot_map"])
        return s["cache"][s["layer"]]
    plan = dict(page_table=s["page_table"], kv_len=s["kv_len"], q_indptr=s["q_indptr"], max_q_len=s["max_q"])
    if s["op"] == "chunk":
        return attention.chunk_attention_paged(s["q"], s["cache"], s["layer"], **plan)
    return attention.window_attention_paged(s["q"], s["cache"], s["layer"], window=s["window"], sinks=s["sinks"], **plan)


def _plain_plan(s):
    dev, pl, table, n_pages, free = s["page_table"].device, s["page_len"], s["page_table"], s["n_pages"], s["free_mask"]
    column = torch.arange(table.shape[1], device=dev)[None, :]
    bits = torch.arange(32, device=dev)
    is_free = ((free.long()[:, None] >> bits) & 1).reshape(-1)
    # the cache is cut back: pages behind the kept rows are free again
    keep = torch.minimum(n_pages.long(), (s["cached"].long() + pl - 1) // pl)
    back = (column >= keep[:, None]) & (column < n_pages[:, None])
    is_free[table[back].long()] = 1
    table.masked_fill_(back, -1)
    # the pages of the new rows: the lowest free ones, requests in order
    length = s["cached"].long() + s["n_new"].long()
    need = (length + pl - 1) // pl
    first = torch.cumsum(need - keep, 0) - (need - keep)
    lowest = torch.nonzero(is_free[:s["pages"]]).reshape(-1)
    fresh = (column >= keep[:, None]) & (column < need[:, None])
    given = lowest[(first[:, None] + column - keep[:, None])[fresh]]
    table[fresh] = given.to(torch.int32)
    is_free[given] = 0
    word = (is_free.view(-1, 32) << bits).sum(1)
    free.copy_(torch.where(word >= 1 << 31, word - (1 << 32), word))
    n_pages.copy_(need)
    s["kv_len"].copy_(length)
    # every new token's request, position and slot
    indptr = torch.zeros(len(need) + 1, dtype=torch.int64, device=dev)
    indptr[1:] = torch.cumsum(s["n_new"].long(), 0)
    token = torch.arange(s["tokens"], device=dev)
    request = (token[:, None] >= indptr[None, 1:]).sum(1)
    position = s["cached"].long()[request] + token - indptr[request]
    slot = table[request, position // pl].long() * pl + position % pl
    return dict(q_indptr=indptr.to(torch.int32), slot_map=slot, positions=position.to(torch.int32),
                batch_indices=request.to(torch.int32), page_table=table, n_pages=n_pages, kv_len=s["kv_len"],
                free_mask=free)


def _plain_append(s):
    cache, slot = s["cache"], s["slot_map"]
    page, row = slot // s["page_len"], slot % s["page_len"]
    cache[s["layer"], page, 0, row] = s["k"]
    cache[s["layer"], page, 1, row] = s["v"]
    return cache[s["layer"]]


def _plain_attention(s):
    """All requests at once, padded to the longest."""
    cache, q, pl = s["cache"], s["q"], s["page_len"]
    dev, h, d = q.device, cache.shape[4], cache.shape[5]
    group = q.shape[1] // h
    begin, n, kv_len = s["q_indptr"][:-1].long(), s["n_new"].long(), s["kv_len"].long()
    i, j = torch.arange(s["max_q"], device=dev), torch.arange(s["max_kv"], device=dev)
    page = s["page_table"].long()[:, j // pl].clamp(min=0)
    k = cache[s["layer"], page, 0, j % pl].float().permute(0, 2, 3, 1)            # [request, kv head, dim, row]
    v = cache[s["layer"], page, 1, j % pl].float().permute(0, 2, 1, 3)            # [request, kv head, row, dim]
    at = torch.minimum(begin[:, None] + i, begin[:, None] + n[:, None] - 1)
    rows = q[at].float().view(len(n), s["max_q"], h, group, d).permute(0, 2, 3, 1, 4).reshape(len(n), h, -1, d)
    score = (rows @ k).view(len(n), h, group, s["max_q"], -1).mul_(1 / math.sqrt(d))
    place = (kv_len - n)[:, None, None] + torch.minimum(i, n[:, None] - 1)[:, :, None]
    seen = j <= place
    if s["op"] == "window":
        seen &= (j > place - s["window"]) | (j < s["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1).view(len(n), h, -1, 1)
    out = (score.view(len(n), h, -1, score.shape[-1]) @ v) / total
    out = out.view(len(n), h, group, s["max_q"], d).permute(0, 3, 1, 2, 4).reshape(len(n), s["max_q"], -1, d)
    token = torch.arange(s["tokens"], device=dev)
    request = (token[:, None] >= begin[None, 1:]).sum(1)
    return out[request, token - begin[request]].to(q.dtype)


def _seen_pairs(new, cached, window, sinks):
    """Pairs of query and visible row of one request."""
    if not window:
        return new * cached + new * (new + 1) // 2
    return sum(min(window, p + 1) + min(sinks, max(0, p + 1 - window)) for p in range(cached, cached + new))


def work(case):
    new, cached = _lengths(case)
    pl, h, hq, d = case["page_len"], case["kv_heads"], case["heads"], case["dim"]
    tokens = sum(new)
    if case["op"] == "plan":
        fresh = sum(_ceil(n + c, pl) - _ceil(c, pl) for n, c in zip(new, cached))
        # lengths in, page list entries, lengths and offsets out, 16 bytes a token, the free pages' bits
        return {"bytes": 8 * case["batch"] + 4 * fresh + 12 * case["batch"] + 16 * tokens + fresh // 4, "flops": tokens}
    if case["op"] == "append":
        return {"bytes": tokens * (8 + 2 * 2 * h * d * 2), "flops": 0}
    pairs = sum(_seen_pairs(n, c, case["window"], case["sinks"]) for n, c in zip(new, cached))
    rows = sum(n + c for n, c in zip(new, cached))
    if case["window"]:
        rows = sum(min(n + c, n + case["window"] - 1 + case["sinks"]) for n, c in zip(new, cached))
    return {"bytes": 2 * tokens * hq * d * 2 + 2 * rows * h * d * 2, "flops": 4 * d * hq * pairs}


def exact(case, seed):
    """From the definition, a request at a time: whole numbers in Python, attention in 64 bits."""
    s = prepare(case, seed)
    new, cached = _lengths(case)
    pl = case["page_len"]
    if case["op"] == "plan":
        return _exact_plan(s, new, cached, pl)
    q, cache, layer = s["q"], s["cache"], s["layer"]
    if case["op"] == "append":
        # rows by their place in the layer's memory: page p holds page_len rows of K, then page_len rows of V
        place = s["slot_map"] // pl * 2 * pl + s["slot_map"] % pl
        flat = cache[layer].double().view(-1, *s["k"].shape[1:])
        flat.index_copy_(0, place, s["k"].double())
        flat.index_copy_(0, place + pl, s["v"].double())
        return flat.view(cache[layer].shape)
    h, d = case["kv_heads"], case["dim"]
    group = case["heads"] // h
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    first = 0
    for b, (n, c) in enumerate(zip(new, cached)):
        kv = torch.cat([cache[layer, p] for p in s["page_table"][b, :_ceil(n + c, pl)].tolist()], 1)[:, :n + c].double()
        step = max(1, (1 << 26) // (group * (n + c)))
        for lo in range(0, n, step):
            hi = min(n, lo + step)
            place = torch.arange(c + lo, c + hi, device=q.device)[:, None]
            row = torch.arange(c + hi, device=q.device)[None, :]
            hidden = row > place
            if case["window"]:
                hidden |= (place - row >= case["window"]) & (row >= case["sinks"])
            for g in range(h):
                x = q[first + lo:first + hi, g * group:(g + 1) * group].double().transpose(0, 1)
                w = torch.softmax((x @ kv[0, :c + hi, g].T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                out[first + lo:first + hi, g * group:(g + 1) * group] = (w @ kv[1, :c + hi, g]).transpose(0, 1)
        first += n
    return out


def _exact_plan(s, new, cached, pl):
    taken = [[p for p in row if p >= 0] for row in s["page_table"].tolist()]
    busy = {p for row in taken for p in row}
    free = iter([p for p in range(s["pages"]) if p not in busy])
    out = dict(q_indptr=[0], slot_map=[], positions=[], batch_indices=[])
    for b, (n, c) in enumerate(zip(new, cached)):
        taken[b] += [next(free) for _ in range(_ceil(n + c, pl) - len(taken[b]))]
        for p in range(c, c + n):
            out["slot_map"].append(taken[b][p // pl] * pl + p % pl)
            out["positions"].append(p)
            out["batch_indices"].append(b)
        out["q_indptr"].append(out["q_indptr"][-1] + n)
    left = set(free)
    words = [sum(1 << (i % 32) for i in range(w, w + 32) if i in left or i >= s["pages"]) for w in range(0, _ceil(s["pages"], 32) * 32, 32)]
    width = s["page_table"].shape[1]
    i32 = dict(dtype=torch.int32, device=s["page_table"].device)
    return dict(q_indptr=torch.tensor(out["q_indptr"], **i32),
                slot_map=torch.tensor(out["slot_map"], dtype=torch.int64, device=i32["device"]),
                positions=torch.tensor(out["positions"], **i32), batch_indices=torch.tensor(out["batch_indices"], **i32),
                page_table=torch.tensor([row + [-1] * (width - len(row)) for row in taken], **i32),
                n_pages=torch.tensor([len(row) for row in taken], **i32),
                kv_len=torch.tensor([n + c for n, c in zip(new, cached)], **i32),
                free_mask=torch.tensor([w - (1 << 32) if w >= 1 << 31 else w for w in words], **i32))
