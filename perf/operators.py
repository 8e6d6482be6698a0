"""The operators that keep and read a serving program's key / value cache: what their speed is judged by.

Attention over the whole prompts of several requests packed one behind the other (prompt_attention), attention of one new
token per request over a paged cache whose requests share long prefixes (paged_attention), the writing of new keys and
values into the cache's pages (cache_write), the step of the page tables between two tokens - requests released, forked
and admitted, pages handed out, half-filled pages copied (cache_step) - and the moving of live pages to the front of the
cache (cache_compact).

The cache of a layer is two tensors [pages][key / value heads][tokens of a page][head size]; all layers together are a pool
[planes][pages][...], two planes a layer.  Row s of `table` lists the pages of request s in order, -1 behind the last one;
`refs` counts the rows that use a page.

listed() holds calls of the ranges' ends and middles, draw() others of the same ranges.  run() computes an operator with
elementary torch operations in 32 bits, or, where `own` is set, calls the package.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # the last 40 tokens of a prompt that is taken in pieces, behind 2900 that are in place: few rows, long keys
        {"name": "prompt_piece_40_of_2940", "op": "prompt", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "seqs": 1,
         "longest": 40, "context": 2900, "causal": True, "fused": False},
        # prompts of 24 users packed together, from nothing to 901 tokens, heads of 64, taken out of one projection's result
        {"name": "prompt_ragged_24x901", "op": "prompt", "type": "f16", "D": 64, "Hq": 32, "Hkv": 32, "seqs": 24,
         "longest": 901, "context": 0, "causal": True, "fused": True},
        # one long document
        {"name": "prompt_long_16384", "op": "prompt", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "seqs": 1,
         "longest": 16384, "context": 0, "causal": True, "fused": False},
        # one user's next token, nothing shared: latency
        {"name": "paged_one_of_333", "op": "paged", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "batch": 1, "groups": 1,
         "shared": 0, "own": 333, "page": 16},
        # 32 users behind one system prompt of 8192 tokens, everyone with a few hundred tokens of their own
        {"name": "paged_32_behind_8192", "op": "paged", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "batch": 32,
         "groups": 1, "shared": 8192, "own": 300, "page": 16},
        # 64 samples of four long documents, a wide model, larger pages
        {"name": "paged_64_in_4_behind_15000", "op": "paged", "type": "f16", "D": 128, "Hq": 64, "Hkv": 8, "batch": 64,
         "groups": 4, "shared": 15000, "own": 1500, "page": 64},
        # every user's next token goes into the cache
        {"name": "write_64x1", "op": "write", "type": "bf16", "D": 128, "Hkv": 8, "rows": 64, "longest": 1, "page": 16},
        # the prompts of five users go into the cache
        {"name": "write_5x4001", "op": "write", "type": "f16", "D": 128, "Hkv": 8, "rows": 5, "longest": 4001, "page": 16},
        # 48 users go on by a token, some leave, some come: tables only, no page is copied
        {"name": "step_48_users", "op": "step", "planes": 16, "page_elems": 4096, "pages": 4096, "rows": 48, "width": 128,
         "page": 16, "longest": 1000, "beams": 1, "kept": 1, "leave": 4, "come": 4},
        # 64 beam searches of four: in each, two of the four go on and every one is forked; one half-filled page each is copied
        {"name": "step_64_searches_of_4", "op": "step", "planes": 32, "page_elems": 16384, "pages": 2048, "rows": 256,
         "width": 24, "page": 16, "longest": 250, "beams": 4, "kept": 2, "leave": 0, "come": 0},
        # a small cache with two holes to fill
        {"name": "compact_300_of_512", "op": "compact", "planes": 8, "page_elems": 8192, "pages": 512, "live": 300,
         "moves": 2, "rows": 16},
        # a large cache, a third of it free: a quarter of its pages move
        {"name": "compact_1365_of_2048", "op": "compact", "planes": 32, "page_elems": 16384, "pages": 2048, "live": 1365,
         "moves": 455, "rows": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice([(32, 32), (32, 8), (64, 8), (16, 2), (28, 4), (14, 2), (8, 8), (12, 1)])


def draw(rng):
    op = rng.choice(["prompt", "prompt", "paged", "paged", "write", "step", "compact"])
    kind = rng.choice(["bf16", "f16"])
    d = rng.choice([64, 128])
    hq, hkv = _heads(rng)
    page = rng.choice([16, 16, 32, 64])
    if op == "prompt":
        seqs = _log(rng, 1, 40)
        # padded, the plain form's scores take seqs * longest * (longest + context) floats a head
        most = math.sqrt(16384 * 16384 * 32 / (2 * hq * seqs))
        longest = _log(rng, 1, max(2, min(16384, most)))
        context = _log(rng, 1, 8192) if rng.random() < 0.4 else 0
        while seqs * hq * longest * (longest + context) > 16384 * 16384 * 32:
            context //= 2
        return {"op": op, "type": kind, "D": d, "Hq": hq, "Hkv": hkv, "seqs": seqs, "longest": longest, "context": context,
                "causal": rng.random() < 0.85, "fused": context == 0 and rng.random() < 0.5}
    if op == "paged":
        batch = _log(rng, 1, 64)
        groups = min(batch, rng.choice([1, 1, 2, 4, batch]))
        shared = 0 if groups == batch else _log(rng, 16, 16000)
        return {"op": op, "type": kind, "D": d, "Hq": hq, "Hkv": hkv, "batch": batch, "groups": groups, "shared": shared,
                "own": _log(rng, 1, 4000 if shared < 4000 else 1500), "page": page}
    if op == "write":
        rows = _log(rng, 1, 64)
        return {"op": op, "type": kind, "D": d, "Hkv": hkv, "rows": rows, "longest": _log(rng, 1, 20000 // rows), "page": page}
    planes = 2 * rng.randint(1, 16)
    elems = page * d * min(hkv, 8)
    pages = min(_log(rng, 64, 2048), (1 << 30) // (planes * elems))
    if op == "compact":
        live = rng.randint(1, pages - 1)
        return {"op": op, "planes": planes, "page_elems": elems, "pages": pages, "live": live,
                "moves": rng.randint(0, min(live, pages - live) // 2), "rows": _log(rng, 1, min(live, 256))}
    beams = rng.choice([1, 1, 2, 4, 8])
    rows = max(1, _log(rng, 1, max(1, min(256, pages // 4 // beams)))) * beams
    # each search: pages that its beams share, a tail and a fresh page for each beam
    width = max(2, min(256, (pages - 3 * rows) * beams // rows if beams > 1 else pages // (2 * rows)))
    longest = max(1, _log(rng, 1, (width - 1) * page))
    return {"op": op, "planes": planes, "page_elems": elems, "pages": pages, "rows": rows, "width": width, "page": page,
            "longest": longest, "beams": beams, "kept": rng.randint(1, beams), "leave": rng.randint(0, rows // 4) if beams == 1 else 0,
            "come": rng.randint(0, rows // 4) if beams == 1 else 0}


def _spread(n, longest, least=0):
    """n lengths from `least` to `longest`, the longest first, spread over the range without a pattern that divides anything."""
    return [longest if i == 0 else least + int((longest + 1 - least) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _prompt_lengths(c):
    new = _spread(c["seqs"], c["longest"])
    return new, [n + (int(c["context"] * (1.0 - 0.4 * ((i * 0.7548776662) % 1.0))) if c["context"] else 0) for i, n in enumerate(new)]


def _step_lengths(c):
    """Length of each search (or, beams 1, request): no whole pages in a search, so that every fork copies one."""
    got = _spread(c["rows"] // c["beams"], c["longest"], 1)
    return [n + 1 if c["beams"] > 1 and n % c["page"] == 0 else n for n in got] if c["page"] > 1 else got


def _cumulated(lengths):
    return np.concatenate([[0], np.cumsum(np.asarray(lengths, np.int64))])


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).cuda()


def _pool(c, g):
    shape = (c["planes"], c["pages"], c["page_elems"])
    return torch.randint(-32768, 32768, shape, generator=g, device="cuda", dtype=torch.int16).view(torch.float16)


def _paged_layout(c, r):
    """Table, lengths, group bounds and the number of pages: a group's first pages are the same in all its rows."""
    b, page, shared = c["batch"], c["page"], c["shared"]
    bounds = [c["batch"] * i // c["groups"] for i in range(c["groups"] + 1)]
    lengths = [shared + n for n in _spread(b, c["own"], 1)]
    width = -(-max(lengths) // page)
    full = shared // page  # the tokens of a half-filled page were copied when the rows were forked: every row has its own
    use = [-(-n // page) for n in lengths]
    pages = full * c["groups"] + sum(u - full for u in use)
    order = r.permutation(pages)
    table = np.full((b, width), -1, np.int32)
    at = 0
    for gi in range(c["groups"]):
        head = order[at:at + full]
        at += full
        for row in range(bounds[gi], bounds[gi + 1]):
            table[row, :full] = head
            table[row, full:use[row]] = order[at:at + use[row] - full]
            at += use[row] - full
    return table, lengths, bounds, pages


def _step_layout(c, r):
    b, page, n = c["beams"], c["page"], c["rows"]
    order = r.permutation(c["pages"])
    table = np.full((n, c["width"]), -1, np.int32)
    lengths, parent, add = np.zeros(n, np.int32), np.arange(n, dtype=np.int32), np.ones(n, np.int32)
    refs = np.zeros(c["pages"], np.int32)
    at = 0
    for i, length in enumerate(_step_lengths(c)):
        rows = np.arange(i * b, (i + 1) * b)
        length = min(length, c["width"] * page - 1)
        full, used = length // page, -(-length // page)
        lengths[rows] = length
        table[rows, :full] = order[at:at + full]
        at += full
        if used > full:
            table[rows, full] = order[at:at + b]
            at += b
        if b > 1:
            kept = r.permutation(rows)[:c["kept"]]
            parent[rows] = r.permutation(np.concatenate([kept, kept[r.integers(0, len(kept), b - len(kept))]]))
    for row in range(n):
        used = -(-int(lengths[row]) // page)
        np.add.at(refs, table[row, :used], 1)
    out = r.permutation(n)
    parent[out[:c["leave"]]] = -1
    add[out[:c["leave"]]] = 0
    come = out[c["leave"]:c["leave"] + c["come"]]
    parent[come] = -1
    add[come] = [min(c["longest"], 1 + int(c["longest"] * ((k * 0.6180339887) % 1.0))) for k in range(len(come))]
    return table, lengths, refs, parent, add


def _compact_layout(c, r):
    live, moves, n = c["live"], c["moves"], c["pages"]
    used = np.zeros(n, bool)
    used[:live] = True
    used[r.permutation(live)[:moves]] = False
    used[live + r.permutation(n - live)[:moves]] = True
    order = r.permutation(np.nonzero(used)[0])
    width = -(-live // c["rows"]) + 1
    table = np.full((c["rows"], width), -1, np.int32)
    for row in range(c["rows"]):
        mine = order[row::c["rows"]]
        table[row, :1 + len(mine)] = np.concatenate([order[:1], mine])  # all of them begin on one page
    refs = np.zeros(n, np.int32)
    np.add.at(refs, table[table >= 0], 1)
    return table, refs


def prepare(case, seed):
    c, g, r = case, _gen(seed), np.random.default_rng(seed)
    s = {"case": c}
    if c["op"] in ("prompt", "paged", "write"):
        kind, d = TYPES[c["type"]], c["D"]
    if c["op"] == "prompt":
        new, keys = _prompt_lengths(c)
        cu_q, cu_k = _cumulated(new), _cumulated(keys)
        tq, tk, hq, hkv = int(cu_q[-1]), int(cu_k[-1]), c["Hq"], c["Hkv"]
        if c["fused"]:
            qkv = _normal(g, (tq, hq + 2 * hkv, d), kind)
            q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            q, k, v = _normal(g, (tq, hq, d), kind, 1.5), _normal(g, (tk, hkv, d), kind), _normal(g, (tk, hkv, d), kind)
        s.update(q=q, k=k, v=v, cu_q=_ints(cu_q), cu_k=_ints(cu_k), most_q=max(new), most_k=max(keys))
    elif c["op"] == "paged":
        table, lengths, bounds, pages = _paged_layout(c, r)
        shape = (pages, c["Hkv"], c["page"], d)
        s.update(q=_normal(g, (c["batch"], c["Hq"], d), kind, 1.5), k=_normal(g, shape, kind), v=_normal(g, shape, kind),
                 table=_ints(table), lengths=_ints(lengths), groups=_ints(bounds),
                 shared=_ints([c["shared"] // c["page"] * c["page"]] * c["groups"]), most_k=max(lengths))
    elif c["op"] == "write":
        new = _spread(c["rows"], c["longest"], 1)
        start = [0 if c["longest"] > 1 else (37 * i + 11) % 500 for i in range(len(new))]
        width = max(-(-(a + n) // c["page"]) for a, n in zip(start, new))
        use = [-(-(a + n) // c["page"]) for a, n in zip(start, new)]
        order, table, at = r.permutation(sum(use) + 7), np.full((len(new), width), -1, np.int32), 0
        for row, u in enumerate(use):
            table[row, :u] = order[at:at + u]
            at += u
        shape = (len(order), c["Hkv"], c["page"], d)
        t = sum(new)
        s.update(k=_normal(g, (t, c["Hkv"], d), kind), v=_normal(g, (t, c["Hkv"], d), kind), k_pages=_normal(g, shape, kind),
                 v_pages=_normal(g, shape, kind), table=_ints(table), starts=_ints(start), cu=_ints(_cumulated(new)))
    elif c["op"] == "step":
        table, lengths, refs, parent, add = _step_layout(c, r)
        s.update(pool=_pool(c, g), table=_ints(table), lengths=_ints(lengths), refs=_ints(refs), parent=_ints(parent), add=_ints(add))
    else:
        table, refs = _compact_layout(c, r)
        s.update(pool=_pool(c, g), table=_ints(table), refs=_ints(refs))
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _softmax_product(scores, seen, v):
    """Rows of `scores` over the keys that they see, times v; a row that sees none gives zeros."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return torch.matmul(scores, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prompt(s):
    c, dev = s["case"], s["q"].device
    hq, hkv, d, lq, lk = c["Hq"], c["Hkv"], c["D"], s["most_q"], s["most_k"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    nq, nk = (cu_q[1:] - cu_q[:-1])[:, None], (cu_k[1:] - cu_k[:-1])[:, None]
    iq, ik = torch.arange(lq, device=dev)[None], torch.arange(lk, device=dev)[None]
    at_q, at_k = torch.where(iq < nq, cu_q[:-1, None] + iq, 0), torch.where(ik < nk, cu_k[:-1, None] + ik, 0)
    n = at_q.shape[0]
    q = s["q"][at_q].float().view(n, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    k = s["k"][at_k].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][at_k].float().permute(0, 2, 1, 3).contiguous()
    seen = (ik < nk)[:, None, :]
    if c["causal"]:
        seen = seen & (ik[:, None, :] <= (iq + nk - nq)[:, :, None])
    seen = seen.expand(n, lq, lk)[:, None, None]
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(d)).view(n, hkv, hq // hkv, lq, lk)
    o = _softmax_product(scores, seen, v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(n * lq, hq, d).to(s["q"].dtype)
    out = torch.empty((s["q"].shape[0] + 1, hq, d), dtype=o.dtype, device=dev)  # the last row takes what is padding
    out[torch.where(iq < nq, at_q, out.shape[0] - 1).view(-1)] = o
    return out[:-1]


def _plain_paged(s):
    c, dev = s["case"], s["q"].device
    b, hq, hkv, d, page = c["batch"], c["Hq"], c["Hkv"], c["D"], c["page"]
    ik = torch.arange(s["most_k"], device=dev)
    seen = ik[None] < s["lengths"].long()[:, None]
    at = s["table"].long()[:, ik // page].clamp(min=0)
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    k = s["k"][at, :, ik % page].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][at, :, ik % page].float().permute(0, 2, 1, 3).contiguous()
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(d))
    return _softmax_product(scores, seen[:, None, None], v).view(b, hq, d).to(s["q"].dtype)


def _plain_write(s):
    t, page = s["k"].shape[0], s["case"]["page"]
    token = torch.arange(t, device=s["k"].device)
    row = torch.searchsorted(s["cu"][1:].long(), token, right=True)
    at = s["starts"].long()[row] + token - s["cu"].long()[row]
    pages = s["table"].long()[row, at // page]
    s["k_pages"][pages, :, at % page] = s["k"]
    s["v_pages"][pages, :, at % page] = s["v"]
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _free_in_order(refs):
    """Pages that nobody uses, lowest first (behind them whatever), and how many there are."""
    free = refs <= 0
    rank = torch.where(free, torch.cumsum(free, 0) - 1, refs.shape[0])
    first = torch.zeros(refs.shape[0] + 1, dtype=torch.long, device=refs.device)
    return first.scatter(0, rank, torch.arange(refs.shape[0], device=refs.device)), free.sum()


def _plain_step(s):
    page, table, pool = s["case"]["page"], s["table"].long(), s["pool"]
    rows, width, pages, dev = table.shape[0], table.shape[1], s["refs"].shape[0], table.device
    j, row = torch.arange(width, device=dev)[None], torch.arange(rows, device=dev)
    parent = s["parent"].long()
    alive, at = (parent >= 0) & (parent < rows), parent.clamp(0, rows - 1)
    old = s["lengths"].long().clamp(0, width * page)
    start = torch.where(alive, old[at], 0)
    full, used = start // page, (start + page - 1) // page
    length = (start + s["add"].long().clamp(min=0)).clamp(max=width * page)
    was = torch.where((j < ((old + page - 1) // page)[:, None]) & (table >= 0) & (table < pages), table, -1)
    got = torch.where(j < used[:, None], was[at], -1)
    first = torch.full((rows,), rows, device=dev).scatter_reduce(0, at, torch.where(alive, row, rows), "amin")
    source = got.gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    copied = alive & (used > full) & (first[at] != row) & (source >= 0)
    new = (copied[:, None] & (j == full[:, None])) | ((j >= used[:, None]) & (j < ((length + page - 1) // page)[:, None]))
    got = torch.where(new, -1, got)
    refs = s["refs"].long()
    count = torch.zeros(pages + 1, dtype=torch.long, device=dev)
    refs = refs - count.scatter_add(0, torch.where(was >= 0, was, pages).view(-1), torch.ones_like(was).view(-1))[:-1]
    refs = refs + count.scatter_add(0, torch.where(got >= 0, got, pages).view(-1), torch.ones_like(got).view(-1))[:-1]
    free, there = _free_in_order(refs)
    ask = torch.cumsum(new.view(-1), 0).view(rows, width) - 1
    have = new & (ask < there)
    took = free[ask.clamp(0, pages - 1)]
    got = torch.where(have, took, got)
    refs = torch.cat([refs, refs[:1]]).scatter(0, torch.where(have, took, pages).view(-1), 1)[:-1]
    lost = torch.where(new & ~have, j, width).amin(1)
    length = torch.minimum(length, lost * page)
    target = torch.where(copied, got.gather(1, full.clamp(max=width - 1)[:, None])[:, 0], -1)
    copied = target >= 0
    one = copied.int().argmax()  # whoever copies nothing writes what the first copy writes; nobody copies: page 0 stays itself
    target = torch.where(copied, target, torch.where(copied[one], target[one], 0))
    source = torch.where(copied, source, torch.where(copied[one], source[one], 0))
    pool[:, target] = pool[:, source]
    return {"table": got.int(), "lengths": length.int(), "refs": refs.int(), "starts": torch.minimum(start, length).int(),
            "missing": (new.sum() - have.sum()).int().view(1), "pool": pool.view(torch.int16)}


def _plain_compact(s):
    pool, table, refs = s["pool"], s["table"].long(), s["refs"].long()
    pages, dev = refs.shape[0], refs.device
    used, at = refs > 0, torch.arange(pages, device=dev)
    live = used.sum()
    hole, mover = ~used & (at < live), used & (at >= live)
    holes = torch.zeros(pages + 1, dtype=torch.long, device=dev)
    holes = holes.scatter(0, torch.where(hole, torch.cumsum(hole, 0) - 1, pages), at)
    to = torch.where(mover, holes[(torch.cumsum(mover, 0) - 1).clamp(min=0)], at)
    source = torch.cat([at, at[:1]]).scatter(0, torch.where(mover, to, pages), at)[:-1]
    pool.copy_(pool[:, source])
    known = (table >= 0) & (table < pages)
    return {"table": torch.where(known, to[table.clamp(0, pages - 1)], table).int(),
            "refs": torch.where(at < live, refs[source], torch.where(used, 0, refs)).int(), "live": live.int().view(1),
            "pool": pool.view(torch.int16)}


def _own(s):
    import hecbench_amd as hq
    op = s["case"]["op"]
    if op == "prompt":
        return hq.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["case"]["causal"])
    if op == "paged":
        return hq.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["groups"], s["shared"])
    if op == "write":
        hq.cache_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["cu"])
        return {"k": s["k_pages"], "v": s["v_pages"]}
    if op == "step":
        table, lengths, refs, starts, missing = hq.cache_step(s["pool"], s["case"]["page"], s["table"], s["lengths"], s["refs"],
                                                              s["parent"], s["add"])
        return {"table": table, "lengths": lengths, "refs": refs, "starts": starts, "missing": missing,
                "pool": s["pool"].view(torch.int16)}
    table, refs, live = hq.cache_compact(s["pool"], s["table"], s["refs"])
    return {"table": table, "refs": refs, "live": live, "pool": s["pool"].view(torch.int16)}


_PLAIN = {"prompt": _plain_prompt, "paged": _plain_paged, "write": _plain_write, "step": _plain_step, "compact": _plain_compact}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    if op == "prompt":
        new, keys = _prompt_lengths(c)
        pairs = 0
        for n, m in zip(new, keys):
            pairs += n * m - n * (n - 1) // 2 if c["causal"] else n * m
        data = 2 * c["D"] * (2 * sum(new) * c["Hq"] + 2 * sum(keys) * c["Hkv"])
        return {"bytes": data + 8 * (len(new) + 1), "flops": 4 * c["D"] * c["Hq"] * pairs}
    if op == "paged":
        shared = c["shared"] // c["page"] * c["page"]
        own_tokens = sum(_spread(c["batch"], c["own"], 1)) + c["batch"] * (c["shared"] - shared)
        data = 2 * c["D"] * (2 * c["batch"] * c["Hq"] + 2 * c["Hkv"] * (c["groups"] * shared + own_tokens))
        entries = (own_tokens + c["groups"] * shared) // c["page"]
        return {"bytes": data + 4 * (entries + c["batch"] + 2 * c["groups"]),
                "flops": 4 * c["D"] * c["Hq"] * (c["batch"] * shared + own_tokens)}
    if op == "write":
        new = _spread(c["rows"], c["longest"], 1)
        return {"bytes": 8 * c["D"] * c["Hkv"] * sum(new) + 4 * (sum(new) // c["page"] + 3 * len(new)), "flops": 0}
    if op == "step":
        tables = 2 * c["rows"] * c["width"] + 2 * c["pages"] + 5 * c["rows"]
        copies = c["rows"] // c["beams"] * (c["beams"] - c["kept"])
        return {"bytes": 4 * tables + 4 * c["planes"] * c["page_elems"] * copies, "flops": 0}
    tables = 2 * c["rows"] * (-(-c["live"] // c["rows"]) + 1) + 2 * c["pages"]
    return {"bytes": 4 * tables + 4 * c["planes"] * c["page_elems"] * c["moves"], "flops": 0}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _attend(q, k, v, seen):
    """q [rows][D] over k, v [keys][D] of one head, all in 64 bits; seen: [rows][keys] or None."""
    w = q @ k.T / math.sqrt(q.shape[1])
    if seen is not None:
        w = torch.where(seen, w, -math.inf)
    return torch.nan_to_num(torch.softmax(w, 1)) @ v  # a row that sees nothing is NaN in the softmax


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "prompt":
        new, keys = _prompt_lengths(c)
        ratio = c["Hq"] // c["Hkv"]
        out = torch.zeros((sum(new), c["Hq"], c["D"]), dtype=torch.float64, device="cuda")
        a = b = 0
        for n, m in zip(new, keys):
            if n:
                seen = None
                if c["causal"]:
                    seen = torch.ones((n, m), dtype=torch.bool, device="cuda").tril(m - n)
                for h in range(c["Hq"]):
                    if m:
                        out[a:a + n, h] = _attend(s["q"][a:a + n, h].double(), s["k"][b:b + m, h // ratio].double(),
                                                  s["v"][b:b + m, h // ratio].double(), seen)
            a, b = a + n, b + m
        return out
    if c["op"] == "paged":
        out = torch.zeros((c["batch"], c["Hq"], c["D"]), dtype=torch.float64, device="cuda")
        ratio = c["Hq"] // c["Hkv"]
        for i, n in enumerate(s["lengths"].tolist()):
            pages = s["table"][i, :-(-n // c["page"])].long()
            k = s["k"][pages].double().transpose(1, 2).reshape(-1, c["Hkv"], c["D"])[:n]
            v = s["v"][pages].double().transpose(1, 2).reshape(-1, c["Hkv"], c["D"])[:n]
            for h in range(c["Hkv"]):
                rows = slice(h * ratio, (h + 1) * ratio)
                out[i, rows] = _attend(s["q"][i, rows].double(), k[:, h].contiguous(), v[:, h].contiguous(), None)
        return out
    if c["op"] == "write":
        got = {}
        table, starts, cu = s["table"].cpu().numpy(), s["starts"].tolist(), s["cu"].tolist()
        where = [(int(table[i, (starts[i] + t) // c["page"]]), (starts[i] + t) % c["page"])
                 for i in range(c["rows"]) for t in range(cu[i + 1] - cu[i])]
        p, o = torch.tensor(where, device="cuda").T
        for name in ("k", "v"):
            full = s[name + "_pages"].double()
            full[p, :, o] = s[name].double()
            got[name] = full
        return got
    if c["op"] == "step":
        return _exact_step(s)
    return _exact_compact(s)


def _exact_step(s):
    page = s["case"]["page"]
    table, lengths, refs, parent, add = (s[n].cpu().numpy().astype(np.int64) for n in ("table", "lengths", "refs", "parent", "add"))
    rows, width = table.shape
    wanted, kept, after = [], set(), np.full_like(table, -1)
    starts, ends = np.zeros(rows, np.int64), np.zeros(rows, np.int64)
    left = refs.copy()
    for i in range(rows):
        for p in table[i, :-(-lengths[i] // page)]:
            left[p] -= 1
    for i in range(rows):
        if parent[i] >= 0:
            starts[i] = lengths[parent[i]]
        ends[i] = min(starts[i] + add[i], width * page)
        used = -(-starts[i] // page)
        for j in range(-(-ends[i] // page)):
            whole = (j + 1) * page <= starts[i]
            if j < used and (whole or parent[i] not in kept):
                after[i, j] = table[parent[i], j]
                left[after[i, j]] += 1
            else:
                wanted.append((i, j, table[parent[i], j] if j < used else -1))
        kept.add(parent[i])
    free, missing = [p for p in range(len(left)) if left[p] == 0], 0
    pool = s["pool"].view(torch.int16).clone()
    for (i, j, source) in wanted:
        if free:
            after[i, j] = free.pop(0)
            left[after[i, j]] = 1
            if source >= 0:
                pool[:, after[i, j]] = s["pool"].view(torch.int16)[:, source]
        else:
            missing += 1
            ends[i] = min(ends[i], j * page)
    return {"table": _ints(after), "lengths": _ints(ends), "refs": _ints(left), "starts": _ints(np.minimum(starts, ends)),
            "missing": _ints([missing]), "pool": pool}


def _exact_compact(s):
    table, refs = s["table"].cpu().numpy(), s["refs"].cpu().numpy()
    live = int((refs > 0).sum())
    holes = [p for p in range(live) if refs[p] <= 0]
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    after, counts, pool = table.copy(), refs.copy(), s["pool"].view(torch.int16).clone()
    for source, target in zip(movers, holes):
        after[table == source] = target
        counts[target], counts[source] = refs[source], 0
        pool[:, target] = pool[:, source]
    return {"table": _ints(after), "refs": _ints(counts), "live": _ints([live]), "pool": pool}
