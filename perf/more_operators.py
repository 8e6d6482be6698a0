"""Operators around a serving program's attention: what their speed is judged by.

Between a layer's projection and its attention the heads of queries and keys are normed and rotated by their tokens'
positions (norm_rotate), in a program with a paged cache on the keys' way into their pages (cache_write_rotated).  Then
the new tokens attend: those of whole prompts packed one behind the other, through a sliding window and a few first tokens
that stay visible (prompt_attention with a window), or those of every request's next piece - one token, a few drafted ones,
a chunk of a long prompt, all in one call - over the paged cache, with such a window or without (chunk_attention).

The cache of a layer is two tensors [pages][key / value heads][tokens of a page][head size]; row s of `table` lists the
pages of request s in order, -1 behind the last one.  cos_sin [positions][rotated elements] holds, for every position, the
cosines of its angles and then their sines, in fp32.

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
        # the prompts of 24 users, packed, heads of 64 of which half of the elements are rotated, neighbours in pairs; no norm
        {"name": "rotate_24x901", "op": "rotate", "type": "f16", "D": 64, "Hq": 32, "Hkv": 32, "seqs": 24, "longest": 901,
         "rotary": 32, "norm": False, "interleaved": True},
        # one long document, queries and keys out of one projection's result
        {"name": "rotate_16384", "op": "rotate", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "seqs": 1, "longest": 16384,
         "rotary": 128, "norm": True, "interleaved": False},
        # one user's next token: latency
        {"name": "write_rotated_1", "op": "write", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "rows": 1, "longest": 1, "page": 16,
         "rotary": 128, "norm": True, "interleaved": False},
        # the next token of 64 users
        {"name": "write_rotated_64x1", "op": "write", "type": "f16", "D": 128, "Hq": 64, "Hkv": 8, "rows": 64, "longest": 1, "page": 16,
         "rotary": 128, "norm": True, "interleaved": False},
        # the prompts of five users go into the cache
        {"name": "write_rotated_5x4001", "op": "write", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "rows": 5, "longest": 4001,
         "page": 16, "rotary": 128, "norm": True, "interleaved": False},
        # one user's next token, a short window: latency
        {"name": "chunk_one_of_333_window_128", "op": "chunk", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "rows": 1, "chunks": 1,
         "new": 1, "context": 332, "page": 16, "window": 128, "sinks": 4},
        # 64 users' next tokens in conversations of up to 16000 tokens, a window of 1024 and four first tokens
        {"name": "chunk_64x1_of_16000_window_1024", "op": "chunk", "type": "f16", "D": 128, "Hq": 32, "Hkv": 8, "rows": 64, "chunks": 64,
         "new": 1, "context": 16000, "page": 16, "window": 1024, "sinks": 4},
        # five drafted tokens each of 16 users are checked at once, in conversations of up to 4000 tokens
        {"name": "chunk_16x5_behind_4000", "op": "chunk", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "rows": 16, "chunks": 16,
         "new": 5, "context": 4000, "page": 16, "window": 0, "sinks": 0},
        # a step of a busy server: the next 509 tokens of one prompt and of another, smaller one, and 30 users' next tokens
        {"name": "chunk_509_and_30x1", "op": "chunk", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "rows": 32, "chunks": 2,
         "new": 509, "context": 3000, "page": 16, "window": 0, "sinks": 0},
        # a piece of a long document behind what is in place
        {"name": "chunk_2048_behind_30000", "op": "chunk", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "rows": 1, "chunks": 1,
         "new": 2048, "context": 30000, "page": 64, "window": 0, "sinks": 0},
        # short prompts of 17 users, heads of 64, taken out of one projection's result
        {"name": "window_17x700_of_128", "op": "prompt", "type": "f16", "D": 64, "Hq": 14, "Hkv": 2, "seqs": 17, "longest": 700,
         "context": 0, "fused": True, "window": 128, "sinks": 4},
        # one long document
        {"name": "window_16384_of_1024", "op": "prompt", "type": "bf16", "D": 128, "Hq": 32, "Hkv": 8, "seqs": 1, "longest": 16384,
         "context": 0, "fused": False, "window": 1024, "sinks": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice([(32, 32), (32, 8), (64, 8), (16, 2), (28, 4), (14, 2), (8, 8), (12, 1)])


def draw(rng):
    op = rng.choice(["rotate", "write", "write", "chunk", "chunk", "chunk", "prompt", "prompt"])
    kind, d, page = rng.choice(["bf16", "f16"]), rng.choice([64, 128]), rng.choice([16, 16, 32, 64])
    hq, hkv = _heads(rng)
    c = {"op": op, "type": kind, "D": d, "Hq": hq, "Hkv": hkv}
    if op in ("rotate", "write"):
        most = 16384 * 40 * 128 // ((hq + hkv) * d)  # tokens: as much data as the largest listed case
        c.update(rotary=rng.choice([d, d, d // 2, 16 * rng.randint(1, d // 16)]), norm=rng.random() < 0.7, interleaved=rng.random() < 0.3)
        n = _log(rng, 1, 64)
        c["longest"] = _log(rng, 1, min(16384, most // n))
        c.update({"seqs": n} if op == "rotate" else {"rows": n, "page": page})
        return c
    window = 0 if op == "chunk" and rng.random() < 0.5 else _log(rng, 16, 4096)
    c.update(window=window, sinks=rng.choice([0, 1, 4, 4, 64]) if window else 0)
    if op == "chunk":
        rows = _log(rng, 1, 64)
        chunks = rng.choice([rows, rows, 1, max(1, rows // 8)])
        new = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 2048)])
        context = _log(rng, 1, 30000)
        # the plain form, padded: scores of rows * new queries a head, and every request's keys in fp32
        while rows * new * hq * (new + context) > 2048 * 32048 * 32 or rows * (new + context) * hkv * d > 1 << 30:
            if new > context:
                new = (new + 1) // 2
            else:
                context //= 2
        c.update(rows=rows, chunks=chunks, new=new, context=context, page=page)
        return c
    seqs = _log(rng, 1, 40)
    longest = _log(rng, 2, max(3, min(16384, math.sqrt(16384 * 16384 * 32 / (2 * hq * seqs)))))
    context = _log(rng, 1, 8192) if rng.random() < 0.3 else 0
    while seqs * hq * longest * (longest + context) > 16384 * 16384 * 32:
        context //= 2
    c.update(seqs=seqs, longest=longest, context=context, fused=context == 0 and rng.random() < 0.5)
    return c


def _spread(n, longest, least=0):
    """n lengths from `least` to `longest`, the longest first, spread over the range without a pattern that divides anything."""
    return [longest if i == 0 else least + int((longest + 1 - least) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _prompt_lengths(c):
    new = _spread(c["seqs"], c["longest"])
    return new, [n + (int(c["context"] * (1.0 - 0.4 * ((i * 0.7548776662) % 1.0))) if c["context"] else 0) for i, n in enumerate(new)]


def _chunk_lengths(c):
    """New tokens of each request, the chunks among requests that go on by one token, and the tokens that it has with them."""
    rows, n = c["rows"], c["chunks"]
    new = [1] * rows
    for i, m in enumerate(_spread(n, c["new"], 1 if c["new"] < 9 else c["new"] // 3)):
        new[i * rows // n] = m
    before = _spread(rows, c["context"])
    return new, [a + b for a, b in zip(before, new)]


def _write_lengths(c):
    new = _spread(c["rows"], c["longest"], 1)
    return new, [0 if c["longest"] > 1 else (37 * i + 411) % 500 for i in range(len(new))]


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


def _paged(lengths, page, r):
    """A table of pages in no order for requests of these lengths, and the number of pages."""
    use = [-(-n // page) for n in lengths]
    order, table, at = r.permutation(sum(use) + 5), np.full((len(lengths), max(use)), -1, np.int32), 0
    for row, u in enumerate(use):
        table[row, :u] = order[at:at + u]
        at += u
    return table, len(order)


def _rotation(c, positions, g):
    """Cosines and sines of a table's positions, and the norms' weights, near one as training leaves them."""
    half = c["rotary"] // 2
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64, device="cuda") / half)
    weights = [(1 + 0.2 * torch.randn(c["D"], generator=g, device="cuda")).to(TYPES[c["type"]]) if c["norm"] else None for _ in range(2)]
    return {"cos_sin": torch.cat([angle.cos(), angle.sin()], 1).float(), "q_weight": weights[0], "k_weight": weights[1]}


def prepare(case, seed):
    c, g, r = case, _gen(seed), np.random.default_rng(seed)
    kind, d, hq, hkv = TYPES[c["type"]], c["D"], c["Hq"], c["Hkv"]
    s = {"case": c}
    if c["op"] in ("rotate", "write"):
        new, start = (_spread(c["seqs"], c["longest"], 1), [0] * c["seqs"]) if c["op"] == "rotate" else _write_lengths(c)
        qkv = _normal(g, (sum(new), hq + 2 * hkv, d), kind, 1.5)
        s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], **_rotation(c, 32768, g))
        if c["op"] == "rotate":
            s.update(positions=_ints(np.concatenate([np.arange(n) for n in new])))
            return s
        table, pages = _paged([a + n for a, n in zip(start, new)], c["page"], r)
        shape = (pages, hkv, c["page"], d)
        s.update(k_pages=_normal(g, shape, kind), v_pages=_normal(g, shape, kind), table=_ints(table), starts=_ints(start),
                 cu=_ints(_cumulated(new)))
    elif c["op"] == "chunk":
        new, lengths = _chunk_lengths(c)
        table, pages = _paged(lengths, c["page"], r)
        shape = (pages, hkv, c["page"], d)
        s.update(q=_normal(g, (sum(new), hq, d), kind, 1.5), k=_normal(g, shape, kind), v=_normal(g, shape, kind), table=_ints(table),
                 lengths=_ints(lengths), cu_q=_ints(_cumulated(new)), most_q=max(new), most_k=max(lengths))
    else:
        new, keys = _prompt_lengths(c)
        cu_q, cu_k = _cumulated(new), _cumulated(keys)
        if c["fused"]:
            qkv = _normal(g, (sum(new), hq + 2 * hkv, d), kind)
            q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            q = _normal(g, (sum(new), hq, d), kind, 1.5)
            k, v = (_normal(g, (sum(keys), hkv, d), kind) for _ in range(2))
        s.update(q=q, k=k, v=v, cu_q=_ints(cu_q), cu_k=_ints(cu_k), most_q=max(new), most_k=max(keys))
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _normed_and_rotated(x, weight, cos, sin, interleaved):
    """x [tokens][heads][D]; cos and sin [tokens][rotated pairs]."""
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    n = cos.shape[1]
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    cos, sin = cos[:, None], sin[:, None]
    turned = [a * cos - b * sin, b * cos + a * sin]
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat([turned, y[..., 2 * n:]], -1).to(x.dtype)


def _plain_rotation(s, positions):
    cos, sin = s["cos_sin"][positions].chunk(2, 1)
    pairs = ((s["q"], s["q_weight"]), (s["k"], s["k_weight"]))
    return [_normed_and_rotated(x, w, cos, sin, s["case"]["interleaved"]) for x, w in pairs]


def _plain_rotate(s):
    return _plain_rotation(s, s["positions"].long())


def _plain_write(s):
    page = s["case"]["page"]
    token = torch.arange(s["k"].shape[0], device=s["k"].device)
    row = torch.searchsorted(s["cu"][1:].long(), token, right=True)
    at = s["starts"].long()[row] + token - s["cu"].long()[row]
    q, k = _plain_rotation(s, at)
    pages = s["table"].long()[row, at // page]
    s["k_pages"][pages, :, at % page] = k
    s["v_pages"][pages, :, at % page] = s["v"]
    return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}


def _softmax_product(scores, seen, v):
    """Rows of `scores` over the keys that they see, times v; a row that sees none gives zeros."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return torch.matmul(scores, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_attention(s, at_q, padding, nq, nk, k, v):
    """Padded: tokens at_q [sequences][most_q] of q over keys and values [sequences][heads][most_k][D] in fp32."""
    c, dev, hq, hkv, d = s["case"], s["q"].device, s["case"]["Hq"], s["case"]["Hkv"], s["case"]["D"]
    n, lq = at_q.shape
    lk = s["most_k"]
    q = s["q"][at_q].float().view(n, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    ik = torch.arange(lk, device=dev)
    place = torch.arange(lq, device=dev)[None] + nk - nq  # of a token among its sequence's keys
    seen = (ik < nk)[:, None, :] & (ik <= place[:, :, None])
    if c["window"]:
        seen &= (ik > place[:, :, None] - c["window"]) | (ik < c["sinks"])
    seen = seen[:, None, None]
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(d)).view(n, hkv, hq // hkv, lq, lk)
    o = _softmax_product(scores, seen, v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(n * lq, hq, d).to(s["q"].dtype)
    out = torch.empty((s["q"].shape[0] + 1, hq, d), dtype=o.dtype, device=dev)  # the last row takes what is padding
    out[torch.where(padding, out.shape[0] - 1, at_q).view(-1)] = o
    return out[:-1]


def _padded(s, cu, most):
    """Tokens of each sequence, padded to the longest; where that is padding; and how many there are."""
    cu = cu.long()
    n, i = (cu[1:] - cu[:-1])[:, None], torch.arange(most, device=cu.device)[None]
    return torch.where(i < n, cu[:-1, None] + i, 0), i >= n, n


def _plain_chunk(s):
    page = s["case"]["page"]
    at_q, padding, nq = _padded(s, s["cu_q"], s["most_q"])
    ik = torch.arange(s["most_k"], device=s["q"].device)
    pages = s["table"].long()[:, ik // page].clamp(min=0)
    k, v = (s[x][pages, :, ik % page].float().permute(0, 2, 1, 3) for x in ("k", "v"))
    return _plain_attention(s, at_q, padding, nq, s["lengths"].long()[:, None], k, v.contiguous())


def _plain_prompt(s):
    at_q, padding, nq = _padded(s, s["cu_q"], s["most_q"])
    at_k, _, nk = _padded(s, s["cu_k"], s["most_k"])
    k, v = (s[x][at_k].float().permute(0, 2, 1, 3) for x in ("k", "v"))
    return _plain_attention(s, at_q, padding, nq, nk, k, v.contiguous())


def _own(s):
    import hecbench_amd as hq
    c, op = s["case"], s["case"]["op"]
    if op == "rotate":
        return hq.norm_rotate(s["q"], s["k"], s["cos_sin"], s["positions"], s["q_weight"], s["k_weight"], interleaved=c["interleaved"])
    if op == "write":
        q = hq.cache_write_rotated(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["cu"], s["cos_sin"],
                                   s["q_weight"], s["k_weight"], interleaved=c["interleaved"])
        return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
    window = c["window"] or None
    if op == "chunk":
        return hq.chunk_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["cu_q"], window=window, sinks=c["sinks"])
    return hq.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], window=window, sinks=c["sinks"])


_PLAIN = {"rotate": _plain_rotate, "write": _plain_write, "chunk": _plain_chunk, "prompt": _plain_prompt}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def _seen(c, nq, nk):
    """Pairs of a token and a key that it sees, and keys that some token sees, in a sequence of nq new tokens among nk."""
    if nq == 0:
        return 0, 0
    w, sinks = c["window"] or nk, c["sinks"]
    places = np.arange(nk - nq, nk)
    first = np.maximum(places - w + 1, 0)
    lowest = int(first[0])
    return int((places - first + 1 + np.minimum(sinks, first)).sum()), nk - lowest + min(sinks, lowest)


def work(case):
    c, d, hq, hkv = case, case["D"], case["Hq"], case["Hkv"]
    if c["op"] in ("rotate", "write"):
        new = _spread(c["seqs"], c["longest"], 1) if c["op"] == "rotate" else _write_lengths(c)[0]
        angles = max(new) if c["op"] == "rotate" or c["longest"] > 1 else len(new)
        heads = hq + hkv + (hkv if c["op"] == "write" else 0)
        small = sum(new) if c["op"] == "rotate" else sum(new) // c["page"] + 3 * len(new)
        return {"bytes": 4 * d * heads * sum(new) + 4 * c["rotary"] * angles + 4 * small + (4 * d if c["norm"] else 0),
                "flops": sum(new) * (hq + hkv) * (3 * c["rotary"] + (4 * d if c["norm"] else 0))}
    new, keys = _chunk_lengths(c) if c["op"] == "chunk" else _prompt_lengths(c)
    pairs, read = (sum(x) for x in zip(*(_seen(c, n, m) for n, m in zip(new, keys))))
    small = 3 * len(new) + (read // c["page"] if c["op"] == "chunk" else 0)
    return {"bytes": 2 * d * (2 * sum(new) * hq + 2 * read * hkv) + 4 * small, "flops": 4 * d * hq * pairs}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_rotated(s, x, weight, where):
    """Every pair of elements is a complex number, turned by one of unit size."""
    c, n = s["case"], s["case"]["rotary"] // 2
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6) * weight.double()
    y = y.clone()
    first = torch.arange(n, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else n)
    rows = s["cos_sin"][where].double()
    turned = torch.complex(y[..., first], y[..., second]) * torch.complex(rows[:, :n], rows[:, n:])[:, None]
    y[..., first], y[..., second] = turned.real, turned.imag
    return y


def _exact_attention(c, q, k, v):
    """Tokens q [n][heads][D], the last of a sequence's keys k, v [m][heads][D], in 64 bits, a head at a time."""
    n, m, ratio = q.shape[0], k.shape[0], c["Hq"] // c["Hkv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    if n == 0 or m == 0:
        return out
    hidden = torch.ones((n, m), dtype=torch.bool, device="cuda").triu(m - n + 1)
    if c["window"]:
        old = torch.ones((n, m), dtype=torch.bool, device="cuda").tril(m - n - c["window"])
        old[:, :c["sinks"]] = False
        hidden |= old
    for h in range(c["Hq"]):
        w = (q[:, h].double() @ k[:, h // ratio].double().T.contiguous()) / math.sqrt(c["D"])
        w.masked_fill_(hidden, -math.inf)
        out[:, h] = torch.nan_to_num(torch.softmax(w, 1)) @ v[:, h // ratio].double()
    return out


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "rotate":
        where = s["positions"].long()
        return [_exact_rotated(s, s["q"], s["q_weight"], where), _exact_rotated(s, s["k"], s["k_weight"], where)]
    if c["op"] == "write":
        table, starts, cu = s["table"].cpu().numpy(), s["starts"].tolist(), s["cu"].tolist()
        at = np.concatenate([starts[i] + np.arange(cu[i + 1] - cu[i]) for i in range(c["rows"])])
        row = np.repeat(np.arange(c["rows"]), np.diff(cu))
        p, o = torch.from_numpy(table[row, at // c["page"]]).long().cuda(), torch.from_numpy(at % c["page"]).cuda()
        at = torch.from_numpy(at).cuda()
        k, v = s["k_pages"].double(), s["v_pages"].double()
        k[p, :, o] = _exact_rotated(s, s["k"], s["k_weight"], at)
        v[p, :, o] = s["v"].double()
        return {"q": _exact_rotated(s, s["q"], s["q_weight"], at), "k": k, "v": v}
    parts, a, b = [], 0, 0
    new, keys = _chunk_lengths(c) if c["op"] == "chunk" else _prompt_lengths(c)
    for i, (n, m) in enumerate(zip(new, keys)):
        if c["op"] == "chunk":
            pages = s["table"][i, :-(-m // c["page"])].long()
            k, v = (s[x][pages].transpose(1, 2).reshape(-1, c["Hkv"], c["D"])[:m] for x in ("k", "v"))
        else:
            k, v = s["k"][b:b + m], s["v"][b:b + m]
        parts.append(_exact_attention(c, s["q"][a:a + n], k, v))
        a, b = a + n, b + m
    return torch.cat(parts)
