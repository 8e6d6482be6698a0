"""Attention of any number of new tokens per request over a paged cache, and through a sliding window with a few first tokens that stay
visible, over the cache and over packed prompts, against the formula in 64 bits.  Bounds as in test_attention_gpu."""
import math

import pytest
import torch

from tests.test_attention_gpu import TYPES, attend, bounds, close, i32, randn

pytestmark = pytest.mark.gpu


def seen_of(n, m, window, sinks):
    """Which of m keys the last n tokens of a sequence see."""
    place = torch.arange(m - n, m, device="cuda")[:, None]
    key = torch.arange(m, device="cuda")[None]
    seen = key <= place
    if window:
        seen &= (key > place - window) | (key < sinks)
    return seen


def check(out, q, k, v, window, sinks, scale, u):
    """One sequence: q [n][heads][D], the last of k, v [m][kv_heads][D]."""
    n, m, r = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    seen = seen_of(n, m, window, sinks)
    for h in range(q.shape[1]):
        want, a, big = attend(q[:, h].double(), k[:, h // r].double(), v[:, h // r].double(), seen, scale)
        close(out[:, h], want, a, big, u)
        assert (out[:, h][~seen.any(1)] == 0).all()


class Cache:
    """Pages in no order; whatever no request uses is NaN."""

    def __init__(self, seed, lengths, kv, page, D, dtype, spare=3, width=None):
        self.page, self.lengths = page, lengths
        use = [-(-max(n, 0) // page) for n in lengths]
        width = width or max(use + [1])
        order = torch.randperm(sum(use) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
        self.rows = [[order.pop() for _ in range(u)] for u in use]
        self.table = i32([r + [-1] * (width - len(r)) for r in self.rows])
        self.k, self.v = (torch.full((sum(use) + spare, kv, page, D), math.nan, dtype=dtype, device="cuda") for _ in range(2))
        self.dense = []
        for i, n in enumerate(lengths):
            k, v = randn(seed + 2 * i, max(n, 0), kv, D).to(dtype), randn(seed + 2 * i + 1, max(n, 0), kv, D).to(dtype)
            self.dense.append((k, v))
            for x, pages in ((k, self.k), (v, self.v)):
                for j, p in enumerate(self.rows[i]):
                    part = x[j * page:(j + 1) * page]
                    pages[p, :, :len(part)] = part.transpose(0, 1)


def run_chunk(hq, cache, new, heads, D, dtype, window=None, sinks=0, scale=None, seed=100, behind=0):
    q = (1.5 * randn(seed, sum(new) + behind, heads, D)).to(dtype)
    out = torch.full_like(q, 7.0)
    got = hq.chunk_attention(q, cache.k, cache.v, cache.table, i32(cache.lengths), i32(bounds(new)), window=window, sinks=sinks, scale=scale, out=out)
    assert got is out and (out[sum(new):] == 7).all()
    return q, out


def check_chunk(q, out, cache, new, window, sinks, scale, u):
    at = 0
    for n, (k, v) in zip(new, cache.dense):
        if n:
            part, o, m = q[at:at + n], out[at:at + n], k.shape[0]
            if n > m:  # tokens before the first one see nothing
                assert (o[:n - m] == 0).all()
                part, o = part[n - m:], o[n - m:]
            if m:
                check(o, part, k, v, window, sinks, scale or 1 / math.sqrt(q.shape[2]), u)
        at += n


# (new tokens, lengths with them)
CHUNKS = [([1], [1]), ([1], [333]), ([1], [3000]), ([5, 1, 0, 3], [700, 9, 50, 3]), ([4], [4]), ([2], [0]), ([9, 40], [5, 300]), ([17], [17]),
          ([33], [1000]), ([200, 1, 1], [200, 1500, 64]), ([129], [129]), ([300], [2200])]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (8, 2), (14, 2), (40, 1)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (100, 4), (64, 64), (37, 130), (1000, 1)])
def test_chunk(hq, kind, D, heads, window, sinks):
    dtype, u = TYPES[kind]
    for n, (new, lengths) in enumerate(CHUNKS):
        cache = Cache(10 * n, lengths, heads[1], (16, 8, 64)[n % 3], D, dtype)
        q, out = run_chunk(hq, cache, new, heads[0], D, dtype, window, sinks, seed=n, behind=n % 2)
        check_chunk(q, out, cache, new, window, sinks, None, u)


@pytest.mark.parametrize("D", [64, 128])
def test_chunk_many_requests(hq, D):
    """More than 64: found by their bounds; some of them chunks, some empty."""
    dtype, u = TYPES["bf16"]
    for rows, heads in ((65, (8, 2)), (150, (6, 1)), (400, (4, 4))):
        new = [(i * 7) % 4 + (37 if i % 50 == 3 else 0) for i in range(rows)]
        lengths = [n + (i * 13) % 90 + (900 if i % 40 == 1 else 0) for i, n in enumerate(new)]
        for window, sinks in ((None, 0), (20, 3)):
            cache = Cache(rows, lengths, heads[1], 16, D, dtype)
            q, out = run_chunk(hq, cache, new, heads[0], D, dtype, window, sinks, behind=2)
            check_chunk(q, out, cache, new, window, sinks, None, u)


def test_chunk_of_one_token_is_paged_attention(hq):
    """The same numbers to rounding, whatever the plan."""
    dtype, u = TYPES["f16"]
    lengths = [1, 900, 4000, 64, 129]
    cache = Cache(3, lengths, 2, 16, 128, dtype)
    q, out = run_chunk(hq, cache, [1] * 5, 8, 128, dtype)
    paged = hq.paged_attention(q, cache.k, cache.v, cache.table, i32(lengths))
    check_chunk(q, out, cache, [1] * 5, None, 0, None, u)
    check_chunk(q, paged, cache, [1] * 5, None, 0, None, u)


def test_chunk_pages_that_nobody_sees(hq):
    """Behind a window pages may have gone; what is needed and no page counts as zeros."""
    dtype, u = TYPES["bf16"]
    lengths, new, window, sinks = [1000, 700], [3, 100], 150, 5
    cache = Cache(5, lengths, 2, 16, 64, dtype)
    q, want = run_chunk(hq, cache, new, 8, 64, dtype, window, sinks)
    for row, n in enumerate(lengths):
        lowest = n - new[row] - window + 1
        cache.table[row, 1:lowest // 16] = -1
    q, out = run_chunk(hq, cache, new, 8, 64, dtype, window, sinks)
    assert torch.equal(out, want)
    cache.table[0, 60] = 9999
    cache.dense[0][0][960:976] = 0
    cache.dense[0][1][960:976] = 0
    q, out = run_chunk(hq, cache, new, 8, 64, dtype, window, sinks)
    check_chunk(q, out, cache, new, window, sinks, None, u)
    none = torch.zeros((0, 2, 16, 64), dtype=dtype, device="cuda")
    out = hq.chunk_attention(q, none, none, cache.table, i32(lengths), i32(bounds(new)))
    assert (out == 0).all()
    out = hq.chunk_attention(q, cache.k, cache.v, cache.table[:, :0].contiguous(), i32(lengths), i32(bounds(new)))
    assert (out == 0).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf, "most"])
@pytest.mark.parametrize("new", [[3, 1], [70, 40], [1, 1]])
def test_what_is_not_seen_has_no_effect(hq, kind, D, what, new):
    """Keys and values that some tokens see and others do not: those that do not give the same bits, those that see a value that is not
    finite give NaN in its element."""
    dtype, _ = TYPES[kind]
    lengths, window, sinks = [400, 333], 120, 6
    heads, kv = 8, 4
    cache = Cache(1, lengths, kv, 16, D, dtype)
    bad = torch.finfo(dtype).max if what == "most" else what
    q, want = run_chunk(hq, cache, new, heads, D, dtype, window, sinks)
    packed = [torch.cat([d[i] for d in cache.dense]) for i in range(2)]
    cu, ck = i32(bounds(new)), i32(bounds(lengths))
    prompt = hq.prompt_attention(q, *packed, cu, ck, window=window, sinks=sinks)
    for key in (6, 7, 8, 100, 400 - 70 - 121, 400 - 3 - 120, 279, 280, 281, 340, 398):
        kc, vc, kp, vp = cache.k.clone(), cache.v.clone(), packed[0].clone(), packed[1].clone()
        page = cache.rows[0][key // 16]
        kc[page, 1, key % 16, 3] = bad
        vc[page, 2, key % 16, 5] = bad
        kp[key, 1, 3] = bad
        vp[key, 2, 5] = bad
        sees = seen_of(new[0], 400, window, sinks)[:, key]
        for got, ref in ((hq.chunk_attention(q, kc, vc, cache.table, i32(lengths), cu, window=window, sinks=sinks), want),
                         (hq.prompt_attention(q, kp, vp, cu, ck, window=window, sinks=sinks), prompt)):
            touched = torch.zeros_like(got, dtype=torch.bool)
            touched[:new[0]][sees, 2:4] = True                       # of key head 1
            touched[:new[0], 4:6, 5] = sees[:, None].expand(-1, 2)   # of value head 2
            assert torch.equal(got[~touched], ref[~touched]), key
            if what != "most":
                assert torch.isnan(got[:new[0]][sees][:, 4:6, 5]).all(), key


def apart(u):
    """How far two results of the same attention may be from each other: both within close()'s bound, values of at most 5.5, scores' sums S of
    at most 16."""
    return 2 * 1.02 * (2 * u + 2.0 ** -13 + 2.0 ** -15 * 16) * 5.5


# ---- prompts through a window ------------------------------------------------------------------------------------------
PROMPTS = [([1], [1]), ([33], None), ([127, 0, 1, 200], None), ([300, 65], None), ([3], [259]), ([40, 1, 0], [700, 64, 9]), ([70], [10]),
           ([5, 6], [0, 6]), ([1], [1025]), ([600], [900])]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (8, 2), (14, 2), (40, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (100, 4), (64, 64), (37, 130), (1000, 1), (8, 8), (200, 1)])
def test_prompt_window(hq, kind, D, heads, window, sinks):
    dtype, u = TYPES[kind]
    for n, (nq, nk) in enumerate(PROMPTS):
        cu_k = nk
        nk = nk or nq
        q, k, v = (randn(n * 10 + i, sum(m), h, D).to(dtype) for i, (m, h) in enumerate(((nq, heads[0]), (nk, heads[1]), (nk, heads[1]))))
        out = hq.prompt_attention(q, k, v, i32(bounds(nq)), None if cu_k is None else i32(bounds(nk)), window=window, sinks=sinks)
        a = b = 0
        for x, y in zip(nq, nk):
            if x > y:
                assert (out[a:a + x - y] == 0).all()
            if min(x, y):
                check(out[a + max(x - y, 0):a + x], q[a + max(x - y, 0):a + x], k[b:b + y], v[b:b + y], window, sinks, 1 / math.sqrt(D), u)
            a, b = a + x, b + y


def test_prompt_window_of_everything(hq):
    """A window as long as the prompts is none: the same bits."""
    q, k, v = (randn(i, 300, h, 128).half() for i, h in enumerate((8, 2, 2)))
    want = hq.prompt_attention(q, k, v, i32([0, 180, 300]))
    for window, sinks in ((300, 0), (2 ** 31 - 1, 5), (2 ** 40, 2 ** 40)):
        assert torch.equal(hq.prompt_attention(q, k, v, i32([0, 180, 300]), window=window, sinks=sinks), want)
    got = hq.prompt_attention(q, k, v, i32([0, 180, 300]), window=180)
    assert (got.float() - want.float()).abs().max().item() <= apart(2.0 ** -11)


def test_prompt_window_parts_of_a_projection(hq):
    dtype, u = TYPES["bf16"]
    n, heads, kv, D = 300, 8, 2, 128
    qkv = randn(1, n, heads + 2 * kv, D).to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    out = torch.full((n, heads, D), 7.0, dtype=dtype, device="cuda")
    assert hq.prompt_attention(q, k, v, i32([0, 190, 250]), out=out, window=50, sinks=2) is out
    for a, b in ((0, 190), (190, 250)):
        check(out[a:b], q[a:b], k[a:b], v[a:b], 50, 2, 1 / math.sqrt(D), u)
    assert (out[250:] == 7.0).all()


# ---- graphs, streams, strides --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("warm", [True, False])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 60, 1]])
def test_graph(hq, warm, new):
    """Captured with and without a workspace to divide keys in, replayed with other lengths, tables and data."""
    dtype, u = TYPES["bf16"]
    lengths = [1500, 900, 64]
    cache = Cache(1, lengths, 2, 16, 128, dtype)
    q, cu, ln = randn(5, sum(new), 8, 128).to(dtype), i32(bounds(new)), i32(lengths)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(stream):
            hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu)
            hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu, window=200, sinks=4)
        stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        a = hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu)
        b = hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu, window=200, sinks=4)
    for i in range(4):
        q.copy_(randn(20 + i, *q.shape))
        now = [n - 13 * i for n in lengths]
        ln.copy_(i32(now))
        a.zero_()
        graph.replay()
        torch.cuda.synchronize()
        cache.lengths = now
        short = Cache.__new__(Cache)
        short.dense = [(k[:n], v[:n]) for (k, v), n in zip(cache.dense, now)]
        check_chunk(q, a, short, new, None, 0, None, u)
        check_chunk(q, b, short, new, 200, 4, None, u)


def test_streams_and_strides(hq):
    """Two streams at once, each with its own workspace; queries out of a projection's rows; a scale."""
    dtype, u = TYPES["f16"]
    new, lengths = [2, 30, 1], [2000, 1100, 700]
    cache = Cache(1, lengths, 2, 32, 64, dtype)
    qkv = randn(9, sum(new), 12, 64).to(dtype)
    q = qkv[:, :8]
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(hq.chunk_attention(q, cache.k, cache.v, cache.table, i32(lengths), i32(bounds(new)), scale=0.3))
    torch.cuda.synchronize()
    check_chunk(q, outs[0][0], cache, new, None, 0, 0.3, u)
    for o in outs[0] + outs[1]:
        assert torch.equal(o, outs[0][0])


def test_bounds_out_of_range_stay_inside(hq):
    """Bounds and lengths that are cut to what there is: negative ones, too large ones; lengths beyond the table."""
    dtype, u = TYPES["bf16"]
    cache = Cache(1, [64, 64, 64], 2, 16, 64, dtype)
    q = randn(3, 10, 4, 64).to(dtype)
    ref = hq.chunk_attention(q, cache.k, cache.v, cache.table, i32([64, 0, 64]), i32([0, 4, 6, 10]))
    got = hq.chunk_attention(q, cache.k, cache.v, cache.table, i32([1000, -5, 2 ** 31 - 1]), i32([-7, 4, 6, 99]))
    assert torch.equal(got, ref)


# ---- together ----------------------------------------------------------------------------------------------------------
def test_a_prompt_in_pieces_equals_the_whole(hq):
    """Norm, rotation and the cache in one pass, attention of the pieces - chunks, drafts, single tokens - over it: what one pass over the
    whole prompts gives, with a window and without."""
    dtype, u = TYPES["f16"]
    heads, kv, D, page = 8, 2, 64, 16
    total = [333, 150]
    qkv = [randn(i, n, heads + 2 * kv, D).to(dtype) for i, n in enumerate(total)]
    qw, kw = ((1 + 0.2 * randn(9 + i, D)).to(dtype) for i in range(2))
    angles = hq.rotary_table(400, D)
    for window, sinks in ((None, 0), (90, 4)):
        whole = torch.cat(qkv)
        positions = i32(list(range(total[0])) + list(range(total[1])))
        rq, rk = hq.norm_rotate(whole[:, :heads], whole[:, heads:heads + kv], angles, positions, qw, kw)
        want = hq.prompt_attention(rq, rk, whole[:, heads + kv:], i32([0] + [sum(total[:1]), sum(total)]), window=window, sinks=sinks)
        want = [want[:total[0]], want[total[0]:]]
        kp, vp = (torch.zeros((40, kv, page, D), dtype=dtype, device="cuda") for _ in range(2))
        table = i32([list(range(0, 22)), list(range(39, 17, -1))])
        table[1, 10:] = -1
        done = [0, 0]
        for new in ([100, 100], [64, 1], [1, 5], [130, 44], [38, 0]):
            part = torch.cat([x[a:a + n] for x, a, n in zip(qkv, done, new)])
            cu = i32(bounds(new))
            q = hq.cache_write_rotated(part[:, :heads], part[:, heads:heads + kv], part[:, heads + kv:], kp, vp, table, i32(done), cu, angles, qw, kw)
            done = [a + n for a, n in zip(done, new)]
            out = hq.chunk_attention(q, kp, vp, table, i32(done), cu, window=window, sinks=sinks)
            for i, o in enumerate((out[:new[0]], out[new[0]:])):
                ref = want[i][done[i] - new[i]:done[i]]
                assert not new[i] or (o.float() - ref.float()).abs().max().item() <= apart(u)
        assert done == total
