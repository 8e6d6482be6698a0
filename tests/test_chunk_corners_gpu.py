"""Corners of attention over the paged cache and of the rotation into it: offsets beyond 32 bits, pages of 1024 tokens, many query heads a key head,
bounds that begin late, scales and scores at the ends, plans of many shapes, workspaces of two graphs.  Bounds as in test_attention_gpu."""
import math

import pytest
import torch

from tests.test_attention_gpu import TYPES, bounds, i32, randn
from tests.test_chunk_gpu import Cache, check, check_chunk, run_chunk, seen_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,D", [(4, 4, 128), (14, 2, 64)])
def test_offsets_beyond_32_bits(hq, heads, kv, D):
    """The last pages of a pool of more than 4 GiB: written and rotated, and attended to by one token and by many."""
    dtype, u = TYPES["bf16"]
    page, bytes_of_page = 16, kv * 16 * D * 2
    pages = 4400000000 // bytes_of_page
    kp, vp = (torch.empty((pages, kv, page, D), dtype=dtype, device="cuda") for _ in range(2))
    rows = [[pages - 1 - i for i in range(20)], [pages // 2 + 3 * i for i in range(20)]]
    table, new = i32(rows), [300, 200]
    qkv = randn(1, sum(new), heads + 2 * kv, D).to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    angles = hq.rotary_table(512, D)
    rq = hq.cache_write_rotated(q, k, v, kp, vp, table, i32([0, 0]), i32(bounds(new)), angles)
    want_q, want_k = hq.norm_rotate(q, k, angles, i32(list(range(300)) + list(range(200))))
    assert torch.equal(rq, want_q)
    for part in ([300, 200], [1, 1], [7, 90]):
        pick = torch.cat([torch.arange(300 - part[0], 300), torch.arange(500 - part[1], 500)]).cuda()
        out = hq.chunk_attention(rq[pick], kp, vp, table, i32(new), i32(bounds(part)))
        for a, b, lo, hi in ((0, part[0], 0, 300), (part[0], sum(part), 300, 500)):
            check(out[a:b], rq[pick][a:b], want_k[lo:hi], v[lo:hi], None, 0, 1 / math.sqrt(D), u)


def test_rows_further_apart_than_32_bits(hq):
    """Tokens of a very wide projection."""
    stride, n = 1 << 28, 9
    flat = torch.empty(stride * n, dtype=torch.float16, device="cuda")
    wide = flat.as_strided((n, 6, 64), (stride, 64, 1))
    wide.copy_(randn(1, n, 6, 64))
    q, k, p = wide[:, :4], wide[:, 4:], i32(list(range(n)))
    angles = hq.rotary_table(16, 64)
    want = hq.norm_rotate(q.contiguous(), k.contiguous(), angles, p)
    got = hq.norm_rotate(q, k, angles, p)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    hq.norm_rotate(q, k, angles, p, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 9)])
def test_large_pages_and_many_heads(hq, D, window, sinks):
    dtype, u = TYPES["f16"]
    for heads, kv in ((200, 1), (34, 2), (17, 1)):
        new, lengths = [1, 2, 30], [2500, 1024, 1300]
        cache = Cache(heads, lengths, kv, 1024, D, dtype)
        q, out = run_chunk(hq, cache, new, heads, D, dtype, window, sinks)
        check_chunk(q, out, cache, new, window, sinks, None, u)


@pytest.mark.parametrize("rows", [3, 70])
def test_bounds_that_begin_late(hq, rows):
    """Tokens before the first request's are left as they were, as are those behind the last one's."""
    dtype, u = TYPES["bf16"]
    new, lengths = [1 + i % 5 + (60 if i == 1 else 0) for i in range(rows)], [40 + 9 * (i % 11) + (800 if i == 2 else 60) for i in range(rows)]
    cache = Cache(3, lengths, 2, 16, 64, dtype)
    before = 137
    q = randn(5, before + sum(new) + 2, 8, 64).to(dtype)
    out = torch.full_like(q, 7.0)
    cu = i32([before + b for b in bounds(new)])
    hq.chunk_attention(q, cache.k, cache.v, cache.table, i32(lengths), cu, out=out)
    assert (out[:before] == 7).all() and (out[before + sum(new):] == 7).all()
    check_chunk(q[before:], out[before:], cache, new, None, 0, None, u)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
def test_scales(hq, kind, D):
    dtype, u = TYPES[kind]
    for scale in (0.0, 2.0, 1e-30):
        for new, lengths in (([3], [900]), ([60], [400]), ([1, 1], [70, 600])):
            cache = Cache(1, lengths, 2, 16, D, dtype)
            for window, sinks in ((None, 0), (90, 4)):
                q, out = run_chunk(hq, cache, new, 8, D, dtype, window, sinks, scale=scale)
                at = 0
                for n, (k, v) in zip(new, cache.dense):
                    check(out[at:at + n], q[at:at + n], k, v, window, sinks, scale, u)
                    at += n


def test_scores_far_from_zero(hq):
    """Scores of 10^7 and masked keys: results are finite, and an equal shift of all scores changes nothing (one key has all the weight)."""
    dtype, _ = TYPES["bf16"]
    for new in ([2], [50]):
        cache = Cache(1, [300], 1, 16, 64, dtype)
        cache.k.nan_to_num_(0)
        cache.k[cache.rows[0][16], 0, 5] = 1000.0  # token 261
        q = torch.full((new[0], 4, 64), 1000.0, dtype=dtype, device="cuda")
        out = hq.chunk_attention(q, cache.k, cache.v, cache.table, i32([300]), i32([0, new[0]]), window=60, sinks=2)
        seen = torch.arange(300 - new[0], 300, device="cuda") >= 261
        assert torch.isfinite(out).all()
        want = cache.dense[0][1][261, 0]
        assert torch.equal(out[seen], want.expand_as(out[seen]))


def test_a_query_that_is_not_finite_stays_alone(hq):
    dtype, _ = TYPES["f16"]
    for new in ([3, 2], [40, 30]):
        cache = Cache(1, [500, 300], 2, 16, 64, dtype)
        q, want = run_chunk(hq, cache, new, 4, 64, dtype, 100, 3)
        bad = q.clone()
        bad[1, 2, 7] = math.nan
        out = hq.chunk_attention(bad, cache.k, cache.v, cache.table, i32([500, 300]), i32(bounds(new)), window=100, sinks=3)
        assert torch.isnan(out[1, 2]).all()
        out[1, 2] = want[1, 2]
        assert torch.equal(out, want)


def test_plans(hq):
    """Requests of one token, drafts and chunks of many shapes beside each other: whatever is divided and whatever is not."""
    dtype, u = TYPES["bf16"]
    g = torch.Generator().manual_seed(5)
    rand = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    for case in range(24):
        heads, kv = ((8, 2), (4, 4), (32, 8), (16, 1), (7, 7))[case % 5]
        rows = rand(1, 64) if case % 3 else rand(1, 4)
        new = [(1, rand(2, 9), rand(0, 70), rand(100, 400))[rand(0, 3) if case % 2 else 0 if rand(0, 7) else 3] for _ in range(rows)]
        lengths = [n + (rand(0, 40), rand(100, 700), rand(2000, 5000))[rand(0, 2) if rows < 9 else rand(0, 1)] for n in new]
        D, page = (64, 128)[case % 2], (8, 16, 128)[case % 3]
        window, sinks = ((None, 0), (rand(1, 600), rand(0, 20)))[case % 4 == 1]
        cache = Cache(case, lengths, kv, page, D, dtype)
        q, out = run_chunk(hq, cache, new, heads, D, dtype, window, sinks, seed=case)
        check_chunk(q, out, cache, new, window, sinks, None, u)
        again = hq.chunk_attention(q, cache.k, cache.v, cache.table, i32(lengths), i32(bounds(new)), window=window, sinks=sinks)
        assert torch.equal(again[:sum(new)], out[:sum(new)]), case  # the same call, the same bits


def test_two_graphs_of_a_stream_in_turn(hq):
    """They share the stream's workspace, counters among it; replayed one after the other, with eager calls between."""
    dtype, u = TYPES["bf16"]
    stream = torch.cuda.Stream()
    calls = []
    for i, (new, lengths) in enumerate((([1, 1], [3000, 700]), ([30, 6, 1], [1200, 2500, 90]))):
        cache = Cache(i, lengths, 2, 16, 128, dtype)
        q = randn(7 + i, sum(new), 8, 128).to(dtype)
        args = (q, cache.k, cache.v, cache.table, i32(lengths), i32(bounds(new)))
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            hq.chunk_attention(*args)
        stream.synchronize()
        calls.append((args, cache, new))
    graphs = []
    for args, cache, new in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = hq.chunk_attention(*args)
        graphs.append((graph, out))
    for i in range(6):
        with torch.cuda.stream(stream):
            graphs[i % 2][1].zero_()
            graphs[i % 2][0].replay()
            eager = hq.chunk_attention(*calls[1 - i % 2][0])
        stream.synchronize()
        for out, (args, cache, new) in ((graphs[i % 2][1], calls[i % 2]), (eager, calls[1 - i % 2])):
            check_chunk(args[0], out, cache, new, None, 0, None, u)


@pytest.mark.parametrize("heads,kv,batch", [(4, 1, 64), (8, 2, 64), (32, 8, 20), (16, 1, 63), (8, 2, 90)])
def test_bounds_that_do_not_ascend(hq, heads, kv, batch):
    """Whatever they are, the call ends, tokens of no request stay as they were, and the next call finds its workspace in order."""
    dtype, u = TYPES["bf16"]
    lengths = [400 + 37 * (i % 5) for i in range(batch)]
    cache = Cache(2, lengths, kv, 16, 128, dtype)
    q = randn(3, 8 + 40, heads, 128).to(dtype)
    for window, sinks in ((None, 0), (150, 5)):
        for cycle in ((0, 4), (4, 8, 0), (0, 8, 3, 8, -5), (8, 0, 10 ** 9, 5, -2 ** 31), (8, 7, 6, 5), (0, 48), (2, 40, 1)):
            cu = [cycle[i % len(cycle)] for i in range(batch + 1)]
            out = torch.full_like(q, 7.0)
            hq.chunk_attention(q, cache.k, cache.v, cache.table, i32(lengths), i32(cu), window=window, sinks=sinks, out=out)
            inside = {t for a, b in zip(cu, cu[1:]) for t in range(max(a, 0), min(b, len(q)))}
            outside = [t for t in range(len(q)) if t not in inside]
            assert (out[outside] == 7).all(), cycle
            new = [1 + (i % 3 == 0) for i in range(batch)]
            good, got = run_chunk(hq, cache, new, heads, 128, dtype, window, sinks)
            check_chunk(good, got, cache, new, window, sinks, None, u)


# Tiles, undivided, of 128 to 256 workgroups, or 64 with few keys: those of twice the waves, and some beside them.
ALONE = [((64, 64), [350], [1500]), ((64, 16), [350], [901]), ((64, 16), [200, 150], [1300, 149]), ((64, 16), [340, 1, 9], [345, 700, 60]),
         ((64, 32), [400, 0], [100, 50]), ((64, 16), [6, 360], [6, 2000]), ((60, 12), [450], [450]),
         ((32, 8), [400], [900]), ((32, 8), [300, 90, 2], [700, 400, 500]), ((32, 8), [257], [300])]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads,new,lengths", ALONE)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (100, 4), (700, 130)])
def test_tiles_that_have_a_compute_unit_each(hq, kind, D, heads, new, lengths, window, sinks):
    dtype, u = TYPES[kind]
    cache = Cache(4, lengths, heads[1], 16, D, dtype)
    q, out = run_chunk(hq, cache, new, heads[0], D, dtype, window, sinks, behind=2)
    check_chunk(q, out, cache, new, window, sinks, None, u)
    again = hq.chunk_attention(q, cache.k, cache.v, cache.table, i32(lengths), i32(bounds(new)), window=window, sinks=sinks)
    assert torch.equal(again[:sum(new)], out[:sum(new)])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf, "most"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 6)])
def test_tiles_that_have_a_compute_unit_each_and_what_is_not_seen(hq, kind, D, what, window, sinks):
    """As test_what_is_not_seen_has_no_effect: pages of keys and values in both halves of a tile, a missing page among them."""
    dtype, _ = TYPES[kind]
    new, length, bad = 350, 800, torch.finfo(dtype).max if what == "most" else what
    cache = Cache(6, [length], 16, 16, D, dtype)
    q, want = run_chunk(hq, cache, [new], 64, D, dtype, window, sinks)
    for key in (3, 6, 63, 64, 301, 450, 451, 512, 600, 640, 700, 799):
        k, v = cache.k.clone(), cache.v.clone()
        page = cache.rows[0][key // 16]
        k[page, 1, key % 16, 3] = bad
        v[page, 2, key % 16, 5] = bad
        sees = seen_of(new, length, window, sinks)[:, key]
        got = hq.chunk_attention(q, k, v, cache.table, i32([length]), i32([0, new]), window=window, sinks=sinks)
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[sees, 4:8] = True
        touched[:, 8:12, 5] = sees[:, None].expand(-1, 4)
        assert torch.equal(got[~touched], want[~touched]), key
        if what != "most":
            assert torch.isnan(got[sees][:, 8:12, 5]).all(), key
    for missing in (0, 20, 38, 40):
        table, k, v = cache.table.clone(), cache.k.clone(), cache.v.clone()
        table[0, missing] = -1
        k[cache.rows[0][missing]] = 0
        v[cache.rows[0][missing]] = 0
        args = (i32([length]), i32([0, new]), window, sinks)
        assert torch.equal(hq.chunk_attention(q, cache.k, cache.v, table, *args), hq.chunk_attention(q, k, v, cache.table, *args))


@pytest.mark.parametrize("D", [64, 128])
def test_tiles_that_have_a_compute_unit_each_in_a_graph(hq, D):
    """Replayed with other lengths, beside eager calls; the stream's first call is the captured one."""
    dtype, u = TYPES["bf16"]
    cache = Cache(8, [1400], 16, 16, D, dtype)
    q, cu, ln = randn(5, 350, 64, D).to(dtype), i32([0, 350]), i32([1400])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu)
    for length in (1400, 350, 777, 20):
        ln.copy_(i32([length]))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu))
        n = min(length, 350)
        assert (out[:350 - n] == 0).all()
        check(out[350 - n:], q[350 - n:], *(x[:length] for x in cache.dense[0]), None, 0, 1 / math.sqrt(D), u)
