"""More than 16 query heads a key / value head: a token by itself is a tile of many rows, whose keys are divided like any others.  Bounds as in
test_attention_gpu."""
import math

import pytest
import torch

from tests.test_attention_gpu import TYPES, attend, bounds, close, i32, randn
from tests.test_chunk_gpu import Cache, run_chunk, seen_of

pytestmark = pytest.mark.gpu


def check_chunk(q, out, cache, new, window, sinks, u):
    """A key / value head at a time, all rows of its group."""
    at, D = 0, q.shape[2]
    for n, (k, v) in zip(new, cache.dense):
        r = q.shape[1] // k.shape[1]
        seen = seen_of(n, k.shape[0], window, sinks).repeat_interleave(r, 0)
        for g in range(k.shape[1] if n else 0):
            rows, got = (x[at:at + n, g * r:(g + 1) * r].reshape(n * r, D) for x in (q, out))
            want, a, big = attend(rows.double(), k[:, g].double(), v[:, g].double(), seen, 1 / math.sqrt(D))
            close(got, want, a, big, u)
        at += n


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads,D", [((17, 1), 64), ((32, 1), 128), ((40, 2), 64), ((128, 4), 128), ((129, 1), 64), ((200, 1), 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (900, 5)])
def test_single_tokens(hq, kind, heads, D, window, sinks):
    dtype, u = TYPES[kind]
    for n, (new, lengths) in enumerate((([1], [9000]), ([1], [513]), ([1, 1, 0, 1], [4000, 1, 77, 650]), ([1] * 20, [300 + 71 * i for i in range(20)]),
                                        ([1, 5, 1], [3000, 2000, 512]), ([1] * 64, [40 + 11 * i for i in range(64)]))):
        cache = Cache(7 * n, lengths, heads[1], 16, D, dtype)
        q, out = run_chunk(hq, cache, new, heads[0], D, dtype, window, sinks, seed=n, behind=1)
        check_chunk(q, out, cache, new, window, sinks, u)
        again = hq.chunk_attention(q, cache.k, cache.v, cache.table, i32(lengths), i32(bounds(new)), window=window, sinks=sinks)
        assert torch.equal(again[:sum(new)], out[:sum(new)])


@pytest.mark.parametrize("warm", [True, False])
def test_graph(hq, warm):
    """Captured with room for shares and without, replayed with other lengths."""
    dtype, u = TYPES["bf16"]
    cache = Cache(1, [5000, 800], 1, 16, 128, dtype)
    q, cu, ln = randn(5, 2, 32, 128).to(dtype), i32([0, 1, 2]), i32([5000, 800])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(stream):
            hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu)
        stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = hq.chunk_attention(q, cache.k, cache.v, cache.table, ln, cu)
    whole = list(cache.dense)
    for now in ([5000, 800], [1, 3], [4000, 640], [513, 129]):
        ln.copy_(i32(now))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        cache.dense = [(k[:n], v[:n]) for (k, v), n in zip(whole, now)]
        check_chunk(q, out, cache, [1, 1], None, 0, u)


def time_of(f):
    for _ in range(3):
        f()
    best = float("inf")
    for _ in range(5):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(10):
            f()
        end.record()
        end.synchronize()
        best = min(best, begin.elapsed_time(end))
    return best


@pytest.mark.parametrize("heads", [(32, 1), (40, 2)])
def test_no_slower_than_a_few_times_the_attention_of_single_tokens(hq, heads):
    """One workgroup a head through all keys takes 27 times as long; divided, the two are about as fast."""
    pages, kv = 1900, heads[1]
    q = randn(1, 1, heads[0], 128).bfloat16()
    k, v = (randn(i, pages, kv, 16, 128).bfloat16() for i in range(2))
    table, lengths, cu = i32([list(range(pages))]), i32([30000]), i32([0, 1])
    chunk = time_of(lambda: hq.chunk_attention(q, k, v, table, lengths, cu))
    paged = time_of(lambda: hq.paged_attention(q, k, v, table, lengths))
    assert chunk <= 4 * paged, (chunk, paged)
