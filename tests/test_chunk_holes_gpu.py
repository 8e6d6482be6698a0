"""Pages behind a window given back while their requests go on: entries of -1 in the tables, counts a row less, through steps, forks and
compactions.  Bounds as in test_attention_gpu."""
import numpy as np
import pytest
import torch

from tests.test_attention_gpu import TYPES, bounds, i32, randn
from tests.test_chunk_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages", [44, 5000])  # the step and the compaction in one launch, and in two
@pytest.mark.parametrize("sinks", [0, 5, 17])
def test_pages_behind_the_window(hq, pages, sinks):
    dtype, u = TYPES["bf16"]
    rows, heads, kv, D, page, window, free = 6, 8, 2, 64, 16, 40, 44
    r = np.random.default_rng(sinks)
    pool = torch.zeros((2, pages, kv, page, D), dtype=dtype, device="cuda")
    table, lengths = torch.full((rows, 24), -1, dtype=torch.int32, device="cuda"), i32([0] * rows)
    refs = i32([0] * free + [1] * (pages - free))  # the others are somebody else's
    kept = [tuple(torch.zeros((0, kv, D), dtype=dtype, device="cuda") for _ in range(2)) for _ in range(rows)]
    parent, given_back = list(range(rows)), 0
    for step in range(60):
        if step:
            parent = list(range(rows))
        if step % 17 == 9:
            parent[int(r.integers(rows))] = int(r.integers(rows))  # a fork in the place of another row
        if step % 23 == 20:
            parent[int(r.integers(rows))] = -1
        add = [int(n) for n in r.integers(0, 11, rows)]
        table, lengths, refs, starts, missing = hq.cache_step(pool, page, table, lengths, refs, i32(parent), i32(add))
        assert missing.item() == 0
        if step % 8 == 5:
            table, refs, live = hq.cache_compact(pool, table, refs)
            assert (refs[:live.item()] > 0).all() and (refs[live.item():] == 0).all()
        n, cu = sum(add), i32(bounds(add))
        k, v, q = (randn(3 * step + i, n, h, D).to(dtype) for i, h in enumerate((kv, kv, heads)))
        hq.cache_write(k, v, pool[0], pool[1], table, starts, cu)
        empty = kept[0][0][:0]
        at = bounds(add)
        old, kept = kept, []
        for s in range(rows):
            before = old[parent[s]] if parent[s] >= 0 else (empty, empty)
            kept.append(tuple(torch.cat([a, x[at[s]:at[s + 1]]]) for a, x in zip(before, (k, v))))
        assert lengths.tolist() == [len(a) for a, _ in kept]
        out = hq.chunk_attention(q, pool[0], pool[1], table, lengths, cu, window=window, sinks=sinks)
        for s in range(rows):
            if add[s]:
                check(out[at[s]:at[s + 1]], q[at[s]:at[s + 1]], *kept[s], window, sinks, D ** -0.5, u)
        # what no token to come sees: keys up to length - window, but the first ones
        t, c = table.cpu().numpy(), refs.cpu().numpy()
        for s, length in enumerate(lengths.tolist()):
            for j in range(-(-sinks // page), (length - window + 1) // page):
                if t[s, j] >= 0:
                    c[t[s, j]] -= 1
                    t[s, j] = -1
                    given_back += 1
        table.copy_(torch.from_numpy(t))
        refs.copy_(torch.from_numpy(c))
        assert (c >= 0).all()
        counts = np.bincount(t[t >= 0], minlength=pages)
        assert c.sum() == counts.sum() + pages - free
    assert given_back > free  # more pages than there are have been used
