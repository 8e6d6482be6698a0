"""The cache's own operators at sizes where there is nothing to copy, or a page's size is none that they take."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("pages", [0, 1, 300, 4096, 4097, 9000])
@pytest.mark.parametrize("planes", [0, 2])
def test_compact_pages_of_no_bytes(hq, pages, planes):
    """Tables are compacted whether there is something to move or not."""
    r = np.random.default_rng(pages)
    refs = [int(n) for n in (r.random(pages) < 0.6) * r.integers(1, 4, pages)]
    pool = torch.zeros((planes, pages, 0), dtype=torch.float16, device="cuda")
    table = r.integers(-2, pages + 2, (5, 11)).tolist()
    live = sum(n > 0 for n in refs)
    holes, movers = [p for p in range(live) if refs[p] <= 0], [p for p in range(live, pages) if refs[p] > 0]
    to, want = dict(zip(movers, holes)), refs[:]
    for source, target in to.items():
        want[target], want[source] = refs[source], 0
    t, n, got = hq.cache_compact(pool, i32(table), i32(refs))
    assert t.tolist() == [[to.get(p, p) for p in row] for row in table] and n.tolist() == want and got.tolist() == [live]


def test_step_pages_of_no_bytes(hq):
    for pages in (40, 5000):
        pool = torch.zeros((2, pages, 0), dtype=torch.float16, device="cuda")
        table, lengths, refs = [[3, 5, -1], [3, 7, -1]], [20, 30], [0] * pages
        refs[3], refs[5], refs[7] = 2, 1, 1
        t, n, c, s, missing = hq.cache_step(pool, 16, i32(table), i32(lengths), i32(refs), i32([0, 0]), i32([1, 1]))
        assert t.tolist() == [[3, 5, -1], [3, 0, -1]] and n.tolist() == [21, 21] and s.tolist() == [20, 20] and missing.tolist() == [0]
        assert c.tolist()[:8] == [1, 0, 0, 2, 0, 1, 0, 0]
