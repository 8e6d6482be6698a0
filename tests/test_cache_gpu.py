"""The cache's own operators against a plain statement of what they do, whole numbers and bytes: equal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def pool_of(seed, planes, pages, elems):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-32768, 32768, (planes, pages, elems), generator=g, device="cuda", dtype=torch.int16)


# ---- tokens into pages -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,D", [(1, 64), (2, 128), (8, 128), (5, 8), (12, 64)])
def test_write(hq, dtype, heads, D):
    for page in (1, 16, 64):
        for new, starts, width in (([1], [0], 4), ([1, 1, 1], [0, 15, 16], 33), ([70, 0, 3], [2, 5, 9], 80), ([0], [0], 2),
                                   ([(i * 3) % 4 for i in range(200)], [(i * 5) % 40 for i in range(200)], 48)):
            width = -(-width * 2 // page)
            rows, pages = len(new), len(new) * width + 5
            table = torch.randperm(pages)[:rows * width].view(rows, width).int().cuda()
            cu = np.concatenate([[0], np.cumsum(new)])
            qkv = torch.randn((int(cu[-1]), 3 * heads, D), device="cuda").to(dtype)
            k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
            kp, vp = torch.randn((pages, heads, page, D), device="cuda").to(dtype), torch.randn((pages, heads, page, D), device="cuda").to(dtype)
            kw, vw, t = kp.clone(), vp.clone(), table.tolist()
            for s in range(rows):
                for i in range(new[s]):
                    p = starts[s] + i
                    kw[t[s][p // page], :, p % page] = k[cu[s] + i]
                    vw[t[s][p // page], :, p % page] = v[cu[s] + i]
            assert hq.cache_write(k, v, kp, vp, table, i32(starts), i32(cu)) is None
            assert torch.equal(kp, kw) and torch.equal(vp, vw)


def test_write_leaves_out_what_has_no_place(hq):
    k, v = torch.randn((12, 2, 64), device="cuda").half(), torch.randn((12, 2, 64), device="cuda").half()
    kp, vp = torch.zeros((4, 2, 8, 64), device="cuda").half(), torch.zeros((4, 2, 8, 64), device="cuda").half()
    # row 0: from -2 on, in page 1; row 1: its second page is missing; row 2: beyond the table; tokens 0 and 11 belong to nobody
    hq.cache_write(k, v, kp, vp, i32([[1, -1], [2, 9], [3, 0]]), i32([-2, 6, 2 ** 31 - 1]), i32([1, 4, 8, 11]))
    kw, vw = torch.zeros_like(kp), torch.zeros_like(vp)
    for src, dst in ((k, kw), (v, vw)):
        dst[1, :, 0] = src[3]
        dst[2, :, 6], dst[2, :, 7] = src[4], src[5]
    assert torch.equal(kp, kw) and torch.equal(vp, vw)


# ---- the step of the tables -------------------------------------------------------------------------------------------------
def step_model(page, table, lengths, refs, parent, add):
    rows, width, pages = len(table), len(table[0]), len(refs)
    cap = width * page
    real = lambda p: 0 <= p < pages  # noqa: E731
    old = [min(max(n, 0), cap) for n in lengths]
    refs = list(refs)
    for s in range(rows):
        for p in table[s][:-(-old[s] // page)]:
            if real(p):
                refs[p] -= 1
    out, starts, ends, asked, seen = [], [], [], [], set()
    for s in range(rows):
        p = parent[s]
        alive = 0 <= p < rows
        start = old[p] if alive else 0
        end = min(start + max(add[s], 0), cap)
        row = [-1] * width
        for j in range(-(-start // page)):
            e = table[p][j] if real(table[p][j]) else -1
            if (j + 1) * page > start and p in seen and e >= 0:
                asked.append((s, j, e))
            else:
                row[j] = e
                if e >= 0:
                    refs[e] += 1
        for j in range(-(-start // page), -(-end // page)):
            asked.append((s, j, -1))
        if alive:
            seen.add(p)
        out.append(row)
        starts.append(start)
        ends.append(end)
    free = [p for p in range(pages) if refs[p] <= 0]
    missing, copies = 0, []
    for s, j, source in asked:
        if free:
            out[s][j] = free.pop(0)
            refs[out[s][j]] = 1
            if source >= 0:
                copies.append((source, out[s][j]))
        else:
            missing += 1
            ends[s] = min(ends[s], j * page)
    return out, ends, refs, [min(a, b) for a, b in zip(starts, ends)], missing, copies


def check_step(hq, seed, page, table, lengths, refs, parent, add, planes=2, elems=24, out=None):
    pages = len(refs)
    pool = pool_of(seed, planes, pages, elems)
    want = step_model(page, table, lengths, refs, parent, add)
    want_pool = pool.clone()
    for source, target in want[5]:
        want_pool[:, target] = pool[:, source]
    got = hq.cache_step(pool, page, i32(table), i32(lengths), i32(refs), i32(parent), i32(add), out=out)
    for name, g, w in zip(("table", "lengths", "refs", "starts", "missing"), got, want[:4] + ([want[4]],)):
        assert g.tolist() == w, name
    assert torch.equal(pool, want_pool)
    return got, pool, want


def random_tables(r, rows, width, page, pages, groups=1):
    """Rows that share their first pages within a group, consistent counts."""
    order, table, lengths, refs = list(r.permutation(pages)), [], [], [0] * pages
    for g in range(groups):
        most = max(1, min(width, (len(order) - rows) // max(1, rows // groups + 1)))
        head = [int(order.pop()) for _ in range(int(r.integers(0, most)))]
        for _ in range(rows // groups):
            row = head[:]
            n = len(head) * page
            if len(row) < width and order and r.random() < 0.9:
                row.append(int(order.pop()))
                n += int(r.integers(1, page + 1))
            table.append(row + [-1] * (width - len(row)))
            lengths.append(n)
            for p in row:
                refs[p] += 1
    return table, lengths, refs


@pytest.mark.parametrize("rows,width,page,pages,groups", [(1, 1, 1, 1, 1), (1, 4, 16, 40, 1), (8, 6, 16, 100, 2), (12, 3, 8, 60, 3), (64, 9, 16, 1000, 8),
                                                          (300, 40, 4, 9000, 10), (33, 2, 64, 35, 1), (7, 500, 16, 5000, 1)])
def test_step(hq, rows, width, page, pages, groups):
    rows = rows // groups * groups
    for seed in range(6):
        r = np.random.default_rng(seed)
        table, lengths, refs = random_tables(r, rows, width, page, pages, groups)
        kind = seed % 3
        if kind == 0:    # everyone goes on by a token
            parent, add = list(range(rows)), [1] * rows
        elif kind == 1:  # anyone from anyone
            parent, add = [int(p) for p in r.integers(-2, rows + 2, rows)], [int(n) for n in r.integers(-3, 3 * page, rows)]
        else:            # beams
            n = rows // groups
            parent, add = [int(g * n + r.integers(0, n)) for g in range(groups) for _ in range(n)], [1] * rows
        got, pool, want = check_step(hq, seed, page, table, lengths, refs, parent, add)
        # and on from there, with fewer tokens, into tensors of ours
        out = [torch.empty_like(t) for t in got]
        parent = [int(p) for p in r.integers(-1, rows, rows)]
        again, _, _ = check_step(hq, seed + 50, page, want[0], want[1], want[2], parent, [2] * rows, out=out)
        assert all(a is b for a, b in zip(again, out))


def test_step_counts_held_by_others_and_numbers_that_are_no_pages(hq):
    refs = [1, 2, 0, 5, 0, -3, 1, 0]
    table = [[0, 1, -1, -1], [99, 6, -7, -1], [3, -1, -1, -1]]
    check_step(hq, 1, 16, table, [30, 40, 10 ** 9], refs, [0, 1, 1], [3, 0, 30])
    check_step(hq, 2, 16, table, [-5, 64, 1], refs, [1, 1, 1], [2 ** 31 - 1, 1, -2 ** 31])
    check_step(hq, 3, 16, table, [17, 17, 17], refs, [0, 0, 0], [1, 16, 32])


def test_step_of_nothing(hq):
    pool = pool_of(1, 2, 4, 8)
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    got = hq.cache_step(pool, 16, z.view(0, 5), z, i32([0, 2, 0, 1]), z, z)
    assert got[2].tolist() == [0, 2, 0, 1] and got[4].tolist() == [0] and got[0].shape == (0, 5)
    got = hq.cache_step(pool, 16, z.view(3, 0), i32([1, 2, 3]), i32([0, 2, 0, 1]), i32([0, 0, -1]), i32([1, 1, 1]))
    assert got[1].tolist() == [0, 0, 0] and got[2].tolist() == [0, 2, 0, 1] and got[4].tolist() == [0]


# ---- live pages to the front -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("pages,share", [(1, 1.0), (1, 0.0), (7, 0.5), (300, 0.3), (300, 0.95), (1000, 0.0), (1000, 1.0), (5003, 0.6)])
@pytest.mark.parametrize("planes,elems", [(1, 8), (6, 1000)])
def test_compact(hq, pages, share, planes, elems):
    for seed in range(3):
        r = np.random.default_rng(seed)
        refs = [int(n) for n in (r.random(pages) < share) * r.integers(1, 4, pages)]
        if seed == 2:
            refs = [n if n else -int(r.integers(0, 2)) for n in refs]
        table = r.integers(-2, pages + 2, (5, 11)).tolist()
        pool = pool_of(seed, planes, pages, elems)
        live = sum(n > 0 for n in refs)
        holes, movers = [p for p in range(live) if refs[p] <= 0], [p for p in range(live, pages) if refs[p] > 0]
        to, want_refs, want_pool = dict(zip(movers, holes)), refs[:], pool.clone()
        for source, target in to.items():
            want_refs[target], want_refs[source] = refs[source], 0
            want_pool[:, target] = pool[:, source]
        t, n, got = hq.cache_compact(pool, i32(table), i32(refs))
        assert t.tolist() == [[to.get(p, p) for p in row] for row in table]
        assert n.tolist() == want_refs and got.tolist() == [live]
        assert torch.equal(pool, want_pool)


def test_pools_of_every_type(hq):
    for dtype in (torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.uint8, torch.int32):
        pool = torch.arange(2 * 6 * 4 * 16, device="cuda").view(2, 6, 4, 16).to(dtype)
        want = pool.clone()
        want[:, 1] = pool[:, 4]
        t, refs, live = hq.cache_compact(pool, i32([[0, 4], [2, 4]]), i32([1, 0, 1, 0, 2, 0]))
        assert torch.equal(pool, want) and t.tolist() == [[0, 1], [2, 1]] and refs.tolist() == [1, 2, 1, 0, 0, 0] and live.tolist() == [3]


def test_other_stream_and_graph(hq):
    r = np.random.default_rng(3)
    table, lengths, refs = random_tables(r, 32, 8, 16, 400, 4)
    args = [i32(table), i32(lengths), i32(refs), i32(r.integers(-1, 32, 32)), i32([1] * 32)]
    s = torch.cuda.Stream()
    for name in ("step", "compact"):
        pool = pool_of(4, 2, 400, 64)
        call = (lambda p: hq.cache_step(p, 16, *args)) if name == "step" else (lambda p: hq.cache_compact(p, args[0], args[2]))
        wpool = pool.clone()
        want = call(wpool)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            mine = pool.clone()
            got = call(mine)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(mine, wpool)
        graph = torch.cuda.CUDAGraph()
        static = pool.clone()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            got = call(static)
        for i in range(3):
            args[3].copy_(i32(np.random.default_rng(i).integers(-1, 32, 32)))
            fresh = pool_of(5 + i, 2, 400, 64)
            static.copy_(fresh)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = call(fresh)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(static, fresh)


def test_a_search_with_forks_end_to_end(hq):
    """Tokens written, rows forked, moved together and attended to, against contiguous keys kept beside."""
    page, heads, D, rows = 16, 2, 64, 6
    r = np.random.default_rng(0)
    pool = torch.zeros((2, 120, heads, page, D), dtype=torch.float16, device="cuda")
    table, lengths, refs = i32([[-1] * 12] * rows), i32([0] * rows), i32([0] * 120)
    kept = [(np.zeros((0, heads, D), np.float32), np.zeros((0, heads, D), np.float32)) for _ in range(rows)]
    add = [int(n) for n in r.integers(1, 60, rows)]
    parent = [-1] * rows
    for step in range(8):
        table, lengths, refs, starts, missing = hq.cache_step(pool, page, table, lengths, refs, i32(parent), i32(add))
        assert missing.item() == 0
        if step % 3 == 2:
            table, refs, live = hq.cache_compact(pool, table, refs)
            assert (refs[:live.item()] > 0).all() and (refs[live.item():] == 0).all()
        n = sum(add)
        k, v = torch.randn((n, heads, D), device="cuda").half(), torch.randn((n, heads, D), device="cuda").half()
        cu = np.concatenate([[0], np.cumsum(add)])
        hq.cache_write(k, v, pool[0], pool[1], table, starts, i32(cu))
        kn, vn = k.float().cpu().numpy(), v.float().cpu().numpy()
        old = kept
        kept = []
        for s in range(rows):
            a, b = old[parent[s]] if parent[s] >= 0 else (kn[:0], vn[:0])
            kept.append((np.concatenate([a, kn[cu[s]:cu[s + 1]]]), np.concatenate([b, vn[cu[s]:cu[s + 1]]])))
        assert lengths.tolist() == [len(a) for a, _ in kept]
        q = torch.randn((rows, 4, D), device="cuda").half()
        out = hq.paged_attention(q, pool[0], pool[1], table, lengths)
        for s, (a, b) in enumerate(kept):
            for h in range(4):
                x = torch.from_numpy(a[:, h // 2]).double().cuda() @ q[s, h].double() / math.sqrt(D)
                want = torch.softmax(x, 0) @ torch.from_numpy(b[:, h // 2]).double().cuda()
                assert (out[s, h].double() - want).abs().max() <= 2.0 ** -9 * float(np.abs(b).max())
        parent, add = [int(p) for p in r.integers(0, rows, rows)], [1] * rows


def test_step_that_hands_out_thousands_of_pages(hq):
    """More than a workgroup lists in its own memory, with enough of them and without, in large and in small tables."""
    for rows, width, pages in ((400, 30, 14000), (400, 30, 9000), (500, 32, 4096), (1024, 16, 4000), (1025, 16, 4000)):
        page = 4
        r = np.random.default_rng(rows + pages)
        table, lengths, refs = random_tables(r, rows, width, page, pages, 1)
        parent = [-1 if r.random() < 0.7 else int(r.integers(0, rows)) for _ in range(rows)]
        add = [int(n) for n in r.integers(0, (width + 2) * page, rows)]
        check_step(hq, 1, page, table, lengths, refs, parent, add, planes=1, elems=8)


def test_pages_of_every_size(hq):
    """Page sizes that are no multiple of what a workgroup copies at a time."""
    for elems in (8, 2040, 2048, 16392, 70000):
        r = np.random.default_rng(elems)
        table, lengths, refs = random_tables(r, 16, 6, 16, 150, 2)
        check_step(hq, 2, 16, table, lengths, refs, [int(p) for p in r.integers(0, 16, 16)], [1] * 16, planes=3, elems=elems)


def test_what_one_step_leaves_the_next_one_finds(hq):
    """A step of large tables leaves its counts at zero for the next, whatever that one's size; other operators in between."""
    r = np.random.default_rng(9)
    big = random_tables(r, 300, 40, 4, 9000, 10)
    small = random_tables(r, 8, 500, 16, 5000, 2)
    for i in range(4):
        for (table, lengths, refs), page in ((big, 4), (small, 16)):
            n = len(table)
            check_step(hq, i, page, table, lengths, refs, [int(p) for p in r.integers(-1, n, n)], [3] * n, planes=1, elems=8)
        x = torch.randn(4096, device="cuda")
        assert hq.q3_matvec(x, torch.zeros((384, 256), dtype=torch.int32, device="cuda"), torch.ones(256, device="cuda"),
                            torch.zeros(256, device="cuda")).abs().max() == 0


def test_large_tables_on_another_stream_and_in_a_graph(hq):
    """The ways of more than one launch, which keep counters between calls."""
    r = np.random.default_rng(8)
    rows, pages = 1100, 7000
    table, lengths, refs = random_tables(r, rows, 4, 16, pages, 2)
    args = [i32(table), i32(lengths), i32(refs), i32(r.integers(-1, rows, rows)), i32([1] * rows)]
    s = torch.cuda.Stream()
    for call in (lambda p: hq.cache_step(p, 16, *args), lambda p: hq.cache_compact(p, args[0], args[2])):
        pool = pool_of(4, 1, pages, 16)
        wpool = pool.clone()
        want = call(wpool)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            mine = pool.clone()
            got = call(mine)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(mine, wpool)
        graph = torch.cuda.CUDAGraph()
        static = pool.clone()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            got = call(static)
        for i in range(3):
            args[3].copy_(i32(np.random.default_rng(i).integers(-1, rows, rows)))
            fresh = pool_of(5 + i, 1, pages, 16)
            static.copy_(fresh)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = call(fresh)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(static, fresh)


@pytest.mark.parametrize("planes,pages,elems", [(4, 1024, 131072), (3, 700, 300008), (64, 4096, 2048)])
def test_compact_of_large_pools(hq, planes, pages, elems):
    """Pools of a gibibyte and more take the way of a plan and then copies; pages of no whole pieces of a workgroup, and many that move."""
    r = np.random.default_rng(pages)
    refs = [int(n) for n in (r.random(pages) < 0.6) * r.integers(1, 4, pages)]
    pool = pool_of(1, planes, pages, elems)
    live = sum(n > 0 for n in refs)
    holes, movers = [p for p in range(live) if refs[p] <= 0], [p for p in range(live, pages) if refs[p] > 0]
    to, want_refs, want_pool = dict(zip(movers, holes)), refs[:], pool.clone()
    for source, target in to.items():
        want_refs[target], want_refs[source] = refs[source], 0
    want_pool[:, holes[:len(movers)]] = pool[:, movers]
    table = r.integers(-2, pages + 2, (5, 11)).tolist()
    t, n, got = hq.cache_compact(pool, i32(table), i32(refs))
    assert t.tolist() == [[to.get(p, p) for p in row] for row in table]
    assert n.tolist() == want_refs and got.tolist() == [live]
    assert torch.equal(pool, want_pool)
