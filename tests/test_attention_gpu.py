"""Attention over packed prompts and over a paged cache against its formula in 64 bits.

Bound of every element, derived before the first run: the result is rounded once (unit roundoff u of its type: 2^-8 bf16, 2^-11
fp16), and so is every weight on its way into the product with the values, which moves a result by at most u * A,
A = sum_j p_j |v_j|.  Scores are fp32 sums of at most 128 products: of magnitude S, the largest sum of |q_d k_d| times scale, they
are off by less than 130 * 2^-24 * S, and the weights by as much relatively, twice (numerator and sum); the rest is fp32 sums,
below 2^-13 in all for the lengths here.  |got - exact| <= u |exact| + (u + 2^-13 + 2^-15 S) A, times 1.02 for what is of second order."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11)}


def attend(q, k, v, seen, scale):
    """Result, A and S of one head: q [n][D], k, v [m][D] in 64 bits, seen [n][m]."""
    s = (q @ k.T) * scale
    big = float(((q.abs() @ k.abs().T) * scale).amax()) if s.numel() else 0.0
    s = torch.where(seen, s, -math.inf)
    top = s.amax(1, keepdim=True) if s.shape[1] else s.new_full((s.shape[0], 1), -math.inf)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    return p @ v, p @ v.abs(), big


def close(got, want, a, big, u):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    bound = 1.02 * (u * want.abs() + (u + 2.0 ** -13 + 2.0 ** -15 * big) * a) + 2.0 ** -24
    worst = (err - bound).max().item()
    assert worst <= 0, (worst, err.max().item())


def bounds(lengths):
    c = [0]
    for n in lengths:
        c.append(c[-1] + n)
    return c


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def check_prompt(out, q, k, v, nq, nk, causal, scale, u):
    r, cq, ck = q.shape[1] // k.shape[1], bounds(nq), bounds(nk)
    for i in range(len(nq)):
        qs, ks = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        seen = torch.ones((nq[i], nk[i]), dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril(nk[i] - nq[i])
        if nq[i] == 0:
            continue
        for h in range(q.shape[1]):
            want, a, big = attend(q[qs, h].double(), k[ks, h // r].double(), v[ks, h // r].double(), seen, scale)
            close(out[qs, h], want, a, big, u)
            assert (out[qs, h][~seen.any(1)] == 0).all()


PROMPTS = [([1], [1]), ([5], None), ([32], None), ([33], None), ([64], None), ([127, 0, 1, 200], None), ([129], None), ([300, 65], None),
           ([3], [259]), ([40, 1, 0], [700, 64, 9]), ([70], [10]), ([5, 6], [0, 6]), ([1], [1025])]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (8, 2), (14, 2), (3, 1), (40, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt(hq, kind, D, heads, causal):
    dtype, u = TYPES[kind]
    for n, (nq, nk) in enumerate(PROMPTS):
        cu_k = nk
        nk = nk or nq
        q, k, v = (randn(n * 10 + i, sum(m), h, D).to(dtype) for i, (m, h) in enumerate(((nq, heads[0]), (nk, heads[1]), (nk, heads[1]))))
        out = hq.prompt_attention(q, k, v, i32(bounds(nq)), None if cu_k is None else i32(bounds(nk)), causal=causal)
        check_prompt(out, q, k, v, nq, nk, causal, 1 / math.sqrt(D), u)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_prompt_long_and_scales(hq, kind):
    dtype, u = TYPES[kind]
    for nq, nk, scale in (([1500], [1500], None), ([1000], [2100], 0.0), ([257], [800], 0.5), ([900], [900], 2.0)):
        q, k, v = randn(1, sum(nq), 4, 128).to(dtype), randn(2, sum(nk), 2, 128).to(dtype), randn(3, sum(nk), 2, 128).to(dtype)
        out = hq.prompt_attention(q, k, v, i32(bounds(nq)), i32(bounds(nk)), scale=scale)
        check_prompt(out, q, k, v, nq, nk, True, 1 / math.sqrt(128) if scale is None else scale, u)


@pytest.mark.parametrize("D", [64, 128])
def test_prompt_scores_that_rise_and_fall(hq, D):
    """The running maximum moves in every tile, by a lot and by a little, up and down."""
    dtype, u = TYPES["f16"]
    n = 700
    for step in (0.2, -0.2, 0.003):
        ramp = torch.arange(n, device="cuda", dtype=torch.float32)[:, None, None] * step
        q = torch.ones((n, 2, D), device="cuda").to(dtype)
        k = (ramp.expand(n, 2, D) / 4 + randn(5, n, 2, D) * 0.1).to(dtype)
        v = randn(6, n, 2, D).to(dtype)
        out = hq.prompt_attention(q, k, v, i32([0, n]), scale=0.25)
        check_prompt(out, q, k, v, [n], [n], True, 0.25, u)


def test_prompt_many_sequences(hq):
    dtype, u = TYPES["bf16"]
    nq = [(i * 7) % 6 for i in range(150)]
    nk = [n + (i * 5) % 4 for i, n in enumerate(nq)]
    q, k, v = randn(1, sum(nq), 6, 64).to(dtype), randn(2, sum(nk), 3, 64).to(dtype), randn(3, sum(nk), 3, 64).to(dtype)
    out = hq.prompt_attention(q, k, v, i32(bounds(nq)), i32(bounds(nk)))
    check_prompt(out, q, k, v, nq, nk, True, 0.125, u)


def test_prompt_parts_of_a_projection_and_given_result(hq):
    dtype, u = TYPES["bf16"]
    n, hq_, hk, D = 200, 8, 2, 128
    qkv = randn(1, n, hq_ + 2 * hk, D).to(dtype)
    q, k, v = qkv[:, :hq_], qkv[:, hq_:hq_ + hk], qkv[:, hq_ + hk:]
    out = torch.full((n, hq_, D), 7.0, dtype=dtype, device="cuda")
    assert hq.prompt_attention(q, k, v, i32([0, 90, 150]), out=out) is out
    check_prompt(out[:150], q[:150], k[:150], v[:150], [90, 60], [90, 60], True, 1 / math.sqrt(D), u)
    assert (out[150:] == 7.0).all()
    assert torch.equal(out[:150], hq.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), i32([0, 90, 150]))[:150])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf, "most"])
def test_prompt_what_is_not_seen_has_no_effect(hq, kind, D, what):
    """Later tokens and the neighbour's tokens hold NaN, infinities or the type's largest numbers: the tokens that do not see them
    give the same bits, those that see a value that is not finite give NaN."""
    dtype, _ = TYPES[kind]
    what = torch.finfo(dtype).max if what == "most" else what
    nq = [150, 131]
    q, k, v = randn(1, 281, 8, D).to(dtype), randn(2, 281, 2, D).to(dtype), randn(3, 281, 2, D).to(dtype)
    cu = i32(bounds(nq))
    want = hq.prompt_attention(q, k, v, cu)
    for at in (0, 3, 70, 149):
        k2, v2 = k.clone(), v.clone()
        k2[at], v2[at] = what, what
        k2[150:], v2[150:] = what, what
        got = hq.prompt_attention(q, k2, v2, cu)
        assert torch.equal(got[:at], want[:at])
        v3 = v.clone()
        v3[at, 1, 5] = what
        got = hq.prompt_attention(q, k, v3, cu)
        assert torch.equal(got[:at], want[:at]) and torch.equal(got[150:], want[150:])
        assert torch.equal(got[at:150, :, 6:], want[at:150, :, 6:]) and torch.equal(got[at:150, :4], want[at:150, :4])
        if not math.isfinite(what):
            assert not torch.isfinite(got[at:150, 4:, 5]).any()


def test_prompt_scores_of_minus_infinity(hq):
    """A key whose score is -inf has no weight; a token all of whose scores are is NaN, as its softmax is."""
    n, D = 80, 64
    q, k, v = torch.ones((n, 1, D), device="cuda").half(), randn(2, n, 1, D).half(), randn(3, n, 1, D).half()
    k[40] = -math.inf
    out = hq.prompt_attention(q, k, v, i32([0, n]), causal=False)
    keep = torch.arange(n, device="cuda") != 40
    want, a, big = attend(q[:, 0].double(), k[keep][:, 0].double(), v[keep][:, 0].double(), torch.ones((n, n - 1), dtype=torch.bool, device="cuda"), 0.125)
    close(out[:, 0], want, a, big, 2.0 ** -11)
    k[:] = -math.inf
    assert torch.isnan(hq.prompt_attention(q, k, v, i32([0, n]), causal=False)).all()


# ---- pages ---------------------------------------------------------------------------------------------------------------
def paged_case(seed, dtype, lengths, heads, D, page, groups=None, shared=None, spare=3):
    """Requests on random pages; what is behind a request's length in its pages, and every spare page, is NaN."""
    g = torch.Generator().manual_seed(seed)
    use = [-(-n // page) for n in lengths]
    width = max(use + [1])
    pages = sum(use) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = [[-1] * width for _ in lengths]
    for s, u in enumerate(use):
        for j in range(u):
            table[s][j] = order.pop()
    if groups:
        for i in range(len(groups) - 1):
            for s in range(groups[i], groups[i + 1]):
                for j in range(-(-shared[i] // page)):
                    if j < use[s]:
                        table[s][j] = table[groups[i]][j] if j < use[groups[i]] else table[s][j]
    k, v = torch.full((pages, heads[1], page, D), math.nan, dtype=dtype, device="cuda"), torch.full((pages, heads[1], page, D), math.nan, dtype=dtype, device="cuda")
    for s, n in enumerate(lengths):
        for j in range(use[s]):
            m = min(page, n - j * page)
            part = randn(seed + 131 * table[s][j] + 7, 2, heads[1], page, D).to(dtype)
            k[table[s][j], :, :m], v[table[s][j], :, :m] = part[0, :, :m], part[1, :, :m]
    q = randn(seed + 1, len(lengths), heads[0], D).to(dtype)
    return q, k, v, table, lengths


def check_paged(out, q, k, v, table, lengths, scale, u):
    r, page = q.shape[1] // k.shape[1], k.shape[2]
    for s, n in enumerate(lengths):
        if n == 0:
            assert (out[s] == 0).all()
            continue
        pages = torch.tensor(table[s][:-(-n // page)], device="cuda")
        ks = k[pages].transpose(1, 2).reshape(-1, k.shape[1], k.shape[3])[:n]
        vs = v[pages].transpose(1, 2).reshape(-1, k.shape[1], k.shape[3])[:n]
        for h in range(k.shape[1]):
            want, a, big = attend(q[s, h * r:(h + 1) * r].double(), ks[:, h].double(), vs[:, h].double(),
                                  torch.ones((r, n), dtype=torch.bool, device="cuda"), scale)
            close(out[s, h * r:(h + 1) * r], want, a, big, u)


LENGTHS = [[1], [0], [15, 16, 17, 0, 300], [129, 4], [700], [1]]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (8, 2), (14, 2), (40, 1)])
def test_paged(hq, kind, D, heads):
    dtype, u = TYPES[kind]
    for n, lengths in enumerate(LENGTHS):
        for page in (8, 16, 128, 1024):
            q, k, v, table, lengths = paged_case(n, dtype, lengths, heads, D, page)
            out = hq.paged_attention(q, k, v, i32(table), i32(lengths))
            check_paged(out, q, k, v, table, lengths, 1 / math.sqrt(D), u)


GROUPS = [  # lengths, bounds, shared
    ([40, 50, 33], [0, 3], [32]),
    ([40, 50, 33], [0, 3], [0]),
    ([40, 50, 20, 0], [0, 4], [35]),                   # shared beyond some requests, and no whole pages of it
    ([40, 50, 33, 70, 80], [0, 2, 5], [16, 64]),
    ([40, 50, 33, 70, 80], [1, 2, 2, 4], [16, 7, 64]),  # requests without a group, a group of one and one of none
    ([600 + i for i in range(45)], [0, 45], [592]),     # more rows than a workgroup has
    ([1500, 1600], [0, 2], [1488]),
    ([100, 101, 102], [0, 1, 2, 3], [96, 0, 1000]),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads,D", [((2, 2), 64), ((8, 2), 128), ((14, 2), 64), ((40, 1), 128)])
def test_paged_shared(hq, kind, heads, D):
    dtype, u = TYPES[kind]
    for n, (lengths, groups, shared) in enumerate(GROUPS):
        q, k, v, table, lengths = paged_case(n, dtype, lengths, heads, D, 16, groups, shared)
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths), i32(groups), i32(shared))
        check_paged(out, q, k, v, table, lengths, 1 / math.sqrt(D), u)
        assert torch.equal(out, hq.paged_attention(q, k, v, i32(table), i32(lengths), i32(groups), i32(shared)))


def test_paged_tables_with_numbers_that_are_no_pages(hq):
    """A needed entry that is no page counts as a page of zeros; lengths beyond the table end with it."""
    dtype, u = TYPES["f16"]
    q, k, v, table, _ = paged_case(3, dtype, [64, 64, 64], (4, 2), 64, 16)
    bad = [row[:] for row in table]
    bad[0][1], bad[1][3], bad[2][0] = -1, 10 ** 6, -2 ** 31
    out = hq.paged_attention(q, k, v, i32(bad), i32([64, 64, 10 ** 9]))
    k0, v0 = torch.cat([k, torch.zeros_like(k[:1])]), torch.cat([v, torch.zeros_like(v[:1])])
    bad[0][1] = bad[1][3] = bad[2][0] = len(k)
    check_paged(out, q, k0, v0, bad, [64, 64, 64], 0.125, u)


def test_other_stream_and_graph(hq):
    dtype, u = TYPES["bf16"]
    q, k, v, table, lengths = paged_case(5, dtype, [900, 950, 20], (8, 2), 128, 16, [0, 2], [896])
    args = (q, k, v, i32(table), i32(lengths), i32([0, 2]), i32([896]))
    pq, pk, pv = randn(1, 300, 8, 128).to(dtype), randn(2, 300, 2, 128).to(dtype), randn(3, 300, 2, 128).to(dtype)
    cu = i32([0, 100, 300])
    want, pwant = hq.paged_attention(*args), hq.prompt_attention(pq, pk, pv, cu)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, pgot = hq.paged_attention(*args), hq.prompt_attention(pq, pk, pv, cu)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(pgot, pwant)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got, pgot = hq.paged_attention(*args), hq.prompt_attention(pq, pk, pv, cu)
    for i in range(4):
        got.zero_()
        pgot.zero_()
        q.copy_(randn(50 + i, *q.shape))
        pq.copy_(randn(60 + i, *pq.shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, hq.paged_attention(*args)) and torch.equal(pgot, hq.prompt_attention(pq, pk, pv, cu))


# ---- the ways through the kernels that the sizes above do not take ---------------------------------------------------------------
def test_prompt_divided_keys_leave_what_is_no_ones(hq):
    """Few rows and many keys: the shares' sums, rows that see nothing, and tokens of no sequence."""
    dtype, u = TYPES["bf16"]
    for heads in ((8, 2), (3, 1)):
        nq, nk = [40, 0, 3, 70], [2500, 100, 1, 60]  # the last one's first tokens see nothing
        q, k, v = randn(1, 120, heads[0], 128).to(dtype), randn(2, sum(nk), heads[1], 128).to(dtype), randn(3, sum(nk), heads[1], 128).to(dtype)
        out = torch.full((120, heads[0], 128), 7.0, dtype=dtype, device="cuda")
        hq.prompt_attention(q, k, v, i32(bounds(nq)), i32(bounds(nk)), out=out)
        check_prompt(out[:113], q[:113], k, v, nq, nk, True, 1 / math.sqrt(128), u)
        assert (out[113:] == 7.0).all()
        k2, v2 = k.clone(), v.clone()
        k2[2480:2500], v2[2480:2500] = math.nan, math.inf  # seen by the last 20 of the 40
        got = hq.prompt_attention(q, k2, v2, i32(bounds(nq)), i32(bounds(nk)))
        assert torch.equal(got[:20], out[:20]) and torch.equal(got[40:113], out[40:113]) and not torch.isfinite(got[21:40]).any()


def test_prompt_rows_far_apart(hq):
    """Offsets beyond 32 bits: tokens 2 MB apart."""
    dtype, u = TYPES["f16"]
    n, D = 2300, 64
    flat = torch.zeros(n << 20, dtype=dtype, device="cuda")
    k = flat.as_strided((n, 1, D), (1 << 20, D, 1))
    v = flat.as_strided((n, 1, D), (1 << 20, D, 1), storage_offset=D)
    k.copy_(randn(2, n, 1, D))
    v.copy_(randn(3, n, 1, D))
    q = randn(1, 5, 2, D).to(dtype)
    out = hq.prompt_attention(q, k, v, i32([0, 5]), i32([0, n]))
    check_prompt(out, q, k, v, [5], [n], True, 0.125, u)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64)])
def test_paged_long_rows_in_one_share(hq, kind, D):
    """So many requests that nobody's keys are divided: a wave's blocks take several sets of page numbers."""
    dtype, u = TYPES[kind]
    lengths = [3333 if i == 3 else 2050 if i == 7 else (i * 37) % 70 for i in range(280)]
    q, k, v, table, lengths = paged_case(1, dtype, lengths, (2, 2), D, 16)
    check_paged(hq.paged_attention(q, k, v, i32(table), i32(lengths)), q, k, v, table, lengths, 1 / math.sqrt(D), u)


@pytest.mark.parametrize("D", [64, 128])
def test_paged_missing_pages_anywhere(hq, D):
    """Entries that are no pages in whole blocks, next to the end, in what is shared and in what is not."""
    dtype, u = TYPES["f16"]
    lengths, groups, shared = [1000, 1003, 990, 700, 20], [0, 3, 5], [640, 16]
    for heads in ((4, 2), (24, 1)):
        q, k, v, table, _ = paged_case(4, dtype, lengths, heads, D, 16, groups, shared)
        zero = len(k)
        k0, v0 = torch.cat([k, torch.zeros_like(k[:1])]), torch.cat([v, torch.zeros_like(v[:1])])
        bad = [row[:] for row in table]
        for s, places in ((0, (41, 50, 51, 61, 62)), (1, (40, 62)), (2, (61,)), (3, (1, 2, 3, 4, 20, 43)), (4, (1,))):
            for j in places:
                bad[s][j] = (-1, zero, 2 ** 31 - 1)[j % 3]
        for row in bad[:3]:
            row[5] = row[39] = -1
        want = [[zero if not 0 <= p < zero else p for p in row] for row in bad]
        out = hq.paged_attention(q, k, v, i32(bad), i32(lengths), i32(groups), i32(shared))
        check_paged(out, q, k0, v0, want, lengths, 1 / math.sqrt(D), u)


def test_paged_many_groups(hq):
    """More groups than a wave has lanes, some of them empty, and requests behind the last."""
    dtype, u = TYPES["bf16"]
    groups, lengths = [0], []
    for g in range(75):
        n = (g * 5) % 3
        lengths += [48 + (g * 11 + i * 7) % 90 for i in range(n)]
        groups.append(len(lengths))
    lengths += [30, 5]
    shared = [(g * 16) % 64 for g in range(75)]
    for heads in ((4, 1), (32, 1)):
        q, k, v, table, _ = paged_case(8, dtype, lengths, heads, 64, 16, groups, shared)
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths), i32(groups), i32(shared))
        check_paged(out, q, k, v, table, lengths, 0.125, u)


def test_paged_beyond_32_bits(hq):
    """A cache of more than 4 GB: the last pages, written and read."""
    dtype, u = TYPES["bf16"]
    pages, heads, page, D = 2200, 8, 1024, 128
    k = torch.zeros((pages, heads, page, D), dtype=dtype, device="cuda")
    v = torch.zeros_like(k)
    n = 1500
    table = [[2199, 2100], [3, 2150]]
    kn, vn = randn(1, 2 * n, heads, D).to(dtype), randn(2, 2 * n, heads, D).to(dtype)
    hq.cache_write(kn, vn, k, v, i32(table), i32([0, 0]), i32([0, n, 2 * n]))
    assert torch.equal(k[2100, :, :n - page], kn[page:n].transpose(0, 1)) and torch.equal(v[2150, :, :n - page], vn[n + page:].transpose(0, 1))
    q = randn(3, 2, 16, D).to(dtype)
    out = hq.paged_attention(q, k, v, i32(table), i32([n, n]))
    check_paged(out, q, k, v, table, [n, n], 1 / math.sqrt(D), u)
    out = hq.paged_attention(q[:1].expand(2, 16, D).contiguous(), k, v, i32([table[1], table[1]]), i32([n, n]), i32([0, 2]), i32([page]))
    check_paged(out, q[:1].expand(2, 16, D), k, v, [table[1], table[1]], [n, n], 1 / math.sqrt(D), u)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (10, 2), (16, 1), (17, 1)])
def test_paged_shares_joined_here_and_in_a_second_launch(hq, kind, D, heads):
    """1 to 64 shares a row, full and without a key, each call twice and on counters that the call before left."""
    dtype, u = TYPES[kind]
    for n, lengths in enumerate([[300], [1500, 2], [4000], [4100, 0, 129], [9000], [130] * 40, [513] * 9]):
        q, k, v, table, lengths = paged_case(20 + n, dtype, lengths, heads, D, 16)
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths))
        check_paged(out, q, k, v, table, lengths, 1 / math.sqrt(D), u)
        assert torch.equal(out, hq.paged_attention(q, k, v, i32(table), i32(lengths)))


def test_paged_shares_joined_in_a_graph(hq):
    dtype, u = TYPES["bf16"]
    q, k, v, table, lengths = paged_case(5, dtype, [2900, 950, 20], (8, 2), 128, 16)
    args = (q, k, v, i32(table), i32(lengths))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        hq.paged_attention(*args)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = hq.paged_attention(*args)
        again = hq.paged_attention(*args)
    for i in range(4):
        got.zero_()
        again.zero_()
        q.copy_(randn(50 + i, *q.shape))
        args[4].copy_(i32([2900 - 700 * i, 950 * (i % 2), 20 + i]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = hq.paged_attention(*args)  # NaN where a request is longer than its tokens
        for x in (got, again):
            torch.testing.assert_close(x, want, rtol=0, atol=0, equal_nan=True)


def test_paged_as_many_groups_as_requests(hq):
    """Some of them empty, the keys of another common."""
    dtype, u = TYPES["bf16"]
    groups, shared = [0, 3, 3, 3], [992, 16, 5]
    q, k, v, table, lengths = paged_case(31, dtype, [1000, 1100, 999], (8, 2), 128, 16, groups, shared)
    out = hq.paged_attention(q, k, v, i32(table), i32(lengths), i32(groups), i32(shared))
    check_paged(out, q, k, v, table, lengths, 1 / math.sqrt(128), u)


def test_paged_infinite_scores_in_one_share(hq):
    """One key of an infinite score among 1000: the row is NaN, whichever share holds it, and the other rows are not touched."""
    dtype, u = TYPES["bf16"]
    for at in (0, 200, 999):
        q, k, v, table, lengths = paged_case(41, dtype, [1000, 1000], (8, 2), 128, 16)
        k[table[0][at // 16], 1, at % 16] = math.inf
        q[0, 4:].abs_()
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths))
        assert torch.isnan(out[0, 4:]).all() and torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("heads,groups", [((64, 8), [0, 16, 32, 48, 64]), ((32, 8), [0, 16, 32, 48, 64]), ((64, 8), [0, 3, 3, 60]), ((32, 8), [0, 64])])
def test_paged_many_rows_joined(hq, heads, groups):
    """2048 and 4096 rows: groups alike, of very different sizes, one of all."""
    dtype, u = TYPES["bf16"]
    shared = [480, 16, 992, 320][:len(groups) - 1]
    lengths = [(s * 37) % 400 + 500 for s in range(64)]
    lengths[5], lengths[63] = 0, 1500
    q, k, v, table, lengths = paged_case(51, dtype, lengths, heads, 128, 16, groups, shared)
    out = hq.paged_attention(q, k, v, i32(table), i32(lengths), i32(groups), i32(shared))
    check_paged(out, q, k, v, table, lengths, 1 / math.sqrt(128), u)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("queries,keys,heads", [([100], [6100], (32, 8)), ([3, 0, 40], [2000, 900, 2500], (8, 8)), ([600], [600], (2, 2)), ([1], [9000], (4, 4))])
def test_prompt_divided_keys_joined(hq, kind, D, queries, keys, heads):
    """Few rows and many, few shares and many, sequences of different lengths whose keys are divided alike."""
    dtype, u = TYPES[kind]
    q, k, v = randn(1, sum(queries), heads[0], D).to(dtype), randn(2, sum(keys), heads[1], D).to(dtype), randn(3, sum(keys), heads[1], D).to(dtype)
    out = hq.prompt_attention(q, k, v, i32(bounds(queries)), i32(bounds(keys)))
    check_prompt(out, q, k, v, queries, keys, True, 1 / math.sqrt(D), u)
