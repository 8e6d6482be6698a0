"""Attention where its results are decided by something else than a sum: no keys, numbers that are not finite in one of several
shares of the keys, weights far below the largest, no room for shares while a stream is being captured."""
import math

import pytest
import torch

from tests.test_attention_gpu import TYPES, attend, bounds, check_paged, check_prompt, close, i32, paged_case, randn

pytestmark = pytest.mark.gpu


# ---- no keys, no pages -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,D", [((8, 2), 128), ((24, 1), 64)])
def test_paged_tables_of_no_width(hq, heads, D):
    """Lengths end with the table: nothing is seen, with and without groups, and the results are zeros."""
    q = randn(1, 5, heads[0], D).bfloat16()
    pages = randn(2, 3, heads[1], 16, D).bfloat16()
    table, lengths = torch.zeros((5, 0), dtype=torch.int32, device="cuda"), i32([7, 100, 0, 1, 2 ** 31 - 1])
    for groups in ((), (i32([0, 5]), i32([64])), (i32([0, 2, 4]), i32([0, 16]))):
        out = torch.full_like(q, 7.0)
        hq.paged_attention(q, pages, pages, table, lengths, *groups, out=out)
        assert (out == 0).all()


def alike(seed, n, heads, dtype, D):
    """A request's keys, of which the first has a score of 200 and all others less than 1 in magnitude: 2^-287 of its weight."""
    k = randn(seed, n, heads, D) * 0.01
    k[0], k[:, :, 0] = 0, 0
    k[0, :, 0] = 100
    q0 = 2.0 * math.sqrt(D)
    return k.to(dtype), q0


# ---- numbers that are not finite, in one share -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads,D", [((8, 2), 128), ((1, 1), 64), ((24, 1), 64)])
@pytest.mark.parametrize("page", [8, 16])
def test_paged_nan_keys_alone_in_the_last_share(hq, kind, heads, D, page):
    """The last share holds nothing but keys of NaN: joined in one launch, in two, and without being divided the request is NaN."""
    dtype, u = TYPES[kind]
    for lengths, bad in (([129], 1), ([257], 1), ([9000], 40), ([129, 300], 1), ([129] + [200] * 300, 1)):
        q, k, v, table, lengths = paged_case(7, dtype, lengths, heads, D, page)
        for t in range(lengths[0] - bad, lengths[0]):
            k[table[0][t // page], :, t % page] = math.nan
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths))
        assert torch.isnan(out[0]).all()
        check_paged(out[1:], q[1:], k, v, table[1:], lengths[1:], 1 / math.sqrt(D), u)


@pytest.mark.parametrize("heads,D", [((8, 2), 128), ((24, 1), 64)])
def test_paged_nan_keys_behind_what_is_common(hq, heads, D):
    """One request's own key is NaN: it is, and the others of its group are not."""
    dtype, u = TYPES["bf16"]
    q, k, v, table, lengths = paged_case(9, dtype, [513, 600, 520], heads, D, 16, [0, 3], [512])
    k[table[0][32], :, 0] = math.nan
    out = hq.paged_attention(q, k, v, i32(table), i32(lengths), i32([0, 3]), i32([512]))
    assert torch.isnan(out[0]).all()
    check_paged(out[1:], q[1:], k, v, table[1:], lengths[1:], 1 / math.sqrt(D), u)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_nan_keys_fill_shares(hq, kind, D):
    dtype, u = TYPES[kind]
    nq, nk = [3, 5], [2500, 900]
    q, k, v = randn(1, 8, 8, D).to(dtype), randn(2, 3400, 2, D).to(dtype), randn(3, 3400, 2, D).to(dtype)
    k[1700:2490, 1] = math.nan
    out = hq.prompt_attention(q, k, v, i32(bounds(nq)), i32(bounds(nk)))
    assert torch.isnan(out[:3, 4:]).all()
    check_prompt(out[:3, :4], q[:3, :4], k[:2500, :1], v[:2500, :1], [3], [2500], True, 1 / math.sqrt(D), u)
    check_prompt(out[3:], q[3:], k[2500:], v[2500:], [5], [900], True, 1 / math.sqrt(D), u)


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,D", [((8, 2), 128), ((1, 1), 64), ((24, 1), 64)])
def test_paged_values_without_weight(hq, what, heads, D):
    """A value that is not finite makes its element NaN, however small its weight and whichever share holds it, and no other."""
    for kind in ("bf16", "f16"):
        dtype, u = TYPES[kind]
        for lengths, groups in (([100], None), ([129], None), ([257], None), ([9000], None), ([129] + [200] * 300, None), ([700, 600], ([0, 2], [512]))):
            q, k, v, table, lengths = paged_case(11, dtype, lengths, heads, D, 16, *(groups or ()))
            rows, q0 = alike(3, lengths[0], heads[1], dtype, D)
            q[0, :, 0] = q0
            for t in range(lengths[0]):
                k[table[0][t // 16], :, t % 16] = rows[t]
            args = (i32(table), i32(lengths)) + (tuple(i32(g) for g in groups) if groups else ())
            want = hq.paged_attention(q, k, v, *args)
            check_paged(want[:1], q[:1], k, v, table[:1], lengths[:1], 1 / math.sqrt(D), u)
            v[table[0][(lengths[0] - 1) // 16], 0, (lengths[0] - 1) % 16, 5] = what
            got = hq.paged_attention(q, k, v, *args)
            r = heads[0] // heads[1]
            assert torch.isnan(got[0, :r, 5]).all()
            got[0, :r, 5] = want[0, :r, 5]
            assert torch.equal(got, want)


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_values_without_weight(hq, what, D):
    for kind in ("bf16", "f16"):
        dtype, u = TYPES[kind]
        for nq, nk in ((3, 2500), (40, 2900), (500, 500)):
            q, v = randn(1, nq, 8, D).to(dtype), randn(3, nk, 2, D).to(dtype)
            k, q0 = alike(2, nk, 2, dtype, D)
            q[:, :, 0] = q0
            cu = i32([0, nq]), i32([0, nk])
            want = hq.prompt_attention(q, k, v, *cu)
            check_prompt(want, q, k, v, [nq], [nk], True, 1 / math.sqrt(D), u)
            v[nk - 2, 1, 5] = what  # seen by the last two tokens
            got = hq.prompt_attention(q, k, v, *cu)
            assert torch.isnan(got[-2:, 4:, 5]).all()
            got[-2:, 4:, 5] = want[-2:, 4:, 5]
            assert torch.equal(got, want)


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_not_finite_are_nan_in_every_tile(hq, what, D):
    """Tiles that all rows see and tiles that some see, keys divided and not, a prompt's and a cache's: one answer."""
    for kind in ("bf16", "f16"):
        dtype, _ = TYPES[kind]
        for nq, nk, heads in ((300, 300, (8, 2)), (5, 2000, (8, 2)), (1000, 1000, (32, 32))):
            q, k, v = randn(1, nq, heads[0], D).to(dtype), randn(2, nk, heads[1], D).to(dtype), randn(3, nk, heads[1], D).to(dtype)
            want = hq.prompt_attention(q, k, v, i32([0, nq]), i32([0, nk]))
            for at in (3, nk - 200, nk - 1):
                v2 = v.clone()
                v2[at, 1, 5] = what
                got = hq.prompt_attention(q, k, v2, i32([0, nq]), i32([0, nk]))
                r, first = heads[0] // heads[1], max(at - (nk - nq), 0)
                assert torch.isnan(got[first:, r:2 * r, 5]).all()
                got[first:, r:2 * r, 5] = want[first:, r:2 * r, 5]
                assert torch.equal(got, want)
        for heads in ((8, 2), (48, 2)):
            for lengths, groups in (([60], None), ([2000, 100], None), ([900] * 20, ([0, 20], [512])), ([600, 560], ([0, 2], [512]))):
                q, k, v, table, lengths = paged_case(13, dtype, lengths, heads, D, 16, *(groups or ()))
                args = (i32(table), i32(lengths)) + (tuple(i32(g) for g in groups) if groups else ())
                want = hq.paged_attention(q, k, v, *args)
                v[table[0][1], 1, 3, 5] = what
                got = hq.paged_attention(q, k, v, *args)
                r, who = heads[0] // heads[1], slice(None) if groups else slice(0, 1)
                assert torch.isnan(got[who, r:, 5]).all()
                got[who, r:, 5] = want[who, r:, 5]
                assert torch.equal(got, want)


def test_keys_of_minus_infinity_in_one_share_and_in_all(hq):
    """Keys whose score is -inf have no weight, also where a share holds nothing else; where all have it the softmax is NaN."""
    dtype, u = TYPES["bf16"]
    D = 64
    q, k, v = torch.ones((4, 4, D), device="cuda").to(dtype), randn(2, 2500, 2, D).to(dtype), randn(3, 2500, 2, D).to(dtype)
    k[1500:2400, 1] = -math.inf
    out = hq.prompt_attention(q, k, v, i32([0, 4]), i32([0, 2500]), causal=False)
    keep = torch.cat([torch.arange(1500), torch.arange(2400, 2500)]).cuda()
    for h in (2, 3):
        want, a, big = attend(q[:, h].double(), k[keep, 1].double(), v[keep, 1].double(), torch.ones((4, 1600), dtype=torch.bool, device="cuda"), 0.125)
        close(out[:, h], want, a, big, u)
    k[:, 0] = -math.inf
    out = hq.prompt_attention(q, k, v, i32([0, 4]), i32([0, 2500]), causal=False)
    assert torch.isnan(out[:, :2]).all() and torch.isfinite(out[:, 2:]).all()
    for n, heads in ((129, (4, 2)), (700, (4, 2)), (9000, (4, 2)), (700, (40, 2))):
        q, k, v, table, lengths = paged_case(3, dtype, [n, n], heads, D, 16)
        q[:] = 1
        for t in range(n):
            k[table[0][t // 16], 1, t % 16] = -math.inf
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths))
        r = heads[0] // 2
        assert torch.isnan(out[0, r:]).all() and torch.isfinite(out[0, :r]).all() and torch.isfinite(out[1]).all()


# ---- weights far below the largest -----------------------------------------------------------------------------------------
GAPS = [12.3, 18.5, 24.4, 26.2]


def sink(gap, n, heads, dtype, D):
    """n keys, of which the first has a score `gap` octaves above the others' and a value of zero; the others' values are about 1.  q0: of
    the query's first element, with the usual scale."""
    k = torch.zeros((n, heads, D), device="cuda")
    k[0, :, 0] = gap * math.log(2) / 4
    v = 1 + 0.01 * randn(5, n, heads, D)
    v[0] = 0
    return k.to(dtype), v.to(dtype), 4 * math.sqrt(D)


def close_to_sink(out, q, k, v, kind):
    """The bound of every element, as for all results, and the rounding of weights that are below fp16's normal numbers: fp16 weights are
    scaled so that the row's largest is 2^11 at least, and of those below 2^-14 each is off by 2^-25 at most, so that a sum is by 2^-36 of
    the sum of |v| at most (the largest weight, and so the sum of the weights, taken as 1)."""
    u = TYPES[kind][1]
    s = (q @ k.T) / math.sqrt(q.shape[1])
    p = torch.softmax(s, 1)
    big = float(((q.abs() @ k.abs().T) / math.sqrt(q.shape[1])).amax())
    want, a = p @ v, p @ v.abs()
    err = (out.double() - want).abs()
    bound = 1.02 * (u * want.abs() + (u + 2.0 ** -13 + 2.0 ** -15 * big) * a) + 2.0 ** -24
    if kind == "f16":
        bound = bound + 2.0 ** -36 * v.abs().sum(0)
    worst = (err - bound).max().item()
    assert worst <= 0, (worst, err.max().item(), want.abs().max().item())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("gap", GAPS)
def test_prompt_small_weights(hq, kind, D, gap):
    dtype = TYPES[kind][0]
    for nq, nk, heads in ((300, 1000, (16, 2)), (2, 100, (2, 2)), (3, 2000, (2, 2))):
        k, v, q0 = sink(gap, nk, heads[1], dtype, D)
        q = torch.zeros((nq, heads[0], D), dtype=dtype, device="cuda")
        q[:, :, 0] = q0
        out = hq.prompt_attention(q, k, v, i32([0, nq]), i32([0, nk]), causal=False)
        for h in (0, heads[0] - 1):
            at = h // (heads[0] // heads[1])
            close_to_sink(out[:, h], q[:, h].double(), k[:, at].double(), v[:, at].double(), kind)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,D", [((8, 2), 128), ((4, 4), 64), ((24, 1), 128), ((40, 2), 64)])
@pytest.mark.parametrize("gap", GAPS)
def test_paged_small_weights(hq, kind, heads, D, gap):
    dtype = TYPES[kind][0]
    for lengths in ([100, 40], [1001, 128], [1001] + [20] * 300):
        q, k, v, table, lengths = paged_case(17, dtype, lengths, heads, D, 16)
        ks, vs, q0 = sink(gap, lengths[0], heads[1], dtype, D)
        q[0] = 0
        q[0, :, 0] = q0
        for t in range(lengths[0]):
            k[table[0][t // 16], :, t % 16], v[table[0][t // 16], :, t % 16] = ks[t], vs[t]
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths))
        for h in range(heads[0]):
            at = h // (heads[0] // heads[1])
            close_to_sink(out[0, h:h + 1], q[0, h:h + 1].double(), ks[:, at].double(), vs[:, at].double(), kind)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_every_magnitude(hq, kind, D):
    """Scores up to 2^40, where fp32 numbers are far further apart than an octave: results stay among the values."""
    dtype, u = TYPES[kind]
    q, k, v = randn(1, 300, 8, D).to(dtype), randn(2, 700, 2, D).to(dtype), randn(3, 700, 2, D).to(dtype)
    pq, pk, pv, table, lengths = paged_case(23, dtype, [700, 100], (8, 2), D, 16)
    for octaves in range(16, 40):
        out = hq.prompt_attention(q, k, v, i32([0, 300]), i32([0, 700]), scale=2.0 ** octaves)
        assert torch.isfinite(out).all() and out.abs().max() <= v.abs().max() * (1 + 2 * u)
        out = hq.paged_attention(pq, pk, pv, i32(table), i32(lengths), scale=2.0 ** octaves)
        assert torch.isfinite(out).all() and out.abs().max() <= torch.nan_to_num(pv).abs().max() * (1 + 2 * u)


def test_scale_of_zero_and_scores_beyond_all_bounds(hq):
    """A scale of zero makes all keys alike, whatever their products with the query."""
    dtype, u = TYPES["bf16"]
    q, k, v = (randn(1, 4, 4, 64) * 2.0 ** 50).to(dtype), (randn(2, 200, 2, 64) * 2.0 ** 50).to(dtype), randn(3, 200, 2, 64).to(dtype)
    out = hq.prompt_attention(q, k, v, i32([0, 4]), i32([0, 200]), causal=False, scale=0.0)
    for h in range(4):
        close(out[:, h], v[:, h // 2].double().mean(0).expand(4, 64), v[:, h // 2].double().abs().mean(0), 0.0, u)


def test_paged_pools_of_no_pages(hq):
    """Every entry that is needed counts as a page of zeros."""
    pages = torch.zeros((0, 2, 16, 128), dtype=torch.float16, device="cuda")
    q = randn(1, 3, 8, 128).half()
    table = i32([[0, 1, 2], [-1, -1, -1], [5, 0, 0]])
    for groups in ((), (i32([0, 3]), i32([16]))):
        out = torch.full_like(q, 7.0)
        hq.paged_attention(q, pages, pages, table, i32([40, 1, 0]), *groups, out=out)
        assert (out == 0).all()


def test_paged_bounds_of_groups_that_do_not_ascend(hq):
    """Whatever they are, the call ends, and requests in no group are what they are without groups."""
    dtype, u = TYPES["bf16"]
    q, k, v, table, lengths = paged_case(70, dtype, [300 + 7 * i for i in range(90)], (8, 2), 128, 16)
    for groups in ([0, 80, 3, 80, -5, 70], [80, 0, 10 ** 9, 5, -2 ** 31, 60], [40, 40, 39, 38, 37, 36]):
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths), i32(groups), i32([64, 0, 16, 2 ** 31 - 1, -1]))
        inside = [any(max(min(a, 90), 0) <= s < max(min(b, 90), min(a, 90), 0) for a, b in zip(groups, groups[1:])) for s in range(90)]
        free = [s for s in range(90) if not inside[s]]
        check_paged(out[free], q[free], k, v, [table[s] for s in free], [lengths[s] for s in free], 1 / math.sqrt(128), u)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("heads", [(12, 1), (1, 1), (16, 2), (3, 1), (24, 1)])
def test_paged_one_long_request_among_short_ones(hq, kind, D, heads):
    """Hundreds of shares of one request where the others have one: joined in several steps, on counters that the call before left."""
    dtype, u = TYPES[kind]
    for n, lengths in enumerate(([20000] + [1] * 16, [0, 3, 30000] + [130] * 17, [100, 4300, 0, 5000] + [7] * 8, [40000] + [50] * 40)):
        q, k, v, table, lengths = paged_case(60 + n, dtype, lengths, heads, D, 16)
        args = (q, k, v, i32(table), i32(lengths))
        out = hq.paged_attention(*args)
        check_paged(out, q, k, v, table, lengths, 1 / math.sqrt(D), u)
        assert torch.equal(out, hq.paged_attention(*args))
        bad = 0 if lengths[0] > 1000 else 2 if n == 1 else 3
        k[table[bad][-3], :, 5] = math.nan
        again = hq.paged_attention(*args)
        assert torch.isnan(again[bad]).all()
        again[bad] = out[bad]
        assert torch.equal(again, out)


# ---- no room for shares -----------------------------------------------------------------------------------------------------
def captured(call, stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    return graph, out


def test_captured_on_a_stream_that_has_no_workspace(hq):
    """A call that would divide the keys does without, where the stream is being captured and nothing has been allocated for it."""
    dtype, u = TYPES["bf16"]
    pq, pk, pv = randn(1, 40, 32, 128).to(dtype), randn(2, 2940, 8, 128).to(dtype), randn(3, 2940, 8, 128).to(dtype)
    cu = i32([0, 40]), i32([0, 2940])
    torch.cuda.synchronize()
    graph, out = captured(lambda: hq.prompt_attention(pq, pk, pv, *cu), torch.cuda.Stream())
    for i in range(3):
        out.zero_()
        pq.copy_(randn(20 + i, *pq.shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_prompt(out, pq, pk, pv, [40], [2940], True, 1 / math.sqrt(128), u)
    for lengths, groups in (([2000], None), ([9000, 17, 400], None), ([900, 1000, 950], ([0, 3], [896]))):
        for heads in ((8, 2), (24, 1)):
            q, k, v, table, _ = paged_case(19, dtype, lengths, heads, 128, 16, *(groups or ()))
            args = (q, k, v, i32(table), i32(lengths)) + (tuple(i32(g) for g in groups) if groups else ())
            torch.cuda.synchronize()
            graph, out = captured(lambda: hq.paged_attention(*args), torch.cuda.Stream())
            for i in range(3):
                out.zero_()
                q.copy_(randn(30 + i, *q.shape))
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                check_paged(out, q, k, v, table, lengths, 1 / math.sqrt(128), u)
