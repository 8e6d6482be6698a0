"""Norms and rotations of queries' and keys' heads, by themselves and into the pages of the cache, against their formula in 64 bits.

Bound of every element, derived before the first run.  y = x * rsqrt(mean(x^2) + eps) * weight in fp32: the sum of up to 128 squares in
chains of at most 20 additions, off by 21 * 2^-24 relatively, half of that behind the root; the root itself 2^-23 and three products
2^-24 each: 2^-19 covers it.  a c - b s: two products and a sum of that, 2^-19 (|a c| + |b s|) covers the 2^-23 that they add; and one
rounding, u of the result (2^-8 bf16, 2^-11 fp16; among fp16's subnormal numbers 2^-25).  |got - want| <= u |want| + 2^-18 (|a c| + |b s|)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11)}


def randn(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def formula(x, weight, cos_sin, positions, eps, interleaved):
    """Result and |a c| + |b s| in 64 bits, pair by pair."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    want, size = y.clone(), y.abs()
    if cos_sin is not None:
        n = cos_sin.shape[1] // 2
        rows = cos_sin.double()[positions.long().clamp(0, len(cos_sin) - 1)][:, None]
        for i in range(n):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
            c, s = rows[..., i], rows[..., n + i]
            want[..., a] = y[..., a] * c - y[..., b] * s
            want[..., b] = y[..., b] * c + y[..., a] * s
            size[..., a] = (y[..., a] * c).abs() + (y[..., b] * s).abs()
            size[..., b] = (y[..., b] * c).abs() + (y[..., a] * s).abs()
    return want, size


def close(got, want, size, u):
    assert got.shape == want.shape
    excess = (got.double() - want).abs() - (u * want.abs() + 2.0 ** -18 * size + 2.0 ** -25)
    assert not torch.isnan(got).any() and excess.max().item() <= 0, excess.max().item()


def weights(seed, D, dtype):
    return [(1 + 0.3 * randn(seed + i, D)).to(dtype) for i in range(2)]


CASES = [(heads, tokens) for heads in ((1, 1), (14, 2), (32, 8), (3, 5), (64, 8)) for tokens in (1, 3, 70)]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rotary", [0, 16, 48, 64, 112, 128])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rotate(hq, kind, D, rotary, interleaved):
    if rotary > D:
        pytest.skip("no such head")
    dtype, u = TYPES[kind]
    table = hq.rotary_table(500, rotary) if rotary else None
    for n, ((h, kv), tokens) in enumerate(CASES):
        q, k = (2 * randn(10 * n, tokens, h, D)).to(dtype), randn(10 * n + 1, tokens, kv, D).to(dtype)
        positions = torch.randint(0, 500, (tokens,), device="cuda", dtype=torch.int32)
        qw, kw = weights(n, D, dtype)
        if n % 4 == 1:
            qw = None
        if n % 4 == 2:
            kw = None
        if n % 4 == 3:
            qw = kw = None
        got = hq.norm_rotate(q, k, table, positions, qw, kw, interleaved=interleaved)
        for g, x, w in ((got[0], q, qw), (got[1], k, kw)):
            close(g, *formula(x, w, table, positions, 1e-6, interleaved), u)


def test_rotary_table(hq):
    """Far positions: the angles themselves are right to 64 bits, their cosines and sines rounded once."""
    t = hq.rotary_table(100001, 64, base=500000.0)
    assert t.shape == (100001, 64) and t.dtype == torch.float32 and t.is_cuda
    for p in (0, 1, 77, 99999, 100000):
        for i in (0, 1, 15, 31):
            angle = p * 500000.0 ** (-2 * i / 64)
            assert abs(t[p, i].item() - math.cos(angle)) <= 2.0 ** -25 + 1e-10
            assert abs(t[p, 32 + i].item() - math.sin(angle)) <= 2.0 ** -25 + 1e-10


def test_positions_beyond_the_table_are_cut(hq):
    q, k = randn(1, 5, 4, 64).half(), randn(2, 5, 2, 64).half()
    table = hq.rotary_table(40, 64)
    got = hq.norm_rotate(q, k, table, i32([-1, -2 ** 31, 40, 2 ** 31 - 1, 39]))
    want = hq.norm_rotate(q, k, table, i32([0, 0, 39, 39, 39]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_parts_of_rows_and_in_place(hq, kind):
    dtype, u = TYPES[kind]
    n, h, kv, D = 37, 12, 3, 128
    qkv = randn(1, n, h + 2 * kv, D).to(dtype)
    before = qkv.clone()
    table, positions = hq.rotary_table(64, D), torch.arange(n, dtype=torch.int32, device="cuda")
    qw, kw = weights(3, D, dtype)
    q, k = qkv[:, :h], qkv[:, h:h + kv]
    want = hq.norm_rotate(q.contiguous(), k.contiguous(), table, positions, qw, kw)
    close(want[0], *formula(q, qw, table, positions, 1e-6, False), u)
    got = hq.norm_rotate(q, k, table, positions, qw, kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(qkv, before)
    wide = torch.full((n, h + kv + 2, D), 7.0, dtype=dtype, device="cuda")
    out = (wide[:, 1:1 + h], wide[:, 1 + h:1 + h + kv])
    got = hq.norm_rotate(q, k, table, positions, qw, kw, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and (wide[:, 0] == 7).all() and (wide[:, -1] == 7).all()
    hq.norm_rotate(q, k, table, positions, qw, kw, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, h + kv:], before[:, h + kv:])


def test_what_shares_memory_is_refused(hq):
    x = torch.zeros((9, 8, 64), dtype=torch.float16, device="cuda")
    flat = torch.zeros(20000, dtype=torch.float16, device="cuda")
    table, p = hq.rotary_table(16, 64), torch.zeros(9, dtype=torch.int32, device="cuda")
    q, k = x[:, :4], x[:, 4:6]
    for out in ((x[:, 1:5], None), (None, x[:, 3:5]), (x[:, 2:6], None), (None, x[:, 0:2]), (x[:, 4:8], None)):
        with pytest.raises(hq.HqError):
            hq.norm_rotate(q, k, table, p, out=out)
    same = flat[:9 * 4 * 64].view(9, 4, 64)
    with pytest.raises(hq.HqError):
        hq.norm_rotate(q, k, table, p, out=(same, same[:, :2]))
    shifted = flat[64:64 + 9 * 4 * 64].view(9, 4, 64)
    with pytest.raises(hq.HqError):  # the same rows, an element's width off, would be read after they are written
        hq.norm_rotate(same, k, table, p, out=(shifted, None))
    hq.norm_rotate(q, k, table, p, out=(None, x[:, 6:8]))
    hq.norm_rotate(x[:, 2:6], k[:, :1].contiguous(), table, p, out=(None, x[:, 0:1]))


def test_numbers_at_the_ends(hq):
    """bf16 values whose squares fp32 does not hold, tiny ones, rows of zeros, infinities and NaN."""
    D, table, p = 128, None, None
    x = randn(1, 6, 1, D).bfloat16()
    big = x.clone()
    big[0] *= 2.0 ** 100
    big[1] *= 2.0 ** 64
    big[2] *= 2.0 ** -80
    big[3] = 0
    big[4, 0, 5] = 3e38
    w = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    got, _ = hq.norm_rotate(big, big, table, p, w, w, eps=1e-6)
    close(got, *formula(big, w, None, None, 1e-6, False), 2.0 ** -8)
    assert (got[3] == 0).all()
    for what in (math.inf, -math.inf, math.nan):
        bad = x.clone()
        bad[2, 0, 9] = what
        got, _ = hq.norm_rotate(bad, bad, table, p, w, w)
        assert torch.isnan(got[2, 0, 9])
        rest = torch.arange(6, device="cuda") != 2
        assert torch.equal(got[rest], hq.norm_rotate(x, x, table, p, w, w)[0][rest])
        assert math.isnan(what) == torch.isnan(got[2, 0, 8]).item()  # an infinite mean makes the others 0, one of NaN NaN
    rotated = hq.rotary_table(8, 64)
    bad = x.clone()
    bad[0, 0, 3] = math.nan  # without a norm its pair alone
    got, _ = hq.norm_rotate(bad, bad, rotated, torch.full((6,), 3, dtype=torch.int32, device="cuda"))
    assert torch.isnan(got[0, 0]).nonzero().view(-1).tolist() == [3, 35] and torch.isfinite(got[1:]).all()


def test_far_weights(hq):
    """Heads of zeros, and of numbers near the ends, beside weights that make 1 / rms times weight larger or smaller than fp32 holds."""
    dtype, u = TYPES["bf16"]
    p = i32([0] * 3)
    for x, w, eps in ((0.0, 2.0 ** 80, 2.0 ** -126), (2.0 ** 60, 2.0 ** -85, 1e-6), (2.0 ** -60, 2.0 ** 70, 2.0 ** -126)):
        q = (x * (0.5 + randn(2, 3, 2, 64).abs())).to(dtype)
        weight = (w * (0.5 + randn(3, 64).abs())).to(dtype)
        got, _ = hq.norm_rotate(q, q[:, :1], None, p, weight, None, eps)
        want, size = formula(q, weight, None, p, eps, False)
        assert torch.isfinite(got).all() and ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -18 * size).all()


def test_nothing(hq):
    table = hq.rotary_table(4, 64)
    q, k = torch.zeros((0, 4, 64), dtype=torch.float16, device="cuda"), torch.zeros((0, 2, 64), dtype=torch.float16, device="cuda")
    got = hq.norm_rotate(q, k, table, i32([]))
    assert got[0].shape == q.shape and got[1].shape == k.shape


# ---- into the cache ----------------------------------------------------------------------------------------------------
def cache(seed, pages, kv, page, D, dtype):
    return [randn(seed + i, pages, kv, page, D).to(dtype) for i in range(2)]


def tables(lengths, page, spare, seed, width=None):
    use = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(use) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max(use + [1])
    rows = []
    for u in use:
        rows.append(order[:u] + [-1] * (width - u))
        order = order[u:]
    return i32(rows), sum(use) + spare


WRITES = [([0], [1]), ([17], [1]), ([0, 5, 30, 7], [40, 0, 1, 3]), ([100] * 70, [1] * 70), ([3, 0], [0, 0]), ([9], [300])]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D,rotary", [(64, 64), (64, 32), (128, 128), (128, 16)])
@pytest.mark.parametrize("heads", [(1, 1), (14, 2), (32, 8)])
@pytest.mark.parametrize("page", [1, 16, 1024])
def test_cache_write_rotated(hq, kind, D, rotary, heads, page):
    dtype, u = TYPES[kind]
    h, kv = heads
    table_of = hq.rotary_table(600, rotary)
    for n, (starts, new) in enumerate(WRITES):
        behind = 3 if n % 2 else 0
        tokens = sum(new) + behind
        qkv = randn(n, tokens, h + 2 * kv, D).to(dtype)
        q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        qw, kw = weights(n, D, dtype) if n % 3 else (None, None)
        table, pages = tables([a + b for a, b in zip(starts, new)], page, 4, n)
        kp, vp = cache(50 + n, pages, kv, page, D, dtype)
        want_k, want_v = kp.clone(), vp.clone()
        cu = [0]
        for m in new:
            cu.append(cu[-1] + m)
        positions = [a + i for a, m in zip(starts, new) for i in range(m)]
        out = torch.full((tokens, h, D), 7.0, dtype=dtype, device="cuda")
        got = hq.cache_write_rotated(q, k, v, kp, vp, table, i32(starts), i32(cu), table_of, qw, kw, interleaved=n % 2 == 1, out=out)
        assert got is out and (out[cu[-1]:] == 7).all()
        if cu[-1]:
            whole = hq.norm_rotate(q[:cu[-1]], k[:cu[-1]], table_of, i32(positions), qw, kw, interleaved=n % 2 == 1)
            assert torch.equal(out[:cu[-1]], whole[0])
            close(out[:cu[-1]], *formula(q[:cu[-1]], qw, table_of, i32(positions), 1e-6, n % 2 == 1), u)
            hq.cache_write(whole[1], v[:cu[-1]], want_k, want_v, table, i32(starts), i32(cu))
        assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


def test_cache_tokens_without_a_place(hq):
    """Pages that are missing or none, places before and behind the row: the queries are there all the same, the pages as they were."""
    h, kv, D, page = 4, 2, 64, 8
    new, starts = [10, 6, 5, 4], [3, -2, 30, 2 ** 31 - 3]
    qkv = randn(1, 25, h + 2 * kv, D).half()
    q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
    table = i32([[2, -1, 0, 5], [1, 99, 3, -7], [6, 6, 6, 4], [0, 0, 0, 0]])
    kp, vp = cache(5, 7, kv, page, D, torch.float16)
    before = kp.clone(), vp.clone()
    positions = [a + i for a, m in zip(starts, new) for i in range(m)]
    angles = hq.rotary_table(64, D)
    got = hq.cache_write_rotated(q, k, v, kp, vp, table, i32(starts), i32([0, 10, 16, 21, 25]), angles)
    want_q, want_k = hq.norm_rotate(q, k, angles, i32([min(max(p, 0), 63) for p in positions]))
    assert torch.equal(got, want_q)
    for t, p in enumerate(positions):
        row = 0 if t < 10 else 1 if t < 16 else 2 if t < 21 else 3
        entry = table[row, p // page].item() if 0 <= p < 32 else -1
        if 0 <= entry < 7:
            before[0][entry, :, p % page], before[1][entry, :, p % page] = want_k[t], v[t]
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
    none = torch.zeros((0, kv, page, D), dtype=torch.float16, device="cuda")
    assert torch.equal(hq.cache_write_rotated(q, k, v, none, none, table, i32(starts), i32([0, 10, 16, 21, 25]), angles), want_q)
    assert torch.equal(hq.cache_write_rotated(q, k, v, kp, vp, table[:, :0].contiguous(), i32(starts), i32([0, 10, 16, 21, 25]), angles), want_q)
    inside = q.clone()
    assert hq.cache_write_rotated(inside, k, v, kp, vp, table, i32(starts), i32([0, 10, 16, 21, 25]), angles, out=inside) is inside
    assert torch.equal(inside, want_q)


def test_graph_and_streams(hq):
    h, kv, D, page, rows = 8, 2, 128, 16, 5
    qkv = randn(1, rows, h + 2 * kv, D).bfloat16()
    q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
    starts, cu = i32([0, 9, 31, 4, 16]), torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    table, pages = tables([40] * rows, page, 0, 1)
    kp, vp = cache(3, pages, kv, page, D, torch.bfloat16)
    angles, (qw, kw) = hq.rotary_table(64, D), weights(1, D, torch.bfloat16)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = hq.cache_write_rotated(q, k, v, kp, vp, table, starts, cu, angles, qw, kw)
        both = hq.norm_rotate(q, k, angles, starts, qw, kw)
    for i in range(4):
        qkv.copy_(randn(10 + i, rows, h + 2 * kv, D))
        starts.copy_(i32([i, 9 + i, 31 - i, 4, 16 + i]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want_k, want_v = kp.clone(), vp.clone()
        want = hq.norm_rotate(q, k, angles, starts, qw, kw)
        hq.cache_write(want[1], v, want_k, want_v, table, starts, cu)
        assert torch.equal(out, want[0]) and torch.equal(both[0], want[0]) and torch.equal(both[1], want[1])
        assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
