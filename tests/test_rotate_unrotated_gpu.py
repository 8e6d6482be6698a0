"""Elements that no rotation reaches: behind the rotated ones, or all of them.  Without a norm they are the input's bits, and what is not finite
among them, or in them, reaches no other element; with a norm an infinity makes every other element of its head 0."""
import math

import pytest
import torch

from tests.test_rotate_gpu import TYPES, i32, randn, weights

pytestmark = pytest.mark.gpu
BAD = [math.nan, math.inf, -math.inf]
# (head size, rotated elements, an element behind them or None, a rotated one or None)
PLACES = [(64, 0, 9, None), (64, 0, 63, None), (64, 16, 16, 3), (64, 16, 40, 15), (64, 48, 55, 20), (64, 64, None, 33), (128, 0, 70, None), (128, 16, 30, 9),
          (128, 64, 70, 40), (128, 64, 127, 0), (128, 112, 120, 60), (128, 128, None, 5)]


def bits(x):
    return x.contiguous().view(torch.int16)


def calls(hq, q, k, rotary, qw, kw, interleaved):
    """Queries and keys of norm_rotate, and of cache_write_rotated."""
    n, D = q.shape[0], q.shape[2]
    angles = hq.rotary_table(64, rotary) if rotary else None
    yield hq.norm_rotate(q, k, angles, i32([5 + i for i in range(n)]), qw, kw, interleaved=interleaved)
    kp, vp = (torch.full((2, k.shape[1], 16, D), 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    rq = hq.cache_write_rotated(q, k, k, kp, vp, i32([[1, 0]]), i32([5]), i32([0, n]), angles, qw, kw, interleaved=interleaved)
    pages = torch.cat([kp[1], kp[0]], 1).transpose(0, 1)[5:5 + n]
    assert torch.equal(bits(torch.cat([vp[1], vp[0]], 1).transpose(0, 1)[5:5 + n]), bits(k))
    yield rq, pages


def partner(at, rotary, interleaved):
    if interleaved:
        return at ^ 1
    return (at + rotary // 2) % rotary


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rotary,behind,within", PLACES)
def test_without_a_norm(hq, kind, interleaved, D, rotary, behind, within):
    dtype, _ = TYPES[kind]
    q, k = randn(1, 6, 14, D).to(dtype), randn(2, 6, 2, D).to(dtype)
    q[0, 0, rotary:] = -0.0
    q[0, 1, rotary::2] = -0.0
    clean = list(calls(hq, q, k, rotary, None, None, interleaved))
    for got in clean:
        for g, x in zip(got, (q, k)):
            assert torch.equal(bits(g[..., rotary:]), bits(x[..., rotary:]))
    for what in BAD:
        for at in (behind, within):
            if at is None:
                continue
            touched = [at] if at >= rotary else [at, partner(at, rotary, interleaved)]
            rest = [i for i in range(D) if i not in touched]
            bq, bk = q.clone(), k.clone()
            bq[3, 13, at] = bk[4, 1, at] = what
            for got, want in zip(calls(hq, bq, bk, rotary, None, None, interleaved), clean):
                for g, w, (token, head) in zip(got, want, ((3, 13), (4, 1))):
                    assert torch.equal(bits(g[token, head, rest]), bits(w[token, head, rest])), (what, at)
                    if at < rotary:  # times a cosine or a sine, of either sign
                        assert not torch.isfinite(g[token, head, touched]).any()
                    else:
                        assert repr(g[token, head, at].item()) == repr(what)
                    g = g.clone()
                    g[token, head] = w[token, head]
                    assert torch.equal(bits(g), bits(w))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rotary,behind,within", PLACES)
def test_with_a_norm(hq, kind, interleaved, D, rotary, behind, within):
    """x * rsqrt(infinity) * weight is 0 but for the infinity itself, which is NaN then, and so is what is rotated against it."""
    dtype, _ = TYPES[kind]
    q, k = randn(1, 6, 14, D).to(dtype), randn(2, 6, 2, D).to(dtype)
    qw, kw = weights(3, D, dtype)
    clean = list(calls(hq, q, k, rotary, qw, kw, interleaved))
    for what in BAD:
        for at in (behind, within):
            if at is None:
                continue
            touched = [at] if at >= rotary else [at, partner(at, rotary, interleaved)]
            rest = [i for i in range(D) if i not in touched]
            bq, bk = q.clone(), k.clone()
            bq[3, 13, at] = bk[4, 1, at] = what
            for got, want in zip(calls(hq, bq, bk, rotary, qw, kw, interleaved), clean):
                for g, w, (token, head) in zip(got, want, ((3, 13), (4, 1))):
                    assert torch.isnan(g[token, head, touched]).all()
                    assert torch.isnan(g[token, head, rest]).all() if math.isnan(what) else (g[token, head, rest] == 0).all(), (what, at)
                    g = g.clone()
                    g[token, head] = w[token, head]
                    assert torch.equal(bits(g), bits(w))
