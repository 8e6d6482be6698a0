"""What norms and rotations refuse, before any pointer reaches a kernel: no GPU."""
import pytest
import torch

import hecbench_amd as hq
from hecbench_amd import _lib


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def refuse(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_norm_rotate():
    q, k, t, p, w = half(6, 8, 64), half(6, 2, 64), torch.zeros(10, 64), i32(6), half(64)
    f = hq.norm_rotate
    refuse("device tensors only", f, q, k, t, p)
    refuse("device tensors only", f, q, k, t, p, w, w, out=(half(6, 8, 64), half(6, 2, 64)))
    refuse("device tensors only", f, q, k, None, None, w, w)
    refuse("q must be float16 or bfloat16", f, q.float(), k, t, p)
    refuse("k must have the type", f, q, k.bfloat16(), t, p)
    refuse("k must be \\[tokens of q\\]", f, q, half(5, 2, 64), t, p)
    refuse("k must be \\[tokens of q\\]", f, q, half(6, 2, 128), t, p)
    refuse("cos_sin must be float32", f, q, k, t.half(), p)
    refuse("cos_sin must be \\[positions\\]", f, q, k, t.view(-1), p)
    refuse("cos_sin must not hold more", f, q, k, torch.zeros(10, 80), p)
    refuse("cos_sin must be contiguous", f, q, k, torch.zeros(10, 80)[:, :64], p)
    refuse("positions is required", f, q, k, t, None)
    refuse("positions must be int32", f, q, k, t, p.long())
    refuse("positions must hold 6", f, q, k, t, i32(5))
    refuse("q_weight must hold 64", f, q, k, t, p, half(128))
    refuse("k_weight must be float16", f, q, k, t, p, w, w.float())
    refuse("one behind the other", f, half(8, 6, 64).transpose(0, 1), k, t, p)
    refuse("not overlap itself", f, half(6 * 8 * 64).as_strided((6, 8, 64), (64, 64, 1)), k, t, p)
    refuse("out\\[0\\] must have the shape", f, q, k, t, p, out=(half(6, 7, 64), None))
    refuse("out\\[1\\] must be float16", f, q, k, t, p, out=(None, k.bfloat16()))
    refuse("too many values", f, q, k, t, p, out=(q, k, k))


def test_cache_write_rotated():
    q, k, t, w = half(6, 8, 64), half(6, 2, 64), torch.zeros(10, 64), half(64)
    pages, table, starts, cu = half(10, 2, 16, 64), i32(3, 4), i32(3), i32(4)
    f = hq.cache_write_rotated
    refuse("device tensors only", f, q, k, k, pages, pages, table, starts, cu, t, w, w)
    refuse("device tensors only", f, q, k, k, pages, pages, table, starts, cu, None, w, w, out=half(6, 8, 64))
    refuse("k must have the type", f, q, k.bfloat16(), k, pages, pages, table, starts, cu, t)
    refuse("v must have the shape", f, q, k, half(6, 3, 64), pages, pages, table, starts, cu, t)
    refuse("v must have the type", f, q, k, k.bfloat16(), pages, pages, table, starts, cu, t)
    refuse("k must be \\[tokens of q\\]", f, half(5, 8, 64), k, k, pages, pages, table, starts, cu, t)
    refuse("k_pages must be \\[pages\\]", f, q, k, k, half(10, 3, 16, 64), pages, table, starts, cu, t)
    refuse("v_pages must", f, q, k, k, pages, half(9, 2, 16, 64), table, starts, cu, t)
    refuse("v_pages must have the shape", f, q, k, k, pages, half(20, 2, 8, 64), table, starts, cu, t)
    refuse("table must be \\[requests\\]", f, q, k, k, pages, pages, i32(12), starts, cu, t)
    refuse("starts must hold 3", f, q, k, k, pages, pages, table, i32(2), cu, t)
    refuse("cu must hold 4", f, q, k, k, pages, pages, table, starts, i32(3), t)
    refuse("out must have the shape", f, q, k, k, pages, pages, table, starts, cu, t, out=half(6, 2, 64))


def rotate(**kw):
    a = dict(q=1 << 40, k=2 << 40, qo=3 << 40, ko=4 << 40, dtype=2, qw=16, kw=16, cs=16, p=16, tokens=6, heads=8, kv=2, d=64, rotary=64, known=10,
             qs=512, ks=128, qos=512, kos=128, eps=1e-6, inter=0, stream=None)
    a.update(kw)
    return _lib.load().hq_norm_rotate(*a.values())


def write(**kw):
    a = dict(q=1 << 40, k=2 << 40, v=3 << 40, qo=4 << 40, kp=5 << 40, vp=6 << 40, dtype=1, qw=16, kw=16, cs=16, table=16, starts=16, cu=16, rows=3,
             tokens=6, width=4, pages=10, page=16, heads=8, kv=2, d=128, rotary=32, known=10, qs=1024, ks=256, vs=256, qos=1024, eps=1e-6, inter=1,
             stream=None)
    a.update(kw)
    return _lib.load().hq_cache_write_rotated(*a.values())


def test_entry_points():
    for f in (rotate, write):
        for kw, rc in (({"tokens": 0}, 0), ({"tokens": -1}, -2), ({"heads": 0}, -2), ({"kv": 0}, -2), ({"d": 96}, -2), ({"rotary": 24}, -2),
                       ({"rotary": 144}, -2), ({"rotary": -16}, -2), ({"known": 0}, -2), ({"known": -1}, -2), ({"eps": 0.0}, -2), ({"eps": -1.0}, -2),
                       ({"eps": float("nan")}, -2), ({"eps": float("inf")}, -2), ({"dtype": 0}, -3), ({"cs": None}, -1), ({"q": None}, -1), ({"k": None}, -1),
                       ({"qo": None}, -1), ({"qs": 500}, -2), ({"qs": 1028}, -4), ({"ks": 100}, -2), ({"q": (1 << 40) + 8}, -4), ({"qw": 8}, -4),
                       ({"kw": 8}, -4), ({"cs": 8}, -4), ({"qos": 1020 if f is write else 516}, -2 if f is write else -4),
                       ({"tokens": 1 << 31}, -6), ({"heads": 1 << 20, "qs": 1 << 27, "qos": 1 << 27}, -6), ({"qs": 1 << 32}, -6),
                       ({"qo": 2 << 40}, -2), ({"qo": (1 << 40) + 512}, -2)):
            assert f(**kw) == rc, (f.__name__, kw)
    for kw, rc in (({"ko": None}, -1), ({"p": None}, -1), ({"p": 18}, -4), ({"ko": 3 << 40}, -2), ({"ko": 1 << 40}, -2), ({"kos": 120}, -2)):
        assert rotate(**kw) == rc, kw
    for kw, rc in (({"v": None}, -1), ({"page": 24}, -2), ({"page": 2048}, -2), ({"page": 0}, -2), ({"rows": -1}, -2), ({"width": -1}, -2), ({"pages": -1}, -2),
                   ({"table": None}, -1), ({"starts": None}, -1), ({"cu": None}, -1), ({"kp": None}, -1), ({"kp": 8}, -4), ({"table": 18}, -4),
                   ({"rows": 0}, 0), ({"qo": 3 << 40}, -2), ({"vs": 100}, -2)):
        assert write(**kw) == rc, kw


def test_columns_of_one_row_are_apart():
    """q, k and their results side by side in rows of 20 heads: refused only where they meet.  (What passes the checks ends at the device.)"""
    base, row = 1 << 40, 20 * 64
    def at(q, k, qo, ko):
        return rotate(q=base + 128 * q, k=base + 128 * k, qo=base + 128 * qo, ko=base + 128 * ko, qs=row, ks=row, qos=row, kos=row)
    ok = at(0, 8, 10, 18)
    assert ok not in (-1, -2, -3, -4, -6)
    assert at(0, 8, 0, 8) == ok and at(0, 8, 0, 10) == ok and at(12, 10, 0, 8) == ok
    for bad in ((0, 8, 1, 10), (0, 8, 10, 17), (0, 8, 2, 10), (0, 8, 9, 18), (0, 8, 10, 7), (0, 8, 10, 9), (0, 8, 13, 10)):
        assert at(*bad) == -2, bad
