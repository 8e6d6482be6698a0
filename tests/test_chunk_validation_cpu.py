"""What attention of chunks and windows refuse, before any pointer reaches a kernel: no GPU."""
import pytest
import torch

import hecbench_amd as hq
from hecbench_amd import _lib

MOST = 2 ** 31 - 1


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def refuse(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_chunk_attention():
    q, p, table, n, cu = half(7, 8, 64), half(10, 2, 16, 64), i32(3, 4), i32(3), i32(4)
    f = hq.chunk_attention
    refuse("device tensors only", f, q, p, p, table, n, cu)
    refuse("device tensors only", f, q, p, p, table, n, cu, 5, 3)
    refuse("device tensors only", f, q, p, p, table, n, cu, 2 ** 70, 2 ** 70)
    refuse("q must be float16 or bfloat16", f, q.float(), p, p, table, n, cu)
    refuse("k_pages must be float16", f, q, p.bfloat16(), p, table, n, cu)
    refuse("k_pages must be \\[pages\\]", f, q, half(10, 2, 16, 128), p, table, n, cu)
    refuse("v_pages must hold", f, q, p, half(9, 2, 16, 64), table, n, cu)
    refuse("v_pages must have the shape", f, q, p, half(10, 16, 2, 64), table, n, cu)
    refuse("table must be \\[requests\\]", f, q, p, p, i32(12), n, cu)
    refuse("lengths must hold 3", f, q, p, p, table, i32(4), cu)
    refuse("cu_q must hold 4", f, q, p, p, table, n, i32(3))
    refuse("cu_q must be int32", f, q, p, p, table, n, cu.long())
    refuse("window must be", f, q, p, p, table, n, cu, 0)
    refuse("window must be", f, q, p, p, table, n, cu, -3)
    refuse("sinks must not be negative", f, q, p, p, table, n, cu, 5, -1)
    refuse("sinks go with", f, q, p, p, table, n, cu, None, 1)
    refuse("out must hold", f, q, p, p, table, n, cu, out=half(6, 8, 64))
    refuse("one behind the other", f, half(8, 7, 64).transpose(0, 1), p, p, table, n, cu)


def test_prompt_window():
    q, k, cu = half(6, 8, 64), half(6, 2, 64), i32(3)
    f = hq.prompt_attention
    refuse("device tensors only", f, q, k, k, cu, window=4, sinks=1)
    refuse("window goes with causal", f, q, k, k, cu, causal=False, window=4)
    refuse("window must be", f, q, k, k, cu, window=0)
    refuse("sinks go with", f, q, k, k, cu, sinks=2)
    refuse("sinks must not be negative", f, q, k, k, cu, window=3, sinks=-2)


def chunk(**kw):
    a = dict(q=16, k=16, v=16, out=16, dtype=2, table=16, lengths=16, cu=16, batch=2, total=9, width=4, pages=9, page=16, heads=8, kv=2, d=128, qs=1024,
             scale=0.1, window=0, sinks=0, stream=None)
    a.update(kw)
    return _lib.load().hq_chunk_attention(*a.values())


def prompt(**kw):
    a = dict(q=16, k=16, v=16, out=16, dtype=1, cu=16, ck=16, seqs=2, tq=9, tk=30, heads=8, kv=2, d=64, qs=512, ks=128, vs=128, scale=0.1, window=5,
             sinks=1, stream=None)
    a.update(kw)
    return _lib.load().hq_prompt_attention_window(*a.values())


def test_entry_points():
    for kw, rc in (({"batch": 0}, 0), ({"total": 0}, 0), ({"batch": -1}, -2), ({"total": -1}, -2), ({"width": -1}, -2), ({"pages": -1}, -2), ({"window": -1}, -2),
                   ({"sinks": -1}, -2), ({"heads": 7}, -2), ({"heads": 0}, -2), ({"kv": 0}, -2), ({"page": 24}, -2), ({"page": 4}, -2), ({"page": 2048}, -2),
                   ({"d": 96}, -2), ({"dtype": 0}, -3), ({"scale": -1.0}, -2), ({"scale": float("nan")}, -2), ({"scale": float("inf")}, -2),
                   ({"q": None}, -1), ({"k": None}, -1), ({"v": None}, -1), ({"out": None}, -1), ({"table": None}, -1), ({"lengths": None}, -1), ({"cu": None}, -1),
                   ({"qs": 1000}, -2), ({"qs": 1028}, -4), ({"q": 24}, -4), ({"k": 24}, -4), ({"out": 8}, -4), ({"cu": 18}, -4), ({"lengths": 18}, -4),
                   ({"width": 2 ** 27}, -6), ({"total": 2 ** 29}, -6), ({"total": MOST + 1, "heads": 2}, -6),
                   ({"page": 1024, "kv": 16384, "heads": 16384, "qs": 16384 * 128}, -6), ({"batch": 2 ** 30, "total": 2 ** 28}, -6)):
        assert chunk(**kw) == rc, kw
    for kw, rc in (({"window": 0}, -2), ({"window": -1}, -2), ({"sinks": -1}, -2), ({"d": 32}, -2), ({"dtype": 5}, -3), ({"q": None}, -1), ({"ks": 1 << 23}, -6),
                   ({"tq": 0}, 0), ({"seqs": 0}, 0), ({"tk": MOST - 200}, -6)):
        assert prompt(**kw) == rc, kw
