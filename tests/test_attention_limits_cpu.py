"""Sizes that attention and the cache refuse because what they are multiplied into would not fit, and page sizes that one operator of the
cache takes and another does not: the C entry points' own checks, before any HIP call."""
import os
import re

from hecbench_amd import _lib

MOST = 2 ** 31 - 1
CSRC = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")


def paged(**kw):
    a = dict(q=16, k=16, v=16, out=16, dtype=2, table=16, lengths=16, groups=None, shared=None, ngroups=0, batch=1, width=4, pages=9, page=16, heads=8,
             kv=2, d=128, qs=1024, scale=0.1, stream=None)
    a.update(kw)
    return _lib.load().hq_paged_attention(*a.values())


def write(**kw):
    a = dict(k=16, v=16, kp=16, vp=16, dtype=1, table=16, starts=16, cu=16, rows=2, tokens=3, width=4, pages=9, page=16, kv=2, d=64, ks=128, vs=128,
             stream=None)
    a.update(kw)
    return _lib.load().hq_cache_write(*a.values())


def step(**kw):
    a = dict(pool=16, planes=2, bytes=32, table=1 << 44, lengths=2 << 44, refs=3 << 44, parent=4 << 44, add=5 << 44, to=6 << 44, lo=7 << 44,
             ro=8 << 44, so=9 << 44, missing=10 << 44, rows=3, width=4, pages=9, page=16, stream=None)
    a.update(kw)
    return _lib.load().hq_cache_step(*a.values())


def test_pages_of_four_gibibytes():
    """Bytes of a page, all heads: kv_heads * head_dim * 2 * page_size in 32 bits."""
    assert paged(page=1024, kv=16384, heads=16384, qs=16384 * 128) == -6
    assert paged(page=1024, kv=32768, heads=32768, d=64, qs=32768 * 64) == -6


def test_tables_within_a_workgroup_of_two_to_the_31():
    """Keys are numbered in 32 bits, and a kernel's loads and shares go some way beyond the last."""
    assert paged(page=1024, width=2 ** 21 - 1) == -6
    assert paged(page=8, width=(MOST - 300) // 8) == -6


def test_prompts_within_a_workgroup_of_two_to_the_31():
    def prompt(tk):
        return _lib.load().hq_prompt_attention(16, 16, 16, 16, 1, 16, 16, 1, 4, tk, 8, 2, 64, 512, 128, 128, 0.1, 1, None)
    assert prompt(MOST - 200) == -6


def test_steps_of_too_many_pages_and_of_pages_too_large():
    """Pages are numbered in 32 bits by loops that go a stretch beyond the last; a length is rounded up to whole pages in 32 bits."""
    assert step(pages=MOST) == -6 and step(pages=MOST - 4095) == -6
    assert step(width=1, page=MOST - 1024) == -6 and step(width=2, page=2 ** 30 - 600) == -6


def test_steps_of_too_many_entries():
    """What is handed out is numbered in 32 bits by loops that go a workgroup beyond the last."""
    assert step(rows=2, width=2 ** 30 - 1, page=1) == -6 and step(rows=16384, width=2 ** 17, page=1) == -6


def test_page_sizes_that_are_not_written():
    """Powers of two up to 1024, as attention takes them from 8 on."""
    assert write(page=24) == -2 and write(page=2048) == -2 and write(page=3) == -2
    assert paged(page=24) == -2 and paged(page=2048) == -2


def test_pools_of_no_pages_are_taken():
    """No refusal for want of pages: the next one in the order of the checks comes."""
    assert paged(pages=0, k=None, v=None, q=24) == -4
    assert paged(pages=9, k=None, q=24) == -1 and paged(pages=0, table=None) == -1


def test_assembly_that_writes_m0_says_so():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".hip", ".h")):
            text = open(os.path.join(CSRC, name)).read()
            for asm in re.findall(r"asm volatile\((.*?)\);", text, re.S):
                if "s_mov_b32 m0" in asm:
                    assert '"m0"' in asm.rsplit(":", 1)[1], (name, asm)
