"""Memory that results of norms and rotations must not share: refused before any pointer reaches a kernel.  No GPU: what passes the checks ends at
the device."""
import pytest

from tests.test_rotate_validation_cpu import rotate, write

pytestmark = pytest.mark.no_gpu
REFUSED = -2
CHECKED = (-1, -2, -3, -4, -6)
Q, K, V, QO, KO, VO = ((i + 1) << 40 for i in range(6))  # as in rotate() and write(): rows of 512 and 128 halves, 1024 and 256; pages of 10 * 2 * 16 * 128


@pytest.mark.parametrize("name,size", [("qw", 128), ("kw", 128), ("cs", 4 * 10 * 64), ("p", 24)])
@pytest.mark.parametrize("out,row", [(QO - (1 << 40), 1024), (KO - (1 << 40), 256)])
def test_norm_rotate(name, size, out, row):
    end = out + 6 * row
    for at in (out, out + 16, out + row - 16, end - 16, out - size + 16):
        assert rotate(**{name: at}) == REFUSED, hex(at)
    for at in (end, out - (size + 15) // 16 * 16):
        assert rotate(**{name: at}) not in CHECKED, hex(at)


def test_between_rows():
    """Weights in the gap that rows leave: read, and not written."""
    wide = dict(qos=512 + 256)
    assert rotate(qw=(3 << 40) + 1024, **wide) not in CHECKED
    assert rotate(qw=(3 << 40) + 1536 + 1024 + 384, **wide) not in CHECKED
    for at in (1008, 1536 - 112, 1536):
        assert rotate(qw=(3 << 40) + at, **wide) == REFUSED
    assert rotate(cs=(3 << 40) + 1024, **wide) == REFUSED  # longer than the gap


def test_what_no_rotation_reads():
    assert rotate(rotary=0, cs=3 << 40, p=3 << 40) not in CHECKED
    assert rotate(qw=None, kw=None) not in CHECKED


@pytest.mark.parametrize("name,size", [("qw", 256), ("kw", 256), ("cs", 4 * 10 * 32), ("table", 48), ("starts", 12), ("cu", 16)])
def test_cache_write_rotated(name, size):
    pages = 10 * 2 * 16 * 128 * 2
    for out, n in ((QO, 6 * 2048), (KO, pages), (VO, pages)):
        for at in (out, out + 2048, out + n - 16, out - (size + 15) // 16 * 16 + 16):
            assert write(**{name: at}) == REFUSED, (name, hex(at))
        assert write(**{name: out + n}) not in CHECKED
        assert write(**{name: out - (size + 15) // 16 * 16}) not in CHECKED


def test_pages():
    pages = 10 * 2 * 16 * 128 * 2
    for name, n in (("q", 6 * 2048), ("k", 6 * 512), ("v", 6 * 512), ("qo", 6 * 2048)):
        for at in (KO, VO, VO + pages - 16, KO - n + 16):
            assert write(**{name: at}) == REFUSED, (name, hex(at))
        assert write(**{name: KO + pages}) not in CHECKED and write(**{name: KO - n}) not in CHECKED
    assert write(vp=KO) == REFUSED and write(vp=KO + pages - 16) == REFUSED and write(vp=KO + pages) not in CHECKED
    assert write(pages=0, kp=QO, vp=QO) not in CHECKED and write(width=0, kp=QO, vp=QO) not in CHECKED
    assert write(q=KO + 4 * (1 << 40), pages=2 ** 31 - 1, page=1024, kv=1 << 16, ks=1 << 23, vs=1 << 23) == REFUSED  # far more than any memory
