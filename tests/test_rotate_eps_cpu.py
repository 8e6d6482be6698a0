"""eps is the norm's: without one it is not looked at.  No GPU: what passes the checks ends at the device."""
import math

import pytest

from tests.test_rotate_validation_cpu import rotate, write

pytestmark = pytest.mark.no_gpu


@pytest.mark.parametrize("f", [rotate, write])
@pytest.mark.parametrize("eps", [0.0, -1.0, 2.0 ** -127, math.inf, math.nan])
def test_eps(f, eps):
    assert f(qw=None, kw=None, eps=eps) not in (-1, -2, -3, -4, -6)
    assert f(eps=eps) == -2 and f(qw=None, eps=eps) == -2 and f(kw=None, eps=eps) == -2
