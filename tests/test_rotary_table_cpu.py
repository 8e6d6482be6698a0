"""The table of angles: what it refuses, and its shape.  On the CPU, which it is made on."""
import pytest
import torch

import hecbench_amd as hq


@pytest.mark.parametrize("rotary", [-16, 1, 8, 17, 33, 65, 127])
def test_refusals(rotary):
    with pytest.raises(ValueError, match="multiple of 16"):
        hq.rotary_table(4, rotary, device="cpu")


@pytest.mark.parametrize("positions", [0, 1, 5])
@pytest.mark.parametrize("rotary", [0, 16, 48, 128])
def test_shapes(positions, rotary):
    t = hq.rotary_table(positions, rotary, device="cpu")
    assert t.shape == (positions, rotary) and t.dtype == torch.float32
    if positions and rotary:
        assert (t[0, :rotary // 2] == 1).all() and (t[0, rotary // 2:] == 0).all()
