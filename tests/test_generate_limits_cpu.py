"""What the example refuses before it touches a device."""
from types import SimpleNamespace

import pytest
import torch

from hecbench_amd.examples import generate


def test_more_tokens_than_positions():
    """Positions beyond the table would be cut to it by the operators, and the tokens there rotated alike."""
    model = SimpleNamespace(angles=torch.zeros(40, 64), layers=[], kv_heads=1, head_dim=64)
    with pytest.raises(ValueError, match="40 positions"):
        generate.Server(model, [torch.zeros(12, 8), torch.zeros(31, 8)], 2, 10)


def test_the_command_asks_for_as_many_as_it_needs(monkeypatch):
    """60 prompts of up to 10407 tokens."""
    asked = {}

    def decoder(layers, **kw):
        asked.update(kw)
        raise KeyboardInterrupt

    monkeypatch.setattr(generate, "Decoder", decoder)
    monkeypatch.setattr(generate.hq, "init", lambda: None)
    monkeypatch.setattr("sys.argv", ["generate", "--prompts", "60", "--tokens", "100"])
    with pytest.raises(KeyboardInterrupt):
        generate.main()
    assert asked["longest"] >= 200 + 173 * 59 + 100
