"""What CachedLM.forward turns down before any layer runs (on the CPU; no kernel is launched)."""

import pytest

torch = pytest.importorskip("torch")

from redline_tiny_b200 import vlm  # noqa: E402


@pytest.mark.parametrize("x,cos,sin,match", [
    (torch.zeros(3, 256), torch.zeros(3, 64), torch.zeros(3, 64), "bf16"),
    (torch.zeros(3, 256, dtype=torch.float16), torch.zeros(3, 64), torch.zeros(3, 64), "bf16"),
    (torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, 64), torch.zeros(3, 64), "256"),
    (torch.zeros(3, 256, 1, dtype=torch.bfloat16), torch.zeros(3, 64), torch.zeros(3, 64), "256"),
    (torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(6, 32), torch.zeros(6, 32), "cos and sin"),
    (torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, 64), torch.zeros(64), "cos and sin"),
    (torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(2, 64), torch.zeros(2, 64), "2 rows"),
])
def test_rows_and_angles(monkeypatch, x, cos, sin, match):
    """A wrong type or shape would be read as if it were the right one."""
    lm = vlm.CachedLM.__new__(vlm.CachedLM)
    lm.cfg, lm.kv, lm.few, lm.layers = vlm.LMConfig(hidden=256, heads=2, kv_heads=1, ffn=256), object(), 64, [{"p_in": None}]

    class Batch:
        kv, rows = lm.kv, 3

    def reached(*a, **k):
        raise AssertionError("a layer was run")
    monkeypatch.setattr(vlm.ops, "ln_mod", reached)
    with pytest.raises(ValueError, match=match):
        lm.forward(x, Batch(), cos, sin)
