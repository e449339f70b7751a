"""Sizes that do not fit the library's 32-bit arguments are refused, not cut off."""
import pytest
import torch

from adkv_b200 import gemv, step

pytestmark = pytest.mark.gpu
HUGE = (1 << 32) + 40        # 40 in 32 bits


def test_rotation_tables():
    qkv, row = torch.randn(1, 3, 3 * 64, device="cuda").half(), torch.ones(1, 8, device="cuda")
    positions = torch.tensor([50], dtype=torch.int32, device="cuda")
    for kw in (dict(start=20), dict(start=50), dict(positions=positions)):
        with pytest.raises(RuntimeError, match="2\\^31 rows"):
            step.norm_rope_qkv(qkv, 1, 1, row.expand(HUGE, 8), row.expand(HUGE, 8), **kw)
    most = row.expand((1 << 31) - 1, 8)
    step.norm_rope_qkv(qkv, 1, 1, most, most, positions=positions)
    assert gemv.device_status() == 0


def test_history():
    logits = torch.randn(1, 100, device="cuda")
    history = torch.empty(HUGE, dtype=torch.int32, device="cuda").view(1, -1)       # 17 GB, of which little is touched
    lens = torch.tensor([50], dtype=torch.int32, device="cuda")
    history[0, :50] = 7
    with pytest.raises(RuntimeError, match="2\\^31 tokens"):
        step.process_logits(logits, history=history, history_lens=lens, frequency=1.0)
    out, _ = step.process_logits(logits, history=history[:, :(1 << 31) - 1], history_lens=lens, frequency=1.0)
    assert abs(float(out[0, 7]) - (float(logits[0, 7]) - 50.0)) <= 50 * 2.0 ** -23
