"""The harness's logit rules on the CPU, with the logit operator restated in torch: what a sequence's history holds and which tokens
are chosen."""
import math

import pytest
import torch

from adkv_b200 import e2e_llama
from adkv_b200.e2e_llama import ADKVLlama, LlamaShape

BARE = LlamaShape(n_layers=0, d_model=32, n_heads=2, n_kv_heads=2, head_dim=128, ffn=64, vocab=50)     # embedding, norm and head only
B = 3


def process_logits(logits, *, history, history_lens, repetition=1.0, presence=0.0, frequency=0.0, bias=None, mask=None):
    x = logits.double()
    for b, n in enumerate(history_lens.tolist()):
        for t in history[b, :n].tolist():
            if 0 <= t < x.shape[1]:
                x[b, t] -= frequency
        for t in {t for t in history[b, :n].tolist() if 0 <= t < x.shape[1]}:
            x[b, t] -= presence
    if bias is not None:
        x = x + bias
    if mask is not None:
        at = torch.arange(x.shape[1])
        x = torch.where((mask[:, at // 32] >> (at % 32).int() & 1).bool(), x, -math.inf)
    top, tokens = x.max(-1)
    return x.to(logits.dtype), torch.where(top == -math.inf, -1, tokens).int()


def model(monkeypatch, max_tokens, shape=BARE, **rules):
    monkeypatch.setattr(e2e_llama.step, "process_logits", process_logits)
    return ADKVLlama(shape, B, max_tokens, device="cpu", logit_rules=rules)


def tokens(seed, *size):
    return torch.randint(0, BARE.vocab, size, generator=torch.Generator().manual_seed(seed))


def test_steps_behind_the_last_place_stay_inside_the_history(monkeypatch):
    """A replayed step cannot know on the host that its sequences are full: its writes must stay inside the rows all the same."""
    m = model(monkeypatch, 4)
    m.prefill(tokens(0, B, 3))
    rows = m.history.shape[1]
    for i in range(rows + 3):
        tok = torch.full((B,), i)
        m._remember(tok)
        n = min(3 + i + 1, rows)
        assert m.history_lens.tolist() == [n] * B and m.history[:, n - 1].tolist() == [i] * B
    assert torch.equal(m.history[:, :3].long(), tokens(0, B, 3))


def test_a_refused_step_leaves_the_history_alone(monkeypatch):
    m = model(monkeypatch, 8, LlamaShape(**{**BARE.__dict__, "n_layers": 1}))
    m.T, before = 4, m.history.clone()
    for _ in range(12):
        with pytest.raises(RuntimeError, match="CUDA tensor"):       # the attention has no CPU path
            m.decode(tokens(1, B))
    assert m.history_lens.tolist() == [0] * B and torch.equal(m.history, before) and m.T == 4
