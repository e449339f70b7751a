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


def allow(*rows):
    """Mask words [B, ceil(V / 32)]: the tokens that each row allows."""
    m = torch.zeros(B, (BARE.vocab + 31) // 32, dtype=torch.int64)
    for b, row in enumerate(rows):
        for t in row:
            m[b, t // 32] |= 1 << (t % 32)
    return torch.where(m >= 1 << 31, m - (1 << 32), m).int()


def test_a_sequence_that_is_left_no_token_has_ended(monkeypatch):
    """Its token is -1 from then on, whatever the rules allow later; no row of the embedding stands for it, and the others go on."""
    mask = allow(range(50), range(50), [7, 40])
    m, other = (model(monkeypatch, 12, mask=x, frequency=0.5) for x in (mask, allow(range(50), range(50), [7, 40])))
    ids = tokens(2, B, 4)
    tok = m.prefill(ids)
    assert torch.equal(tok, other.prefill(ids)) and int(tok[2]) in (7, 40)
    mask[1] = 0
    for i in range(5):
        before = tok
        tok, want = m.decode(tok), other.decode(tok.clamp(min=0))
        assert torch.equal(m.last_logits, other.last_logits)              # taken along with token 0
        assert tok.tolist() == [int(want[0]), -1, int(want[2])]
        assert m.history[:, 4 + i].tolist() == before.tolist()
        if i == 2:
            mask[1] = -1
    assert m.history_lens.tolist() == [9] * B
    mask[0] = 0
    fresh = model(monkeypatch, 12, mask=mask)
    assert int(fresh.prefill(ids)[0]) == -1


def test_without_rules_tokens_are_taken_as_they_are(monkeypatch):
    m = ADKVLlama(BARE, B, 8, device="cpu")
    tok = m.prefill(tokens(3, B, 2))
    assert torch.equal(tok, m.last_logits.argmax(-1)) and torch.equal(m.decode(tok), m.last_logits.argmax(-1))


@pytest.mark.parametrize("rows,vocab", [(1, 1), (5, 5), (4, 50), (7, 3), (9, 1)])
def test_first_tokens_in_turn(rows, vocab):
    """Row b's b-th most likely token, round and round where the vocabulary or what the row allows is smaller than the batch."""
    g = torch.Generator().manual_seed(rows * vocab)
    logits = torch.randn(rows, vocab, generator=g).half()
    allowed = torch.rand(rows, vocab, generator=g) < torch.linspace(0, 1, rows)[:, None]
    for x in (logits, logits[:1].expand(rows, vocab), logits.masked_fill(~allowed, -math.inf)):
        got = e2e_llama._in_turn(x)
        assert got.shape == (rows,) and got.dtype == torch.int64
        for b in range(rows):
            order = sorted((v for v in range(vocab) if x[b, v] > -math.inf), key=lambda v: -float(x[b, v]))
            if not order:
                assert int(got[b]) == -1
            else:
                assert x[b, int(got[b])] == x[b, order[b % len(order)]]      # of equal logits either


def test_shards_stepped_together_keep_the_history(monkeypatch):
    """Prefill and steps of co-resident shards look at the history that one model does; every shard holds it."""
    one = model(monkeypatch, 12, frequency=30.0)
    shards = [ADKVLlama(BARE, B, 12, device="cpu", rank=r, world=2, peers=[], logit_rules=dict(frequency=30.0)) for r in range(2)]
    ids = tokens(6, B, 4)
    tok = one.prefill(ids)
    assert torch.equal(e2e_llama.prefill_together(shards, ids), tok)
    for _ in range(6):
        got = e2e_llama.step_together(shards, tok)
        tok = one.decode(tok)
        assert torch.equal(got, tok)
    for m in shards:
        assert torch.equal(m.history, one.history) and torch.equal(m.history_lens, one.history_lens)
