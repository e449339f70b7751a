"""Logit rules in the harness's steps on the GPU: sequences that are left no token, eager and replayed."""
import pytest
import torch

from adkv_b200 import gemv
from adkv_b200.e2e_llama import ADKVLlama, LlamaShape

pytestmark = pytest.mark.gpu
TINY = LlamaShape(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=128, ffn=512, vocab=503)
WORDS = (TINY.vocab + 31) // 32


def _mask(B, fill=-1):
    return torch.full((B, WORDS), fill, dtype=torch.int32, device="cuda")


def _ids(seed, *size):
    return torch.randint(0, TINY.vocab, size, generator=torch.Generator().manual_seed(seed)).cuda()


def test_a_sequence_that_is_left_no_token_has_ended():
    B, P = 3, 20
    ids = _ids(1, B, P)
    eager, graph = [], []
    masks = [_mask(B) for _ in range(2)]
    a, b = (ADKVLlama(TINY, B, P + 12, device="cuda", seed=3, logit_rules=dict(mask=m, repetition=1.2)) for m in masks)
    tok = a.prefill(ids)
    assert torch.equal(tok, b.prefill(ids))
    got = b.capture_decode(tok, 2)
    for t in range(8):
        if t == 4:
            masks[0][1] = 0
        if t == 6:
            masks[0][1] = -1
        tok = a.decode(tok)
        eager.append(tok.tolist())
    for t in range(2, 8):
        if t == 4:
            masks[1][1] = 0
        if t == 6:
            masks[1][1] = -1
        got = b.decode_replay(got)
        graph.append(got.tolist())
    assert graph == eager[2:]
    assert [row[1] for row in eager[4:]] == [-1] * 4 and all(t >= 0 for row in eager for t in (row[0], row[2]))
    assert torch.equal(a.history, b.history) and a.history[1, P + 5:P + 8].tolist() == [-1] * 3
    assert gemv.device_status() == 0


def test_replayed_steps_behind_the_last_place():
    """They have no results (a position without a row in the tables, later a cache without room), and write nowhere else."""
    B, P, room = 2, 9, 4
    m = ADKVLlama(TINY, B, P + room, device="cuda", seed=3, logit_rules=dict(frequency=0.1))
    tok = m.capture_decode(m.prefill(_ids(2, B, P)), 1)
    for _ in range(room - 1):
        tok = m.decode_replay(tok)
    assert gemv.device_status() == 0
    before = m.history[:, :P + room].clone()
    for _ in range(6):
        tok = m.decode_replay(tok)
    assert m.history_lens.tolist() == [P + room + 1] * B and torch.equal(m.history[:, :P + room], before)
    assert bool(((tok >= -1) & (tok < TINY.vocab)).all()) and gemv.device_status() in (6, 8)


@pytest.mark.parametrize("B", [2, 6])
def test_first_tokens_behind_a_shared_prompt_are_allowed(B):
    mask = _mask(B, 0)
    mask[:, 1] = 0b1110                  # tokens 33, 34, 35
    mask[B - 1] = 0                      # none
    m = ADKVLlama(TINY, B, 8, device="cuda", seed=3, shared_tokens=40, logit_rules=dict(mask=mask))
    tok = m.prefill_shared(_ids(5, 33))
    order = (33 + m.last_logits[0, 33:36].float().argsort(descending=True)).tolist()
    assert tok.tolist() == [order[b % 3] for b in range(B - 1)] + [-1]
    nxt = m.decode(tok)
    assert all(33 <= t <= 35 for t in nxt.tolist()[:-1]) and int(nxt[-1]) == -1 and gemv.device_status() == 0


def test_more_sequences_behind_a_shared_prompt_than_tokens():
    shape = LlamaShape(**{**TINY.__dict__, "vocab": 5})
    m = ADKVLlama(shape, 8, 4, device="cuda", seed=3, shared_tokens=16)
    tok = m.prefill_shared(_ids(5, 9) % 5)
    order = m.last_logits[0].float().argsort(descending=True).tolist()
    assert tok.tolist() == [order[b % 5] for b in range(8)] and m.decode(tok).shape == (8,)
