"""One prompt, several completions, as a program runs them: the cache object's fork, the harness with a shared prompt, rotation and
logit rules in its steps, eager and from a captured graph."""
import pytest
import torch

from adkv_b200 import gemv, synth
from adkv_b200.cache import KVCache, KVCacheLayer
from adkv_b200.e2e_llama import ADKVLlama, LlamaShape

D = 128
TINY = LlamaShape(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=128, ffn=512, vocab=503)


def _flat(params):
    return tuple(p.reshape(-1).cuda() for p in params)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,Hq,Hkv,interval", [(4, 4, 4, 64), (2, 8, 2, 32), (4, 2, 1, 0)])
def test_fork_continues_like_layers_that_hold_everything(bits, Hq, Hkv, interval):
    """Prefill, fork, a second chunk per sequence, steps across a growth of the buffers: codes and tails of a layer per sequence that was
    given the whole token run, results up to the rounding of the shared values (fp16, of values of a few units: 2e-3 as everywhere)."""
    B, P, chunk, steps = 3, 150, 20, 60
    k, v = (synth.gen_kv(s, B, Hkv, P + chunk + steps, D).cuda() for s in (1, 2))
    k[:, :, :P], v[:, :, :P] = k[:1, :, :P], v[:1, :, :P]
    params = (*_flat(synth.gen_params(3, Hkv, D, bits)), *_flat(synth.gen_params(4, Hkv, D, bits)))
    q = torch.randn(steps, B, Hq, 1, D, generator=torch.Generator().manual_seed(0)).half().cuda()
    parent = KVCacheLayer(bits=bits, checkpoint_interval=interval)
    parent.prefill(k[:1, :, :100], v[:1, :, :100], *params)
    parent.prefill(k[:1, :, 100:P], v[:1, :, 100:P], *params)
    child, whole = parent.fork(B), KVCacheLayer(bits=bits)
    assert child.get_seq_length() == P and child.get_mask_sizes(1) == (P + 1, 0)
    whole.prefill(k[:, :, :P + chunk], v[:, :, :P + chunk], *params)
    child.prefill(k[:, :, P:P + 7], v[:, :, P:P + 7], *params)
    child.prefill(k[:, :, P + 7:P + chunk], v[:, :, P + 7:P + chunk], *params)
    for t in range(steps):
        at = slice(P + chunk + t, P + chunk + t + 1)
        args = (q[t], k[:, :, at], v[:, :, at], *params)
        got, weights = child.decode(*args, scaling=0.09)
        want, _ = whole.decode(*args, scaling=0.09)
        assert weights is None
        assert ((got - want).abs() <= 2e-3 + 2e-3 * want.abs()).all()
        if t % 20 == 3:        # the layer that was forked goes on by itself, in the same buffers
            parent.decode(q[t][:1], k[:1, :, at], v[:1, :, at], *params, scaling=0.09)
    assert child.get_seq_length() == whole.get_seq_length() == P + chunk + steps
    for a, b in zip(child.tails, whole.tails):
        assert torch.equal(a, b)
    again = parent.fork(2)     # behind what the parent has appended since
    assert again.get_seq_length() == P + 3
    again.decode(q[0][:2], k[:2, :, :1], v[:2, :, :1], *params, scaling=0.09)
    assert gemv.device_status() == 0


@pytest.mark.gpu
def test_fork_refusals():
    params = (*_flat(synth.gen_params(3, 2, D, 4)), *_flat(synth.gen_params(4, 2, D, 4)))
    x = torch.randn(2, 2, 40, D, device="cuda").half()
    with pytest.raises(ValueError, match="nothing is cached"):
        KVCacheLayer().fork(2)
    for layer, n in ((KVCacheLayer(), 2), (KVCacheLayer(half_state=True), 1), (KVCacheLayer(fused=False), 1)):
        layer.prefill(x[:n], x[:n], *params)
        with pytest.raises(ValueError, match="one sequence with tail states"):
            layer.fork(2)
    layer = KVCacheLayer()
    layer.prefill(x[:1], x[:1], *params)
    with pytest.raises(ValueError, match="at least one"):
        layer.fork(0)
    child = layer.fork(2)
    with pytest.raises(ValueError, match="cannot be forked"):
        child.fork(2)
    with pytest.raises(ValueError, match="no mask"):
        child.decode(x[:, :, :1], x[:, :, :1], x[:, :, :1], *params, attention_mask=torch.zeros(2, 1, 1, 41, device="cuda"))
    caches = KVCache(2)
    for c in caches:
        c.prefill(x[:1], x[:1], *params)
    both = caches.fork(3)
    assert len(both) == 2 and both.get_seq_length(1) == 40


def _model(B, own, shared=0, seed=3, **kw):
    m = ADKVLlama(kw.pop("shape", TINY), B, own, device="cuda", seed=seed, shared_tokens=shared, **kw)
    for L in m.layers:         # random-init attention is nearly uniform and would hide mistakes
        L["wqkv"][: (m.hq + m.hkv) * D] *= 40.0
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
def test_shared_prompt_gives_the_logits_of_a_batch_of_prompts(bits):
    """Steps of the harness with the prompt kept once against the same tokens fed to a model whose sequences hold the prompt each; eager
    and replayed.  Both run in fp16 and lie within 2e-2 of an fp32 restatement (test_gpu_e2e.py), twice that of one another; with 2-bit
    codes, where a flipped code of a new token is a coarse step, twice that again."""
    B, P, gen = 3, 77, 12
    ids = torch.randint(0, TINY.vocab, (P,), generator=torch.Generator().manual_seed(1)).cuda()
    a, b, c = _model(B, gen + 1, P + 3, bits=bits, shared_interval=32), _model(B, P + gen + 1, bits=bits), _model(B, gen + 1, P, bits=bits)
    tok = a.prefill_shared(ids)
    assert len(set(tok.tolist())) == B and int(tok[0]) == int(b.prefill(ids.expand(B, -1))[0])
    assert torch.equal(c.prefill_shared(ids), tok)
    graph_tok, eager = c.capture_decode(tok, 2), []
    for _ in range(gen):
        nxt = a.decode(tok)
        b.decode(tok)
        scale = float(b.last_logits.float().abs().max())
        assert float((a.last_logits.float() - b.last_logits.float()).abs().max()) < 4e-2 * (2 if bits == 2 else 1) * scale
        tok = nxt
        eager.append(tok)
    for t in range(1, gen - 1):    # the same steps from the graph
        assert torch.equal(graph_tok, eager[t])
        graph_tok = c.decode_replay(graph_tok)
    assert gemv.device_status() == 0


@pytest.mark.gpu
def test_graph_replays_are_the_eager_steps():
    B, P = 4, 50
    ids = torch.randint(0, TINY.vocab, (P,), generator=torch.Generator().manual_seed(2)).cuda()
    rules = dict(repetition=1.4, frequency=0.2)
    a, b = (_model(B, 20, P, logit_rules=dict(rules)) for _ in range(2))
    tok = first = a.prefill_shared(ids)
    assert torch.equal(first, b.prefill_shared(ids))
    eager = []
    for _ in range(10):
        tok = a.decode(tok)
        eager.append(tok)
    got = b.capture_decode(first, 3)
    assert torch.equal(got, eager[2])
    for t in range(3, 10):
        got = b.decode_replay(got)
        assert torch.equal(got, eager[t])
    assert torch.equal(a.history[:, :P + 10], b.history[:, :P + 10]) and torch.equal(a.history_lens, b.history_lens)


@pytest.mark.gpu
def test_logit_rules_choose_the_tokens():
    """A hard repetition rule lets no token come twice, a mask only what it allows; the choice is process_logits of the step's logits."""
    B, P, gen = 2, 9, 30
    ids = torch.randint(0, TINY.vocab, (B, P), generator=torch.Generator().manual_seed(4)).cuda()
    allowed = torch.zeros(B, (TINY.vocab + 31) // 32, dtype=torch.int32, device="cuda")
    allowed[:, 2:9] = -1                                                       # tokens 64 .. 287
    m = _model(B, P + gen + 1, logit_rules=dict(presence=1e4, mask=allowed))
    tok = m.prefill(ids)
    seen = [set(row.tolist()) for row in ids]
    for _ in range(gen):
        for b in range(B):
            t = int(tok[b])
            assert 64 <= t < 288 and t not in seen[b]
            seen[b].add(t)
        tok = m.decode(tok)
    assert m.history_lens.tolist() == [P + gen] * B


@pytest.mark.gpu
def test_harness_normalises_queries_and_keys():
    shape = LlamaShape(**{**TINY.__dict__, "qk_norm": True})
    m = _model(2, 40, shape=shape)
    L = m.layers[0]
    L["q_norm"].copy_(1 + 0.1 * torch.randn(D, device="cuda"))
    h = torch.randn(2, 5, TINY.d_model, device="cuda").half()
    q, k, v = m._qkv(L, h, 3)
    x = (h @ L["wqkv"].T).view(2, 5, 8, D).transpose(1, 2)
    for got, part, w in ((q, x[:, :4], L["q_norm"]), (k, x[:, 4:6], L["k_norm"])):
        y = part.double() / torch.sqrt(part.double().pow(2).mean(-1, keepdim=True) + shape.norm_eps) * w.double()
        a, b = y[..., :64], y[..., 64:]
        cos, sin = m.cos[3:8, :64].double(), m.sin[3:8, :64].double()
        want = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -11 + 80 * 2.0 ** -24 * y.abs().amax() + 2.0 ** -25).all()
    assert torch.equal(v, x[:, 6:])
    tok = m.prefill(torch.randint(0, TINY.vocab, (2, 9), device="cuda"))
    m.decode(tok)
    assert torch.isfinite(m.last_logits).all()


def test_shared_prompt_needs_tails():
    for kw in (dict(fused=False), dict(half_state=True), dict(ckpt_interval=32)):
        with pytest.raises(ValueError, match="shared prompt"):
            ADKVLlama(LlamaShape(**{**TINY.__dict__, "n_layers": 0}), 1, 8, device="cpu", shared_tokens=8, **kw)
