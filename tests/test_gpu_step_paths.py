"""Steps behind a shared prefix, rotation and logits where their host and device code can take another way: without the native host path, on
another stream, with pieces of the prefix that cross from one head to the next, long own tokens, counts of 32 bits, offsets behind 2^31."""
import ctypes
import math
import time

import pytest
import torch

from adkv_b200 import _lib, gemv, step
from adkv_b200.cache import KVCacheLayer
from tests.test_gpu_prefix import D, SCALING, Shared
from tests.test_gpu_step import logits_check, logits_inputs, rope_check, rope_inputs, rope_want


def _state(c):
    return [t.clone() for t in (c.kc, c.vc, c.kt, c.vt)]


def _prefix_steps(lens):
    c = Shared(2, 8, 2, 333, 96, lens, seed=21)
    first = c.step(tail_keep=True)
    ints = c.step(T=0, tail_keep=True, scratch=torch.empty(gemv.prefix_scratch_bytes(c.B, 8, c.prefix), dtype=torch.uint8, device="cuda"),
                  out=torch.empty_like(first))
    return [first, ints, c.step()] + _state(c)


@pytest.mark.gpu
def test_python_path_equals_the_native_one(monkeypatch):
    x, kw = logits_inputs(3, 5000, 200, torch.bfloat16, bias="all")
    qkv, cos, sin, wq, wk = rope_inputs(2, 9, 4, 2, 128, 64, torch.bfloat16)
    pos = torch.tensor([5, 100], dtype=torch.int32, device="cuda")

    def everything():
        plain = {k: v for k, v in kw.items() if k not in ("history", "history_lens")}
        return (_prefix_steps([3, 40, 0]) + list(step.process_logits(x, **kw)) + list(step.process_logits(x, **plain)) +
                list(step.norm_rope_qkv(qkv, 4, 2, cos, sin, positions=pos, q_weight=wq, k_weight=wk, interleaved=True, dtype=torch.float16)) +
                list(step.norm_rope_qkv(qkv, 4, 2, cos, sin, start=11)))
    assert _lib.host() is not None
    native = everything()
    monkeypatch.setattr(_lib, "host", lambda: None)
    python = everything()
    assert len(native) == len(python)
    for a, b in zip(native, python):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_what_the_native_path_leaves_alone():
    c = Shared(4, 4, 2, 100, 64, [3, 5], seed=2)
    host, before = _lib.host(), _state(c)
    base = [c.q, c.prefix._native, c.kc, c.vc, *c.new, c.kp, c.vp, c.lens_gpu, SCALING, 0.1, 1.0, c.kt, c.vt, _lib.flags(True), None, None]

    def other(i, x):
        a = list(base)
        a[i] = x
        return host.decode_prefix(*a)
    for i, x in [(0, c.q.float()), (0, c.q[:1]), (0, c.q.cpu()), (1, (0,) * 4), (1, c.prefix._native[:3]), (1, c.prefix._native[:1] + (3,) + c.prefix._native[2:]),
                 (2, c.kc[:, :, :, ::2]), (3, c.vc[:1]), (4, c.new[0][:1]), (5, None), (6, c.kp[:4]), (8, c.lens_gpu.long()), (8, c.lens_gpu[:1]),
                 (8, 8 * c.cap), (8, -1), (8, 2.0), (12, None), (13, c.vt[:1]), (14, "x"), (15, torch.empty(2, 4, D, device="cuda")),
                 (16, torch.empty(1 << 20, dtype=torch.uint8))]:
        done = other(i, x)
        assert done is None or (isinstance(done, int) and done < 0), i
    for t, b in zip(_state(c), before):
        assert torch.equal(t, b)
    assert gemv.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits,Hq,Hkv,P,interval,lens,room", [
    (4, 150, 150, 1000, 96, [0, 7], None),                     # 150 units: the line is cut evenly, most pieces cross from head to head
    (2, 256, 32, 70, 32, [0, 1, 2, 30] * 40, None),            # 320 units of 128 rows, more than CTAs
    (4, 300, 300, 33, 32, [2], None),                          # a piece of several heads
    (4, 8, 1, 100, 32, [5, 700, 1], 130),                      # own tokens in tiles of 64 for eight heads
    (4, 4, 4, 50, 32, [129, 640], None),
    (2, 8, 2, 50, 0, [1500, 3], None)])
def test_pieces_that_cross_and_long_own_tokens(bits, Hq, Hkv, P, interval, lens, room):
    c = Shared(bits, Hq, Hkv, P, interval, lens, seed=P, room=room)
    got = c.step(tail_keep=True)
    c.check(got, c.want())
    assert torch.equal(got, c.step(tail_keep=True))            # sums in a fixed order
    assert gemv.device_status() == 0


@pytest.mark.gpu
def test_two_steps_at_once_and_a_stream_that_is_not_the_first():
    c, d = Shared(4, 32, 32, 3000, 128, [60] * 4, seed=1), Shared(2, 32, 8, 5000, 128, [100] * 8, seed=2)
    want = [x.step(tail_keep=True) for x in (c, d)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, s) in enumerate(zip((c, d), streams)):
            with torch.cuda.stream(s):
                got[i].append(x.step(tail_keep=True))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.gpu
def test_one_prefix_for_calls_of_different_sizes_and_its_owner_going_on():
    """The parent is continued, past a growth of its buffers, while forks of different sizes read what it had."""
    torch.manual_seed(0)
    params = Shared(4, 2, 2, 1, 32, [0]).kp
    params = tuple(params) * 2
    kv = lambda B, T: [torch.randn(B, 2, T, D, device="cuda").half() for _ in range(2)]
    parent = KVCacheLayer(checkpoint_interval=32)
    first, q = kv(1, 77), torch.randn(5, 2, 1, D, device="cuda").half()
    parent.prefill(*first, *params)
    forks = [parent.fork(n) for n in (1, 5)]
    parent.prefill(*kv(1, 900), *params)                       # fills up the last word, then grows
    late = parent.fork(2)
    assert [f.get_seq_length() for f in forks + [late]] == [77, 77, 977]
    new = kv(5, 1)
    for child, B in zip(forks, (1, 5)):
        whole = KVCacheLayer()
        whole.prefill(*(x.expand(B, -1, -1, -1).contiguous() for x in first), *params)
        args = (q[:B], new[0][:B], new[1][:B], *params)
        got, want = child.decode(*args, scaling=SCALING)[0], whole.decode(*args, scaling=SCALING)[0]
        assert ((got - want).abs() <= 2e-3 + 2e-3 * want.abs()).all()
        assert all(torch.equal(a, b) for a, b in zip(child.tails, whole.tails))


@pytest.mark.gpu
@pytest.mark.parametrize("bits,P,interval,B", [(4, 300, 0, 2), (2, 300, 32, 130), (4, 3000, 64, 2)])
def test_waits_that_run_out_end_the_step(bits, P, interval, B):
    """The scans of the prefix's keys do nothing: every wait behind them ends after its second, the results are NaN, the own tokens and
    the new one are cached as always, and the next step is as if nothing had been."""
    c = Shared(bits, 4, 2, P, interval, [3] * B, seed=8)
    before = _state(c)
    good = c.step()
    after = _state(c)
    for t, b in zip((c.kc, c.vc, c.kt, c.vt), before):
        t.copy_(b)
    out = torch.zeros_like(good)
    scratch = torch.zeros(gemv.prefix_scratch_bytes(B, 4, c.prefix), dtype=torch.uint8, device="cuda")
    kp, vp = (_lib.Params(*[t.data_ptr() for t in p]) for p in (c.kp, c.vp))
    assert gemv.device_status() == 0
    t0 = time.perf_counter()
    rc = _lib.load().adkv_decode_attn_prefix(
        c.q.data_ptr(), ctypes.addressof(c.prefix.desc), c.kc.data_ptr(), c.vc.data_ptr(), c.new[0].data_ptr(), c.new[1].data_ptr(), ctypes.addressof(kp),
        ctypes.addressof(vp), c.kt.data_ptr(), c.vt.data_ptr(), c.lens_gpu.data_ptr(), 0, out.data_ptr(), scratch.data_ptr(), scratch.numel(), B, 4, 2, D,
        c.cap, bits, SCALING, *c.bounds, _lib.FLAG_SELFTEST_MUTE_K, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    torch.cuda.synchronize()
    seconds = time.perf_counter() - t0
    assert 1 <= gemv.device_status() <= 4 and gemv.device_status() == 0
    assert torch.isnan(out).all()
    assert 0.9 < seconds < 4.0, seconds
    for t, b in zip(_state(c), after):
        assert torch.equal(t, b)
    for t, b in zip((c.kc, c.vc, c.kt, c.vt), before):
        t.copy_(b)
    assert torch.equal(c.step(scratch=scratch), good)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
def test_first_own_token_by_append_and_by_prefill(bits):
    """A token appended at index 0, quantised as a chunk of one, and appended by the step: the same codes and tails."""
    c = Shared(bits, 4, 2, 100, 64, [0, 0, 0], seed=6)
    tails, caches = [], []
    for how in range(3):
        kt, vt = c.prefix.start_tails(3)
        kc, vc = torch.zeros_like(c.kc), torch.zeros_like(c.vc)
        if how == 0:
            gemv.append_kv_pair(kc, c.new[0], c.kp, kt, vc, c.new[1], c.vp, vt, 0, *c.bounds, bits=bits)
        elif how == 1:
            gemv.encode_kv_pair(kc, c.new[0], c.kp, vc, c.new[1], c.vp, *c.bounds, bits=bits, k_tail=kt, v_tail=vt, from_tail=True)
        else:
            gemv.decode_attn_prefix(c.q, c.prefix, kc, vc, *c.new, c.kp, c.vp, 0, SCALING, *c.bounds, k_tail=kt, v_tail=vt)
        tails.append((kt, vt))
        caches.append((kc, vc))
    for other in (1, 2):
        for a, b in zip(tails[0] + caches[0], tails[other] + caches[other]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_counts_of_32_bits():
    for V, L in ((70, 70000), (40000, 100000)):
        x, kw = logits_inputs(2, V, L, torch.float32)
        kw["history"][0, :66000] = 5                            # more often than 16 bits hold
        kw["history_lens"][0] = L
        kw["frequency"] = 1e-4
        logits_check(x, step.process_logits(x, **kw), kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_logits_in_place_in_parts(dtype):
    """A row that several CTAs share, worked on where it lies."""
    x, kw = logits_inputs(2, 50257, 4000, dtype)
    before = x.clone()
    out, tokens = step.process_logits(x, out=x, **kw)
    assert out is x
    logits_check(before, (x, tokens), kw)
    again = step.process_logits(before, **kw)
    assert torch.equal(again[0].nan_to_num(), x.nan_to_num()) and torch.equal(again[1], tokens)


@pytest.mark.gpu
def test_logits_of_rows_behind_2_to_31():
    B, V = 17000, 128256                                        # 2.18e9 elements
    row, kw = logits_inputs(1, V, 300, torch.float16)
    x = torch.zeros(B, V, dtype=torch.float16, device="cuda")
    x[-1] = row[0]
    history = torch.zeros(B, 300, dtype=torch.int32, device="cuda")
    history[-1] = kw["history"][0]
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    lens[-1] = kw["history_lens"][0]
    out, tokens = step.process_logits(x, out=x, history=history, history_lens=lens, repetition=1.5, bias=kw["bias"])
    want = dict(history=kw["history"], history_lens=kw["history_lens"], repetition=1.5, bias=kw["bias"])
    logits_check(row, (out[-1:], tokens[-1:]), want)
    assert int(tokens[5]) == int(kw["bias"].half().argmax())


@pytest.mark.gpu
def test_rotation_of_tokens_behind_2_to_31():
    T, Hq, Hkv = 180000, 32, 32                                 # 2.2e9 elements
    _, cos, sin, _, _ = rope_inputs(1, 1, 1, 1, 128, 128, torch.float16, rows=10)
    qkv = torch.zeros(1, T, 96 * 128, dtype=torch.float16, device="cuda")
    qkv[:, -3:] = torch.randn(3, 96 * 128, device="cuda")
    pos = torch.zeros(1, T, dtype=torch.int32, device="cuda")
    pos[0, -3:] = torch.tensor([9, 0, 4])
    got = step.norm_rope_qkv(qkv, Hq, Hkv, cos, sin, positions=pos)
    want = rope_want(qkv[:, -3:], Hq, Hkv, cos, sin, pos[:, -3:].cpu().long(), None, None, 1e-6, False)
    rope_check([t[:, :, -3:].contiguous() for t in got], want, torch.float16)
    assert not got[0][:, :, :1000].any()


@pytest.mark.gpu
def test_rotation_positions_at_the_ends_of_32_bits():
    qkv, cos, sin, _, _ = rope_inputs(2, 3, 2, 1, 64, 64, torch.float16, rows=10)
    pos = torch.tensor([2 ** 31 - 2, -2 ** 31], dtype=torch.int32, device="cuda")
    q, k, v = step.norm_rope_qkv(qkv, 2, 1, cos, sin, positions=pos)
    assert gemv.device_status() == 8
    assert torch.isnan(q).all() and torch.isnan(k).all() and not torch.isnan(v).any()
    # rows of zeros with and without eps
    zero = torch.zeros_like(qkv)
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    assert not step.norm_rope_qkv(zero, 2, 1, cos, sin, q_weight=w, k_weight=w)[0].any()


@pytest.mark.gpu
def test_rows_of_queries_that_are_no_numbers_stay_apart():
    """A query of infinities or NaN spoils its own rows only."""
    c = Shared(4, 4, 2, 300, 64, [3, 0, 9], seed=4)
    good = c.step(tail_keep=True)
    c.q[1, 2, 0, 5] = math.nan
    c.q[2, 0, 0, 7] = math.inf
    got = c.step(tail_keep=True)
    spoilt = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    spoilt[1, 2] = spoilt[2, 0] = True
    assert torch.equal(got[~spoilt], good[~spoilt]) and torch.isnan(got[1, 2]).all()
