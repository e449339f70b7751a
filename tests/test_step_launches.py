"""Which kernels the steps behind a shared prefix, the rotation and the logits launch, and what is left where a launch is refused: on the
CPU, with a stand-in for the CUDA runtime."""
import ctypes

import pytest

from adkv_b200 import _lib
from tests.launches import PTR, _pp, run

PLACES = 296       # two CTAs on each of 148 SMs


def prefix(B, Hq, Hkv, P, interval, T=0, lens=PTR, bits=4, room=4096, fail=()):
    words = P // (32 // bits) + 1
    desc = _lib.Prefix(PTR, PTR, PTR, PTR, PTR, PTR, P, words, interval, P // interval + 1 if interval else 0)
    return run("adkv_decode_attn_prefix", PTR, ctypes.addressof(desc), PTR, PTR, PTR, PTR, _pp, _pp, PTR, PTR, lens, T, PTR, PTR, 1 << 60, B, Hq,
               Hkv, 128, room // (32 // bits), bits, 0.1, 0.1, 1.0, 0, None, fail=fail)


def names(got):
    return [next(n for n in ("prefix_kernel", "prefix_own", "prefix_join", "norm_rope", "process_logits") if n in g[0]) for g in got]


def test_three_launches_behind_one_another():
    rc, got = prefix(4, 8, 8, 1000, 64)
    assert rc == 0 and names(got) == ["prefix_kernel", "prefix_own", "prefix_join"]
    assert [g[3] for g in got] == [False, True, True]
    assert [g[1] for g in got[1:]] == [4 * 8, 4 * 8]
    rc, got = prefix(4, 8, 8, 576, 64)                    # nine parts
    assert rc == 0 and len(got) == 3
    rc, got = prefix(4, 8, 8, 512, 64)                    # few parts of a row: no join
    assert rc == 0 and names(got) == ["prefix_kernel", "prefix_own"] and [g[3] for g in got] == [False, True]
    rc, got = prefix(4, 8, 8, 0, 0)                       # nothing in front
    assert rc == 0 and names(got) == ["prefix_own"] and not got[0][3]
    assert prefix(0, 8, 8, 1000, 64) == (0, [])


@pytest.mark.parametrize("fail,left", [(("cudaLaunchKernel", 1), 0), (("cudaFuncSetAttribute", 1), 0)])
def test_refused_before_anything_runs(fail, left):
    rc, got = prefix(4, 8, 8, 1000, 64, fail=[fail])
    assert rc != 0 and len(got) == left
    rc, got = prefix(4, 8, 8, 1000, 64)                   # and no error stays behind
    assert rc == 0 and len(got) == 3


@pytest.mark.parametrize("nth", [1, 2])
def test_refused_beside_follows(nth):
    """Once tokens may be appended the result has to be finished: what is refused beside is launched behind."""
    rc, got = prefix(4, 8, 8, 1000, 64, fail=[("cudaLaunchKernelExC", nth)])
    assert rc == 0 and names(got) == ["prefix_kernel", "prefix_own", "prefix_join"]
    assert [g[3] for g in got[1:]] == [nth != 1, nth != 2]


@pytest.mark.parametrize("B,Hq,Hkv,P,interval,ctas", [
    (1, 1, 1, 1, 0, 1), (1, 1, 1, 100000, 0, 1),          # no checkpoints: one run a head
    (1, 1, 1, 8192, 128, 64), (4, 32, 32, 8192, 128, 256), (4, 32, 32, 9216, 128, 256), (64, 32, 32, 8192, 128, 256), (64, 32, 32, 9216, 128, 288),
    (129, 32, 32, 8192, 128, 256),
    (2, 150, 150, 1000, 96, PLACES), (160, 256, 32, 70, 32, PLACES), (1, 400, 400, 64, 64, PLACES), (1, 200, 200, 640, 64, 200)])
def test_ctas_of_the_prefix(B, Hq, Hkv, P, interval, ctas):
    rc, got = prefix(B, Hq, Hkv, P, interval)
    assert rc == 0 and got[0][1] == ctas


def test_more_than_a_launch_can_hold_is_refused():
    assert prefix(1 << 24, 1, 1, 100, 32)[0] == 0 and prefix((1 << 24) + 1, 1, 1, 100, 32) == (-4, [])
    assert prefix(1 << 20, 1 << 12, 1 << 12, 100, 32) == (-4, [])
    assert run("adkv_decode_attn_prefix_scratch_bytes", 1 << 20, 1 << 12, 1 << 12, 100, 32)[0] == -4
    assert run("adkv_process_logits", PTR, 8, PTR, 7, 0, PTR, None, 0, 0, None, None, 1.0, None, 0.0, None, 0.0, None, 0, None, 0, 2, 8, None) == (-4, [])
    assert run("adkv_process_logits", PTR, 8, PTR, 7, 0, PTR, None, 0, 0, None, None, 1.0, None, 0.0, None, 0.0, None, 0, None, 0, 1, 8, None)[0] == 0


def test_tiles_of_own_tokens():
    """Short sequences take tiles of 32 tokens, by what the cache has room for or the length given."""
    def tok(**kw):
        return prefix(4, kw.pop("Hq", 8), 8, 100, 64, **kw)[1][1][0]
    assert tok(room=128) != tok(room=256) and tok(room=256) == tok(room=4096)
    assert tok(lens=None, T=100) == tok(room=128) and tok(lens=None, T=200) == tok(room=256)
    assert tok(Hq=64, room=1000) != tok(Hq=64, room=1008)


def rope(B, T, Hq, Hkv, D, kinds=(0, 0), fail=()):
    return run("adkv_norm_rope_qkv", PTR, T * (Hq + 2 * Hkv) * D, (Hq + 2 * Hkv) * D, kinds[0], PTR, PTR, PTR, kinds[1], None, None, 1e-6, PTR, PTR,
               D // 2, T, D, None, 0, 0, B, T, Hq, Hkv, D, 0, None, fail=fail)


def logits(B, V, L=0, kind=0, fail=()):
    return run("adkv_process_logits", PTR, V, PTR, V, kind, PTR, PTR if L else None, L, L, None, None, 1.0, None, 0.0, None, 0.0, None, 0, None, 0, B, V,
               None, fail=fail)


def test_one_launch_each():
    for D in (64, 128, 256, 512):
        for kinds in ((0, 0), (1, 0), (1, 1), (2, 0), (2, 2)):
            rc, got = rope(3, 50, 8, 2, D, kinds)
            assert rc == 0 and names(got) == ["norm_rope"]
    for kind in (0, 1, 2):
        for L in (0, 100, 70000):
            rc, got = logits(3, 50257, L, kind)
            assert rc == 0 and names(got) == ["process_logits"]
    assert logits(3, 1000, 65535)[1][0][0] != logits(3, 1000, 65536)[1][0][0]          # counts of 16 bits while they suffice
    for call in (lambda **k: rope(1, 1, 1, 1, 64, **k), lambda **k: logits(1, 100, **k)):
        for function in ("cudaLaunchKernel", "cudaLaunchKernelExC", "cudaFuncSetAttribute"):
            rc, got = call(fail=[(function, 1)])
            assert (rc != 0) == (not got)
        assert call()[0] == 0


@pytest.mark.parametrize("B,V,ctas", [(1, 1000, 1), (1, 4096, 2), (1, 128256, 8), (64, 128256, 256), (148, 50257, 296), (149, 50257, 149), (300, 50257, 300)])
def test_ctas_of_the_logits(B, V, ctas):
    rc, got = logits(B, V)
    assert rc == 0 and got[0][1] == ctas
