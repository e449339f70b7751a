"""Decode steps of sequences that share a packed prefix: against 64 bits, against whole caches, and what the calls refuse."""
import ctypes
import math

import pytest
import torch

from adkv_b200 import _lib, gemv, synth
from tests.util import SMAX, SMIN

D = 128
SCALING = D ** -0.5


class Shared:
    """A prefix of P tokens, B sequences with `lens` own tokens behind it and one step's queries and new tokens."""

    def __init__(self, bits, Hq, Hkv, P, interval, lens, seed=0, bounds=(SMIN, SMAX), room=None, k_size=1.0, dirty=True, params=None):
        B, tpw = len(lens), 32 // bits
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.bits, self.Hq, self.Hkv, self.P, self.interval, self.lens, self.bounds, self.B = bits, Hq, Hkv, P, interval, list(lens), bounds, B
        self.kp, self.vp = params or (synth.gen_params(seed + 1, Hkv, D, bits, device="cuda"), synth.gen_params(seed + 2, Hkv, D, bits, device="cuda"))
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
        mean = 2 * rand(2, Hkv, 1, D)
        T = max(lens) if lens else 0
        # keys and values as one run per sequence: prefix tokens, own tokens, the new one
        self.pre = [(k_size * (rand(1, Hkv, P, D) + mean[i])).half() for i in range(2)]
        self.own = [(k_size * (rand(B, Hkv, T, D) + mean[i])).half() for i in range(2)]
        self.new = [(k_size * (rand(B, Hkv, 1, D) + mean[i])).half() for i in range(2)]
        self.q = rand(B, Hq, 1, D).half()
        ns = max(1, gemv.n_super_for(P, bits)) + 1
        kc, vc = (torch.zeros(1, Hkv, ns, D // 4, 4, 4, dtype=torch.uint8, device="cuda") for _ in range(2))
        kt, vt = (torch.zeros(1, Hkv, 2, D, device="cuda") for _ in range(2))
        ck = dict(k_ckpt=gemv.alloc_ckpt(1, Hkv, D, P, interval, "cuda"), v_ckpt=gemv.alloc_ckpt(1, Hkv, D, P, interval, "cuda"),
                  ckpt_interval=interval) if interval else {}
        gemv.encode_kv_pair(kc, self.pre[0], self.kp, vc, self.pre[1], self.vp, *bounds, bits=bits, k_tail=kt, v_tail=vt, **ck)
        if dirty:   # what lies behind the prefix, in its last word and after it, must not matter
            for c in (kc, vc):
                words = c.view(1, Hkv, ns, D, 4).view(torch.int32).view(1, Hkv, ns, D)
                if P % tpw:
                    keep = (1 << (bits * (P % tpw))) - 1
                    words[:, :, P // tpw] = (words[:, :, P // tpw] & keep) | (0x5A5A5A5A & ~keep)
                words[:, :, gemv.n_super_for(P, bits):] = -1
        self.prefix = gemv.SharedPrefix(kc, vc, P, bits=bits, k_tail=kt, v_tail=vt, **ck)
        self.ck = ck
        self.cap = room or gemv.n_super_for(T + 1, bits)
        self.kc, self.vc = (torch.full((B, Hkv, self.cap, D // 4, 4, 4), 0xC3, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.kt, self.vt = self.prefix.start_tails(B)
        for b, n in enumerate(lens):
            gemv.encode_kv_pair(self.kc[b:b + 1], self.own[0][b:b + 1, :, :n], self.kp, self.vc[b:b + 1], self.own[1][b:b + 1, :, :n], self.vp,
                                *bounds, bits=bits, k_tail=self.kt[b:b + 1], v_tail=self.vt[b:b + 1], from_tail=True)
        self.lens_gpu = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def step(self, T=None, scaling=SCALING, **kw):
        T = self.lens_gpu if T is None else T
        kw = {**dict(k_tail=self.kt, v_tail=self.vt), **kw}
        return gemv.decode_attn_prefix(self.q, self.prefix, self.kc, self.vc, *self.new, self.kp, self.vp, T, scaling, *self.bounds, **kw)

    # ------------------------------------------------------------------ 64 bits, on the CPU
    def _codes(self, cache, n):
        B, H, ns = cache.shape[:3]
        words = cache.cpu().contiguous().view(B, H, ns, D, 4).view(torch.int32).view(B, H, ns, 1, D).long()
        shift = torch.arange(32 // self.bits)[:, None] * self.bits
        return (((words >> shift) & ((1 << self.bits) - 1)) - (1 << (self.bits - 1))).reshape(B, H, -1, D)[:, :, :n].double()

    def _replay(self, codes, zp, s, p):
        """codes [..., T, D] -> values, and the zero points before each token."""
        alpha, beta, target = (t.double().cpu() for t in p[2:])
        x, z = [], []
        for t in range(codes.shape[-2]):
            c = codes[..., t, :]
            r = c * s.clamp(min=1e-8)
            x.append(r + zp)
            z.append(zp)
            zp = zp + alpha * r
            s = (s * (1 + beta * (c.abs() - target))).clamp(min=self.bounds[0]).clamp(max=self.bounds[1])
        shape = codes.shape[:-2] + (0, D)
        return (torch.stack(x, -2), torch.stack(z, -2)) if x else (torch.zeros(shape).double(), torch.zeros(shape).double())

    def values(self):
        """K and V: prefix values and zero points at the start of their checkpoint interval [Hkv, P, D]; own values [B, Hkv, T, D]; new
        values [B, Hkv, D] (codes of the new token in 32 bits, as the definition has them)."""
        out = []
        I = self.interval or max(self.P, 1)
        for i, p in enumerate((self.kp, self.vp)):
            cache = self.prefix._keep[i]
            codes = self._codes(cache, self.P)[0]
            ck = self.prefix._keep[2 + i]
            parts, starts = [], []
            for j in range(0, self.P, I):
                if j == 0:
                    zp, s = (t.double().cpu() for t in p[:2])
                else:
                    zp, s = ck[0, :, j // I - 1].double().cpu().unbind(1)
                x, z = self._replay(codes[:, j:j + I], zp, s, p)
                parts.append(x)
                starts.append(zp[:, None].expand(x.shape))
            pre = torch.cat(parts, 1) if parts else torch.zeros(self.Hkv, 0, D).double()
            start = torch.cat(starts, 1) if parts else pre
            tail = (self.prefix.k_tail, self.prefix.v_tail)[i].double().cpu().expand(self.B, -1, -1, -1)
            own, _ = self._replay(self._codes((self.kc, self.vc)[i], max(self.lens)), tail[:, :, 0], tail[:, :, 1], p)
            zp, s = ((self.kt, self.vt)[i].cpu()).unbind(2)
            code = torch.round((self.new[i][:, :, 0].float().cpu() - zp) / s.clamp(min=1e-8)).clamp(-(1 << (self.bits - 1)), (1 << (self.bits - 1)) - 1)
            out.append((pre, start, own, zp.double() + code.double() * s.double().clamp(min=1e-8)))
        return out

    def want(self, scaling=SCALING):
        """Result in float64, and a bound of what the operands of the products and fp32 sums may add to it.

        Values of the prefix are pairs of fp16 numbers, as differences from the zero point at the start of a run: off by at most half a step of
        the remainder, 2^-22 of the difference, or 2^-21 (half the smallest fp16 step in units of 16).  Runs may span intervals, so differences
        count from any interval's start.  Replays in 32 bits are off by at most 8 roundings of the largest value a token.  A weight is off by
        half a step of fp16, 2^-11; as the denominator adds up the rounded weights, that moves the result by no more than twice that of the
        values' mean distance from it.  The result itself is rounded by half a step."""
        (kp, kz, ko, kn), (vp, vz, vo, vn) = self.values()
        G = self.Hq // self.Hkv
        q = self.q.double().cpu().view(self.B, self.Hkv, G, D)
        out, bound = torch.zeros(self.B, self.Hkv, G, D).double(), torch.zeros(self.B, self.Hkv, G, D).double()

        def far(x, z):   # largest difference of a value from a zero point where a run may have started
            if not x.shape[1]:
                return x
            lo, hi = z.amin(1, keepdim=True), z.amax(1, keepdim=True)
            return torch.maximum((x - lo).abs(), (x - hi).abs())

        kd, vd = far(kp, kz), far(vp, vz)
        steps = (self.interval or self.P) + 600
        drift = 8 * steps * 2.0 ** -24
        for b, n in enumerate(self.lens):
            k = torch.cat([kp, ko[b, :, :n], kn[b, :, None]], 1)
            v = torch.cat([vp, vo[b, :, :n], vn[b, :, None]], 1)
            logits = torch.einsum("hgd,htd->hgt", q[b], k) * scaling
            p = torch.softmax(logits, -1)
            o = p @ v
            # a logit: the values' roundings, sums of D products in 32 bits (towards zero on the tensor cores), replay
            off = torch.zeros_like(k)
            off[:, :self.P] = torch.maximum(kd * 2.0 ** -22, torch.full_like(kd, 2.0 ** -21))
            off = off + (D * 2.0 ** -23 + drift) * k.abs().amax(1, keepdim=True)
            e = abs(scaling) * torch.einsum("hgd,htd->hgt", q[b].abs(), off).amax(-1, keepdim=True)
            away = torch.einsum("hgt,hgtd->hgd", p, (v[:, None] - o[:, :, None]).abs())
            voff = torch.zeros_like(v)
            voff[:, :self.P] = torch.maximum(vd * 2.0 ** -22, torch.full_like(vd, 2.0 ** -21))
            out[b] = o
            bound[b] = (torch.expm1(2 * e) + 2 * 2.0 ** -11) * away + p @ voff + (k.shape[1] * 2.0 ** -23 + drift) * v.abs().amax(1)[:, None] + \
                o.abs() * 2.0 ** -11 + 2.0 ** -25
        return out.view(self.B, self.Hq, D), bound.view(self.B, self.Hq, D)

    def check(self, got, want):
        o, bound = want
        err = (got.double().cpu() - o).abs()
        assert (err <= bound).all(), f"{(err / bound).max():.2f} of the bound"


CASES = [  # bits, Hq, Hkv, P, interval, own tokens
    (4, 2, 2, 1, 32, [0]),
    (4, 1, 1, 7, 0, [3, 0]),
    (2, 4, 2, 17, 32, [0, 20, 1]),
    (4, 8, 8, 64, 64, [5] * 2),
    (4, 4, 4, 65, 32, [70, 0, 33]),
    (2, 8, 1, 300, 128, [9, 130, 0, 64]),
    (4, 8, 2, 777, 96, [0] * 33),                        # 132 rows: two row tiles
    (4, 16, 2, 1000, 64, [1, 2, 3, 200] * 10),           # 320 rows
    (2, 2, 1, 2049, 256, [31, 0]),
    (4, 3, 3, 1500, 0, [12]),                            # no checkpoints: one run
    (4, 32, 32, 600, 128, [40, 100]),
    (4, 2, 1, 0, 64, [0, 10, 65]),                       # no prefix
]


@pytest.mark.gpu
@pytest.mark.parametrize("bits,Hq,Hkv,P,interval,lens", CASES)
def test_against_64_bits(bits, Hq, Hkv, P, interval, lens):
    c = Shared(bits, Hq, Hkv, P, interval, lens, seed=P)
    want = c.want()
    c.check(c.step(tail_keep=True), want)
    assert gemv.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [0.0, -0.3, 1.0])
def test_scaling_of_any_sign(scaling):
    c = Shared(4, 4, 2, 333, 64, [3, 50], seed=5)
    c.check(c.step(tail_keep=True, scaling=scaling), c.want(scaling))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("bounds,k_size", [((0.0, 0.4), 1.0), ((0.3, 0.3), 1.0), ((0.5, 0.1), 1.0), ((0.0, math.inf), 1e-3), ((SMIN, SMAX), 300.0),
                                           ((1.0, 8.0), 1.0), ((0.0, math.inf), 1500.0)])
def test_scales_at_their_bounds_and_values_of_any_size(bits, bounds, k_size):
    """Bounds that every scale meets, no lower bound, none at all; small and large values."""
    c = Shared(bits, 4, 2, 500, 96, [0, 77], seed=11, bounds=bounds, k_size=k_size)
    scaling = SCALING / k_size
    c.check(c.step(tail_keep=True, scaling=scaling), c.want(scaling))


@pytest.mark.gpu
def test_scale_that_starts_at_zero():
    """Zero initial scales: the quantiser's guard acts until the lower bound does."""
    kp, vp = ([t.clone() for t in synth.gen_params(i, 2, D, 4, device="cuda")] for i in (1, 2))
    kp[1].zero_()
    vp[1][:, ::3] = 0
    c = Shared(4, 2, 2, 200, 64, [0, 9], seed=3, params=(kp, vp))
    c.check(c.step(tail_keep=True), c.want())


@pytest.mark.gpu
@pytest.mark.parametrize("bits,G", [(4, 1), (4, 8), (2, 2), (2, 4)])
def test_codes_tails_and_result_are_those_of_whole_caches(bits, G):
    """A cache per sequence that holds prefix and own tokens in one piece gives the same codes, tails and, nearly, results."""
    lens = [0, 5, 64, 31]
    c = Shared(bits, 2 * G, 2, 413, 64, lens, seed=9)
    cap = gemv.n_super_for(c.P + max(lens) + 1, bits)
    kc, vc = (torch.zeros(c.B, 2, cap, D // 4, 4, 4, dtype=torch.uint8, device="cuda") for _ in range(2))
    kt, vt = (torch.zeros(c.B, 2, 2, D, device="cuda") for _ in range(2))
    for b, n in enumerate(lens):
        x = [torch.cat([c.pre[i], c.own[i][b:b + 1, :, :n]], 2) for i in range(2)]
        gemv.encode_kv_pair(kc[b:b + 1], x[0], c.kp, vc[b:b + 1], x[1], c.vp, *c.bounds, bits=bits, k_tail=kt[b:b + 1], v_tail=vt[b:b + 1])
    assert torch.equal(kt, c.kt) and torch.equal(vt, c.vt)
    whole_lens = c.lens_gpu + c.P
    bound = c.want()[1]
    for step in range(3):      # the tails advance, the caches grow
        got = c.step()
        want = gemv.decode_attn_varlen(c.q, kc, vc, *c.new, c.kp, c.vp, whole_lens, SCALING, *c.bounds, bits=bits, k_tail=kt, v_tail=vt)
        assert torch.equal(kt, c.kt) and torch.equal(vt, c.vt)
        if step == 0:
            assert ((got.double() - want.double()).abs().cpu() <= 2 * bound).all()
        for i in range(2):
            mine, all_ = c._codes((c.kc, c.vc)[i], 10 ** 9), c._codes((kc, vc)[i], 10 ** 9)
            for b, n in enumerate(lens):
                assert torch.equal(mine[b, :, :n + step + 1], all_[b, :, c.P:c.P + n + step + 1])
        if max(lens) + step + 2 > c.cap * (32 // bits):
            break
        c.lens_gpu += 1
        whole_lens += 1


@pytest.mark.gpu
def test_int_length_tail_keep_out_and_scratch():
    c = Shared(4, 8, 4, 300, 64, [37] * 3, seed=2)
    tails = c.kt.clone(), c.vt.clone()
    out = torch.empty(3, 8, D, dtype=torch.float16, device="cuda")
    scratch = torch.full((gemv.prefix_scratch_bytes(3, 8, c.prefix),), 0xFF, dtype=torch.uint8, device="cuda")
    a = c.step(T=37, tail_keep=True, out=out, scratch=scratch)
    assert a is out and torch.equal(c.kt, tails[0]) and torch.equal(c.vt, tails[1])
    codes = c.kc.clone(), c.vc.clone()
    b = c.step(tail_keep=True)                              # device lengths, own scratch: the same step again
    assert torch.equal(a, b) and torch.equal(c.kc, codes[0]) and torch.equal(c.vc, codes[1])
    c.step()
    kt, vt = c.kt.clone(), c.vt.clone()
    c.kt.copy_(tails[0])
    c.vt.copy_(tails[1])
    gemv.append_kv_pair(c.kc, c.new[0], c.kp, c.kt, c.vc, c.new[1], c.vp, c.vt, 37, *c.bounds)
    assert torch.equal(c.kt, kt) and torch.equal(c.vt, vt) and torch.equal(c.kc, codes[0]) and torch.equal(c.vc, codes[1])


@pytest.mark.gpu
def test_captured_steps_on_side_streams_with_growing_lengths():
    c = Shared(4, 4, 2, 260, 64, [0, 3, 20], seed=4, room=8)
    d = Shared(2, 4, 4, 700, 128, [1, 0], seed=6, room=4)
    scratch = [torch.empty(gemv.prefix_scratch_bytes(x.B, x.Hq, x.prefix), dtype=torch.uint8, device="cuda") for x in (c, d)]
    want = []
    for x in (c, d):
        save = [t.clone() for t in (x.kc, x.vc, x.kt, x.vt, x.lens_gpu)]
        rows = []
        for _ in range(4):
            rows.append(x.step())
            x.lens_gpu += 1
        want.append((rows, [t.clone() for t in (x.kc, x.vc, x.kt, x.vt)]))
        for t, s in zip((x.kc, x.vc, x.kt, x.vt, x.lens_gpu), save):
            t.copy_(s)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for x, s in zip((c, d), scratch):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(x.step(scratch=s))
            x.lens_gpu += 1
        graphs.append(graph)
    torch.cuda.synchronize()
    for n in range(4):
        for graph, stream in zip(graphs, streams):          # both at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i][0][n])
    for x, (_, state) in zip((c, d), want):
        for t, s in zip((x.kc, x.vc, x.kt, x.vt), state):
            assert torch.equal(t, s)
    assert gemv.device_status() == 0


@pytest.mark.gpu
def test_length_that_does_not_fit_leaves_its_sequence_out():
    c = Shared(4, 4, 2, 100, 64, [3, 5, 2], seed=8)
    assert gemv.device_status() == 0
    before = c.kc.clone(), c.kt.clone()
    c.lens_gpu.copy_(torch.tensor([3, c.cap * 8, -1]))
    got = c.step()
    assert gemv.device_status() == 6 and gemv.device_status() == 0
    assert torch.isnan(got[1:]).all() and torch.isfinite(got[0]).all()
    assert torch.equal(c.kc[1:], before[0][1:]) and torch.equal(c.kt[1:], before[1][1:]) and not torch.equal(c.kt[0], before[1][0])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
def test_prefill_from_a_tail_is_the_next_chunk(bits):
    """Codes quantised from a tail at index 0 are those of the chunk that follows in one cache, in pieces of any size."""
    kp, vp = (synth.gen_params(i, 3, D, bits, device="cuda") for i in (1, 2))
    x = [torch.randn(2, 3, 200, D, device="cuda").half() for _ in range(2)]
    whole, parts = [], []
    for target in (whole, parts):
        for _ in range(2):
            target.append(torch.zeros(2, 3, gemv.n_super_for(200, bits), D // 4, 4, 4, dtype=torch.uint8, device="cuda"))
        for _ in range(2):
            target.append(torch.zeros(2, 3, 2, D, device="cuda"))
    tpw, first = 32 // bits, 64
    def enc(t, lo, hi, **kw):
        gemv.encode_kv_pair(t[0], x[0][:, :, lo:hi], kp, t[1], x[1][:, :, lo:hi], vp, SMIN, SMAX, bits=bits, k_tail=t[2], v_tail=t[3], **kw)
    enc(whole, 0, first)
    for i in (2, 3):
        parts[i].copy_(whole[i])
    enc(whole, first, 200, t_start=first)
    enc(parts, first, first, from_tail=True)                 # nothing: nothing happens
    enc(parts, first, first + 21, from_tail=True)
    enc(parts, first + 21, 200, t_start=21, from_tail=True)
    n = gemv.n_super_for(200 - first, bits)
    for i in range(2):
        assert torch.equal(parts[i][:, :, :n], whole[i][:, :, first // tpw:first // tpw + n]) and torch.equal(parts[2 + i], whole[2 + i])


@pytest.mark.gpu
def test_refusals():
    c = Shared(4, 4, 2, 100, 64, [3, 5], seed=1)
    with pytest.raises(RuntimeError, match="tail"):
        c.step(k_tail=None)
    with pytest.raises(RuntimeError, match="T must be"):
        c.step(T=c.lens_gpu.long())
    with pytest.raises(RuntimeError, match="T must be"):
        c.step(T=c.lens_gpu[:1])
    with pytest.raises(RuntimeError, match="non-negative"):
        c.step(T=-1)
    with pytest.raises(RuntimeError, match="no free"):
        c.step(T=8 * c.cap)
    with pytest.raises(RuntimeError, match="scratch"):
        c.step(scratch=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="out must"):
        c.step(out=torch.empty(2, 4, D, device="cuda"))
    other = Shared(4, 4, 4, 100, 64, [3, 5], seed=1)
    with pytest.raises(RuntimeError, match="match the prefix"):
        gemv.decode_attn_prefix(c.q, other.prefix, c.kc, c.vc, *c.new, c.kp, c.vp, 3, SCALING, SMIN, SMAX, k_tail=c.kt, v_tail=c.vt)
    kc, vc, kck, vck = c.prefix._keep
    make = lambda **kw: gemv.SharedPrefix(**{**dict(k_cache=kc, v_cache=vc, tokens=100, k_tail=c.prefix.k_tail, v_tail=c.prefix.v_tail, k_ckpt=kck,
                                                     v_ckpt=vck, ckpt_interval=64), **kw})
    for kw, text in [(dict(tokens=1000), "hold"), (dict(tokens=-1), "hold"), (dict(ckpt_interval=48), "multiple of 32"), (dict(bits=3), "bits"),
                     (dict(k_cache=c.kc, v_cache=c.vc), "one sequence"), (dict(k_tail=None), "tail"), (dict(k_ckpt=None), "checkpoint"),
                     (dict(k_ckpt=kck[:, :, :0], v_ckpt=vck[:, :, :0]), "reach"), (dict(v_tail=c.vt), "tail"), (dict(v_cache=vc[:, :, :1]), "match")]:
        with pytest.raises(RuntimeError, match=text):
            make(**kw)
    empty = gemv.decode_attn_prefix(c.q[:0], c.prefix, c.kc[:0], c.vc[:0], c.new[0][:0], c.new[1][:0], c.kp, c.vp, 0, SCALING, SMIN, SMAX,
                                    k_tail=c.kt[:0], v_tail=c.vt[:0])
    assert empty.shape == (0, 4, D)


def test_argument_errors_of_the_c_abi():
    """Checked on the host, before anything is launched."""
    lib = _lib.load()
    params = _lib.Params(16, 16, 16, 16, 16)
    pp = ctypes.addressof(params)

    def call(q=16, pre=True, kt=16, lens=None, T=0, scratch=16, room=1 << 40, B=1, Hq=2, Hkv=2, D=128, ns=1, bits=4, flags=0, **fields):
        desc = _lib.Prefix(16, 16, 16, 16, 16, 16, 100, 13, 64, 1)
        for name, value in fields.items():
            setattr(desc, name, value)
        return lib.adkv_decode_attn_prefix(q, ctypes.addressof(desc) if pre else None, 16, 16, 16, 16, pp, pp, kt, 16, lens, T, 16, scratch, room, B, Hq,
                                           Hkv, D, ns, bits, 0.1, 0.1, 1.0, flags, None)
    assert call(q=None) == call(pre=False) == call(kt=None) == call(scratch=None) == call(k_cache=None) == call(v_tail=None) == call(k_ckpt=None) == -1
    assert call(D=256) == -2
    assert call(bits=3) == -3
    assert call(Hq=3) == call(Hq=6) == call(T=-1) == call(tokens=-1) == call(interval=48) == call(interval=-32) == call(B=-1) == -4
    assert call(T=8) == call(n_super_cap=12) == call(n_ckpt_cap=0) == call(ns=0, lens=16) == -5
    assert call(q=20) == call(kt=24) == call(lens=18) == call(k_cache=24) == call(v_ckpt=24) == -6
    assert call(room=16) == -8
    assert call(flags=_lib.FLAG_HALF_STATE) == call(flags=_lib.FLAG_SPLIT_CHANNELS) == -10
    assert call(B=0) == 0
    assert lib.adkv_decode_attn_prefix_scratch_bytes(1, 3, 2, 10, 0) == -4
    assert lib.adkv_decode_attn_prefix_scratch_bytes(2, 4, 2, 0, 0) == 2 * 4 * 132 * 4
    enc = lambda tail, flags, T=8, t_start=0: lib.adkv_encode_kv_flags(16, 16, pp, tail, None, None, None, None, None, None, 0, 0, 1, 1, T, 128, 1, 4, t_start,
                                                                       0.1, 1.0, flags, None)
    assert enc(None, _lib.FLAG_TAIL_START) == -7
    assert enc(16, _lib.FLAG_TAIL_START | _lib.FLAG_HALF_STATE) == -10
    assert enc(16, _lib.FLAG_TAIL_START, T=9) == -5
    assert enc(16, _lib.FLAG_TAIL_START, t_start=-1) == -4
    assert enc(16, _lib.FLAG_TAIL_START, T=0) == 0
