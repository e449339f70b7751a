"""What the softmax weights of a shared prefix keep: many small ones beside a large one, and more bits than an fp16 number holds.

All parameters but the scales are zero, so that a value is its code times the scale and every number below is known exactly."""
import math

import pytest
import torch

from adkv_b200 import gemv
from tests.util import SMAX, SMIN

D = 128
V_SCALE = 32.0


def params(scale):
    zero = torch.zeros(1, D, dtype=torch.float16, device="cuda")
    return (zero, zero + scale, zero, zero, zero)


def step(bits, k_codes, v_codes, q, scaling, interval=0):
    """k_codes, v_codes [P]: the codes of every channel 0 (K) and of all channels (V); q [B]: channel 0 of the queries -> results [B, D].
    The new token has code 0 in K and V."""
    P, B = len(k_codes), len(q)
    k = torch.zeros(1, 1, P, D, dtype=torch.float16, device="cuda")
    k[0, 0, :, 0] = torch.tensor(k_codes, dtype=torch.float16)
    v = (torch.tensor(v_codes, dtype=torch.float16) * V_SCALE)[None, None, :, None].expand(1, 1, P, D).cuda()
    kp, vp = params(1.0), params(V_SCALE)
    cache = [torch.zeros(1, 1, gemv.n_super_for(P, bits), D // 4, 4, 4, dtype=torch.uint8, device="cuda") for _ in range(2)]
    tails = [torch.zeros(1, 1, 2, D, device="cuda") for _ in range(2)]
    ck = dict(k_ckpt=gemv.alloc_ckpt(1, 1, D, P, interval, "cuda"), v_ckpt=gemv.alloc_ckpt(1, 1, D, P, interval, "cuda"),
              ckpt_interval=interval) if interval else {}
    gemv.encode_kv_pair(cache[0], k, kp, cache[1], v, vp, SMIN, SMAX, bits=bits, k_tail=tails[0], v_tail=tails[1], **ck)
    prefix = gemv.SharedPrefix(cache[0], cache[1], P, bits=bits, k_tail=tails[0], v_tail=tails[1], **ck)
    own = [torch.zeros(B, 1, 1, D // 4, 4, 4, dtype=torch.uint8, device="cuda") for _ in range(2)]
    queries = torch.zeros(B, 1, 1, D, dtype=torch.float16, device="cuda")
    queries[:, 0, 0, 0] = q.half()
    new = torch.zeros(B, 1, 1, D, dtype=torch.float16, device="cuda")
    kt, vt = prefix.start_tails(B)
    out = gemv.decode_attn_prefix(queries, prefix, *own, new, new, kp, vp, 0, scaling, SMIN, SMAX, k_tail=kt, v_tail=vt)
    assert gemv.device_status() == 0
    return out[:, 0].double().cpu()


def softmax64(k_codes, q, scaling):
    """Weights of the prefix's tokens and of the new one, the largest 1: [B, P], [B]."""
    logits = q.half().double()[:, None] * torch.tensor(list(k_codes) + [0.0], dtype=torch.float64) * scaling
    p = (logits - logits.amax(1, keepdim=True)).exp()
    return p[:, :-1], p[:, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("interval", [0, 4096])
@pytest.mark.parametrize("large_at", [0, 9000, -1])
@pytest.mark.parametrize("bits", [4, 2])
def test_many_small_weights_beside_a_large_one(bits, large_at, interval):
    """Each of 16000 tokens weighs 2^-24 to 2^-28 of the largest.  A weight is off by 2^-32 of the largest at most (half the smallest step
    of fp16 numbers that begin at 2^7), the logits by some roundings of 28 (in powers of two)."""
    top, P = (7, 1)[bits == 2], 16000
    k, v = [0] * P, [top] * P
    k[large_at], v[large_at] = top, 0
    powers = torch.tensor([24.0, 24.7, 25.4, 26.2, 27.0, 28.0])
    scaling = math.log(2.0) / top
    got = step(bits, k, v, powers, scaling, interval)
    w, new = softmax64(k, powers, scaling)
    value = torch.tensor(v, dtype=torch.float64) * V_SCALE
    total = w.sum(1) + new
    want = (w @ value / total)[:, None]
    bound = (P * 2.0 ** -32 * value.max() / total)[:, None] + want * (28 * 8 * 2.0 ** -24 + P * 2.0 ** -24 + 2.0 ** -11) + 2.0 ** -25
    assert ((got - want).abs() <= bound).all()
    small = torch.where(w < 2.0 ** -20, (w * 2 ** 24).round() / 2 ** 24, w)            # fp16 numbers that begin at 1
    assert (((small @ value / total)[:, None] - want).abs() > bound).any()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
def test_weights_have_more_bits_than_one_fp16_number(bits):
    """Two tokens of nearly the same weight and opposite values: what is left is the weights' difference.  A weight is off by 2^-22, half a
    step of its remainder, and by the roundings of a logit below 2^-5 and of exp2 (2 in the last place); the sums' by one a product."""
    top = (7, 1)[bits == 2]
    k, v = [top, top - 1], [top, -top]
    q = torch.linspace(1.0, 9.0, 60).half().float()
    scaling = 2.0 ** -14 * 1.3
    got = step(bits, k, v, q, scaling)
    w, new = softmax64(k, q, scaling)
    value = torch.tensor(v, dtype=torch.float64) * V_SCALE
    total = w.sum(1) + new
    want = (w @ value / total)[:, None]
    off = 2.0 ** -22 + 2.0 ** -24 + 2 * 2.0 ** -23 + 4 * 2.0 ** -24
    bound = (2 * off * value.max() / total)[:, None] + want.abs() * (2.0 ** -11 + 16 * 2.0 ** -24) + 2.0 ** -25
    assert ((got - want).abs() <= bound).all()
    single = (w.half().double() @ value / total)[:, None]                                # the weights without their remainders
    assert ((single - want).abs() > 4 * bound).float().mean() > 0.5
