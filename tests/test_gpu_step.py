"""Rotation of projected heads and processing of logits against their definitions in 64 bits, and what the calls refuse."""
import ctypes
import math

import pytest
import torch

from adkv_b200 import _lib, e2e_llama, gemv, step

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


# ---------------------------------------------------------------------------------- rotation

def rope_inputs(B, T, Hq, Hkv, D, rot, dtype, rows=300, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").to(dtype)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    weights = (1 + 0.3 * torch.randn(2, D, generator=g, device="cuda")).to(dtype)
    return qkv, ang.cos().float().cuda(), ang.sin().float().cuda(), weights[0].clone(), weights[1].clone()


def rope_want(qkv, Hq, Hkv, cos, sin, pos, wq, wk, eps, interleaved):
    """(value, bound of what fp32 arithmetic may add to the rounding) of q, k, v in float64 on the CPU."""
    B, T, _ = qkv.shape
    H = Hq + 2 * Hkv
    x = qkv.double().cpu().reshape(B, T, H, -1).transpose(1, 2)
    D, rot = x.shape[-1], 2 * cos.shape[1]
    c, s = cos.double().cpu()[pos], sin.double().cpu()[pos]            # [B, T, rot / 2]
    c, s = c[:, None], s[:, None]
    out = []
    for part, w in ((x[:, :Hq], wq), (x[:, Hq:Hq + Hkv], wk)):
        y = part.clone()
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double().cpu()
        i = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
        j = i + 1 if interleaved else i + rot // 2
        z = y.clone()
        z[..., i], z[..., j] = y[..., i] * c - y[..., j] * s, y[..., j] * c + y[..., i] * s
        # sum of D squares, root, three products in front of the rotation, two products and a sum in it
        size = y.abs()
        size[..., i] = size[..., j] = y[..., i].abs() + y[..., j].abs()
        out.append((z, size * (D / 2 + 8 if w is not None else 3) * 2.0 ** -24))
    return out + [(x[:, Hq + Hkv:], 0.0)]


def rope_check(got, want, dtype):
    for g, (w, arithmetic) in zip(got, want):
        assert g.is_contiguous() and g.dtype == dtype and tuple(g.shape) == tuple(w.shape)
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0           # half a step of fp16's smallest numbers
        bound = (w.abs() + arithmetic) * HALF_STEP[dtype] + arithmetic + tiny
        assert ((g.double().cpu() - w).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,rot", [(1, 1, 1, 1, 64, 64), (3, 1, 32, 8, 128, 128), (2, 37, 5, 5, 128, 64), (1, 130, 8, 1, 256, 256),
                                              (2, 3, 7, 2, 512, 512), (1, 5, 33, 3, 64, 8), (2, 2, 64, 8, 512, 72), (128, 1, 4, 4, 128, 128)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_against_64_bits(B, T, Hq, Hkv, D, rot, interleaved, norm):
    for n, (dtype, out) in enumerate([(torch.float16, torch.float16), (torch.bfloat16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                      (torch.float32, torch.float32), (torch.float32, torch.float16)]):
        qkv, cos, sin, wq, wk = rope_inputs(B, T, Hq, Hkv, D, rot, dtype, seed=n)
        wq, wk = (wq, wk) if norm else (None, None)
        got = step.norm_rope_qkv(qkv, Hq, Hkv, cos, sin, start=7, q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved, dtype=out)
        pos = (7 + torch.arange(T)).expand(B, T)
        rope_check(got, rope_want(qkv, Hq, Hkv, cos, sin, pos, wq, wk, 1e-5, interleaved), out)
    assert gemv.device_status() == 0


@pytest.mark.gpu
def test_rotation_positions_strides_and_one_weight():
    B, T, Hq, Hkv, D = 3, 11, 6, 2, 128
    qkv, cos, sin, wq, _ = rope_inputs(B, T, Hq, Hkv, D, 128, torch.bfloat16)
    first = torch.tensor([0, 250, 31], dtype=torch.int32, device="cuda")
    each = torch.randint(0, 300, (B, T), dtype=torch.int32, device="cuda")
    for positions, pos in ((first, first.cpu().long()[:, None] + torch.arange(T)), (each, each.cpu().long())):
        got = step.norm_rope_qkv(qkv, Hq, Hkv, cos, sin, positions=positions, q_weight=wq)       # keys are not normalised
        rope_check(got, rope_want(qkv, Hq, Hkv, cos, sin, pos, wq, None, 1e-6, False), torch.bfloat16)
    # tables of twice the width, as the harness keeps them; rows of a wider buffer; rows that are not aligned; a transposed view
    twice = [torch.cat([t, t], -1) for t in (cos, sin)]
    pos = torch.arange(T).expand(B, T)
    want = rope_want(qkv, Hq, Hkv, cos, sin, pos, None, None, 1e-6, False)
    wide = torch.zeros(B, T + 2, qkv.shape[2] + 8, dtype=qkv.dtype, device="cuda")
    wide[:, 1:T + 1, 4:-4] = qkv
    odd = torch.zeros(qkv.numel() + 1, dtype=qkv.dtype, device="cuda")[1:].view_as(qkv)
    odd.copy_(qkv)
    turned = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    strange = qkv.transpose(1, 2).contiguous().transpose(1, 2)
    for view in (qkv, wide[:, 1:T + 1, 4:-4], odd, turned, strange):
        rope_check(step.norm_rope_qkv(view, Hq, Hkv, twice[0][:, :64], twice[1][:, :64]), want, torch.bfloat16)


@pytest.mark.gpu
def test_rotation_is_the_harness_expression_bit_for_bit():
    shape = e2e_llama.LlamaShape(n_heads=4, n_kv_heads=2, head_dim=128)
    cos, sin = e2e_llama._rope_tables(shape, 100, "cuda")
    qkv = torch.randn(2, 9, 8 * 128, device="cuda").half()
    q, k, v = step.norm_rope_qkv(qkv, 4, 2, cos[:, :64], sin[:, :64], start=50)
    x = qkv.view(2, 9, 8, 128).transpose(1, 2)
    assert torch.equal(q, e2e_llama._apply_rope(x[:, :4], cos[50:59], sin[50:59]))
    assert torch.equal(k, e2e_llama._apply_rope(x[:, 4:6], cos[50:59], sin[50:59]))
    assert torch.equal(v, x[:, 6:])


@pytest.mark.gpu
def test_rotation_position_without_a_row_marks_its_token_only():
    qkv, cos, sin, _, _ = rope_inputs(3, 2, 2, 1, 64, 32, torch.float16, rows=10)
    assert gemv.device_status() == 0
    pos = torch.tensor([[3, 4], [9, 10], [-1, 0]], dtype=torch.int32, device="cuda")
    q, k, v = step.norm_rope_qkv(qkv, 2, 1, cos, sin, positions=pos)
    assert gemv.device_status() == 8 and gemv.device_status() == 0
    bad = torch.tensor([[False, False], [False, True], [True, False]])
    for t in (q, k):
        assert torch.equal(torch.isnan(t).all(-1).all(1).cpu(), bad) and torch.equal(torch.isnan(t).any(-1).any(1).cpu(), bad)
    assert torch.equal(v, qkv.view(3, 2, 4, 64)[:, :, 3:].transpose(1, 2))
    for B, T in ((0, 4), (2, 0)):
        empty = step.norm_rope_qkv(qkv.new_empty(B, T, 256), 2, 1, cos, sin)
        assert [tuple(t.shape) for t in empty] == [(B, 2, T, 64), (B, 1, T, 64), (B, 1, T, 64)]


# ---------------------------------------------------------------------------------- logits

def logits_inputs(B, V, L, dtype, seed=0, bias="row", mask=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (4 * torch.randn(B, V, generator=g, device="cuda")).to(dtype)
    kw = dict(history=torch.randint(0, max(1, min(V, 2 * L)), (B, L), generator=g, device="cuda", dtype=torch.int32),
              history_lens=torch.randint(0, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32),
              repetition=1 + torch.rand(B, generator=g, device="cuda"), presence=torch.rand(B, generator=g, device="cuda"),
              frequency=0.3 * torch.rand(B, generator=g, device="cuda"))
    if bias:
        kw["bias"] = torch.randn(*((B, V) if bias == "all" else (V,)), generator=g, device="cuda")
    if mask:
        kw["mask"] = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, device="cuda").int()
    return x, kw


def logits_want(x, history=None, history_lens=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, mask=None):
    """Value in float64 and the size that fp32 arithmetic rounds, on the CPU."""
    B, V = x.shape
    y = x.double().cpu()
    each = lambda p: p.double().cpu() if isinstance(p, torch.Tensor) else torch.full((B,), float(torch.tensor(p, dtype=torch.float32)), dtype=torch.float64)
    rep, pres, freq = each(repetition), each(presence), each(frequency)
    size = y.abs().nan_to_num(0, 0, 0)
    for b in range(B if history is not None else 0):
        row = history[b].cpu().long()
        row = row[:max(0, min(len(row), int(history_lens[b])))] if history_lens is not None else row
        row = row[(row >= 0) & (row < V)]
        n = torch.bincount(row, minlength=V).double()
        z = torch.where(y[b] > 0, y[b] / rep[b], y[b] * rep[b]) - (freq[b] * n + pres[b])
        size[b] = torch.where(n > 0, size[b] * max(rep[b], 1 / rep[b]) + 2 * (freq[b] * n + pres[b]).abs(), size[b])
        y[b] = torch.where(n > 0, z, y[b])
    if bias is not None:
        y, size = y + bias.double().cpu(), size + bias.double().cpu().abs()
    if mask is not None:
        v = torch.arange(V)
        y = torch.where((mask.cpu().long()[:, v >> 5] >> (v & 31)) & 1 == 1, y, -math.inf)
    return y, size


def logits_check(x, got, kw):
    out, tokens = got
    want, size = logits_want(x, **kw)
    o = out.double().cpu()
    finite = want.isfinite()
    arithmetic = 4 * 2.0 ** -24 * size                 # at most four roundings, each of at most this size
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    bound = (want.abs() + arithmetic) * (HALF_STEP[x.dtype] if x.dtype != torch.float32 else 0) + arithmetic + tiny
    assert ((o - want).abs()[finite] <= bound[finite]).all()
    assert torch.equal(o[~finite].nan_to_num(1e300), want[~finite].nan_to_num(1e300))
    for b in range(x.shape[0]):
        row = o[b]
        nan = row.isnan().nonzero()
        choice = int(nan[0]) if len(nan) else -1 if row.max() == -math.inf else int((row == row.max()).nonzero()[0])
        assert int(tokens[b]) == choice
    assert tokens.dtype == torch.int32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (2, 7, 5), (3, 31, 40), (1, 32, 0), (4, 1000, 300), (2, 4097, 17), (1, 32000, 100), (5, 50257, 2000),
                                   (2, 151937, 5000), (300, 501, 33)])
def test_logits_against_64_bits(B, V, L, dtype):
    for n, (bias, mask) in enumerate([("row", True), ("all", False), (None, True), (None, False)]):
        x, kw = logits_inputs(B, V, L, dtype, seed=n, bias=bias, mask=mask)
        logits_check(x, step.process_logits(x, **kw), kw)


@pytest.mark.gpu
def test_logits_numbers_for_all_rows_and_rows_apart():
    x, kw = logits_inputs(3, 777, 50, torch.float16)
    kw.update(repetition=1.3, presence=0.25, frequency=0.5, history_lens=None)
    kw.pop("history_lens")
    logits_check(x, step.process_logits(x, **kw), kw)
    # no history: the penalties do not matter; nothing at all: a copy and the largest
    plain = dict(repetition=2.0, presence=1.0)
    logits_check(x, step.process_logits(x, **plain), plain)
    # rows of a wider buffer, at any alignment, in and out
    for skew in range(0, 9):
        wide = torch.zeros(3, 800, dtype=torch.float16, device="cuda")
        view = wide[:, skew:skew + 777]
        view.copy_(x)
        target = torch.full((3, 801), 5.0, dtype=torch.float16, device="cuda")
        into = target[:, 3:780]
        logits_check(x, step.process_logits(view, out=into, **kw), kw)
        assert (target[:, :3] == 5).all() and (target[:, 780:] == 5).all()          # what lies around is left alone
    before = x.clone()
    out, tokens = step.process_logits(x, out=x, **kw)                               # in place
    assert out is x
    logits_check(before, (x, tokens), kw)


@pytest.mark.gpu
def test_logits_rows_without_a_token_ties_and_values_that_are_no_numbers():
    x = torch.zeros(6, 70, device="cuda")
    x[0, 40] = x[0, 41] = 3.0                                                       # a tie
    x[1] = -math.inf
    x[2, 69] = math.nan
    x[3] = 1.0
    x[4, 10] = math.nan                                                             # masked away
    x[5] = -0.0
    x[5, 50] = 0.0                                                                  # no larger than -0
    mask = torch.full((6, 3), -1, dtype=torch.int32, device="cuda")
    mask[3] = 0
    mask[4, 0] = ~(1 << 10)
    kw = dict(mask=mask)
    out, tokens = step.process_logits(x, **kw)
    logits_check(x, (out, tokens), kw)
    assert tokens.tolist() == [40, -1, 69, -1, 0, 0]
    # ids that are no tokens, lengths beyond the history or below zero
    history = torch.tensor([[-1, 70, 5, 5], [5, 5, 5, 5], [1, 2, 3, 4]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([9, -3, 2], dtype=torch.int32, device="cuda")
    y = torch.ones(3, 70, device="cuda")
    out, _ = step.process_logits(y, history=history, history_lens=lens, frequency=0.25)
    want = y.clone()
    want[0, 5] = 0.5
    want[2, 1] = want[2, 2] = 0.75
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_logits_captured_with_device_lengths():
    x, kw = logits_inputs(4, 5000, 64, torch.bfloat16)
    kw["history_lens"].fill_(3)
    step.process_logits(x, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step.process_logits(x, **kw)
    kw["history_lens"].copy_(torch.tensor([0, 64, 10, 1]))
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    logits_check(x, got, kw)


# ---------------------------------------------------------------------------------- refusals (no GPU needed)

def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        step.norm_rope_qkv(torch.zeros(1, 1, 384), 1, 1, torch.zeros(4, 64), torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        step.process_logits(torch.zeros(1, 8))


def test_argument_errors_of_the_c_abi():
    lib = _lib.load()

    def rope(qkv=16, sb=4, st=4, it=0, ot=0, cos=16, rows=8, rot=64, pos=None, start=0, B=1, T=1, Hq=1, Hkv=1, D=64):
        return lib.adkv_norm_rope_qkv(qkv, sb, st, it, 16, 16, 16, ot, None, None, 1e-6, cos, 16, rot // 2, rows, rot, pos, 0, start, B, T, Hq, Hkv, D,
                                      0, None)
    assert rope(qkv=None) == rope(cos=None) == -1
    assert rope(D=96) == -2
    assert rope(B=-1) == rope(rot=60) == rope(rot=128) == rope(rot=0) == rope(Hq=0) == rope(Hkv=0) == rope(st=3) == rope(start=-1) == -4
    assert rope(start=8) == rope(T=9) == -5
    assert rope(qkv=20) == rope(it=2, ot=2, qkv=24) == rope(cos=18) == -6
    assert rope(it=0, ot=1) == rope(it=3) == rope(it=1, ot=2) == -11
    assert rope(B=0) == rope(T=0) == 0

    def logits(x=16, out=16, kind=0, B=1, V=8, cap=0, history=None):
        return lib.adkv_process_logits(x, V, out, V, kind, 16, history, cap, cap, None, None, 1.0, None, 0.0, None, 0.0, None, 0, None, 0, B, V, None)
    assert logits(x=None) == logits(out=None) == -1
    assert logits(V=0) == logits(B=-1) == logits(B=65536) == logits(cap=-1) == -4
    assert logits(kind=3) == -11
    assert logits(x=17) == logits(kind=2, x=18) == logits(history=18, cap=4) == -6
    assert logits(B=0) == 0
    assert _lib.strerror(-11).startswith("adkv:")


@pytest.mark.gpu
def test_refusals():
    qkv, cos, sin, wq, wk = rope_inputs(2, 3, 2, 1, 64, 64, torch.float16)
    call = lambda **kw: step.norm_rope_qkv(**{**dict(qkv=qkv, n_heads=2, n_kv_heads=1, cos=cos, sin=sin), **kw})
    for kw, text in [(dict(n_heads=3), "divide"), (dict(qkv=qkv[0]), "qkv must be"), (dict(qkv=qkv.double()), "qkv must be"),
                     (dict(dtype=torch.bfloat16), "dtype"), (dict(cos=cos[:, :31], sin=sin[:, :31]), "multiple of 8"), (dict(cos=cos[:-1]), "two tables"),
                     (dict(cos=cos.double(), sin=sin.double()), "float32"), (dict(cos=cos.cpu(), sin=sin.cpu()), "device"), (dict(start=298), "rows"),
                     (dict(start=-1), "rows"), (dict(q_weight=wq.float()), "q_weight"), (dict(k_weight=wk[:32]), "k_weight"),
                     (dict(positions=torch.zeros(2, dtype=torch.int64, device="cuda")), "positions"),
                     (dict(positions=torch.zeros(3, dtype=torch.int32, device="cuda")), "positions"),
                     (dict(positions=torch.zeros(2, dtype=torch.int32, device="cuda"), start=1), "exclude"), (dict(n_heads=6, n_kv_heads=1), "head_dim")]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    x, kw = logits_inputs(2, 100, 5, torch.float16)
    for change, text in [(dict(history=kw["history"].long()), "history must"), (dict(history=kw["history"][:1]), "history must"),
                         (dict(history=None), "without history"), (dict(history_lens=kw["history_lens"].long()), "history_lens must"),
                         (dict(repetition=0.0), "positive"), (dict(presence=torch.zeros(3, device="cuda")), "presence"),
                         (dict(bias=torch.zeros(99, device="cuda")), "bias"), (dict(bias=kw["bias"].half()), "bias"),
                         (dict(mask=kw["mask"][:, :3]), "mask"), (dict(out=x.float()), "out must"), (dict(out=x[:, :50]), "out must"),
                         (dict(out=x[:1].expand(2, 100)), "out must")]:
        with pytest.raises(RuntimeError, match=text):
            step.process_logits(x, **{**kw, **change})
    with pytest.raises(RuntimeError, match="one piece"):
        step.process_logits(x.t().contiguous().t())
    out, tokens = step.process_logits(x[:0])
    assert out.shape == (0, 100) and tokens.shape == (0,)
