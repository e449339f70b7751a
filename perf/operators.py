"""Operators around a decode step, as measurable cases: attention of many sequences over one shared packed prefix, rotation
(and normalisation) of the projected queries and keys, penalties and masks on the logits with the choice of the next token.

Together they are the step of a server that generates several completions of one prompt.  ``run`` computes each operator in
elementary torch operations (``own`` false) or calls the library (``own`` true); ``exact`` evaluates the definitions in 64 bits.
Head geometry, batches and context lengths are those of the library's other measured cases (32 heads x 128, groups of 1 to 8, 4- and
2-bit codes, batches up to 128); vocabularies and histories are generic.
"""
import math

import torch

own = False

D = 128
SMIN, SMAX = math.exp(-4.0), math.exp(4.0)      # bounds of the scales
EPS = 1e-8                                      # the quantiser's guard
INTERVAL = 128                                  # tokens between the state checkpoints of a prefix
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # two completions of one question over a short instruction: the smallest step, nothing but latency
        dict(name="prefix_b2_p300", kind="prefix", B=2, Hq=32, Hkv=32, P=300, T=9, bits=4),
        # a best-of-16 sampler in mid-generation, ragged lengths
        dict(name="prefix_b16_p2047_t200", kind="prefix", B=16, Hq=32, Hkv=32, P=2047, T=200, bits=4),
        # a batch of users behind one long system prompt
        dict(name="prefix_b64_p8192_t128", kind="prefix", B=64, Hq=32, Hkv=32, P=8192, T=128, bits=4),
        # questions about one long document: grouped queries, 2-bit codes
        dict(name="prefix_gqa_b32_p16000_2bit_t64", kind="prefix", B=32, Hq=32, Hkv=8, P=16000, T=64, bits=2),
        # many users of a model with eight query heads on a KV head, behind a shorter prompt
        dict(name="prefix_gqa8_b128_p1500_t32", kind="prefix", B=128, Hq=64, Hkv=8, P=1500, T=32, bits=4),
        # one decode step of a large batch, as the model harness makes it: rotation only, straight out of the projection
        dict(name="rope_b128_t1", kind="rope", B=128, T=1, Hq=32, Hkv=32, D=128, rot=128, dtype="fp16", norm=False, interleaved=False, start=1536),
        # prefill of one long prompt of a model that normalises queries and keys per head, bf16 activations, fp16 for the cache
        dict(name="norm_rope_b1_t8191_gqa", kind="rope", B=1, T=8191, Hq=32, Hkv=8, D=128, rot=128, dtype="bf16", norm=True, interleaved=False, start=0),
        # prefill of a ragged batch, a quarter of each head rotated in neighbouring pairs
        dict(name="norm_rope_b16_t777_pairs", kind="rope", B=16, T=777, Hq=16, Hkv=16, D=256, rot=64, dtype="fp16", norm=True, interleaved=True, start=5),
        # one sequence, a repetition penalty over a short history: latency
        dict(name="logits_b1_v32000", kind="logits", B=1, V=32000, L=100, dtype="fp16", bias=False, mask=False),
        # sampling with all penalties, a bias and a grammar's mask, large vocabulary, long histories
        dict(name="logits_b64_v128256", kind="logits", B=64, V=128256, L=4000, dtype="bf16", bias=True, mask=True),
        # the largest batch, an odd vocabulary, rows without alignment
        dict(name="logits_b128_v50257_fp32", kind="logits", B=128, V=50257, L=1500, dtype="fp32", bias=False, mask=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above; sizes over their logarithm, no dearer than the dearest listed case of its kind."""
    kind = rng.choice(["prefix", "prefix", "rope", "logits"])
    most = [work(c) for c in listed() if c["kind"] == kind]
    while True:
        if kind == "prefix":
            Hq, Hkv = rng.choice([(32, 32), (32, 8), (16, 8), (16, 16), (64, 8), (8, 8), (5, 5), (12, 6)])
            case = dict(kind=kind, B=_log(rng, 1, 128), Hq=Hq, Hkv=Hkv, P=_log(rng, 1, 16384), T=_log(rng, 1, 400), bits=rng.choice([4, 4, 2]))
        elif kind == "rope":
            Hkv = rng.choice([1, 2, 4, 8, 16, 32])
            width = rng.choice([64, 128, 128, 256])
            case = dict(kind=kind, B=_log(rng, 1, 128), T=rng.choice([1, _log(rng, 1, 8192)]), Hq=Hkv * rng.choice([1, 2, 4, 8]), Hkv=Hkv, D=width,
                        rot=width // rng.choice([1, 1, 2, 4]), dtype=rng.choice(["fp16", "bf16"]), norm=rng.random() < 0.5,
                        interleaved=rng.random() < 0.4, start=rng.randrange(0, 3000))
        else:
            case = dict(kind=kind, B=_log(rng, 1, 128), V=_log(rng, 1000, 160000), L=_log(rng, 1, 8192), dtype=rng.choice(["fp16", "bf16", "fp32"]),
                        bias=rng.random() < 0.5, mask=rng.random() < 0.5)
        w = work(case)
        if all(w[k] <= max(m[k] for m in most) for k in w):
            return case


def _lens(case):
    """Cached tokens of each sequence: all of T for the first, then spread evenly down to none, a sequence about to write its first."""
    B, T = case["B"], case["T"]
    return [T - T * i // max(1, B - 1) for i in range(B)]


def work(case):
    if case["kind"] == "prefix":
        B, Hq, Hkv, P, bits = (case[k] for k in ("B", "Hq", "Hkv", "P", "bits"))
        own_tokens = sum(_lens(case))
        codes = 2 * Hkv * D * (P + own_tokens)
        data = codes * bits // 8 + 2 * 2 * Hkv * D * 4 + 2 * 5 * Hkv * D * 2       # codes; the state they start from; parameters
        data += 2 * B * Hq * D * 2 + 2 * B * Hkv * D * 2 + 2 * 2 * 2 * B * Hkv * D * 4   # queries, results, new tokens, states in and out
        # eight operations replay a value, four use it for a query
        return {"bytes": data, "flops": 8 * codes + 4 * D * Hq * (B * P + own_tokens + B)}
    if case["kind"] == "rope":
        n = case["B"] * case["T"] * (case["Hq"] + 2 * case["Hkv"]) * case["D"]
        tables = 2 * case["T"] * (case["rot"] // 2) * 4
        return {"bytes": 2 * n * 2 + tables, "flops": n * (4 if case["norm"] else 0) + 3 * n * case["rot"] // case["D"]}
    B, V, L = case["B"], case["V"], case["L"]
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    data = 2 * B * V * size + B * L * 4 + (4 * V if case["bias"] else 0) + (B * ((V + 31) // 32) * 4 if case["mask"] else 0) + 4 * B
    return {"bytes": data, "flops": B * V * (2 + int(case["bias"]))}


# ---------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tokens(g, lead, T, means):
    """K or V of T tokens: unit noise around the means of the channels (a few of them far out), as fp16 holds it."""
    x = torch.randn(*lead, T, D, generator=g, device="cuda")
    return (x + means[..., None, :]).half().float()


def _encode(x, state, par, bits, keep=0):
    """Codes of x [..., T, D] from ``state`` = (zp, s), the state behind them, and those before every ``keep``-th token."""
    alpha, beta, target = par
    lo, hi = -float(1 << (bits - 1)), float((1 << (bits - 1)) - 1)
    zp, s = state
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    marks = []
    for t in range(x.shape[-2]):
        guard = s.clamp(min=EPS)
        code = torch.round((x[..., t, :] - zp) / guard).clamp_(lo, hi)
        codes[..., t, :] = code
        zp = zp + alpha * (code * guard)
        s = (s + s * beta * (code.abs() - target)).clamp_(SMIN, SMAX)
        if keep and (t + 1) % keep == 0:
            marks.append(torch.stack([zp, s], -2))
    return codes, (zp, s), marks


def _pack(codes, bits, words):
    """codes [B, H, T, D] -> packed cache [B, H, words, D / 4, 4, 4]: token j of a word at bits j * bits, as code + 2^(bits - 1)."""
    tpw = 32 // bits
    B, H, T, _ = codes.shape
    full = torch.zeros((B, H, words * tpw, D), dtype=torch.int64, device=codes.device)
    full[:, :, :T] = codes.long() + (1 << (bits - 1))
    shift = torch.arange(tpw, device=codes.device)[:, None] * bits
    word = (full.view(B, H, words, tpw, D) << shift).sum(3)
    byte = torch.stack([(word >> (8 * i)) & 255 for i in range(4)], -1).to(torch.uint8)
    return byte.view(B, H, words, D // 4, 4, 4).contiguous()


def _prepare_prefix(case, seed):
    B, Hq, Hkv, P, bits = (case[k] for k in ("B", "Hq", "Hkv", "P", "bits"))
    g = _gen(seed)
    tpw = 32 // bits
    alpha = (1.0 - (0.90 + 0.099 * torch.rand(2, Hkv, D, generator=g, device="cuda"))).half()
    target = ((1 << (bits - 1)) - 1) / 2.0
    params = [tuple(t.contiguous() for t in (torch.zeros_like(alpha[i]), torch.ones_like(alpha[i]), alpha[i], torch.full_like(alpha[i], 0.05),
                                             torch.full_like(alpha[i], target))) for i in range(2)]
    par = tuple(torch.stack([params[0][j], params[1][j]]).float()[:, None] for j in (2, 3, 4))        # [2, 1, Hkv, D]
    far = torch.rand(2, Hkv, D, generator=g, device="cuda") < 4.0 / D
    means = torch.where(far, 20.0, 0.5) * torch.randn(2, Hkv, D, generator=g, device="cuda")
    zero = torch.zeros(2, 1, Hkv, D, device="cuda")
    codes, state, marks = _encode(_tokens(g, (2, 1, Hkv), P, means[:, None]), (zero, zero + 1.0), par, bits, INTERVAL)
    words = (P + tpw - 1) // tpw
    ckpt = torch.stack(marks, 3) if marks else torch.zeros(2, 1, Hkv, 1, 2, D, device="cuda")          # [2, 1, Hkv, n, 2, D]
    lens = _lens(case)
    T = max(lens)
    own_codes = torch.zeros(2, B, Hkv, T, D, dtype=torch.int8, device="cuda")
    tails = torch.empty(2, B, Hkv, 2, D, device="cuda")
    lens_gpu = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # every sequence goes on from the state behind the prefix; its tail is the state behind its last token
    zp, s = (t.expand(2, B, Hkv, D) for t in state)
    tails.copy_(torch.stack([zp, s], -2))
    own_codes, _, marks = _encode(_tokens(g, (2, B, Hkv), T, means[:, None]), (zp, s), par, bits, 1) if T else (own_codes, None, [])
    for b, n in enumerate(lens):
        if n:
            tails[:, b] = marks[n - 1][:, b]
    room = (T + 1 + tpw - 1) // tpw + 1
    st = dict(case=case, params=params, prefix=[_pack(codes[i], bits, words) for i in range(2)],
              caches=[_pack(own_codes[i], bits, room) for i in range(2)], ckpt=ckpt, prefix_tail=torch.stack(state, -2).contiguous(),
              tails0=tails, tails=tails.clone(), lens=lens_gpu,
              q=torch.randn(B, Hq, 1, D, generator=g, device="cuda").half(),
              new=[(torch.randn(B, Hkv, 1, D, generator=g, device="cuda") + means[i][None, :, None]).half() for i in range(2)])
    if own:
        from adkv_b200 import gemv
        st["shared"] = gemv.SharedPrefix(st["prefix"][0], st["prefix"][1], P, bits=bits, k_tail=st["prefix_tail"][0], v_tail=st["prefix_tail"][1],
                                         k_ckpt=st["ckpt"][0], v_ckpt=st["ckpt"][1], ckpt_interval=INTERVAL)
        st["scratch"] = torch.empty(gemv.prefix_scratch_bytes(B, Hq, st["shared"]), dtype=torch.uint8, device="cuda")
    return st


def _prepare_rope(case, seed):
    B, T, Hq, Hkv, width = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    g = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * width, generator=g, device="cuda", dtype=dtype)
    half = case["rot"] // 2
    inv = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    ang = torch.arange(case["start"] + T, device="cuda", dtype=torch.float64)[:, None] * inv
    st = dict(case=case, qkv=qkv, cos=ang.cos().float(), sin=ang.sin().float(), wq=None, wk=None)
    if case["norm"]:
        st["wq"], st["wk"] = (1.0 + 0.1 * torch.randn(2, width, generator=g, device="cuda")).to(dtype).unbind(0)
    return st


def _prepare_logits(case, seed):
    B, V, L = case["B"], case["V"], case["L"]
    g = _gen(seed)
    st = dict(case=case, logits=(3.0 * torch.randn(B, V, generator=g, device="cuda")).to(DTYPES[case["dtype"]]), bias=None, mask=None)
    # words repeat: small ids are frequent
    st["history"] = (V * torch.rand(B, L, generator=g, device="cuda") ** 3).int().clamp_(0, V - 1)
    st["lens"] = torch.randint(0, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    st["lens"][0] = L
    st["repetition"] = 1.0 + 0.5 * torch.rand(B, generator=g, device="cuda")
    st["presence"] = 0.3 * torch.rand(B, generator=g, device="cuda")
    st["frequency"] = 0.2 * torch.rand(B, generator=g, device="cuda")
    if case["bias"]:
        st["bias"] = torch.where(torch.rand(V, generator=g, device="cuda") < 0.01, 4.0, 0.0) * torch.randn(V, generator=g, device="cuda")
    if case["mask"]:
        # a grammar allows a few tokens, a filter forbids a few; one row of a batch is left without any
        share = torch.rand(B, 1, generator=g, device="cuda") ** 2
        allowed = torch.rand(B, (V + 31) // 32 * 32, generator=g, device="cuda") < share
        if B > 3:
            allowed[3] = False
        bit = torch.arange(32, device="cuda")
        word = (allowed.view(B, -1, 32).long() << bit).sum(-1)
        st["mask"] = torch.where(word >= 1 << 31, word - (1 << 32), word).int()
    return st


def prepare(case, seed):
    return {"prefix": _prepare_prefix, "rope": _prepare_rope, "logits": _prepare_logits}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------------- one pass

def _unpack(cache, bits, tokens):
    B, H, words = cache.shape[:3]
    word = cache.view(B, H, words, D, 4).view(torch.int32).view(B, H, words, 1, D)
    shift = torch.arange(32 // bits, device=cache.device, dtype=torch.int32)[:, None] * bits
    code = ((word >> shift) & ((1 << bits) - 1)) - (1 << (bits - 1))
    return code.view(B, H, words * (32 // bits), D)[:, :, :tokens].float()


def _replay(codes, zp, s, par):
    """Values of codes [..., T, D] from the state (zp, s) before the first of them."""
    alpha, beta, target = par
    out = torch.empty_like(codes)
    for t in range(codes.shape[-2]):
        code = codes[..., t, :]
        step = code * s.clamp(min=EPS)
        out[..., t, :] = step + zp
        zp = zp + alpha * step
        s = (s + s * beta * (code.abs() - target)).clamp(SMIN, SMAX)
    return out


def _run_prefix(st):
    case = st["case"]
    B, Hq, Hkv, P, bits = (case[k] for k in ("B", "Hq", "Hkv", "P", "bits"))
    scaling = D ** -0.5
    if own:
        from adkv_b200 import gemv
        st["tails"].copy_(st["tails0"])      # the step advances the tails: each pass starts from the same ones
        out = gemv.decode_attn_prefix(st["q"], st["shared"], st["caches"][0], st["caches"][1], st["new"][0], st["new"][1], st["params"][0],
                                      st["params"][1], st["lens"], scaling, SMIN, SMAX, k_tail=st["tails"][0], v_tail=st["tails"][1],
                                      scratch=st["scratch"])
        return out, st["tails"]
    par = tuple(torch.stack([st["params"][0][j], st["params"][1][j]]).float()[:, None] for j in (2, 3, 4))        # [2, 1, Hkv, D]
    # the prefix between its checkpoints, all intervals side by side
    n = (P + INTERVAL - 1) // INTERVAL
    codes = torch.zeros(2, 1, Hkv, n * INTERVAL, D, device="cuda")
    codes[:, :, :, :P] = torch.stack([_unpack(c, bits, P) for c in st["prefix"]])
    first = torch.stack([torch.stack([st["params"][i][0], st["params"][i][1]], 1) for i in range(2)]).float()[:, None, :, None]   # [2, 1, Hkv, 1, 2, D]
    begin = torch.cat([first, st["ckpt"]], 3)[:, :, :, :n]
    values = _replay(codes.view(2, 1, Hkv, n, INTERVAL, D), begin[..., 0, :], begin[..., 1, :], tuple(p[:, :, :, None] for p in par))
    k_pre, v_pre = values.reshape(2, Hkv, n * INTERVAL, D)[:, :, :P].unbind(0)
    # what each sequence has cached itself, from the state behind the prefix
    room = max(_lens(case))
    codes = torch.stack([_unpack(c, bits, room) for c in st["caches"]])
    end = st["prefix_tail"].expand(2, B, Hkv, 2, D)
    k_own, v_own = _replay(codes, end[..., 0, :], end[..., 1, :], par).unbind(0)
    # the new token, quantised with the tail, which moves on
    alpha, beta, target = par
    zp, s = st["tails0"].unbind(-2)
    guard = s.clamp(min=EPS)
    code = torch.round((torch.stack(st["new"]).float()[..., 0, :] - zp) / guard).clamp(-float(1 << (bits - 1)), float((1 << (bits - 1)) - 1))
    step = code * guard
    k_self, v_self = (step + zp).unbind(0)
    tails = torch.stack([zp + alpha * step, (s + s * beta * (code.abs() - target)).clamp(SMIN, SMAX)], -2)
    G = Hq // Hkv
    q = st["q"].float().view(B, Hkv, G, D)
    by_head = q.transpose(0, 1).reshape(Hkv, B * G, D)
    pre = (by_head @ k_pre.transpose(1, 2)).view(Hkv, B, G, P).transpose(0, 1)
    mine = q @ k_own.transpose(2, 3)
    mine = mine.masked_fill((torch.arange(room, device="cuda") >= st["lens"][:, None])[:, None, None], -math.inf)
    logits = torch.cat([pre, mine, (q * k_self[:, :, None]).sum(-1, keepdim=True)], -1) * scaling
    logits = logits - logits.amax(-1, keepdim=True)
    p = logits.exp()
    p = p / p.sum(-1, keepdim=True)
    out = (p[..., :P].transpose(0, 1).reshape(Hkv, B * G, P) @ v_pre).view(Hkv, B, G, D).transpose(0, 1)
    out = out + p[..., P:P + room] @ v_own + p[..., -1:] * v_self[:, :, None]
    return out.reshape(B, Hq, D).half(), tails


def _run_rope(st):
    case = st["case"]
    B, T, Hq, Hkv, width = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    if own:
        from adkv_b200 import step
        return step.norm_rope_qkv(st["qkv"], Hq, Hkv, st["cos"], st["sin"], start=case["start"], q_weight=st["wq"], k_weight=st["wk"], eps=1e-6,
                                  interleaved=case["interleaved"], dtype=torch.float16)
    x = st["qkv"].view(B, T, Hq + 2 * Hkv, width).transpose(1, 2)
    cos, sin = st["cos"][case["start"]:case["start"] + T], st["sin"][case["start"]:case["start"] + T]
    half = case["rot"] // 2

    def turned(part, weight):
        y = part.float()
        if weight is not None:
            y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * weight.float()
        turn, rest = y[..., :2 * half], y[..., 2 * half:]
        if case["interleaved"]:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turn[..., :half], turn[..., half:]
            turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turn, rest], -1).half()

    return turned(x[:, :Hq], st["wq"]), turned(x[:, Hq:Hq + Hkv], st["wk"]), x[:, Hq + Hkv:].half().contiguous()


def _run_logits(st):
    if own:
        from adkv_b200 import step
        return step.process_logits(st["logits"], history=st["history"], history_lens=st["lens"], repetition=st["repetition"],
                                   presence=st["presence"], frequency=st["frequency"], bias=st["bias"], mask=st["mask"])
    case = st["case"]
    B, V, L = case["B"], case["V"], case["L"]
    x = st["logits"].float()
    there = (torch.arange(L, device="cuda") < st["lens"][:, None]).float()
    count = torch.zeros(B, V, device="cuda").scatter_add_(1, st["history"].long(), there)
    rep = st["repetition"][:, None]
    x = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep) - (st["frequency"][:, None] * count + st["presence"][:, None]), x)
    if st["bias"] is not None:
        x = x + st["bias"]
    if st["mask"] is not None:
        bit = torch.arange(V, device="cuda")
        x = torch.where(((st["mask"][:, bit >> 5] >> (bit & 31).int()) & 1).bool(), x, -math.inf)
    out = x.to(st["logits"].dtype)
    # the token: the lowest index of the largest, -1 where nothing is left
    top = out.amax(-1, keepdim=True)
    token = torch.where(out == top, torch.arange(V, device="cuda"), V).amin(-1)
    return out, torch.where(top[:, 0] == -math.inf, -1, token).int()


def run(state):
    return {"prefix": _run_prefix, "rope": _run_rope, "logits": _run_logits}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------- the definitions, in 64 bits

def _states64(words, bits, begin, const, tokens):
    """x[t] = zp[t] + c[t] * max(s[t], eps) of one run of tokens: words [..., W, D] int64, begin [..., 2, D]."""
    values = []
    zero_point, scale = begin[..., 0, :].clone(), begin[..., 1, :].clone()
    per_word, low = 32 // bits, 1 << (bits - 1)
    for t in range(tokens):
        c = ((words[..., t // per_word, :] >> (bits * (t % per_word))) % (2 * low) - low).double()
        move = c * torch.maximum(scale, torch.full_like(scale, EPS))
        values.append(zero_point + move)
        zero_point = zero_point + const[0] * move
        scale = torch.minimum(torch.maximum(scale * (1.0 + const[1] * (c.abs() - const[2])), torch.full_like(scale, SMIN)),
                              torch.full_like(scale, SMAX))
    return torch.stack(values, -2) if values else begin.new_zeros(*begin.shape[:-2], 0, D)


def _words64(cache):
    byte = cache.long().view(*cache.shape[:3], D, 4)
    return byte[..., 0] + (byte[..., 1] << 8) + (byte[..., 2] << 16) + (byte[..., 3] << 24)


def _exact_prefix(case, st):
    B, Hq, Hkv, P, bits = (case[k] for k in ("B", "Hq", "Hkv", "P", "bits"))
    per_word, top_code = 32 // bits, (1 << (bits - 1)) - 1
    kv, tails = [], []
    for i in range(2):
        const = [st["params"][i][j].double() for j in (2, 3, 4)]
        words = _words64(st["prefix"][i])[0]
        parts = []
        full = P // INTERVAL                      # whole intervals side by side, then what is left
        states = torch.cat([torch.stack(st["params"][i][:2], 1).double()[:, None], st["ckpt"][i][0].double()], 1)   # [Hkv, 1 + n, 2, D]
        if full:
            block = words[:, :full * INTERVAL // per_word].view(Hkv, full, INTERVAL // per_word, D)
            parts.append(_states64(block, bits, states[:, :full], [c[:, None] for c in const], INTERVAL).flatten(1, 2))
        if P % INTERVAL:
            parts.append(_states64(words[:, full * INTERVAL // per_word:], bits, states[:, full], const, P % INTERVAL))
        shared = torch.cat(parts, 1)
        mine = _states64(_words64(st["caches"][i]), bits, st["prefix_tail"][i].double().expand(B, Hkv, 2, D), const, max(_lens(case)))
        # the code of the new token is a 32-bit quotient, rounded to even; what follows from it is not
        zp, s = st["tails0"][i][:, :, 0], st["tails0"][i][:, :, 1]
        code = torch.clip(torch.round((st["new"][i][:, :, 0].float() - zp) / torch.clip(s, min=EPS)), -top_code - 1, top_code).double()
        zp, s = zp.double(), s.double()
        move = code * torch.clip(s, min=EPS)
        tails.append(torch.stack([zp + const[0] * move, torch.clip(s * (1.0 + const[1] * (code.abs() - const[2])), SMIN, SMAX)], 2))
        kv.append((shared, mine, zp + move))
    q = st["q"].double().view(B, Hkv, Hq // Hkv, D) / math.sqrt(D)
    result = torch.empty(B, Hkv, Hq // Hkv, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        k = torch.cat([kv[0][0], kv[0][1][b, :, :n], kv[0][2][b, :, None]], 1)
        v = torch.cat([kv[1][0], kv[1][1][b, :, :n], kv[1][2][b, :, None]], 1)
        result[b] = torch.softmax(torch.einsum("hgd,htd->hgt", q[b], k), -1) @ v
    return result.view(B, Hq, D), torch.stack(tails)


def _exact_rope(case, st):
    B, T, Hq, Hkv, width, rot = (case[k] for k in ("B", "T", "Hq", "Hkv", "D", "rot"))
    heads = st["qkv"].double().reshape(B, T, Hq + 2 * Hkv, width)
    # a pair of channels as one complex number, turned by cos + i sin
    turn = torch.complex(st["cos"].double(), st["sin"].double())[case["start"]:case["start"] + T, None]

    def one(h0, h1, weight):
        y = heads[:, :, h0:h1].clone()
        if weight is not None:
            y = y * weight.double() * ((y * y).sum(-1, keepdim=True) / width + 1e-6) ** -0.5
        if case["interleaved"]:
            even, odd = slice(0, rot, 2), slice(1, rot, 2)
        else:
            even, odd = slice(0, rot // 2), slice(rot // 2, rot)
        z = torch.complex(y[..., even], y[..., odd]) * turn
        y[..., even], y[..., odd] = z.real, z.imag
        return y.permute(0, 2, 1, 3)

    return one(0, Hq, st["wq"]), one(Hq, Hq + Hkv, st["wk"]), heads[:, :, Hq + Hkv:].permute(0, 2, 1, 3)


def _exact_logits(case, st):
    B, V = case["B"], case["V"]
    result = st["logits"].double()
    lens = st["lens"].tolist()
    for b in range(B):
        seen, times = torch.unique(st["history"][b, :lens[b]].long(), return_counts=True)
        x = result[b, seen]
        rep = st["repetition"][b].double()
        x = torch.where(x > 0, x / rep, x * rep)
        result[b, seen] = x - st["presence"][b].double() - st["frequency"][b].double() * times
    if st["bias"] is not None:
        result = result + st["bias"].double()
    if st["mask"] is not None:
        word = st["mask"].long() % (1 << 32)
        allowed = ((word[:, :, None] >> torch.arange(32, device="cuda")) % 2).reshape(B, -1)[:, :V]
        result[allowed == 0] = -math.inf
    return result, None          # the token is chosen among the rounded logits


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    return {"prefix": _exact_prefix, "rope": _exact_rope, "logits": _exact_logits}[case["kind"]](case, state)
