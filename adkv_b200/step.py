"""What a prefill or decode step does around the attention kernels, one launch each.

``norm_rope_qkv`` takes queries, keys and values from the projection to the layout of the caches, normalising and rotating on the way (the
reference does this in torch, ``src/adkv/hf/llama_adkv.py:333-345``); ``process_logits`` applies penalties, biases and masks to the logits
and chooses the next token (no counterpart in the reference).  Both run on the current torch CUDA stream, allocate nothing but
their results and can be captured into a CUDA graph.  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .gemv import _on_device, _require, _stream

__all__ = ["norm_rope_qkv", "process_logits"]

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
HEAD_DIMS = (64, 128, 256, 512)


def _ptr(t):
    return None if t is None else t.data_ptr()


def norm_rope_qkv(qkv, n_heads: int, n_kv_heads: int, cos, sin, *, start: int = 0, positions: torch.Tensor | None = None,
                  q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                  interleaved: bool = False, dtype: torch.dtype | None = None):
    """Queries ``[B, nh, T, DIM]``, keys and values ``[B, nh_kv, T, DIM]`` from ``qkv [B, T, (nh + 2 nh_kv) * DIM]``, contiguous, of ``dtype``:
    the input's (float16, bfloat16 or float32) or float16, which the caches take; default the input's.  Head dims 64, 128, 256, 512.

    ``q_weight`` / ``k_weight`` (``[DIM]``, the input's type): queries / keys become ``x / sqrt(mean(x^2) + eps) * weight`` per head first.
    ``cos`` / ``sin`` (float32 ``[rows, rot / 2]``, a row per position) then rotate the first ``rot`` channels (a multiple of 8): pairs
    ``(i, i + rot / 2)``, or ``(2i, 2i + 1)`` if ``interleaved``; the others pass through.  Token t of a sequence is at position
    ``start + t``, or ``positions[b] + t`` / ``positions[b, t]`` for int32 CUDA tensors ``[B]`` / ``[B, T]``; a position on the device that has
    no row makes queries and keys of its token NaN and ``gemv.device_status`` report 8.  Computed in float32, rounded once at the end."""
    native = _lib.host()
    if native:                                  # plain tensors of the usual layouts: checked and called in native code
        done = native.norm_rope(qkv, n_heads, n_kv_heads, cos, sin, start, positions, q_weight, k_weight, eps, interleaved, dtype)
        if done is not None:
            if isinstance(done, int):
                _lib.check(done, "norm_rope_qkv")
            return done
    _require(qkv.is_cuda, "qkv must be a CUDA tensor (adkv_b200 has no CPU path)")
    _require(qkv.dim() == 3 and qkv.dtype in _TYPES, "qkv must be float16, bfloat16 or float32 [B, T, (nh + 2 nh_kv) * DIM]")
    _require(n_heads > 0 and n_kv_heads > 0 and qkv.shape[2] % (n_heads + 2 * n_kv_heads) == 0, "qkv does not divide into its heads")
    B, T, D = qkv.shape[0], qkv.shape[1], qkv.shape[2] // (n_heads + 2 * n_kv_heads)
    _require(D in HEAD_DIMS, f"head_dim {D} is not served by the kernel (one of {HEAD_DIMS})")
    dtype = qkv.dtype if dtype is None else dtype
    _require(dtype in (qkv.dtype, torch.float16), "dtype must be the input's or float16")
    _require(cos.shape == sin.shape and cos.dim() == 2 and cos.stride() == sin.stride(), "cos and sin must be two tables of one shape and layout")
    _require(cos.shape[0] < 1 << 31, "the tables must have fewer than 2^31 rows")
    rot = 2 * cos.shape[1]
    _require(0 < rot <= D and rot % 8 == 0, "the rotated channels must be a multiple of 8, at most the head dim")
    for t in (cos, sin):
        _require(t.dtype == torch.float32 and t.device == qkv.device and t.stride(1) == 1, "cos and sin must be float32 on qkv's device, channels side by side")
    for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        _require(w is None or (w.dtype == qkv.dtype and w.device == qkv.device and w.is_contiguous() and w.shape == (D,)),
                 f"{n} must be a contiguous [DIM] tensor of qkv's type and device")
    if positions is not None:
        _require(start == 0, "start and positions exclude each other")
        _require(positions.dtype == torch.int32 and positions.device == qkv.device and positions.is_contiguous() and
                 tuple(positions.shape) in ((B,), (B, T)), "positions must be a contiguous int32 [B] or [B, T] tensor on qkv's device")
    else:
        _require(start >= 0 and (start + T <= cos.shape[0] or B * T == 0), f"the tables have {cos.shape[0]} rows, positions {start} to {start + T - 1} were asked for")
    _require(B * T < 1 << 31, "too many tokens for one call")
    # rows of four elements at a time: anything else is copied into place first
    step = 4 * qkv.element_size()
    if qkv.stride(2) != 1 or qkv.stride(0) % 4 or qkv.stride(1) % 4 or qkv.data_ptr() % step:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    q_weight, k_weight = (w.clone() if w is not None and w.data_ptr() % step else w for w in (q_weight, k_weight))
    q = torch.empty((B, n_heads, T, D), dtype=dtype, device=qkv.device)
    k, v = (torch.empty((B, n_kv_heads, T, D), dtype=dtype, device=qkv.device) for _ in range(2))
    with _on_device(qkv.device):
        rc = _lib.load().adkv_norm_rope_qkv(qkv.data_ptr(), qkv.stride(0), qkv.stride(1), _TYPES[qkv.dtype], q.data_ptr(), k.data_ptr(),
                                            v.data_ptr(), _TYPES[dtype], _ptr(q_weight), _ptr(k_weight), eps, cos.data_ptr(), sin.data_ptr(),
                                            cos.stride(0), cos.shape[0], rot, _ptr(positions),
                                            int(positions is not None and positions.dim() == 2), start, B, T, n_heads, n_kv_heads, D,
                                            int(interleaved), _stream(qkv)) if B * T else 0
    _lib.check(rc, "norm_rope_qkv")
    return q, k, v


def _penalty(name, value, B, device):
    """(pointer, number) of a penalty given per sequence or for all."""
    if isinstance(value, torch.Tensor):
        _require(value.dtype == torch.float32 and value.device == device and value.is_contiguous() and value.shape == (B,),
                 f"{name} must be a number or a contiguous float32 [B] tensor on the logits' device")
        return value.data_ptr(), 0.0
    return None, float(value)


def process_logits(logits, *, history: torch.Tensor | None = None, history_lens: torch.Tensor | None = None, repetition=1.0, presence=0.0,
                   frequency=0.0, bias: torch.Tensor | None = None, mask: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """Logits ``[B, V]`` (float16, bfloat16 or float32) under penalties, bias and mask, and the token that they choose: ``(out, tokens)``.

    With n = how often a token occurs in ``history[b, :history_lens[b]]`` (int32 ids ``[B, L]``, others than ``0 .. V - 1`` do not count;
    lengths int32 ``[B]``, default all of L), in float32 and rounded once at the end:

    * n > 0: ``x / repetition`` where x > 0, ``x * repetition`` elsewhere, then minus ``frequency * n + presence`` (numbers, or float32 ``[B]``);
    * plus ``bias`` (float32 ``[V]`` or ``[B, V]``);
    * -inf where bit ``v % 32`` of ``mask[b, v // 32]`` (int32, at least ``ceil(V / 32)`` words a row) is not set.

    ``out``: of the logits' type and shape, may be ``logits`` itself but not overlap them in another way.  ``tokens`` int32 ``[B]``: the lowest index of the largest element of
    ``out`` (a NaN counts as the largest), -1 for a row of nothing but -inf."""
    native = out is None and _lib.host()
    if native:                                  # as in norm_rope_qkv
        done = native.logits(logits, history, history_lens, repetition, presence, frequency, bias, mask)
        if done is not None:
            if isinstance(done, int):
                _lib.check(done, "process_logits")
            return done
    _require(logits.is_cuda, "logits must be a CUDA tensor (adkv_b200 has no CPU path)")
    _require(logits.dim() == 2 and logits.dtype in _TYPES and logits.shape[1] > 0, "logits must be float16, bfloat16 or float32 [B, V]")
    B, V = logits.shape
    _require(B <= 65535 and V <= 0x7fff0000, "too many logits for one call")
    _require(B == 0 or logits.stride(1) == 1 or V == 1, "a row of logits must lie in one piece")
    device = logits.device
    if out is None:
        out = torch.empty((B, V), dtype=logits.dtype, device=device)
    else:
        _require(out.dtype == logits.dtype and out.device == device and out.shape == logits.shape and (out.stride(1) == 1 or V == 1) and
                 (out.stride(0) >= V or B <= 1), "out must match the logits, rows in one piece and apart")
    _require(history is not None or history_lens is None, "history_lens without history")
    if history is not None:
        _require(history.dtype == torch.int32 and history.device == device and history.dim() == 2 and history.shape[0] == B and
                 (history.stride(1) == 1 or history.shape[1] <= 1), "history must be int32 [B, L] on the logits' device, rows in one piece")
        _require(history.shape[1] < 1 << 31, "a history must have fewer than 2^31 tokens a row")
    if history_lens is not None:
        _require(history_lens.dtype == torch.int32 and history_lens.device == device and history_lens.is_contiguous() and
                 history_lens.shape == (B,), "history_lens must be a contiguous int32 [B] tensor on the logits' device")
    rep, rep1 = _penalty("repetition", repetition, B, device)
    pres, pres1 = _penalty("presence", presence, B, device)
    freq, freq1 = _penalty("frequency", frequency, B, device)
    _require(rep is not None or rep1 > 0, "repetition must be positive")
    bias_stride = 0
    if bias is not None:
        _require(bias.dtype == torch.float32 and bias.device == device and tuple(bias.shape) in ((V,), (B, V)) and (bias.stride(-1) == 1 or V == 1),
                 "bias must be float32 [V] or [B, V] on the logits' device, rows in one piece")
        bias_stride = bias.stride(0) if bias.dim() == 2 else 0
    if mask is not None:
        _require(mask.dtype == torch.int32 and mask.device == device and mask.dim() == 2 and mask.shape[0] == B and
                 mask.shape[1] >= (V + 31) // 32 and (mask.stride(1) == 1 or mask.shape[1] == 1),
                 "mask must be int32 [B, at least ceil(V / 32)] on the logits' device, rows in one piece")
    tokens = torch.empty(B, dtype=torch.int32, device=device)
    used = history is not None and history.shape[1] > 0
    with _on_device(device):
        rc = _lib.load().adkv_process_logits(logits.data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0), _TYPES[logits.dtype],
                                             tokens.data_ptr(), history.data_ptr() if used else None, history.stride(0) if used else 0,
                                             history.shape[1] if used else 0, _ptr(history_lens) if used else None, rep, rep1, pres, pres1,
                                             freq, freq1, _ptr(bias), bias_stride, _ptr(mask), mask.stride(0) if mask is not None else 0, B, V,
                                             _stream(logits)) if B else 0
    _lib.check(rc, "process_logits")
    return out, tokens
