"""Results and scratch memory of the native host path under a dispatch mode: made where the mode sees them."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from adkv_b200 import _lib, gemv, step, synth
from tests.util import SMAX, SMIN

pytestmark = pytest.mark.gpu
D = 128


class Made(TorchDispatchMode):
    """Addresses of all tensors that torch makes."""

    def __init__(self):
        super().__init__()
        self.seen = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if isinstance(out, torch.Tensor) and func.namespace == "aten" and "empty" in func.__name__:
            self.seen.add((out.data_ptr(), out.dtype, tuple(out.shape)))
        return out


def _calls():
    qkv = torch.randn(2, 3, 6 * D, device="cuda").half()
    table = torch.randn(8, 32, device="cuda")
    logits, history = torch.randn(2, 500, device="cuda"), torch.randint(0, 500, (2, 9), dtype=torch.int32, device="cuda")
    kp, vp = (synth.gen_params(i, 2, D, 4, device="cuda") for i in range(2))
    x = torch.randn(2, 2, 40, D, device="cuda").half()
    cache = [torch.zeros(1, 2, 5, D // 4, 4, 4, dtype=torch.uint8, device="cuda") for _ in range(2)]
    tails = [torch.zeros(1, 2, 2, D, device="cuda") for _ in range(2)]
    gemv.encode_kv_pair(cache[0], x[:1], kp, cache[1], x[1:], vp, SMIN, SMAX, k_tail=tails[0], v_tail=tails[1])
    prefix = gemv.SharedPrefix(*cache, 40, k_tail=tails[0], v_tail=tails[1])
    own = [torch.zeros(2, 2, 1, D // 4, 4, 4, dtype=torch.uint8, device="cuda") for _ in range(2)]
    kt, vt = prefix.start_tails(2)
    q, new = torch.randn(2, 4, 1, D, device="cuda").half(), x[:, :, :1].contiguous()
    return [lambda: step.norm_rope_qkv(qkv, 4, 1, table, table), lambda: step.process_logits(logits, history=history, repetition=1.3),
            lambda: (gemv.decode_attn_prefix(q, prefix, *own, new, new, kp, vp, 0, 0.1, SMIN, SMAX, k_tail=kt, v_tail=vt, tail_keep=True),)]


def test_a_dispatch_mode_sees_every_result():
    assert _lib.host(), "the native host module must load"
    for call in _calls():
        alone = call()
        with Made() as mode:
            got = call()
            assert {(t.data_ptr(), t.dtype, tuple(t.shape)) for t in got} <= mode.seen
        assert all(torch.equal(a, b) for a, b in zip(alone, got))
    assert any(dtype == torch.uint8 for _, dtype, _ in mode.seen)          # the last call's scratch memory
    assert gemv.device_status() == 0


def test_inside_a_transform_results_are_those_outside():
    rope, logits, _ = _calls()
    for call in (rope, logits):
        alone = call()
        got = []
        torch.func.vmap(lambda t: (got.append(call()), t)[1])(torch.zeros(2, device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(alone, got[0]))
