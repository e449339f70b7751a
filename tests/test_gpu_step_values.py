"""Infinities, NaN and signed zeros in the rotation of projected heads: channels that are not rotated are copied whatever the others hold,
rotated ones follow the formula."""
import math

import pytest
import torch

from adkv_b200 import gemv, step


def bits_equal(got, want):
    """The same numbers, zeros with their signs; a NaN for a NaN."""
    nan = want.isnan()
    whole = {2: torch.int16, 4: torch.int32}[want.element_size()]
    return torch.equal(got.isnan(), nan) and torch.equal(got.view(whole)[~nan], want.view(whole)[~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot", [(64, 8), (64, 40), (64, 64), (128, 32), (128, 72), (128, 128), (256, 64), (512, 504)])
def test_special_values_on_both_sides_of_the_rotated_channels(D, rot, dtype, interleaved):
    """A special value in every channel in turn, one a head and token, so that each meets finite partners; then with partners of their
    kind.  Products and sums of the rotation are rounded one by one, as torch's are, so its expression gives the same bits."""
    Hq, Hkv, T = 5, 2, D
    g = torch.Generator(device="cuda").manual_seed(D + rot)
    qkv = torch.randn(2, T, Hq + 2 * Hkv, D, generator=g, device="cuda")
    special = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 0.0], device="cuda")
    channel = torch.arange(T, device="cuda")
    for h in range(Hq + 2 * Hkv):
        qkv[0, channel, h, channel] = special[(channel + h) % 5]
    many = torch.rand(T, Hq + 2 * Hkv, D, generator=g, device="cuda") < 0.3
    qkv[1] = torch.where(many, special[torch.randint(0, 5, many.shape, generator=g, device="cuda")], qkv[1])
    qkv = qkv.to(dtype)
    angle = torch.arange(T, device="cuda")[:, None] * 10000.0 ** (-torch.arange(rot // 2, device="cuda") / (rot // 2))
    cos, sin = angle.cos(), angle.sin()
    q, k, v = step.norm_rope_qkv(qkv.view(2, T, -1), Hq, Hkv, cos, sin, interleaved=interleaved)
    x = qkv.transpose(1, 2)
    y = x.float()
    i = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    j = i + 1 if interleaved else i + rot // 2
    turned = x.clone()
    turned[..., i] = (y[..., i] * cos - y[..., j] * sin).to(dtype)
    turned[..., j] = (y[..., j] * cos + y[..., i] * sin).to(dtype)
    for got, want in ((q, turned[:, :Hq]), (k, turned[:, Hq:Hq + Hkv]), (v, x[:, Hq + Hkv:])):
        assert bits_equal(got[..., rot:], want[..., rot:].contiguous())
        assert bits_equal(got[..., :rot], want[..., :rot].contiguous())


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_all_channels_of_a_token_without_a_position_are_nan(interleaved):
    qkv = torch.randn(1, 3, 4 * 64, device="cuda").half()
    table = torch.ones(2, 8, device="cuda")
    positions = torch.tensor([[1, 2, -1]], dtype=torch.int32, device="cuda")
    q, k, v = step.norm_rope_qkv(qkv, 2, 1, table, 0 * table, positions=positions, interleaved=interleaved)
    x = qkv.view(1, 3, 4, 64).transpose(1, 2)
    assert q[:, :, 1:].isnan().all() and k[:, :, 1:].isnan().all() and torch.equal(v, x[:, 3:])
    assert torch.equal(q[:, :, 0], x[:, :2, 0]) and torch.equal(k[:, :, 0], x[:, 2:3, 0])
    assert gemv.device_status() == 8
