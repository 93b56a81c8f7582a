"""Attention in fp16 where a probability or a score gradient leaves the range of its 16-bit operand: keys that
hold little of the softmax each and much of it together.  64-bit definitions and their bounds: tests/token_ref.py."""
import math

import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu

F16 = torch.float16
U = R.tiny(F16)


def T():
    from multiyolov5_amd.utils import tokens
    return tokens


def rnd(seed, *shape, dt=F16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dt)


@pytest.mark.parametrize('lq,lk,h', [(1, 40000, 1), (200, 3000, 300), (40, 9000, 2)])
def test_many_keys_of_little_weight(lq, lk, h):
    """one key holds nearly all of every softmax, and its value is zero: the result is what thousands of probabilities of 2^-26 add up to.  As fp16
    operands relative to the largest they would all be nothing"""
    d = 16
    g = torch.Generator().manual_seed(3)
    q = torch.zeros(1, lq, h, d, dtype=F16)
    q[..., 0] = 1.0
    k = torch.zeros(1, lk, h, d, dtype=F16)
    k[..., 0] = -(25.5 + torch.rand(1, lk, h, generator=g)) * math.log(2.0)            # (exact in fp16 as rounded here)
    k[:, 100] = 0.0
    v = 1.0 + torch.rand(1, lk, h, d, generator=g).to(F16)
    v[:, 100] = 0.0
    P = k.double()[..., 0].transpose(1, 2)[:, :, None].softmax(-1)                   # (every query is the first unit vector)
    ref = (P @ v.double().transpose(1, 2)).transpose(1, 2).expand(1, lq, h, d)
    # probabilities relative to the largest are about 2^-26; a rounding to an operand that keeps 11 bits down to 2^-25 (and half a step of 2^-36
    # below) is off by 2^-36 each; sums of lk + 4 terms in 32 bits; scores up to 19, four roundings each; the result's own rounding
    bound = (lk + 4) * R.E * ref.abs() + 80 * R.E * ref.abs() + 2.0 ** -11 * ref.abs() + 2.0 ** -36 * lk * 2.0 + R.half_step(F16) * ref.abs() + U
    assert float((bound / ref).max()) < 0.2
    o = T().window_attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)
    R.within('o', o, ref, bound)
