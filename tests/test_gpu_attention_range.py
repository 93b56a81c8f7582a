"""Attention in fp16 where a probability or a score gradient leaves the range of its 16-bit operand: small and large incoming gradients, keys that
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


def against(q, k, v, go, lift, **kw):
    """outputs for the incoming gradient `go`, whose size is about 1 / lift (a power of two): the gradients are linear in it, so values and bounds
    are the definition's for lift * go, where no rounding of an operand meets a subnormal, and half the smallest subnormal of the result"""
    ref = R.attention(q, k, v, go=go.double() * lift, **kw)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = T().window_attention(*leaves, **kw)
    R.within('o', o, *ref['o'])
    for n, t in zip(('gq', 'gk', 'gv'), torch.autograd.grad(o, leaves, go.cuda())):
        val, bound = ref[n]
        R.within(n, t, val / lift, bound / lift + U)


CASES = [(1, 1024, 1024, 2, 1, 64, dict(window=512, causal=False)), (1, 700, 700, 4, 2, 128, dict(causal=True)),
         (1, 130, 5000, 2, 1, 128, dict(causal=True)), (2, 333, 333, 2, 2, 40, dict(window=90, sinks=3, causal=True)),
         (20, 200, 200, 14, 14, 64, dict(causal=True)), (30, 260, 260, 9, 9, 96, dict(window=100, sinks=2))]


@pytest.mark.parametrize('size', [1e-4, 1e-3, 1.0, 1e3])
@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c[:6])))
def test_gradients_of_any_size(case, size):
    """a mean over a map's pixels hands back gradients of 1e-4, a scaled loss gradients of 1e3: dS = P (dP - delta) is as small as P times that"""
    b, lq, lk, h, hk, d, kw = case
    q, k, v, go = (rnd(i, *s) for i, s in enumerate(((b, lq, h, d), (b, lk, hk, d), (b, lk, hk, d), (b, lq, h, d))))
    go = (go.float() * size).to(F16)
    against(q, k, v, go, 2.0 ** -round(math.log2(size)), **kw)


@pytest.mark.parametrize('lq,lk', [(96, 96), (96, 700)])
def test_score_gradients_past_the_largest_half(lq, lk):
    """|dS| of more than 65504 where every result is representable"""
    b, h, hk, d = 1, 2, 1, 64
    q, k, v, go = (rnd(10 + i, *s) for i, s in enumerate(((b, lq, h, d), (b, lk, hk, d), (b, lk, hk, d), (b, lq, h, d))))
    q, k, v, go = q * 4, k * 4, v * 16, go * 2500
    go[:, ::3] *= 1e-3                                                   # rows of very different sizes side by side
    kw = dict(scale=2.0 ** -6)
    S = (q.double().transpose(1, 2) @ k.double().transpose(1, 2).transpose(2, 3)) * 2.0 ** -6
    P = S.softmax(-1)
    dP = go.double().transpose(1, 2) @ v.double().transpose(1, 2).transpose(2, 3)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    ref = R.attention(q, k, v, go=go, **kw)
    assert float(dS.abs().max()) > 7e4 and all(float(ref[n][0].abs().max()) < 6e4 for n in ('o', 'gq', 'gk', 'gv'))
    against(q, k, v, go, 2.0 ** -11, **kw)


def test_queries_whose_gradients_differ_by_many_orders():
    """one loss on the last tokens, almost none on the others; keys that only the quiet queries see (a window) keep their gradient's precision"""
    b, n, h, hk, d = 1, 1300, 2, 1, 64
    q, k, v, go = (rnd(20 + i, *s) for i, s in enumerate(((b, n, h, d), (b, n, hk, d), (b, n, hk, d), (b, n, h, d))))
    kw = dict(window=300, causal=True)
    go[:, :600] = (go[:, :600].float() * 4e-5).to(F16)
    ref = R.attention(q, k, v, go=go.double(), **kw)
    quiet = go.double() * 0
    quiet[:, :600] = go[:, :600].double()
    up = 2.0 ** 13
    low = R.attention(q, k, v, go=quiet * up, **kw)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    g = torch.autograd.grad(T().window_attention(*leaves, **kw), leaves, go.cuda())
    for i, (name, t) in enumerate(zip(('gq', 'gk', 'gv'), g)):
        R.within(name, t, *ref[name])
        m = 600 if i == 0 else 300                                       # keys [0, 300): seen by queries of small gradient alone
        R.within(name + ' of the quiet tokens', t[:, :m], low[name][0][:, :m] / up, low[name][1][:, :m] / up + U)


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


@pytest.mark.parametrize('d', [24, 48, 64, 80, 96, 128])
@pytest.mark.parametrize('b,hk,causal', [(1, 1, False), (20, 6, True)])
def test_score_gradients_that_climb_from_tile_to_tile(d, b, hk, causal):
    """incoming gradients that grow from query tile to query tile, values that grow from key tile to key tile, each by its own factor: the lift of every
    query and key falls again and again with sums formed before (few blocks: split walks; many: whole ones)"""
    n, h = 330, 2 * hk
    q, k, v, go = (rnd(30 + i, b, n, m, d) for i, m in enumerate((h, hk, hk, h)))
    tile = torch.arange(n) // 64
    go = (go.float() * 2.0 ** (4.0 * tile - 12)[None, :, None, None]).to(F16)
    v = (v.float() * 2.0 ** (3.0 * tile - 9)[None, :, None, None]).to(F16)
    kw = dict(causal=causal)
    ref = R.attention(q, k, v, go=go, **kw)
    assert all(float(ref[name][0].abs().max()) < 6e4 for name in ref)
    against(q, k, v, go, 1.0, **kw)
