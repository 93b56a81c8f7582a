"""The variants of the token operators that large calls run on: attention that nothing splits, walking several key tiles; sink blocks of dk / dv
split beside whole ones; layer norm's loop over rows; the rotary kernel's four heads a thread.  Definitions and bounds: tests/token_ref.py."""
import ctypes as C
import math

import pytest
import torch

from tests import token_ref as R
from tests.test_gpu_tokens import F16, F32, T, cuda, rnd

pytestmark = pytest.mark.gpu
DTS = pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])


# ---- attention -------------------------------------------------------------------------------------------------------------------------
def scratch(b, lq, lk, h, hk, d, window, sinks, causal, dt):
    """(forward's scratch bytes, backward's behind the row sums): what the library splits"""
    from multiyolov5_amd import _lib as L
    a = L.AttnDesc()
    a.b, a.lq, a.lk, a.hq, a.hk, a.d, a.dtype, a.causal, a.window, a.sinks, a.scale = b, lq, lk, h, hk, d, L.DT[dt], causal, window, sinks, 1.0
    ws = [L.lib().myolo_attn_ws_bytes(C.byref(a), i) for i in (0, 1)]
    return ws[0], ws[1] - (b * h * lq * 4 + 15) // 16 * 16


WHOLE = [  # b, lq, lk, h, hk, d, window, sinks, causal: nothing is split, several tiles are walked
    (16, 200, 200, 32, 32, 64, 0, 0, True), (13, 330, 330, 14, 14, 64, 40, 0, False), (9, 300, 300, 20, 20, 64, 70, 0, True), (17, 260, 260, 12, 6, 128, 0, 0, True),
    (16, 201, 333, 20, 20, 32, 0, 0, True), (15, 261, 261, 6, 6, 96, 100, 0, False), (11, 290, 290, 16, 8, 80, 33, 0, True), (30, 131, 131, 18, 9, 40, 0, 0, False)]


@DTS
@pytest.mark.parametrize('case', WHOLE, ids=lambda c: '-'.join(map(str, c)))
def test_attention_unsplit(case, dt):
    b, lq, lk, h, hk, d, window, sinks, causal = case
    assert scratch(*case, dt) == (0, 0)
    run_attention(case, dt)


MIXED = [(18, 330, 330, 12, 12, 64, 8, 3, True), (9, 400, 400, 20, 10, 128, 8, 130, True), (10, 333, 333, 10, 10, 96, 5, 4, False), (16, 290, 290, 18, 18, 48, 9, 2, True)]


@DTS
@pytest.mark.parametrize('case', MIXED, ids=lambda c: '-'.join(map(str, c)))
def test_attention_sink_blocks_split_beside_whole_ones(case, dt):
    b, lq, lk, h, hk, d, window, sinks, causal = case
    fwd, bwd = scratch(*case, dt)
    per = b * hk * 256 * d * 4                                           # one block of 128 keys of every head, one part
    nblk, nsb = -(-lk // 128), -(-sinks // 128)
    assert fwd == 0 and bwd % (per * nsb) == 0 and 1 < bwd // (per * nsb) <= 32 and nsb < nblk
    # (were every block split, the scratch would hold nblk blocks: not a multiple, or more parts than a block has query tiles)
    tiles = -(-lq // (64 if dt == F16 else 32)) * (h // hk)
    assert bwd // (per * nsb) <= tiles
    run_attention(case, dt)


def run_attention(case, dt):
    b, lq, lk, h, hk, d, window, sinks, causal = case
    q, k, v, go = (rnd(i, *s, dt=dt) for i, s in enumerate(((b, lq, h, d), (b, lk, hk, d), (b, lk, hk, d), (b, lq, h, d))))
    kw = dict(window=window, sinks=sinks, causal=causal)
    ref = R.attention(q, k, v, go=go, **kw)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = T().window_attention(*leaves, **kw)
    R.within('o', o, *ref['o'])
    for n, t in zip(('gq', 'gk', 'gv'), torch.autograd.grad(o, leaves, go.cuda())):
        R.within(n, t, *ref[n])


def staircase(lq, lk, h, hk, dt, seed, spread):
    """scores (in powers of two, scale = ln 2) that climb from key tile to key tile by a step of the query's own: from less than the slack of the
    running maximum to hundreds, lanes of one wave apart; within a tile they vary by `spread`"""
    d = 64
    q, k, v, go = (rnd(seed + i, *s, dt=dt) for i, s in enumerate(((1, lq, h, d), (1, lk, hk, d), (1, lk, hk, d), (1, lq, h, d))))
    q, k = q * spread, k * 0.125
    step = torch.tensor([0.5, 3.9, 4.1, 7.9, 8.1, 15.9, 40.0, 300.0, -5.0])
    q[..., 0] = step[(torch.arange(lq)[:, None] * 5 + torch.arange(h)[None]) % len(step)].to(dt)
    k[..., 0] = (torch.arange(lk) // 64).to(dt)[None, :, None]
    return q, k, v, go


@DTS
@pytest.mark.parametrize('b,lq,lk,h,hk,causal', [(6, 300, 300, 16, 16, False), (6, 300, 300, 16, 16, True), (8, 270, 330, 20, 10, True)])
def test_running_maximum_over_several_tiles(b, lq, lk, h, hk, causal, dt):
    assert scratch(b, lq, lk, h, hk, 64, 0, 0, causal, dt)[0] == 0
    parts = [staircase(lq, lk, h, hk, dt, 100 * i, 0.3) for i in range(b)]
    q, k, v, go = (torch.cat(t) for t in zip(*parts))
    kw = dict(causal=causal, scale=math.log(2.0))
    ref = R.attention(q, k, v, go=go, **kw)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = T().window_attention(*leaves, **kw)
    R.within('o', o, *ref['o'])
    for n, t in zip(('gq', 'gk', 'gv'), torch.autograd.grad(o, leaves, go.cuda())):
        R.within(n, t, *ref[n])


@DTS
@pytest.mark.parametrize('lq,h,hk', [(1, 8, 2), (3, 4, 4)])
def test_running_maximum_of_a_split_decode(lq, h, hk, dt):
    """several key tiles a split: the maximum climbs within a split and between splits"""
    lk = 64 * 64 * 3 + 7
    q, k, v, _ = staircase(lq, lk, h, hk, dt, 5, 0.3)
    k[..., 0] = ((torch.arange(lk) // 64) % 7).to(dt)[None, :, None]
    kw = dict(causal=True, scale=math.log(2.0))
    R.within('o', T().window_attention(*cuda(q, k, v), **kw), *R.attention(q, k, v, **kw)['o'])


@pytest.mark.parametrize('case', [(16, 2048, 2048, 4, 4, 64, 256, 4, False), (2, 4096, 4096, 16, 4, 128, 1024, 4, True), (3, 777, 777, 6, 2, 40, 129, 3, True)],
                         ids=lambda c: '-'.join(map(str, c)))
def test_large_calls_repeat_bit_for_bit(case):
    b, lq, lk, h, hk, d, window, sinks, causal = case
    q, k, v, go = (torch.randn(*s, device='cuda').to(F16) for s in ((b, lq, h, d), (b, lk, hk, d), (b, lk, hk, d), (b, lq, h, d)))
    first = None
    for _ in range(4):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = T().window_attention(*leaves, window=window, sinks=sinks, causal=causal)
        got = [o.detach(), *torch.autograd.grad(o, leaves, go)]
        assert first is None or all(torch.equal(a, r) for a, r in zip(got, first))
        first = first or got


@pytest.mark.parametrize('b,lk,h,hk,d,window', [(8, 32768, 32, 8, 128, 0), (1, 700, 8, 2, 64, 512)])
def test_single_tokens_repeat_bit_for_bit(b, lk, h, hk, d, window):
    q, k, v = (torch.randn(*s, device='cuda').to(F16) for s in ((b, 1, h, d), (b, lk, hk, d), (b, lk, hk, d)))
    first = T().window_attention(q, k, v, window=window, sinks=4, causal=True)
    for _ in range(4):
        assert torch.equal(T().window_attention(q, k, v, window=window, sinks=4, causal=True), first)


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------
# rows enough that every workgroup (1024 at most) walks several, the last walk partly empty, forward and backward: narrow rows in lane groups, rows of one
# wave, rows of a whole workgroup; 16-byte and element-wise accesses
@DTS
@pytest.mark.parametrize('rows,c', [(140001, 40), (40003, 33), (5001, 2056), (4999, 1100), (70001, 192), (4600, 1027)])
def test_layer_norm_many_rows(rows, c, dt):
    x, go = rnd(1, rows, c, dt=dt, scale=1.5, shift=0.7), rnd(2, rows, c, dt=dt)
    w, b = rnd(3, c, scale=0.3, shift=1.0), rnd(4, c, scale=0.5)
    ref = R.layer_norm(x, w, b, 1e-5, go)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = T().layer_norm(*leaves)
    for n, t in zip(('y', 'gx', 'gw', 'gb'), (y, *torch.autograd.grad(y, leaves, go.cuda()))):
        R.within(n, t, *ref[n])


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------
@DTS
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('b,l,h,hk', [(3, 9001, 6, 3), (2, 23011, 5, 0), (1, 30011, 4, 9)])
def test_rope_four_heads_a_thread(b, l, h, hk, interleaved, dt):
    """above the size from which a thread takes four heads: head counts that four does not divide, channels that pass through"""
    d, sections = 64, (0, 12, 12)
    assert b * l * (h + hk) * (5 if dt == F16 and not interleaved else 8) >= 1 << 20
    q, k = rnd(1, b, l, h, d, dt=dt), rnd(2, b, l, hk, d, dt=dt) if hk else None
    pos = torch.randint(0, 4000, (b, l, 3), generator=torch.Generator().manual_seed(5))
    a, c = T().rope_axes(q.cuda(), None if k is None else k.cuda(), pos.cuda(), sections, interleaved=interleaved, spectrum='axis')
    R.within('q', a, *R.rope(q, pos, sections, 10000.0, interleaved, 'axis'))
    if hk:
        R.within('k', c, *R.rope(k, pos, sections, 10000.0, interleaved, 'axis'))
