"""Token operators (multiyolov5_amd/utils/tokens.py) against their 64-bit definitions (tests/token_ref.py, which derives the tolerances)."""
import gc
import math

import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def T():
    from multiyolov5_amd.utils import tokens
    return tokens


def rnd(seed, *shape, dt=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dt)


def cuda(*ts):
    out = [None if t is None else t.cuda() for t in ts]
    return out if len(out) > 1 else out[0]


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------
LN_SHAPES = [(1, 1), (3, 2), (1, 512), (5, 8), (7, 31), (64, 32), (33, 64), (130, 96), (65, 128), (257, 192), (100, 256), (9, 1003), (17, 1024),
             (6, 2048), (5, 2056), (3, 4096), (4, 5000), (2, 8192), (2, 8195), (2, 20000), (1, 33001), (700, 40)]


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
@pytest.mark.parametrize('rows,c', LN_SHAPES)
def test_layer_norm(rows, c, dt):
    x, go = rnd(1, rows, c, dt=dt, scale=1.5, shift=0.7), rnd(2, rows, c, dt=dt)
    w, b = rnd(3, c, scale=0.3, shift=1.0), rnd(4, c, scale=0.5)
    ref = R.layer_norm(x, w, b, 1e-5, go)
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x, w, b))
    y = T().layer_norm(xd, wd, bd)
    assert y.dtype == dt and y.is_contiguous()
    g = torch.autograd.grad(y, (xd, wd, bd), go.cuda())
    for n, t in zip(('y', 'gx', 'gw', 'gb'), (y, *g)):
        R.within(n, t, *ref[n])
    with torch.no_grad():
        R.within('inference', T().layer_norm(xd, wd, bd), *ref['y'])
        assert torch.equal(T().layer_norm(xd, wd, bd), y)


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
@pytest.mark.parametrize('c', [24, 40, 33])
def test_layer_norm_views(c, dt):
    """slices of a wider buffer, a channels-last map, transposed channels, odd offsets; parameters missing"""
    x, go = rnd(1, 6, 5, 7, c, dt=dt), rnd(2, 6, 5, 7, c, dt=dt)
    ref = R.layer_norm(x.reshape(-1, c), None, None, 1e-3, go.reshape(-1, c))

    def views():
        for pad, off in ((8, 0), (8, 8), (3, 1)):
            buf = torch.full((6, 5, 9, c + pad), math.nan, dtype=dt, device='cuda')
            v = buf[:, :, 1:8, off:off + c]
            v.copy_(x.cuda())
            yield f'slice {pad} {off}', v
        yield 'channels last', x.cuda().permute(0, 3, 1, 2).contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)
        yield 'channels first', x.cuda().permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
        yield 'swapped axes', x.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    for name, v in views():
        v = v.detach().requires_grad_()
        y = T().layer_norm(v, None, None, 1e-3)
        gx, = torch.autograd.grad(y, v, go.cuda().transpose(1, 2).contiguous().transpose(1, 2))
        assert y.shape == x.shape
        R.within(name + ' y', y.reshape(-1, c), *ref['y'])
        R.within(name + ' gx', gx.reshape(-1, c), *ref['gx'])


def test_layer_norm_extremes():
    """a large common offset (no cancellation of E[x^2] - mean^2), a constant row, a row with an infinity, the largest fp16 values"""
    x = torch.cat([rnd(1, 4, 200, scale=0.01, shift=300.0), torch.full((2, 200), 7.25), rnd(2, 2, 200)])
    x[6, 3] = math.inf
    y = T().layer_norm(x.cuda())
    ref = R.layer_norm(x[[0, 1, 2, 3, 4, 5, 7]], None, None, 1e-5)['y']
    R.within('rows', y[[0, 1, 2, 3, 4, 5, 7]], *ref)
    assert bool(y[6].isnan().all()) and bool((y[4:6] == 0).all())
    z = torch.full((3, 64), 65504.0, dtype=F16)
    z[:, ::2] = -65504.0
    R.within('fp16 range', T().layer_norm(z.cuda()), *R.layer_norm(z, None, None, 1e-5)['y'])


def test_layer_norm_empty_and_partial_gradients():
    x = torch.zeros(0, 16, device='cuda', requires_grad=True)
    w = torch.ones(16, device='cuda', requires_grad=True)
    y = T().layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert gx.shape == (0, 16) and bool((gw == 0).all())
    v, gv = rnd(7, 40).cuda().requires_grad_(), rnd(8, 40)                   # a single row without a row dimension
    y = T().layer_norm(v)
    ref = R.layer_norm(v.detach().cpu()[None], None, None, 1e-5, gv[None])
    R.within('one row', y[None], *ref['y'])
    R.within('one row gx', torch.autograd.grad(y, v, gv.cuda())[0][None], *ref['gx'])
    x, go, w = rnd(1, 50, 24), rnd(2, 50, 24), rnd(3, 24)
    ref = R.layer_norm(x, w, None, 1e-5, go)
    xd, wd = x.cuda(), w.cuda().requires_grad_()
    gw, = torch.autograd.grad(T().layer_norm(xd, wd), wd, go.cuda())
    R.within('gw alone', gw, *ref['gw'])
    xd = x.cuda().requires_grad_()
    gx, = torch.autograd.grad(T().layer_norm(xd, w.cuda()), xd, go.cuda().expand(50, 24))
    R.within('gx alone', gx, *ref['gx'])
    s = rnd(5, 24).cuda()                            # a gradient that is broadcast over the rows (stride 0)
    gx, = torch.autograd.grad(T().layer_norm(xd, w.cuda()), xd, s.expand(50, 24))
    R.within('broadcast', gx, *R.layer_norm(x, w, None, 1e-5, s.cpu().expand(50, 24))['gx'])


def test_layer_norm_c_entry_accumulates_in_place():
    """acc_x / acc_params add to what is there; out may be x, gx may be gout"""
    import ctypes as C
    from multiyolov5_amd import _lib as L
    lib = L.lib()
    for rows, c, dt in ((37, 48, F16), (12, 35, F32), (5, 4000, F16)):
        x, go, w, b = rnd(1, rows, c, dt=dt), rnd(2, rows, c, dt=dt), rnd(3, c), rnd(4, c)
        ref = R.layer_norm(x, w, b, 1e-5, go)
        xd, god, wd, bd = cuda(x, go, w, b)

        def desc(t):
            return L.Tensor(t.data_ptr(), 1, 1, rows, c, rows * c, rows * c, c, L.DT[t.dtype], 0)
        saved = torch.empty(2 * rows, device='cuda')
        y = xd.clone()
        assert lib.myolo_layernorm_fwd(C.byref(desc(y)), L.ptr(wd), L.ptr(bd), 1e-5, C.byref(desc(y)), L.ptr(saved), L.stream_ptr()) == 0
        R.within('in place', y, *ref['y'])
        ws = torch.empty(lib.myolo_layernorm_ws_bytes(rows, c) // 4, device='cuda')
        dg, db = torch.full((c,), 2.0, device='cuda'), torch.full((c,), -3.0, device='cuda')
        assert lib.myolo_layernorm_bwd(C.byref(desc(god)), C.byref(desc(xd)), L.ptr(saved), L.ptr(wd), C.byref(desc(god)), 0, L.ptr(dg), L.ptr(db),
                                       1, L.ptr(ws), ws.numel() * 4, L.stream_ptr()) == 0
        torch.cuda.synchronize()
        # (the backward writes gx over gout only after it has read the row: the parameter sums see the incoming gradient)
        R.within('gx over gout', god, *ref['gx'])
        R.within('dgamma +=', dg.double().cpu() - 2.0, ref['gw'][0], ref['gw'][1] + 4 * R.E * (ref['gw'][0].abs() + 2))
        R.within('dbeta +=', db.double().cpu() + 3.0, ref['gb'][0], ref['gb'][1] + 4 * R.E * (ref['gb'][0].abs() + 3))
        gx = torch.ones(rows, c, dtype=dt, device='cuda')
        god.copy_(go)
        assert lib.myolo_layernorm_bwd(C.byref(desc(god)), C.byref(desc(xd)), L.ptr(saved), L.ptr(wd), C.byref(desc(gx)), 1, None, None,
                                       0, None, 0, L.stream_ptr()) == 0
        v = ref['gx'][0] + 1
        R.within('gx +=', gx, v, ref['gx'][1] + R.half_step(dt) * (v.abs() + 1))


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------
ROPE = [  # b, l, h, hk, d, sections, interleaved, spectrum, far
    (1, 1, 1, 1, 8, (4,), False, 'shared', 0), (1, 1, 32, 8, 128, (16, 24, 24), False, 'shared', 100000), (2, 37, 4, 2, 64, (0, 16, 16), False, 'axis', 50),
    (2, 37, 4, 4, 64, (8, 12, 12), True, 'shared', 1000000), (3, 5, 3, 1, 96, (12, 18, 18), True, 'axis', 7), (1, 130, 2, 2, 40, (2, 3, 5), False, 'shared', 9),
    (2, 9, 5, 5, 22, (3, 2, 4), False, 'axis', 12345678), (2, 9, 5, 5, 23, (3, 2, 4), True, 'shared', 3), (1, 20, 2, 1, 256, (32, 32, 32, 32), False, 'shared', 5),
    (1, 6, 2, 0, 64, (32,), False, 'shared', 1 << 28), (2, 8, 1, 1, 16, (0, 0), False, 'shared', 1), (4, 300, 8, 8, 32, (4, 6, 6), False, 'axis', 100)]


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
@pytest.mark.parametrize('b,l,h,hk,d,sections,interleaved,spectrum,far', ROPE)
def test_rope(b, l, h, hk, d, sections, interleaved, spectrum, far, dt):
    q, k = rnd(1, b, l, h, d, dt=dt), rnd(2, b, l, hk, d, dt=dt) if hk else None
    gq, gk = rnd(3, b, l, h, d, dt=dt), rnd(4, b, l, hk, d, dt=dt) if hk else None
    pos = torch.randint(-(far // 2), far + 1, (b, l, len(sections)), generator=torch.Generator().manual_seed(5))
    kw = dict(interleaved=interleaved, spectrum=spectrum)
    qd, kd = q.cuda().requires_grad_(), k.cuda().requires_grad_() if hk else None
    a, c = T().rope_axes(qd, kd, pos.cuda(), sections, **kw)
    R.within('q', a, *R.rope(q, pos, sections, 10000.0, interleaved, spectrum))
    if hk:
        R.within('k', c, *R.rope(k, pos, sections, 10000.0, interleaved, spectrum))
        g = torch.autograd.grad((a, c), (qd, kd), cuda(gq, gk))
        R.within('gk', g[1], *R.rope(gk, pos, sections, 10000.0, interleaved, spectrum, True))
    else:
        assert c is None
        g = torch.autograd.grad(a, qd, gq.cuda())
    R.within('gq', g[0], *R.rope(gq, pos, sections, 10000.0, interleaved, spectrum, True))


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
def test_rope_views_and_shared_positions(dt):
    """q and k as slices of one projection [B, L, (H + 2 Hk) D]; positions shared by the batch ([L, A] and [1, L, A]) and as transposed views;
    one missing output gradient"""
    b, l, h, hk, d = 2, 19, 4, 2, 32
    qkv = rnd(1, b, l, (h + 2 * hk) * d + 3, dt=dt)
    pos = torch.randint(0, 500, (l, 3), generator=torch.Generator().manual_seed(2))
    for off in (0, 3):                               # 3: rows that start off a 16-byte boundary
        buf = qkv.cuda()
        q = buf[..., off:off + h * d].view(b, l, h, d) if off == 0 else buf[..., off:off + h * d].unflatten(-1, (h, d))
        k = buf[..., off + h * d:off + (h + hk) * d].unflatten(-1, (hk, d))
        for pv in (pos.cuda(), pos.cuda()[None], pos.t().contiguous().t().cuda(), pos.cuda().expand(b, l, 3)):
            a, c = T().rope_axes(q, k, pv, (4, 6, 6))
            p3 = pos.expand(b, l, 3)
            R.within('q', a, *R.rope(q.cpu(), p3, (4, 6, 6), 10000.0, False, 'shared'))
            R.within('k', c, *R.rope(k.cpu(), p3, (4, 6, 6), 10000.0, False, 'shared'))
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    a, _ = T().rope_axes(q, k, pos.cuda(), (4, 6, 6))
    gq, gk = torch.autograd.grad(a.sum(), (q, k))
    assert bool((gk == 0).all()) and gq.shape == q.shape


def test_rope_c_entry_in_place():
    from multiyolov5_amd import _lib as L
    import ctypes as C
    q, k = rnd(1, 2, 11, 3, 48, dt=F16), rnd(2, 2, 11, 1, 48, dt=F16)
    pos = torch.randint(0, 90, (2, 11, 2), generator=torch.Generator().manual_seed(3))
    for sections in ((8, 16), (3, 4)):
        qd, kd, pd = cuda(q, k, pos)
        turns, axis = T().rope_table(sections)
        d = L.RopeDesc()
        d.q, d.qo, d.k, d.ko, d.pos = qd.data_ptr(), qd.data_ptr(), kd.data_ptr(), kd.data_ptr(), pd.data_ptr()
        d.qs = d.qos = (C.c_int64 * 3)(*qd.stride()[:3])
        d.ks = d.kos = (C.c_int64 * 3)(*kd.stride()[:3])
        d.ps, d.turns, d.axis = (C.c_int64 * 3)(*pd.stride()), C.addressof(turns), C.addressof(axis)
        d.b, d.l, d.hq, d.hk, d.d, d.npair, d.naxis, d.dtype = 2, 11, 3, 1, 48, sum(sections), 2, L.DT[F16]
        assert L.lib().myolo_rope(C.byref(d), L.stream_ptr()) == 0
        R.within('q', qd, *R.rope(q, pos, sections, 10000.0, False, 'shared'))
        R.within('k', kd, *R.rope(k, pos, sections, 10000.0, False, 'shared'))


# ---- attention -------------------------------------------------------------------------------------------------------------------------
ATTN = [  # b, lq, lk, h, hk, d, window, sinks, causal, lens, starts
    (1, 1, 1, 1, 1, 8, 0, 0, False, None, None),
    (2, 5, 5, 2, 2, 16, 0, 0, True, None, None),
    (1, 33, 33, 1, 1, 32, 0, 0, False, None, None),
    (2, 64, 64, 4, 2, 64, 0, 0, True, None, None),
    (1, 65, 65, 2, 1, 40, 1, 0, True, None, None),
    (1, 130, 130, 2, 2, 64, 1, 0, False, None, None),
    (2, 129, 129, 3, 1, 96, 17, 3, True, None, None),
    (2, 129, 129, 3, 3, 128, 17, 3, False, None, None),
    (1, 200, 200, 8, 1, 32, 64, 70, True, None, None),
    (1, 257, 257, 2, 1, 128, 100, 1000, False, None, None),
    (1, 300, 300, 6, 2, 72, 33, 5, True, None, None),
    (3, 77, 77, 2, 2, 64, 20, 2, True, (77, 0, 31), (0, 0, 0)),
    (3, 77, 77, 2, 2, 64, 20, 0, False, (77, 0, 31), (0, 0, 0)),
    (2, 40, 90, 4, 2, 64, 0, 0, True, None, None),
    (2, 40, 90, 4, 2, 64, 16, 2, True, (90, 50), (50, 10)),
    (2, 90, 40, 2, 1, 64, 0, 0, True, None, None),          # more queries than keys: the first 50 see nothing
    (2, 90, 40, 2, 1, 64, 8, 4, False, None, None),
    (3, 50, 60, 2, 2, 48, 10, 3, True, None, (-20, 500, 1 << 30)),
    (3, 50, 60, 2, 2, 48, 10, 3, False, (60, 70, -5), (-(1 << 31), (1 << 31) - 1, 0)),
    (2, 3, 0, 2, 1, 64, 0, 0, False, None, None),
    (2, 0, 7, 2, 1, 64, 0, 0, False, None, None),
    (0, 4, 7, 2, 1, 64, 0, 0, False, None, None)]
DECODE = [
    (1, 1, 700, 8, 2, 64, 512, 4, True, None, None),
    (3, 1, 1500, 8, 2, 128, 0, 0, True, (1500, 1, 777), (1499, 0, 776)),
    (2, 1, 999, 4, 4, 32, 0, 0, True, None, None),
    (1, 5, 2000, 12, 4, 96, 300, 7, True, (1203,), (1198,)),
    (1, 1, 64, 1, 1, 8, 0, 0, False, None, None),
    (2, 2, 5000, 16, 1, 128, 0, 0, True, (5000, 0), (4998, -2)),
    (1, 1, 4100, 40, 1, 64, 64, 0, True, None, None),
    (1, 130, 3000, 1, 1, 64, 0, 0, True, None, None)]


def i32(v):
    return None if v is None else torch.tensor(v, dtype=torch.int64).clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)


def attn_inputs(case, dt, seed=1):
    b, lq, lk, h, hk, d = case[:6]
    return [rnd(seed + i, *s, dt=dt) for i, s in enumerate(((b, lq, h, d), (b, lk, hk, d), (b, lk, hk, d), (b, lq, h, d)))]


def attn_kw(case, dev=None):
    kw = dict(window=case[6], sinks=case[7], causal=case[8], lens=i32(case[9]), starts=i32(case[10]))
    if dev:
        kw = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in kw.items()}
    return kw


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
@pytest.mark.parametrize('case', ATTN + DECODE, ids=lambda c: '-'.join(map(str, c[:9])).replace(' ', ''))
def test_attention(case, dt):
    q, k, v, go = attn_inputs(case, dt)
    ref = R.attention(q, k, v, go=go, **attn_kw(case))
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = T().window_attention(*leaves, **attn_kw(case, 'cuda'))
    R.within('o', o, *ref['o'])
    g = torch.autograd.grad(o, leaves, go.cuda())
    for n, t in zip(('gq', 'gk', 'gv'), g):
        R.within(n, t, *ref[n])
    with torch.no_grad():
        assert torch.equal(T().window_attention(*leaves, **attn_kw(case, 'cuda')), o)


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
@pytest.mark.parametrize('case', [ATTN[11], ATTN[14], ATTN[17], DECODE[1], DECODE[3], (2, 70, 130, 2, 1, 64, 0, 0, True, None, (3, 40))],
                         ids=['padded', 'cache', 'far', 'decode', 'window', 'tail'])
def test_attention_ignores_what_nobody_sees(case, dt):
    """NaN and infinities in keys and values behind the valid length, in front of the window, past the last position; NaN in queries that see
    nothing and in their incoming gradient"""
    q, k, v, go = attn_inputs(case, dt)
    kw = attn_kw(case)
    see = R.visible(case[0], case[1], case[2], case[6], case[7], case[8], kw['lens'], kw['starts'])
    unseen = ~see.any(1)
    blind = ~see.any(2)
    assert bool(unseen.any())
    ref = R.attention(q, k, v, go=go, **kw)
    k[unseen], v[unseen] = math.nan, math.inf
    q[blind], go[blind] = math.nan, math.nan
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = T().window_attention(*leaves, **attn_kw(case, 'cuda'))
    R.within('o', o, *ref['o'])
    gq, gk, gv = torch.autograd.grad(o, leaves, go.cuda())
    R.within('gq', gq, *ref['gq'])
    R.within('gk', gk, *ref['gk'])
    R.within('gv', gv, *ref['gv'])


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
def test_attention_views(dt):
    """slices of one projection, [B, H, L, D] layouts, rows off a 16-byte boundary (copied), gradients that arrive transposed or broadcast"""
    b, l, h, hk, d = 2, 70, 4, 2, 32
    qkv = rnd(1, b, l, (h + 2 * hk) * d, dt=dt)
    q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], -1))
    go = rnd(2, b, l, h, d, dt=dt)
    kw = dict(window=13, sinks=2, causal=True)
    ref = R.attention(q, k, v, go=go, **kw)

    def check(name, leaves, g):
        leaves = [t.detach().requires_grad_() for t in leaves]
        o = T().window_attention(*leaves, **kw)
        R.within(name, o, *ref['o'])
        for n, t in zip(('gq', 'gk', 'gv'), torch.autograd.grad(o, leaves, g)):
            R.within(name + ' ' + n, t, *ref[n])
    dev = qkv.cuda()
    check('slices', [t.unflatten(-1, (-1, d)) for t in dev.split([h * d, hk * d, hk * d], -1)], go.cuda())
    check('heads first', [t.cuda().transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)], go.cuda().transpose(1, 2).contiguous().transpose(1, 2))
    off = torch.zeros(b * l * (h + 2 * hk) * d + 1, dtype=dt, device='cuda')[1:].view(b, l, -1)
    off.copy_(qkv)
    check('off a boundary', [t.unflatten(-1, (-1, d)) for t in off.split([h * d, hk * d, hk * d], -1)], go.cuda())
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    g1 = torch.autograd.grad(T().window_attention(*leaves, **kw).sum(), leaves)
    refs = R.attention(q, k, v, go=torch.ones_like(go), **kw)
    for n, t in zip(('gq', 'gk', 'gv'), g1):
        R.within('ones ' + n, t, *refs[n])


def test_attention_partial_gradients_and_scale():
    case = ATTN[6]
    q, k, v, go = attn_inputs(case, F16)
    for scale in (None, 0.01, 1.7):
        ref = R.attention(q, k, v, go=go, scale=scale, **attn_kw(case))
        for which in ((0,), (1,), (2,), (0, 2)):
            leaves = [t.cuda().requires_grad_(i in which) for i, t in enumerate((q, k, v))]
            o = T().window_attention(*leaves, scale=scale, **attn_kw(case, 'cuda'))
            R.within('o', o, *ref['o'])
            g = torch.autograd.grad(o, [leaves[i] for i in which], go.cuda())
            for i, t in zip(which, g):
                R.within('gqgkgv'[2 * i:2 * i + 2], t, *ref['gqgkgv'[2 * i:2 * i + 2]])


@pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])
def test_attention_large_scores(dt):
    """scores of several hundred: the running maximum carries them; rows dominated by one key"""
    q, k, v, go = attn_inputs((1, 150, 150, 2, 1, 64), dt)
    q, k = q * 6, k * 6
    kw = dict(window=90, sinks=2, causal=True)
    ref = R.attention(q, k, v, go=go, **kw)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = T().window_attention(*leaves, **kw)
    R.within('o', o, *ref['o'])
    for n, t in zip(('gq', 'gk', 'gv'), torch.autograd.grad(o, leaves, go.cuda())):
        R.within(n, t, *ref[n])


def test_attention_offsets_past_32_bits():
    """a cache whose rows lie 2^26 elements apart: byte offsets up to 9 * 10^9"""
    lk, d, step = 70, 64, 1 << 26
    buf = torch.empty((lk - 1) * step + 2 * d, dtype=F16, device='cuda')
    k, v = buf.as_strided((1, lk, 1, d), (step, step, d, 1)), buf[d:].as_strided((1, lk, 1, d), (step, step, d, 1))
    q0, k0, v0, go = attn_inputs((1, 3, lk, 2, 1, d), F16)
    k.copy_(k0)
    v.copy_(v0)
    ref = R.attention(q0, k0, v0, causal=True, go=go)
    leaves = [t.requires_grad_() for t in (q0.cuda(), k.detach(), v.detach())]
    o = T().window_attention(*leaves, causal=True)
    R.within('o', o, *ref['o'])
    for n, t in zip(('gq', 'gk', 'gv'), torch.autograd.grad(o, leaves, go.cuda())):
        R.within(n, t, *ref[n])


def test_attention_repeats_bit_for_bit():
    case = (2, 300, 300, 8, 2, 64, 70, 4, True, None, None)
    q, k, v, go = attn_inputs(case, F16)

    def once():
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        o = T().window_attention(*leaves, **attn_kw(case, 'cuda'))
        return [o, *torch.autograd.grad(o, leaves, go.cuda())]
    first = once()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


# ---- gradients against differences -----------------------------------------------------------------------------------------------------
def test_gradients_against_differences():
    """the directional derivative of the 64-bit forward, by central differences, is the inner product with the operators' gradient"""
    eps = 1e-4

    def close(f, xs, grads, seed):
        for i, (x, g) in enumerate(zip(xs, grads)):
            d = rnd(seed + i, *x.shape).double()
            up, dn = ([t + s * eps * d if j == i else t for j, t in enumerate(xs)] for s in (1, -1))
            num = (f(*up) - f(*dn)) / (2 * eps)
            got = (g.double().cpu() * d).sum()
            # central differences: eps^2 of the third derivative (of order of the value); the gradients: 32-bit arithmetic
            assert abs(float(got - num)) <= 1e-5 * float((g.double().cpu() * d).abs().sum()) + 1e-6, (i, float(got), float(num))
    x, w, b, go = rnd(1, 9, 33), rnd(2, 33), rnd(3, 33), rnd(4, 9, 33)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    g = torch.autograd.grad(T().layer_norm(*leaves), leaves, go.cuda())
    close(lambda x, w, b: (R.layer_norm(x, w, b, 1e-5)['y'][0] * go.double()).sum(), [t.double() for t in (x, w, b)], g, 10)
    case = (1, 45, 45, 4, 2, 24, 9, 2, True, None, None)
    q, k, v, go = attn_inputs(case, F32)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    g = torch.autograd.grad(T().window_attention(*leaves, **attn_kw(case)), leaves, go.cuda())
    close(lambda q, k, v: (R.attention(q, k, v, **attn_kw(case))['o'][0] * go.double()).sum(), [t.double() for t in (q, k, v)], g, 20)
    q, k, gq, gk = rnd(1, 1, 6, 2, 16), rnd(2, 1, 6, 1, 16), rnd(3, 1, 6, 2, 16), rnd(4, 1, 6, 1, 16)
    pos = torch.randint(0, 40, (1, 6, 2), generator=torch.Generator().manual_seed(7))
    leaves = [t.cuda().requires_grad_() for t in (q, k)]
    g = torch.autograd.grad(T().rope_axes(*leaves, pos.cuda(), (3, 4)), leaves, cuda(gq, gk))
    close(lambda q, k: (R.rope(q, pos, (3, 4), 1e4, False, 'shared')[0] * gq.double()).sum() +
          (R.rope(k, pos, (3, 4), 1e4, False, 'shared')[0] * gk.double()).sum(), [t.double() for t in (q, k)], g, 30)


# ---- a run of them together, streams, graphs -------------------------------------------------------------------------------------------
def _layer(x, w, b, wqkv, pos, kw, heads, kv, d):
    """norm -> projection -> positions -> attention, as a layer uses them"""
    y = T().layer_norm(x, w, b)
    qkv = y @ wqkv
    q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv.split([heads * d, kv * d, kv * d], -1))
    q, k = T().rope_axes(q, k, pos, (d // 4, d // 4), spectrum='axis')
    return T().window_attention(q, k, v, **kw)


def _layer_inputs():
    b, hh, ww, c, heads, kv, d = 2, 6, 9, 48, 4, 2, 16
    x, w, bb = rnd(1, b, hh * ww, c), rnd(2, c, scale=0.1, shift=1.0), rnd(3, c, scale=0.1)
    wq = rnd(4, c, (heads + 2 * kv) * d, scale=c ** -0.5)
    pos = torch.stack(torch.meshgrid(torch.arange(hh), torch.arange(ww), indexing='ij'), -1).reshape(-1, 2)
    return (x, w, bb, wq), pos, dict(window=2 * ww, sinks=3), (heads, kv, d), rnd(5, b, hh * ww, heads, d)


def test_chain_matches_the_definitions():
    leaves, pos, kw, dims, go = _layer_inputs()
    heads, kv, d = dims
    g64 = [t.double().requires_grad_() for t in leaves]
    x, w, b, wq = g64
    y = torch.nn.functional.layer_norm(x, (x.shape[-1],), w, b, 1e-5)
    q, k, v = (t.unflatten(-1, (-1, d)) for t in (y @ wq).split([heads * d, kv * d, kv * d], -1))
    f = 10000.0 ** -(torch.arange(d // 4, dtype=torch.float64) / (d // 4))
    ang = (pos.double()[:, :, None] * f).flatten(1)[None, :, None]

    def turn(t):
        u, z = t.chunk(2, -1)
        return torch.cat([u * ang.cos() - z * ang.sin(), z * ang.cos() + u * ang.sin()], -1)
    q, k = turn(q), turn(k)
    see = R.visible(1, q.shape[1], q.shape[1], kw['window'], kw['sinks'], False, None, None)[:, None]
    kk, vv = (t.repeat_interleave(heads // kv, 2).transpose(1, 2) for t in (k, v))
    p = (q.transpose(1, 2) @ kk.transpose(2, 3) * d ** -0.5).masked_fill(~see, -math.inf).softmax(-1)
    o = (p @ vv).transpose(1, 2)
    ref = [o, *torch.autograd.grad(o, g64, go.double())]
    dl = [t.cuda().requires_grad_() for t in leaves]
    got = _layer(*dl, pos.cuda(), kw, *dims)
    got = [got, *torch.autograd.grad(got, dl, go.cuda())]
    for n, a, r in zip(('o', 'gx', 'gw', 'gb', 'gwqkv'), got, ref):
        # 32-bit chain of five operators, each good to some tens of 2^-24 of its inputs' size (test_* above): 2^-24 * 1000 of the norm
        r = r.detach()
        assert float((a.detach().double().cpu() - r).norm()) <= 1000 * R.E * float(r.norm()), n


def test_on_another_stream_and_captured():
    """the calls on a side stream; forward and backward captured and replayed with new inputs while an eager graph of other leaves lives"""
    leaves, pos, kw, dims, go = _layer_inputs()
    posd, god = pos.cuda(), go.cuda()
    dl = [t.cuda().requires_grad_() for t in leaves]
    alive = _layer(*dl, posd, kw, *dims)                            # an eager graph that stays alive throughout
    want = [alive.detach().clone(), *torch.autograd.grad(alive, dl, god, retain_graph=True)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sl = [t.detach().clone().requires_grad_() for t in dl]
        o = _layer(*sl, posd, kw, *dims)
        got = [o.detach(), *torch.autograd.grad(o, sl, god)]
    torch.cuda.current_stream().wait_stream(s)
    for a, r in zip(got, want):
        assert torch.equal(a, r)
    static = [t.detach().clone().requires_grad_() for t in dl]
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(_layer(*static, posd, kw, *dims), static, god)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = _layer(*static, posd, kw, *dims)
        res = [o, *torch.autograd.grad(o, static, god)]
    for rep in range(4):
        new = [rnd(50 + 10 * rep + i, *t.shape, scale=0.3, shift=0.2).cuda() for i, t in enumerate(leaves)]
        with torch.no_grad():
            for a, b in zip(static, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        el = [t.requires_grad_() for t in new]
        e = _layer(*el, posd, kw, *dims)
        for a, r in zip(res, [e, *torch.autograd.grad(e, el, god)]):
            assert torch.equal(a, r)
    again = torch.autograd.grad(alive, dl, god)
    assert all(torch.equal(a, r) for a, r in zip(again, want[1:]))


def test_captured_decode_follows_the_lengths():
    """one captured single-token call serves a growing cache: lens and starts are read on the device"""
    b, cap, h, hk, d = 2, 900, 8, 2, 64
    k, v = rnd(1, b, cap, hk, d, dt=F16), rnd(2, b, cap, hk, d, dt=F16)
    kd, vd, q = k.cuda(), v.cuda(), torch.zeros(b, 1, h, d, dtype=F16, device='cuda')
    lens, starts = (torch.zeros(b, dtype=torch.int32, device='cuda') for _ in range(2))
    kw = dict(window=200, sinks=4, causal=True)
    call = lambda: T().window_attention(q, kd, vd, lens=lens, starts=starts, **kw)      # noqa: E731
    call()
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = call()
    with torch.cuda.graph(g2, pool=g1.pool()):
        o2 = call()
    for step, n in enumerate(((1, 900), (64, 65), (205, 1), (899, 333))):
        qn = rnd(9 + step, b, 1, h, d, dt=F16)
        q.copy_(qn)
        lens.copy_(torch.tensor(n))
        starts.copy_(lens - 1)
        ref = R.attention(qn, k, v, lens=torch.tensor(n), starts=torch.tensor(n) - 1, **kw)['o']
        g1.replay()
        R.within('first graph', o1, *ref)
        g2.replay()
        R.within('second graph', o2, *ref)


def test_first_derivatives_only_and_saved_tensors_are_guarded():
    t = T()
    x, pos = torch.randn(1, 4, 2, 16, device='cuda', requires_grad=True), torch.zeros(4, 1, dtype=torch.int64, device='cuda')
    for f in (lambda: t.layer_norm(x), lambda: t.rope_axes(x, None, pos, (8,))[0], lambda: t.window_attention(x, x, x)):
        with pytest.raises(RuntimeError, match='second derivative'):
            torch.autograd.grad(f().sum(), x, create_graph=True)
    y = x.detach().clone().requires_grad_()
    z = y * 1.0
    out = t.layer_norm(z)
    z.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()
    with torch.inference_mode():
        assert not t.window_attention(x, x, x).requires_grad
    assert not t.layer_norm(x.detach()).requires_grad
    out = t.window_attention(x, x, x)                       # one leaf in three places
    g, = torch.autograd.grad(out.sum(), x)
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    gs = torch.autograd.grad(t.window_attention(*parts).sum(), parts)
    assert torch.equal(g, gs[0] + gs[1] + gs[2]) or torch.allclose(g, gs[0] + gs[1] + gs[2], rtol=4 * R.E, atol=1e-6)


# ---- refusals --------------------------------------------------------------------------------------------------------------------------
def test_refusals():
    from multiyolov5_amd._lib import MyoloError
    t = T()
    x = torch.zeros(4, 16, device='cuda')
    for bad in (lambda: t.layer_norm(x.double()), lambda: t.layer_norm(x.long()), lambda: t.layer_norm(x, torch.ones(8, device='cuda')),
                lambda: t.layer_norm(x, torch.ones(16, device='cuda').half()), lambda: t.layer_norm(x, eps=-1.0), lambda: t.layer_norm(x, eps=math.nan),
                lambda: t.layer_norm(x, torch.ones(16)), lambda: t.layer_norm(torch.zeros((), device='cuda')), lambda: t.layer_norm(torch.zeros(3, 0, device='cuda')),
                lambda: t.layer_norm(x.cpu()), lambda: t.layer_norm(None)):
        with pytest.raises(MyoloError):
            bad()
    q, k = torch.zeros(2, 5, 4, 16, device='cuda'), torch.zeros(2, 5, 2, 16, device='cuda')
    pos = torch.zeros(5, 2, dtype=torch.int64, device='cuda')
    t.rope_axes(q, k, pos, (4, 4))
    for a in ((q, k, pos, (4, 5)), (q, k, pos, (4,)), (q, k, pos.int(), (4, 4)), (q, k, pos[:4], (4, 4)), (q, k.half(), pos, (4, 4)), (q, k[:, :4], pos, (4, 4)),
              (q[0], None, pos, (4, 4)), (q, k, pos.cpu(), (4, 4)), (q, k, pos, (-1, 4)), (q, k, pos, ()), (q, k, torch.zeros(3, 5, 2, dtype=torch.int64, device='cuda'), (4, 4)),
              (q, k, torch.zeros(5, 5, dtype=torch.int64, device='cuda'), (1, 1, 1, 1, 1)), (q, k, pos, (4, 4), 0.0), (q, k, pos, (4, 4), 1e4, False, 'other')):
        with pytest.raises(MyoloError):
            t.rope_axes(*a)
    i = torch.zeros(2, dtype=torch.int32, device='cuda')
    t.window_attention(q, k, k, lens=i, starts=i)
    for a, kw in (((q, k, k[:, :4]), {}), ((q, k.half(), k), {}), ((q, k[:1], k[:1]), {}), ((q[..., :12], k[..., :12], k[..., :12]), {}), ((q[:, :, :3], k, k), {}),
                  ((torch.zeros(1, 2, 1, 136, device='cuda'),) * 3, {}), ((q, k, k), dict(window=-1)), ((q, k, k), dict(sinks=-1)), ((q, k, k), dict(scale=0.0)),
                  ((q, k, k), dict(scale=-1.0)), ((q, k, k), dict(scale=math.inf)), ((q, k, k), dict(lens=i.long())), ((q, k, k), dict(lens=i[:1])),
                  ((q, k, k), dict(starts=i.cpu())), ((q, k, k), dict(window=1 << 29)), ((q, k, k), dict(window=1.5)), ((q.cpu(), k, k), {}), ((q[0], k, k), {}),
                  ((q.double(), k.double(), k.double()), {})):
        with pytest.raises(MyoloError):
            t.window_attention(*a, **kw)


def test_capture_beside_an_eager_graph_of_the_same_leaf_is_refused():
    """a leaf whose gradient node stands on the default stream cannot take part in a capture: an error while the capture is whole, nothing worse"""
    t = T()
    x = rnd(1, 2, 6, 2, 16).cuda().requires_grad_()
    pos = torch.arange(6).reshape(6, 1).cuda()
    go = rnd(2, 2, 6, 2, 16).cuda()
    for f in (lambda: t.layer_norm(x), lambda: t.rope_axes(x, None, pos, (8,))[0], lambda: t.window_attention(x, x, x)):
        alive = f()
        want = torch.autograd.grad(alive, x, go, retain_graph=True)[0]
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match='eager graph of the same leaf'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(f(), x, go)
        assert torch.equal(torch.autograd.grad(alive, x, go)[0], want)
        del alive
        gc.collect()                                                # (the error's traceback held the refused graph)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                               # no eager graph left: the same capture is taken
            got = torch.autograd.grad(f(), x, go)[0]
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        del got
