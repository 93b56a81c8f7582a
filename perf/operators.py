"""The cases that time the token operators (multiyolov5_amd.utils.tokens): layer norm, rotary positions with several axes, attention with a
sliding window and leading tokens that stay visible.  `run` computes an operator in elementary torch operations (`own = False`) or by the
framework's call (`own = True`); `exact` gives the operator's definition in 64 bits."""
import math

import numpy as np
import torch

own = False

DT = {'fp16': torch.float16, 'fp32': torch.float32}
ES = {'fp16': 2, 'fp32': 4}


# ---- cases -----------------------------------------------------------------------------------------------------------------------------
def _ln(name, rows, c, dtype, train, slack=0):
    return {'name': name, 'op': 'ln', 'rows': rows, 'c': c, 'dtype': dtype, 'train': train, 'slack': slack}


def _rope(name, b, t, h, w, heads, kv_heads, d, dtype, train, interleaved=False, spectrum='shared', far=0):
    return {'name': name, 'op': 'rope', 'b': b, 't': t, 'h': h, 'w': w, 'heads': heads, 'kv_heads': kv_heads, 'd': d, 'dtype': dtype,
            'train': train, 'interleaved': interleaved, 'spectrum': spectrum, 'far': far}


def _attn(name, b, lq, lk, heads, kv_heads, d, dtype, train, window=0, sinks=0, causal=False, ragged=False):
    return {'name': name, 'op': 'attn', 'b': b, 'lq': lq, 'lk': lk, 'heads': heads, 'kv_heads': kv_heads, 'd': d, 'dtype': dtype,
            'train': train, 'window': window, 'sinks': sinks, 'causal': causal, 'ragged': ragged}


def listed():
    return [
        # one 512x1024 frame at stride 32 (16x32 pixels), inference: the call's latency
        _ln('ln frame', 512, 512, 'fp16', False),
        # the training batch of 16 images of 512x1024 at stride 8 (64x128 pixels each), yolov5m's width there
        _ln('ln train map', 16 * 64 * 128, 192, 'fp16', True),
        # odd channel count, rows that are a slice of a wider buffer, full precision
        _ln('ln train odd', 4097, 1003, 'fp32', True, slack=5),
        # one new token of a stream, 32 + 8 heads
        _rope('rope token', 1, 1, 1, 1, 32, 8, 128, 'fp16', False, far=100000),
        # the training batch at stride 16 (32x64 pixels), two image axes with a spectrum each
        _rope('rope train map', 16, 1, 32, 64, 8, 8, 64, 'fp16', True, spectrum='axis'),
        # a clip of 9 frames of 31x63 pixels late in a long video, neighbouring channels paired, full precision
        _rope('rope train clip', 2, 9, 31, 63, 12, 4, 96, 'fp32', True, interleaved=True, far=1000000),
        # the training batch at stride 16, a band of 4 pixel rows each way and 4 leading tokens
        _attn('attn train map', 16, 2048, 2048, 4, 4, 64, 'fp16', True, window=256, sinks=4),
        # a long prompt-like sequence, grouped heads, causal, everything visible
        _attn('attn long causal', 1, 8192, 8192, 32, 8, 128, 'fp16', False, causal=True),
        # training on sequences, causal sliding window with leading tokens, grouped heads
        _attn('attn train window', 2, 4096, 4096, 16, 4, 128, 'fp16', True, window=1024, sinks=4, causal=True),
        # padded batch of odd lengths, full precision
        _attn('attn train odd', 3, 777, 777, 6, 2, 40, 'fp32', True, window=129, sinks=3, ragged=True),
        # one new token for each of 8 streams over caches of up to 32768 tokens
        _attn('attn token long', 8, 1, 32768, 32, 8, 128, 'fp16', False, causal=True, ragged=True),
        # one new token of one stream, short cache, window with leading tokens: the call's latency
        _attn('attn token', 1, 1, 700, 8, 2, 64, 'fp16', False, window=512, sinks=4, causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['ln', 'rope', 'attn', 'attn', 'token'])
    dtype = rng.choice(['fp16', 'fp16', 'fp32'])
    if kind == 'ln':
        c = _log(rng, 16, 8192)
        if rng.random() < 0.6:
            c = (c + 7) // 8 * 8
        rows = _log(rng, 1, max(1, min(131072, (1 << 25) // c)))
        return _pop(_ln('', rows, c, dtype, rng.random() < 0.6, rng.choice([0, 0, 8, 3])))
    if kind == 'rope':
        kv = rng.choice([1, 2, 4, 8])
        return _pop(_rope('', _log(rng, 1, 8), _log(rng, 1, 12), _log(rng, 1, 40), _log(rng, 1, 64), kv * rng.choice([1, 2, 4]), kv,
                          rng.choice([32, 40, 64, 96, 128]), dtype, rng.random() < 0.5, rng.random() < 0.5, rng.choice(['shared', 'axis']),
                          rng.choice([0, 1000, 1000000])))
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([32, 40, 64, 96, 128])
    if kind == 'token':
        b = _log(rng, 1, 16)
        lk = _log(rng, 64, 32768)
        lq = min(lk, rng.choice([1, 1, 1, 2, 5]))
        return _pop(_attn('', b, lq, lk, heads, kv, d, dtype, False, rng.choice([0, 0, _log(rng, 16, 4096)]), rng.choice([0, 4, 7]),
                          True, rng.random() < 0.5))
    b = _log(rng, 1, 8)
    most = math.sqrt(2.5e8 / (b * heads))
    lq = _log(rng, 17, max(18, min(4096, most)))
    train = rng.random() < 0.6
    lk = lq if train or rng.random() < 0.5 else lq + _log(rng, 1, max(2, min(4096, most)))
    return _pop(_attn('', b, lq, lk, heads, kv, d, dtype, train, rng.choice([0, _log(rng, 1, 1024), _log(rng, 16, 1024)]),
                      rng.choice([0, 1, 4, 16]), rng.random() < 0.5, rng.random() < 0.3))


def _pop(c):
    c.pop('name')
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------
def _sections(c):
    """rotary pairs of the time, height and width axes: a quarter of them time, the rest shared by the image axes (no time axis: half each)"""
    p = c['d'] // 2
    t = p // 4 if c['t'] > 1 else 0
    return (t, (p - t) // 2, p - t - (p - t) // 2)


def prepare(case, seed):
    c, dt = case, DT[case['dtype']]
    g = torch.Generator(device='cuda').manual_seed(seed)

    def rnd(*shape, dtype=dt, scale=1.0, shift=0.0):
        x = torch.empty(*shape, dtype=dtype, device='cuda').normal_(generator=g)
        return x if scale == 1.0 and shift == 0.0 else x.mul_(scale).add_(shift)

    s = {'case': dict(c)}
    if c['op'] == 'ln':
        buf = rnd(c['rows'], c['c'] + c['slack'], scale=1.7, shift=0.4)
        s['x'] = buf[:, :c['c']]
        s['w'] = rnd(c['c'], dtype=torch.float32, scale=0.2, shift=1.0)
        s['b'] = rnd(c['c'], dtype=torch.float32, scale=0.2)
        if c['train']:
            s['go'] = rnd(c['rows'], c['c'])
        return s
    if c['op'] == 'rope':
        n = c['t'] * c['h'] * c['w']
        s['q'], s['k'] = rnd(c['b'], n, c['heads'], c['d']), rnd(c['b'], n, c['kv_heads'], c['d'])
        ax = [torch.arange(v, device='cuda') for v in (c['t'], c['h'], c['w'])]
        grid = torch.stack(torch.meshgrid(*ax, indexing='ij'), -1).reshape(1, n, 3).repeat(c['b'], 1, 1)
        first = torch.randint(0, c['far'] + 1, (c['b'], 1, 1), generator=g, device='cuda')
        s['pos'] = grid + torch.cat([first, first // 64, first // 64], -1)
        if c['train']:
            s['gq'], s['gk'] = torch.empty_like(s['q']).normal_(generator=g), torch.empty_like(s['k']).normal_(generator=g)
        return s
    s['q'] = rnd(c['b'], c['lq'], c['heads'], c['d'])
    s['k'], s['v'] = rnd(c['b'], c['lk'], c['kv_heads'], c['d']), rnd(c['b'], c['lk'], c['kv_heads'], c['d'])
    s['lens'] = s['starts'] = None
    if c['ragged']:
        lens = torch.randint((c['lk'] + 1) // 2, c['lk'] + 1, (c['b'],), generator=g, device='cuda').clamp_(min=c['lq'] if c['lq'] < c['lk'] else 1)
        s['lens'] = lens.to(torch.int32)
        # queries: the whole padded sequence, or the newest tokens of each row
        s['starts'] = torch.zeros_like(s['lens']) if c['lq'] == c['lk'] else s['lens'] - c['lq']
    if c['train']:
        s['go'] = torch.empty_like(s['q']).normal_(generator=g)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s['case']
    return {'ln': _run_ln, 'rope': _run_rope, 'attn': _run_attn}[c['op']](s, c)


def _run_ln(s, c):
    if own:
        from multiyolov5_amd.utils import tokens as T
        if not c['train']:
            return T.layer_norm(s['x'], s['w'], s['b'], 1e-5)
        x, w, b = (s[k].detach().requires_grad_() for k in ('x', 'w', 'b'))
        y = T.layer_norm(x, w, b, 1e-5)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), s['go']))
    x = s['x'].float()
    xc = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(xc.square().mean(-1, keepdim=True) + 1e-5)
    xh = xc * r
    y = (xh * s['w'] + s['b']).to(s['x'].dtype)
    if not c['train']:
        return y
    go = s['go'].float()
    g = go * s['w']
    gx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return y, gx.to(s['x'].dtype), (go * xh).sum(0), go.sum(0)


def _frequencies(c):
    """(frequency of every rotary pair, its axis)"""
    sec = _sections(c)
    axis = torch.cat([torch.full((n,), a, dtype=torch.int64, device='cuda') for a, n in enumerate(sec)])
    if c['spectrum'] == 'shared':
        e = torch.arange(c['d'] // 2, dtype=torch.float64, device='cuda') / (c['d'] // 2)
    else:
        e = torch.cat([torch.arange(n, dtype=torch.float64, device='cuda') / max(n, 1) for n in sec])
    return torch.pow(10000.0, -e), axis


def _rotate(x, cos, sin, interleaved):
    x = x.float()
    u, v = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    a, b = u * cos - v * sin, v * cos + u * sin
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _run_rope(s, c):
    if own:
        from multiyolov5_amd.utils import tokens as T
        kw = dict(theta=10000.0, interleaved=c['interleaved'], spectrum=c['spectrum'])
        if not c['train']:
            return T.rope_axes(s['q'], s['k'], s['pos'], _sections(c), **kw)
        q, k = s['q'].detach().requires_grad_(), s['k'].detach().requires_grad_()
        a, b = T.rope_axes(q, k, s['pos'], _sections(c), **kw)
        return (a.detach(), b.detach(), *torch.autograd.grad((a, b), (q, k), (s['gq'], s['gk'])))
    f, axis = _frequencies(c)
    ang = s['pos'].double()[..., axis] * f                       # [b, n, d/2]: far positions lose their angle in 32 bits
    cos, sin = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]
    dt, il = s['q'].dtype, c['interleaved']
    out = [_rotate(s[k], cos, sin, il).to(dt) for k in ('q', 'k')]
    if c['train']:
        out += [_rotate(s[k], cos, -sin, il).to(dt) for k in ('gq', 'gk')]
    return tuple(out)


def _visible(s, c):
    """[b or 1, lq, lk] truth values: the keys that a query sees"""
    i, j = torch.arange(c['lq'], device='cuda')[:, None], torch.arange(c['lk'], device='cuda')[None]
    p = (i + (c['lk'] - c['lq']))[None] if s['starts'] is None else s['starts'].long()[:, None, None] + i
    see = torch.ones(1, c['lq'], c['lk'], dtype=torch.bool, device='cuda')
    if s['lens'] is not None:
        see = see & (j < s['lens'].long()[:, None, None])
    if c['causal']:
        see = see & (j <= p)
    if c['window']:
        see = see & (((p - j).abs() < c['window']) | (j < c['sinks']))
    return see


def _run_attn(s, c):
    if own:
        from multiyolov5_amd.utils import tokens as T
        kw = dict(window=c['window'], sinks=c['sinks'], causal=c['causal'], lens=s['lens'], starts=s['starts'])
        if not c['train']:
            return T.window_attention(s['q'], s['k'], s['v'], **kw)
        q, k, v = (s[n].detach().requires_grad_() for n in ('q', 'k', 'v'))
        o = T.window_attention(q, k, v, **kw)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), s['go']))
    b, d, h, hk, dt = c['b'], c['d'], c['heads'], c['kv_heads'], s['q'].dtype
    sc = d ** -0.5
    q = s['q'].float().transpose(1, 2).reshape(b, hk, h // hk, c['lq'], d)
    k = s['k'].float().permute(0, 2, 1, 3).contiguous()[:, :, None]                  # [b, hk, 1, lk, d]
    v = s['v'].float().permute(0, 2, 1, 3).contiguous()[:, :, None]
    see = _visible(s, c)[:, None, None]
    lg = (torch.matmul(q, k.transpose(-1, -2)) * sc).masked_fill_(~see, -math.inf)
    m = lg.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = (lg - m).exp_()
    p = p / p.sum(-1, keepdim=True).clamp_(min=1e-30)
    o = torch.matmul(p, v)

    def back(x, n):                                                                   # [b, hk, g, l, d] -> [b, l, n, d]
        return x.reshape(b, n, x.shape[-2], d).transpose(1, 2).to(dt)
    if not c['train']:
        return back(o, h)
    go = s['go'].float().transpose(1, 2).reshape(b, hk, h // hk, c['lq'], d)
    gv = torch.matmul(p.transpose(-1, -2), go).sum(2)
    gl = p * (torch.matmul(go, v.transpose(-1, -2)) - (go * o).sum(-1, keepdim=True)) * sc
    gq = torch.matmul(gl, k)
    gk = torch.matmul(gl.transpose(-1, -2), q).sum(2)
    return back(o, h), back(gq, h), back(gk, hk), back(gv, hk)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------
def _pairs(c):
    """visible (query, key) pairs of one head, summed over the batch; padded rows: three quarters of the keys, the mean of their lengths"""
    lk = c['lk'] if not c['ragged'] else (3 * c['lk']) // 4
    p = np.arange(c['lq'], dtype=np.int64) + (0 if c['lq'] == c['lk'] else lk - c['lq'])
    hi = np.minimum(lk, p + 1) if c['causal'] else np.full_like(p, lk)
    if not c['window']:
        return c['b'] * int(np.maximum(hi, 0).sum())
    lo = np.maximum(p - c['window'] + 1, 0)
    hi2 = np.minimum(hi, p + c['window'])
    band = np.maximum(hi2 - lo, 0)
    first = np.minimum(np.minimum(c['sinks'], hi), np.where(band > 0, lo, hi))
    return c['b'] * int((band + np.maximum(first, 0)).sum())


def work(c):
    e = ES[c['dtype']]
    if c['op'] == 'ln':
        n = c['rows'] * c['c']
        return {'bytes': n * e * (4 if c['train'] else 2) + 8 * c['c'] * (2 if c['train'] else 1), 'flops': n * (25 if c['train'] else 8)}
    if c['op'] == 'rope':
        n = c['b'] * c['t'] * c['h'] * c['w']
        m = n * (c['heads'] + c['kv_heads']) * c['d'] * (2 if c['train'] else 1)
        return {'bytes': 2 * m * e + 24 * n, 'flops': 3 * m}
    pairs = _pairs(c)
    reach = c['lk'] if not c['ragged'] else (3 * c['lk']) // 4
    if c['window'] and c['causal'] and c['lq'] < c['lk']:
        reach = min(reach, c['window'] + c['sinks'] + c['lq'])
    qo, kv = c['b'] * c['lq'] * c['heads'] * c['d'], c['b'] * reach * c['kv_heads'] * c['d']
    return {'bytes': e * (2 * qo + 2 * kv) * (2 if c['train'] else 1), 'flops': pairs * c['heads'] * c['d'] * (14 if c['train'] else 4)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {'ln': _exact_ln, 'rope': _exact_rope, 'attn': _exact_attn}[case['op']](s, case)


def _exact_ln(s, c):
    x, w, b = (s[k].double().requires_grad_() for k in ('x', 'w', 'b'))
    var, mean = torch.var_mean(x, dim=1, unbiased=False)
    y = ((x.t() - mean) / torch.sqrt(var + 1e-5)).t() * w + b
    if not c['train']:
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), s['go'].double()))


def _exact_rope(s, c):
    sec, half = _sections(c), c['d'] // 2
    col, turn = 0, []
    for a, n in enumerate(sec):
        for j in range(n):
            e = col / half if c['spectrum'] == 'shared' else j / n
            turn.append(s['pos'][..., a].double() * math.pow(10000.0, -e))
            col += 1
    z = torch.polar(torch.ones_like(turn[0]), torch.zeros_like(turn[0])) if not turn else torch.exp(1j * torch.stack(turn, -1))[:, :, None]

    def mul(x, by):
        x = x.double()
        w = torch.complex(x[..., 0::2], x[..., 1::2]) if c['interleaved'] else torch.complex(x[..., :half], x[..., half:])
        w = w * by
        return torch.view_as_real(w).flatten(-2) if c['interleaved'] else torch.cat([w.real, w.imag], -1)
    out = [mul(s['q'], z), mul(s['k'], z)]
    if c['train']:
        out += [mul(s['gq'], z.conj()), mul(s['gk'], z.conj())]
    return tuple(out)


def _exact_attn(s, c):
    """one (row, head) at a time: scores of the visible keys, softmax in 64 bits, derivatives by automatic differentiation"""
    g = c['heads'] // c['kv_heads']
    o, gq = (torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda') for _ in range(2))
    gk, gv = (torch.zeros(s['k'].shape, dtype=torch.float64, device='cuda') for _ in range(2))
    i, j = torch.arange(c['lq'], device='cuda').view(-1, 1), torch.arange(c['lk'], device='cuda').view(1, -1)
    for b in range(c['b']):
        n = c['lk'] if s['lens'] is None else int(s['lens'][b])
        p = i + (c['lk'] - c['lq'] if s['starts'] is None else int(s['starts'][b]))
        hide = j >= n
        if c['causal']:
            hide = hide | (j > p)
        if c['window']:
            hide = hide | ((j >= c['sinks']) & ((j <= p - c['window']) | (j >= p + c['window'])))
        none = hide.all(1, keepdim=True)
        for h in range(c['heads']):
            q, k, v = (t.double().requires_grad_(c['train']) for t in (s['q'][b, :, h], s['k'][b, :, h // g], s['v'][b, :, h // g]))
            a = torch.softmax((q @ k.t() / math.sqrt(c['d'])).masked_fill(hide & ~none, -math.inf), 1).masked_fill(none, 0.0)
            y = a @ v
            o[b, :, h] = y.detach()
            if c['train']:
                dq, dk, dv = torch.autograd.grad(y, (q, k, v), s['go'][b, :, h].double())
                gq[b, :, h] = dq
                gk[b, :, h // g] += dk
                gv[b, :, h // g] += dv
    return (o, gq, gk, gv) if c['train'] else o
