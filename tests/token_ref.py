"""64-bit definitions of the token operators (layer norm, rotary positions, windowed attention) and, next to each value, how far a result formed
with 32-bit statistics and sums and rounded to its storage type may be from it.

A rounding to a type is off by at most half a step, h = finfo.eps / 2 of the value (fp16 2^-11, fp32 2^-24) and by u = half of the smallest
subnormal (fp16 2^-25) where the value is that small.  e = 2^-24 is the half step of the 32-bit arithmetic; a sum of n terms formed in any order
is off by at most n e times the sum of their absolute values."""
import math

import torch

E = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else 1e-38


def within(name, got, ref, bound):
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    bound = bound.detach().double().cpu()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), f'{name}: not finite where the definition is'
    off = (got - ref).abs() - bound
    if off.numel() and not bool((off <= 0).all()):
        i = int(off.argmax())
        raise AssertionError(f'{name}: element {i} is {got.reshape(-1)[i]:.9g}, the definition {ref.reshape(-1)[i]:.9g}, '
                             f'allowed {bound.reshape(-1)[i]:.3g}; {int((off > 0).sum())} of {off.numel()} are too far off')


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------
def layer_norm(x, w, b, eps, go=None):
    """{name: (value, bound)} for x [R, C] (and its gradients for go)"""
    dt, c = x.dtype, x.shape[1]
    X = x.double()
    W = torch.ones(c, dtype=torch.float64) if w is None else w.double()
    B = torch.zeros(c, dtype=torch.float64) if b is None else b.double()
    mu = X.mean(1, keepdim=True)
    D = X - mu
    var = D.square().mean(1, keepdim=True)
    r = (var + eps).rsqrt()
    xh = D * r
    # mean: c + 2 roundings of the mean of |x|; the variance takes it twice per term, squares and sums; the root halves a relative error.  a
    # constant row has D = 0 and var = 0: what is left of the mean's error is scaled by r
    emu = (c + 2) * E * X.abs().mean(1, keepdim=True)
    evar = (2 * D.abs().mean(1, keepdim=True) + emu) * emu + (c + 4) * E * (var + emu * emu)
    er = 0.5 * evar / (var + eps).clamp(min=1e-300) + 4 * E
    exh = (emu + E * (X.abs() + mu.abs())) * r + xh.abs() * (er + 2 * E)
    y = xh * W + B
    out = {'y': (y, exh * W.abs() + 3 * E * (xh * W).abs() + 2 * E * y.abs() + half_step(dt) * y.abs() + tiny(dt))}
    if go is None:
        return out
    G = go.double()
    g = G * W
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    gx = r * (g - m1 - xh * m2)
    e1 = (c + 3) * E * g.abs().mean(1, keepdim=True)
    e2 = (c + 5) * E * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * exh).mean(1, keepdim=True)
    egx = r * (e1 + xh.abs() * e2 + exh * m2.abs() + 4 * E * (g.abs() + m1.abs() + (xh * m2).abs())) + gx.abs() * (er + E)
    out['gx'] = (gx, egx + half_step(dt) * gx.abs() + tiny(dt))
    n = x.shape[0]
    out['gw'] = ((G * xh).sum(0), (n + 4) * E * (G * xh).abs().sum(0) + (G.abs() * exh).sum(0))
    out['gb'] = (G.sum(0), (n + 2) * E * G.abs().sum(0))
    return out


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------
def rope(x, pos, sections, theta, interleaved, spectrum, inverse=False):
    """(value, bound) for x [B, L, H, D], pos [B, L, A]"""
    n = sum(sections)
    X = x.double()
    out = X.clone()
    bound = torch.zeros_like(X)
    j = 0
    for a, na in enumerate(sections):
        for i in range(na):
            f = theta ** -(j / n if spectrum == 'shared' else i / na)
            ang = pos[..., a].double()[:, :, None] * f
            c, s = ang.cos(), ang.sin() * (-1 if inverse else 1)
            u, v = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
            out[..., u] = X[..., u] * c - X[..., v] * s
            out[..., v] = X[..., v] * c + X[..., u] * s
            # the reduced angle is off by 2^-24 of half a turn (its rounding to 32 bits) and 2^-50 of the turn count; sine and cosine by 2
            # half steps; three roundings of the sum
            ea = math.pi * E + 2 * math.pi * 2.0 ** -50 * (ang.abs() / (2 * math.pi)) + 1e-13 * ang.abs() / 1e3
            both = X[..., u].abs() + X[..., v].abs()
            bound[..., u] = bound[..., v] = both * (ea + 5 * E)
            j += 1
    return out, bound + half_step(x.dtype) * out.abs() + tiny(x.dtype)


# ---- attention -------------------------------------------------------------------------------------------------------------------------
def visible(b, lq, lk, window, sinks, causal, lens, starts):
    i, j = torch.arange(lq)[:, None], torch.arange(lk)[None]
    see = torch.zeros(b, lq, lk, dtype=torch.bool)
    for n in range(b):
        p = i + (lk - lq if starts is None else int(starts[n]))
        s = (j < (lk if lens is None else int(lens[n]))) & (j >= 0)
        if causal:
            s = s & (j <= p)
        if window:
            s = s & (((p - j).abs() < window) | (j < sinks))
        see[n] = s
    return see


def attention(q, k, v, window=0, sinks=0, causal=False, lens=None, starts=None, scale=None, go=None):
    """{name: (value, bound)} on the CPU: o, and gq, gk, gv for go"""
    dt = q.dtype
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    g = h // hk
    sc = d ** -0.5 if scale is None else scale
    see = visible(b, lq, lk, window, sinks, causal, lens, starts)[:, None]
    seen = see.any(2)[:, 0]                                        # [b, lk]: keys that no query sees may hold anything
    clean = lambda t: torch.where(seen[:, :, None, None], t.double(), torch.zeros((), dtype=torch.float64))      # noqa: E731
    Q = q.double().transpose(1, 2)
    K, V = (clean(t).transpose(1, 2).repeat_interleave(g, 1) for t in (k, v))
    S = Q @ K.transpose(2, 3) * sc
    S = S.masked_fill(~see, -math.inf)
    some = see.any(3, keepdim=True)
    m = torch.where(some, S.amax(3, keepdim=True) if lk else S.new_zeros(b, h, lq, 1), torch.zeros((), dtype=torch.float64))
    P = (S - m).exp().masked_fill(~see, 0.0)
    l = P.sum(3, keepdim=True)
    P = torch.where(some, P / l.clamp(min=1e-300), torch.zeros((), dtype=torch.float64))
    O = P @ V
    hs, u = half_step(dt), tiny(dt)
    # a score: d + 3 roundings of the sum of |q k|, and one of its own size in each of the scaling, the shift by the maximum and the exponential;
    # a probability takes the error of its own score and, through the sum, at most the largest one
    ES = ((d + 3) * E * (Q.abs() @ K.abs().transpose(2, 3)) * sc + 4 * E * torch.where(see, S, torch.zeros_like(S)).abs() + 4 * E).masked_fill(~see, 0.0)
    EP = ES + (ES.amax(3, keepdim=True) if lk else 0.0) + (lk + 4) * E + 4 * E * m.abs()
    rp = hs if dt == torch.float16 else 0.0                        # fp16: probabilities enter the product rounded
    AV = V.abs()
    bo = (P * (EP + rp)) @ AV + (lk + 4) * E * (P @ AV) + 2.0 ** -24 * u * AV.sum(2, keepdim=True) + hs * O.abs() + u
    out = {'o': (O.transpose(1, 2), bo.transpose(1, 2))}
    if go is None:
        return out
    G = torch.where(some, go.double().transpose(1, 2), torch.zeros((), dtype=torch.float64))
    Qc = torch.where(some, Q, torch.zeros((), dtype=torch.float64))
    dP = G @ V.transpose(2, 3)
    delta = (G * O).sum(3, keepdim=True)
    dS = P * (dP - delta)
    ed = (G.abs() * bo).sum(3, keepdim=True) + (d + 2) * E * (G * O).abs().sum(3, keepdim=True)
    edp = (d + 2) * E * (G.abs() @ AV.transpose(2, 3))
    eds = dS.abs() * (EP + rp + 4 * E) + P * (ed + edp + 2 * E * (dP.abs() + delta.abs())) + torch.where(see, u if rp else 0.0, 0.0)
    AK, AQ, AG = K.abs(), Qc.abs(), G.abs()
    gq = dS @ K * sc
    egq = (eds @ AK + (lk + 4) * E * (dS.abs() @ AK)) * sc + hs * gq.abs() + u
    gk = dS.transpose(2, 3) @ Qc * sc
    egk = (eds.transpose(2, 3) @ AQ + (lq * g + 4) * E * (dS.abs().transpose(2, 3) @ AQ)) * sc
    gv = P.transpose(2, 3) @ G
    egv = ((P * (EP + rp)).transpose(2, 3) @ AG) + (lq * g + 4) * E * (P.transpose(2, 3) @ AG) + 2.0 ** -12 * u * AG.sum(2, keepdim=True)
    fold = lambda t: t.reshape(b, hk, g, lk, d).sum(2)             # noqa: E731
    gk, egk, gv, egv = fold(gk), fold(egk), fold(gv), fold(egv)
    out['gq'] = (gq.transpose(1, 2), egq.transpose(1, 2))
    out['gk'] = (gk.transpose(1, 2), (egk + hs * gk.abs() + u).transpose(1, 2))
    out['gv'] = (gv.transpose(1, 2), (egv + hs * gv.abs() + u).transpose(1, 2))
    return out
