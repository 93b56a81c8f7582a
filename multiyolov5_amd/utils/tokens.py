"""Token operators on MI355X: layer norm, rotary positions with several axes, attention with a sliding window -- what a transformer layer
over the pixels of a feature map (or the frames of a clip) needs next to the convolutions (the reference's own is models/common.py:49-92).

The arithmetic is in libmyolo (csrc/layernorm.hip, csrc/rope.hip, csrc/attention.hip); the backward passes are handed to autograd through
`torch.autograd.Function`.  fp16 and fp32 tensors, statistics, sums and parameters in fp32.  Every call works on the current stream of the
tensors' device, allocates its results and scratch with torch's allocator and never synchronises, so all of them can be captured into a
graph.  There is no CPU path.
"""
import contextlib
import ctypes as C
import functools
import math

import torch

from .. import _lib as L

ATTN_MAX_DIM = 128
_P3 = C.c_int64 * 3


def _tensor(t, what, dtype=None, dim=None):
    if not torch.is_tensor(t):
        raise L.MyoloError(f'{what} must be a tensor, got {type(t).__name__}')
    L.require_gpu(t)
    if dtype is None and t.dtype not in (torch.float16, torch.float32):
        raise L.MyoloError(f'{what} must be fp16 or fp32, got {t.dtype}')
    if dtype is not None and t.dtype != dtype:
        raise L.MyoloError(f'{what} must be {dtype}, got {t.dtype}')
    if dim is not None and t.dim() != dim:
        raise L.MyoloError(f'{what} must have {dim} dimensions, got {tuple(t.shape)}')


def _same_device(t, *others):
    for o in others:
        if o is not None and o.device != t.device:
            raise L.MyoloError(f'tensors on {t.device} and {o.device} in one call')


def _on(t):
    """launches go to the tensors' device (and its current stream), whatever the current device is"""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------
def _rows(x):
    """(tensor whose memory the view describes, L.Tensor of its rows): last dimension = channels, the others numbered in order.  A view whose
    leading dimensions do not reduce to three strides, or whose channels are not adjacent, is copied."""
    if x.dim() == 0:
        raise L.MyoloError('layer_norm: a tensor with a channel dimension is needed')
    c = x.shape[-1]
    if c < 1 or c >= 1 << 31:
        raise L.MyoloError(f'layer_norm: {c} channels')
    if x.stride(-1) != 1 and c > 1:
        x = x.contiguous()
    n, s = _lead(x)
    if n is None:
        x = x.contiguous()
        n, s = _lead(x)
    if n is None:
        raise L.MyoloError('layer_norm: more than 2^31 - 1 rows in one dimension')
    return x, L.Tensor(x.data_ptr(), n[0], n[1], n[2], c, s[0], s[1], s[2], L.DT[x.dtype], 0)


def _lead(x):
    """leading dimensions merged where their strides allow, padded to three: (sizes, strides), or (None, None)"""
    sizes, strides = [], []
    for n, s in zip(x.shape[:-1], x.stride()[:-1]):
        if n == 1:
            continue
        if sizes and strides[-1] == n * s and sizes[-1] * n < 1 << 31:
            sizes[-1], strides[-1] = sizes[-1] * n, s
        else:
            sizes.append(n)
            strides.append(s)
    if len(sizes) > 3 or any(n >= 1 << 31 for n in sizes) or math.prod(sizes[-2:]) >= 1 << 31:
        return None, None
    while len(sizes) < 3:
        n, s = (sizes[0], strides[0]) if sizes else (1, x.shape[-1])
        sizes.insert(0, 1)
        strides.insert(0, n * s)
    return sizes, strides


def _param(p, c, x, what):
    if p is None:
        return None
    _tensor(p, what, torch.float32, 1)
    if p.shape[0] != c:
        raise L.MyoloError(f'{what} has {p.shape[0]} values for {c} channels')
    return p.contiguous()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        lib = L.lib()
        x, xd = _rows(x)
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        _, od = _rows(out)
        n, c = xd.n * xd.h * xd.w, xd.c
        od.n, od.h, od.w, od.sn, od.sh, od.sw = xd.n, xd.h, xd.w, xd.h * xd.w * c, xd.w * c, c
        train = any(ctx.needs_input_grad[:3])
        saved = torch.empty(2 * n, dtype=torch.float32, device=x.device) if train else None
        with _on(x):
            L.check(lib.myolo_layernorm_fwd(C.byref(xd), L.ptr(weight), L.ptr(bias), eps, C.byref(od), L.ptr(saved), L.stream_ptr()),
                    'myolo_layernorm_fwd')
        if train:
            ctx.save_for_backward(x, weight, saved)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go):
        lib = L.lib()
        x, weight, saved = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        x, xd = _rows(x)
        go = go.to(x.dtype)
        if go.shape[-1] > 1 and go.stride(-1) != 1 or _lead(go)[0] != [xd.n, xd.h, xd.w]:
            go = go.contiguous()
        n, c = xd.n * xd.h * xd.w, xd.c
        dense = [xd.h * xd.w * c, xd.w * c, c]
        gs = dense if go.is_contiguous() else _lead(go)[1]
        gd = L.Tensor(go.data_ptr(), xd.n, xd.h, xd.w, c, *gs, L.DT[x.dtype], 0)
        gx = torch.empty_like(x, memory_format=torch.contiguous_format) if want_x else None
        gxd = L.Tensor(gx.data_ptr(), xd.n, xd.h, xd.w, c, *dense, L.DT[x.dtype], 0) if want_x else None
        gw = torch.empty(c, dtype=torch.float32, device=x.device) if want_w else None
        gb = torch.empty(c, dtype=torch.float32, device=x.device) if want_b else None
        nb = lib.myolo_layernorm_ws_bytes(n, c) if want_w or want_b else 0
        ws = torch.empty(nb // 4, dtype=torch.float32, device=x.device) if nb else None
        with _on(x):
            L.check(lib.myolo_layernorm_bwd(C.byref(gd), C.byref(xd), L.ptr(saved), L.ptr(weight), C.byref(gxd) if want_x else None, 0,
                                            L.ptr(gw), L.ptr(gb), 0, L.ptr(ws), nb, L.stream_ptr()), 'myolo_layernorm_bwd')
        return gx, gw, gb, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) * (var + eps)^-1/2 * weight + bias over the last dimension of x [..., C] (any C >= 1, any strides; a channels-last feature
    map is x.permute(0, 2, 3, 1)).  weight, bias: fp32 [C] or None.  The result is contiguous, in x's dtype; gradients for x, weight, bias."""
    _tensor(x, 'layer_norm: x')
    if not (isinstance(eps, (int, float)) and eps >= 0.0 and math.isfinite(eps)):
        raise L.MyoloError(f'layer_norm: eps must be a number >= 0, got {eps!r}')
    c = x.shape[-1] if x.dim() else 0
    weight, bias = _param(weight, c, x, 'layer_norm: weight'), _param(bias, c, x, 'layer_norm: bias')
    _same_device(x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, float(eps))


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=64)
def rope_table(sections, theta=10000.0, spectrum='shared'):
    """host table of the rotary pairs: (turns per unit of position, fp64 ctypes array; axis of every pair, int32 ctypes array).  A pure function
    of its arguments.  spectrum 'shared': pair j of all n turns with theta^(-j / n); 'axis': pair j of an axis' n_a with theta^(-j / n_a)."""
    sections = tuple(sections)
    n = sum(sections)
    turns, axis = [], []
    for a, na in enumerate(sections):
        for j in range(na):
            e = len(turns) / n if spectrum == 'shared' else j / na
            turns.append(math.pow(theta, -e) / (2.0 * math.pi))
            axis.append(a)
    return (C.c_double * max(n, 1))(*turns), (C.c_int32 * max(n, 1))(*axis)


def _strides(t):
    """{batch, token, head} strides of [b, l, h, d]; a dimension of one element has none that matters"""
    return [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]


def rope_desc(q, k, qo, ko, pos, table, sections, interleaved, inverse):
    d = L.RopeDesc()
    b, l, hq, dim = q.shape
    d.q, d.qo, d.pos = q.data_ptr(), qo.data_ptr(), pos.data_ptr()
    d.qs, d.qos = _P3(*_strides(q)), _P3(*_strides(qo))
    if k is not None:
        d.k, d.ko, d.hk = k.data_ptr(), ko.data_ptr(), k.shape[2]
        d.ks, d.kos = _P3(*_strides(k)), _P3(*_strides(ko))
    d.ps = _P3(pos.stride(0) if pos.dim() == 3 and pos.shape[0] > 1 else 0, pos.stride(-2), pos.stride(-1))
    d.turns, d.axis = C.cast(table[0], C.c_void_p), C.cast(table[1], C.c_void_p)
    d.b, d.l, d.hq, d.d = b, l, hq, dim
    d.npair, d.naxis, d.interleaved, d.inverse, d.dtype = sum(sections), len(sections), int(interleaved), int(inverse), L.DT[q.dtype]
    return d


def _rope(q, k, pos, spec, inverse):
    sections, theta, interleaved, spectrum = spec
    q = q if q.stride(-1) == 1 or q.shape[-1] == 1 else q.contiguous()
    qo, ko = torch.empty(q.shape, dtype=q.dtype, device=q.device), None
    if k is not None:
        k = k if k.stride(-1) == 1 or k.shape[-1] == 1 else k.contiguous()
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    table = rope_table(sections, theta, spectrum)
    with _on(q):
        L.check(L.lib().myolo_rope(C.byref(rope_desc(q, k, qo, ko, pos, table, sections, interleaved, inverse)), L.stream_ptr()), 'myolo_rope')
    return qo, ko


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, spec):
        ctx.save_for_backward(pos)
        ctx.spec, ctx.like = spec, (q.shape, None if k is None else k.shape, q.dtype, q.device)
        return _rope(q, k, pos, spec, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        pos, = ctx.saved_tensors
        qs, ks, dt, dev = ctx.like
        gq = torch.zeros(qs, dtype=dt, device=dev) if gq is None else gq.to(dt)
        if ks is not None:
            gk = torch.zeros(ks, dtype=dt, device=dev) if gk is None else gk.to(dt)
        gq, gk = _rope(gq, gk if ks is not None else None, pos, ctx.spec, True)
        return gq, gk, None, None


def rope_axes(q, k, pos, sections, theta=10000.0, interleaved=False, spectrum='shared'):
    """rotary positions with several axes on q [B, L, H, D] and k [B, L, Hk, D] (or None), in one launch: (q', k').

    pos: int64 [B or 1, L, A] or [L, A], the position of every token on each of the A = len(sections) <= 4 axes (time, height, width).
    sections: how many of the rotary pairs turn with each axis, in order; 2 * sum(sections) <= D, channels behind them pass through.
    interleaved: pairs are neighbouring channels (2j, 2j + 1) instead of (j, j + sum(sections)).  spectrum: rope_table.
    Angles are formed in fp64: far positions (10^6 and more) lose nothing.  Gradients for q and k; the results are contiguous."""
    _tensor(q, 'rope_axes: q', dim=4)
    if k is not None:
        _tensor(k, 'rope_axes: k', q.dtype, 4)
        if (k.shape[0], k.shape[1], k.shape[3]) != (q.shape[0], q.shape[1], q.shape[3]) or k.shape[2] < 1:
            raise L.MyoloError(f'rope_axes: q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads')
    _tensor(pos, 'rope_axes: pos', torch.int64)
    _same_device(q, k, pos)
    sections = tuple(int(s) for s in sections)
    if not 1 <= len(sections) <= L.ROPE_MAX_AXES or min(sections) < 0:
        raise L.MyoloError(f'rope_axes: sections {sections}: 1 to {L.ROPE_MAX_AXES} axes with counts >= 0')
    if 2 * sum(sections) > q.shape[3] or sum(sections) > L.ROPE_MAX_PAIRS:
        raise L.MyoloError(f'rope_axes: {sum(sections)} pairs in {q.shape[3]} channels (at most {L.ROPE_MAX_PAIRS})')
    if tuple(pos.shape[-2:]) != (q.shape[1], len(sections)) or pos.dim() not in (2, 3) or (pos.dim() == 3 and pos.shape[0] not in (1, q.shape[0])):
        raise L.MyoloError(f'rope_axes: pos {tuple(pos.shape)} for {q.shape[1]} tokens, {len(sections)} axes and a batch of {q.shape[0]}')
    if spectrum not in ('shared', 'axis') or not theta > 0.0:
        raise L.MyoloError(f'rope_axes: spectrum {spectrum!r}, theta {theta!r}')
    if q.shape[2] < 1 or q.shape[3] < 1:
        raise L.MyoloError(f'rope_axes: q {tuple(q.shape)}')
    return _Rope.apply(q, k, pos, (sections, float(theta), bool(interleaved), spectrum))


# ---- attention -------------------------------------------------------------------------------------------------------------------------
def _side(t):
    """[b, l, h, d] as the kernels take it: adjacent channels, 16-byte aligned base and strides"""
    seg = 16 // t.element_size()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % seg for s in _strides(t)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _attn_desc(q, k, v, o, lse, opt):
    window, sinks, causal, lens, starts, scale = opt
    d = L.AttnDesc()
    d.q, d.k, d.v, d.o, d.lse, d.lens, d.starts = (0 if t is None else t.data_ptr() for t in (q, k, v, o, lse, lens, starts))
    d.qs, d.ks, d.vs, d.os = (_P3(*_strides(t)) for t in (q, k, v, o))
    d.b, d.lq, d.hq, d.d = q.shape
    d.lk, d.hk = k.shape[1], k.shape[2]
    d.dtype, d.causal, d.window, d.sinks, d.scale = L.DT[q.dtype], int(causal), window, sinks, scale
    return d


def _scratch(nbytes, t):
    return torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes else None


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, opt):
        lib = L.lib()
        q, k, v = _side(q), _side(k), _side(v)
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        train = any(ctx.needs_input_grad[:3])
        lse = torch.empty(q.shape[0], q.shape[2], q.shape[1], dtype=torch.float32, device=q.device) if train else None
        d = _attn_desc(q, k, v, o, lse, opt)
        d.ws_bytes = lib.myolo_attn_ws_bytes(C.byref(d), 0)
        ws = _scratch(d.ws_bytes, q)
        d.ws = ws.data_ptr() if ws is not None else 0
        with _on(q):
            L.check(lib.myolo_attn_fwd(C.byref(d), L.stream_ptr()), 'myolo_attn_fwd')
        if train:
            ctx.save_for_backward(q, k, v, o, lse, opt[3], opt[4])
            ctx.opt = opt[:3] + (None, None) + opt[5:]
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go):
        lib = L.lib()
        q, k, v, o, lse, lens, starts = ctx.saved_tensors
        opt = ctx.opt[:3] + (lens, starts) + ctx.opt[5:]
        go = _side(go.to(q.dtype))
        want_q, want_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        gq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if want_q else None
        gk, gv = (torch.empty(k.shape, dtype=k.dtype, device=k.device) if want_kv else None for _ in range(2))
        d = _attn_desc(q, k, v, o, lse, opt)
        d.go, d.gos = go.data_ptr(), _P3(*_strides(go))
        if want_q:
            d.gq, d.gqs = gq.data_ptr(), _P3(*_strides(gq))
        if want_kv:
            d.gk, d.gv, d.gks, d.gvs = gk.data_ptr(), gv.data_ptr(), _P3(*_strides(gk)), _P3(*_strides(gv))
        d.ws_bytes = lib.myolo_attn_ws_bytes(C.byref(d), 1)
        ws = _scratch(d.ws_bytes, q)
        d.ws = ws.data_ptr() if ws is not None else 0
        with _on(q):
            L.check(lib.myolo_attn_bwd(C.byref(d), L.stream_ptr()), 'myolo_attn_bwd')
        return gq, gk if ctx.needs_input_grad[1] else None, gv if ctx.needs_input_grad[2] else None, None


def window_attention(q, k, v, window=0, sinks=0, causal=False, lens=None, starts=None, scale=None):
    """softmax attention of q [B, Lq, H, D] over k, v [B, Lk, Hk, D] (H a multiple of Hk: Hk = H / g heads shared by g query heads each; D a
    multiple of 8, at most 128) -> [B, Lq, H, D].

    Query i stands at position p = starts[b] + i (starts None: Lk - Lq + i, the newest tokens of a sequence).  It sees key j when
    j < lens[b] (lens None: Lk), and not causal or j <= p, and window == 0 or |p - j| < window or j < sinks: the first `sinks` keys stay
    visible however far the window has moved.  lens, starts: int32 [B] on the device (a padded batch; a cache longer than what it holds).
    A query that sees nothing gives zeros and takes no gradient.  What keys hold that no query of the call sees does not matter; a key that
    only some of the queries see has to be finite.  scale: default D^-1/2, > 0.  One new token over a long cache is split over the key
    axis.  Gradients for q, k and v, formed without atomics (a run repeats bit for bit)."""
    _tensor(q, 'window_attention: q', dim=4)
    _tensor(k, 'window_attention: k', q.dtype, 4)
    _tensor(v, 'window_attention: v', q.dtype, 4)
    b, lq, hq, dim = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != dim:
        raise L.MyoloError(f'window_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}')
    if k.shape[2] < 1 or hq < 1 or hq % k.shape[2]:
        raise L.MyoloError(f'window_attention: {hq} query heads over {k.shape[2]} key heads')
    if dim % 8 or not 8 <= dim <= ATTN_MAX_DIM:
        raise L.MyoloError(f'window_attention: head dimension {dim} (a multiple of 8 up to {ATTN_MAX_DIM})')
    if max(lq * (hq // k.shape[2]), k.shape[1], window) > L.ATTN_MAX_LEN or b * hq >= 1 << 24:
        raise L.MyoloError('window_attention: sequence, window or batch too long')
    if window < 0 or sinks < 0 or int(window) != window or int(sinks) != sinks:
        raise L.MyoloError(f'window_attention: window {window}, sinks {sinks}')
    for t, n in ((lens, 'lens'), (starts, 'starts')):
        if t is not None:
            _tensor(t, 'window_attention: ' + n, torch.int32, 1)
            if t.shape[0] != b:
                raise L.MyoloError(f'window_attention: {n} has {t.shape[0]} values for a batch of {b}')
    scale = dim ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise L.MyoloError(f'window_attention: scale {scale}')
    _same_device(q, k, v, lens, starts)
    lens, starts = (None if t is None else t.contiguous() for t in (lens, starts))
    return _WindowAttention.apply(q, k, v, (int(window), min(int(sinks), k.shape[1]), bool(causal), lens, starts, scale))
