"""Token operators on MI355X: layer norm, rotary positions with several axes, attention with a sliding window -- what a transformer layer
over the pixels of a feature map (or the frames of a clip) needs next to the convolutions (the reference's own is models/common.py:49-92).

The arithmetic is in libmyolo (csrc/layernorm.hip, csrc/rope.hip, csrc/attention.hip); the backward passes are handed to autograd through
`torch.autograd.Function`.  fp16 and fp32 tensors, statistics, sums and parameters in fp32.  Every call works on the current stream of the
tensors' device, allocates its results and scratch with torch's allocator and never synchronises, so all of them can be captured into a
graph.  There is no CPU path.
"""
import ctypes as C
import functools
import math

import torch

from .. import _lib as L

ATTN_MAX_DIM = 128
_P3 = C.c_int64 * 3
_stream = torch._C._cuda_getCurrentRawStream          # (device index) -> the current stream's handle
# A call's checks and descriptor depend on sizes, strides, types and options alone: they are worked out once per signature (the host's time is
# what bounds small calls), then the addresses are filled in.
_signature = functools.lru_cache(maxsize=1024)


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


def _device(t, *others):
    """the tensors' common device index"""
    dev = t.get_device()
    for o in others:
        if o is not None and o.get_device() != dev:
            raise L.MyoloError(f'tensors on {t.device} and {o.device} in one call')
    return dev


def _launch(dev, name, *args):
    """a library call on `dev` and its current stream, whatever the current device is"""
    fn = getattr(L.lib(), name)
    if dev == torch.cuda.current_device():
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc:
        L.check(rc, name)


def _needs_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _first_order(fn):
    """backward(ctx, *grads) that refuses to be differentiated again; the check costs nothing where no graph is recorded"""
    once = torch.autograd.function.once_differentiable(fn)
    return staticmethod(lambda ctx, *g: once(ctx, *g) if torch.is_grad_enabled() else fn(ctx, *g))


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------
def _lead(shape, stride):
    """leading dimensions merged where their strides allow, padded to three: sizes + strides, or None"""
    sizes, strides = [], []
    for n, s in zip(shape[:-1], stride[:-1]):
        if n == 1:
            continue
        if sizes and strides[-1] == n * s and sizes[-1] * n < 1 << 31:
            sizes[-1], strides[-1] = sizes[-1] * n, s
        else:
            sizes.append(n)
            strides.append(s)
    if len(sizes) > 3 or any(n >= 1 << 31 for n in sizes) or math.prod(sizes[-2:]) >= 1 << 31:
        return None
    while len(sizes) < 3:
        n, s = (sizes[0], strides[0]) if sizes else (1, shape[-1])
        sizes.insert(0, 1)
        strides.insert(0, n * s)
    return sizes, strides


@_signature
def _ln_fields(shape, stride, dtype):
    """L.Tensor fields behind the pointer for the rows of such a tensor (last dimension = channels, the others numbered in order), or None:
    its channels are not adjacent or its leading dimensions do not reduce to three strides"""
    c = shape[-1]
    if c > 1 and stride[-1] != 1:
        return None
    lead = _lead(shape, stride)
    return None if lead is None else (*lead[0][:3], c, *lead[1], L.DT[dtype], 0)


@_signature
def _ln_dense(shape, dtype):
    """(fields of a contiguous tensor of this shape, rows, channels, bytes of backward scratch)"""
    if not shape or not 1 <= shape[-1] < 1 << 31:
        raise L.MyoloError(f'layer_norm: no channels in a tensor of shape {tuple(shape)}')
    stride, n = [], 1
    for d in reversed(shape):
        stride.insert(0, n)
        n *= max(d, 1)
    f = _ln_fields(tuple(shape), tuple(stride), dtype)
    if f is None:
        raise L.MyoloError('layer_norm: more than 2^31 - 1 rows in one dimension')
    rows = f[0] * f[1] * f[2]
    return f, rows, f[3], L.lib().myolo_layernorm_ws_bytes(rows, f[3])


def _ln_rows(x):
    """(tensor to read, its L.Tensor); copied where no descriptor reaches its rows"""
    f = _ln_fields(x.shape, x.stride(), x.dtype)
    if f is None:
        x = x.contiguous()
        f = _ln_dense(x.shape, x.dtype)[0]
    return x, L.Tensor(x.data_ptr(), *f)


def _param(p, c, what):
    if p.dtype != torch.float32 or p.dim() != 1 or p.shape[0] != c or not p.is_cuda:
        _tensor(p, what, torch.float32, 1)
        raise L.MyoloError(f'{what} has {p.shape[0]} values for {c} channels')
    return p if p.is_contiguous() else p.contiguous()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, train):
        dense, n, c, _ = _ln_dense(x.shape, x.dtype)
        x, xd = _ln_rows(x)
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        od = L.Tensor(out.data_ptr(), *dense)
        if xd.n != od.n or xd.h != od.h or xd.w != od.w:         # (the view's dimensions merge less far than the dense result's)
            od = _like_rows(out, xd)
        saved = torch.empty(2 * n, dtype=torch.float32, device=x.device) if train else None
        _launch(x.get_device(), 'myolo_layernorm_fwd', C.byref(xd), weight.data_ptr() if weight is not None else None,
                bias.data_ptr() if bias is not None else None, eps, C.byref(od), saved.data_ptr() if train else None)
        if train:
            ctx.save_for_backward(x, weight, saved)
        return out

    @_first_order
    def backward(ctx, go):
        x, weight, saved = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dense, n, c, nb = _ln_dense(x.shape, x.dtype)
        dev = x.device
        x, xd = _ln_rows(x)
        if go.dtype != x.dtype:
            go = go.to(x.dtype)
        go, gd = _ln_rows(go)
        gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_x else None
        gxd = L.Tensor(gx.data_ptr() if want_x else None, *dense)
        if not (xd.n == gd.n == gxd.n and xd.h == gd.h == gxd.h and xd.w == gd.w == gxd.w):
            gxd = _like_rows(gx, xd) if want_x else gxd
            if (gd.n, gd.h, gd.w) != (xd.n, xd.h, xd.w):
                go = go.contiguous()
                gd = _like_rows(go, xd)
        gw = torch.empty(c, dtype=torch.float32, device=dev) if want_w else None
        gb = torch.empty(c, dtype=torch.float32, device=dev) if want_b else None
        if not (want_w or want_b):
            nb = 0
        ws = torch.empty(nb // 4, dtype=torch.float32, device=dev) if nb else None
        _launch(x.get_device(), 'myolo_layernorm_bwd', C.byref(gd), C.byref(xd), saved.data_ptr(), weight.data_ptr() if weight is not None else None,
                C.byref(gxd) if want_x else None, 0, gw.data_ptr() if want_w else None, gb.data_ptr() if want_b else None, 0,
                ws.data_ptr() if nb else None, nb)
        return gx, gw, gb, None, None


def _like_rows(t, d):
    """the rows of the contiguous tensor t numbered as descriptor d numbers its own"""
    return L.Tensor(t.data_ptr(), d.n, d.h, d.w, d.c, d.h * d.w * d.c, d.w * d.c, d.c, d.dtype, 0)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) * (var + eps)^-1/2 * weight + bias over the last dimension of x [..., C] (any C >= 1, any strides; a channels-last feature
    map is x.permute(0, 2, 3, 1)).  weight, bias: fp32 [C] or None.  The result is contiguous, in x's dtype; gradients for x, weight, bias."""
    _tensor(x, 'layer_norm: x')
    if not (isinstance(eps, (int, float)) and 0.0 <= eps < math.inf):
        raise L.MyoloError(f'layer_norm: eps must be a number >= 0, got {eps!r}')
    c = _ln_dense(x.shape, x.dtype)[2]
    if weight is not None:
        weight = _param(weight, c, 'layer_norm: weight')
    if bias is not None:
        bias = _param(bias, c, 'layer_norm: bias')
    _device(x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, float(eps), _needs_grad(x, weight, bias))


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------
@_signature
def rope_table(sections, theta=10000.0, spectrum='shared'):
    """host table of the rotary pairs: (turns per unit of position, fp64 ctypes array; axis of every pair, int32 ctypes array).  A pure function
    of its arguments.  spectrum 'shared': pair j of all n turns with theta^(-j / n); 'axis': pair j of an axis' n_a with theta^(-j / n_a)."""
    n = sum(sections)
    turns, axis = [], []
    for a, na in enumerate(sections):
        for j in range(na):
            e = len(turns) / n if spectrum == 'shared' else j / na
            turns.append(math.pow(theta, -e) / (2.0 * math.pi))
            axis.append(a)
    return (C.c_double * max(n, 1))(*turns), (C.c_int32 * max(n, 1))(*axis)


def _strides(shape, stride):
    """{batch, token, head} strides of [b, l, h, d]; a dimension of one element has none that matters"""
    return [s if n > 1 else 0 for n, s in zip(shape[:3], stride[:3])]


def _dense_strides(shape):
    return _strides(shape, (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3]))


@_signature
def _rope_desc(qshape, qstride, qostride, kshape, kstride, kostride, pshape, pstride, dtype, sections, theta, interleaved, spectrum, inverse):
    """descriptor without addresses, after all checks"""
    b, l, hq, dim = qshape
    if kshape is not None and ((kshape[0], kshape[1], kshape[3]) != (b, l, dim) or kshape[2] < 1):
        raise L.MyoloError(f'rope_axes: q {tuple(qshape)} and k {tuple(kshape)} differ in more than their heads')
    if not 1 <= len(sections) <= L.ROPE_MAX_AXES or min(sections) < 0:
        raise L.MyoloError(f'rope_axes: sections {sections}: 1 to {L.ROPE_MAX_AXES} axes with counts >= 0')
    if 2 * sum(sections) > dim or sum(sections) > L.ROPE_MAX_PAIRS:
        raise L.MyoloError(f'rope_axes: {sum(sections)} pairs in {dim} channels (at most {L.ROPE_MAX_PAIRS})')
    if len(pshape) not in (2, 3) or tuple(pshape[-2:]) != (l, len(sections)) or (len(pshape) == 3 and pshape[0] not in (1, b)):
        raise L.MyoloError(f'rope_axes: pos {tuple(pshape)} for {l} tokens, {len(sections)} axes and a batch of {b}')
    if spectrum not in ('shared', 'axis') or not 0.0 < theta < math.inf:
        raise L.MyoloError(f'rope_axes: spectrum {spectrum!r}, theta {theta!r}')
    if hq < 1 or dim < 1 or max(b, l, hq, dim) >= 1 << 31:
        raise L.MyoloError(f'rope_axes: q {tuple(qshape)}')
    d = L.RopeDesc()
    d.qs, d.qos = _P3(*_strides(qshape, qstride)), _P3(*_strides(qshape, qostride))
    if kshape is not None:
        d.hk, d.ks, d.kos = kshape[2], _P3(*_strides(kshape, kstride)), _P3(*_strides(kshape, kostride))
    d.ps = _P3(pstride[0] if len(pshape) == 3 and pshape[0] > 1 else 0, pstride[-2], pstride[-1])
    turns, axis = rope_table(sections, theta, spectrum)          # (held by rope_call while the call reads them)
    d.b, d.l, d.hq, d.d = b, l, hq, dim
    d.npair, d.naxis, d.interleaved, d.inverse, d.dtype = sum(sections), len(sections), int(interleaved), int(inverse), L.DT[dtype]
    return bytes(d), turns, axis


def rope_desc(q, k, qo, ko, pos, spec, inverse):
    """myolo_rope's descriptor of q, k -> qo, ko (spec: sections, theta, interleaved, spectrum) and what has to outlive the call"""
    none = (None, None, None)
    raw, turns, axis = _rope_desc(q.shape, q.stride(), qo.stride(), *((k.shape, k.stride(), ko.stride()) if k is not None else none),
                                  pos.shape, pos.stride(), q.dtype, *spec, inverse)
    d = L.RopeDesc.from_buffer_copy(raw)
    d.q, d.qo, d.pos = q.data_ptr(), qo.data_ptr(), pos.data_ptr()
    if k is not None:
        d.k, d.ko = k.data_ptr(), ko.data_ptr()
    d.turns, d.axis = C.addressof(turns), C.addressof(axis)
    return d, (turns, axis)


def _rope(q, k, pos, spec, inverse):
    if q.stride(-1) != 1 and q.shape[-1] > 1:
        q = q.contiguous()
    qo, ko = torch.empty(q.shape, dtype=q.dtype, device=q.device), None
    if k is not None:
        if k.stride(-1) != 1 and k.shape[-1] > 1:
            k = k.contiguous()
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    d, keep = rope_desc(q, k, qo, ko, pos, spec, inverse)
    _launch(q.get_device(), 'myolo_rope', C.byref(d))
    return qo, ko


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, spec):
        ctx.save_for_backward(pos)
        ctx.spec, ctx.like = spec, (q.shape, None if k is None else k.shape, q.dtype, q.device)
        return _rope(q, k, pos, spec, False)

    @_first_order
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
    _tensor(pos, 'rope_axes: pos', torch.int64)
    _device(q, k, pos)
    spec = (tuple(map(int, sections)), float(theta), bool(interleaved), spectrum)
    if not _needs_grad(q, k):
        return _rope(q, k, pos, spec, False)
    return _Rope.apply(q, k, pos, spec)


# ---- attention -------------------------------------------------------------------------------------------------------------------------
@_signature
def _attn_plan(qshape, kshape, vshape, dtype, window, sinks, causal, scale):
    """(descriptor without addresses and input strides, bytes of forward and of backward scratch), after all checks"""
    b, lq, hq, dim = qshape
    lk, hk = kshape[1], kshape[2]
    if kshape != vshape or kshape[0] != b or kshape[3] != dim:
        raise L.MyoloError(f'window_attention: q {tuple(qshape)}, k {tuple(kshape)}, v {tuple(vshape)}')
    if hk < 1 or hq < 1 or hq % hk:
        raise L.MyoloError(f'window_attention: {hq} query heads over {hk} key heads')
    if dim % 8 or not 8 <= dim <= ATTN_MAX_DIM:
        raise L.MyoloError(f'window_attention: head dimension {dim} (a multiple of 8 up to {ATTN_MAX_DIM})')
    if window < 0 or sinks < 0 or int(window) != window or int(sinks) != sinks:
        raise L.MyoloError(f'window_attention: window {window}, sinks {sinks}')
    if max(lq * (hq // hk), lk, window) > L.ATTN_MAX_LEN or b * hq >= 1 << 24:
        raise L.MyoloError('window_attention: sequence, window or batch too long')
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise L.MyoloError(f'window_attention: scale {scale}')
    d = L.AttnDesc()
    d.b, d.lq, d.hq, d.d, d.lk, d.hk = b, lq, hq, dim, lk, hk
    d.dtype, d.causal, d.window, d.sinks, d.scale = L.DT[dtype], int(bool(causal)), int(window), min(int(sinks), lk), scale
    for n in ('qs', 'os', 'gos', 'gqs'):
        setattr(d, n, _P3(*_dense_strides(qshape)))
    for n in ('ks', 'vs', 'gks', 'gvs'):
        setattr(d, n, _P3(*_dense_strides(kshape)))
    return bytes(d), L.lib().myolo_attn_ws_bytes(C.byref(d), 0), L.lib().myolo_attn_ws_bytes(C.byref(d), 1)


@_signature
def _attn_strides(shape, stride, esize):
    """element strides as the kernels take them, or None: channels not adjacent or rows off a 16-byte boundary"""
    s = _strides(shape, stride)
    if (stride[3] != 1 and shape[3] > 1) or any(v * esize % 16 for v in s):
        return None
    return _P3(*s)


def _side(t):
    """(tensor, its strides for the descriptor or None where dense); a copy where the kernels cannot read it in place"""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, None
    s = _attn_strides(t.shape, t.stride(), t.element_size()) if t.data_ptr() % 16 == 0 else None
    return (t.clone(memory_format=torch.contiguous_format), None) if s is None else (t, s)


def _attn_desc(plan, q, k, v, o, lse, lens, starts):
    d = L.AttnDesc.from_buffer_copy(plan)
    for t, p, s in ((q, 'q', 'qs'), (k, 'k', 'ks'), (v, 'v', 'vs')):
        setattr(d, p, t[0].data_ptr())
        if t[1] is not None:
            setattr(d, s, t[1])
    d.o = o.data_ptr()
    if lse is not None:
        d.lse = lse.data_ptr()
    if lens is not None:
        d.lens = lens.data_ptr()
    if starts is not None:
        d.starts = starts.data_ptr()
    return d


def _scratch(d, nbytes, device):
    if not nbytes:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    d.ws, d.ws_bytes = ws.data_ptr(), nbytes
    return ws


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lens, starts, plan, train):
        raw, nf, _ = plan
        q, k, v = _side(q), _side(k), _side(v)
        dev = q[0].device
        o = torch.empty(q[0].shape, dtype=q[0].dtype, device=dev)
        lse = torch.empty(o.shape[0], o.shape[2], o.shape[1], dtype=torch.float32, device=dev) if train else None
        d = _attn_desc(raw, q, k, v, o, lse, lens, starts)
        ws = _scratch(d, nf, dev)
        _launch(o.get_device(), 'myolo_attn_fwd', C.byref(d))
        if train:
            ctx.save_for_backward(q[0], k[0], v[0], o, lse, lens, starts)
            ctx.plan = plan
        return o

    @_first_order
    def backward(ctx, go):
        q, k, v, o, lse, lens, starts = ctx.saved_tensors
        raw, _, nb = ctx.plan
        if go.dtype != q.dtype:
            go = go.to(q.dtype)
        go, gos = _side(go)
        want_q, want_k, want_v = ctx.needs_input_grad[:3]
        dev = q.device
        d = _attn_desc(raw, _side(q), _side(k), _side(v), o, lse, lens, starts)
        d.go = go.data_ptr()
        if gos is not None:
            d.gos = gos
        gq = gk = gv = None
        if want_q:
            gq = torch.empty(q.shape, dtype=q.dtype, device=dev)
            d.gq = gq.data_ptr()
        if want_k or want_v:
            gk, gv = torch.empty(k.shape, dtype=q.dtype, device=dev), torch.empty(k.shape, dtype=q.dtype, device=dev)
            d.gk, d.gv = gk.data_ptr(), gv.data_ptr()
        ws = _scratch(d, nb, dev)
        _launch(q.get_device(), 'myolo_attn_bwd', C.byref(d))
        return gq, gk if want_k else None, gv if want_v else None, None, None, None, None


def _rows32(t, b, what):
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != b or not t.is_cuda:
        _tensor(t, what, torch.int32, 1)
        raise L.MyoloError(f'{what} has {t.shape[0]} values for a batch of {b}')
    return t if t.is_contiguous() else t.contiguous()


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
    plan = _attn_plan(q.shape, k.shape, v.shape, q.dtype, window, sinks, causal, scale)
    if lens is not None:
        lens = _rows32(lens, q.shape[0], 'window_attention: lens')
    if starts is not None:
        starts = _rows32(starts, q.shape[0], 'window_attention: starts')
    _device(q, k, v, lens, starts)
    return _WindowAttention.apply(q, k, v, lens, starts, plan, _needs_grad(q, k, v))
