"""Token operators on MI355X: layer norm, rotary positions with several axes, attention with a sliding window -- what a transformer layer
over the pixels of a feature map (or the frames of a clip) needs next to the convolutions (the reference's own is models/common.py:49-92).

The arithmetic is in libmyolo (csrc/layernorm.hip, csrc/rope.hip, csrc/attention.hip); checks of sizes, descriptors and the autograd nodes are
host C++ over its C ABI (csrc/token_autograd.cpp): a pass over small tensors is bound by the host.  fp16 and fp32 tensors; statistics, sums
and parameters in fp32.  Every call works on the current stream of the tensors' device, allocates its results and scratch with torch's
allocator and never synchronises, so all of them can be captured into a graph (a backward pass not while an eager graph of the same leaves lives
on the default stream: refused).  First derivatives in reverse mode only (second
derivatives, dual tensors and calls inside torch.jit.trace are refused).  There is no CPU path.
"""
import ctypes as C
import functools
import math
import os

import torch

from .. import _lib as L

EXT_PATH = os.path.join(L._HERE, 'lib', '_token_autograd.so')
_module = None


def _ext():
    """the autograd nodes, bound to the library that _lib loaded (once)"""
    global _module
    if _module is None:
        import importlib.machinery
        import importlib.util
        lib = L.lib()
        if not os.path.exists(EXT_PATH):
            raise L.MyoloError(f'{EXT_PATH} not found: run `python -m multiyolov5_amd.build`')
        loader = importlib.machinery.ExtensionFileLoader('_token_autograd', EXT_PATH)
        m = importlib.util.module_from_spec(importlib.util.spec_from_loader('_token_autograd', loader))
        loader.exec_module(m)
        m.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in
                ('myolo_layernorm_fwd', 'myolo_layernorm_bwd', 'myolo_layernorm_ws_bytes', 'myolo_rope', 'myolo_attn_fwd', 'myolo_attn_bwd', 'myolo_attn_ws_bytes')})
        _module = m
    return _module


def _tensor(t, what, dtype=None, dim=None):
    if not torch.is_tensor(t):
        raise L.MyoloError(f'{what} must be a tensor, got {type(t).__name__}')
    if not t.is_cuda:
        L.require_gpu(t)
    if t.dtype is not dtype and (dtype is not None or (t.dtype is not torch.float16 and t.dtype is not torch.float32)):
        raise L.MyoloError(f'{what} must be {dtype or "fp16 or fp32"}, got {t.dtype}')
    if dim is not None and t.dim() != dim:
        raise L.MyoloError(f'{what} must have {dim} dimensions, got {tuple(t.shape)}')


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) * (var + eps)^-1/2 * weight + bias over the last dimension of x [..., C] (1 <= C <= 2^29, any strides; a channels-last feature
    map is x.permute(0, 2, 3, 1)).  weight, bias: fp32 [C] or None.  The result is contiguous, in x's dtype; gradients for x, weight, bias."""
    _tensor(x, 'layer_norm: x')
    return _ext().layer_norm(x, weight, bias, eps)


@functools.lru_cache(maxsize=256)
def rope_table(sections, theta=10000.0, spectrum='shared'):
    """host table of the rotary pairs: (turns per unit of position, fp64 ctypes array; axis of every pair, int32 ctypes array).  A pure function
    of its arguments.  spectrum 'shared': pair j of all n turns with theta^(-j / n); 'axis': pair j of an axis' n_a with theta^(-j / n_a)."""
    if not 1 <= len(sections) <= L.ROPE_MAX_AXES or min(sections) < 0:
        raise L.MyoloError(f'rope_axes: sections {sections}: 1 to {L.ROPE_MAX_AXES} axes with counts >= 0')
    if spectrum not in ('shared', 'axis') or not 0.0 < theta < math.inf:
        raise L.MyoloError(f'rope_axes: spectrum {spectrum!r}, theta {theta!r}')
    n = sum(sections)
    if n > L.ROPE_MAX_PAIRS:
        raise L.MyoloError(f'rope_axes: {n} rotary pairs (at most {L.ROPE_MAX_PAIRS})')
    turns, axis = [], []
    for a, na in enumerate(sections):
        for j in range(na):
            e = len(turns) / n if spectrum == 'shared' else j / na
            turns.append(math.pow(theta, -e) / (2.0 * math.pi))
            axis.append(a)
    return (C.c_double * max(n, 1))(*turns), (C.c_int32 * max(n, 1))(*axis)


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
    sections = tuple(map(int, sections))
    turns, axis = rope_table(sections, float(theta), spectrum)            # (the call copies what it keeps)
    return _ext().rope_axes(q, k, pos, C.addressof(turns), C.addressof(axis), sum(sections), len(sections), bool(interleaved))


def window_attention(q, k, v, window=0, sinks=0, causal=False, lens=None, starts=None, scale=None):
    """softmax attention of q [B, Lq, H, D] over k, v [B, Lk, Hk, D] (H a multiple of Hk: Hk = H / g heads shared by g query heads each; D a
    multiple of 8, at most 128) -> [B, Lq, H, D].

    Query i stands at position p = starts[b] + i (starts None: Lk - Lq + i, the newest tokens of a sequence).  It sees key j when
    j < lens[b] (lens None: Lk), and not causal or j <= p, and window == 0 or |p - j| < window or j < sinks: the first `sinks` keys stay
    visible however far the window has moved.  lens, starts: int32 [B] on the device (a padded batch; a cache longer than what it holds).
    A query that sees nothing gives zeros and takes no gradient.  What keys hold that no query of the call sees, and queries that see nothing,
    does not matter; everything else has to be finite: a NaN in a key that some queries see, or in a query that sees some keys, may also reach
    results up to 128 tokens beyond the mask, and the gradients of the 31 keys behind the sinks, as 0 * NaN does in a product of masked
    probabilities.  scale: default D^-1/2, > 0.
    One new token over a long cache is split over the key axis.  Gradients for q, k and v, formed without atomics (a run repeats bit for bit)."""
    _tensor(q, 'window_attention: q', dim=4)
    _tensor(k, 'window_attention: k', q.dtype, 4)
    _tensor(v, 'window_attention: v', q.dtype, 4)
    if int(window) != window or int(sinks) != sinks:
        raise L.MyoloError(f'window_attention: window {window}, sinks {sinks}')
    return _ext().window_attention(q, k, v, int(window), int(sinks), bool(causal), lens, starts, scale)
