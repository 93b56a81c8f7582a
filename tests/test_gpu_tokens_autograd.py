"""Token operators under what autograd lets a caller do around them: saved-tensor hooks and checkpointing, lazily negated and zero tensors, forward
mode, tracing, captures beside eager graphs.  Definitions and bounds: tests/token_ref.py."""
import gc

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

from tests import token_ref as R
from tests.test_gpu_tokens import F16, F32, T, _layer, _layer_inputs, rnd

pytestmark = pytest.mark.gpu
DTS = pytest.mark.parametrize('dt', [F16, F32], ids=['fp16', 'fp32'])


# ---- saved-tensor hooks ----------------------------------------------------------------------------------------------------------------
def transposed(t):
    """the same values, the last two axes swapped in memory: channels that are not adjacent"""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else torch.stack([t, t], -1)[..., 0]


def shifted(t):
    """the same values, rows off a 16-byte boundary"""
    b = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return b[1:].view(t.shape).copy_(t)


def heads_first(t):
    return t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 4 else t.clone()


class every_other:
    """another layout for every second tensor: what was laid out alike no longer is"""

    def __init__(self):
        self.n = 0

    def __call__(self, t):
        self.n += 1
        return heads_first(t) if self.n % 2 else transposed(t)


HOOKS = {'transposed': lambda: saved_tensors_hooks(lambda t: t.clone(), transposed), 'shifted': lambda: saved_tensors_hooks(lambda t: t.clone(), shifted),
         'heads first': lambda: saved_tensors_hooks(lambda t: t.clone(), heads_first), 'mixed': lambda: saved_tensors_hooks(lambda t: t.clone(), every_other()),
         'on the host': save_on_cpu, 'pinned': lambda: save_on_cpu(pin_memory=True)}


@DTS
@pytest.mark.parametrize('hook', list(HOOKS))
def test_saved_tensors_in_another_layout(hook, dt):
    x, go, w, b = rnd(1, 67, 48, dt=dt), rnd(2, 48, dt=dt).expand(67, 48), rnd(3, 48, shift=1.0), rnd(4, 48)
    ref = R.layer_norm(x, w, b, 1e-5, go)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    with HOOKS[hook]():
        y = T().layer_norm(*leaves)
    for n, t in zip(('gx', 'gw', 'gb'), torch.autograd.grad(y, leaves, go[0].cuda().expand(67, 48))):   # (a broadcast gradient is copied in the backward)
        R.within(n, t, *ref[n])
    q, k, v, go = rnd(1, 2, 70, 4, 32, dt=dt), rnd(2, 2, 90, 2, 32, dt=dt), rnd(3, 2, 90, 2, 32, dt=dt), rnd(4, 2, 70, 4, 32, dt=dt)
    lens, starts = torch.tensor([90, 71], dtype=torch.int32), torch.tensor([20, 1], dtype=torch.int32)
    kw = dict(window=23, sinks=2, causal=True)
    ref = R.attention(q, k, v, go=go, lens=lens, starts=starts, **kw)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    with HOOKS[hook]():
        o = T().window_attention(*leaves, lens=lens.cuda(), starts=starts.cuda(), **kw)
    for n, t in zip(('gq', 'gk', 'gv'), torch.autograd.grad(o, leaves, go.cuda())):
        R.within(n, t, *ref[n])
    pos = torch.randint(0, 90, (2, 70, 2), generator=torch.Generator().manual_seed(3))
    leaf = q.cuda().requires_grad_()
    with HOOKS[hook]():
        a, _ = T().rope_axes(leaf, None, pos.cuda(), (8, 8))
    R.within('rope', torch.autograd.grad(a, leaf, go.cuda())[0], *R.rope(go, pos, (8, 8), 10000.0, False, 'shared', True))


@pytest.mark.parametrize('change', ['dtype', 'shape', 'device'])
def test_saved_tensors_that_come_back_as_something_else_are_refused(change):
    to = {'dtype': lambda t: t.double(), 'shape': lambda t: t[:1], 'device': lambda t: t.cpu()}[change]
    x, w = rnd(1, 2, 6, 4, 16).cuda().requires_grad_(), torch.ones(16, device='cuda', requires_grad=True)
    pos = torch.arange(12).reshape(2, 6, 1).cuda()
    i = torch.tensor([6, 6], dtype=torch.int32, device='cuda')
    for f in (lambda: T().layer_norm(x, w), lambda: T().window_attention(x, x, x, lens=i), lambda: T().rope_axes(x, None, pos, (8,))[0]):
        with saved_tensors_hooks(lambda t: t, to):
            y = f()
        with pytest.raises(RuntimeError, match='came back as'):
            torch.autograd.grad(y, x, torch.ones_like(y))


def test_an_error_in_a_hook_arrives_as_itself():
    def bad(t):
        raise KeyError('mine')
    x = rnd(1, 2, 6, 4, 16).cuda().requires_grad_()
    pos = torch.arange(6).reshape(6, 1).cuda()
    for f in (lambda: T().layer_norm(x), lambda: T().window_attention(x, x, x), lambda: T().rope_axes(x, None, pos, (8,))[0]):
        with pytest.raises(KeyError, match='mine'):
            with saved_tensors_hooks(bad, lambda t: t):
                f()
        with saved_tensors_hooks(lambda t: t, bad):
            y = f()
        with pytest.raises(KeyError, match='mine'):
            torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize('reentrant', [False, True])
def test_checkpointed_layer(reentrant):
    """the forward formed again in the backward, which stops as soon as it has what it needs (inside an operator)"""
    from torch.utils.checkpoint import checkpoint
    leaves, pos, kw, dims, go = _layer_inputs()
    dl = [t.cuda().requires_grad_() for t in leaves]
    posd = pos.cuda()
    want = torch.autograd.grad(_layer(*dl, posd, kw, *dims), dl, go.cuda())
    o = checkpoint(lambda *a: _layer(*a, posd, kw, *dims), *dl, use_reentrant=reentrant)
    o.backward(go.cuda())
    assert all(torch.equal(t.grad, r) for t, r in zip(dl, want))


# ---- lazily negated tensors, tensors without storage -----------------------------------------------------------------------------------
@DTS
def test_negated_views_are_read_as_their_values(dt):
    """(the imaginary part of a conjugate is such a view)"""
    t, neg = T(), torch._neg_view
    x, w, b = rnd(1, 2, 9, 4, 16, dt=dt).cuda(), rnd(2, 16).cuda(), rnd(3, 16).cuda()
    pos = torch.arange(9).reshape(9, 1).cuda()
    n = neg(x)
    assert n.is_neg() and torch.equal(n, -x)
    assert torch.equal(t.layer_norm(n, neg(w), neg(b)), t.layer_norm(-x, -w, -b))
    assert all(torch.equal(a, r) for a, r in zip(t.rope_axes(n, n, neg(pos), (8,)), t.rope_axes(-x, -x, -pos, (8,))))
    assert torch.equal(t.window_attention(n, x, x), t.window_attention(-x, x, x))
    assert torch.equal(t.window_attention(x, n, x), t.window_attention(x, -x, x)) and torch.equal(t.window_attention(x, x, n), t.window_attention(x, x, -x))
    # (one place a leaf: the engine adds the gradients of several in another order behind another graph)
    c = x.clone()
    for f in (lambda x: t.layer_norm(x), lambda x: t.rope_axes(x, None, pos, (8,))[0], lambda x: t.window_attention(x, c, c),
              lambda x: t.window_attention(c, x, c), lambda x: t.window_attention(c, c, x)):
        leaf = x.clone().requires_grad_()
        want, = torch.autograd.grad(f(leaf), leaf, -x)
        got, = torch.autograd.grad(f(leaf), leaf, n)                     # an incoming gradient that is negated lazily
        assert torch.equal(got, want)
        want, = torch.autograd.grad(f(-leaf), leaf, x)
        got, = torch.autograd.grad(f(neg(leaf)), leaf, x)
        assert torch.equal(got, want)


def test_tensors_without_storage_are_refused():
    from multiyolov5_amd._lib import MyoloError
    t = T()
    x, z = torch.ones(2, 6, 4, 16, device='cuda'), torch._efficientzerotensor((2, 6, 4, 16), device='cuda')
    pos = torch.arange(6).reshape(6, 1).cuda()
    for f in (lambda: t.layer_norm(z), lambda: t.layer_norm(x, torch._efficientzerotensor((16,), device='cuda')), lambda: t.rope_axes(z, None, pos, (8,)),
              lambda: t.window_attention(x, z, x), lambda: t.window_attention(z, x, x)):
        with pytest.raises(MyoloError, match='storage'):
            f()


# ---- forward mode, tracing -------------------------------------------------------------------------------------------------------------
def one_input(t, x, w, pos):
    """the operators as functions of one tensor, by the argument it is"""
    return {'layer_norm': lambda x: t.layer_norm(x, w), 'weight': lambda x: t.layer_norm(x, x[0, 0, 0]), 'rope_axes': lambda x: t.rope_axes(x, None, pos, (8,))[0],
            'k': lambda x: t.rope_axes(x.detach(), x, pos, (8,))[1], 'window_attention': lambda x: t.window_attention(x, x.detach(), x.detach()),
            'v': lambda x: t.window_attention(x.detach(), x.detach(), x)}


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw
    x, w, pos = rnd(1, 2, 6, 4, 16).cuda(), torch.ones(16, device='cuda'), torch.arange(6).reshape(6, 1).cuda()
    for name, f in one_input(T(), x, w, pos).items():
        with fw.dual_level():
            with pytest.raises(RuntimeError, match='forward mode'):
                f(fw.make_dual(x, torch.ones_like(x)))
            leaf = x.clone().requires_grad_()
            y = f(leaf)                                                  # (none of it sticks)
            with pytest.raises(RuntimeError, match='forward mode'):
                torch.autograd.grad(y, leaf, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_tracing_is_refused():
    x, w, pos = rnd(1, 2, 6, 4, 16).cuda(), torch.ones(16, device='cuda'), torch.arange(6).reshape(6, 1).cuda()
    for name, f in one_input(T(), x, w, pos).items():
        with pytest.raises(RuntimeError, match='traced'):
            torch.jit.trace(f, x, check_trace=False)
        f(x)


# ---- captures --------------------------------------------------------------------------------------------------------------------------
def test_captured_layer_beside_an_eager_graph_of_its_leaves_is_refused():
    """the leaf's node is behind other operators (a projection, a split): refused all the same, and only where the captured pass would reach it"""
    leaves, pos, kw, dims, go = _layer_inputs()
    posd, god = pos.cuda(), go.cuda()
    dl = [t.cuda().requires_grad_() for t in leaves]
    alive = _layer(*dl, posd, kw, *dims)
    want = torch.autograd.grad(alive, dl, god, retain_graph=True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match='eager graph of the same leaf'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(_layer(*dl, posd, kw, *dims), dl, god)
    gc.collect()
    # another input of its own, the eager graph's projection not differentiated: nothing of the eager graph takes part
    own = [t.detach().clone().requires_grad_() for t in dl[:3]] + [dl[3]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(_layer(*own, posd, kw, *dims), own[:3], god)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(_layer(*own, posd, kw, *dims), own[:3], god)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, r) for a, r in zip(got, want))
    assert all(torch.equal(a, r) for a, r in zip(torch.autograd.grad(alive, dl, god), want))


# ---- layers in launch plans ------------------------------------------------------------------------------------------------------------
def test_attn_layer_with_frozen_parts():
    """no gradient for the input; frozen parameters stay without one and change nothing for the others"""
    from multiyolov5_amd.models.common import AttnLayer
    torch.manual_seed(0)
    m = AttnLayer(32, 2, 1, 2, 3).cuda().train()
    x, go = rnd(1, 2, 32, 5, 7).cuda(), rnd(2, 2, 32, 5, 7).cuda()
    m(x.clone().requires_grad_()).backward(go)
    want = {k: p.grad.clone() for k, p in m.named_parameters()}
    m.zero_grad(set_to_none=True)
    m(x).backward(go)
    for k, p in m.named_parameters():
        assert float((p.grad - want[k]).norm()) <= 1e-5 * float(want[k].norm()), k
    m.zero_grad(set_to_none=True)
    m.norm1.weight.requires_grad_(False)
    m.qkv.bias.requires_grad_(False)
    m(x).backward(go)
    for k, p in m.named_parameters():
        if p.requires_grad:
            assert float((p.grad - want[k]).norm()) <= 1e-5 * float(want[k].norm()), k
        else:
            assert p.grad is None, k


def test_attn_layer_repeats_once_its_plans_are_captured():
    """launch lists run eagerly at first and as graphs from the third pass on: the same gradients, and those of other inputs in between"""
    from multiyolov5_amd.models.common import AttnLayer
    torch.manual_seed(0)
    m = AttnLayer(64, 4, 2, 2, 3).cuda().train()
    first = {}
    for i in range(9):
        x, go = rnd(i % 2, 2, 64, 9, 12).cuda().requires_grad_(), rnd(10 + i % 2, 2, 64, 9, 12).cuda()
        m.zero_grad(set_to_none=True)
        y = m(x)
        y.backward(go)
        got = [y.detach().clone(), x.grad] + [p.grad.clone() for p in m.parameters()]
        want = first.setdefault(i % 2, got)
        for a, r in zip(got, want):
            assert float((a - r).norm()) <= 1e-5 * float(r.norm()), i


def test_attn_layer_in_half_follows_its_weights():
    """the fp32 copies of a half model's norm weights are formed again when the weights change"""
    from multiyolov5_amd.models.common import AttnLayer
    torch.manual_seed(0)
    m = AttnLayer(32, 2, 2, 1, 1).cuda().eval().half()
    x = rnd(1, 1, 32, 6, 8, dt=F16).cuda()
    with torch.no_grad():
        for step in range(3):
            for _ in range(4):
                y = m(x).clone()
            m32 = AttnLayer(32, 2, 2, 1, 1).cuda().eval()
            m32.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
            r = m32(x.float())
            assert float((y.float() - r).norm()) <= 2e-2 * float(r.norm()), step
            m.norm1.weight.mul_(1.5)
            m.norm2.bias.add_(0.7)
        m.float()                                                        # and back: parameters that were allocated again
        assert float((m(x.float()) - m32.cuda().train(False)(x.float())).norm()) > 0
        m32.load_state_dict(m.state_dict())
        r = m32(x.float())
        assert float((m(x.float()) - r).norm()) <= 1e-5 * float(r.norm())


# ---- threads ---------------------------------------------------------------------------------------------------------------------------
def test_calls_of_several_threads():
    """passes of four threads at once, each on a stream of its own, give what one thread gives"""
    import threading
    leaves, pos, kw, dims, go = _layer_inputs()
    posd, god = pos.cuda(), go.cuda()

    def once(k):
        l = [(t * (1 + k)).cuda().requires_grad_() for t in leaves]
        o = _layer(*l, posd, kw, *dims)
        return [o.detach(), *torch.autograd.grad(o, l, god)]
    want = [once(k) for k in range(4)]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(25):
                    got = once(k)
                    s.synchronize()
                    if not all(torch.equal(a, r) for a, r in zip(got, want[k])):
                        bad.append(k)
        except Exception as e:                                           # noqa: BLE001
            bad.append(e)
    ts = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, bad
