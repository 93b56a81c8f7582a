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
