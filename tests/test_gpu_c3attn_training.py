"""C3Attn (models/common.py) in training: transformer layers between Conv + BatchNorm + SiLU blocks, result and every gradient against a plain
restatement in 64 bits.  Tolerances: relative norms of whole modules as everywhere (gpu_util.TOL)."""
import pytest
import torch
import torch.nn.functional as F

from tests.gpu_util import TOL, check
from tests.test_gpu_attn_layer import layer_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dt', [torch.float32, torch.float16], ids=['fp32', 'fp16'])
@pytest.mark.parametrize('c1,c2,n,heads,rows,sinks,shape', [(32, 64, 1, 2, 0, 0, (4, 6, 10)), (64, 128, 2, 4, 2, 3, (2, 16, 20))])
def test_c3attn_training(c1, c2, n, heads, rows, sinks, shape, dt):
    from multiyolov5_amd.models.common import C3Attn
    torch.manual_seed(0)
    m = C3Attn(c1, c2, n, heads, rows=rows, sinks=sinks)
    with torch.no_grad():
        for k, p in m.named_parameters():
            p.add_(torch.randn_like(p) * (0.03 if p.dim() > 1 else 0.1))
    sd = {k: v.detach().double().clone().requires_grad_() for k, v in m.named_parameters()}
    x = torch.randn(shape[0], c1, *shape[1:]).to(dt)
    go = torch.randn(shape[0], c2, *shape[1:]).to(dt)
    xr = x.double().requires_grad_()

    def conv(name, t):
        eps = getattr(m, name).bn.eps
        return F.silu(F.batch_norm(F.conv2d(t, sd[name + '.conv.weight']), None, None, sd[name + '.bn.weight'], sd[name + '.bn.bias'], True, 0.0, eps))
    a = conv('cv1', xr)
    for i in range(n):
        pre = f'm.{i}.'
        a = layer_ref({k[len(pre):]: v for k, v in sd.items() if k.startswith(pre)}, a, heads, heads, rows, sinks)
    ref = conv('cv3', torch.cat([a, conv('cv2', xr)], 1))
    ref.backward(go.double())
    m = m.cuda().train()
    bad = []
    for _ in range(4):                                     # (launch lists first, then their captured graphs)
        xg = x.cuda().requires_grad_()
        m.zero_grad(set_to_none=True)
        y = m(xg)
        y.backward(go.cuda())
        check('y', y, ref, TOL[dt], collect=bad)
        check('gx', xg.grad, xr.grad, TOL[dt], collect=bad)
        for k, p in m.named_parameters():
            if k == f'm.{n - 1}.fc2.bias':
                # a constant added to every pixel of a channel in front of cv3's BatchNorm, which subtracts the batch mean: the gradient is zero (the
                # definition's is what 64 bits leave of it), and what 32-bit sums leave is measured against the gradient of the same layer's weight
                assert float(sd[k].grad.norm()) <= 1e-10 * float(sd['m.%d.fc2.weight' % (n - 1)].grad.norm())
                assert float(p.grad.norm()) <= TOL[dt] * float(sd['m.%d.fc2.weight' % (n - 1)].grad.norm()), float(p.grad.norm())
                continue
            check(k, p.grad, sd[k].grad, TOL[dt], collect=bad)
    assert not bad, bad
