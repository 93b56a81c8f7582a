"""AttnLayer / C3Attn (models/common.py): the token operators inside launch plans, against a plain restatement in 64 bits; the
yolov5s_city_seg_attn configuration end to end.  Tolerances: relative norms of whole modules as everywhere (gpu_util.TOL)."""
import os

import pytest
import torch
import torch.nn.functional as F

from tests import token_ref as R
from tests.gpu_util import TOL, check

pytestmark = pytest.mark.gpu


def layer_ref(sd, x, heads, kv, rows, sinks, theta=100.0):
    """AttnLayer on [N, C, H, W] in the parameters' precision"""
    n, c, h, w = x.shape
    d = c // heads
    t = x.flatten(2).transpose(1, 2)
    y = F.layer_norm(t, (c,), sd['norm1.weight'], sd['norm1.bias'])
    qkv = y @ sd['qkv.weight'].flatten(1).t() + sd['qkv.bias']
    q, k, v = (u.unflatten(-1, (-1, d)) for u in qkv.split([heads * d, kv * d, kv * d], -1))
    pos = torch.stack(torch.meshgrid(torch.arange(h), torch.arange(w), indexing='ij'), -1).reshape(-1, 2).double()
    f = theta ** -(torch.arange(d // 4, dtype=torch.float64) / (d // 4))
    ang = (pos[:, :, None] * f).flatten(1)[None, :, None].to(x.dtype)

    def turn(u):
        p = d // 4 * 2
        a, b = u[..., :p], u[..., p:2 * p]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), u[..., 2 * p:]], -1)
    q, k = turn(q).transpose(1, 2), turn(k).transpose(1, 2).repeat_interleave(heads // kv, 1)
    v = v.transpose(1, 2).repeat_interleave(heads // kv, 1)
    see = R.visible(1, h * w, h * w, rows * w, sinks, False, None, None)[:, None]
    p = (q @ k.transpose(2, 3) * d ** -0.5).masked_fill(~see, float('-inf')).softmax(-1)
    o = (p @ v).transpose(1, 2).flatten(2)
    t = t + o @ sd['proj.weight'].flatten(1).t() + sd['proj.bias']
    y = F.layer_norm(t, (c,), sd['norm2.weight'], sd['norm2.bias'])
    t = t + F.silu(y @ sd['fc1.weight'].flatten(1).t()) @ sd['fc2.weight'].flatten(1).t() + sd['fc2.bias']
    return t.transpose(1, 2).unflatten(2, (h, w))


@pytest.mark.parametrize('dt', [torch.float32, torch.float16], ids=['fp32', 'fp16'])
@pytest.mark.parametrize('c,heads,kv,rows,sinks,shape', [(32, 2, 2, 0, 0, (2, 5, 7)), (64, 4, 2, 2, 3, (2, 9, 12)), (96, 2, 1, 1, 0, (1, 16, 32)),
                                                         (256, 2, 2, 3, 1, (3, 8, 16))])
def test_attn_layer(c, heads, kv, rows, sinks, shape, dt):
    from multiyolov5_amd.models.common import AttnLayer
    torch.manual_seed(0)
    m = AttnLayer(c, heads, kv, rows, sinks)
    with torch.no_grad():
        for k, p in m.named_parameters():
            p.add_(torch.randn_like(p) * 0.1 * (0.3 if p.dim() > 1 else 1.0))
    sd = {k: v.double().clone().requires_grad_() for k, v in m.state_dict().items()}
    x = torch.randn(shape[0], c, *shape[1:]).to(dt)
    go = torch.randn_like(x)
    xr = x.double().requires_grad_()
    yr = layer_ref(sd, xr, heads, kv, rows, sinks)
    yr.backward(go.double())
    m = m.cuda().train()
    xg = x.cuda().requires_grad_()
    for _ in range(2):                                     # the second pass runs the built plan again: gradients are not accumulated into stale ones
        xg.grad = None
        m.zero_grad(set_to_none=True)
        y = m(xg)
        y.backward(go.cuda())
    bad = []
    check('y', y, yr, TOL[dt], collect=bad)
    check('gx', xg.grad, xr.grad, TOL[dt], collect=bad)
    for k, p in m.named_parameters():
        check(k, p.grad, sd[k].grad, TOL[dt], collect=bad)
    assert not bad, bad
    m.eval()
    with torch.no_grad():
        for _ in range(3):                                 # the third forward of a signature replays a graph
            check('eval', m(x.cuda()), yr, TOL[dt])
        if dt == torch.float16:
            check('half', m.half()(x.cuda()), yr, TOL[dt])


def test_c3attn_is_c3_around_the_layers():
    from multiyolov5_amd.models.common import C3Attn
    torch.manual_seed(1)
    m = C3Attn(32, 64, 2, 2, rows=2, sinks=1).eval()
    for mod in m.modules():
        if isinstance(mod, torch.nn.BatchNorm2d):
            mod.running_mean.normal_(0, 0.1)
            mod.running_var.uniform_(0.5, 1.5)
    x = torch.randn(2, 32, 6, 10)

    def conv(cv, t):
        return F.silu(F.batch_norm(F.conv2d(t, cv.conv.weight.double()), cv.bn.running_mean.double(), cv.bn.running_var.double(), cv.bn.weight.double(),
                                   cv.bn.bias.double(), False, 0.0, cv.bn.eps))
    with torch.no_grad():
        a = conv(m.cv1, x.double())
        for lay in m.m:
            a = layer_ref({k: v.double() for k, v in lay.state_dict().items()}, a, 2, 2, 2, 1)
        ref = conv(m.cv3, torch.cat([a, conv(m.cv2, x.double())], 1))
        check('c3attn', m.cuda()(x.cuda()), ref, TOL[torch.float32])


def test_attn_configuration_trains_and_detects():
    """yolov5s_city_seg_attn: one joint training step (finite, every parameter takes a gradient), eval fp32 against eval fp16"""
    from multiyolov5_amd.models.yolo import Model
    from multiyolov5_amd.utils.loss import ComputeLoss, SegmentationLosses
    from oracle import loss_ref, synth
    from tests.util import CFG
    torch.manual_seed(0)
    m = Model(os.path.join(CFG, 'yolov5s_city_seg_attn.yaml')).cuda().train()
    m.hyp, m.gr, m.nc = loss_ref.scaled_hyp(imgsz=128, nc=10, nl=3), 1.0, 10
    x, t, mask = synth.synth_images(2, 64, 128, seed=1).cuda(), synth.synth_det_targets(2, 8, 10, seed=1).cuda(), synth.synth_seg_targets(2, 64, 128, 19, seed=1).cuda()
    det, seg = m(x)
    loss = ComputeLoss(m)(det, t)[0] * 0.6 + SegmentationLosses()(seg, mask) * 0.7
    loss.backward()
    assert bool(torch.isfinite(loss).all())
    for k, p in m.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), k
        if any(s in k for s in ('norm1', 'norm2', 'qkv', 'proj', 'fc1', 'fc2')):
            assert float(p.grad.abs().max()) > 0, k
    m.eval()
    with torch.no_grad():
        d32, s32 = m(x)[0][0].clone(), m(x)[1].clone()
        h = m.half()
        out = h(x.half())
        check('det', out[0][0], d32, 5e-2)
        check('seg', out[1], s32, 5e-2)
