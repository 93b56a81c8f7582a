"""Token operators near the largest sizes: a layer norm whose parameter sums do not fit one launch of a workgroup per 16 channels."""
import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu


def test_layer_norm_of_very_many_channels():
    from multiyolov5_amd.utils import tokens as T
    c = (1 << 25) + 3
    g = torch.Generator(device='cuda').manual_seed(1)
    x, go = (torch.empty(2, c, dtype=torch.float16, device='cuda').normal_(generator=g) for _ in range(2))
    w, b = torch.ones(c, device='cuda', requires_grad=True), torch.zeros(c, device='cuda', requires_grad=True)
    leaf = x.clone().requires_grad_()
    y = T.layer_norm(leaf, w, b)
    gx, gw, gb = torch.autograd.grad(y, (leaf, w, b), go)
    X, G = x.double(), go.double()
    var, mu = torch.var_mean(X, 1, unbiased=False, keepdim=True)
    xh = (X - mu) / (var + 1e-5).sqrt()
    # a thread adds c / 256 values one after the other, then 256 sums are added: (c / 256 + 256) roundings of sums of |x| <= 1 (and squares) a channel
    e = (c / 256 + 256) * R.E
    assert bool(((gb.double() - G.sum(0)).abs() <= 4 * R.E * G.abs().sum(0)).all())
    assert bool(((gw.double() - (G * xh).sum(0)).abs() <= 2 * e * (G.abs() * (1 + xh.abs())).sum(0)).all())
    gxd = (G - G.mean(1, keepdim=True) - xh * (G * xh).mean(1, keepdim=True)) / (var + 1e-5).sqrt()
    for got, ref in ((y, xh), (gx, gxd)):
        assert bool(((got.double() - ref).abs() <= 4 * e * (1 + xh.abs() + G.abs()) + R.half_step(torch.float16) * ref.abs() + R.tiny(torch.float16)).all())
