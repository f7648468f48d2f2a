"""SSIM and its gradient on the GPU (dimo_amd/fused_ssim.py) for one plane per image, against the formula of
src/loss.py:144-175 in float64 on the host."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 1, 16, 16), (1, 1, 11, 40)])
def test_ssim_against_host_reference(shape):
    from dimo_amd.fused_ssim import fused_ssim
    g = torch.Generator().manual_seed(shape[2])
    a = torch.rand(shape, generator=g)
    b = torch.rand(shape, generator=g) * 0.5 + 0.25 * a
    w = torch.tensor(np.exp(-(np.arange(11) - 5) ** 2 / (2 * 1.5 ** 2)))
    w = w / w.sum()
    win = (w[:, None] * w[None, :])[None, None].expand(shape[1], 1, 11, 11)
    x, y = a.double().requires_grad_(True), b.double()
    conv = lambda t: F.conv2d(t, win, padding=5, groups=shape[1])
    mu1, mu2 = conv(x), conv(y)
    s1, s2, s12 = conv(x * x) - mu1 ** 2, conv(y * y) - mu2 ** 2, conv(x * y) - mu1 * mu2
    r = (((2 * mu1 * mu2 + 1e-4) * (2 * s12 + 9e-4)) / ((mu1 ** 2 + mu2 ** 2 + 1e-4) * (s1 + s2 + 9e-4))).mean()
    gr, = torch.autograd.grad(r, x)
    ad = a.cuda().requires_grad_(True)
    s = fused_ssim(ad, b.cuda())
    gs, = torch.autograd.grad(s, ad)
    assert abs(s.item() - r.item()) < 2e-5
    assert (gs.cpu() - gr).abs().sum() / gr.abs().sum() < 1e-3
