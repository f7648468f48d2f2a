"""GaussianModel.quantize_experts on the CPU SIMT emulation: the deformation network of a render-only model."""
import pytest
import torch

from dimo_amd import experts as ex
from dimo_amd import mx4
from tests import expert_emulation


def _model(experts):
    from dimo_amd.gaussian_model import GaussianModel
    torch.manual_seed(0)
    return GaussianModel(0, num_latent_code=2, device="cpu", timenet_experts=experts)


def test_quantized_network(monkeypatch):
    expert_emulation.use(monkeypatch, ex, mx4)
    g = _model(3)
    net = g._timenet
    with torch.no_grad():
        net.experts.w2.copy_(torch.randn(net.experts.w2.shape) / 16)
        for lin in (net.pts_layers[-1], net.rot_layers[-1]):
            lin.weight.copy_(torch.randn(lin.weight.shape))
    pts, t, lat = torch.rand(1, 7, 3), torch.rand(2, 7, 1), torch.randn(2, 7, 32)
    block = net.experts
    with torch.no_grad():
        full = net(pts, t, lat, t_apply=True)
        net.experts = block.quantized()
        want = net(pts, t, lat, t_apply=True)
        net.experts = block
        g.quantize_experts()
        got = net(pts, t, lat, t_apply=True)
    for a, b, f in zip(got, want, full):
        assert torch.equal(a, b) and not torch.equal(a, f)
    assert isinstance(net.experts, ex.QuantizedExpertMLP)
    with pytest.raises(RuntimeError, match="no_grad"):
        net(pts, t, lat, t_apply=True)
    with pytest.raises(ValueError):
        g.quantize_experts()


def test_a_network_without_experts_is_refused():
    with pytest.raises(ValueError):
        _model(0).quantize_experts()
