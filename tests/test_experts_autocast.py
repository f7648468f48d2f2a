"""Expert blocks under torch.autocast, on the CPU SIMT emulation: they work in their parameters' type."""
import pytest
import torch

from dimo_amd import experts as ex
from dimo_amd import mx4
from tests import expert_emulation


@pytest.fixture
def emulated(monkeypatch):
    expert_emulation.use(monkeypatch, ex, mx4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_under_autocast(emulated, dtype):
    torch.manual_seed(0)
    block = ex.ExpertMLP(16, 3, 2)
    with torch.no_grad():
        block.w2.copy_(torch.randn(block.w2.shape))
    h = torch.randn(9, 16).to(dtype)
    for b in (block, block.quantized()):
        want = b(h.float())
        with torch.autocast("cpu", torch.bfloat16):
            got = b(h)
        assert got.dtype == torch.float32 and torch.equal(got, want)


def test_gradients_under_autocast(emulated):
    torch.manual_seed(0)
    block = ex.ExpertMLP(16, 3, 2)
    with torch.no_grad():
        block.w2.copy_(torch.randn(block.w2.shape))
    h, go = torch.randn(9, 16).to(torch.bfloat16).requires_grad_(True), torch.randn(9, 16)
    leaves = [h] + list(block.parameters())
    want = torch.autograd.grad(block(h.float()), leaves, go)
    with torch.autocast("cpu", torch.bfloat16):
        out = block(h)
    for a, b in zip(torch.autograd.grad(out, leaves, go), want):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_timenet_under_autocast(emulated):
    """A whole deformation network: what ran under autocast without experts runs with them."""
    from dimo_amd.deform import TimeNet
    torch.manual_seed(0)
    net = TimeNet(D=2, W=16, skips=(), latent_code_dim=4, experts=3, top_k=2)
    pts, t, lat = torch.rand(1, 5, 3), torch.rand(2, 5, 1), torch.randn(2, 5, 4)
    with torch.autocast("cpu", torch.bfloat16):
        dx, dq = net(pts, t, lat, t_apply=True)
    assert dx.shape == (2, 5, 3) and dq.shape == (2, 5, 4)
    (dx.float().sum() + dq.float().sum()).backward()
