"""How the expert operators stand to autograd beyond their gradients (tests/expert_cases.py): forward-mode derivatives are
refused, never dropped; a grouping that changes between a forward pass and its backward is an error, not another gradient."""
import pytest
import torch
from torch.autograd import forward_ad

from dimo_amd import experts as ex
from dimo_amd import mx4
from tests import expert_emulation


@pytest.fixture
def emulated(monkeypatch):
    expert_emulation.use(monkeypatch, ex, mx4)


def _inputs():
    torch.manual_seed(0)
    return torch.randn(6, 8), torch.randn(6, 3), torch.randn(3, 5, 8), torch.randn(3, 5), torch.randn(3, 8, 5), torch.randn(3, 8)


CALLS = {
    "route_topk": (lambda x, z, w1, b1, w2, b2, g: ex.route_topk(z, 2)[0], (1,)),
    "grouped_linear": (lambda x, z, w1, b1, w2, b2, g: ex.grouped_linear(x, w1, g, b1, "silu", gather=True), (0, 2, 3)),
    "combine_rows": (lambda x, z, w1, b1, w2, b2, g: ex.combine_rows(x.repeat(2, 1), g, z[:, :2].contiguous(), x), (0, 1)),
    "expert_mlp": (lambda x, z, w1, b1, w2, b2, g: ex.expert_mlp(x, z, w1, b1, w2, b2, 2), (0, 1, 2, 3, 4, 5)),
    "quantize_mx4": (lambda x, z, w1, b1, w2, b2, g: mx4.quantize_mx4(x).dequantize(), (0,)),
    "mx4_linear": (lambda x, z, w1, b1, w2, b2, g: mx4.mx4_linear(mx4.quantize_mx4(w2[0]), mx4.quantize_mx4(w1), b1, g4(), None,
                                                                  torch.float32), (3,)),
}


def g4():
    return ex.RowGroups(torch.tensor([0, 4, 4, 8], dtype=torch.int32))


def _call(name, tensors):
    fn, _ = CALLS[name]
    groups = ex.group_rows(ex.route_topk(_inputs()[1], 2)[1], 3)
    if name == "mx4_linear":  # (w2[0] is [8, 5], w1 [3, 5, 8]: equal columns)
        tensors = list(tensors)
        tensors[2] = _inputs()[2][:, :, :5].contiguous()
    return fn(*tensors, groups)


@pytest.mark.parametrize("name,which", [(n, i) for n, (_, at) in CALLS.items() for i in at])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(emulated, name, which, grad):
    tensors = list(_inputs())
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            _call(name, tensors)


@pytest.mark.parametrize("name", list(CALLS))
def test_an_open_level_changes_nothing_without_tangents(emulated, name):
    want = _call(name, _inputs())
    with forward_ad.dual_level():
        got = _call(name, _inputs())
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["offsets", "rows", "position"])
def test_a_grouping_that_changed_is_an_error(emulated, name):
    x, z, w1, b1, _, _ = (t.requires_grad_(True) for t in _inputs())
    groups = ex.group_rows(ex.route_topk(z, 2)[1], 3)
    y = ex.grouped_linear(x, w1, groups, b1, "relu", gather=True)
    out = ex.combine_rows(y, groups, ex.route_topk(z, 2)[0])
    getattr(groups, name).zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out.sum(), (x, w1, z))
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), (x, w1))


def test_a_grouping_that_was_replaced_keeps_the_gradient(emulated):
    x, _, w1, _, _, _ = (t.requires_grad_(True) for t in _inputs())
    groups = g4()
    rows = x.repeat(2, 1)[:8]
    y = ex.grouped_linear(rows, w1, groups)
    want = torch.autograd.grad(y.sum(), w1, retain_graph=True)[0]
    groups.offsets = torch.tensor([0, 0, 8, 8], dtype=torch.int32)
    assert torch.equal(torch.autograd.grad(y.sum(), w1)[0], want)


def test_a_quantized_block_is_not_trained_through(emulated):
    """What lies before a quantized block would get no gradient, silently."""
    torch.manual_seed(0)
    block = ex.ExpertMLP(16, 3, 2)
    q, h = block.quantized(), torch.randn(5, 16)
    want = q(h)
    assert not want.requires_grad
    with pytest.raises(RuntimeError, match="no_grad"):
        q(h.clone().requires_grad_(True))
    with torch.no_grad():
        assert torch.equal(q(h.clone().requires_grad_(True)), want)
