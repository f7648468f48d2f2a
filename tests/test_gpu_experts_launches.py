"""Sizes whose work takes more threads than one launch does (2^32), on the GPU: every row is reached, the ones behind the
first launch's among them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ex():
    from dimo_amd import experts
    return experts


def _random(*shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(shape[0] % 997)).to(BF16)


def test_sum_backward(ex):
    T, N = (1 << 26) + 5, 8
    position = torch.arange(T - 1, -1, -1, dtype=torch.int32, device="cuda")[:, None]
    groups = ex.RowGroups(torch.tensor([0, T], dtype=torch.int32, device="cuda"))
    groups.order, groups.position, groups.rows = position[:, 0], position, position[:, 0]
    y = _random(T, N).requires_grad_(True)
    w = torch.full((T, 1), 0.5, device="cuda").requires_grad_(True)
    out = ex.combine_rows(y, groups, w)
    assert torch.equal(out.detach(), 0.5 * y.detach().flip(0))
    g = _random(T, N)
    gy, gw = torch.autograd.grad(out, (y, w), g)
    assert torch.equal(gy, 0.5 * g.flip(0))
    # (sums of eight products, in another order: each within eight roundings of its terms' sizes)
    terms = y.detach().flip(0).float() * g.float()
    assert bool(((gw[:, 0] - terms.sum(1)).abs() <= 16 * 2.0 ** -24 * terms.abs().sum(1)).all())


def test_activation_backward(ex):
    n = (1 << 32) + 1  # (odd: an element at a time)
    g = torch.full((n,), 2.0, dtype=BF16, device="cuda")
    saved = torch.full((n,), -1.0, dtype=BF16, device="cuda")
    saved[::2] = 1.0
    out = ex._activation_backward(g, saved, 1)
    del g
    saved.clamp_(min=0).mul_(2)
    assert torch.equal(out[-1000:], saved[-1000:]) and torch.equal(out[:1 << 31], saved[:1 << 31])
    assert torch.equal(out[1 << 31:], saved[1 << 31:])


def test_products(ex):
    R = 1 << 30
    x = _random(R, 1).requires_grad_(True)
    w = torch.tensor([[[0.375]]], dtype=BF16, device="cuda")
    y = ex.grouped_linear(x, w, ex.RowGroups(torch.tensor([0, R], dtype=torch.int32, device="cuda")))
    assert torch.equal(y.detach(), x.detach() * w[0, 0, 0])  # (one product each, rounded once)
    g = _random(R, 1)
    gx, = torch.autograd.grad(y, x, g)
    assert torch.equal(gx, g * w[0, 0, 0])


def test_grouping_grows_with_its_places(ex):
    """2^26 places: sorted as a stable sort does, in no more than twice the eightfold time of 2^23 (sums of all workgroups'
    counts by every workgroup would take 64 times as long)."""
    E, times = 128, []
    for S in (1 << 23, 1 << 26):
        experts = torch.randint(0, E, (S, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(S), dtype=torch.int32)
        groups = ex.group_rows(experts, E)
        took = []
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            groups = ex.group_rows(experts, E)
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        times.append(min(took))
        key, order = torch.sort(experts[:, 0], stable=True)
        assert torch.equal(groups.order, order.to(torch.int32)) and torch.equal(groups.rows, groups.order)
        assert torch.equal(groups.offsets, torch.searchsorted(key, torch.arange(E + 1, device="cuda", dtype=torch.int32)).to(torch.int32))
        assert torch.equal(groups.position[:, 0][order], torch.arange(S, device="cuda", dtype=torch.int32))
    print(times)
    assert times[1] <= 16 * times[0], times


def test_captured_grouping_of_many_places(ex):
    """The three launches of a large grouping, captured once and replayed on other places: what the eager call gives."""
    E, S = 128, 300 * 4096 - 7
    experts = torch.zeros(S, 1, dtype=torch.int32, device="cuda")
    draw = lambda seed: torch.randint(-1, E, (S, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed), dtype=torch.int32)
    ex.group_rows(experts, E)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        groups = ex.group_rows(experts, E)
    for seed in range(4):
        experts.copy_(draw(seed))
        graph.replay()
        torch.cuda.synchronize()
        want = ex.group_rows(experts, E)
        for name in ("offsets", "order", "position", "rows"):
            assert torch.equal(getattr(groups, name), getattr(want, name)), (seed, name)
