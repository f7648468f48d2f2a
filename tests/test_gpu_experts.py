"""The expert operators (dimo_amd/experts.py) on the GPU against their float64 definitions (tests/expert_cases.py has the
checks and derives the tolerances), and how they are used: strides, streams, captured graphs, together."""
import math

import pytest
import torch

from tests import expert_cases as cases

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ex():
    from dimo_amd import experts
    return experts


@pytest.mark.parametrize("T,E,k,dtype,normalize,masked,kind,pad", [
    (1, 1, 1, F32, True, False, "normal", 0),
    (0, 4, 2, F32, True, False, "normal", 0),
    (1, 64, 8, F32, True, False, "normal", 0),
    (5, 3, 3, BF16, True, True, "normal", 1),
    (4096, 8, 2, F32, True, False, "normal", 0),
    (4097, 8, 2, F32, False, True, "normal", 0),
    (333, 64, 8, F16, True, False, "ties", 0),
    (333, 17, 5, F32, True, True, "-inf", 3),
    (333, 17, 5, F32, False, False, "-inf", 0),
    (333, 33, 4, BF16, True, False, "lowest", 0),
    (333, 33, 4, F32, True, False, "lowest", 0),
    (9000, 128, 8, BF16, True, True, "ties", 0),
    (257, 256, 256, F32, False, False, "normal", 0),
    (130, 257, 9, BF16, True, True, "ties", 0),
    (77, 1024, 6, F32, True, False, "normal", 0),
    (200000, 4, 1, F32, True, False, "normal", 0),
])
def test_route(ex, T, E, k, dtype, normalize, masked, kind, pad):
    cases.check_route(ex, "cuda", T, E, k, dtype, normalize, masked, kind, pad, seed=T + E)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_route_nan_and_infinities(ex, dtype):
    cases.check_route_special(ex, "cuda", dtype)


@pytest.mark.parametrize("T,k,E,skew", [(0, 2, 3, False), (1, 1, 1, False), (1, 8, 64, False), (63, 1, 5, False),
                                        (4096, 1, 7, True), (2049, 2, 64, False), (50000, 2, 3, True), (7001, 2, 1024, False),
                                        (131072, 4, 128, False), (4096, 2, 8, False), (2730, 3, 1024, True), (8193, 1, 5, True)])
def test_group(ex, T, k, E, skew):
    cases.check_group(ex, "cuda", T, k, E, seed=T + E, skew=skew)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,K,N,act,tail,pad", [
    ([1], 1, 1, None, 0, 0),
    ([0, 3, 0], 8, 5, "silu", 2, 0),
    ([1, 0, 1, 2], 256, 64, "relu", 0, 0),
    ([70, 0, 5, 64], 40, 66, None, 3, 8),
    ([70, 0, 5, 64], 37, 65, "relu", 0, 3),
    ([130, 300], 256, 256, "silu", 1, 0),
    ([513, 0, 1, 255, 128], 360, 257, None, 0, 8),
    ([0, 0], 16, 16, None, 5, 0),
    ([65], 129, 33, "silu", 0, 0),
    ([16], 264, 72, "silu", 0, 0), ([17], 264, 72, "silu", 0, 0),        # at the borders of the kernel for few rows
    ([200, 56], 264, 72, None, 0, 0), ([200, 57], 264, 72, None, 0, 0),
    ([700], 512, 136, "relu", 60, 8),
    ([3] * 150, 72, 96, "silu", 0, 0),
    ([300, 0, 600], 24, 40, None, 0, 0),
    ([2000, 3, 1500], 264, 136, "silu", 9, 0),
    ([48 + i % 7 for i in range(128)], 40, 104, None, 3, 8),
    ([200 + i % 5 for i in range(225)], 200, 200, None, 0, 0),  # 256 x 256 tiles
    ([300, 0, 513, 128, 129, 256, 1, 700], 136, 7200, None, 5, 0),      # ... whole ones, one and two halves (forward)
    ([300, 0, 513, 128, 129, 256, 1, 700], 7200, 72, "silu", 130, 0),   # (gradient of x)
    ([1024] * 8, 136, 1800, "relu", 0, 0),                              # (no halves)
])
def test_products(ex, counts, K, N, dtype, act, tail, pad):
    cases.check_products(ex, "cuda", counts, K, N, dtype, act, tail, pad, seed=K)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,k,E,K,N,pad", [(1, 1, 1, 3, 2, 0), (1, 2, 8, 512, 256, 0), (200, 2, 4, 256, 128, 8), (150, 3, 5, 33, 17, 1)])
def test_products_gathered(ex, T, k, E, K, N, dtype, pad):
    cases.check_gather(ex, "cuda", T, k, E, K, N, dtype, seed=K, pad=pad)


@pytest.mark.parametrize("T,k,E,N,dtype,weighted,residual,pad", [
    (1, 1, 1, 1, F32, True, True, 0), (500, 2, 5, 64, BF16, True, True, 8), (211, 3, 5, 33, F32, False, False, 1),
    (99, 2, 2, 520, F16, True, False, 0), (301, 8, 16, 1024, F32, True, True, 0)])
def test_combine(ex, T, k, E, N, dtype, weighted, residual, pad):
    cases.check_combine(ex, "cuda", T, k, E, N, dtype, weighted, residual, pad, seed=N)


@pytest.mark.parametrize("T,K,F,E,k,act", [(1, 8, 8, 2, 1, "silu"), (126, 24, 40, 5, 2, "silu"), (600, 256, 128, 8, 2, "silu")])
def test_layer(ex, T, K, F, E, k, act):
    cases.check_layer(ex, "cuda", T, K, F, E, k, act)


@pytest.mark.parametrize("T,K,F,E,k,dtype,act,biases", [
    (0, 8, 8, 3, 2, F32, "relu", True), (1, 256, 512, 3, 1, BF16, "silu", True), (700, 256, 256, 8, 2, F32, "silu", True),
    (3000, 256, 512, 8, 2, BF16, "relu", True), (50, 33, 40, 4, 3, F16, "silu", False), (333, 16, 16, 2, 2, BF16, None, False)])
def test_layer_is_its_parts(ex, T, K, F, E, k, dtype, act, biases):
    cases.check_layer_is_its_parts(ex, "cuda", T, K, F, E, k, dtype, act, biases, seed=T)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,K,N,tail", [
    ([0, 1500, 100, 0, 960], 24, 40, 5),    # cut into slices of 256 rows, whole, empty
    ([0, 1500, 100, 0, 960], 23, 41, 0),
    ([256, 512, 257, 1, 1600], 16, 8, 3),   # at the borders of a slice
    ([0] * 30 + [26000] + [500] * 20 + [17] * 19, 16, 24, 0),  # more than 64 groups
    ([6000], 264, 520, 0),                  # one group, wide
])
def test_weight_gradients_of_cut_groups(ex, counts, K, N, dtype, tail):
    cases.check_products(ex, "cuda", counts, K, N, dtype, None, tail, 0, seed=K)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weight_gradients_of_groups_beyond_twice_the_mean(ex, dtype):
    """128 x 128 tiles enough for the chip: only the groups of more than twice the mean are cut."""
    counts = [512] * 120 + [4000, 0, 1100, 30, 1, 1500, 0, 2000]
    cases.check_products(ex, "cuda", counts, 256, 256, dtype, None, 0, 0, seed=8)


def test_weight_gradients_of_cut_groups_gathered(ex):
    cases.check_gather(ex, "cuda", 1100, 2, 4, 24, 16, BF16, seed=5, pad=0)
    cases.check_gather(ex, "cuda", 1100, 2, 4, 200, 136, F16, seed=7, pad=8)
    cases.check_gather(ex, "cuda", 700, 2, 2, 9, 7, F32, seed=6, pad=1)


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (1, 2), (0, 2)])
def test_only_the_gradients_that_are_wanted(ex, wanted):
    cases.check_wanted(ex, "cuda", wanted)


def test_offsets_beyond_32_bits(ex):
    """Rows whose elements lie more than 2^31 behind their matrix' first: products, their gradients, sums and routing of
    the last rows against float64."""
    R, K, N, n = 1_100_000, 2048, 8, 70
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)
    x, w, gy = r(R, K), (r(2, N, K) / 64).requires_grad_(True), r(R, N)
    x.requires_grad_(True)
    groups = ex.RowGroups(torch.tensor([0, 1000, R], dtype=torch.int32, device="cuda"))
    y = ex.grouped_linear(x, w, groups)
    gx, = torch.autograd.grad(y, x, gy)
    X, W, G = x[-n:].detach().double().cpu(), w[1].detach().double().cpu(), gy[-n:].double().cpu()
    cases.near(y[-n:], X @ W.T, BF16, cases.product_slack(K, X.abs() @ W.abs().T), "y")
    cases.near(gx[-n:], G @ W, BF16, cases.product_slack(N, G.abs() @ W.abs()), "g_x")
    del y, gx
    # the weight gradient of a group that lies behind 2^31 elements
    late = ex.RowGroups(torch.tensor([0, R - n, R], dtype=torch.int32, device="cuda"))
    gw, _ = ex._linear_wgrad(gy, x.detach(), (2, N, K), late, False, False)
    cases.near(gw[1], G.T @ X, BF16, cases.product_slack(n, G.abs().T @ X.abs()), "g_w")
    # the last rows brought back to the first places, the first to the last
    position = torch.arange(R - 1, -1, -1, dtype=torch.int32, device="cuda")[:, None]
    late.order, late.position, late.rows = position[:, 0], position, position[:, 0]
    out = ex.combine_rows(x.detach(), late)
    assert torch.equal(out[:n], x[-n:].flip(0)) and torch.equal(out[-n:], x[:n].flip(0))
    del out, x
    z = r(2 ** 21 + 77, 1024)
    weights, experts, _ = ex.route_topk(z, 3)
    some, which, _ = ex.route_topk(z[-n:].clone(), 3)
    assert torch.equal(weights[-n:], some) and torch.equal(experts[-n:], which)


def _layer_leaves(T, K, F, E, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return [t.to(dtype).requires_grad_(True) for t in (r(T, K), r(T, E), r(E, F, K) / math.sqrt(K), r(E, F), r(E, K, F) / math.sqrt(F), r(E, K))]


def test_same_results_every_time_and_on_another_stream(ex):
    """No result depends on the schedule: a second call, and one on another stream, give the same bits."""
    leaves = _layer_leaves(1000, 256, 128, 8, BF16, 3)
    go = torch.ones_like(leaves[0])

    def step():
        out = ex.expert_mlp(*leaves, k=2, activation="silu")
        return (out.detach(),) + torch.autograd.grad(out, leaves, go)
    first = step()
    again = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, again, there):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_steps(ex):
    """Two captured training steps (their workspaces are the graphs' own) replayed in turns, new inputs every time, the
    eager step between them."""
    graphs = []
    for seed in (1, 2):
        leaves = _layer_leaves(700, 128, 64, 4, F32, seed)
        go = torch.randn_like(leaves[0])

        def step(leaves=leaves, go=go):
            out = ex.expert_mlp(*leaves, k=2, activation="silu")
            return (out.detach(),) + torch.autograd.grad(out, leaves, go)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, leaves, step, outs))
    for it in range(3):
        for n, (graph, leaves, step, outs) in enumerate(graphs):
            g = torch.Generator(device="cuda").manual_seed(10 * it + n)
            with torch.no_grad():
                leaves[0].copy_(torch.randn(leaves[0].shape, generator=g, device="cuda"))
                leaves[1].copy_(torch.randn(leaves[1].shape, generator=g, device="cuda"))
        for graph, _, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, _, step, outs in graphs:
            for got, ref in zip(outs, step()):
                assert torch.equal(got, ref)


@pytest.mark.parametrize("W,P,M,E,k", [(64, 2, 70, 4, 2), (256, 4, 128, 8, 2)])
def test_timenet_with_experts(W, P, M, E, k):
    cases.check_timenet_with_experts("cuda", W, P, M, E, k)


def test_quantized_block(ex):
    from dimo_amd import mx4
    cases.check_quantized_block(ex, mx4, "cuda", 300, 256, 8, 2)


@pytest.mark.parametrize("direct", [True, False])
def test_train_step_with_experts(direct):
    """The trainer's own step with an expert block in the deformation network: every parameter of the block moves once
    its second products have left zero."""
    from dimo_amd.rasterizer import CapacityPolicy
    from dimo_amd.renderer import Renderer
    from dimo_amd.synth import init_synthetic_model
    from dimo_amd.trainer import TrainConfig, Trainer
    cfg = TrainConfig(num_pts=2000, num_cpts=64, num_motions=4, resolution=128, motions_per_step=2, views_per_step=1,
                      frames_per_step=2)
    rd = Renderer(sh_degree=0, num_latent_code=4, add_normal=True, device="cuda", capacity=CapacityPolicy(initial=1 << 18),
                  timenet_experts=4, timenet_top_k=2)
    init_synthetic_model(rd, cfg.num_pts, cfg.num_cpts, seed=0, num_latent=4)
    tr = Trainer(cfg, rd, direct=direct)
    block = rd.gaussians._timenet.experts
    before = {n: p.detach().clone() for n, p in block.named_parameters()}
    for _ in range(3):
        tr.train_step()
    torch.cuda.synchronize()
    assert torch.isfinite(rd.gaussians.flat_params).all()
    for n, p in block.named_parameters():
        assert not torch.equal(before[n], p.detach()), n
