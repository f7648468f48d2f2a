"""The expert kernels (dimo_amd/csrc/experts.hip, grouped.hip, as hipcc compiles them) on the CPU SIMT emulation, through
dimo_amd/experts.py, against float64 definitions (tests/expert_cases.py); and what the entry points refuse."""
import math

import pytest
import torch

from dimo_amd import experts as ex
from tests import expert_cases as cases
from tests import expert_emulation

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture
def emulated(monkeypatch):
    expert_emulation.use(monkeypatch, ex)


@pytest.mark.parametrize("T,E,k,dtype,normalize,masked,kind,pad", [
    (1, 1, 1, F32, True, False, "normal", 0),
    (0, 4, 2, F32, True, False, "normal", 0),
    (5, 3, 3, BF16, True, True, "normal", 1),
    (70, 8, 2, F32, True, False, "normal", 0),
    (70, 8, 2, F32, False, True, "normal", 0),
    (33, 64, 8, F16, True, False, "ties", 0),
    (33, 17, 5, F32, True, True, "-inf", 3),
    (33, 17, 5, F32, False, False, "-inf", 0),
    (9, 130, 5, F32, False, False, "normal", 0),
    (9, 33, 4, BF16, True, False, "lowest", 0),
    (9, 33, 4, F32, True, False, "lowest", 0),
    (7, 257, 9, BF16, True, True, "ties", 0),
    (3, 1024, 6, F32, True, False, "normal", 0),
])
def test_route(emulated, T, E, k, dtype, normalize, masked, kind, pad):
    cases.check_route(ex, "cpu", T, E, k, dtype, normalize, masked, kind, pad, seed=T + E)


def test_route_nan_and_infinities(emulated):
    cases.check_route_special(ex, "cpu", F32)


@pytest.mark.parametrize("T,k,E,skew", [(0, 2, 3, False), (1, 1, 1, False), (1, 8, 64, False), (63, 1, 5, False),
                                        (4096, 1, 7, True), (2049, 2, 64, False), (5000, 2, 3, True), (700, 2, 1024, False),
                                        (4096, 2, 8, False), (2730, 3, 1024, True), (8193, 1, 5, True)])
def test_group(emulated, T, k, E, skew):
    cases.check_group(ex, "cpu", T, k, E, seed=T + E, skew=skew)


@pytest.mark.parametrize("counts,K,N,dtype,act,tail,pad", [
    ([1], 1, 1, F32, None, 0, 0),
    ([0, 3, 0], 8, 5, F32, "silu", 2, 0),
    ([70, 0, 5, 64], 40, 66, BF16, None, 3, 8),
    ([70, 0, 5, 64], 37, 65, F16, "relu", 0, 3),
    ([33, 130], 72, 64, F32, "silu", 1, 0),
    ([233, 130], 72, 64, F32, "silu", 1, 0),  # (more rows than the kernel for few of them takes)
    ([0, 0], 16, 16, BF16, None, 5, 0),
    ([65], 129, 33, BF16, "silu", 0, 0),
    ([300, 0, 600], 24, 40, BF16, None, 0, 0),     # weight gradients from slices of the rows
    ([300, 0, 600], 23, 41, F32, None, 7, 0),
    ([48 + i % 7 for i in range(128)], 40, 104, BF16, None, 3, 8),  # 128 x 128 tiles
])
def test_products(emulated, counts, K, N, dtype, act, tail, pad):
    cases.check_products(ex, "cpu", counts, K, N, dtype, act, tail, pad, seed=K)


@pytest.mark.parametrize("T,k,E,K,N,dtype,pad", [(1, 1, 1, 3, 2, F32, 0), (37, 2, 4, 24, 40, BF16, 4), (20, 3, 5, 33, 17, F32, 1)])
def test_products_gathered(emulated, T, k, E, K, N, dtype, pad):
    cases.check_gather(ex, "cpu", T, k, E, K, N, dtype, seed=K, pad=pad)


@pytest.mark.parametrize("T,k,E,N,dtype,weighted,residual,pad", [
    (1, 1, 1, 1, F32, True, True, 0), (21, 2, 5, 64, BF16, True, True, 8), (21, 3, 5, 33, F32, False, False, 1),
    (9, 2, 2, 520, F16, True, False, 0)])
def test_combine(emulated, T, k, E, N, dtype, weighted, residual, pad):
    cases.check_combine(ex, "cpu", T, k, E, N, dtype, weighted, residual, pad, seed=N)


@pytest.mark.parametrize("T,K,F,E,k,act", [(1, 8, 8, 2, 1, "silu"), (26, 24, 40, 5, 2, "silu")])
def test_layer(emulated, T, K, F, E, k, act):
    cases.check_layer(ex, "cpu", T, K, F, E, k, act)


@pytest.mark.parametrize("T,K,F,E,k,dtype,act,biases", [
    (0, 8, 8, 3, 2, F32, "relu", True), (1, 8, 24, 3, 1, BF16, "silu", True), (70, 40, 33, 4, 2, F32, "silu", True),
    (50, 64, 40, 4, 2, BF16, "relu", True), (50, 33, 40, 4, 3, F16, "silu", False), (33, 16, 16, 2, 2, BF16, None, False)])
def test_layer_is_its_parts(emulated, T, K, F, E, k, dtype, act, biases):
    cases.check_layer_is_its_parts(ex, "cpu", T, K, F, E, k, dtype, act, biases, seed=T)


@pytest.mark.parametrize("counts,K,N,dtype,tail", [
    ([0, 1500, 100, 0, 960], 24, 40, BF16, 5),   # cut into slices of 256 rows, whole, empty
    ([0, 1500, 100, 0, 960], 23, 41, F32, 0),
    ([256, 512, 257, 1, 1600], 16, 8, F16, 3),   # at the borders of a slice
])
def test_weight_gradients_of_cut_groups(emulated, counts, K, N, dtype, tail):
    cases.check_products(ex, "cpu", counts, K, N, dtype, None, tail, 0, seed=K)


def test_weight_gradients_of_cut_groups_gathered(emulated):
    cases.check_gather(ex, "cpu", 1100, 2, 4, 24, 16, BF16, seed=5, pad=0)
    cases.check_gather(ex, "cpu", 700, 2, 2, 9, 7, F32, seed=6, pad=1)


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (1, 2), (0, 2)])
def test_only_the_gradients_that_are_wanted(emulated, wanted):
    cases.check_wanted(ex, "cpu", wanted)


def test_bad_offsets_stay_inside_the_weight_gradients(emulated):
    for R, bad in ((40, [0, 100, -5, 40]), (1600, [0, 1600, 10, 1600]), (1600, [7, 2 ** 31 - 1, -2 ** 31, 3]),
                   (1600, [0, 1600, 0, 1600])):
        x, g = torch.randn(R, 8), torch.randn(R, 4)
        w = torch.randn(3, 4, 8, requires_grad=True)
        b = torch.randn(3, 4, requires_grad=True)
        for rows in (None, torch.arange(R, dtype=torch.int32)):
            groups = ex.RowGroups(torch.tensor(bad, dtype=torch.int32))
            if rows is not None:
                groups.order, groups.rows, groups.position = rows, rows, rows[:, None]
            torch.autograd.grad(ex.grouped_linear(x, w, groups, b, gather=rows is not None), (w, b), g)


def test_bad_offsets_stay_inside(emulated):
    """Offsets that the caller got wrong give wrong rows, never an address outside (run under AddressSanitizer too)."""
    x, w = torch.randn(40, 8), torch.randn(3, 4, 8)
    for bad in ([0, 100, -5, 40], [0, 40, 10, 1000], [7, 2 ** 31 - 1, -2 ** 31, 3]):
        groups = ex.RowGroups(torch.tensor(bad, dtype=torch.int32))
        xg = x.clone().requires_grad_(True)
        y = ex.grouped_linear(xg, w, groups)
        torch.autograd.grad(y.sum(), xg)


def test_refusals():
    z = torch.zeros(4, 6)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ex.route_topk(z, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ex.group_rows(torch.zeros(4, 2, dtype=torch.int32), 6)


@pytest.mark.parametrize("call", [
    lambda: ex.route_topk(torch.zeros(4, 6), 0),
    lambda: ex.route_topk(torch.zeros(4, 6), 7),
    lambda: ex.route_topk(torch.zeros(4, 1025), 2),
    lambda: ex.route_topk(torch.zeros(4, 6, dtype=torch.float64), 2),
    lambda: ex.route_topk(torch.zeros(6), 2),
    lambda: ex.route_topk(torch.zeros(4, 6), 2, row_mask=torch.ones(4)),
    lambda: ex.route_topk(torch.zeros(4, 6), 2, row_mask=torch.ones(5, dtype=torch.bool)),
    lambda: ex.group_rows(torch.zeros(4, 2, dtype=torch.int64), 6),
    lambda: ex.group_rows(torch.zeros(4, 2, dtype=torch.int32), 0),
    lambda: ex.RowGroups(torch.zeros(4, dtype=torch.int64)),
    lambda: ex.RowGroups(torch.zeros(1, dtype=torch.int32)),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(3, 5, 9), ex.RowGroups(torch.zeros(4, dtype=torch.int32))),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(2, 5, 8), ex.RowGroups(torch.zeros(4, dtype=torch.int32))),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(3, 5, 8).half(), ex.RowGroups(torch.zeros(4, dtype=torch.int32))),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(3, 5, 8), ex.RowGroups(torch.zeros(4, dtype=torch.int32)),
                              bias=torch.zeros(3, 4)),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(3, 5, 8), ex.RowGroups(torch.zeros(4, dtype=torch.int32)),
                              activation="gelu"),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(3, 5, 8), ex.RowGroups(torch.zeros(4, dtype=torch.int32)),
                              gather=True),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(6, 5, 8), ex.group_rows(torch.zeros(3, 2, dtype=torch.int32), 6),
                              gather=True),
    lambda: ex.grouped_linear(torch.zeros(4, 8), torch.zeros(6, 5, 8), ex.group_rows(torch.zeros(4, 2, dtype=torch.int32), 6)),
    lambda: ex.expert_mlp(torch.zeros(4, 8), torch.zeros(4, 3), torch.zeros(3, 5, 8), None, torch.zeros(3, 8, 5), None, 4),
    lambda: ex.expert_mlp(torch.zeros(4, 8), torch.zeros(5, 3), torch.zeros(3, 5, 8), None, torch.zeros(3, 8, 5), None, 2),
    lambda: ex.expert_mlp(torch.zeros(4, 8), torch.zeros(4, 3), torch.zeros(3, 5, 8), None, torch.zeros(3, 8, 6), None, 2),
    lambda: ex.expert_mlp(torch.zeros(4, 8), torch.zeros(4, 3).half(), torch.zeros(3, 5, 8), None, torch.zeros(3, 8, 5), None, 2),
    lambda: ex.expert_mlp(torch.zeros(4, 8), torch.zeros(4, 3), torch.zeros(3, 5, 8), None, torch.zeros(3, 8, 5),
                          torch.zeros(3, 5), 2),
    lambda: ex.expert_mlp(torch.zeros(4, 8), torch.zeros(4, 3), torch.zeros(3, 5, 8), None, torch.zeros(3, 8, 5), None, 2, "tanh"),
    lambda: ex.expert_mlp(torch.zeros(4, 8), torch.zeros(4, 3), torch.zeros(3, 5, 8), None, torch.zeros(3, 8, 5), None, 2,
                          row_mask=torch.zeros(3, dtype=torch.bool)),
    lambda: ex.combine_rows(torch.zeros(4, 8), ex.RowGroups(torch.zeros(4, dtype=torch.int32))),
    lambda: ex.combine_rows(torch.zeros(4, 8), ex.group_rows(torch.zeros(4, 2, dtype=torch.int32), 6)),
    lambda: ex.combine_rows(torch.zeros(8, 8), ex.group_rows(torch.zeros(4, 2, dtype=torch.int32), 6),
                            weights=torch.zeros(4, 2, dtype=torch.float64)),
    lambda: ex.combine_rows(torch.zeros(8, 8), ex.group_rows(torch.zeros(4, 2, dtype=torch.int32), 6),
                            residual=torch.zeros(4, 7)),
])
def test_bad_arguments(emulated, call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda many: ex.route_topk(torch.zeros(1).expand(many, 2), 1),
    lambda many: ex.group_rows(torch.zeros(1, dtype=torch.int32).expand(many // 2 + 1, 2), 2),
    lambda many: ex.grouped_linear(torch.zeros(1).expand(many, 1), torch.zeros(1, 1, 1), ex.RowGroups(torch.zeros(2, dtype=torch.int32))),
    lambda many: ex.grouped_linear(torch.zeros(1, 1), torch.zeros(1).expand(1, many, 1), ex.RowGroups(torch.zeros(2, dtype=torch.int32))),
    lambda many: ex.expert_mlp(torch.zeros(1).expand(many // 2 + 1, 1), torch.zeros(1).expand(many // 2 + 1, 2), torch.zeros(2, 1, 1),
                               None, torch.zeros(2, 1, 1), None, k=2),
])
def test_sizes_beyond_the_indices(emulated, call):
    with pytest.raises(ValueError, match="rows, places and columns"):
        call(ex.MAX_SIZE + 1)


def test_c_entry_points_refuse_sizes():
    L, many = expert_emulation.emulated_library(), (1 << 30) + 1
    assert L.dimo_route_topk_forward(many, 6, 2, 0, 1, 6, None, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_route_topk_backward(many, 6, 2, 0, 1, 6, None, 1, 1, 1, 1, None, 1, None) == -1
    assert L.dimo_group_rows(many, 6, 2, 1, 1, 1, 1, None, 1, 1 << 60, None) == -1
    for sizes in ((many, 3, 8, 5), (4, 3, many, 5), (4, 3, 8, many)):
        assert L.dimo_grouped_linear_forward(0, *sizes, 1, 1 << 40, None, 1, 1, None, 0, 1, None, None) == -1
        assert L.dimo_grouped_linear_dgrad(0, *sizes, 1, 1, 1, 0, None, 1, None) == -1
        assert L.dimo_grouped_linear_wgrad(0, *sizes, 1, 1, 1 << 40, None, 1, 1, None, 1, 1 << 60, None) == -1
        assert L.dimo_grouped_linear_wgrad_workspace_bytes(0, *sizes) == 0
    assert L.dimo_combine_rows_forward(many, 1, 8, 8, 0, 1, 8, None, 1, None, 0, 1, None) == -1
    assert L.dimo_combine_rows_backward(many, 1, 8, many, 3, 0, 1, 8, 1, 8, 1, 1, 1, 1, 1, None) == -1


def test_c_entry_points_refuse():
    """The C ABI returns an error for what its header does not allow, before it launches anything."""
    L = expert_emulation.emulated_library()
    assert L.dimo_route_topk_forward(4, 6, 7, 0, 1, 6, None, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_route_topk_forward(4, 6, 2, 3, 1, 6, None, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_route_topk_forward(4, 6, 2, 0, 1, 5, None, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_route_topk_forward(4096, 6, 2, 0, 1, 6, None, 1, 1, 1, 1, None, 0, None) == -3
    assert L.dimo_route_topk_forward(4, 6, 2, 0, None, 6, None, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_group_rows(10000, 6, 2, 1, 1, 1, 1, None, None, 0, None) == -3
    assert L.dimo_group_rows(-1, 6, 2, 1, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_group_rows(4, 6, 0, 1, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_group_rows(4, 1025, 1, 1, 1, 1, 1, None, None, 0, None) == -1
    assert L.dimo_grouped_linear_forward(0, 4, 3, 8, 5, 1, 7, None, 1, 1, None, 0, 1, None, None) == -1
    assert L.dimo_grouped_linear_forward(0, 4, 3, 8, 5, 1, 8, None, 1, 1, None, 3, 1, None, None) == -1
    assert L.dimo_grouped_linear_dgrad(0, 4, 0, 8, 5, 1, 1, 1, 0, None, 1, None) == -1
    assert L.dimo_grouped_linear_dgrad(0, 4, 3, 8, 5, 1, 1, 1, 1, None, 1, None) == -1
    assert L.dimo_grouped_linear_wgrad(0, 4, 3, 8, 5, 1, 1, 8, None, None, 1, None, None, 0, None) == -1
    assert L.dimo_grouped_linear_wgrad(1, 4096, 2, 64, 64, 1, 1, 64, None, 1, 1, None, None, 0, None) == -3
    assert L.dimo_activation_backward(0, 0, 8, 1, 1, 1, None) == -1
    assert L.dimo_combine_rows_forward(4, 2, 8, 8, 0, 1, 7, None, 1, None, 0, 1, None) == -1
    assert L.dimo_combine_rows_backward(4, 2, 8, 9, 3, 0, 1, 8, 1, 8, 1, 1, 1, 1, 1, None) == -1
    assert L.dimo_route_topk_forward(0, 6, 2, 0, None, 6, None, 1, None, None, None, None, 0, None) == 0


def test_timenet_with_experts(emulated):
    cases.check_timenet_with_experts("cpu", 32, 2, 9, 4, 2)


def test_quantized_block(emulated, monkeypatch):
    from dimo_amd import mx4
    expert_emulation.use(monkeypatch, mx4)
    cases.check_quantized_block(ex, mx4, "cpu", 40, 64, 4, 2)


def test_timenet_keeps_its_state_dict_without_experts():
    from dimo_amd.deform import TimeNet
    assert not [k for k in TimeNet(D=2, W=8).state_dict() if "experts" in k]
    assert [k for k in TimeNet(D=2, W=8, experts=2, top_k=1).state_dict() if "experts" in k]


def test_fused_timenet_refuses_experts():
    from dimo_amd.batched_render import timenet_fusable
    from dimo_amd.deform import TimeNet
    net = TimeNet(D=2, W=8, skips=(), experts=2, top_k=1)

    class OnGpu:
        is_cuda, dtype = True, F32
    assert not timenet_fusable(net, OnGpu)
    net.experts = None
    assert timenet_fusable(net, OnGpu)
