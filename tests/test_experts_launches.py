"""What the expert entry points launch for sizes at the ends of their documented range, on the CPU: a launch takes fewer than
2^32 threads, so larger work goes in several.  No kernel runs: the emulation notes the launches (simt_dry_run)."""
import ctypes as C

import pytest

from tests import expert_emulation

MOST = 1 << 30
P = 1 << 20  # an address on every boundary the entry points ask for; nothing is read from it


@pytest.fixture
def launched():
    L = expert_emulation.emulated_library()
    L.simt_launched.argtypes = [C.POINTER(C.c_uint64), C.c_int]

    def call(name, *args):
        L.simt_dry_run(1)
        try:
            rc = getattr(L, name)(*args)
            threads = (C.c_uint64 * 4096)()
            n = L.simt_launched(threads, 4096)
        finally:
            L.simt_dry_run(0)
        return rc, list(threads[:n])
    return call


def _whole(result, least):
    rc, threads = result
    assert rc == 0 and threads and max(threads) < 1 << 32
    assert sum(threads) >= least


@pytest.mark.parametrize("T", [(1 << 26) - 4, 1 << 26, (1 << 27) + 5, MOST])
def test_sum_backward(launched, T):
    _whole(launched("dimo_combine_rows_backward", T, 1, 8, T, 3, 1, P, 8, P, 8, P, P, P, P, P, None), 64 * T)
    _whole(launched("dimo_combine_rows_forward", T, 1, 8, T, 1, P, 8, P, P, None, 0, P, None), T)


@pytest.mark.parametrize("T", [(1 << 26) - 4, 1 << 26, MOST])
@pytest.mark.parametrize("E", [4, 513, 1024])
def test_routing(launched, T, E):
    lanes = 1 if E == 4 else 64
    _whole(launched("dimo_route_topk_backward", T, E, 2, 1, P, E, None, 1, P, P, P, None, P, None), lanes * T)
    rc, threads = launched("dimo_route_topk_forward", T, E, 2, 1, P, E, None, 1, P, P, None, None, 0, None)
    assert rc == 0 and len(threads) == 1 and threads[0] < 1 << 32  # (goes over its rows in rounds)
    rc, threads = launched("dimo_route_topk_forward", T, E, 2, 1, P, E, None, 1, P, P, P, P, 1 << 40, None)
    assert rc == 0 and max(threads) < 1 << 32


@pytest.mark.parametrize("n", [(1 << 32) - 257, (1 << 32) + 1, (1 << 35) + 8, (1 << 38) + 1])
def test_activation_backward(launched, n):
    _whole(launched("dimo_activation_backward", 1, 2, n, P, P, P, None), n // 8 if n % 8 == 0 else n)


@pytest.mark.parametrize("R,K,N", [(MOST, 1, 1), (MOST - 3, 8, 40), (1 << 24, 64, 8192), (5, 1, MOST), (200, 8, MOST)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_products(launched, R, K, N, dtype):
    tiles = lambda rows, columns: rows * columns // 65536  # (the largest tile's outputs)
    _whole(launched("dimo_grouped_linear_forward", dtype, R, 2, K, N, P, K, None, P, P, None, 0, P, None, None), 64 * tiles(R, N))
    _whole(launched("dimo_grouped_linear_dgrad", dtype, R, 2, N, K, P, P, P, 0, None, P, None), 64 * tiles(R, N))
    _whole(launched("dimo_grouped_linear_wgrad", dtype, R, 2, K, N, P, P, K, None, P, P, P, P, 1 << 60, None), 64)


@pytest.mark.parametrize("R,K,N", [(MOST, 32, 1), (1 << 24, 64, 8192), (5, 32, MOST), (1 << 22, 512, 1 << 16)])
def test_4bit_products(launched, R, K, N):
    _whole(launched("dimo_mx4_linear", 1, R, 2, K, N, P, P, P, P, P, None, 0, P, None), 64 * (R * N // 65536))


@pytest.mark.parametrize("S,E,launches", [(8192, 1024, 1), (8193, 1024, 2), (256 * 4096, 128, 2), (257 * 4096, 2, 3), (41 * 4096, 1000, 3),
                                          (MOST, 1024, 3)])
def test_grouping(launched, S, E, launches):
    """One launch, two, or (where every workgroup summing all workgroups' counts would be quadratic in the places) three."""
    need = expert_emulation.emulated_library().dimo_group_rows_workspace_bytes(S, E)
    rc, threads = launched("dimo_group_rows", S, E, 2, P, P, P, P, P, P, need, None)
    assert rc == 0 and max(threads) < 1 << 32 and len(threads) == launches
    assert need >= (0 if launches == 1 else (-(-S // 4096) + launches - 2) * (E + 1) * 4)
