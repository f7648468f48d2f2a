"""The slope on the way out of a gradient of x (dimo_grouped_linear_dgrad with an activation), shared by the CPU-emulated and
the GPU tests."""
import math

import torch

from dimo_amd import _lib
from tests import expert_cases as cases


def check_slope_rounds_once(ex, device, counts, K, N, dtype, act, tail=0, seed=0):
    """gx = (g W) act'(saved), rounded once: against float64 within half a step and the sums' own error."""
    E, R = len(counts), sum(counts) + tail
    g = torch.Generator().manual_seed(seed)
    gy = torch.randn(R, N, generator=g).to(dtype)
    w = (torch.randn(E, N, K, generator=g) / math.sqrt(N)).to(dtype)
    saved = (torch.randn(R, K, generator=g) * 2).to(dtype)
    offsets = cases.make_offsets(counts, device)
    dev = [t.to(device) for t in (gy, w, saved)]
    gx = torch.full((R, K), math.nan, dtype=dtype, device=device)
    _lib.check(_lib.lib().dimo_grouped_linear_dgrad(ex._DTYPES[dtype], R, E, K, N, dev[0].data_ptr(), offsets.data_ptr(),
                                                    dev[1].data_ptr(), ex._ACTIVATIONS[act], dev[2].data_ptr(), gx.data_ptr(),
                                                    _lib.current_stream()), "dimo_grouped_linear_dgrad")
    s = saved.double()
    slope = (s > 0).double() if act == "relu" else torch.sigmoid(s) * (1 + s * (1 - torch.sigmoid(s)))
    ref, slack = torch.zeros(R, K).double(), torch.zeros(R, K).double()
    lo = 0
    for e, n in enumerate(counts):
        r = slice(lo, lo + n)
        lo += n
        sums = gy[r].double() @ w[e].double()
        ref[r] = sums * slope[r]
        # the sums' own error times a slope of at most 1.1, and the slope's: its exponential's argument (|s| <= 16) is off by
        # 2^-24 of it, its half a dozen operations by one rounding each of terms up to 1 + |s|
        slack[r] = (1.1 * cases.product_slack(N, gy[r].double().abs() @ w[e].double().abs())
                    + 8 * 2.0 ** -24 * (1 + s[r].abs()) * sums.abs())
    cases.near(gx, ref, dtype, slack, "g_x")
