"""Bounds that the documentation of the expert operators states, shared by the CPU-emulated and the GPU tests."""
import torch


def check_4bit_error(mx4, device, dtype, seed=0):
    """quantize_mx4's error per element against its block's scale s: s / 4, s / 2, s by the steps of e2m1, |x| - 6 s beyond; at
    most a quarter of the block's largest magnitude; and the bounds are reached."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(400, 96, generator=g) * torch.exp2(torch.randint(-8, 9, (400, 1), generator=g).float())).to(dtype)
    x[0, :6] = torch.tensor([7.875, 0.24, 5.0, 2.5, 1.25, 0.74]).to(dtype)
    x[0, 6:32] = 0
    q = mx4.quantize_mx4(x.to(device))
    got, v = q.dequantize().cpu().double().view(400, 3, 32), x.double().view(400, 3, 32)
    s = torch.exp2(q.scales.cpu().double() - 127)[..., None]
    a, error = v.abs() / s, (got - v).abs() / s
    bound = torch.where(a <= 2, 0.25, torch.where(a <= 4, 0.5, torch.where(a <= 6, 1.0, a - 6)))
    assert bool((error <= bound).all()) and float(error.max()) <= 2
    assert bool((error * s <= 0.25 * v.abs().amax(-1, keepdim=True)).all())
    assert got[0, 0, 1] == 0 and error[0, 0, 0] == a[0, 0, 0] - 6 and error[0, 0, 2] == 1  # all of an element; saturation; a tie


def check_fp32_products(ex, device, rows, scale, seed=0):
    """Single fp32 products: 2^-22 of the three products of pieces that are left out, and the roundings of the sum of the other
    six, smallest first -- one of the whole, at most a step (2^-23) should the hardware cut, and those of what lies 2^-7 below --:
    6.1 x 2^-24.  Operands below 2^-110: 2^-134 of the other one besides."""
    g = torch.Generator().manual_seed(seed)
    x = (1 + torch.rand(rows, generator=g) * (0.02 if seed else 1)) * scale * torch.where(torch.rand(rows, generator=g) < 0.5, -1, 1)
    w = 1 + torch.rand(64, generator=g) * (0.02 if seed else 1)
    groups = ex.RowGroups(torch.tensor([0, rows], dtype=torch.int32, device=device))
    y = ex.grouped_linear(x[:, None].to(device), w[None, :, None].to(device), groups).cpu().double()
    ref = x.double()[:, None] * w.double()[None]
    slack = 2.0 ** -134 * w.double() if scale < 2.0 ** -110 else 0.0
    assert bool(((y - ref).abs() <= 6.1 * 2.0 ** -24 * ref.abs() + slack).all())


def check_infinite_operands(ex, device, rows):
    """An infinite fp32 operand: NaN in its row of outputs, nowhere else."""
    x = torch.randn(rows, 8, generator=torch.Generator().manual_seed(0))
    x[1, 3] = float("inf")
    groups = ex.RowGroups(torch.tensor([0, rows], dtype=torch.int32, device=device))
    y = ex.grouped_linear(x.to(device), torch.ones(1, 5, 8, device=device), groups).cpu()
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2:]).all())
