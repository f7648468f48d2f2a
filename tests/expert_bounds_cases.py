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
