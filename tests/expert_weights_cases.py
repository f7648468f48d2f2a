"""Checks of the expert block's weights over the chosen (normalised) and over all experts, shared by the CPU-emulated and the
GPU tests: every check takes the device its tensors live on."""
import math

import torch

from tests import expert_cases as cases


def check_block_with_one_choice(ex, device, T=90, W=24, E=5, seed=0):
    """ExpertMLP(k=1) in fp32 against float64 autograd of h + p_e (w2 relu(w1 h + b1) + b2), p the softmax over all experts:
    output, input gradient and every parameter's, the router's among them and not zero."""
    torch.manual_seed(seed)
    block = ex.ExpertMLP(W, E, 1)
    with torch.no_grad():
        for p in (block.b1, block.w2, block.b2):
            p.copy_(0.3 * torch.randn(p.shape))
    h, go = torch.randn(T, W), torch.randn(T, W)
    ref = {n: p.detach().double().requires_grad_(True) for n, p in block.named_parameters()}
    h64 = h.double().requires_grad_(True)
    w, e, _ = cases.route_reference(h64 @ ref["router.weight"].T, 1, None, normalize=False)
    i = e[:, 0].long()
    pre = torch.einsum("tfk,tk->tf", ref["w1"][i], h64) + ref["b1"][i]
    out64 = h64 + w * (torch.einsum("tkf,tf->tk", ref["w2"][i], pre.clamp_min(0)) + ref["b2"][i])
    # (a hidden value within its own error of relu's kink may have either slope: such rows' gradients are left out)
    keep = (pre.detach().abs().amin(1) > (W + 32) * 2.0 ** -24 * 8)[:, None]
    names = list(ref)
    g64 = torch.autograd.grad(out64, [h64] + [ref[n] for n in names], (go * keep).double())
    block = block.to(device)
    hd = h.to(device).requires_grad_(True)
    out = block(hd)
    params = dict(block.named_parameters())
    grads = torch.autograd.grad(out, [hd] + [params[n] for n in names], (go * keep).to(device))
    # as in expert_cases.check_layer: three products of W or T unit-variance terms after one another, each within
    # (n + 32) 2^-24 of its terms' sizes, which are sqrt(n) times the sum's
    tol = 4 * (max(W, T) + 32) * math.sqrt(max(W, T)) * 2.0 ** -24
    for name, got, want in zip(["out", "h"] + names, (out,) + grads, (out64.detach(),) + g64):
        assert float((got.detach().double().cpu() - want).abs().max()) <= tol * max(1.0, float(want.abs().max())), name
    assert float(dict(zip(names, grads[1:]))["router.weight"].abs().max()) > 1e-3


def check_weights_over_all(ex, device, T, K, F, E, k, dtype, seed=0):
    """expert_mlp(normalize=False) gives what its operators give one by one, masked rows among them."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g)).to(dtype).to(device).requires_grad_(True)
    x, z, w1, w2 = r(T, K), r(T, E), r(E, F, K, scale=K ** -0.5), r(E, K, F, scale=F ** -0.5)
    b1, b2 = r(E, F), r(E, K)
    mask = (torch.rand(T, generator=g) > 0.25).to(device)
    go = torch.randn(T, K, generator=g).to(dtype).to(device)
    leaves = (x, z, w1, b1, w2, b2)
    one = ex.expert_mlp(*leaves, k, "relu", mask, normalize=False)
    with torch.no_grad():
        assert torch.equal(ex.expert_mlp(*leaves, k, "relu", mask, normalize=False), one)
    g_one = torch.autograd.grad(one, leaves, go)
    weights, experts, _ = ex.route_topk(z, k, mask, normalize=False)
    groups = ex.group_rows(experts, E)
    h = ex.grouped_linear(x, w1, groups, b1, "relu", gather=True)
    two = ex.combine_rows(ex.grouped_linear(h, w2, groups, b2), groups, weights, residual=x)
    assert torch.equal(one, two)
    # relu's slope is 0 or 1: its multiplication rounds nothing in either form
    for a, b in zip(g_one, torch.autograd.grad(two, leaves, go)):
        if a is not g_one[0]:
            assert torch.equal(a, b)
    # (x: the block adds the residual's gradient to the places' sum before it rounds, the parts round both and their sum)
    b = torch.autograd.grad(ex.combine_rows(ex.grouped_linear(ex.grouped_linear(x, w1, groups, b1, "relu", gather=True), w2, groups, b2),
                                            groups, weights.detach(), residual=x), x, go)[0]
    size = g_one[0].double().abs() + b.double().abs() + 2 * go.double().abs()
    assert bool(((g_one[0].double() - b.double()).abs() <= 3 * cases.HALF_STEP[dtype] * size).all())


def check_quantized_block_with_one_choice(ex, mx4, device, T=70, W=64, E=4, seed=0):
    """ExpertMLP(k=1).quantized() weighs as its block does."""
    torch.manual_seed(seed)
    block = ex.ExpertMLP(W, E, 1, device=device)
    with torch.no_grad():
        block.w2.copy_(torch.randn(block.w2.shape) / math.sqrt(W))
        h = torch.randn(T, W).to(device)
        weights, experts, _ = ex.route_topk(block.router(h), 1, normalize=False)
        assert float(weights.max()) < 1
        groups = ex.group_rows(experts, E)
        y = mx4.mx4_linear(mx4.quantize_mx4(h, groups), mx4.quantize_mx4(block.w1), block.b1, groups, "relu", torch.float32)
        y = mx4.mx4_linear(mx4.quantize_mx4(y), mx4.quantize_mx4(block.w2), block.b2, groups, None, torch.float32)
        assert torch.equal(block.quantized()(h), ex.combine_rows(y, groups, weights, h))
