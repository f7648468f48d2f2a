"""Checks of the expert operators (dimo_amd/experts.py) against their definitions in float64, shared by the CPU-emulated
and the GPU tests: every check takes the device its tensors live on.

Tolerances are derived, element by element.  A sum of n products computed in fp32 is off by at most about n 2^-24 of the
sum of the products' absolute values; fp32 operands go through three bf16 pieces each, of whose products those below
2^-21 of the product are left out: n + 32 covers both.  Writing a result rounds it by at most half a step of its type."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}  # where steps stop shrinking


def near(got, ref, dtype, slack, what):
    """|got - ref| <= half a step of dtype + slack (fp32 arithmetic's share, a tensor or a number); NaN and inf equal."""
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), f"{what}: infinities differ"
    slack = slack.double().cpu().expand(ref.shape) if torch.is_tensor(slack) else torch.full(ref.shape, float(slack), dtype=torch.float64)
    tol = HALF_STEP[dtype] * (ref.abs() + slack) + slack + TINY[dtype]
    over = ((got - ref).abs() - tol)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max()):.3e} over the tolerance"


def product_slack(n, absolute):
    return (n + 32) * 2.0 ** -24 * absolute


# ---------------------------------------------------------------------------------------------------------- routing
def route_reference(z, k, mask=None, normalize=True):
    """(weights, experts, load) of logits z in float64 by the definition, differentiable (NaN-free logits)."""
    if mask is not None:
        z = z.masked_fill(~mask[:, None], -math.inf)
    T, E = z.shape
    order = torch.sort(z.detach(), dim=1, descending=True, stable=True)[1][:, :k]
    top = torch.gather(z, 1, order)
    live = top.detach() > -math.inf
    m = torch.where(live[:, :1], top.detach()[:, :1], torch.zeros(T, 1, dtype=z.dtype))
    p = torch.exp(z - m)
    total = p.sum(1, keepdim=True)
    p = torch.where(total > 0, p / torch.where(total > 0, total, 1.0), 0.0)
    w = torch.where(live, torch.gather(p, 1, order), 0.0)
    if normalize:
        s = w.sum(1, keepdim=True)
        w = torch.where(s > 0, w / torch.where(s > 0, s, 1.0), 0.0)
    return w, torch.where(live, order, -1).to(torch.int32), p.sum(0) / max(T, 1)


def make_logits(T, E, dtype, seed, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(T, E, generator=g) * 2
    if kind == "ties":
        z = torch.randint(-2, 3, (T, E), generator=g).float()
    if kind == "-inf":
        z[torch.rand(T, E, generator=g) < 0.6] = -math.inf
        z[0] = -math.inf
    if kind == "lowest":
        z[torch.rand(T, E, generator=g) < 0.6] = torch.finfo(dtype).min
        z[0] = torch.finfo(dtype).min
    return z.to(dtype)


def check_route(ex, device, T, E, k, dtype, normalize=True, masked=False, kind="normal", pad=0, seed=0):
    z = make_logits(T, E, dtype, seed, kind)
    g = torch.Generator().manual_seed(seed + 1)
    mask = torch.rand(T, generator=g) > 0.3 if masked else None
    gw, gl = torch.randn(T, k, generator=g), torch.randn(E, generator=g)
    z64 = z.double().requires_grad_(True)
    w, e, load = route_reference(z64, k, mask, normalize)
    wide = torch.full((T, E + pad), 7.0, dtype=dtype)
    wide[:, :E] = z
    zd = wide.to(device)[:, :E].detach().requires_grad_(True)
    md = None if mask is None else mask.to(device)
    weights, experts, got_load = ex.route_topk(zd, k, row_mask=md, normalize=normalize)
    assert experts.dtype == torch.int32 and torch.equal(experts.cpu(), e), "experts"
    # exp(z - m) with |z - m| <= 32 where it counts: 2^-24 of 32 from the argument, a few roundings, a sum over E
    rel = (64 + E) * 2.0 ** -24
    near(weights, w.detach(), torch.float32, rel * w.detach().abs(), "weights")
    near(got_load, load.detach(), torch.float32, rel * load.detach() + (T + 16) * 2.0 ** -24 * load.detach(), "load")
    plain = ex.route_topk(zd.detach(), k, row_mask=md, normalize=normalize)
    assert torch.equal(plain[0], weights) and torch.equal(plain[1], experts) and torch.equal(plain[2], got_load)
    if T == 0:
        return
    for with_w, with_l in ((True, True), (True, False), (False, True)):
        outs = [t for t, on in ((weights, with_w), (got_load, with_l)) if on]
        gs = [t.to(device) for t, on in ((gw, with_w), (gl, with_l)) if on]
        got = torch.autograd.grad(outs, zd, gs, retain_graph=True)[0]
        refs = [t for t, on in ((w, with_w), (load, with_l)) if on]
        ref = torch.autograd.grad(refs, z64, [t.double() for t, on in ((gw, with_w), (gl, with_l)) if on], retain_graph=True)[0]
        ref = torch.nan_to_num(ref, nan=0.0)  # (autograd of exp(-inf - m) is 0 * -inf; the formula's term is 0)
        scale = 4 * gw.abs().sum(1, keepdim=True).double() * with_w + 4 * float(gl.abs().max()) / T * with_l
        near(got, ref, dtype, rel * scale.expand_as(ref) if torch.is_tensor(scale) else rel * scale, f"g_logits {with_w} {with_l}")


def check_route_special(ex, device, dtype):
    """Rows with NaN or +inf: weights NaN, the choice goes by the other logits, nothing is out of range."""
    z = torch.tensor([[1.0, math.nan, 3.0, 2.0, 0.0], [math.inf, 1.0, 2.0, 3.0, 4.0], [0.0, 1.0, 2.0, 3.0, 4.0],
                      [math.nan] * 5, [-math.inf, 5.0, -math.inf, -math.inf, -math.inf]]).to(dtype).to(device)
    w, e, load = ex.route_topk(z, 2)
    assert e.cpu().tolist() == [[2, 3], [0, 4], [4, 3], [-1, -1], [1, -1]]
    w = w.cpu()
    assert torch.isnan(w[0]).all() and torch.isnan(w[1]).any() and w[4].tolist() == [1.0, 0.0] and w[3].tolist() == [0.0, 0.0]
    assert torch.isfinite(w[2]).all() and torch.isnan(load.cpu()).any()
    keep = torch.tensor([False, False, True, False, True], device=device)  # masked rows: whatever they hold counts as nothing
    w, e, load = ex.route_topk(z, 2, row_mask=keep)
    assert e.cpu().tolist() == [[-1, -1], [-1, -1], [4, 3], [-1, -1], [1, -1]]
    assert torch.isfinite(w).all() and torch.isfinite(load).all() and float(w[0].abs().sum()) == 0
    zg = z.clone().requires_grad_(True)
    w, _, load = ex.route_topk(zg, 2, row_mask=keep)
    g = torch.autograd.grad((w, load), zg, (torch.ones_like(w), torch.ones_like(load)))[0].cpu()
    assert torch.isfinite(g).all() and float(g[~keep.cpu()].abs().sum()) == 0


# --------------------------------------------------------------------------------------------------------- grouping
def group_reference(experts, E):
    flat = experts.flatten().tolist()
    buckets = [[] for _ in range(E)]
    for i, e in enumerate(flat):
        if 0 <= e < E:
            buckets[e].append(i)
    order = [i for b in buckets for i in b]
    offsets = [0]
    for b in buckets:
        offsets.append(offsets[-1] + len(b))
    position = [-1] * len(flat)
    for r, i in enumerate(order):
        position[i] = r
    order += [-1] * (len(flat) - len(order))
    as_int = lambda v: torch.tensor(v, dtype=torch.int32)
    return as_int(offsets), as_int(order), as_int(position).view(experts.shape)


def check_group(ex, device, T, k, E, seed=0, skew=False, dropped=True):
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    if skew:
        e = torch.where(torch.rand(T, k, generator=g) < 0.9, min(E - 1, 2), e).to(torch.int32)
    if dropped and T:
        bad = torch.tensor([-1, E, E + 5, -7, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64).to(torch.int32)
        e = torch.where(torch.rand(T, k, generator=g) < 0.2, bad[torch.randint(0, 6, (T, k), generator=g)], e)
    offsets, order, position = group_reference(e, E)
    got = ex.group_rows(e.to(device), E)
    assert torch.equal(got.offsets.cpu(), offsets), "offsets"
    assert torch.equal(got.order.cpu(), order), "order"
    assert torch.equal(got.position.cpu(), position), "position"


# ----------------------------------------------------------------------------------------------------- the products
def activation64(z, act):
    return z.clamp_min(0) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z


def make_offsets(counts, device):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32).to(device)


def check_products(ex, device, counts, K, N, dtype, act=None, tail=0, pad=0, bias=True, seed=0, scale=1.0):
    """grouped_linear on rows in the order of the groups, forward and backward, against float64."""
    E, R = len(counts), sum(counts) + tail
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, K, generator=g) * scale).to(dtype)
    w = (torch.randn(E, N, K, generator=g) / math.sqrt(K)).to(dtype)
    b = torch.randn(E, N, generator=g).to(dtype) if bias else None
    gy = torch.randn(R, N, generator=g).to(dtype)
    wide = torch.full((R, K + pad), math.nan, dtype=dtype)  # (what lies between the rows must not be read into results)
    wide[:, :K] = x
    xd = wide.to(device)[:, :K].detach().requires_grad_(True)
    wd = w.to(device).requires_grad_(True)
    bd = b.to(device).requires_grad_(True) if bias else None
    groups = ex.RowGroups(make_offsets(counts, device))
    y = ex.grouped_linear(xd, wd, groups, bias=bd, activation=act)
    none = ex.grouped_linear(xd.detach(), wd.detach(), groups, bias=None if b is None else bd.detach(), activation=act)
    assert torch.equal(none, y.detach()), "with and without gradients"
    leaves = [xd, wd] + ([bd] if bias else [])
    grads = torch.autograd.grad(y, leaves, gy.to(device))
    X, W, G = x.double(), w.detach().double(), gy.double()
    Y, GX, GW, GB = torch.zeros(R, N).double(), torch.zeros(R, K).double(), torch.zeros(E, N, K).double(), torch.zeros(E, N).double()
    sY, sX, sW, sB = torch.zeros_like(Y), torch.zeros_like(GX), torch.zeros_like(GW), torch.zeros_like(GB)
    lo = 0
    for e, n in enumerate(counts):
        r = slice(lo, lo + n)
        lo += n
        z = X[r] @ W[e].T + (b[e].detach().double() if bias else 0)
        s = product_slack(K, X[r].abs() @ W[e].abs().T + (b[e].detach().double().abs() if bias else 0))
        Y[r], sY[r] = activation64(z, act), 1.1 * s + 8 * 2.0 ** -24 * z.abs()  # (|silu'| <= 1.1; its own roundings)
        gz, gs = G[r], torch.zeros_like(s)
        if act:
            # the slope is taken from what the forward kept in the inputs' type; relu: its output's sign, which may be
            # either within the sum's own error of zero -- those elements are compared with a gradient of both signs allowed
            d = (z > 0).double() if act == "relu" else torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))
            kept = HALF_STEP[dtype] * z.abs() + s
            ds = (z.abs() <= kept).double() if act == "relu" else 0.5 * kept + 8 * 2.0 ** -24 * (1 + z.abs())  # |silu''| <= 1/2
            gz = G[r] * d
            gs = G[r].abs() * ds + HALF_STEP[dtype] * gz.abs() * (1 + 0) + HALF_STEP[dtype] * G[r].abs() * ds + TINY[dtype]
        GX[r] = gz @ W[e]
        sX[r] = product_slack(N, gz.abs() @ W[e].abs()) + gs @ W[e].abs() * 1.01
        GW[e] = gz.T @ X[r]
        sW[e] = product_slack(n, gz.abs().T @ X[r].abs()) + gs.T @ X[r].abs() * 1.01
        GB[e] = gz.sum(0)
        sB[e] = product_slack(n, gz.abs().sum(0)) + gs.sum(0) * 1.01
    near(y, Y, dtype, sY, "y")
    near(grads[0], GX, dtype, sX, "g_x")
    near(grads[1], GW, dtype, sW, "g_w")
    if bias:
        near(grads[2], GB, dtype, sB, "g_b")
    if tail:
        assert float(y[R - tail:].detach().float().abs().sum()) == 0 and float(grads[0][R - tail:].float().abs().sum()) == 0


def check_gather(ex, device, T, k, E, K, N, dtype, seed=0, pad=0):
    """The products reading x through the grouping, places without an expert among them; x's gradient is the sum over
    a row's places."""
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32)
    x = torch.randn(T, K, generator=g).to(dtype)
    w = (torch.randn(E, N, K, generator=g) / math.sqrt(K)).to(dtype)
    wide = torch.full((T, K + pad), math.nan, dtype=dtype)
    wide[:, :K] = x
    xd, wd = wide.to(device)[:, :K].detach().requires_grad_(True), w.to(device).requires_grad_(True)
    groups = ex.group_rows(e.to(device), E)
    y = ex.grouped_linear(xd, wd, groups, gather=True)
    gy = torch.randn(T * k, N, generator=g).to(dtype)
    gx, gw = torch.autograd.grad(y, (xd, wd), gy.to(device))
    offsets, order, position = group_reference(e, E)
    X, W, G = x.double(), w.detach().double(), gy.double()
    Y, sY = torch.zeros(T * k, N).double(), torch.zeros(T * k, N).double()
    GX, sX = torch.zeros(T, K).double(), torch.zeros(T, K).double()
    GW, sW = torch.zeros(E, N, K).double(), torch.zeros(E, N, K).double()
    for r, place in enumerate(order.tolist()):
        if place < 0:
            continue
        t, q = place // k, int(e.flatten()[place])
        Y[r], sY[r] = W[q] @ X[t], product_slack(K, W[q].abs() @ X[t].abs())
        row = G[r] @ W[q]
        GX[t] += row
        sX[t] += product_slack(N, G[r].abs() @ W[q].abs()) + HALF_STEP[dtype] * row.abs() + TINY[dtype] + k * 2.0 ** -24 * row.abs()
        GW[q] += G[r][:, None] * X[t][None]
        sW[q] += (G[r].abs()[:, None] * X[t].abs()[None])
    near(y, Y, dtype, sY, "y")
    near(gx, GX, dtype, 1.01 * sX, "g_x")
    near(gw, GW, dtype, product_slack(T * k, sW), "g_w")


# ---------------------------------------------------------------------------------------------------- bringing together
def check_wanted(ex, device, wanted, seed=0):
    """A call that needs some of the gradients gets the ones (bit for bit) that it would get with all of them."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(device)
    z = r(60, 4)

    def some(fn, tensors, pick):
        leaves = [t.clone().requires_grad_(i in pick) for i, t in enumerate(tensors)]
        out = fn(*leaves)
        return torch.autograd.grad(out, [leaves[i] for i in pick], torch.ones_like(out))
    _, experts, _ = ex.route_topk(z, 2)
    groups = ex.group_rows(experts, 4)
    calls = [(lambda x, w, b: ex.grouped_linear(x, w, groups, b, "silu", gather=True), (r(60, 24), r(4, 16, 24), r(4, 16))),
             (lambda y, w, x: ex.combine_rows(y, groups, w, x), (r(120, 24), r(60, 2), r(60, 24))),
             (lambda x, w1, b2: ex.expert_mlp(x, z, w1, None, w1.mT.contiguous(), b2, 2), (r(60, 24), r(4, 16, 24), r(4, 24))),
             (lambda logits, b1, w2: ex.expert_mlp(z, logits, w2.mT.contiguous(), b1, w2, None, 2, None), (r(60, 3), r(3, 8), r(3, 4, 8)))]
    for fn, tensors in calls:
        every = some(fn, tensors, (0, 1, 2))
        for i, got in zip(wanted, some(fn, tensors, wanted)):
            assert torch.equal(got, every[i])


def check_combine(ex, device, T, k, E, N, dtype, weighted=True, residual=True, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32)
    groups = ex.group_rows(e.to(device), E)
    _, _, position = group_reference(e, E)
    y = torch.randn(T * k, N, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g) if weighted else None
    res = torch.randn(T, N, generator=g).to(dtype) if residual else None
    go = torch.randn(T, N, generator=g).to(dtype)
    wide = torch.full((T * k, N + pad), math.nan, dtype=dtype)
    wide[:, :N] = y
    yd = wide.to(device)[:, :N].detach().requires_grad_(True)
    leaves = [yd] + [t.to(device).requires_grad_(True) for t in (w, res) if t is not None]
    out = ex.combine_rows(yd, groups, leaves[1] if weighted else None, leaves[-1] if residual else None)
    grads = torch.autograd.grad(out, leaves, go.to(device))
    at = position.long().clamp_min(0)
    ys = y.detach().double()[at] * (position >= 0)[..., None]
    W = w.detach().double() if weighted else torch.ones(T, k).double()
    ref = (W[..., None] * ys).sum(1) + (res.detach().double() if residual else 0)
    mag = (W[..., None] * ys.abs()).sum(1) + (res.detach().double().abs() if residual else 0)
    near(out, ref, dtype, (k + 2) * 2.0 ** -24 * mag, "out")
    gy = torch.zeros(T * k, N).double()
    live = position >= 0
    gy[position[live].long()] = (W[..., None] * go.double()[:, None])[live]
    near(grads[0], gy, dtype, 2.0 ** -24 * gy.abs(), "g_y")
    if weighted:
        near(grads[1], (ys * go.double()[:, None]).sum(-1), torch.float32,
             (N + 8) * 2.0 ** -24 * (ys.abs() * go.double()[:, None].abs()).sum(-1), "g_weights")
    if residual:
        assert torch.equal(grads[-1].cpu(), go)


# ------------------------------------------------------------------------------------------------------ used together
def check_layer_is_its_parts(ex, device, T, K, F, E, k, dtype, act, biases=True, seed=0):
    """expert_mlp gives what its operators give one by one: the forward bit by bit, the gradients within one more rounding
    of the hidden gradient (the slope is applied behind its rounding in the one, in a pass of its own in the other)."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g)).to(dtype).to(device).requires_grad_(True)
    x, z, w1, w2 = r(T, K), r(T, E), r(E, F, K, scale=K ** -0.5), r(E, K, F, scale=F ** -0.5)
    b1, b2 = (r(E, F), r(E, K)) if biases else (None, None)
    mask = (torch.rand(T, generator=g) > 0.25).to(device)
    go = torch.randn(T, K, generator=g).to(dtype).to(device)
    leaves = [t for t in (x, z, w1, b1, w2, b2) if t is not None]
    one = ex.expert_mlp(x, z, w1, b1, w2, b2, k, act, mask)
    with torch.no_grad():
        assert torch.equal(ex.expert_mlp(x, z, w1, b1, w2, b2, k, act, mask), one)
    g_one = torch.autograd.grad(one, leaves, go)
    weights, experts, _ = ex.route_topk(z, k, mask)
    groups = ex.group_rows(experts, E)
    h = ex.grouped_linear(x, w1, groups, b1, act, gather=True)
    two = ex.combine_rows(ex.grouped_linear(h, w2, groups, b2), groups, weights, residual=x)
    g_two = torch.autograd.grad(two, leaves, go)
    assert torch.equal(one, two)
    for a, b in zip(g_one, g_two):
        assert a.shape == b.shape and a.dtype == b.dtype
        if b.numel():
            assert float((a - b).float().abs().max()) <= 8 * HALF_STEP[dtype] * max(float(b.float().abs().max()), 1e-6)
    some = torch.autograd.grad(ex.expert_mlp(x, z, w1, b1, w2, b2, k, act, mask), [z, w1], go)
    assert torch.equal(some[0], g_one[1]) and torch.equal(some[1], g_one[2])


def check_layer(ex, device, T, K, F, E, k, act, seed=0):
    """expert_mlp in fp32, masked rows among them: output and every gradient against float64 autograd, and the gradient
    against differences of the float64 form along a random direction."""
    g = torch.Generator().manual_seed(seed)
    names = ("x", "logits", "w1", "b1", "w2", "b2")
    leaf = [torch.randn(T, K, generator=g), torch.randn(T, E, generator=g), torch.randn(E, F, K, generator=g) / math.sqrt(K),
            0.3 * torch.randn(E, F, generator=g), torch.randn(E, K, F, generator=g) / math.sqrt(F), 0.3 * torch.randn(E, K, generator=g)]
    mask = torch.rand(T, generator=g) > 0.2
    go = torch.randn(T, K, generator=g)

    def reference(x, z, w1, b1, w2, b2):
        w, e, _ = route_reference(z, k, mask)
        out = x
        for j in range(k):
            i = e[:, j].long().clamp_min(0)
            h = activation64(torch.einsum("tfk,tk->tf", w1[i], x) + b1[i], act)
            out = out + (w[:, j] * (e[:, j] >= 0))[:, None] * (torch.einsum("tkf,tf->tk", w2[i], h) + b2[i])
        return out

    l64 = [t.double().requires_grad_(True) for t in leaf]
    out64 = reference(*l64)
    g64 = torch.autograd.grad(out64, l64, go.double())
    ld = [t.to(device).requires_grad_(True) for t in leaf]
    out = ex.expert_mlp(*ld, k=k, activation=act, row_mask=mask.to(device))
    grads = torch.autograd.grad(out, ld, go.to(device))
    # two products of K and F terms each way, each within (n + 32) 2^-24 of its terms' sizes: the terms of a sum of n
    # unit-variance products are sqrt(n) times larger than the sum, three such sums follow one another
    tol = 4 * (max(K, F, T) + 32) * math.sqrt(max(K, F)) * 2.0 ** -24
    for name, got, ref in zip(("out",) + names, (out,) + grads, (out64.detach(),) + g64):
        ref = torch.nan_to_num(ref, nan=0.0)
        assert float((got.detach().double().cpu() - ref).abs().max()) <= tol * max(1.0, float(ref.abs().max())), name
    step = 1e-6
    ways = [torch.randn(t.shape, generator=g).double() for t in leaf]
    ways[1] *= mask[:, None]
    with torch.no_grad():
        hi = reference(*[t.detach() + step * d for t, d in zip(l64, ways)])
        lo = reference(*[t.detach() - step * d for t, d in zip(l64, ways)])
    slope = float(((hi - lo) * go.double()).sum()) / (2 * step)
    along = sum(float((gr.double().cpu() * d).sum()) for gr, d in zip(grads, ways))
    size = sum(float((gr.double().cpu() * d).abs().sum()) for gr, d in zip(grads, ways))
    assert abs(along - slope) <= (tol + 1e-5) * size, (along, slope)


# ------------------------------------------------------------------------------------------- microscaled 4-bit values
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize_reference(x):
    """(codes [R, 32 B], scale bytes [R, B], values [R, K]) of x [R, K] in float64, one element at a time by distance."""
    x = x.double().cpu()
    R, K = x.shape
    B = -(-K // 32)
    v = torch.nn.functional.pad(x, (0, 32 * B - K)).view(R, B, 32)
    big = v.abs().amax(-1)
    finite = torch.isfinite(v).all(-1)
    byte = torch.full((R, B), 255, dtype=torch.int64)
    exponent = torch.frexp(torch.where(finite & (big > 0), big, 1.0))[1].long() - 1
    byte = torch.where(finite, torch.where(big > 0, (exponent - 2 + 127).clamp_min(0), 0), byte)
    scale = torch.ldexp(torch.ones(R, B, dtype=torch.float64), (byte - 127).int())
    a = torch.where(finite[..., None], v / scale[..., None], 0.0).abs().clamp_max(6.0)
    off = (a[..., None] - E2M1).abs()
    best = off.amin(-1, keepdim=True)
    tied = off == best
    even = tied & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.to(torch.uint8).argmax(-1), tied.to(torch.uint8).argmax(-1))
    sign = torch.signbit(v).long()
    values = torch.where(finite[..., None], E2M1[code] * torch.where(sign > 0, -1.0, 1.0) * scale[..., None], math.nan)
    return code | (sign << 3), byte, values.reshape(R, -1)[:, :K], finite


def unpacked(codes):
    codes = codes.cpu().long()
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def quantize_inputs(R, K, dtype, seed, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp(2 * torch.randn(1, K, generator=g))
    if kind == "borders":  # every value on or next to a rounding border, the block's largest 4
        borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0, -0.0, 4.0])
        x = borders[torch.randint(0, 12, (R, K), generator=g)] * torch.where(torch.rand(R, K, generator=g) < 0.5, -1.0, 1.0)
        x = x * torch.exp2(torch.randint(-6, 7, (R, 1), generator=g).float())
        if dtype == torch.float32:
            x = x * (1 + (torch.randint(-1, 2, (R, K), generator=g)).float() * 2.0 ** -23)
    if kind == "range":  # from the smallest magnitudes to the largest of the type
        top = {torch.float32: 127, torch.bfloat16: 127, torch.float16: 15}[dtype]
        low = {torch.float32: -149, torch.bfloat16: -133, torch.float16: -24}[dtype]
        x = torch.ldexp(1 + torch.rand(R, K, generator=g) * 0.99, torch.randint(low, top + 1, (R, 1), generator=g).int())
        x[0] = 0
    if kind == "special":
        x[0, 0], x[1, K // 2], x[2, K - 1] = math.inf, -math.inf, math.nan
    return x.to(dtype)


def check_quantize(mx4, device, R, K, dtype, kind="normal", pad=0, seed=0):
    x = quantize_inputs(R, K, dtype, seed, kind)
    code, byte, values, finite = quantize_reference(x)
    wide = torch.full((R, K + pad), math.nan, dtype=dtype)
    wide[:, :K] = x
    q = mx4.quantize_mx4(wide.to(device)[:, :K])
    assert tuple(q.shape) == (R, K)
    assert torch.equal(q.scales.cpu().long(), byte), "scales"
    got = unpacked(q.codes).view(R, -1, 32)
    assert torch.equal(got[finite], code[finite]), "codes"
    for out in (torch.float32, torch.bfloat16, torch.float16):
        d = q.dequantize(out).cpu()
        assert d.dtype == out and torch.equal(torch.isnan(d), torch.isnan(values))
        ref = values.to(torch.float32).to(out)
        assert torch.equal(torch.nan_to_num(d, nan=0.0, posinf=1.0, neginf=-1.0), torch.nan_to_num(ref, nan=0.0, posinf=1.0, neginf=-1.0)), out


def check_mx4_linear(mx4, ex, device, counts, K, N, dtype, act=None, bias=True, tail=0, grouped=True, seed=0):
    E, R = len(counts), sum(counts) + tail
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp(torch.randn(1, K, generator=g))
    w = torch.randn(E, N, K, generator=g) / math.sqrt(K)
    b = torch.randn(E, N, generator=g).to(dtype) if bias else None
    xq, wq = mx4.quantize_mx4(x.to(device)), mx4.quantize_mx4(w.to(device))
    assert tuple(wq.shape) == (E, N, K)
    X = quantize_reference(x)[2]
    W = quantize_reference(w.view(E * N, K))[2].view(E, N, K)
    if grouped:
        groups = ex.RowGroups(make_offsets(counts, device))
        y = mx4.mx4_linear(xq, wq, None if b is None else b.to(device), groups, act, dtype)
    else:
        y = mx4.mx4_linear(xq, mx4.MX4(wq.codes[0], wq.scales[0], K), None if b is None else b[0].to(device), None, act, dtype)
    Y, s = torch.zeros(R, N).double(), torch.zeros(R, N).double()
    lo = 0
    for e, n in enumerate(counts):
        r = slice(lo, lo + n)
        lo += n
        z = X[r] @ W[e].T + (b[e].double() if bias else 0)
        Y[r] = activation64(z, act)
        s[r] = 1.1 * product_slack(K, X[r].abs() @ W[e].abs().T + (b[e].double().abs() if bias else 0)) + 8 * 2.0 ** -24 * z.abs()
    near(y, Y, dtype, s, "y")
    if tail:
        assert float(y[R - tail:].float().abs().sum()) == 0


def check_mx4_layer(mx4, ex, device, T, k, E, K, F, seed=0):
    """Routing, grouping, quantisation through the grouping, two grouped 4-bit products, the weighted sum: as they are
    used together, places without an expert among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g)
    z = torch.randn(T, E, generator=g)
    mask = torch.rand(T, generator=g) > 0.3
    w1, w2 = torch.randn(E, F, K, generator=g) / math.sqrt(K), torch.randn(E, K, F, generator=g) / math.sqrt(F)
    w, e, _ = ex.route_topk(z.to(device), k, row_mask=mask.to(device))
    groups = ex.group_rows(e, E)
    xq = mx4.quantize_mx4(x.to(device), groups)
    assert tuple(xq.shape) == (T * k, K)
    h = mx4.mx4_linear(xq, mx4.quantize_mx4(w1.to(device)), None, groups, "relu", torch.float32)
    y = mx4.mx4_linear(mx4.quantize_mx4(h), mx4.quantize_mx4(w2.to(device)), None, groups, None, torch.float32)
    out = ex.combine_rows(y, groups, w, x.to(device)).cpu().double()
    W, C, _ = route_reference(z.double(), k, mask)
    X = quantize_reference(x)[2]
    W1 = quantize_reference(w1.view(E * F, K))[2].view(E, F, K)
    W2 = quantize_reference(w2.view(E * K, F))[2].view(E, K, F)
    H = h.cpu().double()
    order = groups.order.cpu().tolist()
    ref, slack = x.double().clone(), torch.zeros(T, K).double()
    for r, place in enumerate(order):
        if place < 0:
            assert float(H[r].abs().sum()) == 0 and float(xq.dequantize().cpu()[r].abs().sum()) == 0
            continue
        t, q = place // k, int(C.flatten()[place])
        hr = (W1[q] @ X[t]).clamp_min(0)
        assert float((H[r] - hr).abs().max()) <= float((product_slack(K, W1[q].abs() @ X[t].abs()) + 2.0 ** -23 * hr).max())
        hq = quantize_reference(h[r:r + 1].cpu())[2][0]  # (a hidden value next to a border may round either way: the kernel's own)
        ref[t] += W[t, place % k] * (W2[q] @ hq)
        slack[t] += W[t, place % k] * product_slack(F, W2[q].abs() @ hq.abs()) * 2 + 2.0 ** -20 * (W2[q] @ hq).abs() * W[t, place % k]
    near(out, ref, torch.float32, slack + 2.0 ** -22 * ref.abs(), "out")


def expert_block_reference(block, h):
    """ExpertMLP in float64 on the CPU: h + the weighted experts' rows."""
    w, e, _ = route_reference(h @ block["router.weight"].T, block["k"])
    out = h
    for j in range(block["k"]):
        i = e[:, j].long().clamp_min(0)
        a = activation64(torch.einsum("tfk,tk->tf", block["w1"][i], h) + block["b1"][i], block["activation"])
        out = out + w[:, j:j + 1] * (torch.einsum("tkf,tf->tk", block["w2"][i], a) + block["b2"][i])
    return out


def check_timenet_with_experts(device, W, P, M, E, k, seed=0):
    """deform.TimeNet(experts=E) against its own module in float64 with the block spelled out: outputs and the gradients
    of every parameter.  silu instead of relu inside the block and no relu kinks from it; the rows whose hidden relu
    inputs lie next to zero are left out of the comparison, as in tests/test_gpu_timenet.py."""
    import copy

    from dimo_amd.deform import TimeNet
    torch.manual_seed(seed)
    net = TimeNet(D=3, W=W, skips=(1,), latent_code_dim=8, experts=E, top_k=k)
    net.experts.activation = "silu"
    g = torch.Generator().manual_seed(seed + 1)
    with torch.no_grad():
        for p in (net.experts.w2, net.experts.b1, net.experts.b2):
            p.copy_(torch.randn(p.shape, generator=g) * 0.1)
        for lin in (net.pts_layers[2], net.rot_layers[2]):
            lin.weight.copy_(0.1 * torch.randn(lin.weight.shape, generator=g))
    n64 = copy.deepcopy(net).double()
    block = dict(n64.experts.named_parameters(), k=k, activation="silu")
    n64.experts.forward = lambda h: expert_block_reference(block, h.reshape(-1, W)).view(h.shape)
    pts, t = torch.rand(M, 3, generator=g) - 0.5, torch.rand(P, 1, 1, generator=g).expand(P, M, 1)
    lat = torch.randn(P, 1, 8, generator=g).expand(P, M, 8)
    gx, gr = torch.randn(P, M, 3, generator=g), torch.randn(P, M, 4, generator=g)
    small = []
    hooks = [lin.register_forward_hook(lambda _m, _i, out: small.append(out.detach().abs().amin(-1)))
             for lin in list(n64.deformnet) + [n64.pts_layers[0], n64.rot_layers[0]]]
    dx64, dr64 = n64(pts[None].double(), t.double(), lat.double(), t_apply=True)
    for h in hooks:
        h.remove()
    keep = (torch.stack(small).amin(0) > 2e-5)[..., None]
    gx, gr = gx * keep, gr * keep
    ((dx64 * gx.double()).sum() + (dr64 * gr.double()).sum()).backward()
    net = net.to(device)
    dx, dr = net(pts[None].to(device), t.to(device), lat.to(device), t_apply=True)
    ((dx * gx.to(device)).sum() + (dr * gr.to(device)).sum()).backward()
    assert torch.allclose(dx.detach().cpu().double(), dx64.detach(), rtol=0, atol=1e-4 * float(dx64.abs().max()))
    assert torch.allclose(dr.detach().cpu().double(), dr64.detach(), rtol=0, atol=1e-4 * float(dr64.abs().max()))
    ref = dict(n64.named_parameters())
    for name, p in net.named_parameters():
        r = ref[name].grad
        assert torch.allclose(p.grad.cpu().double(), r, rtol=0, atol=1e-4 * max(float(r.abs().max()), 1e-6)), name


def check_quantized_block(ex, mx4, device, T, W, E, k, seed=0):
    """ExpertMLP.quantized(): what its own 4-bit operators give, and near the block it was made from (each product's
    operands rounded by at most 2^-2 relative: the block's contribution stays within half of its size)."""
    torch.manual_seed(seed)
    block = ex.ExpertMLP(W, E, k, device=device)
    with torch.no_grad():
        block.w2.copy_(torch.randn(block.w2.shape) / math.sqrt(W))
    h = torch.randn(T, W).to(device)
    with torch.no_grad():
        full, q = block(h), block.quantized()
        out = q(h)
        weights, experts, _ = ex.route_topk(block.router(h), k)
        groups = ex.group_rows(experts, E)
        y = mx4.mx4_linear(mx4.quantize_mx4(h, groups), mx4.quantize_mx4(block.w1), block.b1, groups, "relu", torch.float32)
        y = mx4.mx4_linear(mx4.quantize_mx4(y), mx4.quantize_mx4(block.w2), block.b2, groups, None, torch.float32)
        assert torch.equal(out, ex.combine_rows(y, groups, weights, h))
    assert not list(q.parameters())
    assert float((out - full).norm()) <= 0.5 * float((full - h).norm())
