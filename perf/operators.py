"""The expert operators as they are measured: routing rows to experts, the products grouped by expert, microscaled 4-bit
quantisation and the 4-bit products -- each in a plain form (elementary torch operations in 32 bits) and through the
package's own entry points (`own`).

Rows are what the deformation network works on: one per (motion, frame) pair and control point (8 pairs x 512 points in
a training step of the benchmark's size, up to 256 pairs in one call), widths 256 (its hidden layers) and 360 (the skip
layer's input); the wider cases are generic sizes of the same operators.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one row of a served network: latency alone
        {"name": "route one row", "op": "route", "T": 1, "E": 64, "k": 8, "type": "f32", "train": False, "masked": False},
        # the benchmark step's 8 pairs x 512 control points, forward and backward
        {"name": "route a step", "op": "route", "T": 4096, "E": 8, "k": 2, "type": "f32", "train": True, "masked": False},
        # the largest call of the deformation network (256 pairs x 512 points), many experts, some rows padding
        {"name": "route many rows", "op": "route", "T": 131072, "E": 128, "k": 8, "type": "bf16", "train": True, "masked": True},
        # one expert block at the deformation network's width, a training step in its type
        {"name": "layer f32 step", "op": "layer", "T": 4096, "K": 256, "F": 256, "E": 8, "k": 2, "type": "f32", "act": "silu", "train": True},
        # one row through a wide block: what is read is the chosen experts' weights
        {"name": "layer one row", "op": "layer", "T": 1, "K": 2048, "F": 2048, "E": 16, "k": 2, "type": "bf16", "act": "relu", "train": False},
        # a wide block's training step
        {"name": "layer wide step", "op": "layer", "T": 16384, "K": 1024, "F": 4096, "E": 16, "k": 2, "type": "bf16", "act": "relu", "train": True},
        # odd sizes, skewed and empty groups, rows of a wider tensor; 360 = the skip layer's input
        {"name": "products ragged", "op": "products", "R": 5003, "K": 360, "N": 257, "E": 13, "type": "f16", "train": True},
        # large ordinary products, forward
        {"name": "products large", "op": "products", "R": 65536, "K": 2048, "N": 2048, "E": 32, "type": "bf16", "train": False},
        # activations of the largest call
        {"name": "quantise large", "op": "quantise", "R": 131072, "K": 1024, "type": "bf16"},
        # an odd matrix whose rows end inside a block
        {"name": "quantise odd", "op": "quantise", "R": 1001, "K": 1000, "type": "f32"},
        # eight rows to eight experts' 4-bit weights: reading the weights
        {"name": "mx4 eight rows", "op": "mx4", "R": 8, "K": 2048, "N": 2048, "E": 8, "type": "bf16"},
        # large 4-bit products
        {"name": "mx4 large", "op": "mx4", "R": 32768, "K": 4096, "N": 4096, "E": 8, "type": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("route", "layer", "layer", "products", "products", "quantise", "mx4"))
    kind = rng.choice(("f32", "bf16", "f16"))
    if op == "route":
        E = _spread(rng, 2, 256)
        return {"op": op, "T": _spread(rng, 1, 65536), "E": E, "k": rng.randint(1, min(8, E)), "type": kind,
                "train": rng.random() < 0.7, "masked": rng.random() < 0.5}
    if op == "layer":
        E = _spread(rng, 2, 64)
        return {"op": op, "T": _spread(rng, 1, 8192), "K": _spread(rng, 32, 1024), "F": _spread(rng, 32, 2048), "E": E,
                "k": rng.randint(1, min(4, E)), "type": kind, "act": "silu" if kind == "f32" else rng.choice(("relu", "silu")),
                "train": rng.random() < 0.7}
    if op == "products":
        return {"op": op, "R": _spread(rng, 1, 32768), "K": _spread(rng, 16, 2048), "N": _spread(rng, 16, 2048),
                "E": _spread(rng, 1, 64), "type": kind, "train": rng.random() < 0.6}
    if op == "quantise":
        return {"op": op, "R": _spread(rng, 1, 65536), "K": _spread(rng, 16, 2048), "type": kind}
    return {"op": op, "R": _spread(rng, 1, 16384), "K": _spread(rng, 32, 4096), "N": _spread(rng, 16, 4096),
            "E": _spread(rng, 1, 32), "type": kind}


# ---------------------------------------------------------------------------------------------------------- the inputs
class _Inputs:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=self.g, device="cuda") * scale).to(dtype)

    def logits(self, T, E, dtype):
        # some experts are favoured, as a router's are before it is balanced
        return (1.5 * self.normal(T, E) + self.normal(1, E)).to(dtype)

    def offsets(self, R, E):
        """[E + 1] borders of the groups: sizes of an uneven distribution, about a fifth of them empty."""
        share = torch.exp(1.2 * self.normal(E)) * (torch.rand(E, generator=self.g, device="cuda") > 0.2)
        share[0] += 1e-3
        ends = torch.cumsum(share.double(), 0)
        ends = torch.floor(ends / ends[-1] * R + 0.5).clamp_(0, R)
        ends[-1] = R
        return torch.cat([ends.new_zeros(1), ends]).to(torch.int32)


def prepare(case, seed):
    c, i, dt = dict(case), _Inputs(seed), _TYPES[case["type"]]
    s = {"case": c}
    if c["op"] in ("route", "layer"):
        T, E, k = c["T"], c["E"], c["k"]
        s["logits"] = i.logits(T, E, dt)
        if c["op"] == "route":
            s["mask"] = (torch.rand(T, generator=i.g, device="cuda") > 0.125) if c["masked"] else None
            s["g_weights"], s["g_load"] = i.normal(T, k), i.normal(E)
            return s
        K, F = c["K"], c["F"]
        s["x"] = i.normal(T, K, dtype=dt)
        s["w1"], s["b1"] = i.normal(E, F, K, dtype=dt, scale=K ** -0.5), i.normal(E, F, dtype=dt, scale=0.1)
        s["w2"], s["b2"] = i.normal(E, K, F, dtype=dt, scale=F ** -0.5), i.normal(E, K, dtype=dt, scale=0.1)
        s["g_out"] = i.normal(T, K, dtype=dt)
        return s
    R, K = c["R"], c["K"]
    if c["op"] == "quantise":  # columns of very different size, as activations have them
        s["x"] = (i.normal(R, K) * torch.exp(1.5 * i.normal(1, K))).to(dt)
        return s
    N, E = c["N"], c["E"]
    s["offsets"] = i.offsets(R, E)
    if c["op"] == "products":
        s["x"] = i.normal(R, K + 8, dtype=dt)[:, :K]  # the leading columns of a wider tensor
        s["w"], s["b"] = i.normal(E, N, K, dtype=dt, scale=K ** -0.5), i.normal(E, N, dtype=dt, scale=0.1)
        s["g_y"] = i.normal(R, N, dtype=dt)
        return s
    s["x"] = i.normal(R, K, dtype=dt)
    # the weights as a 4-bit checkpoint holds them: two codes a byte (low four bits first), one scale byte per 32
    exponent, codes = _mx4_codes(i.normal(E, N, K, scale=K ** -0.5))
    codes = codes.flatten(-2)
    s["codes"] = (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)
    s["scales"] = (exponent + 127).to(torch.uint8)
    s["b"] = i.normal(E, N, dtype=dt, scale=0.1)
    return s


# ----------------------------------------------------------------------------------------------------- the plain forms
def _route(z, k, mask):
    """(weights, experts, load, probabilities) of the rows' logits z (32 bits)."""
    if mask is not None:
        z = z.masked_fill(~mask[:, None], -math.inf)
    top, at = torch.sort(z, dim=1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    live = top > -math.inf
    experts = torch.where(live, at, -1).to(torch.int32)
    m = torch.where(live[:, :1], top[:, :1], 0.0)
    p = torch.exp(z - m)
    p = p / p.sum(1, keepdim=True).clamp_min(1e-30)
    w = torch.where(live, torch.exp(top - m), 0.0)
    w = w / w.sum(1, keepdim=True).clamp_min(1e-30)
    return w, experts, p.double().sum(0).div(z.shape[0]).to(z.dtype), p


def _route_gradient(w, experts, p, g_weights, g_load):
    g = w * (g_weights - (w * g_weights).sum(1, keepdim=True))
    dense = torch.zeros_like(p).scatter_add_(1, experts.clamp_min(0).long(), torch.where(experts >= 0, g, 0.0))
    if g_load is None:
        return dense
    return dense + p * (g_load - (p * g_load).sum(1, keepdim=True)) / p.shape[0]


def _group(experts, E):
    """(offsets, order, position) of the places sorted by expert, those without one behind the last group."""
    flat = experts.flatten()
    key = torch.where(flat >= 0, flat, E)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=flat.device).index_add_(0, key, torch.ones_like(key, dtype=torch.int64))
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts[:E], 0)])
    order = torch.sort(key, stable=True)[1]
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=flat.device)
    order = torch.where(torch.arange(order.numel(), device=flat.device) < offsets[-1], order, -1)
    return offsets.to(torch.int32), order.to(torch.int32), torch.where(flat >= 0, position, -1).view(experts.shape).to(torch.int32)


def _products(x, w, offsets):
    """x_r W_e^T for every group's rows; rows behind the last group are zero."""
    y = x.new_zeros(x.shape[0], w.shape[1])
    at = offsets.tolist()
    for e in range(w.shape[0]):
        if at[e + 1] > at[e]:
            y[at[e]:at[e + 1]] = x[at[e]:at[e + 1]] @ w[e].T
    return y


def _weight_gradient(g, x, offsets):
    """Every group's (g^T x, column sums of g)."""
    out, sums = g.new_zeros(offsets.numel() - 1, g.shape[1], x.shape[1]), g.new_zeros(offsets.numel() - 1, g.shape[1])
    at = offsets.tolist()
    for e in range(out.shape[0]):
        if at[e + 1] > at[e]:
            mine = g[at[e]:at[e + 1]]
            out[e], sums[e] = mine.T @ x[at[e]:at[e + 1]], mine.sum(0)
    return out, sums


def _group_of_row(offsets, rows):
    return torch.searchsorted(offsets[1:].long(), torch.arange(rows, device=offsets.device), right=True)


def _bias(b, offsets, rows):
    """The bias of every row's group; zero behind the last one."""
    of = _group_of_row(offsets, rows)
    return torch.cat([b, b.new_zeros(1, b.shape[1])])[of]


def _act(z, act):
    return torch.where(z > 0, z, 0.0) if act == "relu" else z / (1 + torch.exp(-z))


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _layer(s, x, logits, w1, b1, w2, b2, g_out):
    """The expert block in the inputs' type (32 or 64 bits): its output and, in training, every gradient."""
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    wt, experts, _, p = _route(logits, k, None)
    offsets, order, position = _group(experts, E)
    token = (order.long() // k)  # every place has an expert here: no logit is -inf
    xs = x[token]
    z = _products(xs, w1, offsets) + _bias(b1, offsets, T * k)
    h = _act(z, c["act"])
    y = _products(h, w2, offsets) + _bias(b2, offsets, T * k)
    ys = y[position.long()]  # [T, k, K]
    out = {"out": x + (wt[..., None] * ys).sum(1)}
    if not c["train"]:
        return out
    gy = (wt.flatten()[order.long()])[:, None] * g_out[token]
    gz = _products(gy, w2.transpose(1, 2), offsets) * _act_slope(z, c["act"])
    gxs = _products(gz, w1.transpose(1, 2), offsets)
    out["g_x"] = g_out + gxs[position.long()].sum(1)
    out["g_logits"] = _route_gradient(wt, experts, p, (g_out[:, None, :] * ys).sum(-1), None)
    out["g_w1"], out["g_b1"] = _weight_gradient(gz, xs, offsets)
    out["g_w2"], out["g_b2"] = _weight_gradient(gy, h, offsets)
    return out


def _mx4_codes(x):
    """(exponent [..., B], code [..., B, 32]) of the blocks of 32 along the last axis (zeros behind its end)."""
    B = -(-x.shape[-1] // 32)
    v = torch.nn.functional.pad(x, (0, 32 * B - x.shape[-1])).unflatten(-1, (B, 32))
    exponent = torch.frexp(v.abs().amax(-1))[1] - 3  # floor(log2(largest)) - 2
    exponent = torch.where(v.abs().amax(-1) > 0, exponent, -127).clamp(-127, 127)
    a = torch.ldexp(v, -exponent[..., None]).abs()
    # ties to the even code
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    return exponent, code | (torch.signbit(v).int() << 3)


def _mx4_values(exponent, code):
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=code.device)
    return torch.ldexp(table[code.long()], exponent[..., None]).flatten(-2)


def _unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).int()


def _plain(s):
    c = s["case"]
    dt = _TYPES[c["type"]]
    if c["op"] == "route":
        w, experts, load, p = _route(s["logits"].float(), c["k"], s["mask"])
        offsets, order, position = _group(experts, c["E"])
        out = {"weights": w, "experts": experts, "load": load, "offsets": offsets, "order": order, "position": position}
        if c["train"]:
            out["g_logits"] = _route_gradient(w, experts, p, s["g_weights"], s["g_load"]).to(dt)
        return out
    if c["op"] == "layer":
        out = _layer(s, *(s[n].float() for n in ("x", "logits", "w1", "b1", "w2", "b2", "g_out")))
        return {n: v.to(dt) for n, v in out.items()}
    if c["op"] == "products":
        x, w = s["x"].float(), s["w"].float()
        out = {"y": (_products(x, w, s["offsets"]) + _bias(s["b"].float(), s["offsets"], c["R"])).to(dt)}
        if c["train"]:
            g = s["g_y"].float()
            out["g_x"] = _products(g, w.transpose(1, 2), s["offsets"]).to(dt)
            out["g_w"], out["g_b"] = (v.to(dt) for v in _weight_gradient(g, x, s["offsets"]))
        return out
    exponent, code = _mx4_codes(s["x"].float())
    x = _mx4_values(exponent, code)[:, :c["K"]]
    if c["op"] == "quantise":
        return {"values": x.to(dt), "scales": (exponent + 127).to(torch.uint8)}
    w = _mx4_values(s["scales"].int() - 127, _unpack(s["codes"]))[..., :c["K"]]
    return {"y": (_products(x, w, s["offsets"]) + _bias(s["b"].float(), s["offsets"], c["R"])).to(dt)}


# ------------------------------------------------------------------------------------------------ the package's own calls
def _own(s):
    from dimo_amd import experts as ex
    from dimo_amd import mx4
    c = s["case"]
    if c["op"] == "route":
        z = s["logits"].detach().requires_grad_(c["train"])
        w, experts, load = ex.route_topk(z, c["k"], row_mask=s["mask"])
        groups = ex.group_rows(experts, c["E"])
        out = {"weights": w, "experts": experts, "load": load, "offsets": groups.offsets, "order": groups.order,
               "position": groups.position}
        if c["train"]:
            out["g_logits"] = torch.autograd.grad((w, load), z, (s["g_weights"], s["g_load"]))[0]
        return out
    if c["op"] == "layer":
        names = ("x", "logits", "w1", "b1", "w2", "b2")
        leaf = [s[n].detach().requires_grad_(c["train"]) for n in names]
        out = {"out": ex.expert_mlp(*leaf, k=c["k"], activation=c["act"])}
        if c["train"]:
            out.update(zip(("g_" + n for n in names), torch.autograd.grad(out["out"], leaf, s["g_out"])))
        return out
    if c["op"] == "products":
        leaf = [s[n].detach().requires_grad_(c["train"]) for n in ("x", "w", "b")]
        out = {"y": ex.grouped_linear(leaf[0], leaf[1], ex.RowGroups(s["offsets"]), bias=leaf[2])}
        if c["train"]:
            out.update(zip(("g_x", "g_w", "g_b"), torch.autograd.grad(out["y"], leaf, s["g_y"])))
        return out
    x = mx4.quantize_mx4(s["x"])
    if c["op"] == "quantise":
        return {"values": x.dequantize(s["x"].dtype), "scales": x.scales}
    w = mx4.MX4(s["codes"], s["scales"], c["K"])
    return {"y": mx4.mx4_linear(x, w, bias=s["b"], groups=ex.RowGroups(s["offsets"]), out_dtype=s["x"].dtype)}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------- what it costs
def work(case):
    c = case
    b = 4 if c["type"] == "f32" else 2
    if c["op"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        n = T * E * b + T * k * (4 + 4 + 4 + 4) + 8 * E + (T if c["masked"] else 0)  # logits; weights, experts, order, position
        f = 5 * T * E
        if c["train"]:
            n, f = n + T * E * b + T * k * 4 + 4 * E, f + 6 * T * E
        return {"bytes": n, "flops": f}
    if c["op"] == "layer":
        T, K, F, E, k = (c[n] for n in ("T", "K", "F", "E", "k"))
        seen = min(E, T * k)  # experts that can have rows
        n = b * (2 * T * K + T * E + seen * (2 * K * F + K + F))
        f = 4 * T * k * K * F
        if c["train"]:
            n, f = n + b * (2 * T * K + T * E + E * (2 * K * F + K + F)), 3 * f
        return {"bytes": n, "flops": f}
    R, K = c["R"], c["K"]
    if c["op"] == "quantise":
        return {"bytes": R * K * (2 * b) + R * (-(-K // 32)), "flops": 4 * R * K}
    N, seen = c["N"], min(c["E"], R)
    if c["op"] == "products":
        n, f = b * (R * K + R * N + seen * N * (K + 1)), 2 * R * N * K
        if c["train"]:
            n, f = n + b * (R * N + R * K + c["E"] * N * (K + 1)), 3 * f
        return {"bytes": n, "flops": f}
    return {"bytes": b * (R * K + R * N + seen * N) + seen * N * K * 17 // 32, "flops": 2 * R * N * K}


# --------------------------------------------------------------------------------------------- the definition in 64 bits
def _route_exact(z, k, mask):
    z = z.clone()
    if mask is not None:
        z[~mask] = -math.inf
    T, E = z.shape
    p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
    left, rows = z.clone(), torch.arange(T, device=z.device)
    chosen, w = [], []
    for _ in range(k):  # the largest that is left, k times over
        best, _ = left.max(1)
        at = (left == best[:, None]).to(torch.uint8).argmax(1)  # the first of equals
        none = best == -math.inf
        chosen.append(torch.where(none, -1, at))
        w.append(torch.where(none, 0.0, p[rows, at]))
        left[rows, at] = -math.inf
    chosen, w = torch.stack(chosen, 1), torch.stack(w, 1)
    total = w.sum(1, keepdim=True)
    return torch.where(total > 0, w / total, 0.0), chosen, p


def _route_gradient_exact(w, chosen, p, g_weights, g_load):
    out = torch.zeros_like(p)
    inner = (w * g_weights).sum(1)
    for j in range(w.shape[1]):
        live = chosen[:, j] >= 0
        out[live, chosen[live, j]] += (w[:, j] * (g_weights[:, j] - inner))[live]
    if g_load is not None:
        out += p * (g_load[None] - (p @ g_load)[:, None]) / p.shape[0]
    return out


def _exact_values(x):
    """The e2m1 values nearest to x / scale, times the scale, block by block of 32."""
    R, K = x.shape
    out = torch.empty_like(x)
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    for lo in range(0, K, 32):
        v = x[:, lo:lo + 32]
        big = v.abs().amax(1, keepdim=True)
        scale = torch.where(big > 0, torch.exp2(torch.floor(torch.log2(big.clamp_min(1e-300))) - 2), 1.0)
        a = (v / scale).abs().clamp_max(6.0)
        up = torch.searchsorted(grid, a.contiguous()).clamp_max(7)  # first value >= a
        down = (up - 1).clamp_min(0)
        to_up, to_down = grid[up] - a, a - grid[down]
        code = torch.where((to_up < to_down) | ((to_up == to_down) & (up % 2 == 0)), up, down)
        out[:, lo:lo + 32] = torch.sign(v) * grid[code] * scale
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "route":
        z = s["logits"].double()
        w, chosen, p = _route_exact(z, c["k"], s["mask"])
        out = {"weights": w, "experts": None, "load": p.sum(0) / c["T"], "offsets": None, "order": None, "position": None}
        if c["train"]:
            out["g_logits"] = _route_gradient_exact(w, chosen, p, s["g_weights"].double(), s["g_load"].double())
        return out
    if c["op"] == "layer":
        x, z, w1, b1, w2, b2, go = (s[n].double() for n in ("x", "logits", "w1", "b1", "w2", "b2", "g_out"))
        w, chosen, p = _route_exact(z, c["k"], None)
        out = {"out": x.clone()}
        g = {n: torch.zeros_like(t) for n, t in (("g_x", x), ("g_w1", w1), ("g_b1", b1), ("g_w2", w2), ("g_b2", b2))}
        g_weights = torch.zeros_like(w)
        for e in range(c["E"]):  # expert by expert on the rows that chose it
            row, slot = torch.nonzero(chosen == e, as_tuple=True)
            if not row.numel():
                continue
            a = x[row] @ w1[e].T + b1[e]
            sig = torch.sigmoid(a)
            h = a.clamp_min(0) if c["act"] == "relu" else a * sig
            y = h @ w2[e].T + b2[e]
            wt = w[row, slot][:, None]
            out["out"].index_add_(0, row, wt * y)
            if c["train"]:
                g_weights[row, slot] = (go[row] * y).sum(1)
                gy = wt * go[row]
                ga = (gy @ w2[e]) * ((a > 0).double() if c["act"] == "relu" else sig + a * sig * (1 - sig))
                g["g_w2"][e], g["g_b2"][e] = gy.T @ h, gy.sum(0)
                g["g_w1"][e], g["g_b1"][e] = ga.T @ x[row], ga.sum(0)
                g["g_x"].index_add_(0, row, ga @ w1[e])
        if c["train"]:
            g["g_x"] += go
            out.update(g, g_logits=_route_gradient_exact(w, chosen, p, g_weights, None))
        return out
    if c["op"] == "quantise":
        return {"values": _exact_values(s["x"].double()), "scales": None}
    at = s["offsets"].tolist()
    if c["op"] == "products":
        x, w, b, gy = (s[n].double() for n in ("x", "w", "b", "g_y"))
        out = {"y": x.new_zeros(c["R"], c["N"])}
        g = {"g_x": torch.zeros_like(x), "g_w": torch.zeros_like(w), "g_b": torch.zeros_like(b)}
        for e in range(c["E"]):
            r = slice(at[e], at[e + 1])
            out["y"][r] = torch.addmm(b[e], x[r], w[e].T)
            if c["train"]:
                g["g_x"][r], g["g_w"][e], g["g_b"][e] = gy[r] @ w[e], gy[r].T @ x[r], gy[r].sum(0)
        return {**out, **g} if c["train"] else out
    x = _exact_values(s["x"].double())
    table = torch.tensor([(-1.0) ** (n >> 3) * _E2M1[n & 7] for n in range(16)], dtype=torch.float64, device=x.device)
    y = x.new_zeros(c["R"], c["N"])
    for e in range(c["E"]):
        r = slice(at[e], at[e + 1])
        byte = s["codes"][e].long()
        w = torch.stack([table[byte & 15], table[byte >> 4]], -1).reshape(c["N"], -1)
        w = w * torch.exp2(s["scales"][e].double() - 127).repeat_interleave(32, 1)
        y[r] = torch.addmm(s["b"][e].double(), x[r], w[:, :c["K"]].T)
    return {"y": y}
