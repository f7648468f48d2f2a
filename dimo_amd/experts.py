"""Expert blocks on the HIP library: top-k routing of rows, products grouped by expert, and the weighted sum that brings
the experts' rows back together (dimo_amd/csrc/experts.hip, grouped.hip; include/dimo_hip.h).

    weights, experts, load = route_topk(logits, k)            # [T, k], [T, k], [E]
    groups = group_rows(experts, E)                           # the T k places, grouped by expert
    h = grouped_linear(x, w1, groups, b1, "relu", gather=True)  # [T k, F]: rows of x, in the order of the groups
    y = grouped_linear(h, w2, groups, b2)                     # [T k, N]
    out = combine_rows(y, groups, weights, residual=x)        # [T, N]

`expert_mlp` is this sequence as one call, `ExpertMLP` the module around it.  Nothing here has a counterpart in the
reference, whose deformation network (renderer/latent_gs_renderer.py:184-245) is one dense MLP for all motions: an
expert block gives that network capacity of which every row uses k parts (`deform.TimeNet(experts=...)`).

Types: fp32, bf16, fp16 (all tensors of a call alike; routing weights, load and their gradients are fp32).  Sums are fp32.
fp32 products are made of bf16 ones: each is off by up to 6.1 x 2^-24 of its size (an fp32 multiplication: 1 x 2^-24) where its
operands are 2^-110 or larger, by up to 2^-134 of the other operand where one is smaller; an infinite operand gives NaN.  The sizes of
the groups stay on the device: no call synchronises, every call may be captured into a graph.  All calls run on the
current stream of the tensors' device.  GPU only.
"""
import ctypes as C

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _lib

MAX_EXPERTS = 1024
MAX_SIZE = 1 << 30  # rows, places and columns of a call
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2}


def _dtype(t, what):
    if t.dtype not in _DTYPES:
        raise ValueError(f"{what}: fp32, bf16 or fp16 expected, got {t.dtype}")
    return _DTYPES[t.dtype]


def _gpu(*tensors):
    """The tensors' common device (a GPU), or an error."""
    first = tensors[0]
    if not first.is_cuda:
        raise RuntimeError("the expert operators need GPU tensors (no CPU fallback in the product path)")
    device = first.device
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on different devices ({device}, {t.device})")
    return device


class _Nothing:
    def __enter__(self):
        pass

    def __exit__(self, *_):
        pass


_HERE = _Nothing()


def _on(device):
    """Makes a tensor's device current for a launch (nothing to do when it is: one query of the runtime)."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _rows(t):
    """A matrix whose rows are contiguous (a view of a wider tensor is taken as it is)."""
    if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _check_sizes(*sizes):
    if max(sizes) > MAX_SIZE:
        raise ValueError(f"up to {MAX_SIZE} rows, places and columns expected, got {max(sizes)}")


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _tracked(*tensors):
    """Whether a call goes through its autograd function: for gradients, and wherever a level of forward-mode derivatives is
    open -- torch then refuses inputs with tangents, which would otherwise be dropped without a word."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_tangents(*tensors):
    """For calls without derivatives of either kind."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("no forward-mode derivative for the 4-bit operators")


# ------------------------------------------------------------------------------------------------ routing
def _route_forward(logits, k, row_mask, normalize):
    T, E = logits.shape
    L = _lib.lib()
    weights = torch.empty(T, k, dtype=torch.float32, device=logits.device)
    experts = torch.empty(T, k, dtype=torch.int32, device=logits.device)
    load = torch.empty(E, dtype=torch.float32, device=logits.device)
    with _on(logits.device):
        nbytes = L.dimo_route_workspace_bytes(T, E)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device) if nbytes else None
        _lib.check(L.dimo_route_topk_forward(T, E, k, _DTYPES[logits.dtype], logits.data_ptr(), _ld(logits),
                                             _lib.ptr(row_mask), int(normalize), weights.data_ptr(), experts.data_ptr(),
                                             load.data_ptr(), _lib.ptr(ws), nbytes, _lib.current_stream()),
                   "dimo_route_topk_forward")
    return weights, experts, load


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, row_mask, normalize):
        weights, experts, load = _route_forward(logits, k, row_mask, normalize)
        ctx.save_for_backward(logits, row_mask, weights, experts)
        ctx.normalize = bool(normalize)
        ctx.mark_non_differentiable(experts)
        ctx.set_materialize_grads(False)
        return weights, experts, load

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_weights, _, g_load):
        logits, row_mask, weights, experts = ctx.saved_tensors
        if g_weights is None and g_load is None:
            return None, None, None, None
        T, E = logits.shape
        g = torch.empty(T, E, dtype=logits.dtype, device=logits.device)
        g_weights = None if g_weights is None else g_weights.contiguous()
        g_load = None if g_load is None else g_load.contiguous()
        with _on(logits.device):
            _lib.check(_lib.lib().dimo_route_topk_backward(
                T, E, weights.shape[1], _DTYPES[logits.dtype], logits.data_ptr(), _ld(logits), _lib.ptr(row_mask),
                int(ctx.normalize), weights.data_ptr(), experts.data_ptr(), _lib.ptr(g_weights), _lib.ptr(g_load),
                g.data_ptr(), _lib.current_stream()), "dimo_route_topk_backward")
        return g, None, None, None


def route_topk(logits, k, row_mask=None, normalize=True):
    """(weights [T, k] fp32, experts [T, k] int32, load [E] fp32) of logits [T, E].

    experts: each row's k largest logits in descending order (ties: the lowest index; -inf and NaN are never chosen;
    -1 with weight 0 where nothing is left, and in rows whose row_mask [T] is False).  weights: softmax over the chosen
    (normalize=False: over all E).  load: the experts' mean softmax probability over the T rows (masked rows count as
    0), for a balancing term.  A row with a NaN or +inf logit has NaN weights.  Differentiable in `logits` through
    weights and load."""
    if logits.dim() != 2:
        raise ValueError("logits: [T, E] expected")
    _gpu(logits, row_mask)
    _dtype(logits, "logits")
    _check_sizes(logits.shape[0])
    if not 1 <= logits.shape[1] <= MAX_EXPERTS or not 1 <= k <= logits.shape[1]:
        raise ValueError(f"1 <= k <= E <= {MAX_EXPERTS} expected, got k = {k}, E = {logits.shape[1]}")
    if row_mask is not None:
        if row_mask.dtype != torch.bool or row_mask.shape != logits.shape[:1]:
            raise ValueError("row_mask: bool [T] expected")
        row_mask = row_mask.contiguous()
    logits = _rows(logits)
    if _tracked(logits):
        return _RouteTopk.apply(logits, k, row_mask, normalize)
    return _route_forward(logits, k, row_mask, normalize)


class RowGroups:
    """Rows grouped by expert.  offsets [E + 1] int32: expert e owns rows offsets[e] .. offsets[e + 1] - 1 (offsets[0]
    = 0); rows behind offsets[E] belong to nobody.  From `group_rows` also order [T k] (which place a row came from) and
    position [T, k] (which row a place went to; -1: none); rows [T k] = order / k."""

    __slots__ = ("offsets", "order", "position", "rows")

    def __init__(self, offsets):
        if offsets.dim() != 1 or offsets.dtype != torch.int32 or not offsets.is_contiguous():
            raise ValueError("offsets: contiguous int32 [E + 1] expected")
        if not 2 <= offsets.shape[0] <= MAX_EXPERTS + 1:
            raise ValueError(f"1 to {MAX_EXPERTS} groups expected")
        self.offsets, self.order, self.position, self.rows = offsets, None, None, None

    @property
    def num_experts(self):
        return self.offsets.shape[0] - 1


def _saved_groups(offsets, rows, position):
    """The grouping of a forward pass from tensors that autograd kept for its backward (and would miss if they had changed)."""
    groups = RowGroups(offsets)
    groups.rows, groups.position = rows, position
    return groups


def group_rows(experts, num_experts):
    """RowGroups of the places of experts [T, k] int32, stable: by expert, then by place.  A place whose value is outside
    0 .. num_experts - 1 belongs to nobody."""
    if experts.dim() != 2 or experts.dtype != torch.int32:
        raise ValueError("experts: int32 [T, k] expected")
    if not 1 <= num_experts <= MAX_EXPERTS or experts.shape[1] < 1:
        raise ValueError(f"1 to {MAX_EXPERTS} experts and k >= 1 expected")
    device = _gpu(experts)
    S = experts.numel()
    _check_sizes(S)
    experts = experts.contiguous()
    L = _lib.lib()
    groups = RowGroups(torch.empty(num_experts + 1, dtype=torch.int32, device=device))
    groups.order = torch.empty(S, dtype=torch.int32, device=device)
    groups.rows = torch.empty(S, dtype=torch.int32, device=device)
    groups.position = torch.empty(experts.shape, dtype=torch.int32, device=device)
    with _on(device):
        nbytes = L.dimo_group_rows_workspace_bytes(S, num_experts)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _lib.check(L.dimo_group_rows(S, num_experts, experts.shape[1], experts.data_ptr(), groups.offsets.data_ptr(),
                                     groups.order.data_ptr(), groups.position.data_ptr(), groups.rows.data_ptr(),
                                     _lib.ptr(ws), nbytes, _lib.current_stream()), "dimo_group_rows")
    return groups


# ------------------------------------------------------------------------------------------------ grouped products
def _linear_forward(x, weight, bias, groups, act, gather, save_z):
    E, N, K = weight.shape
    R = groups.order.shape[0] if gather else x.shape[0]
    y = torch.empty(R, N, dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if save_z else None
    with _on(x.device):
        _lib.check(_lib.lib().dimo_grouped_linear_forward(
            _DTYPES[x.dtype], R, E, K, N, x.data_ptr(), _ld(x), groups.rows.data_ptr() if gather else None,
            groups.offsets.data_ptr(), weight.data_ptr(), _lib.ptr(bias), act, y.data_ptr(), _lib.ptr(z), _lib.current_stream()), "dimo_grouped_linear_forward")
    return y, z


def _linear_dgrad(g, weight, groups):
    E, N, K = weight.shape
    gx = torch.empty(g.shape[0], K, dtype=g.dtype, device=g.device)
    with _on(g.device):
        _lib.check(_lib.lib().dimo_grouped_linear_dgrad(
            _DTYPES[g.dtype], g.shape[0], E, K, N, g.data_ptr(), groups.offsets.data_ptr(), weight.data_ptr(), 0, None,
            gx.data_ptr(), _lib.current_stream()), "dimo_grouped_linear_dgrad")
    return gx


def _linear_wgrad(g, x, shape, groups, gather, need_bias):
    E, N, K = shape
    gw = torch.empty(E, N, K, dtype=g.dtype, device=g.device)
    gb = torch.empty(E, N, dtype=g.dtype, device=g.device) if need_bias else None
    with _on(g.device):
        L = _lib.lib()
        nbytes = L.dimo_grouped_linear_wgrad_workspace_bytes(_DTYPES[g.dtype], g.shape[0], E, K, N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=g.device) if nbytes else None
        _lib.check(L.dimo_grouped_linear_wgrad(
            _DTYPES[g.dtype], g.shape[0], E, K, N, g.data_ptr(), x.data_ptr(), _ld(x),
            groups.rows.data_ptr() if gather else None, groups.offsets.data_ptr(), gw.data_ptr(), _lib.ptr(gb),
            _lib.ptr(ws), nbytes, _lib.current_stream()), "dimo_grouped_linear_wgrad")
    return gw, gb


def _activation_backward(g, saved, act):
    out = torch.empty_like(g)
    with _on(g.device):
        _lib.check(_lib.lib().dimo_activation_backward(_DTYPES[g.dtype], act, g.numel(), g.data_ptr(), saved.data_ptr(),
                                                       out.data_ptr(), _lib.current_stream()), "dimo_activation_backward")
    return out


def _combine_forward(y, weights, groups, residual):
    T, k = groups.position.shape
    out = torch.empty(T, y.shape[1], dtype=y.dtype, device=y.device)
    with _on(y.device):
        _lib.check(_lib.lib().dimo_combine_rows_forward(
            T, k, y.shape[1], y.shape[0], _DTYPES[y.dtype], y.data_ptr(), _ld(y), _lib.ptr(weights),
            groups.position.data_ptr(), _lib.ptr(residual), _ld(residual) if residual is not None else 0, out.data_ptr(),
            _lib.current_stream()), "dimo_combine_rows_forward")
    return out


def _combine_backward(g, y, weights, groups, need_y, need_weights):
    T, k = groups.position.shape
    N = g.shape[1]
    g_y = torch.empty(T * k, N, dtype=g.dtype, device=g.device) if need_y else None
    g_w = torch.empty(T, k, dtype=torch.float32, device=g.device) if need_weights else None
    with _on(g.device):
        _lib.check(_lib.lib().dimo_combine_rows_backward(
            T, k, N, T * k, groups.num_experts, _DTYPES[g.dtype], g.data_ptr(), _ld(g), _lib.ptr(y), _ld(y) if y is not None else 0,
            _lib.ptr(weights), groups.position.data_ptr(), groups.offsets.data_ptr(), _lib.ptr(g_y), _lib.ptr(g_w),
            _lib.current_stream()), "dimo_combine_rows_backward")
    return g_y, g_w


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, act, gather):
        y, z = _linear_forward(x, weight, bias, groups, act, gather, act == 2)
        ctx.save_for_backward(x, weight, z if act == 2 else y if act == 1 else None, groups.offsets, groups.rows, groups.position)
        ctx.act, ctx.gather, ctx.bias = act, gather, bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, weight, saved, *grouping = ctx.saved_tensors
        groups = _saved_groups(*grouping)
        g = g.contiguous()
        if ctx.act:
            g = _activation_backward(g, saved, ctx.act)
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = _linear_dgrad(g, weight, groups)
            if ctx.gather:
                gx = _combine_forward(gx, None, groups, None)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            gw, gb = _linear_wgrad(g, x, weight.shape, groups, ctx.gather, ctx.bias)
        return gx, gw, gb, None, None, None


def _check_linear_groups(E, rows, groups):
    if E != groups.num_experts:
        raise ValueError(f"{E} experts' weights for {groups.num_experts} groups")
    if rows is not None and groups.position is not None and rows != groups.order.shape[0]:
        raise ValueError(f"{rows} rows in the order of the groups, {groups.order.shape[0]} expected")


def _check_linear(x, weight, bias, groups, activation, gather):
    if x.dim() != 2 or weight.dim() != 3:
        raise ValueError("x: [rows, K] and weight: [E, N, K] expected")
    _gpu(x, weight, bias, groups.offsets)
    _dtype(x, "x")
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise ValueError("x, weight and bias must have one type")
    E, N, K = weight.shape
    _check_sizes(x.shape[0], N, K)
    if x.shape[1] != K or K < 1 or N < 1:
        raise ValueError(f"x has {x.shape[1]} columns, weight takes {K}")
    if bias is not None and bias.shape != (E, N):
        raise ValueError("bias: [E, N] expected")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation: one of {list(_ACTIVATIONS)} expected")
    if gather:
        if groups.position is None:
            raise ValueError("gather=True needs groups made by group_rows")
        if x.shape[0] != groups.position.shape[0]:
            raise ValueError(f"{x.shape[0]} rows, {groups.position.shape[0]} were grouped")
    _check_linear_groups(E, None if gather else x.shape[0], groups)


def grouped_linear(x, weight, groups, bias=None, activation=None, gather=False):
    """y[r] = activation(weight[e] @ x[r] + bias[e]) for every row r of group e; zeros behind the last group.

    x [R, K] in the order of the groups, or (gather=True) the [T, K] rows that were routed: row r then reads the row its
    place came from, and x's gradient is the sum over a row's places.  weight [E, N, K], bias [E, N] or None,
    activation None, "relu" or "silu".  Differentiable in x, weight and bias; an expert without rows gets zero
    gradients."""
    _check_linear(x, weight, bias, groups, activation, gather)
    x, weight = _rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if _tracked(x, weight, bias):
        return _GroupedLinear.apply(x, weight, bias, groups, _ACTIVATIONS[activation], gather)
    return _linear_forward(x, weight, bias, groups, _ACTIVATIONS[activation], gather, False)[0]


class _CombineRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual, groups):
        ctx.save_for_backward(y if weights is not None and weights.requires_grad else None, weights, groups.offsets, groups.rows,
                              groups.position)
        return _combine_forward(y, weights, groups, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        y, weights, *grouping = ctx.saved_tensors
        groups = _saved_groups(*grouping)
        g_y = g_w = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            g_y, g_w = _combine_backward(_rows(g), y, weights, groups, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return g_y, g_w, g if ctx.needs_input_grad[2] else None, None


def combine_rows(y, groups, weights=None, residual=None):
    """out[t] = residual[t] + sum_j weights[t, j] y[position[t, j]]: the rows y [T k, N] of the groups, back at their
    places and summed over a row's k places (weights fp32 [T, k], None: 1; places of nobody add nothing).  Differentiable
    in y, weights and residual."""
    if groups.position is None:
        raise ValueError("combine_rows needs groups made by group_rows")
    if y.dim() != 2 or y.shape[0] != groups.order.shape[0]:
        raise ValueError(f"y: [{groups.order.shape[0]}, N] expected")
    _gpu(y, weights, residual, groups.offsets)
    _dtype(y, "y")
    _check_sizes(y.shape[1])
    if weights is not None and (weights.shape != groups.position.shape or weights.dtype != torch.float32):
        raise ValueError("weights: fp32 [T, k] expected")
    if residual is not None and (residual.dtype != y.dtype or residual.shape != (groups.position.shape[0], y.shape[1])):
        raise ValueError("residual: [T, N] of y's type expected")
    y = _rows(y)
    weights = None if weights is None else weights.contiguous()
    residual = None if residual is None else _rows(residual)
    if _tracked(y, weights, residual):
        return _CombineRows.apply(y, weights, residual, groups)
    return _combine_forward(y, weights, groups, residual)


class _ExpertMlpDesc(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("dtype", "T", "K", "F", "E", "k", "act", "normalize")] + [("ld_x", C.c_int64), ("ld_logits", C.c_int64)] \
        + [(n, C.c_void_p) for n in ("x", "logits", "w1", "b1", "w2", "b2", "row_mask")]


def _expert_mlp_desc(x, logits, w1, b1, w2, b2, row_mask, k, act, normalize):
    return _ExpertMlpDesc(_DTYPES[x.dtype], x.shape[0], x.shape[1], w1.shape[1], w1.shape[0], k, act, normalize, _ld(x),
                          _ld(logits), x.data_ptr(), logits.data_ptr(), w1.data_ptr(), _lib.ptr(b1), w2.data_ptr(), _lib.ptr(b2),
                          _lib.ptr(row_mask))


def _expert_mlp_forward(x, logits, w1, b1, w2, b2, row_mask, k, act, normalize, keep):
    L, d = _lib.lib(), _expert_mlp_desc(x, logits, w1, b1, w2, b2, row_mask, k, act, normalize)
    at = C.addressof(d)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _on(x.device):
        nbytes = L.dimo_expert_mlp_workspace_bytes(at, keep)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        _lib.check(L.dimo_expert_mlp_forward(at, keep, out.data_ptr(), ws.data_ptr(), nbytes, _lib.current_stream()),
                   "dimo_expert_mlp_forward")
    return out, ws


class _ExpertMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, logits, w1, b1, w2, b2, row_mask, k, act, normalize):
        out, ws = _expert_mlp_forward(x, logits, w1, b1, w2, b2, row_mask, k, act, normalize, True)
        ctx.save_for_backward(x, logits, w1, b1, w2, b2, row_mask, ws)
        ctx.rest = k, act, normalize
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        *tensors, ws = ctx.saved_tensors
        x, logits, w1, b1, w2, b2, _ = tensors
        L, d = _lib.lib(), _expert_mlp_desc(*tensors, *ctx.rest)
        at, need = C.addressof(d), ctx.needs_input_grad
        g = _rows(g)
        # (a bias gradient comes with its weight's)
        wanted = [need[0], need[1], need[2] or need[3], need[3], need[4] or need[5], need[5]]
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if on else None
                 for t, on in zip((x, logits, w1, b1, w2, b2), wanted)]
        with _on(x.device):
            nbytes = L.dimo_expert_mlp_scratch_bytes(at)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            _lib.check(L.dimo_expert_mlp_backward(at, g.data_ptr(), _ld(g), ws.data_ptr(), scratch.data_ptr(), nbytes,
                                                  *[_lib.ptr(t) for t in grads], _lib.current_stream()),
                       "dimo_expert_mlp_backward")
        return (*[t if on else None for t, on in zip(grads, need)], None, None, None, None)


def expert_mlp(x, logits, w1, b1, w2, b2, k, activation="relu", row_mask=None, normalize=True):
    """x + sum over a row's k experts of weight * (w2 activation(w1 x + b1) + b2): routing (weights normalised over the
    chosen; normalize=False: softmax over all E), both products and the sum as one call per direction -- what route_topk,
    group_rows, grouped_linear (gathering, then plain) and combine_rows give one by one.  x [T, K], logits [T, E], w1 [E, F, K], b1 [E, F] or None, w2 [E, K, F],
    b2 [E, K] or None; row_mask [T]: rows with False come back as they are.  Differentiable in x, logits and the weights.
    With k = 1 a normalised weight is the constant 1, and the logits' gradient zero."""
    if x.dim() != 2 or logits.dim() != 2 or w1.dim() != 3:
        raise ValueError("x: [T, K], logits: [T, E] and w1: [E, F, K] expected")
    _gpu(x, logits, w1, b1, w2, b2, row_mask)
    _dtype(x, "x")
    (T, K), (E, F, _) = x.shape, w1.shape
    for t, shape, what in ((logits, (T, E), "logits: [T, E]"), (w1, (E, F, K), "w1: [E, F, K]"), (w2, (E, K, F), "w2: [E, K, F]"),
                           (b1, (E, F), "b1: [E, F]"), (b2, (E, K), "b2: [E, K]")):
        if t is not None and (t.shape != shape or t.dtype != x.dtype):
            raise ValueError(f"{what} of x's type expected")
    if not 1 <= k <= E <= MAX_EXPERTS or K < 1 or F < 1:
        raise ValueError(f"1 <= k <= E <= {MAX_EXPERTS} and at least one column expected")
    _check_sizes(T * k, K, F)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation: one of {list(_ACTIVATIONS)} expected")
    if row_mask is not None:
        if row_mask.dtype != torch.bool or row_mask.shape != (T,):
            raise ValueError("row_mask: bool [T] expected")
        row_mask = row_mask.contiguous()
    x, logits, w1, w2 = _rows(x), _rows(logits), w1.contiguous(), w2.contiguous()
    b1, b2 = None if b1 is None else b1.contiguous(), None if b2 is None else b2.contiguous()
    if _tracked(x, logits, w1, b1, w2, b2):
        return _ExpertMlp.apply(x, logits, w1, b1, w2, b2, row_mask, k, _ACTIVATIONS[activation], bool(normalize))
    return _expert_mlp_forward(x, logits, w1, b1, w2, b2, row_mask, k, _ACTIVATIONS[activation], bool(normalize), False)[0]


def _without_autocast(block, h, dtype):
    """block(h) in the type of its parameters where autocast is on (which would give the router's product another type than the
    rows'), None elsewhere."""
    if not torch.is_autocast_enabled(h.device.type):
        return None
    with torch.autocast(h.device.type, enabled=False):
        return block(h.to(dtype))


class ExpertMLP(nn.Module):
    """h + the weighted sum of a row's k experts (each width -> hidden -> width), h [..., width].  The weights
    are normalised over the chosen; with k = 1, where that would be the constant 1 and the router would not learn, they are
    the softmax over all experts.  The second products start at zero, so a network that gets such a block starts as it was.
    Under autocast the block works (and answers) in its parameters' type.  Nothing here keeps the experts' load even: a balancing
    term takes `load` of route_topk(block.router(rows), k), differentiable in the router.  `quantized()`: the same block for evaluation
    only, its products in microscaled 4-bit form (dimo_amd/mx4.py)."""

    def __init__(self, width, num_experts, k=2, hidden=None, activation="relu", device=None):
        super().__init__()
        hidden = width if hidden is None else hidden
        if not 1 <= k <= num_experts <= MAX_EXPERTS:
            raise ValueError(f"1 <= k <= num_experts <= {MAX_EXPERTS} expected")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation: one of {list(_ACTIVATIONS)} expected")
        self.k, self.activation, self.normalize = k, activation, k > 1
        self.router = nn.Linear(width, num_experts, bias=False)
        self.w1 = nn.Parameter(torch.empty(num_experts, hidden, width))
        self.b1 = nn.Parameter(torch.zeros(num_experts, hidden))
        self.w2 = nn.Parameter(torch.zeros(num_experts, width, hidden))
        self.b2 = nn.Parameter(torch.zeros(num_experts, width))
        for w in self.w1:
            nn.init.xavier_uniform_(w)
        if device is not None:
            self.to(device)

    def forward(self, h):
        out = _without_autocast(self, h, self.w1.dtype)
        if out is not None:
            return out
        rows = h.reshape(-1, h.shape[-1])
        out = expert_mlp(rows, self.router(rows), self.w1, self.b1, self.w2, self.b2, self.k, self.activation,
                         normalize=self.normalize)
        return out.view(h.shape)

    def quantized(self):
        return QuantizedExpertMLP(self)


class QuantizedExpertMLP(nn.Module):
    """An ExpertMLP's weights of this moment in 4-bit form, for evaluation: no parameters, no gradients (a call that would have
    to give any is refused: use torch.no_grad()); the router stays as it is."""

    def __init__(self, block):
        super().__init__()
        from .mx4 import quantize_mx4
        self.k, self.activation, self.normalize, self.hidden = block.k, block.activation, block.normalize, block.w1.shape[1]
        q1, q2 = quantize_mx4(block.w1), quantize_mx4(block.w2)
        for name, t in (("router", block.router.weight.detach().clone()), ("b1", block.b1.detach().clone()),
                        ("b2", block.b2.detach().clone()), ("w1_codes", q1.codes), ("w1_scales", q1.scales),
                        ("w2_codes", q2.codes), ("w2_scales", q2.scales)):
            self.register_buffer(name, t)

    def forward(self, h):
        from .mx4 import MX4, mx4_linear, quantize_mx4
        if torch.is_grad_enabled() and h.requires_grad:
            raise RuntimeError("a quantized expert block has no gradients: evaluate it under torch.no_grad()")
        out = _without_autocast(self, h, self.router.dtype)
        if out is not None:
            return out
        rows = h.reshape(-1, h.shape[-1])
        weights, experts, _ = route_topk(rows @ self.router.T, self.k, normalize=self.normalize)
        groups = group_rows(experts, self.router.shape[0])
        y = mx4_linear(quantize_mx4(rows, groups), MX4(self.w1_codes, self.w1_scales, rows.shape[1]), self.b1, groups,
                       self.activation, rows.dtype)
        y = mx4_linear(quantize_mx4(y), MX4(self.w2_codes, self.w2_scales, self.hidden), self.b2, groups, None, rows.dtype)
        return combine_rows(y, groups, weights, residual=rows).view(h.shape)
