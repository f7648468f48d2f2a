"""Microscaled 4-bit floating point on the HIP library (dimo_amd/csrc/mx4.hip): quantisation and products for networks
that are only evaluated (render-only use, ExpertMLP.quantized()).

    x4 = quantize_mx4(x)                     # e2m1 elements, one power-of-two scale per 32 values along the last axis
    w4 = quantize_mx4(weight)                # once, when the weights are final
    y = mx4_linear(x4, w4, bias)             # [R, K] x [N, K] -> [R, N]; or grouped: w4 [E, N, K], groups=RowGroups

Products of the quantised values are exact and summed in fp32, so what an `mx4_linear` loses against the product of its
inputs is what `quantize_mx4` rounded.  That is bounded against the block's scale s, not against the element: s / 4 up to 2 s,
s / 2 up to 4 s, s up to 6 s, and |x| - 6 s (below 2 s) beyond, where elements saturate -- at most a quarter of the block's
largest magnitude, and all of an element below s / 4.  No gradients.  GPU only."""
import torch

from . import _lib
from .experts import _ACTIVATIONS, _DTYPES, _check_linear_groups, _check_sizes, _dtype, _gpu, _ld, _on, _refuse_tangents, _rows


class MX4:
    """Values in microscaled 4-bit form.  codes uint8 [..., 16 ceil(K / 32)]: two e2m1 codes to a byte, low four bits
    first; scales uint8 [..., ceil(K / 32)]: 2^(byte - 127), 255 = NaN; columns: K (what lies behind it in the last block
    counts as zero: the codes there have to be 0 or 8)."""

    __slots__ = ("codes", "scales", "columns")

    def __init__(self, codes, scales, columns):
        blocks = -(-columns // 32)
        if columns < 1 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("uint8 codes and scales and at least one column expected")
        if codes.shape[-1] != 16 * blocks or scales.shape[-1] != blocks or codes.shape[:-1] != scales.shape[:-1]:
            raise ValueError(f"{columns} columns: codes [..., {16 * blocks}] and scales [..., {blocks}] expected")
        if codes.device != scales.device:
            raise ValueError("codes and scales on different devices")
        codes, scales = codes.contiguous(), scales.contiguous()
        self.codes, self.scales, self.columns = codes if codes.data_ptr() % 16 == 0 else codes.clone(), scales, columns

    @property
    def shape(self):
        return self.codes.shape[:-1] + (self.columns,)

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32):
        """The values, in fp32, bf16 or fp16 (in bf16 and fp32 exactly, in fp16 where its range allows)."""
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        _gpu(out)
        _dtype(out, "dequantize")
        with _on(self.device):
            _lib.check(_lib.lib().dimo_mx4_dequantize(_DTYPES[dtype], out.numel() // self.columns, self.columns,
                                                      self.codes.data_ptr(), self.scales.data_ptr(), out.data_ptr(),
                                                      _lib.current_stream()), "dimo_mx4_dequantize")
        return out


def quantize_mx4(x, groups=None):
    """MX4 of x [..., K], block by block of 32 along the last axis: scale 2^(floor(log2 max|x|) - 2), elements to the
    nearest e2m1 value (ties to the even code, larger ones to 6); a block with an infinite or NaN value is NaN as a whole.
    groups (from group_rows): x [T, K] is read through the grouping, the result is [T k, K] in the order of the groups
    (zeros behind the last one)."""
    _gpu(x)
    _refuse_tangents(x)
    dtype = _dtype(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x: [..., K] with K >= 1 expected")
    _check_sizes(x.shape[-1])
    x = x.detach()
    K, lead = x.shape[-1], x.shape[:-1]
    flat = _rows(x) if x.dim() == 2 else x.contiguous().view(-1, K)
    rows, source = flat.shape[0], None
    if groups is not None:
        if groups.position is None or x.dim() != 2 or x.shape[0] != groups.position.shape[0]:
            raise ValueError("groups of these rows, made by group_rows, expected")
        _gpu(x, groups.order)
        rows, source = groups.rows.shape[0], groups.rows
        lead = (rows,)
    blocks = -(-K // 32)
    codes = torch.empty(*lead, 16 * blocks, dtype=torch.uint8, device=x.device)
    scales = torch.empty(*lead, blocks, dtype=torch.uint8, device=x.device)
    with _on(x.device):
        _lib.check(_lib.lib().dimo_mx4_quantize(dtype, rows, K, flat.data_ptr(), _ld(flat), _lib.ptr(source),
                                                codes.data_ptr(), scales.data_ptr(), _lib.current_stream()),
                   "dimo_mx4_quantize")
    return MX4(codes, scales, K)


def mx4_linear(x, weight, bias=None, groups=None, activation=None, out_dtype=torch.bfloat16):
    """y[r] = activation(weight[e] @ x[r] + bias[e]) of MX4 x [R, K] and MX4 weight: [N, K] for all rows, or [E, N, K] with
    `groups` (RowGroups of the R rows; zeros behind the last group).  bias [N] or [E, N] in the result's type."""
    if len(x.shape) != 2 or len(weight.shape) != (2 if groups is None else 3):
        raise ValueError("x: [R, K]; weight: [N, K], or [E, N, K] with groups expected")
    if weight.columns != x.columns:
        raise ValueError(f"x has {x.columns} columns, weight takes {weight.columns}")
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype: fp32, bf16 or fp16 expected, got {out_dtype}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation: one of {list(_ACTIVATIONS)} expected")
    R, N, E = x.shape[0], weight.shape[-2], 1
    if N < 1:
        raise ValueError("weight without rows")
    _check_sizes(R, N, x.columns)
    _refuse_tangents(bias)
    _gpu(x.codes, weight.codes, bias, None if groups is None else groups.offsets)
    if groups is not None:
        E = weight.shape[0]
        _check_linear_groups(E, R, groups)
    if bias is not None:
        if bias.dtype != out_dtype or bias.shape != ((N,) if groups is None else (E, N)):
            raise ValueError("bias: one value per output column, of the result's type, expected")
        bias = bias.contiguous()
    y = torch.empty(R, N, dtype=out_dtype, device=x.device)
    with _on(x.device):
        _lib.check(_lib.lib().dimo_mx4_linear(
            _DTYPES[out_dtype], R, E, x.columns, N, x.codes.data_ptr(), x.scales.data_ptr(),
            None if groups is None else groups.offsets.data_ptr(), weight.codes.data_ptr(), weight.scales.data_ptr(),
            _lib.ptr(bias), _ACTIVATIONS[activation], y.data_ptr(), _lib.current_stream()), "dimo_mx4_linear")
    return y
