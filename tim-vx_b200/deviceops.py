"""Operators on torch tensors that are on the GPU already, over the ``*_noalloc`` entry points of include/b2vx.h.

    quantize_fp4 / dequantize_fp4   rows of numbers to 4-bit block floating point and back
    Fp4Weight                       4-bit weights of a layer or of its experts, laid out for the products
    linear                          y = x W^T + bias, W 4-bit (x is quantized on the way in) or 16-bit
    expert_linear                   the same for rows that belong to different experts, optionally gated
    route_experts                   which experts a token goes to, and the pairs sorted by expert
    combine_experts                 the weighted sum of each token's expert rows

Work is queued on the current stream of the tensors' device and nothing waits for it.  Outputs and workspaces come from torch's allocator
(give ``out`` for an output of your own; what quantize_fp4 and route_experts return shares one allocation).  Refused arguments raise pyb2vx.B2vxError with the library's message, tensors of a wrong type,
shape or device raise ValueError; nothing is launched then.  Tensors whose last dimension is contiguous are used where they
lie; a bias, scale or index tensor has to be contiguous.  ``out`` may be the residual of combine_experts, but must not overlap another input.
"""
import collections

import torch

import deviceops_native as _native

FORMATS = {"block32": 1, "block16": 2}
BLOCK = {"block32": 32, "block16": 16}

# codes uint8 [rows][(k rounded up to 32) / 2], scales uint8 [rows][blocks]; scale: the tensor's scale (block16) or None
Fp4Rows = collections.namedtuple("Fp4Rows", "codes scales k format scale")
Routes = collections.namedtuple("Routes", "ids weights offsets row_index slots")


def _format(name):
    if name not in FORMATS:
        raise ValueError("format must be one of %s" % ", ".join(FORMATS))
    return FORMATS[name]


def quantize_fp4(x, format="block32", scale=None, row_index=None):
    """Rows of x [rows][k] (float32, float16, bfloat16) as 4-bit codes with a scale per block.

    row_index (int32): the rows of x to take, in that order; an index outside x gives a row of zeros.
    scale (block16): one float32, the tensor's scale; amax / (6 * 448) uses e4m3's whole range."""
    codes, scales = _native.quantize(x, _format(format), scale, row_index)
    return Fp4Rows(codes, scales, x.shape[1], format, scale)


def dequantize_fp4(q, dtype=torch.float32, out=None):
    """The values of quantize_fp4's rows."""
    return _native.dequantize(q.codes, q.scales, q.k, _format(q.format), q.scale, dtype, out)


class Fp4Weight:
    """4-bit weights [n][k] or, of experts, [experts][n][k] as codes [..][n][k / 2] and scale bytes [..][n][k / block], whose scales are laid
    out for the products here, once.  The codes are used where they lie.

    scale (block16): float32, one for each matrix.  gated: the matrices are [2 n][k], gate rows first, n a multiple of 8."""

    def __init__(self, codes, scales, format="block32", scale=None, gated=False):
        self.code, self.gated = _format(format), bool(gated)
        if codes.dim() not in (2, 3) or codes.dtype != torch.uint8 or not codes.is_contiguous():
            raise ValueError("codes must be a dense uint8 tensor of two or three dimensions")
        rows, k = codes.shape[-2], codes.shape[-1] * 2
        if k % 32:
            raise ValueError("k must be a multiple of 32")
        if gated and rows % 16:
            raise ValueError("the rows of a gated weight must be a multiple of 16")
        if tuple(scales.shape) != tuple(codes.shape[:-1]) + (k // BLOCK[format],) or scales.device != codes.device:
            raise ValueError("scales must have the shape %s on the codes' device" % (tuple(codes.shape[:-1]) + (k // BLOCK[format],),))
        if (scale is not None) != (format == "block16"):
            raise ValueError("scale belongs to block16 and only to it")
        self.codes, self.scale, self.format = codes, scale, format
        self.packed = _native.pack(scales.reshape(codes.shape[0] if codes.dim() == 3 else 1, rows, k // BLOCK[format]), self.code, self.gated)


def _product(x, weight, offsets, row_index, bias, gated, x_scale, out_dtype, out):
    if isinstance(weight, Fp4Weight):
        if weight.gated != bool(gated):
            raise ValueError("the weight was laid out for gated=%s" % weight.gated)
        return _native.product(x, weight.codes, weight.packed, weight.scale, weight.code, gated, offsets, row_index, bias, x_scale, out_dtype, out)
    return _native.product(x, weight, None, None, 0, gated, offsets, row_index, bias, x_scale, out_dtype, out)


def linear(x, weight, bias=None, x_scale=None, out_dtype=None, out=None):
    """y [rows][n] = x [rows][k] W^T + bias.

    weight: Fp4Weight (x is quantized to its format; block16: with the tensor's scale x_scale), or a dense tensor [n][k] of x's 16-bit type.
    bias: float32 [n].  out_dtype: float32, float16 or bfloat16 (x's)."""
    return _product(x, weight, None, None, bias, False, x_scale, out_dtype, out)


def expert_linear(x, weight, offsets, row_index=None, bias=None, gated=False, x_scale=None, out_dtype=None, out=None):
    """y [rows][n]: row m, of expert e with offsets[e] <= m < offsets[e + 1], is x[row_index[m]] W_e^T + bias_e.

    weight: Fp4Weight or dense tensor [experts][n][k].  offsets: int32 [experts + 1], on the GPU.  row_index: int32 [rows] or None (x's own
    rows).  gated: W_e is [2 n][k] and the result silu(of its first half) * (of its second).  bias: float32 [experts][rows of W_e].
    Rows that no expert has are left as they are in ``out`` (without ``out``, undefined)."""
    return _product(x, weight, offsets, row_index, bias, gated, x_scale, out_dtype, out)


def route_experts(logits, top_k, normalize=True):
    """The top_k experts of each row of logits [tokens][experts] and the pairs (token, choice) sorted by expert.

    ids int32, weights float32 [tokens][top_k], largest logit first, ties to the lowest index; normalize: weights over the chosen experts
    instead of all.  offsets int32 [experts + 1], row_index int32 [tokens * top_k]: the token of each sorted row,
    slots int32 [tokens][top_k]: the sorted row of each pair."""
    return Routes(*_native.route(logits, top_k, normalize))


def combine_experts(z, slots, weights, residual=None, out=None):
    """y[t] = residual[t] + sum_j weights[t][j] z[slots[t][j]], summed in float32 and rounded once; a slot outside z adds nothing."""
    return _native.combine(z, slots, weights, residual, out)


def check(device=None):
    """Waits for the current stream of a GPU (the current one, unless device names another); raises where a product there gave up on a barrier."""
    index = None if device is None else torch.device(device).index
    _native.check(torch.cuda.current_device() if index is None else index)
