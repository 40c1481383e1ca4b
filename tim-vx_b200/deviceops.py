"""Operators on torch tensors that are on the GPU already, over the ``*_noalloc`` entry points of include/b2vx.h.

    quantize_fp4 / dequantize_fp4   rows of numbers to 4-bit block floating point and back
    Fp4Weight                       4-bit weights of a layer or of its experts, laid out for the products
    linear                          y = x W^T + bias, W 4-bit (x is quantized on the way in) or 16-bit
    expert_linear                   the same for rows that belong to different experts, optionally gated
    route_experts                   which experts a token goes to, and the pairs sorted by expert
    combine_experts                 the weighted sum of each token's expert rows

Work is queued on the current stream of the tensors' device and nothing waits for it.  Outputs and workspaces come from torch's allocator
(give ``out`` for an output of your own).  Refused arguments raise pyb2vx.B2vxError with the library's message, tensors of a wrong type,
shape or device raise ValueError; nothing is launched then.  Tensors whose last dimension is contiguous are used where they
lie; a bias, scale or index tensor has to be contiguous.
"""
import collections
import ctypes as C

import torch

import pyb2vx

FORMATS = {"block32": 1, "block16": 2}
BLOCK = {"block32": 32, "block16": 16}
_DT = {torch.float32: 9, torch.float16: 8, torch.bfloat16: 16}
MAX_EXPERTS = 1024

_vp, _u64, _u32, _i32, _sz = C.c_void_p, C.c_uint64, C.c_uint32, C.c_int32, C.c_size_t


class QuantizeDesc(C.Structure):
    _fields_ = [("format", _i32), ("scales_layout", _i32), ("x_dtype", _i32), ("x_rows", _u64), ("rows", _u64), ("k", _u64), ("x_stride", _u64),
                ("codes_pitch", _u64), ("scales_pitch", _u64)]


class DequantizeDesc(C.Structure):
    _fields_ = [("format", _i32), ("y_dtype", _i32), ("rows", _u64), ("k", _u64), ("codes_pitch", _u64), ("scales_pitch", _u64), ("y_stride", _u64)]


class LinearDesc(C.Structure):
    _fields_ = [("w_format", _i32), ("x_dtype", _i32), ("y_dtype", _i32), ("gated", _i32), ("experts", _u32), ("x_rows", _u64), ("rows", _u64),
                ("n", _u64), ("k", _u64), ("x_stride", _u64), ("y_stride", _u64)]


class LinearArgs(C.Structure):
    _fields_ = [("x", _vp), ("w", _vp), ("w_scales", _vp), ("x_scale", _vp), ("w_scale", _vp), ("bias", _vp), ("offsets", _vp), ("row_index", _vp),
                ("y", _vp), ("workspace", _vp), ("workspace_bytes", _sz)]


class RouteDesc(C.Structure):
    _fields_ = [("logits_dtype", _i32), ("normalize", _i32), ("experts", _u32), ("top_k", _u32), ("tokens", _u64), ("logits_stride", _u64)]


class CombineDesc(C.Structure):
    _fields_ = [("dtype", _i32), ("top_k", _u32), ("tokens", _u64), ("n", _u64), ("z_rows", _u64), ("z_stride", _u64), ("residual_stride", _u64),
                ("y_stride", _u64)]


_err = [C.c_char_p, _sz]
_SIGNATURES = {
    "b2vx_fp4_quantize_noalloc": [C.POINTER(QuantizeDesc), _vp, _vp, _vp, _vp, _vp, _vp] + _err,
    "b2vx_fp4_dequantize_noalloc": [C.POINTER(DequantizeDesc), _vp, _vp, _vp, _vp, _vp] + _err,
    "b2vx_fp4_packed_scales_size_noalloc": [_i32, _u64, _u64, _u64, C.POINTER(_sz)],
    "b2vx_fp4_pack_scales_noalloc": [_i32, _u64, _u64, _u64, _vp, _vp, _vp] + _err,
    "b2vx_linear_workspace_size_noalloc": [C.POINTER(LinearDesc), C.POINTER(_sz)] + _err,
    "b2vx_linear_noalloc": [C.POINTER(LinearDesc), C.POINTER(LinearArgs), _vp] + _err,
    "b2vx_route_workspace_size_noalloc": [C.POINTER(RouteDesc), C.POINTER(_sz)] + _err,
    "b2vx_route_noalloc": [C.POINTER(RouteDesc)] + [_vp] * 7 + [_sz, _vp] + _err,
    "b2vx_combine_noalloc": [C.POINTER(CombineDesc)] + [_vp] * 6 + _err,
    "b2vx_device_check_noalloc": [_vp] + _err,
}
_lib = None


def library():
    """The product library with these entry points declared; raises where it is not built."""
    global _lib
    if _lib is None:
        lib = C.CDLL(pyb2vx.PRODUCT_LIB)
        for name, args in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = _i32
            fn.argtypes = args
        _lib = lib
    return _lib


def _call(fn, *args):
    err = C.create_string_buffer(256)
    st = fn(*args, err, 256)
    if st:
        raise pyb2vx.B2vxError(st, err.value.decode())


def _need(cond, message):
    if not cond:
        raise ValueError(message)


def _rows(t, what, dtypes=_DT):
    _need(isinstance(t, torch.Tensor) and t.dim() == 2, "%s must be a tensor of two dimensions" % what)
    _need(t.dtype in dtypes, "%s has type %s" % (what, t.dtype))
    _need(t.stride(1) == 1 or t.shape[1] <= 1, "%s must be contiguous along its last dimension" % what)
    return max(t.stride(0), t.shape[1])


def _dense(t, what, dtype, shape, device):
    """The address of an optional dense tensor."""
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and t.dtype == dtype, "%s must be a tensor of %s" % (what, dtype))
    _need(tuple(t.shape) == tuple(shape), "%s must have the shape %s, not %s" % (what, tuple(shape), tuple(t.shape)))
    _need(t.is_contiguous(), "%s must be contiguous" % what)
    _need(t.device == device, "%s is on another device" % what)
    return t.data_ptr()


def _out(out, shape, dtype, device):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _rows(out, "out")
    _need(tuple(out.shape) == tuple(shape) and out.device == device, "out must have the shape %s on %s" % (tuple(shape), device))
    _need(out.shape[0] <= 1 or out.stride(0) >= out.shape[1], "out has rows that overlap")
    return out


class _On:
    """The device of a call as the current one, and its current stream."""

    def __init__(self, device):
        _need(device.type == "cuda", "tensors must be on a GPU")
        self.device = device

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.device.index != self.before:
            torch.cuda.set_device(self.device)
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.device.index != self.before:
            torch.cuda.set_device(self.before)


# codes uint8 [rows][(k rounded up to 32) / 2], scales uint8 [rows][blocks]; scale: the tensor's scale (block16) or None
Fp4Rows = collections.namedtuple("Fp4Rows", "codes scales k format scale")


def _scale(scale, format, count, device, what):
    _need(format in FORMATS, "format must be one of %s" % ", ".join(FORMATS))
    _need((scale is not None) == (format == "block16"), "%s belongs to block16 and only to it" % what)
    return _dense(scale.reshape(-1) if isinstance(scale, torch.Tensor) else scale, what, torch.float32, (count,), device)


def quantize_fp4(x, format="block32", scale=None, row_index=None):
    """Rows of x [rows][k] (float32, float16, bfloat16) as 4-bit codes with a scale per block.

    row_index (int32): the rows of x to take, in that order; an index outside x gives a row of zeros.
    scale (block16): one float32, the tensor's scale; amax / (6 * 448) uses e4m3's whole range."""
    stride = _rows(x, "x")
    rows, k = x.shape[0] if row_index is None else row_index.numel(), x.shape[1]
    scale_ptr = _scale(scale, format, 1, x.device, "scale")
    index = _dense(row_index, "row_index", torch.int32, (rows,), x.device)
    codes = torch.empty(rows, (k + 31) // 32 * 16, dtype=torch.uint8, device=x.device)
    scales = torch.empty(rows, -(-k // BLOCK[format]), dtype=torch.uint8, device=x.device)
    d = QuantizeDesc(FORMATS[format], 0, _DT[x.dtype], x.shape[0], rows, k, stride, codes.shape[1], scales.shape[1])
    with _On(x.device) as stream:
        _call(library().b2vx_fp4_quantize_noalloc, C.byref(d), x.data_ptr(), index, scale_ptr, codes.data_ptr(), scales.data_ptr(), stream)
    return Fp4Rows(codes, scales, k, format, scale)


def dequantize_fp4(q, dtype=torch.float32, out=None):
    """The values of quantize_fp4's rows."""
    device = q.codes.device
    rows = q.codes.shape[0]
    _need(dtype in _DT, "dtype must be float32, float16 or bfloat16")
    codes = _dense(q.codes, "codes", torch.uint8, (rows, (q.k + 31) // 32 * 16), device)
    scale_ptr = _scale(q.scale, q.format, 1, device, "scale")
    scales = _dense(q.scales, "scales", torch.uint8, (rows, -(-q.k // BLOCK[q.format])), device)
    y = _out(out, (rows, q.k), dtype, device)
    d = DequantizeDesc(FORMATS[q.format], _DT[y.dtype], rows, q.k, q.codes.shape[1], q.scales.shape[1], max(y.stride(0), q.k))
    with _On(device) as stream:
        _call(library().b2vx_fp4_dequantize_noalloc, C.byref(d), codes, scales, scale_ptr, y.data_ptr(), stream)
    return y


class Fp4Weight:
    """4-bit weights [n][k] or, of experts, [experts][n][k] as codes [..][n][k / 2] and scale bytes [..][n][k / block], whose scales are laid
    out for the products here, once.  The codes are used where they lie.

    scale (block16): float32, one for each matrix.  gated: the matrices are [2 n][k], gate rows first."""

    def __init__(self, codes, scales, format="block32", scale=None, gated=False):
        _need(codes.dim() in (2, 3) and codes.dtype == torch.uint8 and codes.is_contiguous(), "codes must be a dense uint8 tensor of two or three dimensions")
        self.experts = codes.shape[0] if codes.dim() == 3 else 0
        self.rows, self.k, self.format, self.gated = codes.shape[-2], codes.shape[-1] * 2, format, bool(gated)
        _need(self.k % 32 == 0, "k must be a multiple of 32")
        _need(not gated or self.rows % 2 == 0, "a gated weight has an even number of rows")
        count = max(1, self.experts)
        self.scale_ptr = _scale(scale, format, count, codes.device, "scale")
        src = _dense(scales, "scales", torch.uint8, tuple(codes.shape[:-1]) + (self.k // BLOCK[format],), codes.device)
        self.codes, self.scale, self.device = codes, scale, codes.device
        parts = 2 if gated else 1
        size = _sz()
        st = library().b2vx_fp4_packed_scales_size_noalloc(FORMATS[format], count * parts, self.rows // parts, self.k, C.byref(size))
        if st:
            raise pyb2vx.B2vxError(st, "weights out of range")
        self.packed = torch.empty(max(16, size.value), dtype=torch.uint8, device=codes.device)
        with _On(codes.device) as stream:
            _call(library().b2vx_fp4_pack_scales_noalloc, FORMATS[format], count * parts, self.rows // parts, self.k, src, self.packed.data_ptr(), stream)


def _product(x, weight, offsets, row_index, bias, gated, x_scale, out_dtype, out):
    stride = _rows(x, "x")
    rows = x.shape[0] if row_index is None else row_index.numel()
    fp4 = isinstance(weight, Fp4Weight)
    if fp4:
        experts, w_rows, k, fmt = weight.experts, weight.rows, weight.k, FORMATS[weight.format]
        _need(weight.gated == bool(gated), "the weight was laid out for gated=%s" % weight.gated)
        _need(weight.device == x.device, "the weight is on another device")
        w, w_scales, w_scale = weight.codes.data_ptr(), weight.packed.data_ptr(), weight.scale_ptr
        x_scale_ptr = _scale(x_scale, weight.format, 1, x.device, "x_scale")
    else:
        _need(isinstance(weight, torch.Tensor) and weight.dim() in (2, 3) and weight.dtype == x.dtype and weight.device == x.device,
              "weight must be an Fp4Weight or a tensor of x's type and device with two or three dimensions")
        _need(weight.is_contiguous(), "weight must be contiguous")
        _need(x_scale is None, "x_scale belongs to block16 and only to it")
        experts, w_rows, k, fmt = weight.shape[0] if weight.dim() == 3 else 0, weight.shape[-2], weight.shape[-1], 0
        _need(not gated or w_rows % 2 == 0, "a gated weight has an even number of rows")
        w, w_scales, w_scale, x_scale_ptr = weight.data_ptr(), None, None, None
    _need((offsets is not None) == (experts > 0), "offsets belong to weights of experts and only to them")
    _need(x.shape[1] == k, "x has %d columns, the weight %d" % (x.shape[1], k))
    n = w_rows // 2 if gated else w_rows
    index = _dense(row_index, "row_index", torch.int32, (rows,), x.device)
    starts = _dense(offsets, "offsets", torch.int32, (experts + 1,), x.device)
    b = _dense(bias, "bias", torch.float32, (experts, w_rows) if experts else (w_rows,), x.device)
    y = _out(out, (rows, n), out_dtype or x.dtype, x.device)
    _need(y.dtype in _DT, "the output must be float32, float16 or bfloat16")
    d = LinearDesc(fmt, _DT[x.dtype], _DT[y.dtype], int(bool(gated)), experts, x.shape[0], rows, n, k, stride, max(y.stride(0), n))
    lib = library()
    with _On(x.device) as stream:
        size = _sz()
        _call(lib.b2vx_linear_workspace_size_noalloc, C.byref(d), C.byref(size))
        workspace = torch.empty(size.value + 256, dtype=torch.uint8, device=x.device)
        at = -workspace.data_ptr() % 256
        a = LinearArgs(x.data_ptr(), w, w_scales, x_scale_ptr, w_scale, b, starts, index, y.data_ptr(), workspace.data_ptr() + at, size.value)
        _call(lib.b2vx_linear_noalloc, C.byref(d), C.byref(a), stream)
    return y


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


Routes = collections.namedtuple("Routes", "ids weights offsets row_index slots")


def route_experts(logits, top_k, normalize=True):
    """The top_k experts of each row of logits [tokens][experts] and the pairs (token, choice) sorted by expert.

    ids int32, weights float32 [tokens][top_k], largest logit first, ties to the lowest index; normalize: weights over the chosen experts
    instead of all.  offsets int32 [experts + 1], row_index int32 [tokens * top_k]: the token of each sorted row,
    slots int32 [tokens][top_k]: the sorted row of each pair."""
    stride = _rows(logits, "logits")
    tokens, experts = logits.shape
    dev = logits.device
    d = RouteDesc(_DT[logits.dtype], int(bool(normalize)), experts, top_k, tokens, stride)
    lib = library()
    size = _sz()
    _call(lib.b2vx_route_workspace_size_noalloc, C.byref(d), C.byref(size))
    ids = torch.empty(tokens, top_k, dtype=torch.int32, device=dev)
    weights = torch.empty(tokens, top_k, dtype=torch.float32, device=dev)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    row_index = torch.empty(tokens * top_k, dtype=torch.int32, device=dev)
    slots = torch.empty(tokens, top_k, dtype=torch.int32, device=dev)
    with _On(dev) as stream:
        workspace = torch.empty(size.value + 256, dtype=torch.uint8, device=dev)
        at = -workspace.data_ptr() % 256
        _call(lib.b2vx_route_noalloc, C.byref(d), logits.data_ptr(), ids.data_ptr(), weights.data_ptr(), offsets.data_ptr(), row_index.data_ptr(),
              slots.data_ptr(), workspace.data_ptr() + at, size.value, stream)
    return Routes(ids, weights, offsets, row_index, slots)


def combine_experts(z, slots, weights, residual=None, out=None):
    """y[t] = residual[t] + sum_j weights[t][j] z[slots[t][j]], summed in float32 and rounded once; a slot outside z adds nothing."""
    stride = _rows(z, "z")
    _need(isinstance(slots, torch.Tensor) and slots.dim() == 2, "slots must be a tensor of two dimensions")
    tokens, top_k = slots.shape
    s = _dense(slots, "slots", torch.int32, (tokens, top_k), z.device)
    w = _dense(weights, "weights", torch.float32, (tokens, top_k), z.device)
    n = z.shape[1]
    r_stride = 0
    if residual is not None:
        r_stride = _rows(residual, "residual", (z.dtype,))
        _need(tuple(residual.shape) == (tokens, n) and residual.device == z.device, "residual must have the shape (%d, %d) on z's device" % (tokens, n))
    y = _out(out, (tokens, n), z.dtype, z.device)
    _need(y.dtype == z.dtype, "out must have z's type")
    d = CombineDesc(_DT[z.dtype], top_k, tokens, n, z.shape[0], stride, r_stride, max(y.stride(0), n))
    with _On(z.device) as stream:
        _call(library().b2vx_combine_noalloc, C.byref(d), z.data_ptr(), s, w, None if residual is None else residual.data_ptr(), y.data_ptr(), stream)
    return y


def check(device=None):
    """Waits for the current stream; raises where a product on that GPU gave up on a barrier."""
    with _On(torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)) as stream:
        _call(library().b2vx_device_check_noalloc, stream)
