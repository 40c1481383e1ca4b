"""The b2vx_*_noalloc entry points of the operators on device tensors through ctypes, for tests that pass what torch tensors cannot."""
import ctypes as C

import pyb2vx

_vp, _u64, _u32, _i32, _sz = C.c_void_p, C.c_uint64, C.c_uint32, C.c_int32, C.c_size_t


class QuantizeDesc(C.Structure):
    _fields_ = [("format", _i32), ("x_dtype", _i32), ("x_rows", _u64), ("rows", _u64), ("k", _u64), ("x_stride", _u64),
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
    "b2vx_fp4_packed_scales_size_noalloc": [_i32, _u64, _u64, _i32, _u64, C.POINTER(_sz)],
    "b2vx_fp4_pack_scales_noalloc": [_i32, _u64, _u64, _i32, _u64, _vp, _vp, _vp] + _err,
    "b2vx_linear_workspace_size_noalloc": [C.POINTER(LinearDesc), C.POINTER(_sz)] + _err,
    "b2vx_linear_in_place_noalloc": [C.POINTER(LinearDesc), C.POINTER(LinearArgs)],
    "b2vx_linear_noalloc": [C.POINTER(LinearDesc), C.POINTER(LinearArgs), _vp] + _err,
    "b2vx_route_workspace_size_noalloc": [C.POINTER(RouteDesc), C.POINTER(_sz)] + _err,
    "b2vx_route_noalloc": [C.POINTER(RouteDesc)] + [_vp] * 7 + [_sz, _vp] + _err,
    "b2vx_combine_noalloc": [C.POINTER(CombineDesc)] + [_vp] * 6 + _err,
    "b2vx_device_check_noalloc": [_vp] + _err,
}
_lib = None


def library():
    """The product library with these entry points declared."""
    global _lib
    if _lib is None:
        lib = C.CDLL(pyb2vx.PRODUCT_LIB)
        for name, args in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = _i32
            fn.argtypes = args
        _lib = lib
    return _lib


def call(fn, *args):
    err = C.create_string_buffer(256)
    st = fn(*args, err, 256)
    if st:
        raise pyb2vx.B2vxError(st, err.value.decode())
