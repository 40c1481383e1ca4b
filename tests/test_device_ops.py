"""Refusals of the operators on device tensors, and the sizes they tell: host-side rules, no GPU needed.

Every refusal comes before the first CUDA call, so the pointers here are only numbers."""
import ctypes as C
import os
import re
import subprocess
import sys

import pytest

import device_ops_abi as ABI
import deviceops as D
import pyb2vx

PTR = 1 << 20   # an address that is aligned to everything; never read


def desc(cls, base, **change):
    d = cls()
    for name, value in dict(base, **change).items():
        setattr(d, name, value)
    return d


QUANTIZE = dict(format=1, x_dtype=16, x_rows=8, rows=8, k=96, x_stride=96, codes_pitch=48, scales_pitch=3)
DEQUANTIZE = dict(format=1, y_dtype=16, rows=8, k=96, codes_pitch=48, scales_pitch=3, y_stride=96)
LINEAR = dict(w_format=1, x_dtype=16, y_dtype=16, gated=0, experts=0, x_rows=8, rows=8, n=64, k=96, x_stride=96, y_stride=64)
ROUTE = dict(logits_dtype=9, normalize=1, experts=16, top_k=4, tokens=200, logits_stride=16)
COMBINE = dict(dtype=16, top_k=2, tokens=8, n=64, z_rows=16, z_stride=64, residual_stride=64, y_stride=64)


def refused(fn, *args):
    err = C.create_string_buffer(256)
    st = fn(*args, err, 256)
    assert st == 1, (st, err.value)
    assert err.value
    assert fn(*args, None, 0) == 1      # without a place for the message
    return err.value.decode()


@pytest.mark.parametrize("change,scale,words", [
    (dict(format=0), None, "format"), (dict(format=3), None, "format"), (dict(x_dtype=2), None, "float32"),
    (dict(k=1 << 30), None, "range"), (dict(rows=1 << 30), None, "range"), (dict(x_stride=95), None, "x_stride"), (dict(x_stride=1 << 41), None, "x_stride"),
    (dict(codes_pitch=44), None, "codes_pitch"), (dict(codes_pitch=49), None, "codes_pitch"), (dict(scales_pitch=2), None, "scales_pitch"),
    (dict(format=2, scales_pitch=6), None, "tensor scale"), (dict(), PTR, "tensor scale"), (dict(rows=9), None, "row_index")])
def test_quantize_refuses(change, scale, words):
    fn = ABI.library().b2vx_fp4_quantize_noalloc
    assert words in refused(fn, C.byref(desc(ABI.QuantizeDesc, QUANTIZE, **change)), PTR, None, scale, PTR, PTR, None)


def test_quantize_refuses_pointers():
    fn = ABI.library().b2vx_fp4_quantize_noalloc
    d = C.byref(desc(ABI.QuantizeDesc, QUANTIZE))
    assert "null" in refused(fn, None, PTR, None, None, PTR, PTR, None)
    for args in ((None, None, None, PTR, PTR, None), (PTR, None, None, None, PTR, None), (PTR, None, None, PTR, None, None)):
        assert "null" in refused(fn, d, *args)
    assert "aligned" in refused(fn, d, PTR + 1, None, None, PTR, PTR, None)
    assert "aligned" in refused(fn, d, PTR, None, None, PTR + 2, PTR, None)


@pytest.mark.parametrize("change,scale,words", [
    (dict(format=0), None, "format"), (dict(y_dtype=1), None, "float32"), (dict(rows=1 << 30), None, "range"), (dict(codes_pitch=40), None, "codes_pitch"),
    (dict(scales_pitch=1), None, "scales_pitch"), (dict(y_stride=95), None, "y_stride"), (dict(format=2, scales_pitch=6), None, "tensor scale"),
    (dict(), PTR, "tensor scale")])
def test_dequantize_refuses(change, scale, words):
    fn = ABI.library().b2vx_fp4_dequantize_noalloc
    assert words in refused(fn, C.byref(desc(ABI.DequantizeDesc, DEQUANTIZE, **change)), PTR, PTR, scale, PTR, None)


def test_dequantize_refuses_pointers():
    fn = ABI.library().b2vx_fp4_dequantize_noalloc
    d = C.byref(desc(ABI.DequantizeDesc, DEQUANTIZE))
    for args in ((None, PTR, None, PTR, None), (PTR, None, None, PTR, None), (PTR, PTR, None, None, None)):
        assert "null" in refused(fn, d, *args)
    assert "aligned" in refused(fn, d, PTR, PTR, None, PTR + 1, None)


@pytest.mark.parametrize("change,words", [
    (dict(w_format=4), "w_format"), (dict(x_dtype=1), "float32"), (dict(y_dtype=2), "float32"), (dict(w_format=0, x_dtype=9), "16-bit"),
    (dict(gated=2), "gated"), (dict(gated=1, n=60), "gated"), (dict(experts=1025), "1024"), (dict(n=1 << 30), "range"), (dict(k=0, x_stride=0), "zero"), (dict(k=100, x_stride=100), "multiple"),
    (dict(w_format=0, k=100, x_stride=100), "multiple"), (dict(x_stride=95), "x_stride"), (dict(y_stride=63), "y_stride"),
    (dict(rows=1 << 28, x_rows=1 << 28, n=1 << 20, y_stride=1 << 20), "tiles"), (dict(n=1 << 28, y_stride=1 << 28), "range"),
    (dict(experts=1024, n=1 << 22, k=1 << 16, x_stride=1 << 16, y_stride=1 << 22), "tiles")])
def test_linear_refuses(change, words):
    size = C.c_size_t()
    d = desc(ABI.LinearDesc, LINEAR, **change)
    assert words in refused(ABI.library().b2vx_linear_workspace_size_noalloc, C.byref(d), C.byref(size))
    args = ABI.LinearArgs(PTR, PTR, PTR, None, None, None, None, None, PTR, PTR, 1 << 30)
    assert words in refused(ABI.library().b2vx_linear_noalloc, C.byref(d), C.byref(args), None)


@pytest.mark.parametrize("change,args,words", [
    (dict(), dict(offsets=PTR), "offsets"), (dict(experts=4), dict(), "offsets"), (dict(w_format=2), dict(), "tensor scales"),
    (dict(w_format=2), dict(x_scale=PTR), "tensor scales"), (dict(), dict(w_scale=PTR), "tensor scales"), (dict(rows=9), dict(), "row_index"),
    (dict(), dict(x=None), "null"), (dict(), dict(w=None), "null"), (dict(), dict(y=None), "null"), (dict(), dict(w_scales=None), "null"),
    (dict(), dict(w=PTR + 8), "aligned"), (dict(), dict(w_scales=PTR + 8), "aligned"), (dict(), dict(y=PTR + 1), "aligned"), (dict(), dict(x=PTR + 1), "aligned"),
    (dict(), dict(workspace=None), "workspace"), (dict(), dict(workspace=PTR + 16), "workspace"), (dict(), dict(workspace_bytes=100), "workspace"),
    (dict(w_format=0), dict(row_index=PTR, workspace_bytes=0), "workspace"), (dict(w_format=0, x_stride=100), dict(workspace=None), "workspace")])
def test_linear_refuses_arguments(change, args, words):
    d = desc(ABI.LinearDesc, LINEAR, **change)
    a = desc(ABI.LinearArgs, dict(x=PTR, w=PTR, w_scales=PTR, y=PTR, workspace=PTR, workspace_bytes=1 << 30), **args)
    assert words in refused(ABI.library().b2vx_linear_noalloc, C.byref(d), C.byref(a), None)


@pytest.mark.parametrize("change,words", [
    (dict(experts=0), "experts"), (dict(experts=1025, logits_stride=1025), "experts"), (dict(top_k=0), "top_k"), (dict(top_k=17), "top_k"),
    (dict(experts=64, logits_stride=64, top_k=33), "top_k"), (dict(tokens=1 << 29), "tokens"), (dict(logits_dtype=1), "float32"), (dict(normalize=2), "normalize"),
    (dict(logits_stride=15), "logits_stride")])
def test_route_refuses(change, words):
    d = C.byref(desc(ABI.RouteDesc, ROUTE, **change))
    assert words in refused(ABI.library().b2vx_route_noalloc, d, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 1 << 30, None)


def test_route_refuses_pointers():
    fn, d = ABI.library().b2vx_route_noalloc, C.byref(desc(ABI.RouteDesc, ROUTE))
    for i in range(6):
        args = [PTR] * 6
        args[i] = None
        assert "null" in refused(fn, d, *args, PTR, 1 << 20, None)
    assert "workspace" in refused(fn, d, *[PTR] * 6, None, 1 << 20, None)
    assert "workspace" in refused(fn, d, *[PTR] * 6, PTR + 8, 1 << 20, None)
    assert "workspace" in refused(fn, d, *[PTR] * 6, PTR, 8, None)
    assert "aligned" in refused(fn, d, PTR + 2, *[PTR] * 5, PTR, 1 << 20, None)


@pytest.mark.parametrize("change,words", [
    (dict(dtype=2), "float32"), (dict(tokens=1 << 30), "range"), (dict(z_stride=63), "stride"), (dict(y_stride=63), "stride"), (dict(residual_stride=63), "stride"),
    (dict(z_stride=1 << 41), "stride")])
def test_combine_refuses(change, words):
    d = C.byref(desc(ABI.CombineDesc, COMBINE, **change))
    assert words in refused(ABI.library().b2vx_combine_noalloc, d, PTR, PTR, PTR, PTR, PTR, None)


def test_combine_refuses_pointers():
    fn, d = ABI.library().b2vx_combine_noalloc, C.byref(desc(ABI.CombineDesc, COMBINE))
    for args in ((None, PTR, PTR, PTR, PTR), (PTR, None, PTR, PTR, PTR), (PTR, PTR, None, PTR, PTR), (PTR, PTR, PTR, PTR, None)):
        assert "null" in refused(fn, d, *args, None)
    assert "aligned" in refused(fn, d, PTR + 1, PTR, PTR, PTR, PTR, None)


def test_empty_calls_launch_nothing():
    lib = ABI.library()
    assert lib.b2vx_fp4_quantize_noalloc(C.byref(desc(ABI.QuantizeDesc, QUANTIZE, rows=0)), None, None, None, None, None, None, None, 0) == 0
    assert lib.b2vx_fp4_dequantize_noalloc(C.byref(desc(ABI.DequantizeDesc, DEQUANTIZE, rows=0)), None, None, None, None, None, None, 0) == 0
    assert lib.b2vx_linear_noalloc(C.byref(desc(ABI.LinearDesc, LINEAR, rows=0)), C.byref(ABI.LinearArgs()), None, None, 0) == 0
    assert lib.b2vx_linear_noalloc(C.byref(desc(ABI.LinearDesc, LINEAR, n=0)), C.byref(ABI.LinearArgs()), None, None, 0) == 0
    assert lib.b2vx_combine_noalloc(C.byref(desc(ABI.CombineDesc, COMBINE, tokens=0)), None, None, None, None, None, None, None, 0) == 0


def packed_size(fmt, matrices, n, k, gated=0):
    size = C.c_size_t()
    assert ABI.library().b2vx_fp4_packed_scales_size_noalloc(fmt, matrices, n, gated, k, C.byref(size)) == 0
    return size.value


def test_sizes():
    # tiles of 128 rows x 4 blocks of 512 bytes, K in steps of 256 columns
    assert packed_size(1, 1, 128, 256) == 2 * 512
    assert packed_size(2, 1, 128, 256) == 4 * 512
    assert packed_size(1, 3, 129, 257) == 3 * 2 * 4 * 512
    assert packed_size(1, 0, 5, 64) == 0
    assert ABI.library().b2vx_fp4_packed_scales_size_noalloc(0, 1, 1, 0, 1, C.byref(C.c_size_t())) == 1
    assert packed_size(1, 2, 72, 64, 1) == 2 * 2 * 2 * 512     # gated: 64 features to a tile
    size = C.c_size_t()
    lib = ABI.library()
    # codes of 8 rows, 48 bytes each, and two words of scales for a tile of each expert's
    assert lib.b2vx_linear_workspace_size_noalloc(C.byref(desc(ABI.LinearDesc, LINEAR)), C.byref(size), None, 0) == 0
    assert size.value == 512 + 2 * 512
    assert lib.b2vx_linear_workspace_size_noalloc(C.byref(desc(ABI.LinearDesc, LINEAR, experts=5)), C.byref(size), None, 0) == 0
    assert size.value == 512 + 5 * 2 * 512


@pytest.mark.parametrize("bn", [64, 128, 192, 224])
def test_group_scale_tiles_do_not_overlap(bn):
    """The rule that gives every tile of a group's rows its own scale tiles: group e starts at (lo / bn + e) tiles of bn rows."""
    import random
    rng = random.Random(bn)
    for _ in range(300):
        counts = [rng.choice([0, 0, 1, bn - 1, bn, bn + 1, rng.randrange(2000)]) for _ in range(rng.randrange(1, 40))]
        lo, end = 0, 0
        for e, n in enumerate(counts):
            first = lo // bn + e
            assert first >= end
            end = first + -(-n // bn)
            lo += n
        assert end <= lo // bn + len(counts)


def test_tensors_must_be_on_a_gpu():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="GPU"):
        D.quantize_fp4(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="type"):
        D.quantize_fp4(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(ValueError, match="format"):
        D.quantize_fp4(torch.zeros(2, 32), "block8")
    with pytest.raises(ValueError, match="scale"):
        D.quantize_fp4(torch.zeros(2, 32), "block16")
    with pytest.raises(ValueError, match="last dimension"):
        D.quantize_fp4(torch.zeros(32, 2).t())
    with pytest.raises(ValueError, match="gradient"):
        D.quantize_fp4(torch.zeros(2, 32, requires_grad=True))
    with pytest.raises(ValueError, match="must be a tensor"):
        D.quantize_fp4([[1.0] * 32])
    with pytest.raises(ValueError, match="multiple of 16"):
        D.Fp4Weight(torch.zeros(24, 32, dtype=torch.uint8), torch.zeros(24, 2, dtype=torch.uint8), gated=True)
    with pytest.raises(ValueError, match="shape"):
        D.Fp4Weight(torch.zeros(24, 32, dtype=torch.uint8), torch.zeros(24, 4, dtype=torch.uint8))
    with pytest.raises(ValueError, match="offsets"):
        D.expert_linear(torch.zeros(2, 32, dtype=torch.bfloat16), torch.zeros(3, 8, 32, dtype=torch.bfloat16), None)
    with pytest.raises(ValueError, match="columns"):
        D.linear(torch.zeros(2, 32, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="two dimensions"):
        D.combine_experts(torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32), torch.zeros(4))


def test_addresses_of_words_must_be_aligned():
    lib, odd = ABI.library(), PTR + 2
    d = desc(ABI.QuantizeDesc, QUANTIZE)
    assert "aligned" in refused(lib.b2vx_fp4_quantize_noalloc, d, PTR, odd, None, PTR, PTR, None)
    d = desc(ABI.QuantizeDesc, dict(QUANTIZE, format=2, scales_pitch=6))
    assert "aligned" in refused(lib.b2vx_fp4_quantize_noalloc, d, PTR, None, odd, PTR, PTR, None)
    d = desc(ABI.DequantizeDesc, dict(DEQUANTIZE, format=2, scales_pitch=6))
    assert "aligned" in refused(lib.b2vx_fp4_dequantize_noalloc, d, PTR, PTR, odd, PTR, None)
    d = desc(ABI.LinearDesc, dict(LINEAR, w_format=2, experts=4))
    for name in ("bias", "x_scale", "w_scale", "offsets", "row_index"):
        words = dict(dict(bias=PTR, x_scale=PTR, w_scale=PTR, offsets=PTR, row_index=PTR), **{name: odd})
        a = desc(ABI.LinearArgs, dict(words, x=PTR, w=PTR, w_scales=PTR, y=PTR, workspace=PTR, workspace_bytes=1 << 30))
        assert "aligned" in refused(lib.b2vx_linear_noalloc, C.byref(d), C.byref(a), None)
    d = C.byref(desc(ABI.RouteDesc, ROUTE))
    for i in range(1, 6):
        args = [PTR] * 6
        args[i] = odd
        assert "aligned" in refused(lib.b2vx_route_noalloc, d, *args, PTR, 1 << 20, None)
    d = C.byref(desc(ABI.CombineDesc, COMBINE))
    for args in ((PTR, odd, PTR, PTR, PTR), (PTR, PTR, odd, PTR, PTR)):
        assert "aligned" in refused(lib.b2vx_combine_noalloc, d, *args, None)


def test_derivatives_are_refused_and_not_dropped():
    torch = pytest.importorskip("torch")
    import torch.autograd.forward_ad as forward
    with forward.dual_level():
        dual = forward.make_dual(torch.ones(2, 32), torch.ones(2, 32))
        with pytest.raises(ValueError, match="forward-mode"):
            D.quantize_fp4(dual)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            D.linear(dual.bfloat16(), torch.zeros(8, 32, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="forward-mode"):
            D.combine_experts(torch.zeros(4, 8), torch.zeros(4, 1, dtype=torch.int32), forward.make_dual(torch.ones(4, 1), torch.ones(4, 1)))
        assert forward.unpack_dual(dual).tangent is not None
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):       # a gradient that nobody asks for is no obstacle
        D.quantize_fp4(torch.zeros(2, 32, requires_grad=True))


def test_transformed_tensors_are_refused():
    """torch.func's wrappers have no memory of their own."""
    torch = pytest.importorskip("torch")
    for transformed in (lambda f: torch.func.grad(lambda x: f(x).sum()), lambda f: torch.func.vmap(f), lambda f: (lambda x: torch.func.jvp(f, (x,), (x,)))):
        with pytest.raises(ValueError, match="memory of its own"):
            transformed(lambda x: D.quantize_fp4(x).scales.float())(torch.ones(3, 32))
    with pytest.raises(ValueError, match="memory of its own"):
        D.quantize_fp4(torch.ones(2, 32).to_sparse())


def test_traces_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda x: D.quantize_fp4(x).codes, torch.ones(2, 32))


@pytest.mark.parametrize("change,args,told", [
    (dict(), dict(), 1), (dict(w_format=1), dict(), 0), (dict(), dict(row_index=PTR), 0), (dict(), dict(x=PTR + 2), 0), (dict(x_stride=100), dict(), 0),
    (dict(x_stride=104), dict(x=PTR + 16), 1)])
def test_products_that_need_no_workspace(change, args, told):
    d = desc(ABI.LinearDesc, dict(LINEAR, w_format=0), **change)
    a = desc(ABI.LinearArgs, dict(x=PTR, w=PTR, y=PTR), **args)
    assert ABI.library().b2vx_linear_in_place_noalloc(C.byref(d), C.byref(a)) == told
    assert ABI.library().b2vx_linear_in_place_noalloc(None, C.byref(a)) == 0


def test_the_libraries_are_made_without_torch():
    def commands(python):
        env = {k: v for k, v in os.environ.items() if k not in ("PYTHONPATH", "MAKEFLAGS")}
        return subprocess.run(["make", "-n", "-B", "-C", os.path.dirname(pyb2vx.PRODUCT_LIB), "PYTHON=" + python], capture_output=True, text=True, check=True, env=env).stdout
    with_torch, without = commands(sys.executable), commands(sys.executable + " -S")     # -S: no installed packages
    for text in (with_torch, without):
        assert "-o " + pyb2vx.PRODUCT_LIB in text and "libtim-vx.so" in text
    assert "deviceops_torch.cc" in with_torch and "deviceops_torch.cc" not in without
    assert "has no torch" in without


@pytest.mark.parametrize("name", ["block_linear.cu", "block_linear.cuh", "fp4_quant.cu", "fp4.cuh", "experts.cu", "device_ops.cu"])
def test_launches_count_the_devices_sms(name):
    """No number of SMs is written into the code of these operators; comments say which one figures were measured on."""
    with open(os.path.join(os.path.dirname(pyb2vx.PRODUCT_LIB), name)) as f:
        assert not re.findall(r"\b(?:148|132|160)\b", re.sub(r"//.*", "", f.read()))
