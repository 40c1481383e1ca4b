"""The operators on device tensors against plain restatements in 64 bits.

Quantization is compared code by code and byte by byte.  Products: a kernel adds float32 partial sums, one for every 16 to 64 columns of K, each
rounded (or cut) to 2^-23 of at most S = sum |x w| |alpha| + |bias|, so a result may be off by (k / 16 + 4) 2^-23 S and half a step of its type."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import device_ops_abi as ABI
import deviceops as D
import pyb2vx

pytestmark = pytest.mark.gpu
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m / 512 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)])[:127]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


@pytest.fixture(autouse=True)
def _settled():
    yield
    D.check()


def nearest(table, v):
    """Index of the nearest table entry, ties to the even index, in exact arithmetic of doubles that are far apart enough."""
    hi = np.clip(np.searchsorted(table, v), 1, len(table) - 1)
    lo = hi - 1
    d_lo, d_hi = v - table[lo], table[hi] - v
    return np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)


def quantized(x, fmt, g=None):
    """Codes [rows][k32] and scale bytes [rows][blocks] of x (float64 values of the inputs)."""
    b = D.BLOCK[fmt]
    rows, k = x.shape
    full = np.zeros((rows, (k + 31) // 32 * 32))
    full[:, :k] = x
    blocks = full.reshape(rows, -1, b)
    amax = np.abs(blocks).max(axis=2)
    bad = ~np.isfinite(blocks).all(axis=2)
    amax = np.where(bad, 1.0, amax)
    if fmt == "block32":
        e = np.where(amax > 0, np.frexp(amax)[1] - 1, -200)
        byte = np.clip(e - 2 + 127, 0, 254)
        unit = np.ldexp(1.0, byte - 127)
        byte = np.where(bad, 255, byte)
    else:
        if not (g > 0 and np.isfinite(g)):
            bad[:] = True
            g = 1.0
        byte = nearest(E4M3, amax / (6 * g))
        unit = E4M3[byte] * g
        byte = np.where(bad, 127, byte)
    with np.errstate(divide="ignore", invalid="ignore"):
        v = np.where(unit[..., None] > 0, np.abs(blocks) / unit[..., None], 0.0)
    codes = nearest(E2M1, np.where(bad[..., None], 0.0, v))
    sign = np.signbit(blocks) & ~bad[..., None] & (unit[..., None] > 0)
    codes = (codes + 8 * sign).astype(np.uint8).reshape(rows, -1)
    return codes, byte.astype(np.uint8)[:, :-(-k // b)]


def values(codes, byte, fmt, g=None):
    v = np.where(codes & 8, -1.0, 1.0) * E2M1[codes & 7]
    if fmt == "block32":
        unit = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(int) - 127))
    else:
        unit = np.where(byte >= 127, np.nan, E4M3[np.minimum(byte, 126)]) * g
    return v * np.repeat(unit, D.BLOCK[fmt], axis=1)[:, :v.shape[1]]


def packed_codes(codes):
    return (codes[:, 0::2] | codes[:, 1::2] << 4).astype(np.uint8)


def unpacked(c):
    return np.stack([c & 15, c >> 4], axis=-1).reshape(c.shape[0], -1)


def f64(t):
    return t.double().cpu().numpy()


def scale_for(x, fmt):
    return None if fmt == "block32" else torch.tensor([float(np.float32(np.abs(x).max() / (6 * 448) + 1e-30))], device="cuda")


def gaussian(rows, k, dtype, seed, spread=3.0):
    """Numbers whose blocks differ in size."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda") * torch.exp2(spread * torch.randn(rows, (k + 15) // 16, generator=g, device="cuda")).repeat_interleave(16, dim=1)[:, :k]
    return x.to(dtype)


def same_quantized(q, x, g=None):
    codes, byte = quantized(f64(x), q.format, g)
    assert np.array_equal(q.scales.cpu().numpy(), byte)
    got = unpacked(q.codes.cpu().numpy())
    if q.format == "block16":     # the sign of a zero in a block whose scale is zero is open
        zero = np.repeat(byte == 0, 16, axis=1)
        zero = np.pad(zero, ((0, 0), (0, codes.shape[1] - zero.shape[1])), constant_values=True)
        got, codes = np.where(zero, got & 7, got), np.where(zero, codes & 7, codes)
    assert np.array_equal(got, codes)


# ---- quantization ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["block32", "block16"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 33), (5, 511), (129, 256), (2, 4099), (1000, 96)])
def test_quantize(fmt, dtype, rows, k):
    x = gaussian(rows, k, dtype, rows * 7919 + k, 2.0)
    s = scale_for(f64(x), fmt)
    q = D.quantize_fp4(x, fmt, scale=s)
    g = None if s is None else float(s)
    same_quantized(q, x, g)
    for out_dtype in (torch.float32, torch.float16, torch.bfloat16):
        codes, byte = unpacked(q.codes.cpu().numpy()), q.scales.cpu().numpy()
        want = values(codes[:, :byte.shape[1] * D.BLOCK[fmt]], byte, fmt, g)[:, :k]
        got = f64(D.dequantize_fp4(q, out_dtype))
        ref = torch.from_numpy(want).float().to(out_dtype).double().numpy()   # exact up to the one rounding
        if fmt == "block32":
            assert np.array_equal(got, ref)
        else:
            ok = np.isfinite(ref)
            assert (np.abs(got - want)[ok] <= (HALF_STEP[out_dtype] * (1 + 2.0 ** -12) + 2.0 ** -24) * np.abs(want)[ok] + TINY[out_dtype]).all()


@pytest.mark.parametrize("g", [1.0, 0.0131, 3e-30, 2.5e30])
def test_quantize_borders_block16(g):
    """Numbers on, just below and just above every border between two codes and two scales."""
    g = float(np.float32(g))
    rows = []
    for b in range(1, 127, 5):
        unit = np.float64(E4M3[b]) * g
        mids = (E2M1[1:] + E2M1[:-1]) / 2 * unit
        row = np.zeros(16)
        row[0] = 6 * unit
        row[1:8] = mids
        row[8:15] = -mids
        for shift in (0, 1, -1):
            r = row.astype(np.float32)
            for _ in range(abs(shift)):
                r[1:15] = np.nextafter(r[1:15], np.float32(np.inf if shift > 0 else -np.inf))
            rows.append(r)
        top = np.zeros(16, np.float32)                       # the scale's own borders
        for s in (-1, 0, 1):
            t = np.float32((E4M3[b] + E4M3[b - 1]) / 2 * 6 * g)
            top = top.copy()
            top[3] = t if s == 0 else np.nextafter(t, np.float32(np.inf if s > 0 else 0))
            rows.append(top)
    x = torch.from_numpy(np.stack(rows)).cuda()
    same_quantized(D.quantize_fp4(x, "block16", scale=torch.tensor([g], device="cuda")), x, g)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("g", [1.0, 1 / 56, 0.5, 3 / 1024, 0.0131, 1.0009765625])
def test_quantize_16_bit_numbers_near_borders(dtype, g):
    """16-bit numbers that lie on borders, and the 16-bit numbers next to those that lie near one, for tensor scales of few and of many bits."""
    g = float(np.float32(g))
    rows = []
    for b in list(range(40, 80)) + [1, 7, 8, 126]:
        unit = np.float64(E4M3[b]) * g
        near = np.concatenate([(E2M1[1:] + E2M1[:-1]) / 2 * unit, E2M1 * unit])
        x = torch.from_numpy(near).to(dtype)
        row = torch.zeros(16, dtype=dtype)
        row[:15] = x
        for step in (0, 1, -1):
            r = (row.view(torch.int16) + torch.where(row != 0, step, 0).to(torch.int16)).view(dtype)
            r[15] = torch.tensor(6 * unit, dtype=dtype)
            rows.append(r)
            rows.append(-r)
    x = torch.stack(rows).cuda()
    same_quantized(D.quantize_fp4(x, "block16", scale=torch.tensor([g], device="cuda")), x, g)


def test_quantize_borders_block32():
    rows = []
    for e in (-140, -127, -126, -125, -100, -1, 0, 3, 100, 124, 125):
        unit = np.ldexp(1.0, e)
        mids = (E2M1[1:] + E2M1[:-1]) / 2 * unit
        r = np.zeros(32, np.float32)
        r[0] = np.float32(4 * unit)
        with np.errstate(over="ignore"):
            r[1:8], r[8:15] = mids, -mids
            r[15], r[16] = 7.75 * unit, -7.5 * unit
        if np.isfinite(r).all():
            rows += [r, np.where(np.arange(32) == 0, r, np.nextafter(r, np.float32(1e38))), np.where(np.arange(32) == 0, r, np.nextafter(r, np.float32(-1e38)))]
    x = torch.from_numpy(np.stack(rows)).cuda()
    same_quantized(D.quantize_fp4(x), x)


@pytest.mark.parametrize("fmt", ["block32", "block16"])
def test_quantize_special_values(fmt):
    x = torch.zeros(8, 96)
    x[0, 40] = float("nan")
    x[1, 3], x[1, 70] = float("inf"), 5.0
    x[2, 0] = -float("inf")
    x[3] = -0.0
    x[4, 33] = 2.0 ** -149
    x[5, 33] = 3.4e38
    x[6] = torch.linspace(-7.9, 7.9, 96)
    x[7, 95] = -1e-30
    x = x.cuda()
    s = None if fmt == "block32" else torch.tensor([1.0], device="cuda")
    q = D.quantize_fp4(x, fmt, scale=s)
    same_quantized(q, x, 1.0)
    y = D.dequantize_fp4(q)
    assert torch.isnan(y[0, 32:48]).all() and torch.isfinite(y[0, :32]).all()
    if fmt == "block16":
        for bad in (0.0, -1.0, float("nan"), float("inf")):
            q = D.quantize_fp4(x, fmt, scale=torch.tensor([bad], device="cuda"))
            assert (q.scales == 127).all() and (q.codes == 0).all()


@pytest.mark.parametrize("fmt", ["block32", "block16"])
@pytest.mark.parametrize("dtype,offset,stride", [(torch.bfloat16, 0, 200), (torch.bfloat16, 1, 203), (torch.float32, 3, 190), (torch.float16, 8, 192)])
def test_quantize_views_and_row_index(fmt, dtype, offset, stride):
    k = 185
    store = gaussian(40, stride + offset, dtype, 5).flatten()
    x = store.as_strided((37, k), (stride, 1), offset)
    index = torch.tensor([0, 36, 5, 5, -1, 37, 1 << 30, 20], dtype=torch.int32, device="cuda")
    s = scale_for(f64(x), fmt)
    q = D.quantize_fp4(x, fmt, scale=s, row_index=index)
    rows = torch.zeros(8, k, dtype=dtype, device="cuda")
    for i, r in enumerate(index.tolist()):
        if 0 <= r < 37:
            rows[i] = x[r]
    same_quantized(q, rows, None if s is None else float(s))


@pytest.mark.parametrize("fmt", ["block32", "block16"])
@pytest.mark.parametrize("matrices,n,k,gated", [(1, 1, 32, False), (2, 130, 288, False), (1, 40, 1024, True), (3, 72, 96, True)])
def test_pack_scales(fmt, matrices, n, k, gated):
    """The layout's rule: [stage of 256 columns][128-row tile][tile of four blocks][row % 32][row / 32][block], gated rows eight by eight."""
    f, b = D.FORMATS[fmt], D.BLOCK[fmt]
    scales = torch.randint(0, 255, (matrices, 2 * n if gated else n, k // b), dtype=torch.uint8, device="cuda")
    size = C.c_size_t()
    assert ABI.library().b2vx_fp4_packed_scales_size_noalloc(f, matrices, n, int(gated), k, C.byref(size)) == 0
    packed = torch.full((size.value,), 0xCD, dtype=torch.uint8, device="cuda")
    ABI.call(ABI.library().b2vx_fp4_pack_scales_noalloc, f, matrices, n, int(gated), k, scales.data_ptr(), packed.data_ptr(), None)
    torch.cuda.synchronize()
    per = 256 // (4 * b)                                     # words (four blocks) of a stage
    want = np.zeros((matrices, (k + 255) // 256, -(-n // 64) if gated else -(-n // 128), per, 32, 4, 4), np.uint8)
    byte = scales.cpu().numpy()
    for m in range(matrices):
        for row in range(byte.shape[1]):
            f, up = (row % n, row // n) if gated else (row, 0)
            t, r = (f // 64, f % 64 // 8 * 16 + up * 8 + f % 8) if gated else (f // 128, f % 128)
            for j in range(byte.shape[2]):
                want[m, j // 4 // per, t, j // 4 % per, r % 32, r // 32, j % 4] = byte[m, row, j]
    assert np.array_equal(packed.cpu().numpy(), want.reshape(-1))


def test_quantize_beyond_two_gigaelements():
    rows, k = 70001, 32768
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-1] = gaussian(1, k, torch.bfloat16, 3)[0]
    q = D.quantize_fp4(x)
    codes, byte = quantized(f64(x[-1:]), "block32")
    assert np.array_equal(unpacked(q.codes[-1:].cpu().numpy()), codes) and np.array_equal(q.scales[-1:].cpu().numpy(), byte)
    y = D.dequantize_fp4(q, torch.bfloat16)
    assert np.array_equal(f64(y[-1:]), values(codes, byte, "block32")) and not y[-2].any()


# ---- products ---------------------------------------------------------------------------------------------------------------

def weight_of(lead, n, k, fmt, seed, gated=False):
    """An Fp4Weight and its values in float64, [experts or 1][n][k]."""
    count = lead or 1
    w = gaussian(count * n, k, torch.float32, seed, 1.0) / k ** 0.5
    g = [None] * count if fmt == "block32" else [float(np.float32(v)) for v in np.linspace(0.0007, 0.0011, count)]
    codes, scales, vals = [], [], []
    for e in range(count):
        c, s = quantized(f64(w[e * n:(e + 1) * n]), fmt, g[e])
        codes.append(packed_codes(c))
        scales.append(s)
        vals.append(values(c, s, fmt, g[e]))
    codes, scales = torch.from_numpy(np.stack(codes)).cuda(), torch.from_numpy(np.stack(scales)).cuda()
    scale = None if fmt == "block32" else torch.tensor(g, device="cuda")
    if not lead:
        codes, scales = codes[0], scales[0]
    return D.Fp4Weight(codes, scales, fmt, scale, gated), np.stack(vals)


def operand(x, fmt):
    """The values of x as the product sees them, and its tensor scale."""
    if fmt == "none":
        return f64(x), None
    s = scale_for(f64(x), fmt)
    g = None if s is None else float(s)
    return values(*quantized(f64(x), fmt, g), fmt, g)[:, :x.shape[1]], s


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-v))


def expected(x, w, bias, gated):
    """The product in 64 bits and how far a result may be off before its own rounding."""
    k = x.shape[1]
    y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    off = (k / 16 + 4) * 2.0 ** -23 * size
    if gated:
        n = y.shape[1] // 2
        g, u = y[:, :n], y[:, n:]
        # silu' is at most 1.1; the exponential, the division and two products add a few steps of float32
        off = 1.1 * off[:, :n] * np.abs(u) + np.abs(silu(g)) * off[:, n:] + off[:, :n] * off[:, n:] + 16 * 2.0 ** -24 * np.abs(silu(g) * u)
        y = silu(g) * u
    return y, off


def close(got, want, off):
    half = HALF_STEP[got.dtype]
    d = np.abs(f64(got) - want)
    bad = ~(d <= half * np.abs(want) + off * (1 + half) + TINY[got.dtype])
    assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4].tolist(), d.max())


SHAPES = [(1, 1, 32), (1, 128, 64), (2, 129, 96), (16, 300, 256), (17, 7, 288), (33, 256, 1056), (64, 500, 544), (65, 257, 512), (129, 640, 96), (193, 130, 320),
          (400, 264, 160), (1000, 1032, 64)]


@pytest.mark.parametrize("fmt", ["block32", "block16", "none"])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_linear(fmt, rows, n, k):
    dtype = (torch.bfloat16, torch.float16, torch.float32)[(rows + n) % (2 if fmt == "none" else 3)]
    out_dtype = (torch.bfloat16, torch.float16, torch.float32)[(rows + k // 32) % 3]
    x = gaussian(rows, k, dtype, rows + n, 1.0)
    bias = gaussian(1, n, torch.float32, 3)[0] if n % 2 == 0 else None
    xv, s = operand(x, fmt)
    if fmt == "none":
        w = (gaussian(n, k, torch.float32, n + k, 1.0) / k ** 0.5).to(dtype)
        wv = f64(w)
    else:
        w, wv = weight_of(0, n, k, fmt, n + k)
        wv = wv[0]
    y = D.linear(x, w, bias=bias, x_scale=s, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    close(y, *expected(xv, wv, None if bias is None else f64(bias), False))


@pytest.mark.parametrize("rows,n,k", [(1, 4096, 4096), (8, 2048, 8192), (3, 5000, 6016), (16, 1024, 16384), (300, 8192, 2048), (2100, 4100, 512), (1, 18000, 8192),
                                      (16, 900, 3104), (17, 900, 3104), (64, 20000, 1056), (1, 40, 65536)])
@pytest.mark.parametrize("fmt", ["block32", "block16"])
def test_linear_large(fmt, rows, n, k):
    x = gaussian(rows, k, torch.bfloat16, rows, 1.0)
    xv, s = operand(x, fmt)
    w, wv = weight_of(0, n, k, fmt, n)
    y = D.linear(x, w, x_scale=s)
    some = np.unique(np.linspace(0, rows - 1, 40).astype(int))
    close(y[torch.from_numpy(some).cuda()], *expected(xv[some], wv[0], None, False))
    again = D.linear(x, w, x_scale=s)
    assert torch.equal(y, again)


@pytest.mark.parametrize("fmt", ["block32", "none"])
@pytest.mark.parametrize("offset,x_stride,y_stride", [(0, 96, 140), (8, 104, 133), (3, 101, 131), (1, 96, 130)])
def test_linear_views(fmt, offset, x_stride, y_stride):
    """x and y inside larger buffers, at odd places; what lies between the rows of y stays."""
    rows, n, k = 70, 130, 96
    store = gaussian(rows + 1, x_stride + offset, torch.bfloat16, 9, 1.0).flatten()
    x = store.as_strided((rows, k), (x_stride, 1), offset)
    if fmt == "none":
        w = gaussian(n, k, torch.bfloat16, 4, 0.0)
        wv = f64(w)
    else:
        w, wv = weight_of(0, n, k, fmt, 4)
        wv = wv[0]
    buf = torch.full((rows * y_stride + 7,), -77.0, dtype=torch.bfloat16, device="cuda")
    y = buf.as_strided((rows, n), (y_stride, 1), offset % 7)
    assert D.linear(x, w, out=y) is y
    close(y, *expected(operand(x, fmt)[0], wv, None, False))
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask.as_strided((rows, n), (y_stride, 1), offset % 7).fill_(False)
    assert (buf[mask] == -77.0).all()


@pytest.mark.parametrize("fmt", ["block32", "block16", "none"])
@pytest.mark.parametrize("rows", [1, 5, 20, 64])
def test_linear_views_few_rows(fmt, rows):
    """The same with few rows: products that quantize x themselves, that share K, and that do neither."""
    for n, k, offset, x_stride, y_stride in ((130, 1056, 1, 1061, 131), (19000, 96, 3, 99, 19001)):
        store = gaussian(rows + 1, x_stride + offset, torch.float16, 9, 1.0).flatten()
        x = store.as_strided((rows, k), (x_stride, 1), offset)
        xv, s = operand(x, fmt)
        if fmt == "none":
            w = (gaussian(n, k, torch.float32, 4, 1.0) / k ** 0.5).half()
            wv = f64(w)
        else:
            w, wv = weight_of(0, n, k, fmt, 4)
            wv = wv[0]
        buf = torch.full((rows * y_stride + 7,), -77.0, dtype=torch.float16, device="cuda")
        y = buf.as_strided((rows, n), (y_stride, 1), 3)
        D.linear(x, w, x_scale=s, out=y)
        close(y, *expected(xv, wv, None, False))
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask.as_strided((rows, n), (y_stride, 1), 3).fill_(False)
        assert (buf[mask] == -77.0).all()


def test_linear_row_index_and_types():
    x = gaussian(20, 64, torch.float32, 2, 1.0)
    index = torch.tensor([3, 3, -1, 19, 20, 0], dtype=torch.int32, device="cuda")
    w, wv = weight_of(1, 40, 64, "block32", 6)
    off = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    y = D.expert_linear(x, w, off, row_index=index, out_dtype=torch.float32)
    rows = torch.stack([x[i] if 0 <= i < 20 else torch.zeros_like(x[0]) for i in index.tolist()])
    close(y, *expected(operand(rows, "block32")[0], wv[0], None, False))


@pytest.mark.parametrize("fmt,k", [("block32", 1056), ("block16", 1120)])
def test_expert_linear_rows_taken_several_times(fmt, k):
    """Enough rows that each row of x is quantized once and then copied; indices outside x give rows of zeros."""
    tokens, rows, n, experts = 300, 5000, 72, 5
    x = gaussian(tokens, k, torch.bfloat16, 12, 1.0)
    rng = np.random.default_rng(3)
    index = rng.integers(-2, tokens + 2, rows).astype(np.int32)
    starts = np.array([0, 700, 700, 2001, 4990, 4997], np.int32)
    w, wv = weight_of(experts, n, k, fmt, 6)
    xv, s = operand(x, fmt)
    y = torch.full((rows, n), -77.0, dtype=torch.bfloat16, device="cuda")
    D.expert_linear(x, w, torch.from_numpy(starts).cuda(), row_index=torch.from_numpy(index).cuda(), x_scale=s, out=y)
    there = (index >= 0) & (index < tokens)
    full = np.where(there[:, None], xv[np.where(there, index, 0)], 0.0)
    for e in range(experts):
        lo, hi = starts[e], starts[e + 1]
        if hi > lo:
            close(y[lo:hi], *expected(full[lo:hi], wv[e], None, False))
    assert (y[starts[-1]:] == -77.0).all()


def test_nan_scales_reach_only_their_outputs():
    x = gaussian(5, 128, torch.bfloat16, 1, 0.5)
    x[2, 7] = float("nan")
    w, wv = weight_of(0, 70, 128, "block32", 8)
    y = D.linear(x, w)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]]).all()
    codes = w.codes.clone()
    scales = torch.full((70, 4), 127, dtype=torch.uint8, device="cuda")
    scales[69, 1] = 255
    y = D.linear(x, D.Fp4Weight(codes, scales))
    assert torch.isnan(y[:, 69]).all() and torch.isfinite(y[[0, 1, 3, 4]][:, :69]).all()


COUNTS = {
    "even": [40, 40, 40],
    "ragged": [0, 1, 130, 0, 7, 64, 65, 0],
    "one": [0, 0, 300, 0],
    "single rows": [1] * 40,
    "empty": [0, 0, 0],
    "long": [500, 3, 200, 129],
}


@pytest.mark.parametrize("fmt", ["block32", "block16", "none"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts", sorted(COUNTS))
def test_expert_linear(fmt, gated, counts):
    counts = COUNTS[counts]
    experts, rows, front = len(counts), sum(counts), 3
    n, k = 136, 288
    total = rows + front + 5                      # rows before the first and behind the last expert
    dtype = torch.float16 if fmt == "block16" else torch.bfloat16
    tokens = 50
    x = gaussian(tokens, k, dtype, 21, 1.0)
    index = torch.from_numpy(np.random.default_rng(4).integers(0, tokens, total).astype(np.int32)).cuda()
    wn = 2 * n if gated else n
    if fmt == "none":
        w = (gaussian(experts * wn, k, torch.float32, 5, 1.0) / k ** 0.5).to(dtype).reshape(experts, wn, k)
        wv = f64(w)
    else:
        w, wv = weight_of(experts, wn, k, fmt, 5, gated)
    bias = gaussian(experts, wn, torch.float32, 6, 0.0)
    starts = front + np.concatenate([[0], np.cumsum(counts)])
    offsets = torch.from_numpy(starts.astype(np.int32)).cuda()
    xv, s = operand(x, fmt)
    y = torch.full((total, n), -77.0, dtype=dtype, device="cuda")
    D.expert_linear(x, w, offsets, row_index=index, bias=bias, gated=gated, x_scale=s, out=y)
    assert (y[:front] == -77.0).all() and (y[front + rows:] == -77.0).all()
    b = f64(bias)
    for e in range(experts):
        lo, hi = starts[e], starts[e + 1]
        if hi > lo:
            close(y[lo:hi], *expected(xv[index.cpu().numpy()[lo:hi]], wv[e], b[e], gated))


@pytest.mark.parametrize("fmt", ["block32", "block16", "none"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows", [3, 40, 400])
def test_gated_output_types(fmt, out_dtype, rows):
    """One group of a gated product, few rows (K shared), a narrow tile and tiles of two CTAs; an odd place and stride of y."""
    n, k = 200, 1120
    dtype = torch.float32 if fmt != "none" else torch.bfloat16
    x = gaussian(rows, k, dtype, 31, 1.0)
    xv, s = operand(x, fmt)
    if fmt == "none":
        w = (gaussian(2 * n, k, torch.float32, 5, 1.0) / k ** 0.5).bfloat16().reshape(1, 2 * n, k)
        wv = f64(w)
    else:
        w, wv = weight_of(1, 2 * n, k, fmt, 5, True)
    bias = gaussian(1, 2 * n, torch.float32, 6, 0.0)
    buf = torch.full((rows, n + 5), -77.0, dtype=out_dtype, device="cuda")
    D.expert_linear(x, w, torch.tensor([0, rows], dtype=torch.int32, device="cuda"), bias=bias, gated=True, x_scale=s, out=buf[:, 3:3 + n])
    close(buf[:, 3:3 + n], *expected(xv, wv[0], f64(bias)[0], True))
    assert (buf[:, :3] == -77.0).all() and (buf[:, 3 + n:] == -77.0).all()


@pytest.mark.parametrize("fmt", ["block32", "none"])
def test_expert_linear_many_experts(fmt):
    experts, n, k = 1024, 40, 64
    counts = np.random.default_rng(1).integers(0, 4, experts)
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1])
    x = gaussian(rows, k, torch.bfloat16, 3, 1.0)
    if fmt == "none":
        w = gaussian(experts * n, k, torch.bfloat16, 4, 0.0).reshape(experts, n, k)
        wv = f64(w)
    else:
        w, wv = weight_of(experts, n, k, fmt, 4)
    y = D.expert_linear(x, w, torch.from_numpy(starts.astype(np.int32)).cuda())
    xv = operand(x, fmt)[0]
    for e in range(experts):
        if counts[e]:
            close(y[starts[e]:starts[e + 1]], *expected(xv[starts[e]:starts[e + 1]], wv[e], None, False))


@pytest.mark.parametrize("offsets", [[0, 50, 20, 70], [-5, 10, 1 << 30, 70], [70, 60, 50, 0], [90, 90, 90, 90]])
def test_bad_offsets_stay_inside(offsets):
    """Offsets that fall or lie outside are cut; rows that no expert has after that are left as they are."""
    w, wv = weight_of(3, 40, 64, "block32", 4)
    x = gaussian(70, 64, torch.bfloat16, 3, 1.0)
    buf = torch.full((72, 40), -77.0, dtype=torch.bfloat16, device="cuda")
    D.expert_linear(x, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out=buf[1:71])
    assert (buf[0] == -77.0).all() and (buf[71] == -77.0).all()
    wb = gaussian(3 * 40, 64, torch.bfloat16, 4, 0.0).reshape(3, 40, 64)
    buf.fill_(-77.0)
    D.expert_linear(x, wb, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out=buf[1:71])
    cut = np.maximum.accumulate(np.clip(offsets, 0, 70))
    ref = f64(x)
    got = buf[1:71]
    seen = np.zeros(70, bool)
    for e in range(3):
        lo, hi = int(cut[e]), int(cut[e + 1])
        seen[lo:hi] = True
        if hi > lo:
            close(got[lo:hi], *expected(ref[lo:hi], f64(wb[e]), None, False))
    assert (got[torch.from_numpy(~seen).cuda()] == -77.0).all()


# ---- routing and the weighted sum -------------------------------------------------------------------------------------------------

def routed(z, k, normalize):
    """ids, weights, offsets, row_index, slots of logits z [tokens][experts] in 64 bits."""
    z = np.where(np.isnan(z), -np.inf, z)
    t, e = z.shape
    ids = np.argsort(-z, axis=1, kind="stable")[:, :k]
    top = z.max(axis=1, keepdims=True)
    with np.errstate(invalid="ignore"):
        p = np.where(z == top, 1.0, np.exp(z - top))
    p = np.where(np.isneginf(top), 0.0, p)
    mine = np.take_along_axis(p, ids, axis=1)
    total = (mine if normalize else p).sum(axis=1, keepdims=True)
    weights = np.where(total > 0, mine / np.where(total > 0, total, 1), 0.0)
    pairs = ids.reshape(-1)
    order = np.argsort(pairs, kind="stable")
    slots = np.empty(t * k, np.int64)
    slots[order] = np.arange(t * k)
    return ids, weights, np.searchsorted(pairs[order], np.arange(e + 1)), order // k, slots.reshape(t, k)


def same_routes(r, z, k, normalize):
    ids, weights, offsets, row_index, slots = routed(f64(z), k, normalize)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    # one exponential of two steps, a sum of up to 1024 terms (five levels across lanes, 32 in a row), a division
    assert (np.abs(f64(r.weights) - weights) <= 48 * 2.0 ** -24 * weights + 2.0 ** -126).all()
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.row_index.cpu().numpy(), row_index)
    assert np.array_equal(r.slots.cpu().numpy(), slots)


@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 8, 8), (31, 33, 2), (32, 64, 32), (33, 100, 3), (700, 256, 8), (5000, 512, 4), (100, 1024, 32), (2049, 7, 7)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route(tokens, experts, k, dtype):
    z = gaussian(tokens, experts, dtype, tokens + experts, 0.5)
    for normalize in (True, False):
        same_routes(D.route_experts(z, k, normalize), z, k, normalize)


def test_route_ties_and_special_values():
    inf, nan = float("inf"), float("nan")
    z = torch.zeros(70, 40)
    z[1] = -inf
    z[2] = nan
    z[3, 10:] = -inf
    z[4, 5] = inf
    z[5, 5], z[5, 6] = inf, inf
    z[6, 1], z[6, 2] = nan, 3.0
    z[7] = -0.0
    z[7, 3] = 0.0
    z[8] = torch.linspace(3e38, -3e38, 40)
    z[9, ::2] = 1.0
    z[10, 39] = -3.4e38
    z[10, :39] = -inf
    z = z.cuda()
    for normalize in (True, False):
        for k in (1, 5, 32):
            same_routes(D.route_experts(z, k, normalize), z, k, normalize)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [60, 200])
def test_route_special_values_of_16_bits(dtype, tokens):
    inf, nan = float("inf"), float("nan")
    z = torch.randint(-3, 3, (tokens, 100)).to(dtype)
    z[1] = -inf
    z[2] = nan
    z[3, 10:] = -inf
    z[4, 5], z[4, 6] = inf, inf
    z[5, 1], z[5, 2] = nan, 3.0
    z[6] = -0.0
    z[6, 3] = 0.0
    z[7] = torch.linspace(-1e-7, 1e-7, 100).to(dtype)
    z[8, ::7] = torch.finfo(dtype).max
    z[9] = torch.finfo(dtype).min
    z = z.cuda()
    for normalize in (True, False):
        for k in (1, 6, 32):
            same_routes(D.route_experts(z, k, normalize), z, k, normalize)


def test_route_views_and_empty():
    z = gaussian(50, 90, torch.float32, 8, 0.0)
    same_routes(D.route_experts(z[:, 5:69], 4), z[:, 5:69], 4, True)
    r = D.route_experts(torch.empty(0, 16, device="cuda"), 2)
    assert not r.offsets.any() and r.ids.shape == (0, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,k,n", [(1, 1, 1), (3, 8, 2048), (100, 3, 77), (513, 2, 4096), (7, 0, 16)])
def test_combine(dtype, tokens, k, n):
    rows = tokens * max(1, k)
    z = gaussian(rows, n, dtype, n, 0.5)
    slots = torch.randint(-1, rows + 1, (tokens, k), dtype=torch.int32, device="cuda")
    w = torch.rand(tokens, k, device="cuda")
    for residual in (None, gaussian(tokens, n, dtype, 5, 0.0)):
        y = D.combine_experts(z, slots, w, residual=residual)
        sl = slots.cpu().numpy()
        there = (sl >= 0) & (sl < rows)
        terms = f64(z)[np.where(there, sl, 0)] * (f64(w) * there)[..., None]
        want, size = terms.sum(axis=1), np.abs(terms).sum(axis=1)
        if residual is not None:
            want, size = want + f64(residual), size + np.abs(f64(residual))
        close(y, want, (k + 2) * 2.0 ** -24 * size)
    if k:
        into = residual.clone()
        assert torch.equal(D.combine_experts(z, slots, w, residual=into, out=into), y)


def test_combine_views():
    z = gaussian(21, 50, torch.bfloat16, 1, 0.0)[:, 3:40]
    slots = torch.arange(20, dtype=torch.int32, device="cuda").reshape(10, 2)
    w = torch.rand(10, 2, device="cuda")
    buf = torch.full((10, 41), -77.0, dtype=torch.bfloat16, device="cuda")
    D.combine_experts(z, slots, w, out=buf[:, 2:39])
    want = (f64(z)[slots.cpu().numpy()] * f64(w)[..., None]).sum(axis=1)
    close(buf[:, 2:39], want, 4 * 2.0 ** -24 * (np.abs(f64(z))[slots.cpu().numpy()] * f64(w)[..., None]).sum(axis=1))
    assert (buf[:, :2] == -77.0).all() and (buf[:, 39:] == -77.0).all()


# ---- together --------------------------------------------------------------------------------------------------------------------

class Layer:
    """A router, gated experts and their weighted sum, as a model has them."""

    def __init__(self, fmt, experts, hidden, inter, top_k, seed):
        self.fmt, self.top_k, self.experts, self.inter = fmt, top_k, experts, inter
        self.router = (gaussian(experts, hidden, torch.float32, seed, 0.0) / hidden ** 0.5).bfloat16()
        if fmt == "none":
            self.up = (gaussian(experts * 2 * inter, hidden, torch.float32, seed + 1, 0.0) / hidden ** 0.5).bfloat16().reshape(experts, 2 * inter, hidden)
            self.down = (gaussian(experts * hidden, inter, torch.float32, seed + 2, 0.0) / inter ** 0.5).bfloat16().reshape(experts, hidden, inter)
            self.up_v, self.down_v = f64(self.up), f64(self.down)
        else:
            self.up, self.up_v = weight_of(experts, 2 * inter, hidden, fmt, seed + 1, True)
            self.down, self.down_v = weight_of(experts, hidden, inter, fmt, seed + 2)
        self.s1 = None if fmt != "block16" else torch.tensor([0.002], device="cuda")
        self.s2 = None if fmt != "block16" else torch.tensor([0.003], device="cuda")

    def __call__(self, x):
        r = D.route_experts(D.linear(x, self.router, out_dtype=torch.float32), self.top_k)
        h = D.expert_linear(x, self.up, r.offsets, row_index=r.row_index, gated=True, x_scale=self.s1)
        z = D.expert_linear(h, self.down, r.offsets, x_scale=self.s2)
        return D.combine_experts(z, r.slots, r.weights, residual=x), r, h, z


@pytest.mark.parametrize("fmt", ["none", "block32", "block16"])
@pytest.mark.parametrize("tokens", [1, 5, 150])
def test_expert_layer(fmt, tokens):
    hidden, inter, experts, top_k = 256, 160, 12, 3
    layer = Layer(fmt, experts, hidden, inter, top_k, 30)
    x = gaussian(tokens, hidden, torch.bfloat16, 77, 0.0)
    y, r, h, z = layer(x)
    # each step against its own inputs: what it was given is what the step before stored
    logits = D.linear(x, layer.router, out_dtype=torch.float32)
    close(logits, *expected(f64(x), f64(layer.router), None, False))
    same_routes(r, logits, top_k, True)
    g = lambda s: None if s is None else float(s)
    xv = f64(x) if fmt == "none" else values(*quantized(f64(x), fmt, g(layer.s1)), fmt, g(layer.s1))
    hv = f64(h) if fmt == "none" else values(*quantized(f64(h), fmt, g(layer.s2)), fmt, g(layer.s2))
    off, index = r.offsets.tolist(), r.row_index.cpu().numpy()
    for e in range(experts):
        if off[e + 1] > off[e]:
            part = slice(off[e], off[e + 1])
            close(h[part], *expected(xv[index[part]], layer.up_v[e], None, True))
            close(z[part], *expected(hv[part], layer.down_v[e], None, False))
    terms = f64(z)[r.slots.cpu().numpy()] * f64(r.weights)[..., None]
    close(y, terms.sum(axis=1) + f64(x), 6 * 2.0 ** -24 * (np.abs(terms).sum(axis=1) + np.abs(f64(x))))


def test_nothing_to_do():
    w, _ = weight_of(3, 16, 64, "block32", 1)
    wb = torch.zeros(3, 16, 64, dtype=torch.bfloat16, device="cuda")
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    none = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    for weight in (w, wb):
        assert D.expert_linear(none, weight, offsets).shape == (0, 16)
    assert D.linear(none, torch.zeros(16, 64, dtype=torch.bfloat16, device="cuda")).shape == (0, 16)
    index = torch.full((5,), -1, dtype=torch.int32, device="cuda")
    offsets[1:] = 5
    for weight in (w, wb):                                  # rows, but no row of x behind them
        assert not D.expert_linear(none, weight, offsets, row_index=index).any()
    q = D.quantize_fp4(none)
    assert q.codes.shape == (0, 32) and D.dequantize_fp4(q).shape == (0, 64)
    assert not D.quantize_fp4(none, row_index=index).codes.any()
    assert D.combine_experts(none, torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, 2, device="cuda")).shape == (0, 64)
    y = D.combine_experts(none, torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda"))
    assert y.shape == (3, 64) and not y.any()


def test_outputs_must_not_overlap_inputs():
    x = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        D.linear(x, torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda"), out=x)
    with pytest.raises(ValueError, match="overlaps"):
        D.combine_experts(x, torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda"), out=x[4:])
    with pytest.raises(ValueError, match="overlap"):
        D.linear(x, torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda"), out=torch.zeros(64, dtype=torch.bfloat16, device="cuda").expand(8, 64))


def test_captured_layers():
    """Two captured graphs, each replayed on new inputs, interleaved with eager calls on another stream."""
    layers = [Layer("block32", 9, 256, 96, 2, 40), Layer("block16", 5, 128, 64, 2, 50)]
    inputs = [gaussian(40, 256, torch.bfloat16, 1, 0.0), gaussian(70, 128, torch.bfloat16, 2, 0.0)]
    graphs, outs = [], []
    for layer, x in zip(layers, inputs):
        layer(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(x)[0])
        graphs.append(g)
    side = torch.cuda.Stream()
    for step in range(5):
        fresh = [gaussian(*x.shape, torch.bfloat16, 100 + step, 0.0) for x in inputs]
        want = [layer(f)[0].clone() for layer, f in zip(layers, fresh)]
        for x, f in zip(inputs, fresh):
            x.copy_(f)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = layers[0](fresh[0])[0]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
        assert torch.equal(other, want[0])


def test_two_streams_at_once():
    """Layers on two streams, nothing waited for in between."""
    layers = [Layer("block32", 16, 512, 192, 4, 60), Layer("block16", 16, 512, 192, 4, 70)]
    xs = [gaussian(n, 512, torch.bfloat16, 9 + n, 0.0) for n in (1, 37, 400)]
    want = [[layer(x)[0].clone() for x in xs] for layer in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(6):
        for i, x in enumerate(xs):
            for s in range(2):
                with torch.cuda.stream(streams[s]):
                    got[s].append((i, layers[s](x)[0]))
    torch.cuda.synchronize()
    for s in range(2):
        for i, y in got[s]:
            assert torch.equal(y, want[s][i])


def test_results_do_not_depend_on_the_run():
    layer = Layer("block32", 16, 512, 192, 4, 60)
    x = gaussian(300, 512, torch.bfloat16, 9, 0.0)
    first = [t.clone() for t in (layer(x)[0], *layer(x)[1])]
    for _ in range(10):
        y, r, _, _ = layer(x)
        for a, b in zip(first, (y, *r)):
            assert torch.equal(a, b)


FIRST = """
import sys
sys.path[:0] = %r
import torch, deviceops as D
torch.manual_seed(0)
x, w = (torch.randn(n, 64, device="cuda").bfloat16() for n in (5, 24))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = D.linear(x, w)
g.replay()
D.check("cuda")
want = x.double() @ w.double().T
assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-4).all()
print("same")
"""


def test_the_first_call_of_a_process_may_be_captured():
    # sums of 64 products of at most 25 or so: float32 is off by less than 1e-4
    out = subprocess.run([sys.executable, "-c", FIRST % sys.path], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr


def test_no_memory_is_torchs_own_error():
    x = torch.zeros(8192, 32, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(1 << 17, 32, dtype=torch.bfloat16, device="cuda")
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.005)   # 0.9 GB; the result has 2
    try:
        with pytest.raises(torch.cuda.OutOfMemoryError):
            D.linear(x, w)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert not D.linear(x, w[:64]).any()


@pytest.mark.parametrize("rows,k", [(3, 1024), (40, 64)])
def test_gate_far_below_zero(rows, k):
    """silu of numbers around -88, whose exponentials leave float32's normal range, times numbers that bring the result back into it."""
    # Sums are of one product, exact.  The exponential is off by two steps or half the smallest float32, the division by two steps, two products
    # and a sum by half a step each or half the smallest float32.
    gates = [-126.0, -103.5, -100.0, -90.0, -88.75, -88.5, -88.0, -87.5, -87.0, -20.0, -0.5, 0.0, 0.5, 20.0, 88.5, 126.0]
    n = len(gates)
    u = 2.0 ** 100
    w = torch.zeros(1, 2 * n, k, dtype=torch.bfloat16, device="cuda")
    w[0, :n, 0], w[0, n:, 0] = torch.tensor(gates), u
    g = f64(w[0, :n, 0])                           # -88.75 is -89 in bfloat16
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1.0
    y = D.expert_linear(x, w, torch.tensor([0, rows], dtype=torch.int32, device="cuda"), gated=True, out_dtype=torch.float32)
    want = silu(g) * u
    off = (4 * 2.0 ** -23 + 3 * 2.0 ** -24) * np.abs(want) + (np.abs(g) + 1) * 2.0 ** -150 * u
    assert (np.abs(f64(y) - want) <= off).all()


@pytest.mark.parametrize("fmt", ["block32", "block16"])
@pytest.mark.parametrize("k,pitch,offset", [(96, 48, 4), (96, 48, 0), (96, 52, 4), (1100, 560, 4), (1100, 564, 0)])
def test_codes_at_any_four_byte_address(fmt, k, pitch, offset):
    """Codes that start on 4 bytes but not on 8, and pitches that are a multiple of 4 but not of 8: what quantize_fp4 stores at 256, between bytes that stay."""
    rows = 9
    x = gaussian(rows, k, torch.bfloat16, k, 2.0)
    s = scale_for(f64(x), fmt)
    want = D.quantize_fp4(x, fmt, scale=s)
    width, blocks = want.codes.shape[1], want.scales.shape[1]
    buf = torch.full((rows * pitch + 8,), 0xCD, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, blocks, dtype=torch.uint8, device="cuda")
    d = ABI.QuantizeDesc(D.FORMATS[fmt], 16, rows, rows, k, k, pitch, blocks)
    ABI.call(ABI.library().b2vx_fp4_quantize_noalloc, C.byref(d), x.data_ptr(), None, None if s is None else s.data_ptr(), buf.data_ptr() + offset, scales.data_ptr(), None)
    torch.cuda.synchronize()
    at = buf.as_strided((rows, width), (pitch, 1), offset)
    assert torch.equal(at, want.codes) and torch.equal(scales, want.scales)
    at.fill_(0xCD)
    assert (buf == 0xCD).all()
    d = ABI.DequantizeDesc(D.FORMATS[fmt], 9, rows, k, pitch, blocks, k)
    buf.as_strided((rows, width), (pitch, 1), offset).copy_(want.codes)
    y = torch.empty(rows, k, device="cuda")
    ABI.call(ABI.library().b2vx_fp4_dequantize_noalloc, C.byref(d), buf.data_ptr() + offset, scales.data_ptr(), None if s is None else s.data_ptr(), y.data_ptr(), None)
    torch.cuda.synchronize()
    assert torch.equal(y, D.dequantize_fp4(want))


@pytest.mark.parametrize("fmt", ["block32", "block16"])
@pytest.mark.parametrize("offsets", [[0, 50, 20, 70], [-5, 10, 1 << 30, 70], [70, 60, 50, 0], [90, 90, 90, 90], [-1, -7, 33, -2, 12, 40], [5, 5, 0, 64, 63, 65, 70], [0, 69, 40, 70]])
def test_bad_offsets_of_4_bit_products(fmt, offsets):
    """Rows and their scales belong to the groups of the offsets after these are cut; memory that was used before holds NaN."""
    experts, rows, n, k = len(offsets) - 1, 70, 40, 96
    w, wv = weight_of(experts, n, k, fmt, 4)
    x = gaussian(rows, k, torch.bfloat16, 3, 1.0)
    xv, s = operand(x, fmt)
    cut = np.maximum.accumulate(np.clip(offsets, 0, rows))
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    buf = torch.full((rows + 2, n), -77.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.empty_cache()
    torch.empty(1 << 21, dtype=torch.uint8, device="cuda").fill_(0x7F)
    D.expert_linear(x, w, off, x_scale=s, out=buf[1:-1])
    seen = np.zeros(rows + 2, bool)
    for e in range(experts):
        lo, hi = int(cut[e]), int(cut[e + 1])
        seen[lo + 1:hi + 1] = True
        if hi > lo:
            close(buf[lo + 1:hi + 1], *expected(xv[lo:hi], wv[e], None, False))
    assert (buf[torch.from_numpy(~seen).cuda()] == -77.0).all()


@pytest.mark.parametrize("fmt", ["block32", "none"])
@pytest.mark.parametrize("rows", [40, 70])
@pytest.mark.parametrize("tiles", [0.5, 1, 1.5, 2, 2.5, 3, 5])
def test_tiles_of_a_cta(fmt, rows, tiles):
    """One to five tiles for each CTA or pair of CTAs, some with one more than others: accumulators are handed back for the tiles that come, and only for those."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n, k = int(128 * sms * tiles) - 9, 96                # 128 features of a tile and SM
    x = gaussian(rows, k, torch.bfloat16, 2, 1.0)
    if fmt == "none":
        w = (gaussian(n, k, torch.float32, 4, 1.0) / k ** 0.5).bfloat16()
        wv = f64(w)
    else:
        w, wv = weight_of(0, n, k, fmt, 4)
        wv = wv[0]
    y = D.linear(x, w)
    close(y, *expected(operand(x, fmt)[0], wv, None, False))
    for _ in range(5):
        assert torch.equal(D.linear(x, w), y)


@pytest.mark.parametrize("fmt", ["block32", "block16"])
def test_bad_offsets_of_rows_taken_several_times(fmt):
    """Rows that are quantized once and copied to where falling offsets put them, in tiles of two CTAs."""
    tokens, rows, n, k = 300, 5000, 72, 1056
    offsets = [-3, 2000, 900, 3500, 3400, 1 << 30, 4000]
    experts = len(offsets) - 1
    x = gaussian(tokens, k, torch.bfloat16, 12, 1.0)
    index = np.random.default_rng(3).integers(0, tokens, rows).astype(np.int32)
    w, wv = weight_of(experts, n, k, fmt, 6)
    xv, s = operand(x, fmt)
    y = D.expert_linear(x, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), row_index=torch.from_numpy(index).cuda(), x_scale=s)
    cut = np.maximum.accumulate(np.clip(offsets, 0, rows))
    for e in range(experts):
        lo, hi = int(cut[e]), int(cut[e + 1])
        if hi > lo:
            close(y[lo:hi], *expected(xv[index[lo:hi]], wv[e], None, False))


STALL = """
import sys
sys.path[:0] = %r
import torch, deviceops as D, pyb2vx as B
g = torch.Generator(device="cuda").manual_seed(1)
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")

def case(fmt, rows, n, k, gated=False):
    # numbers that 4 bits hold with a scale of 1, so that sums are exact
    x = torch.tensor([-6.0, -3.0, 0.0, 1.0, 6.0], device="cuda")[torch.randint(0, 5, (rows, k), generator=g, device="cuda")]
    x[:, ::16] = 6.0
    x = x.bfloat16()
    lead, s, off = (2 * n if gated else n,), None, None
    if gated:
        lead, off = (2,) + lead, torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
    if fmt == "none":
        w = torch.randint(-3, 4, lead + (k,), generator=g, device="cuda").bfloat16()
        v = w.double()
    else:
        codes = torch.randint(0, 256, lead + (k // 2,), dtype=torch.uint8, generator=g, device="cuda")
        one = 127 if fmt == "block32" else 0x38
        scale = None if fmt == "block32" else torch.ones(2 if gated else 1, device="cuda")
        s = None if fmt == "block32" else torch.ones(1, device="cuda")
        w = D.Fp4Weight(codes, torch.full(lead + (k // D.BLOCK[fmt],), one, dtype=torch.uint8, device="cuda"), fmt, scale, gated)
        v = torch.stack([E2M1[(codes & 15).long()], E2M1[(codes >> 4).long()]], dim=-1).flatten(-2)
    if not gated:
        return lambda: D.linear(x, w, x_scale=s, out_dtype=torch.float32), x.double() @ v.T
    h = torch.cat([x[:rows // 3].double() @ v[0].T, x[rows // 3:].double() @ v[1].T])
    return lambda: D.expert_linear(x, w, off, gated=True, x_scale=s, out_dtype=torch.float32), torch.nn.functional.silu(h[:, :n]) * h[:, n:]

cases = [case("none", 40, 40000, 96), case("none", 3, 300, 1024), case("block32", 2, 512, 2048), case("block16", 24, 2048, 4096),
         case("block16", 300, 5000, 1056), case("none", 300, 21000, 160), case("block32", 400, 1024, 512, True), case("block32", 40, 512, 544, True)]
assert len(cases) == %d
torch.cuda.synchronize()
for run, _ in cases:
    run()
    torch.cuda.synchronize()
    for again in (run, D.check):
        try:
            again()
            print("no error")
        except B.B2vxError as e:
            assert e.status == 7 and "gave up waiting on a barrier" in str(e), str(e)
    D.check()
for _ in range(3):
    for i, (run, want) in enumerate(cases):
        got = run().double()
        # of a gated product 16 steps of float32 at most, as in expected() above; sums are exact
        assert ((got - want).abs() <= (16 * 2.0 ** -24 * want.abs() + 2.0 ** -126 if i >= 6 else 0 * want)).all(), i
D.check()
print("same")
"""


def test_a_wait_that_runs_out_is_reported_and_the_context_stays_usable():
    """B2VX_TEST_STALL: the first products of the process announce 16 bytes more than they load and give up after a millisecond, in every form of the kernel:
    one CTA to a tile, a cluster that shares K, with x quantized by the product and before it, and two CTAs to a tile, also by expert."""
    env = dict(os.environ, B2VX_TEST_STALL="8")
    out = subprocess.run([sys.executable, "-c", STALL % (sys.path, 8)], capture_output=True, text=True, env=env, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stdout + out.stderr


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g", [2.0 ** -149, 3e-39, 1e-37, 2.0 ** -126, 1e-30, 2.0 ** -61, 2.0 ** -60, 2.0 ** 60, 2.0 ** 61, 3e38])
def test_quantize_at_the_ends_of_float_range(dtype, g):
    """Tensor scales whose blocks' units are subnormal or below, or near float's largest; zeros, tiny and large numbers side by side."""
    g = float(np.float32(g))
    rng = np.random.default_rng(5)
    rows = [np.zeros(16), np.full(16, 2.0 ** -149), np.where(np.arange(16) % 3 == 0, 3.4e38, 1e-40)]
    for unit in (2.0 ** -9, 2.0 ** -8, 2.0 ** -6, 0.40625, 1.0, 13.0, 448.0):
        for spread in (0.0, 1.0, 6.0):
            r = 6 * unit * g * np.exp2(-spread * rng.random(16)) * rng.choice([-1.0, 1.0], 16)
            r[rng.integers(0, 16, 4)] = 0.0
            rows.append(r)
        rows.append(np.append((E2M1[1:] + E2M1[:-1]) / 2, np.append(E2M1, 6.0)) * unit * g)
    with np.errstate(over="ignore"):
        x = torch.from_numpy(np.nan_to_num(np.stack(rows).astype(np.float32), posinf=3.3e38, neginf=-3.3e38)).to(dtype).cuda()
    same_quantized(D.quantize_fp4(x, "block16", scale=torch.tensor([g], device="cuda")), x, g)


def test_linear_with_a_tiny_scale_of_x():
    """A product that quantizes x itself, x and its scale near float's smallest."""
    n, k = 128, 2048
    x = gaussian(1, k, torch.float32, 8, 0.5) * 1e-37
    x[:, ::5] = 0.0
    g = float(np.float32(1e-38))
    w, wv = weight_of(0, n, k, "block16", 9)
    w.scale.mul_(1e30)
    y = D.linear(x, w, x_scale=torch.tensor([g], device="cuda"), out_dtype=torch.float32)
    xv = values(*quantized(f64(x), "block16", g), "block16", g)
    close(y, *expected(xv, wv[0] * (float(w.scale) / float(np.float32(0.0007))), None, False))


def test_outputs_must_not_overlap_any_input():
    pool = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")

    def at(offset, shape, dtype):
        return pool[offset:].view(dtype)[:int(np.prod(shape))].view(shape)

    x = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    codes, scales = at(0, (3, 64, 32), torch.uint8), at(8192, (3, 64, 4), torch.uint8)
    scales.fill_(0x38)
    w_scale, x_scale, bias = at(16384, (3,), torch.float32), at(16400, (1,), torch.float32), at(16416, (3, 64), torch.float32)
    offsets, index = at(20480, (4,), torch.int32), at(20512, (8,), torch.int32)
    w_scale.fill_(1.0), x_scale.fill_(1.0)
    w = D.Fp4Weight(codes, scales, "block16", w_scale)
    args = dict(row_index=index, bias=bias, x_scale=x_scale)
    for offset in (0, 6143 // 16 * 16, 16384, 16400, 16416 + 512, 20480, 20512):        # over each of them
        with pytest.raises(ValueError, match="overlaps"):
            D.expert_linear(x, w, offsets, out=at(offset, (8, 64), torch.bfloat16), **args)
    with pytest.raises(ValueError, match="overlaps"):
        D.expert_linear(x, w, offsets, out=w.packed[:1024].view(torch.bfloat16).view(8, 64), **args)
    D.expert_linear(x, w, offsets, out=at(65536, (8, 64), torch.bfloat16), **args)

    q = D.Fp4Rows(at(0, (4, 32), torch.uint8), at(128, (4, 4), torch.uint8), 64, "block16", at(256, (1,), torch.float32))
    for offset in (0, 64, 128, 256):
        with pytest.raises(ValueError, match="overlaps"):
            D.dequantize_fp4(q, torch.float16, out=at(offset, (4, 64), torch.float16))
    assert D.dequantize_fp4(q, torch.float16, out=at(512, (4, 64), torch.float16)).shape == (4, 64)

    z, slots, weights = torch.zeros(4, 64, device="cuda"), at(0, (4, 2), torch.int32), at(32, (4, 2), torch.float32)
    for offset in (0, 32):
        with pytest.raises(ValueError, match="overlaps"):
            D.combine_experts(z, slots, weights, out=at(offset, (4, 64), torch.float32))
    wide = torch.zeros(9, 64, device="cuda")
    for residual, out in ((wide[:4], wide[1:5]), (wide[1:5], wide[:4]), (wide[:4], wide[:8:2]), (wide.view(-1)[:256].view(4, 64), wide.view(-1)[4:260].view(4, 64))):
        with pytest.raises(ValueError, match="overlaps"):
            D.combine_experts(z, slots, weights, residual=residual, out=out)
    D.combine_experts(z, slots, weights, residual=wide[:4], out=wide[:4])
    D.combine_experts(z, slots, weights, residual=wide[:4], out=wide[4:8])


def test_columns_of_one_tensor_may_be_input_and_output():
    wide = torch.zeros(30, 256, dtype=torch.bfloat16, device="cuda")
    wide[:, 32:128] = gaussian(30, 96, torch.bfloat16, 1, 0.0)
    w = gaussian(64, 96, torch.bfloat16, 2, 0.0)
    want = D.linear(wide[:, 32:128].contiguous(), w)
    for first in (128, 192):
        assert torch.equal(D.linear(wide[:, 32:128], w, out=wide[:, first:first + 64]), want)
    assert not wide[:, :32].any()
    for first in (0, 64, 127):
        with pytest.raises(ValueError, match="overlaps"):
            D.linear(wide[:, 32:128], w, out=wide[:, first:first + 64])
    narrow = wide.view(60, 128)                          # rows of another pitch over the same memory
    with pytest.raises(ValueError, match="overlaps"):
        D.linear(narrow[:, 32:128], w, out=wide.view(60, 128)[:, 64:])
    with pytest.raises(ValueError, match="overlaps"):
        D.linear(wide[:, 32:128], w, out=wide.view(-1)[:30 * 64].view(30, 64))


def test_outputs_of_the_callers_count_as_changed():
    """A graph that saved a tensor refuses its backward pass once one of these operators has written to it."""
    x, w = torch.ones(4, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, 64, dtype=torch.bfloat16, device="cuda")
    q = D.quantize_fp4(x)
    slots, weights = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.ones(4, 1, device="cuda")
    for write in (lambda out: D.linear(x, w, out=out), lambda out: D.dequantize_fp4(q, torch.bfloat16, out=out),
                  lambda out: D.combine_experts(x, slots, weights, out=out), lambda out: D.combine_experts(x, slots, weights, residual=out, out=out)):
        leaf, out = torch.ones(4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True), torch.ones(4, 64, dtype=torch.bfloat16, device="cuda")
        loss = (leaf * out).sum()
        write(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        D.linear(x, w, out=torch.empty(4, 64, dtype=torch.bfloat16, device="cuda"))


def test_no_workspace_where_x_is_read_in_place():
    x, w = gaussian(4096, 4096, torch.bfloat16, 1, 0.0), gaussian(64, 4096, torch.bfloat16, 2, 0.0)
    out = torch.empty(4096, 64, dtype=torch.bfloat16, device="cuda")
    D.linear(x, w, out=out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    D.linear(x, w, out=out)
    assert torch.cuda.max_memory_allocated() == before
    D.linear(x[1:, :], w, out=out[1:])                   # rows of another place on 16 bytes
    assert torch.cuda.max_memory_allocated() == before
    odd = torch.empty(4096 * 4096 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4096, 4096)
    odd.copy_(x)
    want = out.clone()
    assert torch.equal(D.linear(odd, w), want)
    assert torch.cuda.max_memory_allocated() >= before + 2 * x.numel() * 2


def test_route_as_many_pairs_as_32_bits_count():
    tokens, experts = (2 ** 31 - 1) // 32, 32
    if torch.cuda.mem_get_info()[0] < 56 << 30:
        pytest.skip("needs 56 GB")
    z = torch.empty(tokens, experts, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    r = D.route_experts(z, experts)                      # every token to every expert: rows are known
    assert torch.equal(r.offsets, torch.arange(experts + 1, dtype=torch.int64, device="cuda").mul_(tokens).int())
    step = 1 << 21
    for t in range(0, tokens, step):
        ids, m = r.ids[t:t + step].long(), min(step, tokens - t)
        assert torch.equal(ids.sort(dim=1).values, torch.arange(experts, device="cuda").expand(m, -1))
        assert torch.equal(r.slots[t:t + step].long(), ids * tokens + torch.arange(t, t + m, device="cuda")[:, None])
        assert torch.equal(z[t:t + step].gather(1, ids), z[t:t + step].sort(dim=1, descending=True).values)
    for e in range(experts):
        assert torch.equal(r.row_index[e * tokens:(e + 1) * tokens], torch.arange(tokens, dtype=torch.int32, device="cuda"))
    assert ((r.weights[-5:].sum(dim=1) - 1).abs() <= 32 * 2.0 ** -24).all()


def test_weights_of_no_features():
    x = torch.ones(3, 32, dtype=torch.bfloat16, device="cuda")
    w = D.Fp4Weight(torch.zeros(0, 16, dtype=torch.uint8, device="cuda"), torch.zeros(0, 1, dtype=torch.uint8, device="cuda"))
    assert D.linear(x, w).shape == (3, 0)
    w = D.Fp4Weight(torch.zeros(2, 0, 16, dtype=torch.uint8, device="cuda"), torch.zeros(2, 0, 1, dtype=torch.uint8, device="cuda"), gated=True)
    assert D.expert_linear(x, w, torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"), gated=True).shape == (3, 0)


def test_weights_of_too_many_experts():
    with pytest.raises(pyb2vx.B2vxError, match="1024 matrices"):
        D.Fp4Weight(torch.zeros(1025, 8, 16, dtype=torch.uint8, device="cuda"), torch.zeros(1025, 8, 1, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("fmt", ["block32", "block16", "none"])
@pytest.mark.parametrize("rows,n,k", [(1, 8, 32), (1, 72, 2048), (2, 200, 4096), (16, 4104, 512), (5, 1000, 8192), (17, 136, 1056), (100, 264, 288), (300, 1032, 544)])
def test_one_gated_matrix(fmt, rows, n, k):
    """A gated product without experts, in every form: x quantized by the product and by a launch before it, K shared, two CTAs to a tile."""
    dtype = torch.bfloat16
    x = gaussian(rows, k, dtype, rows + n, 1.0)
    xv, s = operand(x, fmt)
    if fmt == "none":
        w = (gaussian(2 * n, k, torch.float32, n, 1.0) / k ** 0.5).to(dtype)
        wv, packed, scale, codes = f64(w), None, None, w
    else:
        w, wv = weight_of(0, 2 * n, k, fmt, n, True)
        wv, packed, scale, codes = wv[0], w.packed, w.scale, w.codes
    bias = gaussian(1, 2 * n, torch.float32, 6, 0.0)[0] if rows != 2 else None
    d = ABI.LinearDesc(D.FORMATS.get(fmt, 0), 16, 9, 1, 0, rows, rows, n, k, k, n + 3)
    size = C.c_size_t()
    ABI.call(ABI.library().b2vx_linear_workspace_size_noalloc, C.byref(d), C.byref(size))
    work = torch.full((max(1, size.value),), 0x7F, dtype=torch.uint8, device="cuda")
    y = torch.full((rows, n + 3), -77.0, device="cuda")
    at = lambda t: None if t is None else t.data_ptr()
    a = ABI.LinearArgs(at(x), at(codes), at(packed), at(s), at(scale), at(bias), None, None, at(y), at(work), size.value)
    ABI.call(ABI.library().b2vx_linear_noalloc, C.byref(d), C.byref(a), torch.cuda.current_stream().cuda_stream)
    close(y[:, :n], *expected(xv, wv, None if bias is None else f64(bias), True))
    assert (y[:, n:] == -77.0).all()
    assert torch.equal(D.expert_linear(x, w, None, bias=bias, gated=True, x_scale=s, out_dtype=torch.float32), y[:, :n])


FIRST_OF_EACH = """
import sys
sys.path[:0] = %r
import torch, deviceops as D
torch.manual_seed(0)
dev = "cuda"
x, xs = torch.randn(300, 256, device=dev).bfloat16(), torch.full((1,), 0.01, device=dev)
codes = torch.randint(0, 256, (6, 128, 128), device=dev).byte()
scales = torch.randint(118, 124, (6, 128, 8), device=dev).byte()
plain = torch.randn(6, 128, 256, device=dev).bfloat16()
logits = torch.randn(300, 6, device=dev)
odd = torch.randn(301, 257, device=dev).bfloat16()[1:, 1:]
torch.cuda.synchronize()

def everything():
    w, one = D.Fp4Weight(codes, scales, gated=True), D.Fp4Weight(codes[0], scales[0])
    r, few = D.route_experts(logits, 2), D.route_experts(logits[:9], 2)
    h = D.expert_linear(x, w, r.offsets, row_index=r.row_index, gated=True)
    outs = [*r, *few, h, D.expert_linear(x, plain, r.offsets, row_index=r.row_index), D.combine_experts(h, r.slots, r.weights)]
    outs += [D.linear(x[:n], one) for n in (1, 20, 300)] + [D.linear(odd, plain[0]), D.linear(odd[:3], one)]
    for q in (D.quantize_fp4(x), D.quantize_fp4(odd, "block16", scale=xs)):
        outs += [q.codes, q.scales, D.dequantize_fp4(q)]
    return outs

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    captured = everything()
g.replay()
D.check("cuda")
for a, b in zip(captured, everything()):
    assert torch.equal(a, b)
print("same")
"""


def test_the_first_call_of_each_operator_may_be_captured():
    out = subprocess.run([sys.executable, "-c", FIRST_OF_EACH % sys.path], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr
