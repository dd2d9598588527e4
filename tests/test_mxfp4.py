"""The microscaled 4-bit format and the products on it, against the format's definition in numpy.

Quantisation, packing and dequantisation are exact: every element is compared bit for bit.  A product is
a sum of K products that are multiples of 2^(ea+eb)/4; each accumulation step (at most K/32 of them,
with the scales applied) may lose 2^-23 of the running sum, which is at most sum |a||b|, and the last
steps (bias, activation, store) a few 2^-24 of the result: (K/32 + 8) 2^-23 (sum |a||b| + |bias|).
"""
import ctypes

import numpy as np
import pytest

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


# ---------------------------------------------------------------------- the format in numpy
def quantize64(x):
    """codes [rows, blocks*32] and scale bytes [rows, blocks] of blocks along the rows."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(axis=2)
    v = np.where(bad[..., None], 0.0, v)
    amax = np.abs(v).max(axis=2)
    e = np.where(amax > 0, np.frexp(np.where(amax > 0, amax, 1.0))[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    a = np.abs(v) / np.exp2(e.astype(np.float64))[..., None]
    step = np.exp2(np.clip(np.floor(np.log2(np.maximum(a, 1.0))), 0, 2) - 1)
    mag = np.minimum(np.rint(a / step) * step, 6.0)
    code = np.searchsorted(VALUES, mag) + 8 * (np.signbit(v) & ~bad[..., None])
    byte = np.where(bad, 255, e + 127)
    return code.reshape(rows, blocks * 32).astype(np.uint8), byte.astype(np.uint8)


def pack(code, byte):
    rows, blocks = byte.shape
    out = (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8).reshape(-1)
    at = -(-out.size // 512) * 512
    tall, wide = -(-rows // 128), -(-blocks // 4)
    scales = np.zeros((tall, wide, 512), np.uint8)
    for r in range(rows):
        for b in range(blocks):
            scales[r // 128, b // 4, (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4] = byte[r, b]
    packed = np.zeros(at + scales.size, np.uint8)
    packed[:out.size] = out
    packed[at:] = scales.reshape(-1)
    return packed, out.size, at


def values64(code, byte, cols):
    rows, blocks = byte.shape
    v = np.where(code >= 8, -VALUES[code & 7], VALUES[code & 7]).reshape(rows, blocks, 32)
    scale = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return (v * scale[..., None]).reshape(rows, -1)[:, :cols]


def through(x):
    return values64(*quantize64(x), x.shape[1])


def upload_packed(g, x):
    return g.Buffer.from_host(pack(*quantize64(x))[0].view(np.float32))


def refused(g, call, code):
    with pytest.raises(g.GonnError) as e:
        call()
    assert e.value.code == code and e.value.message, e.value


class Handle:
    handle = ctypes.c_void_p(0x1234)


# ---------------------------------------------------------------------- CPU
def test_packed_sizes(built_lib):
    g = built_lib
    for rows, cols in ((1, 1), (1, 32), (3, 33), (128, 128), (129, 129), (1000, 784), (5, 4096)):
        code, byte = quantize64(np.ones((rows, cols)))
        assert g.mxfp4_bytes(rows, cols) == pack(code, byte)[0].size
    assert g.mxfp4_bytes(2 ** 31 - 1, 2 ** 20) > 2 ** 50
    for rows, cols in ((0, 4), (4, 0), (-1, 4), (2 ** 31, 4), (2 ** 31 - 1, 2 ** 31 - 1)):
        with pytest.raises(g.GonnError):
            g.mxfp4_bytes(rows, cols)


def test_dimensions_are_refused_before_anything_else(built_lib):
    g, h = built_lib, Handle()
    for rows, cols in ((0, 4), (4, -1), (2 ** 31, 4)):
        refused(g, lambda: g.mxfp4_quantize(h, rows, cols, False, h), -3)
        refused(g, lambda: g.mxfp4_dequantize(h, rows, cols, h), -3)
        refused(g, lambda: g.mxfp4_matmul(h, rows, h, 4, cols, h), -3)
        refused(g, lambda: g.mxfp4_linear(h, 4, cols, h, rows, None, -1, 0.0, h), -3)
    refused(g, lambda: g.mxfp4_quantize(h, 4, 4, False, h), -2)
    refused(g, lambda: g.mxfp4_dequantize(h, 4, 4, h), -2)
    refused(g, lambda: g.mxfp4_matmul(h, 4, h, 4, 4, h), -2)


def test_the_format_rounds_to_the_nearest_code():
    """The numpy definition itself: no code is nearer, ties go to the even code."""
    x = np.concatenate([np.linspace(-6.5, 6.5, 2001), [5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, 7.9]])
    a = np.zeros((x.size, 32))
    a[:, 0], a[:, 1] = x, 4.0                            # the block's scale is 1
    got = through(a)[:, 0]
    far = np.abs(np.abs(np.clip(x, -6, 6))[:, None] - VALUES[None])
    assert np.array_equal(np.abs(np.abs(got) - np.abs(np.clip(x, -6, 6))), far.min(axis=1))
    assert list(got[-8:]) == [4.0, 4.0, 2.0, 2.0, 1.0, 1.0, 0.0, 6.0]


# ---------------------------------------------------------------------- GPU: quantise and back
def spread(rng, rows, cols):
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-30, 30, (rows, 1)))
    return x.astype(np.float32)


SIZES = [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (128, 128), (129, 130), (7, 784), (300, 100), (1, 5000),
         (257, 1001), (1000, 10), (64, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("transposed", [False, True])
def test_quantize_packs_and_dequantizes_exactly(gpu, rows, cols, transposed):
    rng = np.random.default_rng(rows * 7 + cols)
    x = spread(rng, rows, cols)
    logical = np.ascontiguousarray(x.T) if transposed else x
    code, byte = quantize64(logical)
    want, codes, at = pack(code, byte)
    src = gpu.Buffer.from_host(x)
    packed = gpu.Buffer.from_host(np.full(want.size // 4, np.float32(3.3)))  # stale bytes everywhere
    gpu.mxfp4_quantize(src, rows, cols, transposed, packed)
    got = packed.retrieve_bytes()
    assert np.array_equal(got[:codes], want[:codes]) and np.array_equal(got[at:], want[at:])
    r, c = logical.shape
    out = gpu.Buffer.empty(r * c * 4)
    gpu.mxfp4_dequantize(packed, r, c, out)
    assert np.array_equal(out.retrieve((r, c)).astype(np.float64), values64(code, byte, c))


@pytest.mark.gpu
@pytest.mark.parametrize("transposed", [False, True])
def test_quantize_of_ties_extremes_and_spoiled_blocks(gpu, transposed):
    x = np.zeros((40, 96), np.float32)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99])
    x[0, :9], x[0, 9:18], x[0, 18] = ties, -ties, 4.0
    x[1] = np.nextafter(x[0], np.float32(100))
    x[2] = np.nextafter(x[0], np.float32(-100))
    x[3] = np.finfo(np.float32).max
    x[4] = np.finfo(np.float32).tiny
    x[5] = 1e-45
    x[6, 5], x[6, 40] = np.nan, np.inf
    x[7, 95] = -np.inf
    x[8, :] = -0.0
    x[9, ::2] = 1.5 * 2.0 ** -126
    x[10, :] = np.exp2(np.linspace(-140, 120, 96))
    x[11, 31], x[11, 32] = 1e30, 1e-30
    if transposed:
        x = np.ascontiguousarray(x[:32])
    src = gpu.Buffer.from_host(np.ascontiguousarray(x.T) if transposed else x)
    rows, cols = x.shape
    packed, out = gpu.Buffer.empty(gpu.mxfp4_bytes(rows, cols)), gpu.Buffer.empty(x.nbytes)
    gpu.mxfp4_quantize(src, *((cols, rows) if transposed else (rows, cols)), transposed, packed)
    code, byte = quantize64(x)
    want, codes, at = pack(code, byte)
    got = packed.retrieve_bytes()
    assert np.array_equal(got[:codes], want[:codes]) and np.array_equal(got[at:], want[at:])
    gpu.mxfp4_dequantize(packed, rows, cols, out)
    assert np.array_equal(out.retrieve(x.shape).astype(np.float64), values64(code, byte, cols), equal_nan=True)


# ---------------------------------------------------------------------- GPU: products
def tolerance(a, b, bias):
    k = a.shape[1]
    most = np.abs(a) @ np.abs(b).T + (0 if bias is None else np.abs(bias)[None])
    return (k / 32 + 8) * 2.0 ** -23 * most + 1e-37


def activate(y, act, param):
    if act == 0:
        return np.maximum(y, 0)
    if act == 1:
        return np.where(y > 0, y, y * np.float32(param))
    if act == 2:
        return 1 / (1 + np.exp(-y))
    if act == 3:
        return np.tanh(y)
    if act == 4:
        return 0.5 * y * (1 + np.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    return y


PRODUCTS = [(1, 1, 1), (1, 10, 784), (1, 1000, 4096), (2, 129, 100), (3, 64, 33), (4, 300, 2000), (5, 17, 31), (8, 512, 1024),
            (9, 130, 64), (16, 256, 300), (17, 100, 1000), (33, 65, 129), (64, 256, 256), (100, 1000, 784),
            (128, 128, 128), (129, 257, 513), (200, 300, 5000), (256, 256, 2048), (300, 515, 777), (512, 10, 1024),
            (520, 1030, 260), (1000, 2000, 3000), (2048, 2048, 320), (2050, 2100, 1000), (257, 20000, 100),
            (20001, 130, 600)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_and_matmul(gpu, m, n, k, bias):
    rng = np.random.default_rng(m + 10 * n + 100 * k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[:, rng.random(k) < 0.02] *= 30.0
    w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    bv = rng.standard_normal(n).astype(np.float32) if bias else None
    xq, wq = through(x), through(w)
    want = xq @ wq.T + (0 if bv is None else bv.astype(np.float64))
    tol = tolerance(xq, wq, bv)
    bx, bw, bb = gpu.Buffer.from_host(x), upload_packed(gpu, w), gpu.Buffer.from_host(bv) if bias else None
    y = gpu.Buffer.from_host(np.full((m, n), np.float32(-5.0)))
    gpu.mxfp4_linear(bx, m, k, bw, n, bb, gpu.ACT_NONE, 0.0, y)
    got = y.retrieve((m, n))
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
    ba, c = upload_packed(gpu, x), gpu.Buffer.from_host(np.full((m, n), np.float32(-5.0)))
    gpu.mxfp4_matmul(ba, m, bw, n, k, c, bias=bb)
    got = c.retrieve((m, n))
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 40, 300])
@pytest.mark.parametrize("act", [0, 1, 2, 3, 4, 9])
def test_activations(gpu, m, act):
    """An activation adds its own float32 rounding (expf, tanhf: a few 2^-24) to the product's."""
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, 96)).astype(np.float32)
    w = (rng.standard_normal((70, 96)) / 8).astype(np.float32)
    bv = rng.standard_normal(70).astype(np.float32)
    pre = through(x) @ through(w).T + bv
    y = gpu.Buffer.empty(m * 70 * 4)
    gpu.mxfp4_linear(gpu.Buffer.from_host(x), m, 96, upload_packed(gpu, w), 70, gpu.Buffer.from_host(bv), act, 0.1, y)
    want = activate(pre, act, 0.1)
    assert np.all(np.abs(y.retrieve((m, 70)) - want) <= 2 * tolerance(through(x), through(w), bv) + 2.0 ** -20 * (1 + np.abs(want)))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 40, 96), (7, 300, 160), (130, 140, 320), (300, 300, 512)])
def test_products_of_wide_scales_and_spoiled_blocks(gpu, m, n, k):
    """Scales over many binades keep their places; a NaN block spoils its row or column and no other."""
    rng = np.random.default_rng(m)
    x, w = spread(rng, m, k), spread(rng, n, k)
    x[:, 32:64] *= np.float32(2.0 ** -20)
    x[m // 2, 40] = np.nan
    w[n // 3, k - 1] = np.inf
    xq, wq = through(x), through(w)
    y = gpu.Buffer.empty(m * n * 4)
    gpu.mxfp4_linear(gpu.Buffer.from_host(x), m, k, upload_packed(gpu, w), n, None, gpu.ACT_NONE, 0.0, y)
    got = y.retrieve((m, n))
    bad = np.zeros((m, n), bool)
    bad[m // 2], bad[:, n // 3] = True, True
    assert np.all(np.isnan(got[bad]))
    want, tol = np.nan_to_num(xq) @ np.nan_to_num(wq).T, tolerance(np.nan_to_num(xq), np.nan_to_num(wq), None)
    assert np.all(np.abs(got - want)[~bad] <= tol[~bad])


@pytest.mark.gpu
def test_whole_numbers_are_exact(gpu):
    """Sums that fit 24 bits come out exactly, whatever the split of the work."""
    rng = np.random.default_rng(2)
    for m, n, k in ((1, 128, 4096), (3, 100, 999), (40, 256, 2048), (256, 256, 1024), (257, 300, 4000)):
        x = rng.choice([0, 0, 1, -1, 2, 3, -4, 6], (m, k)).astype(np.float32)
        w = rng.choice([0, 0.5, 1, -1, 2, -3, 4, -6], (n, k)).astype(np.float32)
        x[:, ::32], w[:, ::32] = 4.0, 4.0
        y = gpu.Buffer.empty(m * n * 4)
        gpu.mxfp4_linear(gpu.Buffer.from_host(x), m, k, upload_packed(gpu, w), n, None, gpu.ACT_NONE, 0.0, y)
        assert np.array_equal(y.retrieve((m, n)).astype(np.float64), x.astype(np.float64) @ w.T.astype(np.float64))


@pytest.mark.gpu
def test_sizes_alignment_and_overlaps_are_refused(gpu):
    n = gpu.mxfp4_bytes(40, 70)
    x, p, y = gpu.Buffer.empty(40 * 70 * 4), gpu.Buffer.empty(n), gpu.Buffer.empty(40 * 40 * 4)
    short = gpu.Buffer.empty(n - 4)
    refused(gpu, lambda: gpu.mxfp4_quantize(x, 40, 71, False, p), -3)
    refused(gpu, lambda: gpu.mxfp4_quantize(x, 40, 70, False, short), -3)
    refused(gpu, lambda: gpu.mxfp4_dequantize(short, 40, 70, x), -3)
    refused(gpu, lambda: gpu.mxfp4_dequantize(p, 40, 70, y), -3)
    refused(gpu, lambda: gpu.mxfp4_matmul(short, 40, p, 40, 70, y), -3)
    refused(gpu, lambda: gpu.mxfp4_matmul(p, 40, short, 40, 70, y), -3)
    refused(gpu, lambda: gpu.mxfp4_matmul(p, 40, p, 40, 70, short), -3)
    refused(gpu, lambda: gpu.mxfp4_matmul(p, 40, p, 40, 70, y, bias=gpu.Buffer.empty(39 * 4)), -3)
    refused(gpu, lambda: gpu.mxfp4_linear(x, 41, 70, p, 40, None, -1, 0.0, y), -3)
    odd = gpu.Buffer.wrap(p.device_address() + 4, n - 4)
    refused(gpu, lambda: gpu.mxfp4_dequantize(odd, 8, 70, x), -3)
    inside = gpu.Buffer.wrap(x.device_address() + 1024, 4096)
    refused(gpu, lambda: gpu.mxfp4_quantize(x, 40, 70, False, gpu.Buffer.wrap(x.device_address(), n)), -3)
    refused(gpu, lambda: gpu.mxfp4_linear(x, 40, 70, p, 10, None, -1, 0.0, inside), -3)


@pytest.mark.gpu
def test_scratch_that_cannot_be_had_is_reported(gpu):
    x, p, y = gpu.Buffer.empty(40 * 70 * 4), gpu.Buffer.empty(gpu.mxfp4_bytes(40, 70)), gpu.Buffer.empty(6400)
    gpu.mxfp4_quantize(x, 40, 70, False, p)
    gpu.lib().gonngpu_inject_fault(b"alloc", 1)
    try:
        refused(gpu, lambda: gpu.mxfp4_linear(x, 40, 70, p, 40, None, -1, 0.0, y), -5)
    finally:
        gpu.lib().gonngpu_inject_fault(b"alloc", 0)
    gpu.mxfp4_linear(x, 40, 70, p, 40, None, -1, 0.0, y)
