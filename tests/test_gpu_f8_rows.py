"""rms_f8 and quant_f8 on the GPU against the definition in 64 bits (oracle.f8_ref).

Tolerances count roundings of half a step. A code: 2^-4 of the value, or 2^-10 of the scale among e4m3's subnormals.
fp32: 2^-24 each. The norm's factor: the sum of squares passes at most 16 * 4 additions in a thread (D <= 32768), 5
across a warp and 16 across warps, each with its multiply fused, and its error is halved by the root; division by D, eps,
root (2), two multiplications and the scale's division follow: (85 / 2 + 6) * 2^-24 < 49 * 2^-24. silu: the exponent
-g log2(e) is rounded once, which moves e^-g by up to |g| * 2^-24 of itself, |g| < 104 where e^-g is neither 0 nor infinite;
2^x is off by 2^-22, the reciprocal by 2^-23, the constant, the denominator and the three products by 2^-24 each:
(104 + 4 + 2 + 5) * 2^-24."""
import numpy as np
import pytest

from h3metal_b200 import ops, quant
from oracle import f8_ref

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24
NORM_TOL = 49 * HALF
SILU_TOL = 115 * HALF


def as_type(a, dtype):
    """(array to upload, its values in fp32)."""
    if dtype == "bf16":
        bits = quant.bf16_bits(a.astype(np.float32))
        return bits, quant.bf16_to_f32(bits)
    t = a.astype({"f16": np.float16, "f32": np.float32}[dtype])
    return t, t.astype(np.float32)


def to_f32(t):
    a = t.numpy()
    return quant.bf16_to_f32(a) if t.dtype == "bf16" else a.astype(np.float32)


def padded(a, stride):
    out = np.zeros((a.shape[0], stride), a.dtype)
    out[:, :a.shape[1]] = a
    return out


def check(v, codes, sa, D, tol):
    """codes (bytes) and scales stand for the rows v (64 bits), each value of which was computed to within tol."""
    want = f8_ref.scales(v)
    assert np.all(np.abs(sa - want) <= (tol + HALF) * want)
    s = f8_ref.spread(sa.astype(np.float64), D)
    got = quant.e4m3_to_f32(codes[:, :D]).astype(np.float64) * s
    # the code of v * (1 / s): two roundings before e4m3's own
    assert np.all(np.abs(got - v) <= (2.0 ** -4 * np.abs(v) + 2.0 ** -10 * s) * (1 + 8 * (tol + 2 * HALF)) + (tol + 2 * HALF) * np.abs(v))


def buffers(gpu, M, D, rows=None, out_stride=None, sa_stride=None):
    """Codes and scales with two guard rows behind M; every byte starts as 0x55."""
    rows = rows or M + 2
    stride, sas = out_stride or quant.f8_stride(D), sa_stride or M
    out = gpu.upload(np.full((rows, stride), 0x55, np.uint8), "f8")
    sa = gpu.upload(np.full((-(-D // 128), sas), -7.0, np.float32))
    return out, sa


def guards_kept(out, sa, M, D):
    o, s = out.numpy(), sa.numpy()
    assert (o[M:] == 0x55).all() and (o[:M, D:] == 0x55).all() and (s[:, M:] == -7.0).all()
    return o[:M], s[:, :M]


SIZES = [(1, 1), (1, 128), (3, 8), (2, 100), (7, 129), (5, 1000), (33, 3840), (2, 8191), (9, 8192), (3, 16384), (2, 20000),
         (2, 32768), (700, 256)]


@pytest.mark.parametrize("M,D", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("gated", [False, True])
def test_quantiser(gpu, M, D, dtype, gated):
    rng = np.random.default_rng(D + M)
    wide = 2 * D if gated else D
    stride = -(-wide // 8) * 8 + 8
    x = rng.standard_normal((M, wide)) * np.exp(rng.uniform(-3, 3, (M, 1)))
    x[:, ::37] *= 20
    if D >= 256:
        x[0, :128] = 0.0  # a group of zeros
    raw, val = as_type(x, dtype)
    out, sa = buffers(gpu, M, D, sa_stride=M + 3)
    ops.quant_f8(gpu, gpu.upload(padded(raw, stride)), out, sa, M, D, swiglu=gated, x_stride=stride, sa_stride=M + 3)
    gpu.wait()
    codes, scales = guards_kept(out, sa, M, D)
    v = f8_ref.gated_rows(val, D) if gated else val.astype(np.float64)
    check(v, codes, scales, D, SILU_TOL if gated else 0.0)
    if not gated:  # every step is one rounding of fp32: bit for bit
        s = f8_ref.scales(v).astype(np.float32)
        full = f8_ref.spread(s, D).astype(np.float32)
        assert np.array_equal(scales, s)
        assert np.array_equal(codes[:, :D], quant.e4m3_bits((val * (np.float32(1) / full)).astype(np.float32)))


def test_quantiser_edges(gpu):
    """Zeros, the smallest and largest magnitudes, NaN and infinities, the gate's far ends."""
    D = 1024
    x = np.ones((3, D), np.float32)
    x[0, :128] = 0.0
    x[0, 128:256] = 1e-38 * np.linspace(-1, 1, 128)      # scale at its floor
    x[0, 256:384] = 3e38 * np.linspace(-1, 1, 128)
    x[0, 384] = np.nan                                    # alone in its place
    x[0, 512] = np.inf                                    # the group reads back as NaN
    x[0, 640:768] = np.nan                                # a group of nothing else
    x[0, 768] = -0.0
    x[1, :] = 1e-45 * np.arange(D)
    out, sa = buffers(gpu, 3, D)
    ops.quant_f8(gpu, gpu.upload(x), out, sa, 3, D)
    gpu.wait()
    codes, s = guards_kept(out, sa, 3, D)
    back = quant.e4m3_to_f32(codes) * f8_ref.spread(s, D).astype(np.float32)
    assert s[0, 0] == 1.0 and s[1, 0] == np.float32(2.0 ** -126) and (codes[0, :128] == 0).all()
    assert np.isfinite(back[0, :384]).all() and np.abs(back[0, 256:384] - x[0, 256:384]).max() <= 2.0 ** -4 * 3.0001e38
    assert np.isnan(back[0, 384]) and np.isfinite(back[0, 385:512]).all() and s[3, 0] == np.float32(1) / np.float32(448)
    assert np.isnan(back[0, 512:640]).all() and s[4, 0] == np.inf
    assert np.isnan(back[0, 640:768]).all() and s[5, 0] == 1.0
    assert codes[0, 768] == 0x80 and np.isfinite(back[1:]).all()
    g = np.tile(np.array([-np.inf, -200.0, -100.0, -88.0, -20.0, 0.0, 20.0, 200.0], np.float32), D // 8)[None]
    row = np.concatenate([np.full((1, D), 2.0, np.float32), g], 1)
    row[0, D + 128:] = np.where(np.isinf(row[0, D + 128:]), -300.0, row[0, D + 128:])  # infinities in the first group only
    out, sa = buffers(gpu, 1, D)
    ops.quant_f8(gpu, gpu.upload(row), out, sa, 1, D, swiglu=True)
    gpu.wait()
    codes, s = guards_kept(out, sa, 1, D)
    back = quant.e4m3_to_f32(codes) * f8_ref.spread(s, D).astype(np.float32)
    assert np.isnan(back[0, 0]) and np.isfinite(back[0, 1:8]).all()      # -inf * silu's 0 is no number
    assert np.array_equal(back[0, 128:136], np.array([0, 0, 0, 0, 0, 0, 2 * 20.0, 400.0], np.float32)) or \
        np.allclose(back[0, 128:136], [0, 0, 0, 0, 0, 0, 40.0, 400.0], rtol=2.0 ** -4, atol=400 / 448 * 2.0 ** -10)


@pytest.mark.parametrize("M,D", SIZES)
@pytest.mark.parametrize("xt,yt,wt", [("bf16", None, "f32"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "f32"),
                                      ("f16", "f16", "f16"), ("f32", "f32", "f32"), ("f16", "f32", "f32"), ("bf16", "f32", "f32"),
                                      ("f32", None, "f16"), ("f16", "bf16", "f32"), ("bf16", "f16", "f32"), ("f32", "f16", "f32"),
                                      ("f16", None, "f32")])
def test_norm(gpu, M, D, xt, yt, wt):
    rng = np.random.default_rng(D * 3 + M)
    xs, ys, rs = -(-D // 8) * 8, -(-D // 8) * 8 + 8, -(-D // 8) * 8 + 16
    x = rng.standard_normal((M, D)) * 3
    x[:, ::41] *= 20
    xr, xv = as_type(x, xt)
    wr, wv = as_type(1 + 0.3 * rng.standard_normal(D), wt)
    X, W = gpu.upload(padded(xr, xs)), gpu.upload(wr)
    out, sa = buffers(gpu, M, D)
    if yt is None:
        ops.rms_f8(gpu, X, W, out, sa, M, D, eps=1e-5, x_stride=xs)
        h = xv
    else:
        yr, yv = as_type(rng.standard_normal((M, D)), yt)
        fill = np.zeros((M + 1, rs), xr.dtype)
        fill[:] = 3
        R = gpu.upload(fill)
        ops.rms_f8(gpu, X, W, out, sa, M, D, eps=1e-5, x_stride=xs, y=gpu.upload(padded(yr, ys)), y_stride=ys, res=R, res_stride=rs)
        _, h = as_type(xv + yv, xt)  # one fp32 addition, then the stream's rounding
        kept = to_f32(R)
        assert np.array_equal(kept[:M, :D], h)
        rest = R.numpy()
        assert (rest[M:] == 3).all() and (rest[:, D:] == 3).all()
        assert np.array_equal(to_f32(X)[:, :D], xv)
    gpu.wait()
    codes, scales = guards_kept(out, sa, M, D)
    check(f8_ref.norm_rows(h, wv, 1e-5), codes, scales, D, NORM_TOL)


def test_norm_in_place_and_empty_rows(gpu):
    rng = np.random.default_rng(5)
    M, D = 6, 640
    x, y = rng.standard_normal((M, D)).astype(np.float32), rng.standard_normal((M, D)).astype(np.float32)
    x[2], y[2] = 0, 0                       # nothing in the row: codes of zeros, scales of one
    x[3, 5] = np.nan
    x[4, 7] = np.inf
    X, W = gpu.upload(x), gpu.upload(np.ones(D, np.float32))
    out, sa = buffers(gpu, M, D)
    ops.rms_f8(gpu, X, W, out, sa, M, D, eps=1e-6, y=gpu.upload(y))
    gpu.wait()
    codes, s = guards_kept(out, sa, M, D)
    assert np.array_equal(X.numpy(), x + y, equal_nan=True)
    assert (codes[2] == 0).all() and (s[:, 2] == 1.0).all()
    good = [0, 1, 5]
    check(f8_ref.norm_rows((x + y)[good], np.ones(D), 1e-6), codes[good], s[:, good], D, NORM_TOL)
    assert (codes[3] & 0x7F == 0x7F).all()  # a NaN in a row is in its mean square
    assert codes[4, 7] & 0x7F == 0x7F and (np.delete(codes[4], 7) & 0x7F == 0).all()  # inf * 0; the others divided by inf


def test_refusals_of_the_library(gpu):
    from h3metal_b200.gpu import GpuError
    M, D = 4, 256
    x, w, out, sa = gpu.empty((M, 2 * D), "bf16"), gpu.empty((D,), "f32"), gpu.empty((M, D), "f8"), gpu.empty((2, M), "f32")
    off = x.view((M, D), offset_elems=1)
    n = gpu.launch_count
    bad = [lambda: gpu.quant_f8_native(off, D, out, D, sa, M, M - 1, D, 0),
           lambda: gpu.quant_f8_native(x, D + 1, out, D, sa, M, M, D, 0),
           lambda: gpu.quant_f8_native(x, D, out, D + 8, sa, M, M, D, 0),
           lambda: gpu.quant_f8_native(x, D, out, D, sa, M, M, D, 2),
           lambda: gpu.quant_f8_native(x, D, out, D, sa, M - 1, M, D, 0),
           lambda: gpu.quant_f8_native(x, D, out, D, sa, M, 0, D, 0),
           lambda: gpu.quant_f8_native(out, D, out, D, sa, M, M, D, 0),
           lambda: gpu.rms_f8_native(x, D, None, 0, x, D, w, out, D, sa, M, M, D, 1e-6),
           lambda: gpu.rms_f8_native(x, D, None, 0, None, 0, w, out, D, sa, M, M, D, -1.0),
           lambda: gpu.rms_f8_native(x, D, None, 0, None, 0, w, out, D, sa, M, M, D, float("nan")),
           lambda: gpu.rms_f8_native(x, D, off, D, x, D, w, out, D, sa, M, M, D, 1e-6),
           lambda: gpu.rms_f8_native(x, 32784, None, 0, None, 0, w, out, 32784, sa, M, 1, 32784, 1e-6),
           lambda: gpu.rms_f8_native(x, D, None, 0, None, 0, out, out, D, sa, M, M, D, 1e-6)]
    for call in bad:
        with pytest.raises(GpuError):
            call()
    assert gpu.launch_count == n
