"""Host side of the block-scaled e4m3 format: encoding, weight preparation, the launchers' strides and refusals."""
import numpy as np
import pytest

from h3metal_b200 import linear, ops, quant
from tests.fakes import RecordingGpu


class F8Gpu(RecordingGpu):
    def rms_f8_native(self, x, x_stride, y, y_stride, res, res_stride, w, out, out_stride, sa, sa_stride, M, D, eps, name=""):
        self.calls.append(dict(kind="rms", x=x, x_stride=x_stride, y=y, y_stride=y_stride, res=res, res_stride=res_stride,
                               out_stride=out_stride, sa_stride=sa_stride, M=M, D=D, eps=eps))

    def quant_f8_native(self, x, x_stride, out, out_stride, sa, sa_stride, M, D, mode, name=""):
        self.calls.append(dict(kind="quant", x=x, x_stride=x_stride, out_stride=out_stride, sa_stride=sa_stride, M=M, D=D,
                               mode=mode))

    def gemm_f8_native(self, a, a_stride, sa, sa_stride, w, w_stride, sw, sw_stride, bias, out, c_stride, M, N, K, name=""):
        self.calls.append(dict(kind="gemm", a_stride=a_stride, sa_stride=sa_stride, w_stride=w_stride, sw_stride=sw_stride,
                               bias=bias, c_stride=c_stride, M=M, N=N, K=K))


def test_codes_match_torch_and_round_to_even():
    import torch
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(quant.e4m3_to_f32(codes), want, equal_nan=True)
    finite = codes[(codes & 0x7F) != 0x7F]
    assert np.array_equal(quant.e4m3_bits(quant.e4m3_to_f32(finite)), finite)
    rng = np.random.default_rng(0)
    grid = np.sort(np.abs(quant.e4m3_to_f32(finite).astype(np.float64)))
    middles = (grid[1:] + grid[:-1]) / 2
    v = np.concatenate([rng.standard_normal(4000) * 10.0 ** rng.uniform(-4, 2.5, 4000), middles, -middles, [0.0, -0.0, 448, 460,
                        -1e9]]).astype(np.float32)
    want = torch.from_numpy(np.clip(v, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(quant.e4m3_bits(v), want)
    assert quant.e4m3_bits(np.array([np.nan]))[0] == 0x7F


@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 1000), (300, 129)])
def test_weight_blocks(N, K):
    rng = np.random.default_rng(N + K)
    w = (rng.standard_normal((N, K)) * 0.02).astype(np.float32)
    w[:, :K // 3] = 0.0
    codes, scales = quant.quantize("f8", w)
    assert codes.shape == (N, quant.f8_stride(K)) and scales.shape == (-(-N // 128), -(-K // 128))
    back = quant.dequant("f8", codes, scales, N, K)
    s = np.repeat(np.repeat(scales, 128, 0)[:N], 128, 1)[:, :K].astype(np.float64)
    # half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale among its subnormals; the division by the scale and
    # the multiplication back add 2^-24 each
    assert (np.abs(back - w.astype(np.float64)) <= (2.0 ** -4 * np.abs(w) + 2.0 ** -10 * s) * (1 + 2.0 ** -22)).all()
    assert (codes[:, K:] == 0).all()
    if K >= 384:
        assert scales[0, 0] == 1.0  # a block of zeros


def test_launchers_pass_default_and_given_strides():
    g = F8Gpu()
    M, D = 5, 1000
    x, w, out = g.empty((M, D), "bf16"), g.empty((D,), "f32"), g.empty((M, 1008), "f8")
    sa = g.empty((8, M), "f32")
    ops.rms_f8(g, x, w, out, sa, M, D, eps=1e-6)
    assert {k: g.calls[-1][k] for k in ("x_stride", "out_stride", "sa_stride", "y", "res")} == \
        {"x_stride": 1000, "out_stride": 1008, "sa_stride": 5, "y": None, "res": None}
    y = g.empty((M, D), "f16")
    ops.rms_f8(g, x, w, out, sa, M, D, eps=1e-6, y=y)
    assert g.calls[-1]["res"] is x and g.calls[-1]["res_stride"] == 1000
    r = g.empty((M, 1008), "bf16")
    ops.rms_f8(g, x, w, out, sa, M, D, eps=1e-6, y=y, res=r, res_stride=1008)
    assert g.calls[-1]["res"] is r and g.calls[-1]["res_stride"] == 1008
    ops.quant_f8(g, x, out, sa, M, 500, swiglu=True, out_stride=1008)
    assert (g.calls[-1]["mode"], g.calls[-1]["x_stride"]) == (1, 1000)
    wt = linear.upload_weight_f8(g, np.zeros((300, D), np.float32), np.zeros(300))
    c = g.empty((M, 304), "f32")
    ops.gemm_f8(g, out, wt, c, M, sa=sa, c_stride=304)
    call = g.calls[-1]
    assert (call["a_stride"], call["w_stride"], call["sw_stride"], call["c_stride"], call["sa_stride"]) == (1008, 1008, 8, 304, 5)
    assert call["bias"] is wt.bias


def test_layer_uses_its_buffers_for_fewer_rows():
    g = F8Gpu()
    wt = linear.upload_weight_f8(g, np.zeros((256, 320), np.float32))
    layer = linear.BlockScaledLinear(g, wt, 40, swiglu_in=True)
    layer(g.empty((40, 640), "bf16"), 3)
    assert [c["kind"] for c in g.calls] == ["quant", "gemm"] and all((c["M"], c["sa_stride"]) == (3, 40) for c in g.calls)
    with pytest.raises(ValueError):
        layer(g.empty((41, 640), "bf16"), 41)
    with pytest.raises(ValueError):
        layer.normed(g.empty((40, 320), "bf16"), g.empty((320,), "f32"), eps=1e-6)
    plain = linear.BlockScaledLinear(g, wt, 40)
    plain.normed(g.empty((40, 320), "f32"), g.empty((320,), "f32"), eps=1e-6, y=g.empty((40, 320), "bf16"))
    assert [c["kind"] for c in g.calls[-2:]] == ["rms", "gemm"]


def test_refusals():
    g = F8Gpu()
    M, D = 4, 256
    x, w, out, sa = g.empty((M, D), "bf16"), g.empty((D,), "f32"), g.empty((M, D), "f8"), g.empty((2, M), "f32")
    wt = linear.upload_weight_f8(g, np.zeros((128, D), np.float32))
    c = g.empty((M, 128), "bf16")
    bad = [
        lambda: ops.rms_f8(g, x, w, out, sa, 0, D, eps=1e-6),
        lambda: ops.rms_f8(g, x, w, out, sa, M + 1, D, eps=1e-6),                        # buffers end before the last row
        lambda: ops.rms_f8(g, x, w, g.empty((M, D), "i8"), sa, M, D, eps=1e-6),
        lambda: ops.rms_f8(g, x, w, out, g.empty((1, M), "f32"), M, D, eps=1e-6),
        lambda: ops.rms_f8(g, x, g.empty((D - 1,), "f32"), out, sa, M, D, eps=1e-6),
        lambda: ops.rms_f8(g, x, w, out, sa, M, D, eps=1e-6, res=x),                     # res without y
        lambda: ops.rms_f8(g, x, w, out, sa, M, D, eps=1e-6, y=x, res=g.empty((M, D), "f32")),
        lambda: ops.rms_f8(g, g.empty((M, D), "i8"), w, out, sa, M, D, eps=1e-6),
        lambda: ops.quant_f8(g, x, out, sa, M, D, swiglu=True),                          # no gates in the buffer
        lambda: ops.quant_f8(g, x, out, sa, M, D, x_stride=128),
        lambda: ops.quant_f8(g, x, out, sa, M, D, sa_stride=3),
        lambda: ops.quant_f8(g, x, out, sa, M, 0),
        lambda: ops.gemm_f8(g, out, wt, c, M + 1, sa=sa),
        lambda: ops.gemm_f8(g, x, wt, c, M, sa=sa),
        lambda: ops.gemm_f8(g, out, wt, g.empty((M, 128), "i32"), M, sa=sa),
        lambda: ops.gemm_f8(g, out, wt, c, M, sa=g.empty((M,), "f32")),
        lambda: ops.gemm_f8(g, out, ops.QWeight("q8", wt.w, wt.sw, 128, D), c, M, sa=sa),
        lambda: ops.gemm_f8(g, out, ops.QWeight("f8", wt.w, wt.sw, 256, D), c, M, sa=sa),
        lambda: ops.gemm_f8(g, out, ops.QWeight("f8", wt.w, None, 128, D), c, M, sa=sa),
        lambda: ops.gemm_f8(g, out, ops.QWeight("f8", wt.w, wt.sw, 128, D, bias=sa), c, M, sa=sa),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(NotImplementedError):  # the int8 product refuses the e4m3 format, as it refuses every other
        ops.gemm(g, out, wt, c, M, sa=sa)
    assert not g.calls
