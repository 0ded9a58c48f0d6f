"""BlockScaledLinear where widths are no multiple of 16 bytes: rows lie apart, from one layer's output to the next one's input."""
import numpy as np
import pytest

from h3metal_b200 import linear, quant
from oracle import f8_ref
from tests.test_f8_host import F8Gpu


def test_strides_reach_the_calls():
    g = F8Gpu()
    wt = linear.upload_weight_f8(g, np.zeros((1002, 1001), np.float32))
    layer = linear.BlockScaledLinear(g, wt, 7, out_stride=1008)
    assert layer.out.shape == (7, 1008)
    x, y, r = (g.empty((7, 1008), "bf16") for _ in range(3))
    layer.normed(x, g.empty((1001,), "f32"), eps=1e-6, x_stride=1008, y=y, y_stride=1008, res=r, res_stride=1008)
    rms, gemm = g.calls
    assert (rms["x_stride"], rms["y_stride"], rms["res_stride"]) == (1008, 1008, 1008)
    assert gemm["c_stride"] == 1008
    layer.normed(x, g.empty((1001,), "f32"), 3, eps=1e-6, x_stride=1008, y=y, y_stride=1008)
    assert g.calls[-2]["res"] is x and g.calls[-2]["res_stride"] == 1008 and g.calls[-2]["M"] == 3
    packed = linear.BlockScaledLinear(g, wt, 7)
    assert packed.out.shape == (7, 1002) and packed.out_stride == 1002
    with pytest.raises(ValueError):
        linear.BlockScaledLinear(g, wt, 7, out_stride=1000)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 30, 300])
def test_a_gated_mlp_of_odd_widths(gpu, M):
    """norm -> product -> gated quantiser -> product -> norm -> product, 1001 and 333 channels, each step against the definition
    from the codes it left. Tolerances as in test_gpu_f8_gemm's chain."""
    rng = np.random.default_rng(M)
    D, F, Ds, Fs = 1001, 333, 1008, 672
    up = linear.upload_weight_f8(gpu, (rng.standard_normal((2 * F, D)) * 0.04).astype(np.float32))
    down = linear.upload_weight_f8(gpu, (rng.standard_normal((D, F)) * 0.04).astype(np.float32), rng.standard_normal(D))
    last = linear.upload_weight_f8(gpu, (rng.standard_normal((D, D)) * 0.04).astype(np.float32))
    a = linear.BlockScaledLinear(gpu, up, M, out_stride=Fs)
    b = linear.BlockScaledLinear(gpu, down, M, swiglu_in=True, out_stride=Ds)
    c = linear.BlockScaledLinear(gpu, last, M, out_dtype="f32")
    gain = gpu.upload(np.ones(D, np.float32))
    rows = np.full((M, Ds), 7.0, np.float32)                 # what lies behind the rows does not matter, and stays
    rows[:, :D] = rng.standard_normal((M, D))
    x = gpu.upload(quant.bf16_bits(rows))
    h0 = quant.bf16_to_f32(x.numpy())[:, :D]
    y = b(a.normed(x, gain, eps=1e-6, x_stride=Ds), x_stride=Fs)
    out = c.normed(x, gain, eps=1e-6, x_stride=Ds, y=y, y_stride=Ds)
    gpu.wait()

    def product(layer, wt, K):
        want, S = f8_ref.product(layer.codes.numpy(), layer.sa.numpy(), wt.w.numpy(), wt.sw.numpy(), K,
                                 wt.bias.numpy() if wt.bias is not None else None)
        return want, 2e-5 * S

    def coded(layer, v, K):
        s = f8_ref.spread(layer.sa.numpy().astype(np.float64), K)
        back = quant.e4m3_to_f32(layer.codes.numpy()[:, :K]) * s
        assert np.all(np.abs(back - v) <= (2.0 ** -4 + 2.0 ** -20) * np.abs(v) + 2.0 ** -10 * s)

    coded(a, f8_ref.norm_rows(h0, np.ones(D), 1e-6), D)
    mid = quant.bf16_to_f32(a.out.numpy())
    want, tol = product(a, up, D)
    assert np.all(np.abs(mid[:, :2 * F] - want) <= 2.0 ** -8 * np.abs(want) + tol) and (mid[:, 2 * F:] == 0).all()
    coded(b, f8_ref.gated_rows(mid, F), F)
    want, tol = product(b, down, F)
    yv = quant.bf16_to_f32(y.numpy())[:, :D]
    assert np.all(np.abs(yv - want) <= 2.0 ** -8 * np.abs(want) + tol)
    kept = quant.bf16_to_f32(x.numpy())
    h = quant.bf16_to_f32(quant.bf16_bits(h0 + yv))
    assert np.array_equal(kept[:, :D], h) and (kept[:, D:] == 7.0).all()
    coded(c, f8_ref.norm_rows(h, np.ones(D), 1e-6), D)
    want, tol = product(c, last, D)
    assert np.all(np.abs(out.numpy() - want) <= 2.0 ** -24 * np.abs(want) + tol)


@pytest.mark.gpu
def test_rows_off_their_boundary_are_refused(gpu):
    from h3metal_b200.gpu import GpuError
    wt = linear.upload_weight_f8(gpu, np.zeros((64, 1001), np.float32))
    layer = linear.BlockScaledLinear(gpu, wt, 4)
    gain = gpu.upload(np.ones(1001, np.float32))
    n = gpu.launch_count
    with pytest.raises(GpuError, match="16-byte"):
        layer.normed(gpu.empty((4, 1001), "bf16"), gain, eps=1e-6)
    with pytest.raises(GpuError, match="16-byte"):
        layer(gpu.empty((4, 1001), "bf16"))
    assert gpu.launch_count == n
