"""Block-scaled layers in the weight container: what is written can be read back."""
import numpy as np
import pytest

from h3metal_b200 import quant, weights
from tests.fakes import RecordingGpu


@pytest.mark.parametrize("N,K", [(1, 1), (24, 512), (130, 1001)])
def test_round_trip(tmp_path, N, K):
    rng = np.random.default_rng(N + K)
    codes, scales = quant.quantize("f8", (rng.standard_normal((N, K)) * 0.02).astype(np.float32))
    bias = rng.standard_normal(N).astype(np.float32)
    path = str(tmp_path / "w.h3m")
    w = weights.Writer(path, {})
    w.linear("a", "f8", N, K, codes, scales, bias=bias)
    w.linear("b", "f8", N, K, codes.view(np.int8), scales)
    w.close()
    wf = weights.WeightFile(RecordingGpu(), path)
    a, b = wf.linear("a"), wf.linear("b")
    assert (a.fmt, a.N, a.K, a.w.dtype, a.sw.dtype) == ("f8", N, K, "f8", "f32") and b.bias is None
    for lin in (a, b):
        assert lin.w.shape == codes.shape and lin.sw.shape == scales.shape
        assert np.array_equal(lin.w.numpy(), codes) and np.array_equal(lin.sw.numpy(), scales)
    assert np.array_equal(a.bias.numpy(), bias) and wf.linear("a").w is a.w


def test_codes_and_scales_of_other_shapes_are_refused(tmp_path):
    codes, scales = quant.quantize("f8", np.ones((130, 1001), np.float32))
    w = weights.Writer(str(tmp_path / "w.h3m"), {})
    for args in ((130, 990, codes, scales), (129, 1001, codes, scales), (130, 1001, codes[:, :1001], scales),
                 (130, 1001, codes, scales[:1]), (130, 1001, codes, None), (130, 1001, codes, scales.reshape(-1)),
                 (130, 1001, codes.astype(np.float32), scales)):
        with pytest.raises(ValueError):
            w.linear("a", "f8", *args)
    with pytest.raises(ValueError):
        w.linear("a", "f8", 130, 1001, codes, scales, G=64)
    assert not w.entries


@pytest.mark.gpu
def test_a_layer_read_back_multiplies(gpu, tmp_path):
    from h3metal_b200 import linear
    rng = np.random.default_rng(0)
    N, K, M = 300, 512, 5
    values = (rng.standard_normal((N, K)) * 0.02).astype(np.float32)
    path = str(tmp_path / "w.h3m")
    w = weights.Writer(path, {})
    w.linear("a", "f8", N, K, *quant.quantize("f8", values))
    w.close()
    x = gpu.upload(rng.standard_normal((M, K)).astype(np.float32))
    outs = [linear.BlockScaledLinear(gpu, wt, M, out_dtype="f32")(x).numpy()
            for wt in (linear.upload_weight_f8(gpu, values), weights.WeightFile(gpu, path).linear("a"))]
    assert np.array_equal(outs[0], outs[1]) and np.abs(outs[0]).max() > 0
