"""Block-scaled calls one behind the other on the same buffers, without a wait in between: each reads what the one ahead wrote,
also where its launch overlaps the end of that one."""
import numpy as np
import pytest

from h3metal_b200 import linear, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 24, 100, 300, 700])
def test_one_scale_buffer_for_changing_inputs(gpu, request, M):
    """quant_f8 and gemm_f8 in turn, forty times over one buffer of codes and one of scales, the inputs 2^0 .. 2^39 apart: an
    output that used a scale of the call before would be off by a factor."""
    rng = np.random.default_rng(M)
    N, K, turns = 512, 1024, 40
    wt = linear.upload_weight_f8(gpu, (rng.standard_normal((N, K)) * 0.05).astype(np.float32))
    base = rng.standard_normal((M, K)).astype(np.float32)
    xs = [gpu.upload(base * np.float32(2.0 ** (t - 20))) for t in range(turns)]
    codes, sa = gpu.empty((M, K), "f8"), gpu.empty((K // 128, M), "f32")
    outs = [gpu.empty((M, N), "f32") for _ in range(turns)]
    request.addfinalizer(lambda: gpu.set_launch_overlap(True))
    got = {}
    for on in (False, True):
        gpu.set_launch_overlap(on)
        for o in outs:
            o.torch().fill_(-1.0)
        for x, o in zip(xs, outs):
            ops.quant_f8(gpu, x, codes, sa, M, K)
            ops.gemm_f8(gpu, codes, wt, o, M, sa=sa)
        gpu.wait()
        got[on] = [o.numpy() for o in outs]
    for t in range(turns):
        assert np.array_equal(got[True][t], got[False][t])
        # powers of two: the same codes, scales and sums that much larger, exactly
        assert np.array_equal(got[False][t], got[False][0] * np.float32(2.0 ** t))


@pytest.mark.parametrize("M", [2, 200])
def test_norm_and_product_share_one_scale_buffer(gpu, request, M):
    rng = np.random.default_rng(M)
    D, turns = 640, 30
    wt = linear.upload_weight_f8(gpu, (rng.standard_normal((D, D)) * 0.05).astype(np.float32))
    layer = linear.BlockScaledLinear(gpu, wt, M, out_dtype="f32")
    gain = gpu.upload(np.ones(D, np.float32))
    start = rng.standard_normal((M, D)).astype(np.float32)
    request.addfinalizer(lambda: gpu.set_launch_overlap(True))
    ends = []
    for on in (False, True):
        gpu.set_launch_overlap(on)
        x, y = gpu.upload(start), None
        for _ in range(turns):  # the layer's own output is added to the stream that its next call norms
            y = layer.normed(x, gain, eps=1e-6, y=y)
        gpu.wait()
        ends.append((x.numpy(), y.numpy()))
    assert np.isfinite(ends[0][1]).all()
    assert np.array_equal(ends[0][0], ends[1][0]) and np.array_equal(ends[0][1], ends[1][1])
