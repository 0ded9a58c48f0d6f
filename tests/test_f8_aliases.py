"""rms_f8 with the sum kept where an addend was: value by value in the same place, or not at all."""
import numpy as np
import pytest

from h3metal_b200 import ops
from tests.test_f8_host import F8Gpu


def tensors(g, M, D, y="bf16"):
    return (g.empty((M, 2 * D), "bf16"), g.empty((D,), "f32"), g.empty((M, D), "f8"), g.empty((2, M), "f32"), g.empty((M, 2 * D), y))


def test_other_row_strides_are_refused():
    g = F8Gpu()
    M, D = 4, 256
    x, w, out, sa, y = tensors(g, M, D)
    kw = dict(eps=1e-6, x_stride=2 * D, y=y, y_stride=2 * D)
    for res, stride in ((None, D), (x, D), (y, D), (x.view((M, 2 * D)), D)):
        with pytest.raises(ValueError, match="same place"):
            ops.rms_f8(g, x, w, out, sa, M, D, res=res, res_stride=stride, **kw)
    assert not g.calls
    for res in (None, x, y):
        ops.rms_f8(g, x, w, out, sa, M, D, res=res, res_stride=2 * D, **kw)
    ops.rms_f8(g, x, w, out, sa, 1, D, res=x, res_stride=D, **kw)             # one row has no stride
    assert [c["kind"] for c in g.calls] == ["rms"] * len(g.calls) and len(g.calls) == 4


@pytest.mark.parametrize("M", [1, 4])
def test_other_element_sizes_are_refused(M):
    g = F8Gpu()
    D = 256
    x, w, out, sa, y = tensors(g, M, D, "f32")
    with pytest.raises(ValueError, match="same place"):
        ops.rms_f8(g, x, w, out, sa, M, D, eps=1e-6, x_stride=2 * D, y=y, y_stride=2 * D, res=y.view((M, 2 * D), "bf16"),
                   res_stride=2 * D)
    assert not g.calls


@pytest.mark.gpu
def test_the_library_refuses_them_too(gpu):
    from h3metal_b200.gpu import GpuError
    M, D = 4, 256
    x, w, out, sa = gpu.empty((M, 2 * D), "bf16"), gpu.empty((D,), "f32"), gpu.empty((M, D), "f8"), gpu.empty((2, M), "f32")
    y, f = gpu.empty((M, 2 * D), "bf16"), gpu.empty((M, 2 * D), "f32")
    n = gpu.launch_count
    for yy, res, stride in ((y, x, D), (y, y, D), (f, f.view((M, 2 * D), "bf16"), 2 * D)):
        with pytest.raises(GpuError, match="same place"):
            gpu.rms_f8_native(x, 2 * D, yy, 2 * D, res, stride, w, out, D, sa, M, M, D, 1e-6)
    assert gpu.launch_count == n


@pytest.mark.gpu
def test_the_sum_beside_x_in_the_same_rows(gpu):
    """x in the left half of wide rows, the sum in the right half: memory apart, the same stride."""
    rng = np.random.default_rng(0)
    M, D = 300, 256
    x, y = rng.standard_normal((M, D)).astype(np.float32), rng.standard_normal((M, D)).astype(np.float32)
    wide = np.zeros((M, 2 * D), np.float32)
    wide[:, :D] = x
    X = gpu.upload(wide)
    right = X.view(((M - 1) * 2 * D + D,), offset_elems=D)
    out, sa, w = gpu.empty((M, D), "f8"), gpu.empty((2, M), "f32"), gpu.upload(np.ones(D, np.float32))
    ops.rms_f8(gpu, X, w, out, sa, M, D, eps=1e-6, x_stride=2 * D, y=gpu.upload(y), res=right, res_stride=2 * D)
    gpu.wait()
    got = X.numpy()
    assert np.array_equal(got[:, :D], x) and np.array_equal(got[:, D:], x + y)
