"""The int8 product's staged (TMA) stores where N is no multiple of eight: TMA writes whole 16-byte pieces of a row, so such
outputs must take the other way out and leave the columns behind N alone."""
import numpy as np
import pytest

from h3metal_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [412, 516, 1003])
@pytest.mark.parametrize("out_dtype", ["bf16", "f16"])
def test_columns_behind_n_are_left_alone(gpu, request, N, out_dtype):
    rng = np.random.default_rng(N)
    M, K, stride = 512, 256, -(-N // 8) * 8 + 8
    a, w = rng.integers(-127, 128, (M, K), dtype=np.int8), rng.integers(-127, 128, (N, K), dtype=np.int8)
    sa, sw = rng.uniform(0.001, 0.01, M).astype(np.float32), rng.uniform(0.001, 0.01, N).astype(np.float32)
    wt = ops.QWeight("q8", gpu.upload(w), gpu.upload(sw), N, K)
    A, S = gpu.upload(a), gpu.upload(sa)
    outs = []
    request.addfinalizer(gpu.set_policy)
    request.addfinalizer(gpu.set_store_mode)
    gpu.set_policy(pair=1)
    for mode in (1, -1):
        gpu.set_store_mode(mode)
        out = gpu.upload(np.full((M, stride), 3, np.uint16), out_dtype)
        ops.gemm(gpu, A, wt, out, M, sa=S, c_stride=stride, tile=(128, 1, 4))
        gpu.wait()
        outs.append(out.torch().view(__import__("torch").int16).cpu().numpy())
    assert (outs[0][:, N:] == 3).all()
    assert np.array_equal(outs[0], outs[1])
