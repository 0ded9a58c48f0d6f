"""Every kernel that gemm_f8 chooses from, by name, at sizes that end inside its tiles, instructions, groups and 16-byte pieces.
Data and tolerances as in test_gpu_f8_gemm."""
import numpy as np
import pytest

from oracle import f8_ref
from tests.test_gpu_f8_gemm import STEP, exact_case, random_case, run

pytestmark = pytest.mark.gpu

# kernel -> (M, N, K): the few-row kernel by its rows per tile, 256 a CTA pair, 512 two pairs that share K
SIZES = [(16, 9, 300, 1000), (32, 31, 500, 900), (64, 50, 771, 640), (128, 100, 300, 2000),
         (256, 1100, 2304, 640), (256, 2600, 2309, 300),
         (512, 512, 3840, 1152), (512, 300, 3840, 1024), (512, 640, 2560, 2048), (512, 509, 3847, 1000), (512, 700, 2500, 1537),
         (512, 300, 2572, 2304), (512, 256, 3840, 3840)]


@pytest.mark.parametrize("kernel,M,N,K", SIZES)
def test_exact_sums(gpu, kernel, M, N, K):
    assert gpu.gemm_f8_kernel(M, N, K) == kernel
    rng = np.random.default_rng(M * 5 + N + K)
    a, sa, w, sw = exact_case(rng, M, N, K)
    bias = rng.integers(-8, 9, N).astype(np.float32)
    want, _ = f8_ref.product(a, sa, w, sw, K, bias)
    assert np.array_equal(run(gpu, a, sa, w, sw, M, N, K, "f32", bias, c_stride=N + 5, sa_stride=M + 7), want.astype(np.float32))
    assert np.array_equal(run(gpu, a, sa, w, sw, M, N, K, "f32", None, c_stride=-(-N // 4) * 4),
                          (want - bias).astype(np.float32))


@pytest.mark.parametrize("kernel,M,N,K", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_random_values(gpu, kernel, M, N, K, dtype):
    """N a multiple of eight in rows of whole 16-byte pieces goes out by TMA, the others by plain stores."""
    assert gpu.gemm_f8_kernel(M, N, K) == kernel
    rng = np.random.default_rng(M + N * 3 + K)
    a, sa, w, sw = random_case(rng, M, N, K)
    bias = (rng.standard_normal(N) * 0.1).astype(np.float32)
    want, S = f8_ref.product(a, sa, w, sw, K, bias)
    tol = (4 * 33 * 2.0 ** -23 + (-(-K // 128) + 3) * 2.0 ** -24) * S  # two pairs: one more addition, of the bias's kind
    for stride in (-(-N // 8) * 8, N + 1):
        got = run(gpu, a, sa, w, sw, M, N, K, dtype, bias, c_stride=stride)
        assert np.all(np.abs(got - want) <= tol * (1 + STEP[dtype]) + STEP[dtype] * np.abs(want) + 2.0 ** -24 * (dtype == "f16"))


@pytest.mark.parametrize("M,N,K", [(512, 3840, 1152), (300, 2572, 2304)])
def test_two_pairs_give_the_same_every_time(gpu, M, N, K):
    assert gpu.gemm_f8_kernel(M, N, K) == 512
    rng = np.random.default_rng(3)
    a, sa, w, sw = random_case(rng, M, N, K)
    first = run(gpu, a, sa, w, sw, M, N, K, "f32")
    for _ in range(5):
        assert np.array_equal(run(gpu, a, sa, w, sw, M, N, K, "f32"), first)


def test_sizes_that_are_refused(gpu):
    from h3metal_b200.gpu import GpuError
    for sizes in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(GpuError):
            gpu.gemm_f8_kernel(*sizes)
