"""Calls of the block-scaled entries that the library turns down before it launches anything."""
import pytest

from h3metal_b200.gpu import GpuError

pytestmark = pytest.mark.gpu


@pytest.fixture
def rows(gpu):
    M, D = 4, 256
    return dict(M=M, D=D, x=gpu.empty((M, 2 * D), "bf16"), w=gpu.empty((D,), "f32"), out=gpu.empty((M, D), "f8"),
                sa=gpu.empty((3, M), "f32"))


def refused(gpu, call):
    n = gpu.launch_count
    with pytest.raises(GpuError):
        call()
    assert gpu.launch_count == n


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_scales_off_their_alignment(gpu, rows, offset):
    M, D, x, w, out = (rows[k] for k in ("M", "D", "x", "w", "out"))
    sa = rows["sa"].view((12 * M,), "u8").view((8 * M,), "u8", offset).view((2, M), "f32")
    assert sa.ptr % 4 == offset
    refused(gpu, lambda: gpu.quant_f8_native(x, D, out, D, sa, M, M, D, 0))
    refused(gpu, lambda: gpu.rms_f8_native(x, D, None, 0, None, 0, w, out, D, sa, M, M, D, 1e-6))


def test_more_channels_than_a_launch_covers(gpu, rows):
    """Turned down by its size alone: the buffers behind the pointers are never touched."""
    x, out, sa = rows["x"], rows["out"], rows["sa"]
    with pytest.raises(GpuError, match="channels one launch covers"):
        gpu.quant_f8_native(x, 2 ** 28, out, 2 ** 28, sa, 1, 1, 2 ** 28 - 4095, 0)
    refused(gpu, lambda: gpu.quant_f8_native(x, 2 ** 28, out, 2 ** 28, sa, 1, 1, 2 ** 28, 0))
