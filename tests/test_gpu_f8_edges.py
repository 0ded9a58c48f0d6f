"""Calls of the block-scaled operators that the documentation allows and that are easy to get wrong: slices, odd bases, long
strides, aliased buffers, profile mode. Tolerances as in test_gpu_f8_rows and test_gpu_f8_gemm."""
import numpy as np
import pytest

from h3metal_b200 import ops, quant
from oracle import f8_ref
from tests.test_gpu_f8_gemm import exact_case
from tests.test_gpu_f8_rows import NORM_TOL, as_type, buffers, check, guards_kept

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [3, 40, 200, 600])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_product_into_an_unaligned_slice(gpu, M, dtype):
    """C starts one element into its buffer, the bias one element into its own; nothing around them changes."""
    rng = np.random.default_rng(M)
    N, K, stride = 520, 512, 523
    a, sa, w, sw = exact_case(rng, M, N, K)
    bias = rng.integers(-8, 9, N + 1).astype(np.float32)
    want, _ = f8_ref.product(a, sa, w, sw, K, bias[1:])
    fill = np.full((M + 1, stride), 3, {"bf16": np.uint16, "f16": np.float16, "f32": np.float32}[dtype])
    out, b = gpu.upload(fill), gpu.upload(bias)
    wt = ops.QWeight("f8", gpu.upload(w, "f8"), gpu.upload(sw), N, K, bias=b.view((N,), offset_elems=1))
    c = out.view((M * stride,), offset_elems=1)
    ops.gemm_f8(gpu, gpu.upload(a, "f8"), wt, c, M, sa=gpu.upload(sa), c_stride=stride)
    gpu.wait()
    raw = out.numpy()
    got = raw[:M, 1:N + 1]
    got = quant.bf16_to_f32(got) if dtype == "bf16" else got.astype(np.float32)
    half = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 0.0}[dtype]  # sums are exact, the store rounds once
    assert np.all(np.abs(got - want) <= half * np.abs(want))
    assert (raw[:M, 0] == 3).all() and (raw[:M, N + 1:] == 3).all() and (raw[M] == 3).all()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_product_over_a_slice_of_k(gpu, M):
    """Whole groups [g0, g1) of wider codes: A, W and both scales as views into the full tensors."""
    rng = np.random.default_rng(M)
    N, K, g0, g1 = 384, 2048, 3, 11
    a, sa, w, sw = exact_case(rng, M, N, K)
    k0, k1 = g0 * 128, g1 * 128
    want, _ = f8_ref.product(a[:, k0:k1], sa[g0:g1], w[:, k0:k1], sw[:, g0:g1], k1 - k0)
    A, S, W, SW = gpu.upload(a, "f8"), gpu.upload(sa), gpu.upload(w, "f8"), gpu.upload(np.ascontiguousarray(sw[:, g0:g1]))
    out = gpu.empty((M, N), "f32")
    wt = ops.QWeight("f8", W.view((N * K - k0,), offset_elems=k0), SW, N, k1 - k0, ws=K)
    ops.gemm_f8(gpu, A.view((M * K - k0,), offset_elems=k0), wt, out, M, sa=S.row(g0, g1 - g0), a_stride=K)
    gpu.wait()
    assert np.array_equal(out.numpy(), want.astype(np.float32))


def test_rows_and_results_more_than_2_to_31_elements_apart(gpu):
    import torch
    rng = np.random.default_rng(0)
    far = 2 ** 31 + 64
    dev = gpu.torch_device
    M, D = 2, 256
    xv = rng.standard_normal((M, D)).astype(np.float32)
    bits, vals = as_type(xv, "bf16")

    def spread_out(rows, dtype):
        t = torch.zeros(far + 4096, dtype=dtype, device=dev)
        for m in range(M):
            t[m * far:m * far + rows.shape[1]] = torch.from_numpy(rows[m]).to(dev).view(dtype)
        return t

    x = spread_out(bits.view(np.int16), torch.bfloat16)
    codes = torch.zeros(far + 4096, dtype=torch.float8_e4m3fn, device=dev)
    sa = gpu.empty((2, M), "f32")
    X, C = gpu.wrap(x), gpu.wrap(codes)
    ops.quant_f8(gpu, X, C, sa, M, D, x_stride=far, out_stride=far)
    gpu.wait()
    got = np.stack([codes[m * far:m * far + D].view(torch.uint8).cpu().numpy() for m in range(M)])
    check(vals.astype(np.float64), got, sa.numpy(), D, 0.0)
    # the norm reads the same rows, adds, keeps the sum as far apart
    w = gpu.upload(np.ones(D, np.float32))
    ops.rms_f8(gpu, X, w, C, sa, M, D, eps=1e-6, y=X, x_stride=far, y_stride=far, res_stride=far, out_stride=far)
    gpu.wait()
    _, h = as_type(vals + vals, "bf16")
    kept = np.stack([x[m * far:m * far + D].float().cpu().numpy() for m in range(M)])
    assert np.array_equal(kept, h)
    got = np.stack([codes[m * far:m * far + D].view(torch.uint8).cpu().numpy() for m in range(M)])
    check(f8_ref.norm_rows(h, np.ones(D), 1e-6), got, sa.numpy(), D, NORM_TOL)
    # the product reads those codes and writes fp32 rows that far apart
    wc, sw = quant.quant_f8((rng.standard_normal((48, D)) * 0.02).astype(np.float32))
    wt = ops.QWeight("f8", gpu.upload(wc, "f8"), gpu.upload(sw), 48, D)
    del x, X
    out = torch.zeros(far + 4096, dtype=torch.float32, device=dev)
    ops.gemm_f8(gpu, C, wt, gpu.wrap(out), M, sa=sa, a_stride=far, c_stride=far)
    gpu.wait()
    want, S = f8_ref.product(got, sa.numpy(), wc, sw, D)
    res = np.stack([out[m * far:m * far + 48].cpu().numpy() for m in range(M)])
    assert np.all(np.abs(res - want) <= 2e-5 * S)


def test_the_sum_may_go_where_either_addend_was(gpu):
    rng = np.random.default_rng(1)
    M, D = 400, 1280  # more rows than CTAs of one wave have: a row is fetched while the one before is written
    x, y = rng.standard_normal((M, D)).astype(np.float32), rng.standard_normal((M, D)).astype(np.float32)
    w = gpu.upload(np.ones(D, np.float32))
    results = []
    for where in ("own", "x", "y"):
        X, Y = gpu.upload(x), gpu.upload(y)
        res = {"own": gpu.empty((M, D), "f32"), "x": X, "y": Y}[where]
        out, sa = buffers(gpu, M, D)
        ops.rms_f8(gpu, X, w, out, sa, M, D, eps=1e-6, y=Y, res=res)
        gpu.wait()
        assert np.array_equal(res.numpy(), x + y)
        results.append(guards_kept(out, sa, M, D))
    for codes, scales in results[1:]:
        assert np.array_equal(codes, results[0][0]) and np.array_equal(scales, results[0][1])


@pytest.mark.parametrize("offset", [8, 16])
def test_rows_on_16_byte_boundaries_give_the_same_as_on_32(gpu, offset):
    rng = np.random.default_rng(2)
    M, D, stride = 300, 1024, 1048  # a stride of 16-byte but not 32-byte pieces
    x = rng.standard_normal((M, D)).astype(np.float32)
    bits, vals = as_type(x, "bf16")
    wide = np.zeros(M * stride + 64, np.uint16)
    for m in range(M):
        wide[offset + m * stride:offset + m * stride + D] = bits[m]
    X = gpu.upload(wide).view((M * stride,), offset_elems=offset)
    straight, ss = buffers(gpu, M, D)
    out, sa = buffers(gpu, M, D)
    ops.quant_f8(gpu, gpu.upload(bits), straight, ss, M, D)
    ops.quant_f8(gpu, X, out, sa, M, D, x_stride=stride)
    gpu.wait()
    assert np.array_equal(out.numpy(), straight.numpy()) and np.array_equal(sa.numpy(), ss.numpy())
    w = gpu.upload(np.ones(D, np.float32))
    ops.rms_f8(gpu, gpu.upload(bits), w, straight, ss, M, D, eps=1e-6)
    ops.rms_f8(gpu, X, w, out, sa, M, D, eps=1e-6, x_stride=stride)
    gpu.wait()
    assert np.array_equal(out.numpy(), straight.numpy()) and np.array_equal(sa.numpy(), ss.numpy())


def test_profile_mode_names_every_launch(gpu):
    M, D, N = 4, 256, 128
    x, w, out, sa = gpu.empty((M, D), "bf16"), gpu.empty((D,), "f32"), gpu.empty((M, D), "f8"), gpu.empty((2, M), "f32")
    wt = ops.QWeight("f8", gpu.empty((N, D), "f8"), gpu.empty((1, 2), "f32"), N, D)
    gpu.wait()
    gpu.profile(True)
    try:
        ops.rms_f8(gpu, x, w, out, sa, M, D, eps=1e-6, y=x)
        ops.quant_f8(gpu, x, out, sa, M, D // 2, swiglu=True, out_stride=D)
        ops.gemm_f8(gpu, out, wt, gpu.empty((M, N), "f32"), M, sa=sa)
        took = gpu.profile_take()
    finally:
        gpu.profile(False)
    assert [n for n, _ in took] == ["rms_f8(256,add)", "quant_f8(128,swiglu)", "gemm(f8,256->128)"]
    assert all(s > 0 for _, s in took)


def test_a_chain_without_launch_overlap_gives_the_same(gpu, request):
    """Programmatic launches read nothing before the kernel ahead has finished: turned off, the bits are the same."""
    from h3metal_b200 import linear
    rng = np.random.default_rng(4)
    M, D = 24, 768
    wt = linear.upload_weight_f8(gpu, (rng.standard_normal((D, D)) * 0.05).astype(np.float32))
    layers = [linear.BlockScaledLinear(gpu, wt, M) for _ in range(4)]
    gain = gpu.upload(np.ones(D, np.float32))
    start = quant.bf16_bits(rng.standard_normal((M, D)).astype(np.float32))
    request.addfinalizer(lambda: gpu.set_launch_overlap(True))
    outs = []
    for on in (True, False, True):
        gpu.set_launch_overlap(on)
        x = gpu.upload(start)
        y = None
        for layer in layers:
            y = layer.normed(x, gain, eps=1e-6, y=y)
        gpu.wait()
        outs.append((x.numpy(), y.numpy()))
    for x, y in outs[1:]:
        assert np.array_equal(x, outs[0][0]) and np.array_equal(y, outs[0][1])
