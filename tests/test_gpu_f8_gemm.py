"""gemm_f8 on the GPU against the definition in 64 bits, and the block-scaled layers run together.

Two kinds of data. Exact: codes that are small whole numbers and scales that are powers of two, chosen so that every
partial sum is a whole multiple of the smallest product below 2^24 of it - exact in fp32 in any order - and fp32
results must agree bit for bit. Random: a group's 128 products are added by the tensor core in fp32, four
instructions of 32; with S the sum of the magnitudes, 33 truncations of a whole step per instruction bound a group's error
by 4 * 33 * 2^-23 * S, and the scales' product, the running sum over G groups and the bias add (G + 3) * 2^-24 * S; the
result's own rounding is half a step of its type."""
import numpy as np
import pytest

from h3metal_b200 import linear, ops, quant
from oracle import f8_ref

pytestmark = pytest.mark.gpu

STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def store(v, dtype):
    return quant.bf16_to_f32(v) if dtype == "bf16" else v.astype(np.float32)


def exact_case(rng, M, N, K):
    """Codes -2..2 with scales 1, 2 or 4 (activations) and 1/2, 1 (weights): every product is a multiple of 1/2, and the sum
    of K <= 16384 of at most 16 in magnitude stays below 2^18: 19 bits."""
    G = -(-K // 128)
    stride = quant.f8_stride(K)
    a = np.full((M, stride), 0x7F, np.uint8)   # NaN codes behind the row's end: they must not be read
    w = np.full((N, stride), 0x7F, np.uint8)
    a[:, :K] = quant.e4m3_bits(rng.integers(-2, 3, (M, K)))
    w[:, :K] = quant.e4m3_bits(rng.integers(-2, 3, (N, K)))
    sa = 2.0 ** rng.integers(0, 3, (G, M)).astype(np.float32)
    sw = 2.0 ** rng.integers(-1, 1, (-(-N // 128), G)).astype(np.float32)
    return a, sa, w, sw


def random_case(rng, M, N, K):
    x = (rng.standard_normal((M, K)) * np.exp(rng.uniform(-2, 2, (M, 1)))).astype(np.float32)
    x[:, ::61] *= 20
    s = f8_ref.scales(x.astype(np.float64)).astype(np.float32)
    a = np.zeros((M, quant.f8_stride(K)), np.uint8)
    a[:, :K] = quant.e4m3_bits(x / f8_ref.spread(s, K))
    w, sw = quant.quant_f8((rng.standard_normal((N, K)) * 0.02).astype(np.float32))
    return a, s, w, sw


def run(gpu, a, sa, w, sw, M, N, K, dtype, bias=None, c_stride=None, sa_stride=None):
    c_stride, sa_stride = c_stride or N, sa_stride or M
    out = gpu.upload(np.full((M + 2, c_stride), 3, {"bf16": np.uint16, "f16": np.float16, "f32": np.float32}[dtype]))
    full = np.full((sa.shape[0], sa_stride), np.nan, np.float32)  # scales of rows that do not exist: not to be used
    full[:, :M] = sa
    wt = ops.QWeight("f8", gpu.upload(w, "f8"), gpu.upload(sw), N, K, bias=gpu.upload(bias) if bias is not None else None)
    ops.gemm_f8(gpu, gpu.upload(a, "f8"), wt, out, M, sa=gpu.upload(full), sa_stride=sa_stride, c_stride=c_stride)
    gpu.wait()
    raw = out.numpy()
    assert (raw[M:] == 3).all() and (raw[:, N:] == 3).all()
    return store(raw[:M, :N], dtype)


# from one value to several tiles of every kernel; ends inside tiles, instructions, groups and 16-byte pieces
SIZES = [(1, 1, 1), (1, 128, 128), (1, 300, 1000), (2, 129, 127), (5, 64, 3840), (16, 256, 129), (17, 130, 2048), (32, 384, 640),
         (33, 1000, 400), (64, 512, 1024), (65, 257, 777), (100, 771, 1000), (128, 128, 16384), (129, 640, 256), (255, 256, 128),
         (256, 256, 384), (257, 513, 1040), (300, 1280, 512), (700, 700, 300), (1024, 512, 256), (1100, 2304, 640),
         (2600, 2304, 300), (20, 11400, 3840), (64, 9000, 640), (7, 20000, 384), (24, 2048, 8192), (160, 1024, 2048)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_exact_sums(gpu, M, N, K):
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    a, sa, w, sw = exact_case(rng, M, N, K)
    bias = rng.integers(-8, 9, N).astype(np.float32)
    want, _ = f8_ref.product(a, sa, w, sw, K, bias)
    got = run(gpu, a, sa, w, sw, M, N, K, "f32", bias, c_stride=N + 5, sa_stride=M + 7)
    assert np.array_equal(got, want.astype(np.float32))


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_random_values(gpu, M, N, K, dtype):
    rng = np.random.default_rng(M + N + K)
    a, sa, w, sw = random_case(rng, M, N, K)
    bias = None if M % 2 else (rng.standard_normal(N) * 0.1).astype(np.float32)
    want, S = f8_ref.product(a, sa, w, sw, K, bias)
    got = run(gpu, a, sa, w, sw, M, N, K, dtype, bias, c_stride=-(-N // 8) * 8)
    groups = -(-K // 128)
    tol = (4 * 33 * 2.0 ** -23 + (groups + 3) * 2.0 ** -24) * S
    err = np.abs(got - want)
    print(f"largest error / sum of magnitudes: {np.max(np.maximum(0, err - STEP[dtype] * np.abs(want)) / S):.2e}")
    assert np.all(err <= tol * (1 + STEP[dtype]) + STEP[dtype] * np.abs(want) + 2.0 ** -24 * (dtype == "f16"))


def test_results_do_not_vary(gpu):
    rng = np.random.default_rng(9)
    M, N, K = 40, 640, 4096
    a, sa, w, sw = random_case(rng, M, N, K)
    first = run(gpu, a, sa, w, sw, M, N, K, "f32")
    for _ in range(3):
        assert np.array_equal(run(gpu, a, sa, w, sw, M, N, K, "f32"), first)


def test_nan_and_infinite_scales_stay_in_their_rows(gpu):
    rng = np.random.default_rng(10)
    M, N, K = 20, 256, 512
    a, sa, w, sw = exact_case(rng, M, N, K)
    want, _ = f8_ref.product(a, sa, w, sw, K)
    a[3, 5] = 0x7F
    sa[1, 7] = np.inf
    got = run(gpu, a, sa, w, sw, M, N, K, "f32")
    assert np.isnan(got[3]).all() and not np.isfinite(got[7]).any()
    keep = [m for m in range(M) if m not in (3, 7)]
    assert np.array_equal(got[keep], want[keep].astype(np.float32))


@pytest.mark.parametrize("M", [1, 24, 300])
def test_captured_and_replayed_on_another_stream(gpu, M):
    """norm -> product -> gated quantiser -> product of a block's MLP, eager, then captured once and replayed on new inputs."""
    import torch
    rng = np.random.default_rng(M)
    D, F = 640, 1000
    up = linear.upload_weight_f8(gpu, (rng.standard_normal((2 * F, D)) * 0.04).astype(np.float32))
    down = linear.upload_weight_f8(gpu, (rng.standard_normal((D, F)) * 0.04).astype(np.float32), rng.standard_normal(D))
    gain = gpu.upload((1 + 0.1 * rng.standard_normal(D)).astype(np.float32))
    first, second = linear.BlockScaledLinear(gpu, up, M), linear.BlockScaledLinear(gpu, down, M, swiglu_in=True)
    x, y = gpu.empty((M, D), "f32"), gpu.empty((M, D), "bf16")
    kept = gpu.empty((M, D), "f32")

    def step():
        second(first.normed(x, gain, eps=1e-6, y=y, res=kept))

    def fill(seed):
        r = np.random.default_rng(seed)
        xv, yv = r.standard_normal((M, D)).astype(np.float32), quant.bf16_bits(r.standard_normal((M, D)).astype(np.float32))
        x.torch().copy_(torch.from_numpy(xv))
        y.torch().copy_(torch.from_numpy(yv.view(np.int16)).view(torch.bfloat16))
        return xv, quant.bf16_to_f32(yv)

    xv, yv = fill(1)
    step()
    gpu.wait()
    eager = second.out.numpy().copy()
    # against the same chain in 64 bits from the codes each step left behind: no step sees another's rounding
    h = kept.numpy()
    assert np.array_equal(h, xv + yv)
    mid, S = f8_ref.product(first.codes.numpy(), first.sa.numpy(), up.w.numpy(), up.sw.numpy(), D)
    got = quant.bf16_to_f32(first.out.numpy())
    assert np.all(np.abs(got - mid) <= 2.0 ** -8 * np.abs(mid) + 2e-5 * S)
    # the norm's factor and the gate are computed to 49 * 2^-24 (test_gpu_f8_rows): well inside 2^-20
    for layer, v, K in ((first, f8_ref.norm_rows(h, gain.numpy(), 1e-6), D), (second, f8_ref.gated_rows(got, F), F)):
        s = f8_ref.spread(layer.sa.numpy().astype(np.float64), K)
        back = quant.e4m3_to_f32(layer.codes.numpy()[:, :K]) * s
        assert np.all(np.abs(back - v) <= (2.0 ** -4 + 2.0 ** -20) * np.abs(v) + 2.0 ** -10 * s)
    want, S = f8_ref.product(second.codes.numpy(), second.sa.numpy(), down.w.numpy(), down.sw.numpy(), F, down.bias.numpy())
    assert np.all(np.abs(quant.bf16_to_f32(eager) - want) <= 2.0 ** -8 * np.abs(want) + 2e-5 * S)

    side = torch.cuda.Stream(gpu.torch_device)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            gpu.use_stream(side)
            step()
    finally:
        gpu.use_stream(None)
    outs = {}
    for seed in (2, 1, 2):
        fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        outs.setdefault(seed, []).append(second.out.numpy().copy())
    assert np.array_equal(outs[1][0], eager)
    assert np.array_equal(outs[2][0], outs[2][1]) and not np.array_equal(outs[2][0], eager)
    step()  # and eager again: the context is none the worse for the capture
    assert gpu.wait() >= 0
    assert np.array_equal(second.out.numpy(), outs[2][0])
    del graph


def test_two_streams_at_once(gpu):
    """Two chains on streams of their own share nothing but the weight."""
    import torch
    rng = np.random.default_rng(3)
    M, N, K = 8, 2048, 4096
    cases = [random_case(rng, M, 1, K)[:2] for _ in range(2)]
    w, sw = quant.quant_f8((rng.standard_normal((N, K)) * 0.02).astype(np.float32))
    wt = ops.QWeight("f8", gpu.upload(w, "f8"), gpu.upload(sw), N, K)
    ins = [(gpu.upload(a, "f8"), gpu.upload(s)) for a, s in cases]
    outs = [gpu.empty((M, N), "f32") for _ in ins]
    streams = [torch.cuda.Stream(gpu.torch_device) for _ in ins]
    torch.cuda.synchronize()
    try:
        for _ in range(20):
            for (a, s), o, st in zip(ins, outs, streams):
                gpu.use_stream(st)
                ops.gemm_f8(gpu, a, wt, o, M, sa=s)
        torch.cuda.synchronize()
        gpu.wait()
    finally:
        gpu.use_stream(None)
    for (a, s), o in zip(cases, outs):
        want, S = f8_ref.product(a, s, w, sw, K)
        assert np.all(np.abs(o.numpy() - want) <= 2e-5 * S)


def test_refusals_of_the_library(gpu):
    from h3metal_b200.gpu import GpuError
    M, N, K = 4, 256, 256
    a, sa, w, sw = gpu.empty((M, K), "f8"), gpu.empty((2, M), "f32"), gpu.empty((N, K), "f8"), gpu.empty((2, 2), "f32")
    c = gpu.empty((M, N), "bf16")
    n = gpu.launch_count
    ok = dict(a=a, a_stride=K, sa=sa, sa_stride=M, w=w, w_stride=K, sw=sw, sw_stride=2, bias=None, out=c, c_stride=N, M=M, N=N, K=K)
    for change in (dict(M=0), dict(N=0), dict(K=0), dict(a_stride=K - 16), dict(a_stride=K + 8), dict(w_stride=K + 1), dict(c_stride=N - 1),
                   dict(sa_stride=M - 1), dict(sw_stride=1), dict(out=a), dict(a=a.view((M, K), offset_elems=8)),
                   dict(w=w.view((N, K), offset_elems=4))):
        with pytest.raises(GpuError):
            gpu.gemm_f8_native(**{**ok, **change})
    assert gpu.launch_count == n
