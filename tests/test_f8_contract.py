"""The rounding that the block-scaled format promises: codes are e4m3(v * (1 / s)) in fp32 steps, which is the nearest code to
v / s except where v / s lies within 2^-23 of itself of the middle between two codes - there it is one of the two."""
import os

import numpy as np
import pytest

from h3metal_b200 import quant

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rows(dtype, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((400, 128)) * np.exp(rng.uniform(-3, 3, (400, 1)))).astype(np.float32)
    if dtype == "bf16":
        return quant.bf16_to_f32(quant.bf16_bits(x))
    return x.astype({"f16": np.float16, "f32": np.float32}[dtype]).astype(np.float32)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_codes_differ_from_the_division_at_middles_only(dtype):
    v = rows(dtype, 1)
    s = (np.abs(v).max(1, keepdims=True) / np.float32(448)).astype(np.float32)
    codes = quant.f8_codes(v, s)
    exact = v.astype(np.float64) / s.astype(np.float64)          # 24-bit numbers: the quotient to 2^-53
    grid = quant.e4m3_to_f32(np.arange(127, dtype=np.uint8)).astype(np.float64)
    middles = (grid[1:] + grid[:-1]) / 2
    got = quant.e4m3_to_f32(codes).astype(np.float64)
    nearest = grid[np.abs(np.abs(exact)[..., None] - grid).argmin(-1)] * np.sign(exact)
    off = np.abs(got) != np.abs(nearest)
    if dtype == "bf16":
        assert off.any()                                         # values of 8 bits do meet middles
    for q, c in zip(np.abs(exact[off]), np.abs(got[off])):
        mid = middles[np.abs(middles - q).argmin()]
        assert abs(q - mid) <= 2.0 ** -23 * (1 + 2.0 ** -24) * q
        i = np.flatnonzero(grid == c)[0]
        assert mid in (middles[i - 1] if i else None, middles[min(i, 125)])
    # two roundings of 2^-24 (2^-23 of q and a term in 2^-48) move the quotient, then half a step of e4m3
    half = np.maximum(2.0 ** -4 * np.abs(exact) * (1 + 2.0 ** -22), 2.0 ** -10)
    assert (np.abs(got - exact) <= half + 2.0 ** -23 * (1 + 2.0 ** -24) * np.abs(exact)).all()


def test_the_header_states_the_rounding_that_the_kernels_use():
    text = open(os.path.join(ROOT, "include", "h3b200.h")).read()
    kernel = open(os.path.join(ROOT, "h3metal_b200", "csrc", "rows_f8.cu")).read()
    for s in (text, kernel):
        assert "e4m3(v / s)" not in s
    assert "code = e4m3(v * r)" in text and "e4m3(v * (1 / s))" in kernel
