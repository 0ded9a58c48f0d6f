"""quant.quant_f8 where a weight holds NaN, infinities, zeros and the smallest magnitudes: as the kernels treat rows."""
import numpy as np

from h3metal_b200 import quant


def test_a_nan_spoils_its_own_place_only():
    rng = np.random.default_rng(0)
    w = (rng.standard_normal((200, 300)) * 0.02).astype(np.float32)
    clean_codes, clean_scales = quant.quant_f8(w)
    top = np.unravel_index(np.abs(w[:128, :128]).argmax(), (128, 128))
    at = (5, 7) if top != (5, 7) else (6, 7)
    w[at] = np.nan
    codes, scales = quant.quant_f8(w)
    assert np.array_equal(scales, clean_scales)
    assert codes[at] & 0x7F == 0x7F
    codes[at] = clean_codes[at]
    assert np.array_equal(codes, clean_codes)
    w[:128, 128:256] = np.nan                       # a block of nothing else: codes of NaN, a scale of one
    codes, scales = quant.quant_f8(w)
    assert scales[0, 1] == 1.0 and (codes[:128, 128:256] & 0x7F == 0x7F).all()


def test_infinities_and_the_smallest_magnitudes():
    w = np.ones((128, 512), np.float32)
    w[3, 130] = np.inf
    w[:, 256:384] = 0.0
    w[:, 384:] = 1e-45 * np.arange(128)
    with np.errstate(all="raise", under="ignore"):
        codes, scales = quant.quant_f8(w)
    assert list(scales[0]) == [np.float32(1) / np.float32(448), np.inf, 1.0, np.float32(2.0 ** -126)]
    with np.errstate(invalid="ignore"):
        back = quant.dequant("f8", codes, scales, 128, 512)
    assert np.isnan(back[:, 128:256]).all() and (back[:, 256:384] == 0).all() and np.isfinite(back[:, 384:]).all()
    # 2^-126 is the scale's floor: half a step among the subnormal codes is 2^-10 of it
    assert np.abs(back[:, 384:] - w[:, 384:]).max() <= 2.0 ** -136


def test_one_value_per_block():
    codes, scales = quant.quant_f8(np.full((1, 1), -3.5, np.float32))
    assert codes.shape == (1, 16) and codes[0, 0] == 0xFE and scales[0, 0] == np.float32(3.5) / np.float32(448)
