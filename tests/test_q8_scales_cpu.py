"""Q8_0 scales of kv_write, amax * (1 / 127), against those of sessions, amax / 127: the same f16 for every amax.

The two f32 numbers differ (in 4.5 % of all cases, by a step): 127 * f32(1 / 127) is 1 - 2^-28. They round to different f16 only where
amax / 127 lies within 2^-28 above B - u / 2, B a border of f16's rounding and u an f32 step of it, which puts amax between
127 B - 63.5 u and 127 B - 55.5 u. But 127 B is an f32 (B has 12 bits), whose neighbours are 64 or 128 u away."""
import numpy as np
import pytest


def half_up(x):
    """f32 -> f16 bits, half up on the dropped bits, as the rows' codec rounds (numbers of f16's range)."""
    b = x.view(np.uint32)
    e, m = (b >> 23).astype(np.int32) - 127, b & np.uint32(0x7fffff)
    normal = ((e + 15).astype(np.int64) << 10) + ((m.astype(np.int64) + 0x1000) >> 13)
    shift = np.clip(-e - 14, 0, 11)
    small = ((m.astype(np.int64) | 0x800000) + (np.int64(1) << (shift + 12))) >> (shift + 13)
    return np.where(e < -24, 0, np.where(e < -14, small, normal))


def scales(exponent):
    a = ((np.uint32(127 + exponent) << np.uint32(23)) | np.arange(1 << 23, dtype=np.uint32)).view(np.float32)
    return a * (np.float32(1) / np.float32(127)), a / np.float32(127)


@pytest.mark.parametrize("exponent", [-19, -18, -13, -9, -8, -7, -6, 0, 1, 10, 22])
def test_the_inverse_gives_the_same_f16_scales(exponent):
    """Every amax of a power of two: f16's subnormal scales (amax below 2^-7), and normal ones up to the largest."""
    product, quotient = scales(exponent)
    assert np.any(product != quotient)
    assert np.array_equal(half_up(product), half_up(quotient))


def test_the_codec_rounds_like_that(oracle):
    from yuuka_b200 import cuda
    x = np.concatenate([scales(e)[0][::70001] for e in (-19, -13, -7, 0, 15)])
    x = np.ascontiguousarray(x[:x.size // 32 * 32])
    assert np.array_equal(oracle.kv_encode_row(cuda.KV_F16, x).view(np.uint16), half_up(x))
