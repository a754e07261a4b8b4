"""2^x on the multipliers, as pb_prefix_attn's kernel for the prefix computes a quarter of its exponentials, in numpy: its steps, with the coefficients that the
source has, against 2^x in 64 bits over the range that softmax gives it, [-126, 13].

In exact arithmetic the stored polynomial is 2^-22.6 off, relative, and fp32's roundings leave 2^-22.1.  The last step takes away what the range's lower end came to, which
makes all below it nothing and costs its neighbours their digits: less than 2^-125 absolute."""
import pathlib
import re

import numpy as np

SOURCE = pathlib.Path(__file__).parents[1] / "paella_b200" / "csrc" / "lm_attn.cu"
BIG = np.float32(12582912.0)             # 1.5 x 2^23: behind it a sum's last bit is 1


def coefficients():
    """highest power first"""
    body = re.search(r"uint64_t ex2_pair\(uint64_t x\) \{(.*?)\n\}", SOURCE.read_text(), re.S).group(1)
    found = [np.float32(c) for c in re.findall(r"both\(([01]\.\d+)f\)", body)]
    assert len(found) == 6
    return found


def fma(x, y, z):
    """one rounding but for ties of a double one: the product of two fp32 values is exact in 64 bits"""
    return (np.float64(x) * np.float64(y) + np.float64(z)).astype(np.float32)


def ex2(x):
    x = np.maximum(x, np.float32(-126.0))            # (a NaN stays one)
    t = x + BIG
    f = fma(t - BIG, np.float32(-1.0), x)
    r = np.full_like(x, coefficients()[0])
    for c in coefficients()[1:]:
        r = fma(r, f, c)
    whole = (r.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))).view(np.float32)
    return whole + fma(x, np.float32(0.0), np.float32(-2.0 ** -126 * (1 + 2.0 ** -23)))


def test_polynomial():
    f = np.linspace(-0.5, 0.5, 400001).astype(np.float32)
    r = np.zeros(f.shape)
    for c in coefficients():
        r = r * f + np.float64(c)
    assert np.abs(r / np.exp2(np.float64(f)) - 1).max() < 2.0 ** -22.6


def test_powers_of_two():
    x = np.concatenate([np.linspace(-126.0, 13.0, 3000001), np.arange(-126, 14), np.arange(-126, 13) + 0.5]).astype(np.float32)
    ref = np.exp2(np.float64(x))
    assert (np.abs(ex2(x) - ref) <= 2.0 ** -22.1 * ref + 2.0 ** -125).all()
    assert (ex2(np.array([0.0, -1.0, 5.0, 13.0], np.float32)) == np.exp2(np.array([0.0, -1.0, 5.0, 13.0])) * np.float32(1.0000001192092896)).all()


def test_what_is_far_below_is_nothing_and_a_nan_stays_one():
    assert (ex2(np.array([-126.0, -126.5, -127.0, -1e4, -1e30, -np.inf], np.float32)) == 0).all()
    nans = np.array([0x7fffffff, 0x7fc00000, 0xffc00000], np.uint32).view(np.float32)
    assert np.isnan(ex2(nans)).all()


def test_whole_parts_lose_a_nan():
    """Why the last step has the argument in it: adding to the exponent field of the NaN that the GPU's arithmetic gives leaves a finite number."""
    nan = np.uint32(0x7fffffff)
    with np.errstate(over="ignore"):
        assert np.isfinite((nan + (nan << np.uint32(23))).view(np.float32))
