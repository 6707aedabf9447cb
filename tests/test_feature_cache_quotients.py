"""The steps by which the feature cache's kernels divide, in exact arithmetic on a machine without a GPU: on which side of every middle
between two codes they end, for the floats next to it."""
from fractions import Fraction

import numpy as np
import pytest

from oracle import feature_cache as ocache

F = np.float32


def to_float(q, nearest):
    """A fraction to the float32 nearest to it (ties to even) or cut; no case here comes near the ends of the range."""
    if q == 0:
        return Fraction(0)
    a, e = abs(q), 0
    e = a.numerator.bit_length() - a.denominator.bit_length() - 24
    for e in (e - 1, e, e + 1, e + 2):  # units of the last place 2^e: 24 bits in front of it
        units = a / Fraction(2) ** e
        if 2 ** 23 <= units < 2 ** 24:
            break
    n = units.numerator // units.denominator
    if nearest and (units - n > Fraction(1, 2) or units - n == Fraction(1, 2) and n % 2):
        n += 1
    return (1 if q > 0 else -1) * n * Fraction(2) ** e


def quotient(x, s):
    """What the kernel takes for x / s (positive): its steps, one rounding each; also the first guess."""
    inverse = int((F(1) / s).view(np.uint32))
    small, large = (Fraction(float(np.uint32(i).view(F))) for i in (inverse - 3, inverse + 4))
    x, s = Fraction(float(x)), Fraction(float(s))
    t = to_float(-x * small, True)
    y = to_float(-to_float(t * s + x, True) * large + t, False)
    bits = int(F(float(y)).view(np.uint32)) | (1 if y * s + x != 0 else 0)
    return -Fraction(float(np.uint32(bits).view(F))), -t


def middles(code):
    numbers = np.arange(128.0) if code == "int8" else ocache.e4m3_numbers()[:127]
    return (numbers[1:] + numbers[:-1]) / 2


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_quotients_end_on_their_side_of_every_middle(code):
    """A quotient that is not a middle ends strictly on its own side of it, one that is one ends on it: so the code that it rounds to,
    ties to even, is that of the exact quotient."""
    rng = np.random.default_rng(9)
    scales = [F(m) * F(2.0) ** int(e) for m, e in zip(rng.integers(2 ** 23, 2 ** 24, 30), rng.integers(-60, 60, 30))]
    scales += [F(1.0), F(2 ** 24 - 1), F(2 ** 23 + 1), F(1.5326611), F(16700629)]
    for s in scales:
        for m in middles(code):
            near = F(np.float64(m) * np.float64(s))
            for x in (np.nextafter(near, F(0)), near, np.nextafter(near, F(np.inf))):
                exact = Fraction(float(x)) / Fraction(float(s))
                y, t = quotient(x, s)
                middle = Fraction(float(m))
                assert (y > middle) == (exact > middle) and (y < middle) == (exact < middle), (x, s, m)
                assert t <= exact < t + 8 * Fraction(2) ** (int(np.floor(np.log2(float(t)))) - 23), (x, s)


def test_quotients_next_to_a_float():
    """Quotients just below a float (2^-24 and 2.6 2^-24 of a unit here) end on that float and are made odd there: two units above the
    cut quotient where that one was odd.  No code minds: floats next to a middle between codes are even, and no quotient is that
    close to one."""
    for x, s, past in ((F(10683675), F(16700629), 1), (F(2.9060206), F(1.5326611), 2)):
        exact = Fraction(float(x)) / Fraction(float(s))
        y, _ = quotient(x, s)
        cut = to_float(exact, False)
        unit = Fraction(2) ** (int(np.floor(np.log2(float(cut)))) - 23)
        assert y - cut == past * unit and 0 < cut + unit - exact < unit / 2 ** 22
    rng = np.random.default_rng(10)
    for x, s in rng.integers(2 ** 23, 2 ** 24, (3000, 2)):
        exact = Fraction(int(x), int(s))
        y, t = quotient(F(x), F(s))
        unit = Fraction(2) ** (int(np.floor(np.log2(float(exact)))) - 23)
        assert exact - unit < y < exact + 2 * unit and t <= exact
