"""The running maximum of the attention of drafted tokens, restated in 32 bits (no GPU): after m has moved, no score is
above it, whatever the scores' size.

A tile's scores are x = fma(P, b, lg), P the rounded product of the MMA's sum and the key's g, and W's exponent is
y = x + c with c = 9 - m.  m follows while some y is above 15, so the step ends only if y <= 15 holds afterwards for
all that m was made of.
"""
import numpy as np
import pytest

F = np.float32


def fma(a, b, c):
    """fma in 32 bits (by 64: the product is exact there, the sum nearly)."""
    return (a.astype(np.float64) * b.astype(np.float64) + c.astype(np.float64)).astype(F)


def bias_minus(m):
    """9 - m rounded down to 32 bits."""
    d = 9.0 - m.astype(np.float64)  # exact below 2^52; above 2^28, 9 is less than m's last place
    r = d.astype(F)
    r = np.where(r.astype(np.float64) > d, np.nextafter(r, F(-np.inf)), r)
    return np.where(np.abs(m) >= 2.0 ** 40, np.where(m > 0, -m, np.nextafter(-m, F(-np.inf))), r).astype(F)


@pytest.mark.parametrize("exponent", list(range(-8, 60)) + [90, 126])
def test_no_score_is_above_a_maximum_made_of_it(exponent):
    rng = np.random.RandomState(exponent + 10)
    rows, keys = 64, 256
    P = rng.randn(rows, keys).astype(F)
    b = rng.uniform(0.5, 2.0, (rows, 1)).astype(F)
    lg = rng.uniform(-3.0, 3.0, (1, keys)).astype(F)
    big = np.abs(P * b).max(1, keepdims=True)
    P = (P / big * F(2.0) ** F(exponent / 2) * rng.uniform(1, 2, (rows, 1))).astype(F)
    x = fma(P, b * F(2.0) ** F(exponent - exponent / 2) * F(0.5), lg)
    assert np.isfinite(x).all()
    m = x.max(1, keepdims=True)
    y = x + bias_minus(m)
    assert y.dtype == F and (y <= 9.0).all()
    # the key that has the maximum keeps a weight of 2^0 to 2^9
    assert (y.max(1) >= 0.0).all()
