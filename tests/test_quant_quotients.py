"""The paged append forms a bf16 group's codes from a * rcp(step), whose relative error is below
2^-22, in place of the rounded quotient a / step.  That gives the same bf16 quotient for every
pair: checked over all significands (exponents only scale the quotient), and likewise for a / 15
times the rounded 1 / 15."""

import numpy as np


def _bf16(x):
    """float64 -> bf16 (round half to even), as float64; exact for these magnitudes."""
    m, e = np.frexp(x)                       # m in [0.5, 1)
    return np.ldexp(np.rint(np.ldexp(m, 8)), e - 8)


def test_every_bf16_quotient_survives_the_reciprocals_error():
    a = np.arange(128, 256, dtype=np.float64)[:, None]
    step = np.arange(128, 256, dtype=np.float64)[None]
    exact = a / step
    want = _bf16(exact)
    for err in (-2.0 ** -22, 2.0 ** -22):
        assert np.array_equal(_bf16(exact * (1 + err)), want)


def test_every_bf16_fifteenth_survives():
    a = np.arange(128, 256, dtype=np.float64)
    for err in (-2.0 ** -22, 2.0 ** -22):
        assert np.array_equal(_bf16(a / 15 * (1 + err)), _bf16(a / 15))


