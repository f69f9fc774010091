"""The arithmetic of the casts to NVFP4 restated for every 16-bit value and every ue4m3 scale,
with 1 / s rounded up to fp32 as the kernels have it."""
import numpy as np
import pytest

import linear_ops_ref as ref
from test_linear_ops_cpu import _bf16_values, _f16_values


def reciprocal_up(s):
    """The least fp32 that is not below 1 / s; s has four bits, so the check is exact."""
    inv = np.float32(1.0 / s)
    return np.nextafter(inv, np.float32(np.inf)) if float(inv) * s < 1.0 else inv


@pytest.mark.parametrize("values", [_bf16_values, _f16_values])
def test_the_short_quotient_with_a_reciprocal_rounded_up(values):
    x = values()
    for s in ref.E4M3[1:]:
        xs = x[(x > 0.2 * s) & (x < 8 * s)].astype(np.float64)
        snap = (xs * np.float64(reciprocal_up(s)) + 48.0).astype(np.float32) - np.float32(48.0)
        got, want = (ref.nearest(np.minimum(q, 6.0), ref.E2M1) for q in (snap, xs / s))
        assert np.array_equal(got, want), s


@pytest.mark.parametrize("fold", [2.0 ** -12, 1.0, 2.0 ** 8])
@pytest.mark.parametrize("values", [_bf16_values, _f16_values])
def test_the_stochastic_code_of_every_value_at_its_step(values, fold):
    # q = x times fold / s, then q 2^-126 without rounding up: its bits are the code above 22 bits of
    # fraction (below 1 those of a subnormal number), to which 2^14 (r + 1/2) is added
    x = values()
    for s in ref.E4M3[1:]:
        with np.errstate(over="ignore"):
            xs = x[(x * fold >= 2.0 ** -10 * s) & (x * fold <= 6 * s)]
        q = xs * (reciprocal_up(s) * np.float32(fold))
        assert q.dtype == np.float32
        bits = np.where(q >= 1, q.view(np.int32).astype(np.int64) - (126 << 23),
                        np.floor(q.astype(np.float64) * 2.0 ** 23).astype(np.int64))
        exact = xs.astype(np.float64) * fold / s
        lo = np.clip(np.searchsorted(ref.E2M1, exact, side="right") - 1, 0, 6)
        f = (exact - ref.E2M1[lo]) / (ref.E2M1[lo + 1] - ref.E2M1[lo])
        first = np.ceil(256 * (1 - f) - 0.5)  # the least byte that takes the code up
        for r in (first - 1, first):
            r = np.clip(r, 0, 255).astype(np.int64)
            code = np.minimum((bits + 64 * (256 * r + 128)) >> 22, 7)
            assert np.array_equal(code, lo + (f + (r + 0.5) / 256 >= 1)), s
