"""The coefficients of the normal distribution function in product.h against 60 digits (no GPU needed)."""
import importlib.util
import os

import pytest

mp = pytest.importorskip("mpmath")
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def poly():
    spec = importlib.util.spec_from_file_location("cdf_poly", os.path.join(HERE, "..", "scripts", "microbench", "cdf_poly.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_coefficients(poly):
    """Truncation below half a rounding of the result, 2^-54, and each coefficient's rounding, 2^-53 of it, over values
    above 1."""
    with mp.workdps(poly.DIGITS):
        c = poly.committed()
        assert len(c) == poly.DEGREE + 1
        assert poly.worst([mp.mpf(x) for x in c], 801) <= 2.0 ** -54 + 2.0 ** -53 * sum(abs(x) for x in c)
        assert min(poly.exact(mp.mpf(i) / 50 - 1) for i in range(100)) >= 1


def test_fit(poly):
    with mp.workdps(poly.DIGITS):
        assert poly.worst(poly.fit(), 201) <= 2.0 ** -54
