"""The folding of the standardisation into the effects (locus_amd.predict), without a GPU."""
import numpy as np
import pytest


@pytest.mark.parametrize("order", ["C", "F"])
@pytest.mark.parametrize("value", [0.1, 0.3, 1 / 3, 1e-3, 7.7, 2.0, 0.0, 1e9 + 0.1])
def test_columns_of_one_value(order, value):
    """Such a column is kept by scale_rm_ where its rounded mean is off.  Terms of order 1 (raw columns of order 1),
    sums of 6 of them, twice: 1e-13 holds them with room."""
    from locus_amd.predict import _raw_effects
    from locus_amd.prepare import scale_rm_
    kept = 0
    for n in range(20, 120, 3):
        rng = np.random.default_rng(n)
        X = np.array(rng.normal(size=(n, 6)), order=order)
        X[:, 2] = value
        Xs, rmvd = scale_rm_(X)
        kept += not rmvd[2]
        eff = rng.normal(size=(Xs.shape[1], 2))
        out, const = _raw_effects(eff, X, np.nonzero(rmvd)[0])
        assert np.abs(X @ out + const - Xs @ eff).max() <= 1e-13
        new = rng.normal(size=(4, 6))                  # of another value there: the same constant
        same = new.copy()
        same[:, 2] = value
        assert np.abs((new - same) @ out).max() == 0
    assert kept or value in (2.0, 0.0)


def test_a_kept_column_without_deviation_is_refused():
    """The fit cannot have kept it: these are not the covariates it was given (predictions would be NaN)."""
    from locus_amd import Predictor
    X = np.random.default_rng(0).normal(size=(20, 4))
    X[:, 1] = 2.0
    vb = dict(beta_vb=np.ones((4, 2)), alpha_vb=np.zeros((2, 2)), rmvd_x=np.array([], dtype=int))
    with pytest.raises(ValueError, match="do not go with the fit.*1"):
        Predictor(dict(vb, alpha_vb=np.zeros((1, 2))), X, link="probit")
    with pytest.raises(ValueError, match="do not go with the fit.*0"):
        Predictor(vb, np.random.default_rng(1).normal(size=(20, 4)), Z=np.ones((20, 1)), link="probit")
