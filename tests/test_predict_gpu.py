"""Predictions from fitted models (locus_amd.predict) against numpy on what the fits returned.

On the training samples the linear predictor is mat_x_m1 + mat_z_mu of the fit itself; folding the
standardisation into the effects regroups sums of p terms, each off by a few 2^-53 of the largest: 1e-11 of the
values' scale at p below 200.  float32: sums of p terms and the rounded effects, 2 (p + 4) 2^-24 of the terms' sum."""
import numpy as np
import pytest
from scipy.special import expit, ndtr

pytestmark = pytest.mark.gpu
KW = dict(user_seed=4, tol=1e-30, maxit=4, verbose=False, full_output=True)


@pytest.fixture(scope="module")
def data(hip):
    from locus_amd.simulate import simulate
    sim = simulate(90, 60, 7, 5, seed=21)
    X = 3.0 + 2.0 * sim["X"]                                  # raw covariates, not standardised
    X[:, 11] = 1.0                                            # one constant column, one copy: both removed
    X[:, 17] = X[:, 3]
    Z = np.random.default_rng(2).normal(size=(90, 2)) * [1.0, 5.0] + 2.0
    Y = sim["Y"] + 4.0
    return X, Z, Y, (sim["Y"] > np.median(sim["Y"], axis=0)).astype(np.float64)


@pytest.mark.parametrize("with_z", [False, True])
@pytest.mark.parametrize("link", ["identity", "logit", "probit", "mix"])
def test_training_samples(data, link, with_z):
    from locus_amd import Predictor, locus, predict
    X, Z, Yc, Yb = data
    ind_bin = None
    Y = Yc if link == "identity" else Yb
    if link == "mix":
        ind_bin = np.array([1, 4, 6])
        Y = Yc.copy()
        Y[:, ind_bin] = Yb[:, ind_bin]
    vb = locus(Y, X, 5, Z=Z if with_z else None, link=link, ind_bin=ind_bin, **KW)
    assert 11 in vb["rmvd_x"] and 17 in vb["rmvd_x"]
    eta = np.asarray(vb["mat_x_m1"], dtype=np.float64)
    if "mat_z_mu" in vb:
        eta = eta + np.asarray(vb["mat_z_mu"], dtype=np.float64)
    centred = eta.copy()
    if link == "identity":
        eta = eta + Y.mean(axis=0)
    if link == "mix":
        eta[:, [0, 2, 3, 5]] += Y[:, [0, 2, 3, 5]].mean(axis=0)
    want = {"identity": eta, "logit": expit(eta), "probit": ndtr(eta)}.get(link)
    if link == "mix":
        want = eta.copy()
        want[:, ind_bin] = ndtr(eta[:, ind_bin])
    ys = Y if link in ("identity", "mix") else None
    pred = Predictor(vb, X, Z if with_z else None, ys, link, ind_bin)
    zn = Z if with_z else None
    np.testing.assert_allclose(pred(X, zn), want, rtol=1e-10, atol=1e-10)
    np.testing.assert_allclose(pred(X, zn, type="link"), eta, rtol=1e-10, atol=1e-10)
    one = pred(X[7:8], None if zn is None else zn[7:8])       # one new sample
    np.testing.assert_allclose(one, want[7:8], rtol=1e-10, atol=1e-10)
    assert pred(X[:0], None if zn is None else zn[:0]).shape == (0, 7)
    if ys is not None:
        np.testing.assert_allclose(predict(vb, X, X, Z=zn, Z_new=zn, link=link, ind_bin=ind_bin, type="link"), centred,
                                   rtol=1e-10, atol=1e-10)
    small = Predictor(vb, X, zn, ys, link, ind_bin, single=True)(X, zn, type="link")
    eff = np.abs(pred.parts[0][2].cpu().numpy()).max()
    terms = (np.abs(X).sum(axis=1) + (np.abs(Z).sum(axis=1) if with_z else 0)).max() * eff + np.abs(eta).max()
    assert np.abs(small - eta).max() <= 2 * (62 + 4) * 2.0 ** -24 * terms * 4


@pytest.mark.parametrize("link", ["identity", "mix"])
def test_many_fits(data, link):
    """A fit per fold, the samples in any order, one fold without samples."""
    from locus_amd import Predictor, locus
    X, Z, Yc, Yb = data
    ind_bin = None
    Y = Yc
    if link == "mix":
        ind_bin = np.array([0, 2])
        Y = Yc.copy()
        Y[:, ind_bin] = Yb[:, ind_bin]
    fold = np.arange(90) % 3
    fits = [locus(Y[fold != k], X[fold != k], 5, link=link, ind_bin=ind_bin, **KW) for k in range(3)]
    xs, ys = [X[fold != k] for k in range(3)], [Y[fold != k] for k in range(3)]
    pred = Predictor(fits, xs, None, ys, link, ind_bin)
    rng = np.random.default_rng(3)
    for to in (fold, rng.integers(0, 3, size=90), np.where(fold == 1, 2, fold)):
        got = pred(X, fit=to)
        want = np.empty_like(got)
        for k in range(3):
            want[to == k] = Predictor(fits[k], xs[k], None, ys[k], link, ind_bin)(X[to == k])
        np.testing.assert_allclose(got, want, rtol=1e-11, atol=1e-11)
    for bad in (None, fold[:-1], fold + 1, fold - 1, fold.astype(float)):
        with pytest.raises(ValueError):
            pred(X, fit=bad)
    with pytest.raises(ValueError):
        Predictor(fits[0], xs[0], link=link, ind_bin=ind_bin)(X, fit=fold)
