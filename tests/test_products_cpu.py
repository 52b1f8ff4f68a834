"""Refusals of the fused products and of predict() that need no GPU: the library's own checks come before
anything is launched, the Python ones before the library is asked."""
import numpy as np
import pytest

from locus_amd import _lib

torch = pytest.importorskip("torch")
EINVAL, EWORKSPACE = -1, -5


def args(**kw):
    """A packed locus_hip_product_args: 4 x 5 times 5 x 3 on made-up addresses (nothing is ever read)."""
    from locus_amd import products as pr
    d = dict(m=4, n=3, k=5, dtype=0, act=0, mode=0, fill_rest=0, cfg0=0, cfg1=0, alpha=1.0, beta=1.0,
             A=1 << 20, sa_m=5, sa_k=1, B=2 << 20, sb_k=3, sb_n=1, bias=0, sbias_m=0, sbias_n=0, res=0, sr_m=0, sr_n=0,
             C=3 << 20, sc_m=3, sc_n=1, pre=0, sp_m=0, sp_n=0, groups=0, offsets=0, sb_g=0, sbias_g=0, gather=0,
             a_rows=0, workspace=0, workspace_bytes=0)
    d.update(kw)
    return pr._ARGS.pack(*d.values())


def grad(**kw):
    from locus_amd import products as pr
    d = dict(m=4, n=3, k=5, dtype=0, act=0, mode=0, pad=0, cfg0=0, cfg1=0, alpha=1.0, dC=1 << 20, sd_m=3, sd_n=1, pre=0,
             sp_m=0, sp_n=0, A=2 << 20, sa_m=5, sa_k=1, B=3 << 20, sb_k=3, sb_n=1, G=0, dA=4 << 20, dB=5 << 20,
             col_sums=0, row_sums=0, groups=0, offsets=0, sb_g=0, gather=0, a_rows=0, workspace=0, workspace_bytes=0)
    d.update(kw)
    return pr._GRAD_ARGS.pack(*d.values())


BAD = [dict(dtype=2), dict(act=6), dict(act=-1), dict(mode=2), dict(m=-1), dict(n=4194241), dict(k=1 << 30), dict(cfg0=32),
       dict(cfg1=257), dict(cfg1=-1), dict(A=0), dict(B=0), dict(C=0),
       dict(mode=1, groups=0, offsets=1), dict(mode=1, groups=65536, offsets=1), dict(mode=1, groups=2, offsets=0),
       dict(mode=1, groups=2, offsets=9 << 20, gather=8 << 20, a_rows=0),
       dict(mode=1, groups=2, offsets=9 << 20, gather=8 << 20, a_rows=-1),
       dict(sc_m=2), dict(sc_m=0), dict(sc_n=0), dict(sc_m=1, sc_n=3),             # elements of C share memory
       dict(C=(1 << 20) + 8), dict(C=(2 << 20) - 8), dict(pre=3 << 20, sp_m=3, sp_n=1),
       dict(pre=4 << 20, sp_m=1, sp_n=1), dict(bias=(3 << 20) + 16, sbias_n=1),
       dict(res=(3 << 20) + 8, sr_m=3, sr_n=1), dict(res=3 << 20, sr_m=1, sr_n=4)]
BAD_GRAD = [dict(dtype=-1), dict(act=7), dict(mode=3), dict(k=4194241), dict(cfg0=1), dict(act=1), dict(dC=0), dict(A=0),
            dict(B=0), dict(G=6 << 20), dict(mode=1, groups=1, offsets=7 << 20, row_sums=6 << 20), dict(mode=1, groups=1),
            dict(mode=1, groups=2, offsets=7 << 20, gather=8 << 20, a_rows=0),
            dict(dA=(1 << 20) + 88), dict(dB=(2 << 20) - 16), dict(dB=(4 << 20) + 8), dict(col_sums=(3 << 20) + 8),
            dict(row_sums=5 << 20)]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_bad_products_are_refused(kw):
    lib = _lib.lib()
    assert lib.locus_hip_product_dev(args(**kw), None) == EINVAL
    assert b"product" in lib.locus_hip_last_error()


@pytest.mark.parametrize("kw", BAD_GRAD, ids=str)
def test_bad_gradients_are_refused(kw):
    lib = _lib.lib()
    assert lib.locus_hip_product_grad_dev(grad(**kw), None) == EINVAL
    assert b"product_grad" in lib.locus_hip_last_error()


def test_null_arguments_and_missing_workspace(monkeypatch):
    lib = _lib.lib()
    for fn in (lib.locus_hip_product_dev, lib.locus_hip_product_grad_dev):
        assert fn(None, None) == EINVAL
    for fn in (lib.locus_hip_product_workspace_bytes, lib.locus_hip_product_grad_workspace_bytes):
        assert fn(None) == EINVAL
    monkeypatch.setenv("LOCUS_HIP_MFMA_CUS", "256")                   # plans without a device
    split = dict(m=64, n=64, k=4096, sa_m=4096, sb_k=64, sc_m=64, B=16 << 20, C=32 << 20, cfg0=64, cfg1=4)
    need = lib.locus_hip_product_workspace_bytes(args(**split))
    assert need == 4 * 64 * 64 * 8
    assert lib.locus_hip_product_dev(args(**split), None) == need            # what to bring, nothing launched
    assert lib.locus_hip_product_dev(args(**split, workspace=64 << 20, workspace_bytes=need - 1), None) == EWORKSPACE
    g = dict(act=1, pre=6 << 20, sp_m=3, sp_n=1)
    need = lib.locus_hip_product_grad_workspace_bytes(grad(**g))
    assert need >= 4 * 3 * 8
    assert lib.locus_hip_product_grad_dev(grad(**g), None) == need
    assert lib.locus_hip_product_grad_dev(grad(**g, workspace=64 << 20, workspace_bytes=need - 1), None) == EWORKSPACE


@pytest.mark.parametrize("at,ok", [(512, True), (504, False), (1000, True), (1008, False), (1016, False), (1024, False),
                                   (1536, True), (2024, True), (-24, True), (-16, False), (-1024 + 512, True)])
def test_blocks_of_one_matrix_share_no_memory(monkeypatch, at, ok):
    """A: columns 0 .. 63 of rows of 128 (1024 bytes), C: 3 other columns `at` bytes from there, or not quite.  (The
    small workspace stops the calls that pass.)"""
    monkeypatch.setenv("LOCUS_HIP_MFMA_CUS", "256")
    lib = _lib.lib()
    rc = lib.locus_hip_product_dev(args(m=4, n=3, k=64, sa_m=128, sc_m=128, C=(1 << 20) + at, cfg0=64, cfg1=4,
                                        workspace=64 << 20, workspace_bytes=1), None)
    assert rc == (EWORKSPACE if ok else EINVAL)


def test_a_dense_gradient_has_no_runs(monkeypatch):
    monkeypatch.setenv("LOCUS_HIP_MFMA_CUS", "256")
    need = _lib.lib().locus_hip_product_grad_workspace_bytes
    big = dict(m=5000, n=70, k=30, act=1, pre=1 << 40, sp_m=70, sp_n=1, col_sums=1 << 41)
    assert need(grad(**big)) == need(grad(**big, groups=900, offsets=1 << 42, gather=1 << 43, a_rows=9)) > 0


def test_empty_products_do_nothing(monkeypatch):
    monkeypatch.setenv("LOCUS_HIP_MFMA_CUS", "256")
    lib = _lib.lib()
    assert lib.locus_hip_product_dev(args(m=0, A=0, C=0), None) == 0
    assert lib.locus_hip_product_dev(args(n=0, B=0, C=0), None) == 0
    assert lib.locus_hip_product_workspace_bytes(args(m=0)) == 0
    assert lib.locus_hip_product_grad_dev(grad(m=0, n=0, k=0, dC=0, A=0, B=0, dA=0, dB=0), None) == 0


def test_python_refusals():
    from locus_amd import products as pr
    A, B = torch.zeros(4, 5, dtype=torch.float64), torch.zeros(5, 3, dtype=torch.float64)
    with pytest.raises(ValueError, match="GPU"):
        pr.dense_product(A, B)
    with pytest.raises(ValueError, match="float64 or float32"):
        pr.dense_product(A.half(), B.half())
    with pytest.raises(ValueError, match="2-dimensional"):
        pr.dense_product(A[0], B)
    with pytest.raises(ValueError, match="3-dimensional"):
        pr.grouped_product(A, B, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="2-dimensional"):
        pr.dense_product(np.zeros((4, 5)), B)
    with pytest.raises(ValueError, match="negated"):
        pr.dense_product(torch.zeros(4, 5, dtype=torch.complex128).conj().imag, B)


def test_predict_refusals():
    from locus_amd import Predictor
    rng = np.random.default_rng(0)
    X, Y = rng.normal(size=(20, 6)), rng.normal(size=(20, 2))
    vb = dict(beta_vb=np.zeros((6, 2)), rmvd_x=np.array([], dtype=int))
    for kw, match in ((dict(link="cloglog"), "link"), (dict(link="mix"), "ind_bin"), (dict(ind_bin=[0]), "ind_bin"),
                      (dict(Z=X[:, :2]), "Z"), (dict(link="probit"), "intercept"), (dict(link="logit"), "intercept")):
        with pytest.raises(ValueError, match=match):
            Predictor(vb, X, **kw)
    with pytest.raises(ValueError, match="means"):
        Predictor(dict(vb, alpha_vb=np.zeros((1, 2))), X, link="logit", Y=Y)
    with pytest.raises(ValueError, match="beta_vb"):
        Predictor(dict(om_vb=1), X)
    with pytest.raises(ValueError, match="do not go with"):
        Predictor(dict(vb, rmvd_x=np.array([1])), X)
    with pytest.raises(ValueError, match="one length"):
        Predictor([vb, vb], [X])
    with pytest.raises(ValueError, match="one length"):
        Predictor([], [])
    with pytest.raises(ValueError, match="same covariates"):
        Predictor([vb, dict(vb, beta_vb=np.zeros((6, 3)))], [X, X])
    with pytest.raises(ValueError, match="columns"):
        Predictor(vb, X, Y=Y[:, :1])
