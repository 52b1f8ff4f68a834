"""Corners of the fused products' host side that need no GPU: the plan, and which arrays share memory."""
import numpy as np
import pytest

from test_products_cpu import EINVAL, EWORKSPACE, args, grad

from locus_amd import _lib

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("cus", ["1", "2", "3", "64"])
def test_the_sweeps_cu_override_does_not_change_products(monkeypatch, cus):
    """LOCUS_HIP_MFMA_CUS forces launch plans of the sweeps.  The split of a product, and with it its bits, stay (a
    gradient's plan divided by half of it: 0)."""
    lib = _lib.lib()
    monkeypatch.delenv("LOCUS_HIP_MFMA_CUS", raising=False)
    calls = [(lib.locus_hip_product_grad_workspace_bytes, grad(m=m, n=n, k=k, act=1, pre=1 << 40, sp_m=n, sp_n=1, sd_m=n,
                                                              sa_m=k, sb_k=n, dA=4 << 40, dB=5 << 40, col_sums=col))
             for m, n, k in ((300, 200, 100), (4, 3, 5), (5000, 70, 30), (64, 2000, 3000)) for col in (0, 6 << 40)]
    calls += [(lib.locus_hip_product_workspace_bytes, args(m=m, n=n, k=k, sa_m=k, sb_k=n, sc_m=n))
              for m, n, k in ((1, 1000, 20000), (2000, 500, 20000), (64, 64, 100000))]
    want = [fn(a) for fn, a in calls]
    assert min(want) >= 0 and max(want) > 0
    monkeypatch.setenv("LOCUS_HIP_MFMA_CUS", cus)
    assert [fn(a) for fn, a in calls] == want


def shares(kw):
    """Whether the library finds that C shares memory with what is read (a small workspace stops the calls that pass)."""
    rc = _lib.lib().locus_hip_product_dev(args(**kw, cfg0=64, cfg1=4, workspace=64 << 20, workspace_bytes=1), None)
    assert rc in (EINVAL, EWORKSPACE)
    return rc == EINVAL


def own_memory(shape, strides):
    """The library's rule for what is written: rows (or columns) one behind the other."""
    (m, n), (sm, sn) = shape, (abs(strides[0]), abs(strides[1]))
    if m == 1 or n == 1:
        return (m == 1 or sm >= 1) and (n == 1 or sn >= 1)
    return (sm >= 1 and sn > sm * (m - 1)) if sm <= sn else (sn >= 1 and sm > sn * (n - 1))


@pytest.mark.parametrize("seed", range(8))
def test_views_that_share_nothing_are_taken(seed):
    """C and A anywhere in one buffer, any strides, against the sets of their elements: every call that shares nothing
    passes (arrays this small are looked through), every other is refused."""
    rng = np.random.default_rng(seed)
    base, taken = 1 << 20, 0
    for _ in range(1500):
        m, n, k = 4, int(rng.integers(1, 5)), 64
        sa = [int(x) for x in rng.integers(-9, 140, size=2)]
        sc = [int(x) for x in (rng.integers(-9, 140, size=2) if rng.random() < 0.3 else np.array(sa) * rng.choice([1, 1, 2, -1]))]
        if not own_memory((m, n), sc):
            continue
        at = int(rng.integers(-40, 200))
        a = (np.arange(m)[:, None] * sa[0] + np.arange(k) * sa[1]).ravel()
        c = (at + np.arange(m)[:, None] * sc[0] + np.arange(n) * sc[1]).ravel()
        free = not np.isin(c, a).any()
        got = shares(dict(m=m, n=n, k=k, A=base, sa_m=sa[0], sa_k=sa[1], B=9 << 20, sb_k=n, C=base + 8 * at, sc_m=sc[0], sc_n=sc[1]))
        assert got != free, (m, n, k, sa, sc, at)
        taken += free and c.min() <= a.max() and a.min() <= c.max()
    assert taken > 50


@pytest.mark.parametrize("ld", [128, 129, 200])
def test_every_other_column(ld):
    """A: the even columns of a matrix, C: odd ones."""
    kw = dict(m=4, k=64, n=40, sa_m=ld, sa_k=2, B=9 << 20, sb_k=40, sc_m=ld, sc_n=2)
    assert not shares(dict(**kw, C=(1 << 20) + 8))
    assert shares(dict(**kw, C=(1 << 20) + 16))
    assert shares(dict(**kw, C=(1 << 20) + 12))


def test_large_interleaved_views_end_quickly():
    """Strides without a common order: too many places to look through count as shared, and soon."""
    import time
    start = time.perf_counter()
    for _ in range(50):
        shares(dict(m=1 << 20, n=64, k=1 << 16, sa_m=7919, sa_k=104729, B=1 << 45, sb_k=64, C=(1 << 20) + 8, sc_m=65, sc_n=1))
    assert time.perf_counter() - start < 1.0


@pytest.mark.parametrize("kw,ok", [(dict(m=1, sr_m=77, sr_n=1), True), (dict(m=4, n=1, sc_m=3, sr_m=3, sr_n=5), True),
                                   (dict(m=1, n=1, sr_m=0, sr_n=0), True), (dict(m=1, sr_m=77, sr_n=2), False),
                                   (dict(m=4, sr_m=4, sr_n=1), False)])
def test_one_row_in_place_of_its_residual(kw, ok):
    """C is the residual; the stride of a single row or column, which a view may give any value, does not count."""
    kw = dict(dict(n=3, k=64, sa_m=64, res=3 << 20), **kw)
    assert shares(kw) != ok
