"""Corners of the fused products' host side that need no GPU: the plan, and which arrays share memory."""
import pytest

from test_products_cpu import args, grad

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
