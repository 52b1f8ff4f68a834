"""Fused products at the limit of 32-bit offsets: a K-tile whose last element begins 2^31 - sizeof(T) bytes
behind its first one, the last that a 2 GiB window can hold, and the same one row step before and behind."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pr(hip):
    from locus_amd import products
    return products


@pytest.fixture(scope="module")
def big(hip):
    return torch.zeros((2 ** 31 + 2 ** 20) // 8, dtype=torch.float64, device="cuda:0")


# rows (of A) or columns (of B) 4 260 880 float64 or 8 521 760 float32 apart: 63 steps and 16 or 32 elements are
# 2^31 bytes exactly
@pytest.mark.parametrize("step", [-1, 0, 1])
@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("cfg", [(64, 1), (0, 0)])
def test_last_element_of_two_gigabytes(pr, big, dtype, step, cfg):
    t, kt, far = (torch.float64, 16, 4260880) if dtype == "f64" else (torch.float32, 32, 8521760)
    flat = big.view(t)
    assert 63 * far + kt == 2 ** 31 // flat.element_size()
    far += step
    rng = np.random.default_rng(step + 1)
    A = flat.as_strided((64, kt), (far, 1))
    A.copy_(torch.from_numpy(rng.normal(size=(64, kt))))
    other = torch.from_numpy(rng.normal(size=(kt, 70))).to("cuda:0").to(t)
    near = A.contiguous()
    u = torch.finfo(t).eps / 2

    def same(got, want, terms):
        assert ((got.double() - want).abs() <= 2 * (kt + 66) * u * terms).all()

    P, S = near.double() @ other.double(), near.double().abs() @ other.double().abs()
    same(pr.dense_product(A, other, cfg=cfg), P, S)
    same(pr.dense_product(other.t(), A.t(), cfg=cfg), P.t(), S.t())
    off, src = torch.tensor([0, 64], device="cuda:0"), torch.arange(63, -1, -1, device="cuda:0")
    same(pr.grouped_product(A, other[None], off, cfg=cfg), P, S)
    same(pr.grouped_product(A, other[None], off, gather=src, cfg=cfg), P.flip(0), S.flip(0))
    dC = torch.from_numpy(rng.normal(size=(64, 70))).to("cuda:0").to(t)
    P, S = near.double().t() @ dC.double(), near.double().t().abs() @ dC.double().abs()
    for gather in (None, torch.arange(64, device="cuda:0")):
        dA, dB, _ = pr.grouped_product_grad(dC, A, other[None], off, gather=gather, cfg=cfg)
        same(dB[0], P, S)
    same(pr.dense_product_grad(dC, A, other, cfg=cfg)[1], P, S)


@pytest.mark.parametrize("step", [-1, 0, 1])
def test_last_element_of_two_gigabytes_plain_product(hip, big, monkeypatch, step):
    """The same for locus_hip_gemm_dev (K-tiles of 16, rows of A and columns of B)."""
    from locus_amd import device as dv
    monkeypatch.setenv("LOCUS_HIP_GEMM_BK", "16")
    rng = np.random.default_rng(step + 5)
    far = 4260880 + step
    A = big.as_strided((64, 16), (far, 1))
    A.copy_(torch.from_numpy(rng.normal(size=(64, 16))))
    other = torch.from_numpy(rng.normal(size=(16, 70))).to("cuda:0")
    P, S = A.contiguous() @ other, A.contiguous().abs() @ other.abs()
    C = torch.empty((64, 70), dtype=torch.float64, device="cuda:0")
    dv.gemm(64, 70, 16, A, far, 1, other, 70, 1, C, 70, 1)
    assert ((C - P).abs() <= 2 * 82 * 2.0 ** -53 * S).all()
    C = torch.empty((70, 64), dtype=torch.float64, device="cuda:0")
    dv.gemm(70, 64, 16, other, 1, 70, A, 1, far, C, 64, 1)
    assert ((C - P.t()).abs() <= 2 * 82 * 2.0 ** -53 * S.t()).all()
