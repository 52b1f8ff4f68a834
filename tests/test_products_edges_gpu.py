"""Corners of the fused products' calls on the GPU: results in place, concurrent callers, tensors of autograd."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pr(hip):
    from locus_amd import products
    return products


def normal(seed, *shape, dtype=torch.float64):
    return torch.from_numpy(np.random.default_rng(seed).normal(size=shape)).to("cuda:0").to(dtype)


@pytest.mark.parametrize("cfg", [(0, 0), (16, 2), (64, 2), (128, 1)])
def test_one_row_or_column_in_place_of_its_residual(pr, cfg):
    for m, n in ((1, 70), (70, 1), (1, 1)):
        A, B, buf = normal(1, m, 130), normal(2, 130, n), normal(3, 5, 70)
        row = buf[3:4] if m == 1 else buf[3:4].t()
        row = row[:m, :n]
        out = buf.as_strided((m, n), (999 if m == 1 else 1, 999 if n == 1 else 1), 3 * 70)
        want, kept = pr.dense_product(A, B, residual=row.clone(), beta=-1.0, cfg=cfg), buf.clone()
        assert pr.dense_product(A, B, residual=row, beta=-1.0, out=out, cfg=cfg) is out
        assert torch.equal(row, want)
        kept.view(-1)[3 * 70:3 * 70 + m * n] = want.reshape(-1)
        assert torch.equal(buf, kept)
