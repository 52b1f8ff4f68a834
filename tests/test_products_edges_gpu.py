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


def test_callers_on_threads_of_their_own(pr):
    """Two threads on their own streams, 20 calls each; what a thread raises fails the test."""
    from concurrent.futures import ThreadPoolExecutor
    A, B = normal(12, 70, 2003), normal(13, 2003, 65)
    off = torch.tensor([0, 11, 70], device="cuda:0")
    Bg, dC = torch.stack([B, 2 * B]), normal(14, 70, 65)
    calls = [lambda: (pr.dense_product(A, B, act="gelu"), pr.grouped_product(A, Bg, off, cfg=(64, 2))),
             lambda: pr.grouped_product_grad(dC, A, Bg, off, act="probit", pre=dC, need_bias=True)]
    want = [c() for c in calls]
    torch.cuda.synchronize()

    def work(call, ref):
        side, done = torch.cuda.Stream(), 0
        with torch.cuda.stream(side):
            for _ in range(20):
                got = call()
                assert len(got) == len(ref) and all(torch.equal(g, w) for g, w in zip(got, ref))
                done += 1
        side.synchronize()
        return done

    with ThreadPoolExecutor(2) as pool:
        assert [f.result() for f in [pool.submit(work, *x) for x in zip(calls, want)]] == [20, 20]


def test_tensors_that_require_grad_are_refused(pr):
    """The products are outside autograd: a result cut off from the graph would lose its gradient without a word.
    Detached, or under no_grad, the same calls are made."""
    A, B, off = normal(1, 4, 5), normal(2, 5, 3), torch.tensor([0, 1, 4], device="cuda:0")
    bias, res, pre, dC = normal(3, 3), normal(4, 4, 3), normal(5, 4, 3), normal(6, 4, 3)

    def dense(A=A, B=B, bias=bias, residual=res, out=None, pre=pre):
        return pr.dense_product(A, B, bias=bias, residual=residual, out=out, pre=pre)

    def grouped(A=A, B=B, bias=bias, residual=res):
        return pr.grouped_product(A, torch.stack([B.detach(), B.detach()]).requires_grad_(B.requires_grad), off,
                                  bias=torch.stack([bias.detach()] * 2).requires_grad_(bias.requires_grad), residual=residual)

    def grad(A=A, B=B, dC=dC, pre=pre):
        return pr.dense_product_grad(dC, A, B, act="silu", pre=pre, bias_grad="row")[0]

    all_args = dict(A=A, B=B, bias=bias, residual=res, out=torch.zeros_like(res), pre=pre, dC=dC)
    for fn in (dense, grouped, grad):
        want = fn()
        for name in fn.__code__.co_varnames[:fn.__code__.co_argcount]:
            leaf = all_args[name].clone().requires_grad_()
            with pytest.raises(ValueError, match=f"{name} requires grad.*no_grad"):
                fn(**{name: leaf})
            with torch.no_grad():
                assert torch.equal(fn(**{name: leaf}), want)
            assert torch.equal(fn(**{name: leaf.detach()}), want)


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("arg", ["out", "pre"])
def test_autograd_sees_what_was_overwritten(pr, arg, grouped):
    """A tensor that a graph of autograd holds for its backward pass, given as out or pre: the pass fails, as after any
    operation in place, instead of using the new values."""
    A, B, off = normal(1, 4, 5), normal(2, 5, 3), torch.tensor([0, 1, 4], device="cuda:0")
    held, other = normal(3, 4, 3), normal(4, 4, 3)
    leaf = torch.ones((4, 3), dtype=torch.float64, device="cuda:0", requires_grad=True)
    y = (leaf * held).sum()
    kw = {arg: held, "pre" if arg == "out" else "out": other}
    before = other._version
    if grouped:
        pr.grouped_product(A, torch.stack([B, B]), off, **kw)
    else:
        pr.dense_product(A, B, **kw)
    assert other._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():                    # tensors without a version
        kw = {name: torch.empty_like(t) for name, t in kw.items()}
        pr.dense_product(A, B, **kw)


def test_as_many_runs_as_there_may_be(pr):
    """65 535 runs, empty ones among them, rows of no run before and behind.  Sums of k and of a run's rows in float64:
    2 (terms + 4) 2^-53 of the terms' magnitudes."""
    rng = np.random.default_rng(20)
    gr, m, k, n = 65535, 70000, 3, 2
    off = np.sort(rng.integers(5, m - 7, size=gr + 1))
    A, B, dC = rng.normal(size=(m, k)), rng.normal(size=(gr, k, n)), rng.normal(size=(m, n))
    run = np.searchsorted(off, np.arange(m), side="right") - 1
    rows = (run >= 0) & (run < gr)
    g = np.clip(run, 0, gr - 1)
    u, most = 2.0 ** -53, np.diff(off).max()

    def close(got, want, terms, count):
        assert (np.abs(got.cpu().numpy() - want) <= 2 * (count + 4) * u * terms).all()

    up = [torch.from_numpy(x).to("cuda:0") for x in (A, B, off)]
    for cfg in ((0, 0), (64, 1)):
        P = np.einsum("mk,mkn->mn", A, B[g]) * rows[:, None]
        close(pr.grouped_product(*up, cfg=cfg), P, np.einsum("mk,mkn->mn", np.abs(A), np.abs(B[g])) * rows[:, None], k)
        dA, dB, db = pr.grouped_product_grad(torch.from_numpy(dC).to("cuda:0"), *up, need_bias=True, cfg=cfg)
        close(dA, np.einsum("mn,mkn->mk", dC, B[g]) * rows[:, None],
              np.einsum("mn,mkn->mk", np.abs(dC), np.abs(B[g])) * rows[:, None], n)
        for got, each in ((dB, A[:, :, None] * dC[:, None]), (db, dC)):
            want, terms = np.zeros((gr, *each.shape[1:])), np.zeros((gr, *each.shape[1:]))
            np.add.at(want, run[rows], each[rows])
            np.add.at(terms, run[rows], np.abs(each[rows]))
            close(got, want, terms, most)
