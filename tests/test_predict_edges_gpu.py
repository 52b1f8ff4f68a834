"""Predictor.score as a caller on a busy stream uses it, and the corners of its arguments.  The fits are made up."""
import numpy as np
import pytest
from scipy.special import ndtr

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def fits(count, n=40, p=9, d=6, seed=0):
    rng = np.random.default_rng(seed)
    X = [rng.normal(size=(n, p)) * 2 + 1 for _ in range(count)]
    vb = [dict(beta_vb=rng.normal(size=(p, d)), alpha_vb=rng.normal(size=(1, d)), rmvd_x=np.array([], dtype=int))
          for _ in range(count)]
    return vb, X


def eta(vb, X, new):
    return ((new - X.mean(axis=0)) / X.std(axis=0, ddof=1)) @ vb["beta_vb"] + vb["alpha_vb"][0]


@pytest.mark.parametrize("link", ["probit", "mix"])
@pytest.mark.parametrize("many", [False, True])
def test_score_does_not_wait(hip, link, many):
    """The stream is kept busy for some hundred milliseconds; score() returns while it still is."""
    from locus_amd import Predictor
    ind_bin = np.array([1, 4]) if link == "mix" else None
    vb, X = fits(3)
    pred = Predictor(vb, X, link=link, ind_bin=ind_bin) if many else Predictor(vb[0], X[0], link=link, ind_bin=ind_bin)
    rng = np.random.default_rng(1)
    new, to = rng.normal(size=(50, 9)), rng.integers(0, 3, size=50)
    A = torch.from_numpy(new).to("cuda:0")
    fit = to if many else None
    for _ in range(3):
        pred.score(A, fit)
    big = torch.ones((4096, 4096), dtype=torch.float64, device="cuda:0")
    out = torch.empty_like(big)
    torch.mm(big, big, out=out)
    torch.cuda.synchronize()
    for _ in range(100):                       # 1.4e11 operations each: 2 ms
        torch.mm(big, big, out=out)
    done = torch.cuda.Event()
    done.record()
    got = pred.score(A, fit)
    assert not done.query(), "score() waited for the work queued before it"
    torch.cuda.synchronize()
    want = np.stack([eta(vb[g], X[g], new[i:i + 1])[0] for i, g in enumerate(to if many else np.zeros(50, int))])
    cols = np.arange(6) if link == "probit" else ind_bin
    want[:, cols] = ndtr(want[:, cols])
    np.testing.assert_allclose(got.cpu().numpy(), want, rtol=1e-11, atol=1e-11)


@pytest.mark.parametrize("link", ["probit", "mix"])
def test_captured_and_replayed(hip, link):
    """score() of one fit in a graph, new samples in the same memory, eager calls in between; with fit it is refused."""
    from locus_amd import Predictor
    vb, X = fits(2)
    ind_bin = np.array([0, 5]) if link == "mix" else None
    pred = Predictor(vb[0], X[0], link=link, ind_bin=ind_bin)
    A = torch.zeros((33, 9), dtype=torch.float64, device="cuda:0")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pred.score(A)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pred.score(A)
    rng = np.random.default_rng(2)
    for _ in range(4):
        A.copy_(torch.from_numpy(rng.normal(size=(33, 9))))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pred.score(A))
    many = Predictor(vb, X, link=link, ind_bin=ind_bin)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        A + 1
        with pytest.raises(RuntimeError, match="captured"):
            many.score(A, np.arange(33) % 2)


def test_device_without_a_number_is_the_current_one(hip):
    """"cuda" names whatever device is current when it is looked at: the predictor fixes it where its effects are."""
    from locus_amd import Predictor
    vb, X = fits(1)
    for device in (None, "cuda", "cuda:0", torch.device("cuda")):
        pred = Predictor(vb[0], X[0], link="probit", device=device)
        assert pred.device == pred.parts[0][2].device == torch.device("cuda", torch.cuda.current_device())


@pytest.mark.parametrize("link", ["probit", "mix"])
@pytest.mark.parametrize("fit", [[], (), np.array([], dtype=int), np.array([])], ids=["list", "tuple", "int", "float"])
def test_no_samples(hip, link, fit):
    from locus_amd import Predictor
    vb, X = fits(2)
    pred = Predictor(vb, X, link=link, ind_bin=[1] if link == "mix" else None)
    assert pred(np.zeros((0, 9)), fit=fit).shape == (0, 6)
    with pytest.raises(ValueError, match="integers"):
        pred(np.zeros((1, 9)), fit=fit)
