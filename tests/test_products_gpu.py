"""Fused and grouped matrix products and their gradients (locus_amd.products) against plain 64-bit numpy.

Tolerances, per element, derived before the first run (u = eps / 2 of the type).  A sum of k products in any order is off by
at most (k + 1) u sum |a b| (to first order); alpha, the bias and the reference's own sum (float64 runs)
add 3 u and double it, so  |dZ| <= 2 (k + 4) u S  with S = |alpha| |A| |B| + |bias|.  The activations have
slopes below 1.2 and are evaluated to a few units of their own value and of e^x arguments up to z^2 / 2
(whose error the vanishing factor keeps below one unit of 1): 16 u (1 + |act|); the residual adds one
rounding of the result.
"""
import numpy as np
import pytest
from scipy.special import expit, ndtr

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f64": torch.float64, "f32": torch.float32}
ACTS = ("identity", "logistic", "probit", "softplus", "gelu", "silu")
CFGS = [(0, 0), (16, 1), (16, 3), (64, 1), (64, 3), (128, 1), (128, 2)]


@pytest.fixture(scope="module")
def pr(hip):
    from locus_amd import products
    return products


def unit(t):
    return torch.finfo(t.dtype).eps / 2


def dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0").to(dtype)


def host(t):
    return t.detach().to("cpu", torch.float64).numpy()


def act_ref(name, z):
    with np.errstate(invalid="ignore", over="ignore"):
        return {"identity": lambda: z, "logistic": lambda: expit(z), "probit": lambda: ndtr(z),
                "softplus": lambda: np.logaddexp(0.0, z), "gelu": lambda: np.where(z == -np.inf, 0.0, z * ndtr(z)),
                "silu": lambda: np.where(z == -np.inf, 0.0, z * expit(z))}[name]()


def slope_ref(name, z):
    dens = np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)
    return {"identity": lambda: np.ones_like(z), "logistic": lambda: expit(z) * expit(-z), "probit": lambda: dens,
            "softplus": lambda: expit(z), "gelu": lambda: ndtr(z) + z * dens,
            "silu": lambda: expit(z) * (1 + z * expit(-z))}[name]()


def layout(a, kind, dtype):
    """The matrix on the GPU: row-major, column-major, or a window of a larger buffer full of NaN."""
    t = dev(a, dtype)
    if kind == "col":
        return t.t().contiguous().t()
    if kind == "win":
        big = torch.full((a.shape[0] + 3, 2 * a.shape[1] + 5), float("nan"), dtype=dtype, device=t.device)
        w = big[1:1 + a.shape[0], 3:3 + 2 * a.shape[1]:2]
        w.copy_(t)
        return w
    return t


def close(got, want, tol):
    got = host(got)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / tol)} of the tolerance"


def reference(A, B, bias, act, residual, alpha, beta, u, k):
    z = alpha * (A @ B) + (0 if bias is None else bias)
    s = abs(alpha) * (np.abs(A) @ np.abs(B)) + (0 if bias is None else np.abs(bias))
    dz = 2 * (k + 4) * u * s + 1e-300
    v = act_ref(act, z)
    tol = 1.2 * dz + 16 * u * (1 + np.abs(v))
    if residual is not None:
        v = v + beta * residual
        tol = tol + 2 * u * (np.abs(beta * residual) + np.abs(v))
    return z, dz, v, tol


# one, odd and ragged sizes around the tiles of 16, 64 and 128, an empty sum, long sums
SHAPES = [(1, 1, 1), (1, 7, 3), (5, 0, 9), (1, 1037, 70), (16, 64, 64), (33, 17, 65), (67, 130, 1), (70, 133, 67), (129, 259, 131), (300, 31, 258)]


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("cfg", CFGS)
def test_dense_product(pr, dtype, cfg):
    t = DT[dtype]
    u = torch.finfo(t).eps / 2
    for i, (m, k, n) in enumerate(SHAPES):
        for j, lay in enumerate((("row", "row"), ("col", "row"), ("row", "col"), ("win", "win"))):
            rng = np.random.default_rng(1000 * i + j)
            A, B = (rng.normal(size=s).astype(np.float32).astype(np.float64) for s in ((m, k), (k, n)))
            bias = [None, rng.normal(size=n), rng.normal(size=(m, 1)), rng.normal(size=(m, n))][(i + j) % 4]
            res = rng.normal(size=(m, n)) if (i + j) % 2 else None
            if t == torch.float32:
                bias, res = (None if x is None else x.astype(np.float32).astype(np.float64) for x in (bias, res))
            act = ACTS[(i + j) % 6]
            z, dz, v, tol = reference(A, B, bias, act, res, 0.5, -1.5, u, k)
            pre = torch.full((m, n), 7.0, dtype=t, device="cuda:0") if j % 2 else None
            out = torch.empty((n, m), dtype=t, device="cuda:0").t() if j > 1 else None
            got = pr.dense_product(layout(A, lay[0], t), layout(B, lay[1], t), bias=None if bias is None else dev(bias, t),
                                   act=act, residual=None if res is None else layout(res, lay[0], t), alpha=0.5,
                                   beta=-1.5, out=out, pre=pre, cfg=cfg)
            assert out is None or got is out
            close(got, v, tol)
            if pre is not None:
                close(pre, z, dz)


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_activation_values_and_slopes(pr, dtype, act):
    """Z itself (A a column of values, B = 1): both tails, the switch of signs, infinities and NaN."""
    t = DT[dtype]
    u = torch.finfo(t).eps / 2
    z = np.concatenate([np.linspace(-9, 9, 73), [0.0, -0.0, 1e-30, -1e-30, 30, -30, 90, -90, 700, -700, 1e4, -1e4]])
    z = z.astype(np.float32).astype(np.float64)
    col = dev(z[:, None], t)
    one = torch.ones((1, 1), dtype=t, device="cuda:0")
    v = act_ref(act, z)
    close(pr.dense_product(col, one, act=act)[:, 0], v, 16 * u * (1 + np.abs(v)))
    special = np.array([np.inf, -np.inf, np.nan])
    got = host(pr.dense_product(dev(special[:, None], t), one, act=act)[:, 0])
    want = {"identity": [np.inf, -np.inf], "softplus": [np.inf, 0], "gelu": [np.inf, 0], "silu": [np.inf, 0]}.get(act, [1, 0])
    assert np.array_equal(got[:2], want) and np.isnan(got[2])
    _, _, g = pr.dense_product_grad(torch.ones_like(col), col, one, act=act, pre=col, bias_grad="matrix")
    s = slope_ref(act, z)
    close(g[:, 0], s, 16 * u * (1 + np.abs(s)))
    sp = dev(np.array([[np.inf], [-np.inf]]), t)
    _, _, g = pr.dense_product_grad(torch.ones_like(sp), sp, one, act=act, pre=sp, bias_grad="matrix", need_A=False,
                                    need_B=False)
    limit = {"identity": [1, 1], "logistic": [0, 0], "probit": [0, 0]}.get(act, [1, 0])
    assert np.array_equal(host(g)[:, 0], limit)


@pytest.mark.parametrize("cfg", [(16, 1), (16, 2), (64, 2), (128, 1)])
def test_nan_and_inf_stay_in_their_row_and_column(pr, cfg):
    rng = np.random.default_rng(5)
    m, k, n = 70, 45, 66
    A, B = rng.normal(size=(m, k)), rng.normal(size=(k, n))
    A[3, 44], B[0, 65] = np.nan, np.inf
    got = host(pr.dense_product(dev(A, torch.float64), dev(B, torch.float64), cfg=cfg))
    hit = np.zeros((m, n), bool)
    hit[3], hit[:, 65] = True, True
    assert np.isfinite(got[~hit]).all() and not np.isfinite(got[hit]).any()


def runs_of(offsets, m):
    """The documented reading of offsets: a running maximum within [0, m]."""
    o = np.maximum.accumulate(np.clip(offsets, 0, m))
    return list(zip(o[:-1], o[1:]))


OFFSETS = {
    "even": lambda m: [0, m // 3, m // 2, m],
    "empty runs": lambda m: [0, 0, m // 2, m // 2, m, m],
    "one run has all": lambda m: [0, 0, m, m],
    "rows before and behind": lambda m: [min(2, m), min(2, m), max(min(2, m), m - 3)],
    "none": lambda m: [0, 0, 0],
    "out of order and range": lambda m: [-5, m // 2, m // 4, m + 9, 3],
    "many": lambda m: np.sort(np.random.default_rng(0).integers(0, m + 1, size=150)).tolist(),
}


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("cfg", [(0, 0), (16, 1), (16, 3), (64, 1), (64, 2), (128, 1), (128, 3)])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_product(pr, dtype, cfg, gather):
    t = DT[dtype]
    u = torch.finfo(t).eps / 2
    for i, (name, make) in enumerate(OFFSETS.items()):
        for j, (m, k, n) in enumerate([(1, 5, 3), (40, 33, 70), (300, 70, 65)]):
            rng = np.random.default_rng(100 * i + j)
            off = np.array(make(m), dtype=np.int64)
            G = len(off) - 1
            rows = m + 7 if gather else m
            f32 = lambda *s: rng.normal(size=s).astype(np.float32).astype(np.float64)  # noqa: E731
            A, B, bias, res = f32(rows, k), f32(G, k, n), f32(G, n), f32(m, n)
            src = rng.integers(0, rows, size=m) if gather else np.arange(m)      # the same row several times
            act = ACTS[(i + j) % 6]
            want, tol, zw, zt = (np.zeros((m, n)) for _ in range(4))
            inside = np.zeros(m, bool)
            for g, (lo, hi) in enumerate(runs_of(off, m)):
                zw[lo:hi], zt[lo:hi], want[lo:hi], tol[lo:hi] = reference(A[src[lo:hi]], B[g], bias[g], act, res[lo:hi], 1.0, -1.0, u, k)
                inside[lo:hi] = True
            At = layout(A, ("row", "col", "win")[j], t)
            Bt = dev(B, t) if (i + j) % 2 else dev(B.transpose(0, 2, 1), t).transpose(1, 2)
            kw = dict(bias=dev(bias, t), act=act, residual=dev(res, t), beta=-1.0,
                      gather=torch.from_numpy(src).to("cuda:0") if gather else None, cfg=cfg)
            offt = torch.from_numpy(off).to("cuda:0")
            got = pr.grouped_product(At, Bt, offt, **kw)
            close(got, want, tol)                          # rows of no run are 0 where out is made there
            out = torch.full((m, n), 3.0, dtype=t, device="cuda:0")
            pre = torch.full((m, n), 4.0, dtype=t, device="cuda:0")
            pr.grouped_product(At, Bt, offt, out=out, pre=pre, **kw)
            want[~inside], tol[~inside] = 3.0, 0.0         # and left as they were where it is given
            zw[~inside], zt[~inside] = 4.0, 0.0
            close(out, want, tol)
            close(pre, zw, zt)


@pytest.mark.parametrize("cfg", [(16, 1), (16, 2), (64, 1), (128, 2)])
def test_gathered_rows_outside_come_out_nan(pr, cfg):
    rng = np.random.default_rng(1)
    A, B = rng.normal(size=(9, 40)), rng.normal(size=(2, 40, 5))
    src = np.array([0, 9, 3, -1, 8, 2 ** 40, 8])
    off = torch.tensor([0, 3, 7], device="cuda:0")
    at, bt, st = dev(A, torch.float64), dev(B, torch.float64), torch.from_numpy(src).to("cuda:0")
    got = host(pr.grouped_product(at, bt, off, gather=st, cfg=cfg))
    ok = (src >= 0) & (src < 9)
    assert np.isnan(got[~ok]).all() and np.isfinite(got[ok]).all()
    dC = dev(rng.normal(size=(7, 5)), torch.float64)
    dA, dB, db = pr.grouped_product_grad(dC, at, bt, off, gather=st, need_bias=True)
    assert np.isfinite(host(dA)).all() and np.isfinite(host(db)).all()
    assert np.isnan(host(dB)).all()                        # both runs hold such a row
    dB = host(pr.grouped_product_grad(dC, at, bt, torch.tensor([0, 1, 1], device="cuda:0"), gather=st)[1])
    assert np.isfinite(dB[0]).all() and (dB[1] == 0).all()


def grad_reference(dC, A, B, act, pre, alpha, u):
    """G, dA, dB, dbias of one run, each with its tolerance: G is off by 16 u (1 + slope) |dC| <= 40 u |dC| (see
    the top of the file) and one rounding; sums as there."""
    m, k = A.shape
    n = B.shape[1]
    G = dC * slope_ref(act, pre)
    aG = np.abs(G) + 40 * u * np.abs(dC)
    tG = 42 * u * np.abs(dC)
    dA, dB = alpha * G @ B.T, alpha * A.T @ G
    tA = abs(alpha) * (2 * (n + 4) * u * aG + tG) @ np.abs(B).T
    tB = abs(alpha) * np.abs(A).T @ (2 * (m + 4) * u * aG + tG)
    tb = (2 * (m + 4) * u * aG + tG).sum(axis=0)
    return G, tG, dA, tA, dB, tB, G.sum(axis=0), tb, (2 * (n + 4) * u * aG + tG).sum(axis=1, keepdims=True)


GRAD_CFGS = [(0, 0), (16, 0), (64, 1), (64, 2), (128, 1), (128, 2)]


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("cfg", GRAD_CFGS)
def test_dense_product_grad(pr, dtype, act, cfg):
    t = DT[dtype]
    u = torch.finfo(t).eps / 2
    for i, (m, k, n) in enumerate([(1, 1, 1), (1, 50, 33), (67, 5, 20), (200, 130, 70), (700, 20, 3), (130, 33, 300)]):
        rng = np.random.default_rng(i)
        f32 = lambda *s: rng.normal(size=s).astype(np.float32).astype(np.float64)  # noqa: E731
        A, B, dC, pre = f32(m, k), f32(k, n), f32(m, n), 2 * f32(m, n)
        G, tG, dA, tA, dB, tB, db, tb, tr = grad_reference(dC, A, B, act, pre, -0.5, u)
        lay = ("row", "col", "win")[i % 3]
        args = [layout(x, lay, t) for x in (dC, A, B)]
        kw = dict(act=act, pre=layout(pre, lay, t), alpha=-0.5, cfg=cfg)
        ga, gb, gc = pr.dense_product_grad(*args, bias_grad="column", **kw)
        close(ga, dA, tA + 1e-300)
        close(gb, dB, tB + 1e-300)
        close(gc, db, tb)
        ga, gb, gr = pr.dense_product_grad(*args, bias_grad="row", need_A=False, need_B=False, **kw)
        assert ga is None and gb is None
        close(gr, G.sum(axis=1, keepdims=True), tr)
        gm = pr.dense_product_grad(*args, bias_grad="matrix", need_A=False, need_B=False, **kw)[2]
        close(gm, G, tG + 1e-300)
        assert gm.data_ptr() != args[0].data_ptr()


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("name", list(OFFSETS))
@pytest.mark.parametrize("cfg", GRAD_CFGS)
def test_grouped_product_grad(pr, dtype, gather, name, cfg):
    t = DT[dtype]
    u = torch.finfo(t).eps / 2
    for j, (m, k, n) in enumerate([(1, 5, 3), (40, 33, 70), (600, 70, 65), (150, 140, 131)]):
        rng = np.random.default_rng(j)
        off = np.array(OFFSETS[name](m), dtype=np.int64)
        gr = len(off) - 1
        rows = m + 7 if gather else m
        f32 = lambda *s: rng.normal(size=s).astype(np.float32).astype(np.float64)  # noqa: E731
        A, B, dC, pre = f32(rows, k), f32(gr, k, n), f32(m, n), 2 * f32(m, n)
        src = rng.integers(0, rows, size=m) if gather else np.arange(m)
        act = ACTS[(j + len(name)) % 6]
        dA, tA = np.zeros((m, k)), np.full((m, k), 1e-300)
        dB, tB = np.zeros((gr, k, n)), np.full((gr, k, n), 1e-300)
        db, tb = np.zeros((gr, n)), np.full((gr, n), 1e-300)
        for g, (lo, hi) in enumerate(runs_of(off, m)):
            r = grad_reference(dC[lo:hi], A[src[lo:hi]], B[g], act, pre[lo:hi], 2.0, u)
            dA[lo:hi], dB[g], db[g] = r[2], r[4], r[6]
            tA[lo:hi] += r[3]
            tB[g] += r[5]
            tb[g] += r[7]
        got = pr.grouped_product_grad(dev(dC, t), layout(A, ("row", "col", "win", "row")[j], t), dev(B, t),
                                      torch.from_numpy(off).to("cuda:0"), act=act, pre=dev(pre, t), alpha=2.0,
                                      gather=torch.from_numpy(src).to("cuda:0") if gather else None, need_bias=True, cfg=cfg)
        close(got[0], dA, tA)
        close(got[1], dB, tB)
        close(got[2], db, tb)


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(pr, act):
    """(f(x + h e) - f(x - h e)) / 2h of f = sum w C, float64: off by h^2 f''' / 6 and 2^-53 |f| / h; with h = 1e-5,
    third derivatives of order 1 and f of order 100 both stay below 1e-7."""
    rng = np.random.default_rng(11)
    m, k, n = 6, 5, 4
    A, B, b, w = (rng.normal(size=s) for s in ((m, k), (k, n), (n,), (m, n)))
    off = torch.tensor([0, 2, 2, 6], device="cuda:0")
    Bg, bg = rng.normal(size=(3, k, n)), rng.normal(size=(3, n))
    d = lambda x: dev(x, torch.float64)  # noqa: E731

    def f(A, B, b):
        return float((w * host(pr.dense_product(d(A), d(B), bias=d(b), act=act))).sum())

    def fg(A, B, b):
        return float((w * host(pr.grouped_product(d(A), d(B), off, bias=d(b), act=act))).sum())

    pre = torch.empty((m, n), dtype=torch.float64, device="cuda:0")
    pr.dense_product(d(A), d(B), bias=d(b), act=act, pre=pre)
    dense = pr.dense_product_grad(d(w), d(A), d(B), act=act, pre=pre, bias_grad="column")
    preg = torch.empty_like(pre)
    pr.grouped_product(d(A), d(Bg), off, bias=d(bg), act=act, pre=preg)
    grouped = pr.grouped_product_grad(d(w), d(A), d(Bg), off, act=act, pre=preg, need_bias=True)
    h = 1e-5
    for fn, at, grads in ((f, (A, B, b), dense), (fg, (A, Bg, bg), grouped)):
        for which in range(3):
            g = host(grads[which])
            for _ in range(4):
                i = tuple(rng.integers(0, s) for s in g.shape)
                up, dn = [x.copy() for x in at], [x.copy() for x in at]
                up[which][i] += h
                dn[which][i] -= h
                assert abs((fn(*up) - fn(*dn)) / (2 * h) - g[i]) < 1e-7


@pytest.mark.parametrize("cfg", [(16, 1), (16, 2), (64, 1), (128, 2)])
def test_out_may_be_the_residual(pr, cfg):
    rng = np.random.default_rng(2)
    A, B, R = rng.normal(size=(70, 90)), rng.normal(size=(90, 66)), rng.normal(size=(70, 66))
    for buf in (dev(R, torch.float64), layout(R, "col", torch.float64)):
        want = pr.dense_product(dev(A, torch.float64), dev(B, torch.float64), residual=buf.clone(), alpha=-1.0, cfg=cfg)
        got = pr.dense_product(dev(A, torch.float64), dev(B, torch.float64), residual=buf, out=buf, alpha=-1.0, cfg=cfg)
        assert got is buf and torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f64", "f32"])
def test_addresses_beyond_32_bits(pr, dtype):
    """Rows, runs and gathered rows further apart than 2^31 bytes (and 2^31 elements of float32 for the runs)."""
    t = DT[dtype]
    s = torch.finfo(t).bits // 8
    far = (2 ** 31 + 2 ** 20) // s
    big = torch.zeros(3 * far, dtype=t, device="cuda:0")
    k, n = 40, 70
    rng = np.random.default_rng(3)
    A = big.as_strided((3, k), (far, 1))
    A.copy_(dev(rng.normal(size=(3, k)), t))
    B = dev(rng.normal(size=(k, n)), t)
    want = pr.dense_product(A.contiguous(), B)
    for cfg in ((0, 0), (16, 2), (64, 1), (128, 2)):
        assert torch.equal(pr.dense_product(A, B, cfg=cfg), pr.dense_product(A.contiguous(), B, cfg=cfg))
        close(pr.dense_product(A, B, cfg=cfg), host(want), 2 * (k + 4) * unit(want) * (np.abs(host(A)) @ np.abs(host(B))))
    off = torch.tensor([0, 1, 4], device="cuda:0")
    src = torch.tensor([2, 1, 0, 2], device="cuda:0")
    Bs = dev(rng.normal(size=(2, k, n)), t)
    dC = dev(rng.normal(size=(4, n)), t)
    for cfg in ((0, 0), (64, 1), (128, 1)):
        assert torch.equal(pr.grouped_product(A, Bs, off, gather=src, cfg=cfg),
                           pr.grouped_product(A.contiguous(), Bs, off, gather=src, cfg=cfg))
    assert torch.equal(pr.grouped_product_grad(dC, A, Bs, off, gather=src)[1],
                       pr.grouped_product_grad(dC, A.contiguous(), Bs, off, gather=src)[1])
    keep = A.contiguous()
    Bf = big.as_strided((2, k, n), (far, n, 1))
    Bf.copy_(Bs)
    assert torch.equal(pr.grouped_product(keep, Bf, off[:2 + 1], gather=src),
                       pr.grouped_product(keep, Bs, off, gather=src))


def test_same_bits_every_time_and_on_another_stream(pr):
    rng = np.random.default_rng(4)
    A, B = dev(rng.normal(size=(100, 3001)), torch.float32), dev(rng.normal(size=(3001, 90)), torch.float32)
    off = torch.tensor([0, 30, 100], device="cuda:0")
    Bg = torch.stack([B, -B])
    first = pr.dense_product(A, B, act="logistic")
    grouped = pr.grouped_product(A, Bg, off, act="silu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            assert torch.equal(pr.dense_product(A, B, act="logistic"), first)
            assert torch.equal(pr.grouped_product(A, Bg, off, act="silu"), grouped)
    side.synchronize()


def test_captured_and_replayed(pr):
    """Forward and gradient in HIP graphs, two graphs in turn, new inputs in the same buffers, eager work in between."""
    rng = np.random.default_rng(6)
    m, k, n = 90, 2500, 70
    A, B = dev(rng.normal(size=(m, k)), torch.float64), dev(rng.normal(size=(k, n)) / 50, torch.float64)
    Bg = torch.stack([B, 2 * B, -B])
    off = torch.tensor([0, 40, 40, 90], device="cuda:0")
    dC, pre = dev(rng.normal(size=(m, n)), torch.float64), torch.empty((m, n), dtype=torch.float64, device="cuda:0")

    def dense():
        c = pr.dense_product(A, B, act="probit", pre=pre)
        return (c, *pr.dense_product_grad(dC, A, B, act="probit", pre=pre, bias_grad="column"))

    def grouped():
        c = pr.grouped_product(A, Bg, off, act="logistic", pre=pre)
        return (c, *pr.grouped_product_grad(dC, A, Bg, off, act="logistic", pre=pre, need_bias=True))

    graphs = []
    for fn in (dense, grouped):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = fn()
        graphs.append((fn, g, outs))
    for turn in range(4):
        A.copy_(dev(rng.normal(size=(m, k)), torch.float64))
        off.copy_(torch.tensor([[0, 40, 40, 90], [0, 0, 1, 90], [5, 20, 60, 80], [0, 90, 90, 90]][turn]))
        for fn, g, outs in graphs:
            g.replay()
            torch.cuda.synchronize()
            for got, want in zip(outs, fn()):
                assert torch.equal(got, want)


def test_a_run_together(pr):
    """Fold-wise logistic regression by gradient steps, as it would be used: probabilities minus responses by the
    fused forward, the gradient of every fold's effects and intercepts by the grouped products, then new samples scored by
    one fit.  Against the same steps in numpy; three steps of size 0.1 on sums below 100 terms of order 1 amplify
    the roundings of a step (relative 1e-14) by less than 1e3."""
    rng = np.random.default_rng(8)
    m, k, n = 120, 30, 9
    off = np.array([0, 50, 50, 120])
    X = rng.normal(size=(m, k))
    Y = (rng.random((m, n)) < 0.4).astype(np.float64)
    beta, b0 = np.zeros((3, k, n)), np.zeros((3, n))
    Xt, Yt = layout(X, "col", torch.float64), layout(Y, "col", torch.float64)
    bt, b0t, offt = dev(beta, torch.float64), dev(b0, torch.float64), torch.from_numpy(off).to("cuda:0")
    for _ in range(3):
        score = pr.grouped_product(Xt, bt, offt, bias=b0t, act="logistic", residual=Yt, beta=-1.0)
        _, dB, db = pr.grouped_product_grad(score, Xt, bt, offt, need_A=False, need_bias=True)
        bt -= 0.1 * dB
        b0t -= 0.1 * db
        for g, (lo, hi) in enumerate(zip(off, off[1:])):
            s = expit(X[lo:hi] @ beta[g] + b0[g]) - Y[lo:hi]
            beta[g] -= 0.1 * X[lo:hi].T @ s
            b0[g] -= 0.1 * s.sum(axis=0)
    np.testing.assert_allclose(host(bt), beta, rtol=1e-11, atol=1e-11)
    new = rng.normal(size=(1, k))
    got = pr.dense_product(dev(new, torch.float64), bt[2], bias=b0t[2], act="logistic")
    np.testing.assert_allclose(host(got), expit(new @ beta[2] + b0[2]), rtol=1e-11)


@pytest.mark.parametrize("cfg", [(0, 0), (16, 2), (64, 2), (128, 1)])
def test_factors_and_result_as_blocks_of_one_matrix(pr, cfg):
    rng = np.random.default_rng(9)
    m, k, n = 37, 130, 21
    big = dev(rng.normal(size=(m, k + n + 3)), torch.float64)
    kept, B = big.clone(), dev(rng.normal(size=(k, n)), torch.float64)
    A, C = big[:, :k], big[:, k + 1:k + 1 + n]
    want = pr.dense_product(A, B, residual=C.clone(), cfg=cfg)
    pr.dense_product(A, B, residual=C, out=C, cfg=cfg)
    assert torch.equal(C, want)
    kept[:, k + 1:k + 1 + n] = want
    assert torch.equal(big, kept)
    with pytest.raises(Exception, match="shares memory"):
        pr.dense_product(A, B, out=big[:, k - 1:k - 1 + n], cfg=cfg)


@pytest.mark.parametrize("need_A", [False, True])
def test_more_runs_and_parts_than_a_grid_axis(pr, need_A):
    """3000 runs, each asked to be cut into 32 parts."""
    rng = np.random.default_rng(10)
    gr, m, k, n = 3000, 7000, 3, 2
    off = np.sort(rng.integers(0, m + 1, size=gr + 1))
    A, B, dC = rng.normal(size=(m, k)), rng.normal(size=(gr, k, n)), rng.normal(size=(m, n))
    got = pr.grouped_product_grad(dev(dC, torch.float64), dev(A, torch.float64), dev(B, torch.float64),
                                  torch.from_numpy(off).to("cuda:0"), need_A=need_A, need_bias=True, cfg=(64, 32))
    dB, tB = np.zeros((gr, k, n)), np.full((gr, k, n), 1e-300)
    for g, (lo, hi) in enumerate(zip(off, off[1:])):
        r = grad_reference(dC[lo:hi], A[lo:hi], B[g], "identity", dC[lo:hi], 1.0, 2.0 ** -53)
        dB[g], tB[g] = r[4], r[5] + 1e-300
    close(got[1], dB, tB)


def test_a_dense_gradient_ignores_the_fields_of_runs(pr):
    from locus_amd import _lib
    rng = np.random.default_rng(11)
    m, k, n = 700, 20, 33
    A, B, dC, pre = (dev(rng.normal(size=s), torch.float64) for s in ((m, k), (k, n), (m, n), (m, n)))
    want = pr.dense_product_grad(dC, A, B, act="silu", pre=pre, bias_grad="column")
    got = [torch.full_like(w, float("nan")) for w in want]
    off = torch.tensor([3, 5, 9, 40, 60], device="cuda:0")
    src = torch.full((m,), -1, device="cuda:0")
    fields = (m, n, k, 0, pr.ACTS["silu"], 0, 0, 0, 0, 1.0, *pr._at(dC), *pr._at(pre), *pr._at(A), *pr._at(B), 0,
              *(g.data_ptr() for g in got), 0, 4, off.data_ptr(), 7, src.data_ptr(), 5)
    pr._run(pr._GRAD_ARGS.pack, _lib.lib().locus_hip_product_grad_dev, fields, A.device)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_two_threads_on_their_own_streams(pr):
    import threading
    rng = np.random.default_rng(12)
    A, B = dev(rng.normal(size=(70, 2003)), torch.float64), dev(rng.normal(size=(2003, 65)), torch.float64)
    off = torch.tensor([0, 11, 70], device="cuda:0")
    Bg, dC = torch.stack([B, 2 * B]), dev(rng.normal(size=(70, 65)), torch.float64)
    calls = [lambda: (pr.dense_product(A, B, act="gelu"), pr.grouped_product(A, Bg, off, cfg=(64, 2))),
             lambda: pr.grouped_product_grad(dC, A, Bg, off, act="probit", pre=dC, need_bias=True)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    wrong = []

    def work(call, ref):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(20):
                if not all(torch.equal(g, w) for g, w in zip(call(), ref)):
                    wrong.append(call)
        side.synchronize()

    threads = [threading.Thread(target=work, args=x) for x in zip(calls, want)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


@pytest.mark.parametrize("groups", [64, 65, 256, 257, 700])
@pytest.mark.parametrize("cfg", [(0, 0), (16, 1), (64, 1), (64, 2), (128, 1)])
def test_many_runs(pr, groups, cfg):
    """Around the numbers of runs at which a tile's run is looked up in another way."""
    rng = np.random.default_rng(groups)
    m, k, n = 2500, 37, 66
    off = np.sort(rng.integers(3, m - 4, size=groups + 1))
    A, B, dC = rng.normal(size=(m, k)), rng.normal(size=(groups, k, n)), rng.normal(size=(m, n))
    want, tol = np.zeros((m, n)), np.zeros((m, n))
    dA, tA = np.zeros((m, k)), np.zeros((m, k))
    dB, tB = np.zeros((groups, k, n)), np.full((groups, k, n), 1e-300)
    for g, (lo, hi) in enumerate(zip(off, off[1:])):
        _, _, want[lo:hi], tol[lo:hi] = reference(A[lo:hi], B[g], None, "identity", None, 1.0, 0.0, 2.0 ** -53, k)
        _, _, dA[lo:hi], tA[lo:hi], dB[g], t, *_ = grad_reference(dC[lo:hi], A[lo:hi], B[g], "identity", dC[lo:hi], 1.0, 2.0 ** -53)
        tB[g] += t
    args = dev(A, torch.float64), dev(B, torch.float64), torch.from_numpy(off).to("cuda:0")
    close(pr.grouped_product(*args, cfg=cfg), want, tol)
    ga, gb, _ = pr.grouped_product_grad(dev(dC, torch.float64), *args, cfg=cfg)
    close(ga, dA, tA)
    close(gb, dB, tB)


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("cfg", [(0, 0), (64, 1), (64, 3), (128, 1)])
def test_gradients_of_one_and_two_columns(pr, dtype, n, cfg):
    t = DT[dtype]
    u = torch.finfo(t).eps / 2
    for m, k, lay in ((300, 203, "row"), (300, 203, "col"), (33, 1500, "win")):
        rng = np.random.default_rng(m + n)
        f32 = lambda *s: rng.normal(size=s).astype(np.float32).astype(np.float64)  # noqa: E731
        A, B, dC, pre = f32(m, k), f32(k, n), f32(m, n), 2 * f32(m, n)
        for act in ("identity", "logistic"):
            r = grad_reference(dC, A, B, act, pre, 1.0, u)
            for runs in (False, True):
                off = torch.tensor([0, m], device="cuda:0")
                args = [layout(dC, lay, t), layout(A, lay, t), layout(B, lay, t)]
                args = args if not runs else [args[0], args[1], args[2][None], off]
                fn = pr.grouped_product_grad if runs else pr.dense_product_grad
                got = fn(*args, act=act, pre=layout(pre, lay, t), cfg=cfg, **(dict(need_bias=True) if runs else dict(bias_grad="column")))
                close(got[0], r[2], r[3] + 1e-300)
                close(got[1][0] if runs else got[1], r[4], r[5] + 1e-300)
                close(got[2][0] if runs else got[2], r[6], r[7])


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("m,k,n", [(17, 333, 8300), (1, 700, 64), (16, 64, 4099), (33, 1030, 130), (5, 5000, 3)])
@pytest.mark.parametrize("layb", ["row", "col", "win"])
def test_few_rows_long_and_wide(pr, dtype, m, k, n, layb):
    """The kernel for few rows, whole and in slices, on every layout of B, up to 130 workgroups side by side."""
    t = DT[dtype]
    u = torch.finfo(t).eps / 2
    rng = np.random.default_rng(m + k)
    A = rng.normal(size=(m, k)).astype(np.float32).astype(np.float64)
    B = rng.normal(size=(k, n)).astype(np.float32).astype(np.float64)
    bias = rng.normal(size=(1, n)).astype(np.float32).astype(np.float64)
    for act, b, cfg in (("identity", None, (16, 1)), ("softplus", bias, (16, 1)), ("logistic", bias, (16, 3)), ("silu", bias, (0, 0))):
        _, _, want, tol = reference(A, B, b, act, None, 1.0, 0.0, u, k)
        got = pr.dense_product(dev(A, t), layout(B, layb, t), bias=None if b is None else dev(b, t), act=act, cfg=cfg)
        close(got, want, tol)
        off = torch.tensor([0, m], device="cuda:0")
        got = pr.grouped_product(dev(A, t), layout(B, layb, t)[None], off, bias=None if b is None else dev(b, t), act=act, cfg=cfg)
        close(got, want, tol)
