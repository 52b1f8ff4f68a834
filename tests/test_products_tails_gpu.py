"""Relative accuracy of the element functions of the products and their slopes, in the tails too, against values
computed with 40 digits (mpmath).

Z itself goes through (A a column of values, B = 1: no rounding).  Bounds, in units u = eps / 2 of the type, derived
before the first run, for results that are normal numbers:
  exp(-x)          float64 2.3 units in the last place (fastmath.h) = 4.6 u, float32 the library's one = 2 u
  density          exp 4.6, the rounding of z^2 / 2 carried and applied 1, the constant and its product 2: 8 u
  Phi              1 / (u w) 2, t, u, w and their products 5, the polynomial 2, exp 4.6, carried rounding 1, products 2: 16 u
                   float32: erfc 8 (the library's), what its argument lost 1, products 1
  logistic         exp 4.6, the sum 1, the quotient 1: 7 u;  softplus: exp 4.6, log1p 4, the sum 1: 10 u
  gelu, silu       one product more: 16 u bounds all values
Slopes are sums of up to two products of these, bound by 24 u of the sum of the terms' magnitudes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
mp = pytest.importorskip("mpmath")
pytestmark = pytest.mark.gpu

DT = {"f64": torch.float64, "f32": torch.float32}
ACTS = ("logistic", "probit", "softplus", "gelu", "silu")
# how far left results stay normal numbers (z^2 / 2 or |z| of the exponential)
NORMAL = {"f64": {"normal": 37.4, "exp": 700.0}, "f32": {"normal": 12.8, "exp": 85.0}}


@pytest.fixture(scope="module")
def pr(hip):
    from locus_amd import products
    return products


def points(dtype, act):
    far = NORMAL[dtype]["normal" if act in ("probit", "gelu") else "exp"]
    rng = np.random.default_rng(len(act))
    z = np.concatenate([-rng.uniform(0, far, 150), -np.exp(rng.uniform(np.log(1e-3), np.log(far), 150)),
                        -rng.uniform(0, min(far, 12), 60), rng.uniform(0, 9, 60)])
    if act in ("logistic", "probit"):          # whose slopes vanish on both sides
        z = np.concatenate([z, rng.uniform(9, far, 60)])
    return z.astype(np.float32 if dtype == "f32" else np.float64).astype(np.float64)


def value_and_slope(act, z):
    """The value, the slope and the sum of the magnitudes of the slope's terms."""
    with mp.workdps(40):
        z = mp.mpf(z)
        s, cdf, dens = 1 / (1 + mp.exp(-z)), mp.ncdf(z), mp.npdf(z)
        a, ss = abs(z), s / (1 + mp.exp(z))
        return {"logistic": (s, ss, ss), "probit": (cdf, dens, dens), "softplus": (mp.log1p(mp.exp(z)), s, s),
                "gelu": (z * cdf, cdf + z * dens, cdf + a * dens), "silu": (z * s, s + z * ss, s + a * ss)}[act]


def check(got, want, scale, z, bound, u, what):
    """|got - want| <= bound u scale, element by element; prints the worst one."""
    with mp.workdps(40):
        off = [float(abs(mp.mpf(float(g)) - w) / s) / u for g, w, s in zip(got, want, scale)]
    i = int(np.nanargmax(off))
    print(f"{what}: at most {off[i]:.1f} units (at {z[i]})", flush=True)
    assert np.all(np.array(off) <= bound), (off[i], z[i])


@pytest.mark.parametrize("cfg", [(16, 1), (64, 1)])
@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_values(pr, act, dtype, cfg):
    t = DT[dtype]
    z = points(dtype, act)
    col = torch.from_numpy(z[:, None]).to("cuda:0").to(t)
    got = pr.dense_product(col, torch.ones((1, 1), dtype=t, device="cuda:0"), act=act, cfg=cfg)[:, 0].cpu().double()
    want = [value_and_slope(act, x)[0] for x in z]
    check(got.numpy(), want, [abs(v) for v in want], z, 16, torch.finfo(t).eps / 2, f"{act} {dtype} value")


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_slopes(pr, act, dtype):
    t = DT[dtype]
    z = points(dtype, act)
    col = torch.from_numpy(z[:, None]).to("cuda:0").to(t)
    got = pr.dense_product_grad(torch.ones_like(col), col, torch.ones((1, 1), dtype=t, device="cuda:0"), act=act, pre=col,
                                need_A=False, need_B=False, bias_grad="matrix")[2][:, 0].cpu().double()
    want = [value_and_slope(act, x) for x in z]
    check(got.numpy(), [w[1] for w in want], [w[2] for w in want], z, 24, torch.finfo(t).eps / 2, f"{act} {dtype} slope")


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("act", ["probit", "gelu"])
def test_slopes_of_huge_values(pr, act, dtype):
    """Whose squares overflow: 0 on both sides, gelu's 1 on the right; NaN stays."""
    t = DT[dtype]
    far = torch.finfo(t).max
    col = torch.tensor([[39.0], [41.0], [1e10], [far / 2], [far], [float("inf")]], dtype=t, device="cuda:0")
    col = torch.cat([col, -col, col.new_full((1, 1), float("nan"))])
    got = pr.dense_product_grad(torch.ones_like(col), col, col.new_ones((1, 1)), act=act, pre=col, need_A=False,
                                need_B=False, bias_grad="matrix")[2][:, 0].cpu().double().numpy()
    right = got[:6] - (1.0 if act == "gelu" else 0.0)
    assert np.abs(right).max() <= 1e-300 and np.abs(got[6:12]).max() <= 1e-300 and np.isnan(got[12])


def test_values_below_the_normal_numbers(pr):
    """Phi in float64 from -37.5 down, 2^-1022 and less: 8 units relative, and half of 2^-1074 each for the last product
    and the exponential before it, which is larger than the result by 90 and rounded to the same grid at worst."""
    rng = np.random.default_rng(0)
    z = np.concatenate([-rng.uniform(37.4, 38.7, 400), [-38.48, -38.6, -39.0, -40.0, -1e3]])
    col = torch.from_numpy(z[:, None]).to("cuda:0")
    got = pr.dense_product(col, col.new_ones((1, 1)), act="probit")[:, 0].cpu().numpy()
    with mp.workdps(40):
        for zi, g in zip(z, got):
            v = mp.ncdf(mp.mpf(zi))
            assert abs(mp.mpf(float(g)) - v) <= 8 * mp.mpf(2) ** -53 * v + mp.mpf(2) ** -1074, zi
