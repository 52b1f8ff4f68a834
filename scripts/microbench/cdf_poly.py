"""The polynomial of normal_cdf (locus_amd/csrc/product.h): how it is computed, and how far the one there is off.

(1 + 2 x) erfcx(x) as a polynomial in t = (x - 3.75) / (x + 3.75), which takes [0, inf] to [-1, 1] (Shepherd and
Laframboise, Math. Comp. 36, 1981): interpolated at the 24 Chebyshev nodes with 60 digits, then in powers of t.

    python scripts/microbench/cdf_poly.py        # coefficients, and the largest relative error of product.h's
"""
import os
import re

import mpmath as mp

DEGREE, DIGITS = 23, 60
SOURCE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "..", "locus_amd", "csrc", "product.h")


def exact(t):
    """(1 + 2 x) erfcx(x) at t < 1; 2 / sqrt(pi) at t = 1."""
    if t == 1:
        return 2 / mp.sqrt(mp.pi)
    x = mp.mpf("3.75") * (1 + t) / (1 - t)
    return (1 + 2 * x) * mp.exp(x * x) * mp.erfc(x)


def fit(degree=DEGREE):
    """Coefficients of t^0 .. t^degree."""
    n = degree + 1
    nodes = [mp.cos(mp.pi * (2 * k + 1) / (2 * n)) for k in range(n)]
    values = [exact(t) for t in nodes]
    out = [mp.mpf(0)] * n
    older, old = [mp.mpf(1)] + [mp.mpf(0)] * degree, [mp.mpf(0), mp.mpf(1)] + [mp.mpf(0)] * (degree - 1)
    for j in range(n):                                # T_j in powers of t: 1, t, 2 t T_{j-1} - T_{j-2}
        if j == 0:
            power = older
        elif j == 1:
            power = old
        else:
            power = [2 * (old[i - 1] if i else 0) - older[i] for i in range(n)]
            older, old = old, power
        c = sum(v * mp.cos(j * mp.pi * (2 * k + 1) / (2 * n)) for k, v in enumerate(values)) * (1 if j == 0 else 2) / n
        out = [o + c * p for o, p in zip(out, power)]
    return out


def committed():
    """The coefficients in product.h."""
    with open(SOURCE) as f:
        table = f.read().split("kCdfPoly[24] = {")[1].split("};")[0]
    return [float.fromhex(x) for x in re.findall(r"-?0x1\.[0-9a-f]+p[+-]\d+", table)]


def worst(coefficients, points=2001):
    """Largest relative error over [-1, 1)."""
    at = [mp.mpf(2 * i) / points - 1 for i in range(points)]
    return max(abs(mp.polyval(list(reversed(coefficients)), t) / exact(t) - 1) for t in at)


if __name__ == "__main__":
    mp.mp.dps = DIGITS
    new = fit()
    for c in new:
        print(float(c).hex())
    print("truncation", mp.nstr(worst(new, 401), 3), " product.h", mp.nstr(worst([mp.mpf(c) for c in committed()]), 3))
