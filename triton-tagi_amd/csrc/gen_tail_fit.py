"""Coefficients of the lower tail's Mills ratio R(a) and of 1 - a R(a) in tagi_remax.h, both over sqrt(2 pi).

Both are fitted as t p(t) and t^2 q(t) in t = 1 / (1 + a / 4) over 0 <= a <= 9 by least squares
whose weights are raised where the relative error is largest (Lawson's iteration, towards the
minimax fit), p and q of degree 8. R is scaled from scipy's erfcx in float64.

    python gen_tail_fit.py
"""

import numpy as np
from numpy.polynomial import chebyshev, polynomial
from scipy.special import erfcx

SLOPE, FAR, DEGREE = 0.25, 9.0, 8


def mills(a):
    return np.sqrt(np.pi / 2) * erfcx(a / np.sqrt(2))


def fit(fn, power):
    low = 1 / (1 + SLOPE * FAR)
    mid, half = (low + 1) / 2, (1 - low) / 2
    x = np.cos(np.pi * (np.arange(2000) + 0.5) / 2000)
    t = mid + half * x
    y = fn((1 / t - 1) / SLOPE) / t**power
    weight = np.ones_like(y)
    basis = chebyshev.chebvander(x, DEGREE) / y[:, None]
    for _ in range(60):
        c = np.linalg.lstsq(basis * np.sqrt(weight)[:, None], np.sqrt(weight), rcond=None)[0]
        error = np.abs(basis @ c - 1)
        weight = np.maximum(weight * error / (weight * error).max(), 1e-12)
    out = np.zeros(1)
    for a in chebyshev.cheb2poly(c)[::-1]:
        out = polynomial.polyadd(polynomial.polymul(out, [-mid / half, 1 / half]), [a])
    return out, error.max()


if __name__ == "__main__":
    density = 1 / np.sqrt(2 * np.pi)
    for name, fn, power in (("R / t", lambda a: density * mills(a), 1),
                            ("(1 - a R) / t^2", lambda a: density * (1 - a * mills(a)), 2)):
        c, error = fit(fn, power)
        print(f"{name}: relative error {error:.1e}")
        print("  " + ", ".join(f"{a:.9e}f" for a in c[::-1]))
