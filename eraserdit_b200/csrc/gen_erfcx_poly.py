"""Derive the scaled complementary error function used by the GELU epilogue (prints C++).

``exp(z^2) erfc(z)`` for z >= 0 is written as ``t P(t)`` with ``t = 1 / (1 + p z)``
(the form of Hastings' rational approximations, Abramowitz and Stegun 7.1.25-26):
t runs over (0, 1], the function goes to zero like t, and P is smooth.  P has
degree 7; its coefficients minimise the largest relative error, by Lawson's
reweighted least squares on Chebyshev nodes, for the p with the smallest error.
The result (2.5e-7) is a few units in the last place of FP32.
"""

import numpy as np
from scipy.special import erfcx

Z_MAX = 12.0  # exp(-z^2) is zero in FP32 beyond
DEGREE = 7


def fit(p: float, nodes: int = 800) -> tuple[float, np.ndarray]:
    t_min = 1.0 / (1.0 + p * Z_MAX)
    angle = np.pi * (np.arange(nodes) + 0.5) / nodes
    t = (1 + t_min) / 2 + (1 - t_min) / 2 * np.cos(angle)
    g = erfcx((1 / t - 1) / p) / t
    basis = np.polynomial.chebyshev.chebvander(2 * t - 1, DEGREE) / g[:, None]
    w = np.ones(nodes)
    for _ in range(60):
        c, *_ = np.linalg.lstsq(basis * np.sqrt(w)[:, None], np.sqrt(w), rcond=None)
        err = np.abs(basis @ c - 1)
        w *= err / err.max() + 1e-3
        w /= w.sum()
    poly = np.polynomial.chebyshev.Chebyshev(c, domain=[0, 1])
    return float(err.max()), poly.convert(kind=np.polynomial.Polynomial).coef


if __name__ == "__main__":
    err, p, coef = min((fit(p)[0], p, None) for p in np.arange(0.25, 0.8, 0.025))
    err, coef = fit(p)
    print(f"// p = {p:.3f}, max relative error {err:.2e}")
    print(f"constexpr float kErfcxP = {float(np.float32(p / np.sqrt(2.0))).hex()}f;  // p / sqrt(2)")
    for k, c in enumerate(coef):
        print(f"constexpr float kErfcx{k} = {float(np.float32(c)).hex()}f;  // {c:.9g}")
