"""Generate gelu_poly.h: the polynomial of the binary32 GELU default-mode
path (chain.h gelu_fast_f32).

    0.5 erfcx(a / sqrt(2)) ~= sum_d Q[d] u^d,  u = (a - K) / (a + K),  0 <= a <= 13

with K the binary32 nearest 3 sqrt(2) (so u is computed from a = |x|
directly, and z = a / sqrt(2) below).

The variable change u = (z - K') / (z + K') maps [0, inf) onto [-1, 1) and
makes erfcx nearly polynomial in u (Shepherd and Laframboise, "Chebyshev
approximation of (1 + 2x) exp(x^2) erfc x in 0 <= x < inf", Math. Comp. 36
(1981) 249-253). The fit is a relative least-squares fit on 20000
Chebyshev nodes in u against scipy's binary64 erfcx, rounded to binary32;
the rounded polynomial's relative error over the range (printed to stderr
and into the header, about 4.4e-8) is below one binary32 ulp. Run `python gen_gelu_poly.py > gelu_poly.h`.
"""
import struct
import sys

import numpy as np
from scipy.special import erfcx

K = float(np.float32(3.0 * np.sqrt(2.0)))
DEG = 9
AMAX = 13.0


def fit(n=20000):
    umin, umax = -1.0, (AMAX - K) / (AMAX + K)
    t = np.cos(np.pi * (np.arange(n) + 0.5) / n)
    u = (umin + umax) / 2 + (umax - umin) / 2 * t
    a = K * (1 + u) / (1 - u)
    f = 0.5 * erfcx(a / np.sqrt(2.0))
    V = np.vander(u, DEG + 1, increasing=True)
    c, *_ = np.linalg.lstsq(V / f[:, None], np.ones_like(f), rcond=None)
    return c.astype(np.float32)


def hexf(v: np.float32) -> str:
    return float(v).hex() + "f"


def main():
    c = fit()
    a = np.linspace(0.0, AMAX, 400001)
    u = (a - K) / (a + K)
    err = np.abs(np.polyval(c.astype(np.float64)[::-1], u) / (0.5 * erfcx(a / np.sqrt(2.0))) - 1).max()
    print(f"gen_gelu_poly: max relative error of the binary32 coefficients {err:.3e}", file=sys.stderr)
    print("/* Generated by gen_gelu_poly.py: do not edit. */")
    print("#pragma once")
    print(f"/* 0.5 erfcx(a / sqrt(2)) ~= sum_d Q[d] u^d, u = (a - K) / (a + K), K = {float(np.float32(K)).hex()},")
    print(f"   0 <= a <= {AMAX:g};")
    print(f"   max relative error {err:.2e} */")
    print(f"#define CHELIS_GELU_K {hexf(np.float32(K))}")
    print(f"#define CHELIS_GELU_DEG {DEG}")
    print("#define CHELIS_GELU_Q { \\")
    print("    " + ", ".join(hexf(v) for v in c) + " }")


if __name__ == "__main__":
    main()
