"""Generate gelu16_poly.h: the polynomial of the 16-bit operators' GELU and its
slope (dense_tile.h).

    0.5 erfcx(a / sqrt(2)) ~= sum_d Q[d] t^d,  t = K / (a + K),  0 <= a <= 14

The least maximum of the relative error, found by reweighting a least-squares
fit by its own error (Lawson), in the variable in which erfcx is nearly
polynomial (gen_gelu_poly.py); degree 8 is the least that reaches binary32's own
step: the residual may cancel most of the value, and dbias may be stored in binary32.
Run `python gen_gelu16_poly.py > gelu16_poly.h`.
"""
import numpy as np
from scipy.special import erfcx

K, DEG, AMAX = float(np.float32(3.4)), 8, 14.0


def fit(n=8000, rounds=200):
    node = np.cos(np.pi * (np.arange(n) + 0.5) / n)
    lo, hi = K / (AMAX + K), 1.0
    t = (lo + hi) / 2 + (hi - lo) / 2 * node
    a = K / t - K
    V = np.vander(t, DEG + 1, increasing=True) / (0.5 * erfcx(a / np.sqrt(2.0)))[:, None]
    w = np.ones(n)
    for _ in range(rounds):
        c = np.linalg.lstsq(V * np.sqrt(w)[:, None], np.sqrt(w), rcond=None)[0]
        w *= np.abs(V @ c - 1)
        w /= w.sum()
    return c.astype(np.float32)


def main():
    c = fit()
    a = np.linspace(0.0, AMAX, 400001)
    err = np.abs(np.polyval(c.astype(np.float64)[::-1], K / (a + K)) / (0.5 * erfcx(a / np.sqrt(2.0))) - 1).max()
    print("/* Generated by gen_gelu16_poly.py: do not edit. */")
    print("#pragma once")
    print(f"/* 0.5 erfcx(a / sqrt(2)) ~= sum_d Q[d] t^d, t = K / (a + K), 0 <= a <= {AMAX:g};")
    print(f"   max relative error {err:.2e} */")
    print(f"#define CHELIS_GELU16_K {float(np.float32(K)).hex()}f")
    print(f"#define CHELIS_GELU16_DEG {DEG}")
    print("#define CHELIS_GELU16_Q { \\")
    print("    " + ", ".join(float(v).hex() + "f" for v in c) + " }")


if __name__ == "__main__":
    main()
