/* Generated by gen_gelu16_poly.py: do not edit. */
#pragma once
/* 0.5 erfcx(a / sqrt(2)) ~= sum_d Q[d] t^d, t = K / (a + K), 0 <= a <= 14;
   max relative error 6.33e-08 */
#define CHELIS_GELU16_K 0x1.b333340000000p+1f
#define CHELIS_GELU16_DEG 8
#define CHELIS_GELU16_Q { \
    0x1.303ee20000000p-16f, 0x1.dee0aa0000000p-4f, 0x1.f1e8a00000000p-4f, 0x1.55d01c0000000p-4f, 0x1.5a834e0000000p-3f, -0x1.f3ce060000000p-4f, 0x1.1abec80000000p-2f, -0x1.79de700000000p-3f, 0x1.41b9700000000p-5f }
