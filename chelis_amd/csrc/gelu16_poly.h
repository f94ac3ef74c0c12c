/* Generated by gen_gelu16_poly.py: do not edit. */
#pragma once
/* 0.5 erfcx(a / sqrt(2)) ~= sum_d Q[d] t^d, t = K / (a + K), 0 <= a <= 14;
   max relative error 2.50e-06 */
#define CHELIS_GELU16_K 0x1.b333340000000p+1f
#define CHELIS_GELU16_DEG 6
#define CHELIS_GELU16_Q { \
    -0x1.2221140000000p-13f, 0x1.eb0b260000000p-4f, 0x1.91f2560000000p-4f, 0x1.78379e0000000p-3f, -0x1.5e70c00000000p-4f, 0x1.1705680000000p-2f, -0x1.6a7f3e0000000p-4f }
