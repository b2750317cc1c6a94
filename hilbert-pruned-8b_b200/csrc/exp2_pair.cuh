// Pairs of float32 in one 64-bit register (fma.rn.f32x2 and its kin work on both halves in one instruction), and 2^x of a pair
// on the FMA pipe, for kernels whose exponentials are bound by the special-function unit (16 a clock and SM).
#pragma once
#include "common.cuh"

typedef unsigned long long f32x2;

__device__ __forceinline__ f32x2 pair_of(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void pair_parts(f32x2 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ f32x2 pair_fma(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 pair_add(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ f32x2 pair_mul(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 2^x of both halves, x at most 127 (below -125: 2^-125 instead of a smaller number; NaN gives NaN).  x = n + f with n
// the nearest integer (adding and taking away 1.5 * 2^23 rounds to it), 2^f by the polynomial of degree DEG with the smallest largest
// relative error on [-1/2, 1/2] (equal ripples, found by exchanging extrema), times 2^n built from its exponent's bits.  Relative error at
// most 2.7e-6 (degree 4, 4e-8 on average) and 2.2e-7 (degree 5).
template <int DEG>
__device__ __forceinline__ void exp2_pair(f32x2 x, float& a, float& b) {
    static_assert(DEG == 4 || DEG == 5, "built for degrees 4 and 5");
    float x0, x1;
    pair_parts(x, x0, x1);
    x = pair_of(max_or_nan(x0, -125.0f), max_or_nan(x1, -125.0f));
    const f32x2 r = pair_add(x, pair_of(12582912.0f, 12582912.0f));
    const f32x2 n = pair_add(r, pair_of(-12582912.0f, -12582912.0f));
    const f32x2 f = pair_fma(n, pair_of(-1.0f, -1.0f), x);
    f32x2 p;
    if (DEG == 5) {
        p = pair_fma(f, pair_of(0.0013276472454890609f, 0.0013276472454890609f), pair_of(0.009675540961325169f, 0.009675540961325169f));
        p = pair_fma(f, p, pair_of(0.05550713092088699f, 0.05550713092088699f));
        p = pair_fma(f, p, pair_of(0.24022120237350464f, 0.24022120237350464f));
        p = pair_fma(f, p, pair_of(0.6931469440460205f, 0.6931469440460205f));
        p = pair_fma(f, p, pair_of(1.0000001192092896f, 1.0000001192092896f));
    } else {
        p = pair_fma(f, pair_of(0.009570102207362652f, 0.009570102207362652f), pair_of(0.05591785907745361f, 0.05591785907745361f));
        p = pair_fma(f, p, pair_of(0.240247443318367f, 0.240247443318367f));
        p = pair_fma(f, p, pair_of(0.6931217908859253f, 0.6931217908859253f));
        p = pair_fma(f, p, pair_of(0.9999992847442627f, 0.9999992847442627f));
    }
    float r0, r1;
    pair_parts(r, r0, r1);
    const f32x2 two_n = pair_of(__uint_as_float((__float_as_uint(r0) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(r1) << 23) + 0x3f800000u));
    pair_parts(pair_mul(p, two_n), a, b);
}
