// Element types, conversions and activations shared by the row operators (linear.hip, norm.hip).
#pragma once
#include "common.h"

#define ROWOPS_GRID_MAX 0x7fffffffLL

// what one lane of a wave wrote to LDS, another may read behind this (LDS executes a wave's accesses in order: nothing is waited for)
__device__ static inline void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

typedef __attribute__((ext_vector_type(2))) _Float16 srf_f16x2;

// Storage of one element and its conversions.  Every store to 16 bits rounds to nearest even ONCE, from a 32-bit value.
struct TypeF32 {
    typedef float raw;
    static constexpr int code = SCENERF_T_F32;
    __device__ static inline float to_f32(raw v) { return v; }
    __device__ static inline raw from_f32(float v) { return v; }
};
struct TypeBF16 {
    typedef uint16_t raw;
    static constexpr int code = SCENERF_T_BF16;
    __device__ static inline float to_f32(raw v) { return __uint_as_float((uint32_t)v << 16); }
    __device__ static inline raw from_f32(float v) { return (raw)pack_bf16x2(v, 0.f); }
};
struct TypeF16 {
    typedef uint16_t raw;
    static constexpr int code = SCENERF_T_F16;
    __device__ static inline float to_f32(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
    __device__ static inline raw from_f32(float v) { return __builtin_bit_cast(raw, (_Float16)v); }
};
struct TypeE4M3 {
    typedef uint8_t raw;
    static constexpr int code = SCENERF_T_E4M3;
    __device__ static inline float to_f32(raw v) { return __builtin_amdgcn_cvt_f32_fp8((int)v, 0); }
    __device__ static inline raw from_f32(float v) { return (raw)__builtin_amdgcn_cvt_pk_fp8_f32(v, 0.f, 0, false); }
};

// 16 bytes in hand as floats
template <typename E> __device__ static inline void unpack16(uint4 t, float (&v)[16 / sizeof(typename E::raw)]) {
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(typename E::raw) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else if constexpr (sizeof(typename E::raw) == 2) {
            v[2 * i] = E::to_f32((uint16_t)(w[i] & 0xffffu));
            v[2 * i + 1] = E::to_f32((uint16_t)(w[i] >> 16));
        } else {
            v[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0);
            v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1);
            v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2);
            v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3);
        }
    }
}
// 4, 8 or 16 bytes at any address: the target's unaligned access mode moves them in one instruction, so that rows of an odd length, whose
// starts no vector type is aligned to, take the same path as any (element by element they took 4 times as long)
typedef uint32_t srf_u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t srf_u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t srf_u32_any __attribute__((aligned(1)));
__device__ static inline uint4 load16(const void* p) {
    const srf_u32x4_any v = *(const srf_u32x4_any*)p;
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ static inline void store16(void* p, uint4 v) { *(srf_u32x4_any*)p = srf_u32x4_any{v.x, v.y, v.z, v.w}; }

// W consecutive elements as floats: W * sizeof(raw) is a multiple of 16 bytes
template <typename E, int W> __device__ static inline void load_vec(const typename E::raw* p, float (&v)[W]) {
    constexpr int S = 16 / (int)sizeof(typename E::raw);
    static_assert(W % S == 0, "whole 16 bytes");
#pragma unroll
    for (int i = 0; i < W; i += S) {
        float t[S];
        unpack16<E>(load16(p + i), t);
#pragma unroll
        for (int e = 0; e < S; ++e) v[i + e] = t[e];
    }
}
// The first n > 0 of them, zeros behind; tail: the row's length % W.  WHOLE: n is known to be W or more -- where a matrix's length is in
// whole pieces no lane has to branch, and a row's loads go out together (with the branch, 40,001 x 2,480 rows to 8 bits took 97 us instead
// of 76).  A row's last piece moves as 1 to 3 powers of two: element by element it cost a row of 511 twice the rest of it.
template <typename E, int AT, int N, int W> __device__ static inline void load_part(const typename E::raw* p, float (&v)[W]) {
    typedef typename E::raw raw;
    union { raw e[N]; uint8_t b1; uint16_t b2; uint32_t b4; uint64_t b8; uint4 b16; } u;
    typedef uint16_t u16_any __attribute__((aligned(1)));
    typedef uint64_t u64_any __attribute__((aligned(1)));
    constexpr int B = N * (int)sizeof(raw);
    static_assert(B <= 16, "one access");
    if constexpr (B == 1) u.b1 = *(const uint8_t*)(p + AT);
    else if constexpr (B == 2) u.b2 = *(const u16_any*)(p + AT);
    else if constexpr (B == 4) u.b4 = *(const srf_u32_any*)(p + AT);
    else if constexpr (B == 8) u.b8 = *(const u64_any*)(p + AT);
    else u.b16 = load16(p + AT);
#pragma unroll
    for (int e = 0; e < N; ++e) v[AT + e] = E::to_f32(u.e[e]);
}
template <typename E, int AT, int N, int W> __device__ static inline void store_part(typename E::raw* p, const float (&v)[W]) {
    typedef typename E::raw raw;
    union { raw e[N]; uint8_t b1; uint16_t b2; uint32_t b4; uint64_t b8; uint4 b16; } u;
    typedef uint16_t u16_any __attribute__((aligned(1)));
    typedef uint64_t u64_any __attribute__((aligned(1)));
    constexpr int B = N * (int)sizeof(raw);
#pragma unroll
    for (int e = 0; e < N; ++e) u.e[e] = E::from_f32(v[AT + e]);
    if constexpr (B == 1) *(uint8_t*)(p + AT) = u.b1;
    else if constexpr (B == 2) *(u16_any*)(p + AT) = u.b2;
    else if constexpr (B == 4) *(srf_u32_any*)(p + AT) = u.b4;
    else if constexpr (B == 8) *(u64_any*)(p + AT) = u.b8;
    else store16(p + AT, u.b16);
}
template <typename E, int TAIL, int W> __device__ static inline void load_tail(const typename E::raw* p, float (&v)[W]) {
    if constexpr (TAIL >= 4) load_part<E, 0, 4, W>(p, v);
    if constexpr (TAIL & 2) load_part<E, TAIL & 4, 2, W>(p, v);
    if constexpr (TAIL & 1) load_part<E, TAIL & 6, 1, W>(p, v);
}
template <typename E, int TAIL, int W> __device__ static inline void store_tail(typename E::raw* p, const float (&v)[W]) {
    if constexpr (TAIL >= 4) store_part<E, 0, 4, W>(p, v);
    if constexpr (TAIL & 2) store_part<E, TAIL & 4, 2, W>(p, v);
    if constexpr (TAIL & 1) store_part<E, TAIL & 6, 1, W>(p, v);
}
template <typename E, int W, bool WHOLE = false> __device__ static inline void load_some(const typename E::raw* p, int n, int tail, float (&v)[W]) {
    if (WHOLE || n >= W) {
        load_vec<E, W>(p, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = 0.f;
    if (tail == 1) load_tail<E, 1, W>(p, v);
    else if (tail == 2) load_tail<E, 2, W>(p, v);
    else if (tail == 3) load_tail<E, 3, W>(p, v);
    if constexpr (W == 8) {
        if (tail == 4) load_tail<E, 4, W>(p, v);
        else if (tail == 5) load_tail<E, 5, W>(p, v);
        else if (tail == 6) load_tail<E, 6, W>(p, v);
        else if (tail == 7) load_tail<E, 7, W>(p, v);
    }
}
template <typename E> __device__ static inline uint32_t pack2(float a, float b) {
    if constexpr (E::code == SCENERF_T_BF16) {
        return pack_bf16x2(a, b);
    } else {
        srf_f32x2 v = {a, b};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, srf_f16x2));
    }
}
template <typename E, int W> __device__ static inline void store_vec(typename E::raw* p, const float (&v)[W]) {
    if constexpr (sizeof(typename E::raw) == 4) {
#pragma unroll
        for (int i = 0; i < W; i += 4)
            store16(p + i, make_uint4(__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3])));
    } else if constexpr (sizeof(typename E::raw) == 2) {
        static_assert(W == 8, "16-bit types move 8 elements");
        store16(p, make_uint4(pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]), pack2<E>(v[4], v[5]), pack2<E>(v[6], v[7])));
    } else {
        uint32_t w[W / 4];
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[i], v[i + 1], 0, false);
            w[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[i + 2], v[i + 3], t, true);
        }
        if constexpr (W == 8) *(srf_u32x2_any*)p = srf_u32x2_any{w[0], w[1]};
        else *(srf_u32_any*)p = w[0];
    }
}
template <typename E, int W, bool WHOLE = false> __device__ static inline void store_some(typename E::raw* p, int n, int tail, const float (&v)[W]) {
    if (WHOLE || n >= W) {
        store_vec<E, W>(p, v);
        return;
    }
    if (tail == 1) store_tail<E, 1, W>(p, v);
    else if (tail == 2) store_tail<E, 2, W>(p, v);
    else if (tail == 3) store_tail<E, 3, W>(p, v);
    if constexpr (W == 8) {
        if (tail == 4) store_tail<E, 4, W>(p, v);
        else if (tail == 5) store_tail<E, 5, W>(p, v);
        else if (tail == 6) store_tail<E, 6, W>(p, v);
        else if (tail == 7) store_tail<E, 7, W>(p, v);
    }
}

// Activations and their slopes.  relu keeps NaN (a comparison, not fmaxf, which would drop it) and its slope at 0 is 0.
// gelu's normal distribution function: Phi(-x) = t P(t) exp(-x^2 / 2), t = 1 / (1 + p x), x >= 0: one exponential and one reciprocal (1 ulp each) serve
// the value and the slope, whose density is the same exponential.  For results in 16 bits P is of degree 4, Abramowitz & Stegun 7.1.26 with the
// constants of z / sqrt 2 and of the half folded in: off by at most 0.75e-7.  For results in 32 bits (FINE) that is more than their own rounding: in the
// 2-norm over normal z gelu was 8.8e-8 off and its slope 1.1e-7, with a correctly rounded erf 3.7e-8 and 3.9e-8.  There P is of degree 6, fitted here
// to the smallest largest error (least squares, weights moved to where it was largest), 2.1e-9: 4.0e-8 and 5.9e-8.  Everywhere, it would cost
// 4 us of 187 at 153,600 x 512 x 512 bf16.
// The library's erff and expf took 145 us of a step's 153,600 x 512 slopes, bound by the vector units; this takes what the bytes take.
__device__ static inline float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
#define CDF_STEP(expression)                      \
    _Pragma("unroll") for (int i = 0; i < W; ++i) expression; \
    __builtin_amdgcn_sched_barrier(0)
// Phi(z), and the exponential exp(-z^2 / 2) in e, of W values a step at a time: one after the other they are a chain of 16 dependent
// instructions each, which the compiler leaves as they are (153,600 x 512 x 512 bf16 with its sums kept 199 us so, 196 by steps)
template <int W, bool FINE> __device__ static inline void normal_cdf(const float (&z)[W], float (&c)[W], float (&e)[W]) {
    float t[W];
#pragma unroll
    for (int i = 0; i < W; ++i) t[i] = fmaf(FINE ? 0.45f : 0.23164189f, fabsf(z[i]), 1.f);
#pragma unroll
    for (int i = 0; i < W; ++i) e[i] = z[i] * z[i] * -0.72134752f;
#pragma unroll
    for (int i = 0; i < W; ++i) t[i] = __builtin_amdgcn_rcpf(t[i]);
    CDF_STEP(e[i] = __builtin_amdgcn_exp2f(e[i]));
    if constexpr (FINE) {
        CDF_STEP(c[i] = fmaf(-0.0378535874f, t[i], 0.217445642f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], -0.474038959f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], 0.393637121f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], 0.0181375835f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], 0.205400571f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], 0.177271649f) * t[i]);
    } else {
        CDF_STEP(c[i] = fmaf(0.53070271f, t[i], -0.72657601f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], 0.71070687f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], -0.14224837f));
        CDF_STEP(c[i] = fmaf(c[i], t[i], 0.12741480f) * t[i]);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) c[i] *= e[i];
#pragma unroll
    for (int i = 0; i < W; ++i) c[i] = z[i] < 0.f ? c[i] : 1.f - c[i];
}
// W values of the activation, or of its slope, in place; FINE: for results in 32 bits
template <int ACT, int W, bool FINE> __device__ static inline void act_fwd(float (&z)[W]) {
    float c[W], e[W];
    if constexpr (ACT == SCENERF_ACT_GELU) normal_cdf<W, FINE>(z, c, e);
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if constexpr (ACT == SCENERF_ACT_RELU) z[i] = z[i] < 0.f ? 0.f : z[i];
        if constexpr (ACT == SCENERF_ACT_GELU) z[i] *= c[i];
        if constexpr (ACT == SCENERF_ACT_SILU) z[i] *= __builtin_amdgcn_rcpf(1.f + fast_exp(-z[i]));
    }
}
// (A z kept in 16 bits may be the infinity that a finite sum past the type's range rounds to.  The slopes have their limits there, 0 and 1: z's
// factor is held to finite numbers, or it would be infinity times 0.  NaN comes through e, c and p.  Clamping z where it is kept instead cost the
// forward pass 8 us of 185 at 153,600 x 512 x 512 bf16; here HBM hides it.)
template <int ACT, int W, bool FINE> __device__ static inline void act_slope(float (&z)[W]) {
    constexpr float top = 3.4028234663852886e38f;
    float c[W], e[W];
    if constexpr (ACT == SCENERF_ACT_GELU) normal_cdf<W, FINE>(z, c, e);
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if constexpr (ACT == SCENERF_ACT_RELU) z[i] = z[i] > 0.f ? 1.f : 0.f;
        if constexpr (ACT == SCENERF_ACT_GELU) z[i] = fmaf(__builtin_amdgcn_fmed3f(z[i], -top, top) * 0.39894228040143268f, e[i], c[i]);
        if constexpr (ACT == SCENERF_ACT_SILU) {
            const float p = __builtin_amdgcn_rcpf(1.f + fast_exp(-z[i]));
            z[i] = p * fmaf(__builtin_amdgcn_fmed3f(z[i], -top, top), 1.f - p, 1.f);
        }
    }
}
