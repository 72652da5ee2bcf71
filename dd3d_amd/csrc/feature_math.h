// Element types, activations with two derivatives, and the counter-based random words shared by the group-norm and dropout kernels.
#pragma once
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

// dtype / activation codes of include/dd3d.h
#define DD3D_F32 0
#define DD3D_F16 1
#define DD3D_BF16 2
#define DD3D_ACT_NONE 0
#define DD3D_ACT_RELU 1
#define DD3D_ACT_LEAKY 2
#define DD3D_ACT_SILU 3
#define DD3D_ACT_GELU 4
#define DD3D_ACT_LOW_MEANS 16   // with any of them: the group norm's means in two floats

// ---- element types: every value is widened to fp32 on the way in and rounded to nearest even once on the way out ----------------
typedef _Float16 half_t;
struct bf16_t {
    uint16_t bits;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(half_t v) { return (float)v; }
__device__ __forceinline__ float widen(bf16_t v) { return __uint_as_float((uint32_t)v.bits << 16); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ half_t narrow<half_t>(float v) { return (half_t)v; }
template <>
__device__ __forceinline__ bf16_t narrow<bf16_t>(float v) {
    __bf16 h = (__bf16)v;  // gfx950 rounds to nearest even in hardware
    bf16_t r;
    __builtin_memcpy(&r.bits, &h, 2);
    return r;
}

__device__ __forceinline__ float widen_bits(uint16_t h, int dt) {
    half_t f;
    __builtin_memcpy(&f, &h, 2);
    return dt == DD3D_F16 ? (float)f : __uint_as_float((uint32_t)h << 16);
}

// parameter vectors (weight, bias and their gradients) are fp32 or of the rows' type: a code, uniform over the launch
__device__ __forceinline__ void store_param(void* p, int pdt, int64_t i, float v) {
    if (pdt == DD3D_F32) ((float*)p)[i] = v;
    else if (pdt == DD3D_F16) ((half_t*)p)[i] = narrow<half_t>(v);
    else ((bf16_t*)p)[i] = narrow<bf16_t>(v);
}

// ---- activations --------------------------------------------------------------------------------------------------------------
// Three families: piecewise linear (none / ReLU / leaky ReLU: slope 1, 0, s below zero, the border belonging to the lower side),
// SiLU u sigma(u), and GELU u Phi(u) with the normal distribution's Phi.
#define DD3D_FAM_LINEAR 0
#define DD3D_FAM_SILU 1
#define DD3D_FAM_GELU 2

__host__ __device__ __forceinline__ int act_family(int act) { return act <= DD3D_ACT_LEAKY ? DD3D_FAM_LINEAR : act == DD3D_ACT_SILU ? DD3D_FAM_SILU : DD3D_FAM_GELU; }

// The upper tail Q(a) = 1 - Phi(a) of the normal distribution, a = |u|, is n-shaped: Q(a) = exp(-a^2 / 2) t P(t) with t = 1 / (1 + 0.35 a) and P a
// degree-8 polynomial fitted for least relative error over a in [0, 14] (6.1e-8 with the coefficients as printed).  So one exponential serves Phi
// and the density alike, and on either side only one subtraction is left:
//   u Phi(u) = max(u, 0) - a Q(a),   Phi(u) + u n(u) = u > 0 ? 1 + r : -r,  r = a n(a) - Q(a),   2 n - u^2 n = n (2 - u^2).
// The exponent is a product of rounded numbers, off by up to five half steps of a^2 / 2, and so is Q, relative to itself: 3e-6 at a = 6, 1.3e-5 at 13, where
// Q is 1e-9 and 6e-39.  Carrying the square's residual would take five instructions more in every GELU.
// SHORT: results that are rounded to half width take degree 5 over t = 1 / (1 + 0.3 a), relative error 8.2e-6, a sixtieth of fp16's half step.
template <bool SHORT>
__device__ __forceinline__ void normal_tail(float a, float* e, float* pt) {
    const float s = a * 0.84932180f;   // sqrt(log2(e) / 2)
    const float t = __builtin_amdgcn_rcpf(fmaf(SHORT ? 0.3f : 0.35f, a, 1.f));
    float p;
    if (SHORT) {
        p = fmaf(-0.07709760218858719f, t, 0.21603752672672272f);
        p = fmaf(p, t, -0.016948513686656952f);
        p = fmaf(p, t, 0.14419656991958618f);
        p = fmaf(p, t, 0.11374188959598541f);
        p = fmaf(p, t, 0.12007423490285873f);
    } else {
        p = fmaf(-0.029146108776330948f, t, 0.14397257566452026f);
        p = fmaf(p, t, -0.25571608543395996f);
        p = fmaf(p, t, 0.15917624533176422f);
        p = fmaf(p, t, -0.02311127260327339f);
        p = fmaf(p, t, 0.10550861060619354f);
        p = fmaf(p, t, 0.11983271688222885f);
        p = fmaf(p, t, 0.13986189663410187f);
        p = fmaf(p, t, 0.13962140679359436f);
    }
    *e = __builtin_amdgcn_exp2f(-s * s);
    *pt = p * t;   // Q = e pt
}

// phi(u); with ORDER >= 1 also phi'(u) in *d1, with ORDER == 2 phi''(u) in *d2
// SHORT: the value alone, to be rounded to half width
template <int FAM, int ORDER, bool SHORT = false>
__device__ __forceinline__ float activate(float u, float slope, float* d1, float* d2) {
    if (FAM == DD3D_FAM_LINEAR) {
        const bool up = u > 0.f;
        if (ORDER >= 1) *d1 = up ? 1.f : slope;
        if (ORDER == 2) *d2 = 0.f;
        const float low = (slope == 0.f && u == u) ? 0.f : slope * u;  // ReLU of -inf is 0, of NaN is NaN
        return up ? u : low;
    }
    if (FAM == DD3D_FAM_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -1.44269504f));
        const float ds = s * (1.f - s);
        if (ORDER >= 1) *d1 = fmaf(u, ds, s);
        if (ORDER == 2) *d2 = ds * fmaf(u, 1.f - 2.f * s, 2.f);
        return u * s;
    }
    // From 14 on e is zero, so what it multiplies may be bounded there: infinite u give their limits (inf and 0), and u^2 of a huge u does not
    // leave fp32.  (A NaN that a bound swallows is still in e.)
    const float a = fabsf(u), near = fminf(a, 64.f);
    float e, pt;
    normal_tail<SHORT && ORDER == 0>(a, &e, &pt);
    if (ORDER >= 1) {
        const float r = e * fmaf(a, 0.39894228f, -pt);
        *d1 = u > 0.f ? 1.f + r : -r;
    }
    if (ORDER == 2) *d2 = 0.39894228f * e * fmaf(-near, near, 2.f);
    return fmaf(-near, e * pt, fmaxf(u, 0.f));
}

// ---- random words ---------------------------------------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011).  The word of element (row, c) is word
// c % 4 of the block at counter (row * ceil(C / 4) + c / 4, call) under key = seed, so it depends on neither launch shape nor type, and
// whoever needs the mask again computes it again.
struct Drop {
    const int64_t* key;  // device: {seed, call}; NULL: keep everything
    uint32_t thr;        // an element is dropped iff its word < thr, or always with `all`
    int all;
    float scale;         // 1 / (1 - p)
};

struct PhiloxKey {
    uint32_t k0, k1, c2, c3;
};

__device__ __forceinline__ PhiloxKey philox_key(const int64_t* key) {
    PhiloxKey k;
    const uint64_t s = (uint64_t)key[0], c = (uint64_t)key[1];
    const auto uniform = [](uint64_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v); };   // scalar registers
    k.k0 = uniform(s), k.k1 = uniform(s >> 32), k.c2 = uniform(c), k.c3 = uniform(c >> 32);
    return k;
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

__device__ __forceinline__ uint4 philox_block(const PhiloxKey k, uint64_t block) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = k.c2, c3 = k.c3, k0 = k.k0, k1 = k.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = xor3((uint32_t)(b >> 32), c1, k0);
        c1 = (uint32_t)b;
        c2 = xor3((uint32_t)(a >> 32), c3, k1);
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// fills thr / all / scale from p in [0, 1]; false if p is none of that
inline bool make_drop(double p, const int64_t* key, Drop* d) {
    if (!(p >= 0.0 && p <= 1.0) || (p > 0.0 && !key)) return false;
    const double t = __builtin_rint(p * 4294967296.0);
    d->key = p > 0.0 ? key : nullptr;
    d->all = t >= 4294967296.0;
    d->thr = d->all ? 0xFFFFFFFFu : (uint32_t)t;
    d->scale = d->all ? 0.f : (float)(1.0 / (1.0 - p));
    return true;
}
