// Activations of the pointwise linear layer and their derivatives, in fp32.
#pragma once

#include "common.cuh"

namespace spconv {

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == SPCONV_ACT_RELU) return z < 0.f ? 0.f : z;          // NaN stays NaN
    if constexpr (ACT == SPCONV_ACT_GELU) return 0.5f * z * erfcf(z * -0.70710678f);   // 1 + erf would cancel below 0
    if constexpr (ACT == SPCONV_ACT_SILU) return z / (1.f + expf(-z));
    return z;
}

// z as a factor beside an exponential of it that is zero far out: cut off there, so that an infinite z (a kept
// product beyond fp16's range, of a finite forward) times that zero is zero. NaN comes through the exponential.
__device__ __forceinline__ float slope_factor(float z) { return fmaxf(fminf(z, 200.f), -200.f); }

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == SPCONV_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if constexpr (ACT == SPCONV_ACT_GELU)
        return 0.5f * erfcf(z * -0.70710678f) + slope_factor(z) * 0.39894228f * expf(-0.5f * z * z);
    if constexpr (ACT == SPCONV_ACT_SILU) {
        const float s = 1.f / (1.f + expf(-z));
        return s * (1.f + slope_factor(z) * (1.f - s));
    }
    return 1.f;
}

// ---------------------------------------------------------------------------------------
// Two values at a time, for 16-bit features: within 2^-20 of the argument of the functions above.
// The epilogue of a layer over millions of voxels has about 14 issue slots per output before it,
// not HBM, sets the time, so products run as packed fp32 pairs (one slot for two) and the only
// special-function operations are one exponential (GELU) or an exponential and a reciprocal (SiLU).
// ---------------------------------------------------------------------------------------
struct f32x2 { uint64_t v; };
__device__ __forceinline__ f32x2 pack_f32x2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack_f32x2(f32x2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x.v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float relu_nan(float x) {          // max(x, 0), NaN stays NaN
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
    return r;
}

// For t = min(|z|, 16): E = exp(-t^2 / 2) and -q, q = 1 - Phi(t) = E * P(t) with P a degree-9
// polynomial for exp(t^2 / 2) (1 - Phi(t)), fitted here on [0, 4.5] for the least weighted error:
// |dq| <= 6.5e-7 everywhere, and within 6e-4 of q itself up to t = 4. Beyond 16, E is zero.
constexpr float kTailScale = -0.72134752f;                 // -log2(e) / 2
__host__ __device__ constexpr float tail_coef(int k) {      // of -P
    constexpr float c[10] = {-0.49999940f, 0.39890096f, -0.24953401f, 0.13094953f, -0.057988375f,
                             0.020727100f, -0.0055298521f, 9.9795568e-4f, -1.0617938e-4f, 4.9614673e-6f};
    return c[k];
}
__device__ __forceinline__ void normal_tail2(float2 z, f32x2 &t, float2 &e, f32x2 &minus_q) {
    t = pack_f32x2(fminf(fabsf(z.x), 16.f), fminf(fabsf(z.y), 16.f));
    const float2 x = unpack_f32x2(mul2(mul2(t, t), pack_f32x2(kTailScale, kTailScale)));
    e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    f32x2 p = pack_f32x2(tail_coef(9), tail_coef(9));
#pragma unroll
    for (int k = 8; k >= 0; --k) p = fma2(p, t, pack_f32x2(tail_coef(k), tail_coef(k)));
    minus_q = mul2(p, pack_f32x2(e.x, e.y));
}

// For t = -min(|z|, 13): Phi(t) = 2^R(t), R a degree-6 polynomial for log2(Phi), which is nearly
// a parabola there: six products and one exponential, where exp(-t^2 / 2) P(t) takes twelve for the
// same accuracy. Fitted here on [-5.75, 0] for the least weighted error: within 2.6e-7 everywhere and 2^-12.3 of
// Phi itself down to -5.75. It goes on falling to its minimum near -14 (13 % above Phi at -8, where t Phi is
// -5e-15), so from -13 on t Phi counts as -4e-32.
constexpr float kLogTailEnd = 13.f;
__host__ __device__ constexpr float log_tail_coef(int k) {
    constexpr float c[7] = {-0.99999982f, 1.1511294f, -0.45898986f, 0.053147960f, 0.0079413289f, 7.3869905e-4f,
                            3.1020278e-5f};
    return c[k];
}

// act(z) for four pairs, in place, step by step across them: each step's four packed operations are
// independent, which covers one operation's latency without another warp's help. inf and NaN as the
// functions above, but GELU(-inf) = -4e-32 (its limit is 0).
template <int ACT>
__device__ __forceinline__ void act_value8(f32x2 *f) {
    if constexpr (ACT == SPCONV_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 z = unpack_f32x2(f[i]);
            f[i] = pack_f32x2(relu_nan(z.x), relu_nan(z.y));
        }
    }
    if constexpr (ACT == SPCONV_ACT_GELU) {                  // max(z, 0) + t Phi(t), t = -|z|
        f32x2 t[4], p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 z = unpack_f32x2(f[i]);
            t[i] = pack_f32x2(fmaxf(-fabsf(z.x), -kLogTailEnd), fmaxf(-fabsf(z.y), -kLogTailEnd));
            f[i] = pack_f32x2(relu_nan(z.x), relu_nan(z.y));
            p[i] = pack_f32x2(log_tail_coef(6), log_tail_coef(6));
        }
#pragma unroll
        for (int k = 5; k >= 0; --k)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = fma2(p[i], t[i], pack_f32x2(log_tail_coef(k), log_tail_coef(k)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = unpack_f32x2(p[i]);
            p[i] = pack_f32x2(ex2_approx(x.x), ex2_approx(x.y));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = fma2(t[i], p[i], f[i]);
    }
    if constexpr (ACT == SPCONV_ACT_SILU) {                  // z / (1 + exp(-z))
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = unpack_f32x2(mul2(f[i], pack_f32x2(-1.4426950f, -1.4426950f)));
            const float2 d = unpack_f32x2(add2(pack_f32x2(ex2_approx(x.x), ex2_approx(x.y)), pack_f32x2(1.f, 1.f)));
            f[i] = mul2(f[i], pack_f32x2(rcp_approx(d.x), rcp_approx(d.y)));
        }
    }
}

// act'(z) for a pair.
template <int ACT>
__device__ __forceinline__ float2 act_slope2(float2 z) {
    if constexpr (ACT == SPCONV_ACT_RELU) return make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
    if constexpr (ACT == SPCONV_ACT_GELU) {                  // Phi(z) + z phi(z)
        f32x2 t, mq;
        float2 e;
        normal_tail2(z, t, e, mq);
        const float2 u = unpack_f32x2(t), m = unpack_f32x2(mq);
        // for z > 0 the slope is 1 - (q - t phi), else q - t phi
        const float sx = fmaf(u.x * -0.39894228f, e.x, -m.x), sy = fmaf(u.y * -0.39894228f, e.y, -m.y);
        return make_float2(z.x > 0.f ? 1.f - sx : z.x == z.x ? sx : z.x, z.y > 0.f ? 1.f - sy : z.y == z.y ? sy : z.y);
    }
    if constexpr (ACT == SPCONV_ACT_SILU) {
        const float sx = rcp_approx(1.f + ex2_approx(-1.4426950f * z.x)), sy = rcp_approx(1.f + ex2_approx(-1.4426950f * z.y));
        return make_float2(sx * (1.f + slope_factor(z.x) * (1.f - sx)), sy * (1.f + slope_factor(z.y) * (1.f - sy)));
    }
    return make_float2(1.f, 1.f);
}

// Calls f with the activation as a compile-time constant.
template <typename F>
inline int act_dispatch(int activation, F f) {
    switch (activation) {
        case SPCONV_ACT_RELU: return f(std::integral_constant<int, SPCONV_ACT_RELU>{});
        case SPCONV_ACT_GELU: return f(std::integral_constant<int, SPCONV_ACT_GELU>{});
        case SPCONV_ACT_SILU: return f(std::integral_constant<int, SPCONV_ACT_SILU>{});
        default: return f(std::integral_constant<int, SPCONV_ACT_NONE>{});
    }
}

}  // namespace spconv
