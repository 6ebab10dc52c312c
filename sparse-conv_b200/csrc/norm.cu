// The gated residual step between two blocks, with a norm on either side of it, and its
// gradients, for row-major features [M, C] in fp32, fp16 or bf16:
//
//   u = N1(x) * w1 + b1            (the norm after a block; N1 may be absent: u = x)
//   h = alpha * r + g * u          (gate and residual; either may be absent)
//   y = N2(h) * w2 + b2            (the norm before the next block; N2 may be absent: no y)
//
// N is LayerNorm ((t - mean) * rstd) or RMSNorm (t * rstd), rstd = 1 / sqrt(mean square + eps).
// Each of g, w1, b1, w2, b2 is one row of C channels or one row per sample of the batch; the
// rows of sample s are offsets[s] .. offsets[s + 1] - 1.
//
// Backward, from dh and dy (either may be absent), with t = dy * w2:
//   G  = dh + rstd2 * (t - mean(t) - hhat * mean(t * hhat))       (RMS: without mean(t))
//   dr = alpha * G;  du = G * g;  dx = N1's gradient of du * w1, by the same formula
//   dw2 = sum dy * hhat, db2 = sum dy, dg = sum G * u, dw1 = sum du * xhat, db1 = sum du
// over all rows, or over a sample's rows. The forward keeps four fp32 numbers a row (mean and rstd
// of both norms); u and h are recomputed from x and r in fp32, so the forward's rounding of h does
// not enter the gradients, and x and r are as many bytes as x and h would be. Recomputing the
// statistics too would save those 16 bytes a row and cost two more reductions over the row, which
// are what bounds the backward after HBM.
//
// Bound: HBM. Forward reads x, r and writes h, y; backward reads x, r, dh, dy and writes dx, dr.
// All arithmetic is fp32; each output is rounded once. A row lives in the registers of the
// lanes that own it, so every tensor is read once.
#include <algorithm>
#include <numeric>
#include <type_traits>

#include "common.cuh"

namespace spconv {

constexpr int kRnThreads = 256;
constexpr int kRnWarps = kRnThreads / 32;
constexpr int kRnMaxC = 8192;
constexpr int kRnMaxSamples = 65535;   // a grid dimension of the gradient sums
// parameter slots, and the order of their partial sums
enum { kG = 0, kW1 = 1, kB1 = 2, kW2 = 3, kB2 = 4, kRnParams = 5 };
// products the ring kernel keeps beside them: g * w1 and g * b1
enum { kGW = 5, kGB = 6, kRbParams = 7 };

struct RnArgs {
    const void *x, *r;                   // r may be null
    void *h, *y;                         // forward outputs (y null without N2)
    const void *dh, *dy;                 // backward inputs (either may be null)
    void *dx, *dr;                       // backward outputs (either may be null)
    float4 *stats;                       // [M] mean1, rstd1, mean2, rstd2 (forward: may be null)
    const void *p[kRnParams];            // parameters (null: 1 for g, w; 0 for b)
    int p_f32[kRnParams];                // 1: fp32, 0: the features' type
    int64_t p_stride[kRnParams];         // C if there is a row per sample, else 0
    int slot[kRnParams];                 // backward: position among the sums wanted, or -1
    int nslots;
    float *partial;                      // [G + B][nslots][C]
    const int32_t *offsets;              // [B + 1], used when a parameter has a row per sample
    int B;
    int64_t M;
    int C;
    int lpr;                             // lanes per row (unused where a block takes a row)
    int64_t chunk;                       // consecutive rows per CTA
    int norm1, norm2;
    float alpha, eps;
    int32_t *status;
};

// VEC consecutive values of one row: eight (one or two 16-byte loads) or one.
template <typename T, int VEC> struct RnPack;
template <> struct RnPack<float, 8> { uint4 q[2]; };
template <> struct RnPack<__half, 8> { uint4 q[1]; };
template <> struct RnPack<__nv_bfloat16, 8> { uint4 q[1]; };
template <typename T> struct RnPack<T, 1> { T v; };

template <typename T>
__device__ __forceinline__ void rn_load(RnPack<T, 8> &p, const T *src) {
    const uint4 *s = reinterpret_cast<const uint4 *>(src);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(p.q) / 16); ++i) p.q[i] = __ldcs(s + i);
}
template <typename T>
__device__ __forceinline__ void rn_load(RnPack<T, 1> &p, const T *src) { p.v = *src; }

__device__ __forceinline__ void rn_unpack(const RnPack<float, 8> &p, float *f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(p.q[i].x);
        f[4 * i + 1] = __uint_as_float(p.q[i].y);
        f[4 * i + 2] = __uint_as_float(p.q[i].z);
        f[4 * i + 3] = __uint_as_float(p.q[i].w);
    }
}
__device__ __forceinline__ void rn_unpack(const RnPack<__half, 8> &p, float *f) {
    const __half2 *h = reinterpret_cast<const __half2 *>(p.q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(h[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
__device__ __forceinline__ void rn_unpack(const RnPack<__nv_bfloat16, 8> &p, float *f) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(p.q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <typename T>
__device__ __forceinline__ void rn_unpack(const RnPack<T, 1> &p, float *f) { f[0] = dtype_traits<T>::to_f(p.v); }

__device__ __forceinline__ void rn_store(float *dst, const float *f, RnPack<float, 8> *) {
    __stcs(reinterpret_cast<float4 *>(dst), make_float4(f[0], f[1], f[2], f[3]));
    __stcs(reinterpret_cast<float4 *>(dst) + 1, make_float4(f[4], f[5], f[6], f[7]));
}
template <typename T>
__device__ __forceinline__ void rn_store(T *dst, const float *f, RnPack<T, 8> *) {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = dtype_traits<T>::from_f(f[i]);
    uint4 q;
    memcpy(&q, v, 16);
    __stcs(reinterpret_cast<uint4 *>(dst), q);
}
template <typename T>
__device__ __forceinline__ void rn_store(T *dst, const float *f, RnPack<T, 1> *) { *dst = dtype_traits<T>::from_f(f[0]); }

// VEC values of parameter k's row for sample s from column col (its default where it is absent).
template <typename T, int VEC>
__device__ __forceinline__ void rn_param(const RnArgs &a, int k, int s, int col, float *f) {
    if (a.p[k] == nullptr) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = (k == kB1 || k == kB2) ? 0.f : 1.f;
        return;
    }
    const int64_t at = (int64_t)s * a.p_stride[k] + col;
    if (a.p_f32[k]) {
        const float *q = (const float *)a.p[k] + at;
        if constexpr (VEC == 8) {
            const float4 u = __ldg((const float4 *)q), v = __ldg((const float4 *)q + 1);
            f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
            f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
        } else {
            f[0] = __ldg(q);
        }
    } else {
        RnPack<T, VEC> p;
        if constexpr (VEC == 8) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(p.q) / 16); ++i) p.q[i] = __ldg((const uint4 *)((const T *)a.p[k] + at) + i);
        } else {
            p.v = ((const T *)a.p[k])[at];
        }
        rn_unpack(p, f);
    }
}

// Sums of U pairs of values over the lanes that share a row: lpr lanes of a warp (WARPS == 0), or a
// block of WARPS warps, whose sums meet in `scratch` [2][WARPS]. The halves take turns, so that one
// barrier a sum is enough: between two uses of a half lies the other's barrier. Without `both` only the
// second of each pair is summed.
struct RnScratch {
    float2 *part;
    int half;
};
template <int U, int WARPS>
__device__ __forceinline__ void rn_sum2(float (&u)[U], float (&v)[U], bool both, int lpr, RnScratch &scratch) {
    const int top = WARPS ? 16 : lpr >> 1;
    if (both) {
        for (int o = top; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < U; ++i) {
                u[i] += __shfl_xor_sync(0xffffffffu, u[i], o);
                v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
            }
    } else {
        for (int o = top; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < U; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    if constexpr (WARPS > 1) {
        static_assert(U == 1, "a block takes one row at a time");
        float2 *part = scratch.part + scratch.half * WARPS;
        scratch.half ^= 1;
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(u[0], v[0]);
        __syncthreads();
        u[0] = v[0] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            u[0] += part[w].x;
            v[0] += part[w].y;
        }
    }
}

// Sum of a lane's N values, and of their products with n, as trees (short chains).
template <int N>
__device__ __forceinline__ float rn_tree(const float (&t)[N]) {
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = t[i];
#pragma unroll
    for (int n = N; n > 1; n = (n + 1) / 2)
#pragma unroll
        for (int i = 0; i < n / 2; ++i) s[i] += s[i + (n + 1) / 2];
    return s[0];
}
template <int N>
__device__ __forceinline__ float rn_dot(const float (&t)[N], const float (&n)[N]) {
    float p = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        p = fmaf(t[i], n[i], p);
        if (i + 1 < N) q = fmaf(t[i + 1], n[i + 1], q);
    }
    return p + q;
}

// Normalises U rows, N values of each in a lane, in place: (mean, rstd) of each row in st. Columns
// that a lane does not have hold zeros, before and after (FULL: it has them all).
template <typename T, int U, int N, int VEC, int WARPS, bool FULL>
__device__ __forceinline__ void rn_normalise(float (&t)[U][N], float2 (&st)[U], const bool *have, int kind, float inv_c,
                                             float eps, int lpr, RnScratch &scratch) {
    if (kind == SPCONV_NORM_NONE) {
#pragma unroll
        for (int u = 0; u < U; ++u) st[u] = make_float2(0.f, 1.f);
        return;
    }
    // 16-bit features, eight columns a lane: one reduction, of d and d^2 for d = t - c, c the mean of the row's
    // first eight values, which lies within sqrt(C / 8) deviations of the row's mean: mean(d^2) - mean(d)^2
    // then costs at most the factor C / 8 + 1 in the variance's rounding, whatever offset the row has
    // in common; 4e-6 of 1 / deviation measured at C = 256 with the first eight a thousand times the others, under
    // a hundredth of the outputs' rounding. Two reductions, the mean first, then the squares, cost nothing at
    // 64 and 128 channels and 4 to 13 % at 32, 96, 200 and 256 (500,000 x 200 bf16 forward 271 -> 306 us). fp32 takes
    // them (2e-7 for that row; 250,000 x 200 156 -> 183 us, no difference at powers of two), as do single columns a
    // lane and a block a row.
    constexpr bool ONE = sizeof(T) == 2 && VEC == 8 && WARPS == 0;
    float s[U], q[U], shift[U];
    const bool layer = kind == SPCONV_NORM_LAYER;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        shift[u] = s[u] = q[u] = 0.f;
        if (layer) {
            if constexpr (ONE) {
                float head[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) head[i] = t[u][i];
                shift[u] = __shfl_sync(0xffffffffu, rn_tree<8>(head) * 0.125f, 0, lpr);
            } else {
                s[u] = rn_tree<N>(t[u]);
            }
        }
    }
    if (!ONE && layer) {
        rn_sum2<U, WARPS>(s, q, true, lpr, scratch);
#pragma unroll
        for (int u = 0; u < U; ++u) shift[u] = s[u] * inv_c;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (layer) {
#pragma unroll
            for (int i = 0; i < N; ++i) t[u][i] = FULL || have[i / VEC] ? t[u][i] - shift[u] : 0.f;
            s[u] = ONE ? rn_tree<N>(t[u]) : 0.f;
        }
        q[u] = rn_dot<N>(t[u], t[u]);
    }
    rn_sum2<U, WARPS>(s, q, layer && ONE, lpr, scratch);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float m = layer && ONE ? s[u] * inv_c : 0.f;
        const float var = q[u] * inv_c - m * m;
        const float rstd = rsqrtf((var < 0.f ? 0.f : var) + eps);            // NaN stays NaN
        st[u] = make_float2(shift[u] + m, rstd);
        const float offset = -m * rstd;
#pragma unroll
        for (int i = 0; i < N; ++i) t[u][i] = FULL || have[i / VEC] ? fmaf(t[u][i], rstd, offset) : 0.f;
    }
}

// t: gradient at the normalised values n -> gradient at the values before the norm, added to g.
template <int U, int N, int WARPS>
__device__ __forceinline__ void rn_normalise_back(float (&g)[U][N], float (&t)[U][N], const float (&n)[U][N],
                                                  const float (&rstd)[U], int kind, float inv_c, int lpr, RnScratch &scratch) {
    if (kind == SPCONV_NORM_NONE) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) g[u][i] += t[u][i];
        return;
    }
    float s[U], q[U];
    const bool layer = kind == SPCONV_NORM_LAYER;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        s[u] = layer ? rn_tree<N>(t[u]) : 0.f;
        q[u] = rn_dot<N>(t[u], n[u]);
    }
    rn_sum2<U, WARPS>(s, q, layer, lpr, scratch);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float mean = layer ? s[u] * inv_c * rstd[u] : 0.f, along = q[u] * inv_c * rstd[u];
#pragma unroll
        for (int i = 0; i < N; ++i) g[u][i] = fmaf(t[u][i], rstd[u], fmaf(-n[u][i], along, g[u][i] - mean));
    }
}

// The sample of row r (offsets ascending), always in [0, B).
__device__ __forceinline__ int rn_sample(const RnArgs &a, int64_t r) {
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {                        // first s with offsets[s + 1] > r
        const int mid = (lo + hi) >> 1;
        if ((int64_t)__ldg(a.offsets + mid + 1) > r) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Offsets have to ascend from 0 to M; whatever they hold, rows are assigned inside [0, B).
__device__ __forceinline__ void rn_check_offsets(const RnArgs &a) {
    if (blockIdx.x != 0 || !a.offsets) return;
    bool bad = false;
    for (int s = threadIdx.x; s < a.B; s += blockDim.x) {
        const int lo = __ldg(a.offsets + s), hi = __ldg(a.offsets + s + 1);
        bad |= lo > hi || (s == 0 && lo != 0) || (s == a.B - 1 && hi != a.M);
    }
    if (bad) raise_status(a.status, SPCONV_STATUS_OFFSETS);
}

// Direct form: rows from global memory into registers and back, the next row's loads under this one's
// sums. For few rows (short and latency-bound: the ring would not fill), for more than 256 channels,
// where a block of WARPS warps takes a row, and for tensors off 16-byte boundaries.
//
// A block takes `chunk` consecutive rows, sample by sample, and its row groups (lpr lanes, or the
// block) take the rows of a sample in turn. A lane owns at most 8 columns, whose parameters stay in
// registers for a sample's rows, and in the backward their sums too: a block of as many warps as that
// takes beats a warp with more columns a lane (100,000 x 333 fp16: 3.2 ms forward with 32 single
// columns a lane).
template <typename T, int VEC, int VPT, int WARPS>
struct RnDirect {
    static constexpr int N = VEC * VPT;
    static constexpr int kThreads = WARPS ? WARPS * 32 : kRnThreads;
    static_assert(N <= 8, "parameters and sums stay in registers");
};

template <typename T, int VEC, int VPT, int WARPS>
__global__ void __launch_bounds__(RnDirect<T, VEC, VPT, WARPS>::kThreads)
residual_norm_fwd_kernel(const __grid_constant__ RnArgs a) {
    constexpr int N = VEC * VPT, kThreads = RnDirect<T, VEC, VPT, WARPS>::kThreads;
    __shared__ float2 part[2 * (WARPS ? WARPS : 1)];
    RnScratch scratch{part, 0};
    rn_check_offsets(a);
    const int C = a.C, lpr = WARPS ? kThreads : a.lpr;
    const int groups = kThreads / lpr, group = threadIdx.x / lpr, lane = threadIdx.x & (lpr - 1);
    const float inv_c = 1.f / (float)C;
    int col[VPT];
    bool have[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        col[j] = (lane + lpr * j) * VEC;
        have[j] = col[j] < C;
    }
    const int64_t row0 = (int64_t)blockIdx.x * a.chunk, row1 = min(a.M, row0 + a.chunk);
    int s = a.B > 1 && row0 < row1 ? rn_sample(a, row0) : 0;
    for (int64_t seg = row0; seg < row1; ++s) {
        const int64_t end = s < a.B - 1 ? min(row1, (int64_t)__ldg(a.offsets + s + 1)) : row1;
        if (end <= seg) continue;            // an empty sample
        float pg[N], pw1[N], pb1[N], pw2[N], pb2[N];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = have[j] ? col[j] : 0;
            rn_param<T, VEC>(a, kG, s, c, pg + j * VEC);
            rn_param<T, VEC>(a, kW1, s, c, pw1 + j * VEC);
            rn_param<T, VEC>(a, kB1, s, c, pb1 + j * VEC);
            rn_param<T, VEC>(a, kW2, s, c, pw2 + j * VEC);
            rn_param<T, VEC>(a, kB2, s, c, pb2 + j * VEC);
        }
        RnPack<T, VEC> px[VPT], pr[VPT];
        auto fetch = [&](int64_t row) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                px[j] = RnPack<T, VEC>{};
                pr[j] = RnPack<T, VEC>{};
                if (row < end && have[j]) {
                    rn_load(px[j], (const T *)a.x + row * C + col[j]);
                    if (a.r) rn_load(pr[j], (const T *)a.r + row * C + col[j]);
                }
            }
        };
        fetch(seg + group);
        for (int64_t base = seg; base < end; base += groups) {
            const int64_t row = base + group;
            float u[1][N], h[1][N];
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                rn_unpack(px[j], u[0] + j * VEC);
                rn_unpack(pr[j], h[0] + j * VEC);
            }
            fetch(row + groups);
            float2 st1[1], st2[1];
            rn_normalise<T, 1, N, VEC, WARPS, false>(u, st1, have, a.norm1, inv_c, a.eps, lpr, scratch);
#pragma unroll
            for (int n = 0; n < N; ++n)
                h[0][n] = have[n / VEC] ? a.alpha * h[0][n] + pg[n] * (u[0][n] * pw1[n] + pb1[n]) : 0.f;
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if (have[j] && row < end) rn_store((T *)a.h + row * C + col[j], h[0] + j * VEC, (RnPack<T, VEC> *)nullptr);
            rn_normalise<T, 1, N, VEC, WARPS, false>(h, st2, have, a.norm2, inv_c, a.eps, lpr, scratch);
            if (a.norm2 != SPCONV_NORM_NONE) {
#pragma unroll
                for (int n = 0; n < N; ++n) h[0][n] = h[0][n] * pw2[n] + pb2[n];
#pragma unroll
                for (int j = 0; j < VPT; ++j)
                    if (have[j] && row < end) rn_store((T *)a.y + row * C + col[j], h[0] + j * VEC, (RnPack<T, VEC> *)nullptr);
            }
            if (a.stats && lane == 0 && row < end) a.stats[row] = make_float4(st1[0].x, st1[0].y, st2[0].x, st2[0].y);
        }
        seg = end;
    }
}

// As the forward's walk. When a sample's rows in the chunk end, the parameter sums are written as record
// blockIdx + s (added up over the block's warps first, in a fixed order, where those share rows' columns):
// along a walk through the chunks and samples that index only grows, so each (chunk, sample) pair that
// holds rows has a record of its own and at most G + B - 1 are needed.
template <typename T, int VEC, int VPT, int WARPS>
__global__ void __launch_bounds__(RnDirect<T, VEC, VPT, WARPS>::kThreads)
residual_norm_bwd_kernel(const __grid_constant__ RnArgs a) {
    constexpr int N = VEC * VPT, kThreads = RnDirect<T, VEC, VPT, WARPS>::kThreads;
    extern __shared__ float s_acc[];         // WARPS == 0: [kRnWarps][nslots][C]
    __shared__ float2 part[2 * (WARPS ? WARPS : 1)];
    RnScratch scratch{part, 0};
    rn_check_offsets(a);
    const int C = a.C, lpr = WARPS ? kThreads : a.lpr, warp = threadIdx.x >> 5;
    const int groups = kThreads / lpr, group = threadIdx.x / lpr, lane = threadIdx.x & (lpr - 1);
    const float inv_c = 1.f / (float)C;
    int col[VPT];
    bool have[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        col[j] = (lane + lpr * j) * VEC;
        have[j] = col[j] < C;
    }
    const int64_t row0 = (int64_t)blockIdx.x * a.chunk, row1 = min(a.M, row0 + a.chunk);
    int s = a.B > 1 && row0 < row1 ? rn_sample(a, row0) : 0;
    for (int64_t seg = row0; seg < row1; ++s) {
        const int64_t end = s < a.B - 1 ? min(row1, (int64_t)__ldg(a.offsets + s + 1)) : row1;
        if (end <= seg) continue;
        float pg[N], pw1[N], pb1[N], pw2[N];
        float sum_g[N], sum_gn[N], sum_y[N], sum_yn[N];       // of G, G * xhat, dy, dy * hhat
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = have[j] ? col[j] : 0;
            rn_param<T, VEC>(a, kG, s, c, pg + j * VEC);
            rn_param<T, VEC>(a, kW1, s, c, pw1 + j * VEC);
            rn_param<T, VEC>(a, kB1, s, c, pb1 + j * VEC);
            rn_param<T, VEC>(a, kW2, s, c, pw2 + j * VEC);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) sum_g[n] = sum_gn[n] = sum_y[n] = sum_yn[n] = 0.f;
        RnPack<T, VEC> px[VPT], pr[VPT], ph[VPT], py[VPT];
        auto fetch = [&](int64_t row) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                px[j] = RnPack<T, VEC>{};
                pr[j] = RnPack<T, VEC>{};
                ph[j] = RnPack<T, VEC>{};
                py[j] = RnPack<T, VEC>{};
                if (row < end && have[j]) {
                    const int64_t at = row * C + col[j];
                    rn_load(px[j], (const T *)a.x + at);
                    if (a.r) rn_load(pr[j], (const T *)a.r + at);
                    if (a.dh) rn_load(ph[j], (const T *)a.dh + at);
                    if (a.dy) rn_load(py[j], (const T *)a.dy + at);
                }
            }
        };
        fetch(seg + group);
        for (int64_t base = seg; base < end; base += groups) {
            const int64_t row = base + group;
            const bool live = row < end;         // a row past the end holds zeros and adds none
            float n1[1][N], n2[1][N], t[1][N], g[1][N];       // xhat, hhat, dy * w2, dh -> G
            const float4 st = live ? __ldg(a.stats + row) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                rn_unpack(px[j], n1[0] + j * VEC);
                rn_unpack(pr[j], n2[0] + j * VEC);
                rn_unpack(ph[j], g[0] + j * VEC);
                rn_unpack(py[j], t[0] + j * VEC);
            }
            fetch(row + groups);
            const float rstd1[1] = {st.y}, rstd2[1] = {st.w};
#pragma unroll
            for (int n = 0; n < N; ++n) n1[0][n] = have[n / VEC] ? (n1[0][n] - st.x) * st.y : 0.f;
            if (a.norm2 != SPCONV_NORM_NONE && a.dy) {
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const float h = a.alpha * n2[0][n] + pg[n] * (n1[0][n] * pw1[n] + pb1[n]);
                    n2[0][n] = have[n / VEC] ? (h - st.z) * st.w : 0.f;
                    sum_y[n] += t[0][n];
                    sum_yn[n] = fmaf(t[0][n], n2[0][n], sum_yn[n]);
                    t[0][n] *= pw2[n];
                }
                rn_normalise_back<1, N, WARPS>(g, t, n2, rstd2, a.norm2, inv_c, lpr, scratch);
#pragma unroll
                for (int n = 0; n < N; ++n) g[0][n] = have[n / VEC] && live ? g[0][n] : 0.f;
            }
            if (a.dr) {
#pragma unroll
                for (int n = 0; n < N; ++n) t[0][n] = a.alpha * g[0][n];
#pragma unroll
                for (int j = 0; j < VPT; ++j)
                    if (have[j] && live) rn_store((T *)a.dr + row * C + col[j], t[0] + j * VEC, (RnPack<T, VEC> *)nullptr);
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                sum_g[n] += g[0][n];
                sum_gn[n] = fmaf(g[0][n], n1[0][n], sum_gn[n]);
                g[0][n] *= pg[n] * pw1[n];
                t[0][n] = 0.f;
            }
            if (a.dx) {
                rn_normalise_back<1, N, WARPS>(t, g, n1, rstd1, a.norm1, inv_c, lpr, scratch);
#pragma unroll
                for (int j = 0; j < VPT; ++j)
                    if (have[j] && live) rn_store((T *)a.dx + row * C + col[j], t[0] + j * VEC, (RnPack<T, VEC> *)nullptr);
            }
        }
        if (a.nslots > 0) {
            const int n_rec = a.nslots * C;
            float *rec = a.partial + ((int64_t)blockIdx.x + s) * n_rec;
            float *dst = WARPS ? rec : s_acc + (int64_t)warp * n_rec;
            if constexpr (WARPS == 0) {      // lanes of a warp that own the same columns
#pragma unroll
                for (int n = 0; n < N; ++n)
                    for (int o = lpr; o < 32; o <<= 1) {
                        sum_g[n] += __shfl_xor_sync(0xffffffffu, sum_g[n], o);
                        sum_gn[n] += __shfl_xor_sync(0xffffffffu, sum_gn[n], o);
                        sum_y[n] += __shfl_xor_sync(0xffffffffu, sum_y[n], o);
                        sum_yn[n] += __shfl_xor_sync(0xffffffffu, sum_yn[n], o);
                    }
            }
            // G's sums give the gate's, weight's and bias's: u = xhat * w1 + b1 and du = G * g with w1, b1
            // and g the same for all of a sample's rows
            if (WARPS || (int)(threadIdx.x & 31) < lpr) {
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int c = col[n / VEC] + n % VEC;
                    if (!have[n / VEC]) continue;
                    if (a.slot[kG] >= 0) dst[a.slot[kG] * C + c] = pw1[n] * sum_gn[n] + pb1[n] * sum_g[n];
                    if (a.slot[kW1] >= 0) dst[a.slot[kW1] * C + c] = pg[n] * sum_gn[n];
                    if (a.slot[kB1] >= 0) dst[a.slot[kB1] * C + c] = pg[n] * sum_g[n];
                    if (a.slot[kB2] >= 0) dst[a.slot[kB2] * C + c] = sum_y[n];
                    if (a.slot[kW2] >= 0) dst[a.slot[kW2] * C + c] = sum_yn[n];
                }
            }
            if constexpr (WARPS == 0) {
                __syncthreads();
                for (int i = threadIdx.x; i < n_rec; i += kThreads) {
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < kRnWarps; ++w) v += s_acc[(int64_t)w * n_rec + i];
                    rec[i] = v;
                }
                __syncthreads();
            }
        }
        seg = end;
    }
}

// ---------------------------------------------------------------------------------------
// Rows of at most 256 channels, many of them: the streams through shared memory.
//
// Rows are contiguous, so R of them are one untiled bulk copy per tensor whatever the channel
// count. One thread keeps a ring of stages of such copies in flight; the other warps compute in
// place (the outputs take the inputs' slots) and the same thread stores finished stages in bulk.
// The direct kernels above hold what is in flight in registers (two loads a lane); measured
// there and here: 2.0 M x 64 bf16 forward 255 and 172 us (6.0 TB/s), 1.34 M x 128 forward 328 and
// 243 us (5.7 TB/s), backward 738 and 426 us (4.9 TB/s). Nothing is full in the backward: 47 instructions a
// value take 51 % of the issue slots, the bytes 75 % of HBM's copy rate; the 10 warps an SM that its registers
// leave wait for fixed latencies, shared memory and the row reductions' shuffles.
// A tile that crosses a sample's end is worked off in two parts, so tiles stay aligned to 16
// bytes for every channel count; only the last one can end in a few odd bytes, which that thread
// copies itself.
// Waits are bounded: a timeout raises SPCONV_STATUS_WAIT_TIMEOUT and the CTA leaves once its
// copies have landed.
// ---------------------------------------------------------------------------------------
constexpr int kRbMaxStages = 8;
constexpr int kRbTileBytes = 12 * 1024;      // a tensor's share of a stage, about
constexpr int kRbMaxSmem = 226 * 1024;

struct RbArgs {
    int rows;                                // per tile, a multiple of 8
    int stages;
    int tile_bytes;                          // a tensor's slot in a stage
    int cols;                                // columns of the parameters in shared memory: every lane's
    uint64_t wait_ns;
};

template <typename T, int VEC>
__device__ __forceinline__ void rn_load_smem(RnPack<T, VEC> &p, const T *src) {
    if constexpr (VEC == 8) {
        const uint4 *s = reinterpret_cast<const uint4 *>(src);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(p.q) / 16); ++i) p.q[i] = s[i];
    } else {
        p.v = *src;
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void rn_store_smem(T *dst, const float *f) {
    if constexpr (VEC == 8) {
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = dtype_traits<T>::from_f(f[i]);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(v) / 16); ++i) reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<uint4 *>(v)[i];
    } else {
        *dst = dtype_traits<T>::from_f(f[0]);
    }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t mbar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(mbar) : "memory");
}
__device__ __forceinline__ void bulk_store(void *dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" :: "l"(dst), "r"(src), "r"(bytes) : "memory");
}

template <typename T, int VEC, int VPT, bool BWD, bool FULL, int W, int U>
__global__ void __launch_bounds__((W + 1) * 32, 1)
residual_norm_bulk_kernel(const __grid_constant__ RnArgs a, const __grid_constant__ RbArgs rb) {
    constexpr int N = VEC * VPT;
    constexpr int kSums = 4;                 // of G, G * xhat, dy, dy * hhat
    constexpr int kTensors = BWD ? 4 : 2;    // slots of a stage: x (then h or dx), r (then y or dr), dh, dy
    extern __shared__ __align__(128) uint8_t s_raw[];
    uint64_t *full = reinterpret_cast<uint64_t *>(s_raw), *done = full + kRbMaxStages, *flush = done + kRbMaxStages;
    volatile int *s_abort = reinterpret_cast<volatile int *>(flush + 1);
    uint8_t *ring = s_raw + 256;
    const int S = rb.stages, R = rb.rows, C = a.C, lpr = a.lpr;
    const int slot = rb.tile_bytes, stage = kTensors * slot + R * 16;          // the rows' statistics last
    float *s_par = reinterpret_cast<float *>(ring + S * stage);                // [kRbParams][rb.cols]
    float *s_acc = s_par + kRbParams * rb.cols;                                // [W][nslots][C]
    const int tid = threadIdx.x, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&done[i]), W);
        }
        mbar_init(smem_u32(flush), W);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    rn_check_offsets(a);
    __syncthreads();
    auto wait = [&](uint64_t *b, uint32_t parity) { return mbar_wait_suspended(smem_u32(b), parity, s_abort, rb.wait_ns); };
    const int64_t row0 = (int64_t)blockIdx.x * a.chunk, row1 = min(a.M, row0 + a.chunk);
    const int tiles = row0 < row1 ? (int)((row1 - row0 + R - 1) / R) : 0;

    if (warp == W) {
        // ------------------------------------------------------------------ copies
        if ((tid & 31) == 0) {
            const T *in[4] = {(const T *)a.x, (const T *)a.r, BWD ? (const T *)a.dh : nullptr, BWD ? (const T *)a.dy : nullptr};
            T *out[2] = {BWD ? (T *)a.dx : (T *)a.h, BWD ? (T *)a.dr : (T *)a.y};
            auto load = [&](int t, int s) {
                const int64_t row = row0 + (int64_t)t * R;
                const int rows = (int)min((int64_t)R, row1 - row), elems = rows * C;
                const uint32_t whole = (uint32_t)(elems * (int)sizeof(T)) & ~15u, mbar = smem_u32(&full[s]);
                uint8_t *base = ring + s * stage;
                uint32_t total = BWD ? (uint32_t)rows * 16 : 0;
                for (int k = 0; k < kTensors; ++k)
                    if (in[k]) {
                        total += whole;
                        for (int e = (int)(whole / sizeof(T)); e < elems; ++e)
                            reinterpret_cast<T *>(base + k * slot)[e] = in[k][row * C + e];
                    }
                mbar_arrive_expect_tx(mbar, total);
                if (BWD) bulk_load(smem_u32(base + kTensors * slot), a.stats + row, (uint32_t)rows * 16, mbar);
                if (whole > 0)
                    for (int k = 0; k < kTensors; ++k)
                        if (in[k]) bulk_load(smem_u32(base + k * slot), in[k] + row * C, whole, mbar);
            };
            int loaded = 0;
            for (; loaded < min(S, tiles); ++loaded) load(loaded, loaded);
            int s = 0, prev = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = 0; t < tiles; ++t) {
                if (!wait(&done[s], phase)) { ok = false; break; }
                const int64_t row = row0 + (int64_t)t * R;
                const int rows = (int)min((int64_t)R, row1 - row), elems = rows * C;
                const uint32_t whole = (uint32_t)(elems * (int)sizeof(T)) & ~15u;
                uint8_t *base = ring + s * stage;
                for (int k = 0; k < 2; ++k)
                    if (out[k]) {
                        if (whole > 0) bulk_store(out[k] + row * C, smem_u32(base + k * slot), whole);
                        for (int e = (int)(whole / sizeof(T)); e < elems; ++e)
                            out[k][row * C + e] = reinterpret_cast<T *>(base + k * slot)[e];
                    }
                if (!BWD && a.stats) bulk_store(a.stats + row, smem_u32(base + kTensors * slot), (uint32_t)rows * 16);
                bulk_commit();
                // the stage before this one is free once its stores have read it
                if (t > 0 && loaded < tiles) {
                    bulk_wait_read<1>();
                    load(loaded++, prev);
                }
                prev = s;
                if (++s == S) {
                    s = 0;
                    phase ^= 1u;
                }
            }
            if (!ok)                          // loads in flight write shared memory: let them land
                for (int i = 0; i < min(S, loaded); ++i) {
                    const int uses = (loaded - 1 - i) / S;    // completed phases of stage i before its last load
                    mbar_wait_bounded(smem_u32(&full[i]), (uint32_t)(uses & 1), kTmaDrainNs);
                }
            bulk_wait<0>();
        }
    } else {
        // ------------------------------------------------------------------ rows
        const int groups = W * 32 / lpr, group = tid / lpr, lane = tid & (lpr - 1);
        const float inv_c = 1.f / (float)C;
        int col[VPT];
        bool have[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            col[j] = (lane + lpr * j) * VEC;
            have[j] = FULL || col[j] < C;
        }
        float acc[kSums][BWD ? N : 1] = {};
        RnScratch scratch{nullptr, 0};       // rows stay within a warp
        uint32_t flush_phase = 0;
        // All row warps: an mbarrier rather than bar.sync, since its wait is bounded.
        auto meet = [&]() {
            __syncwarp();
            if ((tid & 31) == 0) mbar_arrive(smem_u32(flush));
            const bool ok = __all_sync(0xffffffffu, wait(flush, flush_phase)) != 0;
            flush_phase ^= 1u;
            return ok;
        };
        // Puts the sums of sample `from`'s rows (if any) into record blockIdx + from, and sample
        // `to`'s parameters (if any) into shared memory. False: give up.
        auto turn = [&](int from, int to) -> bool {
            if constexpr (BWD) {
                if (from >= 0) {
                    // G's sums give the gate's, weight's and bias's: u = xhat * w1 + b1 and du = G * g with
                    // w1, b1 and g the same for all of a sample's rows
                    float *mine = s_acc + (int64_t)warp * a.nslots * C;
#pragma unroll
                    for (int k = 0; k < kSums; ++k)
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            for (int o = lpr; o < 32; o <<= 1) acc[k][i] += __shfl_xor_sync(0xffffffffu, acc[k][i], o);
                    if ((tid & 31) < lpr) {
#pragma unroll
                        for (int j = 0; j < VPT; ++j)
                            if (have[j])
#pragma unroll
                                for (int i = 0; i < VEC; ++i) {
                                    const int c = col[j] + i, n = j * VEC + i;
                                    const float g = s_par[kG * rb.cols + c], w = s_par[kW1 * rb.cols + c], b = s_par[kB1 * rb.cols + c];
                                    if (a.slot[kG] >= 0) mine[a.slot[kG] * C + c] = w * acc[1][n] + b * acc[0][n];
                                    if (a.slot[kW1] >= 0) mine[a.slot[kW1] * C + c] = g * acc[1][n];
                                    if (a.slot[kB1] >= 0) mine[a.slot[kB1] * C + c] = g * acc[0][n];
                                    if (a.slot[kB2] >= 0) mine[a.slot[kB2] * C + c] = acc[2][n];
                                    if (a.slot[kW2] >= 0) mine[a.slot[kW2] * C + c] = acc[3][n];
                                }
                    }
                }
            }
            if (!meet()) return false;       // every warp is through with `from`
            if constexpr (BWD) {
                if (from >= 0) {
                    const int n = a.nslots * C;
                    float *rec = a.partial + ((int64_t)blockIdx.x + from) * n;
                    for (int i = tid; i < n; i += W * 32) {
                        float v = 0.f;
#pragma unroll
                        for (int w = 0; w < W; ++w) v += s_acc[(int64_t)w * n + i];
                        rec[i] = v;
                    }
#pragma unroll
                    for (int k = 0; k < kSums; ++k)
#pragma unroll
                        for (int i = 0; i < N; ++i) acc[k][i] = 0.f;
                }
            }
            if (to >= 0)
                for (int c = tid; c < rb.cols; c += W * 32) {
                    float v[kRnParams][1];
#pragma unroll
                    for (int k = 0; k < kRnParams; ++k) {
                        rn_param<T, 1>(a, k, to, c < C ? c : 0, v[k]);
                        s_par[k * rb.cols + c] = v[k][0];
                    }
                    s_par[kGW * rb.cols + c] = v[kG][0] * v[kW1][0];
                    s_par[kGB * rb.cols + c] = v[kG][0] * v[kB1][0];
                }
            return meet();
        };
        // VEC parameters of a kind from the lane's j-th columns (rb.cols covers every lane's)
        auto par = [&](int k, int j, float *f) {
            const float *p = s_par + k * rb.cols + col[j];
            if constexpr (VEC == 8) {
                const float4 u = reinterpret_cast<const float4 *>(p)[0], v = reinterpret_cast<const float4 *>(p)[1];
                f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
                f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
            } else {
                f[0] = *p;
            }
        };
        auto par_all = [&](int k, float (&f)[N]) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) par(k, j, f + j * VEC);
        };
        // rows counted from the chunk's first: 32 bits
        const int rows_here = (int)(row1 - row0);
        int smp = a.B > 1 && tiles > 0 ? rn_sample(a, row0) : 0;
        auto sample_end = [&](int q) {
            return q < a.B - 1 ? (int)max((int64_t)0, min(row1, (int64_t)__ldg(a.offsets + q + 1)) - row0) : rows_here;
        };
        int s_end = tiles > 0 ? sample_end(smp) : 0;
        bool ok = tiles > 0 && turn(-1, smp);
        int s = 0;
        uint32_t phase = 0;
        for (int tile0 = 0; tile0 < rows_here && ok; tile0 += R) {
            ok = __all_sync(0xffffffffu, wait(&full[s], phase)) != 0;
            if (!ok) break;
            const int tile1 = min(rows_here, tile0 + R);
            uint8_t *base_s = ring + s * stage;
            T *tx = reinterpret_cast<T *>(base_s), *tr = reinterpret_cast<T *>(base_s + slot);
            const T *th = reinterpret_cast<const T *>(base_s + (BWD ? 2 * slot : 0));
            const T *ty = reinterpret_cast<const T *>(base_s + (BWD ? 3 * slot : 0));
            float4 *ts = reinterpret_cast<float4 *>(base_s + kTensors * slot);
            // U rows a group, from `base` of the tile on; TAIL: some of them may be past `last`
            auto rows = [&](auto tail, int base, int last) {
                constexpr bool TAIL = decltype(tail)::value;
                int at[U];
                bool live[U];
                float n1[U][N], n2[U][N], p[N], q[N];
                auto read = [&](int u, const T *src, float *f) {
#pragma unroll
                    for (int j = 0; j < VPT; ++j) {
                        RnPack<T, VEC> v;
                        if constexpr (!TAIL && FULL) {
                            rn_load_smem<T, VEC>(v, src + at[u] + col[j]);
                        } else {
                            v = RnPack<T, VEC>{};
                            if (live[u] && have[j]) rn_load_smem<T, VEC>(v, src + at[u] + col[j]);
                        }
                        rn_unpack(v, f + j * VEC);
                    }
                };
                auto write = [&](int u, T *dst, const float *f) {
#pragma unroll
                    for (int j = 0; j < VPT; ++j)
                        if ((!TAIL || live[u]) && have[j]) rn_store_smem<T, VEC>(dst + at[u] + col[j], f + j * VEC);
                };
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int row = base + group + u * groups;
                    live[u] = !TAIL || row < last;
                    at[u] = row * C;
                    read(u, tx, n1[u]);
                    if (a.r) read(u, tr, n2[u]);
                    else
#pragma unroll
                        for (int n = 0; n < N; ++n) n2[u][n] = 0.f;
                }
                // xhat in n1 -> h in n2 (zero in columns a lane does not have)
                auto hidden = [&]() {
                    par_all(kGW, p);
                    par_all(kGB, q);
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int n = 0; n < N; ++n)
                            n2[u][n] = have[n / VEC] ? fmaf(n1[u][n], p[n], fmaf(a.alpha, n2[u][n], q[n])) : 0.f;
                };
                if constexpr (!BWD) {
                    float2 st1[U], st2[U];
                    rn_normalise<T, U, N, VEC, 0, FULL>(n1, st1, have, a.norm1, inv_c, a.eps, lpr, scratch);
                    hidden();
#pragma unroll
                    for (int u = 0; u < U; ++u) write(u, tx, n2[u]);
                    rn_normalise<T, U, N, VEC, 0, FULL>(n2, st2, have, a.norm2, inv_c, a.eps, lpr, scratch);
                    if (a.norm2 != SPCONV_NORM_NONE) {
                        par_all(kW2, p);
                        par_all(kB2, q);
#pragma unroll
                        for (int u = 0; u < U; ++u) {
#pragma unroll
                            for (int n = 0; n < N; ++n) n2[u][n] = fmaf(n2[u][n], p[n], q[n]);
                            write(u, tr, n2[u]);
                        }
                    }
                    if (a.stats && lane == 0) {
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (live[u]) ts[base + group + u * groups] = make_float4(st1[u].x, st1[u].y, st2[u].x, st2[u].y);
                    }
                } else {
                    float g[U][N], t2[U][N], rstd1[U], rstd2[U], shift2[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const float4 st = live[u] ? ts[base + group + u * groups] : make_float4(0.f, 0.f, 0.f, 0.f);
                        rstd1[u] = st.y;
                        rstd2[u] = st.w;
                        shift2[u] = -st.z * st.w;
                        const float shift1 = -st.x * st.y;
#pragma unroll
                        for (int n = 0; n < N; ++n) n1[u][n] = fmaf(n1[u][n], st.y, shift1);
                        if (a.dh) read(u, th, g[u]);
                        else
#pragma unroll
                            for (int n = 0; n < N; ++n) g[u][n] = 0.f;
                    }
                    // dh and dy are zero in rows past the end and in columns a lane does not have, so
                    // those add nothing to any sum
                    if (a.norm2 != SPCONV_NORM_NONE && a.dy) {
                        hidden();
                        par_all(kW2, p);
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            read(u, ty, t2[u]);
#pragma unroll
                            for (int n = 0; n < N; ++n) {
                                n2[u][n] = fmaf(n2[u][n], rstd2[u], shift2[u]);
                                acc[2][n] += t2[u][n];
                                acc[3][n] = fmaf(t2[u][n], n2[u][n], acc[3][n]);
                                t2[u][n] *= p[n];
                            }
                        }
                        rn_normalise_back<U, N, 0>(g, t2, n2, rstd2, a.norm2, inv_c, lpr, scratch);
                        if constexpr (TAIL || !FULL) {
#pragma unroll
                            for (int u = 0; u < U; ++u)
#pragma unroll
                                for (int n = 0; n < N; ++n) g[u][n] = have[n / VEC] && live[u] ? g[u][n] : 0.f;
                        }
                    }
                    if (a.dr) {
#pragma unroll
                        for (int u = 0; u < U; ++u) {
#pragma unroll
                            for (int n = 0; n < N; ++n) t2[u][n] = a.alpha * g[u][n];
                            write(u, tr, t2[u]);
                        }
                    }
                    par_all(kGW, p);
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int n = 0; n < N; ++n) {
                            acc[0][n] += g[u][n];
                            acc[1][n] = fmaf(g[u][n], n1[u][n], acc[1][n]);
                            g[u][n] *= p[n];
                            t2[u][n] = 0.f;
                        }
                    if (a.dx) {
                        rn_normalise_back<U, N, 0>(t2, g, n1, rstd1, a.norm1, inv_c, lpr, scratch);
#pragma unroll
                        for (int u = 0; u < U; ++u) write(u, tx, t2[u]);
                    }
                }
            };
            for (int part = tile0; part < tile1;) {
                if (s_end <= part) {         // the next sample that has rows (the last one takes the rest)
                    const int from = smp;
                    do s_end = sample_end(++smp);
                    while (s_end <= part);
                    if (!turn(from, smp)) { ok = false; break; }
                }
                const int end = min(tile1, s_end), last = end - tile0;
                int base = part - tile0;
                for (; base + groups * U <= last; base += groups * U) rows(std::false_type{}, base, last);
                if (base < last) rows(std::true_type{}, base, last);
                part = end;
            }
            if (!ok) break;
            fence_proxy_async_smem();
            __syncwarp();
            if ((tid & 31) == 0) mbar_arrive(smem_u32(&done[s]));
            if (++s == S) {
                s = 0;
                phase ^= 1u;
            }
        }
        if (BWD && ok) turn(smp, -1);
    }
    __syncthreads();
    if (*s_abort && tid == 0) raise_status(a.status, SPCONV_STATUS_WAIT_TIMEOUT);
}

struct RnGradArgs {
    void *out[kRnParams];                // by slot
    int out_f32[kRnParams], per_sample[kRnParams];
};

// Adds the records of each parameter up: all of them, or a sample's. blockIdx.y is the slot,
// blockIdx.z the sample (only 0 for a parameter of one row). 32 columns x 32 record lanes.
template <typename T>
__global__ void __launch_bounds__(1024)
residual_norm_grad_kernel(const __grid_constant__ RnArgs a, const __grid_constant__ RnGradArgs o) {
    __shared__ float part[32][33];
    const int k = blockIdx.y;
    const int c = blockIdx.x * 32 + threadIdx.x;
    if (!o.per_sample[k] && blockIdx.z != 0) return;
    grid_dependency_wait();
    // Rows before offsets[1] belong to sample 0 and rows from offsets[B - 1] on to the last, as in the walk.
    auto first_row = [&](int s) { return s == 0 ? (int64_t)0 : max((int64_t)0, min(a.M, (int64_t)__ldg(a.offsets + s))); };
    auto end_row = [&](int s) { return s == a.B - 1 ? a.M : max((int64_t)0, min(a.M, (int64_t)__ldg(a.offsets + s + 1))); };
    auto record = [&](int64_t chunk, int s) { return c < a.C ? __ldcg(a.partial + ((chunk + s) * a.nslots + k) * a.C + c) : 0.f; };
    const int64_t chunks = (a.M + a.chunk - 1) / a.chunk;
    float v = 0.f;
    if (o.per_sample[k]) {
        const int s = blockIdx.z;
        const int64_t lo = first_row(s), hi = end_row(s);
        if (lo < hi)
            for (int64_t b = lo / a.chunk + threadIdx.y; b <= (hi - 1) / a.chunk; b += 32) v += record(b, s);
    } else {
        for (int64_t b = threadIdx.y; b < chunks; b += 32) {
            const int64_t r0 = b * a.chunk, r1 = min(a.M, r0 + a.chunk);
            if (a.B == 1) {
                v += record(b, 0);
                continue;
            }
            const int last = rn_sample(a, r1 - 1);
            for (int s = rn_sample(a, r0); s <= last; ++s)
                if (max(r0, first_row(s)) < min(r1, end_row(s))) v += record(b, s);
        }
    }
    part[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && c < a.C) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) sum += part[i][threadIdx.x];
        const int64_t at = (o.per_sample[k] ? (int64_t)blockIdx.z * a.C : 0) + c;
        if (o.out_f32[k]) ((float *)o.out[k])[at] = sum;
        else ((T *)o.out[k])[at] = dtype_traits<T>::from_f(sum);
    }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
static int rn_pow2(int n) {
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}

// Blocks for M rows: enough to fill the SMs, no more than there are row groups. Beyond 256 channels a block takes a row
// at a time, so it is the blocks an SM has room for that keep rows in flight. Forward, LayerNorm on both sides,
// bf16, by blocks per SM: 100,000 x 512 154 us at four, 117 at six, 92 at twelve, no less at more; 50,000 x 1024 160, 106
// and 96 us at two, four and six; 50,000 x 2048 375, 240 and 213 us at one, two and three; 20,000 x 4096 571 us
// at one and at two. The backward, which keeps more registers a thread, is up to 9 % faster with fewer (155 us at
// six and 171 at twelve for 512 channels, 157 at three and 171 at six for 1024, 394 at one and 415 at three for
// 2048), but the workspace is sized for one number. Up to 256 channels few rows come here, and the number hardly
// matters forward (20,000 x 64 10 to 12 us, 40,000 x 256 29 us at one to 24); backward 40,000 x 256 takes 65, 48, 56 and
// 73 us at one, two, four and eight, 20,000 x 64 19, 19, 28 and 30 us.
static int64_t rn_grid(int64_t M, int C, int rows_per_block) {
    const int64_t per_sm = C <= 256 ? 4 : C <= 512 ? 12 : C <= 1024 ? 6 : C <= 2048 ? 3 : 1;
    return std::max<int64_t>(1, std::min<int64_t>(148 * per_sm, (M + rows_per_block - 1) / rows_per_block));
}

template <typename T, int VEC, int VPT, int WARPS>
static int rn_launch(RnArgs &a, bool backward, cudaStream_t st) {
    constexpr int threads = RnDirect<T, VEC, VPT, WARPS>::kThreads;
    int64_t grid = rn_grid(a.M, a.C, WARPS ? 1 : threads / a.lpr);
    a.chunk = (a.M + grid - 1) / grid;
    grid = (a.M + a.chunk - 1) / a.chunk;
    if (!backward) {
        residual_norm_fwd_kernel<T, VEC, VPT, WARPS><<<(unsigned)grid, threads, 0, st>>>(a);
        return check_launch("residual_norm_fwd_kernel");
    }
    const size_t smem = WARPS ? 0 : (size_t)kRnWarps * a.nslots * a.C * sizeof(float);    // at most 40 KB
    residual_norm_bwd_kernel<T, VEC, VPT, WARPS><<<(unsigned)grid, threads, smem, st>>>(a);
    return check_launch("residual_norm_bwd_kernel");
}

// The ring form: C <= 256 (a lane's sums stay in registers), tensors on 16-byte boundaries, and at
// least two tiles per SM, or the ring never fills: below that the direct kernel spreads the rows over
// more blocks.
template <typename T, int VEC, int VPT, bool BWD, bool FULL>
static bool rb_launch(RnArgs &a, cudaStream_t st, int &rc) {
    constexpr bool backward = BWD;
    constexpr int N = VEC * VPT;
    // Warps and rows in hand, measured at 1.34 M x 128 bf16: forward with 12 warps 246 us at two rows of
    // sixteen columns a lane, 340 us at one; backward with 10 warps 438 us at two rows of eight, with
    // 12 (128 registers) 490 us, with 8 504 us, with 20 at one row 769 us.
    constexpr int W = BWD ? 10 : 12, U = 2;
    const int row_bytes = a.C * (int)sizeof(T), groups = W * 32 / a.lpr * U;
    const int unit = std::lcm(groups, 8);    // whole passes, and tiles of whole 16 bytes
    RbArgs rb = {};
    rb.rows = unit * std::max(1, kRbTileBytes / (row_bytes * unit));
    const int64_t tiles = (a.M + rb.rows - 1) / rb.rows;
    if (tiles < 2 * 148) return false;
    rb.tile_bytes = (rb.rows * row_bytes + 127) & ~127;
    rb.cols = a.lpr * VPT * VEC;
    const int extra = 256 + (kRbParams * rb.cols + (backward ? W * a.nslots * a.C : 0)) * (int)sizeof(float);
    const int stage = (backward ? 4 : 2) * rb.tile_bytes + rb.rows * 16;
    rb.stages = std::min(kRbMaxStages, (kRbMaxSmem - extra) / stage);
    if (rb.stages < 3) return false;         // two do not keep HBM busy: 1.34 M x 128 backward 438 -> 663 us
    rb.wait_ns = wait_limit_ns();
    a.chunk = (tiles + 147) / 148 * rb.rows;
    const int grid = (int)((a.M + a.chunk - 1) / a.chunk);
    const int smem = extra + rb.stages * stage;
    auto kern = residual_norm_bulk_kernel<T, VEC, VPT, BWD, FULL, W, U>;
    static std::atomic<uint64_t> set{0};
    if (allow_smem(kern, kRbMaxSmem, set) != cudaSuccess) {
        rc = check_launch("residual_norm_bulk: set max dynamic shared memory");
        return true;
    }
    kern<<<grid, (W + 1) * 32, smem, st>>>(a, rb);
    rc = check_launch("residual_norm_bulk_kernel");
    return true;
}

// Columns a lane owns: eight neighbours at a time where rows and parameters allow 16-byte
// accesses, single columns otherwise; the fewest that cover the row with one warp, and eight with as
// many warps as cover it beyond 256 channels.
template <typename T>
static int rn_dispatch(RnArgs &a, bool vec, bool aligned, bool backward, cudaStream_t st) {
    const int C = a.C;
    int rc = SPCONV_OK;
    if (aligned && C <= 256) {
        // FULL: the lanes' columns are exactly the row's (a power of two): no column is ever checked
        bool ran = false;
        if (vec && !backward && C % 16 == 0 && C >= 64) {    // half the shuffles of eight columns a lane
            a.lpr = rn_pow2(C / 16);
            ran = a.lpr * 16 == C ? rb_launch<T, 8, 2, false, true>(a, st, rc) : rb_launch<T, 8, 2, false, false>(a, st, rc);
        } else if (vec) {
            a.lpr = rn_pow2(C / 8);
            const bool full = a.lpr * 8 == C;
            ran = backward ? (full ? rb_launch<T, 8, 1, true, true>(a, st, rc) : rb_launch<T, 8, 1, true, false>(a, st, rc))
                           : (full ? rb_launch<T, 8, 1, false, true>(a, st, rc) : rb_launch<T, 8, 1, false, false>(a, st, rc));
        } else {
            // single columns: as few lanes a row as eight columns each allow, and no more columns each than
            // that takes (35 channels: 8 lanes of 5)
            a.lpr = 1;
            while ((C + a.lpr - 1) / a.lpr > 8) a.lpr <<= 1;
            auto single = [&](auto per) {
                constexpr int P = decltype(per)::value;
                return backward ? rb_launch<T, 1, P, true, false>(a, st, rc) : rb_launch<T, 1, P, false, false>(a, st, rc);
            };
            const int per = (C + a.lpr - 1) / a.lpr;
            ran = per <= 4 ? single(std::integral_constant<int, 4>{}) : per == 5 ? single(std::integral_constant<int, 5>{})
                : per == 6 ? single(std::integral_constant<int, 6>{}) : per == 7 ? single(std::integral_constant<int, 7>{})
                : single(std::integral_constant<int, 8>{});
        }
        if (ran) return rc;
    }
    a.lpr = std::min(32, rn_pow2(vec ? C / 8 : C));
    if (vec) {
        if (C <= 256) return rn_launch<T, 8, 1, 0>(a, backward, st);
        if (C <= 512) return rn_launch<T, 8, 1, 2>(a, backward, st);
        if (C <= 1024) return rn_launch<T, 8, 1, 4>(a, backward, st);
        if (C <= 2048) return rn_launch<T, 8, 1, 8>(a, backward, st);
        return rn_launch<T, 8, 1, 32>(a, backward, st);
    }
    if (C <= 32) return rn_launch<T, 1, 1, 0>(a, backward, st);
    if (C <= 64) return rn_launch<T, 1, 2, 0>(a, backward, st);
    if (C <= 128) return rn_launch<T, 1, 4, 0>(a, backward, st);
    if (C <= 256) return rn_launch<T, 1, 8, 0>(a, backward, st);
    if (C <= 512) return rn_launch<T, 1, 8, 2>(a, backward, st);
    if (C <= 1024) return rn_launch<T, 1, 8, 4>(a, backward, st);
    if (C <= 2048) return rn_launch<T, 1, 8, 8>(a, backward, st);
    return rn_launch<T, 1, 8, 32>(a, backward, st);
}

static bool rn_aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Checks the call and fills the kernels' arguments (all but lpr and chunk).
static int rn_args(const spconv_residual_norm_args *q, RnArgs &a, bool &vec, bool &aligned, bool backward) {
    SPCONV_REQUIRE(q != nullptr, SPCONV_ERR_ARG, "null argument block");
    SPCONV_REQUIRE(q->dtype == SPCONV_F32 || q->dtype == SPCONV_F16 || q->dtype == SPCONV_BF16, SPCONV_ERR_ARG,
                   "unsupported dtype code %d", q->dtype);
    SPCONV_REQUIRE(q->num_rows >= 0 && q->num_rows < ((int64_t)1 << 31), SPCONV_ERR_ARG, "rows must be in [0, 2^31)");
    SPCONV_REQUIRE(q->channels >= 1 && q->channels <= kRnMaxC, SPCONV_ERR_ARG, "channels must be in [1, %d], got %d",
                   kRnMaxC, q->channels);
    SPCONV_REQUIRE(q->norm >= 0 && q->norm <= 2 && q->next_norm >= 0 && q->next_norm <= 2, SPCONV_ERR_ARG,
                   "unknown norm kind %d / %d", q->norm, q->next_norm);
    SPCONV_REQUIRE(q->num_samples >= 1 && q->num_samples <= kRnMaxSamples, SPCONV_ERR_ARG,
                   "samples must be in [1, %d], got %d", kRnMaxSamples, q->num_samples);
    if (q->num_rows == 0) return SPCONV_OK;
    SPCONV_REQUIRE(q->feats != nullptr, SPCONV_ERR_ARG, "null pointer argument");
    a.x = q->feats;
    a.r = q->residual;
    a.h = q->hidden;
    a.y = q->normed;
    a.dh = q->grad_hidden;
    a.dy = q->grad_normed;
    a.dx = q->grad_feats;
    a.dr = q->grad_residual;
    a.M = q->num_rows;
    a.C = q->channels;
    a.norm1 = q->norm;
    a.norm2 = q->next_norm;
    a.alpha = q->residual_scale;
    a.eps = q->eps;
    a.status = q->status;
    a.stats = (float4 *)q->row_stats;
    SPCONV_REQUIRE(rn_aligned(a.stats), SPCONV_ERR_ARG, "row_stats is not 16-byte aligned");
    a.offsets = nullptr;                     // only read where a parameter has a row per sample
    a.B = 1;
    a.nslots = 0;
    a.partial = (float *)q->workspace;
    const spconv_channel_param *ps[kRnParams] = {&q->gate, &q->weight, &q->bias, &q->next_weight, &q->next_bias};
    vec = q->channels % 8 == 0;
    aligned = true;
    for (const void *p : {a.x, a.r, (const void *)a.h, (const void *)a.y, a.dh, a.dy, (const void *)a.dx, (const void *)a.dr})
        aligned = aligned && rn_aligned(p);
    vec = vec && aligned;
    for (int k = 0; k < kRnParams; ++k) {
        const spconv_channel_param &p = *ps[k];
        a.p[k] = p.data;
        a.p_f32[k] = p.dtype == SPCONV_F32;
        a.p_stride[k] = p.per_sample ? q->channels : 0;
        a.slot[k] = -1;
        if (!p.data) {
            SPCONV_REQUIRE(!p.grad, SPCONV_ERR_ARG, "a gradient of an absent parameter");
            continue;
        }
        SPCONV_REQUIRE(p.dtype == SPCONV_F32 || p.dtype == q->dtype, SPCONV_ERR_ARG,
                       "parameters must be fp32 or of the features' type");
        vec = vec && rn_aligned(p.data);
        if (p.per_sample) {
            a.B = q->num_samples;
            a.offsets = q->offsets;
        }
        if (backward && p.grad) a.slot[k] = a.nslots++;
    }
    for (const auto *p : ps)
        SPCONV_REQUIRE(!p->data || !p->per_sample || a.offsets, SPCONV_ERR_ARG,
                       "a parameter per sample needs the samples' row offsets");
    return SPCONV_OK;
}

template <typename F>
static int rn_by_type(int dtype, F f) {
    if (dtype == SPCONV_F32) return f((float *)nullptr);
    if (dtype == SPCONV_F16) return f((__half *)nullptr);
    return f((__nv_bfloat16 *)nullptr);
}

}  // namespace spconv

using namespace spconv;

extern "C" int64_t spconv_residual_norm_workspace_bytes(int64_t num_rows, int channels, int num_samples) {
    if (num_rows < 0 || channels < 1 || channels > kRnMaxC || num_samples < 1 || num_samples > kRnMaxSamples) return -1;
    return (rn_grid(num_rows, channels, 1) + num_samples) * kRnParams * channels * (int64_t)sizeof(float);
}

extern "C" int spconv_residual_norm_forward(const spconv_residual_norm_args *q, void *stream) {
    RnArgs a = {};
    bool vec = false, aligned = false;
    const int rc = rn_args(q, a, vec, aligned, false);
    if (rc != SPCONV_OK || q->num_rows == 0) return rc;
    SPCONV_REQUIRE(a.h && (a.norm2 == SPCONV_NORM_NONE || a.y), SPCONV_ERR_ARG, "null output pointer");
    return rn_by_type(q->dtype, [&](auto *t) {
        return rn_dispatch<std::remove_pointer_t<decltype(t)>>(a, vec, aligned, false, (cudaStream_t)stream);
    });
}

extern "C" int spconv_residual_norm_backward(const spconv_residual_norm_args *q, void *stream) {
    RnArgs a = {};
    bool vec = false, aligned = false;
    const int rc = rn_args(q, a, vec, aligned, true);
    if (rc != SPCONV_OK) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    spconv_channel_param ps[kRnParams] = {q->gate, q->weight, q->bias, q->next_weight, q->next_bias};
    if (q->num_rows == 0) {                  // sums over no rows
        for (const auto &p : ps)
            if (p.grad && cudaMemsetAsync(p.grad, 0, (size_t)(p.per_sample ? q->num_samples : 1) * q->channels *
                                                        (p.dtype == SPCONV_F32 ? 4 : 2), st) != cudaSuccess)
                return check_launch("residual_norm_backward: clear");
        return SPCONV_OK;
    }
    SPCONV_REQUIRE(a.dh || a.dy, SPCONV_ERR_ARG, "no output gradient given");
    SPCONV_REQUIRE(a.nslots == 0 ||
                       (a.partial && rn_aligned(a.partial) &&
                        q->workspace_bytes >= spconv_residual_norm_workspace_bytes(q->num_rows, q->channels, a.B)),
                   SPCONV_ERR_ARG, "workspace missing, misaligned or too small");
    SPCONV_REQUIRE(a.stats, SPCONV_ERR_ARG, "row_stats of the forward are needed");
    return rn_by_type(q->dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        int e = rn_dispatch<T>(a, vec, aligned, true, st);
        if (e != SPCONV_OK || a.nslots == 0) return e;
        RnGradArgs o = {};
        bool per_sample = false;
        for (int k = 0; k < kRnParams; ++k) {
            if (a.slot[k] < 0) continue;
            o.out[a.slot[k]] = ps[k].grad;
            o.out_f32[a.slot[k]] = a.p_f32[k];
            o.per_sample[a.slot[k]] = a.p_stride[k] != 0;
            per_sample |= a.p_stride[k] != 0;
        }
        const dim3 grid((a.C + 31) / 32, a.nslots, per_sample ? a.B : 1);
        if (launch_pdl(residual_norm_grad_kernel<T>, grid, dim3(32, 32), 0, st, a, o) != cudaSuccess)
            return check_launch("residual_norm_grad_kernel");
        return check_launch("residual_norm_grad_kernel");
    });
}
