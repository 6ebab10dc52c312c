// Attention on the CUDA cores, in exact fp32 products and sums: fp32 tensors, and 16-bit ones that the tensor-core kernels
// do not take. Forward, gradient of the queries and gradients of keys and values, each one sweep over tiles of the
// other side with everything between the inputs and the results in registers and shared memory:
//
//   s = q k scale;  p = exp2(s log2(e) - lse);  out = p v;   dp = grad v;  ds = p (dp - delta)
//   grad_query = scale ds k;  grad_key = scale ds^T q;  grad_value = p^T grad
//
// A block of 256 threads takes BM = 64 rows (32 of heads beyond 128 values) of one head and the opposite side's tiles of as many:
// products of [rows][head] tiles by 16 x 16 threads, 4 x 4 results each (rows 4 ty.., columns tx + 16 j), operands as
// float4 along the head from rows padded by four floats (no bank conflicts), so that 64 FMAs go with 8 loads of 16 bytes;
// products along the tile (p v and the like) take single columns tx + 16 j, which spans any head size in sixteens.
// Bound: the FMA pipe and its operands from shared memory; issue slots 57, 65 and 69 % in use (all 48 columns). 6,001 rows
// in 2 samples, 4 x 35 fp32: 0.62, 0.79 and 1.01 ms for the three sweeps, 17 to 20 TFLOP/s (0.69, 0.85 and 1.06 where products along the head took
// all 48 columns in place of 36; 4 x 64, where none is left out, 0.81, 1.03 and 1.34 against 0.80, 1.06 and 1.33).
#include <algorithm>

#include "activation.cuh"
#include "attention_common.cuh"

namespace spconv {

constexpr int kAsThreads = 256;

template <int DP>
struct AsShape {
    static constexpr int BM = DP > 128 ? 32 : 64;        // rows of a tile, both sides
    static constexpr int R = BM / 16;                    // rows, and columns, of a thread
    static constexpr int C = DP / 16;                    // head columns of a thread
    static constexpr int LD = DP + 4, LP = BM + 4;
    static constexpr int kTile = BM * LD, kScores = BM * LP;
    static constexpr int kPerSm = DP <= 64 ? 2 : 1;      // blocks, by shared memory
};

// Rows [row0, row0 + valid) of a head into a tile, zeros behind them and behind the head's end. Whether one that this thread has
// brought is not finite, if that is asked for.
template <typename T, int DP, bool ASK = false>
__device__ __forceinline__ bool as_load(float *dst, const AtTensor &t, int64_t row0, int valid, int head, int D) {
    using S = AsShape<DP>;
    const T *src = (const T *)t.p + row0 * t.row + head * t.head;
    bool lost = false;
    for (int i = threadIdx.x; i < S::BM * DP; i += kAsThreads) {
        const int r = i / DP, d = i - r * DP;
        const float x = r < valid && d < D ? dtype_traits<T>::to_f(src[r * t.row + d]) : 0.f;
        dst[r * S::LD + d] = x;
        if constexpr (ASK) lost |= !(fabsf(x) < INFINITY);
    }
    return lost;
}
// The tiles are there. Whether, in a causal call, one of the block's threads has brought a value that is not finite: where rows
// of the tile do not see all of its keys, 0 times it must not come into their sums. (Forward and gradients of 6,001 causal rows, 4 x 35
// fp32: 415, 500 and 617 us without this, 412, 492 and 655 with it.)
template <bool CAUSAL>
__device__ __forceinline__ bool as_loaded(bool lost) {
    if constexpr (CAUSAL) return __syncthreads_or(lost) != 0;
    __syncthreads();
    return false;
}

// Two products a slot (fma.rn.f32x2): the pipe's rate is the same, but the loads between them find slots.
__device__ __forceinline__ f32x2 as_pair(const float *p) { return *reinterpret_cast<const f32x2 *>(p); }
__device__ __forceinline__ float as_sum(f32x2 x) {
    const float2 f = unpack_f32x2(x);
    return f.x + f.y;
}

// acc[i][j] = a[4 ty + i][.] . b[tx + 16 j][.], over whole fours of the head's `size` values (zeros behind its end)
template <int DP>
__device__ __forceinline__ void as_dot(const float *a, const float *b, int size, float (&acc)[AsShape<DP>::R][AsShape<DP>::R]) {
    using S = AsShape<DP>;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float *pa = a + ty * S::R * S::LD, *pb = b + tx * S::LD;
    f32x2 sum[S::R][S::R];
#pragma unroll
    for (int i = 0; i < S::R; ++i)
#pragma unroll
        for (int j = 0; j < S::R; ++j) sum[i][j] = pack_f32x2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < size; d += 4) {
        float4 x[S::R], y[S::R];
#pragma unroll
        for (int i = 0; i < S::R; ++i) x[i] = *(const float4 *)(pa + i * S::LD + d);
#pragma unroll
        for (int j = 0; j < S::R; ++j) y[j] = *(const float4 *)(pb + j * 16 * S::LD + d);
#pragma unroll
        for (int i = 0; i < S::R; ++i)
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                sum[i][j] = fma2(as_pair(&x[i].x), as_pair(&y[j].x), sum[i][j]);
                sum[i][j] = fma2(as_pair(&x[i].z), as_pair(&y[j].z), sum[i][j]);
            }
    }
#pragma unroll
    for (int i = 0; i < S::R; ++i)
#pragma unroll
        for (int j = 0; j < S::R; ++j) acc[i][j] = as_sum(sum[i][j]);
}

// acc[i][j] += sum_k p[4 ty + i][k] b[k][tx + 16 j], k < BM, the even and the odd k apart; of `hidden` tiles k < seen[i] alone
template <int DP>
__device__ __forceinline__ void as_rows(const float *p, const float *b, f32x2 (&acc)[AsShape<DP>::R][AsShape<DP>::C], bool hidden,
                                        const int (&seen)[AsShape<DP>::R]) {
    using S = AsShape<DP>;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float *pp = p + ty * S::R * S::LP, *pb = b + tx;
    if (hidden) {
#pragma unroll 1
        for (int k = 0; k < S::BM; ++k)
#pragma unroll
            for (int i = 0; i < S::R; ++i) {
                if (k >= seen[i]) continue;
                const float x = pp[i * S::LP + k];
#pragma unroll
                for (int j = 0; j < S::C; ++j) acc[i][j] = fma2(pack_f32x2(x, 0.f), pack_f32x2(pb[k * S::LD + 16 * j], 0.f), acc[i][j]);
            }
        return;
    }
#pragma unroll 2
    for (int k = 0; k < S::BM; k += 4) {
        float4 x[S::R];
#pragma unroll
        for (int i = 0; i < S::R; ++i) x[i] = *(const float4 *)(pp + i * S::LP + k);
#pragma unroll
        for (int j = 0; j < S::C; ++j) {
            const float *q = pb + k * S::LD + 16 * j;
            const f32x2 y0 = pack_f32x2(q[0], q[S::LD]), y1 = pack_f32x2(q[2 * S::LD], q[3 * S::LD]);
#pragma unroll
            for (int i = 0; i < S::R; ++i) acc[i][j] = fma2(as_pair(&x[i].z), y1, fma2(as_pair(&x[i].x), y0, acc[i][j]));
        }
    }
}

// (acc[i][j]: rows 4 ty + 2 i and 4 ty + 2 i + 1) += sum_q p[q][4 ty + ..] b[q][tx + 16 j], q < BM; of `hidden` tiles those q alone that
// see the key, query number q0 + q seeing up to key number key0 + 4 ty + ..
template <int DP>
__device__ __forceinline__ void as_cols(const AtArgs &a, const float *p, const float *b, f32x2 (&acc)[AsShape<DP>::R / 2][AsShape<DP>::C],
                                        bool hidden, int q0, int key0, int n, int m) {
    using S = AsShape<DP>;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float *pp = p + ty * S::R, *pb = b + tx;
    if (hidden) {
#pragma unroll 1
        for (int q = 0; q < S::BM; ++q) {
            const int seen = at_seen(a, q0 + q, n, m) - key0 - ty * S::R;
#pragma unroll
            for (int i = 0; i < S::R / 2; ++i) {
                if (2 * i >= seen) continue;
                const float2 x = make_float2(pp[q * S::LP + 2 * i], 2 * i + 1 < seen ? pp[q * S::LP + 2 * i + 1] : 0.f);
#pragma unroll
                for (int j = 0; j < S::C; ++j) {
                    const float y = pb[q * S::LD + 16 * j];
                    acc[i][j] = fma2(pack_f32x2(x.x, x.y), pack_f32x2(y, 2 * i + 1 < seen ? y : 0.f), acc[i][j]);
                }
            }
        }
        return;
    }
#pragma unroll 4
    for (int q = 0; q < S::BM; ++q) {
        float x[S::R];
        if constexpr (S::R == 4) *(float4 *)x = *(const float4 *)(pp + q * S::LP);
        else *(float2 *)x = *(const float2 *)(pp + q * S::LP);
#pragma unroll
        for (int j = 0; j < S::C; ++j) {
            const float y = pb[q * S::LD + 16 * j];
            const f32x2 yy = pack_f32x2(y, y);
#pragma unroll
            for (int i = 0; i < S::R / 2; ++i) acc[i][j] = fma2(as_pair(x + 2 * i), yy, acc[i][j]);
        }
    }
}

template <int R, int C>
__device__ __forceinline__ void as_clear(f32x2 (&acc)[R][C]) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j) acc[i][j] = pack_f32x2(0.f, 0.f);
}

// This block's sample, found by its first warp.
__device__ __forceinline__ AtSample as_sample(const AtArgs &a, bool keys, int per_tile, AtSample *shared) {
    at_check_offsets(a);
    if (threadIdx.x < 32) {
        const AtSample s = at_find(a, keys, blockIdx.x, per_tile);
        if (threadIdx.x == 0) *shared = s;
    }
    __syncthreads();
    return *shared;
}

template <typename T, int DP, bool CAUSAL>
__global__ void __launch_bounds__(kAsThreads, AsShape<DP>::kPerSm)
attention_simt_kernel(const __grid_constant__ AtArgs a) {
    using S = AsShape<DP>;
    extern __shared__ __align__(16) float smem[];
    __shared__ AtSample shared;
    const AtSample s = as_sample(a, false, S::BM, &shared);
    const int row0 = s.q0 + s.tile * S::BM, rows = min(S::BM, s.q1 - row0);
    if (s.tile < 0 || rows <= 0) return;
    float *sq = smem, *sk = sq + S::kTile, *sv = sk + S::kTile, *sp = sv + S::kTile;
    const int h = blockIdx.y, kh = h / (a.H / a.K), n = s.q1 - s.q0, m = s.k1 - s.k0;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, i0 = s.tile * S::BM + ty * S::R;
    int first, last;
    at_split(a.splits, blockIdx.z, (at_seen(a, s.tile * S::BM + rows - 1, n, m) + S::BM - 1) / S::BM, first, last);
    as_load<T, DP>(sq, a.q, row0, rows, h, a.D);
    f32x2 acc[S::R][S::C];
    float top[S::R], sum[S::R] = {};
    as_clear(acc);
#pragma unroll
    for (int i = 0; i < S::R; ++i) top[i] = -INFINITY;
    for (int t = first; t < last; ++t) {
        const int key0 = t * S::BM, valid = min(S::BM, m - key0);
        __syncthreads();
        as_load<T, DP>(sk, a.k, s.k0 + key0, valid, kh, a.D);
        const bool lost = as_loaded<CAUSAL>(as_load<T, DP, CAUSAL>(sv, a.v, s.k0 + key0, valid, kh, a.D));
        float x[S::R][S::R];
        int sees[S::R];
        as_dot<DP>(sq, sk, a.D, x);
#pragma unroll
        for (int i = 0; i < S::R; ++i) {
            const int seen = sees[i] = at_seen(a, i0 + i, n, m) - key0;
            float big = top[i];
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                x[i][j] = tx + 16 * j < seen ? x[i][j] * a.c : -INFINITY;
                big = fmaxf(big, x[i][j]);
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            const float base = big == -INFINITY ? 0.f : big;
            const float down = exp2f(top[i] - base);           // top -inf: 0
            top[i] = big;
            float add = 0.f;
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                const float p = exp2f(x[i][j] - base);
                add += p;
                sp[(ty * S::R + i) * S::LP + tx + 16 * j] = p;
            }
            sum[i] = sum[i] * down + add;
#pragma unroll
            for (int j = 0; j < S::C; ++j) acc[i][j] = mul2(acc[i][j], pack_f32x2(down, down));
        }
        __syncwarp();                                          // a row's p are of its own 16 lanes
        as_rows<DP>(sp, sv, acc, lost, sees);
    }
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
#pragma unroll
        for (int o = 8; o; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
        const int r = ty * S::R + i;
        if (r >= rows) continue;
        const int64_t at = (int64_t)(row0 + r) * a.H + h;
        const bool none = at_seen(a, i0 + i, n, m) <= first * S::BM;        // (of this split's keys)
        if (a.splits > 1) {
            const int64_t all = (int64_t)a.M * a.H;
            if (tx == 0) a.part_ml[blockIdx.z * all + at] = make_float2(top[i], none ? -1.f : sum[i]);
#pragma unroll
            for (int j = 0; j < S::C; ++j)
                if (tx + 16 * j < a.D) a.partial[(blockIdx.z * all + at) * a.D + tx + 16 * j] = as_sum(acc[i][j]);
            continue;
        }
        if (tx == 0 && a.lse) a.lse[at] = none ? INFINITY : top[i] + log2f(sum[i]);
        const float inv = 1.f / sum[i];
#pragma unroll
        for (int j = 0; j < S::C; ++j)
            if (tx + 16 * j < a.D) at_put<T>(a, at * a.D + tx + 16 * j, none ? 0.f : as_sum(acc[i][j]) * inv);
    }
}

// p and ds of a tile of queries (rows) and keys (columns) from tiles of q, grad, k and v. The probability of a row that
// sees a single key is 1 whatever its score: ds is zero, not the difference of two roundings of grad . v.
template <int DP>
__device__ __forceinline__ void as_grads(const AtArgs &a, const float *sq, const float *sg, const float *sk, const float *sv,
                                         float *sp, float *sd, const float (&lse)[AsShape<DP>::R],
                                         const float (&delta)[AsShape<DP>::R], const int (&seen)[AsShape<DP>::R],
                                         const bool (&single)[AsShape<DP>::R]) {
    using S = AsShape<DP>;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float x[S::R][S::R], y[S::R][S::R];
    as_dot<DP>(sq, sk, a.D, x);
    as_dot<DP>(sg, sv, a.D, y);
#pragma unroll
    for (int i = 0; i < S::R; ++i)
#pragma unroll
        for (int j = 0; j < S::R; ++j) {
            const bool in = tx + 16 * j < seen[i];
            const float p = in ? exp2f(fmaf(x[i][j], a.c, -lse[i])) : 0.f;
            const int at = (ty * S::R + i) * S::LP + tx + 16 * j;
            if (sp) sp[at] = p;
            sd[at] = in && !single[i] ? p * (y[i][j] - delta[i]) : 0.f;
        }
}

template <typename T, int DP, bool CAUSAL>
__global__ void __launch_bounds__(kAsThreads, AsShape<DP>::kPerSm)
attention_simt_grad_query_kernel(const __grid_constant__ AtArgs a) {
    using S = AsShape<DP>;
    extern __shared__ __align__(16) float smem[];
    __shared__ AtSample shared;
    const AtSample s = as_sample(a, false, S::BM, &shared);
    const int row0 = s.q0 + s.tile * S::BM, rows = min(S::BM, s.q1 - row0);
    if (s.tile < 0 || rows <= 0) return;
    float *sq = smem, *sg = sq + S::kTile, *sk = sg + S::kTile, *sv = sk + S::kTile, *sd = sv + S::kTile;
    const int h = blockIdx.y, kh = h / (a.H / a.K), n = s.q1 - s.q0, m = s.k1 - s.k0;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, i0 = s.tile * S::BM + ty * S::R;
    int first, last;
    at_split(a.splits, blockIdx.z, (at_seen(a, s.tile * S::BM + rows - 1, n, m) + S::BM - 1) / S::BM, first, last);
    as_load<T, DP>(sq, a.q, row0, rows, h, a.D);
    as_load<T, DP>(sg, a.grad, row0, rows, h, a.D);
    f32x2 acc[S::R][S::C];
    float lse[S::R], delta[S::R];
    as_clear(acc);
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        const int r = ty * S::R + i;
        const int64_t at = (int64_t)(row0 + r) * a.H + h;
        lse[i] = r < rows ? a.lse[at] : INFINITY;
        delta[i] = r < rows ? a.delta[at] : 0.f;
    }
    for (int t = first; t < last; ++t) {
        const int key0 = t * S::BM, valid = min(S::BM, m - key0);
        __syncthreads();
        as_load<T, DP>(sv, a.v, s.k0 + key0, valid, kh, a.D);
        const bool lost = as_loaded<CAUSAL>(as_load<T, DP, CAUSAL>(sk, a.k, s.k0 + key0, valid, kh, a.D));
        int seen[S::R];
        bool single[S::R];
#pragma unroll
        for (int i = 0; i < S::R; ++i) {
            const int all = at_seen(a, i0 + i, n, m);
            seen[i] = all - key0;
            single[i] = all == 1;
        }
        as_grads<DP>(a, sq, sg, sk, sv, nullptr, sd, lse, delta, seen, single);
        __syncwarp();
        as_rows<DP>(sd, sk, acc, lost, seen);
    }
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        const int r = ty * S::R + i;
        if (r >= rows) continue;
        const int64_t at = (int64_t)(row0 + r) * a.H + h;
#pragma unroll
        for (int j = 0; j < S::C; ++j) {
            if (tx + 16 * j >= a.D) continue;
            const float g = as_sum(acc[i][j]) * a.scale;
            if (a.splits > 1) a.partial[(blockIdx.z * (int64_t)a.M * a.H + at) * a.D + tx + 16 * j] = g;
            else ((T *)a.gq)[at * a.D + tx + 16 * j] = dtype_traits<T>::from_f(g);
        }
    }
}

template <typename T, int DP, bool CAUSAL>
__global__ void __launch_bounds__(kAsThreads, AsShape<DP>::kPerSm)
attention_simt_grad_key_kernel(const __grid_constant__ AtArgs a) {
    using S = AsShape<DP>;
    extern __shared__ __align__(16) float smem[];
    __shared__ AtSample shared;
    const AtSample s = as_sample(a, true, S::BM, &shared);
    const int key0 = s.tile * S::BM, row0 = s.k0 + key0, rows = min(S::BM, s.k1 - row0);
    if (s.tile < 0 || rows <= 0) return;
    float *sk = smem, *sv = sk + S::kTile, *sq = sv + S::kTile, *sg = sq + S::kTile, *sp = sg + S::kTile, *sd = sp + S::kScores;
    const int kh = blockIdx.y, G = a.H / a.K, n = s.q1 - s.q0, m = s.k1 - s.k0;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    // tiles of queries that see a key of this tile, of each of the group's heads
    const int from = a.causal ? (int)max((int64_t)0, (int64_t)key0 - m + n) / S::BM : 0;
    const int tiles = max(0, (n + S::BM - 1) / S::BM - from);
    int first, last;
    at_split(a.splits, blockIdx.z, tiles * G, first, last);
    as_load<T, DP>(sk, a.k, row0, rows, kh, a.D);
    as_load<T, DP>(sv, a.v, row0, rows, kh, a.D);
    f32x2 gk[S::R / 2][S::C], gv[S::R / 2][S::C];
    as_clear(gk);
    as_clear(gv);
    for (int it = first; it < last; ++it) {
        const int g = it / tiles, t = from + it - g * tiles, h = kh * G + g;
        const int i0 = t * S::BM, valid = min(S::BM, n - i0);
        __syncthreads();
        bool lost = as_load<T, DP, CAUSAL>(sq, a.q, s.q0 + i0, valid, h, a.D);
        lost |= as_load<T, DP, CAUSAL>(sg, a.grad, s.q0 + i0, valid, h, a.D);
        float lse[S::R], delta[S::R];
        int seen[S::R];
        bool single[S::R];
#pragma unroll
        for (int i = 0; i < S::R; ++i) {
            const int r = ty * S::R + i;
            const int64_t at = (int64_t)(s.q0 + i0 + r) * a.H + h;
            lse[i] = r < valid ? a.lse[at] : INFINITY;
            delta[i] = r < valid ? a.delta[at] : 0.f;
            const int all = at_seen(a, i0 + r, n, m);
            seen[i] = r < valid ? min(rows, all - key0) : 0;
            single[i] = all == 1;
        }
        lost = as_loaded<CAUSAL>(lost);
        as_grads<DP>(a, sq, sg, sk, sv, sp, sd, lse, delta, seen, single);
        __syncthreads();
        as_cols<DP>(a, sp, sg, gv, lost, i0, key0, n, m);
        as_cols<DP>(a, sd, sq, gk, lost, i0, key0, n, m);
    }
    auto of = [](f32x2 pair, int i) {
        const float2 f = unpack_f32x2(pair);
        return i & 1 ? f.y : f.x;
    };
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        const int r = ty * S::R + i;
        if (r >= rows) continue;
        const int64_t all = (int64_t)a.N * a.K, at = (int64_t)(row0 + r) * a.K + kh;
#pragma unroll
        for (int j = 0; j < S::C; ++j) {
            const int d = tx + 16 * j;
            if (d >= a.D) continue;
            if (a.splits > 1) {
                a.partial[((2 * blockIdx.z) * all + at) * a.D + d] = of(gk[i / 2][j], i) * a.scale;
                a.partial[((2 * blockIdx.z + 1) * all + at) * a.D + d] = of(gv[i / 2][j], i);
            } else {
                if (a.gk) ((T *)a.gk)[at * a.D + d] = dtype_traits<T>::from_f(of(gk[i / 2][j], i) * a.scale);
                if (a.gv) ((T *)a.gv)[at * a.D + d] = dtype_traits<T>::from_f(of(gv[i / 2][j], i));
            }
        }
    }
}

int at_simt_rows(int D) { return D > 128 ? 32 : 64; }

template <typename T, int DP, bool CAUSAL>
static int as_run(const AtArgs &a, int what) {
    using S = AsShape<DP>;
    static std::atomic<uint64_t> done[3];
    auto kern = what == 0 ? attention_simt_kernel<T, DP, CAUSAL>
                          : what == 1 ? attention_simt_grad_query_kernel<T, DP, CAUSAL> : attention_simt_grad_key_kernel<T, DP, CAUSAL>;
    const int smem = 4 * (what == 0 ? 3 * S::kTile + S::kScores : what == 1 ? 4 * S::kTile + S::kScores : 4 * S::kTile + 2 * S::kScores);
    if (allow_smem(kern, smem, done[what]) != cudaSuccess) return check_launch("attention: shared memory");
    const int64_t tiles = at_tiles(what == 2 ? a.N : a.M, a.B, S::BM);
    kern<<<dim3((unsigned)tiles, what == 2 ? a.K : a.H, a.splits), kAsThreads, smem, a.stream>>>(a);
    return check_launch("attention_simt_kernel");
}

template <typename T, bool CAUSAL>
static int as_size(const AtArgs &a, int what) {
    if (a.D <= 32) return as_run<T, 32, CAUSAL>(a, what);
    if (a.D <= 48) return as_run<T, 48, CAUSAL>(a, what);
    if (a.D <= 64) return as_run<T, 64, CAUSAL>(a, what);
    if (a.D <= 96) return as_run<T, 96, CAUSAL>(a, what);
    if (a.D <= 128) return as_run<T, 128, CAUSAL>(a, what);
    return as_run<T, 256, CAUSAL>(a, what);
}

template <bool CAUSAL>
static int as_type(const AtArgs &a, int what) {
    if (a.dtype == SPCONV_F32) return as_size<float, CAUSAL>(a, what);
    if (a.dtype == SPCONV_F16) return as_size<__half, CAUSAL>(a, what);
    return as_size<__nv_bfloat16, CAUSAL>(a, what);
}

static int as_launch(const AtArgs &a, int what) { return a.causal ? as_type<true>(a, what) : as_type<false>(a, what); }
int launch_at_simt_forward(const AtArgs &a) { return as_launch(a, 0); }
int launch_at_simt_grad_query(const AtArgs &a) { return as_launch(a, 1); }
int launch_at_simt_grad_key(const AtArgs &a) { return as_launch(a, 2); }

}  // namespace spconv
