// Attention's entry points: checks, the choice of kernels and splits, and the small kernels around the products: copies
// of rows that TMA cannot read, delta = grad . out, and the joining of splits.
//
// Splits. A sample whose rows make few tiles (pooling queries, single tokens; for the keys' gradients, few
// conditioning tokens) leaves most SMs idle, so its keys (or queries) are cut into `splits` ranges, each
// with fp32 results of its own, joined in order by a second kernel: the same bits every run.
#include <algorithm>

#include "attention_common.cuh"

namespace spconv {

constexpr int kAtThreads = 256;

// Rows [rows, heads, D] with any strides into rows of `to` values, a multiple of 8, zeros behind the head's end.
template <typename T>
__global__ void __launch_bounds__(kAtThreads)
attention_pack_kernel(AtTensor t, T *out, int64_t rows, int heads, int D, int to) {
    const int64_t total = rows * heads * to;
    for (int64_t i = (int64_t)blockIdx.x * kAtThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kAtThreads) {
        const int64_t rh = i / to, r = rh / heads;
        const int d = (int)(i - rh * to), h = (int)(rh - r * heads);
        out[i] = d < D ? ((const T *)t.p)[r * t.row + h * t.head + d] : dtype_traits<T>::from_f(0.f);
    }
}

// Eight lanes a row and head, of which they have x . y (and x . (y + rest)) and x . x. Bound: HBM.
template <typename T, bool WIDE>
__device__ __forceinline__ void at_dots(const T *x, const T *y, const T *rest, int D, bool in, float &xy, float &xx) {
    const int lane = threadIdx.x & 7;
    xy = xx = 0.f;
    if (in) {
        constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1;
        for (int d = lane * V; d < D; d += 8 * V) {
            T p[V], q[V], r[V];
            if constexpr (WIDE) {
                *(uint4 *)p = *(const uint4 *)(x + d);
                if (y) *(uint4 *)q = *(const uint4 *)(y + d);
                if (rest) *(uint4 *)r = *(const uint4 *)(rest + d);
            } else {
                p[0] = x[d];
                if (y) q[0] = y[d];
                if (rest) r[0] = rest[d];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float f = dtype_traits<T>::to_f(p[i]);
                xx = fmaf(f, f, xx);
                if (y) xy = fmaf(f, dtype_traits<T>::to_f(q[i]), xy);
                if (rest) xy = fmaf(f, dtype_traits<T>::to_f(r[i]), xy);
            }
        }
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) {
        xy += __shfl_xor_sync(0xffffffffu, xy, o);
        xx += __shfl_xor_sync(0xffffffffu, xx, o);
    }
}

// A row's square as the largest are looked for: none where it is not finite, since the row's products are lost as they are, and others
// need their digits all the same.
__device__ __forceinline__ float at_counted(float square) { return square < INFINITY ? square : 0.f; }

// delta[row, head] = grad . (out + what its rounding left out, where that is kept), and grad's square.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kAtThreads)
attention_delta_kernel(const __grid_constant__ AtArgs a) {
    const int64_t rh = ((int64_t)blockIdx.x * kAtThreads + threadIdx.x) >> 3, r = rh / a.H;
    const bool in = rh < (int64_t)a.M * a.H;
    float dot, square;
    at_dots<T, WIDE>((const T *)a.grad.p + r * a.grad.row + (rh - r * a.H) * a.grad.head, (const T *)a.out_in + rh * a.D,
                     a.rest ? (const T *)a.rest + rh * a.D : nullptr, a.D, in, dot, square);
    if (!in || (threadIdx.x & 7) != 0) return;
    a.delta[rh] = dot;
    if (a.peaks) a.squares[rh] = at_counted(square);
}

// Each sample's largest square into peaks[sample * 2], which start at 0: the same whatever the order. A converged warp's, whose rows
// and heads ascend; while they are one sample's that is a comparison.
struct AtPeaks {
    const int32_t *offsets;
    int B, rows, heads;
    float *peaks;
    int b;                               // the sample, and the row and head behind it
    int64_t end;
    uint32_t most;

    __device__ __forceinline__ void begin(int row) {
        b = at_sample_of(offsets, B, rows, row);
        end = b + 1 == B ? INT64_MAX : (int64_t)at_offset(offsets, b + 1, rows) * heads;
        most = 0;
    }
    __device__ __forceinline__ void put(int sample, uint32_t value) const {
        uint32_t *peak = reinterpret_cast<uint32_t *>(peaks + 2 * (int64_t)sample);
        if (value > *(volatile uint32_t *)peak) atomicMax(peak, value);
    }
    __device__ __forceinline__ void flush() const {
        const uint32_t top = __reduce_max_sync(0xffffffffu, most);
        if ((threadIdx.x & 31) == 0) put(b, top);
        __syncwarp();
    }
    // the warp's rows and heads go up to `last`; the lane's own has a square that counts (or 0)
    __device__ __forceinline__ void add(int64_t last, int64_t own, float square) {
        const uint32_t value = __float_as_uint(square);
        if (last < end) {
            most = max(most, value);
            return;
        }
        flush();
        const int row = (int)min(own / heads, (int64_t)rows - 1);
        if (value > 0) {                     // on from the sample before, in steps that double
            int at = b, step = 1;
            for (; at + step < B && at_offset(offsets, at + step, rows) <= row; step *= 2) at += step;
            for (step >>= 1; step > 0; step >>= 1)
                if (at + step < B && at_offset(offsets, at + step, rows) <= row) at += step;
            put(at, value);
        }
        __syncwarp();
        begin(__shfl_sync(0xffffffffu, row, 31));
    }
};

// grad's largest squares of rows that see a key, from those that the pass before wrote (1/32 of the bytes of 16-bit rows of 64; looking
// for the samples in that pass took it from 38 to 57 us over 1,301 windows): a warp takes `share` of them, 128 a step.
__device__ __forceinline__ void at_grad_peaks(const AtArgs &a, int64_t share) {
    const int lane = threadIdx.x & 31;
    const int64_t all = (int64_t)a.M * a.H, first = ((int64_t)blockIdx.x * (kAtThreads / 32) + (threadIdx.x >> 5)) * share;
    if (first >= all) return;
    AtPeaks peaks{a.offsets, a.B, a.M, a.H, a.peaks};
    peaks.begin((int)(first / a.H));
    for (int64_t at = first; at < min(first + share, all); at += 128) {
        float square[4], lse[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t rh = at + 32 * k + lane;
            square[k] = rh < all ? __ldg(a.squares + rh) : 0.f;
            lse[k] = rh < all ? __ldg(a.lse + rh) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) peaks.add(at + 32 * k + 31, at + 32 * k + lane, lse[k] == INFINITY ? 0.f : square[k]);
    }
    peaks.flush();
}

// v's: a block takes `parts` times 128 rows and heads, a warp sixteen of them, eight lanes four at a time, of whole 16 bytes.
__device__ __forceinline__ void at_value_peaks(const AtArgs &a, int64_t parts) {
    constexpr int B = 4;
    const int lane = threadIdx.x & 7, group = (threadIdx.x & 31) >> 3;
    constexpr int kBlock = kAtThreads / 32 * 4 * B;
    const int64_t all = (int64_t)a.N * a.K, begin = blockIdx.x * parts * kBlock, first = begin + (threadIdx.x >> 5) * 4 * B;
    if (first >= all) return;
    AtPeaks peaks{a.key_offsets, a.B, a.N, a.K, a.peaks + 1};
    peaks.begin((int)(first / a.K));
    for (int64_t part = first; part < min(begin + parts * kBlock, all); part += kBlock) {
        float square[B] = {};
        const int64_t row = part / a.K;
        const int head = (int)(part - row * a.K) + group;
        for (int d = lane * 8; d < a.D; d += 64) {
            uint4 x[B];
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const unsigned past = (unsigned)(head + 4 * k) / (unsigned)a.K;          // (32 bits are enough)
                x[k] = make_uint4(0, 0, 0, 0);
                if (part + 4 * k + group < all)
                    x[k] = __ldg((const uint4 *)((const __half *)a.v.p + (row + past) * a.v.row + (head + 4 * k - (int64_t)past * a.K) * a.v.head + d));
            }
#pragma unroll
            for (int k = 0; k < B; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = __half22float2(reinterpret_cast<const __half2 *>(&x[k])[i]);
                    square[k] = fmaf(f.x, f.x, fmaf(f.y, f.y, square[k]));
                }
        }
        __syncwarp();                        // (lanes past the head's end have read less)
#pragma unroll
        for (int k = 0; k < B; ++k) {
#pragma unroll
            for (int o = 4; o; o >>= 1) square[k] += __shfl_xor_sync(0xffffffffu, square[k], o);
            peaks.add(part + 4 * k + 3, part + 4 * k + group, at_counted(square[k]));
        }
    }
    peaks.flush();
}

// Both in one launch, in each other's latency (1,301 windows, 4 x 32: 34 us, 42 one after the other; one largest for the whole call, which
// one sample's rows would set for all others, 23).
__global__ void __launch_bounds__(kAtThreads)
attention_peaks_kernel(const __grid_constant__ AtArgs a, const int64_t parts, const int64_t share) {
    if (blockIdx.y == 0) at_value_peaks(a, parts);
    else at_grad_peaks(a, share);
}

// A row's splits: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, over those that saw a key (others have a sum of -1; scores
// that are all -inf have one of 0, and make the row NaN where no split has another). `share` warps take a row's splits in turn and add up in
// order: all eight of a block where rows are few, one where they are many. Forward by eight warps a row and by one, in us: 8 rows and heads
// over 200,000 keys 55 and 174, 512 over 20,000 35 and 55, 2,048 over 8,000 41 and 41, 4,096 over 4,096 43 and 35, 8,192 61 and 47.
template <typename T>
__global__ void __launch_bounds__(kAtThreads)
attention_join_kernel(const __grid_constant__ AtArgs a, const int share) {
    __shared__ float parts[kAtThreads / 32][256], sums[kAtThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp % share;
    const int64_t all = (int64_t)a.M * a.H, rh = (int64_t)blockIdx.x * (kAtThreads / 32 / share) + warp / share;
    const bool in = rh < all;
    float m = -INFINITY, acc[8] = {}, sum = 0.f;
    bool nan = false, some = false;
    if (in) {
        for (int s = lane; s < a.splits; s += 32) {
            const float2 ml = a.part_ml[s * all + rh];
            m = fmaxf(m, ml.x);
            nan |= isnan(ml.x);
            some |= !(ml.y < 0.f);                              // else it saw no key, and nothing may be written there
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (__any_sync(0xffffffffu, nan)) m = NAN;
        some = __any_sync(0xffffffffu, some);
#pragma unroll 4
        for (int s = w; s < a.splits; s += share) {
            const float2 ml = a.part_ml[s * all + rh];
            const bool there = !(ml.y < 0.f);
            const float weight = there ? exp2f(ml.x - m) : 0.f;
            const float *p = a.partial + (s * all + rh) * a.D;
            sum = fmaf(weight, ml.y, sum);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (lane + 32 * j < a.D) acc[j] = fmaf(weight, there ? p[lane + 32 * j] : 0.f, acc[j]);
        }
    }
    if (share > 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) parts[warp][lane + 32 * j] = acc[j];
        if (lane == 0) sums[warp] = sum;
        __syncthreads();
        if (w != 0) return;
        for (int k = 1; k < share; ++k) {
            sum += sums[warp + k];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += parts[warp + k][lane + 32 * j];
        }
    }
    if (!in) return;
    const float inv = some ? 1.f / sum : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (lane + 32 * j < a.D) at_put<T>(a, rh * a.D + lane + 32 * j, acc[j] * inv);
    if (lane == 0 && a.lse) a.lse[rh] = some ? m + log2f(sum) : INFINITY;
}

// out[i] = sum of the splits' partial[s * stride + i], in order.
template <typename T>
__global__ void __launch_bounds__(kAtThreads)
attention_sum_kernel(const float *partial, int64_t stride, int splits, T *out, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * kAtThreads + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < splits; ++k) s += partial[k * stride + i];
    out[i] = dtype_traits<T>::from_f(s);
}

static unsigned at_blocks(int64_t threads) { return (unsigned)((threads + kAtThreads - 1) / kAtThreads); }

template <typename F>
static int at_by_type(int dtype, F f) {
    if (dtype == SPCONV_F32) return f((float *)nullptr);
    if (dtype == SPCONV_F16) return f((__half *)nullptr);
    return f((__nv_bfloat16 *)nullptr);
}

// Whether TMA can read the tensor as it is: 16-byte strides (none of zero) and address, whole 16-byte heads.
static bool at_tma(const AtTensor &t, int64_t rows, int heads, int D) {
    return D % 8 == 0 && ((uintptr_t)t.p & 15) == 0 && (rows == 1 || (t.row % 8 == 0 && t.row > 0 && t.row < (int64_t)1 << 38)) &&
           (heads == 1 || (t.head % 8 == 0 && t.head > 0 && t.head < (int64_t)1 << 38));
}

// Where things lie in the workspace, and how the work is cut.
struct AtPlan {
    bool tc;
    bool pair;                           // forward: two tiles a CTA
    int splits[3];                       // forward (or queries' gradients), and keys' gradients
    bool pack[4];                        // q, k, v, grad
    int64_t pack_at[4], delta_at, peaks_at, squares_at, ml_at, partial_at, bytes;
};

// Splits of `tiles` steps each of `ctas` CTAs, of which `slots` run at a time: whole waves, none of fewer than `least` steps. A CTA's
// start and end count as two steps, and the joining, in the kernels' own time, as six. What that chooses against the best of every count
// up to 256, in us: one query of 8 heads over 10,000 keys 26.6 and 20.4 (64 splits), over 100,000 41.0 and 41.0, eight over 1.0 M 77.8
// and 77.8; 512 tokens x 16 heads 18.4 and 18.4 (one; two 26.6), 2,048 x 8 47.1 and 45.1, 4,096 x 8 92 and 92 (gradients 82 and 82,
// 100 and 98); keys' gradients of 257 tokens, 10,534 queries 55.3 and 55.3 (one 185), 16 such samples 436 and 436 (one 510); fp32,
// 2,000 x 4, 213 and 211, keys' gradients 342 and 315.
static int at_cut(int64_t ctas, int64_t slots, int64_t tiles, int least) {
    if (ctas == 0 || ctas >= 4 * slots) return 1;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>({tiles / least, 4 * slots / ctas, 256}));
    int64_t best = 1, best_cost = INT64_MAX;
    for (int64_t s = 1; s <= most; ++s) {
        const int64_t cost = ((ctas * s + slots - 1) / slots) * ((tiles + s - 1) / s + 2) + (s > 1 ? 6 : 0);
        if (cost < best_cost) {
            best_cost = cost;
            best = s;
        }
    }
    return (int)best;
}

static AtPlan at_plan(const spconv_attention_args *q, bool backward) {
    AtPlan p = {};
    const int64_t M = q->num_queries, N = q->num_keys, B = q->num_samples;
    p.tc = q->kernel != SPCONV_KERNEL_SIMT && q->dtype != SPCONV_F32 && q->head_size <= 128 && M > 0 && N > 0;
    const int G = q->heads / q->key_heads;
    int P = 1;
    while (P < 128 && G % (2 * P) == 0) P *= 2;
    const int64_t mean_q = (M + B - 1) / B, mean_k = (N + B - 1) / B;
    auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    if (p.tc) {
        const int64_t rows = mean_q * P, heads = q->heads / P;
        // One tile a CTA and two, 4 heads of 128, samples of n rows and keys, in us: 64 of 320 47 and 59, 16 of 512 24.6 and 24.6, 64 of
        // 512 78 and 74, 16 of 768 53 and 47, 16 of 2,048 221 and 166. (Two are faster with fewer of them than SMs as well, from 768 keys
        // on: one sample of 1,024 33 and 27. They are not taken there yet.)
        p.pair = !backward && q->head_size > 64 && rows > 192 && mean_k > 512 && B * up(rows, 256) * heads >= 148;
        // CTAs that run at a time, and what each has to have for itself: 512 keys (a split's rows are written and read once more)
        const int64_t per_sm = q->head_size > 64 ? 1 : 2;
        p.splits[0] = p.pair ? at_cut(B * up(rows, 256) * heads, 148, up(mean_k, 128), 4)
                             : at_cut(B * up(rows, 128) * heads, 148 * (backward ? per_sm : 2 * per_sm), up(mean_k, 128), 4);
        p.splits[1] = at_cut(B * up(mean_k, 128) * q->key_heads, 148 * per_sm, up(rows, 128) * (G / P), 4);
    } else {
        const int64_t R = at_simt_rows(q->head_size);
        p.splits[0] = at_cut(B * up(mean_q, R) * q->heads, 296, up(mean_k, R), 4);
        p.splits[1] = at_cut(B * up(mean_k, R) * q->key_heads, 296, up(mean_q, R) * G, 4);
    }
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const AtTensor t[4] = {{q->query, q->query_row, q->query_head}, {q->key, q->key_row, q->key_head},
                           {q->value, q->value_row, q->value_head}, {q->grad_out, q->grad_row, q->grad_head}};
    for (int i = 0; i < (backward ? 4 : 3); ++i) {
        const bool keys = i == 1 || i == 2;
        p.pack[i] = p.tc && !at_tma(t[i], keys ? N : M, keys ? q->key_heads : q->heads, q->head_size);
        if (p.pack[i]) p.pack_at[i] = take((keys ? N * q->key_heads : M * q->heads) * (int64_t)((q->head_size + 7) / 8 * 16));
    }
    const int64_t rows = M * q->heads, krows = N * q->key_heads;
    if (backward) {
        p.delta_at = take(rows * 4);
        const bool lift = p.tc && q->dtype == SPCONV_F16;
        p.peaks_at = take(lift ? B * 8 : 0);
        p.squares_at = take(lift ? rows * 4 : 0);
        p.partial_at = take(std::max(p.splits[0] > 1 ? p.splits[0] * rows * q->head_size * 4 : 0,
                                     p.splits[1] > 1 ? 2 * p.splits[1] * krows * q->head_size * 4 : 0));
    } else if (p.splits[0] > 1) {
        p.ml_at = take(p.splits[0] * rows * 8);
        p.partial_at = take(p.splits[0] * rows * q->head_size * 4);
    }
    p.bytes = at;
    return p;
}

// A score's factor in powers of two.
static float at_exponent(float scale) { return (float)((double)scale * 1.4426950408889634); }

static int at_check(const spconv_attention_args *q, bool backward) {
    SPCONV_REQUIRE(q != nullptr, SPCONV_ERR_ARG, "null pointer argument");
    SPCONV_REQUIRE(q->dtype == SPCONV_F32 || q->dtype == SPCONV_F16 || q->dtype == SPCONV_BF16, SPCONV_ERR_ARG,
                   "unsupported dtype code %d", q->dtype);
    SPCONV_REQUIRE(q->kernel >= SPCONV_KERNEL_AUTO && q->kernel <= SPCONV_KERNEL_TCGEN05, SPCONV_ERR_ARG,
                   "unknown kernel choice %d", q->kernel);
    constexpr int64_t most = ((int64_t)1 << 31) - 1024;              // a tile's last row, past the tensor's end, fits 32 bits too
    SPCONV_REQUIRE(q->num_queries >= 0 && q->num_queries <= most && q->num_keys >= 0 && q->num_keys <= most, SPCONV_ERR_ARG,
                   "row counts must be in [0, 2^31 - 1024]");
    SPCONV_REQUIRE(q->num_samples >= 1 && q->num_samples < 1 << 24, SPCONV_ERR_ARG, "num_samples must be in [1, 2^24)");
    SPCONV_REQUIRE(q->key_heads >= 1 && q->heads >= q->key_heads && q->heads <= 65535 && q->heads % q->key_heads == 0, SPCONV_ERR_ARG,
                   "heads must be a multiple of key_heads, at most 65535");
    SPCONV_REQUIRE(q->head_size >= 1 && q->head_size <= SPCONV_ATTENTION_MAX_SIZE, SPCONV_ERR_ARG, "head size must be in [1, %d]",
                   SPCONV_ATTENTION_MAX_SIZE);
    SPCONV_REQUIRE(q->scale > 0.f && at_exponent(q->scale) < INFINITY, SPCONV_ERR_ARG, "scale must be positive and finite, its 1.44-fold too");
    SPCONV_REQUIRE((q->offsets && q->key_offsets) || q->num_samples == 1, SPCONV_ERR_ARG, "several samples need the row offsets of both sides");
    SPCONV_REQUIRE(q->kernel != SPCONV_KERNEL_TCGEN05 || (q->dtype != SPCONV_F32 && q->head_size <= 128), SPCONV_ERR_UNSUPPORTED,
                   "the tensor-core kernels take fp16 and bf16 heads of at most 128 values");
    SPCONV_REQUIRE((q->num_queries == 0 || (q->query && q->out)) && (q->num_keys == 0 || (q->key && q->value)), SPCONV_ERR_ARG,
                   "null pointer argument");
    if (backward)
        SPCONV_REQUIRE((q->num_queries == 0 || (q->grad_out && q->row_stats)), SPCONV_ERR_ARG, "null pointer argument");
    const int64_t need = at_plan(q, backward).bytes;
    SPCONV_REQUIRE(need == 0 || (q->workspace && ((uintptr_t)q->workspace & 255) == 0 && q->workspace_bytes >= need), SPCONV_ERR_ARG,
                   "workspace missing, misaligned or too small");
    return SPCONV_OK;
}

static int at_prepare(const spconv_attention_args *q, const AtPlan &p, bool backward, cudaStream_t st, AtArgs &a) {
    a = {};
    a.q = {q->query, q->query_row, q->query_head};
    a.k = {q->key, q->key_row, q->key_head};
    a.v = {q->value, q->value_row, q->value_head};
    a.grad = {q->grad_out, q->grad_row, q->grad_head};
    a.out = q->out;
    a.out_in = q->out;
    a.rest = q->dtype == SPCONV_F32 ? nullptr : q->out_rest;
    a.lse = q->row_stats;
    a.gq = q->grad_query;
    a.gk = q->grad_key;
    a.gv = q->grad_value;
    a.offsets = q->offsets;
    a.key_offsets = q->key_offsets;
    a.B = q->num_samples;
    a.M = (int)q->num_queries;
    a.N = (int)q->num_keys;
    a.H = q->heads;
    a.K = q->key_heads;
    a.D = q->head_size;
    a.causal = q->causal != 0;
    a.scale = q->scale;
    a.c = at_exponent(q->scale);
    a.status = q->status;
    a.wait_ns = wait_limit_ns();
    a.dtype = q->dtype;
    a.stream = st;
    uint8_t *ws = (uint8_t *)q->workspace;
    a.delta = (float *)(ws + p.delta_at);
    a.peaks = backward && p.tc && q->dtype == SPCONV_F16 ? (float *)(ws + p.peaks_at) : nullptr;
    a.squares = (float *)(ws + p.squares_at);
    a.part_ml = (float2 *)(ws + p.ml_at);
    a.partial = (float *)(ws + p.partial_at);
    AtTensor *t[4] = {&a.q, &a.k, &a.v, &a.grad};
    for (int i = 0; i < (backward ? 4 : 3); ++i) {
        if (!p.pack[i]) continue;
        const bool keys = i == 1 || i == 2;
        const int64_t rows = keys ? a.N : a.M;
        const int heads = keys ? a.K : a.H, to = (a.D + 7) / 8 * 8;
        const unsigned blocks = (unsigned)std::min<int64_t>(at_blocks(rows * heads * to), 148 * 16);
        uint16_t *dst = (uint16_t *)(ws + p.pack_at[i]);
        if (a.dtype == SPCONV_F16) attention_pack_kernel<<<blocks, kAtThreads, 0, st>>>(*t[i], (__half *)dst, rows, heads, a.D, to);
        else attention_pack_kernel<<<blocks, kAtThreads, 0, st>>>(*t[i], (__nv_bfloat16 *)dst, rows, heads, a.D, to);
        if (const int rc = check_launch("attention_pack_kernel")) return rc;
        *t[i] = {dst, (int64_t)heads * to, to};
    }
    return SPCONV_OK;
}

// The arguments with heads as wide as their rows of whole 16 bytes (zeros behind a packed head's end).
static AtArgs at_whole(const AtArgs &a) {
    AtArgs w = a;
    w.D = (a.D + 7) / 8 * 8;
    return w;
}

}  // namespace spconv

using namespace spconv;

extern "C" int64_t spconv_attention_workspace_bytes(const spconv_attention_args *q, int backward) {
    if (!q || q->num_queries < 0 || q->num_keys < 0 || q->num_samples < 1 || q->key_heads < 1 || q->heads < q->key_heads ||
        q->heads % q->key_heads || q->head_size < 1 || q->head_size > SPCONV_ATTENTION_MAX_SIZE)
        return -1;
    return at_plan(q, backward != 0).bytes;
}

extern "C" int spconv_attention_forward(const spconv_attention_args *q, void *stream) {
    if (const int rc = at_check(q, false)) return rc;
    if (q->num_queries == 0) return SPCONV_OK;
    const AtPlan p = at_plan(q, false);
    AtArgs a;
    if (const int rc = at_prepare(q, p, false, (cudaStream_t)stream, a)) return rc;
    a.splits = p.splits[0];
    if (const int rc = p.tc ? launch_at_tc_forward(a, p.pair) : launch_at_simt_forward(a)) return rc;
    if (a.splits == 1) return SPCONV_OK;
    return at_by_type(a.dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const int share = (int64_t)a.M * a.H <= 4096 ? kAtThreads / 32 : 1;
        attention_join_kernel<T><<<at_blocks((int64_t)a.M * a.H * share * 32), kAtThreads, 0, a.stream>>>(a, share);
        return check_launch("attention_join_kernel");
    });
}

extern "C" int spconv_attention_backward(const spconv_attention_args *q, void *stream) {
    if (const int rc = at_check(q, true)) return rc;
    const AtPlan p = at_plan(q, true);
    AtArgs a;
    if (const int rc = at_prepare(q, p, true, (cudaStream_t)stream, a)) return rc;
    if (a.M > 0) {
        const bool wide = a.D % 8 == 0 && (((uintptr_t)q->grad_out | (uintptr_t)q->out | (uintptr_t)q->out_rest) & 15) == 0 &&
                          q->grad_row % 8 == 0 && q->grad_head % 8 == 0;
        if (a.peaks && cudaMemsetAsync(a.peaks, 0, (size_t)a.B * 8, a.stream) != cudaSuccess) return check_launch("attention: clear");
        AtArgs d = a;
        d.grad = {q->grad_out, q->grad_row, q->grad_head};
        const int rc = at_by_type(a.dtype, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            auto kern = wide ? attention_delta_kernel<T, true> : attention_delta_kernel<T, false>;
            kern<<<at_blocks((int64_t)a.M * a.H * 8), kAtThreads, 0, a.stream>>>(d);
            return check_launch("attention_delta_kernel");
        });
        if (rc) return rc;
        if (a.peaks) {                       // (a.v as the products read it: packed where its own layout is not aligned)
            const int64_t rows = (int64_t)a.M * a.H, values = (int64_t)a.N * a.K;
            auto share = [](int64_t n, int each, int many) { return std::max<int64_t>(1, (n + (int64_t)each * many - 1) / ((int64_t)each * many)); };
            const int64_t parts = share(values, 128, 148 * 8), steps = share(rows, 128, 148 * 32);
            const int64_t blocks = std::max((values + parts * 128 - 1) / (parts * 128), (rows + steps * 1024 - 1) / (steps * 1024));
            attention_peaks_kernel<<<dim3((unsigned)blocks, 2), kAtThreads, 0, a.stream>>>(at_whole(a), parts, steps * 128);
            if (const int rc2 = check_launch("attention_peaks_kernel")) return rc2;
        }
    }
    auto join = [&](const float *from, int64_t stride, void *to, int64_t n) {
        if (!to || n == 0) return (int)SPCONV_OK;
        return at_by_type(a.dtype, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            attention_sum_kernel<T><<<at_blocks(n), kAtThreads, 0, a.stream>>>(from, stride, a.splits, (T *)to, n);
            return check_launch("attention_sum_kernel");
        });
    };
    if (a.gq && a.M > 0) {
        a.splits = p.splits[0];
        if (const int rc = p.tc ? launch_at_tc_grad_query(a) : launch_at_simt_grad_query(a)) return rc;
        const int64_t n = (int64_t)a.M * a.H * a.D;
        if (a.splits > 1)
            if (const int rc = join(a.partial, n, a.gq, n)) return rc;
    }
    if ((a.gk || a.gv) && a.N > 0) {
        a.splits = p.splits[1];
        if (const int rc = p.tc ? launch_at_tc_grad_key(a) : launch_at_simt_grad_key(a)) return rc;
        const int64_t n = (int64_t)a.N * a.K * a.D;
        if (a.splits > 1) {
            if (const int rc = join(a.partial, 2 * n, a.gk, n)) return rc;
            if (const int rc = join(a.partial + n, 2 * n, a.gv, n)) return rc;
        }
    }
    return SPCONV_OK;
}
