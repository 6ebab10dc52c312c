// Rotary positions: pairs of a head's values turned by an angle that grows with the voxel's coordinates,
//
//   (a, b) -> amplitude * (a cos - b sin, a sin + b cos),   angle = position[axis] * step[pair],
//
// for queries and keys at once (the sines of a row serve all heads of both). Pair i of an axis's n pairs belongs
// to axis i / n; a pair is columns (i, i + half) or (2 i, 2 i + 1) of the head's first 2 * half columns; columns
// behind them, and pairs behind the last axis's, are copied. The gradient is the same turn backwards.
//
// Angles are exact to the last bit that matters at any position: a step is given in 2^-64ths of a full turn, so that
// position * step modulo 2^64 is the fraction of a turn left after all whole ones, without a rounding (fp32
// angles are off by 0.06 at position 2^20, and a product in fp64 would cost 64 times the fp32 one's time).
//
// Bound: HBM, each value read once and written once. A block takes `rows` consecutive rows. Their sines and cosines go to
// shared memory, one pair a thread, while the rows' values are on their way: 16 bytes of each half of a pair (or of
// neighbouring pairs) at a time where half, head size, strides and addresses allow; for other sizes of contiguous
// tensors the block's whole range goes through shared memory in 16-byte pieces; strided ones are taken value by value.
// 84,000 x (8 + 8) x 64 bf16 61 us (70.9 with the sines before the loads), 5.6 TB/s; 168,546 x (3 + 1) x 35 fp32 38 us a
// launch (85 value by value).
#include <algorithm>

#include "common.cuh"

namespace spconv {

constexpr int kRoThreads = 256;
constexpr int kRoMaxPairs = SPCONV_ROTARY_MAX_PAIRS;
constexpr int kRoTable = 2048;               // (cos, sin) pairs of a block: 16 KB

constexpr int kRoSlots = 8;                  // vectors a thread has in flight
constexpr int kRoStaged = 24 * 1024;         // bytes of values a block stages

struct RoTensor {
    const void *in;
    void *out;
    int64_t in_row, in_head, out_row, out_head;
};
// Quotients of small numbers (n < 2^16) by a divisor known to the host.
struct RoDiv {
    uint32_t d, magic;
    __device__ __forceinline__ int operator()(int n) const { return d == 1 ? n : (int)__umulhi((uint32_t)n, magic); }
};
static RoDiv ro_div(int d) { return {(uint32_t)d, (uint32_t)(((1ull << 32) + d - 1) / d)}; }
struct RoArgs {
    RoTensor t[2];
    int heads[2];                            // of t[0] (queries) and t[1] (keys)
    const int32_t *pos;
    int64_t pos_row, pos_col;
    int64_t num_rows;
    int rows;                                // rows of a block
    int axes, per_axis, pairs, half, size;
    int turned, units;                       // units of a head that hold pairs, and all of them
    int heads_here, step_rows;               // heads of a block, and rows that it takes at a time
    RoDiv by_half, by_units, by_heads, by_axis;
    float amplitude;
    int inverse;
    uint64_t step[kRoMaxPairs];              // of an axis's pairs
};

template <typename T, int V>
struct alignas(sizeof(T) * V) RoVec { T x[V]; };

// Cosines and sines of the block's rows, (1, 0) for pairs that no axis turns. FAST: good to 2^-21 of the circle's radius (the
// reduced angle is within half a turn), for values that are rounded to 2^-9 or 2^-12 of their size.
template <bool FAST>
__device__ __forceinline__ void ro_table(const RoArgs &a, float2 *table, int64_t row0, int rows) {
    for (int i = threadIdx.x; i < rows * a.half; i += kRoThreads) {
        const int r = a.by_half(i), p = i - r * a.half;
        float2 cs = make_float2(1.f, 0.f);
        if (p < a.pairs) {
            const int axis = a.by_axis(p);
            const int32_t t = __ldg(a.pos + (row0 + r) * a.pos_row + axis * a.pos_col);
            const uint64_t turn = (uint64_t)(int64_t)t * a.step[p - axis * a.per_axis];
            float s, c;
            if constexpr (FAST) __sincosf((float)(int32_t)(turn >> 32) * 1.4629180792671596e-9f, &s, &c);     // 2 pi / 2^32
            else sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
            cs = make_float2(c * a.amplitude, (a.inverse ? -s : s) * a.amplitude);
        }
        table[i] = cs;
    }
}

template <typename T>
__device__ __forceinline__ void ro_turn(T &x, T &y, float2 w) {
    const float p = dtype_traits<T>::to_f(x), q = dtype_traits<T>::to_f(y);
    x = dtype_traits<T>::from_f(p * w.x - q * w.y);
    y = dtype_traits<T>::from_f(p * w.y + q * w.x);
}

// A unit: V values of each half of V pairs (HALF), V / 2 neighbouring pairs (one where V is 1), or V values to copy. A thread
// keeps its unit and its head and takes every step_rows-th of the block's rows; with V > 1 all of them are on their way
// into its own slots in shared memory at once (eight of 16 bytes a thread, four blocks an SM: what HBM's latency takes)
// while the table is made.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kRoThreads, 4)
rotary_kernel(const __grid_constant__ RoArgs a) {
    using Vec = RoVec<T, V>;
    constexpr bool TWO = HALF || V == 1;                             // a unit of pairs is two vectors
    constexpr int B = kRoSlots / (TWO ? 2 : 1);                      // a thread's rows
    extern __shared__ __align__(16) uint8_t smem[];
    uint4 *slots = reinterpret_cast<uint4 *>(smem) + threadIdx.x;    // [kRoSlots][kRoThreads] (V > 1)
    float2 *table = reinterpret_cast<float2 *>(smem + (V > 1 ? kRoSlots * kRoThreads * 16 : 0));
    const int64_t row0 = (int64_t)blockIdx.x * a.rows;
    const int rows = (int)min((int64_t)a.rows, a.num_rows - row0);
    const int g = a.by_units(threadIdx.x), u = threadIdx.x - g * a.units;
    int r = a.by_heads(g), h = g - r * a.heads_here;
    h += blockIdx.y * a.heads_here;
    if (r >= a.step_rows || h >= a.heads[0] + a.heads[1]) r = rows;   // a thread too many
    const int key = h >= a.heads[0];
    const RoTensor &t = a.t[key];
    const int hh = key ? h - a.heads[0] : h;
    const bool turned = u < a.turned;
    const int at = turned ? u * (HALF || V > 1 ? V : 2) : 2 * a.half + (u - a.turned) * V;   // first value's column, and the
    const int apart = HALF ? a.half : 1;                                                     // second one's distance
    const T *in = (const T *)t.in + (row0 + r) * t.in_row + hh * t.in_head + at;
    T *out = (T *)t.out + (row0 + r) * t.out_row + hh * t.out_head + at;
    const int64_t in_step = a.step_rows * t.in_row, out_step = a.step_rows * t.out_row;
    if constexpr (V > 1) {
#pragma unroll
        for (int k = 0; k < B; ++k) {
            if (r + k * a.step_rows >= rows) break;
            cp_async_16(smem_u32(slots + (TWO ? 2 * k : k) * kRoThreads), in + k * in_step, 16);
            if (TWO && turned) cp_async_16(smem_u32(slots + (2 * k + 1) * kRoThreads), in + k * in_step + apart, 16);
        }
        cp_async_commit();
    }
    ro_table<sizeof(T) == 2>(a, table, row0, rows);
    if constexpr (V > 1) cp_async_wait<0>();
    __syncthreads();
    const float2 *cs = table + r * a.half + u * (TWO ? V : V / 2);
#pragma unroll
    for (int k = 0; k < B; ++k, r += a.step_rows, in += in_step, out += out_step, cs += a.step_rows * a.half) {
        if (r >= rows) break;
        Vec x, y;
        if constexpr (V > 1) {
            x = *reinterpret_cast<const Vec *>(slots + (TWO ? 2 * k : k) * kRoThreads);
            if (TWO && turned) y = *reinterpret_cast<const Vec *>(slots + (2 * k + 1) * kRoThreads);
        } else {
            x = *(const Vec *)in;
            if (turned) y = *(const Vec *)(in + apart);
        }
        if (turned) {
            if constexpr (TWO) {
#pragma unroll
                for (int i = 0; i < V; ++i) ro_turn(x.x[i], y.x[i], cs[i]);
                *(Vec *)(out + apart) = y;
            } else {
#pragma unroll
                for (int i = 0; i < V / 2; ++i) ro_turn(x.x[2 * i], x.x[2 * i + 1], cs[i]);
            }
        }
        *(Vec *)out = x;
    }
}

// Contiguous tensors of any head size: the block's rows, whose number is a multiple of 8, begin on 16-byte boundaries.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kRoThreads)
rotary_staged_kernel(const __grid_constant__ RoArgs a) {
    __shared__ float2 table[kRoTable];
    __shared__ __align__(16) uint8_t staged[kRoStaged];
    constexpr int V = 16 / sizeof(T);
    const int64_t row0 = (int64_t)blockIdx.x * a.rows;
    const int rows = (int)min((int64_t)a.rows, a.num_rows - row0);
    T *part[2];
    part[0] = reinterpret_cast<T *>(staged);
    part[1] = part[0] + a.rows * a.heads[0] * a.size;                // a multiple of 8 values
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int n = rows * a.heads[k] * a.size;
        const T *in = (const T *)a.t[k].in + row0 * a.heads[k] * a.size;
        for (int i = threadIdx.x; i < n / V; i += kRoThreads) cp_async_16(smem_u32(part[k] + i * V), in + i * V, 16);
        for (int i = n / V * V + threadIdx.x; i < n; i += kRoThreads) part[k][i] = in[i];
    }
    cp_async_commit();
    ro_table<sizeof(T) == 2>(a, table, row0, rows);
    cp_async_wait<0>();
    __syncthreads();
    const int heads = a.heads[0] + a.heads[1];
    for (int i = threadIdx.x; i < rows * heads * a.half; i += kRoThreads) {
        const int hr = a.by_half(i), r = a.by_heads(hr), h = hr - r * heads, p = i - hr * a.half;
        T *x = h < a.heads[0] ? part[0] + (r * a.heads[0] + h) * a.size : part[1] + (r * a.heads[1] + h - a.heads[0]) * a.size;
        T &first = x[HALF ? p : 2 * p], &second = x[HALF ? p + a.half : 2 * p + 1];
        ro_turn(first, second, table[r * a.half + p]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int n = rows * a.heads[k] * a.size;
        T *out = (T *)a.t[k].out + row0 * a.heads[k] * a.size;
        for (int i = threadIdx.x; i < n / V; i += kRoThreads) *(uint4 *)(out + i * V) = *(const uint4 *)(part[k] + i * V);
        for (int i = n / V * V + threadIdx.x; i < n; i += kRoThreads) out[i] = part[k][i];
    }
}

template <typename T>
static int ro_launch(RoArgs &a, bool half, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int heads = a.heads[0] + a.heads[1], row = heads * a.size;
    bool wide = a.size % V == 0 && (half ? a.half : 2 * a.half) % V == 0, dense = true;
    for (int i = 0; i < 2; ++i) {
        const RoTensor &t = a.t[i];
        if (a.heads[i] == 0) continue;
        const bool aligned = (((uintptr_t)t.in | (uintptr_t)t.out) & 15) == 0;
        wide = wide && aligned && ((t.in_row | t.in_head | t.out_row | t.out_head) % V) == 0;
        dense = dense && aligned && (t.in_row == t.out_row || a.num_rows == 1) && (t.in_head == t.out_head || a.heads[i] == 1);
    }
    // a thread's batch of units, a table's worth of pairs, no fewer blocks than SMs
    const int64_t spread = (a.num_rows + 147) / 148;
    auto rows_of = [&](int64_t most) { return (int)std::max<int64_t>(1, std::min<int64_t>({most, kRoTable / a.half, spread})); };
    const int staged = std::min<int>(kRoTable / a.half, (int)std::min<int64_t>(kRoStaged / ((int64_t)row * sizeof(T)), 1 << 16)) / 8 * 8;
    void (*kern)(const RoArgs);
    int head_blocks = 1, smem = 0;
    a.heads_here = heads;
    if (!wide && dense && staged >= 8 && (int64_t)staged * heads * a.half < 1 << 16) {
        a.rows = std::min<int>(staged, (int)std::max<int64_t>(8, (spread + 7) / 8 * 8));
        kern = half ? rotary_staged_kernel<T, true> : rotary_staged_kernel<T, false>;
    } else {
        const int v = wide ? V : 1;
        a.turned = half || v == 1 ? a.half / v : 2 * a.half / v;
        a.units = a.turned + (a.size - 2 * a.half) / v;
        const int groups = kRoThreads / a.units;                     // heads that a block takes at a time, of one row or several
        a.heads_here = std::min(heads, groups);
        a.step_rows = groups / a.heads_here;
        head_blocks = (heads + a.heads_here - 1) / a.heads_here;
        a.rows = rows_of((int64_t)a.step_rows * (half || v == 1 ? kRoSlots / 2 : kRoSlots));
        smem = (wide ? kRoSlots * kRoThreads * 16 : 0) + a.rows * a.half * (int)sizeof(float2);
        kern = half ? (wide ? rotary_kernel<T, V, true> : rotary_kernel<T, 1, true>)
                    : (wide ? rotary_kernel<T, V, false> : rotary_kernel<T, 1, false>);
    }
    a.by_half = ro_div(a.half);
    a.by_units = ro_div(std::max(1, a.units));
    a.by_heads = ro_div(a.heads_here);
    a.by_axis = ro_div(a.per_axis);
    kern<<<dim3((unsigned)((a.num_rows + a.rows - 1) / a.rows), head_blocks), kRoThreads, smem, st>>>(a);
    return check_launch("rotary_kernel");
}

}  // namespace spconv

using namespace spconv;

extern "C" int spconv_rotary(const spconv_rotary_args *q, void *stream) {
    SPCONV_REQUIRE(q != nullptr, SPCONV_ERR_ARG, "null pointer argument");
    SPCONV_REQUIRE(q->dtype == SPCONV_F32 || q->dtype == SPCONV_F16 || q->dtype == SPCONV_BF16, SPCONV_ERR_ARG,
                   "unsupported dtype code %d", q->dtype);
    SPCONV_REQUIRE(q->num_rows >= 0 && q->num_rows < (int64_t)1 << 31, SPCONV_ERR_ARG, "num_rows out of range");
    SPCONV_REQUIRE(q->head_size >= 2 && q->head_size <= 2 * kRoMaxPairs, SPCONV_ERR_ARG, "head size must be in [2, %d]",
                   2 * kRoMaxPairs);
    SPCONV_REQUIRE(q->rotary_dim >= 2 && q->rotary_dim <= q->head_size && q->rotary_dim % 2 == 0, SPCONV_ERR_ARG,
                   "rotary_dim must be even and in [2, head size]");
    SPCONV_REQUIRE(q->axes >= 1 && q->axes <= q->rotary_dim / 2, SPCONV_ERR_ARG, "axes must be in [1, rotary_dim / 2]");
    SPCONV_REQUIRE(q->layout == SPCONV_ROTARY_HALF || q->layout == SPCONV_ROTARY_INTERLEAVED, SPCONV_ERR_ARG,
                   "unknown layout %d", q->layout);
    SPCONV_REQUIRE(q->heads >= 0 && q->key_heads >= 0 && (int64_t)q->heads + q->key_heads > 0 && (int64_t)q->heads + q->key_heads <= 65535,
                   SPCONV_ERR_ARG, "heads must be in [1, 65535], of queries and keys together");
    if (q->num_rows == 0) return SPCONV_OK;
    SPCONV_REQUIRE(q->positions && (q->heads == 0 || (q->query && q->query_out)) && (q->key_heads == 0 || (q->key && q->key_out)),
                   SPCONV_ERR_ARG, "null pointer argument");
    RoArgs a = {};
    a.t[0] = {q->query, q->query_out, q->query_row, q->query_head, (int64_t)q->heads * q->head_size, q->head_size};
    a.t[1] = {q->key, q->key_out, q->key_row, q->key_head, (int64_t)q->key_heads * q->head_size, q->head_size};
    a.heads[0] = q->heads;
    a.heads[1] = q->key_heads;
    a.pos = q->positions;
    a.pos_row = q->position_row;
    a.pos_col = q->position_col;
    a.num_rows = q->num_rows;
    a.axes = q->axes;
    a.half = q->rotary_dim / 2;
    a.per_axis = a.half / a.axes;
    a.pairs = a.per_axis * a.axes;
    a.size = q->head_size;
    a.amplitude = q->amplitude;
    a.inverse = q->inverse != 0;
    std::copy(q->steps, q->steps + a.per_axis, a.step);
    const cudaStream_t st = (cudaStream_t)stream;
    const bool half = q->layout == SPCONV_ROTARY_HALF;
    if (q->dtype == SPCONV_F32) return ro_launch<float>(a, half, st);
    if (q->dtype == SPCONV_F16) return ro_launch<__half>(a, half, st);
    return ro_launch<__nv_bfloat16>(a, half, st);
}
