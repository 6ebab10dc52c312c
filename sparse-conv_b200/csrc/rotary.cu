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
// Bound: HBM, each value read once and written once. A block takes `rows` consecutive rows: their sines and cosines go to
// shared memory first (one pair a thread), then the threads walk the rows' heads, 16 bytes of each half of
// a pair at a time where half, head size, strides and addresses allow, else one value.
#include <algorithm>

#include "common.cuh"

namespace spconv {

constexpr int kRoThreads = 256;
constexpr int kRoMaxPairs = SPCONV_ROTARY_MAX_PAIRS;
constexpr int kRoTable = 2048;               // (cos, sin) pairs of a block: 16 KB

struct RoTensor {
    const void *in;
    void *out;
    int64_t in_row, in_head, out_row, out_head;
};
struct RoArgs {
    RoTensor t[2];
    int heads[2];                            // of t[0] (queries) and t[1] (keys)
    const int32_t *pos;
    int64_t pos_row, pos_col;
    int64_t num_rows;
    int rows;                                // rows of a block
    int axes, per_axis, pairs, half, size;
    float amplitude;
    int inverse;
    uint64_t step[kRoMaxPairs];              // of an axis's pairs
};

template <typename T, int V>
struct alignas(sizeof(T) * V) RoVec { T x[V]; };

// V values of each half of V pairs (HALF), V values of V / 2 neighbouring pairs (not HALF), or V to copy, as one unit.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kRoThreads)
rotary_kernel(const __grid_constant__ RoArgs a) {
    __shared__ float2 table[kRoTable];
    using Vec = RoVec<T, V>;
    const int64_t row0 = (int64_t)blockIdx.x * a.rows;
    const int rows = (int)min((int64_t)a.rows, a.num_rows - row0);
    const int tid = threadIdx.x;
    for (int i = tid; i < rows * a.half; i += kRoThreads) {
        const int r = i / a.half, p = i - r * a.half;
        float2 cs = make_float2(1.f, 0.f);
        if (p < a.pairs) {
            const int axis = p / a.per_axis;
            const int32_t t = __ldg(a.pos + (row0 + r) * a.pos_row + axis * a.pos_col);
            const uint64_t turn = (uint64_t)(int64_t)t * a.step[p - axis * a.per_axis];
            float s, c;
            sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
            cs = make_float2(c * a.amplitude, (a.inverse ? -s : s) * a.amplitude);
        }
        table[i] = cs;
    }
    __syncthreads();
    const int turned = HALF ? a.half / V : (V == 1 ? a.half : 2 * a.half / V);   // units of pairs
    const int rest = (a.size - 2 * a.half) / V;                                  // units to copy
    const int units = turned + rest, heads = a.heads[0] + a.heads[1];
    // threads in groups of `units` (or all for one head at a time, where a head has more)
    const int lanes = min(units, kRoThreads), groups = kRoThreads / lanes;
    const int g = tid / lanes;
    if (g >= groups) return;
    int r = g / heads, h = g - r * heads;
    const int dr = groups / heads, dh = groups - dr * heads;
    while (r < rows) {
        const int k = h >= a.heads[0];
        const RoTensor &t = a.t[k];
        const int hh = k ? h - a.heads[0] : h;
        const T *in = (const T *)t.in + (row0 + r) * t.in_row + hh * t.in_head;
        T *out = (T *)t.out + (row0 + r) * t.out_row + hh * t.out_head;
        const float2 *cs = table + r * a.half;
        for (int u = tid - g * lanes; u < units; u += lanes) {
            if (u >= turned) {
                const int c = 2 * a.half + (u - turned) * V;
                *(Vec *)(out + c) = *(const Vec *)(in + c);
            } else if constexpr (HALF) {
                Vec x = *(const Vec *)(in + u * V), y = *(const Vec *)(in + a.half + u * V);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float p = dtype_traits<T>::to_f(x.x[i]), q = dtype_traits<T>::to_f(y.x[i]);
                    const float2 w = cs[u * V + i];
                    x.x[i] = dtype_traits<T>::from_f(p * w.x - q * w.y);
                    y.x[i] = dtype_traits<T>::from_f(p * w.y + q * w.x);
                }
                *(Vec *)(out + u * V) = x;
                *(Vec *)(out + a.half + u * V) = y;
            } else if constexpr (V == 1) {
                const float p = dtype_traits<T>::to_f(in[2 * u]), q = dtype_traits<T>::to_f(in[2 * u + 1]);
                const float2 w = cs[u];
                out[2 * u] = dtype_traits<T>::from_f(p * w.x - q * w.y);
                out[2 * u + 1] = dtype_traits<T>::from_f(p * w.y + q * w.x);
            } else {
                Vec x = *(const Vec *)(in + u * V);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const float p = dtype_traits<T>::to_f(x.x[2 * i]), q = dtype_traits<T>::to_f(x.x[2 * i + 1]);
                    const float2 w = cs[u * (V / 2) + i];
                    x.x[2 * i] = dtype_traits<T>::from_f(p * w.x - q * w.y);
                    x.x[2 * i + 1] = dtype_traits<T>::from_f(p * w.y + q * w.x);
                }
                *(Vec *)(out + u * V) = x;
            }
        }
        r += dr;
        h += dh;
        if (h >= heads) {
            h -= heads;
            ++r;
        }
    }
}

template <typename T>
static int ro_launch(const RoArgs &a, bool half, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool wide = a.size % V == 0 && (half ? a.half : 2 * a.half) % V == 0;
    for (int i = 0; i < 2; ++i) {
        const RoTensor &t = a.t[i];
        if (a.heads[i] == 0) continue;
        wide = wide && (((uintptr_t)t.in | (uintptr_t)t.out) & 15) == 0 &&
               ((t.in_row | t.in_head | t.out_row | t.out_head) % V) == 0;
    }
    const int64_t blocks = (a.num_rows + a.rows - 1) / a.rows;
    auto kern = half ? (wide ? rotary_kernel<T, V, true> : rotary_kernel<T, 1, true>)
                     : (wide ? rotary_kernel<T, V, false> : rotary_kernel<T, 1, false>);
    kern<<<(unsigned)blocks, kRoThreads, 0, st>>>(a);
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
    SPCONV_REQUIRE(q->heads >= 0 && q->key_heads >= 0 && q->heads <= 65535 && q->key_heads <= 65535 && q->heads + q->key_heads > 0,
                   SPCONV_ERR_ARG, "head counts out of range");
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
    // rows of a block: at most a table's worth of pairs, and about 16 KB of values
    const int64_t row_bytes = (int64_t)(q->heads + q->key_heads) * q->head_size * (q->dtype == SPCONV_F32 ? 4 : 2);
    a.rows = (int)std::max<int64_t>(1, std::min<int64_t>({kRoTable / a.half, 16384 / row_bytes, (q->num_rows + 147) / 148}));
    const cudaStream_t st = (cudaStream_t)stream;
    const bool half = q->layout == SPCONV_ROTARY_HALF;
    if (q->dtype == SPCONV_F32) return ro_launch<float>(a, half, st);
    if (q->dtype == SPCONV_F16) return ro_launch<__half>(a, half, st);
    return ro_launch<__nv_bfloat16>(a, half, st);
}
