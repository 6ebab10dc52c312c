// What every attention kernel does with the samples' offsets.
#pragma once

#include "attention_internal.h"
#include "common.cuh"

namespace spconv {

__device__ __forceinline__ int at_offset(const int32_t *offsets, int b, int rows) {
    return offsets ? max(0, min(rows, __ldg(offsets + b))) : (b ? rows : 0);
}

// The sample that a row lies in: the last that begins at or before it. By a converged warp, 32 samples a step; inside [0, B)
// whatever the offsets hold.
__device__ __forceinline__ int at_sample_of(const int32_t *offsets, int B, int rows, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5, at = lo + lane * step;
        const bool in = lane == 0 || (at < hi && at_offset(offsets, at, rows) <= row);
        const int last = 31 - __clz((int)__ballot_sync(0xffffffffu, in));
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

struct AtSample {
    int b, tile;                         // the sample and the tile's number in it
    int q0, q1, k0, k1;                  // its query and key rows
};

// The sample that tile `t` belongs to, where sample b's tiles are numbered from rows(b) / per_tile + b (its rows
// never need more than the next one's number; a tile past a sample's end has nothing to do). By a converged warp, 32 samples
// a step; ends inside [0, B) whatever the offsets hold, with a tile that begins inside the sample's rows, or -1.
__device__ __forceinline__ AtSample at_find(const AtArgs &a, bool keys, int t, int per_tile) {
    const int32_t *by = keys ? a.key_offsets : a.offsets;
    const int rows = keys ? a.N : a.M;
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = a.B;
    // Of many samples first the 32 about where it would be if all were alike, which for windows in their grid's order is mostly the
    // only step: 1,301 of 65 to 194 rows, 4 x 32 fp16, forward 152 -> 145 us, queries' gradients 298 -> 286 (half of
    // them empty 201 -> 195; in the order of their sizes, where the guess fails, 249 -> 253).
    if (hi > 32) {
        const float part = __fdividef((float)t, (float)(rows / per_tile + a.B));
        const int first = max(0, min(a.B - 32, (int)(part * (float)a.B) - 16)), at = first + lane;
        const unsigned in = __ballot_sync(0xffffffffu, at == 0 || at_offset(by, at, rows) / per_tile + at <= t);
        const int last = 31 - __clz((int)in);                        // -1: before them all
        if (last < 0) hi = first;
        else lo = first + last;
        if (last >= 0 && last < 31) hi = lo + 1;
    }
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5, at = lo + lane * step;
        const bool in = lane == 0 || (at < hi && at_offset(by, at, rows) / per_tile + at <= t);
        const int last = 31 - __clz((int)__ballot_sync(0xffffffffu, in));
        lo += last * step;
        hi = min(hi, lo + step);
    }
    AtSample s;
    s.b = lo;
    s.tile = t - (at_offset(by, lo, rows) / per_tile + lo);
    s.q0 = at_offset(a.offsets, lo, a.M);
    s.q1 = max(s.q0, at_offset(a.offsets, lo + 1, a.M));
    s.k0 = at_offset(a.key_offsets, lo, a.N);
    s.k1 = max(s.k0, at_offset(a.key_offsets, lo + 1, a.N));
    const int own = keys ? s.k1 - s.k0 : s.q1 - s.q0;
    if (s.tile < 0 || s.tile >= own / per_tile + (own % per_tile != 0)) s.tile = -1;
    return s;
}

// Offsets have to ascend from 0 to the rows; by the first block.
__device__ __forceinline__ void at_check_offsets(const AtArgs &a) {
    if (blockIdx.x | blockIdx.y | blockIdx.z) return;
    bool bad = false;
    for (int which = 0; which < 2; ++which) {
        const int32_t *o = which ? a.key_offsets : a.offsets;
        const int rows = which ? a.N : a.M;
        if (!o) continue;
        for (int s = threadIdx.x; s < a.B; s += blockDim.x) {
            const int lo = __ldg(o + s), hi = __ldg(o + s + 1);
            bad |= lo > hi || (s == 0 && lo != 0) || (s == a.B - 1 && hi != rows);
        }
    }
    if (bad) raise_status(a.status, SPCONV_STATUS_OFFSETS);
    __syncwarp();                        // lanes have walked different numbers of samples
}

// Keys that query i of a sample of n queries and m keys sees: the last query sees the last key.
__device__ __forceinline__ int at_seen(const AtArgs &a, int i, int n, int m) {
    return a.causal ? (int)max((int64_t)0, min((int64_t)m, (int64_t)i + 1 + m - n)) : m;
}

// Split `s` of `count` tiles: [first, last).
__device__ __forceinline__ void at_split(int splits, int s, int count, int &first, int &last) {
    const int per = (count + splits - 1) / splits;
    first = min(count, s * per);
    last = min(count, first + per);
}

// The power of two by which a sample's ds is lifted where it has to be rounded to fp16: |ds| <= 2 |grad row| |v row|, so the largest
// is at most 2^15, and rows of thousands of keys, or gradients of any size, keep their digits above fp16's smallest values.
__device__ __forceinline__ int at_lift(const AtArgs &a, int b) {
    if (!a.peaks) return 0;
    const float2 squares = __ldg(reinterpret_cast<const float2 *>(a.peaks) + b);
    const float x = sqrtf(squares.x) * sqrtf(squares.y);
    if (!(x > 0.f && x < INFINITY)) return 0;
    int e;
    frexpf(x, &e);                       // x <= 2^e
    return max(-60, min(60, 14 - e));
}

// Stores a result and, where it is kept, what rounding took from it.
template <typename T>
__device__ __forceinline__ void at_put(const AtArgs &a, int64_t i, float x) {
    const T hi = dtype_traits<T>::from_f(x);
    ((T *)a.out)[i] = hi;
    if (a.rest) ((T *)a.rest)[i] = dtype_traits<T>::from_f(x - dtype_traits<T>::to_f(hi));
}

}  // namespace spconv
