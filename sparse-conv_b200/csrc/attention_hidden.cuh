// Results that a hidden value has spoilt. Tiles on a causal sample's diagonal hold keys that a row does not see: p and ds are 0 there,
// and 0 times an infinity or a NaN is NaN. A thread that has stored a result that is not finite looks for such a value among what its
// row (or its key) does not see, and if there is one adds up again what it does see, one by one in fp32. Results that are finite,
// which are all of them unless the inputs are not, cost half a product a value as they are stored, in causal calls: 4 x 128 over 5,000
// tokens 457 -> 460, 575 -> 581 and 816 -> 822 us (forward, queries', keys' gradients); 8 x 64 in scenes of 3,000 to 7,500 768 -> 790,
// 942 -> 946 and 1,307 -> 1,350.
#pragma once

#include "attention_common.cuh"

namespace spconv {

constexpr int kAtAgain = 32;             // sums between two looks whether any of them is still a number

template <typename T>
__device__ __forceinline__ const T *at_row(const AtTensor &t, int64_t row, int head) {
    return (const T *)t.p + row * t.row + head * t.head;
}
template <typename T>
__device__ __forceinline__ float at_dot(const T *x, const T *y, int D) {
    float s = 0.f;
    for (int d = 0; d < D; ++d) s = fmaf(dtype_traits<T>::to_f(x[d]), dtype_traits<T>::to_f(y[d]), s);
    return s;
}
constexpr int kAtSums = 16;              // columns that are added up at a time

__device__ __forceinline__ bool at_is_lost(float x) { return !(fabsf(x) < INFINITY); }
// Whether one of the columns from `c` on is not finite.
template <typename T>
__device__ __forceinline__ bool at_any_lost(const T *x, int c, int D) {
    bool lost = false;
    for (int d = c; d < min(c + kAtSums, D); ++d) lost |= at_is_lost(dtype_traits<T>::to_f(x[d]));
    return lost;
}
template <typename T>
__device__ __forceinline__ void at_add(float (&sums)[kAtSums], float weight, const T *x, int c, int D) {
#pragma unroll
    for (int i = 0; i < kAtSums; ++i)
        if (c + i < D) sums[i] = fmaf(weight, dtype_traits<T>::to_f(x[c + i]), sums[i]);
}
__device__ __forceinline__ bool at_all_lost(const float (&sums)[kAtSums], int c, int D) {
    bool all = true;
#pragma unroll
    for (int i = 0; i < kAtSums; ++i) all &= c + i >= D || sums[i] != sums[i];
    return all;
}

// Where a row's results have been stored, in fp32 or rounded.
template <typename T>
struct AtStored {
    float *part;
    T *out;
    __device__ __forceinline__ bool lost(int c, int D) const { return part ? at_any_lost(part, c, D) : at_any_lost(out, c, D); }
    __device__ __forceinline__ void put(int c, int D, const float (&sums)[kAtSums], float factor) const {
#pragma unroll
        for (int i = 0; i < kAtSums; ++i) {
            if (c + i >= D) continue;
            if (part) part[c + i] = sums[i] * factor;
            else out[c + i] = dtype_traits<T>::from_f(sums[i] * factor);
        }
    }
};

// A query row of a sample whose keys begin at k0, and of those the range that was added up: it sees [lo, seen) of [lo, hi).
struct AtHidden {
    int64_t row;
    int head, key_head, k0, lo, seen, hi;
};

// out = factor sum_j 2^(s_j c + shift) v_j (and what its rounding leaves out).
template <typename T>
__device__ __noinline__ void at_values_again(const AtArgs &a, const AtHidden r, float shift, float factor, float *part) {
    const int64_t at = (r.row * a.H + r.head) * a.D;
    const AtStored<T> to{part, (T *)a.out + at};
    const T *q = at_row<T>(a.q, r.row, r.head);
    for (int c = 0; c < a.D; c += kAtSums) {
        bool lost = false;
        if (to.lost(c, a.D))
            for (int j = r.seen; j < r.hi && !lost; ++j) lost = at_any_lost(at_row<T>(a.v, r.k0 + j, r.key_head), c, a.D);
        if (!lost) continue;
        float sums[kAtSums] = {};
        for (int j = r.lo; j < r.seen; ++j) {
            const float s = at_dot(q, at_row<T>(a.k, r.k0 + j, r.key_head), a.D);
            at_add(sums, exp2f(fmaf(s, a.c, shift)), at_row<T>(a.v, r.k0 + j, r.key_head), c, a.D);
            if (j % kAtAgain == 0 && at_all_lost(sums, c, a.D)) break;
        }
        if (part) to.put(c, a.D, sums, factor);
        else
            for (int i = 0; i < kAtSums && c + i < a.D; ++i) at_put<T>(a, at + c + i, sums[i] * factor);
    }
}

// grad_query = factor sum_j ds_j k_j, ds_j = 2^(s_j c + shift) (grad . v_j - delta), columns [from, end).
template <typename T>
__device__ __noinline__ void at_keys_again(const AtArgs &a, const AtHidden r, float shift, float delta, int from, int end, float factor,
                                           const AtStored<T> to) {
    const T *q = at_row<T>(a.q, r.row, r.head), *g = at_row<T>(a.grad, r.row, r.head);
    for (int c = from; c < min(end, a.D); c += kAtSums) {
        bool lost = false;
        if (to.lost(c, a.D))
            for (int j = r.seen; j < r.hi && !lost; ++j) lost = at_any_lost(at_row<T>(a.k, r.k0 + j, r.key_head), c, a.D);
        if (!lost) continue;
        float sums[kAtSums] = {};
        for (int j = r.lo; j < r.seen; ++j) {
            const T *k = at_row<T>(a.k, r.k0 + j, r.key_head);
            const float p = exp2f(fmaf(at_dot(q, k, a.D), a.c, shift));
            const float ds = p * (at_dot(g, at_row<T>(a.v, r.k0 + j, r.key_head), a.D) - delta);
            at_add(sums, r.seen > 1 ? ds : 0.f, k, c, a.D);          // (a single key's probability is 1)
            if (j % kAtAgain == 0 && at_all_lost(sums, c, a.D)) break;
        }
        to.put(c, a.D, sums, factor);
    }
}

// The query tiles that a block has walked for its keys (attention_tc_grad_key_kernel): of tokens x P heads; tile `it`, in [first, last), is
// number from + it % per_head of the group's block of heads it / per_head.
struct AtWalked {
    int n, m, tokens, P, from, per_head, first, last;
    __device__ __forceinline__ AtWalked(const AtArgs &a, const AtSample &s, int key0, int rows, int log_p) {
        n = s.q1 - s.q0;
        m = s.k1 - s.k0;
        tokens = rows >> log_p;
        P = 1 << log_p;
        from = a.causal ? (int)max((int64_t)0, (int64_t)key0 - m + n) / tokens : 0;
        per_head = max(0, (n + tokens - 1) / tokens - from);
        at_split(a.splits, blockIdx.z, per_head * (a.H / a.K >> log_p), first, last);
    }
};

// A key's grad_value = sum_i p_i grad_i, or grad_key = scale sum_i p_i (grad_i . v - delta_i) q_i, over the rows that see it; columns
// [begin, end).
template <typename T>
__device__ __noinline__ void at_rows_again(const AtArgs &a, const AtSample &s, int tile_keys, int tile_rows, int log_p, bool values, int begin,
                                           int end, const AtStored<T> to) {
    const int key0 = s.tile * tile_keys, key = key0 + (threadIdx.x & (tile_keys - 1)), kh = blockIdx.y, head0 = kh * (a.H / a.K);
    const AtWalked w(a, s, key0, tile_rows, log_p);
    const T *k = at_row<T>(a.k, s.k0 + key, kh), *v = at_row<T>(a.v, s.k0 + key, kh);
    for (int c = begin; c < min(end, a.D); c += kAtSums) {
        if (!to.lost(c, a.D)) continue;
        float sums[kAtSums] = {};
        bool lost = false, done = false;
        for (int again = 0; again < 2 && !done; ++again) {           // first what the key is hidden from, then what it is not
            int count = 0;
            for (int it = w.first; it < w.last && !done; ++it) {
                const int t0 = (w.from + it % w.per_head) * w.tokens, t1 = min(w.n, t0 + w.tokens), h0 = head0 + it / w.per_head * w.P;
                if (!again && key < at_seen(a, t0, w.n, w.m)) continue;
                for (int t = t0; t < t1 && !done; ++t) {
                    const int seen = at_seen(a, t, w.n, w.m);
                    if ((again != 0) != (key < seen)) continue;
                    for (int h = h0; h < h0 + w.P && !done; ++h) {
                        const T *q = at_row<T>(a.q, s.q0 + t, h), *g = at_row<T>(a.grad, s.q0 + t, h);
                        if (!again) {
                            lost |= at_any_lost(values ? g : q, c, a.D);
                            continue;
                        }
                        const int64_t at = (int64_t)(s.q0 + t) * a.H + h;
                        const float p = exp2f(fmaf(at_dot(q, k, a.D), a.c, -a.lse[at]));
                        if (values) at_add(sums, p, g, c, a.D);
                        else if (seen > 1) at_add(sums, p * (at_dot(g, v, a.D) - a.delta[at]), q, c, a.D);
                        done = ++count % kAtAgain == 0 && at_all_lost(sums, c, a.D);
                    }
                }
            }
            if (!again && !lost) break;
        }
        if (lost) to.put(c, a.D, sums, values ? 1.f : a.scale);
    }
}

}  // namespace spconv
