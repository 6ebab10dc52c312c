// The global norm of many gradient tensors and clipping by it:
//
//   n = sqrt(sum over all tensors of g^2)   (or the largest |g|)
//   out = g * min(1, max_norm / (n + 1e-6))
//
// Two launches for any mix of sizes and types: norm_kernel leaves one partial per block,
// scale_kernel starts from the partials (each block adds the few hundred of them itself, in the
// same order) and multiplies. Tensors are described in the kernel's own parameters, so no table
// is copied to the device and a captured graph needs no memory of the host's; lists longer than
// one parameter block holds take several launches of each.
//
// The elements of all tensors, in eights, are cut into one range per block, and a block walks its
// range with eight 16-byte loads a thread in flight, looking up a tensor only where one ends.
//
// Bound: HBM, one read for the norm and one read and write for the scaling; the second pass walks
// each range backwards, so what the first left in the L2 is read from there. Where nothing is
// clipped and the output is the gradient itself, nothing is moved. 97 M bf16 values: 45 us (4.3 TB/s)
// and 69 us (5.7 TB/s); twice the loads in flight change neither.
//
// Squares are added in fp32 eight at a time and the eights in fp64. An eight whose fp32 sum
// left the range in which squares are exact to fp32's precision (over 1e30, or under 1e-30) is
// added again in fp64, so gradients of any finite size have a finite, accurate norm.
#include <algorithm>
#include <vector>

#include "common.cuh"

namespace spconv {

constexpr int kClThreads = 256;
constexpr int kClBlocksPerSm = 4;            // all resident at 64 registers: one wave
constexpr int kClMaxBlocks = 148 * kClBlocksPerSm;
constexpr int kClBatch = 8;                  // 16-byte loads a thread has in flight

// K tensors in one launch's parameters.
template <int K>
struct ClTable {
    const void *grad[K];
    void *out[K];
    int64_t numel[K];
    int64_t first[K + 1];                    // eights of elements in the tensors before it
    uint8_t dtype[K];
    int n;
};
struct ClArgs {
    double *partial;                         // [num_partials]
    int first_partial, num_partials;
    int max_norm_kind;                       // 1: largest |g|
    float max_norm;
    float *total;
};

// The tensor that holds eight number e.
template <int K>
__device__ __forceinline__ int cl_find(const ClTable<K> &t, int64_t e) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {                        // last tensor with first <= e
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= e) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// This block's range of eights.
template <int K>
__device__ __forceinline__ void cl_range(const ClTable<K> &t, int64_t &e0, int64_t &e1) {
    const int64_t per = (t.first[t.n] + gridDim.x - 1) / gridDim.x;
    e0 = min(t.first[t.n], blockIdx.x * per);
    e1 = min(t.first[t.n], e0 + per);
}

template <typename T>
__device__ __forceinline__ void cl_unpack16(const uint4 &q, float *f) {
    const T *v = reinterpret_cast<const T *>(&q);
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) f[i] = dtype_traits<T>::to_f(v[i]);
}

// Adds up to 8 values into the running sum of squares, or the largest magnitude (as bits, above
// which NaN sorts).
__device__ __forceinline__ void cl_add8(const float *f, int n, bool largest, double &sum, uint32_t &top) {
    if (largest) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
        return;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) s = fmaf(f[i], f[i], s);
    if (s < 1e30f && s > 1e-30f) {
        sum += (double)s;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) sum += (double)f[i] * (double)f[i];
}

template <typename T>
__device__ __forceinline__ void cl_norm_chunk(const T *g, int n, bool largest, double &sum, uint32_t &top) {
    constexpr int V = 16 / sizeof(T), R = 8 / V;              // values and loads of 16 bytes in an eight
    int done = 0;
    if (((uintptr_t)g & 15) == 0) {
        const int eights = n / 8;
        const uint4 *q = reinterpret_cast<const uint4 *>(g);
        int e = threadIdx.x;
        constexpr int B = kClBatch / R;
        for (; e + (B - 1) * kClThreads < eights; e += B * kClThreads) {
            uint4 v[B][R];
#pragma unroll
            for (int u = 0; u < B; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) v[u][r] = __ldg(q + (e + u * kClThreads) * R + r);
#pragma unroll
            for (int u = 0; u < B; ++u) {
                float f[8];
#pragma unroll
                for (int r = 0; r < R; ++r) cl_unpack16<T>(v[u][r], f + r * V);
                cl_add8(f, 8, largest, sum, top);
            }
        }
        for (; e < eights; e += kClThreads) {
            float f[8];
#pragma unroll
            for (int r = 0; r < R; ++r) cl_unpack16<T>(__ldg(q + e * R + r), f + r * V);
            cl_add8(f, 8, largest, sum, top);
        }
        done = eights * 8;
    }
    for (int i = done + threadIdx.x; i < n; i += kClThreads) {
        const float f[8] = {dtype_traits<T>::to_f(g[i])};
        cl_add8(f, 1, largest, sum, top);
    }
}

// Backwards: the end of the part was read last by the norm.
template <typename T>
__device__ __forceinline__ void cl_scale_chunk(const T *g, T *out, int n, float coef) {
    constexpr int V = 16 / sizeof(T), kBatch = kClBatch * kClThreads;
    int done = 0;
    if ((((uintptr_t)g | (uintptr_t)out) & 15) == 0) done = n / V * V;
    for (int i = done + threadIdx.x; i < n; i += kClThreads)
        out[i] = dtype_traits<T>::from_f(dtype_traits<T>::to_f(g[i]) * coef);
    const int vecs = done / V, batches = vecs / kBatch;
    const uint4 *q = reinterpret_cast<const uint4 *>(g);
    uint4 *o = reinterpret_cast<uint4 *>(out);
    auto scale = [&](uint4 v) {
        T *x = reinterpret_cast<T *>(&v);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = dtype_traits<T>::from_f(dtype_traits<T>::to_f(x[i]) * coef);
        return v;
    };
    for (int e = batches * kBatch + threadIdx.x; e < vecs; e += kClThreads) __stcs(o + e, scale(__ldcs(q + e)));
    for (int b = batches - 1; b >= 0; --b) {
        const int e = b * kBatch + threadIdx.x;
        uint4 v[kClBatch];
#pragma unroll
        for (int u = 0; u < kClBatch; ++u) v[u] = __ldcs(q + e + u * kClThreads);
#pragma unroll
        for (int u = 0; u < kClBatch; ++u) __stcs(o + e + u * kClThreads, scale(v[u]));
    }
}

// The sum (or the largest) of one value per thread, the same bits in every run.
__device__ __forceinline__ double cl_block_reduce(double v, bool largest) {
    __shared__ double part[kClThreads / 32];
    auto join = [&](double a, double b) { return largest ? (isnan(a) || a > b ? a : b) : a + b; };
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kClThreads / 32; ++w) v = join(v, part[w]);
    return v;
}

template <int K>
__global__ void __launch_bounds__(kClThreads, kClBlocksPerSm)
clip_norm_kernel(const __grid_constant__ ClTable<K> t, const __grid_constant__ ClArgs a) {
    grid_launch_dependents();
    double sum = 0.0;
    uint32_t top = 0;
    const bool largest = a.max_norm_kind != 0;
    int64_t e, end;
    cl_range(t, e, end);
    for (int k = e < end ? cl_find(t, e) : 0; e < end; ++k) {
        const int64_t at = (e - t.first[k]) * 8, stop = min(end, t.first[k + 1]);
        const int n = (int)(min(t.numel[k], (stop - t.first[k]) * 8) - at);
        if (t.dtype[k] == SPCONV_F32) cl_norm_chunk((const float *)t.grad[k] + at, n, largest, sum, top);
        else if (t.dtype[k] == SPCONV_F16) cl_norm_chunk((const __half *)t.grad[k] + at, n, largest, sum, top);
        else cl_norm_chunk((const __nv_bfloat16 *)t.grad[k] + at, n, largest, sum, top);
        e = stop;
    }
    const double v = cl_block_reduce(largest ? (double)__uint_as_float(top) : sum, largest);
    if (threadIdx.x == 0) a.partial[a.first_partial + blockIdx.x] = v;
}

template <int K>
__global__ void __launch_bounds__(kClThreads, kClBlocksPerSm)
clip_scale_kernel(const __grid_constant__ ClTable<K> t, const __grid_constant__ ClArgs a) {
    grid_dependency_wait();
    const bool largest = a.max_norm_kind != 0;
    double v = 0.0;
    for (int i = threadIdx.x; i < a.num_partials; i += kClThreads) {
        const double p = __ldcg(a.partial + i);
        v = largest ? (isnan(v) || v > p ? v : p) : v + p;
    }
    v = cl_block_reduce(v, largest);
    const double total = largest ? v : sqrt(v);
    if (a.total && blockIdx.x == 0 && threadIdx.x == 0) *a.total = (float)total;
    const double ratio = (double)a.max_norm / (total + 1e-6);
    const float coef = ratio >= 1.0 ? 1.f : (float)ratio;     // NaN stays NaN
    int64_t begin, e;
    cl_range(t, begin, e);
    for (int k = begin < e ? cl_find(t, e - 1) : 0; e > begin; --k) {
        const int64_t start = max(begin, t.first[k]), at = (start - t.first[k]) * 8;
        const int n = (int)(min(t.numel[k], (e - t.first[k]) * 8) - at);
        e = start;
        if (coef == 1.f && t.out[k] == t.grad[k]) continue;
        if (t.dtype[k] == SPCONV_F32) cl_scale_chunk((const float *)t.grad[k] + at, (float *)t.out[k] + at, n, coef);
        else if (t.dtype[k] == SPCONV_F16) cl_scale_chunk((const __half *)t.grad[k] + at, (__half *)t.out[k] + at, n, coef);
        else cl_scale_chunk((const __nv_bfloat16 *)t.grad[k] + at, (__nv_bfloat16 *)t.out[k] + at, n, coef);
    }
}

struct ClRange {
    uintptr_t lo, hi;
    int tensor;
    bool operator<(const ClRange &o) const { return lo < o.lo; }
};

// A block per 512 eights, up to four blocks per SM; ranges of 2^28 eights are beyond any memory.
static int cl_blocks(int64_t eights) { return (int)std::max<int64_t>(1, std::min<int64_t>(kClMaxBlocks, (eights + 511) / 512)); }

template <int K>
static int cl_run(const void *const *grads, void *const *outs, const int64_t *numels, const int32_t *dtypes,
                  const std::vector<int> &live, ClArgs a, cudaStream_t st) {
    std::vector<ClTable<K>> tables((live.size() + K - 1) / K);
    int partials = 0;
    for (size_t i = 0; i < live.size(); ++i) {
        ClTable<K> &t = tables[i / K];
        const int j = (int)(i % K), k = live[i];
        if (j == 0) t.first[0] = 0;
        t.grad[j] = grads[k];
        t.out[j] = outs[k];
        t.numel[j] = numels[k];
        t.dtype[j] = (uint8_t)dtypes[k];
        t.first[j + 1] = t.first[j] + (numels[k] + 7) / 8;
        t.n = j + 1;
    }
    for (const auto &t : tables) partials += cl_blocks(t.first[t.n]);
    a.num_partials = partials;
    a.first_partial = 0;
    for (const auto &t : tables) {
        const int blocks = cl_blocks(t.first[t.n]);
        clip_norm_kernel<K><<<blocks, kClThreads, 0, st>>>(t, a);
        if (const int rc = check_launch("clip_norm_kernel")) return rc;
        a.first_partial += blocks;
    }
    // the norm has to be complete before the first value is scaled, so only the first scale
    // launch, which follows the last norm launch, may start under it
    bool first = true;
    for (const auto &t : tables) {
        const int blocks = cl_blocks(t.first[t.n]);
        if (first) launch_pdl(clip_scale_kernel<K>, dim3(blocks), dim3(kClThreads), 0, st, t, a);
        else clip_scale_kernel<K><<<blocks, kClThreads, 0, st>>>(t, a);
        if (const int rc = check_launch("clip_scale_kernel")) return rc;
        first = false;
        a.total = nullptr;
    }
    return SPCONV_OK;
}

}  // namespace spconv

using namespace spconv;

constexpr int kClSmall = 64, kClLarge = 512;

extern "C" int64_t spconv_clip_gradients_workspace_bytes(int num_tensors) {
    if (num_tensors < 0) return -1;
    return (int64_t)(num_tensors / kClLarge + 1) * kClMaxBlocks * (int64_t)sizeof(double);
}

extern "C" int spconv_clip_gradients(const void *const *grads, void *const *outs, const int64_t *numels,
                                     const int32_t *dtypes, int num_tensors, int norm_kind, float max_norm,
                                     float *total_norm, void *workspace, int64_t workspace_bytes, void *stream) {
    SPCONV_REQUIRE(num_tensors >= 0, SPCONV_ERR_ARG, "num_tensors must be >= 0");
    SPCONV_REQUIRE(norm_kind == SPCONV_CLIP_P2 || norm_kind == SPCONV_CLIP_INF, SPCONV_ERR_ARG,
                   "unknown norm kind %d", norm_kind);
    SPCONV_REQUIRE(max_norm >= 0.f, SPCONV_ERR_ARG, "max_norm must be >= 0");
    SPCONV_REQUIRE(total_norm != nullptr, SPCONV_ERR_ARG, "null pointer argument");
    const cudaStream_t st = (cudaStream_t)stream;
    try {
        std::vector<int> live;
        std::vector<ClRange> in, out;
        live.reserve(num_tensors);
        in.reserve(num_tensors);
        out.reserve(num_tensors);
        for (int i = 0; i < num_tensors; ++i) {
            SPCONV_REQUIRE(grads && outs && numels && dtypes, SPCONV_ERR_ARG, "null pointer argument");
            SPCONV_REQUIRE(dtypes[i] == SPCONV_F32 || dtypes[i] == SPCONV_F16 || dtypes[i] == SPCONV_BF16,
                           SPCONV_ERR_ARG, "tensor %d: unsupported dtype code %d", i, dtypes[i]);
            SPCONV_REQUIRE(numels[i] >= 0, SPCONV_ERR_ARG, "tensor %d: negative size", i);
            if (numels[i] == 0) continue;
            SPCONV_REQUIRE(grads[i] && outs[i], SPCONV_ERR_ARG, "tensor %d: null pointer", i);
            const uintptr_t bytes = (uintptr_t)numels[i] * (dtypes[i] == SPCONV_F32 ? 4 : 2);
            live.push_back(i);
            in.push_back({(uintptr_t)grads[i], (uintptr_t)grads[i] + bytes, i});
            out.push_back({(uintptr_t)outs[i], (uintptr_t)outs[i] + bytes, i});
        }
        // Blocks write in no given order, so no output may share memory with another output, or
        // with a gradient other than its own at the same place.
        std::sort(in.begin(), in.end());
        std::sort(out.begin(), out.end());
        for (size_t i = 1; i < out.size(); ++i)
            SPCONV_REQUIRE(out[i].lo >= out[i - 1].hi, SPCONV_ERR_ARG, "tensors %d and %d overlap",
                           out[i - 1].tensor, out[i].tensor);
        uintptr_t reach = 0;                 // the furthest end of a gradient that begins before the output
        int reach_of = -1;
        size_t j = 0;
        auto pass = [&] {
            if (in[j].hi > reach) {
                reach = in[j].hi;
                reach_of = in[j].tensor;
            }
            ++j;
        };
        for (const ClRange &o : out) {
            while (j < in.size() && in[j].lo < o.lo) pass();
            SPCONV_REQUIRE(reach <= o.lo, SPCONV_ERR_ARG, "output %d overlaps gradient %d", o.tensor, reach_of);
            while (j < in.size() && in[j].lo < o.hi) {        // begins inside the output
                SPCONV_REQUIRE(in[j].tensor == o.tensor && in[j].lo == o.lo, SPCONV_ERR_ARG,
                               "output %d overlaps gradient %d", o.tensor, in[j].tensor);
                pass();
            }
        }
        if (live.empty()) {
            if (cudaMemsetAsync(total_norm, 0, sizeof(float), st) != cudaSuccess) return check_launch("clip: clear");
            return SPCONV_OK;
        }
        SPCONV_REQUIRE(workspace && ((uintptr_t)workspace & 7) == 0 &&
                           workspace_bytes >= spconv_clip_gradients_workspace_bytes(num_tensors),
                       SPCONV_ERR_ARG, "workspace missing, misaligned or too small");
        ClArgs a = {};
        a.partial = (double *)workspace;
        a.max_norm_kind = norm_kind == SPCONV_CLIP_INF;
        a.max_norm = max_norm;
        a.total = total_norm;
        // a small list in a small parameter block: less to send with each launch
        if ((int)live.size() <= kClSmall) return cl_run<kClSmall>(grads, outs, numels, dtypes, live, a, st);
        return cl_run<kClLarge>(grads, outs, numels, dtypes, live, a, st);
    } catch (const std::exception &e) {
        set_error("clip: %s", e.what());
        return SPCONV_ERR_ARG;
    }
}
