// Pointwise linear layer over voxel features and its gradients:
//
//   out = residual + act(z),  z = feats W^T + bias          feats [M, Ci], W [Co, Ci]
//   dz = grad_out * act'(z);  grad_feats = dz W;  grad_W = dz^T feats;  grad_bias = sum dz
//
// This file holds the CUDA-core product (exact fp32 FMAs; fp32 features, odd channel counts,
// unaligned pointers), the activation's backward with the bias sums, the sum over splits, and
// the entry points.
#include <algorithm>
#include <type_traits>

#include "activation.cuh"
#include "common.cuh"
#include "linear_internal.h"

namespace spconv {

constexpr int kSimtThreads = 256, kSimtBK = 16;

// Reads rows x BK elements of an operand (K contiguous unless T_) into registers and stores them
// as [k][row] fp32 in shared memory.
template <typename T, int ROWS, bool T_>
struct SimtTile {
    static constexpr int kPer = (ROWS * kSimtBK + kSimtThreads - 1) / kSimtThreads;
    float v[kPer];
    __device__ __forceinline__ static void place(int i, int &row, int &k) {
        if constexpr (T_) { row = i % ROWS; k = i / ROWS; }       // neighbours along the rows
        else { k = i % kSimtBK; row = i / kSimtBK; }              // neighbours along K
    }
    __device__ __forceinline__ void load(const T *p, int64_t rows, int64_t row0, int64_t k0, int64_t k_end, int64_t ld) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = threadIdx.x + j * kSimtThreads;
            int r, k;
            place(i, r, k);
            v[j] = 0.f;
            if (i < ROWS * kSimtBK && row0 + r < rows && k0 + k < k_end)
                v[j] = dtype_traits<T>::to_f(T_ ? p[(k0 + k) * ld + row0 + r] : p[(row0 + r) * ld + k0 + k]);
        }
    }
    __device__ __forceinline__ void store(float (*s)[ROWS + 4]) const {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = threadIdx.x + j * kSimtThreads;
            int r, k;
            place(i, r, k);
            if (i < ROWS * kSimtBK) s[k][r] = v[j];
        }
    }
};

// out[m, n] = epilogue(sum_k A(m, k) B(n, k)): BM x BN outputs per block, TM x TN per thread,
// K in steps of 16 through two shared-memory buffers; the next step's global loads run under
// the current step's FMAs. blockIdx.z is the split of K.
template <typename T, int BM, int BN, int TM, int TN, bool AT, bool BT, int ACT>
__global__ void __launch_bounds__(kSimtThreads)
linear_simt_kernel(GemmArgs g) {
    static_assert(BM * BN == TM * TN * kSimtThreads, "threads cover the tile");
    __shared__ float sa[2][kSimtBK][BM + 4], sb[2][kSimtBK][BN + 4];
    const T *a = (const T *)g.a, *b = (const T *)g.b;
    const int64_t m0 = (int64_t)blockIdx.x * BM, n0 = (int64_t)blockIdx.y * BN;
    const int64_t k_begin = g.splits > 1 ? blockIdx.z * g.k_per_split : 0;
    const int64_t k_end = g.splits > 1 ? min(g.K, k_begin + g.k_per_split) : g.K;
    const int64_t lda = AT ? g.M : g.K, ldb = BT ? g.N : g.K;
    const int tn = threadIdx.x % (BN / TN), tm = threadIdx.x / (BN / TN);
    // A thread's columns: fours, BN / 2 apart where it has eight, so that a quarter-warp's 16-byte reads
    // of B fall on different banks.
    auto col = [&](int j) { return TN <= 4 ? tn * TN + j : (j / 4) * (BN / 2) + tn * 4 + j % 4; };
    float acc[TM][TN] = {};
    SimtTile<T, BM, AT> ta;
    SimtTile<T, BN, BT> tb;
    ta.load(a, g.M, m0, k_begin, k_end, lda);
    tb.load(b, g.N, n0, k_begin, k_end, ldb);
    int buf = 0;
    for (int64_t k = k_begin; k < k_end; k += kSimtBK, buf ^= 1) {
        ta.store(sa[buf]);
        tb.store(sb[buf]);
        __syncthreads();
        if (k + kSimtBK < k_end) {
            ta.load(a, g.M, m0, k + kSimtBK, k_end, lda);
            tb.load(b, g.N, n0, k + kSimtBK, k_end, ldb);
        }
#pragma unroll
        for (int kk = 0; kk < kSimtBK; ++kk) {
            float fa[TM], fb[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[i] = sa[buf][kk][tm * TM + i];
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[j] = sb[buf][kk][col(j)];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = fmaf(fa[i], fb[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t m = m0 + tm * TM + i;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int64_t n = n0 + col(j);
            if (n >= g.N) continue;
            const int64_t at = m * g.N + n;
            float z = acc[i][j];
            if (g.partial) {
                g.partial[(int64_t)blockIdx.z * g.M * g.N + at] = z;
                continue;
            }
            if (g.bias) z += sizeof(T) == 2 && g.bias_f32 ? ((const float *)g.bias)[n] : dtype_traits<T>::to_f(((const T *)g.bias)[n]);
            if (g.preact) ((T *)g.preact)[at] = dtype_traits<T>::from_f(z);
            z = act_value<ACT>(z);
            if (g.residual) z += dtype_traits<T>::to_f(((const T *)g.residual)[at]);
            ((T *)g.out)[at] = dtype_traits<T>::from_f(z);
        }
    }
}

template <typename T, bool AT, bool BT, int ACT>
static int simt_shape(const GemmArgs &g) {
    auto run = [&](auto kern, int bm, int bn) {
        const int64_t gx = (g.M + bm - 1) / bm, gy = (g.N + bn - 1) / bn;
        kern<<<dim3((unsigned)gx, (unsigned)gy, (unsigned)g.splits), kSimtThreads, 0, g.stream>>>(g);
        return check_launch("linear_simt_kernel");
    };
    // narrow outputs (class scores) leave three quarters of a 64-wide tile idle
    if (g.N <= 16) return run(linear_simt_kernel<T, 128, 16, 4, 2, AT, BT, ACT>, 128, 16);
    if (g.M <= 16) return run(linear_simt_kernel<T, 16, 128, 2, 4, AT, BT, ACT>, 16, 128);
    // 128 columns where there are that many and the tiles still fill the SMs: a quarter fewer reads of
    // shared memory for each product
    if (g.N > 64 && (g.M + 127) / 128 * ((g.N + 127) / 128) * g.splits >= 148)
        return run(linear_simt_kernel<T, 128, 128, 8, 8, AT, BT, ACT>, 128, 128);
    return run(linear_simt_kernel<T, 128, 64, 8, 4, AT, BT, ACT>, 128, 64);
}

template <typename T>
static int simt_type(const GemmArgs &g) {
    if (g.a_t) return simt_shape<T, true, true, SPCONV_ACT_NONE>(g);       // weight gradient
    if (g.b_t) return simt_shape<T, false, true, SPCONV_ACT_NONE>(g);      // input gradient
    return act_dispatch(g.activation, [&](auto act) { return simt_shape<T, false, false, act.value>(g); });
}

int launch_gemm_simt(const GemmArgs &g) {
    if (g.dtype == SPCONV_F32) return simt_type<float>(g);
    if (g.dtype == SPCONV_F16) return simt_type<__half>(g);
    return simt_type<__nv_bfloat16>(g);
}

// ---------------------------------------------------------------------------------------
// dz = grad_out * act'(z), rounded to the features' type as the products' operand (half the bytes of
// fp32, and what the tensor cores take; see linear_bwd_tc.cu for what it costs), and its column sums,
// of dz before the rounding. One read of each input, one write of dz; a lane owns VEC neighbouring
// columns of a 32 * VEC column tile and walks the chunk's rows, so the sums stay in registers;
// partial[chunk][Co] holds them per block.
// ---------------------------------------------------------------------------------------
constexpr int kDactThreads = 256;

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kDactThreads)
linear_dact_kernel(const T *__restrict__ gout, const T *__restrict__ z, T *__restrict__ dz, float *__restrict__ partial,
                   int64_t M, int Co, int lpr, int64_t chunk) {
    __shared__ float part[kDactThreads / 32][32 * VEC];
    const int lane = threadIdx.x & (lpr - 1), group = threadIdx.x / lpr, groups = kDactThreads / lpr;
    const int col = (blockIdx.y * 32 + lane) * VEC;
    const bool have = col < Co;
    const int64_t row0 = (int64_t)blockIdx.x * chunk, row1 = min(M, row0 + chunk);
    float acc[VEC] = {};
    if (have) {
#pragma unroll 4
        for (int64_t r = row0 + group; r < row1; r += groups) {
            const int64_t at = r * Co + col;
            alignas(16) T gv[VEC], zv[VEC];
            if constexpr (VEC > 1) {
                *reinterpret_cast<uint4 *>(gv) = __ldg(reinterpret_cast<const uint4 *>(gout + at));
                if constexpr (ACT != SPCONV_ACT_NONE) *reinterpret_cast<uint4 *>(zv) = __ldcs(reinterpret_cast<const uint4 *>(z + at));
            } else {
                gv[0] = gout[at];
                if constexpr (ACT != SPCONV_ACT_NONE) zv[0] = z[at];
            }
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                float d[2] = {dtype_traits<T>::to_f(gv[i]), VEC > 1 ? dtype_traits<T>::to_f(gv[i + (VEC > 1)]) : 0.f};
                if constexpr (ACT != SPCONV_ACT_NONE) {
                    const float z0 = dtype_traits<T>::to_f(zv[i]), z1 = VEC > 1 ? dtype_traits<T>::to_f(zv[i + (VEC > 1)]) : 0.f;
                    const float2 slope = sizeof(T) == 2 ? act_slope2<ACT>(make_float2(z0, z1))
                                                        : make_float2(act_slope<ACT>(z0), act_slope<ACT>(z1));
                    d[0] *= slope.x;
                    d[1] *= slope.y;
                }
#pragma unroll
                for (int k = 0; k < (VEC > 1 ? 2 : 1); ++k) {
                    acc[i + k] += d[k];      // the bias sums take dz before it is rounded
                    if constexpr (ACT != SPCONV_ACT_NONE) gv[i + k] = dtype_traits<T>::from_f(d[k]);
                }
            }
            if constexpr (ACT != SPCONV_ACT_NONE) {
                if constexpr (VEC > 1) *reinterpret_cast<uint4 *>(dz + at) = *reinterpret_cast<uint4 *>(gv);
                else dz[at] = gv[0];
            }
        }
    }
    if (!partial) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        for (int o = lpr; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if ((threadIdx.x & 31) < lpr) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[threadIdx.x >> 5][lane * VEC + i] = acc[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < lpr * VEC; i += kDactThreads) {
        const int c = blockIdx.y * 32 * VEC + i;
        if (c >= Co) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kDactThreads / 32; ++w) v += part[w][i];
        partial[(int64_t)blockIdx.x * Co + c] = v;
    }
}

// out[i] = sum over s of partial[s][i], in the order of s within 16 lanes of splits; two arrays in one
// launch (a weight's and a bias's sums).
struct ReduceSeg {
    const float *partial;
    int splits;
    int64_t n;
    void *out;
    int dtype;
    int blocks;
};

__global__ void __launch_bounds__(512)
linear_reduce_kernel(const ReduceSeg a, const ReduceSeg b) {
    __shared__ float part[16][33];
    const bool second = (int)blockIdx.x >= a.blocks;
    const ReduceSeg &g = second ? b : a;
    const int64_t i = (int64_t)(blockIdx.x - (second ? a.blocks : 0)) * 32 + threadIdx.x;
    grid_dependency_wait();
    float v = 0.f;
    if (i < g.n) {
#pragma unroll 4
        for (int s = threadIdx.y; s < g.splits; s += 16) v += __ldcs(g.partial + (int64_t)s * g.n + i);
    }
    part[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && i < g.n) {
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < 16; ++y) sum += part[y][threadIdx.x];
        if (g.dtype == SPCONV_F32) ((float *)g.out)[i] = sum;
        else if (g.dtype == SPCONV_F16) ((__half *)g.out)[i] = __float2half_rn(sum);
        else ((__nv_bfloat16 *)g.out)[i] = __float2bfloat16_rn(sum);
    }
}

static ReduceSeg reduce_seg(const float *partial, int splits, int64_t n, int dtype, void *out) {
    return {partial, splits, n, out, dtype, out ? (int)((n + 31) / 32) : 0};
}

static int launch_reduce(const ReduceSeg &a, const ReduceSeg &b, cudaStream_t st) {
    if (a.blocks + b.blocks == 0) return SPCONV_OK;
    launch_pdl(linear_reduce_kernel, dim3((unsigned)(a.blocks + b.blocks)), dim3(32, 16), 0, st, a, b);
    return check_launch("linear_reduce_kernel");
}

// Row chunks of the dz / bias pass: about four blocks per SM, at least 32 rows each.
static int dact_chunks(int64_t M) { return (int)std::max<int64_t>(1, std::min<int64_t>(148 * 4, (M + 31) / 32)); }

template <typename T, int VEC>
static int dact_vec(const void *gout, const void *z, void *dz, float *partial, int64_t M, int Co, int activation,
                    cudaStream_t st) {
    const int vecs = (Co + VEC - 1) / VEC;
    int lpr = 1;
    while (lpr < vecs && lpr < 32) lpr <<= 1;
    const int chunks = dact_chunks(M);
    const dim3 grid(chunks, (vecs + 31) / 32);
    const int64_t chunk = (M + chunks - 1) / chunks;
    return act_dispatch(activation, [&](auto act) {
        linear_dact_kernel<T, VEC, act.value><<<grid, kDactThreads, 0, st>>>((const T *)gout, (const T *)z, (T *)dz,
                                                                            partial, M, Co, lpr, chunk);
        return check_launch("linear_dact_kernel");
    });
}

template <typename T>
static int dact_type(const void *gout, const void *z, void *dz, float *partial, int64_t M, int Co, int activation,
                     cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = Co % V == 0 && (((uintptr_t)gout | (uintptr_t)z | (uintptr_t)dz) & 15) == 0;
    return vec ? dact_vec<T, V>(gout, z, dz, partial, M, Co, activation, st)
               : dact_vec<T, 1>(gout, z, dz, partial, M, Co, activation, st);
}

static int launch_dact(int dtype, const void *gout, const void *z, void *dz, float *partial, int64_t M, int Co,
                       int activation, cudaStream_t st) {
    if (dtype == SPCONV_F32) return dact_type<float>(gout, z, dz, partial, M, Co, activation, st);
    if (dtype == SPCONV_F16) return dact_type<__half>(gout, z, dz, partial, M, Co, activation, st);
    return dact_type<__nv_bfloat16>(gout, z, dz, partial, M, Co, activation, st);
}

// Splits of the weight gradient's sum over the rows: enough blocks for four per SM, at least 256
// rows each.
static int wgrad_splits(int64_t M, int Ci, int Co) {
    const int64_t tiles = Ci <= 16 ? (Co + 127) / 128 : Co <= 16 ? (Ci + 127) / 128 : (int64_t)((Co + 127) / 128) * ((Ci + 63) / 64);
    return (int)std::max<int64_t>(1, std::min<int64_t>((148 * 4 + tiles - 1) / tiles, (M + 255) / 256));
}

static int64_t pad256(int64_t n) { return (n + 255) & ~(int64_t)255; }
static int64_t elt(int dtype) { return dtype == SPCONV_F32 ? 4 : 2; }

static int check_linear(int dtype, int64_t M, int Ci, int Co, int activation, int kernel_choice) {
    SPCONV_REQUIRE(dtype == SPCONV_F32 || dtype == SPCONV_F16 || dtype == SPCONV_BF16, SPCONV_ERR_ARG,
                   "unsupported dtype code %d", dtype);
    SPCONV_REQUIRE(M >= 0 && M < ((int64_t)1 << 31), SPCONV_ERR_ARG, "rows must be in [0, 2^31)");
    SPCONV_REQUIRE(Ci >= 1 && Ci <= 65536 && Co >= 1 && Co <= 65536, SPCONV_ERR_ARG,
                   "channels must be in [1, 65536], got %d and %d", Ci, Co);
    SPCONV_REQUIRE(activation >= SPCONV_ACT_NONE && activation <= SPCONV_ACT_SILU, SPCONV_ERR_ARG,
                   "unknown activation %d", activation);
    SPCONV_REQUIRE(kernel_choice >= SPCONV_KERNEL_AUTO && kernel_choice <= SPCONV_KERNEL_TCGEN05, SPCONV_ERR_ARG,
                   "unknown kernel choice %d", kernel_choice);
    return SPCONV_OK;
}

static int launch_gemm(const GemmArgs &g, int kernel_choice) {
    if (kernel_choice != SPCONV_KERNEL_SIMT && gemm_tc_supported(g)) return launch_gemm_tc(g);
    SPCONV_REQUIRE(kernel_choice != SPCONV_KERNEL_TCGEN05, SPCONV_ERR_UNSUPPORTED,
                   "the tensor-core kernel needs fp16 or bf16, channels in eights and 16-byte aligned tensors");
    return launch_gemm_simt(g);
}

// ---------------------------------------------------------------------------------------
// Channel counts that are no multiple of 8, 16-bit: TMA needs rows a multiple of 16 bytes apart, so the
// operands are copied into rows of whole eights (zeros behind) and the results out of such rows,
// where the tensor cores then save more than the copies cost: about 15 TFLOP/s of the CUDA-core kernel
// at such widths against 4 TB/s of copying and 15 us of launches. Measured in bf16, forward and
// backward, CUDA cores and here: 15,000 x 1001 -> 517 625 and 76, 1558 and 191 us; 20,000 x 257 -> 131 91
// and 41, 251 and 87 us.
// ---------------------------------------------------------------------------------------
static int up8(int c) { return (c + 7) & ~7; }

bool linear_padded(int dtype, int64_t M, int Ci, int Co) {
    if ((dtype != SPCONV_F16 && dtype != SPCONV_BF16) || (Ci % 8 == 0 && Co % 8 == 0)) return false;
    const double cuda_cores = 2.0 * Ci * Co / 15e12, copies = (4.0 * up8(Ci) + 6.0 * up8(Co)) / 4e12;
    return M * (cuda_cores - copies) > 15e-6;
}

// dst [rows, dst_cols] = src [rows, src_cols] of 16-bit (or 32-bit) values, cut off or with zeros behind.
template <typename V>
__global__ void __launch_bounds__(256)
linear_repitch_kernel(const V *__restrict__ src, int src_cols, V *__restrict__ dst, int dst_cols, int64_t rows) {
    const int64_t n = rows * dst_cols, step = (int64_t)gridDim.x * blockDim.x;
    int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    int64_t r = i / dst_cols;
    int c = (int)(i - r * dst_cols);
    const int64_t dr = step / dst_cols;
    const int dc = (int)(step - dr * dst_cols);
    for (; i < n; i += step) {
        dst[i] = c < src_cols ? src[r * src_cols + c] : V(0);
        r += dr;
        c += dc;
        if (c >= dst_cols) {
            c -= dst_cols;
            ++r;
        }
    }
}

static int launch_repitch(const void *src, int src_cols, void *dst, int dst_cols, int64_t rows, int bytes, cudaStream_t st) {
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(148 * 16, (rows * dst_cols + 1023) / 1024));
    if (bytes == 2) linear_repitch_kernel<uint16_t><<<grid, 256, 0, st>>>((const uint16_t *)src, src_cols, (uint16_t *)dst, dst_cols, rows);
    else linear_repitch_kernel<uint32_t><<<grid, 256, 0, st>>>((const uint32_t *)src, src_cols, (uint32_t *)dst, dst_cols, rows);
    return check_launch("linear_repitch_kernel");
}

static int64_t padded_forward_bytes(int64_t M, int Ci, int Co, bool residual, bool preact) {
    const int64_t pi = up8(Ci), po = up8(Co);
    return pad256(M * pi * 2) + pad256(po * pi * 2) + pad256(po * 4) + (1 + (residual ? 1 : 0) + (preact ? 1 : 0)) * pad256(M * po * 2);
}

static int64_t separate_backward_bytes(int dtype, int64_t M, int Ci, int Co, int activation) {
    const int64_t separate = pad256(activation == SPCONV_ACT_NONE ? 0 : M * Co * elt(dtype)) + pad256((int64_t)dact_chunks(M) * Co * 4) +
                             pad256((int64_t)std::max(wgrad_splits(M, Ci, Co), gemm_tc_splits(Co, Ci, M)) * Co * Ci * 4);
    // the one pass over the rows keeps sums of every CTA; tensors off 16-byte boundaries take the separate kernels
    if (!bwd_tc_shape(dtype, M, Ci, Co, activation)) return separate;
    const int64_t grid = bwd_tc_grid(M);
    return std::max(separate, pad256(grid * 8 * Co * 4) + pad256(grid * Co * Ci * 4));
}

static int64_t padded_backward_bytes(int dtype, int64_t M, int Ci, int Co, int activation) {
    const int64_t pi = up8(Ci), po = up8(Co);
    return 2 * pad256(M * pi * 2) + 2 * pad256(M * po * 2) + pad256(po * pi * 2) + pad256(po * pi * 4) + pad256(po * 4) +
           separate_backward_bytes(dtype, M, (int)pi, (int)po, activation);
}

static int linear_forward(const void *feats, int dtype, int64_t M, int Ci, const void *weight, const void *bias,
                          int bias_dtype, const void *residual, int Co, int activation, void *out, void *preact, int kernel_choice,
                          int32_t *status, cudaStream_t st) {
    GemmArgs g = {};
    g.a = feats;
    g.b = weight;
    g.dtype = dtype;
    g.M = M;
    g.N = Co;
    g.K = Ci;
    g.bias = bias;
    g.bias_f32 = bias && bias_dtype == SPCONV_F32;
    g.residual = residual;
    g.activation = activation;
    g.out = out;
    g.preact = preact;
    g.splits = 1;
    g.status = status;
    g.stream = st;
    return launch_gemm(g, kernel_choice);
}

static int linear_backward(const void *grad_out, const void *preact, const void *feats, const void *weight, int dtype,
                           int64_t M, int Ci, int Co, int activation, void *grad_feats, void *grad_weight,
                           int weight_dtype, void *grad_bias, int bias_dtype, void *workspace, int kernel_choice,
                           int32_t *status, cudaStream_t st) {
    uint8_t *ws = (uint8_t *)workspace;
    bool aligned = true;
    for (const void *p : {grad_out, preact, feats, weight, (const void *)grad_feats})
        aligned = aligned && ((uintptr_t)p & 15) == 0;
    if (kernel_choice != SPCONV_KERNEL_SIMT && aligned && bwd_tc_shape(dtype, M, Ci, Co, activation)) {
        const int grid = bwd_tc_grid(M);
        BwdArgs q = {grad_out, preact, feats, weight, dtype, M, Ci, Co, activation, grad_feats, nullptr, nullptr, status, st};
        if (grad_bias) q.b_partial = (float *)ws;
        if (grad_weight) q.w_partial = (float *)(ws + pad256((int64_t)grid * 8 * Co * 4));
        if (const int rc = launch_bwd_tc(q)) return rc;
        return launch_reduce(reduce_seg(q.w_partial, grid, (int64_t)Co * Ci, weight_dtype, grad_weight),
                             reduce_seg(q.b_partial, grid * 8, Co, bias_dtype, grad_bias), st);
    }
    const void *dz = grad_out;
    if (activation != SPCONV_ACT_NONE) {
        dz = ws;
        ws += pad256(M * Co * elt(dtype));
    }
    float *bias_part = (float *)ws;
    ws += pad256((int64_t)dact_chunks(M) * Co * 4);
    float *weight_part = (float *)ws;
    if (activation != SPCONV_ACT_NONE || grad_bias) {
        if (const int rc = launch_dact(dtype, grad_out, preact, activation != SPCONV_ACT_NONE ? (void *)dz : nullptr,
                                       grad_bias ? bias_part : nullptr, M, Co, activation, st))
            return rc;
    }
    GemmArgs g = {};
    g.dtype = dtype;
    g.splits = 1;
    g.status = status;
    g.stream = st;
    g.a = dz;
    if (grad_feats) {
        g.b = weight;
        g.b_t = true;
        g.M = M;
        g.N = Ci;
        g.K = Co;
        g.out = grad_feats;
        if (const int rc = launch_gemm(g, kernel_choice)) return rc;
    }
    if (grad_weight) {
        g.a_t = g.b_t = true;
        g.b = feats;
        g.M = Co;
        g.N = Ci;
        g.K = M;
        g.out = nullptr;
        g.partial = weight_part;
        const bool tc = kernel_choice != SPCONV_KERNEL_SIMT && gemm_tc_supported(g);
        g.splits = tc ? gemm_tc_splits(Co, Ci, M) : wgrad_splits(M, Ci, Co);
        const int64_t step = tc ? 64 : 1;    // the tensor-core kernel's K step
        g.k_per_split = ((M + g.splits - 1) / g.splits + step - 1) / step * step;
        g.splits = (int)((M + g.k_per_split - 1) / g.k_per_split);
        if (const int rc = launch_gemm(g, kernel_choice)) return rc;
    }
    return launch_reduce(reduce_seg(weight_part, g.splits, (int64_t)Co * Ci, weight_dtype, grad_weight),
                         reduce_seg(bias_part, dact_chunks(M), Co, bias_dtype, grad_bias), st);
}

}  // namespace spconv

using namespace spconv;

extern "C" int64_t spconv_linear_forward_workspace_bytes(int dtype, int64_t M, int Ci, int Co, int has_residual,
                                                         int has_preact) {
    if (check_linear(dtype, M, Ci, Co, SPCONV_ACT_NONE, SPCONV_KERNEL_AUTO) != SPCONV_OK) return -1;
    return linear_padded(dtype, M, Ci, Co) ? padded_forward_bytes(M, Ci, Co, has_residual != 0, has_preact != 0) : 0;
}

extern "C" int spconv_linear_forward(const void *feats, int dtype, int64_t M, int Ci, const void *weight,
                                     const void *bias, const void *residual, int Co, int activation, void *out,
                                     void *preact, void *workspace, int64_t workspace_bytes, int kernel_choice,
                                     int32_t *status, void *stream) {
    return spconv_linear_forward_ex(feats, dtype, M, Ci, weight, bias, dtype, residual, Co, activation, out, preact,
                                    workspace, workspace_bytes, kernel_choice, status, stream);
}

extern "C" int spconv_linear_forward_ex(const void *feats, int dtype, int64_t M, int Ci, const void *weight,
                                        const void *bias, int bias_dtype, const void *residual, int Co, int activation,
                                        void *out, void *preact, void *workspace, int64_t workspace_bytes,
                                        int kernel_choice, int32_t *status, void *stream) {
    if (const int rc = check_linear(dtype, M, Ci, Co, activation, kernel_choice)) return rc;
    SPCONV_REQUIRE(!bias || bias_dtype == SPCONV_F32 || bias_dtype == dtype, SPCONV_ERR_ARG,
                   "the bias is fp32 or of the features' type");
    if (M == 0) return SPCONV_OK;
    SPCONV_REQUIRE(feats && weight && out, SPCONV_ERR_ARG, "null pointer argument");
    const cudaStream_t st = (cudaStream_t)stream;
    // without the workspace the CUDA-core kernel takes such shapes too
    if (kernel_choice != SPCONV_KERNEL_AUTO || !workspace || !linear_padded(dtype, M, Ci, Co))
        return linear_forward(feats, dtype, M, Ci, weight, bias, bias_dtype, residual, Co, activation, out, preact, kernel_choice, status, st);
    SPCONV_REQUIRE(((uintptr_t)workspace & 255) == 0 &&
                       workspace_bytes >= padded_forward_bytes(M, Ci, Co, residual != nullptr, preact != nullptr),
                   SPCONV_ERR_ARG, "workspace misaligned or too small");
    const int pi = up8(Ci), po = up8(Co);
    uint8_t *ws = (uint8_t *)workspace;
    auto take = [&](int64_t bytes) {
        void *p = ws;
        ws += pad256(bytes);
        return p;
    };
    void *x = take(M * pi * 2), *w = take((int64_t)po * pi * 2), *b = take(po * 4), *y = take(M * po * 2);
    void *r = residual ? take(M * po * 2) : nullptr, *z = preact ? take(M * po * 2) : nullptr;
    int rc = launch_repitch(feats, Ci, x, pi, M, 2, st);
    if (!rc) rc = launch_repitch(weight, Ci, w, pi, Co, 2, st);
    if (!rc && po > Co && cudaMemsetAsync((uint8_t *)w + (int64_t)Co * pi * 2, 0, (size_t)(po - Co) * pi * 2, st) != cudaSuccess)
        rc = check_launch("linear_forward: clear");
    if (!rc && bias) rc = launch_repitch(bias, Co, b, po, 1, (int)elt(bias_dtype), st);
    if (!rc && residual) rc = launch_repitch(residual, Co, r, po, M, 2, st);
    if (!rc) rc = linear_forward(x, dtype, M, pi, w, bias ? b : nullptr, bias_dtype, r, po, activation, y, z, kernel_choice, status, st);
    if (!rc) rc = launch_repitch(y, po, out, Co, M, 2, st);
    if (!rc && preact) rc = launch_repitch(z, po, preact, Co, M, 2, st);
    return rc;
}

extern "C" int64_t spconv_linear_backward_workspace_bytes(int dtype, int64_t M, int Ci, int Co, int activation) {
    if (check_linear(dtype, M, Ci, Co, activation, SPCONV_KERNEL_AUTO) != SPCONV_OK) return -1;
    return linear_padded(dtype, M, Ci, Co) ? padded_backward_bytes(dtype, M, Ci, Co, activation)
                                           : separate_backward_bytes(dtype, M, Ci, Co, activation);
}

extern "C" int spconv_linear_backward(const void *grad_out, const void *preact, const void *feats, const void *weight,
                                      int dtype, int64_t M, int Ci, int Co, int activation, void *grad_feats,
                                      void *grad_weight, int weight_dtype, void *grad_bias, int bias_dtype,
                                      void *workspace, int64_t workspace_bytes, int kernel_choice, int32_t *status,
                                      void *stream) {
    if (const int rc = check_linear(dtype, M, Ci, Co, activation, kernel_choice)) return rc;
    SPCONV_REQUIRE(!grad_weight || weight_dtype == SPCONV_F32 || weight_dtype == dtype, SPCONV_ERR_ARG,
                   "the weight's gradient is fp32 or of the features' type");
    SPCONV_REQUIRE(!grad_bias || bias_dtype == SPCONV_F32 || bias_dtype == dtype, SPCONV_ERR_ARG,
                   "the bias's gradient is fp32 or of the features' type");
    const cudaStream_t st = (cudaStream_t)stream;
    if (M == 0) {                            // sums over no rows
        if (grad_weight && cudaMemsetAsync(grad_weight, 0, (size_t)Co * Ci * elt(weight_dtype), st) != cudaSuccess)
            return check_launch("linear_backward: clear");
        if (grad_bias && cudaMemsetAsync(grad_bias, 0, (size_t)Co * elt(bias_dtype), st) != cudaSuccess)
            return check_launch("linear_backward: clear");
        return SPCONV_OK;
    }
    SPCONV_REQUIRE(grad_out && (preact || activation == SPCONV_ACT_NONE) && (feats || !grad_weight) &&
                       (weight || !grad_feats), SPCONV_ERR_ARG, "null pointer argument");
    SPCONV_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0 &&
                       workspace_bytes >= spconv_linear_backward_workspace_bytes(dtype, M, Ci, Co, activation),
                   SPCONV_ERR_ARG, "workspace missing, misaligned or too small");
    if (activation == SPCONV_ACT_NONE) preact = nullptr;
    if (kernel_choice != SPCONV_KERNEL_AUTO || !linear_padded(dtype, M, Ci, Co))
        return linear_backward(grad_out, preact, feats, weight, dtype, M, Ci, Co, activation, grad_feats, grad_weight,
                               weight_dtype, grad_bias, bias_dtype, workspace, kernel_choice, status, st);
    const int pi = up8(Ci), po = up8(Co);
    uint8_t *ws = (uint8_t *)workspace;
    auto take = [&](int64_t bytes) {
        void *p = ws;
        ws += pad256(bytes);
        return p;
    };
    void *x = take(M * pi * 2), *gx = take(M * pi * 2), *g = take(M * po * 2), *z = take(M * po * 2);
    void *w = take((int64_t)po * pi * 2), *gw = take((int64_t)po * pi * 4), *gb = take(po * 4);
    int rc = launch_repitch(grad_out, Co, g, po, M, 2, st);
    if (!rc && preact) rc = launch_repitch(preact, Co, z, po, M, 2, st);
    if (!rc && grad_weight) rc = launch_repitch(feats, Ci, x, pi, M, 2, st);
    if (!rc && grad_feats) {                 // dz is zero in the columns past Co, W has to be finite there
        rc = launch_repitch(weight, Ci, w, pi, Co, 2, st);
        if (!rc && po > Co && cudaMemsetAsync((uint8_t *)w + (int64_t)Co * pi * 2, 0, (size_t)(po - Co) * pi * 2, st) != cudaSuccess)
            rc = check_launch("linear_backward: clear");
    }
    if (!rc)
        rc = linear_backward(g, preact ? z : nullptr, grad_weight ? x : nullptr, grad_feats ? w : nullptr, dtype, M, pi, po,
                             activation, grad_feats ? gx : nullptr, grad_weight ? gw : nullptr, weight_dtype,
                             grad_bias ? gb : nullptr, bias_dtype, ws, kernel_choice, status, st);
    if (!rc && grad_feats) rc = launch_repitch(gx, pi, grad_feats, Ci, M, 2, st);
    if (!rc && grad_weight) rc = launch_repitch(gw, pi, grad_weight, Ci, Co, (int)elt(weight_dtype), st);
    if (!rc && grad_bias) rc = launch_repitch(gb, po, grad_bias, Co, 1, (int)elt(bias_dtype), st);
    return rc;
}
