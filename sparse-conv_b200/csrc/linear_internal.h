// Interface between the pointwise linear layer's entry points (linear.cu) and its kernels.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace spconv {

// One matrix product out[m, n] = epilogue(sum_k A(m, k) * B(n, k)), fp32 accumulation.
// A is [M, K] row-major, or [K, M] if a_t; B is [N, K], or [K, N] if b_t; out [M, N].
struct GemmArgs {
    const void *a, *b;
    bool a_t, b_t;
    // There is a bias, in fp32 whatever dtype is. It stands in padding: with M, N and K eight bytes on, the CUDA-core
    // kernel was given 134 registers in place of 212 (20,000 x 512 -> 512 fp32 449 us in place of 367).
    bool bias_f32;
    int dtype;                       // of a, b, residual, preact and out
    int64_t M, N, K;
    const void *bias, *residual;     // [N], [M, N], or null
    int activation;
    void *out, *preact;              // preact: [M, N] or null
    // splits > 1: K is cut into `splits` ranges of `k_per_split`; split s writes its fp32 sums to
    // partial + s * M * N and there is no epilogue (linear_reduce adds them)
    int splits = 1;
    int64_t k_per_split = 0;
    float *partial = nullptr;
    int32_t *status = nullptr;
    cudaStream_t stream = nullptr;
};

int launch_gemm_simt(const GemmArgs &g);

// Tensor-core form (linear_tc.cu): fp16 / bf16, rows and pointers aligned for TMA. Splits need
// a_t && b_t, and k_per_split a multiple of 64.
bool gemm_tc_supported(const GemmArgs &g);
int launch_gemm_tc(const GemmArgs &g);
// Splits of K for an [M, N] sum over K.
int gemm_tc_splits(int64_t M, int64_t N, int64_t K);

// The whole backward in one pass over the rows (linear_bwd_tc.cu): grad_feats, and partial sums
// w_partial [bwd_tc_grid(M)][Co][Ci] and b_partial [8 * bwd_tc_grid(M)][Co]; each may be null.
struct BwdArgs {
    const void *grad_out, *preact, *feats, *weight;
    int dtype;
    int64_t M;
    int Ci, Co, activation;
    void *grad_feats;
    float *w_partial, *b_partial;
    int32_t *status;
    cudaStream_t stream;
};
bool bwd_tc_shape(int dtype, int64_t M, int Ci, int Co, int activation);
int bwd_tc_grid(int64_t M);
int launch_bwd_tc(const BwdArgs &q);

}  // namespace spconv
