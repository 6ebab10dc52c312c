// Interface between attention's entry points (attention.cu) and its kernels.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace spconv {

// A tensor [rows, heads, size] whose heads' values are contiguous; strides in elements.
struct AtTensor {
    const void *p;
    int64_t row, head;
};

struct AtArgs {
    AtTensor q, k, v, grad;
    void *out, *gq, *gk, *gv;            // contiguous
    const void *out_in;                  // the backward's: the forward's output, contiguous
    void *rest;                          // what out's rounding left out, or null
    float *lse;                          // [num_queries, heads]: log2 of the row's sum, + inf where it sees no key
    float *delta;                        // [num_queries, heads]: grad . out
    float *peaks;                        // fp16 gradients: [samples, 2] largest squares of a row of grad, and of v; else null
    float *squares;                      // [num_queries, heads], of grad's rows
    const int32_t *offsets, *key_offsets;
    int B, M, N;                         // samples, query rows, key rows
    int H, K, D;                         // heads, key heads, head size
    int causal;
    float scale, c;                      // c = scale * log2(e)
    // split s of a sample's keys (or, for the keys' gradients, queries): fp32 results of its own, joined afterwards
    int splits;
    float *partial;                      // [splits, M, H, D]; the keys' gradients [splits, 2, N, K, D]
    float2 *part_ml;                     // forward: [splits, M, H] (largest score * c, sum; -1: no key seen)
    int32_t *status;
    uint64_t wait_ns;
    int dtype;
    cudaStream_t stream;
};

// Rows of a tile, whichever kernel: samples' tiles are numbered from offsets[b] / rows + b.
inline int64_t at_tiles(int64_t rows, int64_t samples, int per_tile) { return rows / per_tile + samples; }

// CUDA cores, any type and size up to 256.
int launch_at_simt_forward(const AtArgs &a);
int launch_at_simt_grad_query(const AtArgs &a);
int launch_at_simt_grad_key(const AtArgs &a);
int at_simt_rows(int D);                 // rows (and keys) of a tile

// Tensor cores (fp16, bf16; sizes up to 128, whose rows and heads lie whole multiples of 16 bytes apart: the size itself is any).
int launch_at_tc_forward(const AtArgs &a, bool pair);        // pair: of tiles of 128 rows a CTA, not one (sizes over 64)
int launch_at_tc_grad_query(const AtArgs &a);
int launch_at_tc_grad_key(const AtArgs &a);

}  // namespace spconv
