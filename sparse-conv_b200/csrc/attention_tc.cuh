// What the tensor-core attention kernels share: tiles of 128 rows by TMA, products with an operand in TMEM, exponentials.
//
// A tile's rows are the query heads of a group that read one key head, token by token: P = the largest power of
// two that divides the group (up to 128), row r = (token r / P, head r % P). Shared keys are then read once for P
// heads, and a single token of 8 heads fills 8 rows of a tile, not one row of 8 tiles.
#pragma once

#include "activation.cuh"
#include "attention_common.cuh"
#include "linear_epilogue.cuh"
#include "tensor_map.h"

namespace spconv {

constexpr int kAtRows = 128;                         // rows of a tile, and keys
constexpr int kAtBlock = kAtRows * 128;              // 16 KB: 128 rows of 64 values, 128-byte swizzle

// One box of a 3-D tensor (value, head, row).
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void *tmap, int x, int y, int z, uint32_t mbar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];\n"
        :: "r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(mbar) : "memory");
}
// D[tmem] (+)= A[tmem, 128 rows of 16-bit pairs] * B[smem desc]^T.
__device__ __forceinline__ void tc_mma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
        :: "r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 consecutive columns of the lane's row; tc_wait_st before others rely on it.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
           "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
           "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}

// A tile in shared memory: DP / 64 blocks of 128 rows x 64 values. As an operand along the head (K-major) ...
__device__ __forceinline__ uint64_t at_desc_k(uint32_t saddr) { return smem_desc_kmajor_swizzled(saddr, 128); }
// ... and along the rows (MN-major): a step of 16 rows is 2048 bytes on.
__device__ __forceinline__ uint64_t at_desc_mn(uint32_t saddr) { return smem_desc_mn_sw128(saddr, kAtBlock, 1024); }

// D = A B^T over the head, A and B tiles of 128 rows.
template <int DP>
__device__ __forceinline__ void at_mma_head(uint32_t d, uint32_t sa, uint32_t sb, uint32_t idesc, int steps) {
    uint64_t ad = at_desc_k(sa), bd = at_desc_k(sb);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        if (kk >= steps) break;
        if (kk == 4) {                               // the second block of 64 values
            ad = at_desc_k(sa + kAtBlock);
            bd = at_desc_k(sb + kAtBlock);
        }
        tc_mma_f16(d, ad, bd, idesc, kk > 0);
        ad += 2;
        bd += 2;
    }
}
// D (+)= A B over the rows: A 128 x 128 in TMEM (the second half of its columns `skip` columns further on), B a tile.
__device__ __forceinline__ void at_mma_rows(uint32_t d, uint32_t ta, int skip, uint32_t sb, uint32_t idesc, int steps, bool accumulate) {
    uint64_t bd = at_desc_mn(sb);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk, bd += 128) {
        if (kk >= steps) break;
        tc_mma_f16_ta(d, ta + kk * 8 + (kk >= 4 ? skip : 0), bd, idesc, accumulate || kk > 0);
    }
}

// Zeros rows [from, to) of a tile: by a converged warp.
template <int DP>
__device__ __forceinline__ void at_zero_rows(uint32_t saddr, int from, int to) {
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < (to - from) * 8 * (DP / 64); i += 32) {
        const int block = i / ((to - from) * 8), j = i - block * (to - from) * 8;
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n"
                     :: "r"(saddr + block * kAtBlock + from * 128 + j * 16), "r"(0) : "memory");
    }
}

// [rows, heads, size] as a 3-D map with boxes of 64 values x `box_heads` x `box_rows`, zeros outside.
inline bool at_map(CUtensorMap *map, const AtTensor &t, int64_t rows, int heads, int D, int box_heads, int box_rows) {
    const uint64_t head = heads == 1 ? (uint64_t)(D + 7) / 8 * 8 : (uint64_t)t.head;
    const uint64_t row = rows == 1 ? head * (uint64_t)heads : (uint64_t)t.row;
    return make_tmap_3d(map, t.p, (uint64_t)D, (uint64_t)heads, (uint64_t)rows, head * 2, row * 2, 64, (uint32_t)box_heads,
                        (uint32_t)box_rows);
}

}  // namespace spconv
