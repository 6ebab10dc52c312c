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

// Bounded wait, suspended up to 20 us between checks; under a limit of less it polls (these waits are so short that one
// suspended try, however short its hint, would outlast any such limit).
__device__ __forceinline__ bool at_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, uint64_t limit_ns) {
    const uint32_t addr = smem_u32(bar);
    if (mbar_test(addr, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
        if (limit_ns < 20000ull ? mbar_test(addr, parity) : mbar_try_wait_suspended(addr, parity, 20000u)) return true;
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > limit_ns) {
            *abort_flag = 1;
            return false;
        }
    }
}

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
// 16 consecutive columns of the lane's row; tc_wait_st before others rely on it.
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

// 2 N columns of the lane's row, all loads in flight before the first is waited for.
template <int N>
__device__ __forceinline__ void at_load(uint32_t taddr, f32x2 (&x)[N]) {
    uint32_t r[2 * N];
#pragma unroll
    for (int g = 0; g < N / 16; ++g) {
        uint32_t *q = r + 32 * g;
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
            "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
            : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
              "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15]),
              "=r"(q[16]), "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]), "=r"(q[22]), "=r"(q[23]),
              "=r"(q[24]), "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]), "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
            : "r"(taddr + 32 * g) : "memory");
    }
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < N; ++i) {                   // nothing that uses them moves before the wait
        asm volatile("mov.b64 %0, {%1, %2};" : "=l"(x[i].v) : "r"(r[2 * i]), "r"(r[2 * i + 1]));
    }
}

// 32 aligned bytes at once: a sector, which two stores of 16 would write in halves.
__device__ __forceinline__ void at_store32(void *p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
                 :: "l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// 2^x of two values, by the special functions: 16 a clock and SM. (A polynomial on the FMA pipe, degree 4, for one to four of
// eight pairs was 2 % faster at best, in the gradients at one of eight, and slower from three on: a step's time is its
// chain of waits, not the special functions alone.)
__device__ __forceinline__ f32x2 at_exp2(f32x2 x) {
    const float2 f = unpack_f32x2(x);
    return pack_f32x2(ex2_approx(f.x), ex2_approx(f.y));
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A tile in shared memory: DP / 64 blocks of ROWS rows x 64 values. As an operand along the head (K-major) ...
__device__ __forceinline__ uint64_t at_desc_k(uint32_t saddr) { return smem_desc_kmajor_swizzled(saddr, 128); }
// ... and along the rows (MN-major): a step of 16 rows is 2048 bytes on.
template <int ROWS>
__device__ __forceinline__ uint64_t at_desc_mn(uint32_t saddr) { return smem_desc_mn_sw128(saddr, ROWS * 128, 1024); }

// D = A B^T over the head: A a tile of 128 rows, B one of ROWS.
template <int DP, int ROWS>
__device__ __forceinline__ void at_mma_head(uint32_t d, uint32_t sa, uint32_t sb, uint32_t idesc, int steps) {
    uint64_t ad = at_desc_k(sa), bd = at_desc_k(sb);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        if (kk >= steps) break;
        if (kk == 4) {                               // the second block of 64 values
            ad = at_desc_k(sa + kAtBlock);
            bd = at_desc_k(sb + ROWS * 128);
        }
        tc_mma_f16(d, ad, bd, idesc, kk > 0);
        ad += 2;
        bd += 2;
    }
}
// D (+)= A B over B's ROWS rows: A 128 x ROWS in TMEM, in parts of PART columns' values (16 bits each) that begin PART
// TMEM columns apart, where the fp32 values were that they are made of.
template <int PART, int ROWS>
__device__ __forceinline__ void at_mma_rows(uint32_t d, uint32_t ta, uint32_t sb, uint32_t idesc, int steps, bool accumulate) {
    constexpr int kSteps = PART / 16;
    uint64_t bd = at_desc_mn<ROWS>(sb);
#pragma unroll
    for (int kk = 0; kk < ROWS / 16; ++kk, bd += 128) {
        if (kk >= steps) break;
        tc_mma_f16_ta(d, ta + kk / kSteps * PART + kk % kSteps * 8, bd, idesc, accumulate || kk > 0);
    }
}

// Zeros rows [from, to) of a tile of ROWS: by a converged warp.
template <int DP, int ROWS>
__device__ __forceinline__ void at_zero_rows(uint32_t saddr, int from, int to) {
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < (to - from) * 8 * (DP / 64); i += 32) {
        const int block = i / ((to - from) * 8), j = i - block * (to - from) * 8;
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n"
                     :: "r"(saddr + block * ROWS * 128 + from * 128 + j * 16), "r"(0) : "memory");
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
