// Matrix products of the pointwise linear layer on the 5th-generation tensor cores (tcgen05 /
// TMEM), fp16 and bf16 with fp32 accumulation:
//
//   forward         out[M, Co]  = residual + act(feats[M, Ci] W[Co, Ci]^T + bias)   (and its argument)
//   input gradient  gx[M, Ci]   = dz[M, Co] W[Co, Ci]                    B read along its rows
//   weight gradient gw[Co, Ci]  = dz[M, Co]^T feats[M, Ci]               A and B read along their rows
//
// One persistent CTA per SM walks 128 x BN output tiles (BN = 64, 128 or 256, the last tile of a
// row as narrow as the matrix). Operands come by TMA as 128-byte-swizzled tiles of 64 K values:
// a K-contiguous operand as rows of 128 bytes (K-major), the others as blocks of 64 K rows of 64
// columns (MN-major descriptors), so no operand is ever transposed in memory. Roles, coupled by
// mbarriers only:
//   warp 0      loads: A and B tiles of each K step into a ring of stages. Where the whole of B's
//               column block fits beside the ring it is loaded once and stays (few K steps: the
//               layers over millions of voxels, whose bound is HBM);
//   warp 1      MMA: one thread; the accumulators take turns in two (BN = 256), four or eight (64) TMEM
//               buffers. With one K step a tile's cost is this thread's: eight buffers in place of four,
//               descriptors advanced rather than built, and an elected lane took 883,771 x 64 -> 16 with a
//               residual from 44.0 to 34.0 us and 1.34 M x 128 -> 128 with GELU from 127.9 to 114.6;
//   warps 2-17  four epilogue groups of four warps (one per TMEM lane quadrant), a group per
//               buffer in turn, or two that share a buffer's columns: 64 columns at a time from TMEM to
//               registers, + bias, act, + residual, one rounding, into swizzled shared memory and out
//               by TMA (which clips ragged edges). The residual arrives by TMA, ahead of its turn, in
//               the slot the output leaves from. Four warps per scheduler, since GELU and SiLU are
//               dependent chains that two could not hide.
// PAIR: two CTAs of a cluster, on two SMs, share a 256 x 256 tile (cta_group::2). Each holds its 128
// rows of A, half of B's columns and its own rows' accumulators; the first one's MMA thread drives
// both tensor cores, and commits to barriers in both. A K step then brings 32 KB into an SM instead of
// 48. 84,000 x 512 -> 2048 bf16: 183 us unpaired, 170 us paired (152 to 163 since, up to 1.16 PFLOP/s; the library's
// product alone takes 151 us). Keeping a pair's halves of B in shared memory (K <= 512) leaves one output slot a
// warp and is slower, 192 us.
// The weight gradient's K is the voxels: K is cut into splits, each writes fp32 sums of its own,
// and linear_reduce_kernel adds them in a fixed order.
// Measured (bf16): 1.34 M x 128 -> 128 112 us (6.1 TB/s) and its input gradient 112 us; 2 M x 64 -> 256
// 217 to 230 us (5.6 to 5.9 TB/s), 287 to 294 us with GELU, 322 to 330 us with SiLU. Nothing is full in those two: at
// 12.4 instructions a value the issue slots are 59 % in use, the special functions 38 %, the tensor pipe 9 % and HBM
// 42 %; the warps wait for fixed latencies, for their loads from TMEM, each complete before its arithmetic
// begins, and for the roles' barriers.
// Bits: the output is rounded once, from fp32. The activation's argument is kept for the backward in the features'
// type, as many bytes as the output; taking the slope at the rounded argument costs bf16 gradients 5.5e-4 of their norm
// (one rounding of a bf16 result costs 1.7e-3), and in fp32 it would be twice the bytes each way where HBM is the bound.
// Every wait is bounded (the conv kernels' limit); a timeout raises SPCONV_STATUS_WAIT_TIMEOUT and
// the CTA waits (bounded) for its own copies and MMAs before it frees TMEM and exits.
#include <algorithm>
#include <mutex>

#include "activation.cuh"
#include "common.cuh"
#include "linear_epilogue.cuh"
#include "linear_internal.h"
#include "tensor_map.h"

namespace spconv {

constexpr int kLtThreads = 576;
constexpr int kLtBM = 128, kLtBK = 64;
constexpr int kLtABytes = kLtBM * kLtBK * 2;            // 16 KB a stage
constexpr int kLtEpiWarps = 16, kLtEpiGroups = 4;
constexpr int kLtMaxBias = 4096;                        // bias columns kept in shared memory
constexpr int kLtMaxStages = 12;
constexpr int kLtMaxSlots = 4;
constexpr int kLtMaxSmem = 227 * 1024;
// behind the tiles: barriers, TMEM address and abort flag, bias (fp32, at most kLtMaxBias)
constexpr int kLtMaxBufs = 8;
constexpr int kLtBars = 2 * kLtMaxStages + 1 + 2 * kLtMaxBufs + kLtEpiWarps * kLtMaxSlots;
constexpr int kLtTail = (kLtBars * 8 + 8 + 15) & ~15;

struct LtArgs {
    int M, N, K;
    int nb;                                 // column blocks
    int tiles;                              // row tiles * nb
    int items;                              // tiles * splits
    int k_per_split;                        // a multiple of 64 unless splits == 1
    int BN, stages, slots;                  // slots per epilogue warp (outputs; as many again for preact)
    int bufs;                               // TMEM accumulators
    int bias_smem;                          // bias columns in shared memory (N up to whole chunks of 32, or 0)
    int b_resident;                         // K steps of B that stay in shared memory, or 0
    const void *bias;
    int bias_f32;                           // a bias in fp32, else in the features' type (or none)
    int has_residual, has_preact;
    float *partial;
    int32_t *status;
    uint64_t wait_ns;
};

__device__ __forceinline__ void lt_wait_read(int pending) {
    if (pending <= 0) bulk_wait_read<0>();
    else if (pending == 1) bulk_wait_read<1>();
    else if (pending == 2) bulk_wait_read<2>();
    else bulk_wait_read<3>();
}

// CH: columns an epilogue warp takes at a time: 64, or 32 where shared memory has no room for 64.
template <typename T, bool A_T, bool B_T, int ACT, bool PAIR, int CH>
__global__ void __launch_bounds__(kLtThreads, 1)
linear_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_res,
                 const __grid_constant__ CUtensorMap map_pre, const __grid_constant__ LtArgs a) {
    constexpr bool PARTIAL = A_T;           // the weight gradient: fp32 sums of a split
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int BN = a.BN, S = a.stages, NO = a.slots;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const int b_bytes = (PAIR ? BN / 2 : BN) * 128;
    const int stage_bytes = kLtABytes + (a.b_resident ? 0 : b_bytes);
    const uint32_t s_b = smem_u32(base);                               // resident B
    const uint32_t s_stage = s_b + a.b_resident * b_bytes;
    const int warp_slots = NO * (a.has_preact ? 2 : 1);
    constexpr int slot_bytes = 64 * CH;                                // a slot: 32 rows of CH columns
    const uint32_t s_out = s_stage + S * stage_bytes;
    uint8_t *tail = base + a.b_resident * b_bytes + S * stage_bytes + (PARTIAL ? 0 : kLtEpiWarps * warp_slots * slot_bytes);
    uint64_t *bar = reinterpret_cast<uint64_t *>(tail);
    uint64_t *full = bar, *empty = full + kLtMaxStages, *bfull = empty + kLtMaxStages, *accfull = bfull + 1;
    uint64_t *accempty = accfull + kLtMaxBufs, *rbar = accempty + kLtMaxBufs;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(bar + kLtBars);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 1);
    float *s_bias = reinterpret_cast<float *>(tail + kLtTail);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // workers: CTAs, or pairs of them
    const int G = PAIR ? gridDim.x >> 1 : gridDim.x, me = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const uint32_t tmem_cols = 512;                                    // bufs * BN: all there are
    if (a.bias_f32)
        for (int i = tid; i < a.bias_smem; i += kLtThreads) s_bias[i] = i < a.N ? ((const float *)a.bias)[i] : 0.f;
    else
        for (int i = tid; i < a.bias_smem; i += kLtThreads)
            s_bias[i] = i < a.N ? dtype_traits<T>::to_f(((const T *)a.bias)[i]) : 0.f;
    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(bfull), 1);
        for (int g = 0; g < a.bufs; ++g) {
            mbar_init(smem_u32(&accfull[g]), 1);
            mbar_init(smem_u32(&accempty[g]), (PAIR ? 2 : 1) * kLtEpiWarps / min(a.bufs, kLtEpiGroups));
        }
        for (int i = 0; i < kLtEpiWarps * NO; ++i) mbar_init(smem_u32(&rbar[i]), 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(smem_u32(s_tmem), tmem_cols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(s_tmem), tmem_cols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    if constexpr (PAIR) cluster_sync();      // the barriers of both are ready
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    auto wait = [&](uint64_t *b, uint32_t parity) -> bool {
        return mbar_wait_suspended(smem_u32(b), parity, s_abort, a.wait_ns);
    };
    // A walk over every `step`-th item: its tile and its range of K. Divisions only at the start (the
    // single loading and MMA threads would spend longer on them than on a tile's copies).
    struct Walk {
        int item, m, n, split, step, dm, dn;
    };
    auto begin = [&](int first, int step) {
        Walk w;
        w.item = first;
        w.step = step;
        w.split = PARTIAL ? first / a.tiles : 0;
        const int tile = first - w.split * a.tiles;
        w.m = tile / a.nb;
        w.n = tile - w.m * a.nb;
        w.dm = step / a.nb;
        w.dn = step - w.dm * a.nb;
        return w;
    };
    auto advance = [&](Walk &w) {
        w.item += w.step;
        if constexpr (PARTIAL) {
            w = begin(w.item, w.step);
        } else {
            w.m += w.dm;
            w.n += w.dn;
            if (w.n >= a.nb) {
                w.n -= a.nb;
                ++w.m;
            }
        }
    };
    auto row_of = [&](const Walk &w) { return PAIR ? w.m * (2 * kLtBM) + (int)rank * kLtBM : w.m * kLtBM; };
    // an MMA's N: a multiple of 16, and of 32 over a pair
    auto mma_cols = [&](int n0) { return (min(BN, a.N - n0) + (PAIR ? 31 : 15)) & ~(PAIR ? 31 : 15); };
    auto k_begin = [&](const Walk &w) { return PARTIAL ? w.split * a.k_per_split : 0; };
    auto k_end = [&](int k0) { return PARTIAL && a.K - k0 > a.k_per_split ? k0 + a.k_per_split : a.K; };
    // ring position: index and the parity of its current use
    auto next = [](int &i, uint32_t &phase, int n) {
        if (++i == n) {
            i = 0;
            phase ^= 1u;
        }
    };

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        if (elect_one()) {
            auto load = [&](uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t mbar) {
                if constexpr (PAIR) tma_load_2d_pair(dst, map, x, y, mbar);
                else tma_load_2d(dst, map, x, y, mbar);
            };
            auto load_b = [&](uint32_t dst, int k, int n0, uint32_t mbar) {
                if constexpr (PAIR) n0 += (int)rank * (mma_cols(n0) >> 1);    // this CTA's half of B's columns
                if constexpr (B_T) {
                    for (int c = 0; c < b_bytes / 8192; ++c) load(dst + c * 8192, &map_b, n0 + c * 64, k, mbar);
                } else {
                    load(dst, &map_b, k, n0, mbar);
                }
            };
            int st = 0;
            uint32_t phase = 0;
            int issued = 0;                  // stages in use, at most S
            bool ok = true;
            Walk w = begin(me, G);
            if (a.b_resident && w.item < a.items) {           // the grid is a multiple of nb: n never changes
                mbar_arrive_expect_tx(smem_u32(bfull), (uint32_t)(a.b_resident * b_bytes));
                for (int c = 0; c < a.b_resident; ++c) load_b(s_b + c * b_bytes, c * kLtBK, w.n * BN, smem_u32(bfull));
            }
            for (; w.item < a.items && ok; advance(w)) {
                const int m0 = row_of(w), n0 = w.n * BN, k0 = k_begin(w), k1 = k_end(k0);
                for (int k = k0; k < k1; k += kLtBK) {
                    if (issued == S && !wait(&empty[st], phase ^ 1u)) { ok = false; break; }
                    uint32_t mbar = smem_u32(&full[st]);
                    const uint32_t dst = s_stage + st * stage_bytes;
                    if constexpr (PAIR) {    // both CTAs' bytes count on the first one's barrier
                        if (rank == 0) mbar_arrive_expect_tx(mbar, 2 * (uint32_t)stage_bytes);
                        mbar = cluster_addr(mbar, 0);
                    } else {
                        mbar_arrive_expect_tx(mbar, (uint32_t)stage_bytes);
                    }
                    if constexpr (A_T) {
                        load(dst, &map_a, m0, k, mbar);
                        load(dst + 8192, &map_a, m0 + 64, k, mbar);
                    } else {
                        load(dst, &map_a, k, m0, mbar);
                    }
                    if (!a.b_resident) load_b(dst + kLtABytes, k, n0, mbar);
                    if (issued < S) ++issued;
                    next(st, phase, S);
                }
            }
            // every load has landed before the CTA may exit (at once unless the MMA gave up): the
            // stages from st on were last used a phase earlier than those before it
            if constexpr (PAIR) {
                // what landed here is counted on the first CTA's barriers, and the last empties say that it
                // was used; after giving up, the bound of such copies is waited out
                if (!ok) {
                    const uint64_t t0 = globaltimer_ns();
                    while (globaltimer_ns() - t0 < kTmaDrainNs) {}
                } else {
                    for (int i = 0; i < issued; ++i)
                        mbar_wait_bounded(smem_u32(&empty[i]), i < st ? phase : phase ^ 1u, a.wait_ns + kTmaDrainNs);
                }
            } else {
                for (int i = 0; i < issued; ++i)
                    mbar_wait_bounded(smem_u32(&full[i]), i < st ? phase : phase ^ 1u, kTmaDrainNs);
                if (a.b_resident && (int)blockIdx.x < a.items) mbar_wait_bounded(smem_u32(bfull), 0, kTmaDrainNs);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA
        if (rank == 0 && elect_one()) {
            auto commit = [&](uint64_t *b) {
                if constexpr (PAIR) tc_commit_pair(smem_u32(b));
                else tc_commit(smem_u32(b));
            };
            int st = 0, buf = 0, last = -1;
            uint32_t phase = 0, acc_phase = 1;                // the first use of a buffer passes at once
            bool ok = true;
            Walk w = begin(me, G);
            if (a.b_resident && w.item < a.items) ok = wait(bfull, 0);
            for (; w.item < a.items && ok; advance(w)) {
                const int n0 = w.n * BN, k0 = k_begin(w), k1 = k_end(k0);
                if (!wait(&accempty[buf], acc_phase)) { ok = false; break; }
                tc_fence_after();
                const uint32_t idesc = instr_desc_f16(dtype_traits<T>::mma_format, PAIR ? 2 * kLtBM : kLtBM, mma_cols(n0)) |
                                       (A_T ? 1u << 15 : 0u) | (B_T ? 1u << 16 : 0u);
                const uint32_t d = tmem + (uint32_t)(buf * BN);
                uint32_t s_res = s_b;
                for (int k = k0; k < k1; k += kLtBK) {
                    if (!wait(&full[st], phase)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t sa = s_stage + st * stage_bytes;
                    const uint32_t sb = a.b_resident ? s_res : sa + kLtABytes;
                    s_res += b_bytes;
                    const int steps = min(4, (k1 - k + 15) >> 4);     // zeros past K's end are skipped
                    // a K step of 16 moves a descriptor's address field (16-byte units, no carry: < 2^14)
                    uint64_t ad = A_T ? smem_desc_mn_sw128(sa, 8192, 1024) : smem_desc_kmajor_swizzled(sa, 128);
                    uint64_t bd = B_T ? smem_desc_mn_sw128(sb, 8192, 1024) : smem_desc_kmajor_swizzled(sb, 128);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk, ad += A_T ? 128 : 2, bd += B_T ? 128 : 2) {
                        if (kk >= steps) break;
                        if constexpr (PAIR) tc_mma_f16_pair(d, ad, bd, idesc, (k > k0 || kk > 0) ? 1u : 0u);
                        else tc_mma_f16(d, ad, bd, idesc, (k > k0 || kk > 0) ? 1u : 0u);
                    }
                    commit(&empty[st]);
                    last = st;
                    next(st, phase, S);
                }
                if (ok) {
                    commit(&accfull[buf]);
                    next(buf, acc_phase, a.bufs);
                }
            }
            // MMAs in flight read shared memory and write TMEM, and the epilogue may have given up: wait for
            // the last commit (its stage's use ended `phase` if the ring has not wrapped since, else the
            // phase before)
            if (last >= 0) mbar_wait_bounded(smem_u32(&empty[last]), last < st ? phase : phase ^ 1u);
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        const int ew = warp - 2, quad = warp & 3;
        // `turn` tiles are in the groups' hands at a time; with more buffers than that a group alternates
        // between bufs / turn of them
        const int turn = min(a.bufs, kLtEpiGroups), mine = (ew >> 2) % turn, sub = (ew >> 2) / turn, share = kLtEpiGroups / turn;
        const uint32_t slot0 = s_out + (uint32_t)(ew * warp_slots * slot_bytes);
        const uint32_t pre0 = slot0 + (uint32_t)(NO * slot_bytes);
        uint64_t *my_rbar = rbar + ew * NO;
        // rows of 128 (64) bytes: the 16-byte chunk's index XOR-ed with address bits 7 and up
        const uint32_t row_at = (uint32_t)(lane * 2 * CH), row_x = (uint32_t)(CH == 64 ? lane & 7 : (lane >> 1) & 3);
        // one answer for the warp: its lanes must not part before the next warp-wide instruction
        auto all_wait = [&](uint64_t *b, uint32_t parity) { return __all_sync(0xffffffffu, wait(b, parity)) != 0; };
        auto chunks_of = [&](int n0) { return (min(BN, a.N - n0) + CH - 1) / CH; };
        // Residual loads run `ahead` chunks before their use. The slot of load L was last the
        // store of chunk L - NO, and when chunk b begins, b stores have been committed: those after
        // L - NO = b + ahead - NO may still be reading.
        const int ahead = NO >= 3 ? NO - 2 : NO - 1;
        int l_slot = 0, outstanding = 0, l_chunk = sub;
        uint32_t l_phase = 0;
        Walk lw = begin(me + mine * G, turn * G);
        auto load_residual = [&](int behind) {        // the next chunk's, if there is one
            while (lw.item < a.items && l_chunk >= chunks_of(lw.n * BN)) {
                advance(lw);
                l_chunk = sub;
            }
            const bool more = lw.item < a.items;
            if (lane == 0) {
                lt_wait_read(behind);
                if (more) {
                    mbar_arrive_expect_tx(smem_u32(&my_rbar[l_slot]), slot_bytes);
                    tma_load_2d(slot0 + l_slot * slot_bytes, &map_res, lw.n * BN + l_chunk * CH, row_of(lw) + quad * 32,
                                smem_u32(&my_rbar[l_slot]));
                }
            }
            if (more) {
                ++outstanding;
                l_chunk += share;
                next(l_slot, l_phase, NO);
            }
        };
        if (!PARTIAL && a.has_residual)
            for (int i = 0; i < ahead; ++i) load_residual(0);
        int s = 0;
        int buf = mine;
        uint32_t s_phase = 0, use_phase = 0;
        for (Walk w = begin(me + mine * G, turn * G); w.item < a.items; advance(w)) {
            const int m0 = row_of(w), n0 = w.n * BN;
            const int n_cols = min(BN, a.N - n0), chunks = chunks_of(n0);
            if (!all_wait(&accfull[buf], use_phase)) break;
            tc_fence_after();
            const uint32_t t_acc = tmem + (uint32_t)(buf * BN) + ((uint32_t)(quad * 32) << 16);
            bool ok = true;
            for (int j = sub; j < chunks; j += share, next(s, s_phase, NO)) {
                const uint32_t so = slot0 + s * slot_bytes + row_at, sp = pre0 + s * slot_bytes + row_at;
                if constexpr (!PARTIAL) {
                    if (a.has_residual) {
                        load_residual(NO - 1 - ahead);
                        if (all_wait(&my_rbar[s], s_phase)) --outstanding;
                        else ok = false;
                    } else {
                        if (lane == 0) lt_wait_read(NO - 1);
                    }
                    __syncwarp();
                    if (!ok) break;
                }
#pragma unroll 1
                for (int half = 0; half < CH / 32; ++half) {
                    const int c0 = j * CH + half * 32;        // columns within the tile
                    if (c0 >= n_cols) break;
                    f32x2 f[16];
                    lt_load32(t_acc + (uint32_t)c0, f);
                    if constexpr (PARTIAL) {
                        const int row = m0 + quad * 32 + lane;
                        float *dst = a.partial + ((int64_t)w.split * a.M + row) * a.N + n0 + c0;
                        if (row < a.M) {
#pragma unroll
                            for (int v = 0; v < 8; ++v)
                                if (c0 + v * 4 < n_cols) {
                                    const float2 lo = unpack_f32x2(f[2 * v]), hi = unpack_f32x2(f[2 * v + 1]);
                                    __stcg(reinterpret_cast<float4 *>(dst) + v, make_float4(lo.x, lo.y, hi.x, hi.y));
                                }
                        }
                        continue;
                    }
                    if (a.bias_smem) {
                        const uint32_t b = smem_u32(s_bias + n0 + c0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            f32x2 b0, b1;
                            asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];\n" : "=l"(b0.v), "=l"(b1.v) : "r"(b + i * 16));
                            f[2 * i] = add2(f[2 * i], b0);
                            f[2 * i + 1] = add2(f[2 * i + 1], b1);
                        }
                    } else if (a.bias_f32) {
                        const float *b = (const float *)a.bias + n0 + c0;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (c0 + 2 * i < n_cols) f[i] = add2(f[i], pack_f32x2(b[2 * i], b[2 * i + 1]));
                    } else if (a.bias) {
                        const T *b = (const T *)a.bias + n0 + c0;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (c0 + 2 * i < n_cols)
                                f[i] = add2(f[i], pack_f32x2(dtype_traits<T>::to_f(b[2 * i]), dtype_traits<T>::to_f(b[2 * i + 1])));
                    }
                    const uint32_t v0 = (uint32_t)half * 4;
                    if (a.has_preact) {
#pragma unroll
                        for (int v = 0; v < 4; ++v) lt_store8<T>(sp + (((v0 + v) ^ row_x) << 4), f + 4 * v);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 4) act_value8<ACT>(f + i);
                    if (a.has_residual) {
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            uint32_t q[4];
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                                         : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3])
                                         : "r"(so + (((v0 + v) ^ row_x) << 4)) : "memory");
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 x = lt_unpack<T>(q[i]);
                                f[4 * v + i] = add2(f[4 * v + i], pack_f32x2(x.x, x.y));
                            }
                        }
                    }
#pragma unroll
                    for (int v = 0; v < 4; ++v) lt_store8<T>(so + (((v0 + v) ^ row_x) << 4), f + 4 * v);
                }
                if constexpr (!PARTIAL) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (m0 + quad * 32 < a.M) {
                            tma_store_2d(&map_out, n0 + j * CH, m0 + quad * 32, slot0 + s * slot_bytes);
                            if (a.has_preact) tma_store_2d(&map_pre, n0 + j * CH, m0 + quad * 32, pre0 + s * slot_bytes);
                        }
                        bulk_commit();       // one group a chunk, empty or not
                    }
                }
            }
            if (!ok) break;
            tc_fence_before();               // the accumulator has been read: free for the MMA
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(cluster_addr(smem_u32(&accempty[buf]), 0));
                else mbar_arrive(smem_u32(&accempty[buf]));
            }
            if ((buf += turn) >= a.bufs) {
                buf = mine;
                use_phase ^= 1u;
            }
        }
        if (!PARTIAL && lane == 0) {
            for (; outstanding > 0; --outstanding, next(s, s_phase, NO))     // residual loads nobody waited for
                mbar_wait_bounded(smem_u32(&my_rbar[s]), s_phase, kTmaDrainNs);
            bulk_wait<0>();
        }
    }

    __syncwarp();
    tc_fence_before();
    if constexpr (PAIR) cluster_sync();      // neither leaves while the other's MMAs or arrivals may reach it
    __syncthreads();                         // every role has set the flag by now if it gives up
    tc_fence_after();
    if (tid == 0 && *s_abort) raise_status(a.status, SPCONV_STATUS_WAIT_TIMEOUT);
    if (warp == 1) {
        if constexpr (PAIR) tmem_dealloc_pair(tmem, tmem_cols);
        else tmem_dealloc(tmem, tmem_cols);
    }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
static int lt_sms() {
    static std::once_flag once;
    static int sms = 148;
    std::call_once(once, [] {
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    });
    return sms;
}

bool gemm_tc_supported(const GemmArgs &g) {
    if (g.dtype != SPCONV_F16 && g.dtype != SPCONV_BF16) return false;
    // TMA: rows a multiple of 16 bytes apart, 16-byte aligned tensors
    const int64_t a_row = g.a_t ? g.M : g.K, b_row = g.b_t ? g.N : g.K;
    if (a_row % 8 || b_row % 8 || g.N % 8) return false;
    for (const void *p : {g.a, g.b, (const void *)g.out, g.residual, (const void *)g.preact, (const void *)g.partial})
        if ((uintptr_t)p & 15) return false;
    return true;
}

// Columns of a tile: the widest of 256, 128, 64 that the matrix fills to more than half (each
// operand is then read least often), narrowed while the tiles are fewer than the SMs.
static int lt_bn(int64_t M, int64_t N, int splits) {
    int bn = N > 128 ? 256 : N > 64 ? 128 : 64;
    const int64_t mt = (M + kLtBM - 1) / kLtBM * splits;
    while (bn > 64 && mt * ((N + bn - 1) / bn) < lt_sms()) bn >>= 1;
    return bn;
}

int gemm_tc_splits(int64_t M, int64_t N, int64_t K) {
    // whole waves of 148 items; each split costs a write and a read of fp32 sums
    const int64_t tiles = ((M + kLtBM - 1) / kLtBM) * ((N + 255) / 256);
    const int64_t chunks = (K + kLtBK - 1) / kLtBK;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(chunks / 4, lt_sms()));
    int64_t best = 1;
    double best_cost = 1e30;
    for (int64_t s = 1; s <= most; ++s) {
        const int64_t waves = (s * tiles + lt_sms() - 1) / lt_sms();
        const double cost = (double)waves * ((chunks + s - 1) / s + 4) + 0.02 * s * tiles;
        if (cost < best_cost) {
            best_cost = cost;
            best = s;
        }
    }
    return (int)best;
}

// A pair of CTAs takes 256 x 256 tiles where B cannot stay in shared memory anyway and there is a tile
// for every pair of SMs.
static bool lt_pair(const GemmArgs &g) {
    const int64_t nk = (g.K + kLtBK - 1) / kLtBK;
    const int64_t tiles = (g.M + 2 * kLtBM - 1) / (2 * kLtBM) * ((g.N + 255) / 256) * g.splits;
    return g.N >= 256 && g.M >= 256 && nk * 256 * 128 > 96 * 1024 && tiles >= lt_sms() / 2;
}

template <typename T, bool A_T, bool B_T, int ACT, bool PAIR, int CH>
static int lt_launch(const GemmArgs &g) {
    LtArgs a = {};
    a.M = (int)g.M;
    a.N = (int)g.N;
    a.K = (int)g.K;
    a.BN = PAIR ? 256 : A_T ? (g.N > 128 ? 256 : g.N > 64 ? 128 : 64) : lt_bn(g.M, g.N, g.splits);
    a.nb = (int)((g.N + a.BN - 1) / a.BN);
    constexpr int rows = PAIR ? 2 * kLtBM : kLtBM;
    const int64_t items = (g.M + rows - 1) / rows * a.nb * g.splits;
    SPCONV_REQUIRE(items < (int64_t)1 << 30, SPCONV_ERR_ARG, "too many output tiles");
    a.items = (int)items;
    a.tiles = a.items / g.splits;
    a.k_per_split = (int)(g.splits > 1 ? g.k_per_split : g.K);
    a.bufs = 512 / a.BN;
    a.bias = g.bias;
    a.bias_f32 = g.bias_f32;
    a.bias_smem = g.bias && g.N <= kLtMaxBias ? (a.N + 31) & ~31 : 0;
    a.has_residual = g.residual != nullptr;
    a.has_preact = g.preact != nullptr;
    a.partial = g.partial;
    a.status = g.status;
    a.wait_ns = wait_limit_ns();
    const int sms = lt_sms();
    int grid = PAIR ? 2 * std::min(sms / 2, a.items) : std::min(sms, a.items);
    const int64_t nk = (g.K + kLtBK - 1) / kLtBK;
    const int b_bytes = (PAIR ? a.BN / 2 : a.BN) * 128, room = kLtMaxSmem - 1024 - kLtTail - a.bias_smem * 4;
    // output slots and stages beside `resident` K steps of B: four stages at least where that is
    // possible at all, then as many slots as fit
    auto fit = [&](int resident) {
        const int stage = kLtABytes + (resident ? 0 : b_bytes);
        for (int least = 4; least >= 3; --least)
            for (int slots = 4; slots >= 1; slots >>= 1) {
                const int out = A_T ? 0 : kLtEpiWarps * slots * (a.has_preact ? 2 : 1) * 64 * CH;
                const int stages = (room - resident * b_bytes - out) / stage;
                if (stages < least) continue;
                a.slots = slots;
                a.stages = std::min(stages, kLtMaxStages);
                a.b_resident = resident;
                return true;
            }
        return false;
    };
    // B stays where a CTA meets it again (more than one row tile per CTA) and its block fits
    const bool stay = !A_T && !PAIR && a.nb <= sms && a.items > grid && nk * b_bytes <= 96 * 1024 && fit((int)nk);
    if (stay) grid = sms / a.nb * a.nb;
    else if (!fit(0)) {
        if constexpr (CH == 64 && !A_T) return lt_launch<T, A_T, B_T, ACT, PAIR, 32>(g);
        set_error("linear: no shared-memory layout for this shape");
        return SPCONV_ERR_UNSUPPORTED;
    }
    const int smem = 1024 + kLtTail + a.bias_smem * 4 + a.b_resident * b_bytes + a.stages * (kLtABytes + (a.b_resident ? 0 : b_bytes)) +
                     (A_T ? 0 : kLtEpiWarps * a.slots * (a.has_preact ? 2 : 1) * 64 * CH);
    auto kern = linear_tc_kernel<T, A_T, B_T, ACT, PAIR, CH>;
    static std::atomic<uint64_t> set{0};
    if (allow_smem(kern, kLtMaxSmem, set) != cudaSuccess)
        return check_launch("linear_tc: set max dynamic shared memory");
    CUtensorMap ma, mb, mo, mr, mp;
    // K-contiguous operands: boxes of 64 K x rows; the others: 64 columns x 64 K rows
    const bool maps =
        (A_T ? make_tmap_2d(&ma, g.a, g.M, g.K, g.M * 2, 64, 64) : make_tmap_2d(&ma, g.a, g.K, g.M, g.K * 2, 64, kLtBM)) &&
        (B_T ? make_tmap_2d(&mb, g.b, g.N, g.K, g.N * 2, 64, 64) : make_tmap_2d(&mb, g.b, g.K, g.N, g.K * 2, 64, PAIR ? a.BN / 2 : a.BN)) &&
        (A_T || make_tmap_2d(&mo, g.out, g.N, g.M, g.N * 2, CH, 32)) &&
        (!g.residual || make_tmap_2d(&mr, g.residual, g.N, g.M, g.N * 2, CH, 32)) &&
        (!g.preact || make_tmap_2d(&mp, g.preact, g.N, g.M, g.N * 2, CH, 32));
    if (!maps) return SPCONV_ERR_CUDA;
    if (A_T) mo = ma;                       // maps that the kernel does not read
    if (!g.residual) mr = ma;
    if (!g.preact) mp = ma;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kLtThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = g.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {2, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = PAIR ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kern, ma, mb, mo, mr, mp, a);
    return check_launch("linear_tc_kernel");
}

template <typename T, bool PAIR>
static int lt_type(const GemmArgs &g) {
    constexpr int CH = PAIR ? 32 : 64;       // a pair's accumulators leave faster than they fill either way
    if (g.a_t) return lt_launch<T, true, true, SPCONV_ACT_NONE, PAIR, CH>(g);
    if (g.b_t) return lt_launch<T, false, true, SPCONV_ACT_NONE, PAIR, CH>(g);
    return act_dispatch(g.activation, [&](auto act) { return lt_launch<T, false, false, act.value, PAIR, CH>(g); });
}

int launch_gemm_tc(const GemmArgs &g) {
    if (lt_pair(g)) return g.dtype == SPCONV_F16 ? lt_type<__half, true>(g) : lt_type<__nv_bfloat16, true>(g);
    return g.dtype == SPCONV_F16 ? lt_type<__half, false>(g) : lt_type<__nv_bfloat16, false>(g);
}

}  // namespace spconv
