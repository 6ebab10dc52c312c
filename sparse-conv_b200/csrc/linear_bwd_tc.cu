// The pointwise linear layer's backward in one pass over the rows (fp16 / bf16, tcgen05):
//
//   dz = grad_out * act'(z);  grad_feats = dz W;  grad_W += dz^T feats;  grad_bias += sum dz
//
// The separate kernels write dz and read it twice more: 4.5 row passes of Co channels and two of Ci
// against the 2 + 2 here (z and grad_out in, feats in, grad_feats out), and these layers are bound by
// HBM. It applies where W, both accumulators and two stages of 128 rows fit an SM: see
// bwd_tc_shape.
//
// 1.34 M x 128 -> 128 with GELU, bf16: 242 to 247 us (5.6 TB/s) and 473 us for the separate kernels; 2 M x 64 ->
// 256 without activation 259 and 602 us.
// Bits: dz is formed in fp32 and rounded to the features' type to be an operand of the tensor cores, as grad_out is when
// there is no activation; the bias sums take it before. For bf16 with GELU that rounding, the rounded argument's (see
// linear_tc.cu) and the output's own, 1.7e-3 of the norm each but the argument's 5.5e-4, make 2.4e-3 of the
// gradient's. Handing the remainder of dz to the tensor cores as a second operand gave 1.75e-3 and took 1.34 M x 128 ->
// 128 from 245 to 280 us and 883,771 x 64 -> 64 from 122 to 144: not kept.
//
// One CTA per SM takes every G-th tile of 128 rows. Roles, coupled by mbarriers:
//   warp 0       TMA loads of the tile's z, grad_out and feats rows (blocks of 64 columns, 128-byte
//                swizzle) into one of two stages; W once, at the start;
//   warps 6-13   dz in place of grad_out, rounded once, and its column sums, before the rounding,
//                in registers (a lane owns eight columns for good);
//   warp 1       MMA: the dz tile is read twice where it lies, as a K-major A operand (rows x co)
//                against W for grad_feats, and as an MN-major one (co x rows) against the feats tile
//                for grad_W, which stays in TMEM over all the CTA's tiles;
//   warps 2-5    epilogue: grad_feats from TMEM through the stage's own shared memory (free once
//                both products are done) and out by TMA; grad_W at the end, fp32, for
//                linear_reduce_kernel to add over the CTAs in a fixed order.
// Every wait is bounded (the conv kernels' limit); a timeout raises SPCONV_STATUS_WAIT_TIMEOUT and
// the CTA waits (bounded) for its own copies and MMAs before it frees TMEM and exits.
#include <algorithm>

#include "activation.cuh"
#include "common.cuh"
#include "linear_epilogue.cuh"
#include "linear_internal.h"
#include "tensor_map.h"

namespace spconv {

constexpr int kLbThreads = 448;
constexpr int kLbRows = 128;
constexpr int kLbBlock = kLbRows * 128;                 // 128 rows of 64 columns: 16 KB
constexpr int kLbCompute = 8;                           // warps of the dz pass
constexpr int kLbMaxSmem = 227 * 1024;
constexpr int kLbTail = 256;                            // barriers, TMEM address, abort flag

struct LbArgs {
    int M, Ci, Co;
    int ci_blocks, co_blocks;                           // of 64 columns; co_blocks even (M = 128 MMAs)
    int tiles;
    int has_act, want_x, want_w, want_b;
    float *w_partial, *b_partial;                       // [G][Co][Ci], [G * 8][Co]
    int tmem_cols;
    int32_t *status;
    uint64_t wait_ns;
};

template <typename T, int ACT>
__global__ void __launch_bounds__(kLbThreads, 1)
linear_bwd_tc_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_z,
                     const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_gx, const __grid_constant__ LbArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    constexpr bool HAS_ACT = ACT != SPCONV_ACT_NONE;
    const int nci = a.ci_blocks, nco = a.co_blocks;
    const int w_bytes = nco * nci * 8192;
    const int z_bytes = HAS_ACT ? nco * kLbBlock : 0, g_bytes = nco * kLbBlock, x_bytes = nci * kLbBlock;
    const int stage_bytes = z_bytes + g_bytes + x_bytes;
    const uint32_t s_w = smem_u32(base), s_stage = s_w + w_bytes;
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + w_bytes + 2 * stage_bytes);
    uint64_t *full = bar, *ready = full + 2, *accfull = ready + 2, *accempty = accfull + 2, *empty = accempty + 2;
    uint64_t *wfull = empty + 2, *wdone = wfull + 1;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(wdone + 1);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = gridDim.x;
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&ready[s]), kLbCompute);
            mbar_init(smem_u32(&accfull[s]), 1);
            mbar_init(smem_u32(&accempty[s]), 4);
            mbar_init(smem_u32(&empty[s]), 4);
        }
        mbar_init(smem_u32(wfull), 1);
        mbar_init(smem_u32(wdone), 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(s_tmem), (uint32_t)a.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    const uint32_t t_w = tmem + (uint32_t)(2 * nci * 64);             // behind grad_feats' two buffers
    auto wait = [&](uint64_t *b, uint32_t parity) -> bool {
        return mbar_wait_suspended(smem_u32(b), parity, s_abort, a.wait_ns);
    };
    // one answer for a warp: its lanes must not part before the next warp-wide instruction
    auto all_wait = [&](uint64_t *b, uint32_t parity) { return __all_sync(0xffffffffu, wait(b, parity)) != 0; };
    // tile i of this CTA uses stage i & 1 for the (i >> 1)-th time

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        if (elect_one()) {
            int i = 0;
            bool ok = true;
            if (a.want_x && (int)blockIdx.x < a.tiles) {
                mbar_arrive_expect_tx(smem_u32(wfull), (uint32_t)w_bytes);
                for (int c = 0; c < nco; ++c)
                    for (int n = 0; n < nci; ++n)
                        tma_load_2d(s_w + (uint32_t)(c * nci + n) * 8192, &map_w, n * 64, c * 64, smem_u32(wfull));
            }
            for (int t = blockIdx.x; t < a.tiles; t += G, ++i) {
                const int s = i & 1;
                if (i >= 2 && !wait(&empty[s], (uint32_t)(((i >> 1) - 1) & 1))) { ok = false; break; }
                const uint32_t mbar = smem_u32(&full[s]), dst = s_stage + s * stage_bytes;
                mbar_arrive_expect_tx(mbar, (uint32_t)(stage_bytes - (a.want_w ? 0 : x_bytes)));
                if (HAS_ACT)
                    for (int c = 0; c < nco; ++c) tma_load_2d(dst + c * kLbBlock, &map_z, c * 64, t * kLbRows, mbar);
                for (int c = 0; c < nco; ++c) tma_load_2d(dst + z_bytes + c * kLbBlock, &map_g, c * 64, t * kLbRows, mbar);
                if (a.want_w)
                    for (int c = 0; c < nci; ++c)
                        tma_load_2d(dst + z_bytes + g_bytes + c * kLbBlock, &map_x, c * 64, t * kLbRows, mbar);
            }
            // loads in flight write shared memory: let them land (at once unless some role gave up)
            for (int j = max(0, i - 2); j < i; ++j)
                mbar_wait_bounded(smem_u32(&full[j & 1]), (uint32_t)((j >> 1) & 1), kTmaDrainNs);
            if (a.want_x && (int)blockIdx.x < a.tiles) mbar_wait_bounded(smem_u32(wfull), 0, kTmaDrainNs);
            (void)ok;
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA
        if (elect_one()) {
            const int n_mma = (a.Ci + 15) & ~15;
            const uint32_t id_x = instr_desc_f16(dtype_traits<T>::mma_format, kLbRows, n_mma) | (1u << 16);
            const uint32_t id_w = instr_desc_f16(dtype_traits<T>::mma_format, 128, n_mma) | (1u << 15) | (1u << 16);
            const int k_steps = (a.Co + 15) >> 4;
            int i = 0;
            bool ok = !a.want_x || (int)blockIdx.x >= a.tiles || wait(wfull, 0);
            for (int t = blockIdx.x; t < a.tiles && ok; t += G, ++i) {
                const int s = i & 1;
                const uint32_t u = (uint32_t)(i >> 1);
                // with no activation dz is grad_out as loaded; the sums' warps only read it
                if (!wait(HAS_ACT ? &ready[s] : &full[s], u & 1u)) { ok = false; break; }
                if (a.want_x && u > 0 && !wait(&accempty[s], (u - 1) & 1u)) { ok = false; break; }
                tc_fence_after();
                const uint32_t dz = s_stage + s * stage_bytes + z_bytes, x = dz + g_bytes;
                // a K step moves a descriptor's address field (16-byte units; shared addresses do not carry out of it)
                if (a.want_x) {
                    const uint32_t d = tmem + (uint32_t)(s * nci * 64);
                    uint64_t dd = smem_desc_kmajor_swizzled(dz, 128), dw = smem_desc_mn_sw128(s_w, 8192, 1024);
                    for (int k = 0; k < k_steps; k += 4, dd += kLbBlock >> 4, dw += nci * 512) {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            if (k + kk >= k_steps) break;
                            tc_mma_f16(d, dd + kk * 2, dw + kk * 128, id_x, k + kk > 0 ? 1u : 0u);
                        }
                    }
                }
                if (a.want_w) {
                    uint64_t dd = smem_desc_mn_sw128(dz, kLbBlock, 1024);
                    const uint64_t dx = smem_desc_mn_sw128(x, kLbBlock, 1024);
                    for (int m = 0; m < nco / 2; ++m, dd += 2 * kLbBlock >> 4) {
#pragma unroll
                        for (int k = 0; k < kLbRows / 16; ++k)
                            tc_mma_f16(t_w + (uint32_t)(m * nci * 64), dd + k * 128, dx + k * 128, id_w,
                                       (i > 0 || k > 0) ? 1u : 0u);
                    }
                }
                tc_commit(smem_u32(&accfull[s]));
            }
            if (ok) tc_commit(smem_u32(wdone));
            // MMAs in flight read shared memory and write TMEM, and the epilogue may have given up
            if (i > 0) mbar_wait_bounded(smem_u32(&accfull[(i - 1) & 1]), (uint32_t)(((i - 1) >> 1) & 1));
        }
    } else if (warp < 6) {
        // ------------------------------------------------------------------ epilogue
        const int quad = warp & 3;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        int i = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < a.tiles; t += G, ++i) {
            const int s = i & 1;
            const uint32_t u = (uint32_t)(i >> 1);
            ok = all_wait(&accfull[s], u & 1u);
            // without an activation the sums' warps may still be reading the tile
            if (ok && !HAS_ACT && a.want_b) ok = all_wait(&ready[s], u & 1u);
            if (!ok) break;
            tc_fence_after();
            if (a.want_x) {
                const uint32_t out = s_stage + s * stage_bytes + (uint32_t)(quad * 4096 + lane * 128);
                for (int c = 0; c < a.Ci; c += 32) {
                    f32x2 f[16];
                    lt_load32(tmem + (uint32_t)(s * nci * 64 + c) + lanes, f);
                    const uint32_t at = out + (uint32_t)(c >> 6) * kLbBlock;
#pragma unroll
                    for (int v = 0; v < 4; ++v) lt_store8<T>(at + ((((c & 32) >> 3) + v) ^ (lane & 7)) * 16, f + 4 * v);
                }
                tc_fence_before();
                fence_proxy_async_smem();
                __syncwarp();
                if (elect_one()) {
                    mbar_arrive(smem_u32(&accempty[s]));
                    if (t * kLbRows + quad * 32 < a.M)
                        for (int c = 0; c < nci; ++c)
                            tma_store_2d(&map_gx, c * 64, t * kLbRows + quad * 32,
                                         s_stage + s * stage_bytes + c * kLbBlock + quad * 4096);
                    bulk_commit();
                    bulk_wait_read<0>();
                }
            }
            if (elect_one()) mbar_arrive(smem_u32(&empty[s]));
            __syncwarp();
        }
        if (ok && a.want_w && all_wait(wdone, 0)) {
            tc_fence_after();
            for (int m = 0; m < nco / 2; ++m) {
                const int co = m * 128 + quad * 32 + lane;
                float *dst = a.w_partial + ((int64_t)blockIdx.x * a.Co + co) * a.Ci;
                for (int c = 0; c < a.Ci; c += 32) {
                    f32x2 f[16];
                    lt_load32(t_w + (uint32_t)(m * nci * 64 + c) + lanes, f);
                    if (co < a.Co) {
#pragma unroll
                        for (int v = 0; v < 8; ++v)
                            if (c + v * 4 < a.Ci) {
                                const float2 lo = unpack_f32x2(f[2 * v]), hi = unpack_f32x2(f[2 * v + 1]);
                                __stcg(reinterpret_cast<float4 *>(dst + c) + v, make_float4(lo.x, lo.y, hi.x, hi.y));
                            }
                    }
                }
            }
            tc_fence_before();
        }
        if (elect_one()) bulk_wait<0>();
    } else if (HAS_ACT || a.want_b) {
        // ------------------------------------------------------------------ dz and its sums
        const int ct = tid - 6 * 32;
        int lpr = 1;                                                   // lanes per row: chunks of 8 columns
        while (lpr * 8 < a.Co) lpr <<= 1;                              // at most 32 (Co <= 256)
        const int chunk = ct & (lpr - 1), row0 = ct / lpr, step = kLbCompute * 32 / lpr;
        const bool have = chunk * 8 < a.Co;
        f32x2 acc[4] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
        const uint32_t col_at = (uint32_t)(chunk >> 3) * kLbBlock;
        int i = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < a.tiles; t += G, ++i) {
            const int s = i & 1;
            ok = all_wait(&full[s], (uint32_t)((i >> 1) & 1));
            if (!ok) break;
            if (have) {
                const uint32_t zt = s_stage + s * stage_bytes + col_at, gt = zt + z_bytes;
#pragma unroll 2
                for (int r = row0; r < kLbRows; r += step) {
                    const uint32_t at = (uint32_t)(r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
                    uint32_t g[4], z[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                                 : "=r"(g[0]), "=r"(g[1]), "=r"(g[2]), "=r"(g[3]) : "r"(gt + at));
                    if constexpr (HAS_ACT)
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                                     : "=r"(z[0]), "=r"(z[1]), "=r"(z[2]), "=r"(z[3]) : "r"(zt + at));
                    f32x2 d[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 gv = lt_unpack<T>(g[k]);
                        d[k] = pack_f32x2(gv.x, gv.y);
                        if constexpr (HAS_ACT) {
                            const float2 slope = act_slope2<ACT>(lt_unpack<T>(z[k]));
                            d[k] = mul2(d[k], pack_f32x2(slope.x, slope.y));
                        }
                        acc[k] = add2(acc[k], d[k]);
                    }
                    if constexpr (HAS_ACT) lt_store8<T>(gt + at, d);
                }
            }
            if constexpr (HAS_ACT) fence_proxy_async_smem();
            __syncwarp();
            if (elect_one()) mbar_arrive(smem_u32(&ready[s]));
        }
        if (ok && a.want_b) {
            const int cw = warp - 6;
            float v[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = unpack_f32x2(acc[k]);
                v[2 * k] = f.x;
                v[2 * k + 1] = f.y;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                for (int o = lpr; o < 32; o <<= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
            if (lane < lpr && have) {
                float4 *dst = reinterpret_cast<float4 *>(a.b_partial + ((int64_t)blockIdx.x * kLbCompute + cw) * a.Co + chunk * 8);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();                         // every role has set the flag by now if it gives up
    tc_fence_after();
    if (tid == 0 && *s_abort) raise_status(a.status, SPCONV_STATUS_WAIT_TIMEOUT);
    if (warp == 1) tmem_dealloc(tmem, (uint32_t)a.tmem_cols);
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
static int lb_smem(int ci_blocks, int co_blocks, bool act) {
    return 1024 + kLbTail + co_blocks * ci_blocks * 8192 + 2 * (co_blocks * (act ? 2 : 1) + ci_blocks) * kLbBlock;
}

// Whether one pass fits: W and two stages in shared memory, grad_W and two grad_feats buffers in 512
// TMEM columns, at most 256 output channels (eight columns a lane), and rows for two tiles per CTA.
bool bwd_tc_shape(int dtype, int64_t M, int Ci, int Co, int activation) {
    if ((dtype != SPCONV_F16 && dtype != SPCONV_BF16) || Ci % 8 || Co % 8 || Ci > 256 || Co > 256) return false;
    const int nci = (Ci + 63) / 64, nco = (Co + 127) / 128 * 2;
    return M >= 2 * 148 * kLbRows && (nco / 2 + 2) * nci * 64 <= 512 &&
           lb_smem(nci, nco, activation != SPCONV_ACT_NONE) <= kLbMaxSmem;
}

int bwd_tc_grid(int64_t M) { return (int)std::min<int64_t>(148, (M + kLbRows - 1) / kLbRows); }

template <typename T, int ACT>
static int lb_launch(const BwdArgs &q) {
    LbArgs a = {};
    a.M = (int)q.M;
    a.Ci = q.Ci;
    a.Co = q.Co;
    a.ci_blocks = (q.Ci + 63) / 64;
    a.co_blocks = (q.Co + 127) / 128 * 2;
    a.tiles = (int)((q.M + kLbRows - 1) / kLbRows);
    a.want_x = q.grad_feats != nullptr;
    a.want_w = q.w_partial != nullptr;
    a.want_b = q.b_partial != nullptr;
    a.w_partial = q.w_partial;
    a.b_partial = q.b_partial;
    a.status = q.status;
    a.wait_ns = wait_limit_ns();
    const int cols = (a.co_blocks / 2 + 2) * a.ci_blocks * 64;
    a.tmem_cols = cols <= 256 ? 256 : 512;
    auto kern = linear_bwd_tc_kernel<T, ACT>;
    static std::atomic<uint64_t> set{0};
    if (allow_smem(kern, kLbMaxSmem, set) != cudaSuccess)
        return check_launch("linear_bwd_tc: set max dynamic shared memory");
    CUtensorMap mg, mz, mx, mw, mo;
    const bool maps = make_tmap_2d(&mg, q.grad_out, q.Co, q.M, (uint64_t)q.Co * 2, 64, kLbRows) &&
                      (ACT == SPCONV_ACT_NONE || make_tmap_2d(&mz, q.preact, q.Co, q.M, (uint64_t)q.Co * 2, 64, kLbRows)) &&
                      (!a.want_w || make_tmap_2d(&mx, q.feats, q.Ci, q.M, (uint64_t)q.Ci * 2, 64, kLbRows)) &&
                      (!a.want_x || (make_tmap_2d(&mw, q.weight, q.Ci, q.Co, (uint64_t)q.Ci * 2, 64, 64) &&
                                     make_tmap_2d(&mo, q.grad_feats, q.Ci, q.M, (uint64_t)q.Ci * 2, 64, 32)));
    if (!maps) return SPCONV_ERR_CUDA;
    if (ACT == SPCONV_ACT_NONE) mz = mg;    // maps that the kernel does not read
    if (!a.want_w) mx = mg;
    if (!a.want_x) mw = mo = mg;
    const int smem = lb_smem(a.ci_blocks, a.co_blocks, ACT != SPCONV_ACT_NONE);
    kern<<<(unsigned)bwd_tc_grid(q.M), kLbThreads, smem, q.stream>>>(mg, mz, mx, mw, mo, a);
    return check_launch("linear_bwd_tc_kernel");
}

int launch_bwd_tc(const BwdArgs &q) {
    return act_dispatch(q.activation, [&](auto act) {
        return q.dtype == SPCONV_F16 ? lb_launch<__half, act.value>(q) : lb_launch<__nv_bfloat16, act.value>(q);
    });
}

}  // namespace spconv
