// Attention's gradients on the 5th-generation tensor cores (tcgen05 / TMEM), fp16 and bf16, heads of up to 128 values:
//
//   p = 2^(s c - lse);  dp = grad v^T;  ds = p (dp - delta);  delta = grad . out
//   grad_query = scale ds k;   grad_key = scale ds^T q;   grad_value = p^T grad
//
// Two sweeps, each recomputing s and dp: one owns 128 query rows and walks the keys, one owns 128 keys and walks the rows of
// every query head that reads them (so the gradients of shared keys add up in the accumulators). That is seven products
// a tile where one sweep with atomic sums of grad_query would have five, but every sum has one owner and one order: the
// same bits every run, no fp32 copy of a gradient in memory.
//
// The walked side comes W rows at a time. Warps: four for each 32 of the W columns compute, a thread a row and 32 columns; one
// loads (TMA), one issues the products. ds (and p) go back to TMEM in 16 bits, over s and dp, and are the A operand of
// the second products from there; B is the tile that s or dp was made of, read along its rows (MN-major). While the threads
// work on one of s and dp, the products that make the other run.
//
// Heads of up to 64: W = 64, two CTAs an SM, whose chains of waits fill one another's gaps (a step waits some 170 clocks
// for each barrier that another warp completes and 250 for a product's end). One CTA with W = 128 has the better products
// (128 columns of B to a read of A) but idles in its own chain: 84,000 voxels in 16 scenes, 8 x 64 bf16, 1.69 and 2.41 ms
// for the two sweeps, against 1.55 and 2.07; voxels to 257 tokens 0.71 and 0.50, against 0.44 and 0.47; many windows of 130,
// 0.47 and 0.53, against 0.28 and 0.32 (launches apart from one another; back to back, at the clocks that the power limit leaves, the
// scenes' forward and sweeps are 5.7 ms where these add up to 5.0). Wider heads: W = 128, one CTA (their accumulators take half of TMEM): 4 x 128 there
// 1.16 and 1.60 ms, 1.25 and 1.21 PFLOP/s. Nothing is full: at 8,192 tokens x 16 x 64 the tensor pipe is 44 and 43 % in use,
// the special functions 58 and 43 %, the issue slots 50 and 48 %.
//
// In fp16, whose smallest values would else lose bits where a row sees thousands of keys or gradients are small, p of
// the keys' sweep comes times 2^15, and ds times the power of two that its bound allows (at_lift); the results are
// scaled back in fp32. A row that sees a single key has ds = 0 exactly.
// Heads of up to 32: the queries' sweep takes ds in two parts, rounded and what that leaves, a product each. The roundings' errors
// add up along what a row's keys have in common (sum p k), which in narrow heads is much of them: over 257 keys, scores of deviation
// 1.5, the gradients are off by 1.79, 1.62 and 1.52 times their own rounding at 8, 16 and 32 values with one part, by 1.25, 1.13 and
// 1.07 with two, for 12 % of the sweep's time (windows of 130, 4 x 32: 301 and 338 us). From 48 on it is 1.49 and less, and at 64
// over long samples two parts would cost 26 %.
// Rows behind a sample's end are treated as in the forward: zeroed in shared memory where a product sums over rows.
#include <algorithm>

#include "attention_hidden.cuh"
#include "attention_tc.cuh"

namespace spconv {

// W columns (of the side that is walked) a tile: four warps compute 32 of them.
template <int DP, int W>
struct AbShape {
    static constexpr int kWarps = W / 8, kThreads = kWarps * 32 + 64;
    static constexpr int kWarpLoad = kWarps, kWarpMma = kWarps + 1;
    static constexpr int kPerSm = DP == 64 && W == 64 ? 2 : 1, kColumns = 512 / kPerSm;
    static constexpr int kOwn = DP / 64 * kAtBlock, kTile = DP / 64 * W * 128;      // bytes of an own tile, and of a walked one
};
// A row of accumulators [from, to) times `factor`, to a row of D values: rounded, or fp32 where `part` is given; zeros if `none`, and
// without a look at them if `zero`, which holds for the warp. Whether one is not finite, if that is asked for.
template <typename T, bool ASK>
__device__ __forceinline__ bool ab_store_row(uint32_t taddr, int from, int to, int D, bool zero, bool none, float factor, bool mine, T *out, float *part) {
    f32x2 lost = pack_f32x2(0.f, 0.f);                               // NaN once a value was not finite
    const bool wide = (D & 7) == 0 && ((uintptr_t)out & 15) == 0;
#pragma unroll 1
    for (int c = from; c < to && c < D; c += 32) {
        f32x2 o[16];
        __syncwarp();                                                // lanes without a row come here before those that store
        if (!zero) lt_load32(taddr + c, o);
        if (!mine) continue;
        if (ASK && !zero) {
#pragma unroll
            for (int i = 0; i < 16; ++i) lost = fma2(o[i], pack_f32x2(0.f, 0.f), lost);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int d = c + v * 8;
            if (d >= D) break;
            float f[8];
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 u = unpack_f32x2(o[v * 4 + i]);
                f[2 * i] = zero || none ? 0.f : u.x * factor;
                f[2 * i + 1] = zero || none ? 0.f : u.y * factor;
                w[i] = lt_pack<T>(f[2 * i], f[2 * i + 1]);
            }
            if (part && (D & 7) == 0) {                              // (the workspace is aligned, and so are rows of eights)
                *(float4 *)(part + d) = make_float4(f[0], f[1], f[2], f[3]);
                *(float4 *)(part + d + 4) = make_float4(f[4], f[5], f[6], f[7]);
            } else if (part) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (d + i < D) part[d + i] = f[i];
            } else if (wide) {
                *(uint4 *)(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (d + i < D) out[d + i] = dtype_traits<T>::from_f(f[i]);
            }
        }
    }
    const float2 z = unpack_f32x2(lost);
    return !(z.x + z.y == 0.f);
}

template <int DP, int W>
struct AqShape : AbShape<DP, W> {
    static constexpr int kK = DP == 64 ? 4 : 3, kV = DP == 64 ? 4 : 2;              // stages
    static constexpr int kSmem = 1024 + 2 * AbShape<DP, W>::kOwn + (kK + kV) * AbShape<DP, W>::kTile + 512;
};

template <typename T, int DP, int W, bool CAUSAL, bool TWO>
__global__ void __launch_bounds__(AbShape<DP, W>::kThreads, AbShape<DP, W>::kPerSm)
attention_tc_grad_query_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                               const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                               const __grid_constant__ AtArgs a, const int log_p) {
    using S = AqShape<DP, W>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t s_q = smem_u32(base), s_g = s_q + S::kOwn, s_k = s_g + S::kOwn, s_v = s_k + S::kK * S::kTile;
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + 2 * S::kOwn + (S::kK + S::kV) * S::kTile);
    uint64_t *kfull = bar, *kempty = kfull + S::kK, *vfull = kempty + S::kK, *vempty = vfull + S::kV;
    uint64_t *qfull = vempty + S::kV, *tail = qfull + 1, *sfull = tail + 1, *dpfull = sfull + 2, *dsready = dpfull + 1, *finished = dsready + 1;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(finished + 1);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 1);
    AtSample *s_sample = reinterpret_cast<AtSample *>(s_tmem + 2);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int P = 1 << log_p, tokens = kAtRows >> log_p;

    const int head0 = blockIdx.y << log_p, kh = head0 / (a.H / a.K);
    auto load = [&](uint32_t dst, int rows, const CUtensorMap *map, int head, int row, uint32_t mbar) {
        for (int c = 0; c < DP / 64; ++c) tma_load_3d(dst + c * rows * 128, map, c * 64, head, row, mbar);
    };
    // what a sample gives the CTA
    AtSample s = {};
    int n, m, t0, first, last, tiles, end_valid;
    auto share = [&] {
        n = s.q1 - s.q0;
        m = s.k1 - s.k0;
        t0 = s.tile * tokens;
        const int seen_last = at_seen(a, min(n, t0 + tokens) - 1, n, m);
        at_split(a.splits, blockIdx.z, (seen_last + W - 1) / W, first, last);
        tiles = s.tile < 0 || t0 >= n ? -1 : last - first;           // -1: nothing to do at all
        end_valid = min(W, seen_last - (last - 1) * W);
    };

    at_check_offsets(a);
    if (warp == S::kWarpLoad) {                                      // up to the first loads by this warp alone
        if (elect_one()) {
            for (const CUtensorMap *map : {&map_q, &map_k, &map_v, &map_g}) tma_prefetch_desc(map);
            for (int i = 0; i < S::kK; ++i) {
                mbar_init(smem_u32(&kfull[i]), 1);
                mbar_init(smem_u32(&kempty[i]), 1);
            }
            for (int i = 0; i < S::kV; ++i) {
                mbar_init(smem_u32(&vfull[i]), 1);
                mbar_init(smem_u32(&vempty[i]), 1);
            }
            for (uint64_t *b : {qfull, tail, sfull, sfull + 1, dpfull, finished}) mbar_init(smem_u32(b), 1);
            mbar_init(smem_u32(dsready), S::kWarps);
            *s_abort = 0;
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
        s = at_find(a, false, a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x, tokens);
        share();
        if (lane == 0) *s_sample = s;
        if (tiles > 0 && elect_one()) {
            mbar_arrive_expect_tx(smem_u32(qfull), 2 * S::kOwn);
            load(s_q, kAtRows, &map_q, head0, s.q0 + t0, smem_u32(qfull));
            load(s_g, kAtRows, &map_g, head0, s.q0 + t0, smem_u32(qfull));
        }
        __syncwarp();
    } else if (warp == 0) {
        tmem_alloc(smem_u32(s_tmem), S::kColumns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp != S::kWarpLoad) {
        s = *s_sample;
        share();
    }
    const uint32_t tmem = *s_tmem, t_dp = tmem + 2 * W, t_dq = tmem + 3 * W;
    auto wait = [&](uint64_t *b, uint32_t parity) { return at_wait(b, parity, s_abort, a.wait_ns); };
    auto next = [](int &i, uint32_t &phase, int stages) {
        if (++i == stages) {
            i = 0;
            phase ^= 1u;
        }
    };

    if (warp == S::kWarpLoad) {
        // ------------------------------------------------------------------ loads: k, v of each tile in turn
        if (tiles > 0) {
            int ks = 0, vs = 0;
            uint32_t kp = 1, vp = 1;
            bool ok = true;
            for (int j = 0; j < tiles && ok; ++j) {
                const bool cut = j + 1 == tiles && (end_valid & 15);
                const int row = s.k0 + (first + j) * W;
                if (!(ok = __all_sync(0xffffffffu, wait(&kempty[ks], kp)) != 0)) break;
                const uint32_t dst = s_k + ks * S::kTile, mbar = smem_u32(cut ? tail : &kfull[ks]);
                if (elect_one()) {
                    mbar_arrive_expect_tx(mbar, S::kTile);
                    load(dst, W, &map_k, kh, row, mbar);
                }
                __syncwarp();
                if (!(ok = __all_sync(0xffffffffu, wait(&vempty[vs], vp)) != 0)) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(smem_u32(&vfull[vs]), S::kTile);
                    load(s_v + vs * S::kTile, W, &map_v, kh, row, smem_u32(&vfull[vs]));
                }
                __syncwarp();
                if (cut) {
                    ok = __all_sync(0xffffffffu, wait(tail, 0)) != 0;
                    at_zero_rows<DP, W>(dst, end_valid, (end_valid + 15) & ~15);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&kfull[ks]));
                }
                next(ks, kp, S::kK);
                next(vs, vp, S::kV);
            }
        }
    } else if (warp == S::kWarpMma) {
        // ------------------------------------------------------------------ products
        if (tiles > 0 && elect_one()) {
            const uint32_t id_s = instr_desc_f16(dtype_traits<T>::mma_format, 128, W);
            const uint32_t id_o = instr_desc_f16(dtype_traits<T>::mma_format, 128, (a.D + 15) & ~15) | 1u << 16;
            const int steps = (a.D + 15) >> 4;
            int ks = 0, vs = 0, done = 0;                            // next k and v stage; the k stage of ds k
            uint32_t kp = 0, vp = 0, ds_phase = 0;
            bool ok = wait(qfull, 0);
            auto scores = [&](int j) {                               // s of tile j
                if (!(ok = ok && wait(&kfull[ks], kp))) return;
                tc_fence_after();
                at_mma_head<DP, W>(tmem + (j & 1) * W, s_q, s_k + ks * S::kTile, id_s, steps);
                tc_commit(smem_u32(&sfull[j & 1]));
                next(ks, kp, S::kK);
            };
            auto products = [&] {                                    // dp of the next tile
                if (!(ok = ok && wait(&vfull[vs], vp))) return;
                tc_fence_after();
                at_mma_head<DP, W>(t_dp, s_g, s_v + vs * S::kTile, id_s, steps);
                tc_commit(smem_u32(dpfull));
                tc_commit(smem_u32(&vempty[vs]));
                next(vs, vp, S::kV);
            };
            scores(0);
            products();
            if (tiles > 1) scores(1);
            for (int j = 0; j < tiles && ok; ++j, ds_phase ^= 1u) {
                if (!(ok = wait(dsready, ds_phase))) break;
                tc_fence_after();
                const int sum_steps = j + 1 < tiles ? W / 16 : (end_valid + 15) >> 4;
                at_mma_rows<32, W>(t_dq, tmem + (j & 1) * W, s_k + done * S::kTile, id_o, sum_steps, j > 0);
                if constexpr (TWO) at_mma_rows<32, W>(t_dq, tmem + (j & 1) * W + 16, s_k + done * S::kTile, id_o, sum_steps, true);
                tc_commit(smem_u32(j + 1 < tiles ? &kempty[done] : finished));
                if (++done == S::kK) done = 0;
                if (j + 1 < tiles) products();
                if (j + 2 < tiles) scores(j + 2);
            }
        }
    } else if (tiles >= 0) {
        // ------------------------------------------------------------------ a thread a row and 32 columns
        const int part = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int token = t0 + (row >> log_p);
        const bool mine = token < n;
        const int seen = mine ? at_seen(a, token, n, m) : 0;
        const bool some = __any_sync(0xffffffffu, mine);
        const int seen_all = __reduce_min_sync(0xffffffffu, mine ? seen : m);
        const int64_t at = (int64_t)(s.q0 + token) * a.H + head0 + (row & (P - 1));
        const float lse = mine ? a.lse[at] : INFINITY, delta = mine ? a.delta[at] : 0.f;
        const int lift = at_lift(a, s.b);                            // p, and so ds, comes times 2^lift
        const f32x2 c2 = pack_f32x2(a.c, a.c), l2 = pack_f32x2(lift - lse, lift - lse), d2 = pack_f32x2(-delta, -delta);
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const uint32_t t_s = tmem + (j & 1) * W + part * 32 + lanes;
            if (!(ok = __all_sync(0xffffffffu, wait(&sfull[j & 1], (j >> 1) & 1)) != 0)) break;
            tc_fence_after();
            f32x2 x[16];
            if (some) {
                lt_load32(t_s, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = at_exp2(fma2(x[i], c2, l2));
            }
            if (!(ok = __all_sync(0xffffffffu, wait(dpfull, j & 1)) != 0)) break;
            tc_fence_after();
            if (some) {
                uint32_t w[16], rest[16];
                f32x2 y[16];
                lt_load32(t_dp + part * 32 + lanes, y);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 f = unpack_f32x2(mul2(x[i], add2(y[i], d2)));
                    w[i] = lt_pack<T>(f.x, f.y);
                    if constexpr (TWO) {
                        const float2 hi = lt_unpack<T>(w[i]);
                        rest[i] = lt_pack<T>(f.x - hi.x, f.y - hi.y);
                    }
                }
                if ((first + j + 1) * W > seen_all) {          // behind the row's keys; all of a single one
                    const int keep = seen == 1 ? 0 : seen - (first + j) * W - part * 32;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t mask = (2 * i < keep ? 0xffffu : 0u) | (2 * i + 1 < keep ? 0xffff0000u : 0u);
                        w[i] &= mask;
                        if constexpr (TWO) rest[i] &= mask;
                    }
                }
                tmem_st16(t_s, w);
                if constexpr (TWO) tmem_st16(t_s + 16, rest);
                tc_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(dsready));
        }
        if (tiles > 0 && ok) ok = __all_sync(0xffffffffu, wait(finished, 0)) != 0;
        tc_fence_after();
        if (ok && some) {
            constexpr int kCols = DP * 32 / W > 32 ? DP * 32 / W : 32;               // a part's (with more parts than 32s: none)
            float *to = a.splits > 1 ? a.partial + (blockIdx.z * (int64_t)a.M * a.H + at) * a.D : nullptr;
            const AtHidden hidden{s.q0 + token, head0 + (row & (P - 1)), kh, s.k0, first * W, seen, min(m, (first + tiles) * W)};
            const int c0 = part * kCols;
            const bool lost = ab_store_row<T, CAUSAL>(t_dq + lanes, c0, c0 + kCols, a.D, tiles == 0, seen == 0, ldexpf(a.scale, -lift), mine,
                                              (T *)a.gq + at * a.D, to);
            if (CAUSAL && lost && seen > 0 && seen < hidden.hi && (seen == 1 || (lse == lse && delta == delta)))
                at_keys_again<T>(a, hidden, -lse, delta, c0, c0 + kCols, a.scale, {to, (T *)a.gq + at * a.D});
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();                                                 // every role has set the flag by now if it gives up
    if (*s_abort) {                                                  // copies and products in flight end within this
        if (tid == 0) raise_status(a.status, SPCONV_STATUS_WAIT_TIMEOUT);
        const uint64_t begin = globaltimer_ns();
        while (globaltimer_ns() - begin < kTmaDrainNs) {}
        __syncthreads();
    }
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, S::kColumns);
}

template <int DP, int W>
struct AkShape : AbShape<DP, W> {
    static constexpr int kStages = DP == 64 ? (W == 64 ? 3 : 4) : 2;                // of q and grad
    static constexpr int kSmem = 1024 + 2 * AbShape<DP, W>::kOwn + 2 * kStages * AbShape<DP, W>::kTile + kStages * W * 8 + 512;
};

template <typename T, int DP, int W, bool CAUSAL>
__global__ void __launch_bounds__(AbShape<DP, W>::kThreads, AbShape<DP, W>::kPerSm)
attention_tc_grad_key_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                             const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                             const __grid_constant__ AtArgs a, const int log_p) {
    using S = AkShape<DP, W>;
    constexpr float kUp = dtype_traits<T>::mma_format == 0 ? 15.f : 0.f;         // powers of two on p
    constexpr float kDown = dtype_traits<T>::mma_format == 0 ? 0x1p-15f : 1.f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t s_k = smem_u32(base), s_v = s_k + S::kOwn, s_q = s_v + S::kOwn;      // stages of q, grad
    float *s_rows = reinterpret_cast<float *>(base + 2 * S::kOwn + 2 * S::kStages * S::kTile);    // stages of W x -lse, W x -delta
    uint64_t *bar = reinterpret_cast<uint64_t *>(s_rows + S::kStages * 2 * W);
    uint64_t *full = bar, *empty = full + S::kStages, *kvfull = empty + S::kStages, *tail = kvfull + 1, *sfull = tail + 1;
    uint64_t *dpfull = sfull + 1, *pready = dpfull + 1, *dsready = pready + 1, *finished = dsready + 1;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(finished + 1);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 1);
    AtSample *s_sample = reinterpret_cast<AtSample *>(s_tmem + 2);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int P = 1 << log_p, tokens = W >> log_p;

    const int kh = blockIdx.y, G = a.H / a.K;
    auto load = [&](uint32_t dst, int rows, const CUtensorMap *map, int head, int row, uint32_t mbar) {
        for (int c = 0; c < DP / 64; ++c) tma_load_3d(dst + c * rows * 128, map, c * 64, head, row, mbar);
    };
    // what a sample gives the CTA: tiles of queries that see a key of this tile, of each block of P heads of the group
    AtSample s = {};
    int n, m, key0, from, per_head, first, last, tiles;
    auto share = [&] {
        n = s.q1 - s.q0;
        m = s.k1 - s.k0;
        key0 = s.tile * kAtRows;
        from = a.causal ? (int)max((int64_t)0, (int64_t)key0 - m + n) / tokens : 0;
        per_head = max(0, (n + tokens - 1) / tokens - from);
        at_split(a.splits, blockIdx.z, per_head * (G >> log_p), first, last);
        tiles = s.tile < 0 || key0 >= m ? -1 : last - first;         // -1: nothing to do at all
    };

    at_check_offsets(a);
    if (warp == S::kWarpLoad) {                                      // up to the first loads by this warp alone
        if (elect_one()) {
            for (const CUtensorMap *map : {&map_q, &map_k, &map_v, &map_g}) tma_prefetch_desc(map);
            for (int i = 0; i < S::kStages; ++i) {
                mbar_init(smem_u32(&full[i]), 2);                    // the copies' bytes, and the rows' numbers
                mbar_init(smem_u32(&empty[i]), 1);
            }
            for (uint64_t *b : {kvfull, tail, sfull, dpfull, finished}) mbar_init(smem_u32(b), 1);
            mbar_init(smem_u32(pready), S::kWarps);
            mbar_init(smem_u32(dsready), S::kWarps);
            *s_abort = 0;
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
        s = at_find(a, true, blockIdx.x, kAtRows);
        share();
        if (lane == 0) *s_sample = s;
        if (tiles > 0 && elect_one()) {
            mbar_arrive_expect_tx(smem_u32(kvfull), 2 * S::kOwn);
            load(s_k, kAtRows, &map_k, kh, s.k0 + key0, smem_u32(kvfull));
            load(s_v, kAtRows, &map_v, kh, s.k0 + key0, smem_u32(kvfull));
        }
        __syncwarp();
    } else if (warp == 0) {
        tmem_alloc(smem_u32(s_tmem), S::kColumns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp != S::kWarpLoad) {
        s = *s_sample;
        share();
    }
    const uint32_t tmem = *s_tmem, t_dp = tmem + W, t_dv = tmem + 2 * W, t_dk = t_dv + DP;
    struct Walk {
        int head, t;                                                 // the tile's first head, and its number
    };
    auto begin = [&] { return Walk{kh * G + (per_head ? first / per_head : 0) * P, from + (per_head ? first % per_head : 0)}; };
    auto advance = [&](Walk &w) {
        if (++w.t == from + per_head) {
            w.t = from;
            w.head += P;
        }
    };
    auto rows_of = [&](const Walk &w) { return min(tokens, n - w.t * tokens) << log_p; };
    auto wait = [&](uint64_t *b, uint32_t parity) { return at_wait(b, parity, s_abort, a.wait_ns); };
    auto next = [](int &i, uint32_t &phase) {
        if (++i == S::kStages) {
            i = 0;
            phase ^= 1u;
        }
    };

    if (warp == S::kWarpLoad) {
        // ------------------------------------------------------------------ loads: q, grad and the rows' numbers
        if (tiles > 0) {
            int st = 0;
            uint32_t phase = 1, tail_phase = 0;
            bool ok = true;
            Walk w = begin();
            float down = 0.f;
            for (int j = 0; j < tiles; ++j, advance(w), next(st, phase)) {
                const int rows = rows_of(w);
                const bool cut = rows & 15;
                float lse[W / 32], delta[W / 32];
#pragma unroll
                for (int i = 0; i < W / 32; ++i) {                        // on their way while the stage is waited for
                    const int r = lane + 32 * i;
                    const int64_t at = (int64_t)(s.q0 + w.t * tokens + (r >> log_p)) * a.H + w.head + (r & (P - 1));
                    lse[i] = r < rows ? kUp - __ldg(a.lse + at) : -INFINITY;
                    delta[i] = r < rows ? -__ldg(a.delta + at) : 0.f;
                }
                if (!(ok = __all_sync(0xffffffffu, wait(&empty[st], phase)) != 0)) break;
                const uint32_t dst = s_q + st * 2 * S::kTile, mbar = smem_u32(cut ? tail : &full[st]);
                if (elect_one()) {
                    mbar_arrive_expect_tx(mbar, 2 * S::kTile);
                    load(dst, W, &map_q, w.head, s.q0 + w.t * tokens, mbar);
                    load(dst + S::kTile, W, &map_g, w.head, s.q0 + w.t * tokens, mbar);
                }
                if (j == 0) down = ldexpf(kDown, at_lift(a, s.b));   // not before the first copies are on their way
#pragma unroll
                for (int i = 0; i < W / 32; ++i) {
                    s_rows[st * 2 * W + lane + 32 * i] = lse[i];
                    s_rows[st * 2 * W + W + lane + 32 * i] = delta[i] * down;
                }
                __syncwarp();
                if (cut) {
                    if (!(ok = __all_sync(0xffffffffu, wait(tail, tail_phase)) != 0)) break;
                    tail_phase ^= 1u;
                    at_zero_rows<DP, W>(dst, rows, (rows + 15) & ~15);
                    at_zero_rows<DP, W>(dst + S::kTile, rows, (rows + 15) & ~15);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&full[st]));
                }
                if (lane == 0) mbar_arrive(smem_u32(&full[st]));
            }
        }
    } else if (warp == S::kWarpMma) {
        // ------------------------------------------------------------------ products
        if (tiles > 0 && elect_one()) {
            const uint32_t id_s = instr_desc_f16(dtype_traits<T>::mma_format, 128, W);
            const uint32_t id_o = instr_desc_f16(dtype_traits<T>::mma_format, 128, (a.D + 15) & ~15) | 1u << 16;
            const int steps = (a.D + 15) >> 4;
            int st = 0;
            uint32_t phase = 0, t_phase = 0;
            bool ok = wait(kvfull, 0) && wait(&full[0], 0);
            if (ok) {
                tc_fence_after();
                at_mma_head<DP, W>(tmem, s_k, s_q, id_s, steps);
                tc_commit(smem_u32(sfull));
                at_mma_head<DP, W>(t_dp, s_v, s_q + S::kTile, id_s, steps);
                tc_commit(smem_u32(dpfull));
            }
            Walk w = begin();
            for (int j = 0; j < tiles && ok; ++j, t_phase ^= 1u, advance(w)) {
                const int here = st, sum_steps = (rows_of(w) + 15) >> 4;
                const uint32_t s_here = s_q + here * 2 * S::kTile;
                const bool more = j + 1 < tiles;
                next(st, phase);
                const uint32_t s_next = s_q + st * 2 * S::kTile;
                if (!(ok = wait(pready, t_phase))) break;
                tc_fence_after();
                at_mma_rows<32, W>(t_dv, tmem, s_here + S::kTile, id_o, sum_steps, j > 0);
                if (more) {
                    if (!(ok = wait(&full[st], phase))) break;
                    tc_fence_after();
                    at_mma_head<DP, W>(tmem, s_k, s_next, id_s, steps);
                    tc_commit(smem_u32(sfull));
                }
                if (!(ok = wait(dsready, t_phase))) break;
                tc_fence_after();
                at_mma_rows<32, W>(t_dk, t_dp, s_here, id_o, sum_steps, j > 0);
                tc_commit(smem_u32(more ? &empty[here] : finished));
                if (more) {
                    at_mma_head<DP, W>(t_dp, s_v, s_next + S::kTile, id_s, steps);
                    tc_commit(smem_u32(dpfull));
                }
            }
        }
    } else if (tiles >= 0) {
        // ------------------------------------------------------------------ a thread a key and 32 query rows
        const int part = warp >> 2, row = tid & 127, key = key0 + row;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + part * 32 + lanes, t_d = t_dp + part * 32 + lanes;
        const bool mine = key < m;
        const int lift = at_lift(a, s.b);                            // ds comes times 2^lift
        const float down = ldexpf(kDown, lift);
        const f32x2 c2 = pack_f32x2(a.c, a.c), k2 = pack_f32x2(down, down);
        bool ok = true;
        int st = 0;
        uint32_t phase = 0, t_phase = 0;
        Walk w = begin();
        for (int j = 0; j < tiles; ++j, t_phase ^= 1u, next(st, phase), advance(w)) {
            const uint32_t s_lse = smem_u32(s_rows + st * 2 * W + part * 32), s_delta = s_lse + W * 4;
            // columns from `see` on see this key; from `use` on with a gradient of their score
            int see = 0, use = 0;
            bool masked = m == 1;
            if (a.causal) {
                const int64_t before = (int64_t)n - m - (int64_t)w.t * tokens;   // the query that sees key 0 last, in the tile
                masked |= before + key0 + kAtRows - 1 > 0;
                see = (int)max((int64_t)-kAtRows, min((int64_t)kAtRows, before + key)) * P - part * 32;
                use = see + (key == 0 ? P : 0);
            }
            if (m == 1) use = kAtRows;
            if (!(ok = __all_sync(0xffffffffu, wait(&full[st], phase) && wait(sfull, t_phase)) != 0)) break;
            tc_fence_after();
            f32x2 x[16];
            uint32_t u[16];
            lt_load32(t_s, x);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                f32x2 l0, l1;
                asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];\n" : "=l"(l0.v), "=l"(l1.v) : "r"(s_lse + i * 8));
                x[i] = at_exp2(fma2(x[i], c2, l0));
                x[i + 1] = at_exp2(fma2(x[i + 1], c2, l1));
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 f = unpack_f32x2(x[i]);
                u[i] = lt_pack<T>(f.x, f.y);
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i) u[i] &= (2 * i >= see ? 0xffffu : 0u) | (2 * i + 1 >= see ? 0xffff0000u : 0u);
            }
            tmem_st16(t_s, u);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(pready));
            if (!(ok = __all_sync(0xffffffffu, wait(dpfull, t_phase)) != 0)) break;
            tc_fence_after();
            f32x2 y[16];
            lt_load32(t_d, y);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                f32x2 d0, d1;
                asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];\n" : "=l"(d0.v), "=l"(d1.v) : "r"(s_delta + i * 8));
                const float2 f0 = unpack_f32x2(mul2(x[i], fma2(y[i], k2, d0)));
                const float2 f1 = unpack_f32x2(mul2(x[i + 1], fma2(y[i + 1], k2, d1)));
                u[i] = lt_pack<T>(f0.x, f0.y);
                u[i + 1] = lt_pack<T>(f1.x, f1.y);
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i) u[i] &= (2 * i >= use ? 0xffffu : 0u) | (2 * i + 1 >= use ? 0xffff0000u : 0u);
            }
            tmem_st16(t_d, u);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(dsready));
        }
        if (tiles > 0 && ok) ok = __all_sync(0xffffffffu, wait(finished, 0)) != 0;
        tc_fence_after();
        if (ok) {                                                    // half of the parts stores grad_value, half grad_key
            constexpr int kParts = W / 64, kCols = DP / kParts;
            const bool keys = part >= kParts;
            const int64_t all = (int64_t)a.N * a.K, at = (int64_t)(s.k0 + key) * a.K + kh;
            float *to = a.splits > 1 ? a.partial + ((2 * blockIdx.z + !keys) * all + at) * a.D : nullptr;
            T *out = (T *)(keys ? a.gk : a.gv);
            const int c0 = (part & (kParts - 1)) * kCols;
            if (out) out += at * a.D;
            const bool lost = ab_store_row<T, CAUSAL>((keys ? t_dk : t_dv) + lanes, c0, c0 + kCols, a.D, tiles == 0, false,
                                              keys ? ldexpf(a.scale, -lift) : kDown, mine && (out || to), out, to);
            if (CAUSAL && lost) at_rows_again<T>(a, *s_sample, kAtRows, W, log_p, !keys, c0, c0 + kCols, {to, out});
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();                                                 // every role has set the flag by now if it gives up
    if (*s_abort) {                                                  // copies and products in flight end within this
        if (tid == 0) raise_status(a.status, SPCONV_STATUS_WAIT_TIMEOUT);
        const uint64_t begin_ns = globaltimer_ns();
        while (globaltimer_ns() - begin_ns < kTmaDrainNs) {}
        __syncthreads();
    }
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, S::kColumns);
}

template <typename T, int DP, int W, bool KEYS, bool CAUSAL, bool TWO>
static int ab_run(const AtArgs &a) {
    using S = AbShape<DP, W>;
    const int G = a.H / a.K;
    constexpr int rows = KEYS ? W : kAtRows;                         // query rows of a tile
    int log_p = 0;
    while ((2 << log_p) <= rows && G % (2 << log_p) == 0) ++log_p;
    const int P = 1 << log_p, tokens = rows >> log_p, keys = KEYS ? kAtRows : W;
    CUtensorMap mq, mk, mv, mg;
    if (!at_map(&mq, a.q, a.M, a.H, a.D, P, tokens) || !at_map(&mk, a.k, a.N, a.K, a.D, 1, keys) ||
        !at_map(&mv, a.v, a.N, a.K, a.D, 1, keys) || !at_map(&mg, a.grad, a.M, a.H, a.D, P, tokens))
        return SPCONV_ERR_CUDA;
    static std::atomic<uint64_t> done;
    auto kern = KEYS ? attention_tc_grad_key_kernel<T, DP, W, CAUSAL> : attention_tc_grad_query_kernel<T, DP, W, CAUSAL, TWO>;
    // padded so that no more CTAs share an SM than its TMEM columns serve
    constexpr int need = KEYS ? AkShape<DP, W>::kSmem : AqShape<DP, W>::kSmem, least = S::kPerSm == 2 ? 80 * 1024 : 120 * 1024;
    constexpr int smem = need > least ? need : least;
    if (allow_smem(kern, smem, done) != cudaSuccess) return check_launch("attention: shared memory");
    const dim3 grid(KEYS ? (unsigned)at_tiles(a.N, a.B, kAtRows) : (unsigned)at_tiles(a.M, a.B, tokens), KEYS ? a.K : a.H / P, a.splits);
    kern<<<grid, S::kThreads, smem, a.stream>>>(mq, mk, mv, mg, a, log_p);
    return check_launch(KEYS ? "attention_tc_grad_key_kernel" : "attention_tc_grad_query_kernel");
}

template <typename T, bool KEYS, bool CAUSAL>
static int ab_size(const AtArgs &a) {
    if (!KEYS && a.D <= 32) return ab_run<T, 64, 64, KEYS, CAUSAL, !KEYS>(a);
    return a.D <= 64 ? ab_run<T, 64, 64, KEYS, CAUSAL, false>(a) : ab_run<T, 128, 128, KEYS, CAUSAL, false>(a);
}
template <typename T, bool KEYS>
static int ab_causal(const AtArgs &a) {
    return a.causal ? ab_size<T, KEYS, true>(a) : ab_size<T, KEYS, false>(a);
}

int launch_at_tc_grad_query(const AtArgs &a) {
    return a.dtype == SPCONV_F16 ? ab_causal<__half, false>(a) : ab_causal<__nv_bfloat16, false>(a);
}
int launch_at_tc_grad_key(const AtArgs &a) {
    return a.dtype == SPCONV_F16 ? ab_causal<__half, true>(a) : ab_causal<__nv_bfloat16, true>(a);
}

}  // namespace spconv
