// Attention's forward on the 5th-generation tensor cores (tcgen05 / TMEM), fp16 and bf16, heads of up to 128 values:
//
//   s = q k^T (fp32, TMEM);  p = 2^(s c - m);  out = (p v) / sum p,   c = scale log2(e), m a running maximum of s c
//
// A CTA owns NQ tiles of 128 query rows of one key head and walks the sample's keys, 128 at a time. Warps: four a
// tile for the softmax, a thread a row; one that loads (TMA), one that issues the products. Per tile of keys s
// arrives in TMEM, its row goes to registers whole, p goes back over it in 16 bits, and is the A operand of p v from there;
// the rows of v are read along the keys (MN-major), so nothing is transposed. With two tiles (NQ = 2, a CTA an SM) one tile's
// products run under the other's softmax, and keys and values are read once for both; with one (two CTAs an SM) the two
// CTAs do that for one another, which wastes less where samples are short.
//
// The maximum is followed lazily: while a row's new maximum exceeds the one in use by at most 8, the old one
// stays (p up to 2^8, exact in range), so out and the sum are rescaled a few times a row, not once a tile. p is
// rounded to the inputs' type, as the tensor cores' operand; the sum adds p unrounded.
//
// Rows and keys behind a sample's end are other samples': s is replaced by -inf there, p v stops at the last 16 keys that
// hold one of the sample's, and the rows of v behind it in those are zeroed in shared memory (0 times an
// infinity or a NaN of another sample would not be 0).
//
// Every wait is bounded; a timeout raises SPCONV_STATUS_WAIT_TIMEOUT, and the CTA waits out its copies and products
// before it frees TMEM and exits.
#include <algorithm>

#include "attention_tc.cuh"

namespace spconv {

constexpr float kAfSlack = 8.f;                      // by how much the maximum in use may be exceeded, in powers of two

template <int NQ, int DP>
struct AfShape {
    static constexpr int kThreads = NQ * 128 + 64;
    static constexpr int kTile = DP / 64 * kAtBlock;
    static constexpr int kStages = NQ == 2 ? (DP == 64 ? 8 : 4) : (DP == 64 ? 5 : 2);
    static constexpr int kSmem = 1024 + (NQ + kStages) * kTile + 512;
    // no more CTAs than the SM's 512 columns serve
    static constexpr int kSmemLeast = NQ == 2 ? 120 * 1024 : 80 * 1024;
    static constexpr int kColumns = NQ == 2 ? 512 : 256;
    static constexpr int kAcc = NQ * 128;            // first column of the accumulators
};

template <typename T, int NQ, int DP>
__global__ void __launch_bounds__(NQ * 128 + 64, NQ == 2 ? 1 : 2)
attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AtArgs a, const int log_p) {
    using S = AfShape<NQ, DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t s_q = smem_u32(base), s_ring = s_q + NQ * S::kTile;
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + (NQ + S::kStages) * S::kTile);
    uint64_t *full = bar, *empty = full + S::kStages, *qfull = empty + S::kStages, *tail = qfull + 1, *sfull = tail + 1, *pready = sfull + NQ;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(pready + NQ);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 1);
    AtSample *s_sample = reinterpret_cast<AtSample *>(s_tmem + 2);
    constexpr int kWarpLoad = NQ * 4, kWarpMma = NQ * 4 + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int P = 1 << log_p, tokens = kAtRows >> log_p;             // tokens of a tile

    at_check_offsets(a);
    if (warp == kWarpLoad) {
        // the last tiles of a causal sample see most: they go first
        const AtSample s = at_find(a.offsets, a.M, a, a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x, NQ * tokens);
        if (lane == 0) *s_sample = s;
    }
    if (tid == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&empty[i]), 1);
        }
        mbar_init(smem_u32(qfull), 1);
        mbar_init(smem_u32(tail), 1);
        for (int q = 0; q < NQ; ++q) {
            mbar_init(smem_u32(&sfull[q]), 1);
            mbar_init(smem_u32(&pready[q]), 4);
        }
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncthreads();
    const AtSample s = *s_sample;
    const int n = s.q1 - s.q0, m = s.k1 - s.k0, t0 = s.tile * NQ * tokens;        // the CTA's first token in the sample
    if (s.tile < 0 || t0 >= n) return;                                           // uniform over the CTA
    if (warp == kWarpMma) {
        tmem_alloc(smem_u32(s_tmem), S::kColumns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    const int head0 = blockIdx.y << log_p, kh = head0 / (a.H / a.K);
    const int nq = NQ == 2 && t0 + tokens < n ? 2 : 1;               // tiles with a row in them
    const int seen_last = at_seen(a, min(n, t0 + nq * tokens) - 1, n, m);
    int first, last;
    at_split(a.splits, blockIdx.z, (seen_last + kAtRows - 1) / kAtRows, first, last);
    const int tiles = last - first;
    const int end_valid = min(kAtRows, seen_last - (last - 1) * kAtRows);      // keys of the last tile (of this split)
    auto wait = [&](uint64_t *b, uint32_t parity) { return mbar_wait_suspended(smem_u32(b), parity, s_abort, a.wait_ns); };
    auto next = [](int &i, uint32_t &phase) {
        if (++i == S::kStages) {
            i = 0;
            phase ^= 1u;
        }
    };

    if (warp == kWarpLoad) {
        // ------------------------------------------------------------------ loads: q; then k, v of each tile in turn
        if (tiles > 0) {
            if (elect_one()) {
                mbar_arrive_expect_tx(smem_u32(qfull), (uint32_t)(nq * S::kTile));
                for (int q = 0; q < nq; ++q)
                    for (int c = 0; c < DP / 64; ++c)
                        tma_load_3d(s_q + q * S::kTile + c * kAtBlock, &map_q, c * 64, head0, s.q0 + t0 + q * tokens, smem_u32(qfull));
            }
            __syncwarp();
            int st = 0;
            uint32_t phase = 1;                                      // the first use of a stage passes at once
            bool ok = true;
            for (int i = 0; i < 2 * tiles && ok; ++i, next(st, phase)) {
                const bool is_v = i & 1, cut = is_v && i + 1 == 2 * tiles && (end_valid & 15);
                ok = __all_sync(0xffffffffu, wait(&empty[st], phase)) != 0;
                if (!ok) break;
                const uint32_t dst = s_ring + st * S::kTile;
                if (elect_one()) {
                    const uint32_t mbar = smem_u32(cut ? tail : &full[st]);
                    mbar_arrive_expect_tx(mbar, S::kTile);
                    for (int c = 0; c < DP / 64; ++c)
                        tma_load_3d(dst + c * kAtBlock, is_v ? &map_v : &map_k, c * 64, kh, s.k0 + (first + (i >> 1)) * kAtRows, mbar);
                }
                __syncwarp();
                if (cut) {
                    ok = __all_sync(0xffffffffu, wait(tail, 0)) != 0;
                    at_zero_rows<DP>(dst, end_valid, (end_valid + 15) & ~15);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&full[st]));
                }
            }
        }
    } else if (warp == kWarpMma) {
        // ------------------------------------------------------------------ products
        if (tiles > 0 && elect_one()) {
            const uint32_t id_s = instr_desc_f16(dtype_traits<T>::mma_format, 128, 128);
            const uint32_t id_o = instr_desc_f16(dtype_traits<T>::mma_format, 128, (a.D + 15) & ~15) | 1u << 16;
            const int steps = (a.D + 15) >> 4;
            int st = 0;
            uint32_t phase = 0, p_phase = 0;
            bool ok = wait(qfull, 0) && wait(&full[0], 0);
            if (ok) {
                tc_fence_after();
                for (int q = 0; q < nq; ++q) {
                    at_mma_head<DP>(tmem + q * 128, s_q + q * S::kTile, s_ring, id_s, steps);
                    tc_commit(smem_u32(&sfull[q]));
                }
                tc_commit(smem_u32(&empty[0]));
                next(st, phase);
            }
            for (int j = 0; j < tiles && ok; ++j, p_phase ^= 1u) {
                const int v_st = st;
                const uint32_t v_phase = phase;
                next(st, phase);
                const bool more = j + 1 < tiles;
                const int rows = more ? 8 : (end_valid + 15) >> 4;
                if (!(ok = wait(&full[v_st], v_phase))) break;
                for (int q = 0; q < nq; ++q) {
                    if (!(ok = wait(&pready[q], p_phase))) break;
                    if (more && q == 0 && !(ok = wait(&full[st], phase))) break;
                    tc_fence_after();
                    at_mma_rows(tmem + S::kAcc + q * DP, tmem + q * 128, 0, s_ring + v_st * S::kTile, id_o, rows, j > 0);
                    if (more) at_mma_head<DP>(tmem + q * 128, s_q + q * S::kTile, s_ring + st * S::kTile, id_s, steps);
                    tc_commit(smem_u32(&sfull[q]));
                }
                if (!ok) break;
                tc_commit(smem_u32(&empty[v_st]));
                if (more) {
                    tc_commit(smem_u32(&empty[st]));
                    next(st, phase);
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax: a thread a row
        const int q = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + q * 128 + lanes, t_o = tmem + S::kAcc + q * DP + lanes;
        const int token = t0 + q * tokens + (row >> log_p);          // in the sample
        const bool mine = token < n;
        const int seen = mine ? at_seen(a, token, n, m) : 0;
        const bool some = __any_sync(0xffffffffu, mine);
        // keys that every row of the warp sees: tiles up to there need no mask
        const int seen_all = __reduce_min_sync(0xffffffffu, mine ? seen : m);
        float top = -INFINITY, sum = 0.f;                            // of s; of p
        bool ok = true;
        uint32_t phase = 0;
        if (q < nq) {
            for (int j = 0; j < tiles; ++j, phase ^= 1u) {
                if (!(ok = __all_sync(0xffffffffu, wait(&sfull[q], phase)) != 0)) break;
                tc_fence_after();
                if (some) {
                    f32x2 x[64];
#pragma unroll
                    for (int g = 0; g < 4; ++g) lt_load32(t_s + g * 32, *reinterpret_cast<f32x2(*)[16]>(x + g * 16));
                    const int key0 = (first + j) * kAtRows;
                    if (key0 + kAtRows > seen_all) {
                        const int left = seen - key0;
#pragma unroll
                        for (int i = 0; i < 64; ++i) {
                            const float2 f = unpack_f32x2(x[i]);
                            x[i] = pack_f32x2(2 * i < left ? f.x : -INFINITY, 2 * i + 1 < left ? f.y : -INFINITY);
                        }
                    }
                    float big[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        const float2 f = unpack_f32x2(x[i]);
                        big[i & 3] = fmaxf(big[i & 3], fmaxf(f.x, f.y));
                    }
                    const float now = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
                    // a maximum that has grown by more than the slack (from -inf: by any amount) is taken over
                    const bool grown = (now - top) * a.c > kAfSlack;
                    if (__any_sync(0xffffffffu, grown)) {
                        const float down = grown ? ex2_approx((top - now) * a.c) : 1.f;
                        if (grown) top = now;
                        sum *= down;
                        if (j > 0) {                                 // every product that wrote out is done: s came after it
                            const f32x2 d2 = pack_f32x2(down, down);
#pragma unroll 1
                            for (int c = 0; c < DP; c += 32) {
                                f32x2 o[16];
                                lt_load32(t_o + c, o);
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = mul2(o[i], d2);
                                tmem_st32(t_o + c, *reinterpret_cast<const uint32_t(*)[32]>(o));
                            }
                        }
                    }
                    const float shift = top == -INFINITY ? 0.f : -top * a.c;
                    const f32x2 c2 = pack_f32x2(a.c, a.c), s2 = pack_f32x2(shift, shift);
                    f32x2 add[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float2 f = unpack_f32x2(fma2(x[g * 32 + i], c2, s2));
                            const float p0 = ex2_approx(f.x), p1 = ex2_approx(f.y);
                            add[i & 1] = add2(add[i & 1], pack_f32x2(p0, p1));
                            w[i] = lt_pack<T>(p0, p1);
                        }
                        tmem_st32(t_s + g * 32, w);
                    }
                    const float2 f = unpack_f32x2(add2(add[0], add[1]));
                    sum += f.x + f.y;
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&pready[q]));
            }
            if (tiles > 0 && ok) ok = __all_sync(0xffffffffu, wait(&sfull[q], phase)) != 0;    // the last p v
            tc_fence_after();
            if (ok && some) {
                const int64_t all = (int64_t)a.M * a.H, at = (int64_t)(s.q0 + token) * a.H + head0 + (row & (P - 1));
                const bool none = seen == 0;
                float *part = nullptr;
                float inv = none ? 0.f : 1.f / sum;
                if (a.splits > 1) {
                    part = a.partial + (blockIdx.z * all + at) * a.D;
                    inv = 1.f;
                    if (mine) a.part_ml[blockIdx.z * all + at] = make_float2(top * a.c, sum);
                } else if (mine && a.lse) {
                    a.lse[at] = none ? INFINITY : fmaf(top, a.c, log2f(sum));
                }
                T *out = (T *)a.out + at * a.D;
                const bool wide = (a.D & 7) == 0 && ((uintptr_t)a.out & 15) == 0;
#pragma unroll 1
                for (int c = 0; c < a.D; c += 32) {
                    f32x2 o[16];
                    if (tiles > 0) {
                        lt_load32(t_o + c, o);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = pack_f32x2(0.f, 0.f);
                    }
                    if (!mine || (part && tiles == 0)) continue;
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        if (c + v * 8 >= a.D) break;
                        uint32_t w[4];
                        float f[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 u = unpack_f32x2(o[v * 4 + i]);
                            f[2 * i] = none ? 0.f : u.x * inv;
                            f[2 * i + 1] = none ? 0.f : u.y * inv;
                            w[i] = lt_pack<T>(f[2 * i], f[2 * i + 1]);
                        }
                        const int d = c + v * 8;
                        if (part) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (d + i < a.D) part[d + i] = f[i];
                        } else if (wide) {
                            *(uint4 *)(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (d + i < a.D) out[d + i] = dtype_traits<T>::from_f(f[i]);
                        }
                    }
                }
            }
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
    if (warp == kWarpMma) tmem_dealloc(tmem, S::kColumns);
}

template <typename T, int NQ, int DP>
static int af_run(const AtArgs &a) {
    using S = AfShape<NQ, DP>;
    const int G = a.H / a.K;
    int log_p = 0;
    while (log_p < 7 && G % (2 << log_p) == 0) ++log_p;
    const int P = 1 << log_p, tokens = kAtRows >> log_p;
    CUtensorMap mq, mk, mv;
    if (!at_map(&mq, a.q, a.M, a.H, a.D, P, tokens) || !at_map(&mk, a.k, a.N, a.K, a.D, 1, kAtRows) ||
        !at_map(&mv, a.v, a.N, a.K, a.D, 1, kAtRows))
        return SPCONV_ERR_CUDA;
    static std::atomic<uint64_t> done;
    auto kern = attention_tc_kernel<T, NQ, DP>;
    constexpr int smem = S::kSmem > S::kSmemLeast ? S::kSmem : S::kSmemLeast;
    if (allow_smem(kern, smem, done) != cudaSuccess) return check_launch("attention: shared memory");
    kern<<<dim3((unsigned)at_tiles(a.M, a.B, NQ * tokens), a.H / P, a.splits), S::kThreads, smem, a.stream>>>(mq, mk, mv, a, log_p);
    return check_launch("attention_tc_kernel");
}

template <typename T>
static int af_shape(const AtArgs &a, int tiles2) {
    if (a.D <= 64) return tiles2 ? af_run<T, 2, 64>(a) : af_run<T, 1, 64>(a);
    return tiles2 ? af_run<T, 2, 128>(a) : af_run<T, 1, 128>(a);
}

int launch_at_tc_forward(const AtArgs &a, int tiles2) {
    return a.dtype == SPCONV_F16 ? af_shape<__half>(a, tiles2) : af_shape<__nv_bfloat16>(a, tiles2);
}

}  // namespace spconv
