// Attention's forward on the 5th-generation tensor cores (tcgen05 / TMEM), fp16 and bf16, heads of up to 128 values:
//
//   s = q k^T (fp32, TMEM);  p = 2^(s c - m);  out = (p v) / sum p,   c = scale log2(e), m a running maximum of s c
//
// A CTA owns tiles of 128 query rows of one key head and walks the sample's keys; four warps a tile do the softmax, a
// thread a row. s arrives in TMEM, its row goes to registers whole, p goes back over it in 16 bits, and is the A operand of
// p v from there; the rows of v are read along the keys (MN-major), so nothing is transposed.
//
// A step is a chain: products, softmax, products; each barrier that another warp completes costs about 170 clocks, a
// product's end 250, and the 64 exponentials a row 520 of the special functions' time. What fills the gaps is other chains:
//   * attention_tc_kernel: one tile a CTA, 64 keys a step, four CTAs an SM (two for heads over 64): 128 columns of TMEM and
//     48 KB each. A fifth warp does both loads and products. 84,000 voxels in 16 scenes, 8 x 64 bf16: 1.32 ms, 0.73 PFLOP/s, in
//     launches apart from one another (as all times here; back to back, at the clocks that the power limit leaves, 1.45 ms)
//     (three CTAs an SM 1.56; one CTA of two tiles and 128 keys a step, whose two chains fell into step with one another,
//     1.69; the same with the next scores made ahead of p v 1.48; two threads a row 2.02). At 8,192
//     tokens x 16 x 64 the special functions are 67 % in use, the issue slots 49 %, the tensor pipe 33 %. One pooling query a
//     scene over 2.0 M voxels: 120 us, 4.3 TB/s, and 15 to join the splits.
//   * attention_tc_pair_kernel, for long samples of heads over 64, whose accumulators leave TMEM for two chains only: two
//     tiles a CTA, which share k and v, 128 keys a step, and registers dealt out anew so that a row of 128 scores fits: 4 x 128
//     there 0.93 ms, 1.04 PFLOP/s (two CTAs of the kernel above 1.21 ms).
//
// The maximum is followed lazily: while a row's new maximum exceeds the one in use by at most 8, the old one
// stays (p up to 2^8, and 2^15 in fp16, where it comes times 2^7), so out and the sum are rescaled a few times a row, not once a tile. p is
// rounded to the inputs' type, as the tensor cores' operand; the sum adds p unrounded.
//
// Rows and keys behind a sample's end are other samples': s is replaced by -inf there, p v stops at the last 16 keys that
// hold one of the sample's, and the rows of v behind it in those are zeroed in shared memory (0 times an
// infinity or a NaN of another sample would not be 0).
//
// Every wait is bounded; a timeout raises SPCONV_STATUS_WAIT_TIMEOUT, and the CTA waits out its copies and products
// before it frees TMEM and exits.
#include <algorithm>

#include "attention_hidden.cuh"
#include "attention_tc.cuh"

namespace spconv {

constexpr float kAfSlack = 8.f;                      // by how much the maximum in use may be exceeded, in powers of two

// Powers of two on p: fp16 loses p under 2^-25, of which a row of a hundred thousand keys may have many; with 2^7, the most that the
// slack leaves below fp16's largest value, under 2^-32. Exact, and out again with the sum.
template <typename T>
constexpr float kAfUp = dtype_traits<T>::mma_format == 0 ? 7.f : 0.f;

// A row's result: its accumulators over its sum, zeros if it sees no key (of this split); or, where keys are split, the
// accumulators as they are. A warp's lanes together.
template <typename T, bool CAUSAL>
__device__ __forceinline__ void af_store(const AtArgs &a, uint32_t t_o, int size, const AtHidden &row, bool mine, bool nothing, float top,
                                         float sum) {
    const int64_t all = (int64_t)a.M * a.H, at = row.row * a.H + row.head;
    bool none = row.seen <= row.lo;
    f32x2 lost = pack_f32x2(0.f, 0.f);                               // NaN once a value was not finite
    float *part = a.splits > 1 ? a.partial + (blockIdx.z * all + at) * a.D : nullptr;
    const float inv = part ? 1.f : none ? 0.f : 1.f / sum;
    if (mine) {
        if (part) a.part_ml[blockIdx.z * all + at] = make_float2(fmaf(top, a.c, -kAfUp<T>), none ? -1.f : sum);
        else if (a.lse) a.lse[at] = none ? INFINITY : fmaf(top, a.c, log2f(sum) - kAfUp<T>);
    }
    T *out = (T *)a.out + at * a.D;
    const bool wide = (a.D & 7) == 0 && (((uintptr_t)a.out | (uintptr_t)a.rest) & 15) == 0;
    const bool whole = (a.D & 15) == 0 && (((uintptr_t)a.out | (uintptr_t)a.rest) & 31) == 0;
#pragma unroll 1
    for (int c = 0; c < size && c < a.D; c += 16) {
        uint32_t o[16];
        __syncwarp();                                                // lanes without a row come here before those that store
        if (!nothing) {                                              // there were keys, the same for every lane
            tmem_ld16(t_o + c, o);
            tc_wait_ld();
        }
        if (!mine || (part && nothing)) continue;
        none |= nothing;
        if constexpr (CAUSAL) {
#pragma unroll
            for (int i = 0; i < 16; i += 2) lost = fma2(pack_f32x2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), pack_f32x2(0.f, 0.f), lost);
        }
        if (!part && whole) {
            // a lane's 16 values are a sector: out and rest of voxels to 257 tokens 334 -> 252 us (out alone 240 -> 236)
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = none ? 0u : lt_pack<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
            at_store32(out + c, w);
            if (a.rest) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 hi = lt_unpack<T>(w[i]);
                    w[i] = none ? 0u : lt_pack<T>(fmaf(__uint_as_float(o[2 * i]), inv, -hi.x), fmaf(__uint_as_float(o[2 * i + 1]), inv, -hi.y));
                }
                at_store32((T *)a.rest + at * a.D + c, w);
            }
            continue;
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int d = c + v * 8;
            if (d >= a.D) break;
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = none ? 0.f : __uint_as_float(o[v * 8 + i]) * inv;
            if (part && (a.D & 7) == 0) {                            // (the workspace is aligned, and so are rows of eights)
                *(float4 *)(part + d) = make_float4(f[0], f[1], f[2], f[3]);
                *(float4 *)(part + d + 4) = make_float4(f[4], f[5], f[6], f[7]);
            } else if (part) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (d + i < a.D) part[d + i] = f[i];
            } else if (wide) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = lt_pack<T>(f[2 * i], f[2 * i + 1]);
                *(uint4 *)(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
                if (a.rest) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 hi = lt_unpack<T>(w[i]);
                        w[i] = lt_pack<T>(f[2 * i] - hi.x, f[2 * i + 1] - hi.y);
                    }
                    *(uint4 *)((T *)a.rest + at * a.D + d) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (d + i < a.D) at_put<T>(a, at * a.D + d + i, f[i]);
            }
        }
    }
    const float2 z = unpack_f32x2(lost);
    if (CAUSAL && !(z.x + z.y == 0.f) && !none && row.seen < row.hi && sum == sum)
        at_values_again<T>(a, row, fmaf(-top, a.c, kAfUp<T>), inv, part);
}

// A CTA a tile of queries.
template <int DP>
struct AfShape {
    static constexpr int kKeys = 64, kStages = 2, kPerSm = DP == 64 ? 4 : 2;
    static constexpr int kOwn = DP / 64 * kAtBlock, kTile = kOwn / 2;            // bytes of a tile of queries, and of keys or values
    static constexpr int kSmem = 1024 + kOwn + 2 * kStages * kTile + 256, kSmemLeast = 228 * 1024 / (kPerSm + 1);
    static constexpr int kColumns = 512 / kPerSm;    // scores, p over them; accumulators
    static constexpr int kThreads = 160, kControl = 4;
};

template <typename T, int DP, bool CAUSAL>
__global__ void __launch_bounds__(AfShape<DP>::kThreads, AfShape<DP>::kPerSm)
attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AtArgs a, const int log_p) {
    using S = AfShape<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t s_q = smem_u32(base), s_k = s_q + S::kOwn, s_v = s_k + S::kStages * S::kTile;
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + S::kOwn + 2 * S::kStages * S::kTile);
    uint64_t *kfull = bar, *vfull = kfull + S::kStages, *qfull = vfull + S::kStages, *sfull = qfull + 1, *pready = sfull + 1;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(pready + 1);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 1);
    AtSample *s_sample = reinterpret_cast<AtSample *>(s_tmem + 2);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int P = 1 << log_p, tokens = kAtRows >> log_p;             // tokens of a tile

    const int head0 = blockIdx.y << log_p, kh = head0 / (a.H / a.K);
    auto load = [&](uint32_t dst, const CUtensorMap *map, int head, int row, int bytes, uint64_t *b) {
        mbar_arrive_expect_tx(smem_u32(b), bytes);
        for (int c = 0; c < DP / 64; ++c) tma_load_3d(dst + c * (bytes / (DP / 64)), map, c * 64, head, row, smem_u32(b));
    };
    // what a sample gives the CTA: its first token, keys, and tiles of them in this split
    int n, m, t0, first, tiles, end_valid;
    AtSample s = {};
    auto share = [&] {
        n = s.q1 - s.q0;
        m = s.k1 - s.k0;
        t0 = s.tile * tokens;
        const int seen_last = at_seen(a, min(n, t0 + tokens) - 1, n, m);
        int last;
        at_split(a.splits, blockIdx.z, (seen_last + S::kKeys - 1) / S::kKeys, first, last);
        tiles = s.tile < 0 || t0 >= n ? -1 : last - first;           // -1: nothing to do at all
        end_valid = min(S::kKeys, seen_last - (last - 1) * S::kKeys);            // keys of the last tile (of this split)
    };
    auto load_tile = [&](int j) {
        const int row = s.k0 + (first + j) * S::kKeys, st = j & 1;
        load(s_k + st * S::kTile, &map_k, kh, row, S::kTile, &kfull[st]);
        load(s_v + st * S::kTile, &map_v, kh, row, S::kTile, &vfull[st]);
    };

    at_check_offsets(a);
    if (warp == S::kControl) {
        // Everything up to the first loads by this warp alone: a short sample's time is mostly this way (TMEM's
        // allocation, by another warp, and the samples' search go on at the same time).
        if (elect_one()) {
            tma_prefetch_desc(&map_q);
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
            for (int i = 0; i < S::kStages; ++i) {
                mbar_init(smem_u32(&kfull[i]), 1);
                mbar_init(smem_u32(&vfull[i]), 1);
            }
            mbar_init(smem_u32(qfull), 1);
            mbar_init(smem_u32(sfull), 1);
            mbar_init(smem_u32(pready), 4);
            *s_abort = 0;
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
        // the last tiles of a causal sample see most: they go first
        s = at_find(a, false, a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x, tokens);
        share();
        if (lane == 0) *s_sample = s;
        if (tiles > 0 && elect_one()) {
            load(s_q, &map_q, head0, s.q0 + t0, S::kOwn, qfull);
            load_tile(0);
            if (tiles > 1) load_tile(1);
        }
        __syncwarp();
    } else if (warp == 0) {
        tmem_alloc(smem_u32(s_tmem), S::kColumns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp != S::kControl) {
        s = *s_sample;
        share();
    }
    const uint32_t tmem = *s_tmem;
    auto wait = [&](uint64_t *b, uint32_t parity) {
        return __all_sync(0xffffffffu, at_wait(b, parity, s_abort, a.wait_ns)) != 0;
    };

    if (warp == S::kControl) {
        // ------------------------------------------------------------------ loads and products
        if (tiles > 0) {
            const uint32_t id_s = instr_desc_f16(dtype_traits<T>::mma_format, 128, S::kKeys);
            const uint32_t id_o = instr_desc_f16(dtype_traits<T>::mma_format, 128, (a.D + 15) & ~15) | 1u << 16;
            const int steps = (a.D + 15) >> 4;
            bool ok = wait(qfull, 0);
            for (int j = 0; j <= tiles && ok; ++j) {
                const int st = j & 1, v = st ^ 1;
                const bool end = j == tiles;
                // what is waited for first is long there when p is
                if (!end && !(ok = wait(&kfull[st], (j >> 1) & 1))) break;
                if (j > 0) {
                    if (!(ok = wait(&vfull[v], ((j - 1) >> 1) & 1))) break;
                    if (end && (end_valid & 15)) {
                        at_zero_rows<DP, S::kKeys>(s_v + v * S::kTile, end_valid, (end_valid + 15) & ~15);
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (!(ok = wait(pready, (j - 1) & 1))) break;
                }
                tc_fence_after();
                if (elect_one()) {                                   // p v of the tile before, then the next scores over p
                    if (j > 0)
                        at_mma_rows<S::kKeys, S::kKeys>(tmem + S::kKeys, tmem, s_v + v * S::kTile, id_o, end ? (end_valid + 15) >> 4 : S::kKeys / 16, j > 1);
                    if (!end) at_mma_head<DP, S::kKeys>(tmem, s_q, s_k + st * S::kTile, id_s, steps);
                    tc_commit(smem_u32(sfull));
                }
                __syncwarp();
                if (j > 0 && j + 1 < tiles) {                        // the tile before is done with: its stage takes the next
                    if (!(ok = wait(sfull, j & 1))) break;
                    if (elect_one()) load_tile(j + 1);
                    __syncwarp();
                }
            }
        }
    } else if (tiles >= 0) {
        // ------------------------------------------------------------------ softmax: a thread a row
        const uint32_t t_s = tmem + ((uint32_t)(warp * 32) << 16), t_o = t_s + S::kKeys;
        const int token = t0 + (tid >> log_p);                       // in the sample
        const bool mine = token < n;
        const int seen = mine ? at_seen(a, token, n, m) : 0;
        const bool some = __any_sync(0xffffffffu, mine);
        // keys that every row of the warp sees: tiles up to there need no mask
        const int seen_all = __reduce_min_sync(0xffffffffu, mine ? seen : m);
        float top = -INFINITY, sum = 0.f;                            // of s; of p
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            if (!(ok = wait(sfull, j & 1))) break;
            tc_fence_after();
            if (some) {
                f32x2 x[32];
                at_load(t_s, x);
                const int key0 = (first + j) * S::kKeys;
                if (key0 + S::kKeys > seen_all) {
                    const int left = seen - key0;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 f = unpack_f32x2(x[i]);
                        x[i] = pack_f32x2(2 * i < left ? f.x : -INFINITY, 2 * i + 1 < left ? f.y : -INFINITY);
                    }
                }
                float big[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float2 f = unpack_f32x2(x[i]);
                    big[i & 3] = max3_nan(big[i & 3], f.x, f.y);
                }
                const float now = max3_nan(max3_nan(big[0], big[1], big[2]), big[3], big[3]);
                // a maximum that has grown by more than the slack (from -inf: by any amount), or is NaN, is taken over
                const bool grown = !((now - top) * a.c <= kAfSlack) && now != -INFINITY;
                if (__any_sync(0xffffffffu, grown)) {
                    const float down = grown ? ex2_approx((top - now) * a.c) : 1.f;
                    if (grown) top = now;
                    sum *= down;
                    if (j > 0) {                                     // the products before are done: s came after them
                        __syncwarp();
#pragma unroll 1
                        for (int c = 0; c < DP; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(t_o + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
                            tmem_st16(t_o + c, o);
                        }
                    }
                }
                const float shift = top == -INFINITY ? 0.f : fmaf(-top, a.c, kAfUp<T>);
                const f32x2 c2 = pack_f32x2(a.c, a.c), s2 = pack_f32x2(shift, shift);
                f32x2 add[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const f32x2 e = at_exp2(fma2(x[g * 16 + i], c2, s2));
                        const float2 f = unpack_f32x2(e);
                        add[i & 1] = add2(add[i & 1], e);
                        w[i] = lt_pack<T>(f.x, f.y);
                    }
                    tmem_st16(t_s + g * 16, w);
                }
                const float2 f = unpack_f32x2(add2(add[0], add[1]));
                sum += f.x + f.y;
                tc_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(pready));
        }
        if (tiles > 0 && ok) ok = wait(sfull, tiles & 1);            // the last p v
        tc_fence_after();
        if (ok && some)
            af_store<T, CAUSAL>(a, t_o, DP, AtHidden{s.q0 + token, head0 + (tid & (P - 1)), kh, s.k0, first * S::kKeys, seen,
                                             min(m, (first + tiles) * S::kKeys)}, mine, tiles == 0, top, sum);
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

// Heads of more than 64 values: two tiles of queries a CTA, keys 128 at a time.
struct ApShape {
    static constexpr int kThreads = 384, kWarpLoad = 8, kWarpMma = 9;
    // registers: launched with 168 a thread, dealt out anew: 224 x 256 + 56 x 128 = 168 x 384
    static constexpr int kRegs = 224, kRegsOther = 56;
    static constexpr int kTile = 2 * kAtBlock, kStages = 4;
    static constexpr int kSmem = 1024 + (2 + kStages) * kTile + 256, kSmemLeast = 120 * 1024;
    static constexpr int kAcc = 256;                 // first column of the accumulators, behind two tiles' scores
};

template <typename T, bool CAUSAL>
__global__ void __launch_bounds__(ApShape::kThreads, 1)
attention_tc_pair_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AtArgs a, const int log_p) {
    using S = ApShape;
    constexpr int DP = 128;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t s_q = smem_u32(base), s_ring = s_q + 2 * S::kTile;
    uint64_t *bar = reinterpret_cast<uint64_t *>(base + (2 + S::kStages) * S::kTile);
    uint64_t *full = bar, *empty = full + S::kStages, *qfull = empty + S::kStages, *tail = qfull + 1, *sfull = tail + 1;
    uint64_t *pready = sfull + 2, *odone = pready + 2;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(odone + 2);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 1);
    AtSample *s_sample = reinterpret_cast<AtSample *>(s_tmem + 2);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int P = 1 << log_p, tokens = kAtRows >> log_p;             // tokens of a tile

    at_check_offsets(a);
    if (warp == S::kWarpLoad) {
        // the last tiles of a causal sample see most: they go first
        const AtSample s = at_find(a, false, a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x, 2 * tokens);
        if (lane == 0) *s_sample = s;
    }
    if (tid == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&empty[i]), 1);
        }
        mbar_init(smem_u32(qfull), 1);
        mbar_init(smem_u32(tail), 1);
        for (int q = 0; q < 2; ++q) {
            mbar_init(smem_u32(&sfull[q]), 1);
            mbar_init(smem_u32(&pready[q]), 4);
            mbar_init(smem_u32(&odone[q]), 1);
        }
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncthreads();
    const AtSample s = *s_sample;
    const int n = s.q1 - s.q0, m = s.k1 - s.k0, t0 = s.tile * 2 * tokens;        // the CTA's first token in the sample
    if (s.tile < 0 || t0 >= n) return;                                           // uniform over the CTA
    if (warp == S::kWarpMma) {
        tmem_alloc(smem_u32(s_tmem), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    const int head0 = blockIdx.y << log_p, kh = head0 / (a.H / a.K);
    const int nq = t0 + tokens < n ? 2 : 1;               // tiles with a row in them
    const int seen_last = at_seen(a, min(n, t0 + nq * tokens) - 1, n, m);
    int first, last;
    at_split(a.splits, blockIdx.z, (seen_last + kAtRows - 1) / kAtRows, first, last);
    const int tiles = last - first;
    const int end_valid = min(kAtRows, seen_last - (last - 1) * kAtRows);      // keys of the last tile (of this split)
    auto wait = [&](uint64_t *b, uint32_t parity) { return at_wait(b, parity, s_abort, a.wait_ns); };
    auto next = [](int &i, uint32_t &phase) {
        if (++i == S::kStages) {
            i = 0;
            phase ^= 1u;
        }
    };

    // each share of the registers is set inside its roles' branch: behind a join the compiler would keep to the smaller
    if (warp >= S::kWarpLoad) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" :: "n"(S::kRegsOther));
        if (warp == S::kWarpLoad) {
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
                    const bool is_v = i & 1;
                    const int tile = i >> 1;
                    const bool cut = is_v && tile + 1 == tiles && (end_valid & 15);
                    ok = __all_sync(0xffffffffu, wait(&empty[st], phase)) != 0;
                    if (!ok) break;
                    const uint32_t dst = s_ring + st * S::kTile;
                    if (elect_one()) {
                        const uint32_t mbar = smem_u32(cut ? tail : &full[st]);
                        mbar_arrive_expect_tx(mbar, S::kTile);
                        for (int c = 0; c < DP / 64; ++c)
                            tma_load_3d(dst + c * kAtBlock, is_v ? &map_v : &map_k, c * 64, kh, s.k0 + (first + tile) * kAtRows, mbar);
                    }
                    __syncwarp();
                    if (cut) {
                        ok = __all_sync(0xffffffffu, wait(tail, 0)) != 0;
                        at_zero_rows<DP, kAtRows>(dst, end_valid, (end_valid + 15) & ~15);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&full[st]));
                    }
                }
            }
        } else if (warp == S::kWarpMma) {
            // ------------------------------------------------------------------ products
            if (tiles > 0 && elect_one()) {
                const uint32_t id_s = instr_desc_f16(dtype_traits<T>::mma_format, 128, 128);
                const uint32_t id_o = instr_desc_f16(dtype_traits<T>::mma_format, 128, (a.D + 15) & ~15) | 1u << 16;
                const int steps = (a.D + 15) >> 4;
                // the ring holds k0, v0, k1, v1, ..
                auto landed = [&](int at) { return wait(&full[at % S::kStages], (at / S::kStages) & 1); };
                auto release = [&](int at) { tc_commit(smem_u32(&empty[at % S::kStages])); };
                auto stage = [&](int at) { return s_ring + at % S::kStages * S::kTile; };
                bool ok = wait(qfull, 0);
                auto scores = [&](int q, int i) {                        // s of tile i
                    if (!(ok = ok && landed(2 * i))) return;
                    tc_fence_after();
                    at_mma_head<DP, kAtRows>(tmem + q * 128, s_q + q * S::kTile, stage(2 * i), id_s, steps);
                    tc_commit(smem_u32(&sfull[q]));
                    if (q + 1 == nq) release(2 * i);
                };
                for (int q = 0; q < nq; ++q) scores(q, 0);
                for (int i = 0; i < tiles && ok; ++i)
                    for (int q = 0; q < nq && ok; ++q) {                 // p v of tile i, then the next scores over p
                        if (!(ok = wait(&pready[q], i & 1) && landed(2 * i + 1))) break;
                        tc_fence_after();
                        at_mma_rows<128, kAtRows>(tmem + S::kAcc + q * DP, tmem + q * 128, stage(2 * i + 1), id_o,
                                                  i + 1 < tiles ? 8 : (end_valid + 15) >> 4, i > 0);
                        tc_commit(smem_u32(&odone[q]));
                        if (q + 1 == nq) release(2 * i + 1);
                        if (i + 1 < tiles) scores(q, i + 1);
                    }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" :: "n"(S::kRegs));
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
                    at_load(t_s, x);
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
                        big[i & 3] = max3_nan(big[i & 3], f.x, f.y);
                    }
                    const float now = max3_nan(max3_nan(big[0], big[1], big[2]), big[3], big[3]);
                    // a maximum that has grown by more than the slack (from -inf: by any amount), or is NaN, is taken over
                    const bool grown = !((now - top) * a.c <= kAfSlack) && now != -INFINITY;
                    if (__any_sync(0xffffffffu, grown)) {
                        const float down = grown ? ex2_approx((top - now) * a.c) : 1.f;
                        if (grown) top = now;
                        sum *= down;
                        if (j > 0) {                                 // the products before are done: s came after them
                            const f32x2 d2 = pack_f32x2(down, down);
                            __syncwarp();
#pragma unroll 1
                            for (int c = 0; c < DP; c += 32) {
                                f32x2 o[16];
                                lt_load32(t_o + c, o);
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = mul2(o[i], d2);
                                tmem_st16(t_o + c, reinterpret_cast<const uint32_t *>(o));
                                tmem_st16(t_o + c + 16, reinterpret_cast<const uint32_t *>(o + 8));
                            }
                        }
                    }
                    const float shift = top == -INFINITY ? 0.f : fmaf(-top, a.c, kAfUp<T>);
                    const f32x2 c2 = pack_f32x2(a.c, a.c), s2 = pack_f32x2(shift, shift);
                    f32x2 add[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const f32x2 e = at_exp2(fma2(x[g * 16 + i], c2, s2));
                            const float2 f = unpack_f32x2(e);
                            add[i & 1] = add2(add[i & 1], e);
                            w[i] = lt_pack<T>(f.x, f.y);
                        }
                        tmem_st16(t_s + g * 16, w);
                    }
                    const float2 f = unpack_f32x2(add2(add[0], add[1]));
                    sum += f.x + f.y;
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&pready[q]));
            }
            if (tiles > 0 && ok) ok = __all_sync(0xffffffffu, wait(&odone[q], (tiles - 1) & 1)) != 0;     // the last p v
            tc_fence_after();
            if (ok && some)
                af_store<T, CAUSAL>(a, t_o, DP, AtHidden{s.q0 + token, head0 + (row & (P - 1)), kh, s.k0, first * kAtRows, seen,
                                                 min(m, (first + tiles) * kAtRows)}, mine, tiles == 0, top, sum);
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
    if (warp == S::kWarpMma) tmem_dealloc(tmem, 512);
}

template <typename T, typename S, bool PAIR, typename K>
static int af_run(const AtArgs &a, K kern, int keys, std::atomic<uint64_t> &done) {
    const int G = a.H / a.K;
    int log_p = 0;
    while (log_p < 7 && G % (2 << log_p) == 0) ++log_p;
    const int P = 1 << log_p, tokens = kAtRows >> log_p;
    CUtensorMap mq, mk, mv;
    if (!at_map(&mq, a.q, a.M, a.H, a.D, P, tokens) || !at_map(&mk, a.k, a.N, a.K, a.D, 1, keys) ||
        !at_map(&mv, a.v, a.N, a.K, a.D, 1, keys))
        return SPCONV_ERR_CUDA;
    // no more CTAs than the SM's 512 columns serve
    constexpr int least = S::kSmemLeast, smem = S::kSmem > least ? S::kSmem : least;
    if (allow_smem(kern, smem, done) != cudaSuccess) return check_launch("attention: shared memory");
    const dim3 grid((unsigned)at_tiles(a.M, a.B, (PAIR ? 2 : 1) * tokens), a.H / P, a.splits);
    kern<<<grid, S::kThreads, smem, a.stream>>>(mq, mk, mv, a, log_p);
    return check_launch("attention_tc_kernel");
}

template <typename T, bool CAUSAL>
static int af_type(const AtArgs &a, bool pair) {
    static std::atomic<uint64_t> done[3];
    if (a.D <= 64) return af_run<T, AfShape<64>, false>(a, attention_tc_kernel<T, 64, CAUSAL>, AfShape<64>::kKeys, done[0]);
    if (!pair) return af_run<T, AfShape<128>, false>(a, attention_tc_kernel<T, 128, CAUSAL>, AfShape<128>::kKeys, done[1]);
    return af_run<T, ApShape, true>(a, attention_tc_pair_kernel<T, CAUSAL>, kAtRows, done[2]);
}
template <bool CAUSAL>
static int af_causal(const AtArgs &a, bool pair) {
    return a.dtype == SPCONV_F16 ? af_type<__half, CAUSAL>(a, pair) : af_type<__nv_bfloat16, CAUSAL>(a, pair);
}

int launch_at_tc_forward(const AtArgs &a, bool pair) { return a.causal ? af_causal<true>(a, pair) : af_causal<false>(a, pair); }

}  // namespace spconv
