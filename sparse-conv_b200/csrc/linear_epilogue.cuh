// Between accumulators in TMEM, packed fp32 pairs and rounded rows in shared memory.
#pragma once

#include "activation.cuh"
#include "common.cuh"

namespace spconv {

template <typename T>
__device__ __forceinline__ uint32_t lt_pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t lt_pack<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t lt_pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T>
__device__ __forceinline__ float2 lt_unpack(uint32_t v);
template <>
__device__ __forceinline__ float2 lt_unpack<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <>
__device__ __forceinline__ float2 lt_unpack<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// 32 accumulator columns of the lane's row as 16 packed pairs, complete on return. The wait and the
// pairing stand in the same statement as the load so that no copy is needed between them.
__device__ __forceinline__ void lt_load32(uint32_t taddr, f32x2 (&f)[16]) {
    asm volatile(
        "{\n\t.reg .b32 x<32>;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "x0,x1,x2,x3,x4,x5,x6,x7,x8,x9,x10,x11,x12,x13,x14,x15,"
        "x16,x17,x18,x19,x20,x21,x22,x23,x24,x25,x26,x27,x28,x29,x30,x31}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t"
        "mov.b64 %0, {x0,x1}; mov.b64 %1, {x2,x3}; mov.b64 %2, {x4,x5}; mov.b64 %3, {x6,x7}; "
        "mov.b64 %4, {x8,x9}; mov.b64 %5, {x10,x11}; mov.b64 %6, {x12,x13}; mov.b64 %7, {x14,x15}; "
        "mov.b64 %8, {x16,x17}; mov.b64 %9, {x18,x19}; mov.b64 %10, {x20,x21}; mov.b64 %11, {x22,x23}; "
        "mov.b64 %12, {x24,x25}; mov.b64 %13, {x26,x27}; mov.b64 %14, {x28,x29}; mov.b64 %15, {x30,x31}; "
        "}\n"
        : "=l"(f[0].v), "=l"(f[1].v), "=l"(f[2].v), "=l"(f[3].v),
          "=l"(f[4].v), "=l"(f[5].v), "=l"(f[6].v), "=l"(f[7].v),
          "=l"(f[8].v), "=l"(f[9].v), "=l"(f[10].v), "=l"(f[11].v),
          "=l"(f[12].v), "=l"(f[13].v), "=l"(f[14].v), "=l"(f[15].v)
        : "r"(taddr) : "memory");
}

// Eight values, rounded, as one 16-byte store to shared memory.
template <typename T>
__device__ __forceinline__ void lt_store8(uint32_t dst, const f32x2 *f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = unpack_f32x2(f[i]);
        w[i] = lt_pack<T>(x.x, x.y);
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n"
                 :: "r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

}  // namespace spconv
