// Pairs of fp32 values (the f32x2 instructions of sm_100), and 16 bytes of values
// taken apart into pairs and put together again.
#pragma once
#include "common.cuh"

namespace usaf {

// two fp32 values in one register pair
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// 16 bytes of T as pairs, and back (rounded to the nearest)
template <typename T> constexpr int kPairs = 8 / (int)sizeof(T);

__device__ __forceinline__ uint64_t unpack_word(uint32_t u, __nv_bfloat16) {
    return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ uint64_t unpack_word(uint32_t u, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u));
    return pair(f.x, f.y);
}
__device__ __forceinline__ uint32_t pack_word(float2 f, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_word(float2 f, __half) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T> __device__ __forceinline__ void unpack(const uint4 &u, uint64_t *p) {
    if constexpr (sizeof(T) == 4) {
        p[0] = pair(__uint_as_float(u.x), __uint_as_float(u.y));
        p[1] = pair(__uint_as_float(u.z), __uint_as_float(u.w));
    } else {
        p[0] = unpack_word(u.x, T());
        p[1] = unpack_word(u.y, T());
        p[2] = unpack_word(u.z, T());
        p[3] = unpack_word(u.w, T());
    }
}
template <typename T> __device__ __forceinline__ uint4 pack(const uint64_t *p) {
    if constexpr (sizeof(T) == 4) {
        const float2 a = halves(p[0]), b = halves(p[1]);
        return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    } else {
        return make_uint4(pack_word(halves(p[0]), T()), pack_word(halves(p[1]), T()), pack_word(halves(p[2]), T()),
                          pack_word(halves(p[3]), T()));
    }
}
}  // namespace usaf
