// Arithmetic on pairs of fp32 values in 64-bit registers (fma, mul, add .f32x2 of sm_100): one issue slot for two elements, each
// rounded as the scalar operation rounds it.
#pragma once

#include "common.cuh"

namespace cgpt {

using Pair = unsigned long long;         // two fp32 values in a 64-bit register

__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ Pair pair(float a) { return pair(a, a); }
__device__ __forceinline__ float2 both(Pair p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float halves_sum(Pair p) {
    const float2 f = both(p);
    return f.x + f.y;
}

template <typename T> __device__ __forceinline__ Pair pair_of(std::uint32_t two);
template <> __device__ __forceinline__ Pair pair_of<__half>(std::uint32_t two) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
    return pair(f.x, f.y);
}
template <> __device__ __forceinline__ Pair pair_of<__nv_bfloat16>(std::uint32_t two) {
    return pair(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ std::uint32_t two_of(Pair p);
template <> __device__ __forceinline__ std::uint32_t two_of<__half>(Pair p) {
    const float2 f = both(p);
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const std::uint32_t*>(&h);
}
template <> __device__ __forceinline__ std::uint32_t two_of<__nv_bfloat16>(Pair p) {
    const float2 f = both(p);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const std::uint32_t*>(&h);
}

// A 16-byte vector as pairs, and back (one rounding to T).
template <typename T>
__device__ __forceinline__ void to_pairs(Pair (&p)[8 / sizeof(T)], const uint4& raw) {
    if constexpr (sizeof(T) == 4) {
        p[0] = pair(__uint_as_float(raw.x), __uint_as_float(raw.y));
        p[1] = pair(__uint_as_float(raw.z), __uint_as_float(raw.w));
    } else {
        p[0] = pair_of<T>(raw.x);
        p[1] = pair_of<T>(raw.y);
        p[2] = pair_of<T>(raw.z);
        p[3] = pair_of<T>(raw.w);
    }
}
template <typename T>
__device__ __forceinline__ uint4 to_raw(const Pair (&p)[8 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        const float2 a = both(p[0]), b = both(p[1]);
        return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    } else {
        return make_uint4(two_of<T>(p[0]), two_of<T>(p[1]), two_of<T>(p[2]), two_of<T>(p[3]));
    }
}

}  // namespace cgpt
