// Rows of class logits: vectors that need not be aligned, lane groups that share a row, the lists of a teacher.
#pragma once
#include "common.h"

// 16 bytes at any multiple of the element size (global memory takes unaligned vectors; a row of an odd number of
// classes starts anywhere)
typedef unsigned uvec4 __attribute__((ext_vector_type(4), aligned(2)));
template <class TR>
__device__ __forceinline__ uint4 ld_any(const char* p) {
    const uvec4 u = *reinterpret_cast<const uvec4*>(p);
    return make_uint4(u.x, u.y, u.z, u.w);
}
__device__ __forceinline__ void st_any(char* p, const uint4& v) {
    uvec4 u = {v.x, v.y, v.z, v.w};
    *reinterpret_cast<uvec4*>(p) = u;
}
// the same past the caches
template <class TR>
__device__ __forceinline__ uint4 ld_any_nt(const char* p) {
    const uvec4 u = __builtin_nontemporal_load(reinterpret_cast<const uvec4*>(p));
    return make_uint4(u.x, u.y, u.z, u.w);
}
__device__ __forceinline__ void st_any_nt(char* p, const uint4& v) {
    const uvec4 u = {v.x, v.y, v.z, v.w};
    __builtin_nontemporal_store(u, reinterpret_cast<uvec4*>(p));
}
template <class TR>
__device__ __forceinline__ float ld_one(const char* p, int64_t i) {
    if constexpr (TR::ESZ == 2) return bf16_to_f32(reinterpret_cast<const unsigned short*>(p)[i]);
    else return reinterpret_cast<const float*>(p)[i];
}
template <class TR>
__device__ __forceinline__ void st_one(char* p, int64_t i, float v) {
    if constexpr (TR::ESZ == 2) reinterpret_cast<unsigned short*>(p)[i] = f32_to_bf16(v);
    else reinterpret_cast<float*>(p)[i] = v;
}

// a vector moved down by n elements (0 < n < VEC)
template <class TR>
__device__ __forceinline__ uint4 down(uint4 w, int n) {
    const int bits = n * TR::ESZ * 8;
    if (bits & 64) { w.x = w.z; w.y = w.w; }
    if (bits & 32) { w.x = w.y; w.y = w.z; w.z = w.w; }
    if (TR::ESZ == 2 && (bits & 16)) {
        w.x = w.x >> 16 | w.y << 16; w.y = w.y >> 16 | w.z << 16; w.z = w.z >> 16 | w.w << 16; w.w >>= 16;
    }
    return w;
}

// the compiler takes the value as new: what was computed from it before is not kept in registers
__device__ __forceinline__ void hold(uint4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }

// maximum / sum over the L neighbouring lanes that share a row (L a power of two)
__device__ __forceinline__ float lanes_max(float v, int L) {
    for (int o = L >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float lanes_sum(float v, int L) {
    for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
