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

// v joined by f (commutative) over L (a power of two, the same for the whole wave) neighbouring lanes, all of which end with the result:
// lanes at distance 1, then 2, halves and rows mirrored (a quad's lanes agree by then), rows and halves of the wave swapped.  Nothing
// goes through LDS, where an exchange takes a hundred cycles (1000000 rows of 133 fp32 classes, distillation loss: 192 -> 150 us).
template <int CTRL>
__device__ __forceinline__ unsigned lane_move(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <class F>
__device__ __forceinline__ unsigned lanes_join(unsigned v, int L, F f) {
    if (L == 1) return v;
    v = f(v, lane_move<0xB1>(v));                                  // quad: 1 0 3 2
    if (L == 2) return v;
    v = f(v, lane_move<0x4E>(v));                                  // quad: 2 3 0 1
    if (L == 4) return v;
    v = f(v, lane_move<0x141>(v));                                 // eight lanes mirrored
    if (L == 8) return v;
    v = f(v, lane_move<0x140>(v));                                 // sixteen lanes mirrored
    if (L == 16) return v;
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(r[0], r[1]);
    if (L == 32) return v;
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(h[0], h[1]);
}
__device__ __forceinline__ float lanes_max(float v, int L) {
    return __uint_as_float(lanes_join(__float_as_uint(v), L, [](unsigned a, unsigned b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ float lanes_sum(float v, int L) {
    return __uint_as_float(lanes_join(__float_as_uint(v), L, [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ unsigned lanes_max(unsigned v, int L) { return lanes_join(v, L, [](unsigned a, unsigned b) { return max(a, b); }); }
__device__ __forceinline__ unsigned lanes_min(unsigned v, int L) { return lanes_join(v, L, [](unsigned a, unsigned b) { return min(a, b); }); }
// the same for a double, half by half
template <int CTRL>
__device__ __forceinline__ double lane_move(double v) {
    return __hiloint2double((int)lane_move<CTRL>((unsigned)__double2hiint(v)), (int)lane_move<CTRL>((unsigned)__double2loint(v)));
}
__device__ __forceinline__ double lanes_sum(double v, int L) {
    if (L == 1) return v;
    v += lane_move<0xB1>(v);
    if (L == 2) return v;
    v += lane_move<0x4E>(v);
    if (L == 4) return v;
    v += lane_move<0x141>(v);
    if (L == 8) return v;
    v += lane_move<0x140>(v);
    if (L == 16) return v;
    const unsigned hi = (unsigned)__double2hiint(v), lo = (unsigned)__double2loint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(hi, hi, false, false), b = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    v = __hiloint2double((int)a[0], (int)b[0]) + __hiloint2double((int)a[1], (int)b[1]);
    if (L == 32) return v;
    const unsigned hi2 = (unsigned)__double2hiint(v), lo2 = (unsigned)__double2loint(v);
    const auto c = __builtin_amdgcn_permlane32_swap(hi2, hi2, false, false), d = __builtin_amdgcn_permlane32_swap(lo2, lo2, false, false);
    return __hiloint2double((int)c[0], (int)d[0]) + __hiloint2double((int)c[1], (int)d[1]);
}
