// Group norm (affine) + activation (+ residual add), forward and backward, on channels-last tensors.
//
//   xh = (x - mean_ng) * rstd_ng ; u = w_c * xh + b_c ; y = act(u) (+ res)
//   g  = dy * act'(u) ; db_c = sum g ; dw_c = sum g * xh ; dalpha = sum_{u <= 0} dy * u
//   dx = rstd_ng * (w_c * g - mean_ng(w g) - xh * mean_ng(w g xh))
//
// Bandwidth-bound: the forward pass cannot do without one read and one write of the tensor, the backward pass without
// two reads (x, dy) and one write.
//
// Thread layout of every kernel: a pixel is C / VEC vectors of up to 16 bytes; a sweep of the workgroup covers `rows`
// pixels x `cols` vectors, and a thread keeps its vector column for all its pixels, so that the constants of its
// channels live in registers.  VEC is the widest vector that the channel count, the pitches and the addresses of all
// tensors of the call allow; dense tensors of odd channel counts go in runs of VEC pixels (see Runs).
//
// Sums: the statistics are fp64 from the first addition on; the backward pass adds up to CHUNK fp32 gradients in a thread and goes on in fp64.  All
// are joined in a fixed order (no atomics).
#include <string.h>
#include <type_traits>

#include "common.h"
#include "../../include/unet_mi355.h"

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_PRELU = 4 };
constexpr int TPB = 256;
constexpr int U = 4, UB = 2;         // vectors in flight per thread and tensor: forward, backward
constexpr int CHUNK = 256;           // pixels a thread adds in fp32 before the sums move to fp64
constexpr int MAX_C = 8192, MAX_G = 2048;

struct View { char* p; int64_t pitch, image; };   // p: address of the first channel of the first pixel; distances in bytes

struct GnParams {
    View x, dy, res, out;
    const float *w, *b, *alpha;
    float* stats;                // [nb][groups][2] mean, rstd
    double* part;                // forward: [nb][S][groups][2] ; backward: the same, then [nb][S][c][2], then [nb * S] dalpha
    double* part_c;
    double* part_a;
    float *dw, *db, *dalpha;
    int nb, c, groups, cg, act, S, B;   // S: splits of an image in the statistics pass, B: in the apply pass
    int cr, rep, tail;                  // dense tensors of odd channel counts: see Runs
    int64_t npix;
    double eps, count;                  // values per group
};

// Runs: a dense tensor whose channel count is no multiple of the widest vector is taken VEC pixels at a time: c = VEC * cr channels
// side by side (rep = VEC, npix counts whole runs), channel ch of which is channel ch % cr of the tensor.  The pixels behind
// the last whole run are `tail` elements.  Vectors then start at any element.
__device__ __forceinline__ int real_ch(const GnParams& p, int ch) { return p.rep == 1 ? ch : ch % p.cr; }

// VEC elements <-> floats
template <class TR, int VEC>
__device__ __forceinline__ void ldv(const char* p, float* v) {
    if constexpr (VEC * TR::ESZ == 16) {
        load_vec<TR>(p, v);
    } else if constexpr (TR::ESZ == 4) {
        if constexpr (VEC == 2) { const float2 u = *reinterpret_cast<const float2*>(p); v[0] = u.x; v[1] = u.y; }
        else v[0] = *reinterpret_cast<const float*>(p);
    } else {
        if constexpr (VEC == 4) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
            v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
        } else if constexpr (VEC == 2) {
            const unsigned u = *reinterpret_cast<const unsigned*>(p);
            v[0] = __uint_as_float(u << 16); v[1] = __uint_as_float(u & 0xffff0000u);
        } else v[0] = bf16_to_f32(*reinterpret_cast<const unsigned short*>(p));
    }
}
template <class TR, int VEC>
__device__ __forceinline__ void stv(char* p, const float* v) {
    if constexpr (VEC * TR::ESZ == 16) {
        store_vec<TR>(p, v);
    } else if constexpr (TR::ESZ == 4) {
        if constexpr (VEC == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
        else *reinterpret_cast<float*>(p) = v[0];
    } else {
        if constexpr (VEC == 4) {
            uint2 u;
            u.x = (unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16);
            u.y = (unsigned)f32_to_bf16(v[2]) | ((unsigned)f32_to_bf16(v[3]) << 16);
            *reinterpret_cast<uint2*>(p) = u;
        } else if constexpr (VEC == 2) {
            *reinterpret_cast<unsigned*>(p) = (unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16);
        } else *reinterpret_cast<unsigned short*>(p) = f32_to_bf16(v[0]);
    }
}

// 1 / (1 + exp(-u)): both hardware functions are good to one unit in the last place
__device__ __forceinline__ float sigmoid_f(float u) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
}
// Phi(u), the normal distribution function, and e = exp(-u^2 / 2).  With t = 1 / (1 + 0.2828 |u|) the scaled tail
// Phi(-|u|) / (e t) is smooth in t; the polynomial below is a weighted least-squares fit of it in relative error, which is 1.3e-7
// in exact arithmetic and 4.8e-7 in fp32 from 0 to 12.  Phi(-|u|) itself also takes what three roundings of the exponent do to e, at most
// 1.5 u^2 2^-24: 1.9e-6 in all at 4, 1.3e-5 at 12 where Phi is 2e-33.  (The library's erff takes twice the instructions:
// GELU forward 32 x 256^2 x 32 bf16 108 -> 97 us, backward 32 x 256^2 x 16 103 -> 79).
__device__ __forceinline__ float normal_cdf(float u, float& e) {
    e = __builtin_amdgcn_exp2f(u * u * -0.72134752044448170f);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.28284272f, fabsf(u), 1.0f));
    float s = 0.025144234f;
    s = fmaf(s, t, -0.091504857f);
    s = fmaf(s, t, 0.084634006f);
    s = fmaf(s, t, -0.0028852099f);
    s = fmaf(s, t, 0.070756972f);
    s = fmaf(s, t, 0.084259167f);
    s = fmaf(s, t, 0.10392314f);
    s = fmaf(s, t, 0.11283468f);
    s = fmaf(s, t, 0.11283793f);
    const float tail = s * t * e;
    return u > 0.0f ? 1.0f - tail : tail;
}
constexpr float INV_SQRT_2PI = 0.39894228040143268f;

template <int VEC>
__device__ __forceinline__ void act_apply(int act, float alpha, float* u) {
    if (act == ACT_SILU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) u[j] *= sigmoid_f(u[j]);
    } else if (act == ACT_RELU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) u[j] = u[j] < 0.0f ? 0.0f : u[j];      // a NaN stays
    } else if (act == ACT_PRELU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) u[j] = u[j] > 0.0f ? u[j] : alpha * u[j];
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float e;
            u[j] *= normal_cdf(u[j], e);
        }
    }
}
// g[j] = dy[j] * act'(u[j]); returns sum of dy * u over u <= 0 (PReLU's slope gradient)
template <int VEC>
__device__ __forceinline__ float act_grad(int act, float alpha, const float* u, const float* dy, float* g) {
    float da = 0.0f;
    if (act == ACT_SILU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float s = sigmoid_f(u[j]);
            g[j] = dy[j] * (s * fmaf(u[j], 1.0f - s, 1.0f));
        }
    } else if (act == ACT_RELU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = u[j] > 0.0f ? dy[j] : 0.0f;
    } else if (act == ACT_PRELU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            g[j] = u[j] > 0.0f ? dy[j] : alpha * dy[j];
            da = u[j] > 0.0f ? da : fmaf(dy[j], u[j], da);
        }
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float e;
            const float c = normal_cdf(u[j], e);
            g[j] = dy[j] * fmaf(u[j] * INV_SQRT_2PI, e, c);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = dy[j];
    }
    return da;
}

// Raw vectors: what a load leaves in registers, unpacked when it is used
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { typedef uint4 T; };
template <> struct RawOf<8> { typedef uint2 T; };
template <> struct RawOf<4> { typedef unsigned T; };
template <> struct RawOf<2> { typedef unsigned short T; };
template <class TR, int VEC> using Raw = typename RawOf<VEC * TR::ESZ>::T;
typedef unsigned nvec4 __attribute__((ext_vector_type(4), aligned(2)));      // runs start at any element
typedef unsigned nvec2 __attribute__((ext_vector_type(2)));
template <class TR, int VEC>
__device__ __forceinline__ Raw<TR, VEC> ldr(const char* p) {
    if constexpr (VEC * TR::ESZ == 16) {
        const nvec4 v = *reinterpret_cast<const nvec4*>(p);
        return make_uint4(v.x, v.y, v.z, v.w);
    } else {
        return *reinterpret_cast<const Raw<TR, VEC>*>(p);
    }
}
// The second passes read their tensors for the last time and write more than the caches hold of use to the next kernel:
// past the caches (32 x 256^2 x 32 bf16 forward 89 -> 77 us, 32 x 256^2 x 16 backward 72 -> 63, 3-D fp32 backward 60 -> 49; with an
// elementwise reader of the result behind the call 137 -> 130 us at 128 MiB a tensor and no difference from 8 to 96 MiB).
template <class TR, int VEC>
__device__ __forceinline__ Raw<TR, VEC> ldr_nt(const char* p) {
    typedef Raw<TR, VEC> R;
    if constexpr (sizeof(R) == 16) {
        const nvec4 v = __builtin_nontemporal_load(reinterpret_cast<const nvec4*>(p));
        return make_uint4(v.x, v.y, v.z, v.w);
    } else if constexpr (sizeof(R) == 8) {
        const nvec2 v = __builtin_nontemporal_load(reinterpret_cast<const nvec2*>(p));
        return make_uint2(v.x, v.y);
    } else {
        return __builtin_nontemporal_load(reinterpret_cast<const R*>(p));
    }
}
template <class TR, int VEC>
__device__ __forceinline__ void stv_nt(char* p, const float* v) {
    typedef Raw<TR, VEC> R;
    R r;
    stv<TR, VEC>(reinterpret_cast<char*>(&r), v);
    if constexpr (sizeof(R) == 16) {
        const nvec4 v = {r.x, r.y, r.z, r.w};
        __builtin_nontemporal_store(v, reinterpret_cast<nvec4*>(p));
    }
    else if constexpr (sizeof(R) == 8) __builtin_nontemporal_store((nvec2){r.x, r.y}, reinterpret_cast<nvec2*>(p));
    else __builtin_nontemporal_store(r, reinterpret_cast<R*>(p));
}
template <class TR, int VEC>
__device__ __forceinline__ void unraw(const Raw<TR, VEC>& r, float* v) {
    Raw<TR, VEC> t = r;
    ldv<TR, VEC>(reinterpret_cast<const char*>(&t), v);
}

// the first n of VEC elements (the others 0), one by one
template <class TR, int VEC>
__device__ __forceinline__ void ld_some(const char* p, int n, float* v) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        v[j] = 0.0f;
        if (j < n) ldv<TR, 1>(p + j * TR::ESZ, v + j);
    }
}
template <class TR, int VEC>
__device__ __forceinline__ void st_some(char* p, int n, const float* v) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (j < n) stv<TR, 1>(p + j * TR::ESZ, v + j);
}

// Sums of the `rows` threads that share a vector column, in a fixed order: NV doubles per thread in LDS as
// [NV][TPB] (consecutive lanes, consecutive addresses), halved until row 0 holds the totals.
template <int NV>
__device__ __forceinline__ void row_tree(double* sm, int tid, int row, int rows, int cols) {
    for (int r = rows; r > 1;) {
        const int half = (r + 1) >> 1;
        __syncthreads();
        if (row + half < r && row < half) {
#pragma unroll
            for (int k = 0; k < NV; ++k) sm[k * TPB + tid] += sm[k * TPB + tid + half * cols];
        }
        r = half;
    }
    __syncthreads();
}

struct Lane { int cols, rows, col, row; };
__device__ __forceinline__ Lane lane_of(int cols) {
    Lane l;
    l.cols = cols;
    l.rows = TPB / cols;
    l.col = threadIdx.x % cols; l.row = threadIdx.x / cols;
    return l;
}

// After a row_tree: column sums of a run's channels folded onto the channels of the tensor, which then lie where they would
// without runs: channel ch of a slab at [ch % VEC][ch / VEC]
template <int VEC>
__device__ __forceinline__ void fold_runs(const GnParams& p, double* sm) {
    if (p.rep == 1) return;
    const int ch = threadIdx.x;                                     // cr <= TPB
    double a = 0.0, b = 0.0;
    if (ch < p.cr)
        for (int k = ch; k < p.c; k += p.cr) { a += sm[(k % VEC) * TPB + k / VEC]; b += sm[(VEC + k % VEC) * TPB + k / VEC]; }
    __syncthreads();
    if (ch < p.cr) { sm[(ch % VEC) * TPB + ch / VEC] = a; sm[(VEC + ch % VEC) * TPB + ch / VEC] = b; }
    __syncthreads();
}
// For the groups g0 .. g1: f(g, k, step) adds every step-th of the group's (at most len) values from the k-th on; the sums are added to
// gs[2 g].  Neighbouring lanes share a group where there are threads to spare.
template <class F>
__device__ __forceinline__ void each_group(int g0, int g1, int len, double* gs, F f) {
    const int tid = threadIdx.x, ng = g1 - g0 + 1;
    int lanes = 1;
    while (lanes < 64 && 2 * lanes * ng <= TPB && lanes < len) lanes *= 2;
    for (int first = g0; first <= g1; first += TPB / lanes) {
        const int g = first + tid / lanes;
        double2 v = make_double2(0.0, 0.0);
        if (g <= g1) v = f(g, tid % lanes, lanes);
        for (int o = lanes >> 1; o > 0; o >>= 1) { v.x += __shfl_xor(v.x, o, 64); v.y += __shfl_xor(v.y, o, 64); }
        if (g <= g1 && tid % lanes == 0) { gs[2 * g] += v.x; gs[2 * g + 1] += v.y; }
    }
}
// Channel sums (two doubles per channel of the thread's column) of `rows` threads -> sums of the groups added to
// gs[2 g].  Where a vector lies inside a group its channels are added in registers and the tree carries two values, else 2 * VEC.
// `sm`: 2 * VEC * TPB doubles.  c0: first channel of column 0.
template <int VEC>
__device__ __forceinline__ void add_groups(const GnParams& p, double* sm, double* gs, const double* d1, const double* d2, const Lane& l, int c0) {
    const int tid = threadIdx.x, cg = p.cg, c1 = min(c0 + l.cols * VEC, p.cr), g0 = c0 / cg, g1 = (c1 - 1) / cg;
    __syncthreads();
    if (p.rep == 1 && cg % VEC == 0) {
        double a = 0.0, b = 0.0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) { a += d1[j]; b += d2[j]; }
        sm[tid] = a; sm[TPB + tid] = b;
        row_tree<2>(sm, tid, l.row, l.rows, l.cols);
        each_group(g0, g1, cg / VEC, gs, [&](int g, int k, int step) {
            double2 v = make_double2(0.0, 0.0);
            for (int i = max(0, (g * cg - c0) / VEC) + k; i < min(l.cols, ((g + 1) * cg - c0) / VEC); i += step) { v.x += sm[i]; v.y += sm[TPB + i]; }
            return v;
        });
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { sm[j * TPB + tid] = d1[j]; sm[(VEC + j) * TPB + tid] = d2[j]; }
        row_tree<2 * VEC>(sm, tid, l.row, l.rows, l.cols);
        fold_runs<VEC>(p, sm);
        each_group(g0, g1, cg, gs, [&](int g, int k, int step) {
            double2 v = make_double2(0.0, 0.0);
            for (int i = max(c0, g * cg) + k; i < min(c1, (g + 1) * cg); i += step) {
                const int at = ((i - c0) % VEC) * TPB + (i - c0) / VEC;
                v.x += sm[at]; v.y += sm[VEC * TPB + at];
            }
            return v;
        });
    }
    __syncthreads();
}

// The pairs part[s][g], s < S, of an image added up by the whole workgroup: f(g, sum a, sum b) for every group.  Threads
// side by side take neighbouring pairs; the sub-sums of a group are joined in a fixed order.
template <class F>
__device__ __forceinline__ void join_groups(const double* part, int S, int groups, double* sm, F f) {
    const int tid = threadIdx.x;
    const double2* q = reinterpret_cast<const double2*>(part);
    for (int g0 = 0; g0 < groups; g0 += TPB) {
        const Lane l = lane_of(min(groups - g0, TPB));
        double a = 0.0, b = 0.0;
        if (l.row < l.rows) {
#pragma unroll 4
            for (int s = l.row; s < S; s += l.rows) {
                const double2 v = q[(int64_t)s * groups + g0 + l.col];
                a += v.x; b += v.y;
            }
        }
        __syncthreads();
        sm[tid] = a; sm[TPB + tid] = b;
        row_tree<2>(sm, tid, l.row, l.rows, l.cols);
        if (tid < l.cols) f(g0 + tid, sm[tid], sm[TPB + tid]);
    }
    __syncthreads();
}

__device__ __forceinline__ float2 moments(double a, double b, double cnt, double eps) {
    const double m = a / cnt;
    double var = b / cnt - m * m;
    var = var < 0.0 ? 0.0 : var;                                    // a NaN stays
    return make_float2((float)m, (float)(1.0 / sqrt(var + eps)));
}

// sums of values and squares: fp64 holds both exactly.  (fp32 sums about a first value of the thread's own lost 2e-3 of the variance where that value was the
// one bright pixel of an even image.)
template <int VEC>
__device__ __forceinline__ void add_moments(const float* v, double* d1, double* d2) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const double x = v[j];
        d1[j] += x; d2[j] = fma(x, x, d2[j]);
    }
}

// ---- forward, pass 1: sum and sum of squares per (image, split, group) -------------------------------------------
// Bound by the read: 32 x 256^2 x 32 bf16 (134 MB) 30 us, 4.5 TB/s.  Two passes because the chip cannot hold such a tensor: with the
// pixels in registers while the workgroups of an image wait for each other's sums (one read), the exchange past the L2 caches takes
// 10 to 20 us a round and the same call 140 us instead of 77.
template <class TR, int VEC>
__global__ __launch_bounds__(TPB) void gn_stats_kernel(GnParams p) {
    __shared__ double sm[2 * VEC * TPB];
    extern __shared__ double gs[];                                  // [groups][2]
    const int n = blockIdx.x / p.S, s = blockIdx.x % p.S, tid = threadIdx.x;
    const int64_t per = (p.npix + p.S - 1) / p.S;
    const int64_t p0 = s * per, p1 = min(p.npix, p0 + per);
    const char* x = p.x.p + n * p.x.image;
    for (int g = tid; g < 2 * p.groups; g += TPB) gs[g] = 0.0;
    const int cv = p.c / VEC;
    for (int col0 = 0; col0 < cv; col0 += TPB) {
        const Lane l = lane_of(min(cv - col0, TPB));
        const int64_t step = l.rows * p.x.pitch;
        const char* xc = x + (int64_t)(col0 + l.col) * (VEC * TR::ESZ) + (p0 + l.row) * p.x.pitch;
        double d1[VEC], d2[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) d1[j] = d2[j] = 0.0;
        auto take = [&](const Raw<TR, VEC>& r) {
            float v[VEC];
            unraw<TR, VEC>(r, v);
            add_moments<VEC>(v, d1, d2);
        };
        int64_t left = l.row < l.rows && p0 + l.row < p1 ? (p1 - p0 - l.row + l.rows - 1) / l.rows : 0;
        for (; left >= U; left -= U) {
            Raw<TR, VEC> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = ldr<TR, VEC>(xc + u * step);
#pragma unroll
            for (int u = 0; u < U; ++u) take(r[u]);
            xc += U * step;
        }
        for (; left > 0; --left) { take(ldr<TR, VEC>(xc)); xc += step; }
        if (s == p.S - 1 && l.row == 0) {                           // behind the last run
            const int have = p.tail - l.col * VEC;
            float v[VEC];
            if (have > 0) ld_some<TR, VEC>(x + p.npix * p.x.pitch + l.col * (VEC * TR::ESZ), have, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < have) { d1[j] += v[j]; d2[j] = fma((double)v[j], (double)v[j], d2[j]); }
        }
        add_groups<VEC>(p, sm, gs, d1, d2, l, col0 * VEC);
    }
    double* out = p.part + (int64_t)blockIdx.x * p.groups * 2;
    for (int g = tid; g < 2 * p.groups; g += TPB) out[g] = gs[g];
}

// ---- forward, pass 2 ----------------------------------------------------------------------------------------------
// Bound by the read and the write: 268 MB in 45 us, 5.9 TB/s; 3 x 187 x 253 x 30 fp32 with GELU and a residual (51 MB) 15 us.
template <class TR, int VEC>
struct FwdConst {
    float mean[VEC], a[VEC], b[VEC];
    __device__ __forceinline__ void load(const GnParams& p, const float2* mr, int g0, int ch0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int ch = real_ch(p, ch0 + j);
            const float2 m = mr[ch / p.cg - g0];
            mean[j] = m.x;
            a[j] = m.y * (p.w ? p.w[ch] : 1.0f);
            b[j] = p.b ? p.b[ch] : 0.0f;
        }
    }
    __device__ __forceinline__ void apply(int act, float alpha, float* v) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = fmaf(v[j] - mean[j], a[j], b[j]);
        act_apply<VEC>(act, alpha, v);
    }
};

template <class TR, int VEC>
__global__ __launch_bounds__(TPB) void gn_apply_kernel(GnParams p) {
    extern __shared__ float2 mr[];                                  // [groups] mean, rstd
    __shared__ double sm[2 * TPB];
    const int n = blockIdx.x / p.B, bi = blockIdx.x % p.B;
    const double cnt = p.count;
    join_groups(p.part + (int64_t)n * p.S * p.groups * 2, p.S, p.groups, sm, [&](int g, double a, double b) {
        mr[g] = moments(a, b, cnt, p.eps);
        if (bi == 0) reinterpret_cast<float2*>(p.stats)[(int64_t)n * p.groups + g] = mr[g];
    });
    const float alpha = p.alpha ? p.alpha[0] : 0.0f;
    const int64_t per = (p.npix + p.B - 1) / p.B;
    const int64_t p0 = bi * per, p1 = min(p.npix, p0 + per);
    const int cv = p.c / VEC;
    for (int col0 = 0; col0 < cv; col0 += TPB) {
        const Lane l = lane_of(min(cv - col0, TPB));
        if (l.row >= l.rows) continue;
        const int ch0 = (col0 + l.col) * VEC;
        FwdConst<TR, VEC> k;
        k.load(p, mr, 0, ch0);
        const int64_t at = p0 + l.row, off = (int64_t)ch0 * TR::ESZ;
        const char* x = p.x.p + n * p.x.image + at * p.x.pitch + off;
        const char* r = p.res.p ? p.res.p + n * p.res.image + at * p.res.pitch + off : nullptr;
        char* o = p.out.p + n * p.out.image + at * p.out.pitch + off;
        const int64_t xs = l.rows * p.x.pitch, rs = l.rows * p.res.pitch, os = l.rows * p.out.pitch;
        int64_t left = p0 + l.row < p1 ? (p1 - p0 - l.row + l.rows - 1) / l.rows : 0;
        auto batch = [&](auto nu) {
            constexpr int N = decltype(nu)::value;
            Raw<TR, VEC> xv[N], rv[N];
#pragma unroll
            for (int u = 0; u < N; ++u) xv[u] = ldr_nt<TR, VEC>(x + u * xs);
            if (r) {
#pragma unroll
                for (int u = 0; u < N; ++u) rv[u] = ldr_nt<TR, VEC>(r + u * rs);
                r += N * rs;
            }
#pragma unroll
            for (int u = 0; u < N; ++u) {
                float v[VEC];
                unraw<TR, VEC>(xv[u], v);
                k.apply(p.act, alpha, v);
                if (r) {
                    float q[VEC];
                    unraw<TR, VEC>(rv[u], q);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[j] += q[j];
                }
                stv_nt<TR, VEC>(o + u * os, v);
            }
            x += N * xs; o += N * os;
        };
        for (; left >= U; left -= U) batch(std::integral_constant<int, U>{});
        for (; left > 0; --left) batch(std::integral_constant<int, 1>{});
        const int have = p.tail - ch0;
        if (have > 0 && bi == p.B - 1 && l.row == 0) {              // behind the last run
            float v[VEC], q[VEC];
            ld_some<TR, VEC>(p.x.p + n * p.x.image + p.npix * p.x.pitch + off, have, v);
            k.apply(p.act, alpha, v);
            if (p.res.p) {
                ld_some<TR, VEC>(p.res.p + n * p.res.image + p.npix * p.res.pitch + off, have, q);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] += q[j];
            }
            st_some<TR, VEC>(p.out.p + n * p.out.image + p.npix * p.out.pitch + off, have, v);
        }
    }
}

// channel constants of the backward kernels: xh = (x - mean) * rstd, u = xh * w + b
template <int VEC>
struct BwdConst {
    float mean[VEC], rstd[VEC], w[VEC], b[VEC];
    __device__ __forceinline__ void load(const GnParams& p, int n, int ch0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int ch = real_ch(p, ch0 + j);
            const float2 st = reinterpret_cast<const float2*>(p.stats)[(int64_t)n * p.groups + ch / p.cg];
            mean[j] = st.x; rstd[j] = st.y;
            w[j] = p.w ? p.w[ch] : 1.0f;
            b[j] = p.b ? p.b[ch] : 0.0f;
        }
    }
    // v: x -> xh; g: gradient in front of the activation; returns the slope's sum
    __device__ __forceinline__ float grad(int act, float alpha, float* v, const float* dy, float* g) const {
        float u[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { v[j] = (v[j] - mean[j]) * rstd[j]; u[j] = fmaf(v[j], w[j], b[j]); }
        return act_grad<VEC>(act, alpha, u, dy, g);
    }
    // dx from xh and g
    __device__ __forceinline__ void dx(const float* v, const float* g, const float* m0, const float* m1, float* o) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = rstd[j] * (fmaf(w[j], g[j], -m0[j]) - v[j] * m1[j]);
    }
};

// Channel sums of a workgroup (LDS, [2 * VEC][TPB], row 0 holds the totals): written to pc[channel], and weighted into the
// groups' sums gs.
template <int VEC>
__device__ __forceinline__ void spread_channels(const GnParams& p, double* sm, const Lane& l, int c0, double* pc, double* gs, int g00) {
    const int tid = threadIdx.x, c1 = min(c0 + l.cols * VEC, p.cr);
    fold_runs<VEC>(p, sm);
    for (int ch = tid; ch < c1 - c0; ch += TPB)
        reinterpret_cast<double2*>(pc)[ch] = make_double2(sm[(ch % VEC) * TPB + ch / VEC], sm[(VEC + ch % VEC) * TPB + ch / VEC]);
    each_group(c0 / p.cg, (c1 - 1) / p.cg, p.cg, gs - 2 * g00, [&](int g, int k, int step) {
        double2 v = make_double2(0.0, 0.0);
        for (int i = max(c0, g * p.cg) + k; i < min(c1, (g + 1) * p.cg); i += step) {
            const int at = ((i - c0) % VEC) * TPB + (i - c0) / VEC;
            const double w = p.w ? p.w[i] : 1.0f;
            v.x += w * sm[at]; v.y += w * sm[VEC * TPB + at];
        }
        return v;
    });
}

// ---- backward, pass 1: per (image, split) the channel sums of g and g xh, the group sums of w g and w g xh ----------
// Bound by the reads of x and dy: 32 x 256^2 x 16 bf16 (134 MB) 32 us, 4.2 TB/s; 4 x 48^3 x 32 fp32 (113 MB) 25 us, 4.5 TB/s.
template <class TR, int VEC>
__global__ __launch_bounds__(TPB) void gn_bwd_reduce_kernel(GnParams p) {
    __shared__ double sm[2 * VEC * TPB];
    extern __shared__ double gs[];                                  // [groups][2]
    const int n = blockIdx.x / p.S, s = blockIdx.x % p.S, tid = threadIdx.x;
    const int64_t per = (p.npix + p.S - 1) / p.S;
    const int64_t p0 = s * per, p1 = min(p.npix, p0 + per);
    const float alpha = p.alpha ? p.alpha[0] : 0.0f;
    for (int g = tid; g < 2 * p.groups; g += TPB) gs[g] = 0.0;
    const int cv = p.c / VEC;
    double da = 0.0;
    for (int col0 = 0; col0 < cv; col0 += TPB) {
        const Lane l = lane_of(min(cv - col0, TPB));
        const int ch0 = (col0 + l.col) * VEC;
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) sm[j * TPB + tid] = 0.0;  // the thread's own sums
        if (l.row < l.rows) {
            BwdConst<VEC> k;
            k.load(p, n, ch0);
            const int64_t at = p0 + l.row, off = (int64_t)ch0 * TR::ESZ;
            const char* x = p.x.p + n * p.x.image + at * p.x.pitch + off;
            const char* d = p.dy.p + n * p.dy.image + at * p.dy.pitch + off;
            const int64_t xs = l.rows * p.x.pitch, ds = l.rows * p.dy.pitch;
            int64_t left = p0 + l.row < p1 ? (p1 - p0 - l.row + l.rows - 1) / l.rows : 0;
            while (left > 0) {
                const int cnt = (int)min((int64_t)CHUNK, left);
                float s1[VEC], s2[VEC], sa = 0.0f;
#pragma unroll
                for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.0f;
                auto batch = [&](auto nu) {
                    constexpr int N = decltype(nu)::value;
                    Raw<TR, VEC> xv[N], dv[N];
#pragma unroll
                    for (int u = 0; u < N; ++u) { xv[u] = ldr<TR, VEC>(x + u * xs); dv[u] = ldr<TR, VEC>(d + u * ds); }
#pragma unroll
                    for (int u = 0; u < N; ++u) {
                        float v[VEC], dy[VEC], g[VEC];
                        unraw<TR, VEC>(xv[u], v);
                        unraw<TR, VEC>(dv[u], dy);
                        sa += k.grad(p.act, alpha, v, dy, g);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) { s1[j] += g[j]; s2[j] = fmaf(g[j], v[j], s2[j]); }
                    }
                    x += N * xs; d += N * ds;
                };
                int i = 0;
                for (; i + UB <= cnt; i += UB) batch(std::integral_constant<int, UB>{});
                for (; i < cnt; ++i) batch(std::integral_constant<int, 1>{});
#pragma unroll
                for (int j = 0; j < VEC; ++j) { sm[j * TPB + tid] += s1[j]; sm[(VEC + j) * TPB + tid] += s2[j]; }
                da += sa;
                left -= cnt;
            }
            const int have = p.tail - ch0;
            if (have > 0 && s == p.S - 1 && l.row == 0) {           // behind the last run; the gradient of what is not there is 0
                float v[VEC], dy[VEC], g[VEC];
                ld_some<TR, VEC>(p.x.p + n * p.x.image + p.npix * p.x.pitch + off, have, v);
                ld_some<TR, VEC>(p.dy.p + n * p.dy.image + p.npix * p.dy.pitch + off, have, dy);
                da += k.grad(p.act, alpha, v, dy, g);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { sm[j * TPB + tid] += g[j]; sm[(VEC + j) * TPB + tid] += g[j] * v[j]; }
            }
        }
        row_tree<2 * VEC>(sm, tid, l.row, l.rows, l.cols);
        spread_channels<VEC>(p, sm, l, col0 * VEC, p.part_c + ((int64_t)blockIdx.x * p.cr + col0 * VEC) * 2, gs, 0);
        __syncthreads();
    }
    double* out = p.part + (int64_t)blockIdx.x * p.groups * 2;
    for (int g = tid; g < 2 * p.groups; g += TPB) out[g] = gs[g];
    if (p.part_a) {
        sm[tid] = da;
        row_tree<1>(sm, tid, tid, TPB, 1);
        if (tid == 0) p.part_a[blockIdx.x] = sm[0];
    }
}

// Parameter gradients: workgroup k joins the channels [k * JC, (k + 1) * JC) of the n parts; the one behind the last, dalpha.
constexpr int JC = 16;
__device__ __forceinline__ void join_params(const GnParams& p, int k, int n, double* sm) {
    const int tid = threadIdx.x, last = (p.cr + JC - 1) / JC;
    if (k < last) {
        const int ch = k * JC + tid % JC, row = tid / JC;
        double a = 0.0, b = 0.0;
        if (ch < p.cr) {
#pragma unroll 4
            for (int i = row; i < n; i += TPB / JC) {
                const double2 v = reinterpret_cast<const double2*>(p.part_c)[(int64_t)i * p.cr + ch];
                a += v.x; b += v.y;
            }
        }
        sm[tid] = a; sm[TPB + tid] = b;
        row_tree<2>(sm, tid, row, TPB / JC, JC);
        if (row == 0 && ch < p.cr) {
            if (p.db) p.db[ch] = (float)sm[tid];
            if (p.dw) p.dw[ch] = (float)sm[TPB + tid];
        }
    } else {
        double a = 0.0;
        for (int i = tid; i < n; i += TPB) a += p.part_a[i];
        sm[tid] = a;
        row_tree<1>(sm, tid, tid, TPB, 1);
        if (tid == 0) p.dalpha[0] = (float)sm[0];
    }
}

// ---- backward, pass 2: dx; the workgroups behind the nb * B of them join the parameter gradients -------------------
// Bound by two reads and a write: the same tensors 34 us (5.9 TB/s) and 26 us (6.6 TB/s, in part from the last-level cache).
template <class TR, int VEC>
__global__ __launch_bounds__(TPB) void gn_bwd_apply_kernel(GnParams p) {
    extern __shared__ float2 gm[];                                  // [groups] means of w g and w g xh
    __shared__ double sm[2 * TPB];
    if ((int)blockIdx.x >= p.nb * p.B) {
        join_params(p, (int)blockIdx.x - p.nb * p.B, p.nb * p.S, sm);
        return;
    }
    const int n = blockIdx.x / p.B, bi = blockIdx.x % p.B;
    const double cnt = p.count;
    join_groups(p.part + (int64_t)n * p.S * p.groups * 2, p.S, p.groups, sm,
                [&](int g, double a, double b) { gm[g] = make_float2((float)(a / cnt), (float)(b / cnt)); });
    const float alpha = p.alpha ? p.alpha[0] : 0.0f;
    const int64_t per = (p.npix + p.B - 1) / p.B;
    const int64_t p0 = bi * per, p1 = min(p.npix, p0 + per);
    const int cv = p.c / VEC;
    for (int col0 = 0; col0 < cv; col0 += TPB) {
        const Lane l = lane_of(min(cv - col0, TPB));
        if (l.row >= l.rows) continue;
        const int ch0 = (col0 + l.col) * VEC;
        BwdConst<VEC> k;
        k.load(p, n, ch0);
        float m0[VEC], m1[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { const float2 m = gm[real_ch(p, ch0 + j) / p.cg]; m0[j] = m.x; m1[j] = m.y; }
        const int64_t at = p0 + l.row, off = (int64_t)ch0 * TR::ESZ;
        const char* x = p.x.p + n * p.x.image + at * p.x.pitch + off;
        const char* d = p.dy.p + n * p.dy.image + at * p.dy.pitch + off;
        char* o = p.out.p + n * p.out.image + at * p.out.pitch + off;
        const int64_t xs = l.rows * p.x.pitch, ds = l.rows * p.dy.pitch, os = l.rows * p.out.pitch;
        int64_t left = p0 + l.row < p1 ? (p1 - p0 - l.row + l.rows - 1) / l.rows : 0;
        auto batch = [&](auto nu) {
            constexpr int N = decltype(nu)::value;
            Raw<TR, VEC> xv[N], dv[N];
#pragma unroll
            for (int u = 0; u < N; ++u) { xv[u] = ldr_nt<TR, VEC>(x + u * xs); dv[u] = ldr_nt<TR, VEC>(d + u * ds); }
#pragma unroll
            for (int u = 0; u < N; ++u) {
                float v[VEC], dy[VEC], g[VEC];
                unraw<TR, VEC>(xv[u], v);
                unraw<TR, VEC>(dv[u], dy);
                k.grad(p.act, alpha, v, dy, g);
                k.dx(v, g, m0, m1, v);
                stv_nt<TR, VEC>(o + u * os, v);
            }
            x += N * xs; d += N * ds; o += N * os;
        };
        for (; left >= UB; left -= UB) batch(std::integral_constant<int, UB>{});
        for (; left > 0; --left) batch(std::integral_constant<int, 1>{});
        const int have = p.tail - ch0;
        if (have > 0 && bi == p.B - 1 && l.row == 0) {              // behind the last run
            float v[VEC], dy[VEC], g[VEC];
            ld_some<TR, VEC>(p.x.p + n * p.x.image + p.npix * p.x.pitch + off, have, v);
            ld_some<TR, VEC>(p.dy.p + n * p.dy.image + p.npix * p.dy.pitch + off, have, dy);
            k.grad(p.act, alpha, v, dy, g);
            k.dx(v, g, m0, m1, v);
            st_some<TR, VEC>(p.out.p + n * p.out.image + p.npix * p.out.pitch + off, have, v);
        }
    }
}

// ---- small images: one launch, the data stays in registers between the sums and their use ----------------------------
// Workgroup (n, slab) owns all pixels of p.B whole groups of image n (the last slab: what is left); a thread holds up to NV
// vectors.  dynamic LDS: [p.B][2] doubles.
struct Slab { int n, slab, g0, ng, c0; };
__device__ __forceinline__ Slab slab_of(const GnParams& p) {
    Slab b;
    b.n = blockIdx.x / p.S; b.slab = blockIdx.x % p.S;
    b.g0 = b.slab * p.B; b.ng = min(p.B, p.groups - b.g0); b.c0 = b.g0 * p.cg;
    return b;
}

template <class TR, int VEC, int NV>
__global__ __launch_bounds__(TPB) void gn_small_fwd_kernel(GnParams p) {
    __shared__ double sm[2 * VEC * TPB];
    extern __shared__ double gs[];
    const Slab b = slab_of(p);
    const Lane l = lane_of(b.ng * p.cg / VEC);
    const int tid = threadIdx.x, npix = (int)p.npix, ch0 = b.c0 + l.col * VEC;
    const int cnt = l.row < l.rows && l.row < npix ? (npix - l.row + l.rows - 1) / l.rows : 0;
    const int64_t at = l.row, off = (int64_t)ch0 * TR::ESZ;
    const char* x = p.x.p + b.n * p.x.image + at * p.x.pitch + off;
    Raw<TR, VEC> xv[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u)
        if (u < cnt) xv[u] = ldr<TR, VEC>(x + u * (l.rows * p.x.pitch));
    for (int g = tid; g < 2 * b.ng; g += TPB) gs[g] = 0.0;
    double d1[VEC], d2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) d1[j] = d2[j] = 0.0;
#pragma unroll
    for (int u = 0; u < NV; ++u)
        if (u < cnt) {
            float v[VEC];
            unraw<TR, VEC>(xv[u], v);
            add_moments<VEC>(v, d1, d2);
        }
    add_groups<VEC>(p, sm, gs - 2 * b.g0, d1, d2, l, b.c0);
    float2* mr = reinterpret_cast<float2*>(sm);
    for (int g = tid; g < b.ng; g += TPB) {
        mr[g] = moments(gs[2 * g], gs[2 * g + 1], p.count, p.eps);
        reinterpret_cast<float2*>(p.stats)[(int64_t)b.n * p.groups + b.g0 + g] = mr[g];
    }
    __syncthreads();
    if (!cnt) return;
    const float alpha = p.alpha ? p.alpha[0] : 0.0f;
    FwdConst<TR, VEC> c;
    c.load(p, mr, b.g0, ch0);
    const char* r = p.res.p ? p.res.p + b.n * p.res.image + at * p.res.pitch + off : nullptr;
    char* o = p.out.p + b.n * p.out.image + at * p.out.pitch + off;
#pragma unroll
    for (int u = 0; u < NV; ++u)
        if (u < cnt) {
            float v[VEC];
            unraw<TR, VEC>(xv[u], v);
            c.apply(p.act, alpha, v);
            if (r) {
                float q[VEC];
                ldv<TR, VEC>(r + u * (l.rows * p.res.pitch), q);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] += q[j];
            }
            stv<TR, VEC>(o + u * (l.rows * p.out.pitch), v);
        }
}

template <class TR, int VEC, int NV>
__global__ __launch_bounds__(TPB) void gn_small_bwd_kernel(GnParams p) {
    __shared__ double sm[2 * VEC * TPB];
    extern __shared__ double gs[];
    const Slab b = slab_of(p);
    const Lane l = lane_of(b.ng * p.cg / VEC);
    const int tid = threadIdx.x, npix = (int)p.npix, ch0 = b.c0 + l.col * VEC;
    const int cnt = l.row < l.rows && l.row < npix ? (npix - l.row + l.rows - 1) / l.rows : 0;
    const int64_t at = l.row, off = (int64_t)ch0 * TR::ESZ;
    const char* x = p.x.p + b.n * p.x.image + at * p.x.pitch + off;
    const char* d = p.dy.p + b.n * p.dy.image + at * p.dy.pitch + off;
    Raw<TR, VEC> xv[NV], dv[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u)
        if (u < cnt) {
            xv[u] = ldr<TR, VEC>(x + u * (l.rows * p.x.pitch));
            dv[u] = ldr<TR, VEC>(d + u * (l.rows * p.dy.pitch));
        }
    const float alpha = p.alpha ? p.alpha[0] : 0.0f;
    BwdConst<VEC> k;
    if (cnt) k.load(p, b.n, ch0);
    for (int g = tid; g < 2 * b.ng; g += TPB) gs[g] = 0.0;
    float s1[VEC], s2[VEC], sa = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
        if (u < cnt) {
            float v[VEC], dy[VEC], g[VEC];
            unraw<TR, VEC>(xv[u], v);
            unraw<TR, VEC>(dv[u], dy);
            sa += k.grad(p.act, alpha, v, dy, g);
#pragma unroll
            for (int j = 0; j < VEC; ++j) { s1[j] += g[j]; s2[j] = fmaf(g[j], v[j], s2[j]); }
        }
#pragma unroll
    for (int j = 0; j < VEC; ++j) { sm[j * TPB + tid] = s1[j]; sm[(VEC + j) * TPB + tid] = s2[j]; }
    row_tree<2 * VEC>(sm, tid, l.row, l.rows, l.cols);
    spread_channels<VEC>(p, sm, l, b.c0, p.part_c + ((int64_t)b.n * p.c + b.c0) * 2, gs, b.g0);
    __syncthreads();
    if (p.part_a) {
        sm[tid] = sa;
        row_tree<1>(sm, tid, tid, TPB, 1);
        if (tid == 0) p.part_a[blockIdx.x] = sm[0];
    }
    if (!cnt) return;
    const double n = p.count;
    float m0[VEC], m1[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int g = (ch0 + j) / p.cg - b.g0;
        m0[j] = (float)(gs[2 * g] / n); m1[j] = (float)(gs[2 * g + 1] / n);
    }
    char* o = p.out.p + b.n * p.out.image + at * p.out.pitch + off;
#pragma unroll
    for (int u = 0; u < NV; ++u)
        if (u < cnt) {
            float v[VEC], dy[VEC], g[VEC];
            unraw<TR, VEC>(xv[u], v);
            unraw<TR, VEC>(dv[u], dy);
            k.grad(p.act, alpha, v, dy, g);
            k.dx(v, g, m0, m1, v);
            stv<TR, VEC>(o + u * (l.rows * p.out.pitch), v);
        }
}

// parameter gradients behind gn_small_bwd_kernel: p.nb parts per channel, p.nb * p.S of dalpha
__global__ __launch_bounds__(TPB) void gn_join_kernel(GnParams p) {
    __shared__ double sm[2 * TPB];
    const bool slope = (int)blockIdx.x >= (p.c + JC - 1) / JC;
    join_params(p, blockIdx.x, slope ? p.nb * p.S : p.nb, sm);
}

// ---- host side ------------------------------------------------------------------------------------------------------
// Splits of an image in both passes: about two workgroups per compute unit in all, at least 32 KB of the tensor per workgroup, and at
// most 8192 pairs (128 KB, in L2) for a workgroup of the second pass to join.  Every workgroup pays for its sums: 32 x 256^2 x 32 bf16
// forward with 256 / 512 / 1024 / 2048 workgroups 77 / 72 / 74 / 77 us, 4 x 117^2 x 256 with 512 / 852 / 1704 of them 21 / 24 / 36;
// 32 x 256^2 x 16 backward with 256 / 512 / 1024: 81 / 64 / 70.  One split less where the last round over the units would be nearly
// empty: 5 x 200^2 x 64 forward 23.2 -> 21.1, backward 38 -> 34; 60 x 80^2 x 32 22.4 -> 19.2, 36 -> 32.
constexpr int WGS = 512, UNITS = 256;
int splits(int esz, int nb, int64_t npix, int c, int groups) {
    const int64_t bytes = npix * c * esz;
    int64_t s = (WGS + nb - 1) / nb;
    auto load = [&](int64_t n) { return (n * nb + UNITS - 1) / UNITS; };       // n-ths of an image on the busiest unit
    if (s > 1 && load(s - 1) * s < load(s) * (s - 1)) --s;
    s = s < bytes / 32768 ? s : bytes / 32768;
    s = s < 8192 / groups ? s : 8192 / groups;
    s = s < npix ? s : npix;
    return s < 1 ? 1 : (int)s;
}

// Small images: slabs of whole groups at least 64 bytes wide, held by 256 threads with at most `most` vectors each.
// (one image of 16 x 16 x 256 bf16: 7 us of kernel, one round trip to memory and the sums, against 4.5 + 7.5 in two passes.)
struct Small { bool ok; int groups, slabs, nv; };
Small small_of(int esz, int vec, int nb, int64_t npix, int c, int groups, int most) {
    const int cg = c / groups;
    Small q = {false, 1, 1, 1};
    if (npix > 65536) return q;
    while (q.groups < groups && (q.groups * cg * esz < 64 || q.groups * cg % vec)) ++q.groups;
    const int cols = q.groups * cg / vec;                            // groups == all: c is a multiple of vec
    if (cols > TPB) return q;
    const int per = (int)((npix + TPB / cols - 1) / (TPB / cols));
    if (per > most) return q;
    q.slabs = (groups + q.groups - 1) / q.groups;
    if ((int64_t)nb * q.slabs > 1 << 23) return q;                    // a launch has at most 2^32 threads
    while (q.nv < per) q.nv *= 2;
    q.ok = true;
    return q;
}

int check_shape(const char* who, int dtype, int nb, int64_t npix, int c, int groups) {
    auto bad = [&](const char* m) { mi_set_error(std::string(who) + ": " + m); return -1; };
    if (dtype != 0 && dtype != 1) return bad("dtype must be 0 or 1");
    if (nb <= 0 || nb > (1 << 20)) return bad("batch must be in 1 .. 2^20");
    if (npix <= 0 || npix > (1LL << 40)) return bad("bad pixel count");
    if (c <= 0 || c > MAX_C) return bad("channels must be in 1 .. 8192");
    if (groups <= 0 || groups > MAX_G || c % groups) return bad("groups must divide the channels and be at most 2048");
    return 0;
}

// vec: narrowed to what this tensor allows; dense: stays true while the tensors are dense
int view_of(const char* who, const char* name, const mi_tensor* t, int64_t npix, int c, int esz, View& v, int& vec, bool& dense) {
    auto bad = [&](const char* m) { mi_set_error(std::string(who) + ": " + name + ": " + m); return -1; };
    if (!t || !t->ptr) return bad("null tensor");
    if (t->ptr2) return bad("a second source is not supported");
    if (t->coff < 0 || t->pitch < t->coff + c) return bad("pitch must cover the channels");
    v.p = (char*)t->ptr + (int64_t)t->coff * esz;
    v.pitch = (int64_t)t->pitch * esz;
    v.image = v.pitch * npix;
    dense = dense && t->pitch == c;
    if ((uintptr_t)v.p % esz) return bad("address is not a multiple of the element size");
    while (vec > 1 && (c % vec || t->pitch % vec || (uintptr_t)v.p % (vec * esz))) vec >>= 1;
    return 0;
}

// Dense tensors of at most 256 channels whose widest vector is shorter than 16 bytes go in runs: backward of 8 x 200^2 x 33 bf16 61 -> 33 us,
// fp32 73 -> 43, of 64 x 200^2 x 36 bf16 (8 bytes) 212 -> 172; forward 29 -> 22, 36 -> 29, 121 -> 111.  Forward with 8-byte vectors from 32 MB on:
// smaller ones lose with the folding of the runs (8 x 200^2 x 36: 21.1 -> 23.2; 4 x 200^2 x 50 fp32, 32 MB: 25.5 -> 25.0).
void take_runs(GnParams& p, int esz, int& vec, bool dense, bool backward) {
    const int full = 16 / esz;
    if (vec == full || !dense || p.c > TPB || p.npix < full) return;
    if (vec * esz == 8 && !backward && (int64_t)p.nb * p.npix * p.c * esz < 1 << 25) return;
    vec = p.rep = full;
    p.c *= full;
    p.tail = (int)(p.npix % full) * p.cr;
    p.npix /= full;
    for (View* v : {&p.x, &p.dy, &p.res, &p.out}) v->pitch *= full;
}

#define GN_SMALL_VEC(KERN, T, V, grid, lds)                                                                 \
    do {                                                                                                    \
        if (q.nv == 1) KERN<T, V, 1><<<grid, TPB, lds, st>>>(p);                                            \
        else if (q.nv == 2) KERN<T, V, 2><<<grid, TPB, lds, st>>>(p);                                       \
        else if (q.nv == 4) KERN<T, V, 4><<<grid, TPB, lds, st>>>(p);                                       \
        else KERN<T, V, 8><<<grid, TPB, lds, st>>>(p);                                                      \
    } while (0)
#define GN_SMALL(KERN, grid, lds)                                                                           \
    do {                                                                                                    \
        if (dtype == 1) {                                                                                   \
            if (vec == 8) GN_SMALL_VEC(KERN, BF16, 8, grid, lds);                                           \
            else if (vec == 4) GN_SMALL_VEC(KERN, BF16, 4, grid, lds);                                      \
            else if (vec == 2) GN_SMALL_VEC(KERN, BF16, 2, grid, lds);                                      \
            else GN_SMALL_VEC(KERN, BF16, 1, grid, lds);                                                    \
        } else {                                                                                            \
            if (vec == 4) GN_SMALL_VEC(KERN, F32, 4, grid, lds);                                            \
            else if (vec == 2) GN_SMALL_VEC(KERN, F32, 2, grid, lds);                                       \
            else GN_SMALL_VEC(KERN, F32, 1, grid, lds);                                                     \
        }                                                                                                   \
        MI_HIP(hipGetLastError());                                                                          \
    } while (0)

#define GN_LAUNCH(KERN, grid, lds)                                                                          \
    do {                                                                                                    \
        if (dtype == 1) {                                                                                   \
            if (vec == 8) KERN<BF16, 8><<<grid, TPB, lds, st>>>(p);                                         \
            else if (vec == 4) KERN<BF16, 4><<<grid, TPB, lds, st>>>(p);                                    \
            else if (vec == 2) KERN<BF16, 2><<<grid, TPB, lds, st>>>(p);                                    \
            else KERN<BF16, 1><<<grid, TPB, lds, st>>>(p);                                                  \
        } else {                                                                                            \
            if (vec == 4) KERN<F32, 4><<<grid, TPB, lds, st>>>(p);                                          \
            else if (vec == 2) KERN<F32, 2><<<grid, TPB, lds, st>>>(p);                                     \
            else KERN<F32, 1><<<grid, TPB, lds, st>>>(p);                                                   \
        }                                                                                                   \
        MI_HIP(hipGetLastError());                                                                          \
    } while (0)

}  // namespace

extern "C" {

size_t mi_groupnorm_act_workspace_bytes(int dtype, int nb, int64_t npix, int c, int groups, int backward) {
    if (check_shape(__func__, dtype, nb, npix, c, groups)) return 0;
    const size_t s = (size_t)nb * splits(dtype ? 2 : 4, nb, npix, c, groups);
    // a small image's backward pass: [nb][c][2] and at most [nb][groups]
    return (s * groups * 2 + (backward ? s * c * 2 + s : 0)) * sizeof(double);
}

int mi_groupnorm_act_fwd(int dtype, int nb, int64_t npix, int c, int groups, const mi_tensor* x, const float* weight,
                         const float* bias, int act, const float* alpha, const mi_tensor* res, const mi_tensor* out,
                         float eps, float* stats, void* workspace, void* stream) {
    if (int r = check_shape(__func__, dtype, nb, npix, c, groups)) return r;
    MI_CHECK(act >= ACT_NONE && act <= ACT_PRELU, "unknown activation");
    MI_CHECK((act == ACT_PRELU) == (alpha != nullptr), "alpha belongs to prelu");
    MI_CHECK(stats && workspace, "null argument");
    MI_CHECK((uintptr_t)workspace % 16 == 0 && (uintptr_t)stats % 8 == 0, "workspace or stats is not aligned");
    MI_CHECK(eps >= 0.0f, "eps must not be negative");
    GnParams p; memset(&p, 0, sizeof(p));
    const int esz = dtype ? 2 : 4;
    int vec = 16 / esz;
    bool dense = true;
    if (int r = view_of(__func__, "x", x, npix, c, esz, p.x, vec, dense)) return r;
    if (int r = view_of(__func__, "out", out, npix, c, esz, p.out, vec, dense)) return r;
    if (res && res->ptr)
        if (int r = view_of(__func__, "res", res, npix, c, esz, p.res, vec, dense)) return r;
    p.w = weight; p.b = bias; p.alpha = alpha; p.stats = stats; p.part = (double*)workspace;
    p.nb = nb; p.npix = npix; p.c = c; p.groups = groups; p.cg = c / groups; p.act = act; p.eps = eps;
    p.cr = c; p.rep = 1; p.count = (double)npix * p.cg;
    hipStream_t st = (hipStream_t)stream;
    const Small q = small_of(esz, vec, nb, npix, c, groups, 8);
    if (q.ok) {
        p.S = q.slabs; p.B = q.groups;
        GN_SMALL(gn_small_fwd_kernel, nb * p.S, q.groups * 2 * sizeof(double));
        return 0;
    }
    p.S = p.B = splits(esz, nb, npix, c, groups);
    take_runs(p, esz, vec, dense, false);
    GN_LAUNCH(gn_stats_kernel, nb * p.S, groups * 2 * sizeof(double));
    GN_LAUNCH(gn_apply_kernel, nb * p.B, groups * 2 * sizeof(float));
    return 0;
}

int mi_groupnorm_act_bwd(int dtype, int nb, int64_t npix, int c, int groups, const mi_tensor* dy, const mi_tensor* x,
                         const float* stats, const float* weight, const float* bias, int act, const float* alpha,
                         const mi_tensor* dx, float* dweight, float* dbias, float* dalpha, void* workspace, void* stream) {
    if (int r = check_shape(__func__, dtype, nb, npix, c, groups)) return r;
    MI_CHECK(act >= ACT_NONE && act <= ACT_PRELU, "unknown activation");
    MI_CHECK((act == ACT_PRELU) == (alpha != nullptr), "alpha belongs to prelu");
    MI_CHECK(!dalpha || alpha, "a gradient of alpha needs alpha");
    MI_CHECK(stats && workspace, "null argument");
    MI_CHECK((uintptr_t)workspace % 16 == 0 && (uintptr_t)stats % 8 == 0, "workspace or stats is not aligned");
    GnParams p; memset(&p, 0, sizeof(p));
    const int esz = dtype ? 2 : 4;
    int vec = 16 / esz;
    bool dense = true;
    if (int r = view_of(__func__, "dy", dy, npix, c, esz, p.dy, vec, dense)) return r;
    if (int r = view_of(__func__, "x", x, npix, c, esz, p.x, vec, dense)) return r;
    if (int r = view_of(__func__, "dx", dx, npix, c, esz, p.out, vec, dense)) return r;
    p.w = weight; p.b = bias; p.alpha = alpha; p.stats = const_cast<float*>(stats);
    p.dw = dweight; p.db = dbias; p.dalpha = dalpha;
    p.nb = nb; p.npix = npix; p.c = c; p.groups = groups; p.cg = c / groups; p.act = act;
    p.cr = c; p.rep = 1; p.count = (double)npix * p.cg;
    hipStream_t st = (hipStream_t)stream;
    const int joins = dweight || dbias || dalpha ? (c + JC - 1) / JC + (dalpha ? 1 : 0) : 0;
    const Small q = small_of(esz, vec, nb, npix, c, groups, 8);
    if (q.ok) {
        p.S = q.slabs; p.B = q.groups;
        p.part_c = (double*)workspace;
        p.part_a = dalpha ? p.part_c + (size_t)nb * c * 2 : nullptr;
        GN_SMALL(gn_small_bwd_kernel, nb * p.S, q.groups * 2 * sizeof(double));
        if (joins) gn_join_kernel<<<joins, TPB, 0, st>>>(p);
        MI_HIP(hipGetLastError());
        return 0;
    }
    p.S = p.B = splits(esz, nb, npix, c, groups);
    take_runs(p, esz, vec, dense, true);
    const size_t s = (size_t)nb * p.S;
    p.part = (double*)workspace;
    p.part_c = p.part + s * groups * 2;
    p.part_a = dalpha ? p.part_c + s * c * 2 : nullptr;
    GN_LAUNCH(gn_bwd_reduce_kernel, nb * p.S, groups * 2 * sizeof(double));
    GN_LAUNCH(gn_bwd_apply_kernel, nb * p.B + joins, groups * 2 * sizeof(float));
    return 0;
}

}  // extern "C"
