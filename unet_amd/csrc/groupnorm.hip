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
// tensors of the call allow (odd channel counts go element by element: neighbouring lanes still read neighbouring
// addresses).
//
// Sums: a thread adds fp32 differences from its own first value (at most CHUNK of them), so that a mean far from zero
// does not cancel; from there on everything is fp64 plain sums, joined in a fixed order (no atomics).
#include <string.h>

#include "common.h"
#include "../../include/unet_mi355.h"

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_PRELU = 4 };
constexpr int TPB = 256;
constexpr int CHUNK = 256;           // pixels a thread adds in fp32 before the sums move to fp64
constexpr int MAX_C = 8192, MAX_G = 2048;

struct View { char* p; int64_t pitch; };   // p: address of the first channel of the first pixel; pitch in bytes

struct GnParams {
    View x, dy, res, out;
    const float *w, *b, *alpha;
    float* stats;                // [nb][groups][2] mean, rstd
    double* part;                // forward: [nb][S][groups][2] ; backward: the same, then [nb][S][c][2], then [nb * S] dalpha
    double* part_c;
    double* part_a;
    float *dw, *db, *dalpha;
    int nb, c, groups, cg, act, S, B;   // S: splits of an image in the statistics pass, B: in the apply pass
    int64_t npix;
    double eps;
};

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
constexpr float SQRT_HALF = 0.70710678118654752f, INV_SQRT_2PI = 0.39894228040143268f;

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
        for (int j = 0; j < VEC; ++j) u[j] = 0.5f * u[j] * (1.0f + erff(u[j] * SQRT_HALF));
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
            const float phi = INV_SQRT_2PI * __builtin_amdgcn_exp2f(u[j] * u[j] * -0.72134752044448170f);
            g[j] = dy[j] * (0.5f * (1.0f + erff(u[j] * SQRT_HALF)) + u[j] * phi);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = dy[j];
    }
    return da;
}

// Sums of `rows` threads that share a vector column, per channel, in a fixed order: NV doubles per thread in LDS as
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
__device__ __forceinline__ Lane lane_of(int cv, int col0) {
    Lane l;
    l.cols = min(cv - col0, TPB);
    l.rows = TPB / l.cols;
    l.col = threadIdx.x % l.cols; l.row = threadIdx.x / l.cols;
    return l;
}

// ---- forward, pass 1: sum and sum of squares per (image, split, group) -------------------------------------------
template <class TR, int VEC>
__global__ __launch_bounds__(TPB) void gn_stats_kernel(GnParams p) {
    __shared__ double sm[2 * VEC * TPB];
    extern __shared__ double gs[];                                  // [groups][2]
    const int n = blockIdx.x / p.S, s = blockIdx.x % p.S, tid = threadIdx.x;
    const int64_t per = (p.npix + p.S - 1) / p.S;
    const int64_t p0 = s * per, p1 = min(p.npix, p0 + per);
    const char* x = p.x.p + (int64_t)n * p.npix * p.x.pitch;
    for (int g = tid; g < 2 * p.groups; g += TPB) gs[g] = 0.0;
    const int cv = p.c / VEC;
    for (int col0 = 0; col0 < cv; col0 += TPB) {
        const Lane l = lane_of(cv, col0);
        const char* xc = x + (int64_t)(col0 + l.col) * (VEC * TR::ESZ);
        double d1[VEC], d2[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) d1[j] = d2[j] = 0.0;
        int64_t q = l.row < l.rows ? p0 + l.row : p1;
        while (q < p1) {
            const int64_t left = (p1 - q + l.rows - 1) / l.rows;
            const int cnt = (int)min((int64_t)CHUNK, left);
            float k[VEC], s1[VEC], s2[VEC];
            ldv<TR, VEC>(xc + q * p.x.pitch, k);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.0f;
#pragma unroll 4
            for (int i = 1; i < cnt; ++i) {
                float v[VEC];
                ldv<TR, VEC>(xc + (q + (int64_t)i * l.rows) * p.x.pitch, v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float d = v[j] - k[j];
                    s1[j] += d; s2[j] = fmaf(d, d, s2[j]);
                }
            }
            // sum (k + d) = cnt k + s1 ; sum (k + d)^2 = cnt k^2 + 2 k s1 + s2
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const double kk = k[j], a = s1[j];
                d1[j] += cnt * kk + a;
                d2[j] += cnt * kk * kk + 2.0 * kk * a + s2[j];
            }
            q += (int64_t)cnt * l.rows;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) { sm[j * TPB + tid] = d1[j]; sm[(VEC + j) * TPB + tid] = d2[j]; }
        row_tree<2 * VEC>(sm, tid, l.row, l.rows, l.cols);
        // channels of this slab -> their groups, one thread per group, ascending
        const int c0 = col0 * VEC, c1 = c0 + l.cols * VEC;
        for (int g = c0 / p.cg + tid; g <= (c1 - 1) / p.cg; g += TPB) {
            double a = 0.0, b = 0.0;
            for (int ch = max(c0, g * p.cg); ch < min(c1, (g + 1) * p.cg); ++ch) {
                a += sm[((ch - c0) % VEC) * TPB + (ch - c0) / VEC];
                b += sm[(VEC + (ch - c0) % VEC) * TPB + (ch - c0) / VEC];
            }
            gs[2 * g] += a; gs[2 * g + 1] += b;
        }
        __syncthreads();
    }
    double* out = p.part + (int64_t)blockIdx.x * p.groups * 2;
    for (int g = tid; g < 2 * p.groups; g += TPB) out[g] = gs[g];
}

// ---- forward, pass 2 ----------------------------------------------------------------------------------------------
template <class TR, int VEC>
__global__ __launch_bounds__(TPB) void gn_apply_kernel(GnParams p) {
    extern __shared__ float mr[];                                   // [groups][2] mean, rstd
    const int n = blockIdx.x / p.B, bi = blockIdx.x % p.B, tid = threadIdx.x;
    const double cnt = (double)p.npix * p.cg;
    for (int g = tid; g < p.groups; g += TPB) {
        double a = 0.0, b = 0.0;
        const double* q = p.part + ((int64_t)n * p.S * p.groups + g) * 2;
        for (int s = 0; s < p.S; ++s) { a += q[(int64_t)s * p.groups * 2]; b += q[(int64_t)s * p.groups * 2 + 1]; }
        const double m = a / cnt;
        double var = b / cnt - m * m;
        var = var < 0.0 ? 0.0 : var;                                // a NaN stays
        mr[2 * g] = (float)m; mr[2 * g + 1] = (float)(1.0 / sqrt(var + p.eps));
        if (bi == 0) { float* o = p.stats + ((int64_t)n * p.groups + g) * 2; o[0] = mr[2 * g]; o[1] = mr[2 * g + 1]; }
    }
    __syncthreads();
    const float alpha = p.alpha ? p.alpha[0] : 0.0f;
    const int64_t per = (p.npix + p.B - 1) / p.B;
    const int64_t p0 = bi * per, p1 = min(p.npix, p0 + per);
    const int cv = p.c / VEC;
    for (int col0 = 0; col0 < cv; col0 += TPB) {
        const Lane l = lane_of(cv, col0);
        if (l.row >= l.rows) continue;
        const int ch0 = (col0 + l.col) * VEC;
        float mean[VEC], a[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int g = (ch0 + j) / p.cg;
            mean[j] = mr[2 * g];
            a[j] = mr[2 * g + 1] * (p.w ? p.w[ch0 + j] : 1.0f);
            b[j] = p.b ? p.b[ch0 + j] : 0.0f;
        }
        const int64_t base = (int64_t)n * p.npix, off = (int64_t)ch0 * TR::ESZ;
#pragma unroll 4
        for (int64_t q = p0 + l.row; q < p1; q += l.rows) {
            float v[VEC];
            ldv<TR, VEC>(p.x.p + (base + q) * p.x.pitch + off, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = fmaf(v[j] - mean[j], a[j], b[j]);
            act_apply<VEC>(p.act, alpha, v);
            if (p.res.p) {
                float r[VEC];
                ldv<TR, VEC>(p.res.p + (base + q) * p.res.pitch + off, r);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] += r[j];
            }
            stv<TR, VEC>(p.out.p + (base + q) * p.out.pitch + off, v);
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
            const float* st = p.stats + ((int64_t)n * p.groups + (ch0 + j) / p.cg) * 2;
            mean[j] = st[0]; rstd[j] = st[1];
            w[j] = p.w ? p.w[ch0 + j] : 1.0f;
            b[j] = p.b ? p.b[ch0 + j] : 0.0f;
        }
    }
};

// ---- backward, pass 1: per (image, split) the channel sums of g and g xh, the group sums of w g and w g xh ----------
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
        const Lane l = lane_of(cv, col0);
        const int ch0 = (col0 + l.col) * VEC;
        double d1[VEC], d2[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) d1[j] = d2[j] = 0.0;
        if (l.row < l.rows) {
            BwdConst<VEC> k;
            k.load(p, n, ch0);
            const int64_t base = (int64_t)n * p.npix, off = (int64_t)ch0 * TR::ESZ;
            int64_t q = p0 + l.row;
            while (q < p1) {
                const int64_t left = (p1 - q + l.rows - 1) / l.rows;
                const int cnt = (int)min((int64_t)CHUNK, left);
                float s1[VEC], s2[VEC], sa = 0.0f;
#pragma unroll
                for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.0f;
#pragma unroll 2
                for (int i = 0; i < cnt; ++i) {
                    const int64_t at = base + q + (int64_t)i * l.rows;
                    float v[VEC], d[VEC], u[VEC], g[VEC];
                    ldv<TR, VEC>(p.x.p + at * p.x.pitch + off, v);
                    ldv<TR, VEC>(p.dy.p + at * p.dy.pitch + off, d);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) { v[j] = (v[j] - k.mean[j]) * k.rstd[j]; u[j] = fmaf(v[j], k.w[j], k.b[j]); }
                    sa += act_grad<VEC>(p.act, alpha, u, d, g);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) { s1[j] += g[j]; s2[j] = fmaf(g[j], v[j], s2[j]); }
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) { d1[j] += s1[j]; d2[j] += s2[j]; }
                da += sa;
                q += (int64_t)cnt * l.rows;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) { sm[j * TPB + tid] = d1[j]; sm[(VEC + j) * TPB + tid] = d2[j]; }
        row_tree<2 * VEC>(sm, tid, l.row, l.rows, l.cols);
        const int c0 = col0 * VEC, c1 = c0 + l.cols * VEC;
        double* pc = p.part_c + ((int64_t)blockIdx.x * p.c + c0) * 2;
        for (int ch = tid; ch < c1 - c0; ch += TPB) {
            pc[2 * ch] = sm[(ch % VEC) * TPB + ch / VEC];
            pc[2 * ch + 1] = sm[(VEC + ch % VEC) * TPB + ch / VEC];
        }
        for (int g = c0 / p.cg + tid; g <= (c1 - 1) / p.cg; g += TPB) {
            double a = 0.0, b = 0.0;
            for (int ch = max(c0, g * p.cg); ch < min(c1, (g + 1) * p.cg); ++ch) {
                const double w = p.w ? p.w[ch] : 1.0f;
                a += w * sm[((ch - c0) % VEC) * TPB + (ch - c0) / VEC];
                b += w * sm[(VEC + (ch - c0) % VEC) * TPB + (ch - c0) / VEC];
            }
            gs[2 * g] += a; gs[2 * g + 1] += b;
        }
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

// sums of n values at a stride by a whole workgroup, fixed order; thread 0 has the result
__device__ __forceinline__ double block_sum(const double* q, int64_t n, int64_t stride, double* sm) {
    double a = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += TPB) a += q[i * stride];
    __syncthreads();
    sm[threadIdx.x] = a;
    row_tree<1>(sm, threadIdx.x, threadIdx.x, TPB, 1);
    return sm[0];
}

// ---- backward, pass 2: dx; the workgroups behind the nb * B of them join the channel sums of all images --------------
template <class TR, int VEC>
__global__ __launch_bounds__(TPB) void gn_bwd_apply_kernel(GnParams p) {
    extern __shared__ float gm[];                                   // [groups][2] means of w g and w g xh
    __shared__ double sm[TPB];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= p.nb * p.B) {
        const int ch = (int)blockIdx.x - p.nb * p.B;
        const int64_t n = (int64_t)p.nb * p.S;
        if (ch < p.c) {
            const double a = block_sum(p.part_c + 2 * ch, n, 2 * p.c, sm);
            if (tid == 0 && p.db) p.db[ch] = (float)a;
            const double b = block_sum(p.part_c + 2 * ch + 1, n, 2 * p.c, sm);
            if (tid == 0 && p.dw) p.dw[ch] = (float)b;
        } else {
            const double a = block_sum(p.part_a, n, 1, sm);
            if (tid == 0) p.dalpha[0] = (float)a;
        }
        return;
    }
    const int n = blockIdx.x / p.B, bi = blockIdx.x % p.B;
    const double cnt = (double)p.npix * p.cg;
    for (int g = tid; g < p.groups; g += TPB) {
        double a = 0.0, b = 0.0;
        const double* q = p.part + ((int64_t)n * p.S * p.groups + g) * 2;
        for (int s = 0; s < p.S; ++s) { a += q[(int64_t)s * p.groups * 2]; b += q[(int64_t)s * p.groups * 2 + 1]; }
        gm[2 * g] = (float)(a / cnt); gm[2 * g + 1] = (float)(b / cnt);
    }
    __syncthreads();
    const float alpha = p.alpha ? p.alpha[0] : 0.0f;
    const int64_t per = (p.npix + p.B - 1) / p.B;
    const int64_t p0 = bi * per, p1 = min(p.npix, p0 + per);
    const int cv = p.c / VEC;
    for (int col0 = 0; col0 < cv; col0 += TPB) {
        const Lane l = lane_of(cv, col0);
        if (l.row >= l.rows) continue;
        const int ch0 = (col0 + l.col) * VEC;
        BwdConst<VEC> k;
        k.load(p, n, ch0);
        float m0[VEC], m1[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { const int g = (ch0 + j) / p.cg; m0[j] = gm[2 * g]; m1[j] = gm[2 * g + 1]; }
        const int64_t base = (int64_t)n * p.npix, off = (int64_t)ch0 * TR::ESZ;
#pragma unroll 2
        for (int64_t q = p0 + l.row; q < p1; q += l.rows) {
            float v[VEC], d[VEC], u[VEC], g[VEC];
            ldv<TR, VEC>(p.x.p + (base + q) * p.x.pitch + off, v);
            ldv<TR, VEC>(p.dy.p + (base + q) * p.dy.pitch + off, d);
#pragma unroll
            for (int j = 0; j < VEC; ++j) { v[j] = (v[j] - k.mean[j]) * k.rstd[j]; u[j] = fmaf(v[j], k.w[j], k.b[j]); }
            act_grad<VEC>(p.act, alpha, u, d, g);
#pragma unroll
            for (int j = 0; j < VEC; ++j) u[j] = k.rstd[j] * (fmaf(k.w[j], g[j], -m0[j]) - v[j] * m1[j]);
            stv<TR, VEC>(p.out.p + (base + q) * p.out.pitch + off, u);
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
// Splits of an image in the reduction passes: enough workgroups to fill the chip (2048 = 8 per CU), at least 32 KB of
// the tensor per workgroup, and at most 4096 partial pairs for a workgroup of the second pass to join.
int splits(int esz, int nb, int64_t npix, int c, int groups) {
    const int64_t bytes = npix * c * esz;
    int64_t s = (2048 + nb - 1) / nb;
    s = s < bytes / 32768 ? s : bytes / 32768;
    const int64_t cap = 4096 / groups > 8 ? 4096 / groups : 8;
    s = s < cap ? s : cap;
    s = s < npix ? s : npix;
    return s < 1 ? 1 : (int)s;
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

int view_of(const char* who, const char* name, const mi_tensor* t, int c, int esz, View& v, int& vec) {
    auto bad = [&](const char* m) { mi_set_error(std::string(who) + ": " + name + ": " + m); return -1; };
    if (!t || !t->ptr) return bad("null tensor");
    if (t->ptr2) return bad("a second source is not supported");
    if (t->coff < 0 || t->pitch < t->coff + c) return bad("pitch must cover the channels");
    v.p = (char*)t->ptr + (int64_t)t->coff * esz;
    v.pitch = (int64_t)t->pitch * esz;
    if ((uintptr_t)v.p % esz) return bad("address is not a multiple of the element size");
    while (vec > 1 && (c % vec || t->pitch % vec || (uintptr_t)v.p % (vec * esz))) vec >>= 1;
    return 0;
}

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
    return (s * groups * 2 + (backward ? s * c * 2 + s : 0)) * sizeof(double);
}

int mi_groupnorm_act_fwd(int dtype, int nb, int64_t npix, int c, int groups, const mi_tensor* x, const float* weight,
                         const float* bias, int act, const float* alpha, const mi_tensor* res, const mi_tensor* out,
                         float eps, float* stats, void* workspace, void* stream) {
    if (int r = check_shape(__func__, dtype, nb, npix, c, groups)) return r;
    MI_CHECK(act >= ACT_NONE && act <= ACT_PRELU, "unknown activation");
    MI_CHECK((act == ACT_PRELU) == (alpha != nullptr), "alpha belongs to prelu");
    MI_CHECK(stats && workspace, "null argument");
    MI_CHECK(eps >= 0.0f, "eps must not be negative");
    GnParams p; memset(&p, 0, sizeof(p));
    const int esz = dtype ? 2 : 4;
    int vec = 16 / esz;
    if (int r = view_of(__func__, "x", x, c, esz, p.x, vec)) return r;
    if (int r = view_of(__func__, "out", out, c, esz, p.out, vec)) return r;
    if (res && res->ptr)
        if (int r = view_of(__func__, "res", res, c, esz, p.res, vec)) return r;
    p.w = weight; p.b = bias; p.alpha = alpha; p.stats = stats; p.part = (double*)workspace;
    p.nb = nb; p.npix = npix; p.c = c; p.groups = groups; p.cg = c / groups; p.act = act; p.eps = eps;
    p.S = p.B = splits(esz, nb, npix, c, groups);
    hipStream_t st = (hipStream_t)stream;
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
    GnParams p; memset(&p, 0, sizeof(p));
    const int esz = dtype ? 2 : 4;
    int vec = 16 / esz;
    if (int r = view_of(__func__, "dy", dy, c, esz, p.dy, vec)) return r;
    if (int r = view_of(__func__, "x", x, c, esz, p.x, vec)) return r;
    if (int r = view_of(__func__, "dx", dx, c, esz, p.out, vec)) return r;
    p.w = weight; p.b = bias; p.alpha = alpha; p.stats = const_cast<float*>(stats);
    p.dw = dweight; p.db = dbias; p.dalpha = dalpha;
    p.nb = nb; p.npix = npix; p.c = c; p.groups = groups; p.cg = c / groups; p.act = act;
    p.S = p.B = splits(esz, nb, npix, c, groups);
    const size_t s = (size_t)nb * p.S;
    p.part = (double*)workspace;
    p.part_c = p.part + s * groups * 2;
    p.part_a = dalpha ? p.part_c + s * c * 2 : nullptr;
    hipStream_t st = (hipStream_t)stream;
    GN_LAUNCH(gn_bwd_reduce_kernel, nb * p.S, groups * 2 * sizeof(double));
    GN_LAUNCH(gn_bwd_apply_kernel, nb * p.B + ((dweight || dbias || dalpha) ? c + (dalpha ? 1 : 0) : 0), groups * 2 * sizeof(float));
    return 0;
}

}  // extern "C"
