// Distillation from a teacher's top logits: rows of V class logits z, per row a list of k teacher logits t with their
// class indices i; temperature T, weight w.  Slots whose index lies outside [0, V) are unused, and so are those with t = -inf.
//
//   q = softmax over the used slots of t / T ,  log p = z / T - lse(z / T)
//   row loss = w T^2 sum_j q_j (log q_j - log p_{i_j}) ;  dz_v = w T gout (p_v - sum_{j: i_j = v} q_j)
//   mean: over the rows with a used slot; the other rows give a loss and a gradient of exactly 0, whatever z holds there.
//
// With zm = max z, tm = max t, St = sum_j exp((t_j - tm) / T), Sz = sum exp((z - zm) / T) and x_j = log q_j - log p_{i_j}:
//   long rows : w T^2 (A / St - log St + log Sz), A = sum_j exp((t_j - tm) / T) ((t_j - tm) - (z_{i_j} - zm)) / T.  One pass over the list; off by
//               a few 2^-24 T^2, which the loss of a list of at most 256 of so many classes exceeds
//   short rows: a list may hold all classes, and those terms then cancel down to 1 / T^2 of their size (16 of 16 classes: 2e-5 of the loss at
//               T = 1, 4 % at 100).  There sum_j q_j (x_j - 1 + exp(-x_j)) + R, R = 1 - sum_j p_{i_j}, of which no part is negative where no class
//               repeats.  An error d that all x_j share (that of log St - log Sz) comes in as d^2 / 2.  R is what is left of Sz without the listed classes:
//               up to T = WIDE_T fp32 sums, which are off by 32 u at most (u = 2^-24), T^2 32 u = 2^-15 of weight in the loss; what lies below that is set
//               to 0.  Above, Sz and the listed part are added in fp64, where the same fp32 exponentials leave exactly nothing behind, and d is taken
//               out again: h = sum_j q_j expm1(-x_j) + R = -d, which - h^2 / 2 removes (d^2 / 2 alone: 5e-4 of the loss of 16 of 16 classes at T = 1e6)
//
// Bandwidth-bound: the forward pass cannot do without one read of z, the backward pass without one read and one write.
//   short rows (up to 4 KB): L neighbouring lanes share a row and hold it in registers
//   long rows : a wave or a workgroup per row, one pass with a running maximum and sum per thread
//   long rows in training: the workgroup holds the row in registers and writes the gradient for gout = 1 in the same
//                          launch (one read and one write in all); the backward pass recomputes it only for another gout
#include <string.h>
#include <type_traits>

#include "rows.h"
#include "../../include/unet_mi355.h"

namespace {

constexpr int TPB = 256;
constexpr int MAX_K = 256;
constexpr int NVMAX = 4;              // 16-byte vectors of a row that a lane holds
constexpr double LN2 = 0.69314718055994531;
// The loss of short rows adds in fp64 above this temperature: 500000 x 256 bf16 63 -> 69 us, 100000 x 2000 bf16 104 -> 123, 2097152 x 16 bf16 42.5 -> 44.
constexpr float WIDE_T = 4.0f;

struct DistParams {
    const char *z, *t, *idx;
    char* dz;
    int64_t rows, zp, dzp;            // pitches in bytes
    int v, k, t_bf16, i64, red, L;    // red: 0 none, 1 mean, 2 sum
    float temp, c, inv_t, wl, wg;     // T, log2(e) / T, 1 / T, weight * T^2 (loss), weight * T (gradient)
    float* loss;                      // [rows] (none) or [1]
    float2* stat;                     // long rows: {max z, Sz}
    double* sums;                     // {sum of the rows' losses, rows with a used slot}
    double* part;                     // [workgroups][2]
    int nparts;
    double* counts;                   // [ncounts] rows with a used slot (training of long rows)
    int ncounts, done;                // done: dz holds the gradient for gout = 1
    const float* gout;
};

__device__ __forceinline__ float list_t(const DistParams& p, int64_t at) {
    return p.t_bf16 ? bf16_to_f32(reinterpret_cast<const unsigned short*>(p.t)[at]) : reinterpret_cast<const float*>(p.t)[at];
}
// class of a slot, -1: unused
__device__ __forceinline__ int list_i(const DistParams& p, int64_t at) {
    const int64_t i = p.i64 ? reinterpret_cast<const int64_t*>(p.idx)[at] : (int64_t)reinterpret_cast<const int*>(p.idx)[at];
    return i >= 0 && i < p.v ? (int)i : -1;
}

// lanes that look at one list in distill_count
__host__ __device__ inline int count_lanes(int k) {
    int L = 1;
    while (L < 64 && L < k) L *= 2;
    return L;
}

// running maximum, sum and weighted gap of a list; gaps in natural units, not over T (T below 1 would take that of a student's class masked with the
// type's lowest value past the end of fp32)
struct ListSum {
    float m = -INFINITY, s = 0.0f, a = 0.0f;
    bool some = false;
    // gap_z = z - zm
    __device__ __forceinline__ void add(float t, float gap_z, float c) {
        if (t == -INFINITY) return;
        some = true;
        if (t > m) rescale(t, c);
        const float gap = t - m, e = __builtin_amdgcn_exp2f(gap * c);
        if (e != 0.0f) { s += e; a = fmaf(e, gap - gap_z, a); }
    }
    __device__ __forceinline__ void rescale(float to, float c) {
        const float gap = m - to, f = __builtin_amdgcn_exp2f(gap * c);
        if (f == 0.0f) { s *= f; a = s; }                         // also the first slot: m = -inf; a NaN in s stays, an infinite a does not
        else { a = f * fmaf(gap, s, a); s *= f; }
        m = to;
    }
    // join the lists of L neighbouring lanes: every lane ends with the whole list
    __device__ __forceinline__ void join(int L, float c) {
        const float to = lanes_max(m, L);
        some = (bool)lanes_max(some ? 1.0f : 0.0f, L);
        if (some && m != to) rescale(to, c);
        a = lanes_sum(a, L);
        s = lanes_sum(s, L);
    }
    __device__ __forceinline__ float loss(float sz, const DistParams& p) const {
        return fmaf(p.wg, a / s, p.wl * ((__builtin_amdgcn_logf(sz) - __builtin_amdgcn_logf(s)) * (float)LN2));
    }
};

// One row in the registers of L lanes: vector i of lane l is vector i * L + l of the row; classes behind the end are -inf.
// `fetch` only requests it (a row's last, partial vector as the 16 bytes that end with the row), `take` makes floats of it.
template <class TR, int NV>
struct Row {
    float x[NV][TR::VEC];
    static __device__ __forceinline__ void fetch(uint4 (&raw)[NV], const char* z, int v, int L, int l) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e0 = (i * L + l) * TR::VEC;
            if (e0 < v && v >= TR::VEC) raw[i] = ld_any<TR>(z + (int64_t)min(e0, v - TR::VEC) * TR::ESZ);
        }
    }
    __device__ __forceinline__ void take(const uint4 (&raw)[NV], const char* z, int v, int L, int l) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e0 = (i * L + l) * TR::VEC;
            if (v < TR::VEC) {
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) x[i][j] = e0 + j < v ? ld_one<TR>(z, e0 + j) : -INFINITY;
                continue;
            }
            if ((i + 1) * L * TR::VEC <= v) {                     // the same for all lanes: they all hold whole vectors
                unpack_vec<TR>(raw[i], x[i]);
                continue;
            }
            uint4 w = raw[i];
            if (v % TR::VEC) {                                    // the same for all lanes
                const int over = e0 + TR::VEC - v;                // > 0: the partial vector, its first class lies `over` up
                if (over > 0) w = down<TR>(w, over);
            }
            unpack_vec<TR>(w, x[i]);
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) x[i][j] = e0 + j < v ? x[i][j] : -INFINITY;
        }
    }
    __device__ __forceinline__ float max_of(int L) const {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) m = fmaxf(m, x[i][j]);
        return lanes_max(m, L);
    }
    // x <- exp((x - m) / T); returns the sum
    __device__ __forceinline__ float exp_of(float m, float c, int L) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) {
                x[i][j] = __builtin_amdgcn_exp2f((x[i][j] - m) * c);
                s += x[i][j];
            }
        return lanes_sum(s, L);
    }
    // the sum of exp((x - m) / T) in fp64
    __device__ __forceinline__ double exp_sum(float m, float c, int L) const {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) s += (double)__builtin_amdgcn_exp2f((x[i][j] - m) * c);
        return lanes_sum(s, L);
    }
};

// x - 1 + exp(-x) for |x| < 1/2: its series, cut where the next term is less than 2^-24 of the sum
__device__ __forceinline__ float small_part(float x) {
    float s = 1.0f / 40320.0f;
    s = fmaf(s, x, -1.0f / 5040.0f);
    s = fmaf(s, x, 1.0f / 720.0f);
    s = fmaf(s, x, -1.0f / 120.0f);
    s = fmaf(s, x, 1.0f / 24.0f);
    s = fmaf(s, x, -1.0f / 6.0f);
    s = fmaf(s, x, 0.5f);
    return s * x * x;
}

// {a, b} added over a workgroup of T threads in a fixed order; thread 0 has the sums
template <int T>
__device__ __forceinline__ double2 block_sum2(double a, double b) {
    __shared__ double sm[2][T / 64];
    for (int o = 32; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); b += __shfl_xor(b, o, 64); }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { sm[0][threadIdx.x >> 6] = a; sm[1][threadIdx.x >> 6] = b; }
    __syncthreads();
    a = b = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < T / 64; ++w) { a += sm[0][w]; b += sm[1][w]; }
    return make_double2(a, b);
}
// (loss, count) of a workgroup's rows -> part[blockIdx.x]
template <int T>
__device__ __forceinline__ void block_part(const DistParams& p, double loss, double count) {
    const double2 v = block_sum2<T>(loss, count);
    if (threadIdx.x == 0) reinterpret_cast<double2*>(p.part)[blockIdx.x] = v;
}

// ---- short rows -----------------------------------------------------------------------------------------------------
// 524288 rows of 16 bf16 classes, 4 slots: forward 15 us (33 MB), backward 15 us (50 MB); 50001 x 133 fp32, 5 slots: 13 us (29 MB) and
// 17 us (55 MB).  Such calls are bounded by the latency of a row or two per thread (0.3 of the wave cycles issue); 2097152 rows of 16:
// forward 43 us, 3.1 TB/s.
// SL slots of a row's list in the registers of a lane: slot j of the list is slot j / L of lane j % L, or slot j % 4 of lane j / 4 where every lane
// has four (one or two loads in place of four: 2097152 rows of 16 bf16 classes, forward 51 -> 43 us).  `fetch` only requests them.
typedef unsigned word4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned half4 __attribute__((ext_vector_type(2), aligned(2)));
template <int SL>
struct Slots {
    unsigned lo[SL], hi[SL], t[SL];
    __device__ __forceinline__ void fetch(const DistParams& p, int64_t r, bool in, int L, int l) {
        if constexpr (SL == 4)
            if (p.k == 4 * L) {                                    // every lane has four slots: its own are neighbours
                const int64_t at = in ? r * p.k + 4 * l : 4 * l;
                if (p.i64) {
                    const word4 a = *reinterpret_cast<const word4*>(p.idx + at * 8), b = *reinterpret_cast<const word4*>(p.idx + at * 8 + 16);
                    lo[0] = a.x; hi[0] = a.y; lo[1] = a.z; hi[1] = a.w;
                    lo[2] = b.x; hi[2] = b.y; lo[3] = b.z; hi[3] = b.w;
                } else {
                    const word4 a = *reinterpret_cast<const word4*>(p.idx + at * 4);
                    lo[0] = a.x; lo[1] = a.y; lo[2] = a.z; lo[3] = a.w;
                    hi[0] = hi[1] = hi[2] = hi[3] = 0u;
                }
                if (p.t_bf16) {
                    const half4 a = *reinterpret_cast<const half4*>(p.t + at * 2);
                    t[0] = a.x & 0xffffu; t[1] = a.x >> 16; t[2] = a.y & 0xffffu; t[3] = a.y >> 16;
                } else {
                    const word4 a = *reinterpret_cast<const word4*>(p.t + at * 4);
                    t[0] = a.x; t[1] = a.y; t[2] = a.z; t[3] = a.w;
                }
                if (!in) hi[0] = hi[1] = hi[2] = hi[3] = 0xffffffffu;
                return;
            }
#pragma unroll
        for (int n = 0; n < SL; ++n) {
            const int j = n * L + l;
            lo[n] = hi[n] = 0xffffffffu;
            t[n] = 0u;
            if (in && j < p.k) {
                const int64_t at = r * p.k + j;
                if (p.i64) {
                    const uint2 u = reinterpret_cast<const uint2*>(p.idx)[at];
                    lo[n] = u.x; hi[n] = u.y;
                } else {
                    lo[n] = reinterpret_cast<const unsigned*>(p.idx)[at];
                    hi[n] = 0u;
                }
                if (p.t_bf16) t[n] = reinterpret_cast<const unsigned short*>(p.t)[at];
                else t[n] = reinterpret_cast<const unsigned*>(p.t)[at];
            }
        }
    }
    __device__ __forceinline__ float teacher(const DistParams& p, int n) const { return __uint_as_float(p.t_bf16 ? t[n] << 16 : t[n]); }
    // class, -1: unused (v is at most 2^28: a negative 32-bit index is too large as well)
    __device__ __forceinline__ int cls(const DistParams& p, int n) const {
        return hi[n] == 0u && lo[n] < (unsigned)p.v && teacher(p, n) != -INFINITY ? (int)lo[n] : -1;
    }
};

// the logits and the list are requested one row ahead
template <class TR, int NV, int SL, bool WIDE>
__global__ __launch_bounds__(TPB) void distill_short_fwd(DistParams p) {
    const int L = p.L, l = threadIdx.x & (L - 1), per = TPB / L;
    double loss = 0.0, count = 0.0;
    const int64_t step = (int64_t)gridDim.x * per;
    int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / L;
    uint4 raw[NV];
    Slots<SL> next;
    auto fetch = [&](int64_t row) {
        const bool in = row < p.rows;
        Row<TR, NV>::fetch(raw, p.z + (in ? row : 0) * p.zp, p.v, L, l);
        next.fetch(p, row, in, L, l);
    };
    fetch(r);
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += step, r += step) {
        const bool in = r < p.rows;
        const char* z = p.z + (in ? r : 0) * p.zp;
        Row<TR, NV> x;
        x.take(raw, z, p.v, L, l);
        float t[SL], zi[SL];                                      // -inf: not used
#pragma unroll
        for (int n = 0; n < SL; ++n) {
            const int cls = next.cls(p, n);
            t[n] = cls >= 0 ? next.teacher(p, n) : -INFINITY;
            zi[n] = cls >= 0 ? ld_one<TR>(z, cls) : 0.0f;
        }
        if (r0 + step < p.rows) fetch(r + step);
        const float m = x.max_of(L);
        float s = 0.0f;
        double wide = 0.0;
        if constexpr (WIDE) { wide = x.exp_sum(m, p.c, L); s = (float)wide; }
        else s = x.exp_of(m, p.c, L);
        float tm = -INFINITY;
#pragma unroll
        for (int n = 0; n < SL; ++n) tm = fmaxf(tm, t[n]);
        tm = lanes_max(tm, L);
        float et[SL], ez[SL], gap[SL], st = 0.0f;
        std::conditional_t<WIDE, double, float> listed = 0.0f;
#pragma unroll
        for (int n = 0; n < SL; ++n) {
            et[n] = ez[n] = gap[n] = 0.0f;
            if (n && n * L >= p.k) continue;                      // no lane has such a slot
            const bool used = t[n] != -INFINITY;
            const float a = t[n] - tm, b = zi[n] - m;
            et[n] = used ? __builtin_amdgcn_exp2f(a * p.c) : 0.0f;
            ez[n] = used ? __builtin_amdgcn_exp2f(b * p.c) : 0.0f;
            gap[n] = used ? a - b : 0.0f;
            st += et[n]; listed += ez[n];
        }
        st = lanes_sum(st, L);                                    // 0: no slot is used
        listed = lanes_sum(listed, L);
        const float inv_z = __builtin_amdgcn_rcpf(s), inv_q = __builtin_amdgcn_rcpf(st);      // good to one unit; s and st are 1 at least
        float rest;
        if constexpr (WIDE) {
            rest = (float)(wide - listed) * inv_z;
        } else {
            rest = (s - listed) * inv_z;
            if (fabsf(rest) < 0x1p-19f) rest = 0.0f;              // 32 steps of fp32: such sums cannot tell it from nothing
        }
        const float shift = (__builtin_amdgcn_logf(st) - __builtin_amdgcn_logf(s)) * (float)LN2;
        // far: q x T, in natural units (over T a class masked with the type's lowest value could pass the end of fp32)
        float part = 0.0f, small = 0.0f, far = 0.0f;
#pragma unroll
        for (int n = 0; n < SL; ++n) {
            if (n && n * L >= p.k) continue;
            const float q = et[n] * inv_q, d = fmaf(gap[n], p.inv_t, -shift);
            const bool near = fabsf(d) < 0.5f;
            part += near ? q * small_part(d) : fmaf(ez[n], inv_z, -q);
            far += near || q == 0.0f ? 0.0f : q * fmaf(-p.temp, shift, gap[n]);
            if constexpr (WIDE) small += near ? q * d : 0.0f;
        }
        float row;
        if constexpr (WIDE) {
            part = lanes_sum(part, L) + rest;
            const float h = part - lanes_sum(small, L);
            row = fmaf(p.wl, fmaf(-0.5f * h, h, part), p.wg * lanes_sum(far, L));
        } else {
            row = fmaf(p.wl, rest, lanes_sum(fmaf(p.wl, part, p.wg * far), L));
        }
        if (l == 0 && in) {
            const bool some = st != 0.0f;
            if (!some) row = 0.0f;
            if (p.red == 0) p.loss[r] = row;
            if (some) { loss += row; count += 1.0; }
        }
    }
    if (p.red) block_part<TPB>(p, loss, count);
}

// weights of a row's list into LDS (L lanes, k slots): qi class or -1, qw weight, qt teacher logit (may be qw).  Returns whether a slot is used.
__device__ __forceinline__ bool list_weights(const DistParams& p, int64_t r, bool in, int L, int l, int* qi, float* qw, float* qt) {
    float m = -INFINITY;
    bool some = false;
    if (in)
        for (int j = l; j < p.k; j += L) {
            int i = list_i(p, r * p.k + j);
            const float t = list_t(p, r * p.k + j);
            if (t == -INFINITY) i = -1;
            if (i >= 0) { m = fmaxf(m, t); some = true; }
            qi[j] = i; qt[j] = t;
        }
    m = lanes_max(m, L);
    some = (bool)lanes_max(some ? 1.0f : 0.0f, L);
    float s = 0.0f;
    if (in)
        for (int j = l; j < p.k; j += L) {
            const float e = qi[j] >= 0 ? __builtin_amdgcn_exp2f((qt[j] - m) * p.c) : 0.0f;
            qw[j] = e; s += e;
        }
    s = lanes_sum(s, L);
    const float inv = 1.0f / s;
    if (in)
        for (int j = l; j < p.k; j += L) qw[j] *= inv;
    return some;
}
// sum of the weights of the slots of class i, in the order of the list
__device__ __forceinline__ float weight_of(const int* qi, const float* qw, int k, int i) {
    float w = 0.0f;
    for (int j = 0; j < k; ++j) w += qi[j] == i ? qw[j] : 0.0f;
    return w;
}
__device__ __forceinline__ float grad_scale(const DistParams& p, int64_t r) {
    const float g = p.gout[p.red ? 0 : r] * p.wg;
    return p.red == 1 ? g / (float)p.sums[1] : g;
}
// LDS written by lanes of this wave is read by others of the same wave
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}

template <class TR, int NV, class F>
__device__ __forceinline__ void store_row(char* dz, int v, int L, int l, F f) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e0 = (i * L + l) * TR::VEC;
        float __attribute__((aligned(16))) d[TR::VEC];
        f(i, e0, d);
        if ((i + 1) * L * TR::VEC <= v || e0 + TR::VEC <= v) {
            st_any(dz + (int64_t)e0 * TR::ESZ, pack_vec<TR>(d));
        } else {
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j)
                if (e0 + j < v) st_one<TR>(dz, e0 + j, d[j]);
        }
    }
}

// the list in registers; every slot's weight is taken off the class it names by comparing, in the order of the list
template <class TR, int NV, int SL>
__global__ __launch_bounds__(TPB) void distill_short_bwd_reg(DistParams p) {
    const int L = p.L, l = threadIdx.x & (L - 1), per = TPB / L, first = (threadIdx.x & 63) - l;
    const int64_t step = (int64_t)gridDim.x * per;
    int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / L;
    uint4 raw[NV];
    Slots<SL> next;
    auto fetch = [&](int64_t row) {
        const bool in = row < p.rows;
        Row<TR, NV>::fetch(raw, p.z + (in ? row : 0) * p.zp, p.v, L, l);
        next.fetch(p, row, in, L, l);
    };
    fetch(r);
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += step, r += step) {
        const bool in = r < p.rows;
        Row<TR, NV> x;
        x.take(raw, p.z + (in ? r : 0) * p.zp, p.v, L, l);
        const Slots<SL> now = next;
        if (r0 + step < p.rows) fetch(r + step);
        const float m = x.max_of(L), s = x.exp_of(m, p.c, L);
        float tm = -INFINITY, q[SL], total = 0.0f;
        int cls[SL];
        bool some = false;
#pragma unroll
        for (int n = 0; n < SL; ++n) {
            cls[n] = now.cls(p, n);
            if (cls[n] >= 0) { tm = fmaxf(tm, now.teacher(p, n)); some = true; }
        }
        tm = lanes_max(tm, L);
        some = (bool)lanes_max(some ? 1.0f : 0.0f, L);
#pragma unroll
        for (int n = 0; n < SL; ++n) {
            q[n] = cls[n] >= 0 ? __builtin_amdgcn_exp2f((now.teacher(p, n) - tm) * p.c) : 0.0f;
            total += q[n];
        }
        total = lanes_sum(total, L);
        const float g = in ? grad_scale(p, r) : 0.0f, inv = 1.0f / s, qs = 1.0f / total;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) x.x[i][j] *= inv;
#pragma unroll
        for (int n = 0; n < SL; ++n) {
            const float w = q[n] * qs;
            for (int o = 0; o < L && n * L + o < p.k; ++o) {       // the same for all lanes
                const int c = L == 1 ? cls[n] : __shfl(cls[n], first + o, 64);
                const float wo = L == 1 ? w : __shfl(w, first + o, 64);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < TR::VEC; ++j) x.x[i][j] -= c == (i * L + l) * TR::VEC + j ? wo : 0.0f;
            }
        }
        if (in)
            store_row<TR, NV>(p.dz + r * p.dzp, p.v, L, l, [&](int i, int, float* d) {
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) d[j] = some ? g * x.x[i][j] : 0.0f;
            });
    }
}

// floats of LDS per row of the kernel below: class weights (whole vectors), classes and weights of the slots; 16-byte rows
__host__ __device__ __forceinline__ int lds_row(int vec, int v, int k) { return (v + vec - 1) / vec * vec + (2 * k + 3) / 4 * 4; }

// any list: the slots' weights are put down at their classes in LDS.  Logits and list are requested one row ahead: nothing else is read.
template <class TR, int NV>
__global__ __launch_bounds__(TPB) void distill_short_bwd(DistParams p) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int L = p.L, l = threadIdx.x & (L - 1), per = TPB / L, slot = threadIdx.x / L, va = (p.v + TR::VEC - 1) / TR::VEC * TR::VEC;
    float* acc = lds + slot * lds_row(TR::VEC, p.v, p.k);
    int* qi = reinterpret_cast<int*>(acc + va);
    float* qw = reinterpret_cast<float*>(qi) + p.k;
    const int64_t step = (int64_t)gridDim.x * per;
    int64_t r = (int64_t)blockIdx.x * per + slot;
    uint4 raw[NV];
    Slots<4> next;
    auto fetch = [&](int64_t row) {
        const bool in = row < p.rows;
        Row<TR, NV>::fetch(raw, p.z + (in ? row : 0) * p.zp, p.v, L, l);
        next.fetch(p, row, in, L, l);
    };
    fetch(r);
    const bool near = p.k == 4 * L;                               // which slot of the list a lane's n-th is
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += step, r += step) {
        const bool in = r < p.rows;
        for (int i = 4 * l; i < va; i += 4 * L) *reinterpret_cast<float4*>(acc + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        Row<TR, NV> x;
        x.take(raw, p.z + (in ? r : 0) * p.zp, p.v, L, l);
        float q[4], tm = -INFINITY, total = 0.0f;
        int cls[4];
        bool some = false;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            cls[n] = next.cls(p, n);
            q[n] = next.teacher(p, n);
            if (cls[n] >= 0) { tm = fmaxf(tm, q[n]); some = true; }
        }
        if (r0 + step < p.rows) fetch(r + step);
        tm = lanes_max(tm, L);
        some = (bool)lanes_max(some ? 1.0f : 0.0f, L);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            q[n] = cls[n] >= 0 ? __builtin_amdgcn_exp2f((q[n] - tm) * p.c) : 0.0f;
            total += q[n];
        }
        const float qs = 1.0f / lanes_sum(total, L);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int j = near ? 4 * l + n : n * L + l;
            q[n] *= qs;
            if (j < p.k) { qi[j] = cls[n]; qw[j] = q[n]; }
        }
        wave_sync();
        bool twice = false;                                       // a class that already has a weight
#pragma unroll
        for (int n = 0; n < 4; ++n)
            if (cls[n] >= 0) twice |= atomicExch(acc + cls[n], q[n]) != 0.0f;
        if (lanes_max(twice ? 1.0f : 0.0f, L) != 0.0f) {
            wave_sync();
#pragma unroll
            for (int n = 0; n < 4; ++n)
                if (cls[n] >= 0) acc[cls[n]] = weight_of(qi, qw, p.k, cls[n]);
        }
        const float m = x.max_of(L), s = x.exp_of(m, p.c, L);
        wave_sync();
        if (in) {
            const float g = grad_scale(p, r), inv = 1.0f / s;
            store_row<TR, NV>(p.dz + r * p.dzp, p.v, L, l, [&](int i, int e0, float* d) {
                if (e0 < p.v) {
#pragma unroll
                    for (int j = 0; j < TR::VEC; j += 4) *reinterpret_cast<float4*>(d + j) = *reinterpret_cast<const float4*>(acc + e0 + j);
                }
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) d[j] = some ? g * fmaf(x.x[i][j], inv, -d[j]) : 0.0f;
            });
        }
        wave_sync();
    }
}

// ---- long rows: a workgroup per row ---------------------------------------------------------------------------------
// A thread's running {maximum, sum of exp((z - maximum) / T)}.  The sum of a thread that saw nothing above -inf is 0, NaN if it
// saw a NaN.
struct RunMax {
    float m = -INFINITY, s = 0.0f;
    bool nan = false;
    template <int N>
    __device__ __forceinline__ void take(const float* x, float c) {
        float top = x[0];
#pragma unroll
        for (int j = 1; j < N; ++j) top = fmaxf(top, x[j]);
        const float to = fmaxf(m, top);
        if (to == -INFINITY) {
#pragma unroll
            for (int j = 0; j < N; ++j) nan |= x[j] != x[j];
            return;
        }
        float add = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) add += __builtin_amdgcn_exp2f((x[j] - to) * c);
        s = m == to ? s + add : fmaf(s, s != 0.0f ? __builtin_amdgcn_exp2f((m - to) * c) : 1.0f, add);
        m = to;
    }
    __device__ __forceinline__ void join_wave(float c) {
        if (nan) s = NAN;
        const float to = lanes_max(m, 64);
        if (s != 0.0f && m != to) s *= __builtin_amdgcn_exp2f((m - to) * c);
        s = lanes_sum(s, 64);
        m = to;
    }
};
// the waves' {m, s} joined (every thread of the calling wave): Sz of a row without a distribution is NaN
template <int T>
__device__ __forceinline__ float2 join_waves(const float* wm, const float* ws, float c) {
    float bm = -INFINITY, bs = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) bm = fmaxf(bm, wm[w]);
#pragma unroll
    for (int w = 0; w < T / 64; ++w) bs += ws[w] != 0.0f ? ws[w] * __builtin_amdgcn_exp2f((wm[w] - bm) * c) : 0.0f;
    return make_float2(bm, bm == -INFINITY ? NAN : bs);
}
// A long row's vectors, which begin at a cache line (half of one for 64 threads): wherever else the rows begin, loads between two words and
// stores of parts of lines take longer (4096 rows of 32769 bf16 classes: loss 71 -> 60 us, step 145 -> 127).  The classes in front and behind, at
// most 70 (38) in all, belong to a thread each; et is the thread's (>= v: none).
template <class TR> struct Span { const char* x; int head, nv, et; };
template <class TR, int T>
__device__ __forceinline__ Span<TR> span_of(const char* z, int v) {
    Span<TR> s;
    constexpr int A = T >= 256 ? 128 : 64;
    s.head = (int)(-(uintptr_t)z & (A - 1)) / TR::ESZ;
    s.x = z + s.head * TR::ESZ;
    s.nv = (v - s.head) / TR::VEC;
    const int back = T - 1 - (int)threadIdx.x;
    s.et = back < s.head ? back : s.head + s.nv * TR::VEC + (int)threadIdx.x;
    return s;
}
// the loss of a row by one wave, the first 64 entries being in q; lane 0 keeps the books
template <class TR>
__device__ __forceinline__ void row_loss(const DistParams& p, int64_t r, const char* z, float2 st, ListSum& q, double& loss, double& count) {
    for (int j = 64 + (threadIdx.x & 63); j < p.k; j += 64) {
        const int i = list_i(p, r * p.k + j);
        if (i >= 0) q.add(list_t(p, r * p.k + j), ld_one<TR>(z, i) - st.x, p.c);
    }
    q.join(64, p.c);
    if ((threadIdx.x & 63) == 0) {
        const float row = q.some ? q.loss(st.y, p) : 0.0f;
        p.stat[r] = st;
        if (p.red == 0) p.loss[r] = row;
        if (q.some) { loss += row; count += 1.0; }
    }
}

// Loss of long rows, one read.  Loads are in flight eight vectors a thread, the last ones of a row too; the first 64 entries of the list and the
// student's logits of their classes are fetched while the row is on its way.  Bound by the read: 4096 x 32768 bf16 58 us, 4.6 TB/s (lists fetched
// behind the row, four vectors in flight: 64); 5 x 32001 fp32 8 us, the latency of one row.
template <class TR, int T>
__global__ __launch_bounds__(T) void distill_long_fwd(DistParams p) {
    __shared__ float wm[T / 64], ws[T / 64];
    double loss = 0.0, count = 0.0;
    const int tid = threadIdx.x;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const char* z = p.z + r * p.zp;
        const Span<TR> sp = span_of<TR, T>(z, p.v);
        int li = -1;
        float lt = 0.0f, lz = 0.0f;
        if (tid < 64 && tid < p.k) {
            li = list_i(p, r * p.k + tid); lt = list_t(p, r * p.k + tid);
            if (li >= 0) lz = ld_one<TR>(z, li);
        }
        RunMax q;
        int i = tid;
        auto batch = [&](auto nu, int most) {                     // nu vectors, those from `most` on stand for nothing
            constexpr int N = decltype(nu)::value, H = N % 4 ? N : 4;
            constexpr unsigned none = TR::ESZ == 2 ? 0xff80ff80u : 0xff800000u;
            uint4 raw[N];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                raw[u] = make_uint4(none, none, none, none);
                if (u < most) raw[u] = ld_any<TR>(sp.x + (int64_t)(i + u * T) * 16);
            }
#pragma unroll
            for (int h = 0; h < N; h += H) {
                float x[H * TR::VEC];
#pragma unroll
                for (int u = 0; u < H; ++u) unpack_vec<TR>(raw[h + u], x + u * TR::VEC);
                q.take<H * TR::VEC>(x, p.c);
            }
            i += N * T;
        };
        while (i + 7 * T < sp.nv) batch(std::integral_constant<int, 8>{}, 8);
        if (i + 3 * T < sp.nv) batch(std::integral_constant<int, 4>{}, 4);
        if (i < sp.nv) batch(std::integral_constant<int, 3>{}, (sp.nv - i + T - 1) / T);
        if (sp.et < p.v) {
            const float x = ld_one<TR>(z, sp.et);
            q.take<1>(&x, p.c);
        }
        q.join_wave(p.c);
        __syncthreads();
        if ((tid & 63) == 0) { wm[tid >> 6] = q.m; ws[tid >> 6] = q.s; }
        __syncthreads();
        if (tid < 64) {
            const float2 st = join_waves<T>(wm, ws, p.c);
            ListSum l;
            if (li >= 0) l.add(lt, lz - st.x, p.c);
            row_loss<TR>(p, r, z, st, l, loss, count);
        }
    }
    if (p.red) block_part<T>(p, loss, count);
}

// rows with a used slot, per workgroup: up to 64 neighbouring lanes look at a row's list (4096 lists of 32: 7.6 -> 3.5 us, against a thread each)
__global__ __launch_bounds__(TPB) void distill_count(DistParams p) {
    __shared__ int sm[TPB / 64];
    const int L = count_lanes(p.k), l = threadIdx.x & (L - 1), lane = threadIdx.x & 63;
    int n = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * (TPB / L); r0 < p.rows; r0 += (int64_t)gridDim.x * (TPB / L)) {
        const int64_t r = r0 + threadIdx.x / L;
        bool some = false;
        if (r < p.rows)
            for (int j = l; j < p.k; j += L) some |= (list_i(p, r * p.k + j) >= 0) & (list_t(p, r * p.k + j) != -INFINITY);
        const unsigned long long ball = __ballot(some), mine = L == 64 ? ball : ball >> (lane & ~(L - 1)) & ((1ull << L) - 1);
        n += l == 0 && mine != 0 ? 1 : 0;
    }
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (lane == 0) sm[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int w = 0; w < TPB / 64; ++w) all += sm[w];
        p.counts[blockIdx.x] = all;
    }
}

// Loss and gradient for gout = 1 of long rows: up to NV vectors of the row in every thread's registers.  The list and the
// student's logits of its classes are fetched while the row is on its way, so that no wave waits for memory once it is there; as
// a vector's gradient is stored, the same vector of the next row is requested.  The exponentials are taken twice: kept, they
// need twice the registers of the bf16 row, and fewer rows in flight cost more than the arithmetic (4096 x 32768 bf16 step: 160 us
// kept, 138 taken twice, 190 with two passes over memory).  Logits and gradient pass the caches by: 137 -> 123 us (the gradient alone
// 131).  Bound by the read and the write: 108 us of kernel, 5.0 TB/s.
template <class TR, int T, int NV>
__global__ __launch_bounds__(T, 4) void distill_long_step(DistParams p) {
    __shared__ float wm[T / 64], ws[T / 64], qw[MAX_K], qt[MAX_K], qz[MAX_K], scale_s;
    __shared__ int qi[MAX_K], any;
    const int tid = threadIdx.x;
    double n = 0.0;
    if (p.red == 1) {
        for (int i = tid; i < p.ncounts; i += T) n += p.counts[i];
        n = block_sum2<T>(n, 0.0).x;
    }
    if (tid == 0) scale_s = p.red == 1 ? p.wg / (float)(n > 0.0 ? n : 1.0) : p.wg;
    double loss = 0.0, count = 0.0;
    uint4 raw[NV];                                                // vectors behind the end: -inf
    float tail = -INFINITY;
    auto fetch = [&](const Span<TR>& sp, int u) {
        constexpr unsigned none = TR::ESZ == 2 ? 0xff80ff80u : 0xff800000u;
        raw[u] = make_uint4(none, none, none, none);
        if (u * T + tid < sp.nv) raw[u] = ld_any_nt<TR>(sp.x + u * (T * 16) + (unsigned)tid * 16u);
    };
    int64_t r = blockIdx.x;
    if (r < p.rows) {
        const Span<TR> sp = span_of<TR, T>(p.z + r * p.zp, p.v);
#pragma unroll
        for (int u = 0; u < NV; ++u) fetch(sp, u);
        tail = sp.et < p.v ? ld_one<TR>(p.z + r * p.zp, sp.et) : -INFINITY;
    }
    for (; r < p.rows; r += gridDim.x) {
        const char* z = p.z + r * p.zp;
        char* dz = p.dz + r * p.dzp;
        __syncthreads();                                          // the list of the row before has been read
        if (tid < 64) {
            const bool some = list_weights(p, r, true, 64, tid, qi, qw, qt);
            for (int j = tid; j < p.k; j += 64) qz[j] = qi[j] >= 0 ? ld_one<TR>(z, qi[j]) : 0.0f;
            if (tid == 0) any = some;
        }
        // the sum about the thread's own maximum (0 if it saw nothing above -inf), brought to the row's maximum by the join
        RunMax q;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            float x[TR::VEC];
            unpack_vec<TR>(raw[u], x);
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) q.m = fmaxf(q.m, x[j]);
        }
        q.m = fmaxf(q.m, tail);
        const float base = q.m == -INFINITY ? 0.0f : q.m;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            hold(raw[u]);
            float y[TR::VEC];
            unpack_vec<TR>(raw[u], y);
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) { y[j] = __builtin_amdgcn_exp2f((y[j] - base) * p.c); q.s += y[j]; }
        }
        q.s += __builtin_amdgcn_exp2f((tail - base) * p.c);
        q.join_wave(p.c);
        if ((tid & 63) == 0) { wm[tid >> 6] = q.m; ws[tid >> 6] = q.s; }
        __syncthreads();
        const float2 st = join_waves<T>(wm, ws, p.c);
        const bool some = any;
        const float g = scale_s, f = g / st.y;
        const bool more = r + gridDim.x < p.rows;
        const char* zn = p.z + (r + gridDim.x) * p.zp;
        const Span<TR> sp = span_of<TR, T>(z, p.v), next = span_of<TR, T>(zn, p.v);
        char* dv = dz + sp.head * TR::ESZ;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            hold(raw[u]);
            float y[TR::VEC];
            unpack_vec<TR>(raw[u], y);
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) y[j] = some ? f * __builtin_amdgcn_exp2f((y[j] - st.x) * p.c) : 0.0f;
            if (u * T + tid < sp.nv) st_any_nt(dv + u * (T * 16) + (unsigned)tid * 16u, pack_vec<TR>(y));
            if (more) fetch(next, u);
        }
        if (sp.et < p.v) st_one<TR>(dz, sp.et, some ? f * __builtin_amdgcn_exp2f((tail - st.x) * p.c) : 0.0f);
        if (more) tail = next.et < p.v ? ld_one<TR>(zn, next.et) : -INFINITY;
        if (tid < 64) {
            ListSum ls;
            for (int j = tid; j < p.k; j += 64)
                if (qi[j] >= 0) ls.add(qt[j], qz[j] - st.x, p.c);
            ls.join(64, p.c);
            if (tid == 0) {
                p.stat[r] = st;
                if (ls.some) { loss += ls.loss(st.y, p); count += 1.0; }
            }
        }
        __syncthreads();                                          // the classes of the list are written over
        if (some)
            for (int j = tid; j < p.k; j += T) {
                const int i = qi[j];
                if (i >= 0) st_one<TR>(dz, i, g * (__builtin_amdgcn_exp2f((qz[j] - st.x) * p.c) / st.y - weight_of(qi, qw, p.k, i)));
            }
    }
    block_part<T>(p, loss, count);
}

template <class TR>
__global__ __launch_bounds__(TPB) void distill_long_bwd(DistParams p) {
    __shared__ int qi[MAX_K];
    __shared__ float qw[MAX_K];
    __shared__ int any;
    if (p.done && p.gout[0] == 1.0f) return;                      // dz holds this gradient already
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        __syncthreads();
        if (threadIdx.x < 64) {
            const bool some = list_weights(p, r, true, 64, threadIdx.x, qi, qw, qw);
            if (threadIdx.x == 0) any = some;
        }
        __syncthreads();
        const bool some = any;
        const char* z = p.z + r * p.zp;
        char* dz = p.dz + r * p.dzp;
        const float2 st = p.stat[r];
        const float g = grad_scale(p, r), f = g / st.y;
        const int nv = p.v / TR::VEC;
#pragma unroll 4
        for (int i = threadIdx.x; i < nv; i += TPB) {
            float x[TR::VEC];
            unpack_vec<TR>(ld_any_nt<TR>(z + (int64_t)i * 16), x);
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) x[j] = some ? f * __builtin_amdgcn_exp2f((x[j] - st.x) * p.c) : 0.0f;
            st_any_nt(dz + (int64_t)i * 16, pack_vec<TR>(x));
        }
        for (int i = nv * TR::VEC + threadIdx.x; i < p.v; i += TPB)
            st_one<TR>(dz, i, some ? f * __builtin_amdgcn_exp2f((ld_one<TR>(z, i) - st.x) * p.c) : 0.0f);
        __syncthreads();                                          // the classes of the list are written over
        if (some)
            for (int j = threadIdx.x; j < p.k; j += TPB) {
                const int i = qi[j];
                if (i >= 0) {
                    const float pr = __builtin_amdgcn_exp2f((ld_one<TR>(z, i) - st.x) * p.c) / st.y;
                    st_one<TR>(dz, i, g * (pr - weight_of(qi, qw, p.k, i)));
                }
            }
    }
}

// Sums of the workgroups' parts in a fixed order; the loss.  A launch of its own: the last workgroup of the kernel before
// could do it behind a device-wide fence, but that writes the L2 back once per workgroup (4096 x 32768 bf16 step, 512
// workgroups: 182 us against 160).
__global__ __launch_bounds__(1024) void distill_final(DistParams p) {
    double a = 0.0, b = 0.0;
    for (int i = threadIdx.x; i < p.nparts; i += 1024) {
        const double2 v = reinterpret_cast<const double2*>(p.part)[i];
        a += v.x; b += v.y;
    }
    const double2 v = block_sum2<1024>(a, b);
    if (threadIdx.x == 0) {
        const double n = v.y > 0.0 ? v.y : 1.0;                   // no row with a used slot: loss 0
        p.sums[0] = v.x; p.sums[1] = n;
        p.loss[0] = (float)(p.red == 1 ? v.x / n : v.x);
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------
// Short rows: the fewest lanes whose registers (NVMAX vectors each) hold the row and, 4 slots each, its list.  The backward
// pass compares every held class with every slot while that is cheap, slots of other lanes costing their way here as well (not where a lane has few
// rows: 50001 x 133 fp32, 5 slots 17 us, 20 through LDS); else it goes through LDS, with the rows of a workgroup within
// 32 KB, or as few as 64 lanes each leave (four: 40 KB at 2048 bf16 classes and 256 slots).  Steps by comparing and through LDS: 4000000 x 16 bf16, 4 slots (work 64) 173 and 186 us, 2000000 x 21, 4 (96) 143 and 151, 2000000 x 32, 8 (128) 192 and 193; 1000000 x 133 fp32, 5 (60, from many lanes) 526 and 466, 1000000 x 64 fp32, 5 (80) 216
// and 190, 100000 x 1000 bf16, 2 (64) 182 and 167.
// Long rows, forward: a wave per row up to 1024 vectors, 256 threads behind that, 1024 where rows alone do not fill the chip (5 x
// 32001 fp32: 256 threads 13.1 us, 1024 7.8).  Step: the fewest threads of 64, 256, 512, 1024 that hold the row with at
// most 16 vectors each (262144 bytes of row).
constexpr int REG_WORK = 120;
struct Plan {
    bool is_long;
    int L, nv, sl;                   // short rows
    int lds_L, lds_nv;               // the backward pass through LDS; lds_L 0: not used
    int T, blocks;                   // threads and workgroups of the forward pass
    int step_t, step_nv, step_blocks;
    int bwd_blocks, parts;
};
Plan plan_of(int esz, int64_t rows, int v, int k) {
    Plan q;
    memset(&q, 0, sizeof(q));
    const int vec = 16 / esz, nvec = (v + vec - 1) / vec;
    auto least = [&](int64_t per, int64_t cap) { const int64_t b = (rows + per - 1) / per; return (int)(b < cap ? b : cap); };
    auto vectors = [&](int L) { return (nvec + L - 1) / L; };
    q.is_long = nvec > 64 * NVMAX;
    if (!q.is_long) {
        q.L = 1;
        while (q.L < 64 && (nvec > q.L * NVMAX || k > 4 * q.L)) q.L *= 2;
        q.nv = vectors(q.L);
        q.sl = k <= q.L ? 1 : 4;
        q.blocks = q.bwd_blocks = q.parts = least(TPB / q.L, 2048);
        if (k * (q.nv * vec + (q.L > 2 && rows > 4 * (int64_t)q.blocks * (TPB / q.L) ? 32 : 0)) > REG_WORK) {
            q.lds_L = 1;
            while (q.lds_L < 64 && (nvec > q.lds_L * NVMAX || k > 4 * q.lds_L || (TPB / q.lds_L) * lds_row(vec, v, k) * 4 > 32768)) q.lds_L *= 2;
            q.lds_nv = vectors(q.lds_L);
            q.bwd_blocks = least(TPB / q.lds_L, 2048);
        }
        return q;
    }
    q.T = rows < 512 ? 1024 : nvec <= 1024 ? 64 : TPB;
    q.blocks = least(1, q.T == 64 ? 8192 : 2048);
    q.bwd_blocks = least(1, 2048);
    const int full = v / vec;
    if (full <= 16384) {
        q.step_t = rows < 512 ? 1024 : full <= 1024 ? 64 : full <= 4096 ? 256 : full <= 8192 ? 512 : 1024;
        q.step_nv = 2 * ((full + 2 * q.step_t - 1) / (2 * q.step_t));       // empty vectors cost their exponentials: 2048 x 32770 fp32 157 -> 126 us
        if (q.step_t == 64 && q.step_nv < 6) q.step_nv = 6;                 // 256 whole vectors and a bit
        if (q.step_t == 1024 && q.step_nv <= 8) q.step_nv = q.step_nv <= 4 ? 4 : 8;
        q.step_blocks = least(1, q.step_t == 64 ? 4096 : 1024);
    }
    q.parts = q.blocks > q.step_blocks ? q.blocks : q.step_blocks;
    return q;
}
constexpr int COUNTS = 512;

int check_args(const char* who, int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int t_dtype,
               const void* teacher, int i_dtype, const void* index, float temperature, float weight, int reduction) {
    auto bad = [&](const char* m) { mi_set_error(std::string(who) + ": " + m); return -1; };
    if (dtype != 0 && dtype != 1) return bad("dtype must be 0 or 1");
    if (t_dtype != 0 && t_dtype != 1) return bad("teacher dtype must be 0 or 1");
    if (i_dtype != 2 && i_dtype != 3) return bad("index dtype must be 2 (int64) or 3 (int32)");
    if (rows <= 0 || rows > (1LL << 40)) return bad("bad row count");
    if (v <= 0 || v > (1 << 28)) return bad("classes must be in 1 .. 2^28");
    if (k <= 0 || k > MAX_K) return bad("list length must be in 1 .. 256");
    if (pitch < v) return bad("pitch must cover the classes");
    if (!logits || !teacher || !index) return bad("null argument");
    const size_t esz = dtype ? 2 : 4;
    if ((uintptr_t)logits % esz || (uintptr_t)teacher % (t_dtype ? 2 : 4) || (uintptr_t)index % (i_dtype == 2 ? 8 : 4))
        return bad("address is not a multiple of the element size");
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return bad("temperature must be in 1e-6 .. 1e6");
    if (!(weight - weight == 0.0f)) return bad("weight must be finite");
    if (!(fabsf(weight * temperature * temperature) < INFINITY)) return bad("weight * temperature^2 must be within fp32");
    if (reduction < 0 || reduction > 2) return bad("unknown reduction");
    return 0;
}

#define SHORT_NV(KERN, nv, grid, lds, ...)                                                                     \
    do {                                                                                                       \
        if (dtype == 1) {                                                                                      \
            if (nv == 1) KERN<BF16, 1 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                                 \
            else if (nv == 2) KERN<BF16, 2 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                            \
            else if (nv == 3) KERN<BF16, 3 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                            \
            else KERN<BF16, 4 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                                         \
        } else {                                                                                               \
            if (nv == 1) KERN<F32, 1 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                                  \
            else if (nv == 2) KERN<F32, 2 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                             \
            else if (nv == 3) KERN<F32, 3 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                             \
            else KERN<F32, 4 __VA_ARGS__><<<grid, TPB, lds, st>>>(p);                                          \
        }                                                                                                      \
        MI_HIP(hipGetLastError());                                                                             \
    } while (0)
#define COMMA ,

void fill(DistParams& p, const Plan& q, int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int t_dtype,
          const void* teacher, int i_dtype, const void* index, float temperature, float weight, int reduction, void* saved) {
    memset(&p, 0, sizeof(p));
    p.z = (const char*)logits; p.t = (const char*)teacher; p.idx = (const char*)index;
    p.rows = rows; p.v = v; p.k = k; p.zp = pitch * (dtype ? 2 : 4); p.t_bf16 = t_dtype; p.i64 = i_dtype == 2; p.red = reduction;
    p.L = q.L; p.nparts = q.blocks;
    p.temp = temperature; p.wl = weight * temperature * temperature; p.wg = weight * temperature;
    p.inv_t = 1.0f / temperature; p.c = (float)(1.4426950408889634 / (double)temperature);
    p.sums = (double*)saved; p.part = p.sums + 2;
    p.counts = p.part + 2 * q.parts;
    const int64_t per = TPB / count_lanes(k), c = (rows + per - 1) / per;
    p.ncounts = (int)(c < COUNTS ? c : COUNTS);
    p.stat = (float2*)(p.counts + (q.is_long ? COUNTS : 0));
}

}  // namespace

extern "C" {

size_t mi_distill_loss_saved_bytes(int dtype, int64_t rows, int v, int k) {
    if ((dtype != 0 && dtype != 1) || rows <= 0 || v <= 0 || k <= 0 || k > MAX_K) {
        mi_set_error(std::string(__func__) + ": bad sizes");
        return 0;
    }
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    return sizeof(double) * (2 + 2 * (size_t)q.parts) + (q.is_long ? sizeof(double) * COUNTS + sizeof(float2) * (size_t)rows : 0);
}

int mi_distill_loss_fwd(int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int teacher_dtype,
                        const void* teacher, int index_dtype, const void* index, float temperature, float weight, int reduction, float* loss,
                        void* saved, void* stream) {
    if (int r = check_args(__func__, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, weight, reduction)) return r;
    MI_CHECK(loss && saved, "null argument");
    MI_CHECK((uintptr_t)saved % 16 == 0 && (uintptr_t)loss % 4 == 0, "saved or loss is not aligned");
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    DistParams p;
    fill(p, q, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, weight, reduction, saved);
    p.loss = loss;
    hipStream_t st = (hipStream_t)stream;
    if (q.is_long) {
        if (dtype == 1) {
            if (q.T == 64) distill_long_fwd<BF16, 64><<<q.blocks, 64, 0, st>>>(p);
            else if (q.T == TPB) distill_long_fwd<BF16, TPB><<<q.blocks, TPB, 0, st>>>(p);
            else distill_long_fwd<BF16, 1024><<<q.blocks, 1024, 0, st>>>(p);
        } else {
            if (q.T == 64) distill_long_fwd<F32, 64><<<q.blocks, 64, 0, st>>>(p);
            else if (q.T == TPB) distill_long_fwd<F32, TPB><<<q.blocks, TPB, 0, st>>>(p);
            else distill_long_fwd<F32, 1024><<<q.blocks, 1024, 0, st>>>(p);
        }
        MI_HIP(hipGetLastError());
    } else {
        if (temperature > WIDE_T) {
            if (q.sl == 1) SHORT_NV(distill_short_fwd, q.nv, q.blocks, 0, COMMA 1 COMMA true);
            else SHORT_NV(distill_short_fwd, q.nv, q.blocks, 0, COMMA 4 COMMA true);
        } else {
            if (q.sl == 1) SHORT_NV(distill_short_fwd, q.nv, q.blocks, 0, COMMA 1 COMMA false);
            else SHORT_NV(distill_short_fwd, q.nv, q.blocks, 0, COMMA 4 COMMA false);
        }
    }
    if (reduction) {
        distill_final<<<1, 1024, 0, st>>>(p);
        MI_HIP(hipGetLastError());
    }
    return 0;
}

int mi_distill_loss_step_ready(int dtype, int64_t rows, int v, int k, int reduction) {
    if ((dtype != 0 && dtype != 1) || rows <= 0 || v <= 0 || k <= 0 || k > MAX_K || reduction <= 0 || reduction > 2) return 0;
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    return q.step_nv > 0;
}

int mi_distill_loss_step(int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int teacher_dtype,
                         const void* teacher, int index_dtype, const void* index, float temperature, float weight, int reduction, float* loss,
                         void* saved, int64_t dpitch, void* dlogits, void* stream) {
    if (int r = check_args(__func__, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, weight, reduction)) return r;
    MI_CHECK(loss && saved && dlogits, "null argument");
    MI_CHECK((uintptr_t)saved % 16 == 0 && (uintptr_t)loss % 4 == 0, "saved or loss is not aligned");
    MI_CHECK(dpitch >= v, "pitch of the gradient must cover the classes");
    MI_CHECK((uintptr_t)dlogits % (dtype ? 2 : 4) == 0, "address is not a multiple of the element size");
    MI_CHECK(mi_distill_loss_step_ready(dtype, rows, v, k, reduction), "not for these sizes or this reduction (mi_distill_loss_step_ready)");
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    DistParams p;
    fill(p, q, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, weight, reduction, saved);
    p.loss = loss; p.dz = (char*)dlogits; p.dzp = dpitch * (dtype ? 2 : 4);
    hipStream_t st = (hipStream_t)stream;
    p.nparts = q.step_blocks;
    if (reduction == 1) {
        distill_count<<<p.ncounts, TPB, 0, st>>>(p);
        MI_HIP(hipGetLastError());
    }
    bool launched = false;
#define STEP_ONE(TR, T_, NV_)                                                                                  \
    if (q.step_t == T_ && q.step_nv == NV_) { distill_long_step<TR, T_, NV_><<<p.nparts, T_, 0, st>>>(p); launched = true; }
#define STEP_TOP(TR, T_) STEP_ONE(TR, T_, 10) STEP_ONE(TR, T_, 12) STEP_ONE(TR, T_, 14) STEP_ONE(TR, T_, 16)
#define STEP_LAUNCH(TR)                                                                                        \
    do {                                                                                                       \
        STEP_ONE(TR, 64, 6) STEP_ONE(TR, 64, 8) STEP_TOP(TR, 64)                                               \
        STEP_ONE(TR, 256, 6) STEP_ONE(TR, 256, 8) STEP_TOP(TR, 256)                                            \
        STEP_TOP(TR, 512)                                                                                      \
        STEP_ONE(TR, 1024, 4) STEP_ONE(TR, 1024, 8) STEP_TOP(TR, 1024)                                         \
    } while (0)
    if (dtype == 1) STEP_LAUNCH(BF16);
    else STEP_LAUNCH(F32);
    MI_CHECK(launched, "no kernel for this number of classes");
    MI_HIP(hipGetLastError());
    distill_final<<<1, 1024, 0, st>>>(p);
    MI_HIP(hipGetLastError());
    return 0;
}

int mi_distill_loss_bwd(int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int teacher_dtype,
                        const void* teacher, int index_dtype, const void* index, float temperature, float weight, int reduction,
                        const float* grad_out, const void* saved, int after_step, int64_t dpitch, void* dlogits, void* stream) {
    if (int r = check_args(__func__, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, weight, reduction)) return r;
    MI_CHECK(grad_out && saved && dlogits, "null argument");
    MI_CHECK((uintptr_t)saved % 16 == 0 && (uintptr_t)grad_out % 4 == 0, "saved or grad_out is not aligned");
    MI_CHECK(dpitch >= v, "pitch of the gradient must cover the classes");
    MI_CHECK((uintptr_t)dlogits % (dtype ? 2 : 4) == 0, "address is not a multiple of the element size");
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    DistParams p;
    fill(p, q, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, weight, reduction, const_cast<void*>(saved));
    MI_CHECK(!after_step || mi_distill_loss_step_ready(dtype, rows, v, k, reduction), "no mi_distill_loss_step for these arguments");
    p.done = after_step != 0;
    p.gout = grad_out; p.dz = (char*)dlogits; p.dzp = dpitch * (dtype ? 2 : 4);
    hipStream_t st = (hipStream_t)stream;
    if (q.is_long) {
        const int blocks = p.done && q.bwd_blocks > 512 ? 512 : q.bwd_blocks;  // mostly there to leave again
        if (dtype == 1) distill_long_bwd<BF16><<<blocks, TPB, 0, st>>>(p);
        else distill_long_bwd<F32><<<blocks, TPB, 0, st>>>(p);
        MI_HIP(hipGetLastError());
    } else {
        if (q.lds_L) {
            p.L = q.lds_L;
            SHORT_NV(distill_short_bwd, q.lds_nv, q.bwd_blocks, (TPB / q.lds_L) * lds_row(dtype ? 8 : 4, v, k) * 4, );
        } else if (q.sl == 1) {
            SHORT_NV(distill_short_bwd_reg, q.nv, q.bwd_blocks, 0, COMMA 1);
        } else {
            SHORT_NV(distill_short_bwd_reg, q.nv, q.bwd_blocks, 0, COMMA 4);
        }
    }
    return 0;
}

}  // extern "C"
