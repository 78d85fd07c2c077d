// Distillation from a teacher's top logits: rows of V class logits z, per row a list of k teacher logits t with their
// class indices i; temperature T.  Slots whose index lies outside [0, V) are unused, and so are those with t = -inf.
//
//   q = softmax over the used slots of t / T ,  log p = z / T - lse(z / T)
//   row loss = T^2 sum_j q_j (log q_j - log p_{i_j}) ;  dz_v = T gout (p_v - sum_{j: i_j = v} q_j)
//   mean: over the rows with a used slot; the other rows give a loss and a gradient of exactly 0, whatever z holds there.
//
// With zm = max z, tm = max t, e_j = exp((t_j - tm) / T): the row loss is T^2 (A / St - log St + log Sz) where
// A = sum e_j ((t_j - tm) - (z_{i_j} - zm)) / T, St = sum e_j and Sz = sum exp((z - zm) / T): one pass over the row, one
// over the list, nothing that cancels.
//
// Bandwidth-bound: the forward pass cannot do without one read of z, the backward pass without one read and one write.
//   short rows (up to ROW_REG bytes per lane group): L neighbouring lanes share a row and hold it in registers
//   long rows : a workgroup per row, one pass with a running maximum and sum per thread
#include <string.h>

#include "rows.h"
#include "../../include/unet_mi355.h"

namespace {

constexpr int TPB = 256;
constexpr int MAX_K = 256;
constexpr int NVMAX = 4;              // 16-byte vectors of a row that a lane holds
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.69314718055994531;

struct DistParams {
    const char *z, *t, *idx;
    char* dz;
    int64_t rows, zp, dzp;            // pitches in bytes
    int v, k, t_bf16, i64, red, L;    // red: 0 none, 1 mean, 2 sum
    float c, inv_t, T;                // log2(e) / T, 1 / T
    float* loss;                      // [rows] (none) or [1]
    float2* stat;                     // long rows: {max z, Sz}
    double* sums;                     // {sum of the rows' losses, rows with a used slot}
    double* part;                     // [workgroups][2]
    int nparts;
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

// running maximum, sum and weighted gap of a list; natural units (to base 2 a student's class masked with the type's lowest
// value would pass the end of fp32)
struct ListSum {
    float m = -INFINITY, s = 0.0f, a = 0.0f;
    bool some = false;
    // gap_z = (z - zm) / T
    __device__ __forceinline__ void add(float t, float gap_z, float inv_t) {
        if (t == -INFINITY) return;
        some = true;
        if (t > m) rescale(t, inv_t);
        const float x = (t - m) * inv_t, e = __builtin_amdgcn_exp2f(x * LOG2E);
        if (e != 0.0f) { s += e; a = fmaf(e, x - gap_z, a); }
    }
    __device__ __forceinline__ void rescale(float to, float inv_t) {
        const float d = (m - to) * inv_t, f = __builtin_amdgcn_exp2f(d * LOG2E);
        if (f == 0.0f) { s = 0.0f; a = 0.0f; }                    // also the first slot: m = -inf
        else { a = f * fmaf(d, s, a); s *= f; }
        m = to;
    }
    // join the lists of L neighbouring lanes: every lane ends with the whole list
    __device__ __forceinline__ void join(int L, float inv_t) {
        const float to = lanes_max(m, L);
        some = (bool)lanes_max(some ? 1.0f : 0.0f, L);
        if (some && m != to) rescale(to, inv_t);
        a = lanes_sum(a, L);
        s = lanes_sum(s, L);
    }
    __device__ __forceinline__ float loss(float sz, float T) const {
        return T * T * (a / s + (__builtin_amdgcn_logf(sz) - __builtin_amdgcn_logf(s)) * (float)LN2);
    }
};

// one row in the registers of L lanes: vector i of lane l is vector i * L + l of the row; classes behind the end are -inf
template <class TR, int NV>
struct Row {
    float x[NV][TR::VEC];
    __device__ __forceinline__ void load(const char* z, int v, int L, int l) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e0 = (i * L + l) * TR::VEC;
            if (e0 + TR::VEC <= v) {
                unpack_vec<TR>(ld_any<TR>(z + (int64_t)e0 * TR::ESZ), x[i]);
            } else {
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) x[i][j] = e0 + j < v ? ld_one<TR>(z, e0 + j) : -INFINITY;
            }
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
};

// (loss, count) of a workgroup's rows -> part[blockIdx.x]
__device__ __forceinline__ void block_part(const DistParams& p, double loss, double count) {
    __shared__ double sm[2][TPB];
    sm[0][threadIdx.x] = loss; sm[1][threadIdx.x] = count;
    for (int h = TPB / 2; h > 0; h >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < h) {
            sm[0][threadIdx.x] += sm[0][threadIdx.x + h];
            sm[1][threadIdx.x] += sm[1][threadIdx.x + h];
        }
    }
    if (threadIdx.x == 0) { p.part[2 * blockIdx.x] = sm[0][0]; p.part[2 * blockIdx.x + 1] = sm[1][0]; }
}

// ---- short rows -----------------------------------------------------------------------------------------------------
template <class TR, int NV>
__global__ __launch_bounds__(TPB) void distill_short_fwd(DistParams p) {
    const int L = p.L, l = threadIdx.x & (L - 1), per = TPB / L;
    double loss = 0.0, count = 0.0;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += (int64_t)gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / L;
        const bool in = r < p.rows;
        const char* z = p.z + (in ? r : 0) * p.zp;
        Row<TR, NV> x;
        x.load(z, p.v, L, l);
        const float m = x.max_of(L), s = x.exp_of(m, p.c, L);
        ListSum q;
        if (in)
            for (int j = l; j < p.k; j += L) {
                const int i = list_i(p, r * p.k + j);
                if (i >= 0) q.add(list_t(p, r * p.k + j), (ld_one<TR>(z, i) - m) * p.inv_t, p.inv_t);
            }
        q.join(L, p.inv_t);
        if (l == 0 && in) {
            const float row = q.some ? q.loss(s, p.T) : 0.0f;
            if (p.red == 0) p.loss[r] = row;
            if (q.some) { loss += row; count += 1.0; }
        }
    }
    if (p.red) block_part(p, loss, count);
}

// weights of a row's list into LDS (L lanes, k slots): qi class or -1, qw weight summed over the slots of the same class,
// in the order of the list.  Returns whether a slot is used.
__device__ __forceinline__ bool list_weights(const DistParams& p, int64_t r, bool in, int L, int l, int* qi, float* qw) {
    float m = -INFINITY;
    bool some = false;
    if (in)
        for (int j = l; j < p.k; j += L) {
            int i = list_i(p, r * p.k + j);
            const float t = list_t(p, r * p.k + j);
            if (t == -INFINITY) i = -1;
            if (i >= 0) { m = fmaxf(m, t); some = true; }
            qi[j] = i; qw[j] = t;
        }
    m = lanes_max(m, L);
    some = (bool)lanes_max(some ? 1.0f : 0.0f, L);
    float s = 0.0f;
    if (in)
        for (int j = l; j < p.k; j += L) {
            const float e = qi[j] >= 0 ? __builtin_amdgcn_exp2f((qw[j] - m) * p.c) : 0.0f;
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
    const float g = p.gout[p.red ? 0 : r] * p.T;
    return p.red == 1 ? g / (float)p.sums[1] : g;
}
// LDS written by lanes of this wave is read by others of the same wave
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}

template <class TR, int NV>
__global__ __launch_bounds__(TPB) void distill_short_bwd(DistParams p) {
    extern __shared__ float lds[];                                // per row: qi [k], qw [k], acc [v]
    const int L = p.L, l = threadIdx.x & (L - 1), per = TPB / L, slot = threadIdx.x / L;
    int* qi = reinterpret_cast<int*>(lds) + (int64_t)slot * (2 * p.k + p.v);
    float* qw = reinterpret_cast<float*>(qi) + p.k;
    float* acc = qw + p.k;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += (int64_t)gridDim.x * per) {
        const int64_t r = r0 + slot;
        const bool in = r < p.rows;
        Row<TR, NV> x;
        x.load(p.z + (in ? r : 0) * p.zp, p.v, L, l);
        const float m = x.max_of(L), s = x.exp_of(m, p.c, L);
        for (int i = l; i < p.v; i += L) acc[i] = 0.0f;
        const bool some = list_weights(p, r, in, L, l, qi, qw);
        wave_sync();
        if (in && some)
            for (int j = l; j < p.k; j += L)
                if (qi[j] >= 0) acc[qi[j]] = weight_of(qi, qw, p.k, qi[j]);
        wave_sync();
        if (in) {
            const float g = grad_scale(p, r), inv = 1.0f / s;
            char* dz = p.dz + r * p.dzp;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e0 = (i * L + l) * TR::VEC;
                float d[TR::VEC];
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) d[j] = some && e0 + j < p.v ? g * (x.x[i][j] * inv - acc[e0 + j]) : 0.0f;
                if (e0 + TR::VEC <= p.v) {
                    st_any(dz + (int64_t)e0 * TR::ESZ, pack_vec<TR>(d));
                } else {
#pragma unroll
                    for (int j = 0; j < TR::VEC; ++j)
                        if (e0 + j < p.v) st_one<TR>(dz, e0 + j, d[j]);
                }
            }
        }
        wave_sync();
    }
}

// ---- long rows: a workgroup per row ---------------------------------------------------------------------------------
template <class TR>
__global__ __launch_bounds__(TPB) void distill_long_fwd(DistParams p) {
    __shared__ float sm[2][TPB / 64];
    double loss = 0.0, count = 0.0;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const char* z = p.z + r * p.zp;
        float m = -INFINITY, s = 0.0f;
        bool nan = false;
        auto take = [&](const float* x, int n) {
            float top = x[0];
#pragma unroll
            for (int j = 1; j < n; ++j) top = fmaxf(top, x[j]);
            if (top > m) { s *= m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * p.c); m = top; }
            if (m != -INFINITY) {
#pragma unroll
                for (int j = 0; j < n; ++j) s += __builtin_amdgcn_exp2f((x[j] - m) * p.c);
            } else {
#pragma unroll
                for (int j = 0; j < n; ++j) nan |= x[j] != x[j];
            }
        };
        const int nv = p.v / TR::VEC;
#pragma unroll 4
        for (int i = threadIdx.x; i < nv; i += TPB) {
            float x[TR::VEC];
            unpack_vec<TR>(ld_any<TR>(z + (int64_t)i * 16), x);
            take(x, TR::VEC);
        }
        for (int i = nv * TR::VEC + threadIdx.x; i < p.v; i += TPB) {
            const float x = ld_one<TR>(z, i);
            take(&x, 1);
        }
        if (nan) s = NAN;
        const float wm = lanes_max(m, 64);
        s = lanes_sum(m == wm && m != -INFINITY ? s : s * (s != 0.0f ? __builtin_amdgcn_exp2f((m - wm) * p.c) : 1.0f), 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { sm[0][threadIdx.x >> 6] = wm; sm[1][threadIdx.x >> 6] = s; }
        __syncthreads();
        if (threadIdx.x < 64) {
            float bm = -INFINITY, bs = 0.0f;
#pragma unroll
            for (int w = 0; w < TPB / 64; ++w) bm = fmaxf(bm, sm[0][w]);
#pragma unroll
            for (int w = 0; w < TPB / 64; ++w) {
                const float sw = sm[1][w];
                bs += sw != 0.0f ? sw * __builtin_amdgcn_exp2f((sm[0][w] - bm) * p.c) : 0.0f;
            }
            if (bm == -INFINITY) bs = NAN;                        // nothing but -inf (or NaN): no distribution
            const int l = threadIdx.x;
            ListSum q;
            for (int j = l; j < p.k; j += 64) {
                const int i = list_i(p, r * p.k + j);
                if (i >= 0) q.add(list_t(p, r * p.k + j), (ld_one<TR>(z, i) - bm) * p.inv_t, p.inv_t);
            }
            q.join(64, p.inv_t);
            if (l == 0) {
                const float row = q.some ? q.loss(bs, p.T) : 0.0f;
                p.stat[r] = make_float2(bm, bs);
                if (p.red == 0) p.loss[r] = row;
                if (q.some) { loss += row; count += 1.0; }
            }
        }
    }
    if (p.red) block_part(p, loss, count);
}

template <class TR>
__global__ __launch_bounds__(TPB) void distill_long_bwd(DistParams p) {
    __shared__ int qi[MAX_K];
    __shared__ float qw[MAX_K];
    __shared__ int any;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        __syncthreads();
        if (threadIdx.x < 64) {
            const bool some = list_weights(p, r, true, 64, threadIdx.x, qi, qw);
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
            unpack_vec<TR>(ld_any<TR>(z + (int64_t)i * 16), x);
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) x[j] = some ? f * __builtin_amdgcn_exp2f((x[j] - st.x) * p.c) : 0.0f;
            st_any(dz + (int64_t)i * 16, pack_vec<TR>(x));
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

// sums of the workgroups' parts in a fixed order; the loss
__global__ __launch_bounds__(TPB) void distill_final(DistParams p) {
    __shared__ double sm[2][TPB];
    double a = 0.0, b = 0.0;
    for (int i = threadIdx.x; i < p.nparts; i += TPB) { a += p.part[2 * i]; b += p.part[2 * i + 1]; }
    sm[0][threadIdx.x] = a; sm[1][threadIdx.x] = b;
    for (int h = TPB / 2; h > 0; h >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < h) {
            sm[0][threadIdx.x] += sm[0][threadIdx.x + h];
            sm[1][threadIdx.x] += sm[1][threadIdx.x + h];
        }
    }
    if (threadIdx.x == 0) {
        const double n = sm[1][0] > 0.0 ? sm[1][0] : 1.0;         // no row with a used slot: loss 0
        p.sums[0] = sm[0][0]; p.sums[1] = n;
        p.loss[0] = (float)(p.red == 1 ? sm[0][0] / n : sm[0][0]);
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------
struct Plan { bool is_long; int L, nv, blocks; };

// Short rows: the fewest lanes whose registers (NVMAX vectors each) hold the row and whose rows' lists and class
// weights leave the workgroup within 32 KB of LDS.
Plan plan_of(int esz, int64_t rows, int v, int k) {
    Plan q;
    const int vec = 16 / esz, nvec = (v + vec - 1) / vec;
    q.is_long = nvec > 64 * NVMAX;
    q.L = 1;
    while (q.L < 64 && (nvec > q.L * NVMAX || (TPB / q.L) * (2 * k + v) * 4 > 32768)) q.L *= 2;
    q.nv = 1;
    while (q.nv * q.L < nvec) q.nv *= 2;
    const int64_t per = q.is_long ? 1 : TPB / q.L, b = (rows + per - 1) / per;
    q.blocks = (int)(b < 4096 ? b : 4096);
    return q;
}

int check_args(const char* who, int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int t_dtype,
               const void* teacher, int i_dtype, const void* index, float temperature, int reduction) {
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
    if (!(temperature > 0.0f) || !(temperature < INFINITY)) return bad("temperature must be positive and finite");
    if (reduction < 0 || reduction > 2) return bad("unknown reduction");
    return 0;
}

#define SHORT_LAUNCH(KERN, lds)                                                                \
    do {                                                                                       \
        if (dtype == 1) {                                                                      \
            if (q.nv == 1) KERN<BF16, 1><<<q.blocks, TPB, lds, st>>>(p);                       \
            else if (q.nv == 2) KERN<BF16, 2><<<q.blocks, TPB, lds, st>>>(p);                  \
            else KERN<BF16, 4><<<q.blocks, TPB, lds, st>>>(p);                                 \
        } else {                                                                               \
            if (q.nv == 1) KERN<F32, 1><<<q.blocks, TPB, lds, st>>>(p);                        \
            else if (q.nv == 2) KERN<F32, 2><<<q.blocks, TPB, lds, st>>>(p);                   \
            else KERN<F32, 4><<<q.blocks, TPB, lds, st>>>(p);                                  \
        }                                                                                      \
        MI_HIP(hipGetLastError());                                                             \
    } while (0)

void fill(DistParams& p, const Plan& q, int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int t_dtype,
          const void* teacher, int i_dtype, const void* index, float temperature, int reduction, void* saved) {
    memset(&p, 0, sizeof(p));
    p.z = (const char*)logits; p.t = (const char*)teacher; p.idx = (const char*)index;
    p.rows = rows; p.v = v; p.k = k; p.zp = pitch * (dtype ? 2 : 4); p.t_bf16 = t_dtype; p.i64 = i_dtype == 2; p.red = reduction;
    p.L = q.L; p.T = temperature; p.inv_t = 1.0f / temperature; p.c = (float)(1.4426950408889634 / (double)temperature);
    p.sums = (double*)saved; p.part = p.sums + 2; p.nparts = q.blocks;
    p.stat = (float2*)(p.part + 2 * q.blocks);
}

}  // namespace

extern "C" {

size_t mi_distill_loss_saved_bytes(int dtype, int64_t rows, int v, int k) {
    if ((dtype != 0 && dtype != 1) || rows <= 0 || v <= 0 || k <= 0 || k > MAX_K) {
        mi_set_error(std::string(__func__) + ": bad sizes");
        return 0;
    }
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    return sizeof(double) * (2 + 2 * (size_t)q.blocks) + (q.is_long ? sizeof(float2) * (size_t)rows : 0);
}

int mi_distill_loss_fwd(int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int teacher_dtype,
                        const void* teacher, int index_dtype, const void* index, float temperature, int reduction, float* loss,
                        void* saved, void* stream) {
    if (int r = check_args(__func__, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, reduction)) return r;
    MI_CHECK(loss && saved, "null argument");
    MI_CHECK((uintptr_t)saved % 8 == 0 && (uintptr_t)loss % 4 == 0, "saved or loss is not aligned");
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    DistParams p;
    fill(p, q, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, reduction, saved);
    p.loss = loss;
    hipStream_t st = (hipStream_t)stream;
    if (q.is_long) {
        if (dtype == 1) distill_long_fwd<BF16><<<q.blocks, TPB, 0, st>>>(p);
        else distill_long_fwd<F32><<<q.blocks, TPB, 0, st>>>(p);
        MI_HIP(hipGetLastError());
    } else {
        SHORT_LAUNCH(distill_short_fwd, 0);
    }
    if (reduction) {
        distill_final<<<1, TPB, 0, st>>>(p);
        MI_HIP(hipGetLastError());
    }
    return 0;
}

int mi_distill_loss_bwd(int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, int teacher_dtype,
                        const void* teacher, int index_dtype, const void* index, float temperature, int reduction,
                        const float* grad_out, const void* saved, int64_t dpitch, void* dlogits, void* stream) {
    if (int r = check_args(__func__, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, reduction)) return r;
    MI_CHECK(grad_out && saved && dlogits, "null argument");
    MI_CHECK((uintptr_t)saved % 8 == 0 && (uintptr_t)grad_out % 4 == 0, "saved or grad_out is not aligned");
    MI_CHECK(dpitch >= v, "pitch of the gradient must cover the classes");
    MI_CHECK((uintptr_t)dlogits % (dtype ? 2 : 4) == 0, "address is not a multiple of the element size");
    const Plan q = plan_of(dtype ? 2 : 4, rows, v, k);
    DistParams p;
    fill(p, q, dtype, rows, v, pitch, logits, k, teacher_dtype, teacher, index_dtype, index, temperature, reduction, const_cast<void*>(saved));
    p.gout = grad_out; p.dz = (char*)dlogits; p.dzp = dpitch * (dtype ? 2 : 4);
    hipStream_t st = (hipStream_t)stream;
    if (q.is_long) {
        if (dtype == 1) distill_long_bwd<BF16><<<q.blocks, TPB, 0, st>>>(p);
        else distill_long_bwd<F32><<<q.blocks, TPB, 0, st>>>(p);
        MI_HIP(hipGetLastError());
    } else {
        const int lds = (TPB / q.L) * (2 * k + v) * 4;
        SHORT_LAUNCH(distill_short_bwd, lds);
    }
    return 0;
}

}  // extern "C"
