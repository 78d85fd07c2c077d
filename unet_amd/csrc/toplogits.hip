// The k largest values of every row of class logits with their indices, largest first, equal values by ascending index.
//
// A value's key is a whole number that orders like the value (-0 = +0, NaN above everything); a class's full key is
// (key, ~index): all full keys of a row differ, and their descending order is the answer's order.  Key 0 belongs to no
// value and stands for "none".
//
// Bandwidth-bound: the rows have to be read once.
//   short lists of short rows: L neighbouring lanes hold a row in registers and take the largest out k times
//   everything else: a workgroup per row.  Every thread finds the largest key of its part; at least k classes lie at or
//   above the k-th largest of these maxima.  The row is read again and the classes from there on are gathered in LDS;
//   a class's place is the number of gathered full keys above its own.  Rows with so many equal values that they do not
//   fit get the exact k-th largest full key by halving the interval of full keys.
#include <string.h>

#include "rows.h"
#include "../../include/unet_mi355.h"

namespace {

constexpr int TPB = 256;
constexpr int MAX_K = 256;
constexpr int NVMAX = 4;
constexpr int CAP = 1024;             // gathered classes

struct TopParams {
    const char* x;
    char* val;
    int* idx;
    int64_t rows, xp;
    int v, k, L;
};

__device__ __forceinline__ unsigned key_of(float f) {
    const unsigned b = __float_as_uint(f + 0.0f);                  // -0 -> +0
    if (f != f) return 0xffffffffu;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
typedef unsigned long long u64;
__device__ __forceinline__ u64 full_key(unsigned key, int i) { return ((u64)key << 32) | (unsigned)~i; }

// the value itself is copied (a NaN keeps its bits, -0 its sign)
template <class TR>
__device__ __forceinline__ void emit(const TopParams& p, int64_t r, int place, int i) {
    typedef typename TR::elem E;
    const int64_t at = r * p.k + place;
    reinterpret_cast<E*>(p.val)[at] = reinterpret_cast<const E*>(p.x + r * p.xp)[i];
    p.idx[at] = i;
}

template <class TR, int NV>
__global__ __launch_bounds__(TPB) void top_short(TopParams p) {
    const int L = p.L, l = threadIdx.x & (L - 1), per = TPB / L;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += (int64_t)gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / L;
        const bool in = r < p.rows;
        const char* x = p.x + (in ? r : 0) * p.xp;
        unsigned key[NV][TR::VEC];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e0 = (i * L + l) * TR::VEC;
            if (e0 + TR::VEC <= p.v) {
                float f[TR::VEC];
                unpack_vec<TR>(ld_any<TR>(x + (int64_t)e0 * TR::ESZ), f);
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) key[i][j] = key_of(f[j]);
            } else {
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) key[i][j] = e0 + j < p.v ? key_of(ld_one<TR>(x, e0 + j)) : 0u;
            }
        }
        for (int n = 0; n < p.k; ++n) {
            unsigned best = 0;
            int at = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < NV; ++i)                           // ascending classes: the first of equal keys wins
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j)
                    if (key[i][j] > best) { best = key[i][j]; at = (i * L + l) * TR::VEC + j; }
            for (int o = L >> 1; o > 0; o >>= 1) {
                const unsigned ob = __shfl_xor(best, o, 64);
                const int oa = __shfl_xor(at, o, 64);
                if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
            }
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j)
                    if ((i * L + l) * TR::VEC + j == at) key[i][j] = 0u;
            if (in && l == (n & (L - 1))) emit<TR>(p, r, n, at);
        }
    }
}

// f(key, class) for the classes of a row, TPB threads side by side
template <class TR, class F>
__device__ __forceinline__ void each(const char* x, int v, F f) {
    const int nv = v / TR::VEC;
#pragma unroll 4
    for (int i = threadIdx.x; i < nv; i += TPB) {
        float u[TR::VEC];
        unpack_vec<TR>(ld_any<TR>(x + (int64_t)i * 16), u);
#pragma unroll
        for (int j = 0; j < TR::VEC; ++j) f(key_of(u[j]), i * TR::VEC + j);
    }
    for (int i = nv * TR::VEC + threadIdx.x; i < v; i += TPB) f(key_of(ld_one<TR>(x, i)), i);
}

// number of classes of the row with a full key >= lo, in every thread
template <class TR>
__device__ int count_from(const char* x, int v, u64 lo, int* sm) {
    int n = 0;
    each<TR>(x, v, [&](unsigned key, int i) { n += full_key(key, i) >= lo ? 1 : 0; });
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < TPB / 64; ++w) n += sm[w];
    return n;
}

template <class TR>
__global__ __launch_bounds__(TPB) void top_long(TopParams p) {
    __shared__ u64 cand[CAP];
    __shared__ unsigned top[TPB];
    __shared__ unsigned thr_s;
    __shared__ int count_s, sm[TPB / 64];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const char* x = p.x + r * p.xp;
        u64 lo = 0;
        if (p.v > CAP) {
            unsigned best = 0;
            each<TR>(x, p.v, [&](unsigned key, int) { best = key > best ? key : best; });
            top[threadIdx.x] = best;
            __syncthreads();
            if (threadIdx.x < 64) {
                // the k-th largest of the maxima, bit by bit: the largest number that k of them reach
                unsigned t = 0;
                for (int bit = 31; bit >= 0; --bit) {
                    const unsigned want = t | (1u << bit);
                    int n = 0;
#pragma unroll
                    for (int w = 0; w < TPB / 64; ++w) n += __popcll(__ballot(top[w * 64 + threadIdx.x] >= want));
                    if (n >= p.k) t = want;
                }
                if (threadIdx.x == 0) thr_s = t;
            }
            __syncthreads();
            lo = (u64)thr_s << 32;
        }
        int n = 0;
        for (int tries = 0;; ++tries) {
            if (threadIdx.x == 0) count_s = 0;
            __syncthreads();
            each<TR>(x, p.v, [&](unsigned key, int i) {
                const u64 f = full_key(key, i);
                if (f >= lo) {
                    const int at = atomicAdd(&count_s, 1);
                    if (at < CAP) cand[at] = f;
                }
            });
            __syncthreads();
            n = count_s;
            if (n <= CAP || tries) break;                          // the second time exactly k are gathered
            u64 hi = ~0ull;                                        // count(lo) > CAP >= k; full keys differ
            while (lo < hi) {                                      // the largest full key that k classes reach
                const u64 mid = lo + (hi - lo) / 2 + ((hi - lo) & 1);
                if (count_from<TR>(x, p.v, mid, sm) >= p.k) lo = mid;
                else hi = mid - 1;
            }
            __syncthreads();
        }
        n = n < CAP ? n : CAP;
        for (int a = threadIdx.x; a < n; a += TPB) {
            const u64 f = cand[a];
            int place = 0;
            for (int b = 0; b < n; ++b) place += cand[b] > f ? 1 : 0;
            if (place < p.k) emit<TR>(p, r, place, (int)~(unsigned)f);
        }
        __syncthreads();
    }
}

struct Plan { bool is_long; int L, nv, blocks; };
// Taking the largest out costs about 3 operations per held class and 10 per lane exchange for every entry of the list:
// lists of up to 16 entries of rows that 64 lanes hold; everything else is a workgroup's.
Plan plan_of(int esz, int64_t rows, int v, int k) {
    Plan q;
    const int vec = 16 / esz, nvec = (v + vec - 1) / vec;
    q.is_long = nvec > 64 * NVMAX || k > 16;
    q.L = 1;
    while (q.L < 64 && nvec > q.L * NVMAX) q.L *= 2;
    q.nv = 1;
    while (q.nv < NVMAX && q.nv * q.L < nvec) q.nv *= 2;
    const int64_t per = q.is_long ? 1 : TPB / q.L, b = (rows + per - 1) / per;
    q.blocks = (int)(b < 16384 ? b : 16384);
    return q;
}

#define SHORT_LAUNCH(KERN)                                                                     \
    do {                                                                                       \
        if (dtype == 1) {                                                                      \
            if (q.nv == 1) KERN<BF16, 1><<<q.blocks, TPB, 0, st>>>(p);                         \
            else if (q.nv == 2) KERN<BF16, 2><<<q.blocks, TPB, 0, st>>>(p);                    \
            else KERN<BF16, 4><<<q.blocks, TPB, 0, st>>>(p);                                   \
        } else {                                                                               \
            if (q.nv == 1) KERN<F32, 1><<<q.blocks, TPB, 0, st>>>(p);                          \
            else if (q.nv == 2) KERN<F32, 2><<<q.blocks, TPB, 0, st>>>(p);                     \
            else KERN<F32, 4><<<q.blocks, TPB, 0, st>>>(p);                                    \
        }                                                                                      \
    } while (0)

}  // namespace

extern "C" int mi_top_logits(int dtype, int64_t rows, int v, int64_t pitch, const void* logits, int k, void* values, int32_t* index,
                             void* stream) {
    MI_CHECK(dtype == 0 || dtype == 1, "dtype must be 0 or 1");
    MI_CHECK(rows > 0 && rows <= (1LL << 40), "bad row count");
    MI_CHECK(v > 0 && v <= (1 << 28), "classes must be in 1 .. 2^28");
    MI_CHECK(k > 0 && k <= MAX_K && k <= v, "list length must be in 1 .. 256 and at most the number of classes");
    MI_CHECK(pitch >= v, "pitch must cover the classes");
    MI_CHECK(logits && values && index, "null argument");
    const size_t esz = dtype ? 2 : 4;
    MI_CHECK((uintptr_t)logits % esz == 0 && (uintptr_t)values % esz == 0 && (uintptr_t)index % 4 == 0, "address is not a multiple of the element size");
    const Plan q = plan_of((int)esz, rows, v, k);
    TopParams p;
    p.x = (const char*)logits; p.val = (char*)values; p.idx = index;
    p.rows = rows; p.xp = pitch * (int64_t)esz; p.v = v; p.k = k; p.L = q.L;
    hipStream_t st = (hipStream_t)stream;
    if (q.is_long) {
        if (dtype == 1) top_long<BF16><<<q.blocks, TPB, 0, st>>>(p);
        else top_long<F32><<<q.blocks, TPB, 0, st>>>(p);
    } else {
        SHORT_LAUNCH(top_short);
    }
    MI_HIP(hipGetLastError());
    return 0;
}
