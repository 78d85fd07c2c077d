// The k largest values of every row of class logits with their indices, largest first, equal values by ascending index.
//
// A value's key is a whole number that orders like the value (-0 = +0, NaN above everything); a class's full key is
// (key, ~index): all full keys of a row differ, and their descending order is the answer's order.  Key 0 belongs to no
// value and stands for "none".
//
// Bandwidth-bound: the rows have to be read once.
//   top_short: L neighbouring lanes hold a row in registers and take the largest out k times, or order it by networks
//   top_wave : a wave holds the row; the k-th largest key is found bit by bit, by counting the keys from there on, the k classes
//              are gathered in LDS (equal keys by ascending class) and placed by the number of full keys above their own
//   top_long : a workgroup streams the row and keeps the largest key of every thread's part.  At least k classes lie at or above
//              the k-th largest of the maxima of groups of threads; only threads that saw such a class have theirs read again
//              (from L2), the classes from there on are gathered in LDS and placed.  Rows with so many equal values that they do
//              not fit get the exact k-th largest key, the classes above it and the first ones at it
#include <string.h>
#include <type_traits>

#include "rows.h"
#include "../../include/unet_mi355.h"

namespace {

constexpr int TPB = 256;
constexpr int MAX_K = 256;
constexpr int NVMAX = 4;
constexpr int SORT = -1;

struct TopParams {
    const char* x;
    char* val;
    int* idx;
    int64_t rows, xp;
    int v, k, L, G, by_lanes;
};

__device__ __forceinline__ unsigned key_of(float f) {
    const unsigned b = __float_as_uint(f + 0.0f);                  // -0 -> +0
    return f != f ? 0xffffffffu : b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
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

// the keys of a row in the registers of L lanes: vector i of lane l is vector i * L + l; behind the end 0
template <class TR, int NV>
__device__ __forceinline__ void load_keys(const char* x, int v, int L, int l, unsigned (&key)[NV][TR::VEC]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e0 = (i * L + l) * TR::VEC;
        if (e0 + TR::VEC <= v) {
            float f[TR::VEC];
            unpack_vec<TR>(ld_any<TR>(x + (int64_t)e0 * TR::ESZ), f);
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) key[i][j] = key_of(f[j]);
        } else {
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) key[i][j] = e0 + j < v ? key_of(ld_one<TR>(x, e0 + j)) : 0u;
        }
    }
}

// fp32 keys with their classes as doubles in 1 .. 2, which order like their bits: 32 bits of key, 20 of class
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return __builtin_fmin(a, b); }
__device__ __forceinline__ double key_word(unsigned key, int cls) {
    return __hiloint2double((int)(0x3ff00000u | key >> 12), (int)(key << 20 | (0xfffffu - (unsigned)cls)));
}

// Networks on words: a holds the larger one after swap_down.  sort4, sort8: largest first (sort8 by merge exchanges of two sorted halves);
// top_of_two: the N largest of two sorted lists, sorted, in a.
__device__ __forceinline__ void swap_down(unsigned& a, unsigned& b) {
    const unsigned hi = max(a, b), lo = min(a, b);
    a = hi; b = lo;
}
__device__ __forceinline__ void swap_down(double& a, double& b) {
    const double hi = larger(a, b), lo = smaller(a, b);
    a = hi; b = lo;
}
template <class W>
__device__ __forceinline__ void sort4(W* a) {
    swap_down(a[0], a[1]); swap_down(a[2], a[3]);
    swap_down(a[0], a[2]); swap_down(a[1], a[3]);
    swap_down(a[1], a[2]);
}
template <class W>
__device__ __forceinline__ void sort8(W* a) {
    sort4(a); sort4(a + 4);
    swap_down(a[0], a[4]); swap_down(a[1], a[5]); swap_down(a[2], a[6]); swap_down(a[3], a[7]);
    swap_down(a[2], a[4]); swap_down(a[3], a[5]);
    swap_down(a[1], a[2]); swap_down(a[3], a[4]); swap_down(a[5], a[6]);
}
template <int N>
__device__ __forceinline__ void top_of_two(unsigned* a, const unsigned* b) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = max(a[i], b[N - 1 - i]);    // rises, then falls (or a rotation of that)
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(i & o)) swap_down(a[i], a[i + o]);
}

// Sorting over lanes: E = 4 or 8 words a lane, largest first, lane by lane.  Two sorted halves of N lanes each: the first exchange is with the
// mirrored lane and word, the others with lanes at distance N / 2 .. 1, the last ones within the lane.  An exchange takes the larger one
// in the lower lane and the smaller one in the upper; for 32-bit words that is the middle one of the two and of everything or nothing: two
// instructions a word.  67496 rows of 99 classes, 35 of them: bf16 71 -> 17.5 us, fp32 68 -> 36 (found bit by bit before); 300000 x 64, 16:
// 38 -> 27.5 and 57 -> 48 (taken out).
__device__ __forceinline__ unsigned pick(unsigned a, unsigned b, bool upper) {
    const unsigned lim = upper ? 0u : 0xffffffffu;
    return max(min(a, b), min(max(a, b), lim));
}
__device__ __forceinline__ double pick(double a, double b, bool upper) { return (a > b) != upper ? a : b; }
template <int X>
__device__ __forceinline__ unsigned from_lane(unsigned v) {                        // lane ^ X
    if constexpr (X == 1) return lane_move<0xB1>(v);
    else if constexpr (X == 2) return lane_move<0x4E>(v);
    else if constexpr (X == 3) return lane_move<0x1B>(v);
    else if constexpr (X == 4) return lane_move<0x1B>(lane_move<0x141>(v));
    else if constexpr (X == 7) return lane_move<0x141>(v);
    else if constexpr (X == 8) return lane_move<0x128>(v);
    else if constexpr (X == 15) return lane_move<0x140>(v);
    else if constexpr (X == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    } else if constexpr (X == 31) {
        return from_lane<16>(lane_move<0x140>(v));
    } else {
        static_assert(X == 63, "");
        const unsigned m = from_lane<31>(v);
        const auto r = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    }
}
template <int X>
__device__ __forceinline__ double from_lane(double v) {
    return __hiloint2double((int)from_lane<X>((unsigned)__double2hiint(v)), (int)from_lane<X>((unsigned)__double2loint(v)));
}
template <int X, bool MIRROR, int E, class W>
__device__ __forceinline__ void exchange(W* a) {
    const bool upper = threadIdx.x & (MIRROR ? (X + 1) / 2 : X);
    W b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) b[e] = from_lane<X>(a[MIRROR ? E - 1 - e : e]);
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = pick(a[e], b[e], upper);
}
// two sorted halves of N lanes -> one of 2 N
template <int N, int E, class W>
__device__ __forceinline__ void merge_lanes(W* a) {
    exchange<2 * N - 1, true, E>(a);
    if constexpr (N >= 32) exchange<16, false, E>(a);
    if constexpr (N >= 16) exchange<8, false, E>(a);
    if constexpr (N >= 8) exchange<4, false, E>(a);
    if constexpr (N >= 4) exchange<2, false, E>(a);
    if constexpr (N >= 2) exchange<1, false, E>(a);
#pragma unroll
    for (int o = E / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (!(i & o)) swap_down(a[i], a[i + o]);
}
template <int E, class W>
__device__ __forceinline__ void sort_lanes(W* a, int L) {
    if constexpr (E == 8) sort8(a);
    else sort4(a);
    if (L == 1) return;
    merge_lanes<1, E>(a);
    if (L == 2) return;
    merge_lanes<2, E>(a);
    if (L == 4) return;
    merge_lanes<4, E>(a);
    if (L == 8) return;
    merge_lanes<8, E>(a);
    if (L == 16) return;
    merge_lanes<16, E>(a);
    if (L == 32) return;
    merge_lanes<32, E>(a);
}

// The classes found go through LDS (dynamic, [workgroup's rows][k]): the results of a wave's rows are one piece of the output and
// leave it with neighbouring lanes at neighbouring addresses.
// bf16: key and class fit one word, (key, 65535 - class), so that a maximum is one instruction.  Lists of at most K = 4 or 8 come from
// networks: 76 or 108 instructions for the 16 words of two vectors, where taking out costs 40 per entry.  K = 1: the maximum.  K = 0: taken out
// one by one.  2097152 rows of 16 classes, bf16: 4 of them 31 us (3.8 TB/s; taken out 38), 1 of them 21.5 (23), 8 of them 40 (57); 50000 x 512,
// 4 of them: 20 (25).  Bounded by instructions: 380 per row of 16 (630 taken out).
template <class TR, int NV, int K>
__global__ __launch_bounds__(TPB) void top_short(TopParams p) {
    // bf16: (key, class), the key's lower half being that of the value's sign; fp32: the class
    extern __shared__ unsigned found[];
    const int L = p.L, l = threadIdx.x & (L - 1), per = TPB / L, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    unsigned* mine = found + (threadIdx.x / L) * p.k;
    const unsigned* waves = found + wave * (64 / L) * p.k;
    const float inv = 1.0f / (float)p.k;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += (int64_t)gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / L;
        const char* x = p.x + (r < p.rows ? r : 0) * p.xp;
        unsigned key[NV][TR::VEC];
        load_keys<TR, NV>(x, p.v, L, l, key);
        if constexpr (TR::ESZ == 2) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e0 = (i * L + l) * TR::VEC;
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) key[i][j] = (key[i][j] & 0xffff0000u) | (0xffffu - (unsigned)(e0 + j));
                if (e0 + TR::VEC > p.v) {
#pragma unroll
                    for (int j = 0; j < TR::VEC; ++j) key[i][j] = e0 + j < p.v ? key[i][j] : 0u;
                }
            }
        }
        if constexpr (K == SORT) {
            if constexpr (TR::ESZ == 2) {
                sort_lanes<8>(key[0], L);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (l * 8 + e < p.k) mine[l * 8 + e] = key[0][e] ^ 0xffffu;
            } else {
                double w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = key_word(key[0][e], l * 4 + e);
                sort_lanes<4>(w, L);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (l * 4 + e < p.k) mine[l * 4 + e] = 0xfffffu - ((unsigned)__double2loint(w[e]) & 0xfffffu);
            }
        } else if constexpr (K != 0) {
            unsigned* top = key[0];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if constexpr (K == 1) {
#pragma unroll
                    for (int j = 1; j < TR::VEC; ++j) key[i][0] = max(key[i][0], key[i][j]);
                } else if constexpr (K == 8) {
                    sort8(key[i]);
                } else {
                    sort4(key[i]); sort4(key[i] + 4);
                    top_of_two<K>(key[i], key[i] + 4);
                }
                if (i) top_of_two<K>(top, key[i]);
            }
            for (int o = L >> 1; o > 0; o >>= 1) {
                unsigned other[K];
#pragma unroll
                for (int n = 0; n < K; ++n) other[n] = __shfl_xor(top[n], o, 64);
                top_of_two<K>(top, other);
            }
            if (l == 0) {
#pragma unroll
                for (int n = 0; n < K; ++n)
                    if (n < p.k) mine[n] = top[n] ^ 0xffffu;
            }
        } else if constexpr (TR::ESZ == 2) {
            for (int n = 0; n < p.k; ++n) {
                unsigned best = 0;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < TR::VEC; ++j) best = max(best, key[i][j]);
                best = lanes_max(best, L);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < TR::VEC; ++j) key[i][j] = key[i][j] == best ? 0u : key[i][j];
                if (l == 0) mine[n] = best ^ 0xffffu;
            }
        } else {
            for (int n = 0; n < p.k; ++n) {
                unsigned best = 0;
                int at = 0x7fffffff;
#pragma unroll
                for (int i = 0; i < NV; ++i)                       // ascending classes: the first of equal keys wins
#pragma unroll
                    for (int j = 0; j < TR::VEC; ++j)
                        if (key[i][j] > best) { best = key[i][j]; at = (i * L + l) * TR::VEC + j; }
                const unsigned all = lanes_max(best, L);
                at = (int)lanes_min(best == all ? (unsigned)at : 0x7fffffffu, L);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < TR::VEC; ++j)
                        if ((i * L + l) * TR::VEC + j == at) key[i][j] = 0u;
                if (l == 0) mine[n] = (unsigned)at;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        // the wave's rows, from w0 on: their outputs are neighbours.  (o + 1/2) / k is at least 1/(2k) away from a whole number and
        // off by less than 64 * 256 / k * 2^-22
        typedef typename TR::elem E;
        const int64_t w0 = r0 + wave * (64 / L);
        const int outs = (int)max((int64_t)0, min((int64_t)(64 / L), p.rows - w0)) * p.k;
        const char* xw = p.x + w0 * p.xp;
        E* val = reinterpret_cast<E*>(p.val) + w0 * p.k;
        int* idx = p.idx + w0 * p.k;
        for (int o = lane; o < outs; o += 64) {
            const unsigned f = waves[o];
            const int cls = (int)(f & 0xffffu);
            auto value = [&] { return reinterpret_cast<const E*>(xw + (int)(((float)o + 0.5f) * inv) * p.xp)[cls]; };
            if constexpr (TR::ESZ == 2) {
                const unsigned key = f >> 16;
                E v = (E)(key & 0x8000u ? key ^ 0x8000u : ~key);
                if (key == 0x8000u || key == 0xffffu) v = value();         // the value itself: a NaN keeps its bits, -0 its sign
                val[o] = v;
            } else {
                val[o] = value();
            }
            idx[o] = cls;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- a wave per row -----------------------------------------------------------------------------------------------------
// 20000 rows of 1000 fp32 classes, 16 of them: 28 us (2.9 TB/s); 50000 x 512 bf16, 16: 29 us (1.9 TB/s): bounded by instructions, the
// search among the lanes' maxima and the gathering.
// exclusive prefix sum over the lanes; all: the sum
__device__ __forceinline__ int lanes_before(int v, int& all) {
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(s, o, 64);
        s += (int)(threadIdx.x & 63) >= o ? u : 0;
    }
    all = __shfl(s, 63, 64);
    return s - v;
}
// how many of n full keys in LDS lie above f: eight reads on their way at a time (30000 x 4000 bf16, 64 of them: 131 -> 100 us)
__device__ __forceinline__ int above(const u64* list, int n, u64 f) {
    int place = 0, c = 0;
    for (; c + 8 <= n; c += 8) {
        ulonglong2 y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = *reinterpret_cast<const ulonglong2*>(list + c + 2 * u);
#pragma unroll
        for (int u = 0; u < 4; ++u) place += (y[u].x > f ? 1 : 0) + (y[u].y > f ? 1 : 0);
    }
    for (; c < n; ++c) place += list[c] > f ? 1 : 0;
    return place;
}
// the k largest of n full keys in LDS to their places, by one wave
template <class TR>
__device__ __forceinline__ void place_all(const TopParams& p, int64_t r, int l, const u64* mine, int n) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    for (int a = l; a < n; a += 64) {
        const u64 f = mine[a];
        const int place = above(mine, n, f);
        if (place < p.k) emit<TR>(p, r, place, (int)~(unsigned)f);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}

template <class TR, int NV>
__global__ __launch_bounds__(TPB) void top_wave(TopParams p) {
    __shared__ alignas(16) u64 list[TPB / 64][MAX_K];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    u64* mine = list[w];
    for (int64_t r = (int64_t)blockIdx.x * (TPB / 64) + w; r < p.rows; r += (int64_t)gridDim.x * (TPB / 64)) {
        const char* x = p.x + r * p.xp;
        unsigned key[NV][TR::VEC];
        load_keys<TR, NV>(x, p.v, 64, l, key);
        if (p.by_lanes) {
            // at least k classes lie at or above the k-th largest of the lanes' maxima: on average 44 for k = 32
            unsigned best = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) best = max(best, key[i][j]);
            unsigned t = 0;
#pragma unroll 1
            for (int bit = 31; bit >= 32 - 8 * TR::ESZ; --bit) {
                const unsigned want = t | (1u << bit);
                if (__popcll(__ballot(best >= want)) >= p.k) t = want;
            }
            int n = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) {
                    const bool f = key[i][j] >= t && key[i][j];
                    const u64 ball = __ballot(f);
                    const int at = n + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(ball >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)ball, 0));
                    if (f && at < MAX_K) mine[at] = full_key(key[i][j], (i * 64 + l) * TR::VEC + j);
                    n += __popcll(ball);
                }
            if (n <= MAX_K) {                                      // the same for the whole wave
                place_all<TR>(p, r, l, mine, n);
                continue;
            }
        }
        unsigned t = 0;                                            // the largest number that k keys reach
#pragma unroll 1
        for (int bit = 31; bit >= 32 - 8 * TR::ESZ; --bit) {       // the lower half of a bf16 key follows from its sign
            const unsigned want = t | (1u << bit);
            int n = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) n += __popcll(__ballot(key[i][j] >= want));
            if (n >= p.k) t = want;
        }
        // above: keys whose compared bits exceed t; equal: the first ones by class fill the list
        const unsigned mask = TR::ESZ == 2 ? 0xffff0000u : 0xffffffffu;
        int above = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) above += __popcll(__ballot((key[i][j] & mask) > t));
        int na = 0, ne = above;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            int ca = 0, ce = 0;
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) {
                ca += (key[i][j] & mask) > t ? 1 : 0;
                ce += key[i][j] && (key[i][j] & mask) == t ? 1 : 0;
            }
            int all;
            const int before = lanes_before(ca | ce << 16, all);
            int pa = na + (before & 0xffff), pe = ne + (before >> 16);
            na += all & 0xffff; ne += all >> 16;
#pragma unroll
            for (int j = 0; j < TR::VEC; ++j) {
                const unsigned kk = key[i][j] & mask;
                const int cls = (i * 64 + l) * TR::VEC + j;
                if (kk > t) mine[pa++] = full_key(kk, cls);
                else if (key[i][j] && kk == t) { if (pe < p.k) mine[pe] = full_key(kk, cls); ++pe; }
            }
        }
        place_all<TR>(p, r, l, mine, p.k);
    }
}

// ---- a workgroup per row ------------------------------------------------------------------------------------------------
// Bound by the read where the lists are short against the row: 2048 x 50001 bf16, 32 of them 48 us, 4.3 TB/s; 15000 x 8000 fp32, 8 of them
// 86 us, 5.6 TB/s.  200 of 50001: 76 us, half of it for the threads' parts read again and the placing.
// Largest key of 16-byte vectors without making the keys: the bits of a value, with the lower ones turned over if it is
// negative, order as signed numbers, two bf16 at a time, except that NaN with a sign lies below -inf; the smallest such number
// tells whether there is one.  2.5 (bf16) and 5 (fp32) instructions per class instead of 9.
typedef short s2 __attribute__((ext_vector_type(2)));
template <class TR> struct BestOf;
template <> struct BestOf<BF16> {
    s2 hi = {-32768, -32768}, lo = {32767, 32767};
    __device__ __forceinline__ void word(unsigned w) {
        s2 v = __builtin_bit_cast(s2, w);
        v ^= (v >> 15) & (short)0x7fff;
        hi = __builtin_elementwise_max(hi, v);
        lo = __builtin_elementwise_min(lo, v);
    }
    __device__ __forceinline__ unsigned key() const {
        short h = hi.x > hi.y ? hi.x : hi.y;
        const short l = lo.x < lo.y ? lo.x : lo.y;
        if (l < (short)0x807f) return 0xffffffffu;                 // below -inf
        if (h == -32768) return 0;                                 // nothing seen
        h ^= (h >> 15) & 0x7fff;
        return key_of(bf16_to_f32((unsigned short)h));
    }
};
template <> struct BestOf<F32> {
    int hi = (int)0x80000000, lo = 0x7fffffff;
    __device__ __forceinline__ void word(unsigned w) {
        const int v = (int)w ^ (((int)w >> 31) & 0x7fffffff);
        hi = max(hi, v); lo = min(lo, v);
    }
    __device__ __forceinline__ unsigned key() const {
        if (lo < (int)0x807fffff) return 0xffffffffu;
        if (hi == (int)0x80000000) return 0;
        return key_of(__uint_as_float((unsigned)(hi ^ ((hi >> 31) & 0x7fffffff))));
    }
};
template <class TR>
__device__ __forceinline__ void best_vec(BestOf<TR>& b, const uint4& v) { b.word(v.x); b.word(v.y); b.word(v.z); b.word(v.w); }

// the largest number that k of N * 64 keys reach, by one wave (0: fewer than k are there)
template <class TR, int N>
__device__ __forceinline__ unsigned reach(const unsigned* top, int k) {
    unsigned key[N], t = 0;
#pragma unroll
    for (int w = 0; w < N; ++w) key[w] = top[w * 64 + (threadIdx.x & 63)];
#pragma unroll 1
    for (int bit = 31; bit >= 32 - 8 * TR::ESZ; --bit) {           // the lower half of a bf16 key follows from its sign
        const unsigned want = t | (1u << bit);
        int n = 0;
#pragma unroll
        for (int w = 0; w < N; ++w) n += __popcll(__ballot(key[w] >= want));
        if (n >= k) t = want;
    }
    return t;
}

// f(key, class) for the classes of a row, T threads side by side
template <class TR, int T, class F>
__device__ __forceinline__ void each(const char* x, int v, F f) {
    const int nv = v / TR::VEC;
    for (int i = threadIdx.x; i < nv; i += T) {
        float y[TR::VEC];
        unpack_vec<TR>(ld_any<TR>(x + (int64_t)i * 16), y);
#pragma unroll
        for (int j = 0; j < TR::VEC; ++j) f(key_of(y[j]), i * TR::VEC + j);
    }
    for (int i = nv * TR::VEC + threadIdx.x; i < v; i += T) f(key_of(ld_one<TR>(x, i)), i);
}

template <int T>
__device__ __forceinline__ int block_count(int c, int* sm) {
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < T / 64; ++w) c += sm[w];
    return c;
}

// Exactly the k classes of a row with too many classes at or above key t: the k-th largest key by halving, the classes above
// it in any order, and as many at it as are missing, by ascending class, T classes at a time until there are enough.
template <class TR, int T, bool ODD>                               // one for every caller: a shared one costs all of them 26 registers
__device__ __noinline__ void gather_ties(const char* x, int v, int k, unsigned t, u64* cand, int* count, int* sm) {
    unsigned hi = 0xffffffffu;                                     // k classes reach t
    bool first = true;                                             // with many equal values t mostly is the key already
    while (t < hi) {
        const unsigned mid = first ? t + 1 : t + (hi - t) / 2 + ((hi - t) & 1);
        first = false;
        int c = 0;
        each<TR, T>(x, v, [&](unsigned key, int) { c += key >= mid ? 1 : 0; });
        if (block_count<T>(c, sm) >= k) t = mid;
        else hi = mid - 1;
    }
    __syncthreads();
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
    each<TR, T>(x, v, [&](unsigned key, int i) { if (key > t) cand[atomicAdd(count, 1)] = full_key(key, i); });
    __syncthreads();
    int n = *count;                                                // fewer than k
    for (int i0 = 0; n < k && i0 < v; i0 += T) {
        const int i = i0 + threadIdx.x;
        const bool f = i < v && key_of(ld_one<TR>(x, i)) == t;
        const u64 ball = __ballot(f);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = __popcll(ball);
        __syncthreads();
        int at = n + __popcll(ball & ((1ull << (threadIdx.x & 63)) - 1));
        for (int w = 0; w < T / 64; ++w) {
            if (w < (int)threadIdx.x >> 6) at += sm[w];
            n += sm[w];
        }
        if (f && at < k) cand[at] = full_key(t, i);
    }
    __syncthreads();
}

template <class TR, int T, bool ODD>
__global__ __launch_bounds__(T) void top_long(TopParams p) {
    constexpr int CAP = T <= 512 ? 4 * T : 2048;                   // classes gathered, 12 times the usual number
    __shared__ alignas(16) u64 cand[CAP];
    __shared__ unsigned top[T], thr_s;
    __shared__ unsigned short hot[T];
    __shared__ int count_s, hot_s, sm[T / 64];
    const int tid = threadIdx.x;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const char* x = p.x + r * p.xp;
        // Vectors begin at a word: in between, a load takes longer (2048 rows of 50001 bf16 classes 58 us, of 50002 48).  The class in front
        // and those behind the last vector, fewer than a vector's worth, belong to a thread each.  ODD: some rows begin between words (where none
        // does, the head costs 4 %: 4000 x 32000, 32 of them 58 -> 61).
        const int head = ODD ? (int)((uintptr_t)x >> 1) & 1 : 0, nv = (p.v - head) / TR::VEC, per = (nv + T - 1) / T;
        const int et = head && tid == T - 1 ? 0 : head + nv * TR::VEC + tid;
        const char* xv = x + head * TR::ESZ;
        constexpr int UN = 8;                                      // vectors in flight per thread; few at the end cost most (8000 x 16000: 88 -> 71 us)
        BestOf<TR> b;
        int i = tid;
        auto batch = [&](auto nu) {
            constexpr int N = decltype(nu)::value;
            uint4 raw[N];
#pragma unroll
            for (int u = 0; u < N; ++u) raw[u] = ld_any<TR>(xv + (int64_t)(i + u * T) * 16);
#pragma unroll
            for (int u = 0; u < N; ++u) best_vec(b, raw[u]);
            i += N * T;
        };
        while (i + (UN - 1) * T < nv) batch(std::integral_constant<int, UN>{});
        if (i + 4 * T < nv) {                                      // 5 to 7 more: all at once, the last vector standing in for those behind the end
            uint4 raw[UN - 1];
#pragma unroll
            for (int u = 0; u < UN - 1; ++u) raw[u] = ld_any<TR>(xv + (int64_t)min(i + u * T, nv - 1) * 16);
#pragma unroll
            for (int u = 0; u < UN - 1; ++u)
                if (i + u * T < nv) best_vec(b, raw[u]);
        } else if (i + 3 * T < nv) {
            batch(std::integral_constant<int, 4>{});
        } else {
            if (i + T < nv) batch(std::integral_constant<int, 2>{});
            if (i < nv) batch(std::integral_constant<int, 1>{});
        }
        const unsigned tail = et < p.v ? key_of(ld_one<TR>(x, et)) : 0u;
        const unsigned best = max(b.key(), tail);
        // G maxima of T / G neighbouring threads each
        const unsigned group = lanes_max(best, T / p.G);
        if (tid % (T / p.G) == 0) top[tid / (T / p.G)] = group;
        if (tid == 0) count_s = hot_s = 0;
        __syncthreads();
        if (tid < 64) {
            const unsigned t = p.G == 64 ? reach<TR, 1>(top, p.k) : p.G == 128 ? reach<TR, 2>(top, p.k) : p.G == 256 ? reach<TR, 4>(top, p.k) : reach<TR, 8>(top, p.k);
            if (tid == 0) thr_s = t;
        }
        __syncthreads();
        const unsigned t = thr_s;
        auto add = [&](unsigned key, int cls) {
            if (key >= t) {
                const int at = atomicAdd(&count_s, 1);
                if (at < CAP) cand[at] = full_key(key, cls);
            }
        };
        if (best >= t && best) hot[atomicAdd(&hot_s, 1)] = (unsigned short)tid;
        if (tail) add(tail, et);
        __syncthreads();
        const int items = hot_s * per;
        for (int m = tid; m < items; m += T) {
            const int at = (m % per) * T + hot[m / per];
            if (at < nv) {
                float y[TR::VEC];
                unpack_vec<TR>(ld_any<TR>(xv + (int64_t)at * 16), y);
#pragma unroll
                for (int j = 0; j < TR::VEC; ++j) add(key_of(y[j]), head + at * TR::VEC + j);
            }
        }
        __syncthreads();
        int n = count_s;
        if (n > CAP) {
            gather_ties<TR, T, ODD>(x, p.v, p.k, t, cand, &count_s, sm);
            n = p.k;
        }
        for (int a = tid; a < n; a += T) {
            const u64 f = cand[a];
            const int place = above(cand, n, f);
            if (place < p.k) emit<TR>(p, r, place, (int)~(unsigned)f);
        }
        __syncthreads();
    }
}

enum { SHORT, SORTED, WAVE, LONG };
struct Plan { int kind, L, nv, T, G, blocks, by_lanes; };
Plan plan_of(int esz, int64_t rows, int v, int k) {
    Plan q = {SHORT, 1, 1, TPB, 0, 0, 0};
    const int vec = 16 / esz, nvec = (v + vec - 1) / vec;
    int64_t per = 1;
    // From 129 vectors on, lists that a wave would search out bit by bit (and all bf16 lists up to 85) go by workgroups of 128: 20000 rows of 2000
    // bf16 classes, 64 of them: 90 -> 51 us, 8 of them 39 -> 35; of 1000 fp32 classes, 64: 65 -> 45, but 16: 28 -> 34.
    const bool small_groups = nvec > 128 && nvec <= 64 * NVMAX && k <= 85 && (esz == 2 || k > 32);
    if (nvec <= 64 * NVMAX && !small_groups) {
        while (q.L < 64 && nvec > q.L * NVMAX) q.L *= 2;
        // instructions of a wave per row: k times 3 (bf16) or 6 (fp32) per held class and 10 per exchange between
        // lanes (networks: 44 or 70 per vector, 50 or 110 per exchange; sorted: a fixed part, the merges within and between lanes), for
        // 64 / L rows at once, against 4 per bit and 12 per held class (k <= 32, by the lanes' maxima) or 3 per held class and bit, and the placing.
        // 50000 rows of 512 bf16 classes, 16 of them: 50 us by search alone, 29 with the lanes' maxima; 100000 x 133 fp32, 5: 28 taken out
        const int n1 = (nvec + q.L - 1) / q.L, n2 = (nvec + 63) / 64;
        const int e1 = n1 * vec, e2 = n2 * vec;
        int lg = 0;
        while ((1 << lg) < q.L) ++lg;
        q.by_lanes = k <= 32 && 2 * nvec >= 3 * k;                 // enough lanes hold something
        const int nets = esz == 2 && k <= 8 ? k <= 4 ? n1 * 44 + lg * 50 : n1 * 70 + lg * 110 : 0;
        const int64_t take = ((nets ? nets : (int64_t)k * ((esz == 2 ? 3 : 6) * e1 + 10 * lg + 8)) + 8 * e1) * q.L / 64, search = q.by_lanes ? 8 * esz * 4 + 12 * e2 + 6 * k + 100 : 8 * esz * 3 * e2 + 100 + (int64_t)k * ((k + 63) / 64) * 4;
        q.kind = take <= search && k <= 32 ? SHORT : WAVE;             // 32: 32 KB of LDS
        if (k > (esz == 2 ? 8 : 4) && nvec <= 64) {
            int s = 1, ls = 0;
            while (s < nvec) s *= 2, ++ls;
            const int sort = (200 + (esz == 2 ? 24 : 12) * ls + (esz == 2 ? 9 : 13) * ls * (ls + 1)) * s / 64;
            if (sort < (q.kind == SHORT ? take : search)) { q.kind = SORTED; q.L = s; }
        }
        if (q.kind == WAVE) q.L = 64;
        q.nv = (nvec + q.L - 1) / q.L;
        per = TPB / q.L;
    } else {
        // Few rows: up to 1024 threads each, one vector at least (else groups without any would leave fewer than k maxima).  Else about
        // eight vectors a thread, all on their way at once, as many rows as possible beside each other: us with 128 / 256 / 512 / 1024 threads
        // 30000 x 4000 bf16, 8 of them: 63 / 93 / - / -, 15000 x 8000: 49 / 64 / 97 / -, 8000 x 16000, 32: 78 / 64 / 79 / 176,
        // 4000 x 32000: 80 / 68 / 58 / 109, 2048 x 50001: 76 / 63 / 58 / 82 (49 since its vectors begin at words), 1000 x 131072: 86 / 74 / 64 / 59.
        // G maxima, at least 1.5 per entry: the classes gathered are then few (G log(G / (G - k)) of them on average: 44 for k = 32, 355 for 256)
        q.kind = LONG;
        q.T = small_groups ? 128 : rows < 512 ? (nvec >= 1024 ? 1024 : nvec >= 512 || k > 170 ? 512 : 256) : nvec <= 1280 && k <= 85 ? 128 : nvec <= 2560 && k <= 170 ? 256 : nvec <= 12288 ? 512 : 1024;
        q.G = 64;
        while (q.G < q.T && q.G < k + k / 2) q.G *= 2;
    }
    const int64_t b = (rows + per - 1) / per;
    q.blocks = (int)(b < 16384 ? b : 16384);
    return q;
}

#define SHORT_NV(T, K)                                                                            \
    do {                                                                                       \
        const size_t lds = TPB / q.L * k * 4;                                                    \
        if (q.nv == 1) top_short<T, 1, K><<<q.blocks, TPB, lds, st>>>(p);                        \
        else if (q.nv == 2) top_short<T, 2, K><<<q.blocks, TPB, lds, st>>>(p);                   \
        else if (q.nv == 3) top_short<T, 3, K><<<q.blocks, TPB, lds, st>>>(p);                   \
        else top_short<T, 4, K><<<q.blocks, TPB, lds, st>>>(p);                                  \
    } while (0)
#define LONG_T(TR, ODD)                                                                           \
    do {                                                                                       \
        if (q.T == 128) top_long<TR, 128, ODD><<<q.blocks, 128, 0, st>>>(p);                     \
        else if (q.T == 256) top_long<TR, 256, ODD><<<q.blocks, 256, 0, st>>>(p);                \
        else if (q.T == 512) top_long<TR, 512, ODD><<<q.blocks, 512, 0, st>>>(p);                \
        else top_long<TR, 1024, ODD><<<q.blocks, 1024, 0, st>>>(p);                              \
    } while (0)
#define NV_LAUNCH(KERN, lds)                                                                      \
    do {                                                                                       \
        if (dtype == 1) {                                                                      \
            if (q.nv == 1) KERN<BF16, 1><<<q.blocks, TPB, lds, st>>>(p);                         \
            else if (q.nv == 2) KERN<BF16, 2><<<q.blocks, TPB, lds, st>>>(p);                    \
            else if (q.nv == 3) KERN<BF16, 3><<<q.blocks, TPB, lds, st>>>(p);                    \
            else KERN<BF16, 4><<<q.blocks, TPB, lds, st>>>(p);                                   \
        } else {                                                                               \
            if (q.nv == 1) KERN<F32, 1><<<q.blocks, TPB, lds, st>>>(p);                          \
            else if (q.nv == 2) KERN<F32, 2><<<q.blocks, TPB, lds, st>>>(p);                     \
            else if (q.nv == 3) KERN<F32, 3><<<q.blocks, TPB, lds, st>>>(p);                     \
            else KERN<F32, 4><<<q.blocks, TPB, lds, st>>>(p);                                    \
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
    p.rows = rows; p.xp = pitch * (int64_t)esz; p.v = v; p.k = k; p.L = q.L; p.G = q.G; p.by_lanes = q.by_lanes;
    hipStream_t st = (hipStream_t)stream;
    if (q.kind == SORTED) {
        if (dtype == 1) top_short<BF16, 1, SORT><<<q.blocks, TPB, TPB / q.L * k * 4, st>>>(p);
        else top_short<F32, 1, SORT><<<q.blocks, TPB, TPB / q.L * k * 4, st>>>(p);
    } else if (q.kind == SHORT) {
        if (dtype == 0) SHORT_NV(F32, 0);
        else if (k == 1) SHORT_NV(BF16, 1);
        else if (k <= 4) SHORT_NV(BF16, 4);
        else if (k <= 8) SHORT_NV(BF16, 8);
        else SHORT_NV(BF16, 0);
    } else if (q.kind == WAVE) {
        NV_LAUNCH(top_wave, 0);
    } else {
        const bool odd = esz == 2 && (pitch % 2 != 0 || (uintptr_t)logits % 4 != 0);
        if (dtype == 0) LONG_T(F32, false);
        else if (odd) LONG_T(BF16, true);
        else LONG_T(BF16, false);
    }
    MI_HIP(hipGetLastError());
    return 0;
}
