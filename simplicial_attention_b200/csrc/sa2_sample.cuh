// A token for each row of logits: temperature, top-k, top-p, min-p, and one given number of [0, 1) a row.
//
// Order of the tokens: larger logit first, of equal ones the lower index.  What the filters keep is the beginning of that order:
//   top-k: the first k;  top-p: of those, the ones before which less than top_p of their mass has come;  min-p: the ones
//   whose probability is at least min_p times the best one's.  The best token stays in any case.
// The token is the first, by index, at which the running mass of what is kept exceeds u times the whole; its log-probability is the one
// among what is kept.
//
// Masses are whole numbers: exp((z - max) / T) in 64-bit floating point, times 2^S and rounded, S so that a row's sum stays below
// 2^63.  Sums of them are exact in any order, so the result does not depend on how threads, warps and CTAs share a row, and
// counters in shared memory may be atomic.  A weight is off by at most 2^-(S+1) of the best token's: a token would change for a share
// of about 2^-46 vocab of the numbers u.
//
// A cluster of CTAs has a row, a warp of it consecutive indices; a slice that fits into shared memory is read from global memory once.
// (1) The maximum.  (2) A histogram of counts over 512 stretches of 24 max(T, 1) below the maximum brackets the cut: for top-k by its
// counts, for top-p by the least and the largest mass that they can have; min-p says itself how far down it goes.  A warp lists its logits
// down to there, in their order, or goes on with all of them where they are many.  (3) If at most 512 are listed, every CTA sorts all of them and
// adds up the masses before each.  Otherwise what is in the bracket is cut again first, on the bits of the logits mapped to integers in
// their order, with exact masses, 512 stretches at a time.  (4) Warps add the kept masses, and the one that has the drawn mass walks its list.
// Bound: reading the logits once, of which few calls come near: one row of 256 12 us and 64 rows of 32000 21 us (chains of waits), 256 rows of
// 128000 fp32 logits 110 to 175 us and 410 to 470 where the cut lies among many (a floor of 20: the second reading from L2 and HBM, the masses'
// 64-bit arithmetic, and the second row of an SM's two CTAs where 256 rows are no multiple of the places); 16384 rows of 256 logits 182 us (a floor
// of 3: a CTA, its tables and about ten waits for so short a row).
#pragma once
#include "sa2_common.cuh"
#include "sa2_sample_keys.h"
#include <cooperative_groups.h>
#include <math_constants.h>

namespace sa2 {
namespace sample {

constexpr int LIST = 256;                               // logits that a warp lists
constexpr int MAX_CTAS = 8;
constexpr int LOG_TABLE = 5, TABLE = 1 << LOG_TABLE, COPIES = 16;       // of a table entry: a lane and its neighbours read different banks
constexpr int SPLIT = 4;                                // of a counter of the coarse histogram

// N: threads of a CTA, stretches of a histogram (one a thread), logits that are sorted at once
template <int N> constexpr int WARPS = N / 32;
template <int N> constexpr int LOG_BINS = N == 512 ? 9 : 7;

struct Params {
    const void *z;              // [rows][vocab], row stride zs
    const void *uniform;        // [rows], fp32 or fp64
    const float *temperature, *top_p, *min_p;       // [rows], or null: the values below
    const int64_t *top_k;
    int64_t *token;             // [rows]
    float *logprob;             // [rows], may be null
    int64_t rows, zs;
    int64_t top_k_all;
    double temperature_all, top_p_all, min_p_all;
    int vocab, uniform64;
    int slice;                  // logits of a CTA, a multiple of 128
    int shift;                  // S above
};

struct Cut {                    // of the order of the tokens, behind a token of the key `key`
    uint32_t key;
    uint32_t ties;              // tokens of that key that are kept, the lowest indices
    uint32_t equal;             // ... that there are
    unsigned long long mass;    // of what is kept
};

template <int N> struct alignas(16) Shared {             // the slice, or the ring, stands behind it
    double table[TABLE][COPIES];                        // 2^(j / 32)
    uint32_t coarse[N][SPLIT], total[N];          // counts below the maximum: of this CTA, of the cluster
    uint32_t count[N], lo[N], hi[N];           // counts and masses in the bracket
    uint32_t keys[N], all[N], sorted[N];
    unsigned long long warp_mass[WARPS<N>], mass_of[2][MAX_CTAS], above_mass[MAX_CTAS], mass_above, mass_in;
    double warp_low[WARPS<N>], warp_high[WARPS<N>];
    uint32_t warp_count[WARPS<N>], ties_of[MAX_CTAS], above_count[MAX_CTAS], count_above, count_in, bin, other, taken;
    float max_of[MAX_CTAS];
    int first_bin, last_bin;
    uint16_t list[WARPS<N>][LIST];
};
static_assert(sizeof(Shared<512>) % 16 == 0 && sizeof(Shared<128>) % 16 == 0, "16-byte pieces of the slice");
constexpr int RING = 8;                                 // quads of a lane on their way from global memory

// Larger logits have larger keys; -0 and 0 the same one.
template <typename T> __device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t u = __float_as_uint(z + 0.f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return sizeof(T) == 2 ? k >> 16 : k;
}
// the smallest key of a logit that is at least z
template <typename T> __device__ __forceinline__ uint32_t key_from_of(float z) {
    if (sizeof(T) == 4) return key_of<T>(z);
    const uint32_t k = key_of<float>(z);                 // (keys of bf16 end in zeros if positive, in ones if negative)
    return (k & 0x80000000u ? k + 0xffffu : k) >> 16;
}
// the logit of a key
template <typename T> __device__ __forceinline__ float logit_of(uint32_t key) {
    if (sizeof(T) == 2) key = key << 16 | (key & 0x8000u ? 0u : 0xffffu);
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// What a warp goes through, in the order of the indices: a list of places in the slice, or all of its part.
struct View {
    const uint16_t *list;       // from `first` on; or null
    int first, count;
    __device__ __forceinline__ int place(int x) const { return first + (list ? list[x] : x); }
};

// RESIDENT: the slice is in shared memory
template <typename T, bool RESIDENT> struct Row {
    const T *z;                 // this CTA's slice
    T *ring;                    // this warp's
    const double *table;        // this lane's copy
    float best, scale, least;   // the mass of a logit that times `scale` is `least` is 0, and so is that of all logits below it
    double top;                 // best * scale
    double inv_t, steps;        // 1 / T, 32 log2(e) / (scale T)
    int shift;                  // S
    bool quads;                 // four logits at a multiple of four can be loaded at once

    __device__ __forceinline__ double exponent(float v) const { return ((double)v - (double)best) * inv_t; }
    // 2^S exp((v - best) / T), rounded.  2^(k / 32 + r / 32): k >> 5 goes into the exponent, 2^((k & 31) / 32) comes from the table, and
    // for the rest, at most 1 / 64, Taylor's polynomial of degree five is good to 2^-48.  (A table of 128 entries and one copy, with degree
    // four, spent its time on bank conflicts.)
    __device__ __forceinline__ unsigned long long mass(float v) const {
        constexpr double MAGIC = 6755399441055744.;      // 1.5 2^52: the sum's low word is the nearest whole number
        constexpr double L = 0.6931471805599453 / TABLE;
        const double d = (double)fmaxf(v * scale, least) - top, t = fma(d, steps, MAGIC);
        const int k = __double2loint(t);
        const double r = fma(d, steps, -(t - MAGIC));
        double p = fma(r, L * L * L * L * L / 120., L * L * L * L / 24.);
        p = fma(r, p, L * L * L / 6.);
        p = fma(r, p, L * L / 2.);
        p = fma(r, p, L);
        p = fma(r, p, 1.) * table[(k & (TABLE - 1)) * COPIES];
        p = __hiloint2double(__double2hiint(p) + (((k >> LOG_TABLE) + shift) << 20), __double2loint(p));
        // 2^52 more: the low bits are the rounded number (S is at most 51).  No branch and no selection: four of these run side by side
        return (unsigned long long)__double_as_longlong(p + 4503599627370496.) - 0x4330000000000000ull;
    }
    static __device__ __forceinline__ void four(const T *p, float (&v)[4]) {
        if constexpr (sizeof(T) == 4) {
            const float4 t = *reinterpret_cast<const float4 *>(p);
            v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        } else {
            const uint2 t = *reinterpret_cast<const uint2 *>(p);
            v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
            v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
        }
    }
    // logits x0 ... x0 + 3 of a view (x0 a multiple of four), -inf behind its end
    __device__ __forceinline__ void quad(const View &V, int x0, float (&v)[4]) const {
        if (!V.list && (RESIDENT || quads) && x0 + 4 <= V.count) {
            four(z + V.first + x0, v);
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x0 + j < V.count ? (float)z[V.place(x0 + j)] : -CUDART_INF_F;
    }
};

// Calls f(x, logits x ... x + 3) for a warp's view, lane by lane.  A row that is not in shared memory comes from L2 or HBM, 1000 to 2000 cycles
// away: RING quads of a lane are on their way, to shared memory of its own.  (Two or four in registers left the SM waiting for most of a
// pass.)  All lanes make all calls: x may lie behind the end.
template <typename T, bool RESIDENT, typename F> __device__ __forceinline__ void for_quads(const Row<T, RESIDENT> &R, const View &V, F f) {
    const int lane = threadIdx.x & 31;
    if constexpr (!RESIDENT) {
        if (!V.list && R.quads) {
            const T *src = R.z + V.first + lane * 4;
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(R.ring + lane * 4);
            auto fetch = [&](int x0, int slot) {
                if (x0 + lane * 4 + 4 <= V.count) {
                    if constexpr (sizeof(T) == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + slot * 512), "l"(src + x0) : "memory");
                    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + slot * 256), "l"(src + x0) : "memory");
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            for (int i = 0; i < RING; ++i) fetch(i * 128, i);
            int slot = 0;
            for (int x0 = 0; x0 < V.count; x0 += 128) {
                asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
                float v[4];
                const int x = x0 + lane * 4;
                if (x + 4 <= V.count) R.four(R.ring + slot * 128 + lane * 4, v);
                else R.quad(V, x, v);
                f(x, v);
                fetch(x0 + RING * 128, slot);            // (the slot's values are in registers)
                slot = slot + 1 == RING ? 0 : slot + 1;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            return;
        }
    }
    for (int x0 = 0; x0 < V.count; x0 += 128) {
        float v[4];
        R.quad(V, x0 + lane * 4, v);
        f(x0 + lane * 4, v);
    }
}

// 64-bit counter of two words; a carry of the lower one is seen by the addition that makes it
__device__ __forceinline__ void add_mass(uint32_t *lo, uint32_t *hi, unsigned long long w) {
    const uint32_t l = (uint32_t)w;
    uint32_t h = (uint32_t)(w >> 32);
    if (l) h += atomicAdd(lo, l) + l < l ? 1u : 0u;
    if (h) atomicAdd(hi, h);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// sum over this lane and the ones before it
template <typename V> __device__ __forceinline__ V warp_upto(V v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}
// all threads of the row's CTAs
__device__ __forceinline__ void row_sync(int ctas) {
    if (ctas > 1) cooperative_groups::this_cluster().sync();
    else __syncthreads();
}
template <int N> __device__ __forceinline__ Shared<N> &of_cta(Shared<N> &S, int ctas, int r) {
    return ctas > 1 ? *cooperative_groups::this_cluster().map_shared_rank(&S, r) : S;
}

// The keys of [from, to] in the views of all CTAs into S.sorted, largest first.  How many there are; -1 if more than N.
template <typename T, bool RESIDENT, int N> __device__ int gather(const Row<T, RESIDENT> &R, const View &V, Shared<N> &S, int ctas, uint32_t from, uint32_t to) {
    const int t = threadIdx.x;
    if (t == 0) S.taken = 0u;
    __syncthreads();
    for_quads(R, V, [&](int x, float (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t k = key_of<T>(v[j]);
            if (x + j < V.count && k >= from && k <= to) {
                const uint32_t at = atomicAdd(&S.taken, 1u);
                if (at < N) S.keys[at] = k;
            }
        }
    });
    row_sync(ctas);
    int own[MAX_CTAS], n = 0, from_cta = 0, at = 0;
#pragma unroll
    for (int r = 0; r < MAX_CTAS; ++r) own[r] = r < ctas ? (int)of_cta(S, ctas, r).taken : 0;
#pragma unroll
    for (int r = 0; r < MAX_CTAS; ++r) {
        if (t >= n && t < n + own[r]) {
            from_cta = r;
            at = t - n;
        }
        n += own[r];
    }
    if (n > N) {
        row_sync(ctas);
        return -1;
    }
    const uint32_t key = t < n ? of_cta(S, ctas, from_cta).keys[at] : 0u;
    S.all[t] = key;                                      // (0 behind the end: no logit has it)
    row_sync(ctas);                                      // nobody reads another CTA's keys any more
    // a key's place: the keys that are larger, and the equal ones in front of it
    if (t < n) {
        int place = 0;
        for (int x = 0; x < n; x += 4) {
            const uint4 o = *reinterpret_cast<const uint4 *>(S.all + x);
            place += (o.x > key || (o.x == key && x < t)) + (o.y > key || (o.y == key && x + 1 < t)) + (o.z > key || (o.z == key && x + 2 < t)) +
                     (o.w > key || (o.w == key && x + 3 < t));
        }
        S.sorted[place] = key;
    }
    __syncthreads();
    return n;
}

// Adds to cb and mb the counts and masses of the threads before this one.
template <int N> __device__ __forceinline__ void sums_before(Shared<N> &S, uint32_t c, unsigned long long m, uint32_t &cb, unsigned long long &mb) {
    const int warp = threadIdx.x >> 5;
    const uint32_t cw = warp_upto(c);
    const unsigned long long mw = warp_upto(m);
    __syncthreads();
    if ((threadIdx.x & 31) == 31) { S.warp_count[warp] = cw; S.warp_mass[warp] = mw; }
    __syncthreads();
    cb += cw - c;
    mb += mw - m;
    for (int w = 0; w < warp; ++w) { cb += S.warp_count[w]; mb += S.warp_mass[w]; }
}

__device__ __forceinline__ unsigned long long wanted_mass(double top_p, unsigned long long all) {
    const double part = ceil(top_p * (double)all);
    const unsigned long long want = part >= 1. ? (unsigned long long)part : 1ull;
    return want < all ? want : all;
}
__device__ __forceinline__ Cut no_cut(unsigned long long mass) { return Cut{0u, 0xffffffffu, 0u, mass}; }

// Both cuts among at most N logits, all from the key `from` on: behind top_k (0: not) and, of what stays, top_p (1: not) of the mass.
// The row's mass, which counts where top_k is 0, lies between `least` and `most`; `sure`: the cut is the same for both.  A cut that lies further
// down than `from` is none.
template <typename T, bool RESIDENT, int N>
__device__ Cut cut_few(const Row<T, RESIDENT> &R, const View &V, Shared<N> &S, int ctas, uint32_t from, int64_t top_k, double top_p, unsigned long long least,
                       unsigned long long most, bool &sure) {
    const int t = threadIdx.x, n = gather(R, V, S, ctas, from, 0xffffffffu);
    sure = n >= 0;
    if (!sure) return no_cut(0ull);
    const uint32_t key = t < n ? S.sorted[t] : 0u;
    int last = top_k > 0 && top_k <= n ? (int)top_k - 1 : -1;            // the last token that stays
    if (top_p < 1.) {
        const unsigned long long m = t < n ? R.mass(logit_of<T>(key)) : 0ull;
        uint32_t cb = 0u;
        unsigned long long mb = 0ull;
        sums_before(S, 0u, m, cb, mb);
        if (t == 0) { S.bin = 0xffffffffu; S.other = 0xffffffffu; }
        if (t == last) S.mass_in = mb + m;
        __syncthreads();
        if (last >= 0) least = most = S.mass_in;
        const unsigned long long low = wanted_mass(top_p, least), high = wanted_mass(top_p, most);
        if (mb < low && low <= mb + m) S.bin = (uint32_t)t;
        if (mb < high && high <= mb + m) S.other = (uint32_t)t;
        __syncthreads();
        sure = S.bin == S.other;
        if (S.bin != 0xffffffffu) last = (int)S.bin;
    }
    if (last < 0) return no_cut(0ull);
    Cut cut;
    cut.key = S.sorted[last];
    cut.equal = (uint32_t)__syncthreads_count(t < n && key == cut.key);
    cut.ties = (uint32_t)__syncthreads_count(t <= last && key == cut.key);
    cut.mass = 0ull;                                     // (not asked for)
    return cut;
}

// The cut behind `want_count` tokens, or (want_count == 0) where the mass before a token is no longer less than want_mass: a key of
// [from, to], or none.  All logits from `from` on are in the warps' views.
template <typename T, bool RESIDENT, int N>
__device__ Cut find_cut(const Row<T, RESIDENT> &R, const View &V, Shared<N> &S, int rank, int ctas, uint32_t from, uint32_t to, bool masses,
                        unsigned long long want_count, unsigned long long want_mass) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = threadIdx.x;
    uint32_t count_above = 0u;
    unsigned long long mass_above = 0ull;
    for (bool opening = true;; opening = false) {
        const int bits = 32 - __clz(to - from), shift = bits > LOG_BINS<N> ? bits - LOG_BINS<N> : 0;
        S.count[t] = 0u; S.lo[t] = 0u; S.hi[t] = 0u;
        __syncthreads();
        uint32_t ca = 0u;
        unsigned long long ma = 0ull;
        for_quads(R, V, [&](int x, float (&v)[4]) {
            unsigned long long m[4] = {0ull, 0ull, 0ull, 0ull};
            if (masses) {
#pragma unroll
                for (int j = 0; j < 4; ++j) m[j] = R.mass(v[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = key_of<T>(v[j]);
                if (k < from || x + j >= V.count || (k > to && !opening)) continue;
                if (k > to) {
                    ++ca;
                    ma += m[j];
                } else {
                    const uint32_t bin = (k - from) >> shift;
                    atomicAdd(&S.count[bin], 1u);
                    if (masses) add_mass(&S.lo[bin], &S.hi[bin], m[j]);
                }
            }
        });
        if (opening) {
            ca = warp_sum(ca);
            ma = warp_sum(ma);
            if (lane == 0) { S.warp_count[warp] = ca; S.warp_mass[warp] = ma; }
            __syncthreads();
            if (t < ctas) {
                ca = 0u;
                ma = 0ull;
                for (int w = 0; w < WARPS<N>; ++w) { ca += S.warp_count[w]; ma += S.warp_mass[w]; }
                Shared<N> &D = of_cta(S, ctas, t);
                D.above_count[rank] = ca;
                D.above_mass[rank] = ma;
            }
        }
        row_sync(ctas);
        if (opening)
            for (int r = 0; r < ctas; ++r) { count_above += S.above_count[r]; mass_above += S.above_mass[r]; }
        uint32_t c = 0u;
        unsigned long long m = 0ull;
        const int bin = N - 1 - t;                    // from the top down
        for (int r = 0; r < ctas; ++r) {
            Shared<N> &D = of_cta(S, ctas, r);
            c += D.count[bin];
            if (masses) m += (unsigned long long)D.hi[bin] << 32 | D.lo[bin];
        }
        uint32_t cb = count_above;
        unsigned long long mb = mass_above;
        sums_before(S, c, m, cb, mb);
        if (t == 0) S.count_in = 0u;
        __syncthreads();
        if (want_count ? cb < want_count && want_count <= (unsigned long long)cb + c : mb < want_mass && want_mass <= mb + m) {
            S.bin = (uint32_t)bin;
            S.count_in = c; S.mass_in = m; S.count_above = cb; S.mass_above = mb;
        }
        row_sync(ctas);                                  // also: nobody reads another CTA's counters any more
        const uint32_t in = S.count_in;
        if (in == 0u) return no_cut(0ull);
        const uint32_t found = S.bin;
        count_above = S.count_above;
        mass_above = S.mass_above;
        Cut cut;
        if (shift == 0) {
            const unsigned long long each = S.mass_in / in;
            cut.key = from + found;
            cut.equal = in;
            cut.ties = (uint32_t)(want_count ? want_count - count_above : (want_mass - mass_above + each - 1) / each);
            cut.mass = mass_above + each * cut.ties;
            __syncthreads();
            return cut;
        }
        from += found << shift;
        to = min(to, from + ((1u << shift) - 1u));
        if (in <= N) {
            const int n = gather(R, V, S, ctas, from, to);
            const uint32_t key = t < n ? S.sorted[t] : 0u;
            m = masses && t < n ? R.mass(logit_of<T>(key)) : 0ull;
            cb = count_above;
            mb = mass_above;
            sums_before(S, t < n ? 1u : 0u, m, cb, mb);
            if (t < n && (want_count ? cb + 1u == want_count : mb < want_mass && want_mass <= mb + m)) {
                S.bin = (uint32_t)t;
                S.mass_in = mb + m;
            }
            __syncthreads();
            const int last = (int)S.bin;
            cut.key = S.sorted[last];
            cut.mass = S.mass_in;
            cut.equal = (uint32_t)__syncthreads_count(t < n && key == cut.key);
            cut.ties = (uint32_t)__syncthreads_count(t <= last && key == cut.key);
            return cut;
        }
        __syncthreads();
    }
}

// The stretches [S.first_bin, S.last_bin] of the coarse histogram that hold the cut, for a wanted count or mass between `least` and `most`.  A
// stretch's logits are less than (bin + 1) width and at least bin width below the maximum, but for the roundings that the margins cover.
template <int N> __device__ __forceinline__ void bracket(Shared<N> &S, double width, double inv_t, bool by_mass, double least, double most) {
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const double c = (double)S.total[t];
    double low = c, high = c;
    if (by_mass) {
        low = t < N - 1 ? c * (double)exp2f((float)(-(double)(t + 1) * width * 1.00001 * inv_t * 1.4426950408889634)) : 0.;
        high = c * (double)exp2f((float)(-(double)t * width * 0.99999 * inv_t * 1.4426950408889634));
    }
    low = warp_upto(low);
    high = warp_upto(high);
    __syncthreads();
    if (t == 0) { S.first_bin = N - 1; S.last_bin = N - 1; }
    if (lane == 31) { S.warp_low[warp] = low; S.warp_high[warp] = high; }
    __syncthreads();
    for (int w = 0; w < warp; ++w) { low += S.warp_low[w]; high += S.warp_high[w]; }
    // (more than the roundings of masses and of these exponentials; counts are whole)
    const double margin = by_mass ? 1e-5 : 0.;
    if (high >= least * (1. - margin)) atomicMin(&S.first_bin, t);
    if (low >= most * (1. + margin)) atomicMin(&S.last_bin, t);
    __syncthreads();
}

template <typename T, bool RESIDENT, int N>
__global__ void __launch_bounds__(N, 1024 / N) kernel(const __grid_constant__ Params P) {
    extern __shared__ __align__(16) char smem[];
    Shared<N> &S = *reinterpret_cast<Shared<N> *>(smem);
    const int ctas = (int)cooperative_groups::this_cluster().num_blocks(), rank = (int)cooperative_groups::this_cluster().block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x / ctas;
    const int begin = min(P.vocab, rank * P.slice), slice = min(P.slice, P.vocab - begin);
    const T *src = reinterpret_cast<const T *>(P.z) + row * P.zs + begin;
    T *own = reinterpret_cast<T *>(smem + sizeof(Shared<N>));
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    Row<T, RESIDENT> R;
    R.z = RESIDENT ? own : src;
    R.ring = own + warp * RING * 128;
    R.table = &S.table[0][lane % COPIES];
    R.quads = RESIDENT || (reinterpret_cast<uintptr_t>(src) & (4 * sizeof(T) - 1)) == 0;
    if (warp == 0) {
        const double e = exp2((double)lane / TABLE);
        for (int c = 0; c < COPIES; ++c) S.table[lane][c] = e;
    }
    *reinterpret_cast<uint4 *>(S.coarse[threadIdx.x]) = make_uint4(0u, 0u, 0u, 0u);

    // settings: on their way while the row is
    double temperature = P.temperature ? (double)P.temperature[row] : P.temperature_all;
    const double top_p = P.top_p ? (double)P.top_p[row] : P.top_p_all;
    const double min_p = P.min_p ? (double)P.min_p[row] : P.min_p_all;
    int64_t top_k = P.top_k ? P.top_k[row] : P.top_k_all;

    float best = -CUDART_INF_F;
    auto seen = [&](float v) { asm("max.NaN.f32 %0, %0, %1;" : "+f"(best) : "f"(v)); };
    constexpr int PER = 16 / (int)sizeof(T), U = 4;
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        const int pieces = slice / PER;
        done = pieces * PER;
        for (int x0 = threadIdx.x; x0 < pieces; x0 += U * N) {
            uint4 t[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (x0 + u * N < pieces) t[u] = __ldg(reinterpret_cast<const uint4 *>(src) + x0 + u * N);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (x0 + u * N < pieces) {
                    if (RESIDENT) reinterpret_cast<uint4 *>(own)[x0 + u * N] = t[u];
                    const T *v = reinterpret_cast<const T *>(&t[u]);
#pragma unroll
                    for (int z = 0; z < PER; ++z) seen((float)v[z]);
                }
        }
    }
    for (int x0 = done + threadIdx.x; x0 < slice; x0 += 2 * U * N) {
        T t[2 * U];
#pragma unroll
        for (int u = 0; u < 2 * U; ++u)
            if (x0 + u * N < slice) t[u] = src[x0 + u * N];
#pragma unroll
        for (int u = 0; u < 2 * U; ++u)
            if (x0 + u * N < slice) {
                if (RESIDENT) own[x0 + u * N] = t[u];
                seen((float)t[u]);
            }
    }
    if (!(best < CUDART_INF_F)) best = CUDART_INF_F;     // a NaN or +inf
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) S.warp_low[warp] = (double)best;
    __syncthreads();
    for (int w = 0; w < WARPS<N>; ++w) best = fmaxf(best, (float)S.warp_low[w]);
    if (ctas > 1) {
        // (all CTAs of the cluster run: their shared memory may be written)
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (threadIdx.x < ctas) of_cta(S, ctas, threadIdx.x).max_of[rank] = best;
        row_sync(ctas);
        for (int r = 0; r < ctas; ++r) best = fmaxf(best, S.max_of[r]);
    }
    if (best == CUDART_INF_F || best == -CUDART_INF_F) {         // no distribution
        if (rank == 0 && threadIdx.x == 0) {
            P.token[row] = -1;
            if (P.logprob) P.logprob[row] = CUDART_NAN_F;
        }
        return;
    }

    const bool greedy = !(temperature > 0.);
    if (greedy) {
        top_k = 1;
        temperature = 1.;
    }
    const bool by_count = top_k > 0 && top_k < P.vocab, by_mass = top_p < 1. && !greedy, by_floor = min_p > 0. && !greedy;
    // Logits and temperatures at the end of fp32 are scaled, so that there is a finite number without mass.  A temperature at which the next
    // smaller number has none is as good as any lower one, one at which all numbers weigh the same as any higher one.
    const double nats = (P.shift + 2) * 0.6931471805599453;      // below which a mass is 0
    temperature = fmin(temperature, 1e60);
    R.scale = (double)best - nats * temperature < -3e38 ? 1.1754944e-38f : 1.f;
    R.top = (double)(best * R.scale);
    const double gap = R.top - (double)logit_of<float>(key_of<float>((float)R.top) - 1u);
    temperature = fmax(temperature, gap / ((nats + 1.) * (double)R.scale));
    R.best = best;
    R.inv_t = 1. / temperature;
    R.steps = R.inv_t / (double)R.scale * (TABLE * 1.4426950408889634);
    R.shift = P.shift;
    R.least = __double2float_rd(R.top - nats * temperature * (double)R.scale);
    const uint32_t best_key = key_of<T>(best);
    // the smallest key that min-p leaves
    uint32_t floor_key = 0u;
    int floor_bin = N - 1;                            // a stretch of the coarse histogram that is not above it
    const double width = 24. * fmax(temperature, 1.) / N;     // of a stretch, in logits
    if (by_floor) {
        const double least = log(fmin(min_p, 1.));
        auto stays = [&](uint32_t k) { return R.exponent(logit_of<T>(k)) >= least; };
        const float about = (float)((double)best + least * temperature);
        if (about > -CUDART_INF_F) floor_key = first_key(best_key, key_of<T>(about), stays);
        floor_bin = (int)fmin(-least * temperature / width + 2., (double)(N - 1));
    }

    const int per_warp = ((P.slice / 128 + WARPS<N> - 1) / WARPS<N>) * 128;
    View V;
    V.list = nullptr;
    V.first = min(slice, warp * per_warp);
    V.count = min(slice, V.first + per_warp) - V.first;

    const bool small = P.vocab <= N;                  // sorted as a whole
    const double one = (double)(1ull << P.shift);
    int sums = 0;
    // of all threads of the row, in each of them (two sets of slots: a CTA may still read the last one)
    auto row_sum = [&](unsigned long long m) {
        m = warp_sum(m);
        __syncthreads();
        if (lane == 0) S.warp_mass[warp] = m;
        __syncthreads();
        m = 0ull;
        for (int w = 0; w < WARPS<N>; ++w) m += S.warp_mass[w];
        if (ctas == 1) return m;
        unsigned long long *slots = S.mass_of[sums++ & 1];
        if (threadIdx.x < ctas) of_cta(S, ctas, threadIdx.x).mass_of[(sums - 1) & 1][rank] = m;
        row_sync(ctas);
        m = 0ull;
        for (int r = 0; r < ctas; ++r) m += slots[r];
        return m;
    };
    // a warp's list of the logits that are at least `least`, filled a quad at a time
    int listed = 0;
    auto list_quad = [&](int x, const float (&v)[4], float least) {
        uint32_t in = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) in |= (x + j < V.count && v[j] >= least ? 1u : 0u) << j;
        if (!__any_sync(0xffffffffu, in)) return;
        const int n = __popc(in), upto = warp_upto(n);
        int at = listed + upto - n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (in >> j & 1u) {
                if (at < LIST) S.list[warp][at] = (uint16_t)(x + j);
                ++at;
            }
        listed += __shfl_sync(0xffffffffu, upto, 31);
    };
    const View all_logits = V;
    auto use_list = [&]() {
        __syncwarp();
        if (listed <= LIST) {
            V.list = S.list[warp];
            V.count = listed;
        }
    };

    // What min-p drops anyway is in no list (but where top-p takes its part of the mass of what top-k keeps).
    const bool floored = by_floor && !(by_count && by_mass), first_list = floored && floor_key > 0u && per_warp <= 65536;
    const float floor_logit = first_list ? logit_of<T>(floor_key) : 0.f;
    auto row_mass = [&]() {
        unsigned long long m = 0ull;
        for_quads(R, all_logits, [&](int, float (&v)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) m += R.mass(v[j]);
        });
        return row_sum(m);
    };
    // Top-p of the whole row: a sum in fp32 says what the row's mass is to a ten thousandth, which mostly shows the cut already.  With min-p
    // the first round does without the histogram: what min-p leaves is mostly little, and holds the cut or needs none.
    const bool of_row = by_mass && !by_count, cuts = by_count || by_mass;
    // Both take differences of logits in fp32.  Where one beyond fp32 may lie in a stretch, or have a mass (T above 1e37), there is neither: exact
    // masses, and a cut among all keys.
    const bool wide = fmax(width * N, nats * temperature) > 3.4e38;
    bool count = cuts && !small && !(of_row && first_list) && !wide, near = small;   // near: at most N logits are left
    unsigned long long least = 0ull, most = 0ull;        // bounds of the row's mass
    for (bool again = false;; again = true) {
        if (count || of_row || first_list) {
            const float scale = (float)(1. / width), exponent = (float)fmin(R.inv_t * 1.4426950408889634, 3e38);
            float about = 0.f;
            for_quads(R, all_logits, [&](int x, float (&v)[4]) {
                if (count) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // (rounded down by the sum with 2^23, whose low bits are then the whole number)
                        const float bin = __fadd_rd(fminf((best - v[j]) * scale, (float)(N - 1)), 8388608.f);
                        if (x + j < all_logits.count) atomicAdd(&S.coarse[__float_as_uint(bin) & (N - 1)][lane % SPLIT], 1u);
                    }
                }
                if (first_list && !again) list_quad(x, v, floor_logit);
                if (of_row && !again) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) about += ex2(fmaxf((v[j] - best) * exponent, -126.f));
                }
            });
            if (of_row && !again) {
                // off by 2^-22 a term, 2^-23 of the exponent (2^-16.5 at most, where the term counts) and 2^-24 an addition
                const double off = 5e-5 + P.slice * (5.9604645e-8 / N);
                const double row = (double)row_sum((unsigned long long)((double)about * 1073741824.)) / 1073741824.;
                least = (unsigned long long)(row * (1. - off) * one);
                most = (unsigned long long)(row * (1. + off) * one) + (unsigned long long)P.vocab;
            }
            if (first_list && !again) {
                const unsigned long long n = row_sum(lane == 0 ? (unsigned long long)listed : 0ull);
                use_list();
                near = near || n <= (unsigned long long)N;
            }
        }
        if (again || near || count || !cuts || wide) break;
        count = true;
    }
    if (count) {
        row_sync(ctas);
        uint32_t c = 0u;
#pragma unroll
        for (int r = 0; r < MAX_CTAS; ++r)
            if (r < ctas) {
                const uint4 n = *reinterpret_cast<const uint4 *>(of_cta(S, ctas, r).coarse[threadIdx.x]);
                c += n.x + n.y + n.z + n.w;
            }
        S.total[threadIdx.x] = c;
    }
    // (a temperature whose inverse is no fp32 number left that sum without meaning)
    if (of_row && (R.inv_t > 1e38 || wide)) least = most = row_mass();
    // The keys between which a cut lies, from the stretches [first, last]: of the numbers that are not outside of them, so that no more than one
    // stretch more is between the two keys.  Margins: a logit's stretch is found in fp32.
    auto key_from = [&](int last) {
        return last < N - 1 ? key_from_of<T>(fmaxf(__double2float_ru((double)best - (last + 1) * width * 1.00001), -3.402823466e38f)) : 0u;
    };
    auto key_to = [&](int first) { return first > 0 ? min(best_key, key_of<T>(__double2float_rd((double)best - first * width * 0.99999))) : best_key; };
    uint32_t from = floored ? floor_key : 0u, to = best_key;
    int last = floored ? floor_bin : N - 1;
    if (count) {
        bracket(S, width, R.inv_t, !by_count, by_count ? (double)top_k : top_p * (double)least / one, by_count ? (double)top_k : top_p * (double)most / one);
        from = max(from, key_from(S.last_bin));
        to = key_to(S.first_bin);
        last = min(last, S.last_bin);
        if (last < N - 1) {
            const uint32_t own = (int)threadIdx.x <= last + 1 ? S.total[threadIdx.x] : 0u;
            uint32_t before = 0u;
            unsigned long long none = 0ull;
            sums_before(S, own, 0ull, before, none);
            near = __syncthreads_and(before + own <= (uint32_t)N) || near;
        }
    }
    if (!V.list && from > (first_list ? floor_key : 0u) && per_warp <= 65536) {
        listed = 0;
        for_quads(R, V, [&](int x, float (&v)[4]) { list_quad(x, v, logit_of<T>(from)); });
        use_list();
    }
    Cut cut = no_cut(0ull);
    for (bool exact = false; cuts; exact = true) {
        // (not sure: by the estimate of the row's mass; if that is exact, there were too many after all)
        if (exact && (!of_row || least == most)) near = false;
        if (of_row && (exact || !near)) least = most = row_mass();
        bool sure = true;
        if (near) {
            cut = cut_few(R, V, S, ctas, from, by_count ? top_k : 0, by_mass ? top_p : 1., least, most, sure);
        } else {
            cut.mass = least;
            if (by_count) cut = find_cut(R, V, S, rank, ctas, from, max(from, to), by_mass, (unsigned long long)top_k, 0ull);
            if (by_mass) {
                const unsigned long long want = wanted_mass(top_p, cut.mass);
                if (by_count && count) {
                    bracket(S, width, R.inv_t, true, (double)want / one, (double)want / one);
                    from = max(from, key_from(S.last_bin));
                    to = key_to(S.first_bin);
                }
                cut = find_cut(R, V, S, rank, ctas, from, max(from, to), true, 0ull, want);
            }
        }
        if (sure) break;
    }

    uint32_t ties_before = 0u;
    const uint32_t least_key = max(cut.key, floor_key);
    const float least_logit = least_key > 0u ? logit_of<T>(least_key) : -CUDART_INF_F;
    const bool some = cut.ties < cut.equal && cut.key >= floor_key;      // not all tokens of the last key stay
    if (some) {
        uint32_t t = 0u;
        for (int x = lane; x < V.count; x += 32) t += (float)R.z[V.place(x)] == least_logit ? 1u : 0u;
        t = warp_sum(t);
        __syncthreads();
        if (lane == 0) S.warp_count[warp] = t;
        __syncthreads();
        uint32_t here = 0u;
        for (int w = 0; w < WARPS<N>; ++w) {
            ties_before += w < warp ? S.warp_count[w] : 0u;
            here += S.warp_count[w];
        }
        if (ctas > 1) {
            if (threadIdx.x < ctas) of_cta(S, ctas, threadIdx.x).ties_of[rank] = here;
            row_sync(ctas);
            for (int r = 0; r < rank; ++r) ties_before += S.ties_of[r];
        }
    }
    // Masses of logits x ... x + 3 of the view, 0 for those that are not kept.  `ties` counts the ones of the cut's key before these 128.
    auto kept = [&](int x, const float (&v)[4], uint32_t &ties, unsigned long long (&w)[4]) {
        uint32_t same = 0u, before = 0u;
        if (some) {
#pragma unroll
            for (int j = 0; j < 4; ++j) same += x + j < V.count && v[j] == least_logit ? 1u : 0u;
            const uint32_t upto = warp_upto(same);
            before = ties + upto - same;
            ties += __shfl_sync(0xffffffffu, upto, 31);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned long long m = R.mass(v[j]);   // (0 behind the view's end)
            w[j] = v[j] >= least_logit ? m : 0ull;
            if (some && x + j < V.count && v[j] == least_logit && before++ >= cut.ties) w[j] = 0ull;
        }
    };
    unsigned long long m = 0ull;
    uint32_t ties = ties_before;
    for_quads(R, V, [&](int x, float (&v)[4]) {
        unsigned long long w[4];
        kept(x, v, ties, w);
        m += w[0] + w[1] + w[2] + w[3];
    });
    m = warp_sum(m);
    __syncthreads();
    if (lane == 0) S.warp_mass[warp] = m;
    __syncthreads();
    unsigned long long below = 0ull, all = 0ull;
    for (int w = 0; w < WARPS<N>; ++w) {
        below += w < warp ? S.warp_mass[w] : 0ull;
        all += S.warp_mass[w];
    }
    if (ctas > 1) {
        if (threadIdx.x < ctas) of_cta(S, ctas, threadIdx.x).mass_of[sums & 1][rank] = all;
        row_sync(ctas);
        all = 0ull;
        for (int r = 0; r < ctas; ++r) {
            below += r < rank ? S.mass_of[sums & 1][r] : 0ull;
            all += S.mass_of[sums & 1][r];
        }
    }
    const double u = P.uniform64 ? reinterpret_cast<const double *>(P.uniform)[row] : (double)reinterpret_cast<const float *>(P.uniform)[row];
    unsigned long long target = u > 0. ? (u < 1. ? (unsigned long long)(u * (double)all) : all - 1ull) : 0ull;
    if (target >= all) target = all - 1ull;
    if (target < below || target >= below + m) return;
    ties = ties_before;
    for (int x0 = 0; x0 < V.count; x0 += 128) {
        const int x = x0 + lane * 4;
        float v[4];
        unsigned long long w[4];
        R.quad(V, x, v);
        kept(x, v, ties, w);
        const unsigned long long sum = w[0] + w[1] + w[2] + w[3], upto = warp_upto(sum);
        const uint32_t over = __ballot_sync(0xffffffffu, below + upto > target);
        if (over) {
            if (lane == __ffs(over) - 1) {
                unsigned long long at = below + upto - sum;
                int j = 0;
#pragma unroll
                for (int z = 0; z < 3; ++z)
                    if (j == z && at + w[z] <= target) {
                        at += w[z];
                        ++j;
                    }
                const int place = V.place(x + j);
                P.token[row] = begin + place;
                if (P.logprob) P.logprob[row] = (float)(R.exponent((float)R.z[place]) - log((double)all / one));
            }
            return;
        }
        below += __shfl_sync(0xffffffffu, upto, 31);
    }
}

// Rows of at most this many logits go to CTAs of 128 threads where there are more rows than SMs: the waits of eight of them overlap
// (4000 rows of 10000 bf16 logits, top-k 50 and top-p: 262 us with 512 threads, 144 with 128; 16384 rows of 256: 798 and 212).
constexpr int SHORT = 16384;
// CTAs of a row: twice as many while every SM has at most one and a slice keeps 2048 logits (64 rows of 32000: 20 us with two CTAs, 23 with four,
// 45 with eight, 23 with one; 256 rows of 128000: 130 with one, 142 with two, 237 with eight).
inline int ctas_of(int64_t rows, int vocab, int sms) {
    int c = 1;
    while (c < MAX_CTAS && rows * c * 2 <= sms && vocab > c * 4096) c *= 2;
    return c;
}
inline int slice_of(int vocab, int ctas) { return ((vocab + ctas - 1) / ctas + 127) / 128 * 128; }
// 2^(shift + bits of vocab) stays below 2^63, a mass below 2^52
inline int mass_shift(int vocab) {
    int bits = 0;
    while ((1ll << bits) < vocab) ++bits;
    return bits > 11 ? 62 - bits : 51;
}

}  // namespace sample
}  // namespace sa2
