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
// A cluster of CTAs holds a row in shared memory, read from global memory once.  A cut is found on the bits of the logits, mapped to integers
// in their order: a histogram of counts and masses over 2048 stretches of what is left, of which one holds the cut; bf16 takes two rounds
// of that, fp32 three.  Then each warp adds the kept masses of its stretch of indices, and the warp that has the drawn mass walks it.
#pragma once
#include "sa2_common.cuh"
#include <cooperative_groups.h>
#include <math_constants.h>

namespace sa2 {
namespace sample {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int LOG_BINS = 11, BINS = 1 << LOG_BINS, BINS_OF_THREAD = BINS / THREADS;
constexpr int MAX_CTAS = 8;

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
    int slice;                  // logits of a CTA, a multiple of 32
    int shift;                  // S above
    int resident;               // the slice is copied to shared memory
};

struct Cut {                    // of the order of the tokens, behind a token of the key `key`
    uint32_t key;
    uint32_t ties;              // tokens of that key that are kept, the lowest indices
    uint32_t equal;             // ... that there are
    unsigned long long mass;    // of what is kept
};

struct Shared {
    uint32_t count[BINS], lo[BINS], hi[BINS];
    uint32_t warp_count[WARPS];
    unsigned long long warp_mass[WARPS];
    float max_of[MAX_CTAS];
    uint32_t ties_of[MAX_CTAS];
    unsigned long long mass_of[MAX_CTAS];
    // the stretch with the cut, written by CTA 0
    uint32_t from, to, equal, count_above;
    unsigned long long mass_above, mass_in;
};

// Larger logits have larger keys; -0 and 0 the same one.
template <typename T> __device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t u = __float_as_uint(z + 0.f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return sizeof(T) == 2 ? k >> 16 : k;
}
template <typename T> struct Row {
    const T *z;                 // this CTA's slice
    int count;
    float best;
    double inv_t, one;          // 1 / T, 2^S
    __device__ __forceinline__ double exponent(float v) const { return ((double)v - (double)best) * inv_t; }
    __device__ __forceinline__ unsigned long long mass(float v) const { return __double2ull_rn(exp(exponent(v)) * one); }
};

// 64-bit counter of two words; a carry of the lower one is seen by the addition that makes it
__device__ __forceinline__ void add_mass(uint32_t *lo, uint32_t *hi, unsigned long long w) {
    const uint32_t l = (uint32_t)w;
    uint32_t h = (uint32_t)(w >> 32);
    if (l) h += atomicAdd(lo, l) + l < l ? 1u : 0u;
    if (h) atomicAdd(hi, h);
}

// The cut behind `want_count` tokens, or (want_count == 0) where the mass before a token is no longer less than want_mass.
template <typename T>
__device__ Cut find_cut(const Row<T> &R, Shared &S, uint32_t best_key, unsigned long long want_count, unsigned long long want_mass) {
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), ctas = (int)cl.num_blocks(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t from = 0u, to = best_key;
    uint32_t count_above = 0u, equal = 0u;
    unsigned long long mass_above = 0ull;
    while (true) {
        const int bits = 32 - __clz(to - from);
        const int shift = bits > LOG_BINS ? bits - LOG_BINS : 0;
        for (int x = threadIdx.x; x < BINS; x += THREADS) { S.count[x] = 0u; S.lo[x] = 0u; S.hi[x] = 0u; }
        __syncthreads();
        if (rank == 0 && ctas > 1) cl.barrier_arrive();
        for (int x = threadIdx.x; x < R.count; x += THREADS) {
            const float v = (float)R.z[x];
            const uint32_t k = key_of<T>(v);
            if (k < from || k > to) continue;
            const uint32_t bin = (k - from) >> shift;
            atomicAdd(&S.count[bin], 1u);
            add_mass(&S.lo[bin], &S.hi[bin], R.mass(v));
        }
        if (ctas > 1) {
            __syncthreads();
            // the others' counters into those of CTA 0, which are zeros or its own by now
            if (rank != 0) cl.barrier_arrive();
            cl.barrier_wait();
            if (rank != 0) {
                Shared *first = cl.map_shared_rank(&S, 0);
                for (int x = threadIdx.x; x < BINS; x += THREADS)
                    if (S.count[x]) {
                        atomicAdd(&first->count[x], S.count[x]);
                        add_mass(&first->lo[x], &first->hi[x], (unsigned long long)S.hi[x] << 32 | S.lo[x]);
                    }
            }
            cl.sync();
        } else {
            __syncthreads();
        }
        if (rank == 0) {
            // bins from the top down, BINS_OF_THREAD a thread
            uint32_t c[BINS_OF_THREAD], cs = 0u;
            unsigned long long m[BINS_OF_THREAD], ms = 0ull;
#pragma unroll
            for (int z = 0; z < BINS_OF_THREAD; ++z) {
                const int bin = BINS - 1 - (threadIdx.x * BINS_OF_THREAD + z);
                c[z] = S.count[bin];
                m[z] = (unsigned long long)S.hi[bin] << 32 | S.lo[bin];
                cs += c[z];
                ms += m[z];
            }
            uint32_t cb = cs;
            unsigned long long mb = ms;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t tc = __shfl_up_sync(0xffffffffu, cb, o);
                const unsigned long long tm = __shfl_up_sync(0xffffffffu, mb, o);
                if (lane >= o) { cb += tc; mb += tm; }
            }
            if (lane == 31) { S.warp_count[warp] = cb; S.warp_mass[warp] = mb; }
            __syncthreads();
            cb += count_above - cs;
            mb += mass_above - ms;
            for (int w = 0; w < warp; ++w) { cb += S.warp_count[w]; mb += S.warp_mass[w]; }
#pragma unroll
            for (int z = 0; z < BINS_OF_THREAD; ++z) {
                const bool here = want_count ? cb < want_count && want_count <= (unsigned long long)cb + c[z] : mb < want_mass && want_mass <= mb + m[z];
                if (here) {
                    const uint32_t bin = BINS - 1 - (threadIdx.x * BINS_OF_THREAD + z);
                    const uint32_t first = from + (bin << shift);
                    for (int r = 0; r < ctas; ++r) {
                        Shared *D = ctas > 1 ? cl.map_shared_rank(&S, r) : &S;
                        D->from = first;
                        D->to = min(to, first + ((1u << shift) - 1u));
                        D->equal = c[z];
                        D->count_above = cb;
                        D->mass_above = mb;
                        D->mass_in = m[z];
                    }
                }
                cb += c[z];
                mb += m[z];
            }
        }
        if (ctas > 1) cl.sync();
        else __syncthreads();
        from = S.from; to = S.to; equal = S.equal; count_above = S.count_above; mass_above = S.mass_above;
        if (shift == 0) break;
    }
    Cut cut;
    cut.key = from;
    cut.equal = equal;
    const unsigned long long each = S.mass_in / equal;
    if (want_count) cut.ties = (uint32_t)(want_count - count_above);
    else cut.ties = (uint32_t)((want_mass - mass_above + each - 1) / each);
    cut.mass = mass_above + each * cut.ties;
    return cut;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) kernel(const __grid_constant__ Params P) {
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    extern __shared__ __align__(16) char smem[];
    Shared &S = *reinterpret_cast<Shared *>(smem);
    const int rank = (int)cl.block_rank(), ctas = (int)cl.num_blocks(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x / ctas;
    const int begin = min(P.vocab, rank * P.slice);
    Row<T> R;
    R.count = min(P.slice, P.vocab - begin);
    const T *src = reinterpret_cast<const T *>(P.z) + row * P.zs + begin;
    T *own = reinterpret_cast<T *>(smem + sizeof(Shared));
    R.z = P.resident ? own : src;

    float best = -CUDART_INF_F;
    bool bad = false;                                    // a NaN or +inf
    for (int x = threadIdx.x; x < R.count; x += THREADS) {
        const T t = src[x];
        const float v = (float)t;
        if (P.resident) own[x] = t;
        bad |= !(v < CUDART_INF_F);
        best = fmaxf(best, v);
    }
    if (__syncthreads_or(bad)) best = CUDART_INF_F;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) S.warp_mass[warp] = __float_as_uint(best);
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) best = fmaxf(best, __uint_as_float((uint32_t)S.warp_mass[w]));
    if (ctas > 1) {
        if (threadIdx.x < ctas) cl.map_shared_rank(&S, threadIdx.x)->max_of[rank] = best;
        cl.sync();
        for (int r = 0; r < ctas; ++r) best = fmaxf(best, S.max_of[r]);
    }
    if (best == CUDART_INF_F || best == -CUDART_INF_F) {         // no distribution
        if (rank == 0 && threadIdx.x == 0) {
            P.token[row] = -1;
            if (P.logprob) P.logprob[row] = CUDART_NAN_F;
        }
        return;
    }

    const double temperature = P.temperature ? (double)P.temperature[row] : P.temperature_all;
    const double top_p = P.top_p ? (double)P.top_p[row] : P.top_p_all;
    const double min_p = P.min_p ? (double)P.min_p[row] : P.min_p_all;
    int64_t top_k = P.top_k ? P.top_k[row] : P.top_k_all;
    const bool greedy = !(temperature > 0.);
    if (greedy) top_k = 1;
    R.best = best;
    R.inv_t = greedy ? 1. : 1. / temperature;
    R.one = (double)(1ull << P.shift);
    const uint32_t best_key = key_of<T>(best);

    Cut cut;
    cut.key = 0u; cut.ties = 0xffffffffu; cut.equal = 0u; cut.mass = 0ull;
    bool whole = true;                                   // no cut yet
    if (top_k > 0 && top_k < P.vocab) {
        cut = find_cut<T>(R, S, best_key, (unsigned long long)top_k, 0ull);
        whole = false;
    }
    if (top_p < 1. && !greedy) {
        unsigned long long all = cut.mass;
        if (whole) {                                     // of the whole row
            unsigned long long m = 0ull;
            for (int x = threadIdx.x; x < R.count; x += THREADS) m += R.mass((float)R.z[x]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
            __syncthreads();
            if (lane == 0) S.warp_mass[warp] = m;
            __syncthreads();
            m = 0ull;
            for (int w = 0; w < WARPS; ++w) m += S.warp_mass[w];
            if (ctas > 1) {
                if (threadIdx.x < ctas) cl.map_shared_rank(&S, threadIdx.x)->mass_of[rank] = m;
                cl.sync();
                m = 0ull;
                for (int r = 0; r < ctas; ++r) m += S.mass_of[r];
            }
            all = m;
        }
        const double part = ceil(top_p * (double)all);
        unsigned long long want = part >= 1. ? (unsigned long long)part : 1ull;
        if (want > all) want = all;
        const Cut c = find_cut<T>(R, S, best_key, 0ull, want);
        cut = c;
    }
    const double floor_p = min_p > 0. ? fmin(min_p, 1.) : 0.;

    // a warp has consecutive indices
    const int per_warp = ((P.slice / 32 + WARPS - 1) / WARPS) * 32, first = min(R.count, warp * per_warp), last = min(R.count, first + per_warp);
    uint32_t ties_before = 0u;
    const bool some = cut.ties < cut.equal;              // not all tokens of the cut's key stay
    if (some) {
        uint32_t t = 0u;
        for (int x = first + lane; x < last; x += 32) t += key_of<T>((float)R.z[x]) == cut.key ? 1u : 0u;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        __syncthreads();
        if (lane == 0) S.warp_count[warp] = t;
        __syncthreads();
        uint32_t here = 0u;
        for (int w = 0; w < WARPS; ++w) {
            ties_before += w < warp ? S.warp_count[w] : 0u;
            here += S.warp_count[w];
        }
        if (ctas > 1) {
            if (threadIdx.x < ctas) cl.map_shared_rank(&S, threadIdx.x)->ties_of[rank] = here;
            cl.sync();
            for (int r = 0; r < rank; ++r) ties_before += S.ties_of[r];
        }
    }
    // the mass of the logit at x if it is kept; `ties` counts the ones of the cut's key so far
    auto kept = [&](int x, uint32_t &ties) -> unsigned long long {
        const bool on = x < last;
        const float v = on ? (float)R.z[x] : -CUDART_INF_F;
        const uint32_t k = key_of<T>(v);
        bool in = on && k >= cut.key;
        if (some) {
            const uint32_t same = __ballot_sync(0xffffffffu, on && k == cut.key);
            if (k == cut.key && ties + __popc(same & ((1u << lane) - 1u)) >= cut.ties) in = false;
            ties += __popc(same);
        }
        if (!in) return 0ull;
        const double w = exp(R.exponent(v));
        return w >= floor_p || k == best_key ? __double2ull_rn(w * R.one) : 0ull;
    };
    unsigned long long m = 0ull;
    uint32_t ties = ties_before;
    for (int x = first + lane; x - lane < last; x += 32) m += kept(x, ties);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    __syncthreads();
    if (lane == 0) S.warp_mass[warp] = m;
    __syncthreads();
    unsigned long long below = 0ull, all = 0ull;
    for (int w = 0; w < WARPS; ++w) {
        below += w < warp ? S.warp_mass[w] : 0ull;
        all += S.warp_mass[w];
    }
    if (ctas > 1) {
        if (threadIdx.x < ctas) cl.map_shared_rank(&S, threadIdx.x)->mass_of[rank] = all;
        cl.sync();
        all = 0ull;
        for (int r = 0; r < ctas; ++r) {
            below += r < rank ? S.mass_of[r] : 0ull;
            all += S.mass_of[r];
        }
    }
    const double u = P.uniform64 ? reinterpret_cast<const double *>(P.uniform)[row] : (double)reinterpret_cast<const float *>(P.uniform)[row];
    unsigned long long target = u > 0. ? (u < 1. ? (unsigned long long)(u * (double)all) : all - 1ull) : 0ull;
    if (target >= all) target = all - 1ull;
    if (target < below || target >= below + m) return;
    ties = ties_before;
    for (int x = first + lane; x - lane < last; x += 32) {
        const unsigned long long w = kept(x, ties);
        unsigned long long upto = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, below + upto > target);
        if (over) {
            if (lane == __ffs(over) - 1) {
                P.token[row] = begin + x;
                if (P.logprob) P.logprob[row] = (float)(R.exponent((float)R.z[x]) - log((double)all / R.one));
            }
            return;
        }
        below += __shfl_sync(0xffffffffu, upto, 31);
    }
}

// CTAs of a row: slices of at most 96 KB (two CTAs an SM), more CTAs while the rows leave SMs without one and a slice keeps 2048 logits.
inline int ctas_of(int64_t rows, int vocab, int size, int sms) {
    int c = 1;
    while (c < MAX_CTAS && (int64_t)vocab * size > (int64_t)c * 96 * 1024) c *= 2;
    while (c < MAX_CTAS && rows * c * 2 <= 2 * sms && vocab > c * 4096) c *= 2;
    return c;
}
inline int slice_of(int vocab, int ctas) { return ((vocab + ctas - 1) / ctas + 31) / 32 * 32; }
// 2^(shift + bits of vocab) stays below 2^63
inline int mass_shift(int vocab) {
    int bits = 0;
    while ((1ll << bits) < vocab) ++bits;
    return 62 - bits;
}

}  // namespace sample
}  // namespace sa2
