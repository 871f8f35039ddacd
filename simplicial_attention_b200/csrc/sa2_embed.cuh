// Embedding lookup with a scale and learned positions, and the dense gradients of both tables.
//
//   out[b, i] = scale W[token[b, i]] + P[start + i]
//   dW[t] = scale * sum of dout[b, i] over all (b, i) with token[b, i] == t,   dP[start + i] = sum over b of dout[b, i]
// A token outside [0, vocab) reads nothing: its row of out is NaN, and it has no gradient; nor has the padding token.
//
// Forward: HBM-bound copies of rows, 16 bytes a lane and access, four rows of a thread in flight.
//
// Backward, three launches.  (1) One cluster sorts the tokens with their places, stably, while the other CTAs of the launch write
// the zeros of dW: a sort is a chain of latencies that a few SMs do as fast as all of them.  (2) A warp adds a stretch of
// sorted places for 256 channels, rows of dout read whole; a token whose places all lie in the stretch is finished there, one that began or
// goes on elsewhere leaves a partial row.  Other CTAs of the launch add dP over the batch.  (3) Partial rows of a token are
// added in order.  Sums are fp32 and have one order, whatever the run: no atomics.
#pragma once
#include "sa2_common.cuh"
#include "sa2_vec8.cuh"
#include <cooperative_groups.h>

namespace sa2 {
namespace embed {

constexpr int THREADS = 256;

struct Params {
    const void *tokens;         // [rows]
    int tokens64;               // int64 or int32
    const void *weight;         // [vocab][dim]
    const void *positions;      // [.][dim], from row `start` on; may be null
    void *out;                  // [rows][dim]
    int64_t rows, vocab, start;
    int n, dim;                 // rows of a sequence, channels
    float scale;
};

__device__ __forceinline__ int64_t token_at(const void *tokens, int tokens64, int64_t r) {
    return tokens64 ? reinterpret_cast<const int64_t *>(tokens)[r] : (int64_t)reinterpret_cast<const int32_t *>(tokens)[r];
}

// Channels of a lane: eight, or one where rows do not begin on 16-byte boundaries.
template <typename T, int V> __device__ __forceinline__ void load_v(const T *p, float (&v)[V]) {
    if constexpr (V == 8) load8<T>(p, v);
    else v[0] = (float)p[0];
}
template <typename T, int V> __device__ __forceinline__ void store_v(T *p, const float (&v)[V]) {
    if constexpr (V == 8) store8<T>(p, v);
    else p[0] = (T)v[0];
}

// A group of `lanes` threads takes a row, the groups of a CTA four rows each.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) fwd_kernel(const __grid_constant__ Params P, int lanes) {
    constexpr int U = 4;
    const int groups = THREADS / lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
    const int64_t row0 = (int64_t)blockIdx.x * groups * U + group;
    const T *weight = reinterpret_cast<const T *>(P.weight), *positions = reinterpret_cast<const T *>(P.positions);
    int64_t token[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t r = row0 + u * groups;
        token[u] = r < P.rows ? token_at(P.tokens, P.tokens64, r) : -1;
    }
    for (int c = (blockIdx.y * lanes + lane) * V; c < P.dim; c += gridDim.y * lanes * V) {
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool there = token[u] >= 0 && token[u] < P.vocab;
#pragma unroll
            for (int z = 0; z < V; ++z) v[u][z] = __int_as_float(0x7fc00000);
            if (there) load_v<T, V>(weight + token[u] * P.dim + c, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = row0 + u * groups;
            if (r >= P.rows) break;
            if (positions) {
                float p[V];
                load_v<T, V>(positions + (P.start + (uint32_t)r % (uint32_t)P.n) * P.dim + c, p);
#pragma unroll
                for (int z = 0; z < V; ++z) v[u][z] = fmaf(v[u][z], P.scale, p[z]);
            } else {
#pragma unroll
                for (int z = 0; z < V; ++z) v[u][z] *= P.scale;
            }
            store_v<T, V>(reinterpret_cast<T *>(P.out) + r * P.dim + c, v[u]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- backward
constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, MAX_BINS = 512;
constexpr int STRETCH = 32;                             // sorted places of a warp

struct BwdParams {
    const void *tokens;
    int tokens64;
    const void *dout;           // [rows][dim]
    void *dweight;              // [vocab][dim]
    void *dpositions;           // [position_rows][dim], may be null
    uint32_t *key[2], *place[2];        // [rows] each: the two sides of the sort
    float *partial;             // [stretches][2][dim]: of the token that came from before, and of the one that goes on
    int64_t rows, vocab, padding, start, position_rows;
    int n, dim, passes, bits;   // sort: passes of `bits` bits; the sorted keys are in key[passes & 1]
    int vec;                    // rows of dout and dweight begin on 16-byte boundaries
    float scale;
};

template <typename T> struct Word;
__device__ __forceinline__ void zero_fill(char *p, int64_t bytes, int64_t first, int64_t step) {
    const int64_t pieces = bytes / 16;
    for (int64_t x = first; x < pieces; x += step) reinterpret_cast<uint4 *>(p)[x] = make_uint4(0u, 0u, 0u, 0u);
    for (int64_t x = pieces * 16 + first; x < bytes; x += step) p[x] = 0;
}

// Cluster 0 sorts (stable, least significant digits first), the others write zeros.  A CTA of the sort has consecutive places,
// a warp of it consecutive ones of those, so that (CTA, warp, lane) order is the order of the places.
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(const __grid_constant__ BwdParams P, int64_t dweight_bytes) {
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    if ((int)blockIdx.x >= ctas) {
        zero_fill(reinterpret_cast<char *>(P.dweight), dweight_bytes, (int64_t)(blockIdx.x - ctas) * SORT_THREADS + threadIdx.x,
                  (int64_t)(gridDim.x - ctas) * SORT_THREADS);
        return;
    }
    extern __shared__ uint32_t smem[];
    const int bins = 1 << P.bits;
    uint32_t *hist = smem;                               // [warps][bins]: counts, then where the warp's next key of a digit goes
    uint32_t *total = hist + SORT_WARPS * bins;          // [bins] counts of this CTA
    uint32_t *scan = total + bins;                       // [bins] sums over warps of a scan
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t per_warp = ((P.rows + (int64_t)ctas * SORT_THREADS - 1) / ((int64_t)ctas * SORT_THREADS)) * 32;
    const int64_t begin = ((int64_t)rank * SORT_WARPS + warp) * per_warp, end = min(P.rows, begin + per_warp);

    auto key_at = [&](int pass, int64_t x) -> uint32_t {
        if (pass) return P.key[pass & 1][x];
        const int64_t t = token_at(P.tokens, P.tokens64, x);
        return t < 0 || t >= P.vocab || t == P.padding ? (uint32_t)P.vocab : (uint32_t)t;
    };
    for (int pass = 0; pass < P.passes; ++pass) {
        for (int x = threadIdx.x; x < SORT_WARPS * bins; x += SORT_THREADS) hist[x] = 0u;
        __syncthreads();
        uint32_t *own = hist + warp * bins;
        for (int64_t x0 = begin; x0 < end; x0 += 32) {
            const bool on = x0 + lane < end;
            const uint32_t digit = on ? key_at(pass, x0 + lane) >> (pass * P.bits) & (bins - 1) : (uint32_t)bins;
            const uint32_t peers = __match_any_sync(0xffffffffu, digit);
            if (on && lane == __ffs(peers) - 1) own[digit] += __popc(peers);
            __syncwarp();
        }
        __syncthreads();
        // counts of earlier warps, digit by digit
        for (int d = threadIdx.x; d < bins; d += SORT_THREADS) {
            uint32_t s = 0u;
            for (int w = 0; w < SORT_WARPS; ++w) {
                const uint32_t c = hist[w * bins + d];
                hist[w * bins + d] = s;
                s += c;
            }
            total[d] = s;
        }
        cl.sync();
        // all smaller digits everywhere, and the same digit in earlier CTAs
        uint32_t before = 0u, all = 0u;
        const int d = threadIdx.x;
        if (d < bins)
            for (int r = 0; r < ctas; ++r) {
                const uint32_t c = cl.map_shared_rank(total, r)[d];
                before += r < rank ? c : 0u;
                all += c;
            }
        uint32_t upto = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        uint32_t base = upto - all + before;
        for (int w = 0; w < warp; ++w) base += scan[w];
        if (d < bins)
            for (int w = 0; w < SORT_WARPS; ++w) hist[w * bins + d] += base;
        __syncthreads();
        uint32_t *key_out = P.key[(pass + 1) & 1], *place_out = P.place[(pass + 1) & 1];
        for (int64_t x0 = begin; x0 < end; x0 += 32) {
            const bool on = x0 + lane < end;
            const uint32_t key = on ? key_at(pass, x0 + lane) : 0u;
            const uint32_t place = on ? (pass ? P.place[pass & 1][x0 + lane] : (uint32_t)(x0 + lane)) : 0u;
            const uint32_t digit = on ? key >> (pass * P.bits) & (bins - 1) : (uint32_t)bins;
            const uint32_t peers = __match_any_sync(0xffffffffu, digit);
            if (on) {
                const uint32_t to = own[digit] + __popc(peers & ((1u << lane) - 1u));
                key_out[to] = key;
                place_out[to] = place;
            }
            __syncwarp();
            if (on && lane == __ffs(peers) - 1) own[digit] += __popc(peers);
            __syncwarp();
        }
        cl.sync();           // the pass is written, and nobody reads this CTA's counts any more
    }
}

// Warps [0, stretches * tiles): a stretch of sorted places, 32 V channels.  Those behind: a row of dP, 32 V channels.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) sum_kernel(const __grid_constant__ BwdParams P, int64_t stretches, int tiles) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    const int c = (int)(unit % tiles) * 32 * V + lane * V;
    const int64_t item = unit / tiles;
    const bool on = c < P.dim;
    const T *dout = reinterpret_cast<const T *>(P.dout);
    float acc[V];
#pragma unroll
    for (int z = 0; z < V; ++z) acc[z] = 0.f;
    constexpr int U = 8;
    if (item >= stretches) {
        const int64_t p = item - stretches;
        if (p >= P.position_rows || !P.dpositions || !on) return;
        const int64_t i = p - P.start, sequences = P.rows / P.n;
        if (i >= 0 && i < P.n)
            for (int64_t b = 0; b < sequences; b += U) {
                float v[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (b + u < sequences) load_v<T, V>(dout + ((b + u) * P.n + i) * P.dim + c, v[u]);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (b + u < sequences) {
#pragma unroll
                        for (int z = 0; z < V; ++z) acc[z] += v[u][z];
                    }
            }
        store_v<T, V>(reinterpret_cast<T *>(P.dpositions) + p * P.dim + c, acc);
        return;
    }
    const uint32_t *key = P.key[P.passes & 1], *place = P.place[P.passes & 1];
    const int64_t begin = item * STRETCH;
    const int count = (int)min((int64_t)STRETCH, P.rows - begin);
    const uint32_t my_key = lane < count ? key[begin + lane] : 0xffffffffu, my_place = lane < count ? place[begin + lane] : 0u;
    const uint32_t before = begin > 0 ? key[begin - 1] : 0xffffffffu;
    const uint32_t after = begin + count < P.rows ? key[begin + count] : 0xffffffffu;
    uint32_t run = __shfl_sync(0xffffffffu, my_key, 0);
    bool first = true;                                   // no token of this stretch is finished yet
    auto flush = [&](bool goes_on) {
        const bool came = first && run == before;
        first = false;
        if (run < (uint32_t)P.vocab && on) {
            if (came || goes_on) {
                store_v<float, V>(P.partial + (item * 2 + (came ? 0 : 1)) * P.dim + c, acc);
            } else {
#pragma unroll
                for (int z = 0; z < V; ++z) acc[z] *= P.scale;
                store_v<T, V>(reinterpret_cast<T *>(P.dweight) + (int64_t)run * P.dim + c, acc);
            }
        }
#pragma unroll
        for (int z = 0; z < V; ++z) acc[z] = 0.f;
    };
    for (int e0 = 0; e0 < count; e0 += U) {
        float v[U][V];
        uint32_t k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = __shfl_sync(0xffffffffu, my_key, (e0 + u) & 31);
            const int64_t p = __shfl_sync(0xffffffffu, my_place, (e0 + u) & 31);
#pragma unroll
            for (int z = 0; z < V; ++z) v[u][z] = 0.f;
            if (e0 + u < count && k[u] < (uint32_t)P.vocab && on) load_v<T, V>(dout + p * P.dim + c, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (e0 + u >= count) break;
            if (k[u] != run) {
                flush(false);
                run = k[u];
            }
#pragma unroll
            for (int z = 0; z < V; ++z) acc[z] += v[u][z];
        }
    }
    flush(run == after);
}

// A CTA for each (stretch, 32 V channels) in which a token begins that goes on in the next: its eight warps add the partial rows of
// stretch + 1 + warp, + 8, ..., then the warps are added in order.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) join_kernel(const __grid_constant__ BwdParams P, int tiles) {
    const int64_t item = blockIdx.x / tiles;
    const int tile = (int)(blockIdx.x % tiles), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t *key = P.key[P.passes & 1];
    const int64_t begin = item * STRETCH, next = begin + STRETCH;
    if (next >= P.rows) return;
    const uint32_t run = key[next - 1];
    if (run >= (uint32_t)P.vocab || key[next] != run || (begin > 0 && key[begin - 1] == run)) return;
    // where the token ends: the first place with a larger key
    int64_t lo = next, hi = P.rows;
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (key[mid] <= run) lo = mid + 1;
        else hi = mid;
    }
    const int64_t last = (lo - 1) / STRETCH;             // the last stretch that has it
    const int c = tile * 32 * V + lane * V;
    const bool on = c < P.dim;
    __shared__ float sums[THREADS / 32][32][V + 1];
    float acc[V];
#pragma unroll
    for (int z = 0; z < V; ++z) acc[z] = 0.f;
    constexpr int U = 4, W = THREADS / 32;
    if (on)
        for (int64_t s = item + 1 + warp; s <= last; s += U * W) {
            float v[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * W <= last) load_v<float, V>(P.partial + (s + u * W) * 2 * P.dim + c, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * W <= last) {
#pragma unroll
                    for (int z = 0; z < V; ++z) acc[z] += v[u][z];
                }
        }
#pragma unroll
    for (int z = 0; z < V; ++z) sums[warp][lane][z] = acc[z];
    __syncthreads();
    if (warp != 0 || !on) return;
    load_v<float, V>(P.partial + (item * 2 + 1) * P.dim + c, acc);
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int z = 0; z < V; ++z) acc[z] += sums[w][lane][z];
#pragma unroll
    for (int z = 0; z < V; ++z) acc[z] *= P.scale;
    store_v<T, V>(reinterpret_cast<T *>(P.dweight) + (int64_t)run * P.dim + c, acc);
}

inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int64_t stretches(int64_t rows) { return (rows + STRETCH - 1) / STRETCH; }
inline size_t workspace_bytes(int64_t rows, int dim) {
    return 4 * up256((size_t)rows * 4) + up256((size_t)stretches(rows) * 2 * dim * sizeof(float));
}
// bits of keys up to `vocab` (the key of a token that has no gradient), in passes of at most nine
inline void sort_plan(int64_t vocab, int &passes, int &bits) {
    int all = 1;
    while (((int64_t)1 << all) <= vocab) ++all;
    passes = (all + 8) / 9;
    bits = (all + passes - 1) / passes;
}
// CTAs of the sort: 1024 places each, a power of two up to sixteen
inline int sort_ctas(int64_t rows) {
    int c = 1;
    while (c < 16 && rows > (int64_t)c * SORT_THREADS) c *= 2;
    return c;
}
inline size_t sort_smem(int bits) { return ((size_t)SORT_WARPS + 2) * ((size_t)1 << bits) * 4 + SORT_WARPS * 4; }

}  // namespace embed
}  // namespace sa2
