// Embedding lookup with a scale and learned positions, and the dense gradients of both tables.
//
//   out[b, i] = scale W[token[b, i]] + P[start + i]
//   dW[t] = scale * sum of dout[b, i] over all (b, i) with token[b, i] == t,   dP[start + i] = sum over b of dout[b, i]
// A token outside [0, vocab) reads nothing: its row of out is NaN, and it has no gradient; nor has the padding token.
//
// Forward: HBM-bound copies of rows, 16 bytes a lane and access, the pieces of four bf16 or two fp32 rows in flight (16384 rows of 2048 bf16
// channels 20 us, 6.7 TB/s with rows that L2 holds).
//
// Backward, three launches.  (1) One cluster sorts the tokens with their places, stably, while the other CTAs of the launch write the zeros of
// the tokens that are not there - each looks through all tokens for those of its stretch of the table - and add dP over the batch: a sort is a
// chain of latencies that a few SMs do as fast as all of them.  (2) A warp adds a stretch of sorted places for 256 channels, rows of
// dout read whole; a token whose places all lie in the stretch is finished there, one that began or goes on elsewhere leaves a partial row.
// (3) Partial rows of a token are added in order.  16384 tokens, 50001 of 2048 bf16 channels: 40, 27 and 9 us (zeros of the whole table beside
// the sort, written twice where tokens are: 40 and 49); 16384 of 256 tokens, 512 fp32 channels: 13 (10 without the positions' sums), 8 and 4.  Sums are
// fp32 and have one order, whatever the run: no floating-point atomics.
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

// What a lane holds of a row in pieces of 32 V channels: eight consecutive channels, where rows begin on 16-byte boundaries (V == 8), else four, 32
// apart (V == 4).
template <typename T, int V> struct Held;
template <typename T> struct Held<T, 8> {
    Packed<T> x;
    __device__ __forceinline__ void load(const T *row, int c0, int lane, int dim) {
        if (c0 + lane * 8 < dim) x.load(row + c0 + lane * 8);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { x.get(v); }
};
template <typename T> struct Held<T, 4> {
    T x[4];
    __device__ __forceinline__ void load(const T *row, int c0, int lane, int dim) {
#pragma unroll
        for (int z = 0; z < 4; ++z)
            if (c0 + lane + 32 * z < dim) x[z] = row[c0 + lane + 32 * z];
    }
    __device__ __forceinline__ void get(float (&v)[4]) const {
#pragma unroll
        for (int z = 0; z < 4; ++z) v[z] = (float)x[z];
    }
};
template <typename T, int V> __device__ __forceinline__ void put(T *row, int c0, int lane, int dim, const float (&v)[V]) {
    if constexpr (V == 8) {
        if (c0 + lane * 8 < dim) store8<T>(row + c0 + lane * 8, v);
    } else {
#pragma unroll
        for (int z = 0; z < 4; ++z)
            if (c0 + lane + 32 * z < dim) row[c0 + lane + 32 * z] = (T)v[z];
    }
}

template <typename T> constexpr int ROWS = sizeof(T) == 2 ? 4 : 2;       // of a warp
// A warp has pieces of 32 V channels of ROWS rows.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) fwd_kernel(const __grid_constant__ Params P, int tiles) {
    constexpr int U = ROWS<T>;
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5), row0 = unit / tiles * U;
    const int c0 = (int)(unit % tiles) * 32 * V;
    if (row0 >= P.rows) return;
    const T *weight = reinterpret_cast<const T *>(P.weight), *positions = reinterpret_cast<const T *>(P.positions);
    int64_t token[U];
#pragma unroll
    for (int u = 0; u < U; ++u) token[u] = row0 + u < P.rows ? token_at(P.tokens, P.tokens64, row0 + u) : -1;
    Held<T, V> w[U], p[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (positions && row0 + u < P.rows) p[u].load(positions + (P.start + (uint32_t)(row0 + u) % (uint32_t)P.n) * P.dim, c0, lane, P.dim);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (token[u] >= 0 && token[u] < P.vocab) w[u].load(weight + token[u] * P.dim, c0, lane, P.dim);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (row0 + u >= P.rows) break;
        float v[V], q[V];
        w[u].get(v);
        p[u].get(q);
        const bool there = token[u] >= 0 && token[u] < P.vocab;
#pragma unroll
        for (int z = 0; z < V; ++z) {
            v[z] = positions ? fmaf(v[z], P.scale, q[z]) : v[z] * P.scale;
            if (!there) v[z] = __int_as_float(0x7fc00000);
        }
        put<T, V>(reinterpret_cast<T *>(P.out) + (row0 + u) * P.dim, c0, lane, P.dim, v);
    }
}

// ---------------------------------------------------------------------------------------------------------------- backward
constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32, SORT_CTAS = 8;
constexpr int WORDS = 4096;                             // of 32 tokens, that a CTA looks for at a time
constexpr int STRETCH = 32;                             // sorted places of a warp

struct BwdParams {
    const void *tokens;
    int tokens64;
    const void *dout;           // [rows][dim]
    void *dweight;              // [vocab][dim], may be null
    void *dpositions;           // [position_rows][dim], may be null
    uint32_t *key[2], *place[2];        // [rows] each: the two sides of the sort
    float *partial;             // [stretches][2][dim]: of the token that came from before, and of the one that goes on
    int64_t rows, vocab, padding, start, position_rows;
    int n, dim, passes, bits;   // sort: passes of `bits` bits; the sorted keys are in key[passes & 1]
    int tiles;                  // pieces of a row
    int zeroing;                // CTAs that write zeros
    float scale;
};

// dP, a warp for 32 V channels of a row
template <typename T, int V> __device__ __forceinline__ void add_positions(const BwdParams &P, int64_t unit) {
    constexpr int U = V == 8 && sizeof(T) == 4 ? 4 : 8;
    const int lane = threadIdx.x & 31, c0 = (int)(unit % P.tiles) * 32 * V;
    const int64_t p = unit / P.tiles, i = p - P.start, sequences = P.rows / P.n;
    const T *dout = reinterpret_cast<const T *>(P.dout);
    float acc[V];
#pragma unroll
    for (int z = 0; z < V; ++z) acc[z] = 0.f;
    if (i >= 0 && i < P.n)
        for (int64_t b = 0; b < sequences; b += U) {
            Held<T, V> t[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (b + u < sequences) t[u].load(dout + ((b + u) * P.n + i) * P.dim, c0, lane, P.dim);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (b + u < sequences) {
                    float v[V];
                    t[u].get(v);
#pragma unroll
                    for (int z = 0; z < V; ++z) acc[z] += v[z];
                }
        }
    put<T, V>(reinterpret_cast<T *>(P.dpositions) + p * P.dim, c0, lane, P.dim, acc);
}

__device__ __forceinline__ uint32_t key_of(const BwdParams &P, int64_t x) {
    const int64_t t = token_at(P.tokens, P.tokens64, x);
    return t < 0 || t >= P.vocab || t == P.padding ? (uint32_t)P.vocab : (uint32_t)t;
}

__device__ __forceinline__ void warp_zeros(char *p, int64_t bytes) {
    const int lane = threadIdx.x & 31;
    int64_t head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15;
    if (head > bytes) head = bytes;
    if (lane < head) p[lane] = 0;
    p += head;
    bytes -= head;
    for (int64_t x = lane; x < bytes / 16; x += 32) reinterpret_cast<uint4 *>(p)[x] = make_uint4(0u, 0u, 0u, 0u);
    if (lane < (bytes & 15)) p[(bytes & ~(int64_t)15) + lane] = 0;
}

// Zeros of the tokens of [first, last) that are not there: a CTA, `bits` of WORDS words, which say of 32 tokens each that there is nothing to do
__device__ __forceinline__ void zero_absent(const BwdParams &P, int64_t first, int64_t last, uint32_t *bits, int64_t row_bytes) {
    for (int64_t w0 = first / 32; w0 * 32 < last; w0 += WORDS) {
        const int words = (int)min((int64_t)WORDS, (last + 31) / 32 - w0);
        __syncthreads();
        for (int x = threadIdx.x; x < words; x += SORT_THREADS) {
            const int64_t t0 = (w0 + x) * 32;
            bits[x] = (t0 < first ? (1u << (first - t0)) - 1u : 0u) | (t0 + 32 > last ? ~0u << (last - t0) : 0u);
        }
        __syncthreads();
        constexpr int U = 4;
        for (int64_t x0 = threadIdx.x; x0 < P.rows; x0 += U * SORT_THREADS) {
            uint32_t k[U];
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = x0 + u * SORT_THREADS < P.rows ? key_of(P, x0 + u * SORT_THREADS) : (uint32_t)P.vocab;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t w = (int64_t)(k[u] / 32) - w0;
                if (k[u] < (uint32_t)P.vocab && w >= 0 && w < words && !(bits[w] >> (k[u] & 31) & 1u)) atomicOr(bits + w, 1u << (k[u] & 31));
            }
        }
        __syncthreads();
        // a warp has as many neighbouring tokens as 2 KB hold
        int group = 1;
        while (group < 32 && 2 * group * row_bytes <= 2048) group *= 2;
        for (int x = threadIdx.x >> 5; x < words * (32 / group); x += SORT_WARPS) {
            const int64_t t0 = w0 * 32 + (int64_t)x * group;
            uint32_t absent = ~bits[x * group / 32] >> (x * group % 32);
            if (group < 32) absent &= (1u << group) - 1u;
            while (absent) {
                const int from = __ffs(absent) - 1, behind = ~(absent >> from) ? __ffs(~(absent >> from)) - 1 : 32, count = min(behind, 32 - from);
                warp_zeros(reinterpret_cast<char *>(P.dweight) + (t0 + from) * row_bytes, count * row_bytes);
                absent = from + count == 32 ? 0u : absent & ~((1u << (from + count)) - 1u);
            }
        }
    }
}

// The first cluster sorts (stable, least significant digits first), `sorting` CTAs (0: none), the others write zeros and add dP.  A CTA of
// the sort has consecutive places, a warp of it consecutive ones of those, so that (CTA, warp, lane) order is the order of the places.
template <typename T, int V>
__global__ void __launch_bounds__(SORT_THREADS, 2) sort_kernel(const __grid_constant__ BwdParams P, int sorting) {
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    extern __shared__ uint32_t smem[];
    if ((int)blockIdx.x >= sorting) {
        const int64_t cta = blockIdx.x - sorting, others = gridDim.x - sorting;
        if (P.dweight) {
            int64_t each = (P.vocab + P.zeroing - 1) / P.zeroing;
            if (each > SORT_WARPS && each < 4 * SORT_WARPS) each = (each + SORT_WARPS - 1) / SORT_WARPS * SORT_WARPS;
            if (cta < P.zeroing) zero_absent(P, min(P.vocab, cta * each), min(P.vocab, (cta + 1) * each), smem, (int64_t)P.dim * sizeof(T));
        }
        const int64_t units = P.position_rows * P.tiles;
        for (int64_t u = cta * SORT_WARPS + warp; P.dpositions && u < units; u += others * SORT_WARPS) add_positions<T, V>(P, u);
        return;
    }
    const int ctas = (int)cl.num_blocks(), rank = (int)cl.block_rank(), bins = 1 << P.bits;
    uint32_t *hist = smem;                               // [warps][bins]: counts, then where the warp's next key of a digit goes
    uint32_t *total = hist + SORT_WARPS * bins;          // [bins] counts of this CTA
    uint32_t *scan = total + bins;                       // sums over warps of a scan
    const int64_t per_warp = ((P.rows + (int64_t)ctas * SORT_THREADS - 1) / ((int64_t)ctas * SORT_THREADS)) * 32;
    const int64_t begin = ((int64_t)rank * SORT_WARPS + warp) * per_warp, end = min(P.rows, begin + per_warp);
    auto key_at = [&](int pass, int64_t x) -> uint32_t { return pass ? P.key[pass & 1][x] : key_of(P, x); };
    for (int pass = 0; pass < P.passes; ++pass) {
        constexpr int U = 4;                             // keys of a lane on their way
        for (int x = threadIdx.x; x < SORT_WARPS * bins; x += SORT_THREADS) hist[x] = 0u;
        __syncthreads();
        uint32_t *own = hist + warp * bins;
        for (int64_t x0 = begin; x0 < end; x0 += U * 32) {
            uint32_t key[U];
#pragma unroll
            for (int u = 0; u < U; ++u) key[u] = x0 + u * 32 + lane < end ? key_at(pass, x0 + u * 32 + lane) : 0u;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool on = x0 + u * 32 + lane < end;
                const uint32_t digit = on ? key[u] >> (pass * P.bits) & (bins - 1) : (uint32_t)bins;
                const uint32_t peers = __match_any_sync(0xffffffffu, digit);
                if (on && lane == __ffs(peers) - 1) own[digit] += __popc(peers);
                __syncwarp();
            }
        }
        __syncthreads();
        // counts of earlier warps, digit by digit
        for (int d = threadIdx.x; d < bins; d += SORT_THREADS) {
            uint32_t s = 0u;
            for (int w0 = 0; w0 < SORT_WARPS; w0 += 8) {
                uint32_t c[8];
#pragma unroll
                for (int w = 0; w < 8; ++w) c[w] = hist[(w0 + w) * bins + d];
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    hist[(w0 + w) * bins + d] = s;
                    s += c[w];
                }
            }
            total[d] = s;
        }
        cl.sync();
        // all smaller digits everywhere, and the same digit in earlier CTAs (a digit a thread: there are at most 512)
        uint32_t before = 0u, all = 0u;
        const int d = threadIdx.x;
        if (d < bins) {
            uint32_t c[SORT_CTAS];
#pragma unroll
            for (int r = 0; r < SORT_CTAS; ++r) c[r] = r < ctas ? cl.map_shared_rank(total, r)[d] : 0u;
#pragma unroll
            for (int r = 0; r < SORT_CTAS; ++r) {
                before += r < rank ? c[r] : 0u;
                all += c[r];
            }
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
        for (int w = 0; w < warp && w * 32 < bins; ++w) base += scan[w];
        if (d < bins) {
#pragma unroll 8
            for (int w = 0; w < SORT_WARPS; ++w) hist[w * bins + d] += base;
        }
        __syncthreads();
        uint32_t *key_out = P.key[(pass + 1) & 1], *place_out = P.place[(pass + 1) & 1];
        for (int64_t x0 = begin; x0 < end; x0 += U * 32) {
            uint32_t key[U], place[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t x = x0 + u * 32 + lane;
                key[u] = x < end ? key_at(pass, x) : 0u;
                place[u] = x < end ? (pass ? P.place[pass & 1][x] : (uint32_t)x) : 0u;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool on = x0 + u * 32 + lane < end;
                const uint32_t digit = on ? key[u] >> (pass * P.bits) & (bins - 1) : (uint32_t)bins;
                const uint32_t peers = __match_any_sync(0xffffffffu, digit);
                if (on) {
                    const uint32_t to = own[digit] + __popc(peers & ((1u << lane) - 1u));
                    key_out[to] = key[u];
                    place_out[to] = place[u];
                }
                __syncwarp();
                if (on && lane == __ffs(peers) - 1) own[digit] += __popc(peers);
                __syncwarp();
            }
        }
        cl.sync();           // the pass is written, and nobody reads this CTA's counts any more
    }
}

// A warp: a stretch of sorted places, 32 V channels.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) sum_kernel(const __grid_constant__ BwdParams P, int64_t stretches) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    const int64_t item = unit / P.tiles;
    if (item >= stretches) return;
    const int c0 = (int)(unit % P.tiles) * 32 * V;
    const T *dout = reinterpret_cast<const T *>(P.dout);
    const uint32_t *key = P.key[P.passes & 1], *place = P.place[P.passes & 1];
    const int64_t begin = item * STRETCH;
    const int count = (int)min((int64_t)STRETCH, P.rows - begin);
    const uint32_t my_key = lane < count ? key[begin + lane] : 0xffffffffu, my_place = lane < count ? place[begin + lane] : 0u;
    const uint32_t before = begin > 0 ? key[begin - 1] : 0xffffffffu;
    const uint32_t after = begin + count < P.rows ? key[begin + count] : 0xffffffffu;
    uint32_t run = __shfl_sync(0xffffffffu, my_key, 0);
    float acc[V];
#pragma unroll
    for (int z = 0; z < V; ++z) acc[z] = 0.f;
    bool first = true;                                   // no token of this stretch is finished yet
    auto flush = [&](bool goes_on) {
        const bool came = first && run == before;
        first = false;
        if (run < (uint32_t)P.vocab) {
            if (came || goes_on) {
                put<float, V>(P.partial + (item * 2 + (came ? 0 : 1)) * P.dim, c0, lane, P.dim, acc);
            } else {
#pragma unroll
                for (int z = 0; z < V; ++z) acc[z] *= P.scale;
                put<T, V>(reinterpret_cast<T *>(P.dweight) + (int64_t)run * P.dim, c0, lane, P.dim, acc);
            }
        }
#pragma unroll
        for (int z = 0; z < V; ++z) acc[z] = 0.f;
    };
    constexpr int U = V == 8 && sizeof(T) == 4 ? 4 : 8;
    for (int e0 = 0; e0 < count; e0 += U) {
        Held<T, V> t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = __shfl_sync(0xffffffffu, my_key, (e0 + u) & 31);
            const int64_t p = __shfl_sync(0xffffffffu, my_place, (e0 + u) & 31);
            if (e0 + u < count && k < (uint32_t)P.vocab) t[u].load(dout + p * P.dim, c0, lane, P.dim);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = __shfl_sync(0xffffffffu, my_key, (e0 + u) & 31);
            if (e0 + u >= count) break;
            if (k != run) {
                flush(false);
                run = k;
            }
            float v[V];
            t[u].get(v);
#pragma unroll
            for (int z = 0; z < V; ++z) acc[z] += v[z];
        }
    }
    flush(run == after);
}

// A CTA for each (stretch, 32 V channels) in which a token begins that goes on in the next: its eight warps add the partial rows of
// stretch + 1 + warp, + 8, ..., then the warps are added in order.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) join_kernel(const __grid_constant__ BwdParams P) {
    const int64_t item = blockIdx.x / P.tiles;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = (int)(blockIdx.x % P.tiles) * 32 * V;
    const uint32_t *key = P.key[P.passes & 1];
    const int64_t begin = item * STRETCH, next = begin + STRETCH;
    if (next >= P.rows) return;
    const uint32_t run = key[next - 1], then = key[next], came = begin > 0 ? key[begin - 1] : 0xffffffffu;
    if (run >= (uint32_t)P.vocab || then != run || came == run) return;
    // the stretches behind this one that begin with the token
    int64_t more = 0;
    for (int step = THREADS; step == THREADS; more += step) {
        const int64_t at = (item + 1 + more + threadIdx.x) * STRETCH;
        step = __syncthreads_count(at < P.rows && key[at] == run);
    }
    const int64_t last = item + more;
    __shared__ float sums[THREADS / 32][32][V + 1];
    float acc[V];
#pragma unroll
    for (int z = 0; z < V; ++z) acc[z] = 0.f;
    constexpr int U = 4, W = THREADS / 32;
    for (int64_t s = item + 1 + warp; s <= last; s += U * W) {
        Held<float, V> t[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u * W <= last) t[u].load(P.partial + (s + u * W) * 2 * P.dim, c0, lane, P.dim);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u * W <= last) {
                float v[V];
                t[u].get(v);
#pragma unroll
                for (int z = 0; z < V; ++z) acc[z] += v[z];
            }
    }
#pragma unroll
    for (int z = 0; z < V; ++z) sums[warp][lane][z] = acc[z];
    __syncthreads();
    if (warp != 0) return;
    Held<float, V> own;
    own.load(P.partial + (item * 2 + 1) * P.dim, c0, lane, P.dim);
    own.get(acc);
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int z = 0; z < V; ++z) acc[z] += sums[w][lane][z];
#pragma unroll
    for (int z = 0; z < V; ++z) acc[z] *= P.scale;
    put<T, V>(reinterpret_cast<T *>(P.dweight) + (int64_t)run * P.dim, c0, lane, P.dim, acc);
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
// CTAs of the sort: a power of two, up to 512 places each until there are eight
inline int sort_ctas(int64_t rows) {
    int c = 1;
    while (c < SORT_CTAS && rows > (int64_t)c * SORT_THREADS) c *= 2;
    return c;
}
// CTAs beside the sort: two an SM, as many as clusters of that many CTAs find room for
inline int others_at_most(int cluster, int sms) { return cluster == SORT_CTAS ? 216 : 2 * sms - 2 * cluster; }
// CTAs that write zeros: one for 512 tokens; more where rows that no token can name weigh more than 128 KB each of them.  Each looks through all
// tokens: where those are few, CTAs go on coming, 512 KB each, which the SMs take as they get through (32 tokens, 128000 x 4096 fp32 of a
// table: 412 us with 216 CTAs, 352 with 286, 310 with 4000; one token, 8192 x 4096: 142 with 16, 29 with 256; 131072 tokens, 50257 x 768: 189 with 99,
// 199 with 216).
inline int zero_ctas(int64_t rows, int64_t vocab, int64_t row_bytes, int most) {
    const int64_t few = (vocab + 511) / 512, sure = vocab > rows ? (vocab - rows) * row_bytes : 0, heavy = sure / (128 * 1024);
    int64_t c = few > heavy ? few : heavy;
    if (c > most) c = rows <= 4 * SORT_THREADS && sure / (512 * 1024) > most ? sure / (512 * 1024) : most;
    return (int)(c < 65536 ? c : 65536);
}
inline size_t sort_smem(int bits) {
    const size_t sort = ((size_t)SORT_WARPS + 1) * ((size_t)1 << bits) * 4 + SORT_WARPS * 4;
    return sort > WORDS * 4 ? sort : WORDS * 4;
}

}  // namespace embed
}  // namespace sa2
