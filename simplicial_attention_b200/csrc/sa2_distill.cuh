// Distillation from a teacher's largest logits: loss and gradient of the student's logits.
//
//   q = softmax(z / T) over the vocabulary,  p = softmax(t / T) over the teacher's K entries of the row
//   loss_r = T^2 sum_k p_k (log p_k - log q_{i_k}),   dz_j = g T (q_j - sum of p_k over the k with i_k == j)
// Entries with an index outside [0, vocab) are not there, whatever their logit; a row without entries, or whose entries are all -inf, has
// no loss and a gradient of zero, and does not count in the mean.  Entries that name one token twice add up.
//
// teacher_kernel turns the entries into places and probabilities, a warp a row; all others go over rows of z.  Bound: reading z (forward) and
// reading z and writing dz (backward) once.  The forward keeps the running maximum of what a thread has seen and the sum of exponentials
// against it; per bf16 logit a fused product, ex2 and an addition, which 16 ex2 per clock and SM allow at the rate the loads come.  4095
// rows of 32000 fp32 logits: forward 100 us (5.2 TB/s), backward 163 (6.4 TB/s, a copy's rate); 16384 rows of 256: 18 the teacher, 12, 9.
// A row's sum s of exponentials is fp32 and has one order.  The rest of its loss is formed in 64 bits, as  sum_k p_k log p_k + log s -
// sum_k p_k (z_k - max) / T:  it is little, and cancels where the student is good.  What is left then is the rounding of s, at most some 2^-21, and that of
// the p_k of the last sum (fp32, 2^-24 each), times T^2.
#pragma once
#include "sa2_common.cuh"
#include "sa2_vec8.cuh"
#include <math_constants.h>

namespace sa2 {
namespace distill {

constexpr int MAX_K = 1024;

constexpr int TEACHER_ROWS = 32;                        // of a CTA of teacher_kernel

struct Params {
    const void *z;              // [rows][vocab], row stride zs
    const void *teacher;        // [rows][k], row stride ts
    const void *index;          // [rows][k], row stride is
    // what teacher_kernel makes of them
    int *place;                 // [rows][k]: -1 where an entry is not there, has no mass, or names the token of an earlier one
    float *prob;                // [rows][k]: of the token
    double *self;               // [rows]: sum of p log p
    int *there;                 // [rows]: whether the row counts
    int *counts;                // rows that count, of every TEACHER_ROWS
    float *stats;               // [rows][2]: maximum of z, sum of exp((z - maximum) / T)
    float *row_loss;            // [rows]
    void *dz;                   // [rows][vocab], row stride ds
    const float *gout;          // gradient of the loss: one, or one for each row (gs = 1); null: 1
    float *scale;               // 1 / rows that count, from total_kernel; -1 while that has not run.  bwd_kernel: null if the loss is no mean
    float times;                // a factor of the caller
    int64_t rows, zs, ts, is, ds;
    int vocab, k, gs;
    int index64, teacher_bf16;
    float t;                    // temperature
    float hi, lo;               // log2(e) / t in two parts
    int mean;                   // both_kernel: the gradient is divided by the rows that count
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^(d log2(e) / T): the factor in two parts for fp32 logits, whose gradients show the rounding of one
struct Factor { float hi, lo; };
__device__ __forceinline__ Factor factor(const Params &P) { return Factor{P.hi, P.lo}; }
template <typename T> __device__ __forceinline__ float weight(float d, const Factor &f) {
    if constexpr (sizeof(T) == 4) {
        const float y = d * f.hi;                        // (far below, the second part may overflow)
        return ex2(y < -200.f ? y : fmaf(d, f.hi, d * f.lo));
    }
    return ex2(d * f.hi);
}
// bf16 logits, below 2^20 in units of the exponent: v hi - c is rounded once, c being m hi rounded, and what c is off by (`off`) is a factor
// of the whole sum: an instruction less for every logit.
template <typename T> struct Reference {
    float m, c, off;
    bool near;
    __device__ __forceinline__ Reference(float best, const Factor &f) : m(best == -INFINITY ? 0.f : best), c(best * f.hi) {
        near = sizeof(T) == 2 && fabsf(c) < 1048576.f;
        off = near ? fmaf(-m, f.hi, c) : 0.f;
    }
    // of a logit, times 2^-off
    template <bool NEAR> __device__ __forceinline__ float weight_of(float v, const Factor &f) const { return NEAR ? ex2(fmaf(v, f.hi, -c)) : weight<T>(v - m, f); }
};

// Eight values that nobody reads soon
template <typename T> __device__ __forceinline__ void store8_once(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        __stcs(reinterpret_cast<float4 *>(p), make_float4(v[0], v[1], v[2], v[3]));
        __stcs(reinterpret_cast<float4 *>(p + 4), make_float4(v[4], v[5], v[6], v[7]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * z], v[2 * z + 1]);
            w[z] = *reinterpret_cast<const uint32_t *>(&t);
        }
        __stcs(reinterpret_cast<uint4 *>(p), make_uint4(w[0], w[1], w[2], w[3]));
    }
}

// A group is a warp or a CTA.
template <int G> struct Group {
    static constexpr int WARPS = G / 32;
    static __device__ __forceinline__ int rank() { return G == 32 ? threadIdx.x & 31 : threadIdx.x; }
    static __device__ __forceinline__ void sync() {
        if constexpr (G == 32) __syncwarp();
        else __syncthreads();
    }
    // all threads of the group, the same result in each; `s` is scratch of one value a warp
    template <typename V, typename F> static __device__ __forceinline__ V reduce(V v, V *s, F f) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        if constexpr (G > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
            __syncthreads();
            v = s[0];
            for (int w = 1; w < WARPS; ++w) v = f(v, s[w]);
        }
        return v;
    }
};

// Calls f(first element, number, values) for all of a row: pieces of eight from the first 16-byte boundary on, U at a time (half as many of fp32),
// single elements around them.  AHEAD: half of the U are loaded while the other half is used (for loss and gradient at once 105 instead of
// 124 us at 8192 rows of 10000 bf16 logits, 187 instead of 204 at 4096 of 50257; the forward alone, with fewer registers, 239 instead of 224 at
// 4096 of 128000).  BACK: from the last piece to the first.
template <int G, typename T, int U, bool AHEAD, bool BACK = false, typename F> __device__ __forceinline__ void for_row(const T *row, int vocab, F f) {
    constexpr int V = (sizeof(T) == 2 ? U : U / 2) / (AHEAD ? 2 : 1);
    const int rank = Group<G>::rank();
    int head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    if (head > vocab) head = vocab;
    const int pieces = (vocab - head) / 8;
    const T *from = row + head;
    auto piece = [&](int x) { return BACK ? pieces - 1 - x : x; };
    auto one = [&](int x) {
        float v[8] = {(float)row[x]};
        f(x, 1, v);
    };
    auto load = [&](Packed<T> (&t)[V], int x0) {
#pragma unroll
        for (int u = 0; u < V; ++u)
            if (x0 + u * G < pieces) t[u].load(from + piece(x0 + u * G) * 8);
    };
    auto use = [&](const Packed<T> (&t)[V], int x0) {
#pragma unroll
        for (int u = 0; u < V; ++u)
            if (x0 + u * G < pieces) {
                float v[8];
                t[u].get(v);
                f(head + piece(x0 + u * G) * 8, 8, v);
            }
    };
    for (int x = rank; x < head; x += G) one(x);
    Packed<T> t[V], next[V];
    if constexpr (AHEAD) {
        load(t, rank);
        for (int x0 = rank; x0 < pieces; x0 += 2 * V * G) {
            load(next, x0 + V * G);
            use(t, x0);
            load(t, x0 + 2 * V * G);
            use(next, x0 + V * G);
        }
    } else {
        for (int x0 = rank; x0 < pieces; x0 += V * G) {
            load(t, x0);
            use(t, x0);
        }
    }
    for (int x = head + pieces * 8 + rank; x < vocab; x += G) one(x);
}

__device__ __forceinline__ int64_t index_at(const Params &P, int64_t r, int k) {
    const int64_t i = P.index64 ? reinterpret_cast<const int64_t *>(P.index)[r * P.is + k] : (int64_t)reinterpret_cast<const int32_t *>(P.index)[r * P.is + k];
    return i >= 0 && i < P.vocab ? i : -1;
}
__device__ __forceinline__ double teacher_at(const Params &P, int64_t r, int k) {
    return P.teacher_bf16 ? (double)__bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(P.teacher)[r * P.ts + k])
                          : (double)reinterpret_cast<const float *>(P.teacher)[r * P.ts + k];
}

// Words of shared memory that a warp of teacher_kernel has: places, and a table of entries by place
inline __host__ __device__ int table_size(int k) {
    int n = 64;
    while (n < 2 * k) n *= 2;
    return n;
}
inline __host__ __device__ int teacher_words(int k) { return k + table_size(k); }
inline int teacher_warps(int k) { return k <= 512 ? 32 : 16; }
constexpr int AGAIN = 1 << 30;                          // flag of a place: another entry has the same (places are below)

// A warp a row.  Entries that name one token become one: its first, with the sum of their probabilities.  A hash table finds them in
// O(k); for those that have one of the same token the warp looks through all.
__global__ void __launch_bounds__(1024) teacher_kernel(const __grid_constant__ Params P) {
    extern __shared__ int words[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, size = table_size(P.k);
    int *place = words + warp * teacher_words(P.k), *table = place + P.k;
    auto sum = [](double a, double b) { return a + b; };
    auto larger = [](double a, double b) { return fmax(a, b); };
    const double inv_t = 1. / (double)P.t;
    const bool warp_of_entries = P.k <= 32;              // an entry a lane needs no table
    int rows = 0;
    for (int q = warp; q < TEACHER_ROWS; q += blockDim.x / 32) {
        const int64_t r = (int64_t)blockIdx.x * TEACHER_ROWS + q;
        if (r >= P.rows) break;
        double best = -CUDART_INF;
        bool any = false;
        for (int k = lane; k < P.k; k += 32)
            if (index_at(P, r, k) >= 0) {
                const double t = teacher_at(P, r, k);
                any |= t != -CUDART_INF;
                best = fmax(best, t);
            }
        const bool counted = __any_sync(0xffffffffu, any);
        best = Group<32>::reduce(best, (double *)nullptr, larger);
        double mass = 0.;
        for (int k = lane; k < P.k; k += 32)
            if (counted && index_at(P, r, k) >= 0) mass += exp((teacher_at(P, r, k) - best) * inv_t);
        mass = Group<32>::reduce(mass, (double *)nullptr, sum);
        const double log_mass = log(mass);
        double self = 0.;
        for (int x = lane; !warp_of_entries && x < size; x += 32) table[x] = -1;
        for (int k = lane; k < P.k; k += 32) {
            const int64_t i = counted ? index_at(P, r, k) : -1;
            const double y = i >= 0 ? (teacher_at(P, r, k) - best) * inv_t - log_mass : -CUDART_INF, p = exp(y);
            if (p != 0.) self += p * y;
            place[k] = p != 0. ? (int)i : -1;
            P.prob[r * P.k + k] = (float)p;
        }
        self = Group<32>::reduce(self, (double *)nullptr, sum);
        __syncwarp();
        if (warp_of_entries) {
            const int i = lane < P.k ? place[lane] : -1;
            if (__popc(__match_any_sync(0xffffffffu, i)) > 1 && i >= 0) place[lane] = i | AGAIN;
        }
        for (int k = lane; !warp_of_entries && k < P.k; k += 32) {
            const int i = place[k] & ~AGAIN;
            if (place[k] < 0) continue;
            // (a slot keeps the entry that came first, and half of the slots stay free)
            for (uint32_t at = (uint32_t)i * 2654435761u >> 16;; ++at) {
                const int other = atomicCAS(table + (at & (size - 1)), -1, k);
                if (other < 0) break;
                if ((place[other] & ~AGAIN) == i) {
                    atomicOr(place + other, AGAIN);
                    atomicOr(place + k, AGAIN);
                    break;
                }
            }
        }
        __syncwarp();
        for (int k0 = 0; k0 < P.k; k0 += 32) {
            const int k = k0 + lane;
            const int flagged = k < P.k ? place[k] : -1;
            int i = flagged < 0 ? -1 : flagged & ~AGAIN;
            for (uint32_t todo = __ballot_sync(0xffffffffu, flagged >= AGAIN); todo; todo &= todo - 1u) {
                const int owner = __ffs(todo) - 1, both = __shfl_sync(0xffffffffu, flagged, owner);
                float all = 0.f;
                int first = P.k;
                for (int o = lane; o < P.k; o += 32)
                    if (place[o] == both) {
                        first = min(first, o);
                        all += P.prob[r * P.k + o];
                    }
                all = Group<32>::reduce(all, (float *)nullptr, [](float a, float b) { return a + b; });
                first = __reduce_min_sync(0xffffffffu, first);
                __syncwarp();                            // (the first of a token comes first, before one of its probabilities changes)
                if (lane == owner) {
                    if (first == k) P.prob[r * P.k + k] = all;
                    else i = -1;
                }
                __syncwarp();
            }
            if (k < P.k) P.place[r * P.k + k] = i;
        }
        __syncwarp();
        if (lane == 0) {
            P.self[r] = self;
            P.there[r] = counted;
        }
        rows += counted;
    }
    __shared__ int of_warp[32];
    if (lane == 0) of_warp[warp] = rows;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < (int)blockDim.x / 32; ++w) rows += of_warp[w];
        P.counts[blockIdx.x] = rows;
        if (blockIdx.x == 0) *P.scale = -1.f;
    }
}
// An entry's part of the last sum of a row's loss; -inf for a token that the student rules out, also where the probability is 0 in fp32
__device__ __forceinline__ double term(float prob, float logit, float best, double inv_t) {
    const double x = ((double)logit - (double)best) * inv_t;
    return x == -CUDART_INF ? x : (double)prob * x;
}
__device__ __forceinline__ float row_loss(double self, double log_s, double terms, float t) { return (float)((self + log_s - terms) * (double)t * (double)t); }

// Running maximum and sum of exponentials of what a thread has seen
template <typename T> struct Running {
    float s;
    Reference<T> ref;
    float m;
    __device__ __forceinline__ Running(const Factor &f) : s(0.f), ref(0.f, f), m(-INFINITY) { ref.near = false; }
    template <int V> __device__ __forceinline__ void take(const float (&v)[V], const Factor &f) {
        float top = v[0];
#pragma unroll
        for (int z = 1; z < V; ++z) top = fmaxf(top, v[z]);
        if (top > m) {
            const Reference<T> next(top, f);
            s *= sizeof(T) == 4 ? weight<T>(m - top, f) : ex2((m - top) * f.hi + (ref.off - next.off));
            m = top;
            ref = next;
        }
        float e;
        if (ref.near) {
            e = ref.template weight_of<true>(v[0], f);
#pragma unroll
            for (int z = 1; z < V; ++z) e += ref.template weight_of<true>(v[z], f);
        } else {
            e = ref.template weight_of<false>(v[0], f);
#pragma unroll
            for (int z = 1; z < V; ++z) e += ref.template weight_of<false>(v[z], f);
        }
        s += e;
    }
    // the sum against 2^(m log2(e) / T)
    __device__ __forceinline__ float2 result() const { return make_float2(m, sizeof(T) == 4 ? s : s * ex2(ref.off)); }
};

// Maximum and sum against it of all threads of a group, with one wait; -inf and 0 (or NaN) for a row of -inf alone (or NaN)
template <int G, typename T> __device__ __forceinline__ float2 joined(float2 all, float2 *of_warp, const Factor &f) {
    auto join = [&](int lanes) {
        float m = all.x;
#pragma unroll
        for (int o = lanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float s = all.x == m ? all.y : all.y * weight<T>(all.x - m, f);
#pragma unroll
        for (int o = lanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        all = make_float2(m, s);
    };
    join(32);
    if constexpr (G > 32) {
        constexpr int WARPS = G / 32;
        if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = all;
        __syncthreads();
        all = of_warp[threadIdx.x % WARPS];
        join(WARPS);
    }
    return all;
}

// The gradient of a row but for the teacher's part: g 2^((z - best) log2(e) / T), or zeros.  First what few rows need (a function of its own,
// whose registers the other does not have to find room for).
template <int G, typename T> __device__ __noinline__ void gradient_anyhow(const T *row, T *grad, int vocab, bool there, float best, float g, Factor f) {
    for (int x = Group<G>::rank(); x < vocab; x += G) grad[x] = (T)(there ? g * weight<T>((float)row[x] - best, f) : 0.f);
}
template <int G, typename T, int U, bool ONCE> __device__ __forceinline__ void gradient(const T *row, T *grad, int vocab, bool there, float best, float g, const Factor &f) {
    const bool together = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    const Reference<T> ref(best, f);
    if (!there || !together || (sizeof(T) == 2 && !ref.near)) {
        gradient_anyhow<G, T>(row, grad, vocab, there, best, g, f);
        return;
    }
    if (sizeof(T) == 2) g *= ex2(ref.off);
    for_row<G, T, U, true, ONCE>(row, vocab, [&](int x, int count, float (&v)[8]) {
#pragma unroll
        for (int z = 0; z < 8; ++z) v[z] = g * ref.template weight_of<sizeof(T) == 2>(v[z], f);
        if (count != 8) {
            grad[x] = (T)v[0];
        } else if constexpr (ONCE) {
            store8_once<T>(grad + x, v);
        } else {
            store8<T>(grad + x, v);
        }
    });
}

// Rows of any alignment.
template <typename T, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G, G == 32 ? 4 : 1536 / G) fwd_kernel(const __grid_constant__ Params P) {
    __shared__ double scratch[G == 32 ? 1 : G / 32];
    __shared__ float2 of_warp[G == 32 ? 1 : G / 32];
    const int64_t r = G == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= P.rows) return;
    const T *row = reinterpret_cast<const T *>(P.z) + r * P.zs;
    const bool there = P.there[r];                       // (looked at behind the row, whose loads do not wait for it)
    const Factor f = factor(P);
    Running<T> run(f);
    for_row<G, T, 4, false>(row, P.vocab, [&](int, int count, float (&v)[8]) {
        if (count == 8) {
            run.take(v, f);
        } else {
            const float one[1] = {v[0]};
            run.take(one, f);
        }
    });
    if (!there) {
        if (Group<G>::rank() == 0) P.row_loss[r] = 0.f;
        return;
    }
    const float2 all = joined<G, T>(run.result(), of_warp, f);
    const float best = all.x == -CUDART_INF_F ? 0.f : all.x, s = all.y;
    const double log_s = log((double)s), inv_t = 1. / (double)P.t;       // (the logarithm here: behind the sum over warps it made registers spill)
    double terms = 0.;
    for (int k = Group<G>::rank(); k < P.k; k += G) {
        const int i = P.place[r * P.k + k];
        if (i >= 0) terms += term(P.prob[r * P.k + k], (float)row[i], best, inv_t);
    }
    terms = Group<G>::reduce(terms, scratch, [](double a, double b) { return a + b; });
    if (Group<G>::rank() == 0) {
        P.stats[2 * r] = best;
        P.stats[2 * r + 1] = s;
        P.row_loss[r] = row_loss(P.self[r], log_s, terms, P.t);
    }
}

// Loss and gradient: a CTA reads its row twice, the second time from the end to the beginning and from L2, which holds most of the rows of all
// CTAs together (two CTAs of 512 threads an SM, 76 MB at 128000 bf16 logits; in one direction every second read missed it); gradients are stored
// so that they leave L2 first.  4096 such rows: 430 us (450 in one direction), 325 at the rate of a copy; ex2, twice a logit, would take 230 us
// alone.  Slower: rows in the shared memory of clusters of four and eight CTAs, read once (576 us; 1080 with the next row on its way
// meanwhile: waits for the cluster, and for its places in one GPC); two CTAs a row (524); 104 KB of each row kept in shared memory by the threads
// that read it (519, with 484 without at that time).
template <typename T, int G>
__global__ void __launch_bounds__(G, 1024 / G) both_kernel(const __grid_constant__ Params P) {
    __shared__ float2 of_warp[G / 32];
    __shared__ int counted[G / 32];
    __shared__ double terms_of[G / 32];
    const int warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x;
    const T *row = reinterpret_cast<const T *>(P.z) + r * P.zs;
    T *grad = reinterpret_cast<T *>(P.dz) + r * P.ds;
    // on their way while the row is read: an entry of each thread, whether the row counts, and how many do
    const bool there = P.there[r];
    int place = -1, rows = 0;
    float prob = 0.f, logit = 0.f;
    if (threadIdx.x < P.k) {
        place = P.place[r * P.k + threadIdx.x];
        prob = P.prob[r * P.k + threadIdx.x];
    }
    if (P.mean)
        for (int64_t x = threadIdx.x; x < (P.rows + TEACHER_ROWS - 1) / TEACHER_ROWS; x += G) rows += P.counts[x];
    const Factor f = factor(P);
    Running<T> run(f);
    for_row<G, T, 8, true>(row, P.vocab, [&](int, int count, float (&v)[8]) {
        if (count == 8) {
            run.take(v, f);
        } else {
            const float one[1] = {v[0]};
            run.take(one, f);
        }
    });
    if (place >= 0) logit = (float)row[place];
    if (P.mean) {
        rows = __reduce_add_sync(0xffffffffu, rows);
        if (threadIdx.x % 32 == 0) counted[warp] = rows;
    }
    const float2 all = joined<G, T>(run.result(), of_warp, f);
    const float best = all.x == -CUDART_INF_F ? 0.f : all.x, s = all.y;
    rows = P.mean ? 0 : 1;
    for (int w = 0; P.mean && w < G / 32; ++w) rows += counted[w];
    const float coef = 1.f / (float)max(rows, 1) * P.times * P.t, inv = 1.f / s;
    gradient<G, T, 8, true>(row, grad, P.vocab, there, best, coef * inv, f);
    __syncthreads();
    // the teacher's tokens and the loss
    const bool on = there && warp * 32 < P.k;
    if (on) {
        const double inv_t = 1. / (double)P.t;
        double terms = 0.;
        for (int k = threadIdx.x; k < P.k; k += G) {
            if (k >= G) {
                place = P.place[r * P.k + k];
                prob = P.prob[r * P.k + k];
                if (place >= 0) logit = (float)row[place];
            }
            if (place < 0) continue;
            grad[place] = (T)(coef * (weight<T>(logit - best, f) * inv - prob));
            terms += term(prob, logit, best, inv_t);
        }
        terms = Group<32>::reduce(terms, (double *)nullptr, [](double a, double b) { return a + b; });
        if (threadIdx.x % 32 == 0) terms_of[warp] = terms;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double terms = 0.;
        for (int w = 0; there && w < G / 32 && w * 32 < P.k; ++w) terms += terms_of[w];
        P.row_loss[r] = there ? row_loss(P.self[r], log((double)s), terms, P.t) : 0.f;
    }
}

// out: sum of the rows' losses, over the rows that count if `mean`; factor: 1 / these rows, for the gradient of a mean
__global__ void __launch_bounds__(1024) total_kernel(const float *row_loss, const int *counts, int64_t rows, int mean, float *out, float *factor) {
    __shared__ double sums[32];
    __shared__ long long count_of[32];
    double s = 0.;
    long long c = 0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) s += (double)row_loss[r];
    for (int64_t x = threadIdx.x; x < (rows + TEACHER_ROWS - 1) / TEACHER_ROWS; x += 1024) c += counts[x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if ((threadIdx.x & 31) == 0) {
        sums[threadIdx.x >> 5] = s;
        count_of[threadIdx.x >> 5] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) {
            s += sums[w];
            c += count_of[w];
        }
        *out = (float)(mean ? s / (double)(c > 0 ? c : 1) : s);
        *factor = 1.f / (float)(c > 0 ? c : 1);
    }
}

// 1 / rows that count, in each lane of a warp: for a backward whose forward was not asked for their total
__device__ __noinline__ float count_again(const int *counts, int64_t rows) {
    long long c = 0;
    for (int64_t x = threadIdx.x & 31; x < (rows + TEACHER_ROWS - 1) / TEACHER_ROWS; x += 32) c += counts[x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    return 1.f / (float)(c > 0 ? c : 1);
}

template <typename T, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G, G == 32 ? 4 : 1536 / G) bwd_kernel(const __grid_constant__ Params P) {
    const int64_t r = G == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= P.rows) return;
    const T *row = reinterpret_cast<const T *>(P.z) + r * P.zs;
    T *grad = reinterpret_cast<T *>(P.dz) + r * P.ds;
    const bool there = P.there[r];
    float part = P.scale ? *P.scale : 1.f;
    if (part < 0.f) part = count_again(P.counts, P.rows);
    const float coef = there ? (P.gout ? P.gout[r * P.gs] : 1.f) * part * P.times * P.t : 0.f;
    const float best = there ? P.stats[2 * r] : 0.f, inv = there ? 1.f / P.stats[2 * r + 1] : 0.f;
    const Factor f = factor(P);
    gradient<G, T, 4, false>(row, grad, P.vocab, there, best, coef * inv, f);
    Group<G>::sync();
    for (int k = Group<G>::rank(); there && k < P.k; k += G) {
        const int i = P.place[r * P.k + k];
        if (i >= 0) grad[i] = (T)(coef * (weight<T>((float)row[i] - best, f) * inv - P.prob[r * P.k + k]));
    }
}

// scratch of a call, which the backward reads again
inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int64_t teacher_blocks(int64_t rows) { return (rows + TEACHER_ROWS - 1) / TEACHER_ROWS; }
inline size_t workspace_bytes(int64_t rows, int k) {
    return 2 * up256((size_t)rows * k * 4) + 2 * up256((size_t)rows * 4) + 2 * up256((size_t)rows * 8) + up256((size_t)teacher_blocks(rows) * 4) + 256;
}
inline void carve(Params &P, void *workspace) {
    char *p = reinterpret_cast<char *>(workspace);
    auto take = [&](size_t bytes) {
        char *at = p;
        p += up256(bytes);
        return at;
    };
    P.place = reinterpret_cast<int *>(take((size_t)P.rows * P.k * 4));
    P.prob = reinterpret_cast<float *>(take((size_t)P.rows * P.k * 4));
    P.self = reinterpret_cast<double *>(take((size_t)P.rows * 8));
    P.there = reinterpret_cast<int *>(take((size_t)P.rows * 4));
    P.stats = reinterpret_cast<float *>(take((size_t)P.rows * 8));
    P.counts = reinterpret_cast<int *>(take((size_t)teacher_blocks(P.rows) * 4));
    P.row_loss = reinterpret_cast<float *>(take((size_t)P.rows * 4));
    P.scale = reinterpret_cast<float *>(take(4));
}

}  // namespace distill
}  // namespace sa2
