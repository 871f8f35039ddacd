// Distillation from a teacher's largest logits: loss and gradient of the student's logits.
//
//   q = softmax(z / T) over the vocabulary,  p = softmax(t / T) over the teacher's K entries of the row
//   loss_r = T^2 sum_k p_k (log p_k - log q_{i_k}),   dz_j = g T (q_j - sum of p_k over the k with i_k == j)
// Entries with an index outside [0, vocab) are not there, whatever their logit; a row without entries, or whose entries are all -inf, has
// no loss and a gradient of zero, and does not count in the mean.  Entries that name one token twice add up.
//
// teacher_kernel turns the entries into places and probabilities, a warp a row; all others go over rows of z.  Bound: reading z (forward) and
// reading z and writing dz (backward) once.  The forward keeps the running maximum of what a thread has seen and the sum of exponentials
// against it; per element a subtraction, a product, ex2 and an addition, which 16 ex2 per clock and SM allow at the rate the loads
// come.  Sums over a row are fp32 and have one order; the row's K terms, and the sum over rows, are 64 bits: they are few, and
// log p - log q cancels where the student is good.
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
    int *place;                 // [rows][k]: -1 where an entry is not there or has no mass
    float *prob;                // [rows][k]
    float *self;                // [rows]: sum of p log p
    int *there;                 // [rows]: whether the row counts
    int *counts;                // rows that count, of every TEACHER_ROWS
    float *stats;               // [rows][2]: maximum of z, sum of exp((z - maximum) / T)
    float *row_loss;            // [rows]
    void *dz;                   // [rows][vocab], row stride ds
    const float *gout;          // gradient of the loss: one, or one for each row (gs = 1); null: 1
    float *scale;               // two factors more: 1 / rows that count (or null), and one of the caller
    float times;
    int64_t rows, zs, ts, is, ds;
    int vocab, k, gs;
    int index64, teacher_bf16;
    float t;                    // temperature
    int mean;                   // both_kernel: the gradient is divided by the rows that count
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^(d log2(e) / T): the factor in two parts for fp32 logits, whose gradients show the rounding of one
struct Factor { float hi, lo; };
__device__ __forceinline__ Factor factor(float t) {
    const double c = 1.4426950408889634 / (double)t;
    Factor f;
    f.hi = (float)c;
    f.lo = (float)(c - (double)f.hi);
    return f;
}
template <typename T> __device__ __forceinline__ float weight(float d, const Factor &f) {
    if constexpr (sizeof(T) == 4) {
        const float y = d * f.hi;                        // (far below, the second part may overflow)
        return ex2(y < -200.f ? y : fmaf(d, f.hi, d * f.lo));
    }
    else return ex2(d * f.hi);
}

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

// Calls f(first element, number, values) for all of a row: pieces of eight from the first 16-byte boundary on, U loads at a time (half as many
// of fp32), single elements around them.
template <int G, typename T, int U, typename F> __device__ __forceinline__ void for_row(const T *row, int vocab, F f) {
    constexpr int V = sizeof(T) == 2 ? U : U / 2;
    const int rank = Group<G>::rank();
    int head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    if (head > vocab) head = vocab;
    const int pieces = (vocab - head) / 8;
    for (int x = rank; x < head; x += G) {
        float v[8] = {(float)row[x]};
        f(x, 1, v);
    }
    const T *from = row + head;
    for (int x0 = rank; x0 < pieces; x0 += V * G) {
        Packed<T> t[V];
#pragma unroll
        for (int u = 0; u < V; ++u)
            if (x0 + u * G < pieces) t[u].load(from + (x0 + u * G) * 8);
#pragma unroll
        for (int u = 0; u < V; ++u)
            if (x0 + u * G < pieces) {
                float v[8];
                t[u].get(v);
                f(head + (x0 + u * G) * 8, 8, v);
            }
    }
    for (int x = head + pieces * 8 + rank; x < vocab; x += G) {
        float v[8] = {(float)row[x]};
        f(x, 1, v);
    }
}

__device__ __forceinline__ int64_t index_at(const Params &P, int64_t r, int k) {
    const int64_t i = P.index64 ? reinterpret_cast<const int64_t *>(P.index)[r * P.is + k] : (int64_t)reinterpret_cast<const int32_t *>(P.index)[r * P.is + k];
    return i >= 0 && i < P.vocab ? i : -1;
}
__device__ __forceinline__ double teacher_at(const Params &P, int64_t r, int k) {
    return P.teacher_bf16 ? (double)__bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(P.teacher)[r * P.ts + k])
                          : (double)reinterpret_cast<const float *>(P.teacher)[r * P.ts + k];
}

// A warp a row.
__global__ void __launch_bounds__(32 * TEACHER_ROWS) teacher_kernel(const __grid_constant__ Params P) {
    const int lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * TEACHER_ROWS + (threadIdx.x >> 5);
    auto sum = [](double a, double b) { return a + b; };
    auto larger = [](double a, double b) { return fmax(a, b); };
    bool counted = false;
    if (r < P.rows) {
        double best = -CUDART_INF;
        bool any = false;
        for (int k = lane; k < P.k; k += 32)
            if (index_at(P, r, k) >= 0) {
                const double t = teacher_at(P, r, k);
                any |= t != -CUDART_INF;
                best = fmax(best, t);
            }
        counted = __any_sync(0xffffffffu, any);
        best = Group<32>::reduce(best, (double *)nullptr, larger);
        const double inv_t = 1. / (double)P.t;
        double mass = 0.;
        for (int k = lane; k < P.k; k += 32)
            if (counted && index_at(P, r, k) >= 0) mass += exp((teacher_at(P, r, k) - best) * inv_t);
        mass = Group<32>::reduce(mass, (double *)nullptr, sum);
        const double log_mass = log(mass);
        double self = 0.;
        for (int k = lane; k < P.k; k += 32) {
            const int64_t i = counted ? index_at(P, r, k) : -1;
            const double y = i >= 0 ? (teacher_at(P, r, k) - best) * inv_t - log_mass : -CUDART_INF, p = exp(y);
            if (p != 0.) self += p * y;
            P.place[r * P.k + k] = p != 0. ? (int)i : -1;
            P.prob[r * P.k + k] = (float)p;
        }
        self = Group<32>::reduce(self, (double *)nullptr, sum);
        if (lane == 0) {
            P.self[r] = (float)self;
            P.there[r] = counted;
        }
    }
    __shared__ int of_warp[TEACHER_ROWS];
    if (lane == 0) of_warp[threadIdx.x >> 5] = counted;
    __syncthreads();
    if (threadIdx.x == 0) {
        int c = 0;
        for (int w = 0; w < TEACHER_ROWS; ++w) c += of_warp[w];
        P.counts[blockIdx.x] = c;
    }
}
// T^2 KL of a row whose z has the maximum `ref` and the sum of exponentials s, over the threads of a group; `scratch`: a value a warp
template <int G, typename T> __device__ __forceinline__ double loss_of(const Params &P, int64_t r, const T *row, float ref, float s, double *scratch) {
    const double log_s = log((double)s), inv_t = 1. / (double)P.t;
    double loss = 0.;
    for (int k = Group<G>::rank(); k < P.k; k += G) {
        const int i = P.place[r * P.k + k];
        if (i >= 0) loss += (double)P.prob[r * P.k + k] * (log_s - ((double)(float)row[i] - (double)ref) * inv_t);
    }
    loss = Group<G>::reduce(loss, scratch, [](double a, double b) { return a + b; });
    return (loss + (double)P.self[r]) * (double)P.t * (double)P.t;
}

// Running maximum and sum of exponentials of what a thread has seen
template <typename T> struct Running {
    float m, s;
    __device__ __forceinline__ Running() : m(-INFINITY), s(0.f) {}
    template <int V> __device__ __forceinline__ void take(const float (&v)[V], const Factor &f) {
        float top = v[0];
#pragma unroll
        for (int z = 1; z < V; ++z) top = fmaxf(top, v[z]);
        if (top > m) {
            s *= m == -CUDART_INF_F ? 0.f : weight<T>(m - top, f);
            m = top;
        }
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        float e = weight<T>(v[0] - ref, f);
#pragma unroll
        for (int z = 1; z < V; ++z) e += weight<T>(v[z] - ref, f);
        s += e;
    }
};

// Maximum and sum against it of all threads of a group, with one wait; -inf and 0 for a row of -inf alone
template <int G, typename T> __device__ __forceinline__ float2 joined(float2 all, float2 *of_warp, const Factor &f) {
    auto join = [&](float2 a, float2 b) {
        const float m = fmaxf(a.x, b.x);
        if (m == -CUDART_INF_F) return make_float2(m, a.y + b.y);
        // (without a maximum the sum is 0, or NaN)
        return make_float2(m, (a.x == -CUDART_INF_F ? a.y : a.y * weight<T>(a.x - m, f)) + (b.x == -CUDART_INF_F ? b.y : b.y * weight<T>(b.x - m, f)));
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = join(all, make_float2(__shfl_xor_sync(0xffffffffu, all.x, o), __shfl_xor_sync(0xffffffffu, all.y, o)));
    if constexpr (G > 32) {
        constexpr int WARPS = G / 32;
        if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = all;
        __syncthreads();
        all = of_warp[threadIdx.x % WARPS];
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) all = join(all, make_float2(__shfl_xor_sync(0xffffffffu, all.x, o), __shfl_xor_sync(0xffffffffu, all.y, o)));
    }
    return all;
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
    const Factor f = factor(P.t);
    Running<T> run;
    for_row<G, T, 4>(row, P.vocab, [&](int, int count, float (&v)[8]) {
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
    const float2 all = joined<G, T>(make_float2(run.m, run.s), of_warp, f);
    const float ref = all.x == -CUDART_INF_F ? 0.f : all.x, s = all.y;
    const double loss = loss_of<G, T>(P, r, row, ref, s, scratch);
    if (Group<G>::rank() == 0) {
        P.stats[2 * r] = ref;
        P.stats[2 * r + 1] = s;
        P.row_loss[r] = (float)loss;
    }
}

// Loss and gradient: a CTA reads its row twice, the second time from L2, where the rows of all CTAs together have room (two CTAs an SM, 76 MB at
// 128000 bf16 logits); gradients are stored so that they leave L2 first.  (Rows in the shared memory of clusters of four and eight CTAs,
// read once: 576 us for 4096 rows of 128000, and 1080 with the next row on its way meanwhile; the waits for the cluster and for its eight
// places in one GPC cost more than the second read.)
template <typename T, int G>
__global__ void __launch_bounds__(G, 1024 / G) both_kernel(const __grid_constant__ Params P) {
    __shared__ float2 of_warp[G / 32];
    __shared__ int counted[G / 32];
    extern __shared__ __align__(16) char shared[];
    const int64_t r = blockIdx.x;
    const T *row = reinterpret_cast<const T *>(P.z) + r * P.zs;
    T *grad = reinterpret_cast<T *>(P.dz) + r * P.ds;
    int *place = reinterpret_cast<int *>(shared);
    float *prob = reinterpret_cast<float *>(place + P.k);
    const Factor f = factor(P.t);
    Running<T> run;
    for_row<G, T, 8>(row, P.vocab, [&](int, int count, float (&v)[8]) {
        if (count == 8) {
            run.take(v, f);
        } else {
            const float one[1] = {v[0]};
            run.take(one, f);
        }
    });
    const bool there = P.there[r];
    if (P.mean) {                                        // rows that count
        int rows = 0;
        for (int64_t x = threadIdx.x; x < (P.rows + TEACHER_ROWS - 1) / TEACHER_ROWS; x += G) rows += P.counts[x];
        rows = __reduce_add_sync(0xffffffffu, rows);
        if (threadIdx.x % 32 == 0) counted[threadIdx.x / 32] = rows;
    }
    for (int k = threadIdx.x; k < P.k; k += G) {
        place[k] = P.place[r * P.k + k];
        prob[k] = P.prob[r * P.k + k];
    }
    const float2 all = joined<G, T>(make_float2(run.m, run.s), of_warp, f);
    const float ref = all.x == -CUDART_INF_F ? 0.f : all.x, s = all.y;
    int rows = P.mean ? 0 : 1;
    for (int w = 0; P.mean && w < G / 32; ++w) rows += counted[w];
    const float coef = (float)(1. / (double)max(rows, 1)) * P.times * P.t, inv = 1.f / s;
    const bool together = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    for_row<G, T, 8>(row, P.vocab, [&](int x, int count, float (&v)[8]) {
        if (count == 8) {
#pragma unroll
            for (int z = 0; z < 8; ++z) v[z] = there ? coef * (weight<T>(v[z] - ref, f) * inv) : 0.f;
            if (together) {
                store8_once<T>(grad + x, v);
            } else {
#pragma unroll
                for (int z = 0; z < 8; ++z) grad[x + z] = (T)v[z];
            }
        } else {
            grad[x] = (T)(there ? coef * (weight<T>(v[0] - ref, f) * inv) : 0.f);
        }
    });
    __syncthreads();
    // the teacher's tokens, entries of one token store the same value; the loss meanwhile
    if (threadIdx.x >= 32) {
        for (int k = threadIdx.x - 32; there && k < P.k; k += G - 32) {
            const int i = place[k];
            if (i < 0) continue;
            float p = 0.f;
            for (int o = 0; o < P.k; ++o) p += place[o] == i ? prob[o] : 0.f;
            grad[i] = (T)(coef * (weight<T>((float)row[i] - ref, f) * inv - p));
        }
    } else {
        const double loss = there ? loss_of<32, T>(P, r, row, ref, s, nullptr) : 0.;
        if (threadIdx.x == 0) P.row_loss[r] = (float)loss;
    }
}

// out: sum of the rows' losses, over the rows that count if `mean`; factor: of the gradient that goes with it
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
        const double by = mean ? 1. / (double)(c > 0 ? c : 1) : 1.;
        *out = (float)(s * by);
        *factor = (float)by;
    }
}

template <typename T, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G, G == 32 ? 4 : 1536 / G) bwd_kernel(const __grid_constant__ Params P) {
    extern __shared__ __align__(16) char shared[];
    const int64_t r = G == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= P.rows) return;
    int *place = reinterpret_cast<int *>(shared) + (G == 32 ? (threadIdx.x >> 5) * 2 * P.k : 0);
    float *prob = reinterpret_cast<float *>(place + P.k);
    const T *row = reinterpret_cast<const T *>(P.z) + r * P.zs;
    T *grad = reinterpret_cast<T *>(P.dz) + r * P.ds;
    const bool there = P.there[r];
    const float coef = there ? (P.gout ? P.gout[r * P.gs] : 1.f) * (P.scale ? P.scale[0] : 1.f) * P.times * P.t : 0.f;
    const float ref = there ? P.stats[2 * r] : 0.f, inv = there ? 1.f / P.stats[2 * r + 1] : 0.f;
    const Factor f = factor(P.t);
    for (int k = Group<G>::rank(); k < P.k; k += G) {
        place[k] = there ? P.place[r * P.k + k] : -1;
        prob[k] = P.prob[r * P.k + k];
    }
    const bool together = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    for_row<G, T, 4>(row, P.vocab, [&](int x, int count, float (&v)[8]) {
        if (count == 8) {
#pragma unroll
            for (int z = 0; z < 8; ++z) v[z] = there ? coef * (weight<T>(v[z] - ref, f) * inv) : 0.f;
            if (together) {
                store8<T>(grad + x, v);
            } else {
#pragma unroll
                for (int z = 0; z < 8; ++z) grad[x + z] = (T)v[z];
            }
        } else {
            grad[x] = (T)(there ? coef * (weight<T>(v[0] - ref, f) * inv) : 0.f);
        }
    });
    Group<G>::sync();
    // the teacher's tokens; entries of one token store the same value
    for (int k = Group<G>::rank(); k < P.k; k += G) {
        const int i = place[k];
        if (i < 0) continue;
        float p = 0.f;
        for (int o = 0; o < P.k; ++o) p += place[o] == i ? prob[o] : 0.f;
        grad[i] = (T)(coef * (weight<T>((float)row[i] - ref, f) * inv - p));
    }
}

// scratch of a call, which the backward reads again
inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int64_t teacher_blocks(int64_t rows) { return (rows + TEACHER_ROWS - 1) / TEACHER_ROWS; }
inline size_t workspace_bytes(int64_t rows, int k) {
    return 2 * up256((size_t)rows * k * 4) + 3 * up256((size_t)rows * 4) + up256((size_t)rows * 8) + up256((size_t)teacher_blocks(rows) * 4) + 256;
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
    P.self = reinterpret_cast<float *>(take((size_t)P.rows * 4));
    P.there = reinterpret_cast<int *>(take((size_t)P.rows * 4));
    P.stats = reinterpret_cast<float *>(take((size_t)P.rows * 8));
    P.counts = reinterpret_cast<int *>(take((size_t)teacher_blocks(P.rows) * 4));
    P.row_loss = reinterpret_cast<float *>(take((size_t)P.rows * 4));
    P.scale = reinterpret_cast<float *>(take(4));
}

}  // namespace distill
}  // namespace sa2
