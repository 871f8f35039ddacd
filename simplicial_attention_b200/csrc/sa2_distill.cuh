// Distillation from a teacher's largest logits: loss and gradient of the student's logits.
//
//   q = softmax(z / T) over the vocabulary,  p = softmax(t / T) over the teacher's K entries of the row
//   loss_r = T^2 sum_k p_k (log p_k - log q_{i_k}),   dz_j = g T (q_j - sum of p_k over the k with i_k == j)
// Entries with an index outside [0, vocab) are not there, whatever their logit; a row without entries, or whose entries are all -inf, has
// no loss and a gradient of zero, and does not count in the mean.  Entries that name one token twice add up.
//
// Bound: reading z (forward) and reading z and writing dz (backward) once.  The forward keeps the running maximum of what a thread
// has seen and the sum of exponentials against it; per element a subtraction, a product, ex2 and an addition, which 16 ex2 per clock and SM
// allow at the rate the loads come.  A row is a CTA's, or a warp's where rows are short.  Sums over a row are fp32 and have one order;
// the row's K terms, and the sum over rows, are 64 bits: they are few, and log p - log q cancels where the student is good.
#pragma once
#include "sa2_common.cuh"
#include "sa2_vec8.cuh"
#include <math_constants.h>

namespace sa2 {
namespace distill {

constexpr int MAX_K = 1024;

struct Params {
    const void *z;              // [rows][vocab], row stride zs
    const void *teacher;        // [rows][k], row stride ts
    const void *index;          // [rows][k], row stride is
    float *stats;               // [rows][2]: maximum of z, sum of exp((z - maximum) / T)
    float *row_loss;            // [rows]
    int *counted;               // [rows]
    void *dz;                   // [rows][vocab], row stride ds
    const float *gout;          // gradient of the loss: one, or one for each row (gs = 1); null: 1
    const float *scale;         // two factors more: 1 / rows that count (or null), and one of the caller
    float times;
    int64_t rows, zs, ts, is, ds;
    int vocab, k, gs;
    int index64, teacher_bf16;
    float t;                    // temperature
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
    if constexpr (sizeof(T) == 4) return ex2(d == -CUDART_INF_F ? d : fmaf(d, f.hi, d * f.lo));
    else return ex2(d * f.hi);
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

// Calls f(first element, number, values) for all of a row: pieces of eight from the first 16-byte boundary on, single elements around them.
template <int G, typename T, int U, typename F> __device__ __forceinline__ void for_row(const T *row, int vocab, F f) {
    const int rank = Group<G>::rank();
    int head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    if (head > vocab) head = vocab;
    const int pieces = (vocab - head) / 8;
    for (int x = rank; x < head; x += G) {
        float v[8] = {(float)row[x]};
        f(x, 1, v);
    }
    for (int x0 = rank; x0 < pieces; x0 += U * G) {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (x0 + u * G < pieces) load8<T>(row + head + (int64_t)(x0 + u * G) * 8, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (x0 + u * G < pieces) f(head + (x0 + u * G) * 8, 8, v[u]);
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

// Maximum and sum of exponentials of the teacher's entries.  Whether there are any.
template <int G> __device__ __forceinline__ bool teacher_stats(const Params &P, int64_t r, double *s, double &best, double &mass) {
    double m = -CUDART_INF;
    int any = 0;
    for (int k = Group<G>::rank(); k < P.k; k += G)
        if (index_at(P, r, k) >= 0) {
            const double t = teacher_at(P, r, k);
            any |= t != -CUDART_INF;
            m = fmax(m, t);
        }
    best = Group<G>::reduce(m, s, [](double a, double b) { return fmax(a, b); });
    const double there = Group<G>::reduce((double)any, s, [](double a, double b) { return fmax(a, b); });
    double e = 0.;
    for (int k = Group<G>::rank(); k < P.k; k += G)
        if (index_at(P, r, k) >= 0) e += exp((teacher_at(P, r, k) - best) / (double)P.t);
    mass = Group<G>::reduce(e, s, [](double a, double b) { return a + b; });
    return there != 0.;
}

template <typename T, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G) fwd_kernel(const __grid_constant__ Params P) {
    __shared__ double scratch[G == 32 ? 1 : G / 32];
    const int64_t r = G == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= P.rows) return;
    const T *row = reinterpret_cast<const T *>(P.z) + r * P.zs;
    double best, mass;
    const bool there = teacher_stats<G>(P, r, scratch, best, mass);
    if (!there) {
        if (Group<G>::rank() == 0) {
            P.stats[2 * r] = 0.f;
            P.stats[2 * r + 1] = 1.f;
            P.row_loss[r] = 0.f;
            P.counted[r] = 0;
        }
        return;
    }
    const Factor f = factor(P.t);
    float m = -CUDART_INF_F, s = 0.f;
    for_row<G, T, 4>(row, P.vocab, [&](int, int count, float (&v)[8]) {
        float top = v[0];
        if (count == 8) {
#pragma unroll
            for (int z = 1; z < 8; ++z) top = fmaxf(top, v[z]);
        }
        if (top > m) {
            s *= m == -CUDART_INF_F ? 0.f : weight<T>(m - top, f);
            m = top;
        }
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        float e = weight<T>(v[0] - ref, f);
        if (count == 8) {
#pragma unroll
            for (int z = 1; z < 8; ++z) e += weight<T>(v[z] - ref, f);
        }
        s += e;
    });
    float *fs = reinterpret_cast<float *>(scratch);
    const float top = Group<G>::reduce(m, fs, [](float a, float b) { return fmaxf(a, b); });
    const float ref = top == -CUDART_INF_F ? 0.f : top;
    s = Group<G>::reduce(m == -CUDART_INF_F ? s : s * weight<T>(m - ref, f), fs, [](float a, float b) { return a + b; });
    const double log_s = log((double)s), log_mass = log(mass), inv_t = 1. / (double)P.t;
    double loss = 0.;
    for (int k = Group<G>::rank(); k < P.k; k += G) {
        const int64_t i = index_at(P, r, k);
        if (i < 0) continue;
        const double y = (teacher_at(P, r, k) - best) * inv_t - log_mass, p = exp(y);
        if (p > 0.) loss += p * (y - (((double)(float)row[i] - (double)ref) * inv_t - log_s));
        else if (p != p) loss = p;
    }
    loss = Group<G>::reduce(loss, scratch, [](double a, double b) { return a + b; });
    if (Group<G>::rank() == 0) {
        P.stats[2 * r] = ref;
        P.stats[2 * r + 1] = s;
        P.row_loss[r] = (float)(loss * (double)P.t * (double)P.t);
        P.counted[r] = 1;
    }
}

// out[0]: sum of the rows' losses, over the rows that count if `mean`; out[1]: the factor of the gradient that goes with it
__global__ void __launch_bounds__(1024) total_kernel(const float *row_loss, const int *counted, int64_t rows, int mean, float *out) {
    __shared__ double sums[32];
    __shared__ long long counts[32];
    double s = 0.;
    long long c = 0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) {
        s += (double)row_loss[r];
        c += counted[r];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if ((threadIdx.x & 31) == 0) {
        sums[threadIdx.x >> 5] = s;
        counts[threadIdx.x >> 5] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) {
            s += sums[w];
            c += counts[w];
        }
        const double by = mean ? 1. / (double)(c > 0 ? c : 1) : 1.;
        out[0] = (float)(s * by);
        out[1] = (float)by;
    }
}

template <typename T, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G) bwd_kernel(const __grid_constant__ Params P) {
    __shared__ double scratch[G == 32 ? 1 : G / 32];
    extern __shared__ char shared[];
    const int64_t r = G == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= P.rows) return;
    int *place = reinterpret_cast<int *>(shared) + (G == 32 ? (threadIdx.x >> 5) * 2 * P.k : 0);
    float *prob = reinterpret_cast<float *>(place + P.k);
    const T *row = reinterpret_cast<const T *>(P.z) + r * P.zs;
    T *grad = reinterpret_cast<T *>(P.dz) + r * P.ds;
    double best, mass;
    const bool there = teacher_stats<G>(P, r, scratch, best, mass);
    const float coef = there ? (P.gout ? P.gout[r * P.gs] : 1.f) * (P.scale ? P.scale[0] : 1.f) * P.times * P.t : 0.f;
    const float ref = P.stats[2 * r], inv = 1.f / P.stats[2 * r + 1];
    const Factor f = factor(P.t);
    const double inv_t = 1. / (double)P.t;
    for (int k = Group<G>::rank(); k < P.k; k += G) {
        const int64_t i = index_at(P, r, k);
        place[k] = there ? (int)i : -1;
        prob[k] = place[k] < 0 ? 0.f : (float)(exp((teacher_at(P, r, k) - best) * inv_t) / mass);
    }
    const bool together = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    for_row<G, T, 2>(row, P.vocab, [&](int x, int count, float (&v)[8]) {
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

}  // namespace distill
}  // namespace sa2
