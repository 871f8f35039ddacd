// RMSNorm of every query and key head and the rotation by position behind it, forward and backward, one pass each.
//
//   u = x * rstd * gain,  rstd = rsqrt(mean over the head of x^2 + eps)
//   a pair (u_a, u_b) of the first 2 * pairs channels of a head turns by the angle t = 2 pi * position * f:
//       y_a = u_a cos t - u_b sin t,   y_b = u_b cos t + u_a sin t;   the channels behind them stay
//   backward: e = dy turned back,  dgain = sum over rows and heads of e * x * rstd,
//             dx = rstd * (e gain - x rstd * mean over the head of e gain x rstd)
// Pairs are channels (i, i + pairs), or (2 i, 2 i + 1) if interleaved.
//
// Angles: f comes as a 64-bit fraction of a turn, so that position * f modulo one turn is the low word of an integer
// product - exact for every position.  What is left of the nearest quarter turn is at most 1/8 of a turn, and its sine and
// cosine are good to the last place of fp32, with no table to read and no limit to positions.
//
// Bound: reading and writing every head once.  Each (row, pair) has its sine and cosine once, in shared memory, for all heads
// of the row; a lane holds eight channels of a head (16 bytes of bf16), the lanes of a head add their squares and exchange
// pairs by shuffles.  The backward reads x again and forms rstd again, which costs no traffic of its own; gain gradients stay in
// registers over all rows of a CTA, a CTA writes one partial row and a second kernel adds those in order, without atomics.
#pragma once
#include "sa2_common.cuh"
#include "sa2_vec8.cuh"

namespace sa2 {
namespace rotary {

constexpr int THREADS = 256, PER_THREAD = 4;    // (row, head, eight channels) items that a thread has in flight

struct Side {                   // queries, or keys
    const void *x, *dy;         // [b][n][h][d], element strides below
    int64_t sb, sn, sh, db, dn, dh;
    void *y;                    // forward: y; backward: dx.  [b][n][h][d] contiguous
    const void *gain;           // [d]
};
struct Params {
    Side q, k;
    const int64_t *freqs;       // [pairs], 2^-64 turns per position
    const int64_t *positions;   // element strides pb, pn; null: start + row
    int64_t pb, pn, start;
    float *partial;             // backward: [gridDim.x][2][d]
    int64_t rows;               // b * n, below 2^31
    int n, hq, heads, pairs;    // heads: of queries and keys
    int tile;                   // rows of a CTA at a time
    int interleaved, gain_bf16;
    float eps;
};

// Sum over the D / 8 lanes of a head
template <int D> __device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Cosine and sine of position * f turns: of the nearest quarter turn exactly, of the rest by the library
__device__ __forceinline__ void cos_sin(int64_t position, int64_t f, float &c, float &s) {
    const uint64_t phase = (uint64_t)position * (uint64_t)f;
    const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
    const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));
    float rc, rs;
    sincospif((float)rest * 1.0842021724855044e-19f, &rs, &rc);          // 2^-63: half turns
    c = quarter & 1 ? rs : rc;
    s = quarter & 1 ? rc : rs;
    if (quarter == 1 || quarter == 2) c = -c;
    if (quarter == 2 || quarter == 3) s = -s;
}

// cs: cosines [tile][pairs], behind them the sines, of rows [row0, row0 + count)
__device__ __forceinline__ void fill_angles(const Params &P, float *cs, int64_t row0, int count) {
    for (int x = threadIdx.x; x < count * P.pairs; x += THREADS) {
        const uint32_t row = (uint32_t)row0 + x / P.pairs, b = row / (uint32_t)P.n, i = row - b * (uint32_t)P.n;
        const int64_t position = P.positions ? P.positions[b * P.pb + i * P.pn] : P.start + (int64_t)i;
        cos_sin(position, P.freqs[x % P.pairs], cs[x], cs[P.tile * P.pairs + x]);
    }
}

// Turns the eight channels from c0 on by `sign` times the row's angles (cos, sin: those of the row).
__device__ __forceinline__ void turn(float (&v)[8], int c0, const Params &P, const float *cos, const float *sin, float sign) {
    if (P.interleaved) {
        if (c0 < 2 * P.pairs) {
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const float c = cos[c0 / 2 + z], s = sign * sin[c0 / 2 + z], a = v[2 * z], b = v[2 * z + 1];
                v[2 * z] = fmaf(a, c, -b * s);
                v[2 * z + 1] = fmaf(b, c, a * s);
            }
        }
    } else {
        const int lane = threadIdx.x & 31, step = P.pairs / 8;          // lanes between the two channels of a pair
        const bool first = c0 < P.pairs, on = c0 < 2 * P.pairs;
        const int from = on ? (first ? lane + step : lane - step) : lane;
        const int p0 = on ? (first ? c0 : c0 - P.pairs) : 0;
        const float side = first ? -sign : sign;
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const float other = __shfl_sync(0xffffffffu, v[z], from);
            if (on) v[z] = fmaf(v[z], cos[p0 + z], side * other * sin[p0 + z]);
        }
    }
}

template <int D> __device__ __forceinline__ void load_gain(const Params &P, const void *gain, int c0, float (&g)[8]) {
    if (P.gain_bf16) load8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16 *>(gain) + c0, g);
    else load8<float>(reinterpret_cast<const float *>(gain) + c0, g);
}

// item of a tile: lane of the head, head of the row, row
struct Item { int row, head, c0; bool on; };
template <int D> __device__ __forceinline__ Item item_of(const Params &P, int x, int count) {
    constexpr int LANES = D / 8;
    Item t;
    t.c0 = x % LANES * 8;
    t.row = x / (LANES * P.heads);
    t.head = x / LANES - t.row * P.heads;
    t.on = t.row < count;
    return t;
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS) fwd_kernel(const __grid_constant__ Params P) {
    extern __shared__ float cs[];
    const int64_t row0 = (int64_t)blockIdx.x * P.tile;
    const int count = (int)min((int64_t)P.tile, P.rows - row0), items = count * P.heads * (D / 8);
    for (int base = 0; base < items; base += THREADS * PER_THREAD) {
        float v[PER_THREAD][8];
#pragma unroll
        for (int u = 0; u < PER_THREAD; ++u) {
            const Item t = item_of<D>(P, base + u * THREADS + threadIdx.x, count);
#pragma unroll
            for (int z = 0; z < 8; ++z) v[u][z] = 0.f;
            if (t.on) {
                const uint32_t row = (uint32_t)row0 + t.row, b = row / (uint32_t)P.n, i = row - b * (uint32_t)P.n;
                const bool q = t.head < P.hq;
                const Side &S = q ? P.q : P.k;
                load8<T>(reinterpret_cast<const T *>(S.x) + b * S.sb + i * S.sn + (int64_t)(q ? t.head : t.head - P.hq) * S.sh + t.c0, v[u]);
            }
        }
        if (base == 0) {
            fill_angles(P, cs, row0, count);
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < PER_THREAD; ++u) {
            const Item t = item_of<D>(P, base + u * THREADS + threadIdx.x, count);
            if (!__any_sync(0xffffffffu, t.on)) break;
            float ss = 0.f;
#pragma unroll
            for (int z = 0; z < 8; ++z) ss = fmaf(v[u][z], v[u][z], ss);
            const float rstd = rsqrtf(head_sum<D>(ss) / (float)D + P.eps);
            const bool q = t.head < P.hq;
            const Side &S = q ? P.q : P.k;
            float g[8];
            load_gain<D>(P, S.gain, t.c0, g);
#pragma unroll
            for (int z = 0; z < 8; ++z) v[u][z] = v[u][z] * rstd * g[z];
            const float *cos = cs + (t.on ? t.row : 0) * P.pairs;
            turn(v[u], t.c0, P, cos, cos + P.tile * P.pairs, 1.f);
            if (t.on) {
                const int h = q ? P.hq : P.heads - P.hq, head = q ? t.head : t.head - P.hq;
                store8<T>(reinterpret_cast<T *>(S.y) + ((row0 + t.row) * h + head) * D + t.c0, v[u]);
            }
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS) bwd_kernel(const __grid_constant__ Params P) {
    extern __shared__ float cs[];
    constexpr int LANES = D / 8, U = 2;
    const int c0 = threadIdx.x % LANES * 8;              // a thread has the same channels in every item
    float dq[8], dk[8], gq[8], gk[8];
#pragma unroll
    for (int z = 0; z < 8; ++z) { dq[z] = 0.f; dk[z] = 0.f; }
    load_gain<D>(P, P.q.gain, c0, gq);
    load_gain<D>(P, P.k.gain, c0, gk);
    const int64_t tiles = (P.rows + P.tile - 1) / P.tile;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t row0 = tile * P.tile;
        const int count = (int)min((int64_t)P.tile, P.rows - row0), items = count * P.heads * LANES;
        for (int base = 0; base < items; base += THREADS * U) {
            float x[U][8], e[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const Item t = item_of<D>(P, base + u * THREADS + threadIdx.x, count);
#pragma unroll
                for (int z = 0; z < 8; ++z) { x[u][z] = 0.f; e[u][z] = 0.f; }
                if (t.on) {
                    const uint32_t row = (uint32_t)row0 + t.row, b = row / (uint32_t)P.n, i = row - b * (uint32_t)P.n;
                    const bool q = t.head < P.hq;
                    const Side &S = q ? P.q : P.k;
                    const int64_t head = q ? t.head : t.head - P.hq;
                    load8<T>(reinterpret_cast<const T *>(S.x) + b * S.sb + i * S.sn + head * S.sh + c0, x[u]);
                    load8<T>(reinterpret_cast<const T *>(S.dy) + b * S.db + i * S.dn + head * S.dh + c0, e[u]);
                }
            }
            if (base == 0) {
                __syncthreads();                         // the last tile's angles are no longer read
                fill_angles(P, cs, row0, count);
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const Item t = item_of<D>(P, base + u * THREADS + threadIdx.x, count);
                if (!__any_sync(0xffffffffu, t.on)) break;
                float ss = 0.f;
#pragma unroll
                for (int z = 0; z < 8; ++z) ss = fmaf(x[u][z], x[u][z], ss);
                const float rstd = rsqrtf(head_sum<D>(ss) / (float)D + P.eps);
                const float *cos = cs + (t.on ? t.row : 0) * P.pairs;
                turn(e[u], c0, P, cos, cos + P.tile * P.pairs, -1.f);
                const bool q = t.head < P.hq;
                float dot = 0.f;
#pragma unroll
                for (int z = 0; z < 8; ++z) {
                    x[u][z] *= rstd;
                    const float dg = e[u][z] * x[u][z];
                    if (t.on && q) dq[z] += dg;
                    else if (t.on) dk[z] += dg;
                    e[u][z] *= q ? gq[z] : gk[z];
                    dot = fmaf(e[u][z], x[u][z], dot);
                }
                const float m = head_sum<D>(dot) / (float)D;
#pragma unroll
                for (int z = 0; z < 8; ++z) e[u][z] = rstd * (e[u][z] - x[u][z] * m);
                if (t.on) {
                    const Side &S = q ? P.q : P.k;
                    const int h = q ? P.hq : P.heads - P.hq, head = q ? t.head : t.head - P.hq;
                    store8<T>(reinterpret_cast<T *>(S.y) + ((row0 + t.row) * h + head) * D + c0, e[u]);
                }
            }
        }
    }
    // the threads of a channel, in order
    float *part = cs;                                    // [threads][8], queries and then keys
    for (int side = 0; side < 2; ++side) {
        __syncthreads();
        store8<float>(part + threadIdx.x * 8, side ? dk : dq);
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += THREADS) {
            float s = 0.f;
            for (int t = c / 8; t < THREADS; t += LANES) s += part[t * 8 + c % 8];
            P.partial[((int64_t)blockIdx.x * 2 + side) * D + c] = s;
        }
    }
}

// Sum of the partial rows: a CTA has 32 channels of one gain, slice j of 32 adds rows j, j + 32, ... in order, then the slices are
// added in order.
template <typename T>
__global__ void __launch_bounds__(1024) dgain_kernel(const float *partial, T *dq, T *dk, int nparts, int d) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    for (int p = slice; p < nparts; p += 32) s += partial[((int64_t)p * 2 + blockIdx.y) * d + c];
    part[slice][lane] = s;
    __syncthreads();
    if (slice == 0) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) t += part[j][lane];
        (blockIdx.y ? dk : dq)[c] = (T)t;
    }
}

// Rows of a CTA: four items a thread, fewer where the rows would leave SMs without work; at most 16 KB of angles.
inline int tile_rows(int64_t rows, int heads, int d, int pairs, int sms) {
    int64_t t = THREADS * PER_THREAD / ((int64_t)heads * (d / 8));
    if (t > rows / (2 * sms)) t = rows / (2 * sms);
    if (t > 2048 / pairs) t = 2048 / pairs;
    return t < 1 ? 1 : (int)t;
}
inline int bwd_grid(int64_t rows, int tile, int sms) {
    const int64_t tiles = (rows + tile - 1) / tile;
    return (int)(tiles < 4 * sms ? tiles : 4 * sms);
}
inline size_t fwd_smem(int tile, int pairs) { return (size_t)tile * pairs * 2 * sizeof(float); }
inline size_t bwd_smem(int tile, int pairs) {
    const size_t angles = fwd_smem(tile, pairs), sums = THREADS * 8 * sizeof(float);
    return angles > sums ? angles : sums;
}

}  // namespace rotary
}  // namespace sa2
