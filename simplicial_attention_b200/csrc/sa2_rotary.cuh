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
// Bound: reading and writing every head once.  A warp has a row (or, where rows are few, a part of its heads): row, position and addresses
// are the same for its lanes, and each sine and cosine is formed once, in shared memory of the warp, while the loads are on their way.  A lane
// holds eight channels of a head: two groups of four, the second the partners of the first where halves are paired, so that a pair is in
// one lane; the lanes of a head add their squares by shuffles.  A lane has the same channels in all of its heads, and their gains in registers.
// The backward reads x again and forms rstd again, which costs no traffic of its own; gain gradients stay in registers over all rows
// of a CTA, a CTA writes one partial row and a second kernel adds those in order, without atomics.
// b16 n1024, 12 heads of 64 bf16 channels: forward 15.5 us, backward 27 and the gains' sums 3.4 (tiles of rows for a CTA, angles between two
// barriers: 22 and 42): issue slots 70 % busy.  b2 n5001, 20 heads of 128 fp32 channels: forward 37 us, 5.5 TB/s; backward with
// the gains' sums 60 us, 5.1 TB/s.
#pragma once
#include "sa2_common.cuh"
#include "sa2_vec8.cuh"

namespace sa2 {
namespace rotary {

constexpr int THREADS = 256, WARPS = THREADS / 32;
// CTAs of an SM, by registers; a launch has as many, and they go on row by row
template <typename T> constexpr int FWD_CTAS = sizeof(T) == 2 ? 4 : 3;
template <typename T> constexpr int BWD_CTAS = sizeof(T) == 2 ? 3 : 2;

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
    int rows, n;                // b * n; rows of a sequence
    int hq, heads, pairs;       // heads: of queries and keys
    int parts, turns;           // warps of a row; what each has: heads, 256 channels at a time
    int gain_bf16;
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

// The channels of a lane: four from `a` on and four from `b` on.  Lanes behind the rotated channels have eight that stay.
struct Channels { int a, b; bool turned; };
template <bool INTERLEAVED> __device__ __forceinline__ Channels channels_of(const Params &P, int lane) {
    const bool turned = lane * 8 < 2 * P.pairs;
    return turned && !INTERLEAVED ? Channels{4 * lane, P.pairs + 4 * lane, true} : Channels{8 * lane, 8 * lane + 4, turned};
}
// A lane's channels as they come: they stay packed until they are used
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> {
    uint2 a, b;
    __device__ __forceinline__ void clear() { a = make_uint2(0u, 0u); b = a; }
    __device__ __forceinline__ void load(const __nv_bfloat16 *p, const Channels &c) {
        a = __ldg(reinterpret_cast<const uint2 *>(p + c.a));
        b = __ldg(reinterpret_cast<const uint2 *>(p + c.b));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            v[2 * z] = __uint_as_float(w[z] << 16);
            v[2 * z + 1] = __uint_as_float(w[z] & 0xffff0000u);
        }
    }
};
template <> struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void clear() { a = make_float4(0.f, 0.f, 0.f, 0.f); b = a; }
    __device__ __forceinline__ void load(const float *p, const Channels &c) {
        a = __ldg(reinterpret_cast<const float4 *>(p + c.a));
        b = __ldg(reinterpret_cast<const float4 *>(p + c.b));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <typename T> __device__ __forceinline__ void store44(T *p, const Channels &c, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p + c.a) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4 *>(p + c.b) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * z], v[2 * z + 1]);
            w[z] = *reinterpret_cast<const uint32_t *>(&t);
        }
        *reinterpret_cast<uint2 *>(p + c.a) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2 *>(p + c.b) = make_uint2(w[2], w[3]);
    }
}

// Turns a lane's pairs by the angles with these cosines and sines.
template <bool INTERLEAVED> __device__ __forceinline__ void turn(float (&v)[8], const float (&cs)[4], const float (&sn)[4]) {
#pragma unroll
    for (int z = 0; z < 4; ++z) {
        float &first = INTERLEAVED ? v[2 * z] : v[z], &second = INTERLEAVED ? v[2 * z + 1] : v[4 + z];
        const float a = first, b = second;
        first = fmaf(a, cs[z], -b * sn[z]);
        second = fmaf(b, cs[z], a * sn[z]);
    }
}

__device__ __forceinline__ void load_gain(const Params &P, const void *gain, const Channels &c, float (&g)[8]) {
    if (P.gain_bf16) {
        Raw<__nv_bfloat16> r;
        r.load(reinterpret_cast<const __nv_bfloat16 *>(gain), c);
        r.get(g);
    } else {
        Raw<float> r;
        r.load(reinterpret_cast<const float *>(gain), c);
        r.get(g);
    }
}

// A warp's unit: a row, and which of its heads
struct Unit { int row, b, i, begin, end; };
template <int D> __device__ __forceinline__ Unit unit_of(const Params &P, int x) {
    Unit u;
    u.row = P.parts == 1 ? x : x / P.parts;
    u.b = u.row / P.n;
    u.i = u.row - u.b * P.n;
    const int part = x - u.row * P.parts;
    u.begin = part * P.turns * (256 / D);
    u.end = min(P.heads, u.begin + P.turns * (256 / D));
    return u;
}
// sines and cosines of a row's position into a warp's shared memory, cosines first; then this lane's
__device__ __forceinline__ void angles(const Params &P, const Unit &u, float *mine, int lane, bool turned, float (&cs)[4], float (&sn)[4], float sign) {
    const int64_t position = P.positions ? P.positions[u.b * P.pb + u.i * P.pn] : P.start + u.i;
    __syncwarp();                                        // the last row's are read
    for (int x = threadIdx.x & 31; x < P.pairs; x += 32) cos_sin(position, P.freqs[x], mine[x], mine[P.pairs + x]);
    __syncwarp();
    if (turned) {
        const float4 c = *reinterpret_cast<const float4 *>(mine + 4 * lane), t = *reinterpret_cast<const float4 *>(mine + P.pairs + 4 * lane);
        cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
        sn[0] = sign * t.x; sn[1] = sign * t.y; sn[2] = sign * t.z; sn[3] = sign * t.w;
    }
}

template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, FWD_CTAS<T>) fwd_kernel(const __grid_constant__ Params P) {
    extern __shared__ __align__(16) float shared[];
    constexpr int LANES = D / 8, HEADS = 256 / D, U = 3;         // heads of a warp at a time; times
    const int lane = threadIdx.x % LANES, sub = threadIdx.x % 32 / LANES, warp = threadIdx.x >> 5;
    const Channels ch = channels_of<INTERLEAVED>(P, lane);
    float gq[8], gk[8];
    load_gain(P, P.q.gain, ch, gq);
    load_gain(P, P.k.gain, ch, gk);
    const int units = P.rows * P.parts;
    for (int x = blockIdx.x * WARPS + warp; x < units; x += gridDim.x * WARPS) {
        const Unit w = unit_of<D>(P, x);
        const T *xq = reinterpret_cast<const T *>(P.q.x) + w.b * P.q.sb + w.i * P.q.sn, *xk = reinterpret_cast<const T *>(P.k.x) + w.b * P.k.sb + w.i * P.k.sn;
        T *yq = reinterpret_cast<T *>(P.q.y) + (int64_t)w.row * P.hq * D, *yk = reinterpret_cast<T *>(P.k.y) + (int64_t)w.row * (P.heads - P.hq) * D;
        float cs[4], sn[4];
        for (int h0 = w.begin + sub; h0 - sub < w.end; h0 += U * HEADS) {
            Raw<T> x0[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * HEADS;
                x0[u].clear();
                if (h < w.end) x0[u].load(h < P.hq ? xq + h * P.q.sh : xk + (h - P.hq) * P.k.sh, ch);
            }
            if (h0 - sub == w.begin) angles(P, w, shared + warp * 2 * P.pairs, lane, ch.turned, cs, sn, 1.f);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * HEADS;
                if (h - sub >= w.end) break;
                float v[8], ss = 0.f;
                x0[u].get(v);
#pragma unroll
                for (int z = 0; z < 8; ++z) ss = fmaf(v[z], v[z], ss);
                const float rstd = rsqrtf(head_sum<D>(ss) / (float)D + P.eps);
#pragma unroll
                for (int z = 0; z < 8; ++z) v[z] = v[z] * rstd * (h < P.hq ? gq[z] : gk[z]);
                if (ch.turned) turn<INTERLEAVED>(v, cs, sn);
                if (h < w.end) store44<T>(h < P.hq ? yq + h * D : yk + (h - P.hq) * D, ch, v);
            }
        }
    }
}

template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, BWD_CTAS<T>) bwd_kernel(const __grid_constant__ Params P) {
    extern __shared__ __align__(16) float shared[];
    constexpr int LANES = D / 8, HEADS = 256 / D, U = sizeof(T) == 2 ? 2 : 3;
    const int lane = threadIdx.x % LANES, sub = threadIdx.x % 32 / LANES, warp = threadIdx.x >> 5;
    const Channels ch = channels_of<INTERLEAVED>(P, lane);
    float dq[8], dk[8], gq[8], gk[8];
#pragma unroll
    for (int z = 0; z < 8; ++z) { dq[z] = 0.f; dk[z] = 0.f; }
    load_gain(P, P.q.gain, ch, gq);
    load_gain(P, P.k.gain, ch, gk);
    const int units = P.rows * P.parts;
    for (int x = blockIdx.x * WARPS + warp; x < units; x += gridDim.x * WARPS) {
        const Unit w = unit_of<D>(P, x);
        const T *xq = reinterpret_cast<const T *>(P.q.x) + w.b * P.q.sb + w.i * P.q.sn, *xk = reinterpret_cast<const T *>(P.k.x) + w.b * P.k.sb + w.i * P.k.sn;
        const T *eq = reinterpret_cast<const T *>(P.q.dy) + w.b * P.q.db + w.i * P.q.dn, *ek = reinterpret_cast<const T *>(P.k.dy) + w.b * P.k.db + w.i * P.k.dn;
        T *yq = reinterpret_cast<T *>(P.q.y) + (int64_t)w.row * P.hq * D, *yk = reinterpret_cast<T *>(P.k.y) + (int64_t)w.row * (P.heads - P.hq) * D;
        float cs[4], sn[4];
        for (int h0 = w.begin + sub; h0 - sub < w.end; h0 += U * HEADS) {
            Raw<T> x0[U], e0[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * HEADS;
                x0[u].clear();
                e0[u].clear();
                if (h < w.end) {
                    x0[u].load(h < P.hq ? xq + h * P.q.sh : xk + (h - P.hq) * P.k.sh, ch);
                    e0[u].load(h < P.hq ? eq + h * P.q.dh : ek + (h - P.hq) * P.k.dh, ch);
                }
            }
            if (h0 - sub == w.begin) angles(P, w, shared + warp * 2 * P.pairs, lane, ch.turned, cs, sn, -1.f);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * HEADS;
                if (h - sub >= w.end) break;
                const bool q = h < P.hq, on = h < w.end;
                float v[8], e[8], ss = 0.f;
                x0[u].get(v);
                e0[u].get(e);
#pragma unroll
                for (int z = 0; z < 8; ++z) ss = fmaf(v[z], v[z], ss);
                const float rstd = rsqrtf(head_sum<D>(ss) / (float)D + P.eps);
                if (ch.turned) turn<INTERLEAVED>(e, cs, sn);
                float dot = 0.f;
#pragma unroll
                for (int z = 0; z < 8; ++z) {
                    v[z] *= rstd;
                    const float dg = e[z] * v[z];
                    if (on && q) dq[z] += dg;
                    if (on && !q) dk[z] += dg;
                    e[z] *= q ? gq[z] : gk[z];
                    dot = fmaf(e[z], v[z], dot);
                }
                const float m = head_sum<D>(dot) / (float)D;
#pragma unroll
                for (int z = 0; z < 8; ++z) e[z] = rstd * (e[z] - v[z] * m);
                if (on) store44<T>(q ? yq + h * D : yk + (h - P.hq) * D, ch, e);
            }
        }
    }
    // the threads of a channel, in order
    for (int side = 0; side < 2; ++side) {
        __syncthreads();
        store8<float>(shared + threadIdx.x * 8, side ? dk : dq);
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += THREADS) {
            float s = 0.f;
            for (int t = c / 8; t < THREADS; t += LANES) s += shared[t * 8 + c % 8];
            const Channels at = channels_of<INTERLEAVED>(P, c / 8);
            P.partial[((int64_t)blockIdx.x * 2 + side) * D + (c % 8 < 4 ? at.a : at.b) + c % 4] = s;
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

// Warps of a row: one where there are 16 rows an SM, else as many as it takes to load all of its heads at once.
inline void split(int64_t rows, int heads, int d, int sms, int &parts, int &turns) {
    turns = (heads * d + 255) / 256;
    parts = 1;
    if (rows < 16 * (int64_t)sms && turns > 3) {
        parts = (turns + 2) / 3;
        turns = 3;
    }
}
inline int grid(int64_t units, int most) {
    const int64_t want = (units + WARPS - 1) / WARPS;
    return (int)(want < most ? want : most);
}
inline size_t fwd_smem(int pairs) { return (size_t)WARPS * pairs * 2 * sizeof(float); }
inline size_t bwd_smem(int pairs) {
    const size_t angles = fwd_smem(pairs), sums = THREADS * 8 * sizeof(float);
    return angles > sums ? angles : sums;
}

}  // namespace rotary
}  // namespace sa2
