// Eight consecutive channels of a row as fp32, for kernels that move 16 bytes (eight bf16) per lane and access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace sa2 {

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int z = 0; z < 4; ++z) {
        v[2 * z] = __uint_as_float(w[z] << 16);
        v[2 * z + 1] = __uint_as_float(w[z] & 0xffff0000u);
    }
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&v)[8]);
template <> __device__ __forceinline__ void store8<float>(float *p, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16 *p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int z = 0; z < 4; ++z) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * z], v[2 * z + 1]);
        w[z] = *reinterpret_cast<const uint32_t *>(&t);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
// rows whose base or stride is not a multiple of 16 bytes: element by element
template <typename T> __device__ __forceinline__ void load8u(const T *p, bool aligned, float (&v)[8]) {
    if (aligned) { load8<T>(p, v); return; }
#pragma unroll
    for (int z = 0; z < 8; ++z) v[z] = (float)p[z];
}
template <typename T> __device__ __forceinline__ void store8u(T *p, bool aligned, const float (&v)[8]) {
    if (aligned) { store8<T>(p, v); return; }
#pragma unroll
    for (int z = 0; z < 8; ++z) p[z] = (T)v[z];
}

// Eight values as they come: loads stay packed until they are used, so that many fit the registers at a time.
template <typename T> struct Packed;
template <> struct Packed<__nv_bfloat16> {
    uint4 a;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { a = __ldg(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            v[2 * z] = __uint_as_float(w[z] << 16);
            v[2 * z + 1] = __uint_as_float(w[z] & 0xffff0000u);
        }
    }
};
template <> struct Packed<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = __ldg(reinterpret_cast<const float4 *>(p));
        b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};

}  // namespace sa2
