// rope.cuh -- reading a head's elements, turned by their token's position: shared by the rope
// kernel and the cache-write kernel, so that both round alike.
#pragma once
#include "kv_impl.h"

namespace rmoe {

template <typename T> struct Elt;
template <> struct Elt<float> {
    static constexpr int TYPE = T_F32;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elt<__half> {
    static constexpr int TYPE = T_F16;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Elt<__nv_bfloat16> {
    static constexpr int TYPE = T_BF16;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// 8 consecutive elements as f32; vec: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float* v) {
    if (vec) {
        constexpr int W = 16 / sizeof(T);
        T e[8];
#pragma unroll
        for (int i = 0; i < 8 / W; i++) *reinterpret_cast<uint4*>(e + i * W) = *reinterpret_cast<const uint4*>(p + i * W);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = Elt<T>::get(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = Elt<T>::get(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float* v) {
    if (vec) {
        constexpr int W = 16 / sizeof(T);
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = Elt<T>::put(v[i]);
#pragma unroll
        for (int i = 0; i < 8 / W; i++) *reinterpret_cast<uint4*>(p + i * W) = *reinterpret_cast<const uint4*>(e + i * W);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = Elt<T>::put(v[i]);
    }
}

// A unit is the 16 elements that one thread turns: two chunks of 8, at a and b, that hold whole
// pairs.  Half layout, inside the rotated part: chunk u of each half; interleaved, or past the
// rotated part: 16 neighbours.  A head of `dim` elements has dim / 16 units (rot % 16 == 0).
__device__ __forceinline__ void unit_chunks(int u, int rot, int half, int& a, int& b) {
    if (half && u < rot / 16) {
        a = 8 * u;
        b = rot / 2 + 8 * u;
    } else {
        a = 16 * u;
        b = a + 8;
    }
}

// The pair (x0, x1) turned by (c, s): products and sums rounded one by one, so that the result
// does not depend on how a compiler contracts them.
__device__ __forceinline__ void turn(float& x0, float& x1, float c, float s) {
    const float y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
    const float y1 = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s));
    x0 = y0;
    x1 = y1;
}

// Turns unit u (its 16 elements in v: chunk a, then chunk b); row: the token's (cos, sin) pairs,
// 16-byte aligned (rot % 16 == 0).
__device__ __forceinline__ void turn_unit(float* v, int u, const float2* row, int rot, int half, float sign) {
    if (u >= rot / 16) return;
    const float4* cs = reinterpret_cast<const float4*>(row + 8 * u);  // the unit's 8 pairs
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float4 t = __ldg(cs + i);
        if (half) {
            turn(v[2 * i], v[8 + 2 * i], t.x, sign * t.y);
            turn(v[2 * i + 1], v[8 + 2 * i + 1], t.z, sign * t.w);
        } else {
            turn(v[4 * i], v[4 * i + 1], t.x, sign * t.y);
            turn(v[4 * i + 2], v[4 * i + 3], t.z, sign * t.w);
        }
    }
}

}  // namespace rmoe
