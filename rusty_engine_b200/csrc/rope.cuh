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

// The (cos, sin) of unit u's 8 pairs; row: the token's table row, 16-byte aligned (rot % 16 == 0).
__device__ __forceinline__ void unit_angles(const float2* row, int u, float4* cs) {
#pragma unroll
    for (int i = 0; i < 4; i++) cs[i] = __ldg(reinterpret_cast<const float4*>(row + 8 * u) + i);
}
__device__ __forceinline__ void turn_unit_by(float* v, const float4* cs, int half, float sign) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (half) {
            turn(v[2 * i], v[8 + 2 * i], cs[i].x, sign * cs[i].y);
            turn(v[2 * i + 1], v[8 + 2 * i + 1], cs[i].z, sign * cs[i].w);
        } else {
            turn(v[4 * i], v[4 * i + 1], cs[i].x, sign * cs[i].y);
            turn(v[4 * i + 2], v[4 * i + 3], cs[i].z, sign * cs[i].w);
        }
    }
}

// Turns unit u (its 16 elements in v: chunk a, then chunk b); row: the token's (cos, sin) pairs,
// 16-byte aligned (rot % 16 == 0).
__device__ __forceinline__ void turn_unit(float* v, int u, const float2* row, int rot, int half, float sign) {
    if (u >= rot / 16) return;
    float4 cs[4];
    unit_angles(row, u, cs);
    turn_unit_by(v, cs, half, sign);
}

// Turns every unit of q and k: items i0, i0 + step, ... of (token, head, unit), units first.  The
// next item's elements and position are asked for before the current one is turned, so that each
// warp has a load in flight all the time (without, 24 warps on an SM reached half of the memory's
// rate, and the angles, which wait for the position, were what they waited for).
template <typename T>
__device__ __forceinline__ void turn_items(const Rows& q, const Rows& qo, const Rows& k, const Rows& ko, const RopeArg& ra, int T_,
                                           int dim, int64_t i0, int64_t step, unsigned* status) {
    constexpr int W = sizeof(T) / 2;  // 16-byte words of a chunk
    const int units = dim >> 4, per_tok = (q.heads + k.heads) * units;
    const int64_t n = (int64_t)T_ * per_tok;
    uint4 next[2 * W];
    int u = 0, pos = 0, h = 0;
    bool isq = true;
    int64_t t = 0;
    auto fetch = [&](int64_t i) {
        t = (n >> 32) == 0 ? (int64_t)((uint32_t)i / (uint32_t)per_tok) : i / per_tok;
        const int r = (int)(i - t * per_tok);
        h = r / units;
        u = r - h * units;
        isq = h < q.heads;
        if (!isq) h -= q.heads;
        pos = __ldg(ra.pos + t);
        int a, b;
        unit_chunks(u, ra.rot, ra.half, a, b);
        if (isq ? q.vec : k.vec) {
            const T* x = isq ? reinterpret_cast<const T*>(q.p) + t * q.st + h * q.sh : reinterpret_cast<const T*>(k.p) + t * k.st + h * k.sh;
#pragma unroll
            for (int i = 0; i < W; i++) {
                next[i] = *(reinterpret_cast<const uint4*>(x + a) + i);
                next[W + i] = *(reinterpret_cast<const uint4*>(x + b) + i);
            }
        }
    };
    if (i0 < n) fetch(i0);
    for (int64_t i = i0; i < n; i += step) {
        const int cu = u, p = pos, ch = h;
        const bool cq = isq;
        const int64_t ct = t;
        T e[16];
#pragma unroll
        for (int j = 0; j < 2 * W; j++) *(reinterpret_cast<uint4*>(e) + j) = next[j];
        const bool inside = (unsigned)p < (unsigned)ra.max_pos, rot = inside && cu < ra.rot / 16;
        float4 cs[4];
        if (rot) unit_angles(ra.table + (size_t)p * (ra.rot / 2), cu, cs);
        if (!inside && cu == 0 && ch == 0) atomicOr(status, (unsigned)DERR_INDEX);
        if (i + step < n) fetch(i + step);
        int a, b;
        unit_chunks(cu, ra.rot, ra.half, a, b);
        float v[16];
        if (cq ? q.vec : k.vec) {
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] = Elt<T>::get(e[j]);
        } else {
            const T* x = cq ? reinterpret_cast<const T*>(q.p) + ct * q.st + ch * q.sh : reinterpret_cast<const T*>(k.p) + ct * k.st + ch * k.sh;
            load8(x + a, false, v);
            load8(x + b, false, v + 8);
        }
        if (rot) turn_unit_by(v, cs, ra.half, ra.sign);
        T* y = cq ? reinterpret_cast<T*>(qo.p) + ct * qo.st + ch * qo.sh : reinterpret_cast<T*>(ko.p) + ct * ko.st + ch * ko.sh;
        const bool vec = cq ? qo.vec : ko.vec;
        store8(y + a, vec, v);
        store8(y + b, vec, v + 8);
    }
}

}  // namespace rmoe
