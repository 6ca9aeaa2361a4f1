// kv_widen.cuh -- widening cached codes to fp16 (exact for both code types), and the numbers that
// the attention kernels share.
#pragma once
#include "kv_code.cuh"

namespace rmoe {

// 4 codes -> two registers of two fp16 each (elements 0, 1 and 2, 3 of the word), exactly.
template <int CODE>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& a, uint32_t& b) {
    if (CODE == RMOE_KV_INT8) {
        // 0x6400 | u is 1024 + u for a byte u; u = code + 128
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 c = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
        const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), c), q = __hsub2(*reinterpret_cast<const __half2*>(&y), c);
        a = *reinterpret_cast<const uint32_t*>(&p);
        b = *reinterpret_cast<const uint32_t*>(&q);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}\n"
            : "=r"(a), "=r"(b) : "r"(w));
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// The V scale enters the exponent: log2 of it is added to the score, and a row's sum takes its
// reciprocal (to 2^-22: an error of the logarithm changes a block's weights alike in both sums and
// is as small as the weights' own).  Exponentials below 2^-126 are 0, so a key whose weight times its
// block's scale is 2^-126 of another's loses its share of the sum.  Values of 0 have no scale of their
// own: their block counts as 2^-60, where it keeps its share beside scales of 2^46 (values of 9e15) from
// 20 powers of two below them on (counted as 2^-100, zeros beside values of 1e10 lost it), and takes no
// bits from the weights of blocks with scales above 2^-78.  Any other scale below 2^-100 counts as 2^-100.
__device__ __forceinline__ float v_scale_floor(float vs) {
    return vs == 0.0f ? 8.6736173798840355e-19f : fmaxf(vs, 7.8886090522101181e-31f);
}

// The exponent e that brings a row of q whose largest magnitude is mx to mx 2^-e in [2^13, 2^14);
// 0 where there is nothing to scale (0, infinities, NaN).
__device__ __forceinline__ int q_exponent(float mx) {
    const int ex = (int)((__float_as_uint(mx) >> 23) & 0xffu) - 127 - 13;
    return mx > 0.0f && mx <= 3.4e38f ? max(-126, min(113, ex)) : 0;
}

// The weights p = 2^(x - M) of a row go to the tensor cores as fp16, whose smallest step is 2^-24 and
// whose largest value is 2^16: they are carried as p times a power of two, which the output is divided
// by again.  Carried as p itself, the keys behind a dominant one were lost where its value is near 0 (4096
// keys 14 nats below it: 2e-4 of an f32 output, all of it from 20 nats on; times 2^15: 1e-9 and 3e-7).
static constexpr float W_UP = 32768.0f, W_DOWN = 1.0f / 32768.0f;

static constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;

}  // namespace rmoe
