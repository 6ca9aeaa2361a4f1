// kv_code.cuh -- the cache's 8-bit codes: rounding f32 to them and widening them.
#pragma once
#include <cuda_fp8.h>

#include "kv_impl.h"

namespace rmoe {

// int8: codes -127 .. 127.  e4m3: the finite values of the format, largest 448.
template <int CODE> struct Code;
template <> struct Code<RMOE_KV_INT8> {
    static constexpr float PER = 1.0f / 127.0f;  // scale per unit of the largest magnitude
    // x finite or not: NaN to 0, beyond the top to the top; nearest, ties to even
    static __device__ __forceinline__ uint32_t put(float x) {
        x = x != x ? 0.0f : fminf(fmaxf(x, -127.0f), 127.0f);
        return (uint32_t)__float2int_rn(x) & 0xffu;
    }
    static __device__ __forceinline__ float get(uint32_t c) { return (float)(int8_t)(c & 0xffu); }
};
template <> struct Code<RMOE_KV_E4M3> {
    static constexpr float PER = 1.0f / 448.0f;
    static __device__ __forceinline__ uint32_t put(float x) {
        x = x != x ? 0.0f : fminf(fmaxf(x, -448.0f), 448.0f);
        return (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
    }
    static __device__ __forceinline__ float get(uint32_t c) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(c & 0xffu), __NV_E4M3);
        return __half2float(__half(h));
    }
};

}  // namespace rmoe
