// enc_common.cuh -- what the encoder operators (enc_*.cu) share: element types
// as 16-byte units in registers, and the arguments of an attention call.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/d2p_b200.h"
#include "sw_internal.h"

namespace d2pb {
namespace enc {

constexpr float kLog2e = 1.4426950408889634f;

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values as one 32-bit word of a 16-bit type (a in the low half)
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// what that rounding took from a and b, in the same type; p: the two rounded
template <class T>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t p);
template <>
__device__ __forceinline__ uint32_t rest2<__nv_bfloat16>(float a, float b, uint32_t p) {
    return pack2<__nv_bfloat16>(a - __uint_as_float(p << 16), b - __uint_as_float(p & 0xffff0000u));
}
template <>
__device__ __forceinline__ uint32_t rest2<__half>(float a, float b, uint32_t p) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
    return pack2<__half>(a - f.x, b - f.y);
}

// eight consecutive elements at a 16-byte boundary
template <class T>
__device__ __forceinline__ void load8(const T* p, float* v) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f<T>(h[i]);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* v) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float* v) {
    uint4 u = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    *reinterpret_cast<uint4*>(p) = u;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float* v) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

}  // namespace enc
}  // namespace d2pb
