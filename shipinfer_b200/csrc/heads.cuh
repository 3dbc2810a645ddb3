// Shared by the kernels that read a model's scores: element types, and the order of choices.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace shipk {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float* out) { *out = v; }
__device__ __forceinline__ void from_f32(float v, __half* out) { *out = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* out) { *out = __float2bfloat16_rn(v); }

// Order bits: larger values give larger codes, -0 and +0 the same one; never 0 for a number.
__device__ __forceinline__ uint32_t order_bits(float v) {
    uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) == 0) u = 0;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_order_bits(uint32_t ord) {
    return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7fffffffu) : ~ord);
}

// Keys whose descending order is the larger value first and, among equal values, the lower index.
// 0 is no value's key.
__device__ __forceinline__ uint64_t choice_key(float v, int index) {
    return ((uint64_t)order_bits(v) << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }
__device__ __forceinline__ float key_value(uint64_t k) { return from_order_bits((uint32_t)(k >> 32)); }

}  // namespace shipk
