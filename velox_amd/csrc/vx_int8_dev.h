// vx_int8_dev.h -- device helpers of vx_int8.hip and vx_experts.hip: elements of activation rows, LDS within a wave.
#pragma once

#include "vx_int8.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float vx_load(const void* p, size_t i, uint32_t dtype) {
    if (dtype == VELOX_DT_F32) return ((const float*)p)[i];
    if (dtype == VELOX_DT_F16) return (float)((const _Float16*)p)[i];
    return (float)((const __bf16*)p)[i];
}
// The fp32 value rounded once (to nearest even) to the element type.
__device__ __forceinline__ void vx_store(void* p, size_t i, uint32_t dtype, float v) {
    if (dtype == VELOX_DT_F32) ((float*)p)[i] = v;
    else if (dtype == VELOX_DT_F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}

// Four neighbouring values of a row at element i as fp32, and back (rounded once); VEC: at whole 16- or 8-byte places.
template <bool VEC>
__device__ __forceinline__ float4 vx_load4(const void* p, size_t i, uint32_t dtype, uint32_t left) {
    float4 v = make_float4(0, 0, 0, 0);
    if (VEC && left >= 4u) {
        if (dtype == VELOX_DT_F32) return *(const float4*)((const float*)p + i);
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        const uint2 w = *(const uint2*)((const uint16_t*)p + i);
        if (dtype == VELOX_DT_F16) {
            const h4 h = __builtin_bit_cast(h4, w);
            return make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
        }
        const b4 b = __builtin_bit_cast(b4, w);
        return make_float4((float)b[0], (float)b[1], (float)b[2], (float)b[3]);
    }
    if (left > 0u) v.x = vx_load(p, i, dtype);
    if (left > 1u) v.y = vx_load(p, i + 1u, dtype);
    if (left > 2u) v.z = vx_load(p, i + 2u, dtype);
    if (left > 3u) v.w = vx_load(p, i + 3u, dtype);
    return v;
}
template <bool VEC>
__device__ __forceinline__ void vx_store4(void* p, size_t i, uint32_t dtype, uint32_t left, float4 v) {
    if (VEC && left >= 4u) {
        if (dtype == VELOX_DT_F32) {
            *(float4*)((float*)p + i) = v;
            return;
        }
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        if (dtype == VELOX_DT_F16) *(h4*)((uint16_t*)p + i) = h4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
        else *(b4*)((uint16_t*)p + i) = b4{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
        return;
    }
    if (left > 0u) vx_store(p, i, dtype, v.x);
    if (left > 1u) vx_store(p, i + 1u, dtype, v.y);
    if (left > 2u) vx_store(p, i + 2u, dtype, v.z);
    if (left > 3u) vx_store(p, i + 3u, dtype, v.w);
}
// What a lane of the wave wrote to LDS is what the others read behind this.
__device__ __forceinline__ void vx_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace
