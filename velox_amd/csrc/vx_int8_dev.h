// vx_int8_dev.h -- device helpers of vx_int8.hip and vx_experts.hip: elements of activation rows, rows in 8 bits, LDS within a wave.
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

// ---- rows in 8 bits ----
// The nearest whole number (ties to even) of the exact quotient x / s: rint(x * inv), inv = fl(1 / s), is off by one at
// most, and x - r s is exact in fp32 (a multiple of the smaller ulp, below s in size).
__device__ __forceinline__ int vx_code(float x, float s, float inv) {
    float r = rintf(x * inv);
    const float d = 2.0f * __builtin_fmaf(-r, s, x);
    const bool odd = ((int)r & 1) != 0;
    if (d > s || (d == s && odd)) r += 1.0f;
    else if (d < -s || (d == -s && odd)) r -= 1.0f;
    return (int)r;
}

// The same of four values, in the bytes of a word, where no x * inv is near a half; `near` says whether one is (rint is
// right below 0.5 - 2^-15, the error of x * inv).
__device__ __forceinline__ uint32_t vx_codes(const float* x, float inv, float& near) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float r = rintf(x[i] * inv);
        near = fmaxf(near, fabsf(__builtin_fmaf(x[i], inv, -r)));
        w = __builtin_amdgcn_cvt_pk_u8_f32(r + 128.0f, i, w);
    }
    return w ^ 0x80808080u;
}
constexpr float kVxNear = 0.4999f;
// A row's scale from the bits of its largest absolute value (those of an infinity or NaN are above any number's).
struct VxRowScale {
    float s, inv;
    bool none;  // codes are 0
};
__device__ __forceinline__ VxRowScale vx_row_scale(uint32_t top) {
    if (top >= 0x7F800000u) return {NAN, 0.0f, true};
    const float s = __builtin_bit_cast(float, top) / 127.0f;
    if (s < 1.17549435e-38f) return {0.0f, 0.0f, true};
    return {s, 1.0f / s, false};
}
__device__ __forceinline__ uint32_t vx_size_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t vx_max(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The largest word of THREADS threads, in each (`red`: a word for each wave).
template <int THREADS>
__device__ __forceinline__ uint32_t vx_threads_max(uint32_t v, uint32_t* red) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = vx_max(v, (uint32_t)__shfl_xor((int)v, off));
    if constexpr (THREADS > 64) {
        __syncthreads();  // (what was there has been looked at)
        if ((threadIdx.x & 63u) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) v = vx_max(v, red[w]);
    }
    return v;
}

// A row of k values (a whole number of 16-byte vectors, so placed) by THREADS threads, t this one's number, as codes at `to`
// (memory or LDS), k filled up to a multiple of 128; its scale. Up to NV vectors a thread stay in registers between the search
// for the largest value and the rounding, those behind are read again (MORE). Loads behind the row give 0. Values next to
// a half, one in 5000 (bf16: one in 380 of normally distributed ones), are done again by a rolled loop: little code, which comes
// through the instruction cache once.
template <class T, int THREADS, int NV, bool MORE>
__device__ __forceinline__ float vx_hold_row(const T* from, uint32_t k, uint8_t* to, uint32_t t, uint32_t* red) {
    constexpr uint32_t V = 16 / sizeof(T), STEP = THREADS * V;
    struct alignas(16) Vec {
        T v[V];
    };
    const uint32_t kp = vx_i8_pad(k);
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, (int)(k * sizeof(T)), 0x00020000);
    const auto load = [&](uint32_t c) { return __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(c * sizeof(T)), 0, 0)); };
    Vec in[NV];
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) in[j] = load(j * STEP + t * V);
    uint32_t top = 0;
    const auto look = [&](const Vec& v) {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) top = vx_max(top, vx_size_bits((float)v.v[i]));
    };
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) look(in[j]);
    if constexpr (MORE)
        for (uint32_t c = NV * STEP + t * V; c < k; c += STEP) look(load(c));
    const VxRowScale q = vx_row_scale(vx_threads_max<THREADS>(top, red));
    float near = 0.0f;
    const auto put = [&](uint32_t c, const Vec& v) {
        uint32_t w[V / 4];
#pragma unroll
        for (uint32_t i = 0; i < V / 4; ++i) {
            const float f[4] = {(float)v.v[4 * i], (float)v.v[4 * i + 1], (float)v.v[4 * i + 2], (float)v.v[4 * i + 3]};
            w[i] = vx_codes(f, q.inv, near);
            w[i] = q.none ? 0u : w[i];
        }
        if (c >= kp) return;
        if constexpr (V == 8) *(uint2*)(to + c) = make_uint2(w[0], w[1]);
        else *(uint32_t*)(to + c) = w[0];
    };
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) put(j * STEP + t * V, in[j]);
    if constexpr (MORE)
        for (uint32_t c = NV * STEP + t * V; c < kp; c += STEP) put(c, load(c));
    if (near > kVxNear && !q.none) {
#pragma unroll 1
        for (uint32_t c = t * V; c < k; c += STEP) {
            const Vec v = load(c);
#pragma unroll 1
            for (uint32_t i = 0; i < V; ++i) {
                float f = (float)v.v[0];
#pragma unroll
                for (uint32_t j = 1; j < V; ++j) f = i == j ? (float)v.v[j] : f;
                to[c + i] = (uint8_t)vx_code(f, q.s, q.inv);
            }
        }
    }
    return q.s;
}

}  // namespace
