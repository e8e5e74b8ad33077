// vx_int8.hip -- products of 8-bit integers with a scale for each token and channel.
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

// ---- weights ----
__global__ __launch_bounds__(256) void vx_i8_pack_kernel(VxI8Mat m, uint32_t first, const int8_t* __restrict__ src, uint64_t ms,
                                                         uint64_t rs, const float* __restrict__ scales, uint64_t ss) {
    const uint32_t e = blockIdx.z;
    const uint64_t per = (uint64_t)m.n_tiles * m.k_tiles * 64u;
    const uint32_t rows = m.paired ? m.n / 2u : m.n;
    src += e * ms;
    scales += e * ss;
    uint4* codes = (uint4*)m.codes + (first + e) * per;
    float* to = (float*)m.scales + (uint64_t)(first + e) * m.n_tiles * 16u;
    for (uint64_t i = blockIdx.x * 256u + threadIdx.x; i < per; i += gridDim.x * 256u) {
        const uint32_t unit = (uint32_t)(i >> 6), lane = (uint32_t)i & 63u, kt = unit % m.k_tiles, t = unit / m.k_tiles;
        const uint32_t in = 16u * (m.paired ? t >> 1 : t) + (lane & 15u), row = m.paired && (t & 1u) ? rows + in : in;
        const uint32_t c0 = 64u * kt + 16u * (lane >> 4);
        alignas(16) int8_t v[16] = {};
        if (in < rows) {
            const int8_t* from = src + row * rs + c0;
            if (c0 + 16u <= m.k && ((uintptr_t)from & 15u) == 0) *(uint4*)v = *(const uint4*)from;
            else
                for (uint32_t j = 0; j < 16u && c0 + j < m.k; ++j) v[j] = from[j];
        }
        codes[i] = *(const uint4*)v;
        if (kt == 0 && lane < 16u) to[16u * t + lane] = in < rows ? scales[row] : 0.0f;
    }
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

__global__ __launch_bounds__(256) void vx_i8_quantize_kernel(VxI8View x, uint32_t k, VxI8Rows o, const uint32_t* limit) {
    __shared__ float red[4];
    const uint32_t r = blockIdx.x, tid = threadIdx.x, kp = vx_i8_pad(k);
    if (limit && r >= *limit) return;
    const size_t base = (size_t)r * x.rs;
    float top = 0.0f;
    bool bad = false;
    for (uint32_t i = tid; i < k; i += 256u) {
        const float v = fabsf(vx_load(x.data, base + i, x.dtype));
        bad |= !(v < INFINITY);
        top = fmaxf(top, v);
    }
    if (bad) top = INFINITY;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
    if ((tid & 63u) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float s = top / 127.0f;
    const bool nan = top == INFINITY, none = s < 1.17549435e-38f;
    const float inv = 1.0f / s;
    int8_t* to = o.codes + (size_t)r * o.rs;
    for (uint32_t i = tid; i < kp; i += 256u)
        to[i] = i < k && !nan && !none ? (int8_t)vx_code(vx_load(x.data, base + i, x.dtype), s, inv) : (int8_t)0;
    if (tid == 0) o.scales[r] = nan ? NAN : none ? 0.0f : s;
}

// ---- products ----
// One wave: 16 activation rows by two weight tiles (paired: a gate tile and its up tile). The weights are the A operand, so
// that a lane ends with four neighbouring outputs of one row: D[n = 4 (lane / 16) + i][row = lane % 16].
template <int EPI>
__global__ __launch_bounds__(256) void vx_i8_kernel(VxI8Args a, uint32_t row0, uint32_t n_blocks) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t nb = blockIdx.x % n_blocks, item = blockIdx.x / n_blocks;
    const uint32_t t0 = 2u * (nb * 4u + wave);
    constexpr bool kGrouped = EPI == VX_I8_HIDDEN || EPI == VX_I8_SLOT;
    uint32_t e = 0, first = row0 + item * 16u, end = a.n_rows;
    if constexpr (kGrouped) {
        if (item >= *a.g.n_items) return;
        const uint2 it = a.g.items[item];
        e = it.x;
        first = it.y;
        end = a.g.offsets[e + 1u];
    }
    if (t0 >= a.w.n_tiles) return;
    const uint32_t p = first + (lane & 15u);
    const bool live = p < end;
    uint32_t slot = p, row = live ? p : first;
    if constexpr (kGrouped) {
        slot = a.g.order[live ? p : first];
        if constexpr (EPI == VX_I8_HIDDEN) row = slot / a.top;
    }
    const int8_t* x = a.a.codes + (size_t)row * a.a.rs + 16u * (lane >> 4);
    const bool two = t0 + 1u < a.w.n_tiles;
    const uint4* w0 = a.w.codes + ((uint64_t)e * a.w.n_tiles + t0) * a.w.k_tiles * 64u + lane;
    const uint4* w1 = two ? w0 + (uint64_t)a.w.k_tiles * 64u : w0;
    v4i acc0 = {0, 0, 0, 0}, acc1 = {0, 0, 0, 0};
    for (uint32_t kt = 0; kt < a.w.k_tiles; ++kt) {
        const v4i b = *(const v4i*)(x + 64u * kt);
        acc0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, w0[64u * kt]), b, acc0, 0, 0, 0);
        acc1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, w1[64u * kt]), b, acc1, 0, 0, 0);
    }
    if (!live) return;
    const float s = a.a.scales[row];
    const float* ws = a.w.scales + (uint64_t)e * a.w.n_tiles * 16u + 16u * t0 + 4u * (lane >> 4);
    if constexpr (EPI == VX_I8_SWIGLU || EPI == VX_I8_HIDDEN) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const float gate = (float)acc0[i] * ws[i] * s, up = (float)acc1[i] * ws[16u + i] * s;
            const float h = gate / (1.0f + expf(-gate)) * up;
            const uint32_t j = 8u * t0 + 4u * (lane >> 4) + i;
            if (j < a.w.n / 2u) {
                if constexpr (EPI == VX_I8_HIDDEN) a.part[(size_t)p * a.part_stride + j] = h;
                else vx_store(a.out.data, (size_t)p * a.out.rs + j, a.out.dtype, h);
            }
        }
    } else {
#pragma unroll
        for (uint32_t t = 0; t < 2u; ++t) {
            if (t && !two) break;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t n = 16u * (t0 + t) + 4u * (lane >> 4) + i;
                if (n >= a.w.n) continue;
                float y = (float)(t ? acc1 : acc0)[i] * ws[16u * t + i] * s;
                if constexpr (EPI == VX_I8_SLOT) {
                    a.part[(size_t)slot * a.part_stride + n] = y;
                } else {
                    if (a.bias) y += a.bias[n];
                    if (a.res.data) y += vx_load(a.res.data, (size_t)p * a.res.rs + n, a.res.dtype);
                    vx_store(a.out.data, (size_t)p * a.out.rs + n, a.out.dtype, y);
                }
            }
        }
    }
}

template <int EPI>
hipError_t vx_i8_launch(const VxI8Args& a, hipStream_t st) {
    const uint32_t n_blocks = (a.w.n_tiles + 7u) / 8u;
    if (EPI == VX_I8_HIDDEN || EPI == VX_I8_SLOT) {
        hipLaunchKernelGGL((vx_i8_kernel<EPI>), dim3(a.max_items * n_blocks), dim3(256), 0, st, a, 0u, n_blocks);
        return hipGetLastError();
    }
    const uint32_t step = 16u * ((1u << 23) / n_blocks ? (1u << 23) / n_blocks : 1u);  // a launch has fewer than 2^32 threads
    for (uint32_t r = 0; r < a.n_rows; r += step) {
        const uint32_t rows = a.n_rows - r < step ? a.n_rows - r : step;
        hipLaunchKernelGGL((vx_i8_kernel<EPI>), dim3((rows + 15u) / 16u * n_blocks), dim3(256), 0, st, a, r, n_blocks);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace

hipError_t vx_launch_i8_pack(const VxI8Mat& m, uint32_t first, uint32_t number, const int8_t* codes, uint64_t ms, uint64_t rs,
                             const float* scales, uint64_t ss, hipStream_t st) {
    const uint64_t per = (uint64_t)m.n_tiles * m.k_tiles * 64u;
    const uint32_t wgs = per / 256u < 4096u ? (uint32_t)((per + 255u) / 256u) : 4096u;
    hipLaunchKernelGGL(vx_i8_pack_kernel, dim3(wgs, 1, number), dim3(256), 0, st, m, first, codes, ms, rs, scales, ss);
    return hipGetLastError();
}

hipError_t vx_launch_i8_quantize(const VxI8View& x, uint32_t n_rows, uint32_t k, const VxI8Rows& out, const uint32_t* limit,
                                 hipStream_t st) {
    hipLaunchKernelGGL(vx_i8_quantize_kernel, dim3(n_rows), dim3(256), 0, st, x, k, out, limit);
    return hipGetLastError();
}

uint32_t vx_i8_item_rows(uint32_t, uint32_t) { return 16u; }

hipError_t vx_launch_i8_product(const VxI8Args& a, int epi, hipStream_t st) {
    switch (epi) {
        case VX_I8_STORE: return vx_i8_launch<VX_I8_STORE>(a, st);
        case VX_I8_SWIGLU: return vx_i8_launch<VX_I8_SWIGLU>(a, st);
        case VX_I8_HIDDEN: return vx_i8_launch<VX_I8_HIDDEN>(a, st);
        case VX_I8_SLOT: return vx_i8_launch<VX_I8_SLOT>(a, st);
        default: return hipErrorInvalidValue;
    }
}
