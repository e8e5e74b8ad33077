// vx_int8.hip -- products of 8-bit integers with a scale for each token and channel.
#include <atomic>

#include "vx_int8_dev.h"

namespace {

template <int V>
struct vx_int {
    static constexpr int value = V;
};
template <int N, int I = 0, class F>
__device__ __forceinline__ void vx_each(F f) {  // f(vx_int<0>) .. f(vx_int<N - 1>)
    if constexpr (I < N) {
        f(vx_int<I>{});
        vx_each<N, I + 1>(f);
    }
}

// A row's bits do not depend on the kernel that it goes through: sums of whole numbers are exact, and what follows is done by the
// functions here with the roundings as they are written (nothing is contracted into an fma but what says fma).
__device__ __forceinline__ float4 vx_add(const float4& a, const float4& b) {
#pragma clang fp contract(off)
    return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
// Four sums with the weight rows' scales, the row's scale and (BIAS) the bias.
template <bool BIAS>
__device__ __forceinline__ float4 vx_scaled(const v4i& c, const float4& w, float s, const float4& b) {
#pragma clang fp contract(off)
    float y[4];
    const float f[4] = {w.x, w.y, w.z, w.w}, d[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = (float)c[i] * f[i];
        y[i] = BIAS ? __builtin_fmaf(p, s, d[i]) : p * s;
    }
    return make_float4(y[0], y[1], y[2], y[3]);
}
__device__ __forceinline__ float vx_swiglu(float g, float u) {
#pragma clang fp contract(off)
    return g / (1.0f + expf(-g)) * u;
}
__device__ __forceinline__ float4 vx_swiglu(const v4i& g, const float4& wg, const v4i& u, const float4& wu, float s) {
    const float4 none = make_float4(0, 0, 0, 0), a = vx_scaled<false>(g, wg, s, none), b = vx_scaled<false>(u, wu, s, none);
    return make_float4(vx_swiglu(a.x, b.x), vx_swiglu(a.y, b.y), vx_swiglu(a.z, b.z), vx_swiglu(a.w, b.w));
}
// Outputs n .. n + 3 of row r (of `cols` in a row), y their products with the bias: the residual added, stored.
template <bool VEC>
__device__ __forceinline__ void vx_finish(const VxI8Args& a, size_t r, uint32_t n, uint32_t cols, float4 y) {
    const uint32_t left = cols - n;
    if (a.res.data) y = vx_add(y, vx_load4<VEC>(a.res.data, r * a.res.rs + n, a.res.dtype, left));
    vx_store4<VEC>(a.out.data, r * a.out.rs + n, a.out.dtype, left, y);
}
// Outputs c .. c + 3 of a plain product's row r (of `cols` in a row), from their sums.
template <bool SWIGLU>
__device__ __forceinline__ void vx_outputs(const VxI8Args& a, size_t r, uint32_t c, uint32_t cols, const v4i& sum, const v4i& up, const float* ws, float s) {
    const float4 w = *(const float4*)ws;
    float4 y;
    if constexpr (SWIGLU) y = vx_swiglu(sum, w, up, *(const float4*)(ws + 16), s);
    else if (a.bias) y = vx_scaled<true>(sum, w, s, vx_load4<false>(a.bias, c, VELOX_DT_F32, cols - c));
    else y = vx_scaled<false>(sum, w, s, w);
    if (a.vec) vx_finish<true>(a, r, c, cols, y);
    else vx_finish<false>(a, r, c, cols, y);
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
// Scale and codes of a row, which is read once: as many threads a row as hold it in registers (a wave for short rows, which
// then share nothing). Bound by the bytes in fp32 (8192 rows of 14336, 587 MB: 108 us, 5.4 TB/s), in 16 bits by the values that lie next to
// a half, for which a wave goes over its values again: 8192 rows of 29568 bf16, 727 MB, take 157 to 175 us (4.6 to 4.2 TB/s) with a few
// channels far above the others, as hidden states have (one value in 3000), 281 with normally distributed ones (one in 380: bf16 numbers
// are few, and so are their quotients). For few rows by latency (32 rows of 3584 fp32: 4.8 us). 64 values of 16 bits a thread of 1024
// (rows of 32769 to 65536 values) do not all stay in registers (44 to 48 bytes a thread go to memory); they still beat the kernel below
// with the former values (4096 rows of 40960: 166 and 216 us), not with the latter (267 and 215).
template <class T, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void vx_i8_quantize_kernel(VxI8View x, uint32_t n_rows, uint32_t k, VxI8Rows o, const uint32_t* limit) {
    constexpr int WG = TPR < 256 ? 256 : TPR;
    __shared__ uint32_t red[WG / 64];
    const uint32_t r = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * (WG / TPR) + threadIdx.x / TPR)), t = threadIdx.x % TPR;
    if (limit) n_rows = *limit < n_rows ? *limit : n_rows;
    if (r >= n_rows) return;  // (a wave that shares nothing, or the workgroup)
    const float s = vx_hold_row<T, TPR, NV, false>((const T*)x.data + (size_t)r * x.rs, k, (uint8_t*)o.codes + (size_t)r * o.rs, t, red);
    if (t == 0) o.scales[r] = s;
}

// Rows at any place and of any length, value by value: NE of them a thread in registers, those behind read twice. Each value's
// remainder is formed, so the values do not matter: 8192 rows of 4096 bf16 25 us, of 29568 289 (2.5 TB/s), fp32 32 and 414.
template <class T, int NE>
__global__ __launch_bounds__(256) void vx_i8_quantize_any_kernel(VxI8View x, uint32_t k, VxI8Rows o, const uint32_t* limit) {
    __shared__ uint32_t red[4];
    const uint32_t r = blockIdx.x, tid = threadIdx.x, kp = vx_i8_pad(k);
    if (limit && r >= *limit) return;
    const T* from = (const T*)x.data + (size_t)r * x.rs;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, (int)(k * sizeof(T)), 0x00020000);
    const auto load = [&](uint32_t c) -> float {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, (int)(c * 4u), 0, 0));
        else return (float)__builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, (int)(c * 2u), 0, 0));
    };
    float in[NE];
#pragma unroll
    for (uint32_t j = 0; j < NE; ++j) in[j] = load(j * 256u + tid);
    uint32_t top = 0;
#pragma unroll
    for (uint32_t j = 0; j < NE; ++j) top = vx_max(top, vx_size_bits(in[j]));
#pragma unroll 8
    for (uint32_t c = NE * 256u + tid; c < k; c += 256u) top = vx_max(top, vx_size_bits(load(c)));
    const VxRowScale q = vx_row_scale(vx_threads_max<256>(top, red));
    int8_t* to = o.codes + (size_t)r * o.rs;
    const auto put = [&](uint32_t c, float v) {
        const int code = vx_code(v, q.s, q.inv);
        if (c < kp) to[c] = q.none ? (int8_t)0 : (int8_t)code;
    };
#pragma unroll
    for (uint32_t j = 0; j < NE; ++j) put(j * 256u + tid, in[j]);
#pragma unroll 4
    for (uint32_t c = NE * 256u + tid; c < kp; c += 256u) put(c, load(c));
    if (tid == 0) o.scales[r] = q.s;
}

template <class T>
hipError_t vx_quantize_launch(const VxI8View& x, uint32_t n_rows, uint32_t k, const VxI8Rows& o, const uint32_t* limit, hipStream_t st) {
    constexpr uint32_t V = 16 / sizeof(T);
    if (vx_whole_rows(x, k) && vx_i8_pad(k) / V <= 1024u * 8u) {
        const uint32_t vecs = vx_i8_pad(k) / V;  // (the codes behind k are written too)
#define VX_QUANTIZE(TPR, NV)                                                                                                              \
    if (vecs <= TPR * NV) {                                                                                                               \
        constexpr uint32_t wg = TPR < 256 ? 256 : TPR;                                                                                    \
        hipLaunchKernelGGL((vx_i8_quantize_kernel<T, TPR, NV>), dim3((n_rows + wg / TPR - 1) / (wg / TPR)), dim3(wg), 0, st, x, n_rows, k, o, limit); \
        return hipGetLastError();                                                                                                         \
    }
        VX_QUANTIZE(64, 1)
        VX_QUANTIZE(64, 2)
        VX_QUANTIZE(256, 1)
        VX_QUANTIZE(256, 2)
        VX_QUANTIZE(256, 4)
        VX_QUANTIZE(256, 8)
        VX_QUANTIZE(1024, 4)
        VX_QUANTIZE(1024, 8)
#undef VX_QUANTIZE
    }
    if (vx_i8_pad(k) <= 4u * 256u) hipLaunchKernelGGL((vx_i8_quantize_any_kernel<T, 4>), dim3(n_rows), dim3(256), 0, st, x, k, o, limit);
    else hipLaunchKernelGGL((vx_i8_quantize_any_kernel<T, 16>), dim3(n_rows), dim3(256), 0, st, x, k, o, limit);
    return hipGetLastError();
}

// ---- products of few rows: the weights' bytes ----
// A workgroup of NW waves takes NT weight tiles (paired: gate and up tiles by turns) by 16 MT rows. Its waves deal out the 64-column
// tiles in turn, so that the weights stream in order, each lane's 16 bytes being its MFMA operand; U tiles are requested
// while U are multiplied, those behind the last by bounds-checked loads that give zeros. The waves' sums meet in LDS. The
// weights are the A operand, so that a lane ends with four neighbouring outputs: D[n = 4 (lane / 16) + i][row = lane % 16].
// Bound by the weights' bytes: 32 rows of 37888 x 3584 28.4 to 29 us (4.7 TB/s), 32 rows by 8 of 256 experts of 7168 x 2048,
// 64 here, 107 and 56 us for the two products (6.7 TB/s).
template <int NT, int MT, int NW, int EPI>
__global__ __launch_bounds__(64 * NW) void vx_i8_stream_kernel(VxI8Args a, uint32_t n_blocks) {
    constexpr bool kGrouped = EPI == VX_I8_HIDDEN || EPI == VX_I8_SLOT, kSwiglu = EPI == VX_I8_SWIGLU || EPI == VX_I8_HIDDEN;
    constexpr int U = NT + MT <= 3 ? 4 : 2;
    __shared__ v4i sums[NW][NT * MT][64];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    const uint32_t item = uniform(blockIdx.x / n_blocks), t0 = uniform(blockIdx.x % n_blocks) * NT;
    uint32_t e = 0, first = item * 16u * MT, end = a.n_rows;
    if constexpr (kGrouped) {
        if (item >= uniform(*a.g.n_items)) return;
        const uint2 it = a.g.items[item];
        e = uniform(it.x);
        first = uniform(it.y);
        end = uniform(a.g.offsets[e + 1u]);
    }
    const int8_t* x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const uint32_t p = first + 16u * m + (lane & 15u);
        uint32_t row = p < end ? p : end - 1u;
        if constexpr (EPI == VX_I8_HIDDEN) row = a.g.order[row] / a.top;
        x[m] = a.a.codes + (size_t)row * a.a.rs + 16u * (lane >> 4);
    }
    const uint32_t run = a.w.k_tiles * 1024u;  // bytes of a tile row
    const uint8_t* w = (const uint8_t*)a.w.codes + ((uint64_t)e * a.w.n_tiles + t0) * run;
    const uint32_t tiles = a.w.n_tiles - t0 < (uint32_t)NT ? a.w.n_tiles - t0 : (uint32_t)NT;
    __amdgpu_buffer_rsrc_t rs[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) rs[n] = __builtin_amdgcn_make_buffer_rsrc((void*)(w + (uint64_t)n * run), 0, n < (int)tiles ? (int)run : 0, 0x00020000);
    struct Set {
        v4i w[U][NT], x[U][MT];
    };
    const auto load = [&](Set& s, uint32_t kt) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = kt + u * NW, kx = k < a.w.k_tiles ? k : a.w.k_tiles - 1u;
#pragma unroll
            for (int n = 0; n < NT; ++n) s.w[u][n] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rs[n], (int)(k * 1024u + lane * 16u), 0, 2));
#pragma unroll
            for (int m = 0; m < MT; ++m) s.x[u][m] = *(const v4i*)(x[m] + 64u * kx);
        }
    };
    v4i acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = v4i{0, 0, 0, 0};
    const auto multiply = [&](const Set& s) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[n][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.w[u][n], s.x[u][m], acc[n][m], 0, 0, 0);
    };
    Set s0, s1;
    load(s0, wave);
    for (uint32_t kt = wave; kt < a.w.k_tiles; kt += 2u * U * NW) {
        load(s1, kt + U * NW);
        multiply(s0);
        load(s0, kt + 2u * U * NW);
        multiply(s1);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) sums[wave][n * MT + m][lane] = acc[n][m];
    __syncthreads();
    // output tiles (paired: of two weight tiles each) by the waves in turn
    constexpr int OUT = (kSwiglu ? NT / 2 : NT) * MT;
    const uint32_t cols = kSwiglu ? a.w.n / 2u : a.w.n;
#pragma unroll 1
    for (int o = wave; o < OUT; o += NW) {
        const int n = o / MT, m = o % MT;
        const uint32_t p = first + 16u * m + (lane & 15u), c = 16u * (t0 / (kSwiglu ? 2u : 1u) + n) + 4u * (lane >> 4);
        const auto total = [&](int at) {
            v4i v = sums[0][at][lane];
#pragma unroll
            for (int j = 1; j < NW; ++j) v += sums[j][at][lane];
            return v;
        };
        if (p >= end || c >= cols) continue;
        uint32_t row = p, slot = p;
        if constexpr (kGrouped) slot = a.g.order[p];
        if constexpr (EPI == VX_I8_HIDDEN) row = slot / a.top;
        const float s = a.a.scales[row];
        const float* ws = a.w.scales + ((uint64_t)e * a.w.n_tiles + t0 + (kSwiglu ? 2 * n : n)) * 16u + 4u * (lane >> 4);
        const v4i sum = total((kSwiglu ? 2 * n : n) * MT + m), up = kSwiglu ? total((2 * n + 1) * MT + m) : sum;
        if constexpr (kGrouped) {
            const float4 f = *(const float4*)ws;
            *(float4*)(a.part + (size_t)(EPI == VX_I8_SLOT ? slot : p) * a.part_stride + c) =
                kSwiglu ? vx_swiglu(sum, f, up, *(const float4*)(ws + 16), s) : vx_scaled<false>(sum, f, s, f);  // (rows of whole float4)
        } else {
            vx_outputs<kSwiglu>(a, p, c, cols, sum, up, ws, s);
        }
    }
}

template <int NT, int MT, int NW, int EPI>
hipError_t vx_i8_stream_launch(const VxI8Args& a, hipStream_t st) {
    const uint32_t n_blocks = (a.w.n_tiles + NT - 1u) / NT;
    const uint32_t items = EPI == VX_I8_HIDDEN || EPI == VX_I8_SLOT ? a.max_items : (a.n_rows + 16u * MT - 1u) / (16u * MT);
    hipLaunchKernelGGL((vx_i8_stream_kernel<NT, MT, NW, EPI>), dim3(items * n_blocks), dim3(64 * NW), 0, st, a, n_blocks);
    return hipGetLastError();
}

// ---- products of one row, put into 8 bits on the way ----
// NT tile rows of weights by one wave: tiles first, first + step, ... of each, U of them requested at a time, against codes in
// LDS (`x`: this lane's row, 16 (lane / 16) bytes in).
template <int NT>
struct VxStream {
    static constexpr int U = NT == 1 ? 8 : 4;
    __amdgpu_buffer_rsrc_t rs[NT];
    uint32_t k_tiles, lane;
    v4i w[2][U][NT], acc[NT];
    __device__ __forceinline__ VxStream(const VxI8Mat& m, uint32_t e, uint32_t t0) : k_tiles(m.k_tiles), lane(threadIdx.x & 63u) {
        const uint32_t run = m.k_tiles * 1024u;
        const uint8_t* at = (const uint8_t*)m.codes + ((uint64_t)e * m.n_tiles + t0) * run;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            rs[n] = __builtin_amdgcn_make_buffer_rsrc((void*)(at + (uint64_t)n * run), 0, t0 + n < m.n_tiles ? (int)run : 0, 0x00020000);
            acc[n] = v4i{0, 0, 0, 0};
        }
    }
    template <int SET>
    __device__ __forceinline__ void load(uint32_t kt, uint32_t step) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n) w[SET][u][n] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rs[n], (int)((kt + u * step) * 1024u + lane * 16u), 0, 2));
    }
    template <int SET>
    __device__ __forceinline__ void multiply(uint32_t kt, uint32_t step, const uint8_t* x) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = kt + u * step;  // (behind the last the weights are zeros)
            const v4i c = *(const v4i*)(x + 64u * (k < k_tiles ? k : k_tiles - 1u));
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[SET][u][n], c, acc[n], 0, 0, 0);
        }
    }
    // load<0>(first, step) has been called
    __device__ __forceinline__ void run(uint32_t first, uint32_t step, const uint8_t* x) {
        for (uint32_t kt = first; kt < k_tiles; kt += 2u * U * step) {
            load<1>(kt + U * step, step);
            multiply<0>(kt, step, x);
            load<0>(kt + 2u * U * step, step);
            multiply<1>(kt + U * step, step, x);
        }
    }
};

// Lets a kernel take `bytes` of dynamic LDS, once on each device (`allowed`: a bit for each).
hipError_t vx_allow_lds(const void* kernel, uint32_t bytes, std::atomic<uint64_t>& allowed) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess || (allowed.load(std::memory_order_relaxed) >> (device & 63) & 1u)) return e;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess) allowed.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
    return e;
}

constexpr uint32_t kRowWaves = 4;

// One or two rows (STORE, SWIGLU), or one slot's row for its expert (HIDDEN): the first weights are requested, the workgroup
// puts the rows into 8 bits in LDS, its waves take the columns' tiles in turn. Saves the launch that quantizes (one row of 4096 x
// 4096 fp32: 7.6 -> 6.2 us). Bound by latency: the row, its largest value, then 16 KB of weights a wave; one slot's gate and up
// (6 of 64 experts of 2048 x 1408, 35 MB): 9.3 us.
template <class T, int NV, int NT, int EPI>
__global__ __launch_bounds__(64 * kRowWaves) void vx_i8_row_kernel(VxI8Args a, VxI8View x, uint32_t n_blocks) {
    constexpr bool kSwiglu = EPI == VX_I8_SWIGLU || EPI == VX_I8_HIDDEN;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ v4i sums[kRowWaves][NT][64];
    __shared__ uint32_t red[kRowWaves];
    __shared__ float scales[4];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    const uint32_t slot = uniform(blockIdx.x / n_blocks), t0 = uniform(blockIdx.x % n_blocks) * NT, kp = vx_i8_pad(a.w.k);
    uint32_t e = 0, row0 = 0, rows = a.n_rows;
    if constexpr (EPI == VX_I8_HIDDEN) {
        e = uniform(a.ids[slot] - a.first);
        if (e >= a.w.count) return;
        row0 = uniform(slot / a.top);
        rows = 1;
    }
    VxStream<NT> s(a.w, e, t0);
    s.template load<0>(wave, kRowWaves);
    for (uint32_t r = 0; r < rows; ++r) {
        const float f = vx_hold_row<T, 64 * kRowWaves, NV, EPI == VX_I8_HIDDEN && NV == 8>((const T*)x.data + (size_t)(row0 + r) * x.rs, a.w.k, lds + r * kp, threadIdx.x, red);
        if (threadIdx.x == 0) scales[r] = f;
    }
    __syncthreads();
    const uint32_t mine = lane & 15u;
    s.run(wave, kRowWaves, lds + (mine < rows ? mine : 0u) * kp + 16u * (lane >> 4));
#pragma unroll
    for (int n = 0; n < NT; ++n) sums[wave][n][lane] = s.acc[n];
    __syncthreads();
    constexpr uint32_t OUT = kSwiglu ? NT / 2 : NT;
    const uint32_t cols = kSwiglu ? a.w.n / 2u : a.w.n;
    for (uint32_t o = wave; o < OUT; o += kRowWaves) {
        const uint32_t n = kSwiglu ? 2u * o : o, c = 16u * (t0 / (kSwiglu ? 2u : 1u) + o) + 4u * (lane >> 4);
        if (mine >= rows || c >= cols) continue;
        v4i sum = sums[0][n][lane], up = sums[0][kSwiglu ? n + 1u : n][lane];
#pragma unroll
        for (uint32_t w = 1; w < kRowWaves; ++w) {
            sum += sums[w][n][lane];
            if (kSwiglu) up += sums[w][n + 1u][lane];
        }
        const float* ws = a.w.scales + ((uint64_t)e * a.w.n_tiles + t0 + n) * 16u + 4u * (lane >> 4);
        if constexpr (EPI == VX_I8_HIDDEN) *(float4*)(a.part + (size_t)slot * a.part_stride + c) = vx_swiglu(sum, *(const float4*)ws, up, *(const float4*)(ws + 16), scales[0]);
        else vx_outputs<kSwiglu>(a, mine, c, cols, sum, up, ws, scales[mine]);
    }
}

// 16 outputs of a row: each wave takes slots of the row in turn, puts the slot's hidden row into 8 bits in its own piece of LDS
// while its expert's weights are on their way, and multiplies; the answers meet in LDS and are added in the slots' order. Bound by
// latency as above (6 of 64 experts of 2048 x 1408, 17 MB: 9.5 to 10 us by 128 workgroups, half of the CUs).
constexpr uint32_t kAnswerWaves = 8, kAnswerMost = 8u * 4u * 64u;  // values of a hidden row
__global__ __launch_bounds__(64 * kAnswerWaves) void vx_i8_answer_kernel(VxI8Args a, VxCombineArgs c, uint32_t n_blocks) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float answers[kVxMaxTop][16];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    const uint32_t row = uniform(blockIdx.x / n_blocks), t = uniform(blockIdx.x % n_blocks), kp = vx_i8_pad(a.w.k);
    uint8_t* codes = lds + wave * kp;
    for (uint32_t j = wave; j < c.top; j += kAnswerWaves) {
        const uint32_t slot = row * c.top + j, e = uniform(c.ids[slot] - c.first);
        if (e >= c.count) continue;
        VxStream<1> s(a.w, e, t);
        s.load<0>(0, 1);
        const float f = vx_hold_row<float, 64, 8, false>(a.part + (size_t)slot * a.part_stride, (a.w.k + 3u) & ~3u, codes, lane, nullptr);
        vx_wave_sync();
        s.run(0, 1, codes + 16u * (lane >> 4));
        vx_wave_sync();
        if ((lane & 15u) == 0) {
            const float* ws = a.w.scales + ((uint64_t)e * a.w.n_tiles + t) * 16u + 4u * (lane >> 4);
            *(float4*)&answers[j][4u * (lane >> 4)] = vx_scaled<false>(s.acc[0], *(const float4*)ws, f, *(const float4*)ws);
        }
    }
    __syncthreads();
    const uint32_t n = 16u * t + threadIdx.x;
    if (threadIdx.x >= 16u || n >= c.n) return;
    float sum = 0.0f;
    for (uint32_t j = 0; j < c.top; ++j) {
        const uint32_t slot = row * c.top + j;
        if (c.ids[slot] - c.first < c.count) sum = __builtin_fmaf(c.weights[slot], answers[j][threadIdx.x], sum);
    }
    const float res = c.res.data ? vx_load(c.res.data, (size_t)row * c.res.rs + n, c.res.dtype) : 0.0f;
    vx_store(c.out.data, (size_t)row * c.out.rs + n, c.out.dtype, res + sum);
}

template <class T, int NV, int NT, int EPI>
hipError_t vx_i8_row_launch_v(const VxI8Args& a, const VxI8View& x, hipStream_t st) {
    static std::atomic<uint64_t> allowed{0};
    const hipError_t set = vx_allow_lds((const void*)vx_i8_row_kernel<T, NV, NT, EPI>, 1 << 17, allowed);
    if (set != hipSuccess) return set;
    const uint32_t n_blocks = (a.w.n_tiles + NT - 1u) / NT, rows = EPI == VX_I8_HIDDEN ? a.n_rows * a.top : 1u;
    hipLaunchKernelGGL((vx_i8_row_kernel<T, NV, NT, EPI>), dim3(rows * n_blocks), dim3(64 * kRowWaves), vx_i8_pad(a.w.k) * (EPI == VX_I8_HIDDEN ? 1u : a.n_rows), st, a, x, n_blocks);
    return hipGetLastError();
}
template <class T, int NT, int EPI>
hipError_t vx_i8_row_launch(const VxI8Args& a, const VxI8View& x, hipStream_t st) {
    const uint32_t vecs = vx_i8_pad(a.w.k) / (16u / sizeof(T));
    if (vecs <= 64u * kRowWaves) return vx_i8_row_launch_v<T, 1, NT, EPI>(a, x, st);
    if (vecs <= 4u * 64u * kRowWaves) return vx_i8_row_launch_v<T, 4, NT, EPI>(a, x, st);
    return vx_i8_row_launch_v<T, 8, NT, EPI>(a, x, st);
}
template <int NT, int EPI>
hipError_t vx_i8_row_launch_t(const VxI8Args& a, const VxI8View& x, hipStream_t st) {
    if (x.dtype == VELOX_DT_F32) return vx_i8_row_launch<float, NT, EPI>(a, x, st);
    if (x.dtype == VELOX_DT_F16) return vx_i8_row_launch<_Float16, NT, EPI>(a, x, st);
    return vx_i8_row_launch<__bf16, NT, EPI>(a, x, st);
}

// ---- products of many rows: tiles through LDS ----
// A workgroup of WN x WM waves takes 32 WN FN weight rows by 32 WM FM activation rows, a wave 32 FN by 32 FM of them on
// v_mfma_i32_32x32x32_i8 (D[n = 8 (i / 4) + 4 (lane / 32) + i % 4][row = lane % 32]). 128 columns of both go straight to LDS at
// a time, two stages; a column quarter's operands are read while the one before is multiplied, and the barrier between
// two stages stands in front of the last quarter's products, behind which everything of the stage is in registers.
// Weights lie in LDS as in memory (1 KiB tiles, operand reads of 256 neighbouring bytes); an activation row's 16-byte units
// are exchanged by row, so that sixteen rows' reads of one unit meet all 64 banks. What bounds it: at 256 x 256 power (8192 rows of
// 8192 x 29568 in 1480 to 1580 us, 2.5 to 2.7 Pop/s, the matrix cores busy in 74 % of the clocks at 1.4 to 1.7 GHz; 8192 cubed with
// the products removed 371 of 461 us, with the loads removed 388), with few columns the way there and back (64 x 64: 5.2 us).
typedef int v16i __attribute__((ext_vector_type(16)));

// 16 bytes a lane from memory to lds + 16 lane; once: with the non-temporal hint.
__device__ __forceinline__ void vx_to_lds(uint32_t lds, const void* from, uint32_t off, bool once) {
    const uint64_t v = (uint64_t)(uintptr_t)from;  // (a scalar operand, wherever the compiler formed it)
    const uint64_t base = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
    if (once) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
    else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void vx_to_lds(uint32_t lds, const void* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "m0", "memory");
}

// Workgroup b of `total`: the b / 8-th of XCD b % 8 (workgroups are dealt out in turn), each XCD taking a run of neighbours.
__device__ __forceinline__ uint32_t vx_xcd_run(uint32_t b, uint32_t total) {
    const uint32_t x = b & 7u, i = b >> 3, q = total >> 3, r = total & 7u;
    return x * q + (x < r ? x : r) + i;
}

template <int WN, int WM, int FN, int FM, int S, int EPI>
__device__ __forceinline__ void vx_i8_tile(const VxI8Args& a, uint8_t* lds, uint32_t nb, uint32_t e, uint32_t first, uint32_t end, bool once) {
    constexpr int W = WN * WM, TN = 32 * WN * FN, TM = 32 * WM * FM, RB = 128, STAGE = (TN + TM) * RB;  // RB: bytes of a row
    constexpr bool kGrouped = EPI == VX_I8_HIDDEN || EPI == VX_I8_SLOT;
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t wn = wave / WM, wm = wave % WM;
    const uint32_t steps = a.w.k_tiles / 2u, tile0 = nb * (TN / 16);

    // where this wave's share of a stage comes from: weight tiles (two pieces of 1 KiB each), pieces of eight rows
    constexpr int PW = TN / 16 / W, PA = TM / 8 / W, UNITS = RB / 16, AROWS = 64 / UNITS;
    static_assert(PW * 16 * W == TN && PA * 8 * W == TM, "the waves' shares are equal");
    const auto swizzle = [](uint32_t row) { return row >> 1 & 7u; };
    const uint8_t* pw[PW];
    const uint8_t* pa[PA];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const auto piece = [&](int j) { return wave * PA + j; };
#pragma unroll
    for (int j = 0; j < PW; ++j) {
        const uint32_t t = tile0 + wave * PW + j;
        pw[j] = (const uint8_t*)a.w.codes + ((uint64_t)e * a.w.n_tiles + (t < a.w.n_tiles ? t : a.w.n_tiles - 1u)) * a.w.k_tiles * 1024u;
    }
#pragma unroll
    for (int j = 0; j < PA; ++j) {
        const uint32_t p = first + piece(j) * AROWS + lane / UNITS;
        uint32_t row = p < end ? p : end - 1u;
        if constexpr (EPI == VX_I8_HIDDEN) row = a.g.order[row] / a.top;
        pa[j] = (const uint8_t*)a.a.codes + (uint64_t)row * a.a.rs + ((lane % UNITS ^ swizzle(piece(j) * AROWS + lane / UNITS)) * 16u);
    }
    // piece j of this wave's share of a stage into LDS, its pointer moved on
    auto fetch = [&](auto j_, uint32_t stage) {
        constexpr int j = decltype(j_)::value;
        const uint32_t base = lds0 + stage * STAGE;
        if constexpr (j < PW) {
            vx_to_lds(base + (wave * PW + j) * (16u * RB), pw[j], lane * 16u, once);
            vx_to_lds(base + (wave * PW + j) * (16u * RB) + 1024u, pw[j] + 1024, lane * 16u, once);
            pw[j] += 16 * RB;
        } else {
            vx_to_lds(base + TN * RB + piece(j - PW) * 1024u, pa[j - PW]);
            pa[j - PW] += RB;
        }
    };
    // operands of column quarter s: the weights' by tile, the rows' by their unit's place
    const uint32_t w_at = wn * FN * (32u * RB) + ((lane >> 4) & 1u) * (16u * RB) + (lane >> 5) * 256u + (lane & 15u) * 16u;
    uint32_t a_at[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) a_at[s] = TN * RB + (wm * FM * 32u + (lane & 31u)) * RB + (((2u * s + (lane >> 5)) ^ swizzle(lane & 31u)) * 16u);
    // what the epilogue needs: outputs 4 (lane % LANES) .. + 3 of the wave's, the rows lane % 32 of its blocks
    constexpr bool kSwiglu = EPI == VX_I8_SWIGLU || EPI == VX_I8_HIDDEN;
    constexpr int ROW = 32 * FN + 4, LANES = (kSwiglu ? 16 : 32) * FN / 4, AT_ONCE = 64 / LANES;
    const uint32_t cols = kSwiglu ? a.w.n / 2u : a.w.n, col0 = (tile0 * 16u + wn * FN * 32u) / (kSwiglu ? 2u : 1u);
    float4 w0 = make_float4(0, 0, 0, 0), w1 = w0;
    float row_scale[FM];
    uint32_t row_slot[FM];
    {
        const uint32_t c = 4u * (lane % LANES), at = tile0 * 16u + wn * FN * 32u + (kSwiglu ? c / 16u * 32u + c % 16u : c);
        const float* ws = a.w.scales + (uint64_t)e * a.w.n_tiles * 16u + at;
        if (at < a.w.n_tiles * 16u) {
            w0 = *(const float4*)ws;
            if constexpr (kSwiglu) w1 = *(const float4*)(ws + 16);
        }
        if constexpr (EPI == VX_I8_STORE) {
            if (a.bias && at < a.w.n) w1 = vx_load4<false>(a.bias, at, VELOX_DT_F32, a.w.n - at);
        }
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            const uint32_t p = first + (wm * FM + m) * 32u + (lane & 31u), at_p = p < end ? p : end - 1u;
            row_slot[m] = at_p;
            if constexpr (kGrouped) row_slot[m] = a.g.order[at_p];
            row_scale[m] = a.a.scales[EPI == VX_I8_HIDDEN ? row_slot[m] / a.top : at_p];
        }
    }
    v4i fw[2][FN], fa[2][FM];
    v16i acc[FN][FM];
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[n][m][i] = 0;

    // operand r of quarter s: the first of the weights', the rows', the other weights'
    auto read = [&](auto s_, auto r_, uint32_t stage, auto to_) {
        constexpr int s = decltype(s_)::value, r = decltype(r_)::value, to = decltype(to_)::value;
        const uint8_t* base = lds + stage * STAGE;
        if constexpr (r >= 1 && r <= FM) fa[to][r - 1] = *(const v4i*)(base + a_at[s] + (r - 1) * (32 * RB));
        else fw[to][r ? r - FM : 0] = *(const v4i*)(base + w_at + (r ? r - FM : 0) * (32 * RB) + (s >> 1) * 1024 + (s & 1) * 512);
    };
    // The products of the operands in set `from`; between them the next quarter's reads and (LO <= j < HI) the pieces of a
    // stage's fetch. The order is fixed: left to itself the compiler puts the reads together and waits for them.
    auto quarter = [&](auto from_, auto next_, uint32_t stage, auto lo_, auto hi_, uint32_t into) {
        constexpr int from = decltype(from_)::value, next = decltype(next_)::value, LO = decltype(lo_)::value, HI = decltype(hi_)::value;
        constexpr int P = FN * FM, R = FN + FM;
        vx_each<P>([&](auto i_) {
            constexpr int i = decltype(i_)::value, n = i / FM, m = i % FM;
            if constexpr (next >= 0) {
                constexpr int r0 = i * R / P, r1 = (i + 1) * R / P;
                if constexpr (r1 > r0) read(vx_int<(next >= 0 ? next : 0)>{}, vx_int<r0>{}, stage, vx_int<from ^ 1>{});
                if constexpr (r1 > r0 + 1) read(vx_int<(next >= 0 ? next : 0)>{}, vx_int<r0 + 1>{}, stage, vx_int<from ^ 1>{});
            }
            constexpr int d0 = LO + i * (HI - LO) / P, d1 = LO + (i + 1) * (HI - LO) / P;
            if constexpr (d1 > d0) fetch(vx_int<d0>{}, into);
            if constexpr (d1 > d0 + 1) fetch(vx_int<d0 + 1>{}, into);
            static_assert(d1 <= d0 + 2);
            acc[n][m] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[from][n], fa[from][m], acc[n][m], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    constexpr int PIECES = 2 * PW + PA, HALF = (PW + PA) / 2;  // loads of a wave's share of a stage
    auto ready = [&](auto left_) {  // this wave's loads but the last `left` are in LDS, its reads in registers; then everybody's are
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(left_)::value) : "memory");
    };
    uint32_t st = 0;  // stage of step i: i % S
    const auto behind = [&](uint32_t by) { return st + by < (uint32_t)S ? st + by : st + by - (uint32_t)S; };
    // Step i: its stage's quarters. Its own place is free once every wave is past the barrier: stage i + S comes there, half in
    // this step's last quarter (NEXT), half in the next one's first (REST).
    auto step = [&](auto rest_, auto next_) {
        constexpr bool REST = decltype(rest_)::value != 0, NEXT = decltype(next_)::value != 0;
        constexpr int ALL = REST ? PW + PA : HALF;
        quarter(vx_int<0>{}, vx_int<1>{}, st, vx_int<HALF>{}, vx_int<ALL>{}, behind(S - 1));
        quarter(vx_int<1>{}, vx_int<2>{}, st, vx_int<0>{}, vx_int<0>{}, 0);
        quarter(vx_int<0>{}, vx_int<3>{}, st, vx_int<0>{}, vx_int<0>{}, 0);
        ready(vx_int<(REST ? (S - 2) * PIECES : 0)>{});
        quarter(vx_int<1>{}, vx_int<0>{}, behind(1), vx_int<0>{}, vx_int<(NEXT ? HALF : 0)>{}, st);
        st = behind(1);
    };
#pragma unroll
    for (int j = 0; j < S - 1; ++j)
        if ((uint32_t)j < steps) vx_each<PW + PA>([&](auto p) { fetch(p, j); });
    if (steps >= (uint32_t)S) ready(vx_int<(S - 2) * PIECES>{});
    else ready(vx_int<0>{});
    vx_each<FN + FM>([&](auto r) { read(vx_int<0>{}, r, 0, vx_int<0>{}); });
    uint32_t i = 0;
    if (steps >= (uint32_t)S) {
        vx_each<HALF>([&](auto j) { fetch(j, S - 1); });
        for (; i + S < steps; ++i) step(vx_int<1>{}, vx_int<1>{});
        if (S > 1 && i + 1u < steps) {
            step(vx_int<1>{}, vx_int<0>{});
            ++i;
        }
    }
    for (; i + 1u < steps; ++i) step(vx_int<0>{}, vx_int<0>{});
    quarter(vx_int<0>{}, vx_int<1>{}, st, vx_int<0>{}, vx_int<0>{}, 0);
    quarter(vx_int<1>{}, vx_int<2>{}, st, vx_int<0>{}, vx_int<0>{}, 0);
    quarter(vx_int<0>{}, vx_int<3>{}, st, vx_int<0>{}, vx_int<0>{}, 0);
    quarter(vx_int<1>{}, vx_int<-1>{}, 0, vx_int<0>{}, vx_int<0>{}, 0);

    // Epilogue, one block of 32 rows at a time: the sums go through LDS, where the lane of row lane % 32 writes those of n =
    // 8 q + 4 (lane / 32) + 0 .. 3 of every weight block; a row's outputs are then formed by neighbouring lanes, four each, and
    // leave in whole lines. Rolled loops: code that runs once comes through the instruction cache at memory's pace (with the
    // scales applied in front of LDS and everything unrolled a launch took 60 us more).
    static_assert(W * 32 * ROW * 4 <= S * STAGE, "the epilogue's rows lie in the stages");
    int* mine = (int*)lds + wave * 32 * ROW;
    asm volatile("s_barrier" ::: "memory");
    const uint32_t n = col0 + 4u * (lane % LANES);
#pragma unroll 1
    for (int m = 0; m < FM; ++m) {
        vx_each<FM>([&](auto m_) {
            constexpr int mm = decltype(m_)::value;
            if (m == mm) {
#pragma unroll
                for (int b = 0; b < FN; ++b)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *(v4i*)(mine + (lane & 31u) * ROW + 32 * b + 8 * q + 4u * (lane >> 5)) = v4i{acc[b][mm][4 * q], acc[b][mm][4 * q + 1], acc[b][mm][4 * q + 2], acc[b][mm][4 * q + 3]};
            }
        });
        float s = row_scale[0];
        uint32_t slot = row_slot[0];
#pragma unroll
        for (int j = 1; j < FM; ++j) {
            s = m == j ? row_scale[j] : s;
            slot = m == j ? row_slot[j] : slot;
        }
        vx_wave_sync();
        const uint32_t p0 = first + (wm * FM + m) * 32u;
        // DT: an element type (rows of whole vectors), or 3: any type and place
        const auto leave = [&](auto dt_, auto res_) {
            constexpr uint32_t DT = decltype(dt_)::value;
            constexpr bool RES = decltype(res_)::value != 0;
            constexpr int PASSES = 32 / AT_ONCE, TOGETHER = DT < 3u && PASSES > 4 ? 4 : 1;
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += AT_ONCE * TOGETHER) {
                float4 y[TOGETHER], res[TOGETHER];
                uint32_t to[TOGETHER];
                bool live[TOGETHER];
#pragma unroll
                for (int j = 0; j < TOGETHER; ++j) {
                    const uint32_t in = r0 + j * AT_ONCE + lane / LANES;
                    live[j] = p0 + in < end && n < cols;
                    to[j] = EPI == VX_I8_SLOT ? (uint32_t)__shfl((int)slot, (int)in) : p0 + in;
                    if constexpr (RES && DT < 3u) {
                        if (live[j]) res[j] = vx_load4<true>(a.res.data, (size_t)to[j] * a.res.rs + n, DT, cols - n);
                    }
                    const float sr = __shfl(s, (int)in);
                    const int* at = mine + in * ROW;
                    if constexpr (kSwiglu) {
                        const uint32_t c = 4u * (lane % LANES), b = c / 16u * 32u + c % 16u;
                        const v4i g = *(const v4i*)(at + b), u = *(const v4i*)(at + b + 16u);
                        y[j] = vx_swiglu(g, w0, u, w1, sr);
                    } else {
                        const v4i c = *(const v4i*)(at + 4u * (lane % LANES));
                        if (EPI == VX_I8_STORE && a.bias) y[j] = vx_scaled<true>(c, w0, sr, w1);
                        else y[j] = vx_scaled<false>(c, w0, sr, w1);
                    }
                }
#pragma unroll
                for (int j = 0; j < TOGETHER; ++j) {
                    if (!live[j]) continue;
                    if constexpr (kGrouped) {
                        *(float4*)(a.part + (size_t)to[j] * a.part_stride + n) = y[j];  // (rows of whole float4)
                    } else if constexpr (DT < 3u) {
                        if constexpr (RES) y[j] = vx_add(y[j], res[j]);
                        vx_store4<true>(a.out.data, (size_t)to[j] * a.out.rs + n, DT, cols - n, y[j]);
                    } else {
                        vx_finish<false>(a, to[j], n, cols, y[j]);
                    }
                }
            }
        };
        if constexpr (kGrouped) {
            leave(vx_int<VELOX_DT_F32>{}, vx_int<0>{});
        } else {
            const bool res = EPI == VX_I8_STORE && a.res.data;
            if (!a.vec || (res && a.res.dtype != a.out.dtype)) leave(vx_int<3>{}, vx_int<0>{});
            else if (a.out.dtype == VELOX_DT_F32) res ? leave(vx_int<0>{}, vx_int<1>{}) : leave(vx_int<0>{}, vx_int<0>{});
            else if (a.out.dtype == VELOX_DT_F16) res ? leave(vx_int<1>{}, vx_int<1>{}) : leave(vx_int<1>{}, vx_int<0>{});
            else res ? leave(vx_int<2>{}, vx_int<1>{}) : leave(vx_int<2>{}, vx_int<0>{});
        }
        vx_wave_sync();
    }
}

// Plain products: patches of up to 4 row blocks by all weight blocks on an XCD, the rows first.
template <int WN, int WM, int FN, int FM, int S, int EPI>
__global__ __launch_bounds__(64 * WN * WM) void vx_i8_tile_kernel(VxI8Args a, uint32_t row0, uint32_t n_blocks, uint32_t m_blocks) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };  // (quotients are formed in vector registers)
    const uint32_t id = vx_xcd_run(blockIdx.x, n_blocks * m_blocks), patch = id / (4u * n_blocks);
    const uint32_t high = m_blocks - 4u * patch < 4u ? m_blocks - 4u * patch : 4u, in = id - patch * 4u * n_blocks;
    vx_i8_tile<WN, WM, FN, FM, S, EPI>(a, lds, uniform(in / high), 0, uniform(row0 + (4u * patch + in % high) * 32u * WM * FM), a.n_rows, false);
}

// Grouped products: blocks of up to 256 of an expert's positions by 256 weight rows, eight waves of 64 weight rows by half of the
// positions. As many blocks of 64 positions are fetched and multiplied as there are (by tiles of 128, padded, 4096 rows of 8 experts,
// 64 of 256 here, took 978 us, so 830), and the fewer they are, the more stages LDS holds. An expert whose weights one block
// reads passes the caches by (512 rows: 506 -> 465 us). What bounds it there: the weights' way to LDS (the call 839 us; in a build without
// the products, the operands still read, 775, without the rows' loads 801, without the weights' 534, without either 493).
constexpr uint32_t kItemRows = 256u;
template <int L>
struct VxLive {
    static constexpr int stages = L == 1 ? 4 : L == 2 ? 3 : 2;
    static constexpr uint32_t lds = stages * (256 + 64 * L) * 128;
};
template <int EPI>
__global__ __launch_bounds__(512) void vx_i8_items_kernel(VxI8Args a, uint32_t n_blocks) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    if (blockIdx.x >= uniform(*a.g.n_items) * n_blocks) return;
    const uint32_t nb = uniform(blockIdx.x % n_blocks);  // (an item's blocks over all XCDs: items are of unequal length)
    const uint2 it = a.g.items[blockIdx.x / n_blocks];
    const uint32_t e = uniform(it.x), first = uniform(it.y), end = uniform(a.g.offsets[e + 1u]);
    const uint32_t live = end - first < kItemRows ? (end - first + 63u) / 64u : kItemRows / 64u;
    const bool once = end - first <= kItemRows && first == uniform(a.g.offsets[e]);
    vx_each<4>([&](auto l_) {
        constexpr int L = decltype(l_)::value + 1;
        if (live == L) vx_i8_tile<4, 2, 2, L, VxLive<L>::stages, EPI>(a, lds, nb, e, first, end, once);
    });
}

// The same by blocks of 64 positions and 64 weight rows, an item being `parts` of them: for experts so small that the larger
// blocks would leave most CUs idle, and for one product of two whose larger blocks would (below 192 of them: 100 rows, 2 of 4 experts of
// 256 x 14336, 123 -> 58 us by 64 x 64 in the second product; 300 rows, 2 of 8 of 4096 x 8192, 160 blocks, 237 -> 215; 1000 rows,
// 2 of 8 of 4096 x 14336, 240 blocks, 568 -> 641).
constexpr uint32_t kSmallItemRows = 64u;
template <int EPI>
__global__ __launch_bounds__(256) void vx_i8_small_items_kernel(VxI8Args a, uint32_t n_blocks, uint32_t parts) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    const uint32_t block = uniform(blockIdx.x / n_blocks), item = uniform(block / parts);
    if (item >= uniform(*a.g.n_items)) return;
    const uint2 it = a.g.items[item];
    const uint32_t e = uniform(it.x), first = uniform(it.y) + block % parts * kSmallItemRows, end = uniform(a.g.offsets[e + 1u]);
    if (first >= end) return;
    vx_i8_tile<2, 2, 1, 1, 4, EPI>(a, lds, uniform(blockIdx.x % n_blocks), e, uniform(first), end, false);
}

constexpr uint32_t kTileStep = 1u << 20;  // rows of a launch

template <int WN, int WM, int FN, int FM, int S, int EPI>
hipError_t vx_i8_tile_launch(const VxI8Args& a, hipStream_t st) {
    constexpr uint32_t TN = 32 * WN * FN, TM = 32 * WM * FM, lds = S * (TN + TM) * 128;
    static std::atomic<uint64_t> allowed{0};
    const hipError_t set = vx_allow_lds((const void*)vx_i8_tile_kernel<WN, WM, FN, FM, S, EPI>, lds, allowed);
    if (set != hipSuccess) return set;
    const uint32_t n_blocks = (a.w.n_tiles * 16u + TN - 1u) / TN;
    for (uint32_t r = 0; r < a.n_rows; r += kTileStep) {
        const uint32_t rows = a.n_rows - r < kTileStep ? a.n_rows - r : kTileStep, m_blocks = (rows + TM - 1u) / TM;
        hipLaunchKernelGGL((vx_i8_tile_kernel<WN, WM, FN, FM, S, EPI>), dim3(n_blocks * m_blocks), dim3(64 * WN * WM), lds, st, a, r, n_blocks, m_blocks);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}
template <int EPI>
hipError_t vx_i8_items_launch(const VxI8Args& a, hipStream_t st) {
    constexpr uint32_t lds = VxLive<1>::lds, small = 4 * (64 + 64) * 128;
    static_assert(lds <= 160 * 1024 && VxLive<3>::lds <= VxLive<1>::lds && VxLive<2>::lds <= VxLive<1>::lds && VxLive<4>::lds <= VxLive<1>::lds, "a CU's LDS");
    if (a.item_rows == kSmallItemRows || (uint64_t)a.max_items * ((a.w.n_tiles + 15u) / 16u) < 192u) {
        const uint32_t n_blocks = (a.w.n_tiles + 3u) / 4u, parts = a.item_rows / kSmallItemRows;
        hipLaunchKernelGGL((vx_i8_small_items_kernel<EPI>), dim3(a.max_items * parts * n_blocks), dim3(256), small, st, a, n_blocks, parts);
        return hipGetLastError();
    }
    static std::atomic<uint64_t> allowed{0};
    const hipError_t set = vx_allow_lds((const void*)vx_i8_items_kernel<EPI>, lds, allowed);
    if (set != hipSuccess) return set;
    const uint32_t n_blocks = (a.w.n_tiles + 15u) / 16u;
    hipLaunchKernelGGL((vx_i8_items_kernel<EPI>), dim3(a.max_items * n_blocks), dim3(512), lds, st, a, n_blocks);
    return hipGetLastError();
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
    constexpr uint32_t kStep = 1u << 21;  // (a launch has fewer than 2^32 threads, up to 1024 of them a row; limit: fewer rows)
    const uint32_t elt = x.dtype == VELOX_DT_F32 ? 4u : 2u;
    for (uint32_t r = 0; r < n_rows; r += kStep) {
        const VxI8View part{(uint8_t*)x.data + (uint64_t)r * x.rs * elt, x.rs, x.dtype};
        const VxI8Rows to{out.codes + (uint64_t)r * out.rs, out.scales + r, out.rs};
        const uint32_t rows = n_rows - r < kStep ? n_rows - r : kStep;
        const hipError_t e = x.dtype == VELOX_DT_F32   ? vx_quantize_launch<float>(part, rows, k, to, limit, st)
                             : x.dtype == VELOX_DT_F16 ? vx_quantize_launch<_Float16>(part, rows, k, to, limit, st)
                                                       : vx_quantize_launch<__bf16>(part, rows, k, to, limit, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Positions of a block of a grouped product, by the call's slots for each expert held. How many of them go to experts elsewhere is not
// known on the host, so the borders, 12 and 32, lie between what measures best where all are held and where a quarter is. Calls by blocks
// of 16, 32, 64 and 256, us, 8 places a row of experts of 7168 x 2048:
//   slots for each held      64 of 64 here              64 of 256 here
//     8 (64 rows)       453   459   489   508      374   376   418   438
//    16 (128)           650   547   510   530      435   436   481   501
//    32 (256)          1136   867   555   549      471   474   508   526
//    64 (512)          2102  1517   711   606      693   568   528   545
//   128 (1024)         4012  2785  1019   730     1198   906   574   564
// and 6 of 64 of 2048 x 1408, 128 rows (12 slots): 119, 116, 120, 135. What that costs at the borders: all held, 16 to 31 slots, 7 to 12 %
// over blocks of 64; a quarter held, 32 slots, 11 % over blocks of 16. Where blocks of 256 would not even be one for each CU, 64
// (257 rows through 5 experts of 576 x 1100: 36 -> 28 us).
uint32_t vx_i8_item_rows(uint32_t slots, uint32_t count, uint32_t n_tiles) {
    if (slots < 32u * count) return slots >= 12u * count ? 32u : 16u;
    return (uint64_t)(slots / kItemRows + count) * ((n_tiles + 15u) / 16u) < 256u ? kSmallItemRows : kItemRows;
}

// Up to 16 rows the streaming kernel with one weight tile a workgroup (4096 x 4096, one row: two tiles 6.1 us, one 5.0) or,
// where more rows share a tile of a large matrix, two (8192 x 8192, 16 rows: 16.1, 14.2); up to 32 rows two tiles and eight
// waves (8192 x 8192: 17.3, four and four 27.7), four and four from 1024 tiles on (28672 x 4096 paired: 30.0, 23.9), six and four where
// those were over two workgroups a CU (37888 x 3584 paired: 35.6, 31.9, 29.6). From 33 rows on tiles through LDS, as large as
// leave the CUs work: 128 x 32 up to 64 rows (8192 x 8192: 18.1, streaming 21.3), then
//   64 x 64 (four stages) up to 100 tiles of 128 x 128 (1037 rows of 960 x 576: 8.3 -> 4.9 us, 200 of 4096 x 14336: 67 -> 29),
//   128 x 64 (three stages) up to 160 (1000 rows of 2048 x 2048: 10.9 by 64 x 64, 10.1, 16.0 by 128 x 128),
//   128 x 128 (three stages: one workgroup a CU) up to 256 (300 rows of 8192 x 8192: 43 by two stages, 31.6),
//   128 x 128 (two stages: two workgroups a CU) up to 191 tiles of 256 x 256 (2048 rows of 4096 x 4096: 39, by 256 x 256 47),
//   256 x 256: eight waves (8192 rows of 8192 x 8192: 554 by 128 x 128, 466 by four waves, 443), four where the columns are many
//   (of 8192 x 29568: 1555 by eight, 1535; the clock is down to 1.6 GHz then, by power).
template <int EPI>
hipError_t vx_i8_choose(const VxI8Args& a, hipStream_t st) {
    if constexpr (EPI == VX_I8_HIDDEN || EPI == VX_I8_SLOT) {
        if (a.item_rows >= kSmallItemRows) return vx_i8_items_launch<EPI>(a, st);
        return a.item_rows == 32u ? vx_i8_stream_launch<2, 2, 4, EPI>(a, st) : vx_i8_stream_launch<2, 1, 4, EPI>(a, st);
    } else {
        constexpr bool one = EPI == VX_I8_STORE;  // (the others take tiles by pairs)
        const auto tiles = [&](uint32_t by) { return (uint64_t)((a.w.n_tiles * 16u + by - 1u) / by) * ((a.n_rows + by - 1u) / by); };
        if (a.n_rows > 64u) {
            if (tiles(256u) >= 192u)
                return a.w.k > 16384u ? vx_i8_tile_launch<2, 2, 4, 4, 2, EPI>(a, st) : vx_i8_tile_launch<4, 2, 2, 4, 2, EPI>(a, st);
            const uint64_t t = tiles(128u);
            if (t > 256u) return vx_i8_tile_launch<2, 2, 2, 2, 2, EPI>(a, st);
            if (t > 160u) return vx_i8_tile_launch<2, 2, 2, 2, 3, EPI>(a, st);
            if (t > 100u) return vx_i8_tile_launch<2, 2, 2, 1, 3, EPI>(a, st);
            return vx_i8_tile_launch<2, 2, 1, 1, 4, EPI>(a, st);
        }
        if (a.n_rows > 32u) return vx_i8_tile_launch<4, 1, 1, 1, 4, EPI>(a, st);
        if (a.n_rows > 16u) {
            if (a.w.n_tiles > 2048u) return vx_i8_stream_launch<6, 2, 4, EPI>(a, st);
            return a.w.n_tiles >= 1024u ? vx_i8_stream_launch<4, 2, 4, EPI>(a, st) : vx_i8_stream_launch<2, 2, 8, EPI>(a, st);
        }
        if (one && (a.n_rows <= 4u || a.w.n_tiles < 512u)) return vx_i8_stream_launch<one ? 1 : 2, 1, 4, EPI>(a, st);
        return vx_i8_stream_launch<2, 1, 4, EPI>(a, st);
    }
}
hipError_t vx_launch_i8_product(const VxI8Args& a, int epi, hipStream_t st) {
    switch (epi) {
        case VX_I8_STORE: return vx_i8_choose<VX_I8_STORE>(a, st);
        case VX_I8_SWIGLU: return vx_i8_choose<VX_I8_SWIGLU>(a, st);
        case VX_I8_HIDDEN: return vx_i8_choose<VX_I8_HIDDEN>(a, st);
        case VX_I8_SLOT: return vx_i8_choose<VX_I8_SLOT>(a, st);
        default: return hipErrorInvalidValue;
    }
}

// Rows of whole 16-byte vectors.
bool vx_whole_rows(const VxI8View& x, uint32_t k) {
    const uint32_t v = x.dtype == VELOX_DT_F32 ? 4u : 8u;
    return ((uintptr_t)x.data & 15u) == 0 && x.rs % v == 0 && k % v == 0;
}

// One or two rows that stay in the workgroup's registers (4096 x 4096 fp32: one row 7.6 -> 6.2 us, two 8.4 and 8.4 but a launch less
// for the host, four 9.0 -> 12.0; 29568 values, which do not: 44.5 -> 54).
bool vx_i8_by_row(const VxI8View& x, uint32_t n_rows, uint32_t k) {
    return n_rows <= 2u && vx_whole_rows(x, k) && k * (x.dtype == VELOX_DT_F32 ? 4u : 2u) <= 8u * 16u * 64u * kRowWaves;
}
hipError_t vx_launch_i8_row(const VxI8Args& a, const VxI8View& x, int epi, hipStream_t st) {
    if (epi == VX_I8_SWIGLU) return vx_i8_row_launch_t<2, VX_I8_SWIGLU>(a, x, st);
    return vx_i8_row_launch_t<1, VX_I8_STORE>(a, x, st);
}

// Up to four rows whose hidden rows stay in a wave's registers (more: 14336, four rows 121 -> 371 us) and whose slots are dealt to the
// answers' eight waves at most twice (one row, 32 of 64 experts of 1024 x 512: 30.1 and 30.3, all 64 44.7 -> 52.8). It saves three
// launches, up to 8 us, but reads an expert's weights for each slot that names it: worth it while the slots that a choice of the
// held experts at random would give to experts that other rows have too cost less than that again, 4 MB and the weights' bytes
// each, 110 MB in all. Grouped and slot by slot, us (a launch behind the other, weights out of the caches):
//   6 of 64 experts of 2048 x 1408, 1 to 4 rows: 25.8 19.1, 30.8 25.8, 40.5 33.5, 45.7 38.8 (six 52.9 55.9);
//   8 of 8 of 7168 x 2048: 71.4 62.6, by groups from two rows on (74.7 115, 75.0 165, 74.7 214);
//   8 of 32 of 4096 x 1024: 34.5 26.6, 48.6 37.7, 57.0 54.0, four by groups (61.6 70.1);
//   2 of 2 of 4096 x 2048: 24.3 18.2, 25.4 22.6, from three rows on by groups (25.6 30.6, 25.8 35.5);
//   64 places of 5 of 96 x 2048: by groups (25.3 76.5 to 28.9 152).
// Where only a part of the experts is held, fewer slots are here than the rule counts with: 8 of 64 of 2048 x 1408, 8 here, three rows
// go by groups, 17.1 for 12.9.
bool vx_i8_ffn_by_slot(const VxI8View& x, uint32_t n_rows, uint32_t top, uint32_t count, uint32_t hidden, uint32_t inner) {
    if (n_rows > 4u || top > 2u * kAnswerWaves || inner > kAnswerMost || !vx_whole_rows(x, hidden)) return false;
    double unnamed = 1.0;  // the share of the experts that no row names
    for (uint32_t r = 0; r < n_rows; ++r) unnamed *= top < count ? 1.0 - (double)top / count : 0.0;
    const double again = n_rows * top - count * (1.0 - unnamed);
    return again * (3.0 * hidden * inner + 4e6) <= 110e6;
}
hipError_t vx_launch_i8_slots(const VxI8Args& a, const VxI8View& x, hipStream_t st) { return vx_i8_row_launch_t<2, VX_I8_HIDDEN>(a, x, st); }
hipError_t vx_launch_i8_answers(const VxI8Args& a, const VxCombineArgs& c, hipStream_t st) {
    static std::atomic<uint64_t> allowed{0};
    const hipError_t set = vx_allow_lds((const void*)vx_i8_answer_kernel, 1 << 17, allowed);
    if (set != hipSuccess) return set;
    const uint32_t n_blocks = a.w.n_tiles;
    hipLaunchKernelGGL(vx_i8_answer_kernel, dim3(c.n_rows * n_blocks), dim3(64 * kAnswerWaves), vx_i8_pad(a.w.k) * kAnswerWaves, st, a, c, n_blocks);
    return hipGetLastError();
}
