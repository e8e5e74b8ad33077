// vx_paged_attn.hip -- attention over the paged KV cache: one new row per sequence, and prompts' rows.
#include "vx_paged.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float vx_load(const void* p, size_t i, uint32_t dtype) {
    if (dtype == VELOX_DT_F32) return ((const float*)p)[i];
    if (dtype == VELOX_DT_F16) return (float)((const _Float16*)p)[i];
    return (float)((const __bf16*)p)[i];
}
__device__ __forceinline__ void vx_store(void* p, size_t i, uint32_t dtype, float v) {
    if (dtype == VELOX_DT_F32) ((float*)p)[i] = v;
    else if (dtype == VELOX_DT_F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}

// One wave per (row, head): lanes over the head's dimensions, a running maximum and sum over the positions.
template <int D>
__global__ __launch_bounds__(256) void vx_paged_rows_kernel(VxPagedAttnArgs a) {
    constexpr int E = D / 64;
    const uint32_t lane = threadIdx.x & 63u, row = blockIdx.x;
    const uint32_t h = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (h >= a.q.heads) return;
    uint32_t seq = row;
    int64_t t;
    if (a.q_start) {
        seq = a.c.n_seqs;
        for (uint32_t s = 0; s < a.c.n_seqs; ++s)
            if (row >= a.q_start[s] && row < a.q_start[s + 1]) seq = s;
        if (seq == a.c.n_seqs) return;
        t = (int64_t)a.c.lens[seq] - (int64_t)(min(a.q_start[seq + 1], a.n_rows) - row);
        if (t < 0) return;
    } else {
        t = (int64_t)a.c.lens[seq] - 1;
    }
    const uint32_t g = h / (a.q.heads / a.c.hkv);
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) {
        q[e] = vx_load(a.q.data, (size_t)row * a.q.rs + (size_t)h * a.q.hs + lane * E + e, a.q.dtype) * a.scale * kLog2e;
        o[e] = 0.0f;
    }
    const int64_t low = a.window && t + 1 > (int64_t)a.window ? t + 1 - (int64_t)a.window : 0;
    for (int64_t p = 0; p <= t; ++p) {
        if (p < low && p >= (int64_t)a.sinks) p = low;
        const uint64_t j = (uint64_t)p / a.c.page_size;
        const uint32_t in = (uint32_t)((uint64_t)p % a.c.page_size);
        const uint32_t page = j < a.c.max_pages ? a.c.table[(size_t)seq * a.c.table_stride + j] : kVxNoPage;
        if (page >= a.c.n_pages) continue;
        const uint16_t* kp = (const uint16_t*)(a.c.pool + (size_t)page * a.c.page_bytes);
        const uint16_t* vp = kp + ((size_t)a.c.hkv * a.c.page_size + (size_t)g * a.c.page_size + (in & ~31u)) * D;
        kp += ((size_t)g * a.c.page_size + in) * D;
        float s = 0.0f;
        for (int e = 0; e < E; ++e) s += q[e] * vx_load(kp, lane * E + e, a.c.dtype);
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
        const float mn = fmaxf(m, s), r = m == -INFINITY ? 0.0f : exp2f(m - mn), w = exp2f(s - mn);
        l = l * r + w;
        for (int e = 0; e < E; ++e) o[e] = o[e] * r + w * vx_load(vp, (size_t)(lane * E + e) * 32 + vx_vslot(in & 31u), a.c.dtype);
        m = mn;
    }
    for (int e = 0; e < E; ++e)
        vx_store(a.out.data, (size_t)row * a.out.rs + (size_t)h * a.out.hs + lane * E + e, a.out.dtype, l > 0.0f ? o[e] / l : 0.0f);
}

hipError_t launch_rows(const VxPagedAttnArgs& a, hipStream_t st) {
    const dim3 grid(a.n_rows, (a.q.heads + 3) / 4);
    if (a.c.d == 64) vx_paged_rows_kernel<64><<<grid, 256, 0, st>>>(a);
    else vx_paged_rows_kernel<128><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

uint32_t vx_paged_attn_splits(const VxPagedView&, uint32_t, uint32_t, uint32_t) { return 1; }
hipError_t vx_launch_paged_attention(const VxPagedAttnArgs& a, hipStream_t st) { return launch_rows(a, st); }
uint32_t vx_paged_prompt_splits(const VxPagedView&, uint32_t, uint32_t, uint32_t, uint32_t) { return 1; }
hipError_t vx_launch_paged_prompt(const VxPagedAttnArgs& a, hipStream_t st) { return launch_rows(a, st); }
