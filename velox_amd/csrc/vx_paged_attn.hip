// vx_paged_attn.hip -- attention over the paged KV cache: one new row per sequence, and prompts' rows.
//
// Softmax runs once over the positions with a running maximum m and sum l per row, in the log2 domain:
// p_j = 2^(x_j - m), o = sum p_j v_j / sum p_j. A chunk is 32 positions of one page: its scores are K Q^T (K rows
// as the A operand straight from the page), which leaves position 16 b + 4 (lane / 16) + r of row lane % 16 in
// register r of tile b -- the order in which the pages' V blocks hold their positions, so the weights are the B
// operand of V^T P^T as they stand.
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

typedef float vx_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t vx_u4 __attribute__((ext_vector_type(4)));

// Eight elements as they lie in memory, at any alignment, to be widened once they are there.
struct VxEight {
    vx_u4 w[2];
    __device__ __forceinline__ void read(const void* p, size_t i, uint32_t dtype) {
        if (dtype == VELOX_DT_F32) __builtin_memcpy(w, (const float*)p + i, 32);
        else __builtin_memcpy(w, (const uint16_t*)p + i, 16);
    }
    __device__ __forceinline__ float at(int i, uint32_t dtype) const {
        const uint32_t f = w[i / 4][i & 3], h = w[0][i / 2] >> 16 * (i & 1) & 0xFFFFu;
        return dtype == VELOX_DT_F32   ? __builtin_bit_cast(float, f)
               : dtype == VELOX_DT_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h)
                                       : __builtin_bit_cast(float, h << 16);
    }
};

// The cache's element type: eight of them are an MFMA operand.
struct VxBf16 {
    typedef __bf16 elt;
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ vx_f4 mfma(v8 a, v8 b, vx_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
struct VxF16 {
    typedef _Float16 elt;
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ vx_f4 mfma(v8 a, v8 b, vx_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// The positions that the row at t sees, as chunks: those of the sinks, then those from the window's first
// position on.
struct VxChunks {
    int64_t t, low;  // newest position, first of the window
    uint32_t sink, n, low_chunk;  // chunks before the window, chunks in all, the window's first chunk
    uint32_t sinks;
};
__device__ __forceinline__ VxChunks vx_chunks(int64_t t, uint32_t window, uint32_t sinks) {
    VxChunks c;
    c.t = t;
    c.sinks = sinks;
    c.low = window && t + 1 > (int64_t)window ? t + 1 - (int64_t)window : 0;
    c.low_chunk = (uint32_t)(c.low >> 5);
    const uint32_t s = min((uint32_t)((min((int64_t)sinks, c.low) + 31) >> 5), c.low_chunk);
    c.sink = s;
    c.n = t < 0 ? 0 : s + (uint32_t)(t >> 5) - c.low_chunk + 1;
    return c;
}
__device__ __forceinline__ uint32_t vx_chunk_base(const VxChunks& c, uint32_t i) {
    return (i < c.sink ? i : c.low_chunk + (i - c.sink)) << 5;
}

// ---- one new row per sequence ----
// A workgroup takes one split of one sequence's chunks for up to 16 q heads of a KV head (the columns of the score
// tiles); its waves take the split's chunks in turn and meet in LDS. A wave holds one chunk's K and V (16 KB at
// head size 128) in registers while the next one's are on their way. q of another type than the cache's enters as
// QT terms of the cache's type whose sum keeps fp32's precision (three of bf16; two of fp16, of which each
// head's largest value is brought to 2^14 first, so that the second term stays in range), the weights as PT.
constexpr int kTokenWaves = 4;
constexpr int kTokenThreads = 64 * kTokenWaves;

template <class E, int D, int QT, int PT>
__global__ __launch_bounds__(kTokenThreads, 2) void vx_paged_token_kernel(VxPagedAttnArgs a) {
    constexpr int NC = D / 32, NB = D / 16, OP = D + 4;  // OP: row pitch of the waves' sums in LDS
    typedef typename E::v8 v8;
    __shared__ __attribute__((aligned(16))) float s_o[kTokenWaves * 16 * OP];
    __shared__ float s_m[kTokenWaves * 16], s_l[kTokenWaves * 16];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = lane & 15u, grp = lane >> 4;
    const uint32_t G = a.q.heads / a.c.hkv, ng = (G + 15) / 16;
    const uint32_t kvh = blockIdx.y / ng, g0 = blockIdx.y % ng * 16, gn = min(16u, G - g0);
    const uint32_t seq = blockIdx.z, split = blockIdx.x, h0 = kvh * G + g0;
    // q: column col is head h0 + col. The requests go out first; the first chunk's follow before q is widened.
    VxEight raw[NC];
    if (col < gn) {
#pragma unroll
        for (int c = 0; c < NC; ++c) raw[c].read(a.q.data, (size_t)seq * a.q.rs + (size_t)(h0 + col) * a.q.hs + 32 * c + 8 * grp, a.q.dtype);
    }
    const VxChunks ch = vx_chunks((int64_t)a.c.lens[seq] - 1, a.window, a.sinks);
    const uint32_t per = (ch.n + a.splits - 1) / a.splits;
    const uint32_t c0 = min(split * per, ch.n), c1 = min(c0 + per, ch.n);
    const uint32_t* table = a.c.table + (size_t)seq * a.c.table_stride;

    // page and place of the wave's next 64 chunks, one a lane
    uint32_t pages, places;
    const auto look_up = [&](uint32_t k0) {
        const uint32_t i = c0 + wave + kTokenWaves * (k0 + lane);
        pages = kVxNoPage;
        places = 0;
        if (i < c1) {
            const uint32_t base = vx_chunk_base(ch, i), j = base / a.c.page_size;
            places = base - j * a.c.page_size;
            if (j < a.c.max_pages) pages = table[j];
        }
    };
    look_up(0);

    struct Chunk {
        v8 k[2][NC], v[NB];
    };
    const uint32_t n_mine = c1 > c0 + wave ? (c1 - c0 - wave + kTokenWaves - 1) / kTokenWaves : 0;
    const auto load = [&](Chunk& x, uint32_t page, uint32_t place) {
        const uint16_t* kp = (const uint16_t*)(a.c.pool + (size_t)(page < a.c.n_pages ? page : 0u) * a.c.page_bytes);
        const uint16_t* vp = kp + ((size_t)a.c.hkv * a.c.page_size + (size_t)kvh * a.c.page_size + place) * D;
        kp += ((size_t)kvh * a.c.page_size + place) * D;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < NC; ++c) x.k[b][c] = *(const v8*)(kp + (16 * b + col) * D + 32 * c + 8 * grp);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) x.v[nb] = *(const v8*)(vp + (16 * nb + col) * 32 + 8 * grp);
    };
    const auto page_of = [&](uint32_t k) { return (uint32_t)__builtin_amdgcn_readlane((int)pages, (int)(k & 63u)); };
    const auto place_of = [&](uint32_t k) { return (uint32_t)__builtin_amdgcn_readlane((int)places, (int)(k & 63u)); };
    const auto base_of = [&](uint32_t k) { return vx_chunk_base(ch, c0 + wave + kTokenWaves * k); };
    Chunk x, y;
    uint32_t px = kVxNoPage, py = kVxNoPage;
    if (n_mine) {
        px = page_of(0);
        load(x, px, place_of(0));
    }

    v8 qf[QT][NC];  // zero past the last head
    float to_log2 = a.scale * kLog2e;
    {
        float x[NC][8];
        float big = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[c][i] = col < gn ? raw[c].at(i, a.q.dtype) : 0.0f;
                big = fmaxf(big, fabsf(x[c][i]));
            }
        if constexpr (QT == 2) {
            big = fmaxf(big, __shfl_xor(big, 16));
            big = fmaxf(big, __shfl_xor(big, 32));
            const int e = big > 0.0f && big < INFINITY ? 14 - ilogbf(big) : 0;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[c][i] = ldexpf(x[c][i], e);
            to_log2 = ldexpf(to_log2, -e);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float rest = x[c][i];
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    const typename E::elt v = (typename E::elt)rest;
                    qf[t][c][i] = v;
                    rest -= (float)v;
                }
            }
    }

    vx_f4 o[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) o[nb] = vx_f4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    const auto use = [&](Chunk& x, uint32_t page, uint32_t base) {
        if (page >= a.c.n_pages) return;
        vx_f4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            s[b] = vx_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = QT - 1; t >= 0; --t)
#pragma unroll
                for (int c = 0; c < NC; ++c) s[b] = E::mfma(x.k[b][c], qf[t][c], s[b]);
            s[b] *= to_log2;
        }
        if ((int64_t)base < ch.low || (int64_t)base + 31 > ch.t) {  // some positions are hidden: their places may hold anything
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t keep[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t p = (int64_t)base + 16 * b + 4 * grp + r;
                    const bool seen = p <= ch.t && (p >= ch.low || p < (int64_t)ch.sinks);
                    if (!seen) s[b][r] = -INFINITY;
                    keep[r] = seen ? 0xFFFFu : 0u;
                }
                const uint32_t w0 = keep[0] | keep[1] << 16, w1 = keep[2] | keep[3] << 16;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    vx_u4 w = __builtin_bit_cast(vx_u4, x.v[nb]);
                    w[2 * b] &= w0;
                    w[2 * b + 1] &= w1;
                    x.v[nb] = __builtin_bit_cast(v8, w);
                }
            }
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
        const float r = __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        v8 pf[PT];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i / 4][i % 4] - ref);
            sum += p;
            float rest = p;
#pragma unroll
            for (int t = 0; t < PT; ++t) {
                const typename E::elt v = (typename E::elt)rest;
                pf[t][i] = v;
                rest -= (float)v;
            }
        }
        l = l * r + sum;
        if (__ballot(r != 1.0f)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[nb] *= r;
        }
#pragma unroll
        for (int t = PT - 1; t >= 0; --t)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[nb] = E::mfma(x.v[nb], pf[t], o[nb]);
    };
    for (uint32_t k = 0; k < n_mine; k += 2) {
        if (k + 1 < n_mine) {
            py = page_of(k + 1);
            load(y, py, place_of(k + 1));
        }
        use(x, px, base_of(k));
        if (k + 1 >= n_mine) break;
        if (k + 2 < n_mine) {
            if (((k + 2) & 63u) == 0) look_up(k + 2);
            px = page_of(k + 2);
            load(x, px, place_of(k + 2));
        }
        use(y, py, base_of(k + 1));
    }

    // the waves' (m, l, o) meet
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (col < gn) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) *(vx_f4*)(s_o + (wave * 16 + col) * OP + 16 * nb + 4 * grp) = o[nb];
        if (grp == 0) {
            s_m[wave * 16 + col] = m;
            s_l[wave * 16 + col] = l;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < gn * D; i += kTokenThreads) {
        const uint32_t c = i / D, e = i % D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kTokenWaves; ++w) top = fmaxf(top, s_m[w * 16 + c]);
        const float ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kTokenWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w * 16 + c] - ref);
            sum += f * s_l[w * 16 + c];
            acc += f * s_o[(w * 16 + c) * OP + e];
        }
        if (a.splits == 1) {
            vx_store(a.out.data, (size_t)seq * a.out.rs + (size_t)(h0 + c) * a.out.hs + e, a.out.dtype, ch.n && sum != 0.0f ? acc / sum : 0.0f);
        } else {
            const size_t part = ((size_t)seq * a.q.heads + h0 + c) * a.splits + split;
            a.part_o[part * D + e] = acc;
            if (e == 0) {
                a.part_ml[2 * part] = top;
                a.part_ml[2 * part + 1] = sum;
            }
        }
    }
}

// Joins a row's splits: a workgroup per (row, head), each of its waves over a quarter of the splits.
template <int D>
__global__ __launch_bounds__(256) void vx_paged_join_kernel(VxPagedAttnArgs a) {
    constexpr int N = D / 64;
    __shared__ float s_acc[4][D];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t row = blockIdx.x / a.q.heads, h = blockIdx.x % a.q.heads;
    const float* ml = a.part_ml + 2 * (size_t)blockIdx.x * a.splits;
    const float* po = a.part_o + (size_t)blockIdx.x * a.splits * D + lane * N;
    const uint32_t per = (a.splits + 3) / 4, s0 = min(wave * per, a.splits), s1 = min(s0 + per, a.splits);
    float v[16][N];  // per <= 16; requested before the weights are known
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (s0 + i < s1) __builtin_memcpy(v[i], po + (size_t)(s0 + i) * D, 4 * N);
    float m = -INFINITY, sum = 0.0f;
    if (lane < a.splits) {  // at most 64
        m = ml[2 * lane];
        sum = ml[2 * lane + 1];
    }
    float top = m;
#pragma unroll
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
    sum *= f;
#pragma unroll
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (s0 + i < s1) {
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), (int)(s0 + i)));
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += w * v[i][e];
        }
#pragma unroll
    for (int e = 0; e < N; ++e) s_acc[wave][lane * N + e] = acc[e];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < D; e += 256) {
        const float o = (s_acc[0][e] + s_acc[1][e]) + (s_acc[2][e] + s_acc[3][e]);
        vx_store(a.out.data, (size_t)row * a.out.rs + (size_t)h * a.out.hs + e, a.out.dtype, sum != 0.0f ? o / sum : 0.0f);
    }
}

hipError_t launch_join(const VxPagedAttnArgs& a, hipStream_t st) {
    const uint64_t items = (uint64_t)a.n_rows * a.q.heads;
    if (a.c.d == 64) vx_paged_join_kernel<64><<<(uint32_t)items, 256, 0, st>>>(a);
    else vx_paged_join_kernel<128><<<(uint32_t)items, 256, 0, st>>>(a);
    return hipGetLastError();
}

template <class E, int D, int QT, int PT>
hipError_t launch_token(const VxPagedAttnArgs& a, hipStream_t st) {
    const uint32_t G = a.q.heads / a.c.hkv;
    vx_paged_token_kernel<E, D, QT, PT><<<dim3(a.splits, a.c.hkv * ((G + 15) / 16), a.c.n_seqs), kTokenThreads, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || a.splits == 1 ? e : launch_join(a, st);
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

// Splits of the token form: workgroups for about two rounds of the GPU (a sequence's own length decides how many
// chunks a split has, so unequal sequences even out), each with a chunk at least for every wave.
uint32_t vx_paged_attn_splits(const VxPagedView& c, uint32_t heads, uint32_t rows, uint32_t max_len) {
    const uint32_t units = rows * c.hkv * ((heads / c.hkv + 15) / 16), chunks = (max_len + 31) / 32;
    const uint32_t want = (512 + units - 1) / units, most = (chunks + kTokenWaves - 1) / kTokenWaves;
    const uint32_t s = want < most ? want : most;
    return s < 1 ? 1 : s > 64 ? 64 : s;
}

hipError_t vx_launch_paged_attention(const VxPagedAttnArgs& a, hipStream_t st) {
    const bool same = a.q.dtype == a.c.dtype, bf16 = a.c.dtype == VELOX_DT_BF16;
    if (a.c.d == 64) {
        if (bf16) return same ? launch_token<VxBf16, 64, 1, 2>(a, st) : launch_token<VxBf16, 64, 3, 3>(a, st);
        return same ? launch_token<VxF16, 64, 1, 2>(a, st) : launch_token<VxF16, 64, 2, 2>(a, st);
    }
    if (bf16) return same ? launch_token<VxBf16, 128, 1, 2>(a, st) : launch_token<VxBf16, 128, 3, 3>(a, st);
    return same ? launch_token<VxF16, 128, 1, 2>(a, st) : launch_token<VxF16, 128, 2, 2>(a, st);
}

uint32_t vx_paged_prompt_splits(const VxPagedView&, uint32_t, uint32_t, uint32_t, uint32_t) { return 1; }
hipError_t vx_launch_paged_prompt(const VxPagedAttnArgs& a, hipStream_t st) { return launch_rows(a, st); }
