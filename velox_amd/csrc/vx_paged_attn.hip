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
typedef float vx_f16 __attribute__((ext_vector_type(16)));
typedef uint32_t vx_u4 __attribute__((ext_vector_type(4)));

// Eight elements as they lie in memory, at any alignment, to be widened once they are there.
struct VxEight {
    vx_u4 w[2];
};
// N of them, `step` elements apart from element i on. HALF: no fp32. One branch for all, so that no read waits for another.
template <bool HALF, int N>
__device__ __forceinline__ void vx_request(VxEight (&raw)[N], const void* p, size_t i, uint32_t step, uint32_t dtype) {
    if (!HALF && dtype == VELOX_DT_F32) {
#pragma unroll
        for (int c = 0; c < N; ++c) __builtin_memcpy(raw[c].w, (const float*)p + i + step * c, 32);
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) __builtin_memcpy(raw[c].w, (const uint16_t*)p + i + step * c, 16);
    }
}
template <int N>
__device__ __forceinline__ void vx_widen(const VxEight (&raw)[N], uint32_t dtype, float (&x)[N][8]) {
    if (dtype == VELOX_DT_F32) {
        asm volatile("");  // three branches, not selects of three values each
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t f = raw[c].w[i / 4][i & 3];
                x[c][i] = __builtin_bit_cast(float, f);
            }
    } else if (dtype == VELOX_DT_F16) {
        asm volatile("");
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint16_t h = (uint16_t)(raw[c].w[0][i / 2] >> 16 * (i & 1));
                x[c][i] = (float)__builtin_bit_cast(_Float16, h);
            }
    } else {
        asm volatile("");
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t f = i & 1 ? raw[c].w[0][i / 2] & 0xFFFF0000u : raw[c].w[0][i / 2] << 16;
                x[c][i] = __builtin_bit_cast(float, f);
            }
    }
}
// The power of two that brings a head's largest value to [2^13, 2^14) (none for 0, infinities and NaN; of values below
// 2^-87 no more than 2^100, so that it stays a number).
__device__ __forceinline__ int vx_to_2_14(float big) {
    return big > 0.0f && big < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(big), 100) : 0;
}
// Four values side by side, each rounded once, at any alignment.
__device__ __forceinline__ void vx_store4(void* p, size_t i, uint32_t dtype, vx_f4 v) {
    if (dtype == VELOX_DT_F32) {
        __builtin_memcpy((float*)p + i, &v, 16);
    } else if (dtype == VELOX_DT_F16) {
        const _Float16 h[4] = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        __builtin_memcpy((uint16_t*)p + i, h, 8);
    } else {
        const __bf16 h[4] = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        __builtin_memcpy((uint16_t*)p + i, h, 8);
    }
}

// The cache's element type: eight of them are an MFMA operand.
struct VxBf16 {
    typedef __bf16 elt;
    static constexpr uint32_t kExp = 0x7F80u, kOne = 0x0080u;  // the exponent's bits, and the lowest of them
    static constexpr float kUp = 0.0f, kUpTerms = 0.0f;         // the weights are taken times 2^kUp (kUpTerms: in the token form)
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ vx_f4 mfma(v8 a, v8 b, vx_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ vx_f16 mfma(v8 a, v8 b, vx_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
struct VxF16 {
    typedef _Float16 elt;
    static constexpr uint32_t kExp = 0x7C00u, kOne = 0x0400u;
    // fp16 weights lose bits below 2^-14 and are 0 below 2^-25: they are moved up as far as the largest allows
    static constexpr float kUp = 7.0f, kUpTerms = 14.0f;
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ vx_f4 mfma(v8 a, v8 b, vx_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ vx_f16 mfma(v8 a, v8 b, vx_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// The positions that the rows at first .. last see, as chunks: those of the sinks, then those from the first
// row's window on.
struct VxChunks {
    int64_t t, low;               // newest position, first of the first row's window
    uint32_t sink, n, low_chunk;  // chunks before the window, chunks in all, the window's first chunk
    uint32_t sinks;
};
__device__ __forceinline__ int64_t vx_low(int64_t t, uint32_t window) {
    return window && t + 1 > (int64_t)window ? t + 1 - (int64_t)window : 0;
}
// cap: positions the table has entries for; the walk ends there, however long the sequence says it is.
__device__ __forceinline__ VxChunks vx_chunks(int64_t first, int64_t last, uint32_t window, uint32_t sinks, uint64_t cap) {
    VxChunks c;
    c.t = last;
    c.sinks = sinks;
    c.low = vx_low(first, window);
    c.low_chunk = (uint32_t)(c.low >> 5);
    const uint32_t end = (uint32_t)((min((uint64_t)(last + 1), cap) + 31) >> 5);  // chunks in all, the hidden ones too
    c.sink = min(min((uint32_t)((min((int64_t)sinks, c.low) + 31) >> 5), c.low_chunk), end);
    c.n = last < 0 ? 0 : c.sink + (end > c.low_chunk ? end - c.low_chunk : 0u);
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
// head's largest value is brought to 2^13 first, so that the second term stays in range), the weights as PT.
// Bound by the bytes of K and V where there are many: 4 sequences of 107243 to 131000 positions of Llama-3-8B's heads 292 us
// (6.7 TB/s); by latency (lengths, table, first chunk, the join) below: 32 sequences of 600 to 2100 positions of
// Qwen2.5-7B's heads (90 MB) 19.6 us, one SmolLM sequence of 700 7.5 us (21.7 and 8.6 while the waits for a chunk were
// waits for the next one too). Four waves: eight were slower where the GPU is full (25.4 against 22.9 us for 32 sequences
// of 1500); with few workgroups more waves were not tried.
// Non-temporal loads (NT) where the caches cannot hold the K and V anyway: Llama-3-8B's heads, 4 sequences of 107243 to
// 131000 positions 330 -> 292 us (5.9 -> 6.7 TB/s); 32 sequences of Qwen2.5-7B (90 MB, in the memory-side cache from
// one call to the next) 21.8 us without, 23.6 with.
constexpr uint64_t kTokenCached = 256ull << 20;  // bytes of the memory-side cache
constexpr int kTokenWaves = 4;
constexpr int kTokenThreads = 64 * kTokenWaves;

template <class E, int D, int QT, int PT, bool NT>
__global__ __launch_bounds__(kTokenThreads, 2) void vx_paged_token_kernel(VxPagedAttnArgs a) {
    constexpr int NC = D / 32, NB = D / 16, OP = D + 4;  // OP: row pitch of the waves' sums in LDS
    typedef typename E::v8 v8;
    __shared__ __attribute__((aligned(16))) float s_o[kTokenWaves * 16 * OP];
    __shared__ float s_m[kTokenWaves * 16], s_l[kTokenWaves * 16];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t col = lane & 15u, grp = lane >> 4;
    const uint32_t G = a.q.heads / a.c.hkv, ng = (G + 15) / 16;
    const uint32_t kvh = blockIdx.y / ng, g0 = blockIdx.y % ng * 16, gn = min(16u, G - g0);
    const uint32_t seq = blockIdx.z, split = blockIdx.x, h0 = kvh * G + g0;
    // q: column col is head h0 + col. The requests go out first; the first chunk's follow before q is widened.
    VxEight raw[NC] = {};
    if (col < gn) vx_request<QT == 1>(raw, a.q.data, (size_t)seq * a.q.rs + (size_t)(h0 + col) * a.q.hs + 8 * grp, 32, a.q.dtype);
    const int64_t t = (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)a.c.lens[seq]) - 1;
    const VxChunks ch = vx_chunks(t, t, a.window, a.sinks, (uint64_t)a.c.max_pages * a.c.page_size);
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
        // waited for here: at every later use the wait would be for all that is on its way by then, the next chunk too
        asm volatile("" : "+v"(pages));
    };
    look_up(0);

    struct Chunk {
        v8 k[2][NC], v[NB];
    };
    const uint32_t n_mine = c1 > c0 + wave ? (c1 - c0 - wave + kTokenWaves - 1) / kTokenWaves : 0;
    // this lane's bytes of a chunk's K and V. Buffer loads: a uniform base, one offset a lane for all of them, and nothing
    // (0) is read of a page that is not there
    const uint32_t k_at = (col * D + 8 * grp) * 2, v_at = (col * 32 + 8 * grp) * 2;
    const auto load = [&](Chunk& x, uint32_t page, uint32_t place) {
        const bool have = page < a.c.n_pages;
        uint8_t* kp = a.c.pool + (size_t)(have ? page : 0u) * a.c.page_bytes + ((size_t)kvh * a.c.page_size + place) * (D * 2);
        const int bytes = have ? 64 * D : 0;
        const auto kr = __builtin_amdgcn_make_buffer_rsrc(kp, (short)0, bytes, 0x00020000);
        const auto vr = __builtin_amdgcn_make_buffer_rsrc(kp + (size_t)a.c.hkv * a.c.page_size * (D * 2), (short)0, bytes, 0x00020000);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < NC; ++c) x.k[b][c] = __builtin_bit_cast(v8, __builtin_amdgcn_raw_buffer_load_b128(kr, k_at + 64 * c, b * 32 * D, NT ? 2 : 0));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            x.v[nb] = __builtin_bit_cast(v8, __builtin_amdgcn_raw_buffer_load_b128(vr, v_at + nb % 4 * 1024, nb / 4 * 4096, NT ? 2 : 0));
        __builtin_amdgcn_sched_barrier(0);  // requested before the chunk at hand is multiplied
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
        vx_widen(raw, a.q.dtype, x);
        if constexpr (QT == 2) {
            float big = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[c][i]));
            big = fmaxf(big, __shfl_xor(big, 16));
            big = fmaxf(big, __shfl_xor(big, 32));
            const int e = vx_to_2_14(big);
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
        const bool have = page < a.c.n_pages;
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
        if (!have || (int64_t)base < ch.low || (int64_t)base + 31 > ch.t) {  // some positions are hidden: their places may hold anything
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t keep[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t p = (int64_t)base + 16 * b + 4 * grp + r;
                    const bool seen = have & (p <= ch.t) & ((p >= ch.low) | (p < (int64_t)ch.sinks));
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
        const float r = __builtin_amdgcn_exp2f(m - ref), from = ref - E::kUpTerms;
        m = mn;
        v8 pf[PT];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i / 4][i % 4] - from);
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
    // Chunk k + 2 is requested whether there is one or not (then nothing is read): behind a branch the wait for chunk
    // k + 1 would be one for it as well.
    uint32_t k = 0;
    for (; k + 2 <= n_mine; k += 2) {
        py = page_of(k + 1);
        load(y, py, place_of(k + 1));
        use(x, px, base_of(k));
        if (((k + 2) & 63u) == 0) look_up(k + 2);
        px = page_of(k + 2);
        load(x, px, place_of(k + 2));
        use(y, py, base_of(k + 1));
    }
    if (k < n_mine) use(x, px, base_of(k));

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

// Joins a row's splits: W waves for a (row, head), each over its part of the splits: one where there are few splits or many
// rows, which then take few workgroups and no barrier (2000 prompt rows of SmolLM in 3 splits, both kernels, with weights of one term, 29 us by one,
// 43 by four), else four (4 sequences of 2000 positions of Llama-3-8B in 8 splits 9.9 us, by one 10.3). A launch's
// latency where there are few. Maxima and sums are requested first: they are joined while the rest arrives. Of a prompt's
// rows, those of no sequence and those in front of position 0 (their sums say -1) are passed over.
template <int D, int W>
__global__ __launch_bounds__(256) void vx_paged_join_kernel(VxPagedAttnArgs a, uint32_t items) {
    constexpr int N = D / 64;
    __shared__ float s_acc[W == 4 ? 4 : 1][D];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t item = W == 4 ? blockIdx.x : blockIdx.x * 4 + wave;
    if (item >= items) return;
    const uint32_t row = item / a.q.heads, h = item % a.q.heads;
    const float* ml = a.part_ml + 2 * (size_t)item * a.splits;
    float m = -INFINITY, sum = 0.0f;
    if (lane < a.splits) {  // at most 64 (W 1: 16)
        m = ml[2 * lane];
        sum = ml[2 * lane + 1];
    }
    if (a.q_start && (row < vx_word(a.q_start) || row >= vx_word(a.q_start + a.c.n_seqs) || ml[1] < 0.0f)) return;
    const float* po = a.part_o + (size_t)item * a.splits * D + lane * N;
    const uint32_t per = (a.splits + W - 1) / W, s0 = W == 4 ? min(wave * per, a.splits) : 0u, s1 = min(s0 + per, a.splits);
    float v[16][N];  // per <= 16; requested before the weights are known
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (s0 + i < s1) __builtin_memcpy(v[i], po + (size_t)(s0 + i) * D, 4 * N);
    float top = m;
#pragma unroll
    for (int x = W == 4 ? 32 : 8; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
    sum *= f;
#pragma unroll
    for (int x = W == 4 ? 32 : 8; x; x >>= 1) sum += __shfl_xor(sum, x);
    sum = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sum)));
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
    const auto put = [&](uint32_t e, float o) {
        vx_store(a.out.data, (size_t)row * a.out.rs + (size_t)h * a.out.hs + e, a.out.dtype, sum != 0.0f ? o / sum : 0.0f);
    };
    if constexpr (W == 4) {
#pragma unroll
        for (int e = 0; e < N; ++e) s_acc[wave][lane * N + e] = acc[e];
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < D; e += 256) put(e, (s_acc[0][e] + s_acc[1][e]) + (s_acc[2][e] + s_acc[3][e]));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) put(lane * N + e, acc[e]);
    }
}

hipError_t launch_join(const VxPagedAttnArgs& a, hipStream_t st) {
    const uint32_t items = a.n_rows * a.q.heads;
    const auto go = [&](auto kernel, uint32_t grid) { kernel<<<grid, 256, 0, st>>>(a, items); };
    if (a.splits > 16 || (a.splits > 4 && items < 4096)) go(a.c.d == 64 ? vx_paged_join_kernel<64, 4> : vx_paged_join_kernel<128, 4>, items);
    else go(a.c.d == 64 ? vx_paged_join_kernel<64, 1> : vx_paged_join_kernel<128, 1>, (items + 3) / 4);
    return hipGetLastError();
}

template <class E, int D, int QT, int PT>
hipError_t launch_token(const VxPagedAttnArgs& a, bool nt, hipStream_t st) {
    const uint32_t G = a.q.heads / a.c.hkv;
    const dim3 grid(a.splits, a.c.hkv * ((G + 15) / 16), a.c.n_seqs);
    if (nt) vx_paged_token_kernel<E, D, QT, PT, true><<<grid, kTokenThreads, 0, st>>>(a);
    else vx_paged_token_kernel<E, D, QT, PT, false><<<grid, kTokenThreads, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || a.splits == 1 ? e : launch_join(a, st);
}

// ---- prompts' rows ----
// A workgroup takes 128 (row, head) pairs of one sequence and KV head -- pair r is row r / G, head r % G of the G
// heads that share the KV head -- and walks the chunks that any of them sees, two chunks (64 positions) a step,
// K and V staged in two LDS buffers by direct-to-LDS loads. Each of its 4 waves keeps 32 pairs: scores
// S^T = K Q^T on 32x32x16 MFMAs leave a pair's scores in two lanes, so maximum and sum cost one lane swap, and
// the weights are the B operand of O^T = V^T P^T without leaving their lanes: the K row that scores row
// 16 t + 8 a + 4 g + b is position 16 a + 8 t + 4 g + b of the chunk (two bits swapped), which puts position
// order into the order of the pages' V blocks.
// The weights enter as PT terms of the cache's type (q of that type: two, as in the token form), so that they are off by
// 2^-16 (bf16) or 2^-22 (fp16) and the output by its own rounding only. One term made half as many products of the
// weights, 1.38 times as fast, but a bf16 output's error against 64 bits was 1.3 times that rounding.
// Bound by the matrix cores and what shares their issue slots: 8192 rows of Llama-3-8B's heads through a window of 4096
// take 550 to 607 us by the box (680 to 750 TFLOP/s of the visible pairs, half as much again with the second terms'
// products; the matrix cores busy in 58 % of the clocks, at 1.8 GHz); four chunks of 392 to 500 rows
// behind 4000 positions of Qwen2.5-7B's heads 177 to 190 us. Before the second term 64 pairs a wave (616 us), 8 or 2
// waves a workgroup (523, 729 against 471 then) were slower; written orders of products, exponentials and LDS reads took
// as long (391 to 396 us).
constexpr int kPromptWaves = 4;
constexpr int kPromptThreads = 64 * kPromptWaves;
constexpr int kPromptRows = kVxPromptRows;
static_assert(kPromptRows == 32 * kPromptWaves, "each wave has 32 pairs");

template <int N>
__device__ __forceinline__ void vx_wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void vx_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// 16 bytes per lane from base + off (off per lane) to the 1 KiB of LDS at byte offset lds (base and lds uniform). It
// stays between the barrier before it and the wait behind it (volatile statements keep their order); LDS reads may
// pass it, so it must not write what is read before that wait.
__device__ __forceinline__ void vx_load_lds(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
// The other lane of a pair (lane ^ 32) and this one: larger value, sum.
__device__ __forceinline__ float vx_max_pair(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t x = p[0], y = p[1];
    return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float vx_sum_pair(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t x = p[0], y = p[1];
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}

// Row tile `item` (counted over the sequences in order): its sequence, its index there, and the sequence's rows. Every
// workgroup scans the sequences in front of its own, 64 at a time: one row each of 64, 512 and 4096 sequences of 20 positions
// (Qwen2.5-7B's heads) 10, 47 and 770 us, by the token form 5, 20 and 150.
struct VxRowTile {
    uint32_t seq, tile, lo, rows;
    int64_t pos0;  // position of row lo
};
__device__ __forceinline__ bool vx_find_tile(const VxPagedAttnArgs& a, uint32_t item, uint32_t G, VxRowTile& r) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t base = 0;
    for (uint32_t s0 = 0; s0 < a.c.n_seqs; s0 += 64) {
        const uint32_t s = s0 + lane;
        uint32_t n = 0, lo = 0, rows = 0, len = 0;
        if (s < a.c.n_seqs) {
            len = a.c.lens[s];
            lo = min(a.q_start[s], a.n_rows);
            rows = max(min(a.q_start[s + 1], a.n_rows), lo) - lo;
            n = (uint32_t)(((uint64_t)rows * G + kPromptRows - 1) / kPromptRows);
        }
        uint32_t upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(upto, o);
            if (lane >= (uint32_t)o) upto += v;
        }
        const uint64_t hit = __ballot(item < base + upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            r.seq = s0 + (uint32_t)l;
            r.tile = item - base - (uint32_t)(__builtin_amdgcn_readlane((int)upto, l) - __builtin_amdgcn_readlane((int)n, l));
            r.lo = (uint32_t)__builtin_amdgcn_readlane((int)lo, l);
            r.rows = (uint32_t)__builtin_amdgcn_readlane((int)rows, l);
            r.pos0 = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)len, l) - (int64_t)r.rows;
            return true;
        }
        base += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    return false;
}

// LDS places of 16-byte blocks: block b of K row p (position of the chunk) at b ^ vx_k_swizzle, block b of V row e
// (dimension) at b ^ vx_v_swizzle, so that the 8 (of 32 banks) or 16 (of 64) lanes of a read meet in no bank.
template <int D>
__device__ __forceinline__ uint32_t vx_k_swizzle(uint32_t p) {
    const uint32_t far = p >> 4 & 1u;
    return D == 128 ? (p & 7u) | far << 3 : (p & 7u) ^ far;
}
__device__ __forceinline__ uint32_t vx_v_swizzle(uint32_t e) { return (e >> 1 & 3u) ^ (e >> 3 & 1u); }

template <class E, int D, int QT, int PT>
__global__ __launch_bounds__(kPromptThreads, 2) void vx_paged_prompt_kernel(VxPagedAttnArgs a, uint32_t tiles) {
    constexpr int NK = D / 16, NM = D / 32, RB = D / 8;
    constexpr uint32_t kChunk = 32u * D * 2u, kBuf = 4u * kChunk;  // K or V of a chunk; of a step
    constexpr uint32_t kUnits = kChunk / 1024u;                    // 1 KiB units of a chunk's K or V
    typedef typename E::v8 v8;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * kBuf];  // K of two steps, V of two steps
    __shared__ uint32_t s_found;  // settle: 1 + the first chunk of the last step with infinities or NaN, else 0
    if (threadIdx.x == 0) s_found = 0;
    // read anew, as LDS: a generic read would wait for the loads in flight too
    const auto found_now = [&] { return *(volatile __attribute__((address_space(3))) uint32_t*)&s_found; };
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t col = lane & 31u, grp = lane >> 5;
    const uint32_t G = a.q.heads / a.c.hkv, kvh = blockIdx.x % a.c.hkv;
    // the last tiles of a sequence have most to do: they go first
    VxRowTile rt;
    if (!vx_find_tile(a, tiles - 1 - blockIdx.x / a.c.hkv, G, rt)) return;
    const uint32_t r0 = rt.tile * kPromptRows, r1 = min(r0 + kPromptRows, rt.rows * G);  // the workgroup's pairs
    const VxChunks ch = vx_chunks(rt.pos0 + r0 / G, rt.pos0 + (r1 - 1) / G, a.window, a.sinks,
                                  (uint64_t)a.c.max_pages * a.c.page_size);
    const uint32_t per = ((ch.n + a.splits - 1) / a.splits + 1) & ~1u;
    const uint32_t c0 = min(blockIdx.y * per, ch.n), c1 = min(c0 + per, ch.n);
    const uint32_t* table = a.c.table + (size_t)rt.seq * a.c.table_stride;

    // this lane's pair; -1: a position of a pair that is not there
    const uint32_t pr = r0 + 32 * wave + col, row = rt.lo + pr / G, head = kvh * G + pr % G;
    const bool mine = pr < r1;
    const auto position = [&](uint32_t pair) { return (int)max((int64_t)-1, rt.pos0 + pair / G); };
    const int t = mine ? position(pr) : -1, low = (int)vx_low(t, a.window);
    const int sinks = (int)min(a.sinks, 0x7FFFFFFFu);
    // all pairs of the wave see [all_low, all_t]; none of the workgroup sees past last_t or, but for sinks, before ch.low
    const int all_t = position(min(r0 + 32 * wave, r1 - 1)), all_low = (int)vx_low(position(min(r0 + 32 * wave + 31, r1 - 1)), a.window);
    const int first_t = position(r0), last_t = position(r1 - 1), last_low = (int)vx_low(last_t, a.window);

    // q is requested before the table and the first K, and brought into its operands behind them
    VxEight raw[NK] = {};
    if (mine) vx_request<QT == 1>(raw, a.q.data, (size_t)row * a.q.rs + (size_t)head * a.q.hs + 8 * grp, 16, a.q.dtype);

    // where the K of the next 64 chunks lies in the pool, one a lane, and which of them have a page (page 0 stands in
    // for the others, and for chunks past the last)
    uint32_t place_lo, place_hi;
    // chunks with a page; that not all pairs of the wave, of the workgroup see whole; with places that no pair sees
    uint64_t paged, partial, mixed, hidden;
    uint32_t first = 0;               // the step whose chunks are in lanes 0 and 1
    const auto look_up = [&](uint32_t step) {
        const uint32_t i = c0 + 2 * step + lane, base = vx_chunk_base(ch, i);
        uint32_t page = kVxNoPage, place = 0;
        if (i < c1) {
            const uint32_t j = base / a.c.page_size;
            place = base - j * a.c.page_size;
            if (j < a.c.max_pages) page = table[j];
        }
        const bool have = page < a.c.n_pages;
        partial = __ballot(!have || (int)base + 31 > all_t || (int)base < all_low);
        mixed = __ballot(!have || (int)base + 31 > first_t || (int)base < last_low);
        hidden = __ballot(!have || (int)base + 31 > last_t || (int)base < (int)ch.low);
        const uint64_t at = (have ? (uint64_t)page * a.c.page_bytes : 0) + ((uint64_t)kvh * a.c.page_size + place) * (D * 2);
        place_lo = (uint32_t)at;
        place_hi = (uint32_t)(at >> 32);
        paged = __ballot(have);
        first = step;
    };

    // staging: each wave brings a quarter of a step's K and V, KiB by KiB
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
    const uint32_t my_chunk = wave >> 1, my_unit = (wave & 1u) * (kUnits / 2);
    const uint32_t my_lds = lds0 + my_chunk * kChunk + my_unit * 1024u;
    const uint64_t v_from_k = (uint64_t)a.c.hkv * a.c.page_size * (D * 2);
    uint32_t k_off[kUnits / 2];
    const uint32_t v_off = (16u * my_unit + lane / 4) * 64 + 16u * (lane % 4 ^ vx_v_swizzle(lane / 4));  // 16 rows a unit
#pragma unroll
    for (uint32_t j = 0; j < kUnits / 2; ++j) {
        const uint32_t i = 64u * (my_unit + j) + lane, p = i / RB;
        k_off[j] = p * D * 2 + 16u * (i % RB ^ vx_k_swizzle<D>(p));
    }
    const auto source = [&](uint32_t step) {  // this wave's chunk of a step that the lanes hold
        const int l = (int)(2 * (step - first) + my_chunk);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)place_lo, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)place_hi, l);
        return (const uint8_t*)a.c.pool + ((uint64_t)hi << 32 | lo);
    };
    const auto load_k = [&](const uint8_t* from, uint32_t buf, uint32_t j) { vx_load_lds(from, k_off[j], my_lds + buf * (2 * kChunk) + j * 1024u); };
    const auto load_v = [&](const uint8_t* from, uint32_t buf, uint32_t j) {
        vx_load_lds(from + v_from_k + j * 1024u, v_off, my_lds + (4 + 2 * buf) * kChunk + j * 1024u);
    };
    constexpr uint32_t NU = kUnits / 2;

    const uint32_t n_steps = (c1 - c0 + 1) / 2;
    constexpr bool PIPE = QT == 1;
    look_up(0);
    if (n_steps) {  // K and V of the first step, with PIPE K of the second
        const uint8_t *from = source(0), *from1 = source(1);
#pragma unroll
        for (uint32_t j = 0; j < NU; ++j) load_k(from, 0, j);
#pragma unroll
        for (uint32_t j = 0; j < NU; ++j) load_v(from, 0, j);
        if constexpr (PIPE) {
#pragma unroll
            for (uint32_t j = 0; j < NU; ++j) load_k(from1, 1, j);
        }
    }
    v8 qf[QT][NK];
    float to_log2 = fabsf(a.scale) * kLog2e;
    {
        if constexpr (QT == 1) {  // the cache's type: as it lies
            const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
            for (int c = 0; c < NK; ++c) qf[0][c] = __builtin_bit_cast(v8, raw[c].w[0] ^ sign);
        } else {
            float x[NK][8];
            vx_widen(raw, a.q.dtype, x);
            float by = a.scale < 0.0f ? -1.0f : 1.0f;
            if constexpr (QT == 2) {
                float big = 0.0f;
#pragma unroll
                for (int c = 0; c < NK; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[c][i]));
                big = vx_max_pair(big);
                const int e = vx_to_2_14(big);
                by = ldexpf(by, e);
                // never 0, times which a hidden score's infinity is NaN (the products stay below 2^38: at 2^-126 they are nothing)
                to_log2 = fmaxf(ldexpf(to_log2, -e), 0x1p-126f);
            }
#pragma unroll
            for (int c = 0; c < NK; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float rest = x[c][i] * by;
#pragma unroll
                    for (int u = 0; u < QT; ++u) {
                        const typename E::elt v = (typename E::elt)rest;
                        qf[u][c][i] = v;
                        rest -= (float)v;
                    }
                }
        }
    }

    vx_f16 o[NM];
#pragma unroll
    for (int n = 0; n < NM; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // the pair's maximum (as far as the weights are taken against it), this lane's sum
    // where this lane reads its K row (position kp of a chunk; the block of step c of the products at ^ 32 c) and V rows
    const uint32_t kp = (col & 7u) | (col >> 3 & 1u) << 4 | (col >> 4) << 3;
    const uint32_t k_at = kp * D * 2 + 16u * (grp ^ vx_k_swizzle<D>(kp));
    const uint32_t v_at = col * 64 + 16u * (grp ^ vx_v_swizzle(col));

    typedef vx_f16 Scores[2];
    const auto scores = [&](vx_f16& s, int b, uint32_t buf) {  // chunk b of a step
        const unsigned char* kb = lds + buf * (2 * kChunk) + b * kChunk;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            const v8 k = *(const v8*)(kb + (k_at ^ 32u * c));
#pragma unroll
            for (int u = QT - 1; u >= 0; --u) s = E::mfma(k, qf[u][c], s);
        }
    };
    // place of position p in the chunk at base: -1 in front of it, 32 or more behind it
    const auto place_in = [](int p, uint32_t base) { return max(-1, min(64, p - (int)base)); };
    struct Step {  // two chunks of the walk, a bit for each
        uint32_t chunk, have, partial, mixed, hidden;
    };
    const auto step_of = [&](uint32_t step) {
        const uint32_t at = 2 * (step - first);
        return Step{c0 + 2 * step, (uint32_t)(paged >> at) & 3u, (uint32_t)(partial >> at) & 3u, (uint32_t)(mixed >> at) & 3u,
                    (uint32_t)(hidden >> at) & 3u};
    };
    // Hides what the mask hides, and moves the maximum where a score passes it by more than 8 (the weights may pass 1
    // by 2^8 until then: a bf16 or fp16 weight keeps its relative precision, and the rescaling is rare).
    const auto bound = [&](Scores& s, const Step& x) {
        if (x.partial) {
            asm volatile("");  // a branch, not 64 selects in every step
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint32_t base = vx_chunk_base(ch, x.chunk + b);
                const int pt = (x.have >> b & 1u ? place_in(t, base) : -1) - 4 * (int)grp, pl = place_in(low, base) - 4 * (int)grp,
                          ps = place_in(sinks, base) - 4 * (int)grp;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int p = 16 * (r >> 2 & 1) + 8 * (r >> 3) + (r & 3);
                    const bool hidden = (p > pt) | ((p < pl) & (p >= ps));
                    s[b][r] = hidden ? -INFINITY : s[b][r];
                }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
        top = vx_max_pair(top) * to_log2;
        if (__ballot(top > m + 8.0f || (m == -INFINITY && top != -INFINITY))) {
            const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int n = 0; n < NM; ++n) o[n] *= f;
        }
    };
    // V of a step that not every pair of the workgroup sees whole. A weight of 0 does not keep a place out of the sums
    // (0 times NaN is NaN), so places that no pair sees are zeroed in LDS, and infinities and NaN of the others too:
    // the pairs that see those get them behind the walk.
    const auto settle = [&](const Step& x, uint32_t buf) {
        unsigned char* vb = lds + 4 * kChunk + buf * (2 * kChunk);
        uint32_t found = 0;
        for (uint32_t i = threadIdx.x; i < 2 * D * 4; i += kPromptThreads) {
            vx_u4* at = (vx_u4*)(vb + 16 * i);
            vx_u4 v = *at;
            if (x.hidden) {
                const uint32_t b = i / (D * 4), e = i / 4 % D, j = i % 4 ^ vx_v_swizzle(e);  // j: slots 8 j .. 8 j + 7 of row e
                const uint32_t base = vx_chunk_base(ch, x.chunk + b);
                const int pt = x.have >> b & 1u ? place_in(last_t, base) : -1, pl = place_in((int)ch.low, base), ps = place_in(sinks, base);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int p = 16 * (k >> 2) + 4 * (int)j + (k & 3);
                    if ((p > pt) | ((p < pl) & (p >= ps))) v[k / 2] &= k & 1 ? 0xFFFFu : 0xFFFF0000u;
                }
                *at = v;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) found |= (v[k] & (E::kExp | E::kExp << 16)) + (E::kOne | E::kOne << 16);  // all ones carry
        }
        if (found & 0x80008000u) s_found = x.chunk + 1;
        vx_barrier();
        if (found_now() != x.chunk + 1) return;
        for (uint32_t i = threadIdx.x; i < 2 * D * 32; i += kPromptThreads) {
            uint16_t* h = (uint16_t*)vb + i;
            if ((*h & E::kExp) == E::kExp) *h = 0;
        }
        vx_barrier();
    };
    // o += V^T P^T of a chunk, the weights as PT terms, never one: rounded once to bf16 (2^-8) or fp16 (2^-11) they would
    // cost the output as much as its own rounding.
    const auto add = [&](const vx_f16& s, int b, uint32_t buf) {
        const unsigned char* vb = lds + 4 * kChunk + buf * (2 * kChunk) + b * kChunk;
        const float ref = (m == -INFINITY ? 0.0f : m) - E::kUp;
        v8 pf[PT][2];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], to_log2, -ref));
            l += p;
            float rest = p;
#pragma unroll
            for (int u = 0; u < PT; ++u) {
                const typename E::elt v = (typename E::elt)rest;
                pf[u][r >> 3][r & 7] = v;
                rest -= (float)v;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NM; ++n) {
                const v8 v = *(const v8*)(vb + 2048 * n + (v_at ^ 32u * h));
#pragma unroll
                for (int u = PT - 1; u >= 0; --u) o[n] = E::mfma(v, pf[u][h], o[n]);
            }
    };

    // The walk, a step of two chunks at a time: while step i's weights are formed and added, the scores of step
    // i + 1 are multiplied and the loads of what follows go out between the products (issued in one go they held a
    // wave up for 1800 of a step's 4500 clocks). LDS: K of steps i + 1 and i + 2, V of steps i and i + 1, each in two
    // buffers. With q in several terms the next step's scores are not multiplied ahead (PIPE false): at head size 128 the
    // registers do not hold them (240 and 255 of 256 are taken); at 64 (158 and 186) they would, which was not tried.
    if (n_steps) {
        Step now = step_of(0), next = now;
        Scores s;
        if constexpr (PIPE) {
            vx_wait_loads<2 * NU>();  // the first K; the V and the next K may be on their way
            vx_barrier();
            next = step_of(1);
            scores(s[0], 0, 0);
            scores(s[1], 1, 0);
            bound(s, now);
        }
        const auto begin = [&](uint32_t i) {
            vx_wait_loads<0>();
            vx_barrier();  // step i is in LDS, and the buffers of what follows are read by everyone
            if (i + 2 - first >= 32) look_up(i + 1);
        };
        if constexpr (PIPE) {
            // behind the last step the loads and the scores go on with what is there, to no use
            const auto go = [&](uint32_t i, uint32_t buf, Scores& s, Scores& u) {
                begin(i);
                const uint8_t *from1 = source(i + 1), *from2 = source(i + 2);
                const Step after = step_of(i + 2);
                if (now.mixed) settle(now, buf);
                __builtin_amdgcn_s_setprio(1);  // before the other workgroup's waves that stage or take maxima: 479 -> 470 us
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const auto load = [&](uint32_t j) {
                        if (b == 0) load_v(from1, buf ^ 1, j);
                        else load_k(from2, buf, j);
                    };
#pragma unroll
                    for (uint32_t j = 0; j < NU / 2; ++j) load(j);
                    scores(u[b], b, buf ^ 1);
#pragma unroll
                    for (uint32_t j = NU / 2; j < NU; ++j) load(j);
                    add(s[b], b, buf);
                }
                __builtin_amdgcn_s_setprio(0);
                if (i + 1 < n_steps) bound(u, next);
                now = next;
                next = after;
            };
            Scores u;
            for (uint32_t i = 0; i < n_steps; i += 2) {
                go(i, 0, s, u);
                if (i + 1 < n_steps) go(i + 1, 1, u, s);
            }
        } else {
            for (uint32_t i = 0; i < n_steps; ++i) {
                const uint32_t buf = i & 1u;
                begin(i);
                const uint8_t* from1 = source(i + 1);
                next = step_of(i + 1);
#pragma unroll
                for (uint32_t j = 0; j < NU; ++j) {
                    load_k(from1, buf ^ 1, j);
                    load_v(from1, buf ^ 1, j);
                }
                if (now.mixed) settle(now, buf);
                scores(s[0], 0, buf);
                scores(s[1], 1, buf);
                bound(s, now);
                add(s[0], 0, buf);
                add(s[1], 1, buf);
                now = next;
            }
        }
        vx_wait_loads<0>();  // nothing may land in LDS that is another workgroup's by then
    }

    if (n_steps && found_now()) {  // infinities and NaN that settle took out, value by value from the pages
#pragma unroll 1
        for (uint32_t i = 0; i < n_steps; ++i) {
            if (i == 0 || i - first >= 32) look_up(i);
            const Step x = step_of(i);
            if (!x.mixed) continue;
#pragma unroll 1
            for (int j = 0; j < 64; ++j) {
                if (!(x.have >> j / 32 & 1u)) continue;
                const int at = (int)(2 * (i - first)) + j / 32, p = (int)vx_chunk_base(ch, x.chunk + j / 32) + (j & 31);
                const uint32_t lo32 = (uint32_t)__builtin_amdgcn_readlane((int)place_lo, at), hi32 = (uint32_t)__builtin_amdgcn_readlane((int)place_hi, at);
                const uint16_t* v = (const uint16_t*)(a.c.pool + ((uint64_t)hi32 << 32 | lo32) + v_from_k) + vx_vslot(j & 31) + 4 * grp * 32;
                if (p > t || (p < low && p >= sinks)) continue;
#pragma unroll
                for (int n = 0; n < NM; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const uint16_t h = v[(32 * n + 8 * (r >> 2) + (r & 3)) * 32];
                        if ((h & E::kExp) == E::kExp) o[n][r] += (float)__builtin_bit_cast(typename E::elt, h);
                    }
            }
        }
    }
    l = vx_sum_pair(l);
    if (t < 0) {
        if (mine && a.splits > 1 && grp == 0) a.part_ml[2 * (((size_t)row * a.q.heads + head) * a.splits + blockIdx.y) + 1] = -1.0f;
        return;
    }
    if (a.splits == 1) {
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        const size_t to = (size_t)row * a.out.rs + (size_t)head * a.out.hs;
#pragma unroll
        for (int n = 0; n < NM; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                vx_store4(a.out.data, to + 32 * n + 8 * q + 4 * grp, a.out.dtype,
                          vx_f4{o[n][4 * q], o[n][4 * q + 1], o[n][4 * q + 2], o[n][4 * q + 3]} * inv);
    } else {
        const size_t part = ((size_t)row * a.q.heads + head) * a.splits + blockIdx.y;
#pragma unroll
        for (int n = 0; n < NM; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(vx_f4*)(a.part_o + part * D + 32 * n + 8 * q + 4 * grp) = vx_f4{o[n][4 * q], o[n][4 * q + 1], o[n][4 * q + 2], o[n][4 * q + 3]};
        if (grp == 0) {
            a.part_ml[2 * part] = m;
            a.part_ml[2 * part + 1] = l;
        }
    }
}

template <class E, int D, int QT, int PT>
hipError_t launch_prompt(const VxPagedAttnArgs& a, hipStream_t st) {
    const uint64_t G = a.q.heads / a.c.hkv;
    uint64_t tiles = (uint64_t)a.n_rows * G / kPromptRows + a.c.n_seqs;
    const uint64_t most = (uint64_t)a.n_rows * ((G + kPromptRows - 1) / kPromptRows + 1);
    if (tiles > most) tiles = most;
    if (tiles * a.c.hkv > kVxMaxRows) return hipErrorInvalidValue;  // threads of a launch
    vx_paged_prompt_kernel<E, D, QT, PT><<<dim3((uint32_t)(tiles * a.c.hkv), a.splits), kPromptThreads, 0, st>>>(a, (uint32_t)tiles);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || a.splits == 1 ? e : launch_join(a, st);
}

}  // namespace

// Splits of the token form. What a CU has to do is its last workgroup's end: rounds / splits of a sequence's K and V of a
// head, rounds = workgroups / 256 CUs, at 16 us per MB (62 GB/s); lengths differ, which more rounds even out (0.3 of
// one). A round's start costs 1 us, the join 4. 24 sequences of 3000 positions, 4 KV heads of 128: 37.0 us with 3 splits
// (288 workgroups), 32.6 with 6 (576), 29.2 with 8 (768), 31.2 with 11 (1056); 64 of 1000: 23.6 unsplit (256), 28.3 with 2.
// A split has a chunk at least for every wave (one sequence of 2000 positions 8.2 us, with two chunks a wave 9.6).
uint32_t vx_paged_attn_splits(const VxPagedView& c, uint32_t heads, uint32_t rows, uint32_t max_len) {
    const uint32_t units = rows * c.hkv * ((heads / c.hkv + 15) / 16), chunks = max_len / 32 + (max_len % 32 != 0);
    const uint32_t most = (chunks + kTokenWaves - 1) / kTokenWaves, rounds0 = (units + 255) / 256;
    const double whole = 16e-6 * max_len * c.d * 4;
    const auto cost = [&](uint32_t rounds, uint32_t s) { return whole * (rounds + 0.3) / s + rounds; };
    double best = cost(rounds0, 1);
    uint32_t splits = 1;
    for (uint32_t r = rounds0; r <= rounds0 + 8; ++r) {
        uint32_t s = 256 * r / units;  // the most of so many rounds
        if (s > most) s = most;
        if (s > 64) s = 64;
        if (s <= splits) continue;
        const double t = cost((units * s + 255) / 256, s) + 4.0;
        if (t < best) best = t, splits = s;
    }
    return splits;
}

hipError_t vx_launch_paged_attention(const VxPagedAttnArgs& a, hipStream_t st) {
    const bool same = a.q.dtype == a.c.dtype, bf16 = a.c.dtype == VELOX_DT_BF16;
    // more than 16 heads of a KV head read the same K and V
    const bool nt = a.span * a.c.n_seqs * a.c.hkv * a.c.d * 4 > kTokenCached && a.q.heads / a.c.hkv <= 16;
    if (a.c.d == 64) {
        if (bf16) return same ? launch_token<VxBf16, 64, 1, 2>(a, nt, st) : launch_token<VxBf16, 64, 3, 3>(a, nt, st);
        return same ? launch_token<VxF16, 64, 1, 2>(a, nt, st) : launch_token<VxF16, 64, 2, 2>(a, nt, st);
    }
    if (bf16) return same ? launch_token<VxBf16, 128, 1, 2>(a, nt, st) : launch_token<VxBf16, 128, 3, 3>(a, nt, st);
    return same ? launch_token<VxF16, 128, 1, 2>(a, nt, st) : launch_token<VxF16, 128, 2, 2>(a, nt, st);
}

// Splits of the prompt form: where the row tiles alone leave CUs empty, the positions are split until there are two
// workgroups for each, into parts of 512 positions at least. Rows for a workgroup on every CU are not split, as equal parts
// of every tile's positions with every row joined: four chunks of 400 rows behind 4000 positions take 168 us (Qwen2.5-7B)
// and 175 (Llama-3-8B), as two splits 172 and 199; 2000 rows 68 and 69, as two splits 79 and 83 (fp32 rows 297 and 307,
// 274 and 327; 108 and 110, 113 and 125). Below that it pays: 2000 rows of SmolLM (141 workgroups) 33 us in three, 39 whole.
// Causal tiles have unequal walks, and cutting the long ones alone was not tried.
// Every sequence has tiles of its own: rows of at most max_rows a sequence are that many sequences at least, and with two
// workgroups for each CU from them alone nothing is split (64 sequences of 4 rows behind 4096 positions, Llama-3-8B:
// 512 workgroups 210 us, in eight splits 247; 128 behind 2000, Qwen2.5-7B: 107 and 129; fp32 rows 317 and 340, 162
// and 176). With fewer it pays still, though the tiles are more than the rows fill: 64 of 4 rows, Qwen2.5-7B, fp32 rows,
// 256 workgroups 190 us, in eight splits 175.
uint32_t vx_paged_prompt_split_rows(const VxPagedView& c, uint32_t max_rows) {
    const uint64_t rows = max_rows ? (uint64_t)max_rows * (511 / c.hkv) : kVxMaxRows;
    return rows < kVxMaxRows ? (uint32_t)rows : kVxMaxRows;
}
uint32_t vx_paged_prompt_splits(const VxPagedView& c, uint32_t heads, uint32_t n_rows, uint32_t max_rows, uint32_t span) {
    if (n_rows > vx_paged_prompt_split_rows(c, max_rows)) return 1;
    const uint64_t g = heads / c.hkv, tiles = ((uint64_t)n_rows * g + kPromptRows - 1) / kPromptRows * c.hkv;
    const uint64_t want = tiles >= 256 ? 1 : (512 + tiles - 1) / tiles, most = span / 512;
    const uint64_t s = want < most ? want : most;
    return s < 1 ? 1 : s > 64 ? 64 : (uint32_t)s;
}

hipError_t vx_launch_paged_prompt(const VxPagedAttnArgs& a, hipStream_t st) {
    const bool same = a.q.dtype == a.c.dtype, bf16 = a.c.dtype == VELOX_DT_BF16;
    if (a.c.d == 64) {
        if (bf16) return same ? launch_prompt<VxBf16, 64, 1, 2>(a, st) : launch_prompt<VxBf16, 64, 3, 3>(a, st);
        return same ? launch_prompt<VxF16, 64, 1, 2>(a, st) : launch_prompt<VxF16, 64, 2, 2>(a, st);
    }
    if (bf16) return same ? launch_prompt<VxBf16, 128, 1, 2>(a, st) : launch_prompt<VxBf16, 128, 3, 3>(a, st);
    return same ? launch_prompt<VxF16, 128, 1, 2>(a, st) : launch_prompt<VxF16, 128, 2, 2>(a, st);
}
