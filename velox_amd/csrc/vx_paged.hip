// vx_paged.hip -- the paged KV cache: rotary positions, the append to the pages, the pages' bookkeeping.
#include "vx_paged.h"

namespace {

// ---- elements ----
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

// cos and sin of position * f_j, times the amplitude. The angle is position * f_j / 2 pi turns in 64 bits (a
// product in 32 would be off by 2^-24 of a position's whole angle: 0.06 rad at position 10^6); its fraction of
// a turn, at most one half, is exact to 2^-25 in fp32.
__device__ __forceinline__ float2 vx_turn_of(const VxRopeTable& t, double freq, uint32_t pos) {
    const double turns = (double)pos * freq;
    const float f = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.0f * f, &s, &c);
    return make_float2(c * t.amp, s * t.amp);
}
__device__ __forceinline__ float2 vx_turn(const VxRopeTable& t, uint32_t j, uint32_t pos) { return vx_turn_of(t, t.turns[j], pos); }

// A pair turned by cs = (cos, sin); the same roundings wherever it is done (the empty statement keeps the values in
// fp32: a product, a sum and the conversion to fp16 would become one instruction in some places and not in others).
__device__ __forceinline__ float2 vx_rotate(float a, float b, float2 cs) {
    float x = __builtin_fmaf(a, cs.x, -(b * cs.y)), y = __builtin_fmaf(b, cs.x, a * cs.y);
    asm("" : "+v"(x), "+v"(y));
    return make_float2(x, y);
}

// A unit of a head's values with 16-byte loads and stores: V pairs (half layout: V values of each half), or V values
// (interleaved pairs, or values behind rot_dim, which pass).
template <class T>
struct alignas(16) VxVec {
    static constexpr int V = 16 / sizeof(T);
    T v[V];
};
// 16 bytes (or 8) with the non-temporal hint (NT) or without.
template <bool NT, class V>
__device__ __forceinline__ V vx_get(const V* p) {
    typedef uint32_t W __attribute__((ext_vector_type(sizeof(V) / 4)));
    if constexpr (NT) return __builtin_bit_cast(V, __builtin_nontemporal_load((const W*)p));
    else return *p;
}
template <bool NT, class V>
__device__ __forceinline__ void vx_set(V* p, const V& v) {
    typedef uint32_t W __attribute__((ext_vector_type(sizeof(V) / 4)));
    if constexpr (NT) __builtin_nontemporal_store(__builtin_bit_cast(W, v), (W*)p);
    else *p = v;
}
template <class T>
__device__ __forceinline__ uint32_t vx_units(const VxRopeTable& t, uint32_t d) {
    constexpr uint32_t V = VxVec<T>::V;
    return (t.interleaved ? t.rot : t.rot / 2) / V + (d - t.rot) / V;
}
// Unit u of a head: what load reads of the values at x, and turn hands on, turned by the row's cos / sin table cs, V
// values at a time as put(first element, values).
template <class T, bool NT>
struct VxUnit {
    static constexpr uint32_t V = VxVec<T>::V;
    VxVec<T> a, b;  // b: the second half's values of half-layout pairs
    // SAME: as many loads in every lane (a unit that has no b reads a's place), so that no branch stands between the loads
    // of several units.
    template <bool SAME>
    __device__ __forceinline__ void load(const VxRopeTable& t, const T* x, uint32_t u) {
        const uint32_t half = t.rot / 2, pair_units = (t.interleaved ? t.rot : half) / V;
        const uint32_t e = u < pair_units ? u * V : t.rot + (u - pair_units) * V;
        a = vx_get<NT>((const VxVec<T>*)(x + e));
        if constexpr (SAME) {
            if (!t.interleaved) b = vx_get<NT>((const VxVec<T>*)(x + (u < pair_units ? half + e : e)));
        } else if (!t.interleaved && u < pair_units) {
            b = vx_get<NT>((const VxVec<T>*)(x + half + e));
        }
    }
    template <class Put>
    __device__ __forceinline__ void turn(const VxRopeTable& t, uint32_t u, const float2* cs, Put put) const {
        const uint32_t half = t.rot / 2, pair_units = (t.interleaved ? t.rot : half) / V;
        float y[V];
        if (u >= pair_units) {
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) y[i] = (float)a.v[i];
            put(t.rot + (u - pair_units) * V, y);
        } else if (t.interleaved) {
#pragma unroll
            for (uint32_t i = 0; i < V; i += 2) {
                const float2 r = vx_rotate((float)a.v[i], (float)a.v[i + 1], cs[u * (V / 2) + i / 2]);
                y[i] = r.x;
                y[i + 1] = r.y;
            }
            put(u * V, y);
        } else {
            float z[V];
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) {
                const float2 r = vx_rotate((float)a.v[i], (float)b.v[i], cs[u * V + i]);
                y[i] = r.x;
                z[i] = r.y;
            }
            put(u * V, y);
            put(half + u * V, z);
        }
    }
};
constexpr int kUnitsAhead = 4;  // units a thread requests before it turns the first

template <bool NT, class O, int V>
__device__ __forceinline__ void vx_put(O* to, const float* y) {
    struct alignas(V * sizeof(O)) Out {
        O v[V];
    } o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = (O)y[i];
    vx_set<NT>((Out*)to, o);
}

// ---- rotation of rows: a workgroup takes kRows rows, whose cos / sin all heads share through LDS ----
// Bound by its bytes: 4001 rows of 64 heads of 128 (fp16, 131 MB moved, cold) take 24 us (5.4 TB/s; a copy of as much
// 26 us).
constexpr int kRopeThreads = 256;

template <class T, bool NT>
__global__ __launch_bounds__(kRopeThreads) void vx_rope_vec_kernel(VxRopeTable t, VxRowsView x, VxRowsView o, uint32_t n_rows,
                                                                   uint32_t d, const uint32_t* __restrict__ positions, uint32_t per) {
    constexpr int V = VxVec<T>::V;
    __shared__ float2 cs[kRopeThreads > 2 * kVxMaxRopePairs ? kRopeThreads : 2 * kVxMaxRopePairs];
    const uint32_t half = t.rot / 2, row0 = blockIdx.x * per, n = min(per, n_rows - row0);  // n * half <= 256
    const uint32_t units = vx_units<T>(t, d), total = n * x.heads;
    const uint32_t step = units < kRopeThreads ? kRopeThreads / units : 1;  // heads at a time; a thread keeps its unit
    VxUnit<T, false> v[kUnitsAhead];
    const auto load = [&](uint32_t u, uint32_t i) {
#pragma unroll
        for (int k = 0; k < kUnitsAhead; ++k) {
            const uint32_t j = i + k * step, w = j / x.heads, h = j % x.heads;
            if (j < total) v[k].template load<false>(t, (const T*)x.data + (size_t)(row0 + w) * x.rs + (size_t)h * x.hs, u);
        }
    };
    const uint32_t u0 = threadIdx.x % units, i0 = threadIdx.x / units < step ? threadIdx.x / units : total;
    load(u0, i0);  // on its way while the angles are formed
    for (uint32_t i = threadIdx.x; i < n * half; i += kRopeThreads) cs[i] = vx_turn(t, i % half, positions[row0 + i / half]);
    __syncthreads();
    for (uint32_t u = u0; u < units; u += kRopeThreads) {  // (once, unless a head has more units than threads)
        if (u != u0) load(u, i0);
        for (uint32_t i = i0; i < total; i += kUnitsAhead * step) {
            if (i != i0) load(u, i);
#pragma unroll
            for (int k = 0; k < kUnitsAhead; ++k) {
                const uint32_t j = i + k * step, w = j / x.heads, h = j % x.heads;
                T* to = (T*)o.data + (size_t)(row0 + w) * o.rs + (size_t)h * o.hs;
                if (j < total) v[k].turn(t, u, cs + w * half, [&](uint32_t e, const float* y) { vx_put<NT, T, V>(to + e, y); });
            }
        }
    }
}

// The same value by value, for rows without 16-byte alignment and pairs that do not fill vectors. Bound by its loads of one
// value each: 4001 rows of 64 heads of 128 in bf16 44 us at an odd address, 84 with 18 or 34 of 128 turned (by vectors 22;
// the bytes at a copy's rate 27).
__global__ __launch_bounds__(kRopeThreads) void vx_rope_rows_kernel(VxRopeTable t, VxRowsView x, VxRowsView o, uint32_t n_rows,
                                                                    uint32_t d, const uint32_t* __restrict__ positions) {
    __shared__ float2 cs[kVxMaxRopePairs];
    const uint32_t half = t.rot / 2, row = blockIdx.x;
    const uint32_t pos = positions[row];
    for (uint32_t j = threadIdx.x; j < half; j += kRopeThreads) cs[j] = vx_turn(t, j, pos);
    __syncthreads();
    const uint32_t units = half + (d - t.rot);  // a pair, or one value behind them
    for (uint32_t i = threadIdx.x; i < units * x.heads; i += kRopeThreads) {
        const uint32_t h = i / units, u = i % units;
        const size_t xb = (size_t)row * x.rs + (size_t)h * x.hs, ob = (size_t)row * o.rs + (size_t)h * o.hs;
        if (u < half) {
            const uint32_t e0 = t.interleaved ? 2 * u : u, e1 = t.interleaved ? 2 * u + 1 : u + half;
            const float a = vx_load(x.data, xb + e0, x.dtype), b = vx_load(x.data, xb + e1, x.dtype);
            const float2 r = vx_rotate(a, b, cs[u]);
            vx_store(o.data, ob + e0, o.dtype, r.x);
            vx_store(o.data, ob + e1, o.dtype, r.y);
        } else {
            const uint32_t e = t.rot + u - half;
            vx_store(o.data, ob + e, o.dtype, vx_load(x.data, xb + e, x.dtype));
        }
    }
}

// ---- ragged batches ----
// Rows [lo, hi) of sequence s and the position of row lo; positions may be negative.
struct VxSpan {
    uint32_t lo, hi;
    int64_t pos0;
};
__device__ __forceinline__ VxSpan vx_span(const uint32_t* q_start, const uint32_t* lens, uint32_t n_rows, uint32_t s) {
    VxSpan r;
    r.lo = q_start ? min(q_start[s], n_rows) : s;
    r.hi = q_start ? min(q_start[s + 1], n_rows) : min(s + 1u, n_rows);
    r.hi = max(r.hi, r.lo);
    r.pos0 = (int64_t)lens[s] - (int64_t)(r.hi - r.lo);
    return r;
}

// ---- append: workgroups (x) take a 32-position block (a V block of the pages, up to 32 rows) of a sequence each;
// y deals its heads ----
struct VxBlock {
    uint32_t row0, n, i0, pos;  // rows row0 .. row0 + n at places i0 .. of the block, positions pos ..
    uint32_t in_page, page;     // the block's place in its page; no page: >= n_pages
    uint32_t seq;
};
// Block `item` of the batch, blocks counted over the sequences in order; false behind the last. Every wave walks the
// sequences 64 at a time (one row each of 64, 512 and 4096 sequences, Qwen2.5-7B's heads, 5.3, 11.5 and 167 us; without
// q_start, hence without the walk, 4.6, 8.3 and 49). One row each (no q_start): which row it is does not wait for the length; the rest is
// vx_block_place's.
__device__ __forceinline__ bool vx_block(const VxAppendArgs& a, uint32_t item, VxBlock& b) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t seq = item, blk = 0;
    VxSpan r;
    if (!a.q_start) {
        b = VxBlock{item, 1, 0, 0, 0, kVxNoPage, item};
        return true;
    } else {
        uint32_t base = 0;
        bool found = false;
        for (uint32_t s0 = 0; s0 < a.c.n_seqs && !found; s0 += 64) {
            const uint32_t s = s0 + lane;
            uint32_t n = 0;
            VxSpan mine = {0, 0, 0};
            if (s < a.c.n_seqs) {
                mine = vx_span(a.q_start, a.c.lens, a.n_rows, s);
                const int64_t end = mine.pos0 + (mine.hi - mine.lo), from = mine.pos0 > 0 ? mine.pos0 : 0;
                if (end > from) n = (uint32_t)(((end + 31) >> 5) - (from >> 5));
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
                const auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
                seq = s0 + (uint32_t)l;
                blk = item - base - (of(upto) - of(n));
                r.lo = of(mine.lo);
                r.hi = of(mine.hi);
                r.pos0 = (int64_t)((uint64_t)of((uint32_t)(mine.pos0 >> 32)) << 32 | of((uint32_t)mine.pos0));
                found = true;
            }
            base += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        }
        if (!found) return false;
    }
    const int64_t from = r.pos0 > 0 ? r.pos0 : 0, end = r.pos0 + (r.hi - r.lo);
    const int64_t p0 = ((from >> 5) + blk) << 5;  // the block's first position
    const auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    const uint32_t i0 = (uint32_t)((from > p0 ? from : p0) - p0), n = (uint32_t)((end < p0 + 32 ? end : p0 + 32) - p0) - i0;
    b = VxBlock{uniform(r.lo + (uint32_t)(p0 + i0 - r.pos0)), uniform(n), uniform(i0), uniform((uint32_t)p0 + i0), 0, kVxNoPage, uniform(seq)};
    return true;
}
// The block's position (one row each: the length's last) and page; false: in front of position 0.
__device__ __forceinline__ bool vx_block_place(const VxAppendArgs& a, VxBlock& b) {
    if (!a.q_start) {
        const uint32_t len = vx_word(a.c.lens + b.seq);
        if (!len) return false;
        b.pos = len - 1;
        b.i0 = b.pos & 31u;
    }
    const uint32_t p0 = b.pos - b.i0, pi = p0 / a.c.page_size;
    b.page = kVxNoPage;
    if (pi < a.c.max_pages) b.page = vx_word(a.c.table + (size_t)b.seq * a.c.table_stride + pi);
    b.in_page = p0 - pi * a.c.page_size;
    return true;
}
// The block's page: its K, V behind; NULL: none.
__device__ __forceinline__ uint16_t* vx_page(const VxAppendArgs& a, const VxBlock& b) {
    return b.page < a.c.n_pages ? (uint16_t*)(a.c.pool + (size_t)b.page * a.c.page_bytes) : nullptr;
}
// cos and sin of the block's rows w0 .. w1; freq: t.turns[threadIdx.x % half], where there are pairs.
__device__ __forceinline__ void vx_angles(const VxRopeTable& t, const VxBlock& b, uint32_t w0, uint32_t w1, double freq,
                                          float2 (*cs)[kVxMaxRopePairs / 2]) {
    const uint32_t half = t.rot / 2, n = (w1 - w0) * half;
    if (threadIdx.x < n) cs[w0 + threadIdx.x / half][threadIdx.x % half] = vx_turn_of(t, freq, b.pos + w0 + threadIdx.x / half);
    for (uint32_t i = threadIdx.x + 256; i < n; i += 256) cs[w0 + i / half][i % half] = vx_turn(t, i % half, b.pos + w0 + i / half);
    __syncthreads();
}

// Bound by its bytes: 8531 rows of Llama-3-8B's q, k and v (bf16, 210 MB moved) take 43 us (4.8 TB/s), one row each of 32
// sequences of Qwen2.5-7B 3.8 us, a launch and the length, the page number and a line behind each other (47 and 4.6 us
// while branches around the loads made them wait for each other). T: the rows' type, C: the cache's. K and q by units
// of 16 bytes; V by 8 dimensions of the 8 positions that share 16 bytes of a V block, transposed in registers, so that
// whole blocks leave as whole lines.
template <class T, class C, bool NT>
__global__ __launch_bounds__(256) void vx_append_vec_kernel(VxRopeTable t, VxAppendArgs a) {
    constexpr int V = VxVec<T>::V;
    __shared__ float2 cs[32][kVxMaxRopePairs / 2];
    VxBlock b;
    if (!vx_block(a, blockIdx.x, b)) return;
    const uint32_t d = a.c.d, hkv = a.c.hkv, hq = a.q.data ? a.q.heads : 0, heads = hq + hkv;
    const uint32_t units = vx_units<T>(t, d), step = 256 / units;  // d <= 128: at most 32 units
    const uint32_t u = threadIdx.x % units, mine = threadIdx.x / units;
    // the workgroups share the block's (row, head) pairs out in runs, so that each forms its own rows' angles only
    const uint32_t all = b.n * heads, from = all * blockIdx.y / gridDim.y, total = all * (blockIdx.y + 1) / gridDim.y;
    const uint32_t i0 = mine < step ? from + mine : total;
    VxUnit<T, NT> v[kUnitsAhead];
    // pinned: the compiler would otherwise choose between their addresses and read them lane by lane, between the loads
    typedef const T __attribute__((address_space(1)))* Global;
    Global qp = (Global)a.q.data, kp = (Global)a.k.data;
    uint64_t qrs = a.q.rs, qhs = a.q.hs, krs = a.k.rs, khs = a.k.hs;
    asm volatile("" : "+s"(qp), "+s"(kp), "+s"(qrs), "+s"(qhs), "+s"(krs), "+s"(khs));
    const auto load = [&](uint32_t base, uint32_t i) {  // base: i of the first thread
#pragma unroll
        for (int k = 0; k < kUnitsAhead; ++k) {
            if (base + k * step >= total) continue;
            const uint32_t j = min(i + k * step, total - 1), w = j / heads, h = j % heads;
            const bool is_q = h < hq;
            const Global x = (is_q ? qp : kp) + (size_t)(b.row0 + w) * (is_q ? qrs : krs) + (size_t)(is_q ? h : h - hq) * (is_q ? qhs : khs);
            v[k].template load<true>(t, (const T*)x, u);
        }
    };
    const double freq = t.rot ? t.turns[threadIdx.x % (t.rot / 2)] : 0.0;
    load(from, i0);  // on its way while the block is placed, V moved and the angles formed
    if (!vx_block_place(a, b)) return;
    uint16_t* const page = vx_page(a, b);
    const uint32_t groups = d / 8, pieces = page ? hkv * groups * 4 : 0;  // a head's pieces lie in one run: whole rows, whole blocks
    const uint32_t v_to = pieces * (blockIdx.y + 1) / gridDim.y;
    for (uint32_t i = pieces * blockIdx.y / gridDim.y + 255 - threadIdx.x; i < v_to; i += 256) {  // the last threads first: with few rows the others turn
        const uint32_t e0 = i % groups * 8, j = i / groups % 4, h = i / groups / 4;  // slots 8 j .. 8 j + 7 of 8 dimensions
        VxVec<T> y[8][8 / V];  // all requested before one is looked at
        uint32_t there = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t p = 16 * (k >> 2) + 4 * j + (k & 3);  // the position of slot 8 j + k
            const uint32_t w = min(max(p, b.i0) - b.i0, b.n - 1);  // of slots without a row another's (a branch would be a wait)
            there |= (uint32_t)(p - b.i0 < b.n) << k;
            const T* from = (const T*)a.v.data + (size_t)(b.row0 + w) * a.v.rs + (size_t)h * a.v.hs + e0;
#pragma unroll
            for (int q = 0; q < 8 / V; ++q) y[k][q] = ((const VxVec<T>*)from)[q];
        }
        const auto x = [&](int k, int e) { return (C)(float)y[k][e / V].v[e % V]; };
        C* to = (C*)page + ((size_t)(hkv + h) * a.c.page_size + b.in_page) * d + e0 * 32 + 8 * j;
        if (there == 255u) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                struct alignas(16) Out {
                    C v[8];
                } o;
#pragma unroll
                for (int k = 0; k < 8; ++k) o.v[k] = x(k, e);
                *(Out*)(to + e * 32) = o;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (there >> k & 1)
#pragma unroll
                    for (int e = 0; e < 8; ++e) to[e * 32 + k] = x(k, e);
        }
    }
    vx_angles(t, b, from / heads, (total + heads - 1) / heads, freq, cs);
    for (uint32_t base = from, i = i0; base < total; base += kUnitsAhead * step, i += kUnitsAhead * step) {
        if (base != from) load(base, i);
#pragma unroll
        for (int k = 0; k < kUnitsAhead; ++k) {
            const uint32_t j = i + k * step, w = j / heads, h = j % heads;
            if (j >= total) continue;
            if (h < hq) {
                T* to = (T*)a.qo.data + (size_t)(b.row0 + w) * a.qo.rs + (size_t)h * a.qo.hs;
                v[k].turn(t, u, cs[w], [&](uint32_t e, const float* y) { vx_put<NT, T, V>(to + e, y); });
            } else if (page) {
                C* to = (C*)page + ((size_t)(h - hq) * a.c.page_size + b.in_page + b.i0 + w) * d;
                v[k].turn(t, u, cs[w], [&](uint32_t e, const float* y) { vx_put<NT, C, V>(to + e, y); });
            }
        }
    }
}

// The same value by value, for rows of several types or without 16-byte alignment, and pairs that do not fill vectors. 8500
// rows of Llama-3-8B's q, k and v in bf16 take 182 us at odd addresses, 244 with 34 of 128 turned (by vectors 43); fp32 q
// beside bf16 k and v 310 us (348 MB, 71 at a copy's rate).
__global__ __launch_bounds__(256) void vx_append_rows_kernel(VxRopeTable t, VxAppendArgs a) {
    __shared__ float2 cs[32][kVxMaxRopePairs / 2];
    VxBlock b;
    if (!vx_block(a, blockIdx.x, b) || !vx_block_place(a, b)) return;
    vx_angles(t, b, 0, b.n, t.rot ? t.turns[threadIdx.x % (t.rot / 2)] : 0.0, cs);
    uint16_t* const kp = vx_page(a, b);
    uint16_t* const vp = kp + (size_t)a.c.hkv * a.c.page_size * a.c.d;
    const uint32_t half = t.rot / 2, d = a.c.d, hkv = a.c.hkv, hq = a.q.data ? a.q.heads : 0, heads = hq + 2 * hkv;
    const uint32_t units = half + (d - t.rot);
    for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < b.n * heads * units; i += gridDim.y * 256) {
        const uint32_t u = i % units, h = i / units % heads, w = i / units / heads;
        const bool pair = u < half;
        const uint32_t e0 = pair ? (t.interleaved ? 2 * u : u) : t.rot + u - half;
        const uint32_t e1 = pair ? (t.interleaved ? 2 * u + 1 : u + half) : e0;
        const VxRowsView& x = h < hq ? a.q : h < hq + hkv ? a.k : a.v;
        const uint32_t hh = h < hq ? h : h < hq + hkv ? h - hq : h - hq - hkv;
        const size_t xb = (size_t)(b.row0 + w) * x.rs + (size_t)hh * x.hs;
        float y0 = vx_load(x.data, xb + e0, x.dtype), y1 = pair ? vx_load(x.data, xb + e1, x.dtype) : 0.0f;
        if (pair && h < hq + hkv) {
            const float2 r = vx_rotate(y0, y1, cs[w][u]);
            y0 = r.x;
            y1 = r.y;
        }
        if (h < hq) {
            const size_t ob = (size_t)(b.row0 + w) * a.qo.rs + (size_t)hh * a.qo.hs;
            vx_store(a.qo.data, ob + e0, a.qo.dtype, y0);
            if (pair) vx_store(a.qo.data, ob + e1, a.qo.dtype, y1);
        } else if (kp && h < hq + hkv) {
            uint16_t* to = kp + ((size_t)hh * a.c.page_size + b.in_page + b.i0 + w) * d;
            vx_store(to, e0, a.c.dtype, y0);
            if (pair) vx_store(to, e1, a.c.dtype, y1);
        } else if (kp) {
            uint16_t* to = vp + ((size_t)hh * (a.c.page_size / 32) + b.in_page / 32) * d * 32;
            const uint32_t slot = vx_vslot(b.i0 + w);
            vx_store(to, (size_t)e0 * 32 + slot, a.c.dtype, y0);
            if (pair) vx_store(to, (size_t)e1 * 32 + slot, a.c.dtype, y1);
        }
    }
}

// ---- pages ----
constexpr int kPageThreads = 1024;

// Sum over the threads before this one; total: the workgroup's sum. Two barriers.
__device__ __forceinline__ uint32_t vx_scan(uint32_t v, uint32_t& total) {
    __shared__ uint32_t part[kPageThreads / 64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t upto = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t w = __shfl_up(upto, o);
        if (lane >= (uint32_t)o) upto += w;
    }
    __syncthreads();  // part of an earlier call is read
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPageThreads / 64; ++w) {
        if ((uint32_t)w < wave) before += part[w];
        all += part[w];
    }
    total = all;
    return before + upto - v;
}

__global__ void vx_pages_reset_kernel(VxPages p) {
    const size_t n = (size_t)p.n_seqs * p.max_pages, step = (size_t)gridDim.x * blockDim.x;
    const size_t i0 = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (size_t i = i0; i < n; i += step) p.table[i / p.max_pages * p.table_stride + i % p.max_pages] = kVxNoPage;
    for (size_t i = i0; i < p.n_pages; i += step) p.refs[i] = 0;
    for (size_t i = i0; i < p.n_seqs; i += step) p.lens[i] = 0;
    for (size_t i = i0; i < kVxPagesHead; i += step) p.scratch[i] = 0;
}

// Which of the eight pages from `first` on are free, as bits; the loads are in flight until used.
struct VxRefs8 {
    uint4 r[2];
    uint32_t n;  // pages there are
    __device__ __forceinline__ void load(const VxPages& p, uint32_t first) {
        n = first < p.n_pages ? min(8u, p.n_pages - first) : 0u;
        if (n == 8) {
            r[0] = *(const uint4*)(p.refs + first);
            r[1] = *(const uint4*)(p.refs + first + 4);
        } else {
            uint32_t* w = (uint32_t*)r;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) w[k] = k < n ? p.refs[first + k] : 1u;
        }
    }
    __device__ __forceinline__ uint32_t free() const {
        return (uint32_t)(r[0].x == 0) | (uint32_t)(r[0].y == 0) << 1 | (uint32_t)(r[0].z == 0) << 2 | (uint32_t)(r[0].w == 0) << 3 |
               (uint32_t)(r[1].x == 0) << 4 | (uint32_t)(r[1].y == 0) << 5 | (uint32_t)(r[1].z == 0) << 6 | (uint32_t)(r[1].w == 0) << 7;
    }
};

// One workgroup: who needs what (a thread per sequence, or four), the lowest free pages (a scan of refs that ends
// when it has enough), then a thread per page given out. What bounds it is the chain of dependent loads -- length,
// last page, its count -- and a dozen barriers: 8 sequences take 6.2 us, 64 that share pages 8.8 us, so the scan's first
// pages are requested at the start, and the pages found stay in LDS.
constexpr uint32_t kPerThread = kVxMaxPagedSeqs / kPageThreads;
constexpr uint32_t kLooked = 64;
constexpr uint32_t kListed = 4096;  // pages found that LDS holds; the rest lie in the scratch memory

__global__ __launch_bounds__(kPageThreads) void vx_pages_extend_kernel(VxPages p, const uint32_t* __restrict__ add) {
    __shared__ uint32_t s_upto[kVxMaxPagedSeqs];  // pages given to sequences up to this one, itself included
    __shared__ uint32_t s_old[kVxMaxPagedSeqs];   // pages it had; bit 31: its last one is copied
    __shared__ uint32_t s_spot[kVxMaxPagedSeqs];  // the shared last page it would write
    __shared__ uint32_t s_list[kListed];
    __shared__ uint32_t s_moves, s_granted, s_refused;
    const uint32_t tid = threadIdx.x, n = p.n_seqs, per = (n + kPageThreads - 1) / kPageThreads;
    const uint32_t a0 = min(tid * per, n), a1 = min(a0 + per, n);
    uint32_t* src = p.scratch + kVxPagesHead;
    uint32_t* dst = src + vx_pages_moves(p.n_seqs, p.n_pages);
    uint32_t* list = dst + vx_pages_moves(p.n_seqs, p.n_pages);
    VxRefs8 refs;
    refs.load(p, tid * 8);
    uint32_t len[kPerThread], grow[kPerThread], refs_of[kPerThread];
#pragma unroll
    for (uint32_t k = 0; k < kPerThread; ++k) {
        const bool is = a0 + k < a1;
        len[k] = is ? p.lens[a0 + k] : 0u;
        grow[k] = is ? add[a0 + k] : 0u;
    }
    if (tid == 0) s_moves = s_granted = s_refused = 0;
    const auto pages_of = [&](uint64_t x) { return (uint32_t)((x + p.page_size - 1) / p.page_size); };
    uint32_t fits = 0;
    int any = 0;
#pragma unroll
    for (uint32_t k = 0; k < kPerThread; ++k) {
        const uint32_t s = a0 + k;
        refs_of[k] = 0;
        if (s >= a1) continue;
        const uint64_t now = (uint64_t)len[k] + grow[k];
        const bool ok = grow[k] && now < 0x80000000ull && (now + p.page_size - 1) / p.page_size <= p.max_pages;
        const uint32_t old = ok ? pages_of(len[k]) : 0u;
        uint32_t spot = kVxNoPage;
        if (ok && len[k] % p.page_size) {
            const uint32_t last = p.table[(size_t)s * p.table_stride + old - 1];
            if (last < p.n_pages) refs_of[k] = p.refs[last];
            if (refs_of[k] > 1) spot = last;
        }
        s_spot[s] = spot;
        s_old[s] = old;
        fits |= (uint32_t)ok << k;
        any |= spot != kVxNoPage;
    }
    any = __syncthreads_or(any);
    // how many write into a shared page, and the last of them: among few sequences each looks at all the others (8: 6.2 us,
    // by counting 7.3), else they are counted in the moves' memory, a word a page (4096 that share by twos, launches and
    // copies included: 39 us, by looking 584; 200: 16 and 20)
    const bool counted = any && n > kLooked;
    if (counted) {
#pragma unroll
        for (uint32_t k = 0; k < kPerThread; ++k)
            if (a0 + k < a1 && s_spot[a0 + k] != kVxNoPage) {
                __hip_atomic_store(src + s_spot[a0 + k], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(dst + s_spot[a0 + k], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // there before anyone counts: a barrier alone waits for LDS only
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kPerThread; ++k)
            if (a0 + k < a1 && s_spot[a0 + k] != kVxNoPage) {
                atomicAdd(src + s_spot[a0 + k], 1u);
                atomicMax(dst + s_spot[a0 + k], a0 + k);
            }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t k = 0; k < kPerThread; ++k) {
        const uint32_t s = a0 + k;
        if (s >= a1) continue;
        if (fits >> k & 1) {
            mine += pages_of((uint64_t)len[k] + grow[k]) - pages_of(len[k]);
            const uint32_t spot = s_spot[s];
            if (any && spot != kVxNoPage) {
                uint32_t same = 0, last = 0;
                if (counted) {
                    same = __hip_atomic_load(src + spot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    last = __hip_atomic_load(dst + spot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                for (uint32_t j = 0; j < n && !counted; ++j)
                    if (s_spot[j] == spot) {
                        ++same;
                        last = j;
                    }
                if (last != s || same != refs_of[k]) {  // else it is the last of all its holders and keeps the page
                    s_old[s] |= 0x80000000u;
                    ++mine;
                }
            }
        }
        s_upto[s] = mine;  // within this thread's sequences, for now
    }
    uint32_t total;
    const uint32_t before = vx_scan(mine, total);
    for (uint32_t s = a0; s < a1; ++s) s_upto[s] += before;
    // the lowest free pages
    uint32_t found = 0;
    for (uint32_t base = 0; base < p.n_pages && found < total; base += kPageThreads * 8) {
        if (base) refs.load(p, base + tid * 8);
        uint32_t free = refs.free(), got;
        uint32_t rank = found + vx_scan(__popc(free), got);
        for (; free; free &= free - 1, ++rank) {
            if (rank >= total) break;
            const uint32_t page = base + tid * 8 + __builtin_ctz(free);
            if (rank < kListed) s_list[rank] = page;
            else list[rank] = page;
        }
        found += got;
    }
    __syncthreads();
    const auto listed = [&](uint32_t rank) { return rank < kListed ? s_list[rank] : list[rank]; };
    // sequences in order until the pages run out; the refused are then the last that extend
#pragma unroll
    for (uint32_t k = 0; k < kPerThread; ++k) {
        const uint32_t s = a0 + k;
        if (s >= a1 || !grow[k]) continue;
        if (!(fits >> k & 1) || s_upto[s] > found) {
            atomicAdd(&s_refused, 1u);
            continue;
        }
        atomicMax(&s_granted, s_upto[s]);
        p.lens[s] = len[k] + grow[k];
        if (s_old[s] >> 31) {
            const uint32_t from = s_spot[s], to = listed(s ? s_upto[s - 1] : 0u), m = atomicAdd(&s_moves, 1u);
            src[m] = from;
            dst[m] = to;
            p.table[(size_t)s * p.table_stride + (s_old[s] & 0x7FFFFFFFu) - 1] = to;
            p.refs[to] = 1;
            atomicSub(&p.refs[from], 1u);
        }
    }
    __syncthreads();
    for (uint32_t r = tid; r < s_granted; r += kPageThreads) {
        uint32_t lo = 0, hi = n - 1;  // the first sequence with s_upto > r
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (s_upto[mid] > r) hi = mid;
            else lo = mid + 1;
        }
        const uint32_t copied = s_old[lo] >> 31, k = r - (lo ? s_upto[lo - 1] : 0u);
        if (k < copied) continue;  // written above
        const uint32_t page = listed(r);
        p.table[(size_t)lo * p.table_stride + (s_old[lo] & 0x7FFFFFFFu) + k - copied] = page;
        p.refs[page] = 1;
    }
    if (tid == 0) {
        p.scratch[0] = s_refused;
        p.scratch[2] = s_moves;
    }
}

// Copies the moves' pages of every layer. Work items of 16 KiB, dealt over the grid; past the caches (48 pages in 28
// layers, 227 MB moved: a fork and an extend 69 -> 64 us; 2.5 GB moved by a compaction 532 -> 524 us, 4.9 TB/s).
constexpr uint32_t kMoveItem = 16384;
__device__ __forceinline__ void vx_copy_moves(const VxPages& p, uint32_t wg, uint32_t n_wgs) {
    const uint32_t moves = p.scratch[2];
    const uint32_t* src = p.scratch + kVxPagesHead;
    const uint32_t* dst = src + vx_pages_moves(p.n_seqs, p.n_pages);
    const uint32_t parts = (uint32_t)((p.page_bytes + kMoveItem - 1) / kMoveItem);
    const uint64_t items = (uint64_t)moves * p.n_layers * parts;
    for (uint64_t i = wg; i < items; i += n_wgs) {
        const uint32_t part = (uint32_t)(i % parts), layer = (uint32_t)(i / parts % p.n_layers), m = (uint32_t)(i / parts / p.n_layers);
        uint8_t* base = p.pool + (size_t)layer * p.layer_stride + (size_t)part * kMoveItem;
        const uint32_t bytes = (uint32_t)min((uint64_t)kMoveItem, p.page_bytes - (uint64_t)part * kMoveItem);
        const uint4* f = (const uint4*)(base + (size_t)src[m] * p.page_bytes);
        uint4* t = (uint4*)(base + (size_t)dst[m] * p.page_bytes);
        for (uint32_t k = threadIdx.x; k < bytes / 16; k += blockDim.x) vx_set<true>(t + k, vx_get<true>(f + k));
    }
}
__global__ __launch_bounds__(256) void vx_pages_copy_kernel(VxPages p) { vx_copy_moves(p, blockIdx.x, gridDim.x); }

// A workgroup takes a few columns of the table: all its entries are read into LDS before one is written, so
// that every sequence takes its parent's old pages whatever the order. References change by the difference;
// the sums do not depend on the order of the atomics. The last workgroup does the lengths.
constexpr uint32_t kForkWords = 16384;
constexpr int kForkThreads = 512;
__global__ __launch_bounds__(kForkThreads) void vx_pages_fork_kernel(VxPages p, const uint32_t* __restrict__ from, uint32_t cols) {
    __shared__ uint32_t old[kForkWords];
    const uint32_t n = p.n_seqs;
    if (blockIdx.x == gridDim.x - 1) {
        for (uint32_t s = threadIdx.x; s < n; s += kForkThreads) old[s] = p.lens[s];
        __syncthreads();
        for (uint32_t s = threadIdx.x; s < n; s += kForkThreads) {
            const uint32_t f = from[s], len = f < n ? old[f] : 0u;
            if (len != old[s]) p.lens[s] = len;
        }
        return;
    }
    const uint32_t c0 = blockIdx.x * cols, nc = min(cols, p.max_pages - c0);
    for (uint32_t i = threadIdx.x; i < n * nc; i += kForkThreads) old[i] = p.table[(size_t)(i / nc) * p.table_stride + c0 + i % nc];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n * nc; i += kForkThreads) {
        const uint32_t s = i / nc, c = i % nc, f = from[s];
        const uint32_t was = old[i], now = f < n ? old[f * nc + c] : kVxNoPage;
        if (was == now) continue;
        p.table[(size_t)s * p.table_stride + c0 + c] = now;
        if (now < p.n_pages) atomicAdd(&p.refs[now], 1u);
        if (was < p.n_pages) atomicSub(&p.refs[was], 1u);
    }
}

// An entry leaves the table by an exchange, so that a sequence listed twice gives its pages back once.
__device__ __forceinline__ void vx_drop(const VxPages& p, uint32_t s, uint32_t j) {
    const uint32_t was = atomicExch(&p.table[(size_t)s * p.table_stride + j], kVxNoPage);
    if (was < p.n_pages) atomicSub(&p.refs[was], 1u);
}
__global__ void vx_pages_free_kernel(VxPages p, const uint32_t* __restrict__ seqs, uint32_t n) {
    for (uint32_t i = blockIdx.y; i < n; i += gridDim.y) {
        const uint32_t s = seqs[i];
        if (s >= p.n_seqs) continue;
        for (uint32_t j = blockIdx.x * blockDim.x + threadIdx.x; j < p.max_pages; j += gridDim.x * blockDim.x) vx_drop(p, s, j);
        if (blockIdx.x == 0 && threadIdx.x == 0) p.lens[s] = 0;
    }
}
__global__ void vx_pages_trim_kernel(VxPages p, uint32_t window, uint32_t sinks) {
    for (uint32_t s = blockIdx.y; s < p.n_seqs; s += gridDim.y) {
        const uint64_t len = p.lens[s];
        if (len + 1 <= window) continue;
        const uint64_t j0 = ((uint64_t)sinks + p.page_size - 1) / p.page_size;
        const uint64_t j1 = min((len + 1 - window) / p.page_size, (uint64_t)p.max_pages);
        for (uint64_t j = j0 + blockIdx.x * blockDim.x + threadIdx.x; j < j1; j += gridDim.x * blockDim.x) vx_drop(p, s, (uint32_t)j);
    }
}

__global__ __launch_bounds__(kPageThreads) void vx_pages_count_kernel(VxPages p) {
    uint32_t free = 0, total;
    for (uint32_t i = threadIdx.x; i < p.n_pages; i += kPageThreads) free += p.refs[i] == 0;
    vx_scan(free, total);
    if (threadIdx.x == 0) p.scratch[1] = total;
}

// One workgroup plans the moves: with L live pages, the k-th free place below L takes the k-th live page from
// L on (there are as many of the one as of the other), and the map of pages from L on says where each went.
__global__ __launch_bounds__(kPageThreads) void vx_pages_plan_kernel(VxPages p) {
    const uint32_t tid = threadIdx.x;
    uint32_t* src = p.scratch + kVxPagesHead;
    uint32_t* dst = src + vx_pages_moves(p.n_seqs, p.n_pages);
    uint32_t* map = dst + vx_pages_moves(p.n_seqs, p.n_pages);
    uint32_t live = 0, total;
    VxRefs8 refs;
    for (uint32_t base = 0; base < p.n_pages; base += kPageThreads * 8) {
        refs.load(p, base + tid * 8);
        live += refs.n - __popc(refs.free());
    }
    vx_scan(live, total);
    uint32_t holes = 0, moved = 0;
    for (uint32_t base = 0; base < p.n_pages; base += kPageThreads * 8) {
        const uint32_t first = base + tid * 8;
        if (p.n_pages > kPageThreads * 8) refs.load(p, first);
        const uint32_t free = refs.free(), there = (1u << refs.n) - 1u;
        const uint32_t front = first >= total ? 0u : total - first >= 8 ? 255u : (1u << (total - first)) - 1u;  // of the first L pages
        uint32_t hole = free & front, move = ~free & there & ~front;
        for (uint32_t dead = free & ~front; dead; dead &= dead - 1) map[first + __builtin_ctz(dead)] = kVxNoPage;
        // at most 8192 of either in a tile: both counts in one scan
        uint32_t got;
        const uint32_t at = vx_scan(__popc(hole) | __popc(move) << 16, got);
        uint32_t h = holes + (at & 0xFFFFu), m = moved + (at >> 16);
        for (; hole; hole &= hole - 1) dst[h++] = first + __builtin_ctz(hole);
        for (; move; move &= move - 1) src[m++] = first + __builtin_ctz(move);
        holes += got & 0xFFFFu;
        moved += got >> 16;
    }
    __syncthreads();
    for (uint32_t i = tid; i < moved; i += kPageThreads) {
        const uint32_t a = src[i], b = dst[i];
        map[a] = b;
        p.refs[b] = p.refs[a];
        p.refs[a] = 0;
    }
    if (tid == 0) {
        p.scratch[2] = moved;
        p.scratch[3] = total;
    }
}
// The table follows the map, beside the copies of the data.
__global__ __launch_bounds__(256) void vx_pages_move_kernel(VxPages p, uint32_t table_wgs) {
    if (blockIdx.x >= table_wgs) {
        vx_copy_moves(p, blockIdx.x - table_wgs, gridDim.x - table_wgs);
        return;
    }
    const uint32_t live = p.scratch[3];
    const uint32_t* map = p.scratch + kVxPagesHead + 2 * (size_t)vx_pages_moves(p.n_seqs, p.n_pages);
    const size_t n = (size_t)p.n_seqs * p.max_pages;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)table_wgs * 256) {
        uint32_t* e = &p.table[i / p.max_pages * p.table_stride + i % p.max_pages];
        const uint32_t was = *e;
        if (was >= live && was < p.n_pages) *e = map[was];
    }
}

uint32_t grid_of(uint64_t items, uint32_t most) { return (uint32_t)(items < 1 ? 1 : items > most ? most : items); }
uint32_t copy_grid(const VxPages& p, uint64_t moves) {
    return grid_of(moves * p.n_layers * ((p.page_bytes + kMoveItem - 1) / kMoveItem), 2048);
}

}  // namespace

// Rows of more bytes than the XCDs' L2 caches hold go past them (non-temporal): what reads them next finds them in
// memory anyway. 4001 rows of 64 heads of 128 (fp16, 131 MB moved, cold) 31.1 -> 24.3 us by non-temporal stores
// (loads made it 30.9); 8531 rows of Llama-3-8B's q, k and v (210 MB) 63 -> 47 us by both.
static constexpr uint64_t kStreamBytes = 32ull << 20;

// Whether 16-byte loads and stores fit rows of type elements.
static bool vx_vec_rows(const VxRowsView& r) {
    const uint32_t v = r.dtype == VELOX_DT_F32 ? 4 : 8;
    return (uintptr_t)r.data % 16 == 0 && r.rs % v == 0 && (r.heads == 1 || r.hs % v == 0);
}
static bool vx_vec_pairs(const VxRopeTable& t, uint32_t dtype, uint32_t d) {
    const uint32_t v = dtype == VELOX_DT_F32 ? 4 : 8;
    return d % v == 0 && (t.interleaved ? t.rot % v == 0 : t.rot % (2 * v) == 0);
}

hipError_t vx_launch_rope_rows(const VxRopeTable& t, const VxRowsView& x, const VxRowsView& out, uint32_t n_rows,
                               uint32_t d, const uint32_t* positions, hipStream_t st) {
    if (vx_vec_rows(x) && vx_vec_rows(out) && vx_vec_pairs(t, x.dtype, d)) {
        // a thread for every angle where the rows fill the GPU several times over, one row a workgroup below
        const uint32_t most = 2 * kRopeThreads / t.rot, share = n_rows / 1024, per = share < 1 ? 1 : share < most ? share : most;
        const uint32_t grid = (n_rows + per - 1) / per;
        const bool nt = (uint64_t)n_rows * x.heads * d * (x.dtype == VELOX_DT_F32 ? 4 : 2) > kStreamBytes;
        const auto go = [&](auto kernel) { kernel<<<grid, kRopeThreads, 0, st>>>(t, x, out, n_rows, d, positions, per); };
        if (x.dtype == VELOX_DT_F32) go(nt ? vx_rope_vec_kernel<float, true> : vx_rope_vec_kernel<float, false>);
        else if (x.dtype == VELOX_DT_F16) go(nt ? vx_rope_vec_kernel<_Float16, true> : vx_rope_vec_kernel<_Float16, false>);
        else go(nt ? vx_rope_vec_kernel<__bf16, true> : vx_rope_vec_kernel<__bf16, false>);
    } else {
        vx_rope_rows_kernel<<<n_rows, kRopeThreads, 0, st>>>(t, x, out, n_rows, d, positions);
    }
    return hipGetLastError();
}

template <class T>
static void vx_append_vec(const VxRopeTable& t, const VxAppendArgs& a, dim3 grid, hipStream_t st) {
    const bool nt = (uint64_t)a.n_rows * ((a.q.data ? a.q.heads : 0) + 2 * a.c.hkv) * a.c.d * sizeof(T) > kStreamBytes;
    const auto go = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(t, a); };
    if (a.c.dtype == VELOX_DT_F16) go(nt ? vx_append_vec_kernel<T, _Float16, true> : vx_append_vec_kernel<T, _Float16, false>);
    else go(nt ? vx_append_vec_kernel<T, __bf16, true> : vx_append_vec_kernel<T, __bf16, false>);
}

hipError_t vx_launch_rope_append(const VxRopeTable& t, const VxAppendArgs& a, hipStream_t st) {
    // a sequence's rows touch at most rows / 32 + 2 blocks
    const uint64_t bound = (uint64_t)a.n_rows / 32 + 2ull * a.c.n_seqs;
    const uint32_t blocks = (uint32_t)(bound < a.n_rows ? bound : a.n_rows);
    // Heads are shared out over 8 workgroups of a block; over 2 where there are many blocks of few rows (one row each of 512
    // sequences of Qwen2.5-7B 15.5 us by 8, 8.3 by 2; of 8 sequences 3.6 and 3.8; prompts of 8531 rows 43.6 and 51.6).
    const dim3 grid(blocks, blocks > 64 && a.n_rows < 4 * (uint64_t)blocks ? 2 : 8);
    const bool vec = (!a.q.data || (vx_vec_rows(a.q) && vx_vec_rows(a.qo) && a.q.dtype == a.k.dtype)) && vx_vec_rows(a.k) &&
                     vx_vec_rows(a.v) && a.k.dtype == a.v.dtype && vx_vec_pairs(t, a.k.dtype, a.c.d);
    if (!vec) vx_append_rows_kernel<<<grid, 256, 0, st>>>(t, a);
    else if (a.k.dtype == VELOX_DT_F32) vx_append_vec<float>(t, a, grid, st);
    else if (a.k.dtype == VELOX_DT_F16) vx_append_vec<_Float16>(t, a, grid, st);
    else vx_append_vec<__bf16>(t, a, grid, st);
    return hipGetLastError();
}

hipError_t vx_launch_pages_reset(const VxPages& p, hipStream_t st) {
    const uint64_t n = (uint64_t)p.n_seqs * p.max_pages;
    vx_pages_reset_kernel<<<grid_of(((n > p.n_pages ? n : p.n_pages) + 255) / 256, 1024), 256, 0, st>>>(p);
    return hipGetLastError();
}

hipError_t vx_launch_pages_extend(const VxPages& p, const uint32_t* add, hipStream_t st) {
    vx_pages_extend_kernel<<<1, kPageThreads, 0, st>>>(p, add);
    vx_pages_copy_kernel<<<copy_grid(p, p.n_seqs), 256, 0, st>>>(p);
    return hipGetLastError();
}

hipError_t vx_launch_pages_fork(const VxPages& p, const uint32_t* src, hipStream_t st) {
    // about 2048 entries a workgroup, in runs of four columns at least (n_seqs <= 4096: they fit)
    uint32_t cols = 2048 / p.n_seqs;
    if (cols < 4) cols = 4;
    if (cols > p.max_pages) cols = p.max_pages;
    vx_pages_fork_kernel<<<(p.max_pages + cols - 1) / cols + 1, kForkThreads, 0, st>>>(p, src, cols);
    return hipGetLastError();
}

hipError_t vx_launch_pages_free(const VxPages& p, const uint32_t* seqs, uint32_t n, hipStream_t st) {
    vx_pages_free_kernel<<<dim3(grid_of((p.max_pages + 255) / 256, 64), grid_of(n, 4096)), 256, 0, st>>>(p, seqs, n);
    return hipGetLastError();
}

hipError_t vx_launch_pages_trim(const VxPages& p, uint32_t window, uint32_t sinks, hipStream_t st) {
    vx_pages_trim_kernel<<<dim3(grid_of((p.max_pages + 255) / 256, 64), grid_of(p.n_seqs, 4096)), 256, 0, st>>>(p, window, sinks);
    return hipGetLastError();
}

hipError_t vx_launch_pages_compact(const VxPages& p, hipStream_t st) {
    vx_pages_plan_kernel<<<1, kPageThreads, 0, st>>>(p);
    const uint32_t table_wgs = grid_of(((uint64_t)p.n_seqs * p.max_pages + 1023) / 1024, 256);
    vx_pages_move_kernel<<<table_wgs + copy_grid(p, p.n_pages / 2), 256, 0, st>>>(p, table_wgs);
    return hipGetLastError();
}

hipError_t vx_launch_pages_count(const VxPages& p, hipStream_t st) {
    vx_pages_count_kernel<<<1, kPageThreads, 0, st>>>(p);
    return hipGetLastError();
}
