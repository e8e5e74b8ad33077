// vx_experts.hip -- the choice of experts, the grouping of rows by expert, the sum of the experts' answers.
#include "vx_int8_dev.h"

namespace {

// ---- routing ----
constexpr uint32_t kRouteItems = kVxI8MaxCount / 64u;  // experts of a lane at most

// One wave per row; lane l holds experts l, l + 64, ... Choice values are 64-bit numbers; an expert that takes no part has
// -infinity.
template <uint32_t ITEMS>
__global__ __launch_bounds__(256) void vx_route_kernel(VxRouteArgs a) {
    __shared__ double all[4][ITEMS * 64u];
    __shared__ double marks[4][kVxMaxGroups];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, r = blockIdx.x * 4u + wave;
    const bool live = r < a.n_rows;  // (barriers below: every wave goes on)
    double score[ITEMS], pick[ITEMS];
    double top = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < ITEMS; ++i) {
        const uint32_t e = lane + 64u * i;
        float x = -INFINITY;
        if (live && e < a.n_experts) x = vx_load(a.x.data, (size_t)r * a.x.rs + e, a.x.dtype);
        x = x > -INFINITY ? fminf(x, 3.40282347e38f) : -INFINITY;  // (NaN too)
        score[i] = x;
        top = fmax(top, score[i]);
    }
    const bool by_logits = !a.sigmoid && !a.bias && !a.two;
    if (a.sigmoid) {
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) {
            const double x = score[i];
            score[i] = 1.0 / (1.0 + exp(-x));
            pick[i] = x > -INFINITY ? score[i] : -INFINITY;
        }
    } else {
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = fmax(top, __shfl_xor(top, off));
        double sum = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) {
            const double x = score[i];
            score[i] = x > -INFINITY ? exp(x - top) : 0.0;
            sum += score[i];
            pick[i] = x;
        }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) {
            score[i] = sum > 0.0 ? score[i] / sum : 0.0;
            if (!by_logits) pick[i] = pick[i] > -INFINITY ? score[i] : -INFINITY;
        }
    }
    if (a.bias) {
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) {
            const uint32_t e = lane + 64u * i;
            const float b = e < a.n_experts ? a.bias[e] : 0.0f;
            pick[i] = pick[i] > -INFINITY && fabsf(b) < INFINITY ? pick[i] + b : -INFINITY;
        }
    }
    if (a.groups > 1u) {
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) all[wave][lane + 64u * i] = pick[i];
        __syncthreads();
        const uint32_t size = a.n_experts / a.groups;
        double best = -INFINITY, next = -INFINITY;
        if (lane < a.groups)
            for (uint32_t j = 0; j < size; ++j) {
                const double v = all[wave][lane * size + j];
                next = fmax(next, fmin(best, v));
                best = fmax(best, v);
            }
        const double mark = a.two && next > -INFINITY ? best + next : best;
        marks[wave][lane] = mark;
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t g = 0; g < a.groups; ++g) {
            const double m = marks[wave][g];
            before += m > mark || (m == mark && g < lane);
        }
        const uint64_t open = __ballot(lane < a.groups && before < a.top_groups);
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) {
            const uint32_t e = lane + 64u * i;
            if (e < a.n_experts && !(open >> (e / size) & 1u)) pick[i] = -INFINITY;
        }
    }
    double mine = 0.0, total = 0.0;  // lane j: the j-th score
    uint32_t id = kVxNoExpert;
    for (uint32_t j = 0; j < a.top; ++j) {
        double best = -INFINITY, s = 0.0;
        uint32_t at = 0xFFFFFFFFu;
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i)
            if (pick[i] > best) {
                best = pick[i];
                s = score[i];
                at = lane + 64u * i;
            }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double ob = __shfl_xor(best, off), os = __shfl_xor(s, off);
            const uint32_t oa = __shfl_xor(at, off);
            if (ob > best || (ob == best && oa < at)) {
                best = ob;
                s = os;
                at = oa;
            }
        }
        if (at == 0xFFFFFFFFu) break;  // (uniform)
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i)
            if (at == lane + 64u * i) pick[i] = -INFINITY;
        if (lane == j) {
            id = at;
            mine = s;
        }
        total += s;
    }
    if (!live || lane >= a.top) return;
    if (a.renorm) mine = total > 0.0 ? mine / total : 0.0;
    a.ids[(size_t)r * a.top + lane] = id;
    a.weights[(size_t)r * a.top + lane] = (float)(mine * a.scale);
}

// ---- grouping: a stable counting sort of the slots by expert ----
// A workgroup takes kGroupSlots slots, a wave kGroupRun neighbours of them. Slots of one expert within a wave find each other by
// ballots of their keys' bits, so that ranks follow the slots' order; waves' and workgroups' counts are summed in order.
// Several workgroups count first (their counts through memory), then place; one does both at once.
constexpr uint32_t kGroupWaves = 4, kGroupRun = 256, kGroupSlots = kGroupWaves * kGroupRun, kGroupSteps = kGroupRun / 64u;
constexpr uint32_t kGroupThreads = 64u * kGroupWaves;

// A wave's keys: slot run + 64 i + lane's expert, or a.count (none of ours).
struct VxKeys {
    uint32_t key[kGroupSteps];
    uint32_t steps;  // those with slots
};
__device__ __forceinline__ VxKeys vx_keys(const VxGroupArgs& a, uint32_t run) {
    const uint32_t lane = threadIdx.x & 63u;
    VxKeys k;
    k.steps = run < a.n_slots ? (a.n_slots - run + 63u) / 64u : 0u;
    k.steps = k.steps < kGroupSteps ? k.steps : kGroupSteps;
#pragma unroll
    for (uint32_t i = 0; i < kGroupSteps; ++i) {
        const uint32_t slot = run + 64u * i + lane, e = slot < a.n_slots ? a.ids[slot] - a.first : a.count;
        k.key[i] = e < a.count ? e : a.count;
    }
    return k;
}
// The lanes of the wave whose key is this lane's.
__device__ __forceinline__ uint64_t vx_peers(uint32_t key, uint32_t bits) {
    uint64_t m = ~0ull;
    for (uint32_t b = 0; b < bits; ++b) {
        const bool mine = key >> b & 1u;
        const uint64_t v = __ballot(mine);
        m &= mine ? v : ~v;
    }
    return m;
}
// How many slots of each expert every wave's run holds: tally[wave][count + 1].
__device__ __forceinline__ void vx_tally(const VxGroupArgs& a, const VxKeys& k, uint32_t* tally) {
    const uint32_t lane = threadIdx.x & 63u, n = a.count + 1u;
    uint32_t* mine = tally + (threadIdx.x >> 6) * n;
    for (uint32_t i = lane; i < n; i += 64u) mine[i] = 0;
    vx_wave_sync();
#pragma unroll
    for (uint32_t i = 0; i < kGroupSteps; ++i) {
        if (i >= k.steps) break;
        const uint64_t peers = vx_peers(k.key[i], a.key_bits);
        if (lane == (uint32_t)__builtin_ctzll(peers)) mine[k.key[i]] += (uint32_t)__popcll(peers);
        vx_wave_sync();
    }
    __syncthreads();
}
__global__ __launch_bounds__(kGroupThreads) void vx_group_count_kernel(VxGroupArgs a) {
    __shared__ uint32_t tally[kGroupWaves * (kVxI8MaxCount + 1u)];
    vx_tally(a, vx_keys(a, blockIdx.x * kGroupSlots + (threadIdx.x >> 6) * kGroupRun), tally);
    for (uint32_t e = threadIdx.x; e < a.count; e += kGroupThreads) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t w = 0; w < kGroupWaves; ++w) n += tally[w * (a.count + 1u) + e];
        a.hist[(size_t)blockIdx.x * a.count + e] = n;
    }
}
// Exclusive sums of u and v (the latter below 2^32) over the workgroup's threads, and the totals; room: 2 kGroupWaves words.
__device__ __forceinline__ uint2 vx_scan(uint2 v, uint32_t* room, uint2& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint2 s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t x = __shfl_up(s.x, off), y = __shfl_up(s.y, off);
        if (lane >= (uint32_t)off) {
            s.x += x;
            s.y += y;
        }
    }
    if (lane == 63u) {
        room[2u * wave] = s.x;
        room[2u * wave + 1u] = s.y;
    }
    __syncthreads();
    uint2 before = make_uint2(0, 0);
    total = before;
#pragma unroll
    for (uint32_t w = 0; w < kGroupWaves; ++w) {
        if (w < wave) before = make_uint2(before.x + room[2u * w], before.y + room[2u * w + 1u]);
        total = make_uint2(total.x + room[2u * w], total.y + room[2u * w + 1u]);
    }
    return make_uint2(before.x + s.x - v.x, before.y + s.y - v.y);
}
// PER: experts of a thread, neighbours.
template <uint32_t PER>
__global__ __launch_bounds__(kGroupThreads) void vx_group_place_kernel(VxGroupArgs a) {
    __shared__ uint32_t tally[kGroupWaves * (kVxI8MaxCount + 1u)];
    __shared__ uint32_t room[2u * kGroupWaves];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, n = a.count + 1u, block = blockIdx.x, blocks = gridDim.x;
    const uint32_t run = block * kGroupSlots + wave * kGroupRun;
    const VxKeys k = vx_keys(a, run);
    uint32_t mine[PER], front[PER];
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        mine[j] = front[j] = 0;
        if (blocks > 1u && e < a.count) {
#pragma unroll 16
            for (uint32_t b = 0; b < blocks; ++b) {
                const uint32_t c = a.hist[(size_t)b * a.count + e];
                front[j] += b < block ? c : 0u;
                mine[j] += c;
            }
        }
    }
    vx_tally(a, k, tally);
    uint2 sum = make_uint2(0, 0);  // slots and blocks of a grouped product
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        if (blocks == 1u && e < a.count) {
#pragma unroll
            for (uint32_t w = 0; w < kGroupWaves; ++w) mine[j] += tally[w * n + e];
        }
        sum.x += mine[j];
        sum.y += (mine[j] + a.item_rows - 1u) / a.item_rows;
    }
    uint2 total, at = vx_scan(sum, room, total);
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        if (e < a.count) {
            if (block == 0) {
                a.offsets[e] = at.x;
                if (a.items)
                    for (uint32_t p = 0; p < mine[j]; p += a.item_rows) a.items[at.y++] = make_uint2(e, at.x + p);
            }
            uint32_t place = at.x + front[j];  // each wave's first place of the expert
#pragma unroll
            for (uint32_t w = 0; w < kGroupWaves; ++w) {
                const uint32_t c = tally[w * n + e];
                tally[w * n + e] = place;
                place += c;
            }
        }
        at.x += mine[j];
    }
    if (block == 0 && threadIdx.x == 0) {
        a.offsets[a.count] = total.x;
        if (a.items) *a.n_items = total.y;
    }
    __syncthreads();
    uint32_t* places = tally + wave * n;
#pragma unroll
    for (uint32_t i = 0; i < kGroupSteps; ++i) {
        if (i >= k.steps) break;
        const uint32_t key = k.key[i];
        const uint64_t peers = vx_peers(key, a.key_bits);
        const uint32_t rank = (uint32_t)__popcll(peers & ((1ull << lane) - 1ull)), place = places[key];
        vx_wave_sync();
        if (key < a.count) {
            a.order[place + rank] = run + 64u * i + lane;
            if (rank == 0) places[key] = place + (uint32_t)__popcll(peers);
        }
        vx_wave_sync();
    }
    for (uint32_t p = total.x + block * kGroupThreads + threadIdx.x; p < a.n_slots; p += blocks * kGroupThreads) a.order[p] = kVxNoExpert;
}

// ---- the sum of a row's experts ----
// A workgroup takes 1024 outputs of a row, a thread four. Lane j of a wave looks at the row's slot j; the slots of our
// experts are then added in order, four of their answers on the way at a time.
constexpr uint32_t kCombineCols = 1024u;
template <bool VEC>
__global__ __launch_bounds__(256) void vx_combine_kernel(VxCombineArgs a, uint32_t blocks) {
    const uint32_t r = blockIdx.x / blocks, c = blockIdx.x % blocks * kCombineCols + 4u * threadIdx.x, lane = threadIdx.x & 63u;
    const size_t slot0 = (size_t)r * a.top;
    const bool mine = lane < a.top && a.ids[slot0 + lane] - a.first < a.count;
    const float w = mine ? a.weights[slot0 + lane] : 0.0f;
    uint64_t left = __ballot(mine);
    if (c >= a.n) return;
    float4 res = make_float4(0, 0, 0, 0);
    if (a.res.data) res = vx_load4<VEC>(a.res.data, (size_t)r * a.res.rs + c, a.res.dtype, a.n - c);
    const float* part = a.part + slot0 * a.part_stride + c;
    float4 sum = make_float4(0, 0, 0, 0);
    while (left) {
        float4 v[4];
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t at = left ? (uint32_t)__builtin_ctzll(left) : 0u;
            f[j] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), (int)at));
            v[j] = make_float4(0, 0, 0, 0);
            if (left) v[j] = *(const float4*)(part + at * a.part_stride);
            else f[j] = 0.0f;
            left &= left - 1u;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            sum = make_float4(__builtin_fmaf(f[j], v[j].x, sum.x), __builtin_fmaf(f[j], v[j].y, sum.y), __builtin_fmaf(f[j], v[j].z, sum.z), __builtin_fmaf(f[j], v[j].w, sum.w));
    }
    vx_store4<VEC>(a.out.data, (size_t)r * a.out.rs + c, a.out.dtype, a.n - c, make_float4(res.x + sum.x, res.y + sum.y, res.z + sum.z, res.w + sum.w));
}

}  // namespace

hipError_t vx_launch_route(const VxRouteArgs& a, hipStream_t st) {
    const dim3 grid((a.n_rows + 3u) / 4u);
    if (a.n_experts <= 64u) hipLaunchKernelGGL((vx_route_kernel<1>), grid, dim3(256), 0, st, a);
    else if (a.n_experts <= 256u) hipLaunchKernelGGL((vx_route_kernel<4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((vx_route_kernel<kRouteItems>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

uint32_t vx_group_blocks(uint32_t n_slots) { return n_slots ? (n_slots + kGroupSlots - 1u) / kGroupSlots : 1u; }

hipError_t vx_launch_group(const VxGroupArgs& args, hipStream_t st) {
    VxGroupArgs a = args;
    a.key_bits = 32u - (uint32_t)__builtin_clz(a.count);  // keys 0 .. count
    const uint32_t blocks = vx_group_blocks(a.n_slots);
    if (blocks > 1u) {
        hipLaunchKernelGGL(vx_group_count_kernel, dim3(blocks), dim3(kGroupThreads), 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (a.count <= kGroupThreads) hipLaunchKernelGGL((vx_group_place_kernel<1>), dim3(blocks), dim3(kGroupThreads), 0, st, a);
    else hipLaunchKernelGGL((vx_group_place_kernel<kVxI8MaxCount / kGroupThreads>), dim3(blocks), dim3(kGroupThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t vx_launch_combine(const VxCombineArgs& a, hipStream_t st) {
    const uint32_t blocks = (a.n + kCombineCols - 1u) / kCombineCols;
    if (a.vec) hipLaunchKernelGGL((vx_combine_kernel<true>), dim3(a.n_rows * blocks), dim3(256), 0, st, a, blocks);
    else hipLaunchKernelGGL((vx_combine_kernel<false>), dim3(a.n_rows * blocks), dim3(256), 0, st, a, blocks);
    return hipGetLastError();
}
