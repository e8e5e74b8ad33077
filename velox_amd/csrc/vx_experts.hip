// vx_experts.hip -- the choice of experts, the grouping of rows by expert, the sum of the experts' answers.
#include "vx_int8.h"

namespace {

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
constexpr uint32_t kGroupWaves = 4, kGroupRun = 512, kGroupSlots = kGroupWaves * kGroupRun;  // a wave's, a workgroup's slots

// The expert of slot i of a run (count: none of ours).
__device__ __forceinline__ uint32_t vx_key(const VxGroupArgs& a, uint32_t i) {
    if (i >= a.n_slots) return a.count;
    const uint32_t e = a.ids[i] - a.first;
    return e < a.count ? e : a.count;
}
// The lanes of the wave whose key is this lane's.
__device__ __forceinline__ uint64_t vx_peers(uint32_t key) {
    uint64_t m = ~0ull;
#pragma unroll
    for (int b = 0; b < 11; ++b) {
        const uint64_t v = __ballot(key >> b & 1u);
        m &= key >> b & 1u ? v : ~v;
    }
    return m;
}
// What a lane of the wave wrote to LDS is what the others read behind this.
__device__ __forceinline__ void vx_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// How many slots of each expert every wave's run holds: tally[wave][count + 1].
__device__ __forceinline__ void vx_tally(const VxGroupArgs& a, uint32_t block, uint32_t* tally) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, n = a.count + 1u;
    for (uint32_t i = threadIdx.x; i < kGroupWaves * n; i += 64u * kGroupWaves) tally[i] = 0;
    __syncthreads();
    const uint32_t run = block * kGroupSlots + wave * kGroupRun;
    for (uint32_t i = 0; i < kGroupRun; i += 64u) {
        const uint32_t key = vx_key(a, run + i + lane);
        const uint64_t peers = vx_peers(key);
        if (lane == (uint32_t)__builtin_ctzll(peers)) tally[wave * n + key] += (uint32_t)__popcll(peers);
        vx_wave_sync();
    }
    __syncthreads();
}
__global__ __launch_bounds__(64 * kGroupWaves) void vx_group_count_kernel(VxGroupArgs a) {
    __shared__ uint32_t tally[kGroupWaves * (kVxI8MaxCount + 1u)];
    vx_tally(a, blockIdx.x, tally);
    for (uint32_t e = threadIdx.x; e < a.count; e += 64u * kGroupWaves) {
        uint32_t n = 0;
        for (uint32_t w = 0; w < kGroupWaves; ++w) n += tally[w * (a.count + 1u) + e];
        a.hist[(size_t)blockIdx.x * a.count + e] = n;
    }
}
// Exclusive sums of v over the workgroup's threads, the total in `total`; room: kGroupWaves words.
__device__ __forceinline__ uint32_t vx_scan(uint32_t v, uint32_t* room, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(s, off);
        if (lane >= (uint32_t)off) s += o;
    }
    if (lane == 63u) room[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < kGroupWaves; ++w) {
        if (w < wave) before += room[w];
        total += room[w];
    }
    __syncthreads();
    return before + s - v;
}
__global__ __launch_bounds__(64 * kGroupWaves) void vx_group_place_kernel(VxGroupArgs a) {
    __shared__ uint32_t tally[kGroupWaves * (kVxI8MaxCount + 1u)];
    __shared__ uint32_t room[kGroupWaves];
    constexpr uint32_t T = 64u * kGroupWaves, PER = kVxI8MaxCount / T;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, n = a.count + 1u, block = blockIdx.x, blocks = gridDim.x;
    vx_tally(a, block, tally);
    // thread t: experts PER t .. + PER - 1
    uint32_t mine[PER], front[PER], sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        mine[j] = front[j] = 0;
        if (e < a.count) {
            if (blocks == 1u) {
                for (uint32_t w = 0; w < kGroupWaves; ++w) mine[j] += tally[w * n + e];
            } else {
                for (uint32_t b = 0; b < blocks; ++b) {
                    const uint32_t c = a.hist[(size_t)b * a.count + e];
                    if (b < block) front[j] += c;
                    mine[j] += c;
                }
            }
        }
        sum += mine[j];
    }
    uint32_t total;
    uint32_t at = vx_scan(sum, room, total);
    uint32_t items = 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) items += (mine[j] + a.item_rows - 1u) / a.item_rows;
    uint32_t n_items;
    uint32_t item = vx_scan(items, room, n_items);
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        if (e < a.count) {
            if (block == 0) {
                a.offsets[e] = at;
                if (a.items)
                    for (uint32_t p = 0; p < mine[j]; p += a.item_rows) a.items[item++] = make_uint2(e, at + p);
            }
            // each wave's first place of the expert
            uint32_t place = at + front[j];
            for (uint32_t w = 0; w < kGroupWaves; ++w) {
                const uint32_t c = tally[w * n + e];
                tally[w * n + e] = place;
                place += c;
            }
        }
        at += mine[j];
    }
    if (block == 0 && threadIdx.x == 0) {
        a.offsets[a.count] = total;
        if (a.items) *a.n_items = n_items;
    }
    __syncthreads();
    const uint32_t run = block * kGroupSlots + wave * kGroupRun;
    for (uint32_t i = 0; i < kGroupRun; i += 64u) {
        const uint32_t slot = run + i + lane, key = vx_key(a, slot);
        const uint64_t peers = vx_peers(key);
        const uint32_t rank = (uint32_t)__popcll(peers & ((1ull << lane) - 1ull));
        if (key < a.count) {
            const uint32_t place = tally[wave * n + key];
            a.order[place + rank] = slot;
            vx_wave_sync();
            if (rank == 0) tally[wave * n + key] = place + (uint32_t)__popcll(peers);
        }
        vx_wave_sync();
    }
    for (uint32_t p = total + block * T + threadIdx.x; p < a.n_slots; p += blocks * T) a.order[p] = kVxNoExpert;
}

// ---- the sum of a row's experts ----
__global__ __launch_bounds__(256) void vx_combine_kernel(VxCombineArgs a) {
    const uint32_t r = blockIdx.x;
    for (uint32_t c = threadIdx.x; c < a.n; c += 256u) {
        float y = a.res.data ? vx_load(a.res.data, (size_t)r * a.res.rs + c, a.res.dtype) : 0.0f;
        float sum = 0.0f;
        for (uint32_t j = 0; j < a.top; ++j) {
            const size_t slot = (size_t)r * a.top + j;
            if (a.ids[slot] - a.first < a.count) sum = __builtin_fmaf(a.weights[slot], a.part[slot * a.part_stride + c], sum);
        }
        vx_store(a.out.data, (size_t)r * a.out.rs + c, a.out.dtype, y + sum);
    }
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

hipError_t vx_launch_group(const VxGroupArgs& a, hipStream_t st) {
    const uint32_t blocks = vx_group_blocks(a.n_slots);
    if (blocks > 1u) {
        hipLaunchKernelGGL(vx_group_count_kernel, dim3(blocks), dim3(64 * kGroupWaves), 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(vx_group_place_kernel, dim3(blocks), dim3(64 * kGroupWaves), 0, st, a);
    return hipGetLastError();
}

hipError_t vx_launch_combine(const VxCombineArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(vx_combine_kernel, dim3(a.n_rows), dim3(256), 0, st, a);
    return hipGetLastError();
}
