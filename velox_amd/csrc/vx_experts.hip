// vx_experts.hip -- the choice of experts, the grouping of rows by expert, the sum of the experts' answers.
#include "vx_int8_dev.h"

namespace {

// ---- routing ----
// The largest of the wave's values, in every lane's reach as a scalar.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t vx_max_dpp(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
    return v > o ? v : o;
}
__device__ __forceinline__ uint32_t vx_wave_max(uint32_t v) {
    v = vx_max_dpp<0x111, 0xF>(v);  // from the lanes 1, 2, 4, 8 below in a row of 16, then from the rows below
    v = vx_max_dpp<0x112, 0xF>(v);
    v = vx_max_dpp<0x114, 0xF>(v);
    v = vx_max_dpp<0x118, 0xF>(v);
    v = vx_max_dpp<0x142, 0xA>(v);
    v = vx_max_dpp<0x143, 0xC>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// Numbers as unsigned words of the same order (-0 below +0: callers add 0), and back.
__device__ __forceinline__ uint32_t vx_word_of(float f) {
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float vx_float_of(uint32_t w) { return __builtin_bit_cast(float, w & 0x80000000u ? w & 0x7FFFFFFFu : ~w); }
// Whether a is above b for certain, where they are sums of numbers of sizes as and bs, each off by less than kVxOff (1 + its
// size): a score in fp32 is off by 22 of its half steps at most (a sum of 1024), its sum with a bias by one more.
constexpr float kVxOff = 1.9073486e-6f;  // 2^-19
__device__ __forceinline__ bool vx_above(float a, float as, float b, float bs) { return a - b > kVxOff * (4.0f + as + bs); }

// A row's groups that take part, as a mask, by marks of the choice values in `all` (LDS, one wave's). L lanes a group.
template <class F>
__device__ __forceinline__ uint64_t vx_open_groups(const VxRouteArgs& a, const F* all, F* marks, bool& unsure) {
    const uint32_t lane = threadIdx.x & 63u, size = a.group_size, L = 1u << a.group_lanes, g = lane >> a.group_lanes, sub = lane & (L - 1u);
    F best = -INFINITY, next = -INFINITY;
    if (g < a.groups)
        for (uint32_t j = sub; j < size; j += L) {
            const F v = all[g * size + j];
            const F low = best < v ? best : v;
            next = next > low ? next : low;
            best = best > v ? best : v;
        }
    for (uint32_t off = 1; off < L; off <<= 1) {
        const F ob = __shfl_xor(best, (int)off), on = __shfl_xor(next, (int)off);
        const F low = best < ob ? best : ob, high = next > on ? next : on;
        next = low > high ? low : high;
        best = best > ob ? best : ob;
    }
    const F mark = a.two && next > -INFINITY ? best + next : best;
    if (sub == 0 && g < a.groups) {
        marks[g] = mark;
        if constexpr (sizeof(F) == 4) marks[kVxMaxGroups + g] = best > -INFINITY ? fabsf(best) + (a.two && next > -INFINITY ? fabsf(next) : 0.0f) : 0.0f;
    }
    vx_wave_sync();
    uint32_t before = 0;  // lane g: the marks in front of group g's
    const F my = marks[lane < a.groups ? lane : 0u];
    for (uint32_t j = 0; j < a.groups; ++j) {
        const F m = marks[j];
        before += m > my || (m == my && j < lane);
    }
    const bool in = lane < a.groups && before < a.top_groups;
    const uint64_t open = __ballot(in);
    if constexpr (sizeof(F) == 4) {
        // The least that a group that is in may be has to be above the most that one that is out may be: not the neighbours' in the
        // order alone, since a mark of two may be off by far more than it is (1e7 + -1e7). One whose parts, or whose sum, overflow may
        // be anything; a group without an expert is -infinity.
        const float size = marks[kVxMaxGroups + (lane < a.groups ? lane : 0u)], off = kVxOff * (2.0f + size);
        const bool known = size < INFINITY;
        const float low = known ? my - off : -INFINITY, high = in || lane >= a.groups ? -INFINITY : known ? my + off : INFINITY;
        const uint32_t out = vx_wave_max(vx_word_of(high));
        unsure = out > vx_word_of(-INFINITY) && __ballot(in && vx_word_of(low) <= out);
    }
    vx_wave_sync();
    return open;
}

// One wave per row; lane l holds experts l, l + 64, ... Without a bias the order is the logits'. With one, and for sums of two
// marks, choice values are first formed in fp32. Where two marks that decide are too near to each other for that, the groups are chosen
// again in 64 bits; where two choices are (about one row in 300 of 256 experts), the experts that may be among the chosen are
// ordered again in 64 bits, each by how many are above it (all experts again, one choice after the other, took 10 us, which a launch
// with one such row waited for: 4096 rows 18.7 -> 9.9 us). The largest is found top_k times: by DPP in the wave, its place
// by ballots. The chosen scores are formed in 64 bits. What bounds it: instructions, about 800 of the vector unit and 350 of the
// scalar one a row (16384 rows of 256 experts, 8 of them in 4 of 8 groups: 28 us, of which reading takes 4); one row 5.1 us.
template <class T, uint32_t ITEMS>
__global__ __launch_bounds__(256) void vx_route_kernel(VxRouteArgs a) {
    __shared__ double room[4][ITEMS * 64u + kVxMaxGroups];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), r = blockIdx.x * 4u + wave;
    if (r >= a.n_rows) return;  // (waves share nothing)
    // (all of a row's loads are requested at once: what is not there they give as 0)
    const T* row = (const T*)a.x.data + (size_t)r * a.x.rs;
    const auto xs = __builtin_amdgcn_make_buffer_rsrc((void*)row, 0, (int)(a.n_experts * sizeof(T)), 0x00020000);
    const auto bs = __builtin_amdgcn_make_buffer_rsrc((void*)a.bias, 0, a.bias ? (int)(a.n_experts * 4u) : 0, 0x00020000);
    const auto logit = [&](uint32_t e) -> float {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(xs, (int)(e * 4u), 0, 0));
        else return (float)__builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(xs, (int)(e * 2u), 0, 0));
    };
    float x[ITEMS], bias[ITEMS];
#pragma unroll
    for (uint32_t i = 0; i < ITEMS; ++i) x[i] = logit(lane + 64u * i);
#pragma unroll
    for (uint32_t i = 0; i < ITEMS; ++i) bias[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(bs, (int)((lane + 64u * i) * 4u), 0, 0));
#pragma unroll
    for (uint32_t i = 0; i < ITEMS; ++i) x[i] = lane + 64u * i < a.n_experts ? x[i] : -INFINITY;
    float top = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < ITEMS; ++i) {
        x[i] = x[i] > -INFINITY ? fminf(x[i], 3.40282347e38f) + 0.0f : -INFINITY;  // (NaN too)
        top = fmaxf(top, x[i]);
    }
    if (!a.sigmoid) top = vx_float_of(vx_wave_max(vx_word_of(top)));
    const auto out = [&](uint32_t i) { return !(x[i] > -INFINITY) || !(fabsf(bias[i]) < INFINITY); };
    const bool by_logits = !a.bias, marked = a.groups > 1u;

    float pick[ITEMS];
    bool unsure = false;
    if (!by_logits || a.two) {
        constexpr float kLog2e = 1.44269504f;
        float score[ITEMS], sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) {
            const float p = __builtin_amdgcn_exp2f((a.sigmoid ? -x[i] : x[i] - top) * kLog2e);
            score[i] = a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + p) : x[i] > -INFINITY ? p : 0.0f;
            sum += score[i];
        }
        if (!a.sigmoid) {
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
            sum = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < ITEMS; ++i) score[i] *= sum;
        }
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) pick[i] = out(i) ? -INFINITY : score[i] + bias[i];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) pick[i] = x[i];
    }
    uint64_t open = ~0ull;
    const auto shut = [&](uint32_t e) { return marked && !(open >> (e * a.by_size >> 20 & 63u) & 1u); };
    if (marked) {
        float* all = (float*)room[wave];
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) all[lane + 64u * i] = pick[i];
        vx_wave_sync();
        open = vx_open_groups<float>(a, all, all + ITEMS * 64u, unsure);
    }
    // 64-bit scores. The softmax's sum is formed where it is wanted, once.
    const auto exact = [&](float v) { return a.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : v > -INFINITY ? exp((double)v - (double)top) : 0.0; };
    double all_sum = 0.0;
    bool summed = a.sigmoid != 0;
    // (a rolled loop's numbers come from LDS: with an index that is not a constant the registers' arrays would go to memory)
    const auto spread = [&](double* all) {
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) all[lane + 64u * i] = __builtin_bit_cast(double, make_float2(x[i], bias[i]));
    };
    const auto sum_all = [&](double* all) {
        summed = true;
        spread(all);
#pragma unroll 1
        for (uint32_t i = 0; i < ITEMS; ++i) all_sum += exact(__builtin_bit_cast(float2, all[lane + 64u * i]).x);
#pragma unroll 1
        for (int off = 1; off < 64; off <<= 1) all_sum += __shfl_xor(all_sum, off);
    };
    const auto score = [&](float v) { return a.sigmoid ? exact(v) : all_sum > 0.0 ? exact(v) / all_sum : 0.0; };
    const auto choices = [&](double* all) {
        if (!summed) sum_all(all);
        spread(all);
#pragma unroll 1
        for (uint32_t i = 0; i < ITEMS; ++i) {
            const float2 v = __builtin_bit_cast(float2, all[lane + 64u * i]);
            all[lane + 64u * i] = v.x > -INFINITY && fabsf(v.y) < INFINITY ? score(v.x) + (double)v.y : -INFINITY;
        }
        vx_wave_sync();
    };
    if (unsure && (!by_logits || a.two)) {
        double* all = room[wave];
        bool never = false;
        choices(all);
        open = vx_open_groups<double>(a, all, all + ITEMS * 64u, never);
    }
    uint32_t id = kVxNoExpert;  // lane j: the j-th choice
    {
        uint32_t key[ITEMS];
        const uint32_t none = vx_word_of(-INFINITY);
        const auto value = [&](uint32_t i) {
            const uint32_t e = lane + 64u * i;
            return e >= a.n_experts || shut(e) ? -INFINITY : by_logits ? x[i] : pick[i] + 0.0f;
        };
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) key[i] = vx_word_of(value(i));
        constexpr bool kSorted = ITEMS <= 4;  // each lane's experts from the largest down, equal ones by index: its first is looked at
        uint32_t place[ITEMS];
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) place[i] = lane + 64u * i;
        if constexpr (kSorted) {
#pragma unroll
            for (uint32_t end = ITEMS - 1u; end > 0u; --end)
#pragma unroll
                for (uint32_t i = 0; i < end; ++i) {
                    const bool turn = key[i + 1] > key[i];
                    const uint32_t k0 = key[i], p0 = place[i];
                    key[i] = turn ? key[i + 1] : k0;
                    key[i + 1] = turn ? k0 : key[i + 1];
                    place[i] = turn ? place[i + 1] : p0;
                    place[i + 1] = turn ? p0 : place[i + 1];
                }
        }
        uint32_t found = 0, mine = 0, next = 0;  // lane j: the key of the j-th choice; the one behind the last
        for (;; ++found) {
            uint32_t best = key[0];
            if constexpr (!kSorted) {
#pragma unroll
                for (uint32_t i = 1; i < ITEMS; ++i) best = best > key[i] ? best : key[i];
            }
            best = vx_wave_max(best);
            if (best <= none) break;
            if (found == a.top) {
                next = best;
                break;
            }
            uint32_t e;
            if constexpr (kSorted) {
                uint64_t lanes = __ballot(key[0] == best);
                if (ITEMS > 1 && (lanes & (lanes - 1u))) {  // the lowest index that has it
                    for (uint32_t end = 64u;; end += 64u) {
                        const uint64_t m = __ballot(key[0] == best && place[0] < end);
                        if (!m) continue;
                        lanes = m;
                        break;
                    }
                }
                const uint32_t l = (uint32_t)__builtin_ctzll(lanes);
                e = (uint32_t)__builtin_amdgcn_readlane((int)place[0], (int)l);
                const bool taken = lane == l;
#pragma unroll
                for (uint32_t i = 0; i < ITEMS; ++i) {
                    key[i] = taken ? (i + 1 < ITEMS ? key[i + 1 < ITEMS ? i + 1 : i] : 0u) : key[i];
                    if (i + 1 < ITEMS) place[i] = taken ? place[i + 1 < ITEMS ? i + 1 : i] : place[i];
                }
            } else {
                uint32_t at = 0;  // the lowest index that has it
                uint64_t lanes = 0;
#pragma unroll
                for (uint32_t i = 0; i < ITEMS; ++i) {
                    const uint64_t m = __ballot(key[i] == best);
                    at = lanes ? at : i;
                    lanes = lanes ? lanes : m;
                }
                const uint32_t l = (uint32_t)__builtin_ctzll(lanes);
#pragma unroll
                for (uint32_t i = 0; i < ITEMS; ++i) key[i] = i == at && lane == l ? 0u : key[i];
                e = l + 64u * at;
            }
            id = lane == found ? e : id;
            mine = lane == found ? best : mine;
            if (by_logits && found + 1u == a.top) break;
        }
        if (!by_logits) {  // neighbours in the order, and the last that is in and the first that is out, have to be apart
            const float v = vx_float_of(mine), up = __shfl_up(v, 1), last = __shfl(v, (int)(a.top - 1u)), first_out = vx_float_of(next);
            const bool near = (lane && lane < found && !vx_above(up, fabsf(up), v, fabsf(v))) || (next && !vx_above(last, fabsf(last), first_out, fabsf(first_out)));
            if (__ballot(near)) {
                // Again, in 64 bits: of the experts that are not certainly below the last choice, as a list by index, each lane's
                // goes behind as many as are above it.
                const auto candidate = [&](uint32_t i) {
                    const float c = value(i);
                    return c > -INFINITY && (found < a.top || !vx_above(last, fabsf(last), c, fabsf(c)));
                };
                uint32_t n = 0;
#pragma unroll
                for (uint32_t i = 0; i < ITEMS; ++i) n += (uint32_t)__popcll(__ballot(candidate(i)));
                if (!summed) sum_all(room[wave]);
                id = kVxNoExpert;
                if (n <= 64u) {
                    uint4* list = (uint4*)room[wave];  // {index, logit, bias}
                    uint32_t front = 0;
#pragma unroll
                    for (uint32_t i = 0; i < ITEMS; ++i) {
                        const bool in = candidate(i);
                        const uint64_t m = __ballot(in);
                        if (in) list[front + (uint32_t)__popcll(m & ((1ull << lane) - 1ull))] =
                            make_uint4(lane + 64u * i, __builtin_bit_cast(uint32_t, x[i]), __builtin_bit_cast(uint32_t, bias[i]), 0u);
                        front += (uint32_t)__popcll(m);
                    }
                    vx_wave_sync();
                    const uint4 c = list[lane < n ? lane : 0u];
                    const double d = score(__builtin_bit_cast(float, c.y)) + (double)__builtin_bit_cast(float, c.z);
                    vx_wave_sync();
                    double* values = room[wave];
                    uint32_t* order = (uint32_t*)(values + 64);
                    values[lane] = d;
                    vx_wave_sync();
                    uint32_t above = 0;
                    for (uint32_t j = 0; j < n; ++j) {
                        const double o = values[j];
                        above += o > d || (o == d && j < lane);
                    }
                    if (lane < n) order[above] = c.x;
                    vx_wave_sync();
                    if (lane < a.top && lane < n) id = order[lane];
                } else {
                    double* all = room[wave];
                    choices(all);
                    for (uint32_t j = 0; j < a.top; ++j) {
                        double most = -INFINITY;
                        uint32_t at = 0xFFFFFFFFu;
                        for (uint32_t e = lane; e < a.n_experts; e += 64u) {
                            const double o = shut(e) ? -INFINITY : all[e];
                            if (o > most) {
                                most = o;
                                at = e;
                            }
                        }
#pragma unroll
                        for (int off = 1; off < 64; off <<= 1) {
                            const double ob = __shfl_xor(most, off);
                            const uint32_t oa = __shfl_xor(at, off);
                            if (ob > most || (ob == most && oa < at)) {
                                most = ob;
                                at = oa;
                            }
                        }
                        if (at == 0xFFFFFFFFu) break;
                        if ((at & 63u) == lane) all[at] = -INFINITY;
                        if (lane == j) id = at;
                    }
                }
            }
        }
    }
    const bool whole = !a.sigmoid && !a.renorm;
    if (whole && !summed) {
#pragma unroll
        for (uint32_t i = 0; i < ITEMS; ++i) all_sum += exact(x[i]);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) all_sum += __shfl_xor(all_sum, off);
    }
    double s = 0.0;
    if (id != kVxNoExpert) {
        s = exact(fminf(logit(id), 3.40282347e38f));
        if (whole) s = all_sum > 0.0 ? s / all_sum : 0.0;
    }
    if (a.renorm) {
        double sum = s;
        for (uint32_t off = 1; off < a.top; off <<= 1) sum += __shfl_xor(sum, (int)off);  // (behind lane top - 1 all are 0)
        s = sum > 0.0 ? s / sum : 0.0;
    }
    if (lane >= a.top) return;
    a.ids[(size_t)r * a.top + lane] = id;
    a.weights[(size_t)r * a.top + lane] = (float)(s * (double)a.scale);
}

// ---- grouping: a stable counting sort of the slots by expert ----
// A workgroup takes kGroupSlots slots, a wave kGroupRun neighbours of them. Slots of one expert within a wave find each other by
// ballots of their keys' bits, so that ranks follow the slots' order; waves' and workgroups' counts are summed in order.
// Several workgroups count first (their counts through memory), then place; one does both at once. Bound by latency: one workgroup
// 3.1 us, 131072 slots of 256 experts 4.6 and 9.5 us (each workgroup sums the counts of those in front of it).
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
#pragma unroll
    for (uint32_t w = 0; w < kGroupWaves; ++w) {
        if (w < wave) before += room[w];
        total += room[w];
    }
    return before + s - v;
}
// Experts by size, in steps of 32 slots: their blocks of a grouped product are listed from the largest class down, so that the
// last workgroups of a launch are short ones (the order within a class is any: blocks do not depend on each other).
__device__ __forceinline__ uint32_t vx_size_class(uint32_t slots) {
    const uint32_t c = (slots + 31u) / 32u;
    return c < 63u ? c : 63u;
}
// PER: experts of a thread, neighbours. Workgroup `block` of `blocks`.
template <uint32_t PER>
__device__ __forceinline__ void vx_group_place(const VxGroupArgs& a, uint32_t block, uint32_t blocks) {
    __shared__ uint32_t tally[kGroupWaves * (kVxI8MaxCount + 1u)];
    __shared__ uint32_t room[kGroupWaves], sizes[64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, n = a.count + 1u;
    const uint32_t run = block * kGroupSlots + wave * kGroupRun;
    const VxKeys k = vx_keys(a, run);
    if (threadIdx.x < 64u) sizes[threadIdx.x] = 0;
    uint32_t mine[PER], front[PER];
    // 32 workgroups' counts on the way at a time (behind the last they are 0)
    const auto hist = __builtin_amdgcn_make_buffer_rsrc((void*)a.hist, 0, blocks > 1u ? (int)(blocks * a.count * 4u) : 0, 0x00020000);
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        mine[j] = front[j] = 0;
        if (blocks > 1u && e < a.count) {
            for (uint32_t b0 = 0; b0 < blocks; b0 += 32u) {
                uint32_t c[32];
#pragma unroll
                for (uint32_t b = 0; b < 32u; ++b) c[b] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(hist, (int)(((b0 + b) * a.count + e) * 4u), 0, 0);
#pragma unroll
                for (uint32_t b = 0; b < 32u; ++b) {
                    front[j] += b0 + b < block ? c[b] : 0u;
                    mine[j] += c[b];
                }
            }
        }
    }
    vx_tally(a, k, tally);
    uint32_t sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        if (blocks == 1u && e < a.count) {
#pragma unroll
            for (uint32_t w = 0; w < kGroupWaves; ++w) mine[j] += tally[w * n + e];
        }
        sum += mine[j];
    }
    uint32_t total, at = vx_scan(sum, room, total);
    const bool items = a.items && block == 0;
    uint32_t rank[PER];
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j, c = (mine[j] + a.item_rows - 1u) / a.item_rows;
        rank[j] = items && e < a.count && c ? atomicAdd(&sizes[vx_size_class(mine[j])], c) : 0u;
    }
    if (items) {  // (the workgroup)
        __syncthreads();
        if (wave == 0) {  // lane l: the items of larger classes than l's
            const uint32_t c = sizes[63u - lane];
            uint32_t s = c;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = __shfl_up(s, off);
                if (lane >= (uint32_t)off) s += o;
            }
            sizes[63u - lane] = s - c;
            if (lane == 63u) *a.n_items = s;
        }
        __syncthreads();
    }
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = threadIdx.x * PER + j;
        if (e < a.count) {
            if (block == 0) a.offsets[e] = at;
            if (items && mine[j]) {
                uint2* to = a.items + sizes[vx_size_class(mine[j])] + rank[j];
                for (uint32_t p = 0; p < mine[j]; p += a.item_rows) *to++ = make_uint2(e, at + p);
            }
            uint32_t place = at + front[j];  // each wave's first place of the expert
#pragma unroll
            for (uint32_t w = 0; w < kGroupWaves; ++w) {
                const uint32_t c = tally[w * n + e];
                tally[w * n + e] = place;
                place += c;
            }
        }
        at += mine[j];
    }
    if (block == 0 && threadIdx.x == 0) a.offsets[a.count] = total;
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
    for (uint32_t p = total + block * kGroupThreads + threadIdx.x; p < a.n_slots; p += blocks * kGroupThreads) a.order[p] = kVxNoExpert;
}

template <uint32_t PER>
__global__ __launch_bounds__(kGroupThreads) void vx_group_place_kernel(VxGroupArgs a) {
    vx_group_place<PER>(a, blockIdx.x, gridDim.x);
}
// Few slots and their rows, which do not need each other, in one launch: workgroup 0 groups, r + 1 puts row r into 8 bits.
template <class T, int NV, uint32_t PER>
__global__ __launch_bounds__(kGroupThreads) void vx_prepare_kernel(VxGroupArgs a, VxI8View x, uint32_t k, VxI8Rows o) {
    __shared__ uint32_t red[kGroupWaves];
    if (blockIdx.x == 0) {
        vx_group_place<PER>(a, 0, 1);
        return;
    }
    const uint32_t r = blockIdx.x - 1u;
    const float s = vx_hold_row<T, kGroupThreads, NV, false>((const T*)x.data + (size_t)r * x.rs, k, (uint8_t*)o.codes + (size_t)r * o.rs, threadIdx.x, red);
    if (threadIdx.x == 0) o.scales[r] = s;
}

// ---- the sum of a row's experts ----
// A workgroup takes 1024 outputs of a row, a thread four. Lane j of a wave looks at the row's slot j; the slots of our
// experts are then added in order, four of their answers on the way at a time. Bound by the answers' bytes (8656 of 7168 fp32 for 4096
// rows, 248 MB and the residual and sum: 61 us).
constexpr uint32_t kCombineCols = 1024u;
template <bool VEC>
__global__ __launch_bounds__(256) void vx_combine_kernel(VxCombineArgs a) {
    const uint32_t r = blockIdx.x, c = blockIdx.y * kCombineCols + 4u * threadIdx.x, lane = threadIdx.x & 63u;
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

template <class T>
static hipError_t vx_route_launch(const VxRouteArgs& a, hipStream_t st) {
    const dim3 grid((a.n_rows + 3u) / 4u);
    if (a.n_experts <= 64u) hipLaunchKernelGGL((vx_route_kernel<T, 1>), grid, dim3(256), 0, st, a);
    else if (a.n_experts <= 128u) hipLaunchKernelGGL((vx_route_kernel<T, 2>), grid, dim3(256), 0, st, a);
    else if (a.n_experts <= 256u) hipLaunchKernelGGL((vx_route_kernel<T, 4>), grid, dim3(256), 0, st, a);
    else if (a.n_experts <= 512u) hipLaunchKernelGGL((vx_route_kernel<T, 8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((vx_route_kernel<T, 16>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}
hipError_t vx_launch_route(const VxRouteArgs& args, hipStream_t st) {
    VxRouteArgs a = args;
    a.group_size = a.n_experts / a.groups;
    a.by_size = (1u << 20) / a.group_size + 1u;  // (too large by less than 1023 / 2^20 of a group, below 1 / group_size)
    a.group_lanes = 0;
    while ((2u << a.group_lanes) * a.groups <= 64u) ++a.group_lanes;
    if (a.x.dtype == VELOX_DT_F32) return vx_route_launch<float>(a, st);
    if (a.x.dtype == VELOX_DT_F16) return vx_route_launch<_Float16>(a, st);
    return vx_route_launch<__bf16>(a, st);
}

uint32_t vx_group_blocks(uint32_t n_slots) { return n_slots ? (n_slots + kGroupSlots - 1u) / kGroupSlots : 1u; }

namespace {
VxGroupArgs vx_keyed(VxGroupArgs a) {
    a.key_bits = 32u - (uint32_t)__builtin_clz(a.count);  // keys 0 .. count
    return a;
}
template <class T, int NV>
hipError_t vx_prepare(const VxGroupArgs& a, const VxI8View& x, uint32_t n_rows, uint32_t k, const VxI8Rows& o, hipStream_t st) {
    if (a.count <= kGroupThreads) hipLaunchKernelGGL((vx_prepare_kernel<T, NV, 1>), dim3(n_rows + 1u), dim3(kGroupThreads), 0, st, a, x, k, o);
    else hipLaunchKernelGGL((vx_prepare_kernel<T, NV, kVxI8MaxCount / kGroupThreads>), dim3(n_rows + 1u), dim3(kGroupThreads), 0, st, a, x, k, o);
    return hipGetLastError();
}
template <class T>
hipError_t vx_prepare_t(const VxGroupArgs& a, const VxI8View& x, uint32_t n_rows, uint32_t k, const VxI8Rows& o, hipStream_t st) {
    return vx_i8_pad(k) * sizeof(T) <= 2u * 16u * kGroupThreads ? vx_prepare<T, 2>(a, x, n_rows, k, o, st) : vx_prepare<T, 8>(a, x, n_rows, k, o, st);
}
}  // namespace

hipError_t vx_launch_group_and_quantize(const VxGroupArgs& args, const VxI8View& x, uint32_t n_rows, uint32_t k, const VxI8Rows& o, hipStream_t st) {
    if (vx_group_blocks(args.n_slots) > 1u || !vx_whole_rows(x, k) || vx_i8_pad(k) * (x.dtype == VELOX_DT_F32 ? 4u : 2u) > 8u * 16u * kGroupThreads) {
        const hipError_t e = vx_launch_group(args, st);
        return e != hipSuccess ? e : vx_launch_i8_quantize(x, n_rows, k, o, nullptr, st);
    }
    const VxGroupArgs a = vx_keyed(args);
    if (x.dtype == VELOX_DT_F32) return vx_prepare_t<float>(a, x, n_rows, k, o, st);
    if (x.dtype == VELOX_DT_F16) return vx_prepare_t<_Float16>(a, x, n_rows, k, o, st);
    return vx_prepare_t<__bf16>(a, x, n_rows, k, o, st);
}

hipError_t vx_launch_group(const VxGroupArgs& args, hipStream_t st) {
    const VxGroupArgs a = vx_keyed(args);
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
    if (a.vec) hipLaunchKernelGGL((vx_combine_kernel<true>), dim3(a.n_rows, blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((vx_combine_kernel<false>), dim3(a.n_rows, blocks), dim3(256), 0, st, a);
    return hipGetLastError();
}
