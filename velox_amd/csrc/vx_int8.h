// vx_int8.h -- device views and launchers of the 8-bit integer products (vx_int8.hip) and the experts (vx_experts.hip), used
// by vx_int8_host.cpp, which has checked every argument.
#pragma once

#include "vx_common.h"

constexpr uint32_t kVxI8MaxCount = 1024;            // matrices of a descriptor, experts of a routing
constexpr uint32_t kVxI8MaxRows = (1u << 24) - 1u;
constexpr uint32_t kVxMaxSlots = 1u << 20;          // (row, expert) pairs of a call
constexpr uint32_t kVxMaxTop = 64, kVxMaxGroups = 64;
constexpr uint32_t kVxNoExpert = VELOX_HIP_NO_EXPERT;

// Laid-out matrices: `count` of n_tiles x k_tiles tiles of 16 rows x 64 columns, 1 KiB each.
struct VxI8Mat {
    const uint4* codes;
    const float* scales;       // [count][16 n_tiles]
    uint32_t n, k, n_tiles, k_tiles, paired, count;
};
VX_HD uint32_t vx_i8_tiles(uint32_t n, uint32_t paired) { return paired ? 2u * ((n / 2u + 15u) / 16u) : (n + 15u) / 16u; }
VX_HD uint32_t vx_i8_pad(uint32_t k) { return (k + 127u) & ~127u; }

struct VxI8View {              // plain rows by a stride in elements
    void* data;
    uint64_t rs;
    uint32_t dtype;
};
struct VxI8Rows {              // rows in 8 bits
    int8_t* codes;
    float* scales;
    uint64_t rs;               // bytes, a multiple of 128
};

// The rows of a product by expert. Position p of the grouped order is slot order[p]; the positions of expert e are
// offsets[e] .. offsets[e + 1]. items[i] = {expert, first position}: the blocks of up to item_rows positions, n_items of
// them at [0] of n_items.
struct VxGrouped {
    const uint32_t* order;
    const uint32_t* offsets;
    const uint2* items;
    const uint32_t* n_items;
};

enum { VX_I8_STORE = 0, VX_I8_SWIGLU = 1, VX_I8_HIDDEN = 2, VX_I8_SLOT = 3 };
struct VxI8Args {
    VxI8Mat w;
    VxI8Rows a;
    uint32_t n_rows;           // plain products
    VxGrouped g;               // HIDDEN, SLOT
    uint32_t top;              // HIDDEN: position p reads row order[p] / top of a
    uint32_t max_items, item_rows;
    const uint32_t* ids;       // slots one by one: slot s is expert ids[s] - first's, of row s / top
    uint32_t first;
    const float* bias;         // STORE
    VxI8View res, out;         // STORE (res.data NULL: none), SWIGLU
    uint32_t vec;              // 1: res and out rows begin at whole multiples of four elements
    float* part;               // HIDDEN: h of position p at part + p * part_stride; SLOT: the answer of slot s at s
    uint64_t part_stride;      // elements, a multiple of 4
};

struct VxRouteArgs {
    VxI8View x;
    const float* bias;
    uint32_t n_rows, n_experts, top, sigmoid, groups, top_groups, two, renorm;
    float scale;
    uint32_t* ids;
    float* weights;
    // set by the launcher: 2^group_lanes lanes for each group; experts of one; e < 1024 is of group e * by_size >> 20
    uint32_t group_lanes, group_size, by_size;
};

struct VxGroupArgs {
    const uint32_t* ids;
    uint32_t n_slots, first, count;
    uint32_t* order;
    uint32_t* offsets;
    uint32_t* hist;            // [blocks][count], vx_group_blocks(n_slots) of them where more than one
    uint2* items;              // NULL: none
    uint32_t* n_items;
    uint32_t item_rows;
    uint32_t key_bits;         // set by the launcher
};

struct VxCombineArgs {
    const uint32_t* ids;
    const float* weights;
    uint32_t n_rows, top, first, count, n;
    const float* part;         // [slot][part_stride]
    uint64_t part_stride;      // a multiple of 4
    VxI8View res, out;
    uint32_t vec;              // 1: res and out rows begin at whole multiples of four elements
};

hipError_t vx_launch_i8_pack(const VxI8Mat& m, uint32_t first, uint32_t number, const int8_t* codes, uint64_t ms, uint64_t rs,
                             const float* scales, uint64_t ss, hipStream_t st);
bool vx_whole_rows(const VxI8View& x, uint32_t k);
// rows < *limit where limit is set
hipError_t vx_launch_i8_quantize(const VxI8View& x, uint32_t n_rows, uint32_t k, const VxI8Rows& out, const uint32_t* limit,
                                 hipStream_t st);
hipError_t vx_launch_i8_product(const VxI8Args& a, int epi, hipStream_t st);
uint32_t vx_i8_item_rows(uint32_t slots, uint32_t count, uint32_t n_tiles);  // positions of a block of a grouped product
// Few rows, quantized by the workgroups that multiply them: whether x's rows are; plain products, the hidden values of
// every slot (a.part: [slot]), the experts' answers and their sum.
bool vx_i8_by_row(const VxI8View& x, uint32_t n_rows, uint32_t k);
hipError_t vx_launch_i8_row(const VxI8Args& a, const VxI8View& x, int epi, hipStream_t st);
bool vx_i8_ffn_by_slot(const VxI8View& x, uint32_t n_rows, uint32_t top, uint32_t count, uint32_t hidden, uint32_t inner);
hipError_t vx_launch_i8_slots(const VxI8Args& a, const VxI8View& x, hipStream_t st);
hipError_t vx_launch_i8_answers(const VxI8Args& a, const VxCombineArgs& c, hipStream_t st);
hipError_t vx_launch_route(const VxRouteArgs& a, hipStream_t st);
uint32_t vx_group_blocks(uint32_t n_slots);
hipError_t vx_launch_group(const VxGroupArgs& a, hipStream_t st);
// Both, in one launch where the slots are few (they do not need each other).
hipError_t vx_launch_group_and_quantize(const VxGroupArgs& a, const VxI8View& x, uint32_t n_rows, uint32_t k, const VxI8Rows& out, hipStream_t st);
hipError_t vx_launch_combine(const VxCombineArgs& a, hipStream_t st);
