// vx_paged.h -- the paged KV cache's device views and launchers (vx_paged.hip, vx_paged_attn.hip), used by
// vx_paged_host.cpp, which has checked every argument.
#pragma once

#include "vx_common.h"

constexpr uint32_t kVxNoPage = VELOX_HIP_NO_PAGE;
constexpr uint32_t kVxMaxRopePairs = 128;   // rot_dim <= 256
constexpr uint32_t kVxMaxRows = (1u << 24) - 1u;  // a launch has fewer than 2^32 threads, 256 of them for a row at most
constexpr uint32_t kVxPromptRows = 128;     // (row, head) pairs of a workgroup of the prompt attention
constexpr uint32_t kVxMaxPagedSeqs = 4096;  // the extend kernel keeps a few words per sequence in LDS

// One layer of a cache.
struct VxPagedView {
    uint8_t* pool;  // the layer's page 0
    const uint32_t* table;
    const uint32_t* lens;
    uint64_t page_bytes;
    uint32_t n_pages, page_size, n_seqs, max_pages, table_stride, hkv, d, dtype;
};

struct VxRowsView {
    void* data;
    uint64_t rs, hs;  // elements
    uint32_t heads, dtype;
};

// Turns per position of every pair (f_j / 2 pi) and the amplitude, as kernel arguments: the handle then holds
// no device memory and serves every device.
struct VxRopeTable {
    double turns[kVxMaxRopePairs];
    float amp;
    uint32_t rot, interleaved;
};

struct VxAppendArgs {
    VxPagedView c;
    VxRowsView q, k, v, qo;  // q.data NULL: k and v only
    const uint32_t* q_start;  // NULL: row s is sequence s's
    uint32_t n_rows;
};

struct VxPagedAttnArgs {
    VxPagedView c;
    VxRowsView q, out;
    const uint32_t* q_start;  // prompt form; NULL: row s is the newest position of sequence s
    uint32_t n_rows;
    uint32_t window, sinks;
    float scale;
    uint32_t splits;
    uint64_t span;   // token form: positions of a row at most, as planned
    float* part_o;   // [row][head][split][d]
    float* part_ml;  // [row][head][split][2]: maximum (log2 domain), sum
};

struct VxPages {
    uint8_t* pool;
    uint64_t page_bytes, layer_stride;
    uint32_t *table, *lens, *refs, *scratch;
    uint32_t n_layers, n_pages, page_size, n_seqs, max_pages, table_stride;
};
// Scratch words: [0] sequences the last extend refused, [1] free pages (status), [2] page moves to copy,
// [3] live pages (compact); then the moves' sources and targets, then one word per page (extend: the free
// pages it takes, compact: where a page went).
constexpr uint32_t kVxPagesHead = 64;
VX_HD uint32_t vx_pages_moves(uint32_t n_seqs, uint32_t n_pages) { return n_seqs > n_pages ? n_seqs : n_pages; }

#ifdef __HIP_DEVICE_COMPILE__
// A word at a uniform address that no kernel in flight writes, by a scalar load: it waits for no vector load.
__device__ __forceinline__ uint32_t vx_word(const uint32_t* p) {
    return *(const __attribute__((address_space(4))) uint32_t*)(uintptr_t)p;
}
#else
__device__ uint32_t vx_word(const uint32_t* p);
#endif

hipError_t vx_launch_rope_rows(const VxRopeTable& t, const VxRowsView& x, const VxRowsView& out, uint32_t n_rows,
                               uint32_t d, const uint32_t* positions, hipStream_t st);
hipError_t vx_launch_rope_append(const VxRopeTable& t, const VxAppendArgs& a, hipStream_t st);
uint32_t vx_paged_attn_splits(const VxPagedView& c, uint32_t heads, uint32_t rows, uint32_t max_len);
hipError_t vx_launch_paged_attention(const VxPagedAttnArgs& a, hipStream_t st);
uint32_t vx_paged_prompt_split_rows(const VxPagedView& c, uint32_t max_rows);  // the most rows that are split
uint32_t vx_paged_prompt_splits(const VxPagedView& c, uint32_t heads, uint32_t n_rows, uint32_t max_rows, uint32_t span);
hipError_t vx_launch_paged_prompt(const VxPagedAttnArgs& a, hipStream_t st);

hipError_t vx_launch_pages_reset(const VxPages& p, hipStream_t st);
hipError_t vx_launch_pages_extend(const VxPages& p, const uint32_t* add, hipStream_t st);
hipError_t vx_launch_pages_fork(const VxPages& p, const uint32_t* src, hipStream_t st);
hipError_t vx_launch_pages_free(const VxPages& p, const uint32_t* seqs, uint32_t n, hipStream_t st);
hipError_t vx_launch_pages_trim(const VxPages& p, uint32_t window, uint32_t sinks, hipStream_t st);
hipError_t vx_launch_pages_compact(const VxPages& p, hipStream_t st);
hipError_t vx_launch_pages_count(const VxPages& p, hipStream_t st);
