// vx_int8_host.cpp -- C entry points of the 8-bit integer products and the experts: argument checks, workspaces, launches.
#include <cmath>
#include <cstring>

#include "vx_int8.h"

namespace {

bool aligned(const void* p, uint64_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
uint64_t up(uint64_t v) { return (v + 255u) & ~255ull; }

// Shapes of a matrix; its pointers are the entry points' to check.
bool shape_ok(const VeloxHipInt8Matrix* m) {
    return m && m->n && m->n <= (1u << 20) && m->k && m->k <= VELOX_HIP_INT8_MAX_K && m->count && m->count <= kVxI8MaxCount &&
           m->paired <= 1u && !(m->paired && m->n % 2u);
}
bool matrix_ok(const VeloxHipInt8Matrix* m) {
    return shape_ok(m) && m->codes && m->scales && aligned(m->codes, 16) && aligned(m->scales, 16);
}
VxI8Mat view(const VeloxHipInt8Matrix* m) {
    VxI8Mat w;
    w.codes = (const uint4*)m->codes;
    w.scales = m->scales;
    w.n = m->n;
    w.k = m->k;
    w.n_tiles = vx_i8_tiles(m->n, m->paired);
    w.k_tiles = vx_i8_pad(m->k) / 64u;
    w.paired = m->paired;
    w.count = m->count;
    return w;
}

uint32_t elt(uint32_t dtype) { return dtype == VELOX_DT_F32 ? 4u : 2u; }
bool rows_ok(const VeloxHipRows* r) {
    return r && r->data && r->dtype <= VELOX_DT_BF16 && r->heads == 1 && aligned(r->data, elt(r->dtype));
}
// Rows that are written: each has a place of its own.
bool out_ok(const VeloxHipRows* r, uint32_t n_rows, uint32_t cols) { return rows_ok(r) && (n_rows <= 1u || r->row_stride >= cols); }
VxI8View view(const VeloxHipRows* r) { return VxI8View{r->data, r->row_stride, r->dtype}; }
bool q_ok(const VeloxHipInt8Rows* q, uint32_t k) {
    return q && q->codes && q->scales && aligned(q->codes, 16) && aligned(q->scales, 4) && q->row_stride % 128u == 0 &&
           q->row_stride >= vx_i8_pad(k);
}
// b is memory of its own, or a's rows as they lie.
bool same_or_apart(const VeloxHipRows* a, const VeloxHipRows* b, uint32_t n_rows) {
    return a->data != b->data || (elt(a->dtype) == elt(b->dtype) && (n_rows <= 1u || a->row_stride == b->row_stride));
}

// Whether [at, at + bytes) and n_rows rows of `len` bytes, `stride` bytes apart, have a byte in common.
bool meet(const void* at, uint64_t bytes, const void* rows, uint64_t n_rows, uint64_t len, uint64_t stride) {
    const uint64_t lo = (uint64_t)(uintptr_t)at, base = (uint64_t)(uintptr_t)rows;
    if (!bytes || !n_rows || !len || base >= lo + bytes) return false;
    if (base + len > lo) return true;
    if (!stride) return false;
    const uint64_t r = (lo - base - len) / stride + 1u;  // the first row that ends behind lo
    return r < n_rows && base + r * stride < lo + bytes;
}
bool meet(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) { return meet(a, a_bytes, b, 1, b_bytes, 0); }

// Every row begins at a whole multiple of four elements.
bool whole(const VeloxHipRows* r) { return aligned(r->data, 4u * elt(r->dtype)) && r->row_stride % 4u == 0; }

// A workspace's regions, each from a multiple of 256 bytes on.
struct Space {
    uint8_t* base;
    uint64_t used = 0;
    explicit Space(void* p) : base((uint8_t*)p) {}
    template <class T>
    T* take(uint64_t n) {
        T* p = (T*)(base + used);
        used += up(n * sizeof(T));
        return p;
    }
};

uint64_t group_words(uint32_t n_slots, uint32_t count) {
    const uint32_t b = vx_group_blocks(n_slots);
    return b > 1u ? (uint64_t)b * count : 0u;
}

bool route_ok(const VeloxHipRouteConfig* c) {
    if (!c || !c->n_experts || c->n_experts > kVxI8MaxCount || !c->top_k || c->top_k > kVxMaxTop) return false;
    if (c->scores > VELOX_ROUTE_SIGMOID || c->group_by > VELOX_GROUP_TWO || c->renormalize > 1u || !std::isfinite(c->scale)) return false;
    if (!c->groups || c->groups > kVxMaxGroups || c->n_experts % c->groups || !c->top_groups || c->top_groups > c->groups) return false;
    return c->top_k <= c->n_experts / c->groups * c->top_groups;
}

struct FfnSpace {
    VxI8Rows x, h;
    uint32_t *order, *offsets, *hist, *n_items;
    uint2* items;
    float *hidden, *part;
    uint64_t hidden_stride, part_stride, bytes;
};
uint32_t max_items(uint32_t slots, uint32_t count, uint32_t rows) {
    const uint32_t most = slots / rows + count;
    return slots < most ? slots : most;
}
FfnSpace ffn_space(const VxI8Mat& gu, const VxI8Mat& down, uint32_t n_rows, uint32_t top, void* memory) {
    Space s(memory);
    FfnSpace f;
    const uint32_t slots = n_rows * top;
    f.x.rs = vx_i8_pad(gu.k);
    f.h.rs = f.hidden_stride = vx_i8_pad(down.k);
    f.part_stride = (down.n + 3u) & ~3u;
    f.x.codes = s.take<int8_t>(n_rows * f.x.rs);
    f.x.scales = s.take<float>(n_rows);
    f.order = s.take<uint32_t>(slots);
    f.offsets = s.take<uint32_t>(gu.count + 1u);
    f.hist = s.take<uint32_t>(group_words(slots, gu.count));
    f.n_items = s.take<uint32_t>(1);
    f.items = s.take<uint2>(max_items(slots, gu.count, 16u));
    f.hidden = s.take<float>(slots * f.hidden_stride);
    f.h.codes = s.take<int8_t>(slots * f.h.rs);
    f.h.scales = s.take<float>(slots);
    f.part = s.take<float>(slots * f.part_stride);
    f.bytes = s.used;
    return f;
}
bool ffn_ok(const VeloxHipInt8Matrix* gu, const VeloxHipInt8Matrix* down, uint32_t n_rows, uint32_t top) {
    return shape_ok(gu) && shape_ok(down) && gu->paired && !down->paired && gu->count == down->count && gu->n / 2u == down->k &&
           gu->k == down->n && top && top <= kVxMaxTop && (uint64_t)n_rows * top <= kVxMaxSlots;
}

}  // namespace

extern "C" {

int velox_hip_int8_layout(const VeloxHipInt8Matrix* m, uint64_t* code_bytes, uint64_t* scale_bytes) {
    if (!shape_ok(m)) return VELOX_HIP_EINVAL;
    const VxI8Mat w = view(m);
    if (code_bytes) *code_bytes = (uint64_t)w.count * w.n_tiles * w.k_tiles * 1024u;
    if (scale_bytes) *scale_bytes = (uint64_t)w.count * w.n_tiles * 64u;
    return VELOX_HIP_OK;
}

int velox_hip_int8_pack(const VeloxHipInt8Matrix* m, uint32_t first, uint32_t number, const int8_t* d_codes, uint64_t matrix_stride,
                        uint64_t row_stride, const float* d_scales, uint64_t scale_stride, hipStream_t st) {
    if (!matrix_ok(m) || first > m->count || number > m->count - first) return VELOX_HIP_EINVAL;
    if (!number) return VELOX_HIP_OK;
    if (!d_codes || !d_scales || !aligned(d_scales, 4)) return VELOX_HIP_EINVAL;
    return (int)vx_launch_i8_pack(view(m), first, number, d_codes, matrix_stride, row_stride, d_scales, scale_stride, st);
}

int velox_hip_int8_quantize(const VeloxHipRows* x, uint32_t n_rows, uint32_t k, const VeloxHipInt8Rows* out, hipStream_t st) {
    if (!k || k > VELOX_HIP_INT8_MAX_K || n_rows > kVxI8MaxRows || !rows_ok(x) || !q_ok(out, k)) return VELOX_HIP_EINVAL;
    if (!n_rows) return VELOX_HIP_OK;
    return (int)vx_launch_i8_quantize(view(x), n_rows, k, VxI8Rows{out->codes, out->scales, out->row_stride}, nullptr, st);
}

int velox_hip_int8_product_bytes(const VeloxHipInt8Matrix* m, uint32_t n_rows, uint64_t* bytes) {
    if (!shape_ok(m) || m->count != 1 || n_rows > kVxI8MaxRows || !bytes) return VELOX_HIP_EINVAL;
    *bytes = up((uint64_t)n_rows * vx_i8_pad(m->k)) + up(4ull * n_rows);
    return VELOX_HIP_OK;
}

int velox_hip_int8_product(const VeloxHipInt8Matrix* m, const VeloxHipRows* x, const VeloxHipInt8Rows* q, uint32_t n_rows,
                           const float* d_bias, const VeloxHipRows* residual, const VeloxHipRows* out, int mode, void* workspace,
                           uint64_t workspace_bytes, hipStream_t st) {
    if (!matrix_ok(m) || m->count != 1 || n_rows > kVxI8MaxRows || !x == !q || !out_ok(out, n_rows, m->paired ? m->n / 2u : m->n))
        return VELOX_HIP_EINVAL;
    if (mode < VELOX_GEMV_STORE || mode > VELOX_GEMV_SWIGLU || (mode == VELOX_GEMV_SWIGLU) != (m->paired != 0)) return VELOX_HIP_EINVAL;
    if ((mode == VELOX_GEMV_RESIDUAL) != (residual != nullptr) || (d_bias && mode == VELOX_GEMV_SWIGLU) || !aligned(d_bias, 4))
        return VELOX_HIP_EINVAL;
    if (residual && (!rows_ok(residual) || !same_or_apart(residual, out, n_rows))) return VELOX_HIP_EINVAL;
    if (x ? !rows_ok(x) : !q_ok(q, m->k)) return VELOX_HIP_EINVAL;
    if (!n_rows) return VELOX_HIP_OK;
    VxI8Args a;
    std::memset(&a, 0, sizeof(a));
    a.w = view(m);
    a.n_rows = n_rows;
    a.bias = d_bias;
    if (residual) a.res = view(residual);
    a.out = view(out);
    a.vec = whole(out) && (!residual || whole(residual));
    const int epi = m->paired ? VX_I8_SWIGLU : VX_I8_STORE;
    if (!x) {
        a.a = VxI8Rows{q->codes, q->scales, q->row_stride};
        return (int)vx_launch_i8_product(a, epi, st);
    }
    Space s(workspace);
    a.a.rs = vx_i8_pad(m->k);
    a.a.codes = s.take<int8_t>(n_rows * a.a.rs);
    a.a.scales = s.take<float>(n_rows);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < s.used) return VELOX_HIP_EINVAL;
    if (x->data != out->data && vx_i8_by_row(view(x), n_rows, m->k)) return  // (every workgroup reads x)
            (int)vx_launch_i8_row(a, view(x), epi, st);
    const hipError_t e = vx_launch_i8_quantize(view(x), n_rows, m->k, a.a, nullptr, st);
    return e != hipSuccess ? (int)e : (int)vx_launch_i8_product(a, epi, st);
}

int velox_hip_expert_route(const VeloxHipRouteConfig* cfg, const VeloxHipRows* logits, const float* d_bias, uint32_t n_rows,
                           uint32_t* d_ids, float* d_weights, hipStream_t st) {
    if (!route_ok(cfg) || !rows_ok(logits) || n_rows > kVxI8MaxRows || !aligned(d_bias, 4)) return VELOX_HIP_EINVAL;
    if (!n_rows) return VELOX_HIP_OK;
    if (!d_ids || !d_weights || !aligned(d_ids, 4) || !aligned(d_weights, 4)) return VELOX_HIP_EINVAL;
    const uint64_t words = 4ull * n_rows * cfg->top_k, e = elt(logits->dtype);  // (waves read while others write)
    if (meet(d_ids, words, d_weights, words)) return VELOX_HIP_EINVAL;
    for (const void* to : {(const void*)d_ids, (const void*)d_weights})
        if (meet(to, words, logits->data, n_rows, e * cfg->n_experts, e * logits->row_stride) ||
            (d_bias && meet(to, words, d_bias, 4ull * cfg->n_experts)))
            return VELOX_HIP_EINVAL;
    VxRouteArgs a;
    std::memset(&a, 0, sizeof(a));
    a.x = view(logits);
    a.bias = d_bias;
    a.n_rows = n_rows;
    a.n_experts = cfg->n_experts;
    a.top = cfg->top_k;
    a.sigmoid = cfg->scores == VELOX_ROUTE_SIGMOID;
    a.groups = cfg->groups;
    a.top_groups = cfg->top_groups;
    a.two = cfg->group_by == VELOX_GROUP_TWO && cfg->groups > 1u;
    a.renorm = cfg->renormalize;
    a.scale = cfg->scale;
    a.ids = d_ids;
    a.weights = d_weights;
    return (int)vx_launch_route(a, st);
}

int velox_hip_expert_group_bytes(uint32_t n_slots, uint32_t count, uint64_t* bytes) {
    if (n_slots > kVxMaxSlots || !count || count > kVxI8MaxCount || !bytes) return VELOX_HIP_EINVAL;
    *bytes = 4ull * group_words(n_slots, count);
    return VELOX_HIP_OK;
}

int velox_hip_expert_group(const uint32_t* d_ids, uint32_t n_slots, uint32_t first, uint32_t count, uint32_t* d_order,
                           uint32_t* d_offsets, void* workspace, uint64_t workspace_bytes, hipStream_t st) {
    if (n_slots > kVxMaxSlots || !count || count > kVxI8MaxCount || (uint64_t)first + count > kVxNoExpert) return VELOX_HIP_EINVAL;
    if (!d_offsets || !aligned(d_offsets, 4) || (n_slots && (!d_ids || !d_order)) || !aligned(d_ids, 4) || !aligned(d_order, 4))
        return VELOX_HIP_EINVAL;
    const uint64_t need = 4ull * group_words(n_slots, count);
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) return VELOX_HIP_EINVAL;
    const void* const at[4] = {d_ids, d_order, d_offsets, workspace};  // (workgroups read while others write)
    const uint64_t bytes[4] = {4ull * n_slots, 4ull * n_slots, 4ull * (count + 1u), need};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j)
            if (meet(at[i], bytes[i], at[j], bytes[j])) return VELOX_HIP_EINVAL;
    VxGroupArgs a;
    std::memset(&a, 0, sizeof(a));
    a.ids = d_ids;
    a.n_slots = n_slots;
    a.first = first;
    a.count = count;
    a.order = d_order;
    a.offsets = d_offsets;
    a.hist = (uint32_t*)workspace;
    a.item_rows = 16u;
    return (int)vx_launch_group(a, st);
}

int velox_hip_expert_ffn_bytes(const VeloxHipInt8Matrix* gate_up, const VeloxHipInt8Matrix* down, uint32_t n_rows, uint32_t top_k,
                               uint64_t* bytes) {
    if (!ffn_ok(gate_up, down, n_rows, top_k) || !bytes) return VELOX_HIP_EINVAL;
    *bytes = ffn_space(view(gate_up), view(down), n_rows, top_k, nullptr).bytes;
    return VELOX_HIP_OK;
}

int velox_hip_expert_ffn(const VeloxHipInt8Matrix* gate_up, const VeloxHipInt8Matrix* down, uint32_t first, const VeloxHipRows* x,
                         const uint32_t* d_ids, const float* d_weights, uint32_t n_rows, uint32_t top_k, const VeloxHipRows* residual,
                         const VeloxHipRows* out, void* workspace, uint64_t workspace_bytes, hipStream_t st) {
    if (!ffn_ok(gate_up, down, n_rows, top_k) || !matrix_ok(gate_up) || !matrix_ok(down) || !rows_ok(x) ||
        !out_ok(out, n_rows, down->n))
        return VELOX_HIP_EINVAL;
    if ((uint64_t)first + gate_up->count > kVxNoExpert || !same_or_apart(x, out, n_rows)) return VELOX_HIP_EINVAL;
    if (residual && (!rows_ok(residual) || !same_or_apart(residual, out, n_rows))) return VELOX_HIP_EINVAL;
    if (!n_rows) return VELOX_HIP_OK;
    if (!d_ids || !d_weights || !aligned(d_ids, 4) || !aligned(d_weights, 4)) return VELOX_HIP_EINVAL;
    const VxI8Mat gu = view(gate_up), dn = view(down);
    const FfnSpace f = ffn_space(gu, dn, n_rows, top_k, workspace);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < f.bytes) return VELOX_HIP_EINVAL;
    const uint32_t slots = n_rows * top_k;
    VxI8Args a;
    std::memset(&a, 0, sizeof(a));
    a.w = gu;
    a.n_rows = n_rows;
    a.top = top_k;
    a.part = f.hidden;
    a.part_stride = f.hidden_stride;
    VxCombineArgs c;
    std::memset(&c, 0, sizeof(c));
    c.ids = d_ids;
    c.weights = d_weights;
    c.n_rows = n_rows;
    c.top = top_k;
    c.first = first;
    c.count = gu.count;
    c.n = dn.n;
    c.part = f.part;
    c.part_stride = f.part_stride;
    if (residual) c.res = view(residual);
    c.out = view(out);
    c.vec = whole(out) && (!residual || whole(residual));
    if (vx_i8_ffn_by_slot(view(x), n_rows, top_k, gu.count, gu.k, dn.k)) {
        a.ids = d_ids;
        a.first = first;
        hipError_t e = vx_launch_i8_slots(a, view(x), st);
        a.w = dn;
        if (e == hipSuccess) e = vx_launch_i8_answers(a, c, st);
        return (int)e;
    }
    VxGroupArgs g;
    g.ids = d_ids;
    g.n_slots = slots;
    g.first = first;
    g.count = gu.count;
    g.order = f.order;
    g.offsets = f.offsets;
    g.hist = f.hist;
    g.items = f.items;
    g.n_items = f.n_items;
    g.item_rows = vx_i8_item_rows(slots, gu.count, gu.n_tiles > dn.n_tiles ? gu.n_tiles : dn.n_tiles);
    hipError_t e = vx_launch_group_and_quantize(g, view(x), n_rows, gu.k, f.x, st);
    a.a = f.x;
    a.g = VxGrouped{f.order, f.offsets, f.items, f.n_items};
    a.max_items = max_items(slots, gu.count, g.item_rows);
    a.item_rows = g.item_rows;
    if (e == hipSuccess) e = vx_launch_i8_product(a, VX_I8_HIDDEN, st);
    if (e == hipSuccess)
        e = vx_launch_i8_quantize(VxI8View{f.hidden, f.hidden_stride, VELOX_DT_F32}, slots, (dn.k + 3u) & ~3u, f.h, f.offsets + gu.count, st);
    a.w = dn;
    a.a = f.h;
    a.part = f.part;
    a.part_stride = f.part_stride;
    if (e == hipSuccess) e = vx_launch_i8_product(a, VX_I8_SLOT, st);
    if (e == hipSuccess) e = vx_launch_combine(c, st);
    return (int)e;
}

}  // extern "C"
