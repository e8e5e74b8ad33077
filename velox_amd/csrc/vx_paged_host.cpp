// vx_paged_host.cpp -- C entry points of the paged KV cache: argument checks, the rotary frequencies, launches.
#include <cmath>
#include <cstring>
#include <new>

#include "vx_paged.h"

struct VeloxHipRope {
    VeloxHipRopeConfig cfg;
    double freq[kVxMaxRopePairs];
    double amplitude;
    VxRopeTable table;
};

namespace {

bool aligned(const void* p, uint64_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

uint64_t page_bytes(const VeloxHipPagedCache& c) {
    return 4ull * c.num_kv_heads * c.page_size * c.head_dim;  // K and V, 2 bytes each
}

// Shapes of a description; its pointers are the entry points' to check.
bool shape_ok(const VeloxHipPagedCache* c) {
    if (!c || c->reserved) return false;
    if (c->dtype != VELOX_DT_F16 && c->dtype != VELOX_DT_BF16) return false;
    if (c->head_dim != 64 && c->head_dim != 128) return false;
    if (!c->num_layers || !c->num_kv_heads || c->num_kv_heads > 1024) return false;
    if (!c->n_pages || c->n_pages >= 0x7FFFFFFFu || !c->page_size || c->page_size % 32 || c->page_size > (1u << 24)) return false;
    if (!c->n_seqs || c->n_seqs > kVxMaxPagedSeqs || !c->max_pages || c->max_pages >= 0x7FFFFFFFu) return false;
    return c->table_stride >= c->max_pages && (uint64_t)c->n_seqs * c->max_pages < 0x80000000ull;
}

bool layers_ok(const VeloxHipPagedCache* c) {
    if (!c->pool || !aligned(c->pool, 16)) return false;
    return c->num_layers == 1 || (c->layer_stride % 16 == 0 && c->layer_stride / page_bytes(*c) >= c->n_pages);
}

bool table_ok(const VeloxHipPagedCache* c) {
    return c->table && c->lens && aligned(c->table, 4) && aligned(c->lens, 4);
}

uint32_t elt(uint32_t dtype) { return dtype == VELOX_DT_F32 ? 4u : 2u; }

bool rows_ok(const VeloxHipRows* r) {
    if (!r || !r->data || r->dtype > VELOX_DT_BF16 || !r->heads || r->heads > 65535u) return false;
    return aligned(r->data, elt(r->dtype));
}

VxRowsView view(const VeloxHipRows* r) { return VxRowsView{r->data, r->row_stride, r->head_stride, r->heads, r->dtype}; }

VxPagedView view(const VeloxHipPagedCache* c, uint32_t layer) {
    VxPagedView v;
    v.pool = (uint8_t*)c->pool + (layer ? (uint64_t)layer * c->layer_stride : 0);
    v.table = c->table;
    v.lens = c->lens;
    v.page_bytes = page_bytes(*c);
    v.n_pages = c->n_pages;
    v.page_size = c->page_size;
    v.n_seqs = c->n_seqs;
    v.max_pages = c->max_pages;
    v.table_stride = c->table_stride;
    v.hkv = c->num_kv_heads;
    v.d = c->head_dim;
    v.dtype = c->dtype;
    return v;
}

uint32_t max_positions(const VeloxHipPagedCache* c, uint32_t max_len) {
    const uint64_t cap = (uint64_t)c->max_pages * c->page_size;
    const uint64_t n = max_len && max_len < cap ? max_len : cap;
    return n > 0x7FFFFFFFull ? 0x7FFFFFFFu : (uint32_t)n;
}

// Bytes of the split partials of `rows` rows: an (m, l) pair and d values for each head and split.
uint64_t part_bytes(uint32_t rows, uint32_t heads, uint32_t splits, uint32_t d) {
    return splits > 1 ? (uint64_t)rows * heads * splits * (d + 2u) * 4u : 0;
}

// out is q, or memory of its own: rows at one address have to lie alike.
bool attn_ok(const VeloxHipPagedCache* c, uint32_t layer, const VeloxHipRows* q, const VeloxHipRows* out, uint32_t n_rows, float scale) {
    if (!shape_ok(c) || !layers_ok(c) || !table_ok(c) || layer >= c->num_layers || !rows_ok(q) || !rows_ok(out)) return false;
    if (q->data == out->data && (elt(q->dtype) != elt(out->dtype) || (n_rows > 1 && q->row_stride != out->row_stride) ||
                                 (q->heads > 1 && q->head_stride != out->head_stride)))
        return false;
    return q->heads == out->heads && q->heads % c->num_kv_heads == 0 && std::isfinite(scale);
}

bool pages_ok(const VeloxHipPagedCache* c) {
    return shape_ok(c) && table_ok(c) && c->refs && c->scratch && aligned(c->refs, 16) && aligned(c->scratch, 16);
}

VxPages pages(const VeloxHipPagedCache* c) {
    VxPages p;
    p.pool = (uint8_t*)c->pool;
    p.page_bytes = page_bytes(*c);
    p.layer_stride = c->layer_stride;
    p.table = c->table;
    p.lens = c->lens;
    p.refs = c->refs;
    p.scratch = c->scratch;
    p.n_layers = c->num_layers;
    p.n_pages = c->n_pages;
    p.page_size = c->page_size;
    p.n_seqs = c->n_seqs;
    p.max_pages = c->max_pages;
    p.table_stride = c->table_stride;
    return p;
}

}  // namespace

extern "C" {

int velox_hip_paged_bytes(const VeloxHipPagedCache* c, uint64_t* page, uint64_t* pool, uint64_t* table, uint64_t* refs,
                          uint64_t* scratch) {
    if (!shape_ok(c)) return VELOX_HIP_EINVAL;
    const uint64_t pb = page_bytes(*c);
    if (page) *page = pb;
    if (pool) *pool = c->num_layers == 1 ? pb * c->n_pages : (uint64_t)(c->num_layers - 1) * c->layer_stride + pb * c->n_pages;
    if (table) *table = 4ull * c->n_seqs * c->table_stride;
    if (refs) *refs = 4ull * c->n_pages;
    if (scratch) *scratch = 4ull * (kVxPagesHead + 2ull * vx_pages_moves(c->n_seqs, c->n_pages) + c->n_pages);
    return VELOX_HIP_OK;
}

int velox_hip_rope_create(const VeloxHipRopeConfig* cfg, VeloxHipRope** out) {
    if (!cfg || !out) return VELOX_HIP_EINVAL;
    *out = nullptr;
    const uint32_t r = cfg->rot_dim;
    if (!r || r % 2 || r > 2 * kVxMaxRopePairs || cfg->layout > VELOX_ROPE_INTERLEAVED || cfg->scaling > VELOX_ROPE_YARN)
        return VELOX_HIP_EINVAL;
    if (!std::isfinite(cfg->theta) || cfg->theta <= 0.0) return VELOX_HIP_EINVAL;
    const bool scaled = cfg->scaling != VELOX_ROPE_PLAIN;
    if (scaled && !(std::isfinite(cfg->factor) && cfg->factor >= 1.0)) return VELOX_HIP_EINVAL;
    const bool by_turns = cfg->scaling == VELOX_ROPE_BANDS || cfg->scaling == VELOX_ROPE_YARN;
    double low = cfg->low_turns, high = cfg->high_turns;
    if (low == 0.0 && high == 0.0) {
        low = 1.0;
        high = cfg->scaling == VELOX_ROPE_YARN ? 32.0 : 4.0;
    }
    if (by_turns && (!cfg->original_len || !std::isfinite(high) || !(low > 0.0 && high > low))) return VELOX_HIP_EINVAL;
    if (cfg->scaling == VELOX_ROPE_YARN && cfg->theta == 1.0) return VELOX_HIP_EINVAL;
    if (!std::isfinite(cfg->amplitude) || cfg->amplitude < 0.0) return VELOX_HIP_EINVAL;
    VeloxHipRope* h = new (std::nothrow) VeloxHipRope;
    if (!h) return VELOX_HIP_ENOMEM;
    std::memset(h, 0, sizeof(*h));
    h->cfg = *cfg;
    const double two_pi = 6.283185307179586476925, len = (double)cfg->original_len;
    double first = 0.0, last = 0.0;
    if (cfg->scaling == VELOX_ROPE_YARN) {
        const auto pair = [&](double turns) { return r * std::log(len / (two_pi * turns)) / (2.0 * std::log(cfg->theta)); };
        first = std::fmax(std::floor(pair(high)), 0.0);
        last = std::fmin(std::ceil(pair(low)), (double)r - 1.0);
    }
    for (uint32_t j = 0; j < r / 2; ++j) {
        const double f = std::pow(cfg->theta, -2.0 * j / (double)r);
        double keep = 1.0;  // the share of f that stays; the rest is divided by factor
        if (cfg->scaling == VELOX_ROPE_LINEAR) keep = 0.0;
        if (cfg->scaling == VELOX_ROPE_BANDS) keep = std::fmin(1.0, std::fmax(0.0, (len * f / two_pi - low) / (high - low)));
        if (cfg->scaling == VELOX_ROPE_YARN)
            keep = 1.0 - std::fmin(1.0, std::fmax(0.0, (j - first) / std::fmax(last - first, 0.001)));
        h->freq[j] = scaled ? keep * f + (1.0 - keep) * f / cfg->factor : f;
        h->table.turns[j] = h->freq[j] / two_pi;
    }
    h->amplitude = cfg->amplitude != 0.0 ? cfg->amplitude : cfg->scaling == VELOX_ROPE_YARN ? 0.1 * std::log(cfg->factor) + 1.0 : 1.0;
    h->table.amp = (float)h->amplitude;
    h->table.rot = r;
    h->table.interleaved = cfg->layout;
    *out = h;
    return VELOX_HIP_OK;
}

void velox_hip_rope_destroy(VeloxHipRope* r) { delete r; }

int velox_hip_rope_frequencies(const VeloxHipRope* r, double* freq, double* amplitude) {
    if (!r) return VELOX_HIP_EINVAL;
    if (freq) std::memcpy(freq, r->freq, sizeof(double) * (r->cfg.rot_dim / 2));
    if (amplitude) *amplitude = r->amplitude;
    return VELOX_HIP_OK;
}

int velox_hip_rope_rows(const VeloxHipRope* r, const VeloxHipRows* x, const VeloxHipRows* out, uint32_t n_rows,
                        uint32_t head_dim, const uint32_t* d_positions, hipStream_t st) {
    if (!r || !rows_ok(x) || !rows_ok(out) || x->dtype != out->dtype || x->heads != out->heads || head_dim > 65536u ||
        r->cfg.rot_dim > head_dim || n_rows > kVxMaxRows)
        return VELOX_HIP_EINVAL;
    if (x->data == out->data && (x->row_stride != out->row_stride || x->head_stride != out->head_stride)) return VELOX_HIP_EINVAL;
    if (!n_rows) return VELOX_HIP_OK;
    if (!d_positions || !aligned(d_positions, 4)) return VELOX_HIP_EINVAL;
    return (int)vx_launch_rope_rows(r->table, view(x), view(out), n_rows, head_dim, d_positions, st);
}

int velox_hip_rope_append(const VeloxHipPagedCache* c, uint32_t layer, const VeloxHipRope* rope, const VeloxHipRows* q,
                          const VeloxHipRows* k, const VeloxHipRows* v, const VeloxHipRows* q_out,
                          const uint32_t* d_q_start, uint32_t n_rows, hipStream_t st) {
    if (!shape_ok(c) || !layers_ok(c) || !table_ok(c) || layer >= c->num_layers || !rows_ok(k) || !rows_ok(v))
        return VELOX_HIP_EINVAL;
    if (k->heads != c->num_kv_heads || v->heads != c->num_kv_heads || (rope && rope->cfg.rot_dim > c->head_dim))
        return VELOX_HIP_EINVAL;
    if (!q != !q_out) return VELOX_HIP_EINVAL;
    if (q && (!rows_ok(q) || !rows_ok(q_out) || q->heads != q_out->heads || q->dtype != q_out->dtype)) return VELOX_HIP_EINVAL;
    if (q && q->data == q_out->data && (q->row_stride != q_out->row_stride || q->head_stride != q_out->head_stride))
        return VELOX_HIP_EINVAL;
    if (!d_q_start && n_rows > c->n_seqs) return VELOX_HIP_EINVAL;
    if ((d_q_start && !aligned(d_q_start, 4)) || n_rows > kVxMaxRows) return VELOX_HIP_EINVAL;
    if (!n_rows) return VELOX_HIP_OK;
    VxAppendArgs a;
    std::memset(&a, 0, sizeof(a));
    a.c = view(c, layer);
    if (q) {
        a.q = view(q);
        a.qo = view(q_out);
    }
    a.k = view(k);
    a.v = view(v);
    a.q_start = d_q_start;
    a.n_rows = n_rows;
    VxRopeTable none;
    std::memset(&none, 0, sizeof(none));
    return (int)vx_launch_rope_append(rope ? rope->table : none, a, st);
}

int velox_hip_paged_attention_bytes(const VeloxHipPagedCache* c, uint32_t heads, uint32_t max_len, uint64_t* bytes) {
    if (!shape_ok(c) || !bytes || !heads || heads > 65535u || heads % c->num_kv_heads) return VELOX_HIP_EINVAL;
    const uint32_t s = vx_paged_attn_splits(view(c, 0), heads, c->n_seqs, max_positions(c, max_len));
    *bytes = part_bytes(c->n_seqs, heads, s, c->head_dim);
    return VELOX_HIP_OK;
}

int velox_hip_paged_attention(const VeloxHipPagedCache* c, uint32_t layer, const VeloxHipRows* q, const VeloxHipRows* out,
                              VeloxHipAttnMask mask, float scale, uint32_t max_len, void* workspace,
                              uint64_t workspace_bytes, hipStream_t st) {
    if (!attn_ok(c, layer, q, out, c ? c->n_seqs : 0, scale)) return VELOX_HIP_EINVAL;
    VxPagedAttnArgs a;
    std::memset(&a, 0, sizeof(a));
    a.c = view(c, layer);
    a.q = view(q);
    a.out = view(out);
    a.n_rows = c->n_seqs;
    a.window = mask.window;
    a.sinks = mask.sinks;
    a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt((float)c->head_dim);
    // positions a row sees: the window's and the sinks', each up to a 32-position block's end more
    uint32_t span = max_positions(c, max_len);
    if (mask.window && (uint64_t)mask.window + mask.sinks + 64u < span) span = mask.window + mask.sinks + 64u;
    a.span = span;
    a.splits = vx_paged_attn_splits(a.c, q->heads, c->n_seqs, span);
    const uint32_t planned = vx_paged_attn_splits(a.c, q->heads, c->n_seqs, max_positions(c, max_len));  // the workspace's
    if (a.splits > planned) a.splits = planned;
    const uint64_t need = part_bytes(c->n_seqs, q->heads, a.splits, c->head_dim);
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) return VELOX_HIP_EINVAL;
    a.part_o = (float*)workspace;
    a.part_ml = need ? a.part_o + (uint64_t)c->n_seqs * q->heads * a.splits * c->head_dim : nullptr;
    return (int)vx_launch_paged_attention(a, st);
}

int velox_hip_paged_prompt_attention_bytes(const VeloxHipPagedCache* c, uint32_t heads, uint32_t n_rows, uint32_t max_rows,
                                           uint32_t max_len, uint64_t* bytes) {
    if (!shape_ok(c) || !bytes || !heads || heads > 65535u || heads % c->num_kv_heads) return VELOX_HIP_EINVAL;
    if (n_rows > kVxMaxRows) return VELOX_HIP_EINVAL;
    // Fewer rows are split more: the largest need of up to n_rows rows. It is that of rows that just fill their tiles, or
    // of as many as are split at all. A window shortens a call's span, which splits less.
    const VxPagedView v = view(c, 0);
    const uint32_t g = heads / c->num_kv_heads, span = max_positions(c, max_len), split_rows = vx_paged_prompt_split_rows(v, max_rows);
    const uint32_t last = n_rows < split_rows ? n_rows : split_rows;
    uint64_t most = 0;
    if (!last) {
        *bytes = 0;
        return VELOX_HIP_OK;
    }
    for (uint32_t tiles = 1; ; ++tiles) {
        const uint64_t fill = (uint64_t)tiles * kVxPromptRows / g;
        const uint32_t rows = fill < last ? (uint32_t)fill : last;
        if (rows) {
            const uint32_t s = vx_paged_prompt_splits(v, heads, rows, max_rows, span);
            const uint64_t need = part_bytes(rows, heads, s, c->head_dim);
            if (need > most) most = need;
            if (rows == last || s == 1) break;
        }
    }
    *bytes = most;
    return VELOX_HIP_OK;
}

int velox_hip_paged_prompt_attention(const VeloxHipPagedCache* c, uint32_t layer, const VeloxHipRows* q,
                                     const VeloxHipRows* out, const uint32_t* d_q_start, uint32_t n_rows,
                                     VeloxHipAttnMask mask, float scale, uint32_t max_rows, uint32_t max_len,
                                     void* workspace, uint64_t workspace_bytes, hipStream_t st) {
    if (!attn_ok(c, layer, q, out, n_rows, scale) || !d_q_start || !aligned(d_q_start, 4) || n_rows > kVxMaxRows) return VELOX_HIP_EINVAL;
    if (!n_rows) return VELOX_HIP_OK;
    VxPagedAttnArgs a;
    std::memset(&a, 0, sizeof(a));
    a.c = view(c, layer);
    a.q = view(q);
    a.out = view(out);
    a.q_start = d_q_start;
    a.n_rows = n_rows;
    a.window = mask.window;
    a.sinks = mask.sinks;
    a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt((float)c->head_dim);
    uint32_t span = max_positions(c, max_len);
    const uint64_t seen = (uint64_t)mask.window + mask.sinks + (max_rows && max_rows < n_rows ? max_rows : n_rows) + 64u;
    if (mask.window && seen < span) span = (uint32_t)seen;
    a.splits = vx_paged_prompt_splits(a.c, q->heads, n_rows, max_rows, span);
    const uint64_t need = part_bytes(n_rows, q->heads, a.splits, c->head_dim);
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) return VELOX_HIP_EINVAL;
    a.part_o = (float*)workspace;
    a.part_ml = need ? a.part_o + (uint64_t)n_rows * q->heads * a.splits * c->head_dim : nullptr;
    return (int)vx_launch_paged_prompt(a, st);
}

int velox_hip_pages_reset(const VeloxHipPagedCache* c, hipStream_t st) {
    if (!pages_ok(c)) return VELOX_HIP_EINVAL;
    return (int)vx_launch_pages_reset(pages(c), st);
}

int velox_hip_pages_extend(const VeloxHipPagedCache* c, const uint32_t* d_add, hipStream_t st) {
    if (!pages_ok(c) || !layers_ok(c) || !d_add || !aligned(d_add, 4)) return VELOX_HIP_EINVAL;
    return (int)vx_launch_pages_extend(pages(c), d_add, st);
}

int velox_hip_pages_fork(const VeloxHipPagedCache* c, const uint32_t* d_src, hipStream_t st) {
    if (!pages_ok(c) || !d_src || !aligned(d_src, 4)) return VELOX_HIP_EINVAL;
    return (int)vx_launch_pages_fork(pages(c), d_src, st);
}

int velox_hip_pages_free(const VeloxHipPagedCache* c, const uint32_t* d_seqs, uint32_t n, hipStream_t st) {
    if (!pages_ok(c) || (n && (!d_seqs || !aligned(d_seqs, 4))) || n > 0x7FFFFFFFu) return VELOX_HIP_EINVAL;
    if (!n) return VELOX_HIP_OK;
    return (int)vx_launch_pages_free(pages(c), d_seqs, n, st);
}

int velox_hip_pages_trim(const VeloxHipPagedCache* c, uint32_t window, uint32_t sinks, hipStream_t st) {
    if (!pages_ok(c) || !window) return VELOX_HIP_EINVAL;
    return (int)vx_launch_pages_trim(pages(c), window, sinks, st);
}

int velox_hip_pages_compact(const VeloxHipPagedCache* c, hipStream_t st) {
    if (!pages_ok(c) || !layers_ok(c)) return VELOX_HIP_EINVAL;
    return (int)vx_launch_pages_compact(pages(c), st);
}

int velox_hip_pages_status(const VeloxHipPagedCache* c, uint32_t* refused, uint32_t* free_pages, hipStream_t st) {
    if (!pages_ok(c)) return VELOX_HIP_EINVAL;
    hipError_t e = vx_launch_pages_count(pages(c), st);
    uint32_t w[2] = {0, 0};
    if (e == hipSuccess) e = hipMemcpyAsync(w, c->scratch, sizeof(w), hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess) return (int)e;
    if (refused) *refused = w[0];
    if (free_pages) *free_pages = w[1];
    return VELOX_HIP_OK;
}

}  // extern "C"
