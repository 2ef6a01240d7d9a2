// Entry points of the decoder step (include/ingot_rocm.h): checks of the
// arguments, and the launches of rotary.hip, kv_pages.hip, tree_attention.hip,
// prefix_attention.hip and verify.hip on the session's stream.

#include "decoder.hpp"

#include <algorithm>
#include <cmath>

#include "runtime.hpp"

using namespace ingot;

namespace {

constexpr int64_t kMaxCount = 0x7FFFFFFF;

int check_cache(const char* what, const ingot_rocm_kv_cache* c) {
    if (!c) return fail(INGOT_EINVAL, "%s: nil cache", what);
    if (c->dtype != INGOT_DT_F32 && c->dtype != INGOT_DT_BF16)
        return fail(INGOT_EINVAL, "%s: cache must be f32 or bf16, got dtype %d", what, c->dtype);
    if (c->kv_heads < 1 || c->head_dim < 1 || c->page_size < 1 || c->layers < 1 || c->pages < 1 || c->pages > kMaxCount)
        return fail(INGOT_EINVAL, "%s: bad cache sizes (kv_heads=%d head_dim=%d page_size=%d layers=%lld pages=%lld)", what,
                    c->kv_heads, c->head_dim, c->page_size, (long long)c->layers, (long long)c->pages);
    if (!c->d_k || !c->d_v) return fail(INGOT_EINVAL, "%s: nil cache pages", what);
    const int64_t strides[4] = {c->stride_layer, c->stride_page, c->stride_head, c->stride_slot};
    const int64_t counts[4] = {c->layers, c->pages, c->kv_heads, c->page_size};
    for (int i = 0; i < 4; ++i)
        if (counts[i] > 1 && strides[i] < c->head_dim)
            return fail(INGOT_EINVAL, "%s: cache stride %lld < head_dim %d", what, (long long)strides[i], c->head_dim);
    for (int i = 0; i < 4; ++i)
        if (strides[i] % 8) return fail(INGOT_EDECLINED, "%s: cache strides must be multiples of 8", what);
    if (c->head_dim % 8 || ((uintptr_t)c->d_k & 15) || ((uintptr_t)c->d_v & 15))
        return fail(INGOT_EDECLINED, "%s: head_dim must be a multiple of 8 and the cache 16-byte aligned", what);
    return INGOT_OK;
}

int check_table(const char* what, const ingot_rocm_kv_table* t, bool refs) {
    if (!t) return fail(INGOT_EINVAL, "%s: nil table", what);
    if (t->rows < 1 || t->rows > kMaxCount || t->max_pages < 1 || t->max_pages > kMaxCount)
        return fail(INGOT_EINVAL, "%s: bad table sizes (rows=%lld max_pages=%lld)", what, (long long)t->rows,
                    (long long)t->max_pages);
    if (!t->d_pages || !t->d_len) return fail(INGOT_EINVAL, "%s: nil page table or lengths", what);
    if (refs && !t->d_refs) return fail(INGOT_EINVAL, "%s: nil reference counts", what);
    return INGOT_OK;
}

int check_batch(const char* what, const ingot_rocm_kv_batch* b, const ingot_rocm_kv_cache* c) {
    if (!b) return fail(INGOT_EINVAL, "%s: nil batch", what);
    if (b->batch < 0 || b->batch > kMaxCount || b->tokens < 0 || b->tokens > kMaxCount)
        return fail(INGOT_EINVAL, "%s: bad batch sizes (batch=%lld tokens=%lld)", what, (long long)b->batch,
                    (long long)b->tokens);
    if (b->layer < 0 || b->layer >= c->layers)
        return fail(INGOT_EINVAL, "%s: layer %lld of %lld", what, (long long)b->layer, (long long)c->layers);
    if (b->tokens && (!b->batch || !b->d_starts)) return fail(INGOT_EINVAL, "%s: tokens without a batch", what);
    return INGOT_OK;
}

// Heads that are read (any strides) or written (heads and tokens apart).
int check_heads(const char* what, const char* name, const ingot_rocm_heads* h, int64_t tokens, int64_t heads, int64_t dim,
                bool written) {
    if (!h) return fail(INGOT_EINVAL, "%s: nil %s", what, name);
    if (tokens && heads && !h->data) return fail(INGOT_EINVAL, "%s: nil %s", what, name);
    if (h->token < 0 || h->head < 0) return fail(INGOT_EINVAL, "%s: negative stride of %s", what, name);
    if (written && ((tokens > 1 && h->token < dim) || (heads > 1 && h->head < dim)))
        return fail(INGOT_EINVAL, "%s: strides of %s overlap (token=%lld head=%lld)", what, name, (long long)h->token,
                    (long long)h->head);
    return INGOT_OK;
}

int check_rotary(const char* what, const ingot_rocm_rotary* r, int64_t tokens, int64_t dim) {
    if (!r) return fail(INGOT_EINVAL, "%s: nil rotary", what);
    if (r->rot_dim < 0 || r->rot_dim % 2 || r->rot_dim > dim)
        return fail(INGOT_EINVAL, "%s: rot_dim %d must be even and at most head_dim %lld", what, r->rot_dim,
                    (long long)dim);
    if (r->rows < 0) return fail(INGOT_EINVAL, "%s: negative table rows", what);
    if (tokens && r->rot_dim && (!r->d_positions || (r->rows && (!r->d_cos || !r->d_sin))))
        return fail(INGOT_EINVAL, "%s: nil positions or tables", what);
    return INGOT_OK;
}

int check_norm(const char* what, const char* name, const ingot_rocm_head_norm* n, int64_t heads, int64_t dim) {
    if (!n) return INGOT_OK;  // not normed
    if (!(n->eps >= 0.f) || !std::isfinite(n->eps))
        return fail(INGOT_EINVAL, "%s: eps of %s must be finite and not negative", what, name);
    if (n->head < 0 || (n->d_weight && heads > 1 && n->head && n->head < dim))
        return fail(INGOT_EINVAL, "%s: weights of %s %lld elements apart", what, name, (long long)n->head);
    return INGOT_OK;
}

int check_dtype(const char* what, int32_t dtype) {
    if (dtype != INGOT_DT_F32 && dtype != INGOT_DT_BF16)
        return fail(INGOT_EINVAL, "%s: heads must be f32 or bf16, got dtype %d", what, dtype);
    return INGOT_OK;
}

HeadsView heads_view(const ingot_rocm_heads* h) { return {(char*)h->data, h->token, h->head}; }

RotaryView rotary_view(const ingot_rocm_rotary* r, int inverse) {
    return {r->d_cos, r->d_sin, r->d_positions, r->rows, r->rot_dim / 2, r->interleaved != 0, inverse != 0};
}

KvView kv_view(const ingot_rocm_kv_cache* c, const ingot_rocm_kv_table* t, const ingot_rocm_kv_batch* b) {
    KvView v = {};
    const int64_t at = (b ? b->layer : 0) * c->stride_layer * (c->dtype == INGOT_DT_F32 ? 4 : 2);
    v.k = (char*)c->d_k + at;
    v.v = (char*)c->d_v + at;
    v.stride_page = c->stride_page;
    v.stride_head = c->stride_head;
    v.stride_slot = c->stride_slot;
    v.pages = t->d_pages;
    v.len = t->d_len;
    v.page_size = c->page_size;
    v.num_pages = (int32_t)c->pages;
    v.kv_heads = c->kv_heads;
    v.max_pages = (int32_t)t->max_pages;
    v.rows = (int32_t)t->rows;
    v.by_page = FastDiv(c->page_size);
    if (b) {
        v.starts = b->d_starts;
        v.row = b->d_row;
        v.batch = (int32_t)b->batch;
        v.tokens = (int32_t)b->tokens;
    }
    return v;
}

PagesView pages_view(const ingot_rocm_kv_cache* c, const ingot_rocm_kv_table* t) {
    PagesView v = {};
    const int esz = c->dtype == INGOT_DT_F32 ? 4 : 2;
    const bool together = c->kv_heads > 1 && c->stride_head == c->head_dim;  // a slot's heads are neighbours
    v.k = (char*)c->d_k;
    v.v = (char*)c->d_v;
    v.stride_layer = c->stride_layer * esz;
    v.stride_page = c->stride_page * esz;
    v.stride_seg = together ? 0 : c->stride_head * esz;
    v.stride_slot = c->stride_slot * esz;
    v.layers = (int32_t)c->layers;
    v.segs = together ? 1 : c->kv_heads;
    v.row_chunks = (together ? c->kv_heads : 1) * c->head_dim * esz / 16;
    v.page_size = c->page_size;
    v.num_pages = (int32_t)c->pages;
    v.by_page = FastDiv(c->page_size);
    if (t) {
        v.rows = (int32_t)t->rows;
        v.max_pages = (int32_t)t->max_pages;
        v.pages = t->d_pages;
        v.len = t->d_len;
        v.refs = t->d_refs;
        v.missing = t->d_missing;
    }
    return v;
}

// The checks the page operations share: lists of n entries, and a cache whose
// chunks of a page can be counted in 31 bits.
int check_pages(const char* what, const ingot_rocm_kv_cache* c, int64_t n, const void* a, const void* b) {
    int rc = check_cache(what, c);
    if (rc) return rc;
    if (n < 0 || n > (1 << 20)) return fail(INGOT_EINVAL, "%s: %lld list entries", what, (long long)n);
    if (n && (!a || !b)) return fail(INGOT_EINVAL, "%s: nil list", what);
    const int64_t row = (int64_t)c->head_dim * (c->dtype == INGOT_DT_F32 ? 4 : 2) / 16 * c->kv_heads;
    if (c->layers > (1 << 16) || row > (1 << 24) || row * c->page_size > (1 << 28) ||
        row * c->page_size * c->layers > (1ll << 29))
        return fail(INGOT_EDECLINED, "%s: a page of more than 2^29 16-byte chunks over the layers", what);
    return INGOT_OK;
}

// The checks of a rotation, and its launch arguments (tokens 0: nothing to do).
int apply_args(const char* what, const ingot_rocm_rotary* rot, int64_t tokens, int64_t heads, int64_t head_dim,
               int32_t dtype, const ingot_rocm_heads* x, const ingot_rocm_heads* y, int32_t inverse, RotaryArgs& a) {
    int rc;
    if (tokens < 0 || tokens > kMaxCount || heads < 0 || head_dim < 0 || heads > (1 << 20) || head_dim > (1 << 16) ||
        heads * head_dim > (1 << 26))
        return fail(INGOT_EINVAL, "%s: bad sizes (tokens=%lld heads=%lld head_dim=%lld)", what, (long long)tokens,
                    (long long)heads, (long long)head_dim);
    if ((rc = check_dtype(what, dtype)) || (rc = check_rotary(what, rot, tokens, head_dim)) ||
        (rc = check_heads(what, "x", x, tokens, heads, head_dim, false)) ||
        (rc = check_heads(what, "y", y, tokens, heads, head_dim, true)))
        return rc;
    if (x->data == y->data && tokens && heads && (x->token != y->token || x->head != y->head))
        return fail(INGOT_EINVAL, "%s: x in place needs y's strides", what);
    if (!heads || !head_dim) return INGOT_OK;
    a.rot = rotary_view(rot, inverse);
    a.x = heads_view(x);
    a.y = heads_view(y);
    a.tokens = tokens;
    a.heads = (int32_t)heads;
    a.dim = (int32_t)head_dim;
    return INGOT_OK;
}

// The checks of a rotation with its append, and its launch arguments.
int append_args(const char* what, const ingot_rocm_rotary* rot, const ingot_rocm_kv_cache* cache,
                const ingot_rocm_kv_table* table, const ingot_rocm_kv_batch* batch, int64_t heads, int32_t dtype,
                const ingot_rocm_heads* q, const ingot_rocm_heads* k, const ingot_rocm_heads* v,
                const ingot_rocm_heads* y, RotaryArgs& a) {
    int rc;
    if ((rc = check_cache(what, cache)) || (rc = check_table(what, table, false)) ||
        (rc = check_batch(what, batch, cache)) || (rc = check_dtype(what, dtype)))
        return rc;
    const int64_t dim = cache->head_dim, kv_heads = cache->kv_heads;
    if (heads < 0 || heads > (1 << 20) || heads + 2 * kv_heads > (1 << 20) || dim > (1 << 16) ||
        (heads + 2 * kv_heads) * dim > (1 << 26))
        return fail(INGOT_EINVAL, "%s: bad sizes (heads=%lld kv_heads=%d head_dim=%lld)", what, (long long)heads,
                    cache->kv_heads, (long long)dim);
    if ((rc = check_rotary(what, rot, batch->tokens, dim)) ||
        (rc = check_heads(what, "q", q, batch->tokens, heads, dim, false)) ||
        (rc = check_heads(what, "k", k, batch->tokens, cache->kv_heads, dim, false)) ||
        (rc = check_heads(what, "v", v, batch->tokens, cache->kv_heads, dim, false)) ||
        (rc = check_heads(what, "y", y, batch->tokens, heads, dim, true)))
        return rc;
    if (heads && q->data == y->data && batch->tokens && (q->token != y->token || q->head != y->head))
        return fail(INGOT_EINVAL, "%s: q in place needs y's strides", what);
    a.rot = rotary_view(rot, 0);
    a.x = heads_view(q);
    a.y = heads_view(y);
    a.k = heads_view(k);
    a.v = heads_view(v);
    a.tokens = batch->tokens;
    a.heads = (int32_t)heads;
    a.kv_heads = cache->kv_heads;
    a.dim = (int32_t)dim;
    a.kv = kv_view(cache, table, batch);
    return INGOT_OK;
}

// The checks of attention over the cache, and its launch arguments (heads 0: nothing
// to do).
int attention_args(const char* what, const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                   const ingot_rocm_kv_batch* batch, const ingot_rocm_tree_attention_args* args, TreeAttnArgs& a) {
    int rc;
    if ((rc = check_cache(what, cache)) || (rc = check_table(what, table, false)) ||
        (rc = check_batch(what, batch, cache)))
        return rc;
    if (!args) return fail(INGOT_EINVAL, "%s: nil arguments", what);
    const ingot_rocm_tree_attention_args& g = *args;
    if ((rc = check_dtype(what, g.dtype))) return rc;
    if (g.heads < 0 || g.heads > (1 << 20) || g.heads % cache->kv_heads)
        return fail(INGOT_EINVAL, "%s: %lld heads over %d key heads", what, (long long)g.heads, cache->kv_heads);
    if (g.max_nodes < 0 || g.max_nodes > kMaxCount || g.max_tokens < 0 || g.max_tokens > kMaxCount || g.mask_words < 0 ||
        g.mask_words > (1 << 26))
        return fail(INGOT_EINVAL, "%s: bad sizes (max_nodes=%lld max_tokens=%lld mask_words=%lld)", what,
                    (long long)g.max_nodes, (long long)g.max_tokens, (long long)g.mask_words);
    if (g.d_mask && !g.mask_words && batch->tokens) return fail(INGOT_EINVAL, "%s: a mask of no words", what);
    if (!std::isfinite(g.scale)) return fail(INGOT_EINVAL, "%s: scale must be finite", what);
    if ((rc = check_heads(what, "q", &g.q, batch->tokens, g.heads, cache->head_dim, false)) ||
        (rc = check_heads(what, "y", &g.y, batch->tokens, g.heads, cache->head_dim, true)))
        return rc;
    if (g.q.data == g.y.data && batch->tokens && g.heads && (g.q.token != g.y.token || g.q.head != g.y.head))
        return fail(INGOT_EINVAL, "%s: q in place needs y's strides", what);
    if (cache->head_dim > 256) return fail(INGOT_EDECLINED, "%s: head_dim %d > 256", what, cache->head_dim);
    if (!batch->tokens || !g.heads || !g.max_nodes) return INGOT_OK;
    a.kv = kv_view(cache, table, batch);
    a.q = heads_view(&g.q);
    a.y = heads_view(&g.y);
    a.mask = g.d_mask;
    a.mask_words = g.mask_words;
    a.heads = (int32_t)g.heads;
    a.group = (int32_t)(g.heads / cache->kv_heads);
    a.by_group = FastDiv(a.group);
    a.dim = cache->head_dim;
    a.max_nodes = (int32_t)std::min(g.max_nodes, batch->tokens);
    const int64_t held = std::min(kMaxCount, table->max_pages * cache->page_size);
    a.max_tokens = (int32_t)(g.max_tokens ? std::min(g.max_tokens, held) : held);
    if (cache->stride_slot > (1 << 28) || cache->page_size > (1 << 30))
        return fail(INGOT_EDECLINED, "%s: slots %lld elements apart, %d to a page", what, (long long)cache->stride_slot,
                    cache->page_size);
    if (a.max_tokens > (1 << 30))  // positions plus a block stay within 31 bits
        return fail(INGOT_EDECLINED, "%s: max_tokens %d > 2^30", what, a.max_tokens);
    if ((int64_t)a.max_nodes * a.group > (1 << 28)) return fail(INGOT_EDECLINED, "%s: too many rows", what);
    a.q_bf16 = g.dtype == INGOT_DT_BF16;
    const int esz = a.q_bf16 ? 2 : 4, quad = 4 * esz;
    a.q_vec = ((uintptr_t)g.q.data % 16 == 0) && (g.q.token * esz) % 16 == 0 && (g.q.head * esz) % 16 == 0;
    a.y_vec = ((uintptr_t)g.y.data % quad == 0) && g.y.token % 4 == 0 && g.y.head % 4 == 0;
    // scores are taken to powers of two by one multiply-add with a positive factor;
    // with a scale of 0 the least one, so that hidden scores (−Inf) stay −Inf
    a.flip = g.scale < 0.f;
    a.scale = std::max(std::fabs(g.scale) * 1.4426950408889634f, 0x1p-126f);
    return INGOT_OK;
}

void set_norms(NormRotaryArgs& a, const ingot_rocm_head_norm* q, const ingot_rocm_head_norm* k) {
    a.inv_dim = 1.f / (float)a.dim;
    a.norm_q = q != nullptr;
    a.norm_k = k != nullptr;
    if (q) a.weight_q = q->d_weight, a.weight_q_head = q->head, a.eps_q = q->eps;
    if (k) a.weight_k = k->d_weight, a.weight_k_head = k->head, a.eps_k = k->eps;
}

}  // namespace

extern "C" {

int ingot_rocm_rotary_table(ingot_rocm_session* s, const ingot_rocm_rotary_table_args* a) {
    int rc = session_enter(s);
    if (rc) return rc;
    if (!a) return fail(INGOT_EINVAL, "rotary_table: nil arguments");
    if (a->rows < 0 || a->rows > kMaxCount || a->first < 0 || a->first > kMaxCount - a->rows || a->rot_dim < 0 ||
        a->rot_dim % 2 || a->rot_dim > 65536)
        return fail(INGOT_EINVAL, "rotary_table: bad sizes (first=%lld rows=%lld rot_dim=%d)", (long long)a->first,
                    (long long)a->rows, a->rot_dim);
    if (a->scaling < INGOT_ROTARY_PLAIN || a->scaling > INGOT_ROTARY_BY_PARTS)
        return fail(INGOT_EINVAL, "rotary_table: unknown scaling %d", a->scaling);
    if (!(a->base > 0) || !std::isfinite(a->base) || !std::isfinite(a->amplitude))
        return fail(INGOT_EINVAL, "rotary_table: base must be positive and finite, amplitude finite");
    if (a->scaling != INGOT_ROTARY_PLAIN && (!(a->factor > 0) || !std::isfinite(a->factor)))
        return fail(INGOT_EINVAL, "rotary_table: factor must be positive and finite");
    if (a->scaling == INGOT_ROTARY_BY_PARTS &&
        (!(a->trained > 0) || !std::isfinite(a->trained) || !std::isfinite(a->low) || !std::isfinite(a->high) || !(a->high > a->low)))
        return fail(INGOT_EINVAL, "rotary_table: by parts needs trained > 0 and low < high");
    if (!a->rows || !a->rot_dim) return INGOT_OK;
    if (!a->d_cos || !a->d_sin) return fail(INGOT_EINVAL, "rotary_table: nil tables");
    if (a->rows * (a->rot_dim / 2) > (int64_t)1 << 38) return fail(INGOT_EINVAL, "rotary_table: too many angles");
    hipError_t e = launch_rotary_table(*a, s->stream);
    if (e != hipSuccess) return hip_fail(e, "rotary_table launch");
    return INGOT_OK;
}

int ingot_rocm_rotary_apply(ingot_rocm_session* s, const ingot_rocm_rotary* rot, int64_t tokens, int64_t heads,
                            int64_t head_dim, int32_t dtype, const ingot_rocm_heads* x, const ingot_rocm_heads* y,
                            int32_t inverse) {
    static const char* what = "rotary_apply";
    int rc = session_enter(s);
    if (rc) return rc;
    RotaryArgs a = {};
    if ((rc = apply_args(what, rot, tokens, heads, head_dim, dtype, x, y, inverse, a)) || !a.tokens) return rc;
    hipError_t e = launch_rotary(a, dtype, dtype, s->stream);
    if (e != hipSuccess) return hip_fail(e, "rotary launch");
    return INGOT_OK;
}

int ingot_rocm_rotary_append(ingot_rocm_session* s, const ingot_rocm_rotary* rot, const ingot_rocm_kv_cache* cache,
                             const ingot_rocm_kv_table* table, const ingot_rocm_kv_batch* batch, int64_t heads,
                             int32_t dtype, const ingot_rocm_heads* q, const ingot_rocm_heads* k,
                             const ingot_rocm_heads* v, const ingot_rocm_heads* y) {
    static const char* what = "rotary_append";
    int rc = session_enter(s);
    if (rc) return rc;
    RotaryArgs a = {};
    if ((rc = append_args(what, rot, cache, table, batch, heads, dtype, q, k, v, y, a)) || !a.tokens) return rc;
    hipError_t e = launch_rotary(a, dtype, cache->dtype, s->stream);
    if (e != hipSuccess) return hip_fail(e, "rotary_append launch");
    return INGOT_OK;
}

int ingot_rocm_norm_rotary_apply(ingot_rocm_session* s, const ingot_rocm_head_norm* norm, const ingot_rocm_rotary* rot,
                                 int64_t tokens, int64_t heads, int64_t head_dim, int32_t dtype,
                                 const ingot_rocm_heads* x, const ingot_rocm_heads* y) {
    static const char* what = "norm_rotary_apply";
    int rc = session_enter(s);
    if (rc) return rc;
    NormRotaryArgs a = {};
    if ((rc = apply_args(what, rot, tokens, heads, head_dim, dtype, x, y, 0, a))) return rc;
    if (!norm) return fail(INGOT_EINVAL, "%s: nil norm", what);
    if ((rc = check_norm(what, "x", norm, heads, head_dim)) || !a.tokens) return rc;
    set_norms(a, norm, nullptr);
    hipError_t e = launch_norm_rotary(a, dtype, dtype, s->stream);
    if (e != hipSuccess) return hip_fail(e, "norm_rotary launch");
    return INGOT_OK;
}

int ingot_rocm_norm_rotary_append(ingot_rocm_session* s, const ingot_rocm_head_norm* norm_q,
                                  const ingot_rocm_head_norm* norm_k, const ingot_rocm_rotary* rot,
                                  const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                                  const ingot_rocm_kv_batch* batch, int64_t heads, int32_t dtype,
                                  const ingot_rocm_heads* q, const ingot_rocm_heads* k, const ingot_rocm_heads* v,
                                  const ingot_rocm_heads* y) {
    static const char* what = "norm_rotary_append";
    int rc = session_enter(s);
    if (rc) return rc;
    NormRotaryArgs a = {};
    if ((rc = append_args(what, rot, cache, table, batch, heads, dtype, q, k, v, y, a))) return rc;
    if ((rc = check_norm(what, "q", norm_q, heads, cache->head_dim)) ||
        (rc = check_norm(what, "k", norm_k, cache->kv_heads, cache->head_dim)) || !a.tokens)
        return rc;
    set_norms(a, norm_q, norm_k);
    hipError_t e = launch_norm_rotary(a, dtype, cache->dtype, s->stream);
    if (e != hipSuccess) return hip_fail(e, "norm_rotary_append launch");
    return INGOT_OK;
}

int ingot_rocm_kv_copy(ingot_rocm_session* s, const ingot_rocm_kv_cache* cache, const int32_t* d_src,
                       const int32_t* d_dst, int64_t n) {
    static const char* what = "kv_copy";
    int rc = session_enter(s);
    if (rc) return rc;
    if ((rc = check_pages(what, cache, n, d_src, d_dst))) return rc;
    if (!n) return INGOT_OK;
    hipError_t e = launch_kv_copy(pages_view(cache, nullptr), d_src, d_dst, n, s->stream);
    if (e != hipSuccess) return hip_fail(e, "kv_copy launch");
    return INGOT_OK;
}

int ingot_rocm_kv_reserve(ingot_rocm_session* s, const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                          const int32_t* d_row, const int32_t* d_tokens, int64_t n) {
    static const char* what = "kv_reserve";
    int rc = session_enter(s);
    if (rc) return rc;
    if ((rc = check_pages(what, cache, n, d_row, d_tokens)) || (rc = check_table(what, table, true))) return rc;
    if (!table->d_missing) return fail(INGOT_EINVAL, "%s: nil missing count", what);
    void* ws;
    if ((rc = ws_reserve(s, kv_alloc_ws(n, cache->pages), &ws))) return rc;
    hipError_t e = launch_kv_reserve(pages_view(cache, table), d_row, d_tokens, (int)n, ws, s->stream);
    if (e != hipSuccess) return hip_fail(e, "kv_reserve launch");
    return INGOT_OK;
}

int ingot_rocm_kv_fork(ingot_rocm_session* s, const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                       const int32_t* d_src, const int32_t* d_dst, int64_t n) {
    static const char* what = "kv_fork";
    int rc = session_enter(s);
    if (rc) return rc;
    if ((rc = check_pages(what, cache, n, d_src, d_dst)) || (rc = check_table(what, table, true))) return rc;
    if (!table->d_missing) return fail(INGOT_EINVAL, "%s: nil missing count", what);
    void* ws;
    if ((rc = ws_reserve(s, kv_alloc_ws(n, cache->pages), &ws))) return rc;
    hipError_t e = launch_kv_fork(pages_view(cache, table), d_src, d_dst, (int)n, ws, s->stream);
    if (e != hipSuccess) return hip_fail(e, "kv_fork launch");
    return INGOT_OK;
}

int ingot_rocm_kv_free(ingot_rocm_session* s, const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                       const int32_t* d_row, int64_t n) {
    static const char* what = "kv_free";
    int rc = session_enter(s);
    if (rc) return rc;
    if ((rc = check_pages(what, cache, n, d_row, d_row)) || (rc = check_table(what, table, true))) return rc;
    if (!n) return INGOT_OK;
    hipError_t e = launch_kv_free(pages_view(cache, table), d_row, (int)n, s->stream);
    if (e != hipSuccess) return hip_fail(e, "kv_free launch");
    return INGOT_OK;
}

int ingot_rocm_kv_compact(ingot_rocm_session* s, const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                          const int32_t* d_row, const int32_t* d_accept, const int32_t* d_count, int64_t n,
                          int64_t max_accept, int32_t* d_new_len) {
    static const char* what = "kv_compact";
    int rc = session_enter(s);
    if (rc) return rc;
    if ((rc = check_pages(what, cache, n, d_row, d_count)) || (rc = check_table(what, table, false))) return rc;
    if (max_accept < 0 || max_accept > (1 << 20)) return fail(INGOT_EINVAL, "%s: max_accept %lld", what, (long long)max_accept);
    if (!n) return INGOT_OK;
    if (!d_new_len || (max_accept && !d_accept)) return fail(INGOT_EINVAL, "%s: nil list", what);
    if (d_new_len == table->d_len) return fail(INGOT_EINVAL, "%s: the new lengths must not be the table's", what);
    hipError_t e = launch_kv_compact(pages_view(cache, table), d_row, d_accept, d_count, (int)n, (int)max_accept,
                                     d_new_len, s->stream);
    if (e != hipSuccess) return hip_fail(e, "kv_compact launch");
    return INGOT_OK;
}

int ingot_rocm_tree_attention(ingot_rocm_session* s, const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                              const ingot_rocm_kv_batch* batch, const ingot_rocm_tree_attention_args* args) {
    static const char* what = "tree_attention";
    int rc = session_enter(s);
    if (rc) return rc;
    TreeAttnArgs a = {};
    if ((rc = attention_args(what, cache, table, batch, args, a)) || !a.heads) return rc;
    const size_t need = plan_tree_attention(a, cache->dtype, s->num_cus);
    if (a.items < 1) return fail(INGOT_EDECLINED, "%s: too many tiles", what);
    if (need) {
        void* ws;
        if ((rc = ws_reserve(s, need, &ws))) return rc;
        place_tree_attention(a, cache->dtype, ws);
    }
    hipError_t e = launch_tree_attention(a, cache->dtype, s->stream);
    if (e != hipSuccess) return hip_fail(e, "tree_attention launch");
    return INGOT_OK;
}

int ingot_rocm_prefix_attention(ingot_rocm_session* s, const ingot_rocm_kv_cache* cache, const ingot_rocm_kv_table* table,
                                const ingot_rocm_kv_batch* batch, const ingot_rocm_kv_prefix* prefix,
                                const ingot_rocm_tree_attention_args* args) {
    static const char* what = "prefix_attention";
    int rc = session_enter(s);
    if (rc) return rc;
    TreeAttnArgs a = {};
    if ((rc = attention_args(what, cache, table, batch, args, a))) return rc;
    if (!prefix) return fail(INGOT_EINVAL, "%s: nil prefix", what);
    if (prefix->groups < 0 || prefix->groups > batch->batch || prefix->max_tokens < 0 || prefix->max_tokens > kMaxCount)
        return fail(INGOT_EINVAL, "%s: bad sizes (groups=%lld of %lld sequences, max_tokens=%lld)", what,
                    (long long)prefix->groups, (long long)batch->batch, (long long)prefix->max_tokens);
    if (prefix->groups && (!prefix->d_first || !prefix->d_tokens)) return fail(INGOT_EINVAL, "%s: nil groups", what);
    if (!a.heads) return INGOT_OK;
    if (!prefix->groups) return ingot_rocm_tree_attention(s, cache, table, batch, args);
    PrefixArgs p = {};
    p.t = a;
    p.first = prefix->d_first;
    p.shared = prefix->d_tokens;
    p.prefix.count = (int32_t)prefix->groups;
    p.max_shared = (int32_t)(prefix->max_tokens ? std::min<int64_t>(prefix->max_tokens, a.max_tokens) : a.max_tokens);
    size_t need = 0;  // of a launch for prefixes, if one is known to pay and is not too large
    if (s->prefix_path ? s->prefix_path != 1 : prefix->max_tokens && prefix_pays(p, cache->dtype))
        need = plan_prefix_attention(p, cache->dtype, s->num_cus);
    if (!need) return ingot_rocm_tree_attention(s, cache, table, batch, args);
    void* ws;
    if ((rc = ws_reserve(s, need, &ws))) return rc;
    hipError_t e = launch_prefix_attention(p, cache->dtype, ws, s->stream);
    if (e != hipSuccess) return hip_fail(e, "prefix_attention launch");
    return INGOT_OK;
}

int ingot_rocm_verify_drafts(ingot_rocm_session* s, const ingot_rocm_verify_args* args) {
    static const char* what = "verify_drafts";
    int rc = session_enter(s);
    if (rc) return rc;
    if (!args) return fail(INGOT_EINVAL, "%s: nil arguments", what);
    const ingot_rocm_verify_args& g = *args;
    if (g.batch < 0 || g.batch > kMaxCount || g.tokens < 0 || g.tokens > kMaxCount || g.vocab < 1 || g.max_accept < 1 ||
        g.max_accept > kMaxCount)
        return fail(INGOT_EINVAL, "%s: bad sizes (batch=%lld tokens=%lld vocab=%lld max_accept=%lld)", what,
                    (long long)g.batch, (long long)g.tokens, (long long)g.vocab, (long long)g.max_accept);
    if (g.dtype != INGOT_DT_F32 && g.dtype != INGOT_DT_BF16)
        return fail(INGOT_EINVAL, "%s: logits must be f32 or bf16, got dtype %d", what, g.dtype);
    if (g.logits_ld < g.vocab || (g.d_draft && g.draft_ld < g.vocab))
        return fail(INGOT_EINVAL, "%s: rows of %lld and %lld elements for %lld tokens", what, (long long)g.logits_ld,
                    (long long)g.draft_ld, (long long)g.vocab);
    if (g.d_draft && g.d_parents) return fail(INGOT_EINVAL, "%s: draft logits go with a chain (no parents)", what);
    if (!g.batch) return INGOT_OK;
    if (!g.d_starts || !g.d_accepted || !g.d_counts || !g.d_next) return fail(INGOT_EINVAL, "%s: nil starts or outputs", what);
    if (g.tokens && (!g.d_logits || !g.d_tokens)) return fail(INGOT_EINVAL, "%s: nil logits or tokens", what);
    if (g.d_temperature && (!g.d_sample_u || (g.tokens && !g.d_accept_u)))
        return fail(INGOT_EINVAL, "%s: temperatures without random numbers", what);
    if (g.vocab > (1 << 24)) return fail(INGOT_EDECLINED, "%s: vocabulary of %lld > 2^24", what, (long long)g.vocab);
    if (g.logits_ld > (int64_t)1 << 30 || (g.d_draft && g.draft_ld > (int64_t)1 << 30))
        return fail(INGOT_EDECLINED, "%s: rows more than 2^30 elements apart", what);
    VerifyArgs a = {};
    a.logits = g.d_logits;
    a.draft = g.d_draft;
    a.logits_ld = g.logits_ld;
    a.draft_ld = g.draft_ld;
    a.starts = g.d_starts;
    a.draft_tokens = g.d_tokens;
    a.parents = g.d_parents;
    a.temperature = g.d_temperature;
    a.accept_u = g.d_accept_u;
    a.sample_u = g.d_sample_u;
    a.accepted = g.d_accepted;
    a.counts = g.d_counts;
    a.next = g.d_next;
    a.batch = (int32_t)g.batch;
    a.tokens = (int32_t)g.tokens;
    a.vocab = (int32_t)g.vocab;
    a.max_accept = (int32_t)g.max_accept;
    a.bf16 = g.dtype == INGOT_DT_BF16;
    const size_t need = plan_verify(a);
    if (!need) return fail(INGOT_EDECLINED, "%s: too many logits", what);
    void* ws;
    if ((rc = ws_reserve(s, need, &ws))) return rc;
    place_verify(a, ws);
    hipError_t e = launch_verify(a, s->stream);
    if (e != hipSuccess) return hip_fail(e, "verify_drafts launch");
    return INGOT_OK;
}

}  // extern "C"
