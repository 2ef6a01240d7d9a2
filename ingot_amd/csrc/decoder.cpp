// Entry points of the decoder step (include/ingot_rocm.h): checks of the
// arguments, and the launches of rotary.hip, kv_pages.hip and
// tree_attention.hip on the session's stream.

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

}  // namespace

extern "C" {

int ingot_rocm_rotary_table(ingot_rocm_session* s, const ingot_rocm_rotary_table_args* a) {
    int rc = session_enter(s);
    if (rc) return rc;
    if (!a) return fail(INGOT_EINVAL, "rotary_table: nil arguments");
    if (a->rows < 0 || a->first < 0 || a->first + a->rows > kMaxCount || a->rot_dim < 0 || a->rot_dim % 2 ||
        a->rot_dim > 65536)
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
    if (!tokens || !heads || !head_dim) return INGOT_OK;
    RotaryArgs a = {};
    a.rot = rotary_view(rot, inverse);
    a.x = heads_view(x);
    a.y = heads_view(y);
    a.tokens = tokens;
    a.heads = (int32_t)heads;
    a.dim = (int32_t)head_dim;
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
    if ((rc = check_cache(what, cache)) || (rc = check_table(what, table, false)) ||
        (rc = check_batch(what, batch, cache)) || (rc = check_dtype(what, dtype)))
        return rc;
    const int64_t dim = cache->head_dim, all = heads + 2 * (int64_t)cache->kv_heads;
    if (heads < 0 || all > (1 << 20) || dim > (1 << 16) || all * dim > (1 << 26))
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
    if (!batch->tokens) return INGOT_OK;
    RotaryArgs a = {};
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
    hipError_t e = launch_rotary(a, dtype, cache->dtype, s->stream);
    if (e != hipSuccess) return hip_fail(e, "rotary_append launch");
    return INGOT_OK;
}

}  // extern "C"
