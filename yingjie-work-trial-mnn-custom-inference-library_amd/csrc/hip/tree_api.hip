// tree_api.hip - entry points of the decode step over a tree of drafted tokens
// (declared in include/xqhip.h): argument checks and launch descriptions.
#include "xqhip.h"
#include "xqhip_kernels.hpp"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <string>

namespace xqhip {
void set_last_error(const std::string& msg);  // xqhip_api.hip
}  // namespace xqhip

namespace {

int refuse(const char* fmt, ...) {
    char buf[384];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    xqhip::set_last_error(buf);
    return XQHIP_EINVAL;
}

int check(hipError_t e, const char* what) {
    if (e == hipSuccess) return XQHIP_OK;
    xqhip::set_last_error(std::string(what) + ": " + hipGetErrorString(e));
    return XQHIP_EDEVICE;
}

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

constexpr int kMaxCapacity = 1 << 20, kMaxVocab = 1 << 24;
static_assert(XQHIP_TREE_MAX == xqhip::kTreeMax, "one mask word per row");

const char* tree_fault(const xqhip_tree* t) {
    if (t->nodes < 1 || t->nodes > XQHIP_TREE_MAX) return "1 to 64 rows";
    if (t->parent[0] != -1) return "row 0 is a root";
    for (int i = 0; i < t->nodes; ++i) {
        if (t->parent[i] < -1 || t->parent[i] >= i) return "a row's parent comes before it";
        if (t->depth[i] != (t->parent[i] < 0 ? 0 : t->depth[t->parent[i]] + 1)) return "depths as xqhip_tree_init sets them";
    }
    return nullptr;
}

const char* kv_fault(const xqhip_kv* kv) {
    if (kv->type != XQHIP_KV_F16 && kv->type != XQHIP_KV_I8) return "cache type";
    if (kv->nkv <= 0 || kv->nkv > 65535 || kv->head_dim <= 0 || kv->head_dim > 1024) return "cache heads";
    if (kv->capacity <= 0 || kv->capacity > kMaxCapacity) return "cache capacity (1 to 2^20 positions)";
    if (!kv->k || !kv->v) return "cache pointers";
    if (kv->type == XQHIP_KV_I8 && (!kv->k_scale || !kv->v_scale)) return "cache scales";
    return nullptr;
}

xqhip::KvCache cache_of(const xqhip_kv* kv) {
    return xqhip::KvCache{kv->k, kv->v, kv->k_scale, kv->v_scale, kv->type == XQHIP_KV_I8, kv->nkv, kv->head_dim,
                          kv->capacity};
}

xqhip::TreeLinks links_of(const xqhip_tree* t) {
    xqhip::TreeLinks l{};
    for (int i = 0; i < t->nodes; ++i) l.words[i / 4] |= static_cast<uint32_t>(t->parent[i] & 0xff) << 8 * (i % 4);
    return l;
}

bool workspace_ok(const void* ws, size_t have, size_t need) {
    return need == 0 || (ws && (reinterpret_cast<uintptr_t>(ws) & 15u) == 0 && have >= need);
}

}  // namespace

extern "C" {

int xqhip_tree_init(const int32_t* parent, int nodes, xqhip_tree* out) {
    if (!parent || !out || nodes < 1 || nodes > XQHIP_TREE_MAX)
        return refuse("xqhip_tree_init: 1 to %d rows (nodes=%d)", XQHIP_TREE_MAX, nodes);
    xqhip_tree t{};
    t.nodes = nodes;
    for (int i = 0; i < nodes; ++i) {
        const int p = parent[i];
        if (p < -1 || p >= i || (i == 0 && p != -1))
            return refuse("xqhip_tree_init: row %d continues row %d", i, p);
        t.parent[i] = p;
        t.depth[i] = p < 0 ? 0 : t.depth[p] + 1;
        t.mask[i] = (p < 0 ? 0 : t.mask[p]) | uint64_t(1) << i;
    }
    *out = t;
    return XQHIP_OK;
}

int xqhip_attn_prep_kv(const float* q_src, const float* k_src, const float* v_src, int gated, int nq, int rotary_dim,
                       const float* q_norm, const float* k_norm, float eps, const float* rope_cs, const int32_t* pos0,
                       const xqhip_tree* tree, int tokens, int src_stride, int out_stride, float* q_out,
                       float* gate_out, const xqhip_kv* kv, void* stream) {
    if (!q_src || !k_src || !v_src || !q_norm || !k_norm || !pos0 || !q_out || !kv || (gated && !gate_out) ||
        nq <= 0 || nq > 65535 || (rotary_dim > 0 && !rope_cs) || tokens <= 0 || tokens > 65535)
        return refuse("xqhip_attn_prep_kv: bad args");
    if (const char* f = kv_fault(kv)) return refuse("xqhip_attn_prep_kv: %s", f);
    const int hd = kv->head_dim;
    if (out_stride < static_cast<int64_t>(nq) * hd || src_stride < 0)
        return refuse("xqhip_attn_prep_kv: row strides");
    if (tree) {
        if (const char* f = tree_fault(tree)) return refuse("xqhip_attn_prep_kv: tree: %s", f);
        if (tree->nodes != tokens) return refuse("xqhip_attn_prep_kv: %d tokens, a tree of %d", tokens, tree->nodes);
    }
    xqhip::KvPrepLaunch p{};
    p.q_src = q_src;
    p.k_src = k_src;
    p.v_src = v_src;
    p.gated = gated != 0;
    p.nq = nq;
    p.rope_pairs = std::max(0, std::min(hd, rotary_dim)) / 2;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.eps = eps;
    p.rope_cs = rope_cs;
    p.pos0 = pos0;
    p.tokens = tokens;
    p.src_stride = src_stride;
    p.out_stride = out_stride;
    p.q_out = q_out;
    p.gate_out = gate_out;
    p.kv = cache_of(kv);
    p.has_tree = tree != nullptr;
    for (int i = 0; tree && i < tokens; ++i) p.depth[i] = static_cast<int8_t>(tree->depth[i]);
    return check(xqhip::launch_kv_prep(p, as_stream(stream)), "attn_prep_kv launch");
}

int xqhip_kv_read(const xqhip_kv* kv, int first, int count, int out_type, void* k_out, void* v_out, void* stream) {
    if (!kv || (out_type != XQHIP_F32 && out_type != XQHIP_F16)) return refuse("xqhip_kv_read: bad args");
    if (const char* f = kv_fault(kv)) return refuse("xqhip_kv_read: %s", f);
    if (kv->type != XQHIP_KV_I8) return refuse("xqhip_kv_read: an 8-bit cache");
    if (first < 0 || count < 0 || first > kv->capacity - count)
        return refuse("xqhip_kv_read: positions %d + %d of %d", first, count, kv->capacity);
    if (count == 0 || (!k_out && !v_out)) return XQHIP_OK;
    return check(xqhip::launch_kv_read({cache_of(kv), first, count, out_type == XQHIP_F16, k_out, v_out},
                                       as_stream(stream)),
                 "kv_read launch");
}

size_t xqhip_tree_attention_workspace_bytes(int nq, int nkv, int head_dim, int tokens) {
    if (tokens <= 0 || tokens > 65535 || !xqhip::tree_attn_supported(nq, nkv, head_dim)) return 0;
    return xqhip::tree_attn_workspace_bytes(nq, nkv, head_dim, tokens);
}

int xqhip_tree_attention(const float* q, const float* gate, const xqhip_kv* kv, int nq, const xqhip_tree* tree,
                         int tokens, int q_stride, const int32_t* pos0, float* out, int out_stride, void* workspace,
                         size_t workspace_bytes, void* stream) {
    if (!q || !kv || !pos0 || !out || tokens <= 0 || tokens > 65535) return refuse("xqhip_tree_attention: bad args");
    if (const char* f = kv_fault(kv)) return refuse("xqhip_tree_attention: %s", f);
    if (!xqhip::tree_attn_supported(nq, kv->nkv, kv->head_dim))
        return refuse("xqhip_tree_attention: heads (nq=%d nkv=%d hd=%d)", nq, kv->nkv, kv->head_dim);
    const int64_t width = static_cast<int64_t>(nq) * kv->head_dim;
    if (q_stride < width || out_stride < width) return refuse("xqhip_tree_attention: row strides");
    if (tree) {
        if (const char* f = tree_fault(tree)) return refuse("xqhip_tree_attention: tree: %s", f);
        if (tree->nodes != tokens) return refuse("xqhip_tree_attention: %d tokens, a tree of %d", tokens, tree->nodes);
    }
    const size_t need = xqhip::tree_attn_workspace_bytes(nq, kv->nkv, kv->head_dim, tokens);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("xqhip_tree_attention: a 16-byte aligned workspace of %zu bytes (%zu given)", need, workspace_bytes);
    xqhip::TreeAttnLaunch p{};
    p.q = q;
    p.gate = gate;
    p.kv = cache_of(kv);
    p.nq = nq;
    p.tokens = tokens;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.pos0 = pos0;
    p.out = out;
    p.ws = static_cast<float*>(workspace);
    p.has_tree = tree != nullptr;
    const uint64_t rows = tokens >= 64 ? ~uint64_t(0) : (uint64_t(1) << tokens) - 1;
    for (int i = 0; tree && i < tokens; ++i) p.masks.m[i] = tree->mask[i] & rows;
    return check(xqhip::launch_tree_attn(p, as_stream(stream)), "tree attention launch");
}

size_t xqhip_linear_attn_tree_workspace_bytes(int nodes, int lk_n, int lk_hd, int lv_n, int lv_hd) {
    if (nodes < 1 || nodes > XQHIP_TREE_MAX || !xqhip::tree_linear_supported(lk_n, lk_hd, lv_n, lv_hd, 1)) return 0;
    return xqhip::tree_linear_workspace_bytes(nodes, lk_n, lk_hd, lv_n, lv_hd);
}

int xqhip_linear_attn_tree(const float* mixed, const float* a, const float* b, int stride, const float* conv_state,
                           const int32_t* pos0, const float* conv_w, const float* a_log, const float* dt_bias,
                           const float* state, int lk_n, int lk_hd, int lv_n, int lv_hd, int ksize,
                           const xqhip_tree* tree, float* out, int out_stride, void* workspace, size_t workspace_bytes,
                           void* stream) {
    if (!mixed || !a || !b || !conv_state || !pos0 || !conv_w || !a_log || !dt_bias || !state || !tree || !out)
        return refuse("xqhip_linear_attn_tree: bad args");
    if (!xqhip::tree_linear_supported(lk_n, lk_hd, lv_n, lv_hd, ksize))
        return refuse("xqhip_linear_attn_tree: shape (lk %d x %d, lv %d x %d, ksize %d)", lk_n, lk_hd, lv_n, lv_hd, ksize);
    if (stride < 0 || out_stride < lv_n * lv_hd) return refuse("xqhip_linear_attn_tree: row strides");
    if (const char* f = tree_fault(tree)) return refuse("xqhip_linear_attn_tree: tree: %s", f);
    const size_t need = xqhip::tree_linear_workspace_bytes(tree->nodes, lk_n, lk_hd, lv_n, lv_hd);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("xqhip_linear_attn_tree: a 16-byte aligned workspace of %zu bytes (%zu given)", need,
                      workspace_bytes);
    xqhip::TreeLinearLaunch p{mixed, a, b, stride, conv_state, pos0, conv_w, a_log, dt_bias, state, lk_n, lk_hd,
                              lv_n, lv_hd, ksize, tree->nodes, out, out_stride, static_cast<float*>(workspace),
                              links_of(tree), {}, 0};
    for (int i = 0; i < tree->nodes; ++i)
        if (const int up = tree->parent[i]; up >= 0) {
            p.above.m[i] = p.above.m[up] | uint64_t(1) << up;
            p.inner |= uint64_t(1) << up;
        }
    return check(xqhip::launch_tree_linear(p, as_stream(stream)), "linear attention tree launch");
}

size_t xqhip_spec_verify_workspace_bytes(int nodes, int vocab) {
    if (nodes < 1 || nodes > XQHIP_TREE_MAX || vocab < 1 || vocab > kMaxVocab) return 0;
    return xqhip::verify_workspace_bytes(nodes, vocab);
}

int xqhip_spec_verify(const float* logits, int ld_logits, int vocab, const xqhip_tree* tree, const int32_t* tokens,
                      const float* draft, int ld_draft, float inv_temperature, const float* u_accept,
                      const float* u_sample, int32_t* out_count, int32_t* out_path, int32_t* out_tokens,
                      void* workspace, size_t workspace_bytes, void* stream) {
    if (!logits || !tree || !tokens || !out_count || !out_path || !out_tokens || vocab < 1 ||
        vocab > kMaxVocab)
        return refuse("xqhip_spec_verify: bad args");
    if (!(inv_temperature >= 0.0f && inv_temperature <= 3.0e38f))
        return refuse("xqhip_spec_verify: inverse temperature %g", inv_temperature);
    const bool sampled = inv_temperature > 0.0f;
    if (sampled && (!u_accept || !u_sample)) return refuse("xqhip_spec_verify: sampling takes random numbers");
    if (ld_logits < vocab || (sampled && draft && ld_draft < vocab)) return refuse("xqhip_spec_verify: row strides");
    if (const char* f = tree_fault(tree)) return refuse("xqhip_spec_verify: tree: %s", f);
    int children[XQHIP_TREE_MAX] = {}, most = 0;
    for (int i = 1; i < tree->nodes; ++i) {
        if (tree->parent[i] < 0) return refuse("xqhip_spec_verify: the tree has one root (row %d is another)", i);
        most = std::max(most, ++children[tree->parent[i]]);
    }
    const size_t need = xqhip::verify_workspace_bytes(tree->nodes, vocab);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("xqhip_spec_verify: a 16-byte aligned workspace of %zu bytes (%zu given)", need, workspace_bytes);
    xqhip::VerifyLaunch p{logits, ld_logits, vocab, tree->nodes, most, tokens, sampled ? draft : nullptr, ld_draft,
                          inv_temperature, u_accept, u_sample, out_count, out_path, out_tokens, workspace,
                          links_of(tree), {}};
    for (int i = 1; i < tree->nodes; ++i) p.kids[tree->parent[i]] |= uint64_t(1) << i;
    return check(xqhip::launch_verify(p, as_stream(stream)), "verify launch");
}

int xqhip_tree_keep(const xqhip_rows* sets, int n_sets, const int32_t* path, const int32_t* count, int max_rows,
                    void* stream) {
    if (n_sets < 0 || (n_sets > 0 && !sets) || !path || !count || max_rows < 1 || max_rows > XQHIP_TREE_MAX)
        return refuse("xqhip_tree_keep: bad args");
    for (int i = 0; i < n_sets; ++i) {
        if (!sets[i].base || sets[i].row_bytes == 0 || sets[i].row_bytes > uint64_t(1) << 30 || sets[i].rows < 0 ||
            sets[i].rows > int64_t(1) << 32)
            return refuse("xqhip_tree_keep: buffer %d", i);
        const auto begin = [&](int j) { return reinterpret_cast<uintptr_t>(sets[j].base); };
        const auto end = [&](int j) { return begin(j) + sets[j].row_bytes * static_cast<uint64_t>(sets[j].rows); };
        for (int j = 0; j < i; ++j)
            if (begin(i) < end(j) && begin(j) < end(i)) return refuse("xqhip_tree_keep: buffers %d and %d overlap", j, i);
    }
    for (int i0 = 0; i0 < n_sets; i0 += xqhip::kKeepSets) {
        const int n = std::min(n_sets - i0, xqhip::kKeepSets);
        xqhip::KeepLaunch p{};
        for (int i = 0; i < n; ++i)
            p.sets[i] = {static_cast<uint8_t*>(sets[i0 + i].base), sets[i0 + i].row_bytes, sets[i0 + i].rows,
                         sets[i0 + i].first};
        p.path = path;
        p.count = count;
        p.max_rows = max_rows;
        if (int rc = check(xqhip::launch_tree_keep(p, n, as_stream(stream)), "tree keep launch")) return rc;
    }
    return XQHIP_OK;
}

}  // extern "C"
