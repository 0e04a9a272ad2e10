// paged_api.hip - entry points of a step over several sequences (declared in
// include/xqhip.h): argument checks and launch descriptions.
#include "xqhip.h"
#include "xqhip_kernels.hpp"

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
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kMaxPositions = 1 << 20, kMaxVocab = 1 << 24, kMaxRows = 65535;

bool workspace_ok(const void* ws, size_t have, size_t need) { return ws && aligned16(ws) && have >= need; }

const char* pages_fault(const xqhip_pages* kv, bool opens) {
    if (kv->type != XQHIP_PAGES_F16 && kv->type != XQHIP_PAGES_I8) return "page type";
    if (kv->nkv <= 0 || kv->nkv > 256) return "kv heads (1 to 256)";
    if (kv->head_dim <= 0 || kv->head_dim > 256 || kv->head_dim % 16) return "head_dim (a multiple of 16, up to 256)";
    if (kv->page != 32 && kv->page != 64 && kv->page != 128) return "page (32, 64 or 128 positions)";
    if (kv->pages <= 0) return "pages of the pool";
    if (!kv->k || !kv->v || !aligned16(kv->k) || !aligned16(kv->v)) return "page pointers (16-byte aligned)";
    if (kv->type == XQHIP_PAGES_I8) {
        if (!kv->k_scale || !kv->v_scale) return "page scales";
        if (opens && (kv->opens <= 0 || !kv->k_open || !kv->v_open || !aligned16(kv->k_open) || !aligned16(kv->v_open)))
            return "open pages (16-byte aligned)";
    }
    return nullptr;
}

const char* step_fault(const xqhip_step* st, const xqhip_pages* kv, bool opens) {
    if (st->seqs < 1 || st->seqs > XQHIP_STEP_SEQS) return "sequences (1 to 1024)";
    if (st->rows < 1 || st->rows > kMaxRows) return "rows (1 to 65535)";
    if (st->max_rows < 1 || st->max_rows > st->rows) return "max_rows (1 to rows)";
    if (st->max_pages < 1 || st->max_pages > kMaxPositions / kv->page) return "max_pages (up to 2^20 positions)";
    if (!st->row0 || !st->past || !st->table) return "row0, past and table";
    if (opens && kv->type == XQHIP_PAGES_I8 && !st->open) return "open pages' numbers";
    return nullptr;
}

const char* rotary_fault(const xqhip_rotary* r) {
    if (r->rotary_dim < 0 || r->rotary_dim > 2 * XQHIP_ROTARY_PAIRS || r->rotary_dim % 2) return "rotary_dim (even, up to 256)";
    if (r->rotary_dim == 0) return nullptr;
    if (!r->cs || (reinterpret_cast<uintptr_t>(r->cs) & 7u) || r->positions <= 0) return "table (8-byte aligned)";
    if (r->axes < 1 || r->axes > 4) return "axes (1 to 4)";
    for (int i = 0; i < r->rotary_dim / 2; ++i)
        if (r->axis[i] >= r->axes) return "axis of a pair";
    return nullptr;
}

xqhip::PagedCache cache_of(const xqhip_pages* kv) {
    return xqhip::PagedCache{kv->k, kv->v, kv->k_scale, kv->v_scale, static_cast<_Float16*>(kv->k_open),
                             static_cast<_Float16*>(kv->v_open), kv->type == XQHIP_PAGES_I8, kv->nkv, kv->head_dim, kv->page,
                             kv->pages, kv->opens};
}

xqhip::PagedStep step_of(const xqhip_step* st) {
    return xqhip::PagedStep{st->seqs, st->rows, st->max_rows, st->max_pages, st->row0, st->past, st->table, st->open};
}

}  // namespace

extern "C" {

int xqhip_rotary_init(const float* cs, int positions, int rotary_dim, const int32_t* sections, int axes, int interleaved,
                      const int32_t* pos, xqhip_rotary* out) {
    if (!out || !sections || axes < 1 || axes > 4 || rotary_dim < 0 || rotary_dim % 2 || rotary_dim > 2 * XQHIP_ROTARY_PAIRS)
        return refuse("xqhip_rotary_init: bad args");
    xqhip_rotary r{};
    r.cs = cs;
    r.positions = positions;
    r.rotary_dim = rotary_dim;
    r.axes = axes;
    r.pos = pos;
    const int pairs = rotary_dim / 2;
    int64_t sum = 0;
    for (int a = 0; a < axes; ++a) {
        if (sections[a] < 0) return refuse("xqhip_rotary_init: section %d", a);
        sum += sections[a];
    }
    if (sum != pairs) return refuse("xqhip_rotary_init: sections of %lld pairs, a rotation of %d", static_cast<long long>(sum), pairs);
    int count[4] = {}, a = 0, left = sections[0];
    for (int i = 0; i < pairs; ++i) {
        if (interleaved) {
            r.axis[i] = static_cast<uint8_t>(i < axes * sections[i % axes] ? i % axes : 0);
        } else {
            while (left == 0) left = sections[++a];
            --left;
            r.axis[i] = static_cast<uint8_t>(a);
        }
        ++count[r.axis[i]];
    }
    for (int b = 0; b < axes; ++b)
        if (count[b] != sections[b])
            return refuse("xqhip_rotary_init: %d interleaved pairs on axis %d, %d asked for", count[b], b, sections[b]);
    *out = r;
    if (const char* f = rotary_fault(&r)) {
        *out = xqhip_rotary{};
        return refuse("xqhip_rotary_init: %s", f);
    }
    return XQHIP_OK;
}

int xqhip_attn_prep_paged(const float* q_src, const float* k_src, const float* v_src, int gated, int nq, const float* q_norm,
                          const float* k_norm, float eps, const xqhip_rotary* rotary, const xqhip_step* step, int src_stride,
                          int out_stride, float* q_out, float* gate_out, const xqhip_pages* kv, void* stream) {
    if (!q_src || !k_src || !v_src || !q_norm || !k_norm || !step || !q_out || !kv || (gated && !gate_out) || nq <= 0 || nq > 65535)
        return refuse("xqhip_attn_prep_paged: bad args");
    if (const char* f = pages_fault(kv, true)) return refuse("xqhip_attn_prep_paged: %s", f);
    if (const char* f = step_fault(step, kv, true)) return refuse("xqhip_attn_prep_paged: %s", f);
    if (rotary) {
        if (const char* f = rotary_fault(rotary)) return refuse("xqhip_attn_prep_paged: rotation: %s", f);
        if (rotary->rotary_dim > kv->head_dim) return refuse("xqhip_attn_prep_paged: rotation: %d of %d dims", rotary->rotary_dim, kv->head_dim);
    }
    if (out_stride < static_cast<int64_t>(nq) * kv->head_dim || src_stride < 0) return refuse("xqhip_attn_prep_paged: row strides");
    xqhip::PagedPrepLaunch p{};
    p.q_src = q_src;
    p.k_src = k_src;
    p.v_src = v_src;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.q_out = q_out;
    p.gate_out = gate_out;
    p.gated = gated != 0;
    p.nq = nq;
    p.src_stride = src_stride;
    p.out_stride = out_stride;
    p.eps = eps;
    p.inv_hd = 1.0 / kv->head_dim;
    if (rotary && rotary->rotary_dim) {
        p.rot.cs = reinterpret_cast<const float2*>(rotary->cs);
        p.rot.pos = rotary->pos;
        p.rot.positions = rotary->positions;
        p.rot.pairs = rotary->rotary_dim / 2;
        p.rot.axes = rotary->axes;
        for (int i = 0; i < p.rot.pairs; ++i) {
            p.rot.axis[i / 16] |= static_cast<uint32_t>(rotary->axis[i]) << 2 * (i % 16);
            p.rot.used |= 1 << rotary->axis[i];
        }
    }
    p.step = step_of(step);
    p.kv = cache_of(kv);
    return check(xqhip::launch_paged_prep(p, as_stream(stream)), "attn_prep_paged launch");
}

int xqhip_paged_read(const xqhip_pages* kv, const xqhip_step* step, int out_type, void* k_out, void* v_out, void* stream) {
    if (!kv || !step || (out_type != XQHIP_F32 && out_type != XQHIP_F16)) return refuse("xqhip_paged_read: bad args");
    if (const char* f = pages_fault(kv, false)) return refuse("xqhip_paged_read: %s", f);
    if (const char* f = step_fault(step, kv, false)) return refuse("xqhip_paged_read: %s", f);
    if (!k_out && !v_out) return XQHIP_OK;
    return check(xqhip::launch_paged_read({cache_of(kv), step_of(step), out_type == XQHIP_F16, k_out, v_out}, as_stream(stream)),
                 "paged_read launch");
}

size_t xqhip_paged_attention_workspace_bytes(int nq, int nkv, int head_dim) {
    return xqhip::paged_attn_workspace_bytes(nq, nkv, head_dim);
}

int xqhip_paged_attention(const float* q, const float* gate, const xqhip_pages* kv, int nq, const xqhip_step* step, int q_stride,
                          float* out, int out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    if (!q || !kv || !step || !out) return refuse("xqhip_paged_attention: bad args");
    if (const char* f = pages_fault(kv, false)) return refuse("xqhip_paged_attention: %s", f);
    if (const char* f = step_fault(step, kv, false)) return refuse("xqhip_paged_attention: %s", f);
    const size_t need = xqhip::paged_attn_workspace_bytes(nq, kv->nkv, kv->head_dim);
    if (need == 0) return refuse("xqhip_paged_attention: heads (nq=%d nkv=%d)", nq, kv->nkv);
    const int64_t width = static_cast<int64_t>(nq) * kv->head_dim;
    if (q_stride < width || out_stride < width) return refuse("xqhip_paged_attention: row strides");
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("xqhip_paged_attention: a 16-byte aligned workspace of %zu bytes (%zu given)", need, workspace_bytes);
    return check(xqhip::launch_paged_attn({q, gate, cache_of(kv), step_of(step), nq, q_stride, out_stride, out,
                                           static_cast<float*>(workspace)},
                                          as_stream(stream)),
                 "paged attention launch");
}

size_t xqhip_token_logprobs_workspace_bytes(int rows, int vocab, int top) {
    if (rows < 1 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab || top < 0 || top > XQHIP_TOP_MAX) return 0;
    return xqhip::logprobs_workspace_bytes(rows, vocab, top);
}

int xqhip_token_logprobs(const void* logits, int type, int ld, int rows, int vocab, float inv_temperature, const int32_t* tokens,
                         int top, float* out_logprob, float* out_entropy, int32_t* out_rank, int32_t* out_top,
                         float* out_top_logprob, void* workspace, size_t workspace_bytes, void* stream) {
    if (!logits || (type != XQHIP_F32 && type != XQHIP_F16) || rows < 1 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab ||
        ((out_logprob || out_rank) && !tokens))
        return refuse("xqhip_token_logprobs: bad args");
    if (ld < vocab) return refuse("xqhip_token_logprobs: row stride %d of %d logits", ld, vocab);
    if (!(inv_temperature > 0.0f && inv_temperature <= 3.0e38f))
        return refuse("xqhip_token_logprobs: inverse temperature %g", inv_temperature);
    if (top < 0 || top > XQHIP_TOP_MAX) return refuse("xqhip_token_logprobs: %d alternatives (up to %d)", top, XQHIP_TOP_MAX);
    if (!out_top && !out_top_logprob) top = 0;
    if (!out_logprob && !out_entropy && !out_rank && top == 0) return XQHIP_OK;
    const size_t need = xqhip::logprobs_workspace_bytes(rows, vocab, top);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("xqhip_token_logprobs: a 16-byte aligned workspace of %zu bytes (%zu given)", need, workspace_bytes);
    return check(xqhip::launch_logprobs({logits, type == XQHIP_F16, ld, rows, vocab, inv_temperature, tokens, top, out_logprob,
                                         out_entropy, out_rank, out_top, out_top_logprob, workspace},
                                        as_stream(stream)),
                 "token_logprobs launch");
}

}  // extern "C"
