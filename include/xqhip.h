/* xqhip.h - thin C ABI between the C++ host runtime (libxqwen35.so) and the
 * hand-written gfx950 HIP kernels (libxqhip.so).
 *
 * Everything here is plain C: device pointers are `void*`, streams are `void*`
 * (a hipStream_t; NULL means the library's own stream on the current device),
 * every call returns 0 on success or a negative XQHIP_E* code, with the message
 * available from xqhip_last_error().  No torch or HIP types appear in the
 * signatures.
 *
 * This layer is the MI355X replacement of the reference's per-op GPU seam
 * (customlib/runtime/vulkan_backend.hpp:21-121, `bool op(..., timing, error)`),
 * re-designed so that weights, KV cache, recurrent state and activations stay
 * resident in HBM and no op uploads or downloads per call.  The CPU kernel each
 * entry point replaces is cited beside it.
 */
#ifndef XQHIP_H_
#define XQHIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define XQHIP_API __attribute__((visibility("default")))

enum {
    XQHIP_OK = 0,
    XQHIP_EINVAL = -1,   /* bad argument or unsupported shape */
    XQHIP_EDEVICE = -2,  /* HIP runtime error (message in xqhip_last_error) */
    XQHIP_ENOMEM = -3,
    XQHIP_ENOTSUP = -4   /* valid arguments this entry point cannot run on this
                            matrix or device (the caller uses the separate calls) */
};

/* Element types of activation vectors. */
enum { XQHIP_F32 = 0, XQHIP_F16 = 1 };

/* Epilogues fused into the GEMV store. */
enum {
    XQHIP_EPI_STORE = 0,     /* y[r] = acc                                           */
    XQHIP_EPI_ADD = 1,       /* y[r] += acc (fp32 residual add, custom_model.cpp:294) */
    XQHIP_EPI_SILU_PAIR = 2  /* rows interleaved (gate_i, up_i): y[i] = silu(g)*u    */
};

/* Device layouts of a W4A16 matrix. */
enum {
    XQHIP_LAYOUT_TILED64 = 0, /* group 64, cols % 64 == 0: 16-byte chunks of each row
                                 permuted so a wave's loads are contiguous; per-group
                                 (fp16 scale, fp16 zero) packed in one u32          */
    XQHIP_LAYOUT_GENERIC = 1, /* any group size: reference row-major nibbles, fp32
                                 scales and zeros (used only for tiny shapes)        */
    XQHIP_LAYOUT_TILED64_F32META = 2, /* TILED64 codes with the reference's fp32
                                 (scale, zero) per group (8 bytes): chosen when a
                                 value is not exact in fp16 (e.g. asymmetric scales
                                 (max - min) / 15)                                  */
    XQHIP_LAYOUT_TILED64_SCALE16 = 3, /* TILED64 codes with one fp16 scale per group
                                 (2 bytes): chosen for 4-bit format-v1 matrices whose
                                 zeros are all 8 (the symmetric quantiser, the
                                 synthetic weights) and whose scales fp16 holds; the
                                 zero point is implied                              */
    XQHIP_LAYOUT_TILED64_F32S_Z4 = 4 /* TILED64 codes with the fp32 scale and a 4-bit
                                 zero code per group (4.5 bytes: fp32 scales
                                 [rows][G], then per row ceil(G/8) u32 words, nibble
                                 k of word j = zero of group 8j+k): chosen for 4-bit
                                 format-v1 matrices whose zeros are integers 0..15
                                 and whose scales fp16 cannot hold (the reference
                                 packer's asymmetric quantiser,
                                 pack_qwen35_xq4_numpy.py:218-247)                  */
};

/* A W4A16 matrix resident in HBM.  Semantics of the reference QuantizedMatrix
 * (customlib/kernels/kernels.hpp:11-21): rows x cols unsigned 4-bit codes, even
 * column in the low nibble, one (scale, zero) per `group` columns of a row;
 * affine == 0: w = (q - zero) * scale (XQ4 version 1), affine == 1:
 * w = q * scale + zero (version 2). */
typedef struct xqhip_w4 {
    int32_t rows;
    int32_t cols;
    int32_t group;
    int32_t affine;
    int32_t layout;
    int32_t inexact_meta; /* scales/zeros fp16 cannot hold exactly: kept in fp32
                             (layouts TILED64_F32META, TILED64_F32S_Z4)          */
    int32_t bits;         /* code width: 4 (xqhip_w4_upload), 3 or 2 (xqhip_wlb_upload) */
    int32_t zero_is_8;    /* affine == 0 and every zero is 8: w = (q - 8) s, so the
                             zero-point term of the prefill GEMM vanishes          */
    void* nib;            /* device codes                                         */
    void* meta;           /* device per-group metadata                            */
    uint64_t nib_bytes;
    uint64_t meta_bytes;
} xqhip_w4;

/* ---- device, memory, streams, events ---------------------------------- */
XQHIP_API const char* xqhip_last_error(void);
XQHIP_API int xqhip_device_count(void);
XQHIP_API int xqhip_set_device(int device);
XQHIP_API int xqhip_device_name(char* out, size_t capacity);
XQHIP_API int xqhip_malloc(void** ptr, size_t bytes);
XQHIP_API int xqhip_free(void* ptr);
XQHIP_API int xqhip_memcpy_h2d(void* dst, const void* src, size_t bytes, void* stream);
XQHIP_API int xqhip_memcpy_d2h(void* dst, const void* src, size_t bytes, void* stream);
XQHIP_API int xqhip_memcpy_d2d(void* dst, const void* src, size_t bytes, void* stream);
/* Asynchronous copies (no synchronisation); host memory should be pinned. */
XQHIP_API int xqhip_memcpy_h2d_async(void* dst, const void* src, size_t bytes, void* stream);
XQHIP_API int xqhip_memcpy_d2h_async(void* dst, const void* src, size_t bytes, void* stream);
/* Pinned host memory (hipHostMalloc). */
XQHIP_API int xqhip_host_alloc(void** ptr, size_t bytes);
XQHIP_API int xqhip_host_free(void* ptr);
/* Pinned host memory that kernels may store to directly (hipHostMalloc,
 * mapped and coherent): a kernel's system-scope store reaches the host
 * without a copy on the stream. */
XQHIP_API int xqhip_host_alloc_coherent(void** ptr, size_t bytes);
/* Byte fill done by a kernel (safe inside captured graphs). */
XQHIP_API int xqhip_fill_u8(void* dst, uint8_t value, size_t bytes, void* stream);
/* Device-to-device copy as one plain kernel dispatch (graph-capturable; also
 * the known-size copy that HBM byte counters are calibrated on).  16-byte
 * aligned pointers. */
XQHIP_API int xqhip_copy(void* dst, const void* src, size_t bytes, void* stream);
XQHIP_API int xqhip_stream_synchronize(void* stream);
/* 1 once all work enqueued on `stream` has finished, 0 while some is pending,
 * a negative XQHIP_E* code on a device error.  Does not block. */
XQHIP_API int xqhip_stream_query(void* stream);
XQHIP_API int xqhip_device_synchronize(void);
XQHIP_API int xqhip_event_create(void** ev);
XQHIP_API int xqhip_event_destroy(void* ev);
XQHIP_API int xqhip_event_record(void* ev, void* stream);
/* Blocks the host until the work recorded before `ev` has finished. */
XQHIP_API int xqhip_event_synchronize(void* ev);
XQHIP_API int xqhip_event_elapsed_ms(void* start, void* stop, float* ms);
/* 1 once the work recorded before `ev` has finished, 0 while it is pending,
 * a negative XQHIP_E* code on a device error.  Does not block. */
XQHIP_API int xqhip_event_query(void* ev);

/* ---- W4A16 weights ----------------------------------------------------- */
/* Repack a reference-format matrix (packed[rows][ceil(cols/2)], fp32
 * scales/zeros[rows][ceil(cols/group)], as read by custom_model.cpp:218-262)
 * into the device layout and upload it.  group == 64 and cols % 64 == 0 give a
 * TILED64 layout, with the smallest metadata that holds every scale and zero
 * exactly: SCALE16 (format v1, zeros all 8, fp16 scales), TILED64 (fp16 scale
 * and zero), F32S_Z4 (format v1, integer zeros 0..15, fp32 scales) or
 * F32META (fp32 pair); anything else gives GENERIC. */
XQHIP_API int xqhip_w4_upload(const uint8_t* packed, const float* scales, const float* zeros, int rows, int cols,
                              int group, int affine, xqhip_w4* out);
/* 3- and 2-bit matrices (W3A16 / W2A16): the reference's low-bit format
 * (QuantizedMatrix with bits 3 or 2, kernels/kernels.hpp:11-21; packed by
 * quantizeLowBit, read by readBits / dequantizeValue, ref_gemv.cpp:10-30,
 * 38-87): one LSB-first bitstream, code of (r, c) at bit (r * cols + c) * bits,
 * no row padding; scales/zeros as for 4 bits.  Replaces the matrix side of
 * gemvW3A16Neon / gemvW2A16Neon (arm64_neon/xq_gemv_w{3,2}a16_neon.cpp:6-8);
 * the result works with xqhip_gemv_w4a16 and xqhip_gemv_w4a16_argmax (not
 * with xqhip_gemm_w4a16).  group 64 with cols % 64 == 0 gives the TILED64
 * layout (codes split into bit planes, fp16 metadata), anything else the
 * GENERIC one (the bitstream as given, fp32 metadata).  The reference's
 * per-row bias is always zero (quantizeLowBit, and no file format sets it)
 * and is not carried. */
XQHIP_API int xqhip_wlb_upload(const uint8_t* bitstream, const float* scales, const float* zeros, int rows, int cols,
                               int group, int bits, int affine, xqhip_w4* out);
XQHIP_API int xqhip_w4_free(xqhip_w4* w);
/* Bytes the GEMV must read per call for this matrix (nibbles + metadata). */
XQHIP_API uint64_t xqhip_w4_weight_bytes(const xqhip_w4* w);

/* ---- fused dequant GEMV ------------------------------------------------ */
/* Normalisation applied to the GEMV input inside the kernel prologue. */
enum {
    XQHIP_PRO_NONE = 0,
    XQHIP_PRO_RMS = 1,        /* x * inv * weight[c], inv = 1/sqrt(mean(x^2) + eps)
                                 (rmsnormReference, ref_rmsnorm.cpp:8-17)          */
    XQHIP_PRO_GATED_HEAD = 2, /* per head of head_dim values:
                                 x * inv_h * weight[c % head_dim] * silu(gate[c])
                                 (applyGatedHeadRms, custom_model.cpp:329-349)     */
    XQHIP_PRO_GATED_HEAD_ACT = 3 /* GATED_HEAD with gate[c] already holding
                                 silu(gate[c]) (as xqhip_linear_attn_step_act
                                 leaves it): the GEMV entry points only        */
};
typedef struct xqhip_prologue {
    int32_t mode;
    int32_t head_dim;     /* GATED_HEAD only                                      */
    const float* weight;  /* device: RMS [cols], GATED_HEAD [head_dim]             */
    const float* gate;    /* device: GATED_HEAD [cols]                             */
    float eps;
} xqhip_prologue;

/* y = W x, replacing gemvW4A16Neon
 * (customlib/kernels/generated/arm64_neon/xq_gemv_w4a16_neon.cpp:259-291), and
 * gemvW3A16Neon / gemvW2A16Neon for matrices from xqhip_wlb_upload.
 * x: `cols` values of x_type, optionally normalised by `pro` (NULL = none).
 * y: `rows` values of y_type (EPI_SILU_PAIR: rows/2 values).  Inputs must not
 * alias outputs. */
XQHIP_API int xqhip_gemv_w4a16(const xqhip_w4* w, const void* x, int x_type, const xqhip_prologue* pro, void* y,
                               int y_type, int epilogue, void* stream);

/* Workspace bytes xqhip_gemv_w4a16_argmax needs for a matrix of `rows` rows. */
XQHIP_API size_t xqhip_argmax_workspace_bytes(int rows);
/* Greedy lm_head: argmax_r (W x)[r] without materialising logits, ties to the
 * lowest row, replacing gemvW4A16ArgmaxNeon (xq_gemv_w4a16_neon.cpp:293-348)
 * and sampleGreedy (custom_model.cpp:1281-1338).  Every GEMV block stores its
 * best (value, row) key in the workspace, then a one-block kernel reduces them.
 * workspace: device memory of xqhip_argmax_workspace_bytes(rows), no
 * initialisation needed.  out_index / out_value: device. */
XQHIP_API int xqhip_gemv_w4a16_argmax(const xqhip_w4* w, const void* x, int x_type, const xqhip_prologue* pro,
                                      void* workspace, int32_t* out_index, float* out_value, void* stream);

/* xqhip_gemv_w4a16_argmax that also advances a device position and hands the
 * result to the host without a copy: no counterpart in the reference, whose
 * decodeOne samples on the calling thread (custom_model.cpp:1281-1356).  After
 * the argmax, the finishing kernel adds 1 to *position (device int32) and
 * stores ((uint64_t)(uint32_t)new_position << 32) | (uint32_t)index to
 * *host_slot (8-byte aligned memory from xqhip_host_alloc_coherent) in one
 * system-scope store.  A host thread polls the slot for the position it
 * expects, so sampling, the next token's position and its forward pass can be
 * one captured graph with no copies between them. */
XQHIP_API int xqhip_gemv_w4a16_argmax_publish(const xqhip_w4* w, const void* x, int x_type, const xqhip_prologue* pro,
                                              void* workspace, int32_t* out_index, float* out_value,
                                              int32_t* position, uint64_t* host_slot, void* stream);

/* xqhip_gemv_w4a16_argmax_publish whose finishing kernel also writes the
 * winner's embedding row, the next position's input: sampleGreedy followed by
 * loadEmbeddingRow (custom_model.cpp:1281-1338, 569-608) in the same two
 * launches instead of three.  embed_out[0 .. hidden) = the bf16 row
 * table[index] widened to fp32, bit for bit what xqhip_embed_bf16 writes for
 * *out_index (ids past the table wrap to index % vocab).  table: device
 * [vocab][hidden] bf16; embed_out: device, may be the buffer x points to (the
 * GEMV has finished reading x when the row is written). */
XQHIP_API int xqhip_gemv_w4a16_argmax_publish_embed(const xqhip_w4* w, const void* x, int x_type,
                                                    const xqhip_prologue* pro, void* workspace, int32_t* out_index,
                                                    float* out_value, int32_t* position, uint64_t* host_slot,
                                                    const uint16_t* table, int vocab, int hidden, float* embed_out,
                                                    void* stream);

/* xqhip_gemv_w4a16_argmax without a workspace argument and without any
 * allocation: no counterpart in the reference.  For callers that cannot
 * allocate device memory (code under HIP graph capture, serving loops or
 * harnesses that forbid hipMalloc).  The per-block keys go to a 16 KiB array
 * of the library's own device memory (one per GPU, held until the process
 * ends; any matrix size fits, the launch caps its blocks), which keeps the last
 * call's contents and needs no clearing.  Calls that overlap on one GPU (other
 * streams, other threads) race on that array: serialise them.  The array used
 * is the current device's: a non-NULL `stream` must belong to that device
 * (XQHIP_EINVAL otherwise).  Same results as xqhip_gemv_w4a16_argmax. */
XQHIP_API int xqhip_gemv_w4a16_argmax_static(const xqhip_w4* w, const void* x, int x_type, const xqhip_prologue* pro,
                                             int32_t* out_index, float* out_value, void* stream);

/* ---- decode-step ops (all device pointers; `pos` is a device int32) ----- */
/* out[hidden] = bf16 table row of *token as fp32; ids outside [0, vocab) wrap
 * to |id| % vocab (loadEmbeddingRow, custom_model.cpp:569-608). */
XQHIP_API int xqhip_embed_bf16(const uint16_t* table, int vocab, int hidden, const int32_t* token, float* out,
                               void* stream);

/* Host helper: the RoPE (cos, sin) table [max_pos][rotary_dim/2] for
 * applyRopeVector (custom_model.cpp:351-370), computed with the host libm in
 * the reference's float operation order: inv_freq = powf(theta, -2i/rd),
 * angle = pos * inv_freq, (cosf(angle), sinf(angle)).  out: host floats,
 * 2 * max_pos * (rotary_dim/2) of them. */
XQHIP_API int xqhip_rope_table(float theta, int rotary_dim, int max_pos, float* out);

/* Full-attention head preparation for position *pos: per query head, split
 * the gated q_proj output into (q, gate) (custom_model.cpp:740-753), per-head
 * RMSNorm of q and k (custom_model.cpp:301-313, weights already +1), partial
 * RoPE from rope_cs (device copy of xqhip_rope_table), then k and v appended
 * as fp16 at cache slot *pos of the [t][kv_head][head_dim] caches
 * (appendKv, custom_model.cpp:673-733).  q_out, gate_out: nq*head_dim fp32
 * (gate_out is 0 when gated == 0, matching custom_model.cpp:750-753). */
XQHIP_API int xqhip_attn_prep(const float* q_src, const float* k_src, const float* v_src, int gated, int nq, int nkv,
                              int head_dim, int rotary_dim, const float* q_norm, const float* k_norm, float eps,
                              const float* rope_cs, const int32_t* pos, float* q_out, float* gate_out, void* k_cache,
                              void* v_cache, void* stream);

/* GQA decode over the fp16 caches for context *pos + 1 (scores, softmax and
 * V reduction of custom_model.cpp:840-928) followed by the sigmoid output gate
 * (custom_model.cpp:929-951): out = softmax(q k^T / sqrt(d)) v * sigmoid(gate).
 * Two kernels: per-(kv head, 64-token chunk) partial softmax-attention into the
 * workspace, then a per-query-head merge.  max_ctx <= 16384.
 * workspace: xqhip_gqa_workspace_bytes() (sized for 16384 tokens), no
 * initialisation needed. */
XQHIP_API size_t xqhip_gqa_workspace_bytes(int nq, int nkv, int head_dim);
XQHIP_API int xqhip_gqa_decode(const float* q, const void* k_cache, const void* v_cache, const float* gate, int nq,
                               int nkv, int head_dim, int max_ctx, const int32_t* pos, float* out, void* workspace,
                               void* stream);

/* xqhip_attn_prep followed by xqhip_gqa_decode in two launches: the q/k
 * RMSNorm + RoPE, the fp16 append of the new key/value at slot *pos and the
 * gated GQA of custom_model.cpp:740-951 (the decode half of
 * CustomModel::forwardAttention).  q_src is the q_proj output ([q | gate] per
 * head when gated, gate 0 otherwise); same caches, limits and workspace as
 * xqhip_gqa_decode. */
XQHIP_API int xqhip_attn_decode(const float* q_src, const float* k_src, const float* v_src, int gated, int nq,
                                int nkv, int head_dim, int rotary_dim, const float* q_norm, const float* k_norm,
                                float eps, const float* rope_cs, const int32_t* pos, void* k_cache, void* v_cache,
                                int max_ctx, float* out, void* workspace, void* stream);
/* The same step in one launch and no workspace: one block per query head
 * reads its kv head's whole context (in passes of 1024 tokens merged with a
 * running max) and writes the gated output.  head_dim 128 only; any context
 * the caches hold.  Same cache layout, append and numerics as
 * xqhip_attn_decode; faster where the context is short (the slot kernel
 * spreads long contexts over more CUs).  Replaces the same reference code
 * (custom_model.cpp:740-951). */
XQHIP_API int xqhip_attn_decode_head(const float* q_src, const float* k_src, const float* v_src, int gated, int nq,
                                     int nkv, int head_dim, int rotary_dim, const float* q_norm, const float* k_norm,
                                     float eps, const float* rope_cs, const int32_t* pos, void* k_cache,
                                     void* v_cache, float* out, void* stream);
/* The same step with the cached context split over `splits` (1..8) blocks per
 * query head: split s takes the positions [s per, (s + 1) per), per =
 * ceil(pos / splits), the last split also the new token (appended as above).
 * Each block writes its partial (running max, exp sum, exp-weighted value
 * sums) to the workspace and counts itself on its head's counter; the block
 * completing the count merges the head's partials and writes the gated output
 * to `out` (no block waits for another, no merge kernel).  One split gives
 * xqhip_attn_decode_head's result bit for bit.  workspace:
 * xqhip_attn_split_workspace_bytes(nq) bytes, 16-byte aligned, zero-filled
 * once before the first call: partials [XQHIP_ATTN_MAX_SPLITS][nq]
 * [XQHIP_ATTN_PART_STRIDE] floats, then one counter per head 128 bytes apart;
 * every call leaves the counters at zero again, and calls that overlap on one
 * device race on them.  Replaces the same reference code as
 * xqhip_attn_decode_head (custom_model.cpp:740-951). */
#define XQHIP_ATTN_PART_STRIDE 160 /* floats per (split, head): m, l, 2 pad, o[128], pad to
                                      five 128-byte lines (no line holds two records) */
#define XQHIP_ATTN_MAX_SPLITS 8
XQHIP_API size_t xqhip_attn_split_workspace_bytes(int nq);
XQHIP_API int xqhip_attn_decode_split(const float* q_src, const float* k_src, const float* v_src, int gated, int nq,
                                      int nkv, int head_dim, int rotary_dim, const float* q_norm, const float* k_norm,
                                      float eps, const float* rope_cs, const int32_t* pos, void* k_cache,
                                      void* v_cache, int splits, void* workspace, float* out, void* stream);

/* Linear attention: conv1d + SiLU over the mixed q|k|v channels with the
 * [channels][ksize-1] history updated in place, then L2-normalised q and k
 * heads (custom_model.cpp:961-1047).  out: conv_dim fp32. */
XQHIP_API int xqhip_linear_conv(const float* mixed, float* conv_state, const float* conv_w, int lk_n, int lk_hd,
                                int lv_n, int lv_hd, int ksize, float* out, void* stream);
/* Gated delta rule per value head on the fp32 state [lv_n][lk_hd][lv_hd]
 * (custom_model.cpp:1074-1096, gatedDeltaDecodeReference ref_delta.cpp:8-41),
 * with beta = sigmoid(b), g = -exp(a_log) * softplus(a + dt_bias).
 * conv: output of xqhip_linear_conv; out: lv_n * lv_hd fp32. */
XQHIP_API int xqhip_gated_delta(const float* conv, const float* a, const float* b, const float* a_log,
                                const float* dt_bias, float* state, int lk_n, int lv_n, int lk_hd, int lv_hd,
                                float* out, void* stream);
/* One decode step of the linear-attention state update in a single kernel:
 * conv1d + SiLU with L2-normalised q/k heads (as xqhip_linear_conv) feeding the
 * gated delta rule (as xqhip_gated_delta), custom_model.cpp:961-1096.
 * conv_state holds TWO copies of the [conv_dim][ksize-1] history: copy
 * (*pos & 1) is read and copy ((*pos + 1) & 1) written, so consecutive
 * positions alternate (zero both copies to reset).  mixed: conv_dim channels
 * (q | k | v); a, b: lv_n gate inputs; out: lv_n * lv_hd. */
XQHIP_API int xqhip_linear_attn_step(const float* mixed, float* conv_state, const float* conv_w, const float* a,
                                     const float* b, const float* a_log, const float* dt_bias, float* state, int lk_n,
                                     int lk_hd, int lv_n, int lv_hd, int ksize, const int32_t* pos, float* out,
                                     void* stream);
/* The same step that also replaces `gate` (lv_n * lv_hd, the gated output
 * norm's z) by silu(gate) in place, once per step, so that the output
 * projection's XQHIP_PRO_GATED_HEAD_ACT prologue reads it instead of every one
 * of its blocks evaluating the 4096 SiLUs (custom_model.cpp:329-349). */
XQHIP_API int xqhip_linear_attn_step_act(const float* mixed, float* conv_state, const float* conv_w, const float* a,
                                         const float* b, const float* a_log, const float* dt_bias, float* state,
                                         int lk_n, int lk_hd, int lv_n, int lv_hd, int ksize, const int32_t* pos,
                                         float* out, float* gate, void* stream);

/* The linear-attention decode step and the output projection that consumes
 * it, as one launch: the same results, bit for bit, as
 *   xqhip_linear_attn_step_act(mixed, ..., pos, out, gate, stream);
 *   xqhip_prologue pro = {XQHIP_PRO_GATED_HEAD_ACT, lv_hd, norm_weight, gate, eps};
 *   xqhip_gemv_w4a16(w, out, XQHIP_F32, &pro, y, XQHIP_F32, XQHIP_EPI_ADD, stream);
 * (the step, applyGatedHeadRms, out_proj and addResidual of a linear-attention
 * layer, customlib/runtime/custom_model.cpp:1074-1135, 1179), with the
 * projection's weights requested while the step runs instead of after a
 * kernel boundary.  One 1024-thread block per CU (every block must be resident
 * at once: each waits, boundedly, for the step's output of all of them).
 * w: a 4-bit TILED64 matrix (any of its metadata forms) with lv_n * lv_hd <=
 * 4096 columns; ksize 4.  sync: xqhip_step_outproj_sync_bytes() bytes of
 * device memory, 128-byte aligned, zero-filled once before the first launch;
 * every launch leaves it zeroed, launches sharing it must be ordered (one
 * stream).  Graph-capturable.  Returns XQHIP_ENOTSUP when the matrix or the
 * device does not allow the combination (xqhip_step_outproj_supported says so
 * beforehand).  No counterpart in the reference, which runs the two ops one
 * after the other.  Measured on MI355X (9B shapes) slower than the two calls,
 * 15.9 against 11.0 us: the hand-off between CUs of different XCDs inside one
 * launch costs more than a kernel boundary. */
XQHIP_API size_t xqhip_step_outproj_sync_bytes(void);
XQHIP_API int xqhip_step_outproj_supported(const xqhip_w4* w, int lk_n, int lk_hd, int lv_n, int lv_hd, int ksize);
XQHIP_API int xqhip_linear_attn_step_outproj(const float* mixed, float* conv_state, const float* conv_w,
                                             const float* a, const float* b, const float* a_log,
                                             const float* dt_bias, float* state, int lk_n, int lk_hd, int lv_n,
                                             int lv_hd, int ksize, const int32_t* pos, float* out, float* gate,
                                             const xqhip_w4* w, const float* norm_weight, float eps, float* y,
                                             void* sync, void* stream);
/* Reads the sync block's error word (synchronous copy): 0, or nonzero after a
 * launch whose wait gave up (its results are then invalid; zero-fill the block
 * again before the next launch). */
XQHIP_API int xqhip_step_outproj_error(const void* sync, int* error);
/* y = x * inv * w (rmsnormReference, ref_rmsnorm.cpp:8-17). */
XQHIP_API int xqhip_rmsnorm(const float* x, const float* w, int n, float eps, float* y, void* stream);

/* ---- prefill: a prompt chunk of m tokens at once ------------------------- */
/* The reference prefills token by token (CustomModel::prefill,
 * custom_model.cpp:610-640, each token through runLayer :1138-1256); these run
 * the same per-token arithmetic for a chunk: the projections as GEMMs on the
 * matrix cores, attention and the linear-attention recurrence as batched
 * kernels.  Row-major [token][...] activations with explicit row strides. */

/* Workspace bytes xqhip_gemm_w4a16 needs for m tokens of `cols` columns and a
 * matrix of `rows` rows (the staged x, plus the partial products of a launch
 * whose columns are split over several blocks when it has too few blocks to
 * fill the device; a workspace sized for the largest rows of a set of
 * matrices serves them all). */
XQHIP_API size_t xqhip_gemm_workspace_bytes(int m, int cols, int rows);
/* y[t] (op)= W prologue(x[t]) for t < m: every token as xqhip_gemv_w4a16 does it
 * (same epilogues; EPI_SILU_PAIR writes rows/2 values per token), on a TILED64
 * matrix.  Per 64-column group the codes q - 8 (exact in fp16) multiply x held
 * as fp16 hi + lo halves on fp16 MFMA with fp32 accumulation, the group sum is
 * scaled by the group scale, and the zero-point term is added as the product of
 * the per-group offsets with the per-token group sums of x.  GATED_HEAD reads the gate
 * of token t at pro->gate + t * ld_gate.  workspace: 16-byte aligned, of
 * workspace_bytes >= xqhip_gemm_workspace_bytes(m, cols, rows of w) (checked:
 * XQHIP_EINVAL when smaller). */
XQHIP_API int xqhip_gemm_w4a16(const xqhip_w4* w, const float* x, int m, int ldx, const xqhip_prologue* pro,
                               int ld_gate, float* y, int ldy, int epilogue, void* workspace, size_t workspace_bytes,
                               void* stream);
/* xqhip_embed_bf16 for n tokens (device ids) into out[n][hidden]. */
XQHIP_API int xqhip_embed_bf16_batch(const uint16_t* table, int vocab, int hidden, const int32_t* tokens, int n,
                                     float* out, void* stream);
/* xqhip_attn_prep for tokens consecutive positions *pos0 .. *pos0 + tokens - 1:
 * token t reads its projections at q_src/k_src/v_src + t * src_stride and writes
 * q and gate at t * out_stride; k and v are appended at cache slot *pos0 + t. */
XQHIP_API int xqhip_attn_prep_batch(const float* q_src, const float* k_src, const float* v_src, int gated, int nq,
                                    int nkv, int head_dim, int rotary_dim, const float* q_norm, const float* k_norm,
                                    float eps, const float* rope_cs, const int32_t* pos0, int tokens, int src_stride,
                                    int out_stride, float* q_out, float* gate_out, void* k_cache, void* v_cache,
                                    void* stream);
/* Causal GQA for the chunk: token t (position *pos0 + t) attends to cache slots
 * 0 .. *pos0 + t, then the sigmoid output gate (custom_model.cpp:840-951 per
 * token).  q, gate: [tokens][q_stride]; out: [tokens][out_stride]. */
XQHIP_API int xqhip_prefill_attention(const float* q, const float* gate, const void* k_cache, const void* v_cache,
                                      int nq, int nkv, int head_dim, int tokens, int q_stride, const int32_t* pos0,
                                      float* out, int out_stride, void* stream);
/* xqhip_linear_attn_step for tokens consecutive positions pos0 .. pos0+tokens-1
 * (pos0 given on the host) in one kernel: mixed, a, b rows of token t at
 * t * stride; conv_state holds the two parity copies of xqhip_linear_attn_step
 * and is left as that step expects for position pos0 + tokens. */
XQHIP_API int xqhip_linear_attn_scan(const float* mixed, const float* a, const float* b, int stride,
                                     float* conv_state, int pos0, const float* conv_w, const float* a_log,
                                     const float* dt_bias, float* state, int lk_n, int lk_hd, int lv_n, int lv_hd,
                                     int ksize, int tokens, float* out, int out_stride, void* stream);
/* xqhip_linear_attn_scan with a workspace of xqhip_linear_scan_workspace_bytes()
 * (16-byte aligned): the conv1d + SiLU, q/k L2 norms and gates of all tokens
 * run first as one token-parallel pass; for key heads of 128 dims the state
 * recurrence then runs in 64-token chunks (the per-token update unrolled over a
 * chunk into products with a triangular solve, parallel over chunks except one
 * pass per value head and 16 columns).  Same mathematics as the per-token scan,
 * a different fp32 summation order.  No counterpart in the reference (which
 * prefills token by token, custom_model.cpp:610-640); same contract as
 * xqhip_linear_attn_scan. */
XQHIP_API size_t xqhip_linear_scan_workspace_bytes(int tokens, int lk_n, int lk_hd, int lv_n, int lv_hd);
XQHIP_API int xqhip_linear_attn_scan_ws(const float* mixed, const float* a, const float* b, int stride,
                                        float* conv_state, int pos0, const float* conv_w, const float* a_log,
                                        const float* dt_bias, float* state, int lk_n, int lk_hd, int lv_n, int lv_hd,
                                        int ksize, int tokens, float* out, int out_stride, void* workspace,
                                        void* stream);

/* ---- drafted tokens: one decode step over a tree of them ----------------- */
/* Checks several drafted tokens in one forward pass; no counterpart in the
 * reference, which decodes one token at a time (CustomModel::decodeOne,
 * custom_model.cpp:1340-1356).  A step's rows are the token sampled last (row
 * 0, the root) and drafted continuations of it: row i continues row parent[i]
 * < i and stands at position *pos0 + depth[i]; its key and value go to cache
 * slot *pos0 + i.  Full-attention layers run xqhip_attn_prep_kv and
 * xqhip_tree_attention, linear-attention layers xqhip_linear_attn_tree (the
 * state stays as it is), the lm_head's logits go to xqhip_spec_verify, and
 * xqhip_tree_keep moves the rows on the accepted path together: cache slots
 * *pos0 .. *pos0 + count - 1, and the rows over which xqhip_linear_attn_scan
 * then advances each linear-attention state (the scan takes position and count
 * as host integers: *out_count is copied back before it).  No call's outputs
 * may overlap its inputs. */
#define XQHIP_TREE_MAX 64
typedef struct xqhip_tree {
    int32_t nodes;                   /* rows, 1 .. XQHIP_TREE_MAX                  */
    int32_t parent[XQHIP_TREE_MAX];  /* -1: continues the cached context           */
    int32_t depth[XQHIP_TREE_MAX];   /* rows above it on its path                  */
    uint64_t mask[XQHIP_TREE_MAX];   /* bit j: row i's attention reads row j       */
} xqhip_tree;
/* Host helper: the tree with `nodes` rows and these parents (parent[0] = -1,
 * -1 <= parent[i] < i): depths, and masks of each row's path with the row
 * itself.  A caller may set other masks afterwards (only
 * xqhip_tree_attention reads them: a padding row with mask 0, say).  Calls
 * that take a tree copy it: it may be changed as soon as they return, and a
 * captured graph keeps the one it was captured with. */
XQHIP_API int xqhip_tree_init(const int32_t* parent, int nodes, xqhip_tree* out);

/* Key/value cache of one full-attention layer, [position][kv head][head_dim]
 * as appendKv keeps it (custom_model.cpp:673-733).
 * KV_F16: fp16 values, the caches of the entry points above.
 * KV_I8: signed 8-bit codes and one fp32 scale per position and kv head
 * ([position][kv head]): scale = max |x| / 127 over the head's values, code =
 * x / scale rounded to the nearest (ties to even), value = code * scale; half
 * the bytes.  A head with a value that is not finite gets the scale NaN and
 * reads back as NaN. */
enum { XQHIP_KV_F16 = 0, XQHIP_KV_I8 = 1 };
typedef struct xqhip_kv {
    int32_t type;
    int32_t nkv, head_dim;
    int32_t capacity;  /* positions, <= 2^20 */
    void* k;           /* device */
    void* v;
    float* k_scale;    /* KV_I8 only */
    float* v_scale;
} xqhip_kv;

/* xqhip_attn_prep_batch for a cache of either type and rows of a tree: per
 * query head (q, gate) split, q and k RMSNorm, partial RoPE at position *pos0 +
 * depth (tree == NULL: *pos0 + t), k and v written to slot *pos0 + t of `kv`
 * (custom_model.cpp:301-370, 673-753).  tokens: the tree's nodes (tree == NULL:
 * up to 65535).  rope_cs: `kv->capacity` positions of xqhip_rope_table.
 * gate_out may be NULL when gated == 0.  A token whose slot or position lies
 * outside the cache's capacity writes no cache row, and NaN as its q. */
XQHIP_API int xqhip_attn_prep_kv(const float* q_src, const float* k_src, const float* v_src, int gated, int nq,
                                 int rotary_dim, const float* q_norm, const float* k_norm, float eps,
                                 const float* rope_cs, const int32_t* pos0, const xqhip_tree* tree, int tokens,
                                 int src_stride, int out_stride, float* q_out, float* gate_out, const xqhip_kv* kv,
                                 void* stream);
/* Positions first .. first + count - 1 of a KV_I8 cache as values of out_type
 * (XQHIP_F32 or XQHIP_F16: code * scale in fp32, then rounded once), for the
 * kernels that take fp16 caches.  k_out, v_out: [count][nkv][head_dim], either
 * may be NULL. */
XQHIP_API int xqhip_kv_read(const xqhip_kv* kv, int first, int count, int out_type, void* k_out, void* v_out,
                            void* stream);

/* Attention of the rows over a cache of either type:
 *   out[t] = softmax_s(q[t] k[s] / sqrt(head_dim)) v[s] * sigmoid(gate[t])
 * over s in [0, *pos0) and the rows of the tree's mask (slot *pos0 + j for bit
 * j; tree == NULL: the rows 0 .. t of up to 65535 tokens: a prompt chunk).  A
 * row that sees nothing, or scores of minus infinity only, gives 0; what a row
 * does not see never reaches it, infinities and NaN included.  q, gate:
 * [tokens][q_stride], gate may be NULL (no gate); out: [tokens][out_stride].
 * Scores, weights and sums are held to fp32 accuracy.  The cache must hold the
 * rows: slots past its capacity are not read.  workspace: 16-byte aligned, of
 * workspace_bytes >= xqhip_tree_attention_workspace_bytes(...) for this call's
 * tokens (fewer tokens can take more: one workspace for several lengths has
 * the largest of their sizes), no initialisation; calls that can overlap need
 * one each.  Limits, with g = nq / nkv: g <= 8, head_dim <= 1024 and g * (2 *
 * head_dim + 67) <= 16384; the size is 0 for shapes and token counts that are refused.
 * Made for heads of 128 and 256 dims, q, gate and out 16-byte aligned with
 * strides that are multiples of 4.  Other calls give the same results in a
 * general form that reads each row's whole context in one block per kv head
 * (one row after 8100 positions 2 to 4 ms instead of 13 us); so does a row
 * beside which an infinity or NaN lies in an fp16 cache's values. */
XQHIP_API size_t xqhip_tree_attention_workspace_bytes(int nq, int nkv, int head_dim, int tokens);
XQHIP_API int xqhip_tree_attention(const float* q, const float* gate, const xqhip_kv* kv, int nq,
                                   const xqhip_tree* tree, int tokens, int q_stride, const int32_t* pos0, float* out,
                                   int out_stride, void* workspace, size_t workspace_bytes, void* stream);

/* The linear-attention step (xqhip_linear_attn_step) for every row of a tree,
 * each from its parent's state and convolution window, without changing
 * either: conv_state ([2][conv_dim][ksize - 1], copy *pos0 & 1 is read) and
 * state ([lv_n][lk_hd][lv_hd]) are read only.  mixed, a, b: rows at i * stride;
 * out: rows at i * out_stride, lv_n * lv_hd values (custom_model.cpp:961-1096
 * per row).  The same mathematics as a scan down each path, in another fp32
 * summation order; decays are summed in 64 bits.  workspace: 16-byte aligned,
 * of workspace_bytes >= xqhip_linear_attn_tree_workspace_bytes(...), no
 * initialisation; calls that can overlap need one each. */
XQHIP_API size_t xqhip_linear_attn_tree_workspace_bytes(int nodes, int lk_n, int lk_hd, int lv_n, int lv_hd);
XQHIP_API int xqhip_linear_attn_tree(const float* mixed, const float* a, const float* b, int stride,
                                     const float* conv_state, const int32_t* pos0, const float* conv_w,
                                     const float* a_log, const float* dt_bias, const float* state, int lk_n,
                                     int lk_hd, int lv_n, int lv_hd, int ksize, const xqhip_tree* tree, float* out,
                                     int out_stride, void* workspace, size_t workspace_bytes, void* stream);

/* Verification of the drafts: walks from row 0 to the rows the target model
 * accepts and samples the token after the last of them.
 *   logits    [nodes][ld_logits]: row i's `vocab` logits (the token after row i)
 *   tokens    [nodes]: the rows' token ids (row 0's is not read)
 *   draft     [nodes][ld_draft]: the distribution that row i's children were
 *             drawn from (sums to 1), or NULL: drafts taken without chance
 *             (looked up, greedy), as if drawn from a point mass
 *   inv_temperature  1 / T; 0: greedy (draft, u_accept, u_sample not read)
 *   u_accept  [nodes], u_sample [1]: uniform numbers in [0, 1)
 * With p = softmax(logits / T) of the current row and q its draft row, its
 * children are tried in order: child j with token x is accepted when
 * u_accept[j] * q(x) < p(x) (q(x) = 1 for a point mass); a rejection replaces p
 * by the normalised max(p - q, 0) (point mass: p without x).  When no child is
 * left the token comes from p by inverse CDF in index order: the first i with
 * p(0) + .. + p(i) > u_sample * sum.  (Should a rejection leave nothing, p
 * itself is sampled.)  Greedy: the child whose token is the row's argmax (ties
 * to the lowest index) is accepted, the last token is that argmax.  The
 * outcome is distributed as sampling from the target alone where a row's
 * children were drawn from its q independently of each other (a token may then
 * come twice; siblings that were drawn to differ, a top-k of q say, are not),
 * or, without q, chosen in any way that the random numbers here have no part
 * in.  NaN logits count as minus infinity; a row with no finite or
 * plus-infinite logit accepts nothing and samples -1.  Tokens outside [0,
 * vocab) are never accepted, and a rejected child takes q off whatever its
 * token: a padding row of a sampled step with draft probabilities continues a
 * row without drafted children whose draft row holds zeros, which changes
 * nothing.  Sums and probabilities are held in 64 bits, the exponentials to
 * 1e-11 of their value.
 * out_count: rows kept, row 0 included = new tokens, 1 .. nodes.  out_path
 * [nodes]: the kept rows, then -1.  out_tokens [nodes]: the new tokens (the
 * kept drafts', then the sampled one), then -1.  The tree has one root.
 * workspace: 16-byte aligned, of workspace_bytes >=
 * xqhip_spec_verify_workspace_bytes(...), no initialisation; calls that can
 * overlap need one each. */
XQHIP_API size_t xqhip_spec_verify_workspace_bytes(int nodes, int vocab);
XQHIP_API int xqhip_spec_verify(const float* logits, int ld_logits, int vocab, const xqhip_tree* tree,
                                const int32_t* tokens, const float* draft, int ld_draft, float inv_temperature,
                                const float* u_accept, const float* u_sample, int32_t* out_count, int32_t* out_path,
                                int32_t* out_tokens, void* workspace, size_t workspace_bytes, void* stream);

/* Moves kept rows together in n_sets buffers: in each, row
 * first + path[j] replaces row first + j for j < *count (path: strictly
 * increasing, path[j] >= j, as xqhip_spec_verify leaves it; path, count:
 * device; at most max_rows <= XQHIP_TREE_MAX rows).  first: *sets[i].first
 * (device), or 0 when that is NULL.  Buffers of one call that overlap are
 * refused.  Rows outside [0, sets[i].rows) and paths that do not increase are
 * left alone from there on. */
typedef struct xqhip_rows {
    void* base;            /* device */
    uint64_t row_bytes;
    int64_t rows;
    const int32_t* first;  /* device, or NULL */
} xqhip_rows;
XQHIP_API int xqhip_tree_keep(const xqhip_rows* sets, int n_sets, const int32_t* path, const int32_t* count,
                              int max_rows, void* stream);

/* ---- several sequences in one step: caches in pages ----------------------- */
/* Decodes and prefills several sequences at once; no counterpart in the
 * reference, whose session holds one sequence (session.cpp:304-421).  A step's
 * rows are the new tokens of its sequences, one sequence behind the other: one
 * row for a sequence that decodes, many for a prompt chunk.  Full-attention
 * layers run xqhip_attn_prep_paged and xqhip_paged_attention, the lm_head's
 * logits go to xqhip_token_logprobs where a program answers with
 * probabilities.  No call's outputs may overlap its inputs. */
#define XQHIP_STEP_SEQS 1024
typedef struct xqhip_step {
    int32_t seqs;          /* sequences, 1 .. XQHIP_STEP_SEQS                       */
    int32_t rows;          /* rows that the activations hold, 1 .. 65535            */
    int32_t max_rows;      /* most rows of one sequence, 1 .. rows; rows past it are
                              left as they were                                     */
    int32_t max_pages;     /* entries of a row of the table, max_pages * page <= 2^20 */
    const int32_t* row0;   /* device [seqs + 1], never falling: sequence s has the rows
                              row0[s] .. row0[s + 1] - 1 (none: it takes no part);
                              rows from row0[seqs] on are left as they were         */
    const int32_t* past;   /* device [seqs]: positions held before the step: row j of
                              sequence s goes to position past[s] + j (negative: its
                              rows have no position)                                */
    const int32_t* table;  /* device [seqs][max_pages]: page of the positions page * i
                              .. page * i + page - 1; entries past a sequence's
                              positions are not read                                */
    const int32_t* open;   /* device [seqs]: each sequence's open page (PAGES_I8: its
                              row of k_open and v_open, another for every sequence) */
} xqhip_step;

/* Key/value cache of one full-attention layer in pages of `page` positions, in
 * pieces of 16 bytes that are operands of the matrix cores as they lie (e = 8
 * fp16 values or 16 codes):
 *   k [pages][nkv][head_dim / e][page][e]    v [pages][nkv][page / e][head_dim][e]
 * A page may stand in several sequences' tables (a prompt they share); a step
 * writes a page for one sequence only.
 * PAGES_F16: fp16 values (rounded from fp32).
 * PAGES_I8: signed 8-bit codes of the fp16 values, with one fp32 scale per page
 * and kv head ([pages][nkv]): scale = max |x| / 127 over the page's positions
 * so far, code = 127 x / max |x| to the nearest (ties to even), value = code *
 * scale.  k_open and v_open ([opens][nkv][page][head_dim]) keep the fp16 values
 * of the page that a sequence's last append ended in: when a later position
 * raises the maximum, or a step goes on into the next page, the page's codes
 * are taken anew from them, so they do not depend on the steps that a page came
 * in.  A scale never falls while its page is filled.  A sequence may go back (a
 * smaller past[s]) within the page that its last append ended in, or to any
 * page's first position (so a step that went on into another page is not
 * repeated from where it began).
 * A row that is not held (xqhip_attn_prep_paged) changes neither codes nor
 * scale; its place in the open page becomes 0, and its position holds no value
 * that may be read once a later row of its page is held.  Such rows count among
 * a step's: it ends in the page of its last row.  A row held at a page's first
 * position begins the page; where that one is not held, the maximum that the
 * page's scale records counts on.
 * Infinities and values past fp16's range are held as fp16's largest value,
 * values that are no numbers as 0.
 * One step's appends to one open page must not overlap. */
enum { XQHIP_PAGES_F16 = 0, XQHIP_PAGES_I8 = 1 };
typedef struct xqhip_pages {
    int32_t type;
    int32_t nkv, head_dim; /* head_dim: a multiple of 16, up to 256; nkv up to 256   */
    int32_t page;          /* 32, 64 or 128                                         */
    int32_t pages;         /* of the pool                                           */
    int32_t opens;         /* PAGES_I8: open pages                                  */
    void* k;               /* device, 16-byte aligned                               */
    void* v;
    float* k_scale;        /* PAGES_I8 only, as what follows                        */
    float* v_scale;
    void* k_open;          /* fp16, 16-byte aligned                                 */
    void* v_open;
} xqhip_pages;

/* Rotation over one or several position axes: pair i (dims i and i +
 * rotary_dim / 2 of a head) is turned by the angles of row pos[axis[i]] of the
 * table, as applyRopeVector does with one position (custom_model.cpp:351-370).
 * Axes are time, height and width of an image's or video's patches, say. */
#define XQHIP_ROTARY_PAIRS 128
typedef struct xqhip_rotary {
    const float* cs;      /* device: xqhip_rope_table of `positions` positions       */
    int32_t positions;
    int32_t rotary_dim;
    int32_t axes;         /* 1 .. 4                                                  */
    uint8_t axis[XQHIP_ROTARY_PAIRS];
    const int32_t* pos;   /* device [axes][rows of the step], or NULL: each row's
                             position in its sequence on every axis                  */
} xqhip_rotary;
/* Host helper: sections[a] pairs for axis a, their sum rotary_dim / 2.
 * interleaved == 0: one axis' pairs after the other's.  interleaved != 0: pair
 * i belongs to axis a = i % axes while i < axes * sections[a], to axis 0
 * otherwise (refused where that gives other numbers of pairs). */
XQHIP_API int xqhip_rotary_init(const float* cs, int positions, int rotary_dim, const int32_t* sections, int axes,
                                int interleaved, const int32_t* pos, xqhip_rotary* out);

/* xqhip_attn_prep_batch for a step over several sequences: per query head (q,
 * gate) split, q and k RMSNorm, rotation, k and v written to their positions'
 * pages (custom_model.cpp:301-370, 673-753).  Row r reads its projections at
 * q_src/k_src/v_src + r * src_stride and writes q and gate at r * out_stride.
 * rotary == NULL: no rotation.  gate_out may be NULL when gated == 0 (else 0 is
 * written there).  The normalised and rotated key is computed in 64 bits and
 * rounded to fp32, then to fp16.  A row without a position or whose position has
 * no page (a table entry outside [0, pages), a position past the table, an open
 * page outside [0, opens)) or whose rotary positions lie outside the table writes no cache
 * row, and NaN as its q. */
XQHIP_API int xqhip_attn_prep_paged(const float* q_src, const float* k_src, const float* v_src, int gated, int nq,
                                    const float* q_norm, const float* k_norm, float eps, const xqhip_rotary* rotary,
                                    const xqhip_step* step, int src_stride, int out_stride, float* q_out,
                                    float* gate_out, const xqhip_pages* kv, void* stream);
/* The step's positions read back: row r of the outputs ([rows][nkv][head_dim] of
 * out_type, XQHIP_F32 or XQHIP_F16: code * scale in fp32, then rounded once)
 * holds the key and value of its position.  With row0 and past of a program's
 * choice this reads any positions of any sequences (to move a cache, say);
 * max_rows counts here too, `open` is not read.  k_out, v_out: either may be
 * NULL.  Rows without a page read 0. */
XQHIP_API int xqhip_paged_read(const xqhip_pages* kv, const xqhip_step* step, int out_type, void* k_out, void* v_out,
                               void* stream);

/* Attention of the step's rows over their sequences' pages, as they stand:
 *   out[r] = softmax_p(q[r] k[p] / sqrt(head_dim)) v[p] * sigmoid(gate[r])
 * row j of sequence s over the positions p = 0 .. past[s] + j.  Positions
 * without a page (as above) are not seen; a row that sees nothing, or scores of
 * minus infinity only, gives 0; what a row does not see never reaches it,
 * infinities and NaN included.  q, gate: [rows][q_stride], gate may be NULL (no
 * gate); out: [rows][out_stride].  Scores, weights and sums are held to fp32
 * accuracy.  nq / nkv <= 16.  workspace: 16-byte aligned, of workspace_bytes >=
 * xqhip_paged_attention_workspace_bytes(...) (0 for refused shapes), no
 * initialisation, one size for every step; calls that can overlap need one
 * each.  Graph-capturable: lengths, rows and tables may change between replays
 * within seqs, rows, max_rows and max_pages. */
XQHIP_API size_t xqhip_paged_attention_workspace_bytes(int nq, int nkv, int head_dim);
XQHIP_API int xqhip_paged_attention(const float* q, const float* gate, const xqhip_pages* kv, int nq,
                                    const xqhip_step* step, int q_stride, float* out, int out_stride, void* workspace,
                                    size_t workspace_bytes, void* stream);

/* Log probabilities of given tokens: with p = softmax(logits * inv_temperature)
 * of a row (logits [rows][ld] of type XQHIP_F32 or XQHIP_F16, `vocab` of each),
 *   out_logprob[r]   log p(tokens[r])
 *   out_entropy[r]   - sum p log p
 *   out_rank[r]      how many tokens come before tokens[r]: a larger logit, or
 *                    the same at a lower index
 *   out_top, out_top_logprob [rows][top]: the `top` <= XQHIP_TOP_MAX first
 *                    tokens in that order and their log probabilities
 * Any output may be NULL (tokens too, when neither log probabilities of them
 * nor ranks are asked for).  The reference's only such output is the debug
 * JSON's top logits (custom_model.cpp:1281-1338).  NaN logits count as minus
 * infinity.  Plus infinities share the probability.  In a row that has nothing
 * above minus infinity every token's log probability is minus infinity, the
 * entropy 0.  Tokens of probability zero because of their logit are not listed:
 * places of out_top that are left hold -1 and minus infinity.  A token outside
 * [0, vocab) has log probability minus infinity and the rank -1.  Sums are held
 * without the maximum's own term, so log probabilities near 0 keep their
 * digits.  inv_temperature > 0.  rows <= 65535, vocab <= 2^24.  workspace:
 * 16-byte aligned, of workspace_bytes >= xqhip_token_logprobs_workspace_bytes
 * (...), no initialisation; calls that can overlap need one each. */
#define XQHIP_TOP_MAX 64
XQHIP_API size_t xqhip_token_logprobs_workspace_bytes(int rows, int vocab, int top);
XQHIP_API int xqhip_token_logprobs(const void* logits, int type, int ld, int rows, int vocab, float inv_temperature,
                                   const int32_t* tokens, int top, float* out_logprob, float* out_entropy,
                                   int32_t* out_rank, int32_t* out_top, float* out_top_logprob, void* workspace,
                                   size_t workspace_bytes, void* stream);

/* One kernel of one thread that stores the device's 100 MHz realtime counter
 * (s_memrealtime) to *slot with a system-scope store; slot may be device or
 * coherent host memory (xqhip_host_alloc_coherent).  Between two kernels on a
 * stream it marks the end of the first; graph-capturable.  Times the ops of
 * traced decode-step graphs (the kernel trace's per-op rows, after
 * custom_model.cpp:374-417). */
XQHIP_API int xqhip_timestamp(uint64_t* slot, void* stream);
/* Test diagnostic, no counterpart in the reference: fills the LDS of every CU
 * with `value` (blocks holding a CU's whole 160 KiB), so that a kernel
 * launched next on the same stream finds that value wherever it reads LDS it
 * has not written itself (LDS keeps its contents between kernels).  The
 * attention tests run the decode attention right after it. */
XQHIP_API int xqhip_lds_fill(float value, void* stream);

/* ---- decode chains: consecutive projections in one persistent launch --- */
/* A chain runs a sequence of decode-step GEMVs (the projections between two
 * non-GEMV ops of the reference's runLayer, customlib/runtime/custom_model.cpp
 * :1138-1256: o/out_proj -> gate/up -> down -> the next layer's input
 * projection) as one launch of one block per CU.  Each CU keeps streaming
 * weights across the op boundaries (the next op's first weights are requested
 * before the current op's output is complete), and an op reads its input
 * vector from the previous op through a hand-off arena of 8-byte records
 * (value, launch sequence number) stored write-through, polled with bounded
 * waits: no kernel boundary and no grid barrier between the ops.  Results are
 * those of xqhip_gemv_w4a16 on the same operands, bit for bit.
 *
 * Every matrix of a chain must be a 4-bit TILED64 matrix with fp16, fp32-pair
 * or fp16-scale metadata (layouts TILED64, TILED64_F32META, TILED64_SCALE16,
 * not TILED64_F32S_Z4), all in one of them; cols <= 16384. */
typedef struct xqhip_chain_src {
    const float* plain; /* a device fp32 vector complete before the launch, or */
    int32_t op;         /* (plain == NULL) the output of op `op` of the chain */
    int32_t offset;     /* first element taken from that output */
} xqhip_chain_src;

typedef struct xqhip_chain_op {
    const xqhip_w4* w;
    int32_t epi;          /* XQHIP_EPI_STORE / ADD / SILU_PAIR                  */
    int32_t pro;          /* XQHIP_PRO_NONE / RMS / GATED_HEAD_ACT              */
    const float* pro_w;   /* RMS: [cols]; GATED_HEAD_ACT: [head_dim]            */
    int32_t head_dim;     /* GATED_HEAD_ACT                                     */
    float eps;
    xqhip_chain_src x;    /* input, cols values                                */
    xqhip_chain_src gate; /* GATED_HEAD_ACT: silu(gate), cols values            */
    xqhip_chain_src res;  /* ADD: the residual added to                         */
    float* y_plain;       /* also store the output here (NULL: later ops only)  */
} xqhip_chain_op;

/* Validates the ops and uploads a device description; *chain receives an
 * opaque handle.  XQHIP_EINVAL when a matrix or shape is not supported. */
XQHIP_API int xqhip_chain_create(const xqhip_chain_op* ops, int n_ops, void** chain);
XQHIP_API int xqhip_chain_destroy(void* chain);
/* Hand-off records a launch of this chain needs (8 bytes each). */
XQHIP_API size_t xqhip_chain_arena_records(const void* chain);
/* Bytes of the synchronisation block shared by the chains of one stream
 * (zero-filled once before the first launch, then left alone). */
XQHIP_API size_t xqhip_chain_sync_bytes(void);
/* One launch: arena of at least xqhip_chain_arena_records records (zero-filled
 * once before first use), sync block as above.  Graph-capturable.  Launches
 * sharing an arena or sync block must be ordered (one stream). */
XQHIP_API int xqhip_chain_launch(const void* chain, void* arena, void* sync, void* stream);
/* The same launch recording per op and block the device's 100 MHz realtime
 * counter when the op's input is staged and when its last output is stored:
 * stamps[(op * grid + block) * 2 + {0, 1}] (uint64), grid = xqhip_chain_grid. */
XQHIP_API int xqhip_chain_launch_stamped(const void* chain, void* arena, void* sync, void* stamps, void* stream);
XQHIP_API int xqhip_chain_grid(const void* chain);
/* Reads the sync block's error word (synchronous copy): 0, or nonzero after a
 * launch whose hand-off wait gave up (its results are then invalid). */
XQHIP_API int xqhip_chain_error(const void* sync, int* error);

/* ---- streams and graphs ------------------------------------------------ */
XQHIP_API int xqhip_stream_create(void** stream);
XQHIP_API int xqhip_stream_destroy(void* stream);
XQHIP_API int xqhip_graph_begin(void* stream);
XQHIP_API int xqhip_graph_end(void* stream, void** graph_exec);
XQHIP_API int xqhip_graph_launch(void* graph_exec, void* stream);
XQHIP_API int xqhip_graph_destroy(void* graph_exec);

#ifdef __cplusplus
}
#endif

#endif /* XQHIP_H_ */
