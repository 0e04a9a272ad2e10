// tree_attn.hip - attention of a decode step's rows (a tree of drafted tokens,
// or a prompt chunk) over an fp16 or 8-bit key/value cache.
#include <algorithm>

#include <type_traits>

#include "attn_mfma.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

constexpr int kTreeMaxGroup = 8;
constexpr int kTreeChunk = 64;

__device__ __forceinline__ int clamp_pos0(const TreeAttnLaunch& p) {
    return max(0, min(*p.pos0, p.kv.capacity));
}

constexpr size_t tree_row_lds(int group, int hd) {
    return 2 * static_cast<size_t>(group) * hd + static_cast<size_t>(group) * (kTreeChunk + 3);
}

// ---------------------------------------------------------------------------
// One row t and the `group` query heads of kv head kh, for any head size: the
// context in 64-key chunks with a running max and sum (rescaled by exp(m_old -
// m_new)), then the drafted rows as one chunk more under their mask.  Every
// key that the row does not see is passed over, so nothing in it can reach the
// row; a chunk without a score above minus infinity leaves the sums as they are.
// ---------------------------------------------------------------------------
template <int THREADS, bool I8>
__device__ void attend_row(const TreeAttnLaunch& p, int t, int kh, float* smem) {
    static_assert(THREADS >= 4 * kTreeChunk, "four threads per key");
    const int hd = p.kv.head_dim, nkv = p.kv.nkv, group = p.nq / nkv;
    const int pos0 = clamp_pos0(p);
    const int rows = min(p.has_tree ? p.tokens : t + 1, p.kv.capacity - pos0);
    float* qs = smem;                       // [group][hd]
    float* sc = qs + group * hd;            // [group][64]
    float* osum = sc + group * kTreeChunk;  // [group][hd] running output
    float* ml = osum + group * hd;          // [group][2] running max, sum
    float* fac = ml + 2 * group;            // [group] rescale of this chunk
    const size_t head = static_cast<size_t>(kh) * group * hd;
    const float* qrow = p.q + static_cast<size_t>(t) * p.q_stride + head;
    for (int i = threadIdx.x; i < group * hd; i += THREADS) {
        qs[i] = qrow[i];
        osum[i] = 0.0f;
    }
    if (threadIdx.x < group) {
        ml[2 * threadIdx.x] = -INFINITY;
        ml[2 * threadIdx.x + 1] = 0.0f;
    }
    __syncthreads();
    const float rscale = 1.0f / sqrtf(static_cast<float>(hd));
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    const _Float16* kf = static_cast<const _Float16*>(p.kv.k);
    const _Float16* vf = static_cast<const _Float16*>(p.kv.v);
    const int8_t* kc = static_cast<const int8_t*>(p.kv.k);
    const int8_t* vc = static_cast<const int8_t*>(p.kv.v);
    // chunks of the context, then those of the drafted rows (a tree's fit one)
    const int before = (pos0 + kTreeChunk - 1) / kTreeChunk, after = (rows + kTreeChunk - 1) / kTreeChunk;
    for (int c = 0; c < before + after; ++c) {
        const int c0 = c < before ? c * kTreeChunk : pos0 + (c - before) * kTreeChunk;
        const int n = min(kTreeChunk, (c < before ? pos0 : pos0 + rows) - c0);
        uint64_t see = n == 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
        if (c >= before && p.has_tree) see &= p.masks.m[t];
        if (!see) continue;  // block-uniform
        {
            const int sub = threadIdx.x & 3, tt = threadIdx.x >> 2;
            const int dq = (hd + 3) / 4, d0 = sub * dq, d1 = min(hd, d0 + dq);
            const bool valid = tt < kTreeChunk && (see >> (tt & 63) & 1);
            const size_t row = static_cast<size_t>(c0 + (valid ? tt : 0)) * nkv + kh;
            const float ks = I8 ? p.kv.k_scale[row] : 1.0f;
            for (int g = 0; g < group; ++g) {
                float dot = 0.0f;
                if (valid)
                    for (int d = d0; d < d1; ++d)
                        dot += qs[g * hd + d] * (I8 ? static_cast<float>(kc[row * hd + d]) : static_cast<float>(kf[row * hd + d]));
                dot = lanes_sum<4>(dot);
                if (valid && sub == 0) sc[g * kTreeChunk + tt] = dot * ks * rscale;
            }
        }
        __syncthreads();
        for (int g = wid; g < group; g += THREADS / kWave) {
            const bool on = see >> lane & 1;
            const float sv = on ? sc[g * kTreeChunk + lane] : -INFINITY;
            const bool nan = __builtin_amdgcn_ballot_w64(sv != sv) != 0;
            const float m_old = ml[2 * g];
            const float m_new = nan ? __builtin_nanf("") : fmaxf(m_old, wave_max(sv));
            const float e = sv == -INFINITY ? 0.0f : expf(sv - m_new);
            const float lsum = wave_sum(e);
            sc[g * kTreeChunk + lane] = e;
            if (lane == 0) {
                const float f = m_old == -INFINITY ? 0.0f : expf(m_old - m_new);
                fac[g] = f;
                ml[2 * g] = m_new;
                ml[2 * g + 1] = ml[2 * g + 1] * f + lsum;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < group * hd; i += THREADS) {
            const int g = i / hd, d = i % hd;
            float o = osum[i] * fac[g];
            for (int j = 0; j < n; ++j) {
                if (!(see >> j & 1)) continue;
                const float w = sc[g * kTreeChunk + j];
                const size_t row = static_cast<size_t>(c0 + j) * nkv + kh;
                o += I8 ? w * p.kv.v_scale[row] * static_cast<float>(vc[row * hd + d]) : w * static_cast<float>(vf[row * hd + d]);
            }
            osum[i] = o;
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < group * hd; i += THREADS) {
        const float l = ml[2 * (i / hd) + 1];
        const float r = l == 0.0f ? 0.0f : osum[i] / l;
        const float gate = p.gate ? sigmoid_dev(p.gate[static_cast<size_t>(t) * p.q_stride + head + i]) : 1.0f;
        p.out[static_cast<size_t>(t) * p.out_stride + head + i] = r * gate;
    }
}

template <bool I8>
__global__ void __launch_bounds__(256) tree_attn_row_kernel(TreeAttnLaunch p) {
    extern __shared__ float smem[];
    attend_row<256, I8>(p, blockIdx.x, blockIdx.y, smem);
}

// ---------------------------------------------------------------------------
// Matrix-core forms, heads of 128 and 256 dims.  A block takes some columns of
// one kv head and one split of its keys, a column being one (row, query head)
// pair: column c of C is head c / T of the kv head's `group` and row t0 + c % T,
// T = C / group.  Its waves share the keys in 32-key tiles, each with its own
// running max, sum and output, joined through LDS at the end.  An 8-bit cache's
// codes become fp16 integers, exactly, and its scales enter as factors of the
// scores and of the weights.
//
// Scores are formed transposed, S^T = K Q^T (keys are the MFMA rows): lane l
// holds column l & 31 and the keys 8 (v / 4) + 4 (l >> 5) + v % 4 of its tile,
// so its weights are already the B operand of O^T = V^T P^T.  V stays
// [key][dim]; ds_read_tr16_b64 hands each lane four keys of its dim.
//
// Precision: q (scaled per column by a power of two to [2^12, 2^13)) and the
// weights (times 2^6) are split into fp16 hi + lo, 22 bits together; fp32
// accumulation.  One fp16 each would leave errors of 2^-12 of the weights, where
// the caches' own values are exact.  The exponents' reference m is a column's
// largest score so far, or up to 2^6 less; over an 8-bit cache the largest of
// score + log2 of V's scale, since the weights carry V's scales and must stay in
// fp16's range: the output is off by 2^-22 of the largest weight times |v|.
//
// A masked key has weight 0, but 0 times an infinity is not 0, and neither hi +
// lo nor the finite start of the running max can carry infinities.  Where that
// happens a sum is not finite or the weights sum to 0: the block that writes
// such an output computes its rows again by attend_row.
//
// Times here and below are of whole calls, one behind the other in a graph, with
// 32 / 8 heads of 128 dims where nothing else is said.
//
// tree_attn_narrow_kernel: calls of up to 16 or 32 columns (a decode step's few
//   rows).  What bounds it: the cache's bytes in long contexts (one row after
//   120000 positions of an 8-bit cache: 253 MB in 56 us, 4.5 TB/s), a chain of a
//   launch's latencies in short ones (4 rows at position 0: 7.5 us).
// tree_attn_wide_kernel: 64 columns, or 128.  What bounds it: the two products'
//   two passes each and, beside them, the weights' exponentials and splits, which
//   issue in turn with the MFMAs (46 and 49 % of the time; a tree of 64 rows after
//   131000 positions of an 8-bit cache: 2.75e11 operations in the two passes,
//   285 to 291 us, 0.95 PFLOP/s; 500 rows after 3584 81 us, of an fp16
//   cache 70: converting the codes is the difference).  A wave with two column
//   tiles of its own read K and V half as often and, when it was tried, was slower
//   below 100000 positions: twice the registers, half the waves.
// ---------------------------------------------------------------------------
constexpr int kTreeMaxSplits = 64;
// A narrow call's splits hold two tiles or more: 8 rows of 16 / 4 heads of 256 dims after 540 positions 12.8 us (one tile
// 13.5, four 14.7), after 2000 15.1 (17.7, 15.6); a wave each of one block, where that is all, needs no join.
constexpr int kMinTiles = 2;

// Columns, waves and output rows of a block: CT column tiles x KS key waves.
template <int HD, int CT, int KS, int COLS>
struct TreeBlock {
    static constexpr int kThreads = kWave * CT * KS;
    static constexpr int kCols = COLS, kKeys = kTTile * KS;
    static constexpr int kLdo = HD + 4;                   // floats per column of a wave's output
    static constexpr int kQuads = HD / 4;                 // float4 of an output row
    static constexpr int kMergeCols = kThreads / kQuads;  // columns per pass of the merge
    static constexpr int kPasses = kCols / kMergeCols;
    static constexpr size_t kOutBytes = static_cast<size_t>(kCols) * (KS * (kLdo + 3) + 1) * 4;
    static constexpr int kLdv = HD + 16;  // halves per V row: the 4 rows of a transposed read in distinct banks
    static_assert(kPasses * kThreads == kCols * kQuads, "merge");
    static_assert(kOutBytes >= tree_row_lds(kTreeMaxGroup, HD) * 4, "the general form runs in it");
};

// bits b .. b + 31 of a row's mask, with the context (negative positions) visible
__device__ __forceinline__ uint32_t mask_window(uint64_t m, int b) {
    if (b <= -32) return ~0u;
    if (b < 0) return static_cast<uint32_t>(m) << -b | ((1u << -b) - 1u);
    return b < 64 ? static_cast<uint32_t>(m >> b) : 0u;
}

struct TreeGrid {
    int tiles, splits;  // row tiles, key splits
};

// pieces [begin, end) of split s of n
__device__ __forceinline__ void split_range(int pieces, int n, int s, int& begin, int& end) {
    const int per = pieces / n, more = pieces - per * n;
    begin = s * per + min(s, more);
    end = s < n ? begin + per + (s < more ? 1 : 0) : begin;
}

template <int HD, bool I8, int CT, int KS>
struct WideTile : TreeBlock<HD, CT, KS, kTTile * CT> {
    using B = TreeBlock<HD, CT, KS, kTTile * CT>;
    static constexpr int kLdk = HD + 8;             // halves per K row: 16-byte rows shifted by 4 banks
    static constexpr int kPieceDims = I8 ? 16 : 8;  // values of a 16-byte piece
    static constexpr int kRowPieces = HD / kPieceDims;
    static constexpr int kPieces = B::kKeys * kRowPieces / B::kThreads;  // pieces of K (or V) per thread and chunk
    static constexpr int kKeyStep = B::kThreads / kRowPieces;
    static constexpr int kScales = I8 ? 3 * B::kKeys : 0;
    static constexpr size_t kKvBytes = 2 * (static_cast<size_t>(B::kKeys) * (kLdk + B::kLdv) * 2 + kScales * 4);
    static constexpr size_t kLds = kKvBytes > B::kOutBytes ? kKvBytes : B::kOutBytes;
    static_assert(kPieces * B::kThreads == B::kKeys * kRowPieces && kPieces > 0, "K / V staging");
    static_assert(!I8 || 2 * B::kKeys <= B::kThreads, "one scale per thread");
    static_assert(kLds + 64 <= 160 * 1024, "LDS");
    static_assert(QueryStage<B, HD>::kBytes <= kLds, "q fits");
    // splits that hold keys, of `splits`: whole chunks
    static __host__ __device__ __forceinline__ int used_splits(int last, int splits) {
        return last / B::kKeys + 1 < splits ? last / B::kKeys + 1 : splits;
    }
};

template <int HD, bool I8, int KS, int COLS>
struct NarrowTile : TreeBlock<HD, 1, KS, COLS> {
    using B = TreeBlock<HD, 1, KS, COLS>;
    static constexpr int kPieces = HD / (I8 ? 32 : 16);     // 16-byte pieces of K (or V) per lane and tile
    static constexpr int kRowPieces = HD / (I8 ? 16 : 8);   // ... of a row
    static constexpr int kScales = I8 ? 3 * kTTile : 0;     // floats per wave
    static constexpr size_t kWaveBytes = static_cast<size_t>(kTTile) * B::kLdv * 2 + kScales * 4;
    static constexpr size_t kKvBytes = KS * kWaveBytes + QueryStage<B, HD>::kBytes;
    static constexpr size_t kLds = kKvBytes > B::kOutBytes ? kKvBytes : B::kOutBytes;
    static_assert(kWave % kRowPieces == 0 && kWaveBytes % 16 == 0, "V staging");
    // splits that hold keys, of `splits`: one while each of its waves has one tile at most
    static __host__ __device__ __forceinline__ int used_splits(int last, int splits) {
        const int tiles = last / kTTile + 1, n = (tiles + kMinTiles - 1) / kMinTiles;
        return tiles <= KS ? 1 : n < splits ? n : splits;
    }
    static_assert(kLds + 64 <= 160 * 1024, "LDS");
};

// The key waves of a block's columns joined, then written: the partial output of one split of several, or the output.
template <typename F, bool I8, int CT, int KS, bool HALF, int N>
__device__ __forceinline__ void finish_columns(const TreeAttnLaunch& p, const TreeGrid& grid, bool whole, int waves, int sp, int kh, int t0,
                                               int ntok, int T, uint32_t inv_t, bool live, const floatx16 (&o)[N], float m, float l,
                                               void* lds, int* redo) {
    constexpr int HD = 32 * N;
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, cl = lane & 31, g = lane >> 5;
    const int group = p.nq / p.kv.nkv;
    float* Ol = static_cast<float*>(lds);          // [waves][columns][kLdo]: column c of key wave s is s kCols + c
    float* Ml = Ol + KS * F::kCols * F::kLdo;      // [waves][columns][2]
    const __amdgpu_buffer_rsrc_t rg = buf_rsrc(p.gate ? p.gate + static_cast<size_t>(t0) * p.q_stride : p.q,
                                               p.gate ? static_cast<uint32_t>(ntok) * p.q_stride * 4u : 0u);
    u32x4 gt[F::kPasses];
    if (whole)
#pragma unroll
        for (int u = 0; u < F::kPasses; ++u) {
            const int c = threadIdx.x / F::kQuads + u * F::kMergeCols, hc = static_cast<int>(c * inv_t >> 16), tc = c - hc * T;
            const uint32_t at = tc * p.q_stride + (kh * group + hc) * HD + 4 * (threadIdx.x % F::kQuads);
            gt[u] = __builtin_amdgcn_raw_buffer_load_b128(rg, hc < group && tc < ntok ? at * 4u : kBufOOB, 0, 0);
        }
    l = xor_pair_sum<32>(l);
    if constexpr (HALF) l = xor_pair_sum<16>(l);
    const int cw = HALF ? cl & 15 : cl, part = HALF ? cl >> 4 : 0;
    if (live && wid / CT < waves) {
        const int at = wid * (F::kCols / CT) + cw;
        float* oc = Ol + at * F::kLdo + 4 * g + 16 * part;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int a = 0; a < (HALF ? 2 : 4); ++a) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = HALF ? rows_sum(o[j][4 * a + e], o[j][(8 + 4 * a + e) % 16]) : o[j][4 * a + e];
                *reinterpret_cast<float4*>(oc + 32 * j + 8 * a) = make_float4(v[0], v[1], v[2], v[3]);
            }
        if (g == 0 && part == 0) *reinterpret_cast<float2*>(Ml + at * 2) = make_float2(m, l);
    }
    __syncthreads();
    // a thread per column: the factors of its waves' outputs, and their sum
    float* Fl = Ml + KS * F::kCols * 2;  // [waves][columns]
    float* Ll = Fl + KS * F::kCols;      // [columns] the sums
    auto row_of = [&](int c, int& hc, int& tc) {
        hc = static_cast<int>(c * inv_t >> 16);
        tc = c - hc * T;
        return hc < group && tc < ntok;
    };
    if (threadIdx.x < F::kCols) {
        const int c = threadIdx.x;
        float M = -INFINITY, L = 0.0f;
        for (int s = 0; s < waves; ++s) M = fmaxf(M, Ml[(c + s * F::kCols) * 2]);
        for (int s = 0; s < waves; ++s) {
            const float f = __builtin_amdgcn_exp2f(Ml[(c + s * F::kCols) * 2] - M);
            L += f * Ml[(c + s * F::kCols) * 2 + 1];
            Fl[c + s * F::kCols] = f;
        }
        Ll[c] = L;
        int hc, tc;
        if (!whole && row_of(c, hc, tc)) {
            float2* pm = reinterpret_cast<float2*>(p.ws + static_cast<size_t>(grid.splits) * p.tokens * p.nq * HD) +
                         static_cast<size_t>(sp) * p.tokens * p.nq;
            pm[static_cast<size_t>(t0 + tc) * p.nq + kh * group + hc] = make_float2(M, L);
        }
    }
    __syncthreads();
    const int c0 = threadIdx.x / F::kQuads, d = 4 * (threadIdx.x % F::kQuads);
    float4 r[F::kPasses] = {};
    for (int s = 0; s < waves; ++s)
#pragma unroll
        for (int u = 0; u < F::kPasses; ++u) {
            const int c = c0 + u * F::kMergeCols + s * F::kCols;
            add_scaled(r[u], Fl[c], *reinterpret_cast<const float4*>(Ol + c * F::kLdo + d));
        }
    float* po = p.ws + static_cast<size_t>(sp) * p.tokens * p.nq * HD;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < F::kPasses; ++u) {
        int hc, tc;
        if (!row_of(c0 + u * F::kMergeCols, hc, tc)) continue;
        if (!whole) {
            const size_t row = static_cast<size_t>(t0 + tc) * p.nq + kh * group + hc;
            *reinterpret_cast<float4*>(po + row * HD + d) = r[u];
            continue;
        }
        bad |= write_quad(r[u], Ll[c0 + u * F::kMergeCols], p.gate, as_float4(gt[u]),
                          p.out + static_cast<size_t>(t0 + tc) * p.out_stride + (kh * group + hc) * HD + d);
    }
    if (!whole) return;
    if (bad) *redo = 1;
    __syncthreads();
    if (__builtin_expect(!*redo, 1)) return;  // block-uniform
    for (int t = t0; t < t0 + ntok; ++t) {
        __syncthreads();
        attend_row<F::kThreads, I8>(p, t, kh, static_cast<float*>(lds));
    }
}

// One column tile, and no barrier before the waves join.  Each wave takes its own 32-key tiles: K straight into registers
// as the A operand (16-byte pieces; the order of the dims within a step is free as long as q's is the same), V through
// the wave's own LDS, the next tile's K and V on their way meanwhile.
// HALF: up to 16 columns, q's hi parts in the tile's first 16 columns and its lo parts in the others.  One MFMA then does
// what two do, a lane and its neighbour 16 lanes on add their scores and take eight keys each, and the weights' hi and lo
// parts go back into the two halves.  One row after 8100 positions 11.7 us, in 32 columns 13.3.
template <int HD, bool I8, int KS, bool HALF>
__global__ void __launch_bounds__(kWave* KS, (KS + 3) / 4) tree_attn_narrow_kernel(TreeAttnLaunch p, TreeGrid grid) {
    using F = NarrowTile<HD, I8, KS, HALF ? 16 : 32>;
    using Q = QueryStage<typename F::B, HD>;
    constexpr int kSteps = HD / 16, kDimTiles = HD / 32, kSlots = HALF ? 8 : 16;
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    extern __shared__ uint4 flash_lds[];
    __shared__ int redo;
    const int nkv = p.kv.nkv, kh = blockIdx.x % nkv, sp = static_cast<int>(blockIdx.x) / nkv;
    const int group = p.nq / nkv, T = F::kCols / group, ntok = p.tokens;
    const int lane = threadIdx.x & (kWave - 1), ks = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int cl = lane & 31, g = lane >> 5;
    const uint32_t inv_t = (65535u + T) / T;
    const int col = HALF ? cl & 15 : cl, part = HALF ? cl >> 4 : 0;
    const int ch = static_cast<int>(col * inv_t >> 16), ctok = col - ch * T;
    const bool live = ch < group && ctok < ntok;
    if (threadIdx.x == 0) redo = 0;
    Q query;
    query.load(p.q, p.q_stride, kh, ntok, group, T, inv_t);
    const int pos0 = __builtin_amdgcn_readfirstlane(clamp_pos0(p));
    const int last = min(pos0 + ntok, p.kv.capacity) - 1;
    const int sure = min(p.has_tree ? pos0 - 1 : pos0, last);  // every column sees the keys up to here
    const int qpos = live ? pos0 + ctok : -1;
    const uint64_t mask = live && p.has_tree ? p.masks.m[ctok] : 0;
    int begin, end;
    const int splits = F::used_splits(last, grid.splits);
    split_range(last / kTTile + 1, splits, sp, begin, end);  // tiles
    begin = __builtin_amdgcn_readfirstlane(begin);
    end = __builtin_amdgcn_readfirstlane(end);
    if (begin >= end) return;  // fewer tiles than splits
    const int waves = min(KS, end - begin), first = begin + ks;

    const uint32_t es = I8 ? 1u : 2u, krow = static_cast<uint32_t>(nkv) * HD * es;  // bytes per cache position
    u32x4 kr[F::kPieces], vr[F::kPieces];
    const float *k_scale = p.kv.k_scale, *v_scale = p.kv.v_scale;
    asm("" : "+s"(k_scale), "+s"(v_scale));  // (else each lane fetches its pointer from the arguments, chunk by chunk)
    const uint32_t kat = cl * krow + 16u * g, vat = lane / F::kRowPieces * krow + lane % F::kRowPieces * 16u;
    auto rows_of = [&](const void* cache, int tile) {  // keys past `last`, tiles past `end` read 0
        const int key0 = tile * kTTile;
        const int n = __builtin_amdgcn_readfirstlane(tile < end ? max(0, min(kTTile, last - key0 + 1)) : 0);
        const uint8_t* base = static_cast<const uint8_t*>(cache) +
                              static_cast<size_t>(__builtin_amdgcn_readfirstlane(min(key0, last))) * krow +
                              static_cast<uint32_t>(kh) * HD * es;
        return buf_rsrc(base, static_cast<uint32_t>(n) * krow);
    };
    const float* scales = I8 && g ? v_scale : k_scale;  // lanes 0 - 31 hold K's of key cl, 32 - 63 V's
    float sr = 0.0f;
    auto load_k = [&](int tile) {
        const __amdgpu_buffer_rsrc_t rs = rows_of(p.kv.k, tile);
#pragma unroll
        for (int u = 0; u < F::kPieces; ++u) kr[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, kat + 32u * u, 0, 0);
        if constexpr (I8) {
            const int key = tile * kTTile + cl;
            sr = tile < end && key <= last ? scales[static_cast<size_t>(key) * nkv + kh] : 0.0f;
        }
    };
    auto load_v = [&](int tile) {
        const __amdgpu_buffer_rsrc_t rs = rows_of(p.kv.v, tile);
#pragma unroll
        for (int u = 0; u < F::kPieces; ++u)
            vr[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, vat + static_cast<uint32_t>(u * (kWave / F::kRowPieces)) * krow, 0, 0);
    };
    load_k(first);
    load_v(first);
    uint8_t* Ql = reinterpret_cast<uint8_t*>(flash_lds) + KS * F::kWaveBytes;
    query.store(Ql);
    __syncthreads();
    half8 qhi[HALF ? 1 : kSteps], qlo[kSteps];  // (HALF: qlo is the lane's own part, hi or lo)
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int d = I8 ? 32 * (s / 2) + 16 * g + 8 * (s % 2) : 16 * s + 8 * g;
        if constexpr (!HALF) qhi[s] = Q::part(Ql, 0, col, d);
        qlo[s] = Q::part(Ql, HALF ? part : 1, col, d);
    }
    const float sscale = Q::scale(Ql, col);
    _Float16* Vl = reinterpret_cast<_Float16*>(reinterpret_cast<uint8_t*>(flash_lds) + ks * F::kWaveBytes);  // [32][kLdv]
    float* Sl = reinterpret_cast<float*>(Vl + kTTile * F::kLdv);  // [3][32]: scales of K, of V, exponents of V's
    float m = -1.0e30f, l = 0.0f;  // reference of the exponents, this lane's part of the sum
    floatx16 o[kDimTiles];
#pragma unroll
    for (int j = 0; j < kDimTiles; ++j) o[j] = floatx16{};
    for (int tile = first; tile < end; tile += KS) {
        const int key0 = tile * kTTile;
        floatx16 st = floatx16{};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            half8 a;
            if constexpr (I8) {
                const u32x2 w0 = codes_to_half(kr[s / 2][2 * (s % 2)]), w1 = codes_to_half(kr[s / 2][2 * (s % 2) + 1]);
                a = __builtin_bit_cast(half8, u32x4{w0.x, w0.y, w1.x, w1.y});
            } else {
                a = __builtin_bit_cast(half8, kr[s]);
            }
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qlo[s], st, 0, 0, 0);
            if constexpr (!HALF) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qhi[s], st, 0, 0, 0);
        }
        if constexpr (I8) {
            Sl[lane] = sr;
            if (g) Sl[kTTile + lane] = scale_exponent(sr);
        }
        load_k(tile + KS);
#pragma unroll
        for (int u = 0; u < F::kPieces; ++u) {
            _Float16* at = Vl + (lane / F::kRowPieces + u * (kWave / F::kRowPieces)) * F::kLdv + lane % F::kRowPieces * (I8 ? 16 : 8);
            if constexpr (I8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x2 a = codes_to_half(vr[u][2 * h]), b = codes_to_half(vr[u][2 * h + 1]);
                    *reinterpret_cast<u32x4*>(at + 8 * h) = u32x4{a.x, a.y, b.x, b.y};
                }
            } else {
                *reinterpret_cast<u32x4*>(at) = vr[u];
            }
        }
        load_v(tile + KS);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // LDS takes a wave's accesses in their order
        __builtin_amdgcn_wave_barrier();
        float sc[kSlots], vs[kSlots], lv[kSlots], mc = -INFINITY;  // of keys 16 part + 8 (v / 4) + 4 g + v % 4
#pragma unroll
        for (int v = 0; v < kSlots; ++v) sc[v] = HALF ? rows_sum(st[v], st[(v + 8) % 16]) : st[v];
        if constexpr (I8) {
#pragma unroll
            for (int a = 0; a < kSlots / 4; ++a) {
                const float* at = Sl + 16 * part + 8 * a + 4 * g;
                const f32x4 k4 = *reinterpret_cast<const f32x4*>(at);
                const f32x4 v4 = *reinterpret_cast<const f32x4*>(at + kTTile);
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(at + 2 * kTTile);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[4 * a + e] *= k4[e];
                    vs[4 * a + e] = v4[e];
                    lv[4 * a + e] = l4[e];
                }
            }
        }
        if (key0 + kTTile - 1 > sure) {  // wave-uniform: keys that some column does not see
            uint32_t see;
            const int from = key0 + 16 * part + 4 * g;
            if (p.has_tree) {
                see = mask_window(mask, from - pos0);
            } else {
                const int b = qpos - from;
                see = b < 0 ? 0u : (b >= 31 ? ~0u : (2u << b) - 1u);
            }
            const int left = last - from;  // (rows and positions past the capacity)
            see &= left < 0 ? 0u : (left >= 31 ? ~0u : (2u << left) - 1u);
#pragma unroll
            for (int v = 0; v < kSlots; ++v)
                if (!(see >> (8 * (v >> 2) + (v & 3)) & 1u)) {
                    sc[v] = -INFINITY;
                    if constexpr (I8) vs[v] = 0.0f;  // (its scale may be NaN)
                }
        }
#pragma unroll
        for (int v = 0; v < kSlots; ++v) mc = fmaxf(mc, I8 ? fmaf(sc[v], sscale, lv[v]) : sc[v]);
        if constexpr (HALF) mc = xor16_max(mc);
        mc = pair32_max(mc) * (I8 ? 1.0f : sscale);
        // the reference moves only when a column's max has outgrown it (rarely after the first tiles)
        const bool up = mc > m + kSlack;
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float to = up ? mc : m, f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int j = 0; j < kDimTiles; ++j) o[j] *= f;
        }
        const float off = kRaise - m;
        half8 phi[2], plo[2];  // (HALF: plo is the lane's own part)
#pragma unroll
        for (int h = 0; h < kSlots / 8; ++h) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = __builtin_amdgcn_exp2f(fmaf(sc[8 * h + e], sscale, off));
                l += w[e];
                if constexpr (I8) {
                    w[e] *= vs[8 * h + e];
                    // the rounded product: hi and lo would else be taken from two roundings of it
                    asm("" : "+v"(w[e]));
                }
            }
            split8(w, phi[h], plo[h]);
        }
        if constexpr (HALF) {  // lanes of the hi columns give their lo for the other 8 keys' hi
            const u32x4 hi = __builtin_bit_cast(u32x4, phi[0]), lo = __builtin_bit_cast(u32x4, plo[0]);
            u32x4 w[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const auto r = __builtin_amdgcn_permlane16_swap(hi[i], lo[i], false, false);
                w[0][i] = r[0];
                w[1][i] = r[1];
            }
            plo[0] = __builtin_bit_cast(half8, w[0]);
            plo[1] = __builtin_bit_cast(half8, w[1]);
        }
        // transposed reads: 16 lanes cover four keys x 16 dims, lane i gets dim i of the four
        const _Float16* vb = Vl + (4 * g + ((lane & 15) >> 2)) * F::kLdv + (lane & 16) + 4 * (lane & 3);
#pragma unroll
        for (int j = 0; j < kDimTiles; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                typedef __attribute__((address_space(3))) short4_t lds_s4;
                const _Float16* q0 = vb + 16 * h * F::kLdv + 32 * j;
                const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q0));
                const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q0 + 8 * F::kLdv));
                const half8 a = __builtin_bit_cast(half8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, plo[h], o[j], 0, 0, 0);
                if constexpr (!HALF) o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, phi[h], o[j], 0, 0, 0);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();  // every wave is done with its V
    finish_columns<F, I8, 1, KS, HALF>(p, grid, splits == 1, waves, sp, kh, 0, ntok, T, inv_t, live, o, m, l, flash_lds, &redo);
}

// CT column tiles x KS key waves.  K and V are staged chunk by chunk (32 KS keys, shared by the column tiles) in LDS,
// twice each: one barrier a chunk, the next chunk's loads over a whole chunk ahead, and a chunk's products with V beside
// the next one's softmax.
template <int HD, bool I8, int CT, int KS>
__global__ void __launch_bounds__(kWave* CT* KS, (CT * KS + 3) / 4) tree_attn_wide_kernel(TreeAttnLaunch p, TreeGrid grid) {
    using F = WideTile<HD, I8, CT, KS>;
    using Q = QueryStage<typename F::B, HD>;
    constexpr int kSteps = HD / 16, kDimTiles = HD / 32;
    extern __shared__ uint4 flash_lds[];
    __shared__ int redo;
    constexpr int kKBuf = F::kKeys * F::kLdk, kVBuf = F::kKeys * F::kLdv, kSBuf = F::kScales;
    _Float16* Kl = reinterpret_cast<_Float16*>(flash_lds);       // [2][kKeys][kLdk]
    _Float16* Vl = Kl + 2 * kKBuf;                               // [2][kKeys][kLdv]
    float* Sl = reinterpret_cast<float*>(Vl + 2 * kVBuf);        // [2][3][kKeys]: scales of K, of V, exponents of V's
    const int nkv = p.kv.nkv, kh = blockIdx.x % nkv;
    const int rest = static_cast<int>(blockIdx.x) / nkv, tile = grid.tiles - 1 - rest % grid.tiles, sp = rest / grid.tiles;
    const int group = p.nq / nkv, T = F::kCols / group;
    const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int ct = wid % CT, ks = wid / CT;
    const int cl = lane & 31, g = lane >> 5;
    const uint32_t inv_t = (65535u + T) / T;  // c / T = c inv_t >> 16 for c < 128, T <= 128
    const int t0 = tile * T, ntok = min(T, p.tokens - t0);
    Q query;
    query.load(p.q + static_cast<size_t>(t0) * p.q_stride, p.q_stride, kh, ntok, group, T, inv_t);
    const int pos0 = __builtin_amdgcn_readfirstlane(clamp_pos0(p));
    const int col = ct * kTTile + cl, ch = static_cast<int>(col * inv_t >> 16), ctok = col - ch * T;
    const bool live = ch < group && ctok < ntok;
    const int last = min(pos0 + (p.has_tree ? p.tokens : t0 + ntok), p.kv.capacity) - 1;  // any column's last key
    const int sure = min(p.has_tree ? pos0 - 1 : pos0 + t0, last);  // every column sees the keys up to here
    const int qpos = live ? pos0 + t0 + ctok : -1;
    const uint64_t mask = live && p.has_tree ? p.masks.m[t0 + ctok] : 0;
    int begin, end;
    const int splits = F::used_splits(last, grid.splits);
    split_range(last / F::kKeys + 1, splits, sp, begin, end);
    begin = __builtin_amdgcn_readfirstlane(begin);
    end = __builtin_amdgcn_readfirstlane(end);
    if (begin >= end) return;

    const uint32_t es = I8 ? 1u : 2u, krow = static_cast<uint32_t>(nkv) * HD * es;  // bytes per cache position
    const int pk = threadIdx.x / F::kRowPieces, pd = threadIdx.x % F::kRowPieces;
    u32x4 kr[F::kPieces], vr[F::kPieces];
    auto load = [&](const void* cache, int c, u32x4 (&r)[F::kPieces]) {  // keys past `last` read 0
        const int c0 = c * F::kKeys;
        const int n = __builtin_amdgcn_readfirstlane(max(0, min(F::kKeys, last - c0 + 1)));
        const uint8_t* base = static_cast<const uint8_t*>(cache) +
                              static_cast<size_t>(__builtin_amdgcn_readfirstlane(max(0, min(c0, last)))) * krow +
                              static_cast<uint32_t>(kh) * HD * es;
        const __amdgpu_buffer_rsrc_t rs = buf_rsrc(base, static_cast<uint32_t>(n) * krow);
#pragma unroll
        for (int u = 0; u < F::kPieces; ++u)
            r[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, static_cast<uint32_t>(pk + u * F::kKeyStep) * krow + pd * 16u,
                                                         0, 0);
    };
    auto store = [&](_Float16* d, int ld, const u32x4 (&r)[F::kPieces]) {
#pragma unroll
        for (int u = 0; u < F::kPieces; ++u) {
            _Float16* at = d + (pk + u * F::kKeyStep) * ld + F::kPieceDims * pd;
            if constexpr (I8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x2 a = codes_to_half(r[u][2 * h]), b = codes_to_half(r[u][2 * h + 1]);
                    *reinterpret_cast<u32x4*>(at + 8 * h) = u32x4{a.x, a.y, b.x, b.y};
                }
            } else {
                *reinterpret_cast<u32x4*>(at) = r[u];
            }
        }
    };
    // scales: thread i < kKeys holds K's of key i, the next kKeys threads V's
    const float *k_scale = p.kv.k_scale, *v_scale = p.kv.v_scale;
    asm("" : "+s"(k_scale), "+s"(v_scale));  // (else each lane fetches its pointer from the arguments, chunk by chunk)
    const float* scales = threadIdx.x < F::kKeys ? k_scale : v_scale;
    float sr = 0.0f;
    auto load_scale = [&](int c) {
        if constexpr (I8) {
            const int key = c * F::kKeys + static_cast<int>(threadIdx.x) % F::kKeys;
            sr = threadIdx.x < 2 * F::kKeys && key <= last ? scales[static_cast<size_t>(key) * nkv + kh] : 0.0f;
        }
    };
    auto store_scale = [&](int buf) {
        if constexpr (I8) {
            if (threadIdx.x >= 2 * F::kKeys) return;  // wave-uniform
            float* at = Sl + buf * kSBuf;
            at[threadIdx.x] = sr;
            if (threadIdx.x >= F::kKeys) at[F::kKeys + threadIdx.x] = scale_exponent(sr);
        }
    };
    load(p.kv.k, begin, kr);
    load_scale(begin);
    load(p.kv.v, begin, vr);
    half8 qhi[kSteps], qlo[kSteps];  // lane supplies dims 16 s + 8 g .. + 7 of its column
    query.store(flash_lds);
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        qhi[s] = Q::part(flash_lds, 0, col, 16 * s + 8 * g);
        qlo[s] = Q::part(flash_lds, 1, col, 16 * s + 8 * g);
    }
    const float sscale = Q::scale(flash_lds, col);
    __syncthreads();  // every wave has its q: K and V may take its place
    store(Kl + (begin & 1) * kKBuf, F::kLdk, kr);
    store_scale(begin & 1);
    __syncthreads();
    load(p.kv.k, begin + 1, kr);
    load_scale(begin + 1);
    float m = -1.0e30f, l = 0.0f;  // reference of the exponents, this lane's part of the sum
    floatx16 o[kDimTiles];
#pragma unroll
    for (int j = 0; j < kDimTiles; ++j) o[j] = floatx16{};
    half8 phi[2], plo[2];  // the weights of the chunk before
    auto add_values = [&](int c) {
        // transposed reads: 16 lanes cover four keys x 16 dims, lane i gets dim i of the four
        const _Float16* vb = Vl + (c & 1) * kVBuf + (ks * kTTile + 4 * g + ((lane & 15) >> 2)) * F::kLdv + (lane & 16) + 4 * (lane & 3);
#pragma unroll
        for (int j = 0; j < kDimTiles; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                typedef __attribute__((address_space(3))) short4_t lds_s4;
                const _Float16* q0 = vb + 16 * h * F::kLdv + 32 * j;
                const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q0));
                const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q0 + 8 * F::kLdv));
                const half8 a = __builtin_bit_cast(half8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, plo[h], o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, phi[h], o[j], 0, 0, 0);
            }
    };
    // One chunk: its scores, the values of the chunk before (the matrix cores work on them while the softmax runs),
    // the next keys and this chunk's values into LDS.  One barrier: both are double-buffered.
    auto chunk = [&](int c, auto first, auto masked) {
        constexpr bool FIRST = decltype(first)::value, MASKED = decltype(masked)::value;
        const int key0 = c * F::kKeys + ks * kTTile;
        floatx16 st = floatx16{};
        const _Float16* krow_l = Kl + (c & 1) * kKBuf + (ks * kTTile + cl) * F::kLdk + 8 * g;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const half8 a = *reinterpret_cast<const half8*>(krow_l + 16 * s);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qlo[s], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qhi[s], st, 0, 0, 0);
        }
        // (past `end`: loads read 0 or rows that no one asks for, into buffers that no one reads)
        store(Kl + (c + 1 & 1) * kKBuf, F::kLdk, kr);
        store_scale(c + 1 & 1);
        store(Vl + (c & 1) * kVBuf, F::kLdv, vr);
        load(p.kv.v, c + 1, vr);
        load(p.kv.k, c + 2, kr);
        load_scale(c + 2);
        if constexpr (!FIRST) add_values(c - 1);
        float sc[16], vs[16], lv[16], mc = -INFINITY;
        if constexpr (I8) {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            const float* at = Sl + (c & 1) * kSBuf;
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const f32x4 k4 = *reinterpret_cast<const f32x4*>(at + ks * kTTile + 8 * a + 4 * g);
                const f32x4 v4 = *reinterpret_cast<const f32x4*>(at + F::kKeys + ks * kTTile + 8 * a + 4 * g);
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(at + 2 * F::kKeys + ks * kTTile + 8 * a + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[4 * a + e] = st[4 * a + e] * k4[e];
                    vs[4 * a + e] = v4[e];
                    lv[4 * a + e] = l4[e];
                }
            }
        } else {
#pragma unroll
            for (int v = 0; v < 16; ++v) sc[v] = st[v];
        }
        if constexpr (MASKED) {
            uint32_t see;
            if (p.has_tree) {
                see = mask_window(mask, key0 + 4 * g - pos0);
            } else {
                const int b = qpos - (key0 + 4 * g);
                see = b < 0 ? 0u : (b >= 31 ? ~0u : (2u << b) - 1u);
            }
            const int left = last - (key0 + 4 * g);  // (rows and positions past the capacity)
            see &= left < 0 ? 0u : (left >= 31 ? ~0u : (2u << left) - 1u);
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (!(see >> (8 * (v >> 2) + (v & 3)) & 1u)) {
                    sc[v] = -INFINITY;
                    if constexpr (I8) vs[v] = 0.0f;  // (its scale may be NaN)
                }
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) mc = fmaxf(mc, I8 ? fmaf(sc[v], sscale, lv[v]) : sc[v]);
        mc = pair32_max(mc) * (I8 ? 1.0f : sscale);
        // the reference moves only when a column's max has outgrown it (rarely after the first chunks)
        const bool up = mc > m + kSlack;
        const float to = up ? mc : m, f = __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= f;
        const float off = kRaise - m;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(fmaf(sc[8 * h + e], sscale, off));
                l += x[e];
                if constexpr (I8) {
                    x[e] *= vs[8 * h + e];
                    // the rounded product: hi and lo would else be taken from two roundings of it
                    asm("" : "+v"(x[e]));
                }
            }
            split8(x, phi[h], plo[h]);
        }
        if (__builtin_amdgcn_ballot_w64(up)) {
#pragma unroll
            for (int j = 0; j < kDimTiles; ++j) o[j] *= f;
        }
        __syncthreads();  // the next keys and these values are staged; every wave is done with the buffers they replace
    };
    const int clear = min(end, max(begin, (sure + 1) / F::kKeys));  // chunks [begin, clear) that every column sees whole
    int c = begin;
    if (c < clear)
        chunk(c++, std::true_type{}, std::false_type{});
    else
        chunk(c++, std::true_type{}, std::true_type{});
    for (; c < clear; ++c) chunk(c, std::false_type{}, std::false_type{});
    for (; c < end; ++c) chunk(c, std::false_type{}, std::true_type{});
    add_values(end - 1);
    __syncthreads();
    finish_columns<F, I8, CT, KS, false>(p, grid, splits == 1, KS, sp, kh, t0, ntok, T, inv_t, live, o, m, l, flash_lds, &redo);
}

// What the merge kernels share: the keys' splits of row t, and an output quad from its sums.
constexpr int kMergeThreads = 512;
constexpr int kFewSplits = 4;
template <typename F>
__device__ __forceinline__ int used_splits(const TreeAttnLaunch& p, const TreeGrid& grid, int t, int T) {
    const int pos0 = clamp_pos0(p), t0 = t / T * T;
    return F::used_splits(min(pos0 + (p.has_tree ? p.tokens : min(t0 + T, p.tokens)), p.kv.capacity) - 1, grid.splits);
}
struct TreeParts {
    __amdgpu_buffer_rsrc_t o, st;
    uint32_t rows;  // of a split's
};
__device__ __forceinline__ TreeParts tree_parts(const TreeAttnLaunch& p, const TreeGrid& grid, int hd) {
    const uint32_t rows = static_cast<uint32_t>(p.tokens) * p.nq, all = grid.splits * rows;
    return TreeParts{buf_rsrc(p.ws, all * hd * 4u), buf_rsrc(p.ws + static_cast<size_t>(all) * hd, all * 8u), rows};
}

// The splits' partial outputs of one row and kv head joined, normalised and gated (nothing to do where one split held
// every key): 4 us, a launch and two round trips.  `slices` threads share an output's splits; their first loads go out before the position has come.
template <typename F, int HD, bool I8>
__global__ void __launch_bounds__(kMergeThreads) tree_attn_merge_kernel(TreeAttnLaunch p, TreeGrid grid, int T) {
    extern __shared__ float smem[];  // attend_row's
    __shared__ float factor[kTreeMaxGroup][kTreeMaxSplits], total[kTreeMaxGroup];
    __shared__ float4 partial[kMergeThreads];
    __shared__ int redo;
    constexpr int kBatch = 8;
    const int t = blockIdx.x, kh = blockIdx.y, group = p.nq / p.kv.nkv;
    const int items = group * (HD / 4), slices = kMergeThreads / items;  // items <= 8 * 64
    const int slice = threadIdx.x / items, item = threadIdx.x - slice * items, h = item / (HD / 4), d = 4 * (item % (HD / 4));
    const TreeParts in = tree_parts(p, grid, HD);
    const uint32_t row0 = static_cast<uint32_t>(t) * p.nq + kh * group;
    u32x4 v[kBatch];
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int s = s0 + i * slices;
            v[i] = __builtin_amdgcn_raw_buffer_load_b128(in.o, slice < slices && s < grid.splits ? ((s * in.rows + row0 + h) * HD + d) * 4u : kBufOOB, 0, 0);
        }
    };
    load(slice);  // (a split without keys holds anything)
    const int wid = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const u32x2 st = __builtin_amdgcn_raw_buffer_load_b64(in.st, wid < group && lane < grid.splits ? (lane * in.rows + row0 + wid) * 8u : kBufOOB, 0, 0);
    const size_t at = static_cast<size_t>(kh * group + h) * HD + d;
    const float4 gt = p.gate ? *reinterpret_cast<const float4*>(p.gate + static_cast<size_t>(t) * p.q_stride + at) : float4{};
    const int splits = used_splits<F>(p, grid, t, T);
    if (splits == 1) return;
    if (wid < group) {
        const float M = wave_max(lane < splits ? __uint_as_float(st.x) : -INFINITY);
        const float f = lane < splits ? __builtin_amdgcn_exp2f(__uint_as_float(st.x) - M) : 0.0f;
        const float L = wave_sum(lane < splits ? f * __uint_as_float(st.y) : 0.0f);
        factor[wid][lane] = f;
        if (lane == 0) total[wid] = L;
    }
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
    float4 r = float4{};
    if (slice < slices)
        for (int s0 = slice;;) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int s = s0 + i * slices;
                if (s < splits) add_scaled(r, factor[h][s], as_float4(v[i]));
            }
            s0 += kBatch * slices;
            if (s0 >= splits) break;
            load(s0);
        }
    partial[threadIdx.x] = r;
    __syncthreads();
    if (slice == 0) {
        for (int i = 1; i < slices; ++i) add_scaled(r, 1.0f, partial[i * items + item]);
        if (write_quad(r, total[h], p.gate, gt, p.out + static_cast<size_t>(t) * p.out_stride + at)) redo = 1;
    }
    __syncthreads();
    if (redo) attend_row<kMergeThreads, I8>(p, t, kh, smem);  // block-uniform
}

// ... of up to kFewSplits splits (calls of many rows): each thread has an output's partials by itself, a block several
// kv heads of a row.  256 rows at position 0, two splits: 16.1 us in all, with the kernel above 22.3.
template <typename F, int HD, bool I8>
__global__ void __launch_bounds__(kMergeThreads) tree_attn_merge_few_kernel(TreeAttnLaunch p, TreeGrid grid, int T) {
    extern __shared__ float smem[];  // attend_row's
    __shared__ uint32_t redo;        // a bit per kv head of the block
    const int t = blockIdx.x, group = p.nq / p.kv.nkv;
    const int items = group * (HD / 4), heads = kMergeThreads / items, k0 = blockIdx.y * heads;
    const int kl = threadIdx.x / items, item = threadIdx.x - kl * items, h = item / (HD / 4), d = 4 * (item % (HD / 4));
    const bool on = kl < heads && k0 + kl < p.kv.nkv;
    const TreeParts in = tree_parts(p, grid, HD);
    const uint32_t head = (k0 + kl) * group + h, row = static_cast<uint32_t>(t) * p.nq + head;
    u32x4 v[kFewSplits];
    u32x2 st[kFewSplits];
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        const bool has = on && s < grid.splits;
        v[s] = __builtin_amdgcn_raw_buffer_load_b128(in.o, has ? ((s * in.rows + row) * HD + d) * 4u : kBufOOB, 0, 0);
        st[s] = __builtin_amdgcn_raw_buffer_load_b64(in.st, has ? (s * in.rows + row) * 8u : kBufOOB, 0, 0);
    }
    const size_t at = static_cast<size_t>(head) * HD + d;
    const float4 gt = p.gate && on ? *reinterpret_cast<const float4*>(p.gate + static_cast<size_t>(t) * p.q_stride + at) : float4{};
    const int splits = used_splits<F>(p, grid, t, T);
    if (splits == 1) return;
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
    if (on) {
        float M = -INFINITY, L = 0.0f;
        float4 r = float4{};
#pragma unroll
        for (int s = 0; s < kFewSplits; ++s)
            if (s < splits) M = fmaxf(M, __uint_as_float(st[s].x));
#pragma unroll
        for (int s = 0; s < kFewSplits; ++s)
            if (s < splits) {
                const float f = __builtin_amdgcn_exp2f(__uint_as_float(st[s].x) - M);
                L += f * __uint_as_float(st[s].y);
                add_scaled(r, f, as_float4(v[s]));
            }
        if (write_quad(r, L, p.gate, gt, p.out + static_cast<size_t>(t) * p.out_stride + at)) atomicOr(&redo, 1u << kl);
    }
    __syncthreads();
    for (uint32_t again = redo; again; again &= again - 1) {  // block-uniform
        attend_row<kMergeThreads, I8>(p, t, k0 + __builtin_ctz(again), smem);
        __syncthreads();
    }
}

bool tree_attn_supported(int nq, int nkv, int head_dim) {
    return nkv > 0 && nq > 0 && nq % nkv == 0 && nq / nkv <= kTreeMaxGroup && head_dim > 0 && head_dim <= 1024 &&
           sizeof(float) * tree_row_lds(nq / nkv, head_dim) <= 64 * 1024;
}

// The columns of a call's blocks.  Few rows are bound by latency and bytes, where the narrow kernel's waves run apart:
// 4 rows after 8100 positions of an 8-bit cache 12.6 us in 16 columns, 14.1 in 32, 15.8 in the wide kernel's 64; 8 rows
// 14.7 in 32, 16.5 in 64.
// With 128 columns each key and value is staged (8-bit codes converted) for four column tiles instead of two, but there
// are half as many row tiles.  Where those still give every CU a block: 2048 rows after 2000 positions 220 us (64 columns
// 251), 1024 after 4000 170 (180), after none 42 (38).  Where they take splits that have to be joined it depends on the
// context: 64 rows after 131000 positions of an 8-bit cache 291 us (321), 512 after 16000 278 (304), 64 after 8000 33.9
// (32.7), 64 after 1000 23.4 (18.6), 512 after none 27.3 (18.2); over fp16 caches the same by ratio.  How long it is only
// the device knows; a cache that can hold kFar positions is taken for one that does.  So a cache allocated for long
// contexts pays the larger figure of the last two cases while its context is short.
constexpr int kFar = 1 << 15;
static int tree_cols(int nq, int nkv, int hd, int tokens, bool far) {
    const int group = nq / nkv, cols = tokens * group, T = 128 / group;
    if (cols <= kTTile) return cols <= 16 ? 16 : 32;
    const bool full = static_cast<int64_t>((tokens + T - 1) / T) * nkv >= 256;
    return (far || full) && cols >= 128 && hd == 128 ? 128 : 64;
}
// Row tiles, and key splits that give every CU a block.  Twice or half as many blocks: one row after 8100 positions 11.7 us
// (16.2, 12.9), 64 rows after 8000 32.7 (38.8, 43.2), after 131000 293 (304, 450), 128 rows after 2000 23.6 (34.5, 29.3);
// half as many is better only where there is next to no context (256 rows at position 0 15.7, 13.5).
static TreeGrid tree_grid(int nq, int nkv, int hd, int tokens, bool far) {
    const int T = tree_cols(nq, nkv, hd, tokens, far) / (nq / nkv);
    const int tiles = (tokens + T - 1) / T;
    const int64_t blocks = static_cast<int64_t>(tiles) * nkv;
    return TreeGrid{tiles, static_cast<int>(std::min<int64_t>(kTreeMaxSplits, std::max<int64_t>(1, 256 / blocks)))};
}

size_t tree_attn_workspace_bytes(int nq, int nkv, int head_dim, int tokens) {
    if (head_dim != 128 && head_dim != 256) return 16;
    const int splits = std::max(tree_grid(nq, nkv, head_dim, tokens, false).splits, tree_grid(nq, nkv, head_dim, tokens, true).splits);
    return splits == 1 ? 16 : static_cast<size_t>(splits) * tokens * nq * (head_dim + 2) * sizeof(float);
}

template <typename F, int HD, bool I8, typename Kernel>
static hipError_t launch_tree(const TreeAttnLaunch& p, Kernel kernel, hipStream_t s) {
    const TreeGrid g = tree_grid(p.nq, p.kv.nkv, HD, p.tokens, p.kv.capacity >= kFar);
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(F::kLds));
        e != hipSuccess)
        return e;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(g.tiles * g.splits) * p.kv.nkv), dim3(F::kThreads), F::kLds, s, p, g);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || g.splits == 1) return e;
    const int group = p.nq / p.kv.nkv, T = F::kCols / group;
    const size_t lds = sizeof(float) * tree_row_lds(group, HD);  // attend_row's
    if (g.splits <= kFewSplits) {
        const int heads = kMergeThreads / (group * (HD / 4));
        hipLaunchKernelGGL((tree_attn_merge_few_kernel<F, HD, I8>), dim3(p.tokens, (p.kv.nkv + heads - 1) / heads),
                           dim3(kMergeThreads), lds, s, p, g, T);
    } else {
        hipLaunchKernelGGL((tree_attn_merge_kernel<F, HD, I8>), dim3(p.tokens, p.kv.nkv), dim3(kMergeThreads), lds, s, p,
                           g, T);
    }
    return hipGetLastError();
}
template <int HD, bool I8, int CT, int KS>
static hipError_t launch_wide(const TreeAttnLaunch& p, hipStream_t s) {
    return launch_tree<WideTile<HD, I8, CT, KS>, HD, I8>(p, &tree_attn_wide_kernel<HD, I8, CT, KS>, s);
}
template <int HD, bool I8, int KS, bool HALF>
static hipError_t launch_narrow(const TreeAttnLaunch& p, hipStream_t s) {
    return launch_tree<NarrowTile<HD, I8, KS, HALF ? 16 : 32>, HD, I8>(p, &tree_attn_narrow_kernel<HD, I8, KS, HALF>, s);
}
template <int HD, bool I8>
static hipError_t launch_tree_heads(const TreeAttnLaunch& p, hipStream_t s) {
    constexpr int KS = HD == 128 ? 8 : 4;
    switch (tree_cols(p.nq, p.kv.nkv, HD, p.tokens, p.kv.capacity >= kFar)) {
        case 16: return launch_narrow<HD, I8, KS, true>(p, s);
        case 32: return launch_narrow<HD, I8, KS, false>(p, s);
        case 64: return launch_wide<HD, I8, 2, KS / 2>(p, s);
        default:
            if constexpr (HD == 128) return launch_wide<HD, I8, 4, KS / 4>(p, s);
            return hipErrorInvalidValue;  // (128 columns are for 128 dims)
    }
}

hipError_t launch_tree_attn(const TreeAttnLaunch& p, hipStream_t s) {
    const int hd = p.kv.head_dim;
    // the matrix-core kernels take rows in 16-byte pieces, the caches in whole words
    const bool al = ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.gate) |
                      reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0 && p.q_stride % 4 == 0 && p.out_stride % 4 == 0 &&
                    ((reinterpret_cast<uintptr_t>(p.kv.k) | reinterpret_cast<uintptr_t>(p.kv.v)) & 3u) == 0;
    const bool in32 = p.q_stride < 1 << 21 && p.out_stride < 1 << 21;  // offsets within a block's (at most 128) rows
    const bool kv32 = static_cast<int64_t>(p.kv.nkv) * hd * 2 * 256 < int64_t(1) << 31;  // ... and its keys
    if (al && in32 && kv32 && hd == 128) return p.kv.i8 ? launch_tree_heads<128, true>(p, s) : launch_tree_heads<128, false>(p, s);
    if (al && in32 && kv32 && hd == 256) return p.kv.i8 ? launch_tree_heads<256, true>(p, s) : launch_tree_heads<256, false>(p, s);
    const size_t lds = sizeof(float) * tree_row_lds(p.nq / p.kv.nkv, hd);
    const dim3 grid(p.tokens, p.kv.nkv);
    if (p.kv.i8)
        hipLaunchKernelGGL((tree_attn_row_kernel<true>), grid, dim3(256), lds, s, p);
    else
        hipLaunchKernelGGL((tree_attn_row_kernel<false>), grid, dim3(256), lds, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
