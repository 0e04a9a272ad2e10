// paged_attn.hip - attention of a step's rows over their sequences' pages.
#include <algorithm>

#include "attn_mfma.hpp"
#include "paged_common.hpp"

namespace xqhip {

constexpr int kPagedMaxGroup = 16;
constexpr int kRowChunk = 32;  // keys: a page holds whole chunks

constexpr size_t paged_row_lds(int group, int hd) {
    return (2 * static_cast<size_t>(group) * hd + static_cast<size_t>(group) * (kRowChunk + 3)) * sizeof(float);
}

// ---------------------------------------------------------------------------
// One row and the `group` query heads of kv head kh (of which h0 .. h1 - 1 are
// written), any head size: the positions in chunks of 32 with a running max and
// sum (rescaled by exp(m_old - m_new)).  What the row does not see is passed over,
// so nothing in it can reach the row; a chunk without a score above minus infinity
// leaves the sums.  Left simple: 32 sequences of 4000 positions take 2.7 ms.
// ---------------------------------------------------------------------------
template <int THREADS>
__device__ void attend_paged_row(const PagedAttnLaunch& p, int s, const SeqRows& sr, int row, int kh, float* smem, int h0 = 0, int h1 = kPagedMaxGroup) {
    static_assert(THREADS >= 8 * kRowChunk, "eight threads per key");
    const int hd = p.kv.head_dim, nkv = p.kv.nkv, group = p.nq / nkv;
    const int64_t want = static_cast<int64_t>(max(sr.past, 0)) + (row - sr.row0) + 1;
    const int seen = sr.past < 0 ? 0 : static_cast<int>(min(want, static_cast<int64_t>(table_positions(p.step, p.kv))));
    float* qs = smem;                      // [group][hd]
    float* sc = qs + group * hd;           // [group][32]
    float* osum = sc + group * kRowChunk;  // [group][hd] running output
    float* ml = osum + group * hd;         // [group][2] running max, sum
    float* fac = ml + 2 * group;           // [group] rescale of this chunk
    const size_t head = static_cast<size_t>(kh) * group * hd;
    const float* qrow = p.q + static_cast<size_t>(row) * p.q_stride + head;
    __syncthreads();
    for (int i = threadIdx.x; i < group * hd; i += THREADS) {
        qs[i] = qrow[i];
        osum[i] = 0.0f;
    }
    if (static_cast<int>(threadIdx.x) < group) {
        ml[2 * threadIdx.x] = -INFINITY;
        ml[2 * threadIdx.x + 1] = 0.0f;
    }
    __syncthreads();
    const float rscale = 1.0f / sqrtf(static_cast<float>(hd));
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    for (int c0 = 0; c0 < seen; c0 += kRowChunk) {
        const int page = page_at(p.step, p.kv, s, c0 / p.kv.page);
        if (page < 0) continue;  // block-uniform
        const int at = c0 % p.kv.page, n = min(kRowChunk, seen - c0);
        const size_t base = page_head(p.kv, page, kh);
        const int8_t* kc = static_cast<const int8_t*>(p.kv.k) + base;
        const int8_t* vc = static_cast<const int8_t*>(p.kv.v) + base;
        const _Float16* kf = static_cast<const _Float16*>(p.kv.k) + base;
        const _Float16* vf = static_cast<const _Float16*>(p.kv.v) + base;
        const size_t sat = static_cast<size_t>(page) * nkv + kh;
        const float ks = p.kv.i8 ? p.kv.k_scale[sat] : 1.0f, vs = p.kv.i8 ? p.kv.v_scale[sat] : 1.0f;
        {
            const int sub = threadIdx.x & 7, tt = threadIdx.x >> 3;
            const bool valid = tt < n;
            for (int g = 0; g < group; ++g) {
                float dot = 0.0f;
                if (valid)
                    for (int d = sub; d < hd; d += 8)
                        dot += qs[g * hd + d] * (p.kv.i8 ? static_cast<float>(kc[k_offset<16>(p.kv, at + tt, d)])
                                                         : static_cast<float>(kf[k_offset<8>(p.kv, at + tt, d)]));
                dot = lanes_sum<8>(dot);
                if (valid && sub == 0) sc[g * kRowChunk + tt] = dot * ks * rscale;
            }
        }
        __syncthreads();
        for (int g = wid; g < group; g += THREADS / kWave) {
            const float sv = lane < n ? sc[g * kRowChunk + lane] : -INFINITY;
            const bool nan = __builtin_amdgcn_ballot_w64(sv != sv) != 0;
            const float m_old = ml[2 * g];
            const float m_new = nan ? __builtin_nanf("") : fmaxf(m_old, wave_max(sv));
            const float e = sv == -INFINITY ? 0.0f : expf(sv - m_new);
            const float lsum = wave_sum(e);
            if (lane < kRowChunk) sc[g * kRowChunk + lane] = e;
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
            float o = 0.0f;
            for (int j = 0; j < n; ++j)
                o += sc[g * kRowChunk + j] * (p.kv.i8 ? static_cast<float>(vc[v_offset<16>(p.kv, at + j, d)])
                                                      : static_cast<float>(vf[v_offset<8>(p.kv, at + j, d)]));
            osum[i] = osum[i] * fac[g] + o * vs;
        }
        __syncthreads();
    }
    for (int i = h0 * hd + threadIdx.x; i < min(h1, group) * hd; i += THREADS) {
        const float l = ml[2 * (i / hd) + 1];
        const float r = l == 0.0f ? 0.0f : osum[i] / l;
        const float gate = p.gate ? sigmoid_dev(p.gate[static_cast<size_t>(row) * p.q_stride + head + i]) : 1.0f;
        p.out[static_cast<size_t>(row) * p.out_stride + head + i] = r * gate;
    }
}

__global__ void __launch_bounds__(256) paged_attn_row_kernel(PagedAttnLaunch p) {
    extern __shared__ float smem[];
    const int row = blockIdx.x;
    const int s = __builtin_amdgcn_readfirstlane(seq_of_row(p.step, row));
    if (s >= p.step.seqs) return;
    const SeqRows sr = seq_rows(p.step, s);
    if (row < sr.row0 || row - sr.row0 >= sr.rows) return;
    attend_paged_row<256>(p, s, sr, row, blockIdx.y, smem);
}

// ---------------------------------------------------------------------------
// Matrix-core forms, heads of 128 and 256 dims: narrow_block for sequences of up
// to 8 or 16 columns (single tokens), wide_block for the others (prompt chunks),
// 64 or 128 columns a block.  A block takes some columns of one sequence and kv
// head and a range of its keys, a column being one (row, query head) pair: column
// c of C is head c / T of the kv head's `group` and row t0 + c % T, T = C / group.
// Its waves share the keys in 32-key tiles, each with its own running max, sum and
// output, joined through LDS at the end; blocks' parts of the same columns are
// joined by paged_merge_kernel.
//
// Scores are formed transposed, S^T = K Q^T (keys are the MFMA rows).  The pages
// hold keys and values as the operands are: a lane's eight (or sixteen) values
// are 16 bytes in a row, 32 lanes' 512 bytes, so K and V go from memory to the
// matrix cores without a transposition.  An MFMA leaves a lane some rows of its
// column; the order in which a tile's keys are given to the rows is chosen so that
// those are eight keys in a row, the ones whose values the lane loads.
//
// An 8-bit page's codes become fp16 integers, exactly; its scales enter as one
// factor of a tile's scores and of its weights.
//
// Precision: q (scaled per column by a power of two to [2^12, 2^13)) and the
// weights (times 2^6) are split into fp16 hi + lo, 22 bits together; fp32
// accumulation.  The exponents' reference m is a column's largest score so far,
// or up to 2^6 less; over 8-bit pages the largest of score + log2 of V's scale.
//
// A masked key has weight 0, but 0 times an infinity is not 0; values behind the
// last position are replaced by 0, and where a sum is not finite for another
// reason or the weights sum to 0 the block that writes such an output computes
// its rows again by attend_paged_row.
// ---------------------------------------------------------------------------
template <int HD>
constexpr int kBlockWaves = HD == 128 ? 8 : 4;  // of a wide block: registers for two waves, or one, per SIMD
template <int HD, bool I8, int NT>
constexpr int kNarrowPerSimd = HD == 128 || (I8 && NT == 1) ? 2 : 1;  // narrow waves that a SIMD has registers for
constexpr int kNarrowWaves = 4;  // of a narrow block (8, one block on a CU: 45 sequences of 500 27.4 us, not 18.5)
constexpr int kNarrowCols = 16;      // sequences of up to 8 or 16 columns: narrow_block
constexpr int kNarrowBlocks = 512;  // blocks that share their tiles, at most
constexpr int kLeastCols = 64, kMostCols = 128;  // columns of other sequences' blocks: wide_block
constexpr int kWideBlocks = 256;    // blocks that few row tiles' keys are split over
constexpr int kMostUnits = 65535 * kPagedMaxGroup / kLeastCols + 1024 + kWideBlocks;  // row tiles and splits of a step

// the key of a tile that row r of a 32-row MFMA stands for: a lane's slots are then keys 16 (slot / 8) + 8 (lane / 32) + slot % 8
__device__ __forceinline__ int key_of_row(int r) {
    const int e = r & 3, g = r >> 2 & 1, a0 = r >> 3 & 1, a1 = r >> 4;
    return 16 * a1 + 8 * g + 4 * a0 + e;
}

// Rows and keys of a sequence in an attention call.
struct SeqKeys {
    SeqRows r;
    int cap;  // positions that the table holds
    __device__ __forceinline__ SeqKeys(const PagedAttnLaunch& p, int s) : r(seq_rows(p.step, s)), cap(table_positions(p.step, p.kv)) {}
    __device__ __forceinline__ SeqKeys(const PagedAttnLaunch& p, const SeqRows& rows) : r(rows), cap(table_positions(p.step, p.kv)) {}
    // last position that row j sees, -1: none
    __device__ __forceinline__ int last(int j) const {
        return r.past < 0 ? -1 : static_cast<int>(min(static_cast<int64_t>(r.past) + j, static_cast<int64_t>(cap) - 1));
    }
};

// (cols: 8 or 16, the narrow blocks' of the call)
__device__ __forceinline__ bool is_narrow(int rows, int group, int cols) { return rows > 0 && rows * group <= cols; }
__device__ __forceinline__ int tiles_of(int last) { return max(0, last) / kTTile + 1; }

// The narrow kernel's work: sequences of up to 16 columns, their 32-key tiles in units of q, for each kv head, one behind
// the other; `blocks` blocks take equal numbers of units.
// Units: a unit lies in one sequence and head and has a block of its own: a CU's only one, or where those are too few one
// of two.  A whole sequence and head where that is not much longer: it needs no joining.
// Ranges (q = 1): a block's tiles may end inside a sequence and head and go on in the next, where some unit would be over
// kApart tiles more than its share.  Every sequence a block goes on to costs it some tiles' time (its place, queries, join).
// (Whole calls, us: 45 sequences of 500 positions in units 17.9, in ranges 22.6; 60 of 1500, 8 bits 27.5, 30.8; 32 of
// 4000, where a unit of 81 tiles stands against ranges of 41, 83, 69.  32 of 1000, 16 / 4 heads, in units of a CU each 14.6,
// of two 16.1; 32 / 8 heads 20.1 either way.)
// Each wave finds its block's place by itself, 64 sequences in its lanes at a time: no barrier, no launch before.
constexpr int kMinTiles = 4;  // smallest unit, a tile for every wave (one sequence of 700 11.1 us, with 8 11.7)
constexpr int kApart = 32;    // (24: one of 60000, 8 bits 30.0 us instead of 27.9; 16: 60 sequences of 1500 31.7, not 27.4)
constexpr int kCus = 256;
struct NarrowItem {
    int s, kh, unit, units;  // of the sequence and head: the unit asked for, and how many there are
};
struct NarrowWork {
    int q, blocks, units, per, rem;  // units: all sequences, one kv head; a block has per, the first rem one more
    int group, nkv, cols;
    int before;           // lane c: units of the sequences up to 64 c + 63
    int held, in, tiles;  // sequences 64 held + lane: units up to it, its tiles

    __device__ __forceinline__ int load(const PagedAttnLaunch& p, int c) const {
        const int s = c * kWave + static_cast<int>(threadIdx.x & (kWave - 1));
        if (s >= p.step.seqs) return 0;
        const SeqKeys k(p, s);
        return is_narrow(k.r.rows, group, cols) ? tiles_of(k.last(k.r.rows - 1)) : 0;
    }
    __device__ __forceinline__ NarrowWork(const PagedAttnLaunch& p, int group_, int cols_, int most) : group(group_), nkv(p.kv.nkv), cols(cols_) {
        const int lane = threadIdx.x & (kWave - 1), chunks = (p.step.seqs + kWave - 1) / kWave;
        int active = 0, sum = 0, longest = 0;
        for (int c = 0; c < chunks; ++c) {
            tiles = load(p, c);
            sum += tiles;
            longest = max(longest, tiles);
            active += __popcll(__builtin_amdgcn_ballot_w64(tiles > 0));
        }
        const int64_t all = static_cast<int64_t>(__builtin_amdgcn_readlane(wave_scan_int(sum), kWave - 1)) * nkv;
        longest = static_cast<int>(wave_max(static_cast<float>(longest)));
        // a block of its own for every unit: on a CU of its own, else beside another
        const int pairs = active * nkv, some = static_cast<int>(min(all, int64_t(1) << 30)), share = some / most;
        q = 0;
        for (int n = min(kCus, most); q == 0 && n <= most; n *= 2) {
            if (pairs > n) continue;
            int u = pairs < n ? max((some + n - pairs - 1) / (n - pairs), kMinTiles) : longest;
            if (2 * longest <= 3 * u) u = longest;
            if (min(u, longest) <= share + kApart) q = u;
        }
        if (q == 0) q = 1 + static_cast<int>(all >> 30);  // (units are counted in 32 bits)
        before = 0;
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) tiles = load(p, c);
            in = wave_scan_int((tiles + q - 1) / q);
            const int n = __builtin_amdgcn_readlane(in, kWave - 1);
            before += lane >= c ? n : 0;
        }
        held = chunks - 1;
        units = __builtin_amdgcn_readlane(before, kWave - 1);
        const int total = units * nkv;
        blocks = min(most, total);
        per = total / max(blocks, 1);
        rem = total - per * blocks;
    }
    __device__ __forceinline__ int begin(int b) const { return b * per + min(b, rem); }
    __device__ __forceinline__ int block_of(int x) const {
        const int edge = rem * (per + 1);
        return x < edge ? x / (per + 1) : rem + (x - edge) / per;
    }
    __device__ __forceinline__ NarrowItem find(const PagedAttnLaunch& p, int x) {
        const int y = x / nkv;
        const int c = __popcll(__builtin_amdgcn_ballot_w64(before <= y));
        const int base = c ? __builtin_amdgcn_readlane(before, c - 1) : 0;
        if (c != held) {
            tiles = load(p, c);
            in = wave_scan_int((tiles + q - 1) / q);
            held = c;
        }
        const int n = __popcll(__builtin_amdgcn_ballot_w64(base + in <= y));
        const int pre = n ? __builtin_amdgcn_readlane(in, n - 1) : 0;
        NarrowItem it;
        it.s = c * kWave + n;
        it.units = __builtin_amdgcn_readlane(in, n) - pre;
        const int at = x - (base + pre) * nkv;
        it.kh = at / it.units;
        it.unit = at - it.kh * it.units;
        return it;
    }
};

// Chunks [begin, end) of the keys of a row tile; its `splits` units lie one behind the other, and of a tile with several
// so do their partial outputs' slots.
struct alignas(16) WideUnit {
    int seq, tile, begin, end;
    int splits, split, slot;  // of the row tile: units, which of them this is, the first's slot
    SeqRows rows;             // the sequence's
};
// Workspace: where the merge finds the narrow sequences' parts, the wide kernel's units, partial outputs.
struct PagedWs {
    int* head;        // [0] wide units, [1] their slots, [2] blocks of the narrow work, [3] columns of a wide block
    int4* narrow_at;  // [seqs][nkv]: blocks that share the sequence's tiles, the first of them and its slot, whether a single
                      // block's output has to be computed again
    int4* wide_at;    // [wide units][nkv], of those without splits: as above
    WideUnit* units;
    WideUnit* split;  // [slots]: their units
    float* narrow;    // [2 blocks][columns][hd + 2]
    float* wide;      // [slots][nkv][columns][hd + 2]
    int narrow_cols, narrow_blocks;  // of the call
    int group, narrow_rows, least_rows, most_rows;  // query heads of a kv head; rows whose heads fill a block's columns
};
// Kernel arguments that are needed at any rate, all on their way at once: where they are first used, behind branches, each
// would be waited for alone.
template <typename... Ts>
__device__ __forceinline__ void fetch_args(Ts... v) {
    (..., [](auto x) { asm volatile("" ::"s"(x)); }(v));
}
constexpr size_t kWsHead = 16;

template <int HD, int KS, int COLS>
struct PagedBlock {
    static constexpr int kThreads = kWave * KS, kCols = COLS;
    static constexpr int kLdo = HD + 4;                                            // floats per column of a wave's output
    static constexpr int kQuads = HD / 4;                                          // float4 of an output row
    static constexpr size_t kOutBytes = static_cast<size_t>(kCols) * (KS * (kLdo + 3) + 1) * 4;
};

__device__ __forceinline__ bool write_paged_quad(float4 r, float L, const float* gate, float* out) {
    return write_quad(r, L, gate != nullptr, gate ? *reinterpret_cast<const float4*>(gate) : float4{}, out);
}

// The key waves of a block's columns joined, then written: a partial output (to part_out: [COLS][HD], then [COLS][2]), or
// the output, and to *entry whether it has to be computed again.  The waves' outputs, maxima and sums lie in LDS; the block
// has passed no barrier since.
template <int HD, int KS, int COLS, int THREADS>
__device__ __forceinline__ void join_paged(const PagedAttnLaunch& p, const SeqRows& sr, int kh, int group, int t0, int ntok, int T,
                                           uint32_t inv_t, float* part_out, int4* entry, void* lds, int* redo) {
    using F = PagedBlock<HD, KS, COLS>;
    const float* Ol = static_cast<float*>(lds);         // [KS][columns][kLdo]
    const float* Ml = Ol + KS * F::kCols * F::kLdo;     // [KS][columns][2]
    float* Fl = const_cast<float*>(Ml) + KS * F::kCols * 2;  // [KS][columns]
    float* Ll = Fl + KS * F::kCols;                     // [columns] the sums
    if (threadIdx.x == 0) *redo = 0;
    __syncthreads();
    auto row_of = [&](int c, int& hc, int& tc) {
        hc = static_cast<int>(c * inv_t >> 16);
        tc = c - hc * T;
        return hc < group && tc < ntok;
    };
    if (threadIdx.x < F::kCols) {  // a thread per column: the factors of its waves' outputs, and their sum
        const int c = threadIdx.x;
        int hc, tc;
        if (row_of(c, hc, tc)) {
            float M = -INFINITY, L = 0.0f;
            for (int i = 0; i < KS; ++i) M = fmaxf(M, Ml[(c + i * F::kCols) * 2]);
            for (int i = 0; i < KS; ++i) {
                const float f = __builtin_amdgcn_exp2f(Ml[(c + i * F::kCols) * 2] - M);
                L += f * Ml[(c + i * F::kCols) * 2 + 1];
                Fl[c + i * F::kCols] = f;
            }
            Ll[c] = L;
            if (part_out) reinterpret_cast<float2*>(part_out + F::kCols * HD)[c] = make_float2(M, L);
        }
    }
    __syncthreads();
    bool bad = false;
    for (int i = threadIdx.x; i < F::kCols * F::kQuads; i += THREADS) {
        const int c = i / F::kQuads, d = 4 * (i % F::kQuads);
        int hc, tc;
        if (!row_of(c, hc, tc)) continue;
        float4 r = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) add_scaled(r, Fl[c + k * F::kCols], *reinterpret_cast<const float4*>(Ol + (c + k * F::kCols) * F::kLdo + d));
        if (part_out) {
            *reinterpret_cast<float4*>(part_out + c * HD + d) = r;
            continue;
        }
        const size_t row = sr.row0 + t0 + tc, col = static_cast<size_t>(kh * group + hc) * HD + d;
        bad |= write_paged_quad(r, Ll[c], p.gate ? p.gate + row * p.q_stride + col : nullptr, p.out + row * p.out_stride + col);
    }
    if (part_out) return;
    if (bad) *redo = 1;
    __syncthreads();
    if (threadIdx.x == 0) *entry = make_int4(1, 0, 0, *redo);
}

// Where the tiles of a wave lie: lane i holds the page (and its scales) of the wave's tile i, of 64.
struct TilePages {
    int page, first, step, end;  // tiles first, first + step, .. < end
    float ks, vs;
    __device__ __forceinline__ void fill(const PagedAttnLaunch& p, int s, int kh, int i0, int last) {
        const int tile = first + (i0 + static_cast<int>(threadIdx.x & (kWave - 1))) * step;
        page = tile < end && tile * kTTile <= last ? page_at(p.step, p.kv, s, tile * kTTile / p.kv.page) : -1;
        if (p.kv.i8) {
            const size_t at = static_cast<size_t>(max(page, 0)) * p.kv.nkv + kh;
            ks = page >= 0 ? p.kv.k_scale[at] : 1.0f;
            vs = page >= 0 ? p.kv.v_scale[at] : 0.0f;
        }
    }
};

template <bool I8, int HD>
struct TileBase {
    __amdgpu_buffer_rsrc_t k, v;
    int valid;
};
// the resources of tile i of a wave's (empty where it has no page: loads then read 0)
template <bool I8, int HD>
__device__ __forceinline__ TileBase<I8, HD> tile_base(const PagedAttnLaunch& p, TilePages& tp, int s, int kh, int i, int last) {
    constexpr uint32_t es = I8 ? 1u : 2u;
    if ((i & 63) == 0) tp.fill(p, s, kh, i, last);  // wave-uniform
    TileBase<I8, HD> b;
    const int page = __builtin_amdgcn_readlane(tp.page, i & 63);
    b.valid = page >= 0;
    const int off = (tp.first + i * tp.step) * kTTile & (p.kv.page - 1);
    const size_t head = page_head(p.kv, max(page, 0), kh) * es;
    const uint32_t kskip = off * 16u, vskip = static_cast<uint32_t>(off) * HD * es;
    const uint32_t all = b.valid ? static_cast<uint32_t>(p.kv.page) * HD * es : 0u;
    b.k = buf_rsrc(static_cast<const uint8_t*>(p.kv.k) + head + kskip, b.valid ? all - kskip : 0u);
    b.v = buf_rsrc(static_cast<const uint8_t*>(p.kv.v) + head + vskip, b.valid ? all - vskip : 0u);
    return b;
}

// The factor of a tile's scores in the exponent of 2.  A page of zeros has the scale 0, and a masked score of minus
// infinity times 0 is no number: another factor of its scores, all 0, does as well.
__device__ __forceinline__ float tile_scale(float column, float page) {
    const float f = column * page;
    return f == 0.0f ? 1.0e-37f : f;
}

// the first n of eight fp16 values, 0 for the others
__device__ __forceinline__ u32x4 first_halves(u32x4 v, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] &= n > 2 * i + 1 ? ~0u : (n > 2 * i ? 0xffffu : 0u);
    return v;
}

template <int HD, int CT>
struct WideShape {
    static constexpr int KS = kBlockWaves<HD> / CT;
    static constexpr int kThreads = kWave * CT * KS, kKeys = kTTile * KS, kCols = kTTile * CT;
    using F = PagedBlock<HD, KS, kCols>;
    struct Q {  // of QueryStage
        static constexpr int kThreads = WideShape::kThreads, kCols = WideShape::kCols;
    };
    static constexpr int kBuf = kKeys * HD;  // halves
    static constexpr size_t kKvBytes = 4 * static_cast<size_t>(kBuf) * 2;
    static constexpr size_t kLds = kKvBytes > F::kOutBytes ? kKvBytes : F::kOutBytes;
    static_assert(QueryStage<Q, HD>::kBytes <= kLds && kLds + 64 <= 160 * 1024, "LDS");
};

// The units of the sequences that the narrow kernel does not take, by one block: of one wave where that has a lane per
// sequence and few row tiles (13 rows beside 13 tokens 22.9 us; by sixteen waves, with their barriers, 24.5).
//
// Columns of a block: with 128 each key and value is staged for four column tiles instead of two, but there are half as many
// row tiles.  128 where those still give every block of a round its own (calls one after the other on the same data: three
// chunks of 512 rows after 2300 beside 21 tokens 139 us, with 64 columns 162; 2000 rows after 2000 208, 233), or where a
// round's blocks have over kLong chunks each, so that splits cost little beside them (512 rows after 16000 268, 283; 64 after
// 131000 267, 291); elsewhere 64 (500 rows after 3584 81, with 128 columns 85; 64 after 1000 23, 26).
constexpr int kLong = 60;
constexpr int kPlanTiles = 256;  // row tiles, at most, for one wave
template <int HD, int WAVES>
__global__ void __launch_bounds__(WAVES* kWave) paged_plan_kernel(PagedAttnLaunch p, PagedWs ws) {
    constexpr int kWaves = WAVES, kThreads = WAVES * kWave;
    __shared__ int pre[kThreads], red[3][kWaves], length;
    __shared__ SeqRows seq[kThreads];
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, s = threadIdx.x;
    const int nkv = p.kv.nkv, group = ws.group, seqs = p.step.seqs, cap = table_positions(p.step, p.kv);
    const int room = max(1, kWideBlocks / nkv);  // units of a round of blocks
    int mine = 0, keys = 0;                      // rows of this thread's sequence, positions
    if (s < seqs) {
        const SeqRows r = seq_rows(p.step, s);
        if (r.rows > 0 && !is_narrow(r.rows, group, ws.narrow_cols)) mine = r.rows;
        seq[s] = r;
        keys = r.past < 0 ? 0 : min(cap, r.past);
    }
    if (wid == kWaves - 1) {
        const NarrowWork w(p, ws.group, ws.narrow_cols, ws.narrow_blocks);
        if (lane == 0) ws.head[2] = w.blocks;
    }
    auto wave_total = [&](int v) { return __builtin_amdgcn_readlane(wave_scan_int(v), kWave - 1); };
    auto tiles_of_rows = [&](int n, int rows) { return (n + rows - 1) / rows; };
    int cols = kLeastCols;
    const int n64 = tiles_of_rows(mine, ws.least_rows), n128 = tiles_of_rows(mine, ws.most_rows);
    {
        // (chunks of 128 keys, in the order of their number)
        const int chunks = n64 ? min(n64 * ((keys + mine / 2) / 128 + 1), 1 << 20) : 0;
        const int a = wave_total(n64), b = wave_total(n128), c = wave_total(chunks);
        if (lane == 0) {
            red[0][wid] = a;
            red[1][wid] = b;
            red[2][wid] = c;
        }
    }
    __syncthreads();
    int tiles = 0, tiles128 = 0, before = 0, before128 = 0;
    int64_t chunks = 0;
    for (int i = 0; i < kWaves; ++i) {
        before += i < wid ? red[0][i] : 0;
        before128 += i < wid ? red[1][i] : 0;
        tiles += red[0][i];
        tiles128 += red[1][i];
        chunks += red[2][i];
    }
    if (HD == 128 && (tiles128 >= room || chunks * nkv > static_cast<int64_t>(kLong) * kWideBlocks)) {
        cols = kMostCols;
        tiles = tiles128;
        before = before128;
    }
    const int own = cols == kMostCols ? n128 : n64, T = cols == kMostCols ? ws.most_rows : ws.least_rows, chunk = kBlockWaves<HD> * kTTile * kTTile / cols;
    // any division of the rows has no more; sequences that claim the same rows (row0 falls) have as many, and units and slots
    // stay within the workspace
    tiles = min(tiles, p.step.rows / T + min(seqs, p.step.rows));
    pre[s] = before + wave_scan_int(own) - own;
    __syncthreads();
    auto tile_at = [&](int f, int& q, int& tile) {  // chunks of row tile f
        int lo = 0, hi = seqs - 1;                  // the last sequence with pre <= f
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (pre[mid] <= f)
                lo = mid;
            else
                hi = mid - 1;
        }
        q = lo;
        tile = f - pre[lo];
        const SeqRows r = seq[lo];
        const int seen = r.past < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(r.past) + min((tile + 1) * T, r.rows), static_cast<int64_t>(cap)));
        return max(0, seen - 1) / chunk + 1;
    };
    // Splits: whole rounds of blocks take whole tiles; the others, no more than three eighths of a round, are split to the
    // shortest length with which their units fit one (two chunks of 600 rows after 1500, heads of 256, 8 bits, 127 us, by whole
    // tiles 154; with half a round the three chunks above 144 instead of 138, with more 900 rows after 500 59 instead of 54).
    const int rest = tiles < room ? tiles : 8 * (tiles % room) <= 3 * room ? tiles % room : 0;
    constexpr int kHeld = kWideBlocks / kWave;
    if (wid == 0) {
        int per = 1 << 20;  // (no tile has so many chunks)
        if (rest > 0) {
            int c[kHeld], most = 0, sum = 0;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const int f = i * kWave + lane;
                int q, tile;
                c[i] = 0;
                if (f < rest) c[i] = tile_at(f, q, tile);
                most = max(most, c[i]);
                sum += c[i];
            }
            most = static_cast<int>(wave_max_u64(most));
            int low = max(1, (wave_total(sum) + room - 1) / room), high = max(most, low);
            while (low < high) {
                const int mid = (low + high) / 2;
                int n = 0;
#pragma unroll
                for (int i = 0; i < kHeld; ++i)
                    if (i * kWave < rest) n += (c[i] + mid - 1) / mid;  // wave-uniform
                if (wave_total(n) <= room)
                    high = mid;
                else
                    low = mid + 1;
            }
            per = low;
        }
        if (lane == 0) length = per;
    }
    __syncthreads();
    const int per = length;
    int units = 0;  // unit count, slots << 16
    for (int f0 = 0; f0 < tiles; f0 += kThreads) {
        const int f = tiles - 1 - (f0 + static_cast<int>(threadIdx.x));  // later rows, which see more, first
        int q = 0, tile = 0, n = 0, c = 0;
        if (f >= 0) {
            c = tile_at(f, q, tile);
            n = f < rest ? (c + per - 1) / per : 1;
        }
        const int v = n + (n > 1 ? n << 16 : 0), in = wave_scan_int(v);
        __syncthreads();
        if (lane == kWave - 1) red[0][wid] = in;
        __syncthreads();
        int at = units + in - v;
        for (int i = 0; i < kWaves; ++i) {
            at += i < wid ? red[0][i] : 0;
            units += red[0][i];
        }
        for (int i = 0; i < n; ++i) {
            // (c < 2^15 chunks, n <= 2^8)
            const WideUnit un{q, tile, c * i / n, c * (i + 1) / n, n, i, at >> 16, seq[q]};
            ws.units[(at & 0xffff) + i] = un;
            if (n > 1) ws.split[(at >> 16) + i] = un;
        }
    }
    if (threadIdx.x == 0) {
        ws.head[0] = units & 0xffff;
        ws.head[1] = units >> 16;
        ws.head[3] = cols;
    }
}

// Up to 8 columns, or 16 (NT tiles of 8): bounded by memory, with short contexts by the chain of loads from the step's
// tables to the values (one sequence of 700 positions 6.9 us; 32 of 4000, 336 MB, 64, 5.3 TB/s).  MFMA tiles of 16 columns: q's hi parts in a tile's first eight, its lo parts in
// the others.  One MFMA then does what two do.  A wave takes 32 keys at a time as two tiles of 16 rows; a lane and its
// neighbour eight lanes on add their scores and take four keys each, and the weights' hi and lo parts go back into the two
// halves.  MFMA row i of tile h stands for key 8 (i / 4) + 4 h + i % 4, so that a lane's part of the weights, four keys of
// each tile, is the eight positions of a piece of V.  K and V go straight into registers, the next keys' on their way
// meanwhile; no barrier before the waves join.
typedef float floatx4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ float other_half(float v) { return dpp_f32<0x128>(v); }  // of lane l ^ 8

template <int HD, bool I8, int KS, int NT>
__device__ __forceinline__ void narrow_block(const PagedAttnLaunch& p, const PagedWs& ws, int block, uint4* paged_lds) {
    constexpr int kCols = 8 * NT;
    using F = PagedBlock<HD, KS, kCols>;
    using Q = QueryStage<F, HD>;
    constexpr int kSteps = HD / 32, kDimTiles = HD / 16, kKPieces = HD / (I8 ? 64 : 32);
    typedef typename std::conditional<I8, u32x2, u32x4>::type VPiece;  // eight positions of a dim
    __shared__ int redo;
    const int nkv = p.kv.nkv, group = ws.group, T = ws.narrow_rows;
    const int lane = threadIdx.x & (kWave - 1), ks = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int i16 = lane & 15, j = lane >> 4, part = i16 >> 3;
    const uint32_t inv_t = (65535u + T) / T;
    NarrowWork w(p, ws.group, kCols, ws.narrow_blocks);
    if (block >= w.blocks) return;
    const int begin = w.begin(block), end = w.begin(block + 1);
    const uint32_t kat = (static_cast<uint32_t>(j) * p.kv.page + 8 * (i16 >> 2) + (i16 & 3)) * 16u, kstep = 64u * p.kv.page;
    const uint32_t vat = I8 ? (static_cast<uint32_t>(j >> 1) * HD + i16) * 16u + 8u * (j & 1) : (static_cast<uint32_t>(j) * HD + i16) * 16u;
    const int lane_key = 8 * j + 4 * part;  // of the lane's four slots
    for (int at = begin; at < end;) {
        const NarrowItem it = w.find(p, at);
        const int s = it.s, kh = it.kh, u0 = it.unit, u1 = min(it.units, u0 + (end - at));
        const bool whole = u0 == 0 && u1 == it.units;
        const int slot = at == begin ? 0 : 1;
        float* part_out = whole ? nullptr : ws.narrow + (2 * static_cast<size_t>(block) + slot) * kCols * (HD + 2);
        int4* entry = ws.narrow_at + s * nkv + kh;
        if (u0 == 0 && !whole && threadIdx.x == 0) *entry = make_int4(w.block_of(at + it.units - 1) - block + 1, block, slot, 0);
        at += u1 - u0;
        const SeqKeys sk(p, s);
        const int ntok = sk.r.rows, last = sk.last(ntok - 1), sure = sk.last(0);
        TilePages tp;
        tp.first = u0 * w.q + ks;
        tp.step = KS;
        tp.end = min(u1 * w.q, tiles_of(last));
        const int n = __builtin_amdgcn_readfirstlane(max(0, (tp.end - tp.first + KS - 1) / KS));
        Q query;
        query.load(p.q + static_cast<size_t>(sk.r.row0) * p.q_stride, p.q_stride, kh, ntok, group, T, inv_t);
        u32x4 kr[2][kKPieces];
        VPiece vr[kDimTiles];
        TileBase<I8, HD> next = tile_base<I8, HD>(p, tp, s, kh, 0, last);
        auto load_k = [&] {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int u = 0; u < kKPieces; ++u) kr[h][u] = __builtin_amdgcn_raw_buffer_load_b128(next.k, kat + 64u * h, u * kstep, 0);
        };
        auto load_v = [&] {
#pragma unroll
            for (int d = 0; d < kDimTiles; ++d) {
                if constexpr (I8)
                    vr[d] = __builtin_amdgcn_raw_buffer_load_b64(next.v, vat + 256u * d, 0, 0);
                else
                    vr[d] = __builtin_amdgcn_raw_buffer_load_b128(next.v, vat + 256u * d, 0, 0);
            }
        };
        load_k();
        load_v();
        query.store(paged_lds);
        __syncthreads();
        half8 qf[NT][kSteps];  // the lane's own part, hi or lo
        float sscale[NT], m[NT], l[NT];
        int qpos[NT];
        floatx4 o[NT][kDimTiles];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c = 8 * t + (i16 & 7), hc = static_cast<int>(c * inv_t >> 16), tc = c - hc * T;
#pragma unroll
            for (int u = 0; u < kSteps; ++u) qf[t][u] = Q::part(paged_lds, part, c, I8 ? 64 * (u / 2) + 16 * j + 8 * (u % 2) : 32 * u + 8 * j);
            sscale[t] = Q::scale(paged_lds, c);
            qpos[t] = hc < group && tc < ntok ? sk.last(tc) : -1;
            m[t] = -1.0e30f;  // reference of the exponents
            l[t] = 0.0f;      // this lane's part of the sum
#pragma unroll
            for (int d = 0; d < kDimTiles; ++d) o[t][d] = floatx4{};
        }
        for (int i = 0; i < n; ++i) {
            const int key0 = (tp.first + i * KS) * kTTile;
            const float pscale = I8 ? readlane_f32(tp.ks, i & 63) : 1.0f, vscale = I8 ? readlane_f32(tp.vs, i & 63) : 1.0f;
            const bool valid = next.valid;
            floatx4 st[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) st[t][0] = st[t][1] = floatx4{};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int u = 0; u < kSteps; ++u) {
                    half8 a;
                    if constexpr (I8) {
                        const u32x2 w0 = codes_to_half(kr[h][u / 2][2 * (u % 2)]), w1 = codes_to_half(kr[h][u / 2][2 * (u % 2) + 1]);
                        a = __builtin_bit_cast(half8, u32x4{w0.x, w0.y, w1.x, w1.y});
                    } else {
                        a = __builtin_bit_cast(half8, kr[h][u]);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) st[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[t][u], st[t][h], 0, 0, 0);
                }
            next = tile_base<I8, HD>(p, tp, s, kh, i + 1, last);
            load_k();
            const bool masked = key0 + kTTile - 1 > sure || !valid;  // wave-uniform: keys that some column does not see
            if (!I8 && masked)
#pragma unroll
                for (int d = 0; d < kDimTiles; ++d)
                    if constexpr (!I8) vr[d] = first_halves(vr[d], last + 1 - (key0 + 8 * j));
            half8 pw[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float sc[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float mine = part ? st[t][1][e] : st[t][0][e], yours = part ? st[t][0][e] : st[t][1][e];
                    sc[e] = mine + other_half(yours);
                }
                const float kscale = I8 ? tile_scale(sscale[t], pscale) : sscale[t];
                if (masked) {
                    const int see = valid ? qpos[t] - (key0 + lane_key) : -1;  // slots up to here
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[e] = e <= see ? sc[e] : -INFINITY;
                }
                float mc = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
                mc = fmaxf(mc, other_half(mc));
                mc = pair32_max(xor16_max(mc)) * kscale;
                if constexpr (I8) mc += scale_exponent(vscale);
                // the reference moves only when a column's max has outgrown it (rarely after the first tiles)
                const bool up = mc > m[t] + kSlack;
                if (__builtin_amdgcn_ballot_w64(up)) {
                    const float to = up ? mc : m[t], f = __builtin_amdgcn_exp2f(m[t] - to);
                    m[t] = to;
                    l[t] *= f;
#pragma unroll
                    for (int d = 0; d < kDimTiles; ++d) o[t][d] *= f;
                }
                const float off = kRaise - m[t];
                typedef float f2 __attribute__((ext_vector_type(2)));
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    float x[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        x[k] = __builtin_amdgcn_exp2f(fmaf(sc[e + k], kscale, off));
                        l[t] += x[k];
                        if constexpr (I8) {
                            x[k] *= vscale;
                            asm("" : "+v"(x[k]));  // the rounded product: hi and lo would else be taken from two roundings of it
                        }
                    }
                    const h2 a = __builtin_convertvector((f2{x[0], x[1]}), h2);
                    const h2 b = __builtin_convertvector((f2{x[0] - static_cast<float>(a[0]), x[1] - static_cast<float>(a[1])}), h2);
                    hi[e / 2] = as_u32(a);
                    lo[e / 2] = as_u32(b);
                }
                // a hi lane takes the other's hi, a lo lane the other's lo
                u32x4 y;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t own = part ? lo[e] : hi[e], got = static_cast<uint32_t>(dpp_i32<0x128>(static_cast<int>(part ? hi[e] : lo[e])));
                    y[e] = part ? got : own;
                    y[2 + e] = part ? own : got;
                }
                pw[t] = __builtin_bit_cast(half8, y);
            }
#pragma unroll
            for (int d = 0; d < kDimTiles; ++d) {
                half8 a;
                if constexpr (I8) {
                    const u32x2 w0 = codes_to_half(vr[d].x), w1 = codes_to_half(vr[d].y);
                    a = __builtin_bit_cast(half8, u32x4{w0.x, w0.y, w1.x, w1.y});
                } else {
                    a = __builtin_bit_cast(half8, vr[d]);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pw[t], o[t][d], 0, 0, 0);
            }
            load_v();
        }
        __syncthreads();  // every wave has its q: the outputs take its place
        float* Ol = reinterpret_cast<float*>(paged_lds);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int col = ks * kCols + 8 * t + (i16 & 7);
            float sum = l[t] + other_half(l[t]);
            sum = xor_pair_sum<32>(xor_pair_sum<16>(sum));
#pragma unroll
            for (int d = 0; d < kDimTiles; d += 2) {  // the hi and lo columns' sums, a dim tile in each half
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (part ? o[t][d + 1][e] : o[t][d][e]) + other_half(part ? o[t][d][e] : o[t][d + 1][e]);
                *reinterpret_cast<float4*>(Ol + col * F::kLdo + 16 * (d + part) + 4 * j) = make_float4(v[0], v[1], v[2], v[3]);
            }
            if (lane < 8) *reinterpret_cast<float2*>(Ol + KS * kCols * F::kLdo + col * 2) = make_float2(m[t], sum);
        }
        join_paged<HD, KS, kCols, F::kThreads>(p, sk.r, kh, group, 0, ntok, T, inv_t, part_out, entry, paged_lds, &redo);
        __syncthreads();
    }
}

// The partial outputs of a sequence and kv head joined (nothing to do where one block had all of its tiles).
constexpr int kMergeThreads = 512;
template <int HD>
__device__ void merge_narrow(const PagedAttnLaunch& p, const PagedWs& ws, int s, int kh, float* smem) {
    __shared__ float fac[kNarrowCols][kNarrowBlocks], total[kNarrowCols];
    __shared__ float4 sums[kMergeThreads];
    __shared__ int redo;
    constexpr int kQuads = HD / 4, kBatch = 4;
    const int nkv = p.kv.nkv, group = ws.group, all_cols = ws.narrow_cols, T = ws.narrow_rows, kSlot = all_cols * (HD + 2);
    fetch_args(p.gate, p.q_stride, p.out, p.out_stride, ws.narrow, group, T);
    const int4 at = ws.narrow_at[s * nkv + kh];
    const SeqRows sr = seq_rows(p.step, s);
    if (!is_narrow(sr.rows, group, all_cols)) return;
    const int n = at.x;
    if (n == 1) {
        if (__builtin_expect(at.w != 0, 0))
            for (int t = 0; t < sr.rows; ++t) attend_paged_row<kMergeThreads>(p, s, sr, sr.row0 + t, kh, smem);
        return;
    }
    // the first block's part, and the following blocks' first ones
    const float* base = ws.narrow + (2 * static_cast<size_t>(at.y) + at.z) * kSlot;
    auto part = [&](int b) { return base + (2 * b - (b ? at.z : 0)) * kSlot; };
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, cols = sr.rows * group;
    auto column = [&](int i) { return i / sr.rows * T + i % sr.rows; };  // live column i
    const int items = cols * kQuads, slices = max(1, kMergeThreads / items);
    const int first = slices > 1 ? threadIdx.x % items : threadIdx.x, slice = slices > 1 ? threadIdx.x / items : 0;
    float4 v[kBatch];
    auto load = [&](int item, int b0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int b = b0 + u * slices;
            v[u] = item < items && slice < slices && b < n ? *reinterpret_cast<const float4*>(part(b) + column(item / kQuads) * HD + 4 * (item % kQuads)) : float4{};
        }
    };
    load(first, slice);
    // a quad's row, and its place in it
    auto place = [&](int item, size_t& row) {
        const int i = item / kQuads, head = i / sr.rows;
        row = static_cast<size_t>(sr.row0 + i - head * sr.rows);
        return static_cast<size_t>(kh * group + head) * HD + 4 * (item % kQuads);
    };
    float4 gates = {};  // of the first quad, on their way with its parts
    if (p.gate && slice == 0 && first < items) {
        size_t row;
        const size_t at_col = place(first, row);
        gates = *reinterpret_cast<const float4*>(p.gate + row * p.q_stride + at_col);
    }
    for (int i = wid; i < cols; i += kMergeThreads / kWave) {
        const int c = column(i);
        float M = -INFINITY, L = 0.0f;
        float2 ml[kNarrowBlocks / kWave];
#pragma unroll
        for (int u = 0; u < kNarrowBlocks / kWave; ++u) {
            const int b = lane + u * kWave;
            ml[u] = b < n ? *reinterpret_cast<const float2*>(part(b) + all_cols * HD + 2 * c) : make_float2(-INFINITY, 0.0f);
            M = fmaxf(M, ml[u].x);
        }
        M = wave_max(M);
#pragma unroll
        for (int u = 0; u < kNarrowBlocks / kWave; ++u) {
            const float f = __builtin_amdgcn_exp2f(ml[u].x - M);
            if (lane + u * kWave < n) fac[i][lane + u * kWave] = f;
            L += f * ml[u].y;
        }
        L = wave_sum(L);
        if (lane == 0) total[i] = L;
    }
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
    bool bad = false;
    for (int item = first; item < items; item += kMergeThreads) {  // (more than one round only without slices)
        const int i = item / kQuads;
        float4 r = {};
        size_t row;
        const size_t col = place(item, row);
        if (item != first) {
            load(item, 0);
            if (p.gate) gates = *reinterpret_cast<const float4*>(p.gate + row * p.q_stride + col);
        }
        if (slice < slices)
            for (int b0 = slice;;) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
                    if (b0 + u * slices < n) add_scaled(r, fac[i][b0 + u * slices], v[u]);
                b0 += kBatch * slices;
                if (b0 >= n) break;
                load(item, b0);
            }
        if (slices > 1) {
            sums[threadIdx.x] = r;
            __syncthreads();
            if (slice == 0)
                for (int k = 1; k < slices; ++k) add_scaled(r, 1.0f, sums[k * items + item]);
        }
        if (slice == 0) bad |= write_quad(r, total[i], p.gate != nullptr, gates, p.out + row * p.out_stride + col);
    }
    if (bad) redo = 1;
    __syncthreads();
    if (__builtin_expect(!redo, 1)) return;
    for (int t = 0; t < sr.rows; ++t) attend_paged_row<kMergeThreads>(p, s, sr, sr.row0 + t, kh, smem);
}

// 64 or 128 columns: CT column tiles x KS key waves.  500 rows after 3584, 8-bit pages: 81 to 85 us, 0.75 PFLOP/s of fp16 hi +
// lo passes; the matrix cores are busy for 34 % of the cycles, the vector units for 45 %: neither is full, but the waves of a
// SIMD pass each chunk's barrier together, so products and softmax alternate, and blocks differ in length.  K and V are staged chunk by chunk (32 KS keys, shared by the column tiles) in
// LDS as the pages hold them (8-bit codes as fp16), twice each: one barrier a chunk, the next chunk's loads over a whole
// chunk ahead, and a chunk's products with V beside the next one's softmax.
template <int HD, bool I8, int CT>
__device__ __forceinline__ void wide_block(const PagedAttnLaunch& p, const PagedWs& ws, int index, uint4* paged_lds) {
    using S = WideShape<HD, CT>;
    using Q = QueryStage<typename S::Q, HD>;
    constexpr int KS = S::KS, kSteps = HD / 16, kDimTiles = HD / 32, kKeys = S::kKeys;
    constexpr uint32_t es = I8 ? 1u : 2u;
    constexpr int kKLoads = HD / (I8 ? 32 : 16) / CT, kVLoads = (I8 ? 2 : 4) * HD / 64 / CT;  // of a wave and chunk, 1 KiB each
    __shared__ int redo;
    const int nkv = p.kv.nkv, kh = index % nkv, group = ws.group, T = S::kCols == kMostCols ? ws.most_rows : ws.least_rows;
    const int unit = index / nkv;
    const WideUnit un = ws.units[min(unit, kMostUnits - 1)];  // (on its way with the number of them)
    if (unit >= ws.head[0]) return;
    const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int ct = wid % CT, ks = wid / CT, cl = lane & 31, g = lane >> 5;
    const uint32_t inv_t = (65535u + T) / T;  // c / T = c inv_t >> 16 for c < 128, T <= 128
    const int s = __builtin_amdgcn_readfirstlane(un.seq), t0 = __builtin_amdgcn_readfirstlane(un.tile) * T;
    const int begin = __builtin_amdgcn_readfirstlane(un.begin), end = __builtin_amdgcn_readfirstlane(un.end);
    const SeqKeys sk(p, un.rows);
    const int ntok = min(T, sk.r.rows - t0);
    Q query;
    query.load(p.q + static_cast<size_t>(sk.r.row0 + t0) * p.q_stride, p.q_stride, kh, ntok, group, T, inv_t);
    const int col = ct * kTTile + cl, ch = static_cast<int>(col * inv_t >> 16), ctok = col - ch * T;
    const bool live = ch < group && ctok < ntok;
    const int last = sk.last(t0 + ntok - 1), sure = sk.last(t0), qpos = live ? sk.last(t0 + ctok) : -1;
    TilePages tp;
    tp.first = begin * KS + ks;
    tp.step = KS;
    tp.end = end * KS;
    struct Ref {  // a wave's 32 keys of a chunk
        int page;
        float ks, vs;
    };
    auto ref_of = [&](int c) {
        const int i = c - begin;
        if ((i & 63) == 0) tp.fill(p, s, kh, i, last);  // wave-uniform; chunks are asked for in their order
        Ref r;
        r.page = __builtin_amdgcn_readlane(tp.page, i & 63);
        r.ks = I8 ? readlane_f32(tp.ks, i & 63) : 1.0f;
        r.vs = I8 ? readlane_f32(tp.vs, i & 63) : 1.0f;
        return r;
    };
    // (without a page, or past `end`: loads read 0)
    auto rows_of = [&](const void* pool, const Ref& r, int c, uint32_t skip) {
        const uint32_t off = static_cast<uint32_t>((c * KS + ks) * kTTile & (p.kv.page - 1)) * skip;
        return buf_rsrc(static_cast<const uint8_t*>(pool) + page_head(p.kv, max(r.page, 0), kh) * es + off,
                        r.page >= 0 ? static_cast<uint32_t>(p.kv.page) * HD * es - off : 0u);
    };
    u32x4 kr[kKLoads], vr[kVLoads];
    auto load_k = [&](const Ref& r, int c) {
        const __amdgpu_buffer_rsrc_t rs = rows_of(p.kv.k, r, c, 16u);
        const uint32_t at = (static_cast<uint32_t>(2 * ct * kKLoads + g) * p.kv.page + cl) * 16u;
#pragma unroll
        for (int u = 0; u < kKLoads; ++u) kr[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, at, u * 32u * p.kv.page, 0);
    };
    auto load_v = [&](const Ref& r, int c) {
        const __amdgpu_buffer_rsrc_t rs = rows_of(p.kv.v, r, c, HD * es);
#pragma unroll
        for (int u = 0; u < kVLoads; ++u)
            vr[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, static_cast<uint32_t>(ct * kVLoads * kWave + lane) * 16u, u * 1024, 0);
    };
    // LDS, in halves: K [2][KS][HD / 8][32][8], V [2][KS][4][HD][8]
    _Float16* Kl = reinterpret_cast<_Float16*>(paged_lds);
    _Float16* Vl = Kl + 2 * S::kBuf;
    auto both_halves = [&](_Float16* at, int next, u32x4 c) {  // sixteen codes: two pieces, `next` halves apart
        const u32x2 a = codes_to_half(c[0]), b = codes_to_half(c[1]), d = codes_to_half(c[2]), e = codes_to_half(c[3]);
        *reinterpret_cast<u32x4*>(at) = u32x4{a.x, a.y, b.x, b.y};
        *reinterpret_cast<u32x4*>(at + next) = u32x4{d.x, d.y, e.x, e.y};
    };
    auto store_k = [&](int c) {
        _Float16* d = Kl + (c & 1) * S::kBuf + ks * kTTile * HD;
#pragma unroll
        for (int u = 0; u < kKLoads; ++u) {
            const int b = 2 * (ct * kKLoads + u);  // block of dims of lane 0
            if constexpr (I8)
                both_halves(d + (2 * (b + g) * 32 + cl) * 8, 256, kr[u]);
            else
                *reinterpret_cast<u32x4*>(d + (b * 32 + lane) * 8) = kr[u];
        }
    };
    auto store_v = [&](int c, bool masked) {
        _Float16* d = Vl + (c & 1) * S::kBuf + ks * kTTile * HD;
#pragma unroll
        for (int u = 0; u < kVLoads; ++u) {
            const int i = ct * kVLoads + u, pb = i / (HD / 64), dim = i % (HD / 64) * 64 + lane;
            if constexpr (I8) {
                both_halves(d + (2 * pb * HD + dim) * 8, HD * 8, vr[u]);
            } else {
                if (masked) vr[u] = first_halves(vr[u], last + 1 - ((c * KS + ks) * kTTile + 8 * pb));
                *reinterpret_cast<u32x4*>(d + (pb * HD + dim) * 8) = vr[u];
            }
        }
    };
    Ref r0 = ref_of(begin), r1;
    load_k(r0, begin);
    load_v(r0, begin);
    half8 qhi[kSteps], qlo[kSteps];  // lane supplies dims 16 t + 8 g .. + 7 of its column
    query.store(paged_lds);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
        qhi[t] = Q::part(paged_lds, 0, col, 16 * t + 8 * g);
        qlo[t] = Q::part(paged_lds, 1, col, 16 * t + 8 * g);
    }
    const float sscale = Q::scale(paged_lds, col);
    __syncthreads();  // every wave has its q: K and V may take its place
    store_k(begin);
    r1 = ref_of(begin + 1);
    __syncthreads();
    load_k(r1, begin + 1);
    float m = -1.0e30f, l = 0.0f;  // reference of the exponents, this lane's part of the sum
    floatx16 o[kDimTiles];
#pragma unroll
    for (int j = 0; j < kDimTiles; ++j) o[j] = floatx16{};
    half8 phi[2], plo[2];  // the weights of the chunk before
    auto add_values = [&](int c) {
        const _Float16* vb = Vl + (c & 1) * S::kBuf + (ks * 4 * HD + g * HD + cl) * 8;
#pragma unroll
        for (int j = 0; j < kDimTiles; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const half8 a = *reinterpret_cast<const half8*>(vb + (2 * h * HD + 32 * j) * 8);
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, plo[h], o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, phi[h], o[j], 0, 0, 0);
            }
    };
    const int krow = (ks * (HD / 8) + g) * 32 + key_of_row(cl);
    // One chunk: its scores, the values of the chunk before (the matrix cores work on them while the softmax runs), the
    // next keys and this chunk's values into LDS.  One barrier: both are double-buffered.
    auto chunk = [&](int c, auto first, auto masked) {
        constexpr bool FIRST = decltype(first)::value, MASKED = decltype(masked)::value;
        const int key0 = c * kKeys + ks * kTTile;
        floatx16 st = floatx16{};
        const _Float16* kb = Kl + (c & 1) * S::kBuf + krow * 8;
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            const half8 a = *reinterpret_cast<const half8*>(kb + t * 512);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qlo[t], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qhi[t], st, 0, 0, 0);
        }
        // (past `end`: loads read 0 into buffers that no one reads)
        store_k(c + 1);
        store_v(c, MASKED);
        const Ref r2 = ref_of(c + 2);
        load_v(r1, c + 1);
        load_k(r2, c + 2);
        if constexpr (!FIRST) add_values(c - 1);
        const float kscale = I8 ? tile_scale(sscale, r0.ks) : sscale, vscale = r0.vs;
        if (MASKED || r0.page < 0) {
            const int see = r0.page < 0 ? -1 : qpos - (key0 + 8 * g);
#pragma unroll
            for (int v = 0; v < 16; ++v) st[v] = 16 * (v / 8) + v % 8 <= see ? st[v] : -INFINITY;
        }
        float mc = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; ++v) mc = fmaxf(mc, st[v]);
        mc = pair32_max(mc) * kscale;
        if constexpr (I8) mc += scale_exponent(vscale);
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
                x[e] = __builtin_amdgcn_exp2f(fmaf(st[8 * h + e], kscale, off));
                l += x[e];
                if constexpr (I8) {
                    x[e] *= vscale;
                    asm("" : "+v"(x[e]));  // the rounded product: hi and lo would else be taken from two roundings of it
                }
            }
            split8(x, phi[h], plo[h]);
        }
        if (__builtin_amdgcn_ballot_w64(up)) {
#pragma unroll
            for (int j = 0; j < kDimTiles; ++j) o[j] *= f;
        }
        r0 = r1;
        r1 = r2;
        __syncthreads();  // the next keys and these values are staged; every wave is done with the buffers they replace
    };
    const int clear = min(end, max(begin, (sure + 1) / kKeys));  // chunks [begin, clear) that every column sees whole
    int c = begin;
    if (c < clear)
        chunk(c++, std::true_type{}, std::false_type{});
    else
        chunk(c++, std::true_type{}, std::true_type{});
    for (; c < clear; ++c) chunk(c, std::false_type{}, std::false_type{});
    for (; c < end; ++c) chunk(c, std::false_type{}, std::true_type{});
    add_values(end - 1);
    float* part_out = un.splits > 1 ? ws.wide + (static_cast<size_t>(un.slot + un.split) * nkv + kh) * S::kCols * (HD + 2) : nullptr;
    l = xor_pair_sum<32>(l);
    __syncthreads();  // every wave is done with K and V: the outputs take their place
    {
        using F = typename S::F;
        float* Ol = reinterpret_cast<float*>(paged_lds);
        const int at = ks * F::kCols + ct * kTTile + cl;
        float* oc = Ol + at * F::kLdo + 4 * g;
        if (live) {
#pragma unroll
            for (int j = 0; j < kDimTiles; ++j)
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    *reinterpret_cast<float4*>(oc + 32 * j + 8 * a) = make_float4(o[j][4 * a], o[j][4 * a + 1], o[j][4 * a + 2], o[j][4 * a + 3]);
            if (g == 0) *reinterpret_cast<float2*>(Ol + KS * F::kCols * F::kLdo + at * 2) = make_float2(m, l);
        }
    }
    join_paged<HD, KS, S::kCols, S::kThreads>(p, sk.r, kh, group, t0, ntok, T, inv_t, part_out, ws.wide_at + unit * nkv + kh, paged_lds, &redo);
}

// The splits of a row tile joined, the blocks of each slot (as many as there are for it) a share of the columns (13 rows after
// 200 18.8 us, by one block for each slot 20.7); and outputs that have to be computed again.
template <int HD>
__device__ void merge_wide(const PagedAttnLaunch& p, const PagedWs& ws, int group_of, int groups, int kh, float* smem) {
    __shared__ float fac[kMostCols + kWideBlocks], total[kMostCols];  // a block's columns times the splits
    __shared__ float2 sums[kMostCols + kWideBlocks];
    __shared__ int list[kMergeThreads], count, redo;
    static_assert(kMergeThreads >= kMostCols + kWideBlocks, "a thread per column and split");
    constexpr int kQuads = HD / 4;
    const int nkv = p.kv.nkv;
    WideUnit un = ws.split[group_of];  // (on its way with the number of them: right if each slot has one block)
    const int cols = ws.head[3], slot_size = cols * (HD + 2), group = ws.group, T = cols == kMostCols ? ws.most_rows : ws.least_rows;
    const int units = ws.head[0], slots = ws.head[1];
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    int each = 1, slot = group_of;
    if (2 * slots <= groups) {
        each = groups / max(slots, 1);
        slot = group_of / each;
        if (slot < slots) un = ws.split[slot];
    }
    const int which = group_of - slot * each;
    if (slot < slots) {
        const SeqRows sr = un.rows;
        const int n = un.splits, t0 = un.tile * T, ntok = min(T, sr.rows - t0);
        const int share = un.split * each + which, c0 = cols * share / (n * each), c1 = cols * (share + 1) / (n * each);
        const size_t stride = static_cast<size_t>(nkv) * slot_size;
        const float* base = ws.wide + (static_cast<size_t>(un.slot) * nkv + kh) * slot_size;
        if (static_cast<int>(threadIdx.x) < (c1 - c0) * n) {  // all splits' maxima and sums at once
            const int c = c0 + static_cast<int>(threadIdx.x) / n, b = static_cast<int>(threadIdx.x) % n;
            const bool on = c / T < group && c % T < ntok;  // (others' were not written)
            sums[threadIdx.x] = on ? *reinterpret_cast<const float2*>(base + b * stride + cols * HD + 2 * c) : make_float2(-INFINITY, 0.0f);
        }
        __syncthreads();
        for (int c = wid; c < c1 - c0; c += kMergeThreads / kWave) {
            float M = -INFINITY, L = 0.0f;
            for (int b = lane; b < n; b += kWave) M = fmaxf(M, sums[c * n + b].x);
            M = wave_max(M);
            for (int b = lane; b < n; b += kWave) {
                const float2 ml = sums[c * n + b];
                const float f = __builtin_amdgcn_exp2f(ml.x - M);
                fac[c * n + b] = f;
                L += f * ml.y;
            }
            L = wave_sum(L);
            if (lane == 0) total[c] = L;
        }
        if (threadIdx.x == 0) redo = 0;
        __syncthreads();
        bool bad = false;
        for (int i = threadIdx.x; i < (c1 - c0) * kQuads; i += kMergeThreads) {
            const int c = c0 + i / kQuads, d = 4 * (i % kQuads), hc = c / T, tc = c % T;
            if (hc >= group || tc >= ntok) continue;
            float4 r = {};
#pragma unroll 4
            for (int b = 0; b < n; ++b) add_scaled(r, fac[(c - c0) * n + b], *reinterpret_cast<const float4*>(base + b * stride + c * HD + d));
            const size_t row = sr.row0 + t0 + tc, colm = static_cast<size_t>(kh * group + hc) * HD + d;
            bad |= write_paged_quad(r, total[c - c0], p.gate ? p.gate + row * p.q_stride + colm : nullptr, p.out + row * p.out_stride + colm);
        }
        if (bad) redo = 1;
        __syncthreads();
        // (another block of the tile may write the same rows' other columns: the general form writes them all, with values
        // that differ from the joined ones by roundings only, so each block takes its own columns' rows)
        if (__builtin_expect(redo, 0)) {
            for (int c = c0; c < c1; ++c)
                if (c / T < group && c % T < ntok) attend_paged_row<kMergeThreads>(p, un.seq, sr, sr.row0 + t0 + c % T, kh, smem, c / T, c / T + 1);
        }
        __syncthreads();
    }
    // the units without a split, a share of them by each block
    const int block = group_of * nkv + kh, blocks = groups * nkv, all = units * nkv, per = (all + blocks - 1) / blocks;
    for (int i0 = block * per; i0 < min(all, (block + 1) * per); i0 += kMergeThreads) {
        const int i = i0 + threadIdx.x;
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        if (i < min(all, (block + 1) * per) && ws.units[i / nkv].splits == 1 && ws.wide_at[i].w) list[atomicAdd(&count, 1)] = i;
        __syncthreads();
        const int n = count;
        for (int j = 0; j < n; ++j) {
            const int at = list[j];
            const WideUnit u = ws.units[at / nkv];
            for (int t = u.tile * T; t < min((u.tile + 1) * T, u.rows.rows); ++t) attend_paged_row<kMergeThreads>(p, u.seq, u.rows, u.rows.row0 + t, at % nkv, smem);
        }
        __syncthreads();
    }
}

// Grid: kv heads, then sequences and behind them the groups of a wide block per kv head.
template <int HD, bool WIDE>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(PagedAttnLaunch p, PagedWs ws) {
    extern __shared__ float smem[];  // attend_paged_row's
    const int s = blockIdx.y, kh = blockIdx.x;
    if (!WIDE || s < p.step.seqs)
        merge_narrow<HD>(p, ws, s, kh, smem);
    else if constexpr (WIDE)
        merge_wide<HD>(p, ws, s - p.step.seqs, gridDim.y - p.step.seqs, kh, smem);
}

static PagedWs paged_ws(float* base, int hd, int nkv, size_t* bytes) {
    PagedWs w{};
    char* at = reinterpret_cast<char*>(base);
    auto take = [&](size_t n) {
        char* r = at;
        at += (n + 15) / 16 * 16;
        return r;
    };
    w.head = reinterpret_cast<int*>(take(kWsHead));
    w.narrow_at = reinterpret_cast<int4*>(take(sizeof(int4) * 1024 * nkv));
    w.wide_at = reinterpret_cast<int4*>(take(sizeof(int4) * kMostUnits * nkv));
    w.units = reinterpret_cast<WideUnit*>(take(sizeof(WideUnit) * kMostUnits));
    w.split = reinterpret_cast<WideUnit*>(take(sizeof(WideUnit) * kWideBlocks));
    w.narrow = reinterpret_cast<float*>(take(sizeof(float) * 2 * kNarrowBlocks * kNarrowCols * (hd + 2)));
    w.wide = reinterpret_cast<float*>(take(sizeof(float) * kWideBlocks * (hd == 128 ? kMostCols : kLeastCols) * (hd + 2)));
    if (bytes) *bytes = at - reinterpret_cast<char*>(base);
    return w;
}

size_t paged_attn_workspace_bytes(int nq, int nkv, int head_dim) {
    if (nkv <= 0 || nkv > 256 || nq <= 0 || nq % nkv || nq / nkv > kPagedMaxGroup || head_dim <= 0 || head_dim > 256 || head_dim % 16) return 0;
    if (head_dim != 128 && head_dim != 256) return 16;
    size_t n;
    paged_ws(nullptr, head_dim, nkv, &n);
    return n;
}

// Steps of few rows per sequence.
template <int HD, bool I8, int NT>
__global__ void __launch_bounds__((kWave * kNarrowWaves), (kNarrowPerSimd<HD, I8, NT>)) paged_narrow_kernel(PagedAttnLaunch p, PagedWs ws) {
    extern __shared__ uint4 paged_lds[];
    narrow_block<HD, I8, kNarrowWaves, NT>(p, ws, blockIdx.x, paged_lds);
}
// Steps with longer ones.  Among the first blocks every fifth eight (one block on each XCD) are narrow ones, as many as there is
// work for: those wait for memory, the others for the matrix cores.  (Every fourth eight would all go to the same quarter
// of an XCD.)  Few wide blocks: every third, so that fewer blocks without work are launched (50
// sequences of up to 200 positions, one of 9 rows: 35 us, with every fifth 37; every second 42).
template <int HD, bool I8>
__global__ void __launch_bounds__(kWave* kBlockWaves<HD>, kBlockWaves<HD> / 4) paged_mixed_kernel(PagedAttnLaunch p, PagedWs ws, int turn) {
    extern __shared__ uint4 paged_lds[];
    const int b = blockIdx.x, all = ws.head[2];
    const int at = b % turn - (turn - 8), n = b / turn * 8 + max(0, at);  // narrow ones before this, if they do not end
    if (at >= 0 && n < all) {
        if (ws.narrow_cols == 8)
            narrow_block<HD, I8, kBlockWaves<HD>, 1>(p, ws, n, paged_lds);
        else
            narrow_block<HD, I8, kBlockWaves<HD>, 2>(p, ws, n, paged_lds);
    } else if (HD == 128 && ws.head[3] == kMostCols) {
        if constexpr (HD == 128) wide_block<HD, I8, kMostCols / kTTile>(p, ws, b - min(n, all), paged_lds);
    } else {
        wide_block<HD, I8, kLeastCols / kTTile>(p, ws, b - min(n, all), paged_lds);
    }
}

template <typename Kernel>
static hipError_t allow_lds(Kernel kernel, size_t bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

template <int HD>
constexpr size_t kWideLds = std::max(WideShape<HD, kLeastCols / kTTile>::kLds, WideShape<HD, (HD == 128 ? kMostCols : kLeastCols) / kTTile>::kLds);

template <int HD, bool I8, int NT>
static hipError_t launch_narrow(const PagedAttnLaunch& p, PagedWs& ws, hipStream_t s) {
    using F = PagedBlock<HD, kNarrowWaves, 8 * NT>;
    constexpr size_t kLds = std::max(F::kOutBytes, QueryStage<F, HD>::kBytes);
    ws.narrow_cols = 8 * NT;
    ws.narrow_rows = ws.narrow_cols / ws.group;
    ws.narrow_blocks = 256 * 4 * kNarrowPerSimd<HD, I8, NT> / kNarrowWaves;
    static_assert(256 * 4 * kNarrowPerSimd<HD, I8, NT> / kNarrowWaves <= kNarrowBlocks, "partial outputs");
    if (hipError_t e = allow_lds(&paged_narrow_kernel<HD, I8, NT>, kLds); e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_narrow_kernel<HD, I8, NT>), dim3(ws.narrow_blocks), dim3(F::kThreads), kLds, s, p, ws);
    return hipGetLastError();
}

template <int HD, bool I8>
static hipError_t launch_paged_heads(const PagedAttnLaunch& p, hipStream_t s) {
    const int nkv = p.kv.nkv, group = p.nq / nkv;
    const int64_t most = p.step.max_rows * static_cast<int64_t>(group);  // columns of a sequence
    PagedWs ws = paged_ws(p.ws, HD, nkv, nullptr);
    ws.group = group;
    ws.least_rows = kLeastCols / group;
    ws.most_rows = kMostCols / group;
    const size_t row_lds = paged_row_lds(group, HD);
    int wide_groups = 0;  // of merge blocks, one per kv head
    if (most > kNarrowCols) {
        ws.narrow_cols = group <= 8 ? 8 : 16;
        ws.narrow_rows = ws.narrow_cols / group;
        ws.narrow_blocks = 256;
        static_assert(kWideLds<HD> >= PagedBlock<HD, kBlockWaves<HD>, kNarrowCols>::kOutBytes, "narrow blocks among them");
        // row tiles of any division of the rows among the sequences, and the splits on top of them
        const int tiles = p.step.rows / (kLeastCols / group) + std::min(p.step.seqs, p.step.rows);
        const unsigned wide = static_cast<unsigned>(tiles + kWideBlocks / nkv) * nkv, narrow = ws.narrow_blocks;
        if (p.step.seqs <= kWave && tiles <= kPlanTiles)
            hipLaunchKernelGGL((paged_plan_kernel<HD, 1>), dim3(1), dim3(kWave), 0, s, p, ws);
        else
            hipLaunchKernelGGL((paged_plan_kernel<HD, 16>), dim3(1), dim3(16 * kWave), 0, s, p, ws);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        const unsigned every = wide >= 4 * narrow ? 5 : 3;
        if (hipError_t e = allow_lds(&paged_mixed_kernel<HD, I8>, kWideLds<HD>); e != hipSuccess) return e;
        hipLaunchKernelGGL((paged_mixed_kernel<HD, I8>), dim3(std::max(wide, (every - 1) * narrow) + narrow), dim3(kWave * kBlockWaves<HD>), kWideLds<HD>, s, p, ws, 8 * every);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        wide_groups = std::max(1, kWideBlocks / nkv);
    } else if (hipError_t e = most <= 8 ? launch_narrow<HD, I8, 1>(p, ws, s) : launch_narrow<HD, I8, 2>(p, ws, s); e != hipSuccess) {
        return e;
    }
    auto merge = [&](auto kernel) {
        if (hipError_t e = allow_lds(kernel, row_lds); e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, dim3(nkv, p.step.seqs + wide_groups), dim3(kMergeThreads), row_lds, s, p, ws);
        return hipGetLastError();
    };
    return wide_groups ? merge(&paged_merge_kernel<HD, true>) : merge(&paged_merge_kernel<HD, false>);
}

hipError_t launch_paged_attn(const PagedAttnLaunch& p, hipStream_t s) {
    const int hd = p.kv.head_dim;
    // the matrix-core kernels take rows in 16-byte pieces and their offsets within 64 rows in 32 bits
    const bool al = ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0 &&
                    p.q_stride % 4 == 0 && p.out_stride % 4 == 0 && p.q_stride < 1 << 21 && p.out_stride < 1 << 21;
    if (al && hd == 128) return p.kv.i8 ? launch_paged_heads<128, true>(p, s) : launch_paged_heads<128, false>(p, s);
    if (al && hd == 256) return p.kv.i8 ? launch_paged_heads<256, true>(p, s) : launch_paged_heads<256, false>(p, s);
    hipLaunchKernelGGL(paged_attn_row_kernel, dim3(p.step.rows, p.kv.nkv), dim3(256), paged_row_lds(p.nq / p.kv.nkv, hd), s, p);
    return hipGetLastError();
}

}  // namespace xqhip
