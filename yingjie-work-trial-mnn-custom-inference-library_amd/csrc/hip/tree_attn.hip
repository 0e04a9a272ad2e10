// tree_attn.hip - attention of a decode step's rows (a tree of drafted tokens,
// or a prompt chunk) over an fp16 or 8-bit key/value cache.
#include <algorithm>

#include <type_traits>

#include "xqhip_common.hpp"
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
// Matrix-core form, heads of 128 and 256 dims.  A block takes 32 CT columns of
// one kv head and one split of its keys, a column being one (row, query head)
// pair: column c is head c / T of the kv head's `group` and row t0 + c % T, T =
// 32 CT / group.  CT x KS waves: wave (ct, ks) owns the 32 columns of tile ct
// and every KS-th 32-key tile, with its own running max, sum and output, merged
// through LDS at the end.  K and V are staged chunk by chunk (32 KS keys, shared
// by all column tiles) as fp16 in LDS; an 8-bit cache's codes become fp16
// integers there, exactly, and the scales enter as factors of the scores and
// of the weights.
//
// Scores are formed transposed, S^T = K Q^T (keys are the MFMA rows): lane l
// holds column l & 31 and the keys 8 (v / 4) + 4 (l >> 5) + v % 4 of its tile,
// so its weights are already the B operand of O^T = V^T P^T.  V stays
// [key][dim]; ds_read_tr16_b64 hands each lane four keys of its dim.
//
// Precision: q (scaled per column by a power of two to [2^12, 2^13)) and the
// weights (times 2^6, within 2^6 of the column's running max) are split into
// fp16 hi + lo, 22 bits together; fp32 accumulation.  One fp16 each would leave
// errors of 2^-12 of the weights, where the caches' own values are exact.  An
// 8-bit V's weights carry its scale over a power of two R at or above the
// split's largest scale (moved when one outgrows it), so they stay in fp16's
// range: the output is off by 2^-31 sqrt(keys) of the largest |v| at most.
//
// A masked key has weight 0, but 0 times an infinity is not 0, and neither hi +
// lo nor the finite start of the running max can carry infinities.  Where that
// happens a sum is not finite or the weights sum to 0: the block that writes
// such an output computes its rows again by attend_row.
// ---------------------------------------------------------------------------
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));
constexpr int kTTile = 32;  // keys and columns of an MFMA tile
constexpr int kTreeMaxSplits = 64;

template <int HD, bool I8, int CT, int KS, int BUFS = 1>
struct TreeTile {
    static constexpr int kThreads = kWave * CT * KS;
    static constexpr int kCols = kTTile * CT, kKeys = kTTile * KS;
    static constexpr int kLdk = HD + 8;   // halves per K row: 16-byte rows shifted by 4 banks
    static constexpr int kLdv = HD + 16;  // halves per V row: the 4 rows of a transposed read in distinct banks
    static constexpr int kLdo = HD + 4;   // floats per column of a wave's output
    static constexpr int kPieceDims = I8 ? 16 : 8;  // values of a 16-byte piece
    static constexpr int kRowPieces = HD / kPieceDims;
    static constexpr int kPieces = kKeys * kRowPieces / kThreads;  // pieces of K (or V) per thread and chunk
    static constexpr int kKeyStep = kThreads / kRowPieces;
    static constexpr int kQuads = HD / 4;                 // float4 of an output row
    static constexpr int kMergeCols = kThreads / kQuads;  // columns per pass of the merge
    static constexpr int kPasses = kCols / kMergeCols;
    // scales of K and V, then each wave's V scales over its R
    static constexpr size_t kScaleBytes = !I8 ? 0 : BUFS == 1 ? static_cast<size_t>(kKeys) * 2 * 4 + static_cast<size_t>(CT * KS) * kTTile * 4
                                                              : static_cast<size_t>(BUFS) * (2 * kKeys + KS) * 4;
    static constexpr size_t kKvBytes = static_cast<size_t>(BUFS) * kKeys * (kLdk + kLdv) * 2 + kScaleBytes;
    static constexpr size_t kOutBytes = static_cast<size_t>(CT * KS) * kTTile * (kLdo + 2) * 4;
    static constexpr size_t kLds = kKvBytes > kOutBytes ? kKvBytes : kOutBytes;
    static_assert(kPieces * kThreads == kKeys * kRowPieces && kPieces > 0, "K / V staging");
    static_assert(kPasses * kThreads == kCols * kQuads, "merge");
    static_assert(!I8 || 2 * kKeys <= kThreads, "one scale per thread");
    static_assert(kLds + 64 <= 160 * 1024, "LDS");
    static_assert(BUFS > 1 || static_cast<size_t>(kKeys) * kLdk * 2 + static_cast<size_t>(kCols) * kLdo * 4 <= kLds, "q fits behind K");
    static_assert(static_cast<size_t>(kCols) * kLdo * 4 <= kLds, "q fits");
    static_assert(kLds >= tree_row_lds(kTreeMaxGroup, HD) * 4, "the general form runs in it");
};

__device__ __forceinline__ float pair32_max(float v) {  // of v[l] and v[l ^ 32]
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
                 __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}

// fp32 -> fp16 hi + fp16 lo (x - hi) of 8 values
__device__ __forceinline__ void split8(const float (&x)[8], half8& hi, half8& lo) {
    typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f2 v = {x[e], x[e + 1]};
        const h2 h = __builtin_convertvector(v, h2);
        hi[e] = h[0];
        hi[e + 1] = h[1];
        const f2 d = {x[e] - static_cast<float>(h[0]), x[e + 1] - static_cast<float>(h[1])};
        const h2 l = __builtin_convertvector(d, h2);
        lo[e] = l[0];
        lo[e + 1] = l[1];
    }
}

// four signed 8-bit codes as fp16 integers: 0x6400 | (c + 128) is 1152 + c
__device__ __forceinline__ u32x2 codes_to_half(uint32_t c) {
    c ^= 0x80808080u;
    const h2 bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const h2 a = as_h2(__builtin_amdgcn_perm(0x64646464u, c, 0x04010400u)) + bias;
    const h2 b = as_h2(__builtin_amdgcn_perm(0x64646464u, c, 0x04030402u)) + bias;
    return u32x2{as_u32(a), as_u32(b)};
}

// bits b .. b + 31 of a row's mask, with the context (negative positions) visible
__device__ __forceinline__ uint32_t mask_window(uint64_t m, int b) {
    if (b <= -32) return ~0u;
    if (b < 0) return static_cast<uint32_t>(m) << -b | ((1u << -b) - 1u);
    return b < 64 ? static_cast<uint32_t>(m >> b) : 0u;
}

struct TreeGrid {
    int tiles, splits;  // row tiles, key splits
};

// key chunks [begin, end) of split s of `chunks`: the first min(splits, chunks) splits have some
__device__ __forceinline__ void split_range(int chunks, int splits, int s, int& begin, int& end) {
    const int n = min(splits, chunks), per = chunks / n, more = chunks - per * n;
    begin = s * per + min(s, more);
    end = s < n ? begin + per + (s < more ? 1 : 0) : begin;
}

template <int HD, bool I8, int CT, int KS>
__global__ void __launch_bounds__(kWave* CT* KS, (CT * KS + 3) / 4) tree_attn_mfma_kernel(TreeAttnLaunch p, TreeGrid grid) {
    using F = TreeTile<HD, I8, CT, KS>;
    constexpr int kSteps = HD / 16, kDimTiles = HD / 32;
    constexpr float kLog2e = 1.44269504088896340736f;
    constexpr float kRaise = 6.0f;  // weights are held times 2^kRaise
    constexpr float kSlack = 6.0f;  // the max may outgrow the reference by 2^kSlack before it is moved
    constexpr float kScaleSlack = 8.0f;
    extern __shared__ uint4 flash_lds[];
    __shared__ int redo;
    _Float16* Kl = reinterpret_cast<_Float16*>(flash_lds);  // [kKeys][kLdk]
    _Float16* Vl = Kl + F::kKeys * F::kLdk;                 // [kKeys][kLdv]
    float* Sl = reinterpret_cast<float*>(Vl + F::kKeys * F::kLdv);  // [2][kKeys] scales of K, V
    // the kv heads of a tile are neighbours in launch order (8 heads: an XCD each), then the row tiles of the
    // same keys, so that a head's blocks read its K / V from one L2
    const int nkv = p.kv.nkv, kh = blockIdx.x % nkv;
    const int rest = static_cast<int>(blockIdx.x) / nkv, tile = grid.tiles - 1 - rest % grid.tiles, sp = rest / grid.tiles;
    const int group = p.nq / nkv, T = F::kCols / group;
    const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int ct = wid % CT, ks = wid / CT;
    const int cl = lane & 31, g = lane >> 5;
    const int pos0 = __builtin_amdgcn_readfirstlane(clamp_pos0(p));
    const uint32_t inv_t = (65535u + T) / T;  // c / T = c inv_t >> 16 for c < 128, T <= 128
    const int t0 = tile * T, ntok = min(T, p.tokens - t0);
    const int col = ct * kTTile + cl, ch = static_cast<int>(col * inv_t >> 16), ctok = col - ch * T;
    const bool live = ch < group && ctok < ntok;
    const int last = min(pos0 + (p.has_tree ? p.tokens : t0 + ntok), p.kv.capacity) - 1;  // any column's last key
    const int sure = p.has_tree ? pos0 - 1 : pos0 + t0;  // every column sees the keys up to here
    const int qpos = live ? pos0 + t0 + ctok : -1;
    const uint64_t mask = live && p.has_tree ? p.masks.m[t0 + ctok] : 0;
    int begin, end;
    split_range(last / F::kKeys + 1, grid.splits, sp, begin, end);
    begin = __builtin_amdgcn_readfirstlane(begin);
    end = __builtin_amdgcn_readfirstlane(end);
    if (begin >= end) return;  // fewer chunks than splits (or no key at all: the merge sees to it)

    const uint32_t es = I8 ? 1u : 2u, krow = static_cast<uint32_t>(nkv) * HD * es;  // bytes per cache position
    const int pk = threadIdx.x / F::kRowPieces, pd = threadIdx.x % F::kRowPieces;
    u32x4 kr[F::kPieces], vr[F::kPieces];
    auto load = [&](const void* cache, int c0, u32x4 (&r)[F::kPieces]) {  // keys past `last` read 0
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
    const bool k_half = threadIdx.x < F::kKeys;
    float sr = 0.0f;
    auto load_scale = [&](int c0) {
        if constexpr (I8) {
            const int key = threadIdx.x % F::kKeys;
            if (threadIdx.x < 2 * F::kKeys)
                sr = c0 + key <= last ? (k_half ? p.kv.k_scale : p.kv.v_scale)[static_cast<size_t>(c0 + key) * nkv + kh] : 0.0f;
        }
    };
    auto store_scale = [&](bool k) {
        if constexpr (I8)
            if (threadIdx.x < 2 * F::kKeys && k_half == k) Sl[threadIdx.x] = sr;
    };
    // rows of q, the gate and the output: thread i takes float4 i % kQuads of columns i / kQuads, + kMergeCols, ...
    auto place = [&](int tid, int u, int stride) {  // float offset of the pass's column from row t0, or -1
        const int c = tid / F::kQuads + u * F::kMergeCols;
        const int hc = static_cast<int>(c * inv_t >> 16), tc = c - hc * T;
        return hc < group && tc < ntok ? tc * stride + (kh * group + hc) * HD + 4 * (tid % F::kQuads) : -1;
    };
    u32x4 qr[F::kPasses];
    {
        const __amdgpu_buffer_rsrc_t rq =
            buf_rsrc(p.q + static_cast<size_t>(t0) * p.q_stride, static_cast<uint32_t>(ntok) * p.q_stride * 4u);
#pragma unroll
        for (int u = 0; u < F::kPasses; ++u) {  // columns without a row read 0
            const int at = place(threadIdx.x, u, p.q_stride);
            qr[u] = __builtin_amdgcn_raw_buffer_load_b128(rq, at >= 0 ? static_cast<uint32_t>(at) * 4u : kBufOOB, 0, 0);
        }
    }
    load(p.kv.k, begin * F::kKeys, kr);
    load_scale(begin * F::kKeys);
    float* Ql = reinterpret_cast<float*>(Vl);  // [kCols][kLdo]
#pragma unroll
    for (int u = 0; u < F::kPasses; ++u)
        *reinterpret_cast<u32x4*>(Ql + (threadIdx.x / F::kQuads + u * F::kMergeCols) * F::kLdo +
                                  4 * (threadIdx.x % F::kQuads)) = qr[u];
    store(Kl, F::kLdk, kr);
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
    half8 qhi[kSteps], qlo[kSteps];  // lane supplies dims 16 s + 8 g .. + 7 of its column
    float sscale;                    // score scale in the exponent of 2
    {
        float x[kSteps][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 v = *reinterpret_cast<const float4*>(Ql + col * F::kLdo + 16 * s + 8 * g + e);
                x[s][e] = v.x;
                x[s][e + 1] = v.y;
                x[s][e + 2] = v.z;
                x[s][e + 3] = v.w;
            }
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[s][e]));
        mx = pair32_max(mx);
        // a power of two brings the column's largest magnitude into [2^12, 2^13); an infinity or 0 stays
        int ex = 13;
        if (mx > 0.0f && mx < INFINITY) frexpf(mx, &ex);
        ex = max(ex, -100);  // 2^(13 - ex) stays finite
        const float down = ldexpf(1.0f, 13 - ex);
        sscale = ldexpf(kLog2e / sqrtf(static_cast<float>(HD)), ex - 13);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] *= down;
            split8(x[s], qhi[s], qlo[s]);
        }
    }
    __syncthreads();  // every wave has its q: V (and the scales behind it) may take its place
    store_scale(true);
    store_scale(false);
    __syncthreads();
    float m = -1.0e30f, l = 0.0f;  // reference of the exponents, this lane's part of the sum
    float R = 0.0f;                // 8-bit V: the weights' scales are held over R (a power of two)
    floatx16 o[kDimTiles];
#pragma unroll
    for (int j = 0; j < kDimTiles; ++j) o[j] = floatx16{};
    for (int c = begin; c < end; ++c) {  // block-uniform
        const int c0 = c * F::kKeys;
        load(p.kv.v, c0, vr);
        const int key0 = c0 + ks * kTTile;
        const bool any = key0 <= last;  // wave-uniform: this wave's tile holds a key
        half8 phi[2], plo[2];
        if (any) {
            floatx16 st = floatx16{};
            const _Float16* krow_l = Kl + (ks * kTTile + cl) * F::kLdk + 8 * g;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const half8 a = *reinterpret_cast<const half8*>(krow_l + 16 * s);
                st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qlo[s], st, 0, 0, 0);
                st = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qhi[s], st, 0, 0, 0);
            }
            float sc[16], vs[16], mc = -INFINITY;
            if constexpr (I8) {
                // V's scales of the tile over R; R moves (rarely after the first tile) when one outgrows it
                const float mine = Sl[F::kKeys + ks * kTTile + cl];
                const float top = wave_max(mine);
                if (top > R * kScaleSlack) {
                    int ex;
                    frexpf(top, &ex);
                    const float to = top < INFINITY ? ldexpf(1.0f, min(ex, 127)) : R;
                    const float f = R > 0.0f ? R / to : 0.0f;
#pragma unroll
                    for (int j = 0; j < kDimTiles; ++j) o[j] *= f;
                    R = to;
                }
                float* over = Sl + 2 * F::kKeys + wid * kTTile;
                over[cl] = R > 0.0f ? mine / R : mine;
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    typedef float f32x4 __attribute__((ext_vector_type(4)));
                    const f32x4 k4 = *reinterpret_cast<const f32x4*>(Sl + ks * kTTile + 8 * a + 4 * g);
                    const f32x4 v4 = *reinterpret_cast<const f32x4*>(over + 8 * a + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[4 * a + e] = st[4 * a + e] * k4[e];
                        vs[4 * a + e] = v4[e];
                    }
                }
            } else {
#pragma unroll
                for (int v = 0; v < 16; ++v) sc[v] = st[v];
            }
            if (key0 + kTTile - 1 > sure || key0 + kTTile - 1 > last) {  // wave-uniform: keys that some column does not see
                uint32_t see;
                if (p.has_tree) {
                    see = mask_window(mask, key0 + 4 * g - pos0);
                } else {
                    const int b = qpos - (key0 + 4 * g);
                    see = b < 0 ? 0u : (b >= 31 ? ~0u : (2u << b) - 1u);
                }
                const int left = last - (key0 + 4 * g);  // (tree rows and positions past the capacity)
                see &= left < 0 ? 0u : (left >= 31 ? ~0u : (2u << left) - 1u);
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (!(see >> (8 * (v >> 2) + (v & 3)) & 1u)) {
                        sc[v] = -INFINITY;
                        if constexpr (I8) vs[v] = 0.0f;  // (its scale may be NaN)
                    }
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) mc = fmaxf(mc, sc[v]);
            mc = pair32_max(mc) * sscale;
            // the reference moves only when a column's max has outgrown it (rarely after the first tiles)
            const bool up = mc > m + kSlack;
            if (__builtin_amdgcn_ballot_w64(up)) {
                const float to = up ? mc : m, f = exp2f(m - to);
                m = to;
                l *= f;
#pragma unroll
                for (int j = 0; j < kDimTiles; ++j) o[j] *= f;
            }
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
        }
        store(Vl, F::kLdv, vr);
        const bool more = c + 1 < end;  // block-uniform
        if (more) {
            load(p.kv.k, c0 + F::kKeys, kr);
            load_scale(c0 + F::kKeys);
        }
        __syncthreads();  // V is staged; every wave has read K and the scales
        if (any) {
            // transposed reads: 16 lanes cover four keys x 16 dims, lane i gets dim i of the four
            const _Float16* vb = Vl + (ks * kTTile + 4 * g + ((lane & 15) >> 2)) * F::kLdv + (lane & 16) + 4 * (lane & 3);
#pragma unroll
            for (int j = 0; j < kDimTiles; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    typedef __attribute__((address_space(3))) short4_t lds_s4;
                    const _Float16* q0 = vb + 16 * h * F::kLdv + 32 * j;
                    const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q0));
                    const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q0 + 8 * F::kLdv));
                    const half8 a = __builtin_bit_cast(half8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, phi[h], o[j], 0, 0, 0);
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, plo[h], o[j], 0, 0, 0);
                }
        }
        if (more) {
            store(Kl, F::kLdk, kr);
            store_scale(true);
            store_scale(false);
        }
        __syncthreads();  // the next K is staged; every wave has read V
    }
    // merge the key waves of each column tile that had a key: outputs, then (reference, sum)
    const int key_waves = min(KS, (last - begin * F::kKeys) / kTTile + 1);
    float* Ol = reinterpret_cast<float*>(flash_lds);  // [waves][32][kLdo]
    float* Ml = Ol + CT * KS * kTTile * F::kLdo;      // [waves][32][2]
    l = xor_pair_sum<32>(l);
    const float back = I8 ? R : 1.0f;
    if (ks < key_waves) {
        float* oc = Ol + (wid * kTTile + cl) * F::kLdo + 4 * g;
#pragma unroll
        for (int j = 0; j < kDimTiles; ++j)
#pragma unroll
            for (int a = 0; a < 4; ++a)
                *reinterpret_cast<float4*>(oc + 32 * j + 8 * a) =
                    make_float4(o[j][4 * a] * back, o[j][4 * a + 1] * back, o[j][4 * a + 2] * back, o[j][4 * a + 3] * back);
        if (g == 0) *reinterpret_cast<float2*>(Ml + (wid * kTTile + cl) * 2) = make_float2(m, l);
    }
    __syncthreads();
    const bool whole = grid.splits == 1;  // this block has all the keys of its rows
    const __amdgpu_buffer_rsrc_t rg = buf_rsrc(p.gate ? p.gate + static_cast<size_t>(t0) * p.q_stride : p.q,
                                               p.gate ? static_cast<uint32_t>(ntok) * p.q_stride * 4u : 0u);
    float* po = p.ws + static_cast<size_t>(sp) * p.tokens * p.nq * HD;
    float2* pm = reinterpret_cast<float2*>(p.ws + static_cast<size_t>(grid.splits) * p.tokens * p.nq * HD) +
                 static_cast<size_t>(sp) * p.tokens * p.nq;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < F::kPasses; ++u) {
        const int c = threadIdx.x / F::kQuads + u * F::kMergeCols;
        const int hc = static_cast<int>(c * inv_t >> 16), tc = c - hc * T;
        if (hc >= group || tc >= ntok) continue;
        const int at = tc * p.out_stride + (kh * group + hc) * HD + 4 * (threadIdx.x % F::kQuads);
        const int gat = tc * p.q_stride + (kh * group + hc) * HD + 4 * (threadIdx.x % F::kQuads);
        const int w0 = (c / kTTile) * kTTile + (c % kTTile);  // column c of wave (ct, ks): w0 + ks CT 32
        float ml[KS], ll[KS], M = -INFINITY;
#pragma unroll
        for (int s = 0; s < KS; ++s)
            if (s < key_waves) {
                const float2 v = *reinterpret_cast<const float2*>(Ml + (w0 + s * F::kCols) * 2);
                ml[s] = v.x;
                ll[s] = v.y;
                M = fmaxf(M, v.x);
            }
        float L = 0.0f;
        float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int s = 0; s < KS; ++s)
            if (s < key_waves) {
                const float f = exp2f(ml[s] - M);
                const float4 v = *reinterpret_cast<const float4*>(Ol + (w0 + s * F::kCols) * F::kLdo + 4 * (threadIdx.x % F::kQuads));
                L += f * ll[s];
                r.x += f * v.x;
                r.y += f * v.y;
                r.z += f * v.z;
                r.w += f * v.w;
            }
        if (!whole) {
            const size_t row = static_cast<size_t>(t0 + tc) * p.nq + kh * group + hc;
            *reinterpret_cast<float4*>(po + row * HD + 4 * (threadIdx.x % F::kQuads)) = r;
            if (threadIdx.x % F::kQuads == 0) pm[row] = make_float2(M, L);
            continue;
        }
        const u32x4 gt = __builtin_amdgcn_raw_buffer_load_b128(rg, static_cast<uint32_t>(gat) * 4u, 0, 0);
        const float inv = L > 0.0f ? 1.0f / L : 0.0f;
        bad |= !(L > 0.0f && fabsf(r.x) + fabsf(r.y) + fabsf(r.z) + fabsf(r.w) < INFINITY);
        float4 y = make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
        if (p.gate) {
            y.x *= sigmoid_dev(__uint_as_float(gt[0]));
            y.y *= sigmoid_dev(__uint_as_float(gt[1]));
            y.z *= sigmoid_dev(__uint_as_float(gt[2]));
            y.w *= sigmoid_dev(__uint_as_float(gt[3]));
        }
        *reinterpret_cast<float4*>(p.out + static_cast<size_t>(t0) * p.out_stride + at) = y;
    }
    if (!whole) return;
    if (bad) redo = 1;
    __syncthreads();
    if (__builtin_expect(!redo, 1)) return;  // block-uniform
    for (int t = t0; t < t0 + ntok; ++t) {
        __syncthreads();
        attend_row<F::kThreads, I8>(p, t, kh, reinterpret_cast<float*>(flash_lds));
    }
}

// max over aligned groups of 32 lanes
__device__ __forceinline__ float half_max(float v) {
    v = lanes_max<16>(v);
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}

template <int HD, bool I8, int CT, int KS>
__global__ void __launch_bounds__(kWave* CT* KS, (CT * KS + 3) / 4) tree_attn_wide_kernel(TreeAttnLaunch p, TreeGrid grid) {
    using F = TreeTile<HD, I8, CT, KS, 2>;
    constexpr int kSteps = HD / 16, kDimTiles = HD / 32;
    constexpr float kLog2e = 1.44269504088896340736f;
    constexpr float kRaise = 6.0f;  // weights are held times 2^kRaise
    constexpr float kSlack = 6.0f;  // the max may outgrow the reference by 2^kSlack before it is moved
    extern __shared__ uint4 flash_lds[];
    __shared__ int redo;
    constexpr int kKBuf = F::kKeys * F::kLdk, kVBuf = F::kKeys * F::kLdv, kSBuf = 2 * F::kKeys + KS;
    _Float16* Kl = reinterpret_cast<_Float16*>(flash_lds);       // [2][kKeys][kLdk]
    _Float16* Vl = Kl + 2 * kKBuf;                               // [2][kKeys][kLdv]
    float* Sl = reinterpret_cast<float*>(Vl + 2 * kVBuf);        // [2]: scales of K, of V, exponent of V's per key tile
    const int nkv = p.kv.nkv, kh = blockIdx.x % nkv;
    const int rest = static_cast<int>(blockIdx.x) / nkv, tile = grid.tiles - 1 - rest % grid.tiles, sp = rest / grid.tiles;
    const int group = p.nq / nkv, T = F::kCols / group;
    const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int ct = wid % CT, ks = wid / CT;
    const int cl = lane & 31, g = lane >> 5;
    const int pos0 = __builtin_amdgcn_readfirstlane(clamp_pos0(p));
    const uint32_t inv_t = (65535u + T) / T;  // c / T = c inv_t >> 16 for c < 128, T <= 128
    const int t0 = tile * T, ntok = min(T, p.tokens - t0);
    const int col = ct * kTTile + cl, ch = static_cast<int>(col * inv_t >> 16), ctok = col - ch * T;
    const bool live = ch < group && ctok < ntok;
    const int last = min(pos0 + (p.has_tree ? p.tokens : t0 + ntok), p.kv.capacity) - 1;  // any column's last key
    const int sure = min(p.has_tree ? pos0 - 1 : pos0 + t0, last);  // every column sees the keys up to here
    const int qpos = live ? pos0 + t0 + ctok : -1;
    const uint64_t mask = live && p.has_tree ? p.masks.m[t0 + ctok] : 0;
    int begin, end;
    split_range(last / F::kKeys + 1, grid.splits, sp, begin, end);
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
    // scales: thread i < kKeys holds K's of key i, the next kKeys threads V's, of which each 32-key tile's exponent
    // goes along (0 for a tile of zeros)
    float sr = 0.0f;
    auto load_scale = [&](int c) {
        if constexpr (I8) {
            const int key = c * F::kKeys + static_cast<int>(threadIdx.x) % F::kKeys;
            const float* from = threadIdx.x < F::kKeys ? p.kv.k_scale : p.kv.v_scale;
            sr = threadIdx.x < 2 * F::kKeys && key <= last ? from[static_cast<size_t>(key) * nkv + kh] : 0.0f;
        }
    };
    auto store_scale = [&](int buf) {
        if constexpr (I8) {
            if (threadIdx.x >= 2 * F::kKeys) return;  // wave-uniform
            float* at = Sl + buf * kSBuf;
            at[threadIdx.x] = sr;
            if (threadIdx.x < F::kKeys) return;
            const float top = half_max(sr);
            int ex = 0;
            if (top > 0.0f) frexpf(top, &ex);
            if (lane % kTTile == 0) at[2 * F::kKeys + (threadIdx.x - F::kKeys) / kTTile] = fminf(fmaxf(ex, -100.0f), 100.0f);
        }
    };
    auto place = [&](int tid, int u, int stride) {  // float offset of the pass's column from row t0, or -1
        const int c = tid / F::kQuads + u * F::kMergeCols;
        const int hc = static_cast<int>(c * inv_t >> 16), tc = c - hc * T;
        return hc < group && tc < ntok ? tc * stride + (kh * group + hc) * HD + 4 * (tid % F::kQuads) : -1;
    };
    load(p.kv.k, begin, kr);
    load_scale(begin);
    load(p.kv.v, begin, vr);
    half8 qhi[kSteps], qlo[kSteps];  // lane supplies dims 16 s + 8 g .. + 7 of its column
    float sscale;                    // score scale in the exponent of 2
    {
        float* Ql = reinterpret_cast<float*>(flash_lds);  // [kCols][kLdo]
        const __amdgpu_buffer_rsrc_t rq =
            buf_rsrc(p.q + static_cast<size_t>(t0) * p.q_stride, static_cast<uint32_t>(ntok) * p.q_stride * 4u);
        u32x4 qr[F::kPasses];
#pragma unroll
        for (int u = 0; u < F::kPasses; ++u) {  // columns without a row read 0
            const int at = place(threadIdx.x, u, p.q_stride);
            qr[u] = __builtin_amdgcn_raw_buffer_load_b128(rq, at >= 0 ? static_cast<uint32_t>(at) * 4u : kBufOOB, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < F::kPasses; ++u)
            *reinterpret_cast<u32x4*>(Ql + (threadIdx.x / F::kQuads + u * F::kMergeCols) * F::kLdo +
                                      4 * (threadIdx.x % F::kQuads)) = qr[u];
        if (threadIdx.x == 0) redo = 0;
        __syncthreads();
        float x[kSteps][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 v = *reinterpret_cast<const float4*>(Ql + col * F::kLdo + 16 * s + 8 * g + e);
                x[s][e] = v.x;
                x[s][e + 1] = v.y;
                x[s][e + 2] = v.z;
                x[s][e + 3] = v.w;
            }
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[s][e]));
        mx = pair32_max(mx);
        // a power of two brings the column's largest magnitude into [2^12, 2^13); an infinity or 0 stays
        int ex = 13;
        if (mx > 0.0f && mx < INFINITY) frexpf(mx, &ex);
        ex = max(ex, -100);  // 2^(13 - ex) stays finite
        const float down = ldexpf(1.0f, 13 - ex);
        sscale = ldexpf(kLog2e / sqrtf(static_cast<float>(HD)), ex - 13);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] *= down;
            split8(x[s], qhi[s], qlo[s]);
        }
        __syncthreads();  // every wave has its q: K and V may take its place
    }
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
        float sc[16], vs[16], mc = -INFINITY, ev = 0.0f;
        if constexpr (I8) {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            const float* at = Sl + (c & 1) * kSBuf;
            ev = at[2 * F::kKeys + ks];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const f32x4 k4 = *reinterpret_cast<const f32x4*>(at + ks * kTTile + 8 * a + 4 * g);
                const f32x4 v4 = *reinterpret_cast<const f32x4*>(at + F::kKeys + ks * kTTile + 8 * a + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[4 * a + e] = st[4 * a + e] * k4[e];
                    vs[4 * a + e] = v4[e];
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
        for (int v = 0; v < 16; ++v) mc = fmaxf(mc, sc[v]);
        mc = pair32_max(mc) * sscale + ev;
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
    // merge the key waves of each column tile: outputs, then (reference, sum)
    float* Ol = reinterpret_cast<float*>(flash_lds);  // [waves][32][kLdo]
    float* Ml = Ol + CT * KS * kTTile * F::kLdo;      // [waves][32][2]
    l = xor_pair_sum<32>(l);
    {
        float* oc = Ol + (wid * kTTile + cl) * F::kLdo + 4 * g;
#pragma unroll
        for (int j = 0; j < kDimTiles; ++j)
#pragma unroll
            for (int a = 0; a < 4; ++a)
                *reinterpret_cast<float4*>(oc + 32 * j + 8 * a) =
                    make_float4(o[j][4 * a], o[j][4 * a + 1], o[j][4 * a + 2], o[j][4 * a + 3]);
        if (g == 0) *reinterpret_cast<float2*>(Ml + (wid * kTTile + cl) * 2) = make_float2(m, l);
    }
    __syncthreads();
    const bool whole = grid.splits == 1;  // this block has all the keys of its rows
    const __amdgpu_buffer_rsrc_t rg = buf_rsrc(p.gate ? p.gate + static_cast<size_t>(t0) * p.q_stride : p.q,
                                               p.gate ? static_cast<uint32_t>(ntok) * p.q_stride * 4u : 0u);
    float* po = p.ws + static_cast<size_t>(sp) * p.tokens * p.nq * HD;
    float2* pm = reinterpret_cast<float2*>(p.ws + static_cast<size_t>(grid.splits) * p.tokens * p.nq * HD) +
                 static_cast<size_t>(sp) * p.tokens * p.nq;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < F::kPasses; ++u) {
        const int cc = threadIdx.x / F::kQuads + u * F::kMergeCols;
        const int hc = static_cast<int>(cc * inv_t >> 16), tc = cc - hc * T;
        if (hc >= group || tc >= ntok) continue;
        const int at = tc * p.out_stride + (kh * group + hc) * HD + 4 * (threadIdx.x % F::kQuads);
        const int gat = tc * p.q_stride + (kh * group + hc) * HD + 4 * (threadIdx.x % F::kQuads);
        const int w0 = (cc / kTTile) * kTTile + (cc % kTTile);  // column cc of wave (ct, ks): w0 + ks CT 32
        float ml[KS], ll[KS], M = -INFINITY;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const float2 v = *reinterpret_cast<const float2*>(Ml + (w0 + s * F::kCols) * 2);
            ml[s] = v.x;
            ll[s] = v.y;
            M = fmaxf(M, v.x);
        }
        float L = 0.0f;
        float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const float f = exp2f(ml[s] - M);
            const float4 v = *reinterpret_cast<const float4*>(Ol + (w0 + s * F::kCols) * F::kLdo + 4 * (threadIdx.x % F::kQuads));
            L += f * ll[s];
            r.x += f * v.x;
            r.y += f * v.y;
            r.z += f * v.z;
            r.w += f * v.w;
        }
        if (!whole) {
            const size_t row = static_cast<size_t>(t0 + tc) * p.nq + kh * group + hc;
            *reinterpret_cast<float4*>(po + row * HD + 4 * (threadIdx.x % F::kQuads)) = r;
            if (threadIdx.x % F::kQuads == 0) pm[row] = make_float2(M, L);
            continue;
        }
        const u32x4 gt = __builtin_amdgcn_raw_buffer_load_b128(rg, static_cast<uint32_t>(gat) * 4u, 0, 0);
        const float inv = L > 0.0f ? 1.0f / L : 0.0f;
        bad |= !(L > 0.0f && fabsf(r.x) + fabsf(r.y) + fabsf(r.z) + fabsf(r.w) < INFINITY);
        float4 y = make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
        if (p.gate) {
            y.x *= sigmoid_dev(__uint_as_float(gt[0]));
            y.y *= sigmoid_dev(__uint_as_float(gt[1]));
            y.z *= sigmoid_dev(__uint_as_float(gt[2]));
            y.w *= sigmoid_dev(__uint_as_float(gt[3]));
        }
        *reinterpret_cast<float4*>(p.out + static_cast<size_t>(t0) * p.out_stride + at) = y;
    }
    if (!whole) return;
    if (bad) redo = 1;
    __syncthreads();
    if (__builtin_expect(!redo, 1)) return;  // block-uniform
    for (int t = t0; t < t0 + ntok; ++t) {
        __syncthreads();
        attend_row<F::kThreads, I8>(p, t, kh, reinterpret_cast<float*>(flash_lds));
    }
}

// The splits' partial outputs of one row and kv head joined, normalised and gated.
template <int HD, bool I8, int KEYS>
__global__ void __launch_bounds__(256) tree_attn_merge_kernel(TreeAttnLaunch p, TreeGrid grid, int T) {
    extern __shared__ float smem[];  // attend_row's
    __shared__ float2 stat[kTreeMaxSplits * kTreeMaxGroup];
    __shared__ int redo;
    const int t = blockIdx.x, kh = blockIdx.y, group = p.nq / p.kv.nkv, t0 = t / T * T;
    const int pos0 = clamp_pos0(p);
    const int last = min(pos0 + (p.has_tree ? p.tokens : min(t0 + T, p.tokens)), p.kv.capacity) - 1;
    const int splits = last < 0 ? 0 : min(grid.splits, last / KEYS + 1);
    const size_t rows = static_cast<size_t>(p.tokens) * p.nq, row0 = static_cast<size_t>(t) * p.nq + kh * group;
    const float2* pm = reinterpret_cast<const float2*>(p.ws + grid.splits * rows * HD);
    for (int i = threadIdx.x; i < splits * group; i += 256) stat[i] = pm[(i / group) * rows + row0 + i % group];
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
    bool bad = false;
    for (int i = threadIdx.x; i < group * HD / 4; i += 256) {
        const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
        float M = -INFINITY, L = 0.0f;
        for (int s = 0; s < splits; ++s) M = fmaxf(M, stat[s * group + h].x);
        float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float* po = p.ws + (row0 + h) * HD + d;
        for (int s = 0; s < splits; ++s) {
            const float2 st = stat[s * group + h];
            const float f = exp2f(st.x - M);
            const float4 v = *reinterpret_cast<const float4*>(po + s * rows * HD);
            L += f * st.y;
            r.x += f * v.x;
            r.y += f * v.y;
            r.z += f * v.z;
            r.w += f * v.w;
        }
        const float inv = L > 0.0f ? 1.0f / L : 0.0f;
        bad |= !(L > 0.0f && fabsf(r.x) + fabsf(r.y) + fabsf(r.z) + fabsf(r.w) < INFINITY);
        float4 y = make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
        if (p.gate) {
            const float4 gt = *reinterpret_cast<const float4*>(p.gate + static_cast<size_t>(t) * p.q_stride + (kh * group + h) * HD + d);
            y.x *= sigmoid_dev(gt.x);
            y.y *= sigmoid_dev(gt.y);
            y.z *= sigmoid_dev(gt.z);
            y.w *= sigmoid_dev(gt.w);
        }
        *reinterpret_cast<float4*>(p.out + static_cast<size_t>(t) * p.out_stride + (kh * group + h) * HD + d) = y;
    }
    if (bad) redo = 1;
    __syncthreads();
    if (redo) attend_row<256, I8>(p, t, kh, smem);  // block-uniform
}

bool tree_attn_supported(int nq, int nkv, int head_dim) {
    return nkv > 0 && nq > 0 && nq % nkv == 0 && nq / nkv <= kTreeMaxGroup && head_dim > 0 && head_dim <= 1024 &&
           sizeof(float) * tree_row_lds(nq / nkv, head_dim) <= 64 * 1024;
}

// The kernel of a call: column tiles of a block and key waves.
struct TreeShape {
    int ct, ks, keys;
};
static TreeShape tree_shape(int group, int hd, int tokens) {
    const int cols = tokens * group;
    if (cols <= kTTile) return hd == 128 ? TreeShape{1, 8, 256} : TreeShape{1, 4, 128};
    return hd == 128 ? TreeShape{2, 4, 128} : TreeShape{2, 2, 64};
}
// Row tiles, and key splits that give every CU a block.
static TreeGrid tree_grid(int nq, int nkv, int hd, int tokens) {
    const int T = kTTile * tree_shape(nq / nkv, hd, tokens).ct / (nq / nkv);
    const int tiles = (tokens + T - 1) / T;
    const int64_t blocks = static_cast<int64_t>(tiles) * nkv;
    return TreeGrid{tiles, static_cast<int>(std::min<int64_t>(kTreeMaxSplits, std::max<int64_t>(1, 256 / blocks)))};
}

size_t tree_attn_workspace_bytes(int nq, int nkv, int head_dim, int tokens) {
    if (head_dim != 128 && head_dim != 256) return 16;
    const TreeGrid g = tree_grid(nq, nkv, head_dim, tokens);
    return g.splits == 1 ? 16 : static_cast<size_t>(g.splits) * tokens * nq * (head_dim + 2) * sizeof(float);
}

template <typename F, int HD, bool I8, typename Kernel>
static hipError_t launch_tree(const TreeAttnLaunch& p, Kernel kernel, hipStream_t s) {
    const TreeGrid g = tree_grid(p.nq, p.kv.nkv, HD, p.tokens);
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(F::kLds));
        e != hipSuccess)
        return e;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(g.tiles * g.splits) * p.kv.nkv), dim3(F::kThreads), F::kLds, s, p, g);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || g.splits == 1) return e;
    const int group = p.nq / p.kv.nkv;
    hipLaunchKernelGGL((tree_attn_merge_kernel<HD, I8, F::kKeys>), dim3(p.tokens, p.kv.nkv), dim3(256),
                       sizeof(float) * tree_row_lds(group, HD), s, p, g, F::kCols / group);
    return hipGetLastError();
}
template <int HD, bool I8, int CT, int KS, bool WIDE>
static hipError_t launch_tree_mfma(const TreeAttnLaunch& p, hipStream_t s) {
    if constexpr (WIDE)
        return launch_tree<TreeTile<HD, I8, CT, KS, 2>, HD, I8>(p, &tree_attn_wide_kernel<HD, I8, CT, KS>, s);
    else
        return launch_tree<TreeTile<HD, I8, CT, KS>, HD, I8>(p, &tree_attn_mfma_kernel<HD, I8, CT, KS>, s);
}
template <bool I8>
static hipError_t launch_tree_heads(const TreeAttnLaunch& p, hipStream_t s) {
    const TreeShape t = tree_shape(p.nq / p.kv.nkv, p.kv.head_dim, p.tokens);
    if (p.kv.head_dim == 256) return t.ct == 1 ? launch_tree_mfma<256, I8, 1, 4, false>(p, s) : launch_tree_mfma<256, I8, 2, 2, true>(p, s);
    if (t.ct == 1) return launch_tree_mfma<128, I8, 1, 8, false>(p, s);
    return launch_tree_mfma<128, I8, 2, 4, true>(p, s);
}

hipError_t launch_tree_attn(const TreeAttnLaunch& p, hipStream_t s) {
    const int hd = p.kv.head_dim;
    // the matrix-core kernels take rows in 16-byte pieces, the caches in whole words
    const bool al = ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.gate) |
                      reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0 && p.q_stride % 4 == 0 && p.out_stride % 4 == 0 &&
                    ((reinterpret_cast<uintptr_t>(p.kv.k) | reinterpret_cast<uintptr_t>(p.kv.v)) & 3u) == 0;
    const bool in32 = p.q_stride < 1 << 22 && p.out_stride < 1 << 22;  // offsets within a block's (at most 64) rows
    const bool kv32 = static_cast<int64_t>(p.kv.nkv) * hd * 2 * 256 < int64_t(1) << 31;  // ... and its keys
    if (al && in32 && kv32 && (hd == 128 || hd == 256)) return p.kv.i8 ? launch_tree_heads<true>(p, s) : launch_tree_heads<false>(p, s);
    const size_t lds = sizeof(float) * tree_row_lds(p.nq / p.kv.nkv, hd);
    const dim3 grid(p.tokens, p.kv.nkv);
    if (p.kv.i8)
        hipLaunchKernelGGL((tree_attn_row_kernel<true>), grid, dim3(256), lds, s, p);
    else
        hipLaunchKernelGGL((tree_attn_row_kernel<false>), grid, dim3(256), lds, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
