// tree_linear.hip - the linear-attention step of every row of a tree of
// drafted tokens, each from its parent's state, the state itself unchanged.
//
// With g_i = exp(gate_i) the decay of row i, L_i the sum of the log gates over
// its path, S0 the state and j over the rows of the path above i:
//   delta_i = beta_i (v_i - e^{L_i} k_i S0 - sum_j e^{L_i - L_j} (k_i.k_j) delta_j)
//   o_i     = (e^{L_i} q_i S0 + sum_{j, i} e^{L_i - L_j} (q_i.k_j) delta_j) / sqrt(dk)
// which is S_i = g_i S_parent + k_i delta_i^T unrolled (custom_model.cpp:
// 1074-1096 per row).  L in 64 bits: differences of sums over a long path lose
// the digits that its length costs.  (Log gates below -1000 count as -1000: the
// decay is 0 either way, and differences stay finite.  NaN stays NaN, as in the
// single-token step.)
#include <algorithm>

#include "xqhip_common.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

constexpr int kTreeLinCols = 16;
constexpr int kTreeLinMaxDim = 256;
constexpr int kTreeLinMaxTaps = 8;

namespace {
// workspace: normalised q and k [nodes][lk_n][lk_hd], v [nodes][lv_n][lv_hd]
struct LinWs {
    float *q, *k, *v;
};
__host__ __device__ inline LinWs lin_ws(const TreeLinearLaunch& p) {
    const size_t nk = static_cast<size_t>(p.nodes) * p.lk_n * p.lk_hd;
    return LinWs{p.ws, p.ws + nk, p.ws + 2 * nk};
}
}  // namespace

__device__ __forceinline__ float log_gate(const TreeLinearLaunch& p, int vh, float a) {
    const float g = -expf(p.a_log[vh]) * softplus_dev(a + p.dt_bias[vh]);
    return g < -1000.0f ? -1000.0f : g;  // (fmaxf would take -1000 for NaN)
}

// conv1d + SiLU of one head's channels of one row over its path (then the
// history), q and k heads L2-normalised.  One wave per (row, head).
__global__ void __launch_bounds__(kWave) tree_conv_kernel(TreeLinearLaunch p) {
    const int lane = threadIdx.x, i = blockIdx.y, u = blockIdx.x;
    const bool is_q = u < p.lk_n, is_k = !is_q && u < 2 * p.lk_n;
    const int h = is_q ? u : (is_k ? u - p.lk_n : u - 2 * p.lk_n);
    const int hd = is_q || is_k ? p.lk_hd : p.lv_hd;
    const int ch0 = (is_q ? 0 : (is_k ? p.lk_n * p.lk_hd : 2 * p.lk_n * p.lk_hd)) + h * hd;
    const int hist = p.ksize - 1, conv_dim = 2 * p.lk_n * p.lk_hd + p.lv_n * p.lv_hd;
    const float* hs = p.conv_state + static_cast<size_t>(*p.pos0 & 1) * conv_dim * hist;
    const LinWs ws = lin_ws(p);
    float* out = is_q ? ws.q + (static_cast<size_t>(i) * p.lk_n + h) * hd
                      : (is_k ? ws.k + (static_cast<size_t>(i) * p.lk_n + h) * hd
                              : ws.v + (static_cast<size_t>(i) * p.lv_n + h) * hd);
    float y[kTreeLinMaxDim / kWave], ss = 0.0f;
#pragma unroll
    for (int e = 0; e < kTreeLinMaxDim / kWave; ++e) {
        const int d = lane + kWave * e;
        y[e] = 0.0f;
        if (d >= hd) continue;
        const int c = ch0 + d;
        float acc = 0.0f;
        int row = i, back = 0;  // the row of this tap, or the steps behind the last history entry
        float tap[kTreeLinMaxTaps];
        for (int t = hist; t >= 0; --t) {
            tap[t] = row >= 0 ? p.mixed[static_cast<size_t>(row) * p.stride + c] : hs[static_cast<size_t>(c) * hist + hist - 1 - back++];
            if (row >= 0) row = static_cast<int8_t>(p.links.words[row / 4] >> 8 * (row % 4));
        }
        for (int t = 0; t <= hist; ++t) acc += tap[t] * p.conv_w[static_cast<size_t>(c) * p.ksize + t];
        y[e] = silu_dev(acc);
        ss += y[e] * y[e];
    }
    const float inv = is_q || is_k ? 1.0f / sqrtf(wave_sum(ss) + 1.0e-6f) : 1.0f;
#pragma unroll
    for (int e = 0; e < kTreeLinMaxDim / kWave; ++e)
        if (lane + kWave * e < hd) out[lane + kWave * e] = y[e] * inv;
}

// Value head vh, kTreeLinCols columns of it.
__global__ void __launch_bounds__(256) tree_delta_kernel(TreeLinearLaunch p) {
    __shared__ double L[kTreeMax];
    __shared__ float beta[kTreeMax], from0[kTreeMax];
    __shared__ uint64_t path[kTreeMax];  // rows above row i
    __shared__ float kk[kTreeMax][kTreeMax], qk[kTreeMax][kTreeMax];  // decay * (k_i.k_j), decay * (q_i.k_j)
    __shared__ float kS[kTreeMax][kTreeLinCols], qS[kTreeMax][kTreeLinCols], delta[kTreeMax][kTreeLinCols];
    const int vh = blockIdx.x, j0 = blockIdx.y * kTreeLinCols, tid = threadIdx.x;
    const int n = p.nodes, dk = p.lk_hd, dv = p.lv_hd;
    const int kh = min(p.lk_n - 1, vh / max(1, p.lv_n / p.lk_n));
    const LinWs ws = lin_ws(p);
    if (tid < n) {
        const float a = p.a[static_cast<size_t>(tid) * p.stride + vh], b = p.b[static_cast<size_t>(tid) * p.stride + vh];
        beta[tid] = sigmoid_dev(b);
        L[tid] = log_gate(p, vh, a);
    }
    __syncthreads();
    double sum = 0.0;
    uint64_t above = 0;
    if (tid < n)
        for (int r = tid; r >= 0; r = static_cast<int8_t>(p.links.words[r / 4] >> 8 * (r % 4))) {
            sum += L[r];
            if (r != tid) above |= uint64_t(1) << r;
        }
    __syncthreads();
    if (tid < n) {
        L[tid] = sum;
        from0[tid] = static_cast<float>(exp(sum));
        path[tid] = above;
    }
    __syncthreads();
    for (int x = tid; x < n * n; x += 256) {
        const int i = x / n, j = x % n;
        float dk_ = 0.0f, dq = 0.0f;
        if (i == j || (path[i] >> j & 1)) {
            const float* ki = ws.k + (static_cast<size_t>(i) * p.lk_n + kh) * dk;
            const float* qi = ws.q + (static_cast<size_t>(i) * p.lk_n + kh) * dk;
            const float* kj = ws.k + (static_cast<size_t>(j) * p.lk_n + kh) * dk;
            for (int d = 0; d < dk; ++d) {
                dk_ += ki[d] * kj[d];
                dq += qi[d] * kj[d];
            }
            const float decay = static_cast<float>(exp(L[i] - L[j]));
            dk_ *= decay;
            dq *= decay;
        }
        kk[i][j] = dk_;
        qk[i][j] = dq;
    }
    const float* S = p.state + static_cast<size_t>(vh) * dk * dv;
    for (int x = tid; x < n * kTreeLinCols; x += 256) {
        const int i = x / kTreeLinCols, c = j0 + x % kTreeLinCols;
        float sk = 0.0f, sq = 0.0f;
        if (c < dv)
            for (int d = 0; d < dk; ++d) {
                const float s = S[static_cast<size_t>(d) * dv + c];
                sk += ws.k[(static_cast<size_t>(i) * p.lk_n + kh) * dk + d] * s;
                sq += ws.q[(static_cast<size_t>(i) * p.lk_n + kh) * dk + d] * s;
            }
        kS[i][x % kTreeLinCols] = sk;
        qS[i][x % kTreeLinCols] = sq;
    }
    __syncthreads();
    const float rs = 1.0f / sqrtf(static_cast<float>(dk));
    if (tid < kTreeLinCols && j0 + tid < dv)
        for (int i = 0; i < n; ++i) {
            float pred = from0[i] * kS[i][tid], o = from0[i] * qS[i][tid];
            for (uint64_t above = path[i]; above; above &= above - 1) {  // (rows elsewhere may hold anything)
                const int j = __builtin_ctzll(above);
                pred += kk[i][j] * delta[j][tid];
                o += qk[i][j] * delta[j][tid];
            }
            const float dl = beta[i] * (ws.v[(static_cast<size_t>(i) * p.lv_n + vh) * dv + j0 + tid] - pred);
            delta[i][tid] = dl;
            p.out[static_cast<size_t>(i) * p.out_stride + static_cast<size_t>(vh) * dv + j0 + tid] = (o + qk[i][i] * dl) * rs;
        }
}

// ---------------------------------------------------------------------------
// Heads of 128 dims and four taps: two launches, or one (below) for up to 16 rows.
//
// tree_linear_prep_kernel: one wave per (row, head): the convolution over the
//   row's path, SiLU and L2 norm; q and k go out as fp16 hi + lo of 2^10 times
//   their values (22 bits: a unit vector's entries), the operands of what
//   follows.  One wave per value head, a row a lane: beta and L (in powers of 2).
// tree_linear_rows_kernel: one block per value head and 16 columns.  The products
//   with the state (k_i S0, q_i S0) and among the rows (k_i.k_j, q_i.k_j) on
//   fp16 MFMA, hi hi + hi lo + lo hi, S0 scaled per column by a power of two and
//   split likewise.  Then a wave has two columns and a lane a row: for each row j
//   that others continue, in order, delta_j goes to all lanes as a scalar and the
//   rows below j add its part: steps as many as inner rows, each a dozen
//   dependent instructions, no barrier.
//
// What bounds it: latency (a launch, rounds of loads, the steps); the bytes (the
// state, 2 MB for 32 heads, and 128 KB a row) are 1 us.  With 16 / 32 heads: 6 rows
// 5.8 us, a tree of 64 rows (three children a row) 14.4, a chain of 64 19.2.  Weights
// with decay and mask applied beforehand left the chain's step as long.
// ---------------------------------------------------------------------------
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
constexpr int kTL = 128;          // head dims
constexpr int kTLCols = 16;       // columns of a block
constexpr int kTLWaves = 8;       // of a block, kTLCols / kTLWaves columns each
constexpr int kTLPitch = kTreeMax + 4;
constexpr float kTLRaise = 1024.0f;

namespace {
struct FastWs {
    _Float16 *q, *k;  // [lk_n][2 (hi, lo)][rows][128], rows to a multiple of 16
    float* v;         // [lv_n][rows][128]
    double* L;        // [lv_n][64]: log2 of the decay from the state to each row
    float* beta;      // [lv_n][64]
};
__host__ __device__ inline int fast_rows(int nodes) { return (nodes + 15) / 16 * 16; }
__host__ __device__ inline size_t fast_bytes(int nodes, int lk_n, int lv_n) {
    const size_t rows = fast_rows(nodes);
    return 2 * (static_cast<size_t>(lk_n) * 2 * rows * kTL * 2) + static_cast<size_t>(lv_n) * rows * kTL * 4 +
           static_cast<size_t>(lv_n) * kTreeMax * 12;
}
__device__ inline FastWs fast_ws(const TreeLinearLaunch& p) {
    const size_t rows = fast_rows(p.nodes), half = static_cast<size_t>(p.lk_n) * 2 * rows * kTL;
    FastWs w;
    w.q = reinterpret_cast<_Float16*>(p.ws);
    w.k = w.q + half;
    w.v = reinterpret_cast<float*>(w.k + half);
    w.L = reinterpret_cast<double*>(w.v + static_cast<size_t>(p.lv_n) * rows * kTL);
    w.beta = reinterpret_cast<float*>(w.L + static_cast<size_t>(p.lv_n) * kTreeMax);
    return w;
}
}  // namespace

// Row r's parent, r < 4 WORDS, each lane for its own r: the words as scalars.  (Indexed by lane, each step up a path would
// be a memory round trip.)
template <int WORDS>
__device__ __forceinline__ int parent_in(const TreeLinks& links, int r) {
    uint32_t w = links.words[0];
#pragma unroll
    for (int i = 1; i < WORDS; ++i) w = r / 4 == i ? links.words[i] : w;
    return static_cast<int8_t>(w >> 8 * (r % 4));
}

// beta and L of every row (a lane each) of value head vh, by one wave
__device__ __forceinline__ void row_gates(const TreeLinearLaunch& p, int vh, double* L, float* beta) {
    const int lane = threadIdx.x & (kWave - 1);
    const bool on = lane < p.nodes;
    const size_t at = static_cast<size_t>(on ? lane : 0) * p.stride + vh;
    const float a = p.a[at], b = p.b[at];
    const double mine = on ? static_cast<double>(log_gate(p, vh, a)) * 1.44269504088896340736 : 0.0;
    // path sums by doubling: before step s a lane has the sum of the last s rows of its path
    int up = on ? static_cast<int8_t>(p.links.words[lane / 4] >> 8 * (lane % 4)) : -1;
    double sum = mine;
    for (int s = 1; s < p.nodes; s *= 2) {
        const double add = __shfl(sum, up < 0 ? lane : up, kWave);
        const int next = __shfl(up, up < 0 ? lane : up, kWave);
        if (up >= 0) {
            sum += add;
            up = next;
        }
    }
    L[lane] = sum;
    beta[lane] = sigmoid_dev(b);
}

__device__ __forceinline__ int conv_channels(const TreeLinearLaunch& p) { return (2 * p.lk_n + p.lv_n) * kTL; }
// What the convolution of channels c and c + 1 takes besides rows: the weights, and the history's three newest steps
// (oldest first) in both copies.  Which copy counts is known when the position has come; no load waits for it.
struct ConvTaps {
    float w[8], past[2][6] = {};
    __device__ __forceinline__ void load_weights(const TreeLinearLaunch& p, int c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = p.conv_w[4 * c + i];
    }
    __device__ __forceinline__ void load_past(const TreeLinearLaunch& p, int c) {
        const float* h = p.conv_state + static_cast<size_t>(c) * 3;
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            past[0][i] = h[i];
            past[1][i] = h[static_cast<size_t>(conv_channels(p)) * 3 + i];
        }
    }
};
// Row i's newest four rows of its path, itself first, in channels c and c + 1; how many there are
template <typename Parent>
__device__ __forceinline__ int path_window(const TreeLinearLaunch& p, int i, int c, Parent parent, float2 (&x)[4]) {
    int r = i, have = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        x[t] = make_float2(0.0f, 0.0f);
        if (r >= 0) {
            const float* row = p.mixed + static_cast<size_t>(r) * p.stride + c;
            x[t] = make_float2(row[0], row[1]);
            r = parent(r);
            ++have;
        }
    }
    return have;
}
// x / (1 + e^-x) by the hardware's exponential and reciprocal, an ulp each: off by |x| 2^-24 of itself at most where it
// is small, by 2^-22 elsewhere.  (The exact division and exponential were half of what few rows take.)
__device__ __forceinline__ float silu_fast(float x) {
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}
__device__ __forceinline__ float2 conv_silu(const float2 (&x)[4], int have, const ConvTaps& taps, bool odd) {
    float y[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        float past[3];  // newest first
#pragma unroll
        for (int i = 0; i < 3; ++i) past[i] = odd ? taps.past[1][3 * e + 2 - i] : taps.past[0][3 * e + 2 - i];
#pragma unroll
        for (int t = 3; t >= 0; --t) {
            float v = e ? x[t].y : x[t].x;
#pragma unroll
            for (int i = 0; i < t; ++i) v = have == t - i ? past[i] : v;
            y[e] += v * taps.w[4 * e + 3 - t];
        }
    }
    return make_float2(silu_fast(y[0]), silu_fast(y[1]));
}
// y over its norm (a wave has the row, two dims a lane), times kTLRaise, as hi + lo
__device__ __forceinline__ void unit_split(float2 y, h2& hi, h2& lo) {
    const float inv = __builtin_amdgcn_rsqf(wave_sum(y.x * y.x + y.y * y.y) + 1.0e-6f);
    float z[2] = {y.x * inv * kTLRaise, y.y * inv * kTLRaise};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        asm("" : "+v"(z[e]));  // (one rounding for hi and for what lo is taken from)
        hi[e] = static_cast<_Float16>(z[e]);
        lo[e] = static_cast<_Float16>(z[e] - static_cast<float>(hi[e]));
    }
}

constexpr int kTLPrepWaves = 4;
__global__ void __launch_bounds__(kWave* kTLPrepWaves) tree_linear_prep_kernel(TreeLinearLaunch p, int row_blocks) {
    const int lane = threadIdx.x & (kWave - 1);
    const FastWs ws = fast_ws(p);
    if (static_cast<int>(blockIdx.x) >= row_blocks) {
        const int vh = (static_cast<int>(blockIdx.x) - row_blocks) * kTLPrepWaves + threadIdx.x / kWave;
        if (vh < p.lv_n) row_gates(p, vh, ws.L + vh * kTreeMax, ws.beta + vh * kTreeMax);
        return;
    }
    const int units = 2 * p.lk_n + p.lv_n, rows = fast_rows(p.nodes);
    const int id = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * kTLPrepWaves + static_cast<int>(threadIdx.x) / kWave);
    const int i = id / units, u = id % units;
    if (i >= p.nodes) return;
    const bool is_q = u < p.lk_n, is_k = !is_q && u < 2 * p.lk_n;
    const int h = is_q ? u : (is_k ? u - p.lk_n : u - 2 * p.lk_n);
    const int c = u * kTL + 2 * lane;
    ConvTaps taps;
    float2 x[4];
    taps.load_weights(p, c);
    const int have = path_window(
        p, i, c, [&](int r) { return static_cast<int>(static_cast<int8_t>(p.links.words[r / 4] >> 8 * (r % 4))); }, x);
    if (have < 4) taps.load_past(p, c);
    const float2 y = conv_silu(x, have, taps, *p.pos0 & 1);
    if (!is_q && !is_k) {
        *reinterpret_cast<float2*>(ws.v + (static_cast<size_t>(h) * rows + i) * kTL + 2 * lane) = y;
        return;
    }
    h2 hi, lo;
    unit_split(y, hi, lo);
    _Float16* out = (is_q ? ws.q : ws.k) + (static_cast<size_t>(h) * 2 * rows + i) * kTL + 2 * lane;
    *reinterpret_cast<h2*>(out) = hi;
    *reinterpret_cast<h2*>(out + static_cast<size_t>(rows) * kTL) = lo;
}

constexpr int kTLLd = kTL + 8;  // halves per operand row: 16-byte rows shifted by 4 banks
struct RowsSmem {
    float kk[kTreeMax][kTLPitch], qk[kTreeMax][kTLPitch];  // [j][i]: k_i.k_j, q_i.k_j
    float kS[kTLCols][kTLPitch], qS[kTLCols][kTLPitch];    // [column][i]
};
// behind it the operands: [q, k][hi, lo][rows][kTLLd]
inline size_t rows_lds(int nodes) { return sizeof(RowsSmem) + static_cast<size_t>(4) * fast_rows(nodes) * kTLLd * 2; }

// ALONE: up to 16 rows, without the first launch: each block convolves its own key head's rows and its own columns of v,
// 16 times over in all, which costs less than a launch and its round trip: with 16 / 32 heads 1 row 4.5 us (two launches
// 7.2), 6 rows 5.8 (7.5), a chain of 16 8.5 (9.1).
constexpr int kTLAlone = 16;
template <bool ALONE>
__global__ void __launch_bounds__(kWave* kTLWaves, 2) tree_linear_rows_kernel(TreeLinearLaunch p) {
    extern __shared__ uint4 tree_lds[];
    __shared__ float v_own[ALONE ? kTLAlone : 1][kTLCols + 2], beta_own[ALONE ? kTreeMax : 1];
    __shared__ double L_own[ALONE ? kTreeMax : 1];
    RowsSmem& sm = *reinterpret_cast<RowsSmem*>(tree_lds);
    _Float16* ops = reinterpret_cast<_Float16*>(&sm + 1);
    const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int vh = blockIdx.x, j0 = blockIdx.y * kTLCols, kh = vh / (p.lv_n / p.lk_n);
    const int n = p.nodes, rows = fast_rows(n), tiles = rows / 16;
    const int g = lane / 16, cl = lane % 16;
    // every load first: the state's columns, the operands, the wave's two columns of v and its rows' gates
    float s0[4][8];
    const bool has_tile = wid < 2 * tiles;  // (q or k, row tile) of this wave
    const bool has_rows = ALONE ? wid / 2 == 1 : has_tile;  // ... of which it does the products among the rows
    {
        const float* S = p.state + (static_cast<size_t>(vh) * kTL + 8 * g) * kTL + j0 + cl;
        if (has_tile)
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) s0[s][e] = S[(32 * s + e) * kTL];
    }
    const int row = lane < n ? lane : n - 1, col = j0 + 2 * wid;
    const uint64_t above = p.above.m[lane];
    float2 v;
    double L;
    float beta;
    if constexpr (ALONE) {
        // this wave's rows of q (even waves) or k, 4 apart; v eight rows a wave and the gates by the last ones
        constexpr int kRounds = kTLAlone / (kTLWaves / 2);
        const int c = ((wid & 1) * p.lk_n + kh) * kTL + 2 * lane;
        ConvTaps taps;
        float2 x[kRounds][4];
        int have[kRounds] = {};
        taps.load_weights(p, c);
        taps.load_past(p, c);
        const int up = parent_in<kTLAlone / 4>(p.links, lane);  // (of the first 16 lanes' rows)
#pragma unroll
        for (int u = 0; u < kRounds; ++u)
            if (const int i = wid / 2 + u * (kTLWaves / 2); i < n)
                have[u] = path_window(p, i, c, [&](int r) { return __builtin_amdgcn_readlane(up, r); }, x[u]);
        const bool odd = *p.pos0 & 1;
        if (const int t = kTLWaves - 1 - wid; 8 * t < n) {
            const int i = min(8 * t + lane / 8, n - 1), at = 2 * (lane % 8), vc = (2 * p.lk_n + vh) * kTL + j0 + at;
            ConvTaps vtaps;
            float2 xv[4];
            vtaps.load_weights(p, vc);
            vtaps.load_past(p, vc);
            const int vhave = path_window(p, i, vc, [&](int r) { return parent_in<kTLAlone / 4>(p.links, r); }, xv);
            *reinterpret_cast<float2*>(&v_own[i][at]) = conv_silu(xv, vhave, vtaps, odd);
        }
        if (wid == kTLWaves - 3) row_gates(p, vh, L_own, beta_own);
#pragma unroll
        for (int u = 0; u < kRounds; ++u)
            if (const int i = wid / 2 + u * (kTLWaves / 2); i < n) {
                h2 hi, lo;
                unit_split(conv_silu(x[u], have[u], taps, odd), hi, lo);
                _Float16* out = ops + (static_cast<size_t>(wid & 1) * 2 * rows + i) * kTLLd + 2 * lane;
                *reinterpret_cast<h2*>(out) = hi;
                *reinterpret_cast<h2*>(out + rows * kTLLd) = lo;
            }
        __syncthreads();
        v = *reinterpret_cast<const float2*>(&v_own[row][2 * wid]);
        L = L_own[lane];
        beta = beta_own[lane];
    } else {
        const FastWs ws = fast_ws(p);
        v = *reinterpret_cast<const float2*>(ws.v + (static_cast<size_t>(vh) * rows + row) * kTL + col);
        L = ws.L[vh * kTreeMax + lane];
        beta = ws.beta[vh * kTreeMax + lane];
        // a quarter of the operands is rows * 16 pieces of 16 bytes: q hi, q lo, k hi, k lo
        const int quarter = rows * (kTL / 8);
        u32x4 piece[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int at = threadIdx.x + u * kWave * kTLWaves, part = at / quarter, in = at % quarter;
            const _Float16* src = (part < 2 ? ws.q : ws.k) + (static_cast<size_t>(kh) * 2 + (part & 1)) * rows * kTL;
            if (part < 4) piece[u] = *reinterpret_cast<const u32x4*>(src + 8 * in);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int at = threadIdx.x + u * kWave * kTLWaves, part = at / quarter, in = at % quarter;
            if (part < 4)
                *reinterpret_cast<u32x4*>(ops + (static_cast<size_t>(part) * rows + in / (kTL / 8)) * kTLLd + 8 * (in % (kTL / 8))) = piece[u];
        }
        __syncthreads();
    }
    // operand fragments of 16 rows: lane holds row cl, dims 32 s + 8 g .. + 7
    auto frag = [&](bool of_k, int t, half8 (&hi)[4], half8 (&lo)[4]) {
        const _Float16* at = ops + (static_cast<size_t>(of_k ? 2 : 0) * rows + 16 * t + cl) * kTLLd + 8 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            hi[s] = *reinterpret_cast<const half8*>(at + 32 * s);
            lo[s] = *reinterpret_cast<const half8*>(at + rows * kTLLd + 32 * s);
        }
    };
    auto product = [&](const half8 (&ah)[4], const half8 (&al)[4], const half8 (&bh)[4], const half8 (&bl)[4]) {
        floatx4 c = {0.0f, 0.0f, 0.0f, 0.0f}, d = c, e = c;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[s], bh[s], c, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[s], bl[s], d, 0, 0, 0);
            e = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[s], bh[s], e, 0, 0, 0);
        }
        return c + d + e;
    };
    const bool of_k = ALONE ? wid % 2 == 0 : wid < tiles;
    const int ta = wid % tiles;
    half8 ah[4], al[4], bh[4], bl[4];
    if (has_tile || has_rows) frag(of_k, ta, ah, al);
    if (has_tile) {
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(s0[s][e]));
        mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
        mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
        int ex = 13;  // a power of two brings the column's largest magnitude into [2^12, 2^13)
        if (mx > 0.0f && mx < INFINITY) frexpf(mx, &ex);
        ex = max(ex, -100);
        const float up = ldexpf(1.0f, 13 - ex), down = ldexpf(1.0f / kTLRaise, ex - 13);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = s0[s][e] * up;
                bh[s][e] = static_cast<_Float16>(x);
                bl[s][e] = static_cast<_Float16>(x - static_cast<float>(bh[s][e]));
            }
        *reinterpret_cast<floatx4*>(&(of_k ? sm.kS : sm.qS)[cl][16 * ta + 4 * g]) = product(ah, al, bh, bl) * down;
    }
    if (has_rows) {  // with the k rows of every tile that holds a row above one of this tile's, or the rows themselves
        for (int b = 0; b <= ta; ++b) {
            if (b < ta && !__builtin_amdgcn_ballot_w64(lane / 16 == ta && (above >> 16 * b & 0xffff))) continue;
            frag(true, b, bh, bl);
            *reinterpret_cast<floatx4*>(&(of_k ? sm.kk : sm.qk)[16 * b + cl][16 * ta + 4 * g]) =
                product(ah, al, bh, bl) * (1.0f / (kTLRaise * kTLRaise));
        }
    }
    __syncthreads();
    // lane: a row; two columns
    const float from0 = __builtin_amdgcn_exp2f(static_cast<float>(L));
    float pred[2], o[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        pred[e] = from0 * sm.kS[2 * wid + e][row];
        o[e] = from0 * sm.qS[2 * wid + e][row];
    }
    const float self = sm.qk[row][row];
    const long long lb = __double_as_longlong(L);
    uint64_t left = p.inner;
    int j = left ? __builtin_ctzll(left) : 0;
    float a = sm.kk[j][row], b = sm.qk[j][row];
    while (left) {
        const int at = j;
        const float ka = a, qa = b;
        left &= left - 1;
        j = left ? __builtin_ctzll(left) : 0;
        a = sm.kk[j][row];  // the next step's
        b = sm.qk[j][row];
        const double Lj = __hiloint2double(__builtin_amdgcn_readlane(static_cast<int>(lb >> 32), at),
                                           __builtin_amdgcn_readlane(static_cast<int>(lb), at));
        const float decay = __builtin_amdgcn_exp2f(static_cast<float>(L - Lj));
        const bool below = above >> at & 1;  // (rows elsewhere may hold anything)
        const float ck = decay * ka, cq = decay * qa;
        const float d0 = readlane_f32(beta * (v.x - pred[0]), at), d1 = readlane_f32(beta * (v.y - pred[1]), at);
        if (below) {
            pred[0] += ck * d0;
            pred[1] += ck * d1;
            o[0] += cq * d0;
            o[1] += cq * d1;
        }
    }
    if (lane >= n) return;
    const float rs = 0.08838834764831845f;  // 1 / sqrt(128)
    float* out = p.out + static_cast<size_t>(lane) * p.out_stride + vh * kTL + col;
    out[0] = (o[0] + self * (beta * (v.x - pred[0]))) * rs;
    out[1] = (o[1] + self * (beta * (v.y - pred[1]))) * rs;
}

static bool linear_fast(int lk_hd, int lv_hd) { return lk_hd == kTL && lv_hd == kTL; }

bool tree_linear_supported(int lk_n, int lk_hd, int lv_n, int lv_hd, int ksize) {
    return lk_n > 0 && lv_n > 0 && lk_n <= 4096 && lv_n <= 4096 && lv_n % lk_n == 0 && lk_hd > 0 && lv_hd > 0 &&
           lk_hd <= kTreeLinMaxDim && lv_hd <= kTreeLinMaxDim && ksize > 0 && ksize <= kTreeLinMaxTaps;
}

size_t tree_linear_workspace_bytes(int nodes, int lk_n, int lk_hd, int lv_n, int lv_hd) {
    if (linear_fast(lk_hd, lv_hd)) return fast_bytes(nodes, lk_n, lv_n);  // (more than the general form takes)
    return static_cast<size_t>(nodes) * (2 * lk_n * lk_hd + lv_n * lv_hd) * sizeof(float);
}

hipError_t launch_tree_linear(const TreeLinearLaunch& p, hipStream_t s) {
    if (linear_fast(p.lk_hd, p.lv_hd) && p.ksize == 4) {
        const dim3 grid(p.lv_n, kTL / kTLCols), block(kWave * kTLWaves);
        if (p.nodes <= kTLAlone) {
            hipLaunchKernelGGL(tree_linear_rows_kernel<true>, grid, block, rows_lds(p.nodes), s, p);
            return hipGetLastError();
        }
        const int row_blocks = ((2 * p.lk_n + p.lv_n) * p.nodes + kTLPrepWaves - 1) / kTLPrepWaves;
        hipLaunchKernelGGL(tree_linear_prep_kernel, dim3(row_blocks + (p.lv_n + kTLPrepWaves - 1) / kTLPrepWaves),
                           dim3(kWave * kTLPrepWaves), 0, s, p, row_blocks);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&tree_linear_rows_kernel<false>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(rows_lds(kTreeMax)));
            e != hipSuccess)
            return e;
        hipLaunchKernelGGL(tree_linear_rows_kernel<false>, grid, block, rows_lds(p.nodes), s, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(tree_conv_kernel, dim3(2 * p.lk_n + p.lv_n, p.nodes), dim3(kWave), 0, s, p);
    hipLaunchKernelGGL(tree_delta_kernel, dim3(p.lv_n, (p.lv_hd + kTreeLinCols - 1) / kTreeLinCols), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
