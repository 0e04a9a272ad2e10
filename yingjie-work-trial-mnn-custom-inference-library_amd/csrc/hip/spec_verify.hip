// spec_verify.hip - verification of a tree of drafted tokens against the
// target's probabilities, from given random numbers.
//
// With p = softmax(logits / T) of a row and q its children's draft
// distribution, the distribution left after s rejections is the normalised
// max(p_{s-1} - q, 0).  Unrolled it is p_s = (p - c_s q)+ / d_s, (x)+ = max(x,
// 0), with
//   c_0 = 0, d_0 = 1, c_{s+1} = c_s + d_s, d_{s+1} = sum (p - c_{s+1} q)+
// (((p - c q)+ / d - q)+ = (p - (c + d) q)+ / d: where p < c q the left side is
// 0 as well), so a rejection costs one sum over the vocabulary and stores no
// distribution.  For point masses p_s is p without the rejected tokens and d_s
// = 1 - their probabilities: no sum at all.
//
// verify_stats_kernel: every row's maximum and sum of exponentials, piece by
//   piece (all rows: which of them the walk visits is not known yet); greedy:
//   its argmax.
// verify_rest_kernel: d_s of the rows with more than s children, one launch per
//   s < the most children of a row; chains and point masses need none.
// verify_walk_kernel: each block walks the tree (a wave decides for every row at
//   once which child it would accept, then follows the links).  The token comes
//   from the last row's piece sums, which the first pass left, less the rejected
//   tokens: one block.  Where a draft distribution was taken off each block
//   sums its piece of the rest, and the last to finish picks the token.
// Exponentials, sums and comparisons in 64 bits: a token's share of a flat
// distribution over 2^18 tokens is 2^-18, and the sampled token is the one
// whose share the random number falls into.  What bounds it: the logits are read
// once; the exponentials' fp64 work (15 operations a logit) takes about as long
// as the memory and half hides behind it (40 rows of 248320 logits: 15 us for
// 39.7 MB, 2.6 TB/s); the walk is a chain of a dozen steps that wait for each
// other (11 to 13 us for 6 as for 40 rows).  Greedy calls take 7.6 us for 6 rows
// and 16.0 for 40, walk and all.
#include <algorithm>

#include "xqhip_common.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

constexpr int kPiece = 4096;  // logits of one block
constexpr int kStatThreads = 256, kWalkThreads = 1024;
constexpr int kWalkLanes = kWalkThreads / kTreeMax;  // lanes that sum one row's pieces

struct Stat {
    double sum;   // of exp((l - m) / T) over the piece
    float m;      // its maximum, NaN as -inf
    int32_t arg;  // greedy: lowest index of it
};

struct VerifyWs {
    Stat* stat;      // [nodes][pieces]
    double* rest;    // [max_children][nodes][pieces]: partial d_s
    double* weight;  // [pieces] of the walk's last row
    uint32_t* done;
};

__host__ __device__ inline int verify_pieces(int vocab) { return (vocab + kPiece - 1) / kPiece; }

__host__ __device__ inline VerifyWs verify_ws(void* ws, int nodes, int vocab) {
    const size_t n = static_cast<size_t>(nodes) * verify_pieces(vocab);
    VerifyWs w;
    w.stat = static_cast<Stat*>(ws);
    w.rest = reinterpret_cast<double*>(w.stat + n);
    w.weight = w.rest + n * nodes;
    w.done = reinterpret_cast<uint32_t*>(w.weight + verify_pieces(vocab));
    return w;
}

size_t verify_workspace_bytes(int nodes, int vocab) {
    const size_t pieces = verify_pieces(vocab), n = pieces * nodes;
    return n * sizeof(Stat) + (n * nodes + pieces) * sizeof(double) + 16;
}

// 2^t for -1001 <= t <= 0: 2^f as the Taylor polynomial of exp(f ln 2) for f = t - rint(t), |f| <= 1/2 (its next
// term is 7e-12 of the value), the whole part (by the addition of 1.5 2^52, whose low word it then is) into the exponent.
__device__ __forceinline__ double exp2_f64(double t) {
    constexpr double kRound = 6755399441055744.0;
    const double b = t + kRound, f = t - (b - kRound);
    double r = 1.01780860092396999e-07;  // ln2^k / k!, k = 9 .. 0
    r = fma(r, f, 1.32154867901443095e-06);
    r = fma(r, f, 1.52527338040598411e-05);
    r = fma(r, f, 1.54035303933816088e-04);
    r = fma(r, f, 1.33335581464284433e-03);
    r = fma(r, f, 9.61812910762847688e-03);
    r = fma(r, f, 5.55041086648215831e-02);
    r = fma(r, f, 2.40226506959100722e-01);
    r = fma(r, f, 6.93147180559945286e-01);
    r = fma(r, f, 1.0);
    return __hiloint2double(__double2hiint(r) + (__double2loint(b) << 20), __double2loint(r));
}

constexpr double kLog2e = 1.44269504088896340736;

// exp((l - m) / T), scale = log2(e) / T, l <= m.  Under 2^-1000 of the maximum it is 0, at the maximum itself (an
// infinity among them) 1.
__device__ __forceinline__ double weight_of(float l, float m, double scale) {
    const double t = (static_cast<double>(l) - static_cast<double>(m)) * scale;
    const double w = exp2_f64(fmax(t, -1000.0));
    return l == m ? 1.0 : (t > -1000.0 ? w : 0.0);
}

// A lane's parent, from the launch's arguments as scalars: indexed by lane they would be one more memory round trip.
__device__ __forceinline__ int parent_of(const TreeLinks& l, int row) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < kTreeMax / 4; ++i) w = row / 4 == i ? l.words[i] : w;
    return static_cast<int8_t>(w >> 8 * (row % 4));
}

// four values of a row at v; past the row's end `pad`, NaN as pad
__device__ __forceinline__ void load4(const float* row, int vocab, int v, bool al, float pad, float (&x)[4]) {
    float4 f = make_float4(pad, pad, pad, pad);
    if (al && v + 3 < vocab) {
        f = *reinterpret_cast<const float4*>(row + v);
    } else {
        if (v < vocab) f.x = row[v];
        if (v + 1 < vocab) f.y = row[v + 1];
        if (v + 2 < vocab) f.z = row[v + 2];
        if (v + 3 < vocab) f.w = row[v + 3];
    }
    x[0] = f.x == f.x ? f.x : pad;
    x[1] = f.y == f.y ? f.y : pad;
    x[2] = f.z == f.z ? f.z : pad;
    x[3] = f.w == f.w ? f.w : pad;
}
// a piece by 256 threads: 4 values at 4 (256 u + tid)
constexpr int kPer = kPiece / kStatThreads;
__device__ __forceinline__ int at_of(int v0, int u) { return v0 + 4 * (kStatThreads * u + static_cast<int>(threadIdx.x)); }
__device__ __forceinline__ void load_piece(const float* row, int vocab, int v0, bool al, float pad, float (&x)[kPer / 4][4]) {
#pragma unroll
    for (int u = 0; u < kPer / 4; ++u) load4(row, vocab, at_of(v0, u), al, pad, x[u]);
}

template <int CTRL, bool ZERO>
__device__ __forceinline__ double dpp_f64(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xF, 0xF, ZERO);
    const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xF, 0xF, ZERO);
    return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
    const long long b = __double_as_longlong(v);
    return __hiloint2double(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane),
                            __builtin_amdgcn_readlane(static_cast<int>(b), lane));
}
// sum over each aligned group of 16 lanes, over the wave
__device__ __forceinline__ double row_sum_f64(double v) {
    v += dpp_f64<kDppXor1, false>(v);
    v += dpp_f64<kDppXor2, false>(v);
    v += dpp_f64<kDppHalfMirror, false>(v);
    return v + dpp_f64<kDppMirror, false>(v);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v = row_sum_f64(v);
    return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}
// inclusive sum over the wave's lanes: within rows of 16 (lanes before a row's first read 0), then the rows' totals
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_f64<0x111, true>(v);  // row_shr:1, 2, 4, 8
    v += dpp_f64<0x112, true>(v);
    v += dpp_f64<0x114, true>(v);
    v += dpp_f64<0x118, true>(v);
    const double a = readlane_f64(v, 15), b = a + readlane_f64(v, 31), c = b + readlane_f64(v, 47);
    const int row = (threadIdx.x & (kWave - 1)) >> 4;
    return v + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? b : c);
}

// sum over the block's up to 16 waves in a fixed order; each wave's first 16 lanes get it
template <int THREADS>
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
    const int lane = threadIdx.x & (kWave - 1);
    v = wave_sum_f64(v);
    __syncthreads();
    if (lane == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    return row_sum_f64(lane < THREADS / kWave ? red[lane] : 0.0);
}

__device__ __forceinline__ bool aligned_rows(const float* base, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && ld % 4 == 0;
}

// One piece of a row.  Each wave takes its own quarter's maximum and sum, so that no wave waits for another before the end.
// (With the walk, when it was chosen, 64 rows of 248320 logits took 32.4 us and 40 rows 26.2, now 31.7 and 25.1; two pieces
// a block 34.4 and 26.0, blocks that go from piece to piece with the next one's loads under way 32.3 and 25.6.)
template <bool GREEDY>
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(VerifyLaunch p, int pieces) {
    constexpr int kWaves = kStatThreads / kWave;
    __shared__ Stat part[kWaves];
    __shared__ uint64_t best[kWaves];
    const int node = blockIdx.y, piece = blockIdx.x, v0 = piece * kPiece, wid = threadIdx.x / kWave;
    const VerifyWs ws = verify_ws(p.ws, p.nodes, p.vocab);
    float x[kPer / 4][4];
    load_piece(p.logits + node * p.ld, p.vocab, v0, aligned_rows(p.logits, p.ld), -INFINITY, x);
    const double scale = p.inv_t * kLog2e;
    if constexpr (GREEDY) {
        uint64_t key = 0;
#pragma unroll
        for (int u = 0; u < kPer / 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) key = u64_max(key, argmax_key(x[u][e], static_cast<uint32_t>(at_of(v0, u) + e)));
        key = wave_max_u64(key);
        if ((threadIdx.x & (kWave - 1)) == 0) best[wid] = key;
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < kPer / 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, x[u][e]);
        m = wave_max(m);
        double sum = 0.0;
        // (fp64 operations are what this pass waits for: the clamp in fp32, one multiply-add for the exponent.
        // Logits at the clamp, minus infinity among them, add 2^-1000 of the maximum: nothing.  Up to 2^16 in `off`, a
        // maximum of 45 at T = 0.001, the clamp's rounding to fp32 moves the exponent by 0.004 and the rounding of `off`
        // by 4e-12; where it is larger the one would leave exp2_f64's range and the other show in the sum.  A clamp of
        // minus infinity, T above 4e35, holds nothing back.  40 rows of 248320 logits with the walk: 25.1 us, with the
        // other branch 26.1.)
        const float low = m - static_cast<float>(1000.0 / scale);
        const double off = m * scale;
        if (low > -INFINITY && fabs(off) <= 65536.0) {  // wave-uniform
#pragma unroll
            for (int u = 0; u < kPer / 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += exp2_f64(fma(static_cast<double>(fmaxf(x[u][e], low)), scale, -off));
        } else if (m > -INFINITY) {
#pragma unroll
            for (int u = 0; u < kPer / 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += weight_of(x[u][e], m, scale);
        }
        sum = wave_sum_f64(sum);
        if ((threadIdx.x & (kWave - 1)) == 0) part[wid] = Stat{sum, m, 0};
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    Stat r{0.0, -INFINITY, 0};
    if constexpr (GREEDY) {
        uint64_t key = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) key = u64_max(key, best[i]);
        r.m = float_from_order_key(static_cast<uint32_t>(key >> 32));
        r.arg = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
    } else {
#pragma unroll
        for (int i = 0; i < kWaves; ++i) r.m = fmaxf(r.m, part[i].m);
#pragma unroll
        for (int i = 0; i < kWaves; ++i)
            if (part[i].m > -INFINITY) r.sum += part[i].sum * weight_of(part[i].m, r.m, scale);
    }
    ws.stat[node * static_cast<size_t>(pieces) + piece] = r;
    if (piece == 0 && node == 0) *ws.done = 0;
}

// maximum, argmax and exponential sum of a row from its pieces, by LANES consecutive lanes (all of them get it)
struct RowStat {
    float m;
    int32_t arg;
    double z;
};
// shares: where the first 64 pieces' parts of z go, or nullptr
template <int LANES>
__device__ __forceinline__ RowStat row_stat(const VerifyWs& ws, int node, int pieces, bool greedy, double scale,
                                            double* shares) {
    const Stat* s = ws.stat + static_cast<size_t>(node) * pieces;
    const int sub = threadIdx.x & (LANES - 1);
    constexpr int kHeld = 64 / LANES;  // pieces of a lane kept in registers
    Stat h[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
        h[u] = sub + u * LANES < pieces ? s[sub + u * LANES] : Stat{0.0, -INFINITY, 0x7fffffff};
    RowStat r{-INFINITY, 0, 0.0};
    if (greedy) {
        uint64_t key = 0;
#pragma unroll
        for (int u = 0; u < kHeld; ++u) key = u64_max(key, argmax_key(h[u].m, static_cast<uint32_t>(h[u].arg)));
        for (int i = sub + kHeld * LANES; i < pieces; i += LANES) key = u64_max(key, argmax_key(s[i].m, static_cast<uint32_t>(s[i].arg)));
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) key = u64_max(key, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(key), o, kWave)));
        r.m = float_from_order_key(static_cast<uint32_t>(key >> 32));
        r.arg = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
        return r;
    }
#pragma unroll
    for (int u = 0; u < kHeld; ++u) r.m = fmaxf(r.m, h[u].m);
    for (int i = sub + kHeld * LANES; i < pieces; i += LANES) r.m = fmaxf(r.m, s[i].m);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) r.m = fmaxf(r.m, __shfl_xor(r.m, o, kWave));
    if (r.m > -INFINITY) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const double z = h[u].m > -INFINITY ? h[u].sum * weight_of(h[u].m, r.m, scale) : 0.0;
            r.z += z;
            if (shares) shares[sub + u * LANES] = z;
        }
        for (int i = sub + kHeld * LANES; i < pieces; i += LANES)
            if (s[i].m > -INFINITY) r.z += s[i].sum * weight_of(s[i].m, r.m, scale);
    }
    if constexpr (LANES == 16) {
        r.z = row_sum_f64(r.z);
    } else {
        static_assert(LANES == kWave, "a row of lanes, or the wave");
        r.z = wave_sum_f64(r.z);
    }
    return r;
}

// d_s of a row from its pieces, by LANES consecutive lanes
template <int LANES>
__device__ __forceinline__ double rest_sum(const VerifyWs& ws, int s, int node, int nodes, int pieces) {
    const double* r = ws.rest + (static_cast<size_t>(s - 1) * nodes + node) * pieces;
    double d = 0.0;
    for (int i = threadIdx.x & (LANES - 1); i < pieces; i += LANES) d += r[i];
    return LANES == 16 ? row_sum_f64(d) : wave_sum_f64(d);
}

// (p - c q)+ of one token
__device__ __forceinline__ double rest_of(float l, float q, const RowStat& r, double inv_z, double c, double scale) {
    return fmax(weight_of(l, r.m, scale) * inv_z - c * static_cast<double>(q), 0.0);
}

// the partial sums of d_s, s >= 1, for the rows with more than s children
__global__ void __launch_bounds__(kStatThreads) verify_rest_kernel(VerifyLaunch p, int s) {
    __shared__ double red[kStatThreads / kWave];
    const int piece = blockIdx.x, node = blockIdx.y, v0 = piece * kPiece, pieces = gridDim.x;
    const int lane = threadIdx.x & (kWave - 1);
    const int mine = lane < p.nodes ? parent_of(p.links, lane) : -2;
    if (__popcll(__builtin_amdgcn_ballot_w64(mine == node)) <= s) return;  // block-uniform
    const VerifyWs ws = verify_ws(p.ws, p.nodes, p.vocab);
    const double scale = p.inv_t * kLog2e;
    float l[kPer / 4][4], q[kPer / 4][4];
    load_piece(p.logits + node * p.ld, p.vocab, v0, aligned_rows(p.logits, p.ld), -INFINITY, l);
    load_piece(p.draft + node * p.ld_draft, p.vocab, v0, aligned_rows(p.draft, p.ld_draft), 0.0f, q);
    const RowStat r = row_stat<kWave>(ws, node, pieces, false, scale, nullptr);
    double c = 1.0;  // c_1 = 1, c_{s+1} = c_s + d_s
    for (int i = 1; i < s; ++i) c += rest_sum<kWave>(ws, i, node, p.nodes, pieces);
    const double inv_z = r.z > 0.0 ? 1.0 / r.z : 0.0;
    double sum = 0.0;
    if (r.m > -INFINITY)
#pragma unroll
        for (int u = 0; u < kPer / 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += rest_of(l[u][e], q[u][e], r, inv_z, c, scale);
    sum = block_sum_f64<kStatThreads>(sum, red);
    if (threadIdx.x == 0) ws.rest[(static_cast<size_t>(s - 1) * p.nodes + node) * pieces + piece] = sum;
}

__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(VerifyLaunch p) {
    __shared__ RowStat row[kTreeMax];
    __shared__ int tok[kTreeMax], path[kTreeMax];
    __shared__ double prob[kTreeMax], prop[kTreeMax], cut[kTreeMax], over[kTreeMax];
    __shared__ float chance[kTreeMax];
    __shared__ uint64_t kids[kTreeMax];
    __shared__ double rest[kTreeMax - 1][kTreeMax];
    __shared__ double shares[kTreeMax][kWave];  // of a row's z: its first 64 pieces
    __shared__ int dup[kTreeMax];               // the token of a sibling before it
    __shared__ int kept_s, last_s, pick_s, ends_s, whole_s;
    __shared__ double want_s, before_s, red[kWalkThreads / kWave];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const int n = p.nodes, pieces = verify_pieces(p.vocab);
    const VerifyWs ws = verify_ws(p.ws, n, p.vocab);
    const bool greedy = p.inv_t == 0.0f, draft = p.draft != nullptr;
    const double scale = p.inv_t * kLog2e;
    // every row's statistics, and every drafted token's logit, draft probability and random number
    {
        const int node = tid / kWalkLanes, sub = tid % kWalkLanes;
        const bool mine = sub == 0 && node > 0 && node < n;
        const int par = mine ? parent_of(p.links, node) : 0, t = mine ? p.tokens[node] : -1;
        const bool valid = mine && !greedy && t >= 0 && t < p.vocab;
        const float l = valid ? p.logits[par * p.ld + t] : -INFINITY;
        const float q = valid ? (draft ? p.draft[par * p.ld_draft + t] : 1.0f) : 0.0f;
        const float u = mine && !greedy ? p.u_accept[node] : 0.0f;
        if (sub == 1) kids[node] = p.kids[node];
        if (node < n) {
            const RowStat r = row_stat<kWalkLanes>(ws, node, pieces, greedy, scale, greedy ? nullptr : shares[node]);
            if (sub == 0) row[node] = r;
            if (draft)
                for (int s = 1; s < p.max_children; ++s) {
                    const double d = rest_sum<kWalkLanes>(ws, s, node, n, pieces);  // (read only where it was written)
                    if (sub == 0) rest[s - 1][node] = d;
                }
        }
        if (sub == 0 && node < n) {
            tok[node] = t;
            chance[node] = u;
            prop[node] = q;
            prob[node] = l == l ? l : -INFINITY;  // (the logit still)
        }
    }
    __syncthreads();
    if (wid == 0) {  // lane i: row i, and its children in order
        const int par = lane < n ? parent_of(p.links, lane) : -2;
        const uint64_t my_kids = kids[lane];
        if (lane > 0 && lane < n) {
            const RowStat r = row[par];
            const float l = static_cast<float>(prob[lane]);
            prob[lane] = !greedy && l > -INFINITY && r.m > -INFINITY ? weight_of(l, r.m, scale) / r.z : 0.0;
            const int t = tok[lane];
            bool again = false;
            for (uint64_t e = kids[par] & ((uint64_t(1) << lane) - 1); e; e &= e - 1) again |= tok[__builtin_ctzll(e)] == t;
            dup[lane] = again;
        }
        __builtin_amdgcn_wave_barrier();
        int next = -1;
        double c = 0.0, d = 1.0;
        int rejected = 0;
        for (uint64_t left = my_kids; left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            if (greedy) {
                if (row[lane].m > -INFINITY && tok[j] == row[lane].arg) {
                    next = j;
                    break;
                }
                continue;
            }
            const bool again = !draft && dup[j];  // a rejected sibling's token: nothing is left of a point mass
            // u q < (p - c q)+ / d
            const double have = again || !(d > 0.0) ? 0.0 : (draft ? fmax(prob[j] - c * prop[j], 0.0) : prob[j]);
            if (static_cast<double>(chance[j]) * prop[j] * d < have) {
                next = j;
                break;
            }
            ++rejected;
            if (draft) {
                c += d;
                if (left & (left - 1)) d = rest[rejected - 1][lane];  // (no child comes after the last rejection)
            } else if (!again) {
                d -= prob[j];
            }
        }
        cut[lane] = c;
        over[lane] = d;
        int at = 0, kept = 1, here = lane == 0 ? 0 : -1;
        for (;;) {
            const int nx = __builtin_amdgcn_readlane(next, __builtin_amdgcn_readfirstlane(at));
            if (nx < 0) break;
            at = nx;
            if (lane == kept) here = at;
            ++kept;
        }
        path[lane] = here;
        if (lane == 0) kept_s = kept;
    }
    __syncthreads();
    const int kept = kept_s, stop = path[kept - 1];
    const RowStat r = row[stop];
    if (blockIdx.x == 0) {
        if (tid < n) {
            p.out_path[tid] = path[tid];
            if (tid + 1 != kept) p.out_tokens[tid] = tid + 1 < kept ? tok[path[tid + 1]] : -1;
        }
        if (tid == 0) *p.out_count = kept;
    }
    if (greedy || !(r.m > -INFINITY)) {  // one block, or nothing to sample
        if (blockIdx.x == 0 && tid == 0) p.out_tokens[kept - 1] = r.m > -INFINITY ? r.arg : -1;
        return;
    }
    // this thread's four weights of a piece of the last row: what is left of it, or (whole) all of it
    const double c = cut[stop], inv_z = 1.0 / r.z;
    const uint64_t refused = kids[stop];
    const bool al = aligned_rows(p.logits, p.ld), ald = draft && aligned_rows(p.draft, p.ld_draft);
    auto weights = [&](int piece, bool whole, double (&w)[4]) {
        const int v = piece * kPiece + 4 * tid;
        float l[4], q[4];
        load4(p.logits + stop * p.ld, p.vocab, v, al, -INFINITY, l);
        const bool off = draft && c > 0.0 && !whole;
        if (off) load4(p.draft + stop * p.ld_draft, p.vocab, v, ald, 0.0f, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = off ? rest_of(l[e], q[e], r, inv_z, c, scale) : weight_of(l[e], r.m, scale);
        if (!draft && !whole)
            for (uint64_t e = refused; e; e &= e - 1) {
                const int at = tok[__builtin_ctzll(e)] - v;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = at == i ? 0.0 : w[i];
            }
    };
    // Sums of the pieces.  Without a draft distribution to take off they are the first pass's, less the rejected
    // tokens (their exponentials are 7e-12 exact: the first block sums the rejected tokens' pieces again where little
    // else is left).  Otherwise every block sums its piece of the rest and the last one to finish goes on.
    const bool cutting = draft && c > 0.0, known = !cutting && over[stop] > 0x1p-7;
    double w[4];
    if (cutting) {
        weights(blockIdx.x, false, w);
        const double sum = block_sum_f64<kWalkThreads>((w[0] + w[1]) + (w[2] + w[3]), red);
        if (tid == 0) {
            __hip_atomic_store(ws.weight + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_s = __hip_atomic_fetch_add(ws.done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        }
        __syncthreads();
        if (!last_s) return;
    } else {
        if (blockIdx.x != 0) return;
        if (!known)
            for (uint64_t e = refused; e; e &= e - 1) {
                const int t = tok[__builtin_ctzll(e)];
                if (t < 0 || t >= p.vocab) continue;
                weights(t / kPiece, false, w);
                const double sum = block_sum_f64<kWalkThreads>((w[0] + w[1]) + (w[2] + w[3]), red);
                if (tid == 0) __hip_atomic_store(ws.weight + t / kPiece, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        __syncthreads();
    }
    // the piece that the random number falls into, then the token
    const Stat* st = ws.stat + static_cast<size_t>(stop) * pieces;
    bool whole = false;
    if (wid == 0) {
        auto share = [&](int i, bool all) {
            if (i >= pieces) return 0.0;
            auto summed = [&] { return __hip_atomic_load(ws.weight + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
            if (cutting && !all) return summed();
            const double z = i < kWave ? shares[stop][i] : (st[i].m > -INFINITY ? st[i].sum * weight_of(st[i].m, r.m, scale) : 0.0);
            if (draft || all) return z;
            double less = 0.0;
            bool hit = false;
            for (uint64_t e = refused; e; e &= e - 1) {
                const int j = __builtin_ctzll(e), t = tok[j];
                if (t < 0 || t >= p.vocab || t / kPiece != i) continue;
                hit = true;
                if (!dup[j]) less += prob[j] * r.z;
            }
            if (!hit) return z;
            if (!known) return summed();
            return z - less > 1e-10 * z ? z - less : 0.0;
        };
        const double want_of = static_cast<double>(*p.u_sample);
        double first = share(lane, false), total = first;
        for (int i = lane + kWave; i < pieces; i += kWave) total += share(i, false);
        total = wave_sum_f64(total);
        if (!(total > 0.0)) {  // a draft that covers the target leaves nothing: the target itself
            whole = true;
            total = r.z;
            first = share(lane, true);
        }
        const double want = want_of * total;
        double before = 0.0;
        int pick = -1, last_with = 0;
        for (int i0 = 0; i0 < pieces && pick < 0; i0 += kWave) {
            const double mine = i0 == 0 ? first : share(i0 + lane, whole), upto = before + wave_scan(mine);
            const uint64_t past = __builtin_amdgcn_ballot_w64(mine > 0.0 && upto > want);
            const uint64_t some = __builtin_amdgcn_ballot_w64(mine > 0.0);
            if (some) last_with = i0 + 63 - __builtin_clzll(some);
            if (past) {
                pick = i0 + __builtin_ctzll(past);
                before = readlane_f64(upto - mine, pick - i0);
            } else {
                before = readlane_f64(upto, kWave - 1);
            }
        }
        if (lane == 0) {
            pick_s = pick < 0 ? last_with : pick;
            ends_s = pick < 0;  // a random number of 1 or more, or NaN: the last token with a weight
            before_s = before;
            want_s = want;
            whole_s = whole;
        }
    }
    __syncthreads();
    whole = whole_s != 0;
    const int pick = pick_s;
    const bool ends = ends_s != 0;
    weights(pick, whole, w);
    const double s4 = (w[0] + w[1]) + (w[2] + w[3]), upto = wave_scan(s4);
    if (lane == kWave - 1) red[wid] = upto;
    __syncthreads();
    // each wave has the waves' sums, one a lane; the first that passes `want` has the token (rounding can leave none: the
    // last token with a weight then)
    constexpr int kWaves = kWalkThreads / kWave;
    const double want = want_s, part = lane < kWaves ? red[lane] : 0.0, end = before_s + wave_scan(part);
    const uint64_t holds = __builtin_amdgcn_ballot_w64(part > 0.0), passes = __builtin_amdgcn_ballot_w64(part > 0.0 && end > want);
    const bool to_the_end = ends || !passes;
    const int owner = to_the_end ? 63 - __builtin_clzll(holds | 1) : __builtin_ctzll(passes);
    if (wid != owner || !holds) return;
    double pre = readlane_f64(end - part, wid) + (upto - s4);
    int found = -1, at_least = -1;  // first token past `want`, last token with a weight
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        pre += w[e];
        if (w[e] > 0.0) {
            at_least = e;
            if (pre > want && found < 0) found = e;
        }
    }
    const uint64_t past = to_the_end ? 0 : __builtin_amdgcn_ballot_w64(found >= 0), some = __builtin_amdgcn_ballot_w64(at_least >= 0);
    const int who = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    if (lane == who) p.out_tokens[kept - 1] = pick * kPiece + 4 * tid + (past ? found : at_least);
}

hipError_t launch_verify(const VerifyLaunch& p, hipStream_t s) {
    const int pieces = verify_pieces(p.vocab);
    const dim3 grid(pieces, p.nodes);
    if (p.inv_t > 0.0f)
        hipLaunchKernelGGL(verify_stats_kernel<false>, grid, dim3(kStatThreads), 0, s, p, pieces);
    else
        hipLaunchKernelGGL(verify_stats_kernel<true>, grid, dim3(kStatThreads), 0, s, p, pieces);
    if (p.draft)
        for (int r = 1; r < p.max_children; ++r)
            hipLaunchKernelGGL(verify_rest_kernel, dim3(pieces, p.nodes), dim3(kStatThreads), 0, s, p, r);
    hipLaunchKernelGGL(verify_walk_kernel, dim3(p.draft ? pieces : 1), dim3(kWalkThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
