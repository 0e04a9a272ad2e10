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
//   piece (all rows: which of them the walk visits is not known yet).
// verify_rest_kernel: d_s of the rows with more than s children, one launch per
//   s < the most children of a row; chains and point masses need none.
// verify_walk_kernel: each block walks the tree (a few hundred operations on
//   values of the first pass), then takes its piece of the last row's rest;
//   the last block to finish picks the token from the pieces' sums.
// Exponentials, sums and comparisons in 64 bits: a token's share of a flat
// distribution over 2^18 tokens is 2^-18, and the sampled token is the one
// whose share the random number falls into.
#include <algorithm>

#include "xqhip_common.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

constexpr int kPiece = 8192;  // logits of one block
constexpr int kVThreads = 256;
constexpr int kPer = kPiece / kVThreads;  // values of a thread: 4 at 4 (256 u + tid)

struct Stat {
    double sum;   // of exp((l - m) / T) over the piece
    float m;      // its maximum, NaN as -inf
    int32_t arg;  // lowest index of it
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

// exp((l - m) / T), 1 at the maximum itself (an infinity among them)
__device__ __forceinline__ double weight_of(float l, float m, double inv_t) {
    return l == m ? 1.0 : exp((static_cast<double>(l) - static_cast<double>(m)) * inv_t);
}

// the thread's 32 values of a row's piece; past the row's end `pad`, NaN as pad
__device__ __forceinline__ void load_piece(const float* row, int vocab, int v0, bool al, float pad, float (&x)[kPer]) {
#pragma unroll
    for (int u = 0; u < kPer / 4; ++u) {
        const int v = v0 + 4 * (kVThreads * u + static_cast<int>(threadIdx.x));
        float4 f = make_float4(pad, pad, pad, pad);
        if (al && v + 3 < vocab) {
            f = *reinterpret_cast<const float4*>(row + v);
        } else {
            if (v < vocab) f.x = row[v];
            if (v + 1 < vocab) f.y = row[v + 1];
            if (v + 2 < vocab) f.z = row[v + 2];
            if (v + 3 < vocab) f.w = row[v + 3];
        }
        x[4 * u] = f.x == f.x ? f.x : pad;
        x[4 * u + 1] = f.y == f.y ? f.y : pad;
        x[4 * u + 2] = f.z == f.z ? f.z : pad;
        x[4 * u + 3] = f.w == f.w ? f.w : pad;
    }
}
__device__ __forceinline__ int index_of(int v0, int e) {
    return v0 + 4 * (kVThreads * (e / 4) + static_cast<int>(threadIdx.x)) + e % 4;
}

// sum over the block in a fixed order; every thread gets it
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < kVThreads / kWave; ++i) t += red[i];
    return t;
}

__device__ __forceinline__ bool aligned_rows(const float* base, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && ld % 4 == 0;
}

__global__ void __launch_bounds__(kVThreads) verify_stats_kernel(VerifyLaunch p) {
    __shared__ uint64_t best[kVThreads / kWave];
    __shared__ double red[kVThreads / kWave];
    const int piece = blockIdx.x, node = blockIdx.y, v0 = piece * kPiece;
    const VerifyWs ws = verify_ws(p.ws, p.nodes, p.vocab);
    float x[kPer];
    load_piece(p.logits + node * p.ld, p.vocab, v0, aligned_rows(p.logits, p.ld), -INFINITY, x);
    uint64_t key = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) key = u64_max(key, argmax_key(x[e], static_cast<uint32_t>(index_of(v0, e))));
    key = wave_max_u64(key);
    if ((threadIdx.x & (kWave - 1)) == 0) best[threadIdx.x / kWave] = key;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kVThreads / kWave; ++i) key = u64_max(key, best[i]);
    const float m = float_from_order_key(static_cast<uint32_t>(key >> 32));
    double sum = 0.0;
    if (p.inv_t > 0.0f && m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += x[e] > -INFINITY ? weight_of(x[e], m, p.inv_t) : 0.0;
        sum = block_sum_f64(sum, red);
    }
    if (threadIdx.x == 0) {
        ws.stat[node * static_cast<size_t>(gridDim.x) + piece] = Stat{sum, m, static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key))};
        if (piece == 0 && node == 0) *ws.done = 0;
    }
}

// maximum, argmax and exponential sum of a row from its pieces, by 4 lanes each (all four get them)
struct RowStat {
    float m;
    int32_t arg;
    double z;
};
__device__ __forceinline__ RowStat row_stat(const VerifyWs& ws, int node, int pieces, double inv_t) {
    const Stat* s = ws.stat + static_cast<size_t>(node) * pieces;
    const int sub = threadIdx.x & 3;
    uint64_t key = 0;
    for (int i = sub; i < pieces; i += 4) key = u64_max(key, argmax_key(s[i].m, static_cast<uint32_t>(s[i].arg)));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) key = u64_max(key, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(key), o, kWave)));
    RowStat r{float_from_order_key(static_cast<uint32_t>(key >> 32)), static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key)), 0.0};
    if (inv_t > 0.0 && r.m > -INFINITY)
        for (int i = sub; i < pieces; i += 4)
            if (s[i].m > -INFINITY) r.z += s[i].sum * weight_of(s[i].m, r.m, inv_t);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) r.z += __shfl_xor(r.z, o, kWave);
    return r;
}

// c_s of a row: c_1 = 1, c_{s+1} = c_s + d_s with d_s summed over the pieces (by every lane alike)
__device__ __forceinline__ double rest_sum(const VerifyWs& ws, int s, int node, int nodes, int pieces) {
    const double* r = ws.rest + (static_cast<size_t>(s - 1) * nodes + node) * pieces;
    double d = 0.0;
    for (int i = 0; i < pieces; ++i) d += r[i];
    return d;
}

// (p - c q)+ of one token
__device__ __forceinline__ double rest_of(float l, float q, const RowStat& r, double c, double inv_t) {
    const double w = (l > -INFINITY ? weight_of(l, r.m, inv_t) / r.z : 0.0) - c * static_cast<double>(q);
    return w > 0.0 ? w : 0.0;
}

// the partial sums of d_s, s >= 1, for the rows with more than s children
__global__ void __launch_bounds__(kVThreads) verify_rest_kernel(VerifyLaunch p, int s) {
    __shared__ double red[kVThreads / kWave];
    const int piece = blockIdx.x, node = blockIdx.y, v0 = piece * kPiece, pieces = gridDim.x;
    int children = 0;
    for (int j = node + 1; j < p.nodes; ++j) children += p.links.parent[j] == node;
    if (children <= s) return;  // block-uniform
    const VerifyWs ws = verify_ws(p.ws, p.nodes, p.vocab);
    const double inv_t = p.inv_t;
    const RowStat r = row_stat(ws, node, pieces, inv_t);
    double c = 1.0;
    for (int i = 1; i < s; ++i) c += rest_sum(ws, i, node, p.nodes, pieces);
    float l[kPer], q[kPer];
    load_piece(p.logits + node * p.ld, p.vocab, v0, aligned_rows(p.logits, p.ld), -INFINITY, l);
    load_piece(p.draft + node * p.ld_draft, p.vocab, v0, aligned_rows(p.draft, p.ld_draft), 0.0f, q);
    double sum = 0.0;
    if (r.m > -INFINITY)
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += rest_of(l[e], q[e], r, c, inv_t);
    sum = block_sum_f64(sum, red);
    if (threadIdx.x == 0) ws.rest[(static_cast<size_t>(s - 1) * p.nodes + node) * pieces + piece] = sum;
}

// Weights of the sampled distribution over a thread's values of a piece.
// excluded: bit e set where the token was rejected (point masses).
__device__ __forceinline__ double sample_weight(float l, float q, bool excluded, const RowStat& r, double c,
                                                bool draft, double inv_t) {
    if (draft && c > 0.0) return rest_of(l, q, r, c, inv_t);
    return l > -INFINITY && !excluded ? weight_of(l, r.m, inv_t) : 0.0;
}

__global__ void __launch_bounds__(kVThreads) verify_walk_kernel(VerifyLaunch p) {
    __shared__ RowStat row[kTreeMax];
    __shared__ int tok[kTreeMax], next[kTreeMax], tried[kTreeMax];
    __shared__ double prob[kTreeMax], prop[kTreeMax], cut[kTreeMax];
    __shared__ int path[kTreeMax + 1];
    __shared__ int kept_s, last_s;
    __shared__ double red[kVThreads / kWave], scan[kVThreads];
    const int tid = threadIdx.x, n = p.nodes, pieces = verify_pieces(p.vocab);
    const VerifyWs ws = verify_ws(p.ws, n, p.vocab);
    const double inv_t = p.inv_t;
    const bool draft = p.draft != nullptr;
    if (tid / 4 < n) {
        const RowStat r = row_stat(ws, tid / 4, pieces, inv_t);
        if ((tid & 3) == 0) row[tid / 4] = r;
    }
    __syncthreads();
    if (tid < n) {
        const int par = p.links.parent[tid], t = tid > 0 ? p.tokens[tid] : -1;
        tok[tid] = t;
        prob[tid] = prop[tid] = 0.0;
        if (tid > 0 && t >= 0 && t < p.vocab && p.inv_t > 0.0f) {
            const float l = p.logits[par * p.ld + t];
            if (l > -INFINITY && row[par].m > -INFINITY) prob[tid] = weight_of(l, row[par].m, inv_t) / row[par].z;
            prop[tid] = draft ? static_cast<double>(p.draft[par * p.ld_draft + t]) : 1.0;
        }
    }
    __syncthreads();
    if (tid < n) {  // the row's children, in order
        const int i = tid;
        int nx = -1, rejected = 0;
        double c = 0.0, d = 1.0;
        for (int j = i + 1; j < n && nx < 0; ++j) {
            if (p.links.parent[j] != i) continue;
            if (p.inv_t == 0.0f) {
                if (row[i].m > -INFINITY && tok[j] == row[i].arg) nx = j;
                continue;
            }
            bool again = false;  // a rejected sibling's token (point masses: nothing is left of it)
            if (!draft)
                for (int k = i + 1; k < j; ++k) again |= p.links.parent[k] == i && tok[k] == tok[j];
            const double left = again || !(d > 0.0) ? 0.0 : (draft ? fmax(prob[j] - c * prop[j], 0.0) : prob[j]) / d;
            if (static_cast<double>(p.u_accept[j]) * prop[j] < left) {
                nx = j;
                continue;
            }
            ++rejected;
            if (draft) {
                c += d;
                // (d_s is there for s < the row's number of children: no child comes after the last rejection)
                bool more = false;
                for (int k = j + 1; k < n; ++k) more |= p.links.parent[k] == i;
                if (more) d = rest_sum(ws, rejected, i, n, pieces);
            } else if (!again) {
                d -= prob[j];
            }
        }
        next[i] = nx;
        tried[i] = rejected;
        cut[i] = c;
    }
    __syncthreads();
    if (tid == 0) {
        int at = 0, kept = 0;
        path[kept++] = 0;
        while (next[at] >= 0) {
            at = next[at];
            path[kept++] = at;
        }
        kept_s = kept;
    }
    __syncthreads();
    const int kept = kept_s, stop = path[kept - 1];
    const RowStat r = row[stop];
    if (blockIdx.x == 0) {
        if (tid < n) {
            p.out_path[tid] = tid < kept ? path[tid] : -1;
            if (tid + 1 != kept) p.out_tokens[tid] = tid + 1 < kept ? tok[path[tid + 1]] : -1;
        }
        if (tid == 0) *p.out_count = kept;
    }
    if (p.inv_t == 0.0f || !(r.m > -INFINITY)) {  // one block, or nothing to sample
        if (blockIdx.x == 0 && tid == 0) p.out_tokens[kept - 1] = r.m > -INFINITY ? r.arg : -1;
        return;
    }
    const double c = cut[stop];
    const bool al = aligned_rows(p.logits, p.ld), ald = draft && aligned_rows(p.draft, p.ld_draft);
    float l[kPer], q[kPer];
    uint32_t excluded = 0;
    auto load = [&](int v0) {
        load_piece(p.logits + stop * p.ld, p.vocab, v0, al, -INFINITY, l);
        if (draft) load_piece(p.draft + stop * p.ld_draft, p.vocab, v0, ald, 0.0f, q);
        excluded = 0;
        if (!draft)
            for (int j = stop + 1; j < n; ++j) {
                if (p.links.parent[j] != stop) continue;
                const int at = tok[j] - v0;
                if (at >= 0 && at < kPiece && (at / 4) % kVThreads == tid) excluded |= 1u << (4 * (at / 4 / kVThreads) + at % 4);
            }
    };
    const int v0 = blockIdx.x * kPiece;
    load(v0);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum += sample_weight(l[e], draft ? q[e] : 0.0f, excluded >> e & 1, r, c, draft, inv_t);
    sum = block_sum_f64(sum, red);
    if (tid == 0) {
        __hip_atomic_store(ws.weight + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_s = __hip_atomic_fetch_add(ws.done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last_s) return;
    // the last block: the piece that the random number falls into, then the token
    auto piece_sum = [&](int i) { return __hip_atomic_load(ws.weight + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    double total = 0.0;
    for (int i = 0; i < pieces; ++i) total += piece_sum(i);
    // nothing left of it (a draft that covers the target): the target itself
    const bool whole = !(total > 0.0);
    const Stat* st = ws.stat + static_cast<size_t>(stop) * pieces;
    auto share = [&](int i) { return whole ? (st[i].m > -INFINITY ? st[i].sum * weight_of(st[i].m, r.m, inv_t) : 0.0) : piece_sum(i); };
    if (whole) total = r.z;
    const double want = static_cast<double>(*p.u_sample) * total;
    double before = 0.0;
    int pick = -1, fallback = 0;
    for (int i = 0; i < pieces; ++i) {
        const double w = share(i);
        if (w > 0.0) fallback = i;
        if (pick < 0 && before + w > want) pick = i;
        if (pick < 0) before += w;
    }
    if (pick < 0) {  // u_sample >= 1 or NaN: the last token with a weight
        pick = fallback;
        before = -INFINITY;
    }
    load(pick * kPiece);
    double w[kPer];
    const bool ends = before == -INFINITY;
    int found = 0x7fffffff, at_least = -1;  // first token past `want`, last token with a weight
#pragma unroll
    for (int u = 0; u < kPer / 4; ++u) {
        double s4 = 0.0;
#pragma unroll
        for (int e = 4 * u; e < 4 * u + 4; ++e) {
            w[e] = sample_weight(l[e], draft && !whole ? q[e] : 0.0f, !whole && (excluded >> e & 1), r, whole ? 0.0 : c, draft, inv_t);
            s4 += w[e];
        }
        __syncthreads();
        scan[tid] = s4;
        __syncthreads();
        double pre = ends ? 0.0 : before, all = 0.0;
        for (int i = 0; i < kVThreads; ++i) {
            if (i < tid) pre += scan[i];
            all += scan[i];
        }
#pragma unroll
        for (int e = 4 * u; e < 4 * u + 4; ++e) {
            pre += w[e];
            if (w[e] > 0.0) {
                at_least = max(at_least, index_of(pick * kPiece, e));
                if (!ends && pre > want) found = min(found, index_of(pick * kPiece, e));
            }
        }
        if (!ends) before += all;
    }
    __shared__ int lo, hi;
    if (tid == 0) {
        lo = 0x7fffffff;
        hi = -1;
    }
    __syncthreads();
    atomicMin(&lo, found);
    atomicMax(&hi, at_least);
    __syncthreads();
    if (tid == 0) p.out_tokens[kept - 1] = lo != 0x7fffffff ? lo : hi;
}

hipError_t launch_verify(const VerifyLaunch& p, hipStream_t s) {
    const int pieces = verify_pieces(p.vocab);
    hipLaunchKernelGGL(verify_stats_kernel, dim3(pieces, p.nodes), dim3(kVThreads), 0, s, p);
    if (p.draft)
        for (int r = 1; r < p.max_children; ++r)
            hipLaunchKernelGGL(verify_rest_kernel, dim3(pieces, p.nodes), dim3(kVThreads), 0, s, p, r);
    hipLaunchKernelGGL(verify_walk_kernel, dim3(p.inv_t > 0.0f ? pieces : 1), dim3(kVThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
