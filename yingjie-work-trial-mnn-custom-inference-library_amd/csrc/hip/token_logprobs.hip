// token_logprobs.hip - log probabilities of given tokens, entropy, rank and the
// first alternatives of rows of logits.
#include <algorithm>
#include <type_traits>

#include "xqhip_common.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

// ---------------------------------------------------------------------------
// With m the largest logit, d_i = (x_i - m) / T and s' the sum of exp(d_i)
// without one term of the maximum: log p_t = d_t - log1p(s'), entropy =
// log1p(s') - sum exp(d_i) d_i / (1 + s').  Without the 1 in the sum a
// probability near 1 keeps its digits.  Two parts of a row, m1 >= m2, join as
//   s' = s1' + (s2' + 1) exp((m2 - m1) / T).
// Equal infinities differ by 0.
//
// logprobs_part_kernel: one pass over the logits.  A wave takes a segment of
//   1024 (more where the row would have over 1024 segments), held in registers:
//   its maximum and where it is, s', the sum of exp(d) d, how many logits come
//   before the given token's.  No barrier, no LDS.
// logprobs_row_kernel: a block per row joins the segments.  The k first tokens
//   lie in the k segments with the first maxima; of those, in the k threads'
//   shares with the first maxima: the rest is never looked at again.
// What bounds it: the logits' bytes, and for one row a chain of two launches.
// ---------------------------------------------------------------------------
constexpr int kSegment = 1024;   // logits of a wave's pass
constexpr int kMostSegments = 1024;
constexpr int kPartWaves = 4;
constexpr int kRowThreads = 512, kFewThreads = 256;
constexpr int kCandidates = 2048;  // candidates of a row that are held
constexpr int kMany = 512;         // ... that are put in order as they are
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LogPart {
    float m, s, h;  // maximum, s', sum of exp(d) d in units of ln 2
    int32_t before;
};

// log2 of the passes of 1024 that a segment holds
__host__ __device__ inline int segment_shift(int vocab) {
    int n = 0;
    while ((static_cast<int64_t>(kSegment) << n) * kMostSegments < vocab) ++n;
    return n;
}
__host__ __device__ inline int segment_count(int vocab) {
    const int size = kSegment << segment_shift(vocab);
    return (vocab + size - 1) / size;
}
size_t logprobs_workspace_bytes(int rows, int vocab, int) {
    return static_cast<size_t>(rows) * segment_count(vocab) * (sizeof(LogPart) + sizeof(int32_t)) + 16;
}

// (x - m) / T in units of ln 2, 2^-200 and less is nothing (minus infinity, and infinity less infinity too)
__device__ __forceinline__ float gap2(float x, float m, float c) { return fmaxf((x - m) * c, -200.0f); }
__device__ __forceinline__ float logit_gap(float x, float m, float inv_t) { return x == m ? 0.0f : (x - m) * inv_t; }
template <bool F16>
__device__ __forceinline__ float logit_at(const void* row, int i) {
    const float x = F16 ? static_cast<float>(static_cast<const _Float16*>(row)[i]) : static_cast<const float*>(row)[i];
    return fmaxf(x, -INFINITY);  // NaN counts as minus infinity
}
template <bool F16>
__device__ __forceinline__ const void* logit_row(const LogprobsLaunch& p, int row) {
    const size_t at = static_cast<size_t>(row) * p.ld;
    return F16 ? static_cast<const void*>(static_cast<const _Float16*>(p.logits) + at)
               : static_cast<const void*>(static_cast<const float*>(p.logits) + at);
}

__device__ __forceinline__ int wave_min_int(int v) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) v = min(v, __shfl_xor(v, o, kWave));
    return v;
}

// 16 logits of a lane: index of element e
template <bool F16, bool VEC>
__device__ __forceinline__ int element(int lane, int e) {
    constexpr int N = F16 ? 8 : 4;  // of a 16-byte load
    return VEC ? (e / N * kWave + lane) * N + e % N : e * kWave + lane;
}

template <bool F16, bool VEC>
__global__ void __launch_bounds__(kWave* kPartWaves) logprobs_part_kernel(LogprobsLaunch p, int segments, int shift) {
    constexpr int E = kSegment / kWave, N = F16 ? 8 : 4;
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, row = blockIdx.y;
    const int seg = __builtin_amdgcn_readfirstlane(blockIdx.x * kPartWaves + wid);
    if (seg >= segments) return;
    const void* x0 = logit_row<F16>(p, row);
    const float c = p.inv_t * kLog2e;
    float M = -INFINITY, S = 0.0f, H = 0.0f;  // the segment so far
    int arg = 0x7fffffff, before = 0;
    int t = -1;
    float xt = 0.0f;
    bool has = false;
    for (int it = 0; it < 1 << shift; ++it) {
        const int i0 = ((seg << shift) + it) * kSegment;
        if (i0 >= p.vocab) break;
        float x[E];
        if (i0 + kSegment <= p.vocab) {
            if constexpr (VEC) {
#pragma unroll
                for (int u = 0; u < E / N; ++u) {
                    if constexpr (F16) {
                        typedef _Float16 half8 __attribute__((ext_vector_type(8)));
                        const half8 v = *reinterpret_cast<const half8*>(static_cast<const _Float16*>(x0) + i0 + (u * kWave + lane) * N);
#pragma unroll
                        for (int e = 0; e < N; ++e) x[u * N + e] = static_cast<float>(v[e]);
                    } else {
                        const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(x0) + i0 + (u * kWave + lane) * N);
                        x[u * N] = v.x;
                        x[u * N + 1] = v.y;
                        x[u * N + 2] = v.z;
                        x[u * N + 3] = v.w;
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    x[e] = F16 ? static_cast<float>(static_cast<const _Float16*>(x0)[i0 + element<F16, VEC>(lane, e)])
                               : static_cast<const float*>(x0)[i0 + element<F16, VEC>(lane, e)];
            }
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = fmaxf(x[e], -INFINITY);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = i0 + element<F16, VEC>(lane, e);
                x[e] = i < p.vocab ? logit_at<F16>(x0, i) : -INFINITY;
            }
        }
        if (it == 0 && p.out_rank) {  // (after the segment's own loads: two round trips beside them)
            t = p.tokens[row];
            has = t >= 0 && t < p.vocab;
            xt = logit_at<F16>(x0, has ? t : 0);
        }
        float m = x[0];
#pragma unroll
        for (int e = 1; e < E; ++e) m = fmaxf(m, x[e]);
        m = wave_max(m);
        if (has && m >= xt) {  // wave-uniform
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = i0 + element<F16, VEC>(lane, e);
                before += __popcll(__builtin_amdgcn_ballot_w64(i < p.vocab && (x[e] > xt || (x[e] == xt && i < t))));
            }
        }
        int at = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < E; ++e) at = x[e] == m ? min(at, i0 + element<F16, VEC>(lane, e)) : at;
        at = wave_min_int(at);
        float s = 0.0f, h = 0.0f;
        int same = 0;
        if (m > -INFINITY) {  // wave-uniform
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = gap2(x[e], m, c);
                const bool top = x[e] == m;
                same += __popcll(__builtin_amdgcn_ballot_w64(top));
                const float w = top ? 0.0f : __builtin_amdgcn_exp2f(d);
                s += w;
                h = fmaf(w, d, h);
            }
            s = wave_sum(s) + static_cast<float>(same - 1);
            h = wave_sum(h);
            if (M == -INFINITY) {
                M = m;
                S = s;
                H = h;
                arg = at;
            } else {  // (the earlier part keeps ties)
                const bool up = m > M;
                const float d = m == M ? 0.0f : gap2(fminf(m, M), fmaxf(m, M), c), w = __builtin_amdgcn_exp2f(d);
                const float s1 = up ? s : S, h1 = up ? h : H, s2 = up ? S : s, h2 = up ? H : h;
                S = s1 + (s2 + 1.0f) * w;
                H = h1 + w * (h2 + d * (s2 + 1.0f));
                M = up ? m : M;
                arg = up ? at : arg;
            }
        }
    }
    if (lane == 0) {
        const size_t o = static_cast<size_t>(row) * segments + seg;
        static_cast<LogPart*>(p.ws)[o] = LogPart{M, S, H, before};
        reinterpret_cast<int32_t*>(static_cast<LogPart*>(p.ws) + static_cast<size_t>(p.rows) * segments)[o] = arg;
    }
}

// A threshold that the k largest of the wave's keys reach and no other (0 where there are no more than k).  Keys that are
// not 0 differ.
template <int R>
__device__ __forceinline__ uint64_t kth_largest(const uint64_t (&key)[R], int k) {
    auto count = [&](auto reaches) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(reaches(key[i])));
        return n;
    };
    if (count([](uint64_t v) { return v != 0; }) <= k) return 0;
    uint32_t h = 0;
    for (int b = 31; b >= 0; --b) {
        const uint32_t to = h | 1u << b;
        const int n = count([&](uint64_t v) { return static_cast<uint32_t>(v >> 32) >= to; });
        if (n == k) return static_cast<uint64_t>(to) << 32;
        if (n > k) h = to;
    }
    const int left = k - count([&](uint64_t v) { return static_cast<uint32_t>(v >> 32) > h; });
    uint32_t l = 0;
    for (int b = 31; b >= 0; --b) {
        const uint32_t to = l | 1u << b;
        const int n = count([&](uint64_t v) { return static_cast<uint32_t>(v >> 32) == h && static_cast<uint32_t>(v) >= to; });
        if (n >= left) l = to;
    }
    return static_cast<uint64_t>(h) << 32 | l;
}

template <int THREADS>
__device__ __forceinline__ float block_total(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) t += red[i];
    return t;
}
template <int THREADS>
__device__ __forceinline__ uint64_t block_most(uint64_t v, uint64_t* red) {
    v = wave_max_u64(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < THREADS / kWave; ++i) v = u64_max(v, red[i]);
    return v;
}

template <bool F16, bool VEC, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS) logprobs_row_kernel(LogprobsLaunch p, int segments, int shift) {
    constexpr int kPer = kMostSegments / THREADS;
    __shared__ uint64_t red[THREADS / kWave];
    __shared__ float fred[THREADS / kWave];
    const int row = blockIdx.x, lane = threadIdx.x & (kWave - 1);
    const void* x0 = logit_row<F16>(p, row);
    const LogPart* parts = static_cast<const LogPart*>(p.ws) + static_cast<size_t>(row) * segments;
    const int32_t* args = reinterpret_cast<const int32_t*>(static_cast<const LogPart*>(p.ws) + static_cast<size_t>(p.rows) * segments) +
                          static_cast<size_t>(row) * segments;
    const int t = p.tokens ? p.tokens[row] : -1;
    const bool has = t >= 0 && t < p.vocab;
    const float xt = has ? logit_at<F16>(x0, t) : 0.0f;
    LogPart part[kPer];
    uint64_t key[kPer], best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int s = i * THREADS + threadIdx.x;
        part[i] = LogPart{-INFINITY, 0.0f, 0.0f, 0};
        key[i] = 0;
        if (s < segments) {
            part[i] = parts[s];
            key[i] = part[i].m > -INFINITY ? argmax_key(part[i].m, args[s]) : 0;
        }
        best = u64_max(best, key[i]);
    }
    best = block_most<THREADS>(best, red);
    const bool any = best != 0;
    const float m = any ? float_from_order_key(static_cast<uint32_t>(best >> 32)) : -INFINITY, c = p.inv_t * kLog2e;
    float s = 0.0f, h = 0.0f;
    int before = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        before += part[i].before;
        if (key[i] == 0) continue;
        const float d = part[i].m == m ? 0.0f : gap2(part[i].m, m, c), w = __builtin_amdgcn_exp2f(d);
        s += (part[i].s + (key[i] == best ? 0.0f : 1.0f)) * w;
        h += w * (part[i].h + d * (part[i].s + 1.0f));
    }
    s = block_total<THREADS>(s, fred);
    h = block_total<THREADS>(h, fred);
    const float lz = log1pf(s);
    if (p.out_rank) {
        // (vocab <= 2^24: a sum of counts is exact)
        const float n = block_total<THREADS>(static_cast<float>(before), fred);
        if (threadIdx.x == 0) p.out_rank[row] = has ? static_cast<int32_t>(n) : -1;
    }
    if (threadIdx.x == 0) {
        if (p.out_logprob) p.out_logprob[row] = any && has ? logit_gap(xt, m, p.inv_t) - lz : -INFINITY;
        if (p.out_entropy) p.out_entropy[row] = any ? lz - kLn2 * h / (1.0f + s) : 0.0f;
    }
    if constexpr (TOP) {
        __shared__ uint64_t keys[kMostSegments];  // of segments, then of threads
        __shared__ uint64_t cand[kCandidates];
        __shared__ uint64_t limit;
        __shared__ int list[64], count;
        static_assert(THREADS <= kMostSegments, "one key a thread");
        const int k = p.top, size = kSegment << shift;
#pragma unroll
        for (int i = 0; i < kPer; ++i) keys[i * THREADS + threadIdx.x] = key[i];
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        if (threadIdx.x < kWave) {
            uint64_t l = 0;
            if (segments > k) {
                if (segments <= 4 * kWave) {
                    uint64_t v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = keys[i * kWave + lane];
                    l = kth_largest(v, k);
                } else {
                    uint64_t v[kMostSegments / kWave];
#pragma unroll
                    for (int i = 0; i < kMostSegments / kWave; ++i) v[i] = keys[i * kWave + lane];
                    l = kth_largest(v, k);
                }
            }
            if (lane == 0) limit = l;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (key[i] != 0 && key[i] >= limit) list[atomicAdd(&count, 1)] = i * THREADS + threadIdx.x;
        __syncthreads();
        // the segments' logits by the block, kBatch loads of a thread in flight: each(logit, index)
        constexpr int N = VEC ? (F16 ? 8 : 4) : 1, kBatch = 8;
        const int loads = (count << (shift + 10)) / N, per = size / N;
        auto walk = [&](auto each) {
            for (int e0 = threadIdx.x; e0 < loads; e0 += kBatch * THREADS) {
                int at[kBatch];
                float x[kBatch][N];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int e = e0 + u * THREADS;
                    at[u] = e < loads ? list[e / per] * size + e % per * N : p.vocab;
#pragma unroll
                    for (int i = 0; i < N; ++i) x[u][i] = -INFINITY;
                    if (at[u] + N <= p.vocab) {
                        typedef typename std::conditional<F16, _Float16, float>::type T;
                        typedef T piece __attribute__((ext_vector_type(N)));
                        const piece v = *reinterpret_cast<const piece*>(static_cast<const T*>(x0) + at[u]);
#pragma unroll
                        for (int i = 0; i < N; ++i) x[u][i] = fmaxf(static_cast<float>(v[i]), -INFINITY);
                    } else {
                        for (int i = 0; i < N; ++i)
                            if (at[u] + i < p.vocab) x[u][i] = logit_at<F16>(x0, at[u] + i);
                    }
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
#pragma unroll
                    for (int i = 0; i < N; ++i) each(x[u][i], at[u] + i);
            }
        };
        // the candidates: logits that the k-th segment's maximum does not pass, not many more than k as a rule
        auto collect = [&](uint64_t least) {
            const float low = float_from_order_key(static_cast<uint32_t>(least >> 32));
            walk([&](float x, int i) {
                if (x < low || x == -INFINITY) return;
                const uint64_t v = argmax_key(x, i);
                if (v < least) return;
                const int at = atomicAdd(&count, 1);
                if (at < kCandidates) cand[at] = v;
            });
        };
        const uint64_t reached = limit;
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        if (reached) collect(reached);
        __syncthreads();
        if (!reached || count > kMany) {  // few segments, or many candidates in one: the same once more with the threads' shares
            __syncthreads();
            uint64_t mine = 0;
            walk([&](float x, int i) { mine = u64_max(mine, x > -INFINITY ? argmax_key(x, i) : 0); });
            keys[threadIdx.x] = mine;
            if (threadIdx.x == 0) count = 0;
            __syncthreads();
            if (threadIdx.x < kWave) {
                uint64_t v[THREADS / kWave];
#pragma unroll
                for (int i = 0; i < THREADS / kWave; ++i) v[i] = keys[i * kWave + lane];
                const uint64_t l = kth_largest(v, k);
                if (lane == 0) limit = l;
            }
            __syncthreads();
            const uint64_t least = u64_max(limit, 1);
            if (mine >= least) collect(least);
            __syncthreads();
        }
        const int n = count;
        auto put = [&](int place, uint64_t v) {
            const size_t o = static_cast<size_t>(row) * k + place;
            if (p.out_top) p.out_top[o] = v ? static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(v)) : -1;
            if (p.out_top_logprob)
                p.out_top_logprob[o] = v ? logit_gap(float_from_order_key(static_cast<uint32_t>(v >> 32)), m, p.inv_t) - lz : -INFINITY;
        };
        if (n <= kCandidates) {
            for (int i = threadIdx.x; i < n; i += THREADS) {
                const uint64_t v = cand[i];
                int place = 0;
                for (int j = 0; j < n; ++j) place += cand[j] > v;
                if (place < k) put(place, v);
            }
            for (int i = n + threadIdx.x; i < k; i += THREADS) put(i, 0);
            return;
        }
        // (a few threads' shares hold more than the list: rows whose largest logits lie at the threads' stride)
        uint64_t before_it = ~uint64_t(0);
        for (int i = 0; i < k; ++i) {
            uint64_t next = 0;
            walk([&](float x, int at) {
                const uint64_t v = x > -INFINITY ? argmax_key(x, at) : 0;
                next = v < before_it ? u64_max(next, v) : next;
            });
            before_it = block_most<THREADS>(next, red);
            if (threadIdx.x == 0) put(i, before_it);
        }
    }
}

hipError_t launch_logprobs(const LogprobsLaunch& p, hipStream_t s) {
    const int segments = segment_count(p.vocab), shift = segment_shift(p.vocab);
    const dim3 grid((segments + kPartWaves - 1) / kPartWaves, p.rows), block(kWave * kPartWaves);
    const bool vec = (reinterpret_cast<uintptr_t>(p.logits) & 15u) == 0 && p.ld % (p.f16 ? 8 : 4) == 0;
    if (p.f16 && vec)
        hipLaunchKernelGGL((logprobs_part_kernel<true, true>), grid, block, 0, s, p, segments, shift);
    else if (p.f16)
        hipLaunchKernelGGL((logprobs_part_kernel<true, false>), grid, block, 0, s, p, segments, shift);
    else if (vec)
        hipLaunchKernelGGL((logprobs_part_kernel<false, true>), grid, block, 0, s, p, segments, shift);
    else
        hipLaunchKernelGGL((logprobs_part_kernel<false, false>), grid, block, 0, s, p, segments, shift);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    auto rows = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(p.rows), dim3(threads), 0, s, p, segments, shift); };
    if (p.top == 0)
        p.f16 ? rows(logprobs_row_kernel<true, false, false, kFewThreads>, kFewThreads) : rows(logprobs_row_kernel<false, false, false, kFewThreads>, kFewThreads);
    else if (vec)
        p.f16 ? rows(logprobs_row_kernel<true, true, true, kRowThreads>, kRowThreads) : rows(logprobs_row_kernel<false, true, true, kRowThreads>, kRowThreads);
    else
        p.f16 ? rows(logprobs_row_kernel<true, false, true, kRowThreads>, kRowThreads) : rows(logprobs_row_kernel<false, false, true, kRowThreads>, kRowThreads);
    return hipGetLastError();
}

}  // namespace xqhip
