// token_logprobs.hip - log probabilities of given tokens, entropy, rank and the
// first alternatives of rows of logits.
#include <algorithm>
#include <type_traits>

#include "xqhip.h"
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
// logprobs_small_kernel: rows of up to 16384 logits, a block per row, the row in
//   registers: one launch (one row of 8192 4.1 us, by two launches 6.0; 200 fp16
//   rows of 16000, 20 alternatives 11.9, 14.5; one of 16384 6.4, 6.1).  One wave
//   for up to 1024 (5000 rows of 100 7.5 us, by eight waves 31), 16 logits a
//   thread for up to 8192 (one row of 8000, 5 alternatives 6.9 us; 32 a thread 9.8).
// logprobs_part_kernel: one pass over the logits.  A wave takes a segment (16
//   fp32 logits a lane or 32 fp16 ones; more where the row would have over 1024
//   segments) in registers: its maximum, s', the sum of exp(d) d, how many
//   logits come before the given token's, and each lane's maximum.  No barrier,
//   no LDS.
// logprobs_row_kernel: a block per row joins the segments.  A value that k
//   segments' maxima reach is reached by the k first tokens: the lanes whose
//   maxima reach it, in those segments, are all that is looked at again.  With
//   fewer than 8 k segments (of up to 256) the threads' shares of all lanes'
//   maxima stand in for the segments: 200 rows of 25 segments, 20 alternatives
//   19.5 us (by segments 28.8); one row of 243 segments, 20 alternatives, by
//   segments 9.8 (so 11.2).  Between them the sides are close: 48 rows of 122
//   segments with 64 alternatives 22.3 (by segments 23.9), with 20 19.2 (17.7).
// What bounds it: the logits' bytes (500 fp32 rows of 248320, 497 MB, 83 us, 6.0
// TB/s); with fp16 logits the vector units are busy for half of the time (48 rows
// 9 to 10 us; 15 instructions a logit, 4.7 us of them) and the waves, which are all on
// the card at once, wait for their loads in the other; for one row a chain of two
// launches, 3.7 and 5.5 us.
// ---------------------------------------------------------------------------
constexpr int kMostSegments = 1024, kFewSegments = 256;
constexpr int kPartWaves = 4;
constexpr int kRun = 8;  // logits of a lane
constexpr int kRowThreads = 512, kFewThreads = 256;
constexpr int kCandidates = 2048;  // candidates of a row that are held
constexpr int kMany = 512;         // ... that are put in order as they are
constexpr int kMostLanes = 1024;   // lanes of a row that are looked at again
constexpr float kTwoLog2e = 2 * 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// Segments of a row.
struct Segments {
    int count, shift;  // each of 64 E << shift logits
};
template <bool F16>
constexpr int kLaneLogits = F16 ? 32 : 16;  // E, of a lane and pass
__host__ __device__ inline Segments segments_of(int vocab, bool f16) {
    const int64_t pass = f16 ? kLaneLogits<true> * kWave : kLaneLogits<false> * kWave;
    int n = 0;
    while ((pass << n) * kMostSegments < vocab) ++n;
    return Segments{static_cast<int>((vocab + (pass << n) - 1) / (pass << n)), n};
}

struct LogPart {
    float m, s, h;  // maximum, s', sum of exp(d) d in units of ln 2
    int32_t before;
};
static_assert(sizeof(LogPart) == 16, "the lanes' maxima follow, 16-byte aligned");

size_t logprobs_workspace_bytes(int rows, int vocab, int top) {
    const size_t n = static_cast<size_t>(rows) * std::max(segments_of(vocab, false).count, segments_of(vocab, true).count);
    return n * (sizeof(LogPart) + (top ? kWave * sizeof(float) : 0));
}

// (x - m) / T in units of ln 2 (c: 2 / (T ln 2)), 2^-200 and less is nothing (minus infinity, no number, and infinity less infinity too).
// Half the difference: of two logits it is in fp32's range, and rounded as the whole one.
__device__ __forceinline__ float half_gap(float x, float m) { return fmaf(x, 0.5f, -0.5f * m); }
__device__ __forceinline__ float gap2(float x, float m, float c) { return fmaxf(half_gap(x, m) * c, -200.0f); }
__device__ __forceinline__ float logit_gap(float x, float m, float inv_t) { return x == m ? 0.0f : 2.0f * (half_gap(x, m) * inv_t); }
template <bool F16>
using logit_t = typename std::conditional<F16, _Float16, float>::type;
template <bool F16>
__device__ __forceinline__ const logit_t<F16>* logit_row(const LogprobsLaunch& p, int row) {
    return static_cast<const logit_t<F16>*>(p.logits) + static_cast<size_t>(row) * p.ld;
}
// NaN counts as minus infinity
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }

// a lane's logit e of a pass: VEC: in 16-byte pieces
template <bool F16, bool VEC>
__device__ __forceinline__ int element(int lane, int e) {
    constexpr int N = F16 ? 8 : 4;
    return VEC ? (e / N * kWave + lane) * N + e % N : e * kWave + lane;
}

template <bool F16, bool VEC>
__global__ void __launch_bounds__(kWave* kPartWaves) logprobs_part_kernel(LogprobsLaunch p, Segments sg) {
    typedef logit_t<F16> L;
    constexpr int E = kLaneLogits<F16>, N = 16 / sizeof(L), kPass = E * kWave;
    typedef L piece __attribute__((ext_vector_type(N)));
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, row = blockIdx.y;
    const int seg = __builtin_amdgcn_readfirstlane(blockIdx.x * kPartWaves + wid);
    if (seg >= sg.count) return;
    const L* x0 = logit_row<F16>(p, row);
    const float c = p.inv_t * kTwoLog2e;
    float M = -INFINITY, S = 0.0f, H = 0.0f, mine = -INFINITY;  // the segment so far, this lane's maximum
    int before = 0, t = -1;
    float xt = 0.0f;
    for (int it = 0; it < 1 << sg.shift; ++it) {
        const int i0 = ((seg << sg.shift) + it) * kPass;
        if (i0 >= p.vocab) break;
        float x[E];
        if (VEC && i0 + kPass <= p.vocab) {
            piece v[E / N];
#pragma unroll
            for (int u = 0; u < E / N; ++u) v[u] = *reinterpret_cast<const piece*>(x0 + i0 + (u * kWave + lane) * N);
            if (it == 0 && p.out_rank) t = p.tokens[row];  // (behind the segment's loads, beside which it comes)
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = static_cast<float>(v[e / N][e % N]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = i0 + element<F16, VEC>(lane, e);
                const float v = static_cast<float>(x0[min(i, p.vocab - 1)]);  // (no branches: the loads go out together)
                x[e] = i < p.vocab ? v : -INFINITY;
            }
            if (it == 0 && p.out_rank) t = p.tokens[row];
        }
        const bool has = t >= 0 && t < p.vocab;  // wave-uniform
        if (it == 0 && has) xt = clean(static_cast<float>(x0[t]));
        float lm = -INFINITY, rm[E / kRun];  // of a lane, of its runs
#pragma unroll
        for (int r = 0; r < E / kRun; ++r) {
            rm[r] = x[kRun * r];
#pragma unroll
            for (int e = 1; e < kRun; ++e) rm[r] = fmaxf(rm[r], x[kRun * r + e]);
            lm = fmaxf(lm, rm[r]);
        }
        mine = fmaxf(mine, lm);
        const float m = wave_max(lm);
        if (has && m >= xt) {  // wave-uniform
#pragma unroll
            for (int e = 0; e < E; ++e) before += __popcll(__builtin_amdgcn_ballot_w64(x[e] > xt));
            uint64_t ties = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) ties |= __builtin_amdgcn_ballot_w64(clean(x[e]) == xt);
            if (ties)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    before += __popcll(__builtin_amdgcn_ballot_w64(clean(x[e]) == xt && i0 + element<F16, VEC>(lane, e) < t));
        }
        if (m > -INFINITY) {  // wave-uniform
            float s = 0.0f, h = 0.0f;
            int same = 0;
#pragma unroll
            for (int r = 0; r < E / kRun; ++r) {
                if (__builtin_amdgcn_ballot_w64(rm[r] == m)) {  // wave-uniform: only there the maximum is looked for
#pragma unroll
                    for (int e = kRun * r; e < kRun * (r + 1); ++e) {
                        const float d = gap2(x[e], m, c);
                        const bool top = x[e] == m;
                        same += __popcll(__builtin_amdgcn_ballot_w64(top));
                        const float w = top ? 0.0f : __builtin_amdgcn_exp2f(d);
                        s += w;
                        h = fmaf(w, d, h);
                    }
                } else {
#pragma unroll
                    for (int e = kRun * r; e < kRun * (r + 1); ++e) {
                        const float d = gap2(x[e], m, c), w = __builtin_amdgcn_exp2f(d);
                        s += w;
                        h = fmaf(w, d, h);
                    }
                }
            }
            s = wave_sum(s) + static_cast<float>(same - 1);
            h = wave_sum(h);
            if (M == -INFINITY) {
                M = m;
                S = s;
                H = h;
            } else {
                const bool up = m > M;
                const float d = m == M ? 0.0f : gap2(fminf(m, M), fmaxf(m, M), c), w = __builtin_amdgcn_exp2f(d);
                const float s1 = up ? s : S, h1 = up ? h : H, s2 = up ? S : s, h2 = up ? H : h;
                S = s1 + (s2 + 1.0f) * w;
                H = h1 + w * (h2 + d * (s2 + 1.0f));
                M = up ? m : M;
            }
        }
    }
    LogPart* parts = static_cast<LogPart*>(p.ws);
    const size_t at = static_cast<size_t>(row) * sg.count + seg;
    if (lane == 0) parts[at] = LogPart{M, S, H, before};
    if (p.top) reinterpret_cast<float*>(parts + static_cast<size_t>(p.rows) * sg.count)[at * kWave + lane] = mine;
}

// A threshold that the k largest of the wave's keys reach and no other (0 where there are no more than k).  Keys that are
// not 0 differ.
template <int R>
__device__ __forceinline__ uint64_t kth_largest(const uint64_t (&key)[R], int k) {
    auto count = [&](auto reaches) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(reaches(static_cast<uint32_t>(key[i] >> 32), static_cast<uint32_t>(key[i]))));
        return n;
    };
    if (count([](uint32_t v, uint32_t) { return v != 0; }) <= k) return 0;
    uint32_t h = 0;
    for (int b = 31; b >= 0; --b) {
        const uint32_t to = h | 1u << b;
        const int n = count([&](uint32_t v, uint32_t) { return v >= to; });
        if (n == k) return static_cast<uint64_t>(to) << 32;
        if (n > k) h = to;
    }
    const int left = k - count([&](uint32_t v, uint32_t) { return v > h; });
    uint32_t l = 0;
    for (int b = 31; b >= 0; --b) {
        const uint32_t to = l | 1u << b;
        const int n = count([&](uint32_t v, uint32_t i) { return v == h && i >= to; });
        if (n >= left) l = to;
    }
    return static_cast<uint64_t>(h) << 32 | l;
}

// A value that at least k and not many more of the wave's order keys reach, by halving the range between the least and the
// largest; 0 where fewer than k are above 0, or ties leave no such value.
template <int R>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&v)[R], int k) {
    const int most = k + 4 + k / 4;
    auto count = [&](uint32_t to) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(v[i] >= to));
        return n;
    };
    uint32_t low = ~0u, high = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        low = v[i] ? min(low, v[i]) : low;
        high = max(high, v[i]);
    }
    low = ~static_cast<uint32_t>(wave_max_u64(~low));
    high = static_cast<uint32_t>(wave_max_u64(high));
    const int all = count(1);
    if (all < k) return 0;
    if (all <= most) return low;
    while (low < high) {  // more than `most` reach low, fewer than k reach high + 1
        const uint32_t mid = low + (high - low + 1) / 2;
        const int n = count(mid);
        if (n >= k && n <= most) return mid;
        if (n > k)
            low = mid;
        else
            high = mid - 1;
    }
    return 0;
}

// The first of a row's n candidates, by a block of `threads`.
__device__ __forceinline__ void put_in_order(const LogprobsLaunch& p, int row, const uint64_t* cand, int n, float m, float lz, int threads) {
    const int k = p.top;
    auto put = [&](int place, uint64_t v) {
        const size_t o = static_cast<size_t>(row) * k + place;
        if (p.out_top) p.out_top[o] = v ? static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(v)) : -1;
        if (p.out_top_logprob)
            p.out_top_logprob[o] = v ? logit_gap(float_from_order_key(static_cast<uint32_t>(v >> 32)), m, p.inv_t) - lz : -INFINITY;
    };
    for (int i = threadIdx.x; i < n; i += threads) {
        const uint64_t v = cand[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += cand[j] > v;
        if (place < k) put(place, v);
    }
    for (int i = n + threadIdx.x; i < k; i += threads) put(i, 0);
}

template <bool F16, bool VEC, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS) logprobs_row_kernel(LogprobsLaunch p, Segments sg) {
    typedef logit_t<F16> L;
    constexpr int kPer = kMostSegments / THREADS, kWaves = THREADS / kWave;
    __shared__ uint64_t red[kWaves];
    __shared__ float4 sums[kWaves];
    const int row = blockIdx.x, lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    const L* x0 = logit_row<F16>(p, row);
    const LogPart* parts = static_cast<const LogPart*>(p.ws) + static_cast<size_t>(row) * sg.count;
    LogPart part[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int s = i * THREADS + threadIdx.x;
        part[i] = LogPart{-INFINITY, 0.0f, 0.0f, 0};
        if (s < sg.count) part[i] = parts[s];
    }
    const int t = p.tokens ? p.tokens[row] : -1;
    const bool has = t >= 0 && t < p.vocab;
    const float xt = has ? clean(static_cast<float>(x0[t])) : 0.0f;
    uint64_t key[kPer], best = 0;  // of the maximum and the segment
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        key[i] = part[i].m > -INFINITY ? argmax_key(part[i].m, i * THREADS + threadIdx.x) : 0;
        best = u64_max(best, key[i]);
    }
    best = wave_max_u64(best);
    if (lane == 0) red[wid] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) best = u64_max(best, red[i]);
    const bool any = best != 0;
    const float m = any ? float_from_order_key(static_cast<uint32_t>(best >> 32)) : -INFINITY, c = p.inv_t * kTwoLog2e;
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
    s = wave_sum(s);
    h = wave_sum(h);
    const float ahead = wave_sum(static_cast<float>(before));  // (vocab <= 2^24: a sum of counts is exact)
    if (lane == 0) sums[wid] = make_float4(s, h, ahead, 0.0f);
    if constexpr (!TOP) {
        __syncthreads();
        if (threadIdx.x != 0) return;
    }
    auto finish = [&] {  // log of the sum; the row's own outputs by thread 0
        float4 a = sums[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) {
            a.x += sums[i].x;
            a.y += sums[i].y;
            a.z += sums[i].z;
        }
        const float lz = log1pf(a.x);
        if (threadIdx.x == 0) {
            if (p.out_rank) p.out_rank[row] = has ? static_cast<int32_t>(a.z) : -1;
            if (p.out_logprob) p.out_logprob[row] = any && has ? logit_gap(xt, m, p.inv_t) - lz : -INFINITY;
            if (p.out_entropy) p.out_entropy[row] = any ? lz - kLn2 * a.y / (1.0f + a.x) : 0.0f;
        }
        return lz;
    };
    if constexpr (!TOP) {
        finish();
    } else {
        __shared__ uint64_t keys[kMostSegments];  // of segments, then of threads
        __shared__ uint64_t cand[kCandidates];
        __shared__ int list[kMostSegments], lanes[kMostLanes];
        __shared__ uint64_t limit;
        __shared__ int counts[3];  // segments, lanes, candidates
        constexpr int E = kLaneLogits<F16>, kPass = E * kWave;
        const int k = p.top;
        if (threadIdx.x < 3) counts[threadIdx.x] = 0;
        __syncthreads();
        const float lz = finish();
        const float* maxima = reinterpret_cast<const float*>(static_cast<const LogPart*>(p.ws) + static_cast<size_t>(p.rows) * sg.count) +
                              static_cast<size_t>(row) * sg.count * kWave;
        auto add_lane = [&](int e) {
            const int at = atomicAdd(&counts[1], 1);
            if (at < kMostLanes) lanes[at] = e;
        };
        uint32_t value;  // at least k logits reach it: order key
        if (sg.count <= kFewSegments && sg.count < 8 * k) {  // block-uniform
            // the threads' maxima of some lanes' each, in their order
            constexpr int kMine = kFewSegments * kWave / THREADS;
            float v[kMine];
            const int all = sg.count * kWave;
            float most = -INFINITY;
#pragma unroll
            for (int u = 0; u < kMine; ++u) {
                const int e = u * THREADS + threadIdx.x;
                v[u] = e < all ? maxima[e] : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < kMine; ++u) most = fmaxf(most, v[u]);
            keys[threadIdx.x] = most > -INFINITY ? float_order_key(most) : 0;
            __syncthreads();
            if (wid == 0) {
                uint32_t w[kWaves];
#pragma unroll
                for (int i = 0; i < kWaves; ++i) w[i] = static_cast<uint32_t>(keys[i * kWave + lane]);
                const uint32_t l = reached_by(w, k);
                if (lane == 0) limit = l;
            }
            __syncthreads();
            value = static_cast<uint32_t>(limit);
            const float low = value ? float_from_order_key(value) : -INFINITY;
#pragma unroll
            for (int u = 0; u < kMine; ++u)
                if (v[u] > -INFINITY && v[u] >= low) add_lane(u * THREADS + threadIdx.x);
        } else {  // many more segments than alternatives: their maxima, then the lanes of those that reach
#pragma unroll
            for (int i = 0; i < kPer; ++i) keys[i * THREADS + threadIdx.x] = key[i];
            __syncthreads();
            if (wid == 0) {
                auto reached = [&](auto tag) {
                    constexpr int R = decltype(tag)::value;
                    uint32_t w[R];
#pragma unroll
                    for (int i = 0; i < R; ++i) w[i] = static_cast<uint32_t>(keys[i * kWave + lane] >> 32);
                    return reached_by(w, k);
                };
                const uint32_t l = sg.count <= kFewSegments ? reached(std::integral_constant<int, kFewSegments / kWave>{})
                                                            : reached(std::integral_constant<int, kMostSegments / kWave>{});
                if (lane == 0) limit = l;
            }
            __syncthreads();
            value = static_cast<uint32_t>(limit);
            const float low = value ? float_from_order_key(value) : -INFINITY;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (key[i] != 0 && part[i].m >= low) list[atomicAdd(&counts[0], 1)] = i * THREADS + threadIdx.x;
            __syncthreads();
            const int all = counts[0] * kWave;
            for (int e0 = threadIdx.x; e0 < all; e0 += 4 * THREADS) {
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = e0 + u * THREADS;
                    v[u] = e < all ? maxima[list[e / kWave] * kWave + e % kWave] : -INFINITY;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = e0 + u * THREADS;
                    if (v[u] > -INFINITY && v[u] >= low) add_lane(list[e / kWave] * kWave + e % kWave);
                }
            }
        }
        __syncthreads();
        // a logit of a lane
        auto index_of = [&](int ln, int e) { return (((ln >> 6) << sg.shift) + e / E) * kPass + element<F16, VEC>(ln & 63, e % E); };
        const int n_lanes = counts[1], each = E << sg.shift;
        auto hold = [&](uint64_t v) {
            const int at = atomicAdd(&counts[2], 1);
            if (at < kCandidates) cand[at] = v;
        };
        auto key_at = [&](int i) {
            const float x = i < p.vocab ? clean(static_cast<float>(x0[i])) : -INFINITY;
            return x > -INFINITY ? argmax_key(x, i) : uint64_t(0);
        };
        bool many = n_lanes > kMostLanes;  // block-uniform
        if (!many) {
            const uint64_t least = u64_max(static_cast<uint64_t>(value) << 32, 1);
            for (int e = threadIdx.x; e < n_lanes * each; e += THREADS) {
                const uint64_t v = key_at(index_of(lanes[e / each], e % each));
                if (v >= least) hold(v);
            }
            __syncthreads();
            many = counts[2] > kMany;
            __syncthreads();
        }
        if (many) {  // ties, or many large logits in a few lanes: the whole row once more, with the k-th of the threads' shares
            uint64_t mine = 0;
#pragma unroll 8
            for (int i = threadIdx.x; i < p.vocab; i += THREADS) mine = u64_max(mine, key_at(i));
            keys[threadIdx.x] = mine;
            if (threadIdx.x == 0) counts[2] = 0;
            __syncthreads();
            if (wid == 0) {
                uint64_t v[kWaves];
#pragma unroll
                for (int i = 0; i < kWaves; ++i) v[i] = keys[i * kWave + lane];
                const uint64_t l = kth_largest(v, k);
                if (lane == 0) limit = u64_max(l, 1);
            }
            __syncthreads();
            const uint64_t least = limit;
            if (mine >= least)
#pragma unroll 8
                for (int i = threadIdx.x; i < p.vocab; i += THREADS) {
                    const uint64_t v = key_at(i);
                    if (v >= least) hold(v);
                }
            __syncthreads();
            if (counts[2] > kCandidates) {  // (a few threads' shares hold them all)
                uint64_t last = ~uint64_t(0);
                for (int i = 0; i < k; ++i) {
                    uint64_t next = 0;
#pragma unroll 8
                    for (int j = threadIdx.x; j < p.vocab; j += THREADS) {
                        const uint64_t v = key_at(j);
                        next = v < last ? u64_max(next, v) : next;
                    }
                    next = wave_max_u64(next);
                    __syncthreads();
                    if (lane == 0) red[wid] = next;
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < kWaves; ++j) next = u64_max(next, red[j]);
                    last = next;
                    if (threadIdx.x == 0) cand[i] = last;
                }
                __syncthreads();
                if (threadIdx.x == 0) counts[2] = k;  // (as many are left: over kCandidates reach the threshold)
                __syncthreads();
            }
        }
        put_in_order(p, row, cand, counts[2], m, lz, THREADS);
    }
}

// A row of few logits, in a block's registers: one launch and no workspace.  VEC: the threads' pieces, and the logits behind
// the last whole piece, one for each of the first threads.
template <bool F16, bool VEC, bool TOP, int THREADS, int E>
__global__ void __launch_bounds__(THREADS) logprobs_small_kernel(LogprobsLaunch p) {
    typedef logit_t<F16> L;
    constexpr int N = VEC ? 16 / sizeof(L) : 1, kWaves = THREADS / kWave;
    typedef L piece __attribute__((ext_vector_type(N)));
    __shared__ float maxima[kWaves];
    __shared__ float4 sums[kWaves];
    __shared__ uint64_t cand[(XQHIP_TOP_MAX + XQHIP_TOP_MAX / 4 + 4) * (E + 1)];  // as many threads, at most, hold any
    __shared__ uint64_t best[THREADS];
    __shared__ uint32_t keys[THREADS];
    __shared__ int count;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave, vocab = p.vocab;
    const L* x0 = logit_row<F16>(p, row);
    const int t = p.tokens ? p.tokens[row] : -1;
    const bool has = t >= 0 && t < vocab;
    const int whole = vocab / N, rest = VEC ? vocab - whole * N : 0;
    auto index = [&](int e) {  // past the row's end: no token's
        const int at = e / N * THREADS + tid;
        return e < E ? (!VEC || at < whole ? at * N : vocab) + e % N : whole * N + tid;
    };
    float x[E + 1];
#pragma unroll
    for (int u = 0; u < E / N; ++u) {  // (no branches: the loads go out together)
        const int at = u * THREADS + tid;
        const piece v = *reinterpret_cast<const piece*>(x0 + min(at, whole - 1) * N);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float y;
            if constexpr (VEC)
                y = static_cast<float>(v[e]);
            else
                y = static_cast<float>(v[0]);
            x[u * N + e] = at < whole ? y : -INFINITY;
        }
    }
    x[E] = static_cast<float>(x0[min(whole * N + tid, vocab - 1)]);
    if (tid >= rest) x[E] = -INFINITY;
    const float xt = clean(static_cast<float>(x0[has ? t : 0])), c = p.inv_t * kTwoLog2e;
    float lm = x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) lm = fmaxf(lm, x[e]);
    lm = clean(lm);
    const float wm = wave_max(lm);
    if (lane == 0) maxima[wid] = wm;
    if (TOP) keys[tid] = lm > -INFINITY ? float_order_key(lm) : 0;
    if (tid == 0) count = 0;
    __syncthreads();
    float m = maxima[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) m = fmaxf(m, maxima[i]);
    const bool any = m > -INFINITY;
    float s = 0.0f, h = 0.0f;
    int same = 0, before = 0;
#pragma unroll
    for (int e = 0; e <= E; ++e) {
        const bool top = x[e] == m;
        const float d = gap2(x[e], m, c), w = top ? 0.0f : __builtin_amdgcn_exp2f(d), y = clean(x[e]);
        same += __popcll(__builtin_amdgcn_ballot_w64(top));
        s += w;
        h = fmaf(w, d, h);
        before += __popcll(__builtin_amdgcn_ballot_w64(y > xt || (y == xt && index(e) < t)));
    }
    s = wave_sum(s);
    h = wave_sum(h);
    if (lane == 0) sums[wid] = make_float4(s, h, static_cast<float>(before), static_cast<float>(same));
    uint64_t least = 1;
    if constexpr (TOP) {  // a value that `top` threads' maxima reach, found by every wave for itself
        uint32_t w[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) w[i] = keys[i * kWave + lane];
        least = static_cast<uint64_t>(reached_by(w, p.top)) << 32;
        if (least == 0) {  // block-uniform: fewer threads have any, or ties
            uint64_t mine = 0;
#pragma unroll
            for (int e = 0; e <= E; ++e) mine = clean(x[e]) > -INFINITY ? u64_max(mine, argmax_key(clean(x[e]), index(e))) : mine;
            best[tid] = mine;
            __syncthreads();
            uint64_t v[kWaves];
#pragma unroll
            for (int i = 0; i < kWaves; ++i) v[i] = best[i * kWave + lane];
            least = u64_max(kth_largest(v, p.top), 1);
        }
#pragma unroll
        for (int e = 0; e <= E; ++e) {
            const float y = clean(x[e]);
            if (y > -INFINITY && float_order_key(y) >= static_cast<uint32_t>(least >> 32)) {
                const uint64_t v = argmax_key(y, index(e));
                if (v >= least) cand[atomicAdd(&count, 1)] = v;
            }
        }
    }
    __syncthreads();
    float4 a = sums[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
        a.x += sums[i].x;
        a.y += sums[i].y;
        a.z += sums[i].z;
        a.w += sums[i].w;
    }
    const float rs = a.x + (a.w - 1.0f), lz = log1pf(rs);
    if (tid == 0) {
        if (p.out_rank) p.out_rank[row] = has ? static_cast<int32_t>(a.z) : -1;
        if (p.out_logprob) p.out_logprob[row] = any && has ? logit_gap(xt, m, p.inv_t) - lz : -INFINITY;
        if (p.out_entropy) p.out_entropy[row] = any ? lz - kLn2 * a.y / (1.0f + rs) : 0.0f;
    }
    if constexpr (TOP) put_in_order(p, row, cand, count, m, lz, THREADS);
}

template <bool F16, bool VEC, int THREADS, int E>
static void launch_small(const LogprobsLaunch& p, hipStream_t s) {
    if (p.top)
        hipLaunchKernelGGL((logprobs_small_kernel<F16, VEC, true, THREADS, E>), dim3(p.rows), dim3(THREADS), 0, s, p);
    else
        hipLaunchKernelGGL((logprobs_small_kernel<F16, VEC, false, THREADS, E>), dim3(p.rows), dim3(THREADS), 0, s, p);
}

template <bool F16, bool VEC>
static void launch_rows(const LogprobsLaunch& p, hipStream_t s) {
    if (p.vocab <= 16 * kWave) return launch_small<F16, VEC, kWave, 16>(p, s);
    if (p.vocab <= 16 * kRowThreads) return launch_small<F16, VEC, kRowThreads, 16>(p, s);
    if (p.vocab <= 32 * kRowThreads) return launch_small<F16, VEC, kRowThreads, 32>(p, s);
    const Segments sg = segments_of(p.vocab, F16);
    hipLaunchKernelGGL((logprobs_part_kernel<F16, VEC>), dim3((sg.count + kPartWaves - 1) / kPartWaves, p.rows), dim3(kWave * kPartWaves), 0, s, p, sg);
    if (hipPeekAtLastError() != hipSuccess) return;
    if (p.top)
        hipLaunchKernelGGL((logprobs_row_kernel<F16, VEC, true, kRowThreads>), dim3(p.rows), dim3(kRowThreads), 0, s, p, sg);
    else
        hipLaunchKernelGGL((logprobs_row_kernel<F16, VEC, false, kFewThreads>), dim3(p.rows), dim3(kFewThreads), 0, s, p, sg);
}

hipError_t launch_logprobs(const LogprobsLaunch& p, hipStream_t s) {
    const int piece = p.f16 ? 8 : 4;
    const bool vec = (reinterpret_cast<uintptr_t>(p.logits) & 15u) == 0 && p.ld % piece == 0 && p.vocab >= piece;
    if (p.f16)
        vec ? launch_rows<true, true>(p, s) : launch_rows<true, false>(p, s);
    else
        vec ? launch_rows<false, true>(p, s) : launch_rows<false, false>(p, s);
    return hipGetLastError();
}

}  // namespace xqhip
