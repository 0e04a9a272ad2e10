// token_logprobs.hip - log probabilities of given tokens, entropy, rank and the
// first alternatives of rows of logits.
#include "xqhip_common.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

// ---------------------------------------------------------------------------
// With m the largest logit, d_i = (x_i - m) / T and s' the sum of exp(d_i)
// without one term of the maximum: log p_t = d_t - log1p(s'), entropy =
// log1p(s') - sum exp(d_i) d_i / (1 + s').  Without the 1 in the sum a
// probability near 1 keeps its digits.  Equal infinities differ by 0.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float logit_at(const void* row, bool f16, int i) {
    const float x = f16 ? static_cast<float>(static_cast<const _Float16*>(row)[i]) : static_cast<const float*>(row)[i];
    return x == x ? x : -INFINITY;
}
__device__ __forceinline__ float logit_gap(float x, float m, float inv_t) { return x == m ? 0.0f : (x - m) * inv_t; }

constexpr int kLogThreads = 1024;
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* red) {
    v = wave_max_u64(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < kLogThreads / kWave; ++i) v = u64_max(v, red[i]);
    return v;
}

__global__ void __launch_bounds__(kLogThreads) logprobs_row_kernel(LogprobsLaunch p) {
    __shared__ uint64_t red[kLogThreads / kWave];
    __shared__ float fred[16];
    const int row = blockIdx.x;
    const bool f16 = p.f16;
    const void* x = f16 ? static_cast<const void*>(static_cast<const _Float16*>(p.logits) + row * p.ld)
                        : static_cast<const void*>(static_cast<const float*>(p.logits) + row * p.ld);
    uint64_t best = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kLogThreads) best = u64_max(best, argmax_key(logit_at(x, f16, i), i));
    best = block_max_u64(best, red);
    const float m = float_from_order_key(static_cast<uint32_t>(best >> 32));
    const int arg = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
    const bool any = m > -INFINITY;
    const int t = p.tokens ? p.tokens[row] : -1;
    const bool has = t >= 0 && t < p.vocab;
    const float xt = has ? logit_at(x, f16, t) : 0.0f;
    float sum = 0.0f, mean = 0.0f;
    int before = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kLogThreads) {
        const float v = logit_at(x, f16, i), d = logit_gap(v, m, p.inv_t);
        before += has && (v > xt || (v == xt && i < t));
        if (i == arg || !any || v == -INFINITY) continue;
        const float e = expf(d);
        sum += e;
        if (e > 0.0f) mean += e * d;
    }
    sum = block_sum_t<kLogThreads / kWave>(sum, fred);
    mean = block_sum_t<kLogThreads / kWave>(mean, fred);
    const float rank = block_sum_t<kLogThreads / kWave>(static_cast<float>(before), fred);  // vocab <= 2^24: exact
    const float lz = log1pf(sum);
    if (threadIdx.x == 0) {
        if (p.out_logprob) p.out_logprob[row] = any && has ? logit_gap(xt, m, p.inv_t) - lz : -INFINITY;
        if (p.out_entropy) p.out_entropy[row] = any ? lz - mean / (1.0f + sum) : 0.0f;
        if (p.out_rank) p.out_rank[row] = has ? static_cast<int32_t>(rank) : -1;
    }
    for (int k = 0; k < p.top; ++k) {
        const float v = float_from_order_key(static_cast<uint32_t>(best >> 32));
        const bool none = best == 0 || v == -INFINITY;
        if (threadIdx.x == 0) {
            const size_t o = static_cast<size_t>(row) * p.top + k;
            if (p.out_top) p.out_top[o] = none ? -1 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
            if (p.out_top_logprob) p.out_top_logprob[o] = none ? -INFINITY : logit_gap(v, m, p.inv_t) - lz;
        }
        if (none) {
            best = 0;
            continue;
        }
        uint64_t next = 0;
        for (int i = threadIdx.x; i < p.vocab; i += kLogThreads) {
            const uint64_t key = argmax_key(logit_at(x, f16, i), i);
            if (key < best) next = u64_max(next, key);
        }
        best = block_max_u64(next, red);
    }
}

size_t logprobs_workspace_bytes(int, int, int) { return 16; }

hipError_t launch_logprobs(const LogprobsLaunch& p, hipStream_t s) {
    hipLaunchKernelGGL(logprobs_row_kernel, dim3(p.rows), dim3(kLogThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
