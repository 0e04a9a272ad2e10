// tree_attn.hip - attention of a decode step's rows (a tree of drafted tokens,
// or a prompt chunk) over an fp16 or 8-bit key/value cache.
#include <algorithm>

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

bool tree_attn_supported(int nq, int nkv, int head_dim) {
    return nkv > 0 && nq > 0 && nq % nkv == 0 && nq / nkv <= kTreeMaxGroup && head_dim > 0 && head_dim <= 1024 &&
           sizeof(float) * tree_row_lds(nq / nkv, head_dim) <= 64 * 1024;
}

size_t tree_attn_workspace_bytes(int nq, int nkv, int head_dim, int tokens) {
    (void)nq; (void)nkv; (void)head_dim; (void)tokens;
    return 16;
}

hipError_t launch_tree_attn(const TreeAttnLaunch& p, hipStream_t s) {
    const size_t lds = sizeof(float) * tree_row_lds(p.nq / p.kv.nkv, p.kv.head_dim);
    const dim3 grid(p.tokens, p.kv.nkv);
    if (p.kv.i8)
        hipLaunchKernelGGL((tree_attn_row_kernel<true>), grid, dim3(256), lds, s, p);
    else
        hipLaunchKernelGGL((tree_attn_row_kernel<false>), grid, dim3(256), lds, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
