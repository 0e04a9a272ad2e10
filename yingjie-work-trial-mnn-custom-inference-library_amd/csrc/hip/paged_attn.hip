// paged_attn.hip - attention of a step's rows over their sequences' pages.
#include <algorithm>

#include "paged_common.hpp"

namespace xqhip {

constexpr int kPagedMaxGroup = 16;
constexpr int kRowChunk = 32;  // keys: a page holds whole chunks

constexpr size_t paged_row_lds(int group, int hd) {
    return (2 * static_cast<size_t>(group) * hd + static_cast<size_t>(group) * (kRowChunk + 3)) * sizeof(float);
}

// ---------------------------------------------------------------------------
// One row and the `group` query heads of kv head kh, any head size: the
// positions in chunks of 32 with a running max and sum (rescaled by exp(m_old -
// m_new)).  What the row does not see is passed over, so nothing in it can reach
// the row; a chunk without a score above minus infinity leaves the sums.
// ---------------------------------------------------------------------------
template <int THREADS>
__device__ void attend_paged_row(const PagedAttnLaunch& p, int s, const SeqRows& sr, int row, int kh, float* smem) {
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
    for (int i = threadIdx.x; i < group * hd; i += THREADS) {
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

size_t paged_attn_workspace_bytes(int nq, int nkv, int head_dim) {
    if (nkv <= 0 || nq <= 0 || nq % nkv || nq / nkv > kPagedMaxGroup || head_dim <= 0 || head_dim > 256 || head_dim % 16) return 0;
    return 16;
}

hipError_t launch_paged_attn(const PagedAttnLaunch& p, hipStream_t s) {
    hipLaunchKernelGGL(paged_attn_row_kernel, dim3(p.step.rows, p.kv.nkv), dim3(256), paged_row_lds(p.nq / p.kv.nkv, p.kv.head_dim), s, p);
    return hipGetLastError();
}

}  // namespace xqhip
