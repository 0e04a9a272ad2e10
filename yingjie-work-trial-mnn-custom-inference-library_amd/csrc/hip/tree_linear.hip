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
// decay is 0 either way, and differences stay finite.)
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
        L[tid] = fmaxf(-expf(p.a_log[vh]) * softplus_dev(a + p.dt_bias[vh]), -1000.0f);
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

bool tree_linear_supported(int lk_n, int lk_hd, int lv_n, int lv_hd, int ksize) {
    return lk_n > 0 && lv_n > 0 && lk_n <= 4096 && lv_n <= 4096 && lv_n % lk_n == 0 && lk_hd > 0 && lv_hd > 0 &&
           lk_hd <= kTreeLinMaxDim && lv_hd <= kTreeLinMaxDim && ksize > 0 && ksize <= kTreeLinMaxTaps;
}

size_t tree_linear_workspace_bytes(int nodes, int lk_n, int lk_hd, int lv_n, int lv_hd) {
    return static_cast<size_t>(nodes) * (2 * lk_n * lk_hd + lv_n * lv_hd) * sizeof(float);
}

hipError_t launch_tree_linear(const TreeLinearLaunch& p, hipStream_t s) {
    hipLaunchKernelGGL(tree_conv_kernel, dim3(2 * p.lk_n + p.lv_n, p.nodes), dim3(kWave), 0, s, p);
    hipLaunchKernelGGL(tree_delta_kernel, dim3(p.lv_n, (p.lv_hd + kTreeLinCols - 1) / kTreeLinCols), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
