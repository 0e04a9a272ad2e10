// attn_mfma.hpp - what the matrix-core attention kernels share: operands in two
// fp16 parts, q's columns in LDS, outputs.
#pragma once

#include "xqhip_common.hpp"

namespace xqhip {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));
constexpr int kTTile = 32;  // keys and columns of an MFMA tile

__device__ __forceinline__ float pair32_max(float v) {  // of v[l] and v[l ^ 32]
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
                 __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}

__device__ __forceinline__ float xor16_max(float v) {  // of v[l] and v[l ^ 16]
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
                 __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
// even rows of 16 lanes: a[l] + a[l ^ 16]; odd rows: b[l] + b[l ^ 16]
__device__ __forceinline__ float rows_sum(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
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

// exponent of a V scale, for the reference of its key's weights
__device__ __forceinline__ float scale_exponent(float s) {
    return fabsf(s) > 0.0f ? fminf(fmaxf(static_cast<float>(__builtin_amdgcn_frexp_expf(s)), -90.0f), 100.0f) : -90.0f;
}

// The block's columns of q as fp16 hi + lo in LDS, each scaled by a power of two into [2^12, 2^13), and the factor of
// each column's scores in the exponent of 2.
template <typename F, int HD>
struct QueryStage {
    static constexpr int kLanes = HD / 8, kStep = F::kThreads / kLanes;  // eight dims a thread
    static constexpr int kPasses = (F::kCols + kStep - 1) / kStep;
    static constexpr int kLd = HD + 8;  // halves per column: 16-byte rows shifted by 4 banks
    static constexpr size_t kBytes = static_cast<size_t>(F::kCols) * (2 * kLd * 2 + 4);
    u32x4 r[kPasses][2];

    // rows: the first of `ntok` rows
    __device__ __forceinline__ void load(const float* rows, int q_stride, int kh, int ntok, int group, int T, uint32_t inv_t) {
        const __amdgpu_buffer_rsrc_t rq = buf_rsrc(rows, static_cast<uint32_t>(ntok) * q_stride * 4u);
#pragma unroll
        for (int u = 0; u < kPasses; ++u) {  // columns without a row read 0
            const int c = threadIdx.x / kLanes + u * kStep, hc = static_cast<int>(c * inv_t >> 16), tc = c - hc * T;
            const uint32_t at = tc * q_stride + (kh * group + hc) * HD + 8 * (threadIdx.x % kLanes);
            const bool on = c < F::kCols && hc < group && tc < ntok;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                r[u][i] = __builtin_amdgcn_raw_buffer_load_b128(rq, on ? at * 4u + 16u * i : kBufOOB, 0, 0);
        }
    }
    __device__ __forceinline__ void store(void* lds) const {
        constexpr float kLog2e = 1.44269504088896340736f;
        _Float16* Q = static_cast<_Float16*>(lds);  // [2][kCols][kLd]
        float* S = reinterpret_cast<float*>(Q + 2 * F::kCols * kLd);
#pragma unroll
        for (int u = 0; u < kPasses; ++u) {
            const int c = threadIdx.x / kLanes + u * kStep;
            if (c >= F::kCols) break;  // wave-uniform
            float x[8], mx = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __uint_as_float(r[u][e / 4][e % 4]);
                mx = fmaxf(mx, fabsf(x[e]));
            }
            mx = lanes_max<16>(mx);
            if constexpr (kLanes == 32) mx = xor16_max(mx);
            int ex = 13;  // an infinity or 0 stays
            if (mx > 0.0f && mx < INFINITY) frexpf(mx, &ex);
            ex = max(ex, -100);  // 2^(13 - ex) stays finite
            const float down = ldexpf(1.0f, 13 - ex);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= down;
            half8 hi, lo;
            split8(x, hi, lo);
            _Float16* at = Q + c * kLd + 8 * (threadIdx.x % kLanes);
            *reinterpret_cast<half8*>(at) = hi;
            *reinterpret_cast<half8*>(at + F::kCols * kLd) = lo;
            if (threadIdx.x % kLanes == 0) S[c] = ldexpf(kLog2e / sqrtf(static_cast<float>(HD)), ex - 13);
        }
    }
    // dims d .. d + 7 of column c
    static __device__ __forceinline__ half8 part(const void* lds, int low, int c, int d) {
        return *reinterpret_cast<const half8*>(static_cast<const _Float16*>(lds) + (low * F::kCols + c) * kLd + d);
    }
    static __device__ __forceinline__ float scale(const void* lds, int c) {
        return reinterpret_cast<const float*>(static_cast<const _Float16*>(lds) + 2 * F::kCols * kLd)[c];
    }
};

__device__ __forceinline__ void add_scaled(float4& r, float f, float4 v) {
    r.x += f * v.x;
    r.y += f * v.y;
    r.z += f * v.z;
    r.w += f * v.w;
}

__device__ __forceinline__ float4 as_float4(u32x4 v) {
    return make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
}
// writes the quad at `out`; whether its row has to be computed again
__device__ __forceinline__ bool write_quad(float4 r, float L, bool gated, float4 gt, float* out) {
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    float4 y = make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
    if (gated) {
        y.x *= sigmoid_dev(gt.x);
        y.y *= sigmoid_dev(gt.y);
        y.z *= sigmoid_dev(gt.z);
        y.w *= sigmoid_dev(gt.w);
    }
    *reinterpret_cast<float4*>(out) = y;
    return !(L > 0.0f && fabsf(r.x) + fabsf(r.y) + fabsf(r.z) + fabsf(r.w) < INFINITY);
}

constexpr float kRaise = 6.0f;  // weights are held times 2^kRaise
constexpr float kSlack = 6.0f;  // the max may outgrow the reference by 2^kSlack before it is moved

}  // namespace xqhip
