// paged_cache.hip - the paged key/value cache of a step over several sequences:
// head preparation with the append, and read-back.
#include <algorithm>

#include "paged_common.hpp"

namespace xqhip {

// ---------------------------------------------------------------------------
// Head preparation (custom_model.cpp:301-370, 673-753): y = x / sqrt(mean x^2 +
// eps) * w, then pair i (dims i and i + pairs) turned by the angles of its
// axis' position.  In 64 bits: a key that is held in 8 bits has to fall on the
// right side of a code's border, and an fp32 rounding on the way moves one code
// of 10^5 by a whole step.
//
// A head's values lie in a wave's lanes: lane l has the dims E l .. E l + E - 1
// (VEC, one load) or l, l + 64, .. (other sizes).
// ---------------------------------------------------------------------------
constexpr int kPagedWaves = 4;
constexpr int kPagedMaxDim = 256;

__device__ __forceinline__ double wave_sum_double(double v) {
    v += __builtin_bit_cast(double, dpp_u64<kDppXor1>(__builtin_bit_cast(uint64_t, v)));
    v += __builtin_bit_cast(double, dpp_u64<kDppXor2>(__builtin_bit_cast(uint64_t, v)));
    v += __builtin_bit_cast(double, dpp_u64<kDppHalfMirror>(__builtin_bit_cast(uint64_t, v)));
    v += __builtin_bit_cast(double, dpp_u64<kDppMirror>(__builtin_bit_cast(uint64_t, v)));
    double r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(u)), 16 * i);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(u >> 32)), 16 * i);
        r[i] = __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
    }
    return (r[0] + r[1]) + (r[2] + r[3]);
}

// LDS written by a wave, then read by it: the accesses of a wave reach LDS in their order
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int E, bool VEC>
struct HeadLanes {
    static __device__ __forceinline__ int dim(int lane, int e) { return VEC ? lane * E + e : lane + kWave * e; }
    static __device__ __forceinline__ bool in(int lane, int e, int hd) { return VEC || dim(lane, e) < hd; }
    static __device__ __forceinline__ void load(const float* s, int lane, int hd, float (&x)[E]) {
        if constexpr (VEC) {
            typedef float fv __attribute__((ext_vector_type(E)));
            const fv v = *reinterpret_cast<const fv*>(s + lane * E);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = in(lane, e, hd) ? s[dim(lane, e)] : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(float* d, int lane, int hd, const float (&x)[E]) {
        if constexpr (VEC) {
            typedef float fv __attribute__((ext_vector_type(E)));
            fv v;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = x[e];
            *reinterpret_cast<fv*>(d + lane * E) = v;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (in(lane, e, hd)) d[dim(lane, e)] = x[e];
        }
    }
};

// The angles of a row: whether all of its positions lie in the table.
template <int E, bool VEC>
__device__ __forceinline__ bool row_angles(const PagedPrepLaunch& p, int row, int pos, int lane, float2 (&cs)[E]) {
    typedef HeadLanes<E, VEC> L;
    const int half = p.rot.pairs;
    bool good = true;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = L::dim(lane, e);
        cs[e] = make_float2(1.0f, 0.0f);
        if (d >= 2 * half) continue;
        const int i = d < half ? d : d - half, a = p.rot.axis[i / 16] >> 2 * (i % 16) & 3;
        const int at = p.rot.pos ? p.rot.pos[static_cast<size_t>(a) * p.step.rows + row] : pos;
        if (at >= 0 && at < p.rot.positions)
            cs[e] = p.rot.cs[static_cast<size_t>(at) * half + i];
        else
            good = false;
    }
    return __builtin_amdgcn_ballot_w64(!good) == 0;
}

// x normalised and turned, by a whole wave; turn: the wave's kPagedMaxDim doubles of LDS
template <int E, bool VEC>
__device__ __forceinline__ void turn_head(const float (&x)[E], const float (&w)[E], const float2 (&cs)[E], int hd, int half, float eps,
                                          int lane, double* turn, float (&y)[E]) {
    typedef HeadLanes<E, VEC> L;
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) ss += static_cast<double>(x[e]) * x[e];
    const double inv = 1.0 / sqrt(wave_sum_double(ss) / hd + static_cast<double>(eps));
    double v[E];
    wave_lds_sync();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = static_cast<double>(x[e]) * inv * w[e];
        if (L::in(lane, e, hd)) turn[L::dim(lane, e)] = v[e];
    }
    wave_lds_sync();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = L::dim(lane, e);
        if (d < half)
            v[e] = v[e] * cs[e].x - turn[half + d] * cs[e].y;
        else if (d < 2 * half)
            v[e] = v[e] * cs[e].x + turn[d - half] * cs[e].y;
        y[e] = static_cast<float>(v[e]);
    }
}

// Whether a row's key and value have a place: sequence s, position pos.
__device__ __forceinline__ int place_of(const PagedPrepLaunch& p, int s, int64_t pos) {
    if (pos < 0 || pos >= table_positions(p.step, p.kv)) return -1;
    if (p.kv.i8) {
        const int o = p.step.open[s];
        if (o < 0 || o >= p.kv.opens) return -1;
    }
    return page_at(p.step, p.kv, s, static_cast<int>(pos) / p.kv.page);
}

// One head of one row per wave: q, gate, and k and v of fp16 pages.
template <int E, bool VEC>
__device__ void prep_unit(const PagedPrepLaunch& p, int unit, int row, double* turn) {
    typedef HeadLanes<E, VEC> L;
    const int lane = threadIdx.x & (kWave - 1), hd = p.kv.head_dim, nkv = p.kv.nkv;
    const bool is_q = unit < p.nq, is_k = !is_q && unit < p.nq + nkv;
    const int h = is_q ? unit : (is_k ? unit - p.nq : unit - p.nq - nkv);
    const size_t off = static_cast<size_t>(row) * p.src_stride;
    const float* src = is_q ? p.q_src + off + static_cast<size_t>(h) * (p.gated ? 2 * hd : hd)
                            : (is_k ? p.k_src : p.v_src) + off + static_cast<size_t>(h) * hd;
    const int s = __builtin_amdgcn_readfirstlane(seq_of_row(p.step, row));
    if (s >= p.step.seqs) return;
    const SeqRows sr = seq_rows(p.step, s);
    const int j = row - sr.row0;
    if (j < 0 || j >= sr.rows) return;
    float x[E], w[E], gate[E] = {};
    L::load(src, lane, hd, x);
    if (is_q && p.gated) L::load(src + hd, lane, hd, gate);
    if (is_q || is_k) L::load(is_q ? p.q_norm : p.k_norm, lane, hd, w);
    const int64_t pos = sr.past < 0 ? -1 : static_cast<int64_t>(sr.past) + j;
    const int page = place_of(p, s, pos);
    float2 cs[E];
    const bool held = row_angles<E, VEC>(p, row, static_cast<int>(pos), lane, cs) && page >= 0;
    if (is_q || is_k) {
        float y[E];
        turn_head<E, VEC>(x, w, cs, hd, p.rot.pairs, p.eps, lane, turn, y);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = y[e];
    }
    if (is_q) {
        const size_t o = static_cast<size_t>(row) * p.out_stride + static_cast<size_t>(h) * hd;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = held ? x[e] : __builtin_nanf("");
        L::store(p.q_out + o, lane, hd, x);
        if (p.gate_out) L::store(p.gate_out + o, lane, hd, gate);
        return;
    }
    if (!held) return;
    const int at = static_cast<int>(pos) % p.kv.page;
    _Float16* d = static_cast<_Float16*>(is_k ? p.kv.k : p.kv.v) + page_head(p.kv, page, h);
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (L::in(lane, e, hd)) {
            const int dim = L::dim(lane, e);
            d[is_k ? k_offset<8>(p.kv, at, dim) : v_offset<8>(p.kv, at, dim)] = static_cast<_Float16>(x[e]);
        }
}

// The fp16 value that 8 bits are taken of: no infinities, no NaN.
__device__ __forceinline__ _Float16 held_value(float x) {
    return static_cast<_Float16>(x == x ? fminf(fmaxf(x, -65504.0f), 65504.0f) : 0.0f);
}
// 127 x / mx to the nearest: 127 x is exact (18 bits), and the division correctly rounded: its quotient is half a code's
// step exactly where the true one is
__device__ __forceinline__ int8_t code_of(_Float16 x, float mx) {
    const float c = mx > 0.0f ? rintf(__fdiv_rn(127.0f * static_cast<float>(x), mx)) : 0.0f;
    return static_cast<int8_t>(fminf(fmaxf(c, -127.0f), 127.0f));  // (a row that was never written may pass the maximum)
}

// One 8-bit page that the step touches, one kv head, k or v, by a block: the new rows' fp16 values into LDS and their
// maximum taken, then codes of them, or of the whole page where the maximum rose.
template <int E, bool VEC>
__device__ void hold_page(const PagedPrepLaunch& p, const SeqRows& sr, int s, int index, int h, bool is_k, _Float16* vals, double* turn) {
    typedef HeadLanes<E, VEC> L;
    __shared__ float wave_mx[kPagedWaves];
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, hd = p.kv.head_dim, nkv = p.kv.nkv, P = p.kv.page;
    const int page = place_of(p, s, static_cast<int64_t>(index) * P);
    if (page < 0) return;  // block-uniform
    const int open = p.step.open[s];
    const int base = index * P;                                                       // position of the page's first
    const int lead = max(0, sr.past - base), end = min(P, sr.past + sr.rows - base);  // new ones: [lead, end)
    const bool last = base + P >= sr.past + sr.rows;
    const size_t head = page_head(p.kv, page, h);
    _Float16* kept = (is_k ? p.kv.k_open : p.kv.v_open) + (static_cast<size_t>(open) * nkv + h) * P * hd;
    float* scale = (is_k ? p.kv.k_scale : p.kv.v_scale) + static_cast<size_t>(page) * nkv + h;
    float w[E], mx = 0.0f;
    if (is_k) L::load(p.k_norm, lane, hd, w);
    for (int t = lead + wid; t < end; t += kPagedWaves) {
        const int row = sr.row0 + base + t - sr.past;
        float x[E];
        float2 cs[E];
        L::load((is_k ? p.k_src : p.v_src) + static_cast<size_t>(row) * p.src_stride + static_cast<size_t>(h) * hd, lane, hd, x);
        const bool held = row_angles<E, VEC>(p, row, base + t, lane, cs);
        if (is_k) {
            float y[E];
            turn_head<E, VEC>(x, w, cs, hd, p.rot.pairs, p.eps, lane, turn, y);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = y[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!L::in(lane, e, hd)) continue;
            const int d = L::dim(lane, e);
            // (a row that is not held leaves what is there: NaN marks it)
            const _Float16 v = held ? held_value(x[e]) : static_cast<_Float16>(__builtin_nanf(""));
            vals[t * hd + d] = v;
            if (held) {
                mx = fmaxf(mx, fabsf(static_cast<float>(v)));
                if (last) kept[static_cast<size_t>(t) * hd + d] = v;
            }
        }
    }
    mx = wave_max(mx);
    if (lane == 0) wave_mx[wid] = mx;
    const float was = lead ? *scale : 0.0f;
    __syncthreads();
    mx = fmaxf(fmaxf(wave_mx[0], wave_mx[1]), fmaxf(wave_mx[2], wave_mx[3]));
    const float before = static_cast<float>(static_cast<_Float16>(was * 127.0f));  // the maximum, an fp16 value, exactly
    const bool grew = mx > before;
    mx = grew ? mx : before;
    int from = lead;
    if (grew && lead) {
        from = 0;
        for (int i = threadIdx.x; i < lead * hd; i += kWave * kPagedWaves) vals[i] = kept[i];
        __syncthreads();
    }
    if (threadIdx.x == 0) *scale = mx / 127.0f;
    int8_t* d = static_cast<int8_t*>(is_k ? p.kv.k : p.kv.v) + head;
    for (int i = from * hd + threadIdx.x; i < end * hd; i += kWave * kPagedWaves) {
        const int t = i / hd, dim = i - t * hd;
        const _Float16 v = vals[i];
        if (t >= lead && v != v) continue;
        d[is_k ? k_offset<16>(p.kv, t, dim) : v_offset<16>(p.kv, t, dim)] = code_of(v, mx);
    }
}

// The 8-bit pages of a sequence, a block per page, kv head and k or v.  The first page and the last are one block's: the
// first's earlier values lie where the last's are kept.
template <int E, bool VEC>
__device__ void hold_unit(const PagedPrepLaunch& p, int unit, _Float16* vals, double* turn) {
    const bool is_k = (unit & 1) == 0;
    unit >>= 1;
    const int h = unit % p.kv.nkv;
    unit /= p.kv.nkv;
    const int s = unit % p.step.seqs, nth = unit / p.step.seqs;
    const SeqRows sr = seq_rows(p.step, s);
    // (positions past the table have no page: the sum stays in 32 bits)
    if (sr.rows == 0 || sr.past < 0 || sr.past >= table_positions(p.step, p.kv)) return;
    const int first = sr.past / p.kv.page, last = (sr.past + sr.rows - 1) / p.kv.page;
    if (nth && first + nth >= last) return;
    hold_page<E, VEC>(p, sr, s, first + nth, h, is_k, vals, turn);
    if (nth || first == last) return;
    __syncthreads();
    hold_page<E, VEC>(p, sr, s, last, h, is_k, vals, turn);
}

template <int E, bool VEC>
__global__ void __launch_bounds__(kWave* kPagedWaves) paged_prep_kernel(PagedPrepLaunch p, int hold_blocks, int row_blocks) {
    extern __shared__ _Float16 page_vals[];
    __shared__ double turn[kPagedWaves][kPagedMaxDim];
    const int wid = threadIdx.x / kWave;
    if (static_cast<int>(blockIdx.x) < hold_blocks) {
        hold_unit<E, VEC>(p, blockIdx.x, page_vals, turn[wid]);
        return;
    }
    const int b = blockIdx.x - hold_blocks, row = b / row_blocks, unit = (b - row * row_blocks) * kPagedWaves + wid;
    if (unit < p.nq + (p.kv.i8 ? 0 : 2 * p.kv.nkv)) prep_unit<E, VEC>(p, unit, row, turn[wid]);
}

hipError_t launch_paged_prep(const PagedPrepLaunch& p, hipStream_t s) {
    const int hd = p.kv.head_dim, P = p.kv.page;
    const int64_t touched = (p.step.max_rows + P - 2) / P + 1;  // most pages that one sequence's rows touch
    const int64_t hold = p.kv.i8 ? 2 * std::max<int64_t>(1, touched - 1) * p.kv.nkv * p.step.seqs : 0;
    const int row_blocks = (p.nq + (p.kv.i8 ? 0 : 2 * p.kv.nkv) + kPagedWaves - 1) / kPagedWaves;
    const int64_t blocks = hold + static_cast<int64_t>(row_blocks) * p.step.rows;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    const size_t lds = p.kv.i8 ? static_cast<size_t>(P) * hd * 2 : 0;
    const uintptr_t ptrs = reinterpret_cast<uintptr_t>(p.q_src) | reinterpret_cast<uintptr_t>(p.k_src) |
                           reinterpret_cast<uintptr_t>(p.v_src) | reinterpret_cast<uintptr_t>(p.q_norm) |
                           reinterpret_cast<uintptr_t>(p.k_norm) | reinterpret_cast<uintptr_t>(p.q_out) |
                           reinterpret_cast<uintptr_t>(p.gate_out);
    const bool al = (ptrs & 15u) == 0 && p.src_stride % 4 == 0 && p.out_stride % 4 == 0;
    auto go = [&](auto kernel) {
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(lds));
            e != hipSuccess)
            return e;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kWave * kPagedWaves), lds, s, p, static_cast<int>(hold),
                           row_blocks);
        return hipGetLastError();
    };
    if (hd == 128 && al) return go(paged_prep_kernel<2, true>);
    if (hd == 256 && al) return go(paged_prep_kernel<4, true>);
    return go(paged_prep_kernel<kPagedMaxDim / kWave, false>);
}

// ---------------------------------------------------------------------------
// Positions read back: a block per row, k or v.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) paged_read_kernel(PagedReadLaunch p) {
    const int row = blockIdx.x, hd = p.kv.head_dim, nkv = p.kv.nkv;
    const bool is_v = blockIdx.y != 0;
    T* out = static_cast<T*>(is_v ? p.v_out : p.k_out);
    if (!out) return;
    const int s = __builtin_amdgcn_readfirstlane(seq_of_row(p.step, row));
    if (s >= p.step.seqs) return;
    const SeqRows sr = seq_rows(p.step, s);
    const int j = row - sr.row0;
    if (j < 0 || j >= sr.rows) return;
    const int64_t pos = sr.past < 0 ? -1 : static_cast<int64_t>(sr.past) + j;
    const int page = pos < 0 || pos >= table_positions(p.step, p.kv) ? -1 : page_at(p.step, p.kv, s, static_cast<int>(pos) / p.kv.page);
    const int at = page < 0 ? 0 : static_cast<int>(pos) % p.kv.page;
    const void* pool = is_v ? p.kv.v : p.kv.k;
    const float* scale = is_v ? p.kv.v_scale : p.kv.k_scale;
    for (int i = threadIdx.x; i < nkv * hd; i += 256) {
        const int h = i / hd, d = i - h * hd;
        float x = 0.0f;
        if (page >= 0) {
            const size_t head = page_head(p.kv, page, h);
            if (p.kv.i8) {
                x = static_cast<float>(static_cast<const int8_t*>(pool)[head + (is_v ? v_offset<16>(p.kv, at, d) : k_offset<16>(p.kv, at, d))]) *
                    scale[static_cast<size_t>(page) * nkv + h];
                asm("" : "+v"(x));  // the fp32 product is a value of its own (else it is rounded to fp16 without it)
            } else {
                x = static_cast<float>(static_cast<const _Float16*>(pool)[head + (is_v ? v_offset<8>(p.kv, at, d) : k_offset<8>(p.kv, at, d))]);
            }
        }
        out[(static_cast<size_t>(row) * nkv + h) * hd + d] = static_cast<T>(x);
    }
}

hipError_t launch_paged_read(const PagedReadLaunch& p, hipStream_t s) {
    if (p.f16)
        hipLaunchKernelGGL(paged_read_kernel<_Float16>, dim3(p.step.rows, 2), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL(paged_read_kernel<float>, dim3(p.step.rows, 2), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
