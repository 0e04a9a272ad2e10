// kv_cache.hip - the key/value cache of a decode step over a tree of drafted
// tokens: head preparation with the (fp16 or 8-bit) write, read-back of 8-bit
// caches, and moving the kept rows together.
#include <algorithm>

#include "xqhip_common.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

// ---------------------------------------------------------------------------
// Head preparation (custom_model.cpp:301-370, 673-753): y = x / sqrt(mean x^2 +
// eps) * w, the first 2 rope_pairs dims turned by the position's angles (dim d
// with dim d + rope_pairs), q to q_out, k and v into the cache.
//
// 8-bit rows: scale = max |y| / 127 and code = y / scale to the nearest.  The
// division is the correctly rounded one, and 127 the largest code: a
// reciprocal would move values on a border to the other code.
//
// One wave per (token, head), a head's values in its lanes (lane l: dims E l
// .. E l + E - 1, VEC: in one load; STRIDED, for sizes that are no multiple of
// 64: dims l, l + 64, ..), so the sums and maxima are lane reductions and only
// the rotary partners pass through LDS.  Nothing is read twice; a decode
// step's 48 heads are one round of loads, a launch's latency is its time (3.6
// us).  Prompt chunks are bound by memory: 509 rows of 16 / 4 gated 256-wide
// heads, 39 MB in and out, 9.7 us.
// ---------------------------------------------------------------------------
constexpr int kPrepWaves = 4;
constexpr int kPrepMaxDim = 1024;

template <int E, bool STRIDED, bool VEC>
__global__ void __launch_bounds__(kWave* kPrepWaves) kv_prep_kernel(KvPrepLaunch p) {
    constexpr int kDims = STRIDED ? kPrepMaxDim : E * kWave;
    __shared__ float turn[kPrepWaves][kDims];
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    const int hd = STRIDED ? p.kv.head_dim : kDims, nkv = p.kv.nkv;
    const int unit = blockIdx.x * kPrepWaves + wid, t = blockIdx.y;
    const bool is_q = unit < p.nq, is_k = !is_q && unit < p.nq + nkv;
    const bool on = unit < p.nq + 2 * nkv;
    const int h = is_q ? unit : (is_k ? unit - p.nq : unit - p.nq - nkv);
    const size_t src_off = static_cast<size_t>(t) * p.src_stride;
    const float* src = is_q ? p.q_src + src_off + static_cast<size_t>(h) * (p.gated ? 2 * hd : hd)
                            : (is_k ? p.k_src : p.v_src) + src_off + static_cast<size_t>(h) * hd;
    auto dim = [&](int e) { return STRIDED ? lane + kWave * e : lane * E + e; };
    auto in = [&](int e) { return on && (!STRIDED || dim(e) < hd); };
    auto load = [&](const float* s, float (&x)[E]) {
        if constexpr (VEC) {
            typedef float fv __attribute__((ext_vector_type(E)));
            const fv v = on ? *reinterpret_cast<const fv*>(s + lane * E) : fv(0.0f);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = in(e) ? s[dim(e)] : 0.0f;
        }
    };
    auto put = [&](auto* row, const auto (&v)[E]) {
        if constexpr (VEC) {
            typedef std::remove_pointer_t<decltype(row)> T;
            struct alignas(E * sizeof(T)) Piece {
                T v[E];
            };
            Piece piece;
#pragma unroll
            for (int e = 0; e < E; ++e) piece.v[e] = v[e];
            *reinterpret_cast<Piece*>(row + lane * E) = piece;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (in(e)) row[dim(e)] = v[e];
        }
    };
    float x[E], w[E], gate[E] = {};
    load(src, x);
    if (is_q && p.gated) load(src + hd, gate);
    const float* norm = is_q ? p.q_norm : p.k_norm;
    if (is_q || is_k) load(norm, w);
    // (64 bits: *pos0 is the caller's)
    const int64_t slot = static_cast<int64_t>(*p.pos0) + t;
    const int64_t pos = static_cast<int64_t>(*p.pos0) + (p.has_tree ? p.depth[t] : t);
    const bool held = slot >= 0 && slot < p.kv.capacity && pos >= 0 && pos < p.kv.capacity;
    if (is_q || is_k) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += x[e] * x[e];
        ss = wave_sum(ss);
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(hd) + p.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] *= inv * w[e];
            if (in(e)) turn[wid][dim(e)] = x[e];
        }
    }
    __syncthreads();
    if ((is_q || is_k) && held) {
        const int half = p.rope_pairs;
        const float2* cs = reinterpret_cast<const float2*>(p.rope_cs) + static_cast<size_t>(pos) * half;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = dim(e);
            if (!in(e) || d >= 2 * half) continue;
            const float2 c = cs[d < half ? d : d - half];
            x[e] = d < half ? x[e] * c.x - turn[wid][half + d] * c.y : x[e] * c.x + turn[wid][d - half] * c.y;
        }
    }
    if (!on) return;
    if (is_q) {
        const size_t o = static_cast<size_t>(t) * p.out_stride + static_cast<size_t>(h) * hd;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = held ? x[e] : __builtin_nanf("");
            gate[e] = p.gated ? gate[e] : 0.0f;
        }
        put(p.q_out + o, x);
        if (p.gate_out) put(p.gate_out + o, gate);
        return;
    }
    if (!held) return;
    const size_t head = static_cast<size_t>(slot) * nkv + h;
    if (!p.kv.i8) {
        _Float16 v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = static_cast<_Float16>(x[e]);
        put(static_cast<_Float16*>(is_k ? p.kv.k : p.kv.v) + head * hd, v);
        return;
    }
    float mx = 0.0f;
    bool fine = true;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        mx = fmaxf(mx, fabsf(x[e]));
        fine = fine && fabsf(x[e]) < INFINITY;
    }
    mx = wave_max(mx);
    fine = __builtin_amdgcn_ballot_w64(!fine) == 0;
    const float scale = fine ? mx / 127.0f : __builtin_nanf("");
    int8_t code[E];
#pragma unroll
    for (int e = 0; e < E; ++e)  // (a tiny scale is a denormal with few bits: the quotient can pass 127)
        code[e] = static_cast<int8_t>(fine && scale > 0.0f ? fminf(fmaxf(rintf(x[e] / scale), -127.0f), 127.0f) : 0.0f);
    put(static_cast<int8_t*>(is_k ? p.kv.k : p.kv.v) + head * hd, code);
    if (lane == 0) (is_k ? p.kv.k_scale : p.kv.v_scale)[head] = scale;
}

hipError_t launch_kv_prep(const KvPrepLaunch& p, hipStream_t s) {
    const int hd = p.kv.head_dim, units = p.nq + 2 * p.kv.nkv;
    const dim3 grid((units + kPrepWaves - 1) / kPrepWaves, p.tokens), block(kWave * kPrepWaves);
    const uintptr_t ptrs = reinterpret_cast<uintptr_t>(p.q_src) | reinterpret_cast<uintptr_t>(p.k_src) |
                           reinterpret_cast<uintptr_t>(p.v_src) | reinterpret_cast<uintptr_t>(p.q_norm) |
                           reinterpret_cast<uintptr_t>(p.k_norm) | reinterpret_cast<uintptr_t>(p.q_out) |
                           reinterpret_cast<uintptr_t>(p.gate_out) | reinterpret_cast<uintptr_t>(p.kv.k) |
                           reinterpret_cast<uintptr_t>(p.kv.v);
    const bool al = (ptrs & 15u) == 0 && p.src_stride % 4 == 0 && p.out_stride % 4 == 0;
    if (hd == 128 && al)
        hipLaunchKernelGGL((kv_prep_kernel<2, false, true>), grid, block, 0, s, p);
    else if (hd == 256 && al)
        hipLaunchKernelGGL((kv_prep_kernel<4, false, true>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((kv_prep_kernel<kPrepMaxDim / kWave, true, false>), grid, block, 0, s, p);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// 8-bit rows read back: value = code * scale, in fp32, rounded once for fp16.
// Memory-bound: 1 byte in, 2 or 4 out per value.  A thread takes the codes of one
// 16-byte piece of the output at a time (a wave then writes 1 KiB in a row), four
// pieces in flight.  General form: value by value.  16380 positions of 8 x 128, 102 MB: 16 us, 6.3 TB/s; in
// 8-byte pieces of codes, value by value, it was 55.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ T read_value(int code, float scale) {
    float x = static_cast<float>(code) * scale;
    asm("" : "+v"(x));  // the fp32 product is a value of its own (else it is rounded to fp16 without it)
    return static_cast<T>(x);
}

template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(KvReadLaunch p) {
    const int hd = p.kv.head_dim;
    const size_t first = static_cast<size_t>(p.first) * p.kv.nkv, heads = static_cast<size_t>(p.count) * p.kv.nkv;
    const bool v = blockIdx.y != 0;
    const int8_t* code = static_cast<const int8_t*>(v ? p.kv.v : p.kv.k) + first * hd;
    const float* scale = (v ? p.kv.v_scale : p.kv.k_scale) + first;
    T* out = static_cast<T*>(v ? p.v_out : p.k_out);
    if (!out) return;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < heads * hd;
         i += static_cast<size_t>(gridDim.x) * 256)
        out[i] = read_value<T>(code[i], scale[i / hd]);
}

constexpr int kReadPieces = 4;  // pieces of a thread
template <typename T>
__global__ void __launch_bounds__(256) kv_read_pieces_kernel(KvReadLaunch p, uint32_t pieces, uint32_t per_head, int shift) {
    constexpr int N = 16 / sizeof(T);
    typedef T out_t __attribute__((ext_vector_type(N)));
    typedef signed char code_t __attribute__((ext_vector_type(N)));
    const size_t first = static_cast<size_t>(p.first) * p.kv.nkv;
    const bool v = blockIdx.y != 0;
    const code_t* code = reinterpret_cast<const code_t*>(static_cast<const int8_t*>(v ? p.kv.v : p.kv.k) + first * p.kv.head_dim);
    const float* scale = (v ? p.kv.v_scale : p.kv.k_scale) + first;
    out_t* out = static_cast<out_t*>(v ? p.v_out : p.k_out);
    if (!out) return;
    const uint32_t i0 = blockIdx.x * (256u * kReadPieces) + threadIdx.x;
    code_t c[kReadPieces];
    float f[kReadPieces];
#pragma unroll
    for (int u = 0; u < kReadPieces; ++u) {
        const uint32_t i = i0 + 256u * u;
        if (i < pieces) {
            c[u] = code[i];
            f[u] = scale[shift >= 0 ? i >> shift : i / per_head];
        }
    }
#pragma unroll
    for (int u = 0; u < kReadPieces; ++u) {
        const uint32_t i = i0 + 256u * u;
        if (i >= pieces) return;
        out_t o;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = read_value<T>(c[u][e], f[u]);
        out[i] = o;
    }
}

template <typename T>
static void launch_read(const KvReadLaunch& p, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const int hd = p.kv.head_dim;
    const size_t n = static_cast<size_t>(p.count) * p.kv.nkv * hd;
    const uintptr_t outs = reinterpret_cast<uintptr_t>(p.k_out) | reinterpret_cast<uintptr_t>(p.v_out);
    const uintptr_t codes = reinterpret_cast<uintptr_t>(p.kv.k) | reinterpret_cast<uintptr_t>(p.kv.v);
    if (hd % N == 0 && (outs & 15u) == 0 && codes % N == 0 && n / N < (size_t(1) << 31)) {
        const uint32_t pieces = static_cast<uint32_t>(n / N), per = hd / N;
        const int shift = (per & (per - 1)) == 0 ? __builtin_ctz(per) : -1;
        hipLaunchKernelGGL(kv_read_pieces_kernel<T>, dim3((pieces + 256 * kReadPieces - 1) / (256 * kReadPieces), 2), dim3(256),
                           0, s, p, pieces, per, shift);
        return;
    }
    hipLaunchKernelGGL(kv_read_kernel<T>, dim3(static_cast<unsigned>(std::min<size_t>((n + 255) / 256, 16384)), 2), dim3(256),
                       0, s, p);
}

hipError_t launch_kv_read(const KvReadLaunch& p, hipStream_t s) {
    if (p.f16)
        launch_read<_Float16>(p, s);
    else
        launch_read<float>(p, s);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Kept rows moved together, in place.  A thread owns one column piece of a
// buffer's rows and takes the moves in their order: row j is written after row
// path[j] >= j was read, and no later move reads a row <= j, so no thread
// waits for another.  Eight rows are loaded before the first of them is written,
// and a wave has the whole path in its lanes: nine rows in 40 buffers, 18 MB, 6
// us (with the path read row by row 10).
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void keep_column(const KeepSet& s, int path, int from, int count, int64_t first, size_t at) {
    constexpr int kBatch = 8;  // rows in flight
    uint8_t* col = s.base + static_cast<size_t>(first) * s.row_bytes + at * sizeof(T);
    for (int j0 = from; j0 < count; j0 += kBatch) {
        T v[kBatch] = {};
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (j0 + u < count)
                v[u] = *reinterpret_cast<const T*>(col + static_cast<size_t>(__builtin_amdgcn_readlane(path, j0 + u)) * s.row_bytes);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (j0 + u < count) *reinterpret_cast<T*>(col + static_cast<size_t>(j0 + u) * s.row_bytes) = v[u];
    }
}

__global__ void __launch_bounds__(256) tree_keep_kernel(KeepLaunch p) {
    const KeepSet& s = p.sets[blockIdx.y];
    const bool wide = ((reinterpret_cast<uintptr_t>(s.base) | s.row_bytes) & 15u) == 0;
    const size_t pieces = wide ? s.row_bytes / 16 : s.row_bytes;
    if (static_cast<size_t>(blockIdx.x) * 256 >= pieces) return;
    // lane j holds path[j]; the moves go up to the first that is none: a row outside the buffer, a path that does not
    // increase (read one after the other they would be a memory round trip each)
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t first = s.first ? *s.first : 0;
    const int want = min(*p.count, p.max_rows);
    const int path = lane < p.max_rows ? p.path[lane] : -1;
    int before = __shfl_up(path, 1, kWave);
    if (lane == 0) before = -1;
    const uint64_t good = __builtin_amdgcn_ballot_w64(lane < want && path > before && first >= 0 && first + path < s.rows);
    const int count = ~good ? __builtin_ctzll(~good) : kWave;
    const uint64_t moved = __builtin_amdgcn_ballot_w64(path != lane);  // the rows before the first such one are in place
    const int from = moved ? __builtin_ctzll(moved) : kWave;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < pieces;
         i += static_cast<size_t>(gridDim.x) * 256) {
        if (wide)
            keep_column<u32x4>(s, path, from, count, first, i);
        else
            keep_column<uint8_t>(s, path, from, count, first, i);
    }
}

hipError_t launch_tree_keep(const KeepLaunch& p, int n_sets, hipStream_t s) {
    size_t most = 0;
    for (int i = 0; i < n_sets; ++i) {
        const KeepSet& k = p.sets[i];
        const bool wide = ((reinterpret_cast<uintptr_t>(k.base) | k.row_bytes) & 15u) == 0;
        most = std::max<size_t>(most, wide ? k.row_bytes / 16 : k.row_bytes);
    }
    const dim3 grid(static_cast<unsigned>(std::min<size_t>((most + 255) / 256, 256)), n_sets);
    hipLaunchKernelGGL(tree_keep_kernel, grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace xqhip
