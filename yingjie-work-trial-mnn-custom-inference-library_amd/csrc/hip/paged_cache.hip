// paged_cache.hip - the paged key/value cache of a step over several sequences:
// head preparation with the append, and read-back.
#include <algorithm>
#include <type_traits>

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
//
// What bounds it: loads that wait for each other (the step's tables, the rotary
// positions, the angles, the rows) and the barrier before the codes.  All blocks are
// on the card at once, so a step takes as long as one block's chain: 509 rows of 16 /
// 4 heads of 256 into 8-bit pages 15.7 us, in which the vector units are busy for a
// third of the cycles (13 % of their instructions are 64-bit ones) and the waves wait
// for half of them; 5.6 for the read-back.  512 rows of 32 / 8 heads of 128 with their
// read-back 17.3 us; single tokens 3.8 to 4.7 us.
// ---------------------------------------------------------------------------
constexpr int kPagedMaxDim = 256;
constexpr int kPagedMaxPage = 128;

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


// The positions of a row on its axes (wave-uniform), and whether all that its pairs use lie in the table.
// (The first's, and what the others are more: a choice between four values held in an object becomes an indexed load of
// it, from LDS, at an offset that takes the dispatch packet in host memory: 13 us.)
struct RowAxes {
    int a0, d1, d2, d3;
    bool fine;
    __device__ __forceinline__ void load(const RotaryAxes& r, int rows, int row, int pos) {
        auto at = [&](int a) { return r.pos && a < r.axes ? r.pos[static_cast<size_t>(a) * rows + row] : pos; };
        auto in = [&](int a, int p) { return !(r.used >> a & 1) || (p >= 0 && p < r.positions); };
        const int p0 = at(0), p1 = at(1), p2 = at(2), p3 = at(3);
        fine = in(0, p0) && in(1, p1) && in(2, p2) && in(3, p3);
        auto less = [](int a, int b) { return static_cast<int>(static_cast<uint32_t>(a) - static_cast<uint32_t>(b)); };  // (of an axis without pairs it may wrap)
        a0 = fine ? p0 : 0;  // (the angles of a row that is not: those of position 0)
        d1 = fine ? less(p1, p0) : 0;
        d2 = fine ? less(p2, p0) : 0;
        d3 = fine ? less(p3, p0) : 0;
    }
    __device__ __forceinline__ int of(int axis) const { return a0 + (axis == 1 ? d1 : 0) + (axis == 2 ? d2 : 0) + (axis == 3 ? d3 : 0); }
};

// The pairs of a lane's dims and their axes, the same for every row.
template <int E, bool VEC>
struct LanePairs {
    int pair[E], axis[E];  // pair -1: a dim that is not turned
    __device__ __forceinline__ LanePairs(const RotaryAxes& r, int lane) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = HeadLanes<E, VEC>::dim(lane, e), i = d < r.pairs ? d : d - r.pairs;
            uint32_t bits = 0;  // (selected from the arguments: indexed by lane they would be a load)
#pragma unroll
            for (int k = 0; k < 8; ++k) bits = i / 16 == k ? r.axis[k] : bits;
            pair[e] = d < 2 * r.pairs ? i : -1;
            axis[e] = bits >> 2 * (i % 16) & 3;
        }
    }
    __device__ __forceinline__ void angles(const RotaryAxes& r, const RowAxes& row, float2 (&cs)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            cs[e] = make_float2(1.0f, 0.0f);
            if (pair[e] >= 0) cs[e] = r.cs[static_cast<size_t>(row.of(axis[e])) * r.pairs + pair[e]];
        }
    }
};

// 1 / sqrt(v): the hardware's estimate and two steps of Newton's, within 2^-50 (what is kept of it has 24 bits).  Of infinity
// 0, the estimate, which the steps leave with a number in its place (chosen behind them 0.3 us more in a step of 16 rows).
__device__ __forceinline__ double inverse_sqrt(double v) {
    double y = __builtin_amdgcn_rsq(v);
    v = fmin(v, 1.0e300);
#pragma unroll
    for (int i = 0; i < 2; ++i) y = fma(0.5 * y, fma(-v * y, y, 1.0), y);
    return y;
}

__device__ __forceinline__ double lane_value(double v, int from) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_ds_bpermute(4 * from, static_cast<int>(static_cast<uint32_t>(u)));
    const uint32_t hi = __builtin_amdgcn_ds_bpermute(4 * from, static_cast<int>(static_cast<uint32_t>(u >> 32)));
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// B rows of a head normalised and turned, by a whole wave, their chains of 64-bit operations beside each other.  A dim's
// partner in its pair lies `half` dims on: in another lane (VEC, half a multiple of E), or it is fetched through the wave's
// kPagedMaxDim doubles of LDS, `turn`.
template <int B, int E, bool VEC>
__device__ __forceinline__ void turn_heads(float (&x)[B][E], const float (&w)[E], const float2 (&cs)[B][E], int hd, int half, double inv_hd,
                                           float eps, int lane, double* turn) {
    typedef HeadLanes<E, VEC> L;
    double v[B][E], inv[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
        inv[b] = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) inv[b] += static_cast<double>(x[b][e]) * x[b][e];
    }
#pragma unroll
    for (int b = 0; b < B; ++b) inv[b] = wave_sum_double(inv[b]);
#pragma unroll
    for (int b = 0; b < B; ++b) inv[b] = inverse_sqrt(fma(inv[b], inv_hd, static_cast<double>(eps)));
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int e = 0; e < E; ++e) v[b][e] = static_cast<double>(x[b][e]) * inv[b] * w[e];
    const bool by_lanes = VEC && half % E == 0;  // block-uniform
    auto turned = [&](double a, double other, float2 c, int d) { return d < half ? a * c.x - other * c.y : (d < 2 * half ? a * c.x + other * c.y : a); };
    if (by_lanes) {
        const int from = lane * E < half ? lane + half / E : lane - half / E;
        double other[B][E];
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int e = 0; e < E; ++e) other[b][e] = lane_value(v[b][e], from & (kWave - 1));
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int e = 0; e < E; ++e) x[b][e] = static_cast<float>(turned(v[b][e], other[b][e], cs[b][e], L::dim(lane, e)));
    } else {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            wave_lds_sync();
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (L::in(lane, e, hd)) turn[L::dim(lane, e)] = v[b][e];
            wave_lds_sync();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = L::dim(lane, e);
                const double other = d < half ? turn[half + d] : (d < 2 * half ? turn[d - half] : 0.0);
                x[b][e] = static_cast<float>(turned(v[b][e], other, cs[b][e], d));
            }
        }
    }
}

// Where a sequence's position goes: its page, and its open page (-1: none).  (Both loads go out at once, from places that
// exist.)
struct Place {
    int page, open;
    __device__ __forceinline__ Place(const PagedPrepLaunch& p, int s, int64_t pos) {
        const int at = static_cast<int>(max(int64_t(0), min(pos, static_cast<int64_t>(table_positions(p.step, p.kv)) - 1))) / p.kv.page;
        page = p.step.table[static_cast<size_t>(s) * p.step.max_pages + at];
        open = p.kv.i8 ? p.step.open[s] : 0;
        if (pos != at * static_cast<int64_t>(p.kv.page) + (pos & (p.kv.page - 1)) || (p.kv.i8 && open >= p.kv.opens)) open = -1;
        if (page >= p.kv.pages || open < 0) page = -1;
    }
    __device__ __forceinline__ bool none() const { return page < 0; }
};

// `per` query heads of one row by a wave, from h0 on: q and their gates.
constexpr int kQueryHeads = 4;
template <int E, bool VEC>
__device__ __forceinline__ void query_unit(const PagedPrepLaunch& p, int h0, int per, int row, double* turn) {
    typedef HeadLanes<E, VEC> L;
    const int lane = threadIdx.x & (kWave - 1), hd = p.kv.head_dim;
    const LanePairs<E, VEC> pairs(p.rot, lane);
    const float* src = p.q_src + static_cast<size_t>(row) * p.src_stride;
    float x[kQueryHeads][E], gate[kQueryHeads][E], w[E];
    auto on = [&](int i) { return i < per && h0 + i < p.nq; };  // wave-uniform
#pragma unroll
    for (int i = 0; i < kQueryHeads; ++i)
        if (on(i)) {
            const float* at = src + static_cast<size_t>(h0 + i) * (p.gated ? 2 * hd : hd);
            L::load(at, lane, hd, x[i]);
            if (p.gated) L::load(at + hd, lane, hd, gate[i]);
        }
    L::load(p.q_norm, lane, hd, w);
    const int s = __builtin_amdgcn_readfirstlane(seq_of_row(p.step, row));
    if (s >= p.step.seqs) return;
    const SeqRows sr = seq_rows(p.step, s);
    const int j = row - sr.row0;
    if (j < 0 || j >= sr.rows || sr.rows == 1) return;  // (token_unit's)
    const int64_t pos = sr.past < 0 ? -1 : static_cast<int64_t>(sr.past) + j;
    RowAxes axes;
    axes.load(p.rot, p.step.rows, row, static_cast<int>(pos));
    const Place place(p, s, pos);
    const bool turned = axes.fine;
    float2 cs[1][E] = {};
    pairs.angles(p.rot, axes, cs[0]);
    const bool held = turned && !place.none();
    const size_t o = static_cast<size_t>(row) * p.out_stride;
#pragma unroll
    for (int i = 0; i < kQueryHeads; ++i) {
        if (!on(i)) break;
        float y[1][E];
#pragma unroll
        for (int e = 0; e < E; ++e) y[0][e] = x[i][e];
        turn_heads<1, E, VEC>(y, w, cs, hd, p.rot.pairs, p.inv_hd, p.eps, lane, turn);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            y[0][e] = held ? y[0][e] : __builtin_nanf("");
            if (!p.gated) gate[i][e] = 0.0f;
        }
        const size_t at = o + static_cast<size_t>(h0 + i) * hd;
        L::store(p.q_out + at, lane, hd, y[0]);
        if (p.gate_out) L::store(p.gate_out + at, lane, hd, gate[i]);
    }
}

// The fp16 value that 8 bits are taken of: no infinities, no NaN.
__device__ __forceinline__ _Float16 held_value(float x) {
    return static_cast<_Float16>(x == x ? fminf(fmaxf(x, -65504.0f), 65504.0f) : 0.0f);
}
// 127 x / mx to the nearest, inv near 1 / mx: 127 x is exact (18 bits), the quotient's error is taken off by its exact
// remainder, so it is half a code's step exactly where the true one is (which is then a number of few bits), and
// elsewhere further from it (2^-12) than its own rounding
__device__ __forceinline__ int code_of(_Float16 x, float mx, float inv) {
    const float n = 127.0f * static_cast<float>(x);
    float q = n * inv;
    q = fmaf(fmaf(-mx, q, n), inv, q);
    return static_cast<int>(__builtin_amdgcn_fmed3f(rintf(q), -127.0f, 127.0f));  // (a position never written may pass the maximum)
}

// A step's rows of one page, one kv head, k or v, as the page holds them, by a block (four rows' loads of a wave at a time):
// those at [from, end) of the page with the first position `base`; to(t, held, v) takes row t.  before(): what is fetched
// beside the first ones.
template <int W, int E, bool VEC, bool I8, typename Before, typename To>
__device__ __forceinline__ void page_rows(const PagedPrepLaunch& p, const SeqRows& sr, int base, int from, int end, int h, bool is_k, double* turn, Before before,
                                          To to) {
    typedef HeadLanes<E, VEC> L;
    constexpr int kBatch = E == 2 ? 4 : 2;
    const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), hd = p.kv.head_dim;
    const LanePairs<E, VEC> pairs(p.rot, lane);
    float x[kBatch][E], w[E];
    RowAxes axes[kBatch];
    auto load = [&](int t0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {  // (rows behind the last: the last again)
            const int row = sr.row0 + base + min(t0 + b * W, end - 1) - sr.past;
            L::load((is_k ? p.k_src : p.v_src) + static_cast<size_t>(row) * p.src_stride + static_cast<size_t>(h) * hd, lane, hd, x[b]);
            axes[b].load(p.rot, p.step.rows, row, base + min(t0 + b * W, end - 1));
        }
    };
    load(from + wid);
    if (is_k) L::load(p.k_norm, lane, hd, w);
    if (!before()) return;  // block-uniform
    for (int t0 = from + wid; t0 < end; t0 += kBatch * W) {
        float2 cs[kBatch][E];
        bool held[kBatch];
        float y[kBatch][E];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            held[b] = t0 + b * W < end && axes[b].fine;
            if (is_k) pairs.angles(p.rot, axes[b], cs[b]);
#pragma unroll
            for (int e = 0; e < E; ++e) y[b][e] = x[b][e];
        }
        if (t0 + kBatch * W < end) load(t0 + kBatch * W);  // (wave-uniform; they come while these are turned)
        if (is_k) turn_heads<kBatch, E, VEC>(y, w, cs, hd, p.rot.pairs, p.inv_hd, p.eps, lane, turn);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int t = t0 + b * W;
            if (t >= end) break;  // wave-uniform
            _Float16 v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = I8 ? held_value(y[b][e]) : static_cast<_Float16>(y[b][e]);
            to(t, held[b], v);
        }
    }
}

template <int E, bool VEC>
__device__ __forceinline__ void put_row(const _Float16 (&v)[E], int lane, int hd, _Float16* d) {
    typedef HeadLanes<E, VEC> L;
    if constexpr (VEC) {
        typedef _Float16 hv __attribute__((ext_vector_type(E)));
        hv y;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = v[e];
        *reinterpret_cast<hv*>(d + lane * E) = y;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (L::in(lane, e, hd)) d[L::dim(lane, e)] = v[e];
    }
}

// a row's fp16 values for the open page, zeros where it is not held
template <int E, bool VEC>
__device__ __forceinline__ void keep_row(const _Float16 (&v)[E], bool held, int lane, int hd, _Float16* d) {
    _Float16 y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = held ? v[e] : static_cast<_Float16>(0.0f);
    put_row<E, VEC>(y, lane, hd, d);
}
// rows [from, end) of an open page, by a block
template <int THREADS>
__device__ __forceinline__ void keep_zeros(_Float16* kept, int from, int end, int hd) {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    for (int i = from * (hd / 8) + threadIdx.x; i < end * (hd / 8); i += THREADS) reinterpret_cast<half8*>(kept)[i] = half8{};
}
// a head's rows in the open page, nullptr: none
__device__ __forceinline__ _Float16* open_rows(const PagedPrepLaunch& p, const Place& place, int h, bool is_k) {
    if (place.open < 0) return nullptr;
    return (is_k ? p.kv.k_open : p.kv.v_open) + (static_cast<size_t>(place.open) * p.kv.nkv + h) * p.kv.page * p.kv.head_dim;
}

// The largest magnitude that a page's scale stands for: an fp16 value, exactly.  (A page that no row began may have any scale.)
__device__ __forceinline__ float recorded_max(float scale) {
    return static_cast<float>(static_cast<_Float16>(fminf(fmaxf(scale * 127.0f, 0.0f), 65504.0f)));
}

// One page that the step touches, one kv head, k or v, by a block.  The new rows' fp16 values go to LDS, then to the page in
// 16-byte pieces; 8 bits: their maximum is taken on the way, and where it rose, or the step leaves the page, the page's
// earlier values are fetched and the codes of all of them written.  A page of which no row is held stays as it is, and only a
// row that is held at its first position begins it anew.  The last page's rows from keep_from on are kept, as zeros where they
// are not held: what another sequence left there would count in the page's maximum.
template <int W, int E, bool VEC, bool I8>
__device__ __forceinline__ void hold_page(const PagedPrepLaunch& p, const SeqRows& sr, int s, int index, int keep_from, int h, bool is_k, _Float16* vals, double* turn) {
    typedef HeadLanes<E, VEC> L;
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    constexpr int kThreads = kWave * W;
    __shared__ float wave_mx[W];
    __shared__ uint8_t ok[kPagedMaxPage];
    const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int hd = p.kv.head_dim, nkv = p.kv.nkv, P = p.kv.page;
    const int base = index * P, ld = hd + 8;                                          // position of the page's first
    const int lead = max(0, sr.past - base), end = min(P, sr.past + sr.rows - base);  // new ones: [lead, end)
    const bool last = base + P >= sr.past + sr.rows;
    int page = -1;
    size_t sat = 0;
    _Float16* kept = nullptr;
    float was = 0.0f, mx = 0.0f;
    auto before = [&] {
        const Place place(p, s, base);
        page = place.page;
        if constexpr (I8) kept = open_rows(p, place, h, is_k);
        if (place.none()) return false;  // block-uniform
        sat = static_cast<size_t>(page) * nkv + h;
        if (I8 && lead) was = (is_k ? p.kv.k_scale : p.kv.v_scale)[sat];
        return true;
    };
    page_rows<W, E, VEC, I8>(p, sr, base, lead, end, h, is_k, turn, before, [&](int t, bool held, const _Float16(&v)[E]) {
        if (lane == 0) ok[t] = held;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (I8 && held && L::in(lane, e, hd)) mx = fmaxf(mx, fabsf(static_cast<float>(v[e])));
        put_row<E, VEC>(v, lane, hd, vals + t * ld);
        if (I8 && last && t >= keep_from) keep_row<E, VEC>(v, held, lane, hd, kept + static_cast<size_t>(t) * hd);
    });
    if (page < 0) {
        if (I8 && last && kept) keep_zeros<kThreads>(kept, max(lead, keep_from), end, hd);
        return;
    }
    int from = lead;
    float inv = 0.0f;
    auto earlier = [&] {  // the page's values before the step, in fp16
        for (int i = threadIdx.x; i < lead * (hd / 8); i += kThreads) {
            const int t = i / (hd / 8), b = i - t * (hd / 8);
            const half8 y = *reinterpret_cast<const half8*>(kept + static_cast<size_t>(t) * hd + 8 * b);
            *reinterpret_cast<half8*>(vals + t * ld + 8 * b) = y;
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(static_cast<float>(y[e])));
        }
    };
    if constexpr (I8) {
        if (lead && !last) {  // the step leaves the page: it is written as it will stay
            earlier();
            from = 0;
        }
        mx = wave_max(mx);
        if (lane == 0) wave_mx[wid] = mx;
    }
    __syncthreads();
    uint64_t on[2];  // new positions that are held
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = i * kWave + lane;
        on[i] = __builtin_amdgcn_ballot_w64(t >= lead && t < end && ok[t] != 0);
    }
    if ((on[0] | on[1]) == 0) return;  // block-uniform
    if constexpr (I8) {
#pragma unroll
        for (int i = 0; i < W; ++i) mx = fmaxf(mx, wave_mx[i]);
        if (!lead && !(on[0] & 1)) was = (is_k ? p.kv.k_scale : p.kv.v_scale)[sat];  // block-uniform
        const float before = recorded_max(was);
        const bool grew = mx > before;
        mx = grew ? mx : before;
        inv = mx > 0.0f ? 1.0f / mx : 0.0f;
        if (grew && lead && last) {
            const float all = mx;
            earlier();
            mx = all;
            from = 0;
            __syncthreads();
        }
        if (threadIdx.x == 0) (is_k ? p.kv.k_scale : p.kv.v_scale)[sat] = mx / 127.0f;
    }
    // positions to write: [from, lead) and the new ones that are held
    uint64_t go[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = i * kWave + lane;
        go[i] = on[i] | __builtin_amdgcn_ballot_w64(t >= from && t < lead);
    }
    auto writes = [&](int t) { return (t < kWave ? go[0] >> t : go[1] >> (t - kWave)) & 1; };
    constexpr int N = I8 ? 16 : 8;  // values of a piece
    typedef typename std::conditional<I8, int8_t, _Float16>::type T;
    union Piece {
        T v[N];
        u32x4 all;
    };
    auto value = [&](_Float16 v) -> T {
        if constexpr (I8)
            return static_cast<T>(code_of(v, mx, inv));
        else
            return v;
    };
    T* d = static_cast<T*>(is_k ? p.kv.k : p.kv.v) + page_head(p.kv, page, h);
    if (is_k) {  // lanes over positions, then blocks of dims
        const int n = end - from;
        for (int i = threadIdx.x; i < n * (hd / N); i += kThreads) {
            const int b = i / n, t = from + i - b * n;
            if (!writes(t)) continue;
            Piece o;
#pragma unroll
            for (int u = 0; u < N / 8; ++u) {
                const half8 y = *reinterpret_cast<const half8*>(vals + t * ld + b * N + 8 * u);
#pragma unroll
                for (int e = 0; e < 8; ++e) o.v[8 * u + e] = value(y[e]);
            }
            *reinterpret_cast<u32x4*>(d + (static_cast<size_t>(b) * P + t) * N) = o.all;
        }
    } else {  // lanes over dims, then blocks of positions
        const int b0 = from / N, n = (end - 1) / N + 1 - b0;
        for (int i = threadIdx.x; i < n * hd; i += kThreads) {
            const int b = b0 + i / hd, dim = i % hd, t0 = b * N;
            const uint32_t on = static_cast<uint32_t>((t0 < kWave ? go[0] >> t0 : go[1] >> (t0 - kWave)) & ((1u << N) - 1));
            T* at = d + (static_cast<size_t>(b) * hd + dim) * N;
            if (on == (1u << N) - 1) {
                Piece o;
#pragma unroll
                for (int e = 0; e < N; ++e) o.v[e] = value(vals[(t0 + e) * ld + dim]);
                *reinterpret_cast<u32x4*>(at) = o.all;
            } else {
                for (int e = 0; e < N; ++e)
                    if (on >> e & 1) at[e] = value(vals[(t0 + e) * ld + dim]);
            }
        }
    }
}

// The pages that the step touches, a block per page, kv head and k or v, in the order of the sequences.  The earlier values of
// an 8-bit page that the step leaves lie where those of its last page are kept: the block of the first has fetched them
// before it keeps those rows of the last, which it computes too, and the last's block the others.
__device__ __forceinline__ int hold_blocks_of(const PagedPrepLaunch& p, const SeqRows& r) {
    // (positions past the table have no page: the sums stay in 32 bits)
    if (r.rows <= 1 || r.past < 0 || r.past >= table_positions(p.step, p.kv)) return 0;
    return (r.past + r.rows - 1) / p.kv.page - r.past / p.kv.page + 1;
}
template <int W, int E, bool VEC, bool I8>
__device__ __forceinline__ void hold_unit(const PagedPrepLaunch& p, int unit, _Float16* vals, double* turn) {
    const bool is_k = (unit & 1) == 0;
    unit >>= 1;
    const int h = unit % p.kv.nkv, nth = unit / p.kv.nkv;  // block `nth` of the head
    int before = 0, s = -1, first_block = 0;
    for (int c = 0; c < p.step.seqs && s < 0; c += kWave) {  // each wave by itself
        const int q = c + static_cast<int>(threadIdx.x & (kWave - 1));
        const int in = before + wave_scan_int(q < p.step.seqs ? hold_blocks_of(p, seq_rows(p.step, q)) : 0);
        const int n = __popcll(__builtin_amdgcn_ballot_w64(in <= nth));
        if (n < kWave) {
            s = c + n;
            first_block = n ? __builtin_amdgcn_readlane(in, n - 1) : before;
        }
        before = __builtin_amdgcn_readlane(in, kWave - 1);
    }
    if (s < 0) return;  // fewer pages than blocks
    const SeqRows sr = seq_rows(p.step, s);
    const int P = p.kv.page, lead = sr.past % P, first = sr.past / P, last = (sr.past + sr.rows - 1) / P, index = first + nth - first_block;
    hold_page<W, E, VEC, I8>(p, sr, s, index, index == first ? 0 : lead, h, is_k, vals, turn);
    if constexpr (I8)
        if (index == first && first < last && lead) {
            __syncthreads();
            const int end = min(lead, sr.past + sr.rows - last * P), lane = threadIdx.x & (kWave - 1), hd = p.kv.head_dim;
            _Float16* kept = nullptr;
            bool none = true;
            auto before = [&] {
                const Place place(p, s, static_cast<int64_t>(last) * P);
                kept = open_rows(p, place, h, is_k);
                none = place.none();
                return !none;
            };
            page_rows<W, E, VEC, I8>(p, sr, last * P, 0, end, h, is_k, turn, before,
                                     [&](int t, bool held, const _Float16(&v)[E]) { keep_row<E, VEC>(v, held, lane, hd, kept + static_cast<size_t>(t) * hd); });
            if (none && kept) keep_zeros<kWave * W>(kept, 0, end, hd);
        }
}

// A sequence that brings one row: a head by a wave (query heads, then keys, then values).
template <int E, bool VEC, bool I8>
__device__ __forceinline__ void token_unit(const PagedPrepLaunch& p, int s, int unit, double* turn) {
    typedef HeadLanes<E, VEC> L;
    const int lane = threadIdx.x & (kWave - 1), hd = p.kv.head_dim, nkv = p.kv.nkv, P = p.kv.page;
    const SeqRows sr = seq_rows(p.step, s);
    if (sr.rows != 1) return;
    const int row = sr.row0;
    const bool is_q = unit < p.nq, is_k = !is_q && unit < p.nq + nkv;
    const int h = is_q ? unit : (is_k ? unit - p.nq : unit - p.nq - nkv);
    const float* src = (is_q ? p.q_src : is_k ? p.k_src : p.v_src) + static_cast<size_t>(row) * p.src_stride +
                       static_cast<size_t>(h) * (is_q && p.gated ? 2 * hd : hd);
    float in[1][E], gate[E] = {}, w[E];
    float(&x)[E] = in[0];
    L::load(src, lane, hd, x);
    if (is_q && p.gated) L::load(src + hd, lane, hd, gate);
    if (is_q || is_k) L::load(is_q ? p.q_norm : p.k_norm, lane, hd, w);
    const int64_t pos = sr.past < 0 ? -1 : sr.past;
    RowAxes axes;
    axes.load(p.rot, p.step.rows, row, static_cast<int>(pos));
    const Place place(p, s, pos);
    const bool turned = axes.fine;
    float2 cs[1][E] = {};
    if (is_q || is_k) LanePairs<E, VEC>(p.rot, lane).angles(p.rot, axes, cs[0]);
    const bool held = turned && !place.none();
    const int t = static_cast<int>(pos) & (P - 1);
    float was = 0.0f;
    const size_t sat = static_cast<size_t>(max(place.page, 0)) * nkv + h;
    float* scale = is_k ? p.kv.k_scale : p.kv.v_scale;
    if (I8 && !is_q && held && t) was = scale[sat];
    if (is_q || is_k) turn_heads<1, E, VEC>(in, w, cs, hd, p.rot.pairs, p.inv_hd, p.eps, lane, turn);
    if (is_q) {
        const size_t o = static_cast<size_t>(row) * p.out_stride + static_cast<size_t>(h) * hd;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = held ? x[e] : __builtin_nanf("");
        L::store(p.q_out + o, lane, hd, x);
        if (p.gate_out) L::store(p.gate_out + o, lane, hd, gate);
        return;
    }
    if (!held) {
        if (I8 && place.open >= 0) {
            const _Float16 zeros[E] = {};
            put_row<E, VEC>(zeros, lane, hd, open_rows(p, place, h, is_k) + static_cast<size_t>(t) * hd);
        }
        return;
    }
    constexpr int N = I8 ? 16 : 8;
    auto offset = [&](int pos_in, int dim) { return is_k ? k_offset<N>(p.kv, pos_in, dim) : v_offset<N>(p.kv, pos_in, dim); };
    const size_t head = page_head(p.kv, place.page, h);
    if constexpr (!I8) {
        _Float16* d = static_cast<_Float16*>(is_k ? p.kv.k : p.kv.v) + head;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (L::in(lane, e, hd)) d[offset(t, L::dim(lane, e))] = static_cast<_Float16>(x[e]);
    } else {
        int8_t* d = static_cast<int8_t*>(is_k ? p.kv.k : p.kv.v) + head;
        _Float16* kept = open_rows(p, place, h, is_k);
        _Float16 v[E];
        float mx = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = held_value(x[e]);
            if (!L::in(lane, e, hd)) continue;
            mx = fmaxf(mx, fabsf(static_cast<float>(v[e])));
            kept[static_cast<size_t>(t) * hd + L::dim(lane, e)] = v[e];
        }
        mx = wave_max(mx);
        const float before = recorded_max(was);
        const bool grew = mx > before;
        mx = grew ? mx : before;
        const float inv = mx > 0.0f ? 1.0f / mx : 0.0f;
        if (lane == 0) scale[sat] = mx / 127.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (L::in(lane, e, hd)) d[offset(t, L::dim(lane, e))] = static_cast<int8_t>(code_of(v[e], mx, inv));
        if (grew) {  // wave-uniform: the page's earlier codes anew (of 64 positions a maximum rises at five or so)
#pragma unroll 4
            for (int i = 0; i < t; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (L::in(lane, e, hd))
                        d[offset(i, L::dim(lane, e))] = static_cast<int8_t>(code_of(kept[static_cast<size_t>(i) * hd + L::dim(lane, e)], mx, inv));
        }
    }
}

// Steps with longer sequences: blocks of pages, then waves of the sequences with one row, then of the others' query heads
// (with its read-back a step of 59 tokens and 30 rows 22.5 us; the tokens by page and row too 28.6).
template <int W, int E, bool VEC, bool I8>
__global__ void __launch_bounds__(kWave* W, 4) paged_prep_kernel(PagedPrepLaunch p, int hold_blocks, int token_blocks, int row_units, int per) {
    extern __shared__ uint4 page_lds[];
    _Float16* page_vals = reinterpret_cast<_Float16*>(page_lds);
    __shared__ double turn[W][kPagedMaxDim];
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (static_cast<int>(blockIdx.x) < hold_blocks) {
        hold_unit<W, E, VEC, I8>(p, blockIdx.x, page_vals, turn[wid]);
        return;
    }
    if (static_cast<int>(blockIdx.x) < hold_blocks + token_blocks) {
        const int heads = p.nq + 2 * p.kv.nkv, unit = (static_cast<int>(blockIdx.x) - hold_blocks) * W + wid, s = unit / heads;
        if (s < p.step.seqs) token_unit<E, VEC, I8>(p, s, unit - s * heads, turn[wid]);
        return;
    }
    const int unit = (static_cast<int>(blockIdx.x) - hold_blocks - token_blocks) * W + wid, row = unit / row_units;
    if (row < p.step.rows) query_unit<E, VEC>(p, (unit - row * row_units) * per, per, row, turn[wid]);
}

// Steps of single tokens: no barrier between a block's waves (with the read-back of that time 32 tokens 10.3 us, by page and
// row 16.1; one token 7.8, 11.1; with today's 9.4 and 8.3).
constexpr int kTokenWaves = 4;
template <int E, bool VEC, bool I8>
__global__ void __launch_bounds__(kWave* kTokenWaves) paged_token_kernel(PagedPrepLaunch p, int row_blocks) {
    __shared__ double turn[kTokenWaves][kPagedMaxDim];
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int s = blockIdx.x / row_blocks, unit = (static_cast<int>(blockIdx.x) - s * row_blocks) * kTokenWaves + wid;
    if (unit < p.nq + 2 * p.kv.nkv) token_unit<E, VEC, I8>(p, s, unit, turn[wid]);
}

hipError_t launch_paged_prep(const PagedPrepLaunch& p, hipStream_t s) {
    const int hd = p.kv.head_dim, P = p.kv.page;
    const uintptr_t ptrs = reinterpret_cast<uintptr_t>(p.q_src) | reinterpret_cast<uintptr_t>(p.k_src) |
                           reinterpret_cast<uintptr_t>(p.v_src) | reinterpret_cast<uintptr_t>(p.q_norm) |
                           reinterpret_cast<uintptr_t>(p.k_norm) | reinterpret_cast<uintptr_t>(p.q_out) |
                           reinterpret_cast<uintptr_t>(p.gate_out);
    const bool al = (ptrs & 15u) == 0 && p.src_stride % 4 == 0 && p.out_stride % 4 == 0;
    if (p.step.max_rows == 1) {
        const int row_blocks = (p.nq + 2 * p.kv.nkv + kTokenWaves - 1) / kTokenWaves;
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.step.seqs) * row_blocks), dim3(kWave * kTokenWaves), 0, s, p, row_blocks);
            return hipGetLastError();
        };
        constexpr int E = kPagedMaxDim / kWave;
        if (hd == 128 && al) return p.kv.i8 ? go(paged_token_kernel<2, true, true>) : go(paged_token_kernel<2, true, false>);
        if (hd == 256 && al) return p.kv.i8 ? go(paged_token_kernel<4, true, true>) : go(paged_token_kernel<4, true, false>);
        return p.kv.i8 ? go(paged_token_kernel<E, false, true>) : go(paged_token_kernel<E, false, false>);
    }
    // (with the read-back: 512 rows with one head a wave 23.2 us, with four 17.3; 51 rows 13.4 either way)
    const int per = p.step.rows >= 128 ? std::min(kQueryHeads, p.nq) : 1;
    const int row_units = (p.nq + per - 1) / per;
    // pages of any division of the rows among the sequences: n rows reach over n / P page borders, and one more; one more
    // page than borders
    const int64_t hold = 2 * static_cast<int64_t>(p.kv.nkv) * (p.step.rows / P + 2 * std::min(p.step.seqs, p.step.rows));
    // Waves of a block: eight; sixteen where pages take many passes of eight and there are few of them (with the read-back: 500
    // rows, fp16 pages of 128, heads of 128 20.2 us, by eight waves 25.0; 139 rows in 8 bits, heads of 256 29.2, 32.8; four
    // chunks of 512, 8-bit pages of 64, 45.3, 42.2, fp16 pages of 128 47.8, 42.9).
    const bool long_pages = std::min(P, p.step.max_rows) * (hd > 128 ? 2 : 1) >= 128, few = 2 * p.kv.nkv * p.step.rows <= 128 * P;
    const int waves = long_pages && few ? 16 : 8;
    const int64_t tokens = (static_cast<int64_t>(p.step.seqs) * (p.nq + 2 * p.kv.nkv) + waves - 1) / waves;
    const int64_t blocks = hold + tokens + (static_cast<int64_t>(row_units) * p.step.rows + waves - 1) / waves;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    const size_t lds = static_cast<size_t>(P) * (hd + 8) * 2;
    auto go = [&](auto kernel) {
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(lds));
            e != hipSuccess)
            return e;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kWave * waves), lds, s, p, static_cast<int>(hold), static_cast<int>(tokens), row_units, per);
        return hipGetLastError();
    };
    auto by_waves = [&](auto w) {
        constexpr int W = decltype(w)::value, E = kPagedMaxDim / kWave;
        if (hd == 128 && al) return p.kv.i8 ? go(paged_prep_kernel<W, 2, true, true>) : go(paged_prep_kernel<W, 2, true, false>);
        if (hd == 256 && al) return p.kv.i8 ? go(paged_prep_kernel<W, 4, true, true>) : go(paged_prep_kernel<W, 4, true, false>);
        return p.kv.i8 ? go(paged_prep_kernel<W, E, false, true>) : go(paged_prep_kernel<W, E, false, false>);
    };
    return waves == 16 ? by_waves(std::integral_constant<int, 16>{}) : by_waves(std::integral_constant<int, 8>{});
}

// ---------------------------------------------------------------------------
// Positions read back, a block per sequence, 16 positions in a row of a page, kv
// head, and k or v: four 16-byte pieces in flight in a thread (3.9 to 5.8 us: a launch
// and three loads that wait for each other).
// ---------------------------------------------------------------------------
constexpr int kReadRows = 16, kReadThreads = 128;
template <typename T>
__device__ __forceinline__ T paged_value(float x, float scale) {
    float y = x * scale;
    asm("" : "+v"(y));  // the fp32 product is a value of its own (else it is rounded to fp16 without it)
    return static_cast<T>(y);
}

template <typename T, bool I8, bool VEC>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(PagedReadLaunch p) {
    constexpr int N = I8 ? 16 : 8;
    typedef typename std::conditional<I8, int8_t, _Float16>::type V;
    typedef V piece __attribute__((ext_vector_type(N)));
    const int s = blockIdx.z, hd = p.kv.head_dim, nkv = p.kv.nkv, h = blockIdx.x >> 1;
    const bool is_v = blockIdx.x & 1;
    T* out = static_cast<T*>(is_v ? p.v_out : p.k_out);
    if (!out) return;
    const SeqRows sr = seq_rows(p.step, s);
    // rows [j0, j1) of the sequence lie in one group of 16 positions; without a position they are grouped from the first
    const int past = max(sr.past, 0);
    const int64_t g0 = (static_cast<int64_t>(past / kReadRows) + blockIdx.y) * kReadRows;
    const int j0 = static_cast<int>(max(g0 - past, int64_t(0))), j1 = static_cast<int>(min(g0 + kReadRows - past, static_cast<int64_t>(sr.rows)));
    if (j0 >= j1) return;
    const int page = sr.past < 0 || g0 >= table_positions(p.step, p.kv) ? -1 : page_at(p.step, p.kv, s, static_cast<int>(g0) / p.kv.page);
    const size_t width = static_cast<size_t>(nkv) * hd;
    T* rows = out + static_cast<size_t>(sr.row0 + j0) * width + h * hd;
    const int n = j1 - j0;
    if (page < 0) {
        for (int i = threadIdx.x; i < n * hd; i += kReadThreads) rows[i / hd * width + i % hd] = static_cast<T>(0.0f);
        return;
    }
    const int t0 = static_cast<int>(g0 % p.kv.page) + (past + j0 - static_cast<int>(g0));  // position of row j0 in the page
    const V* pool = static_cast<const V*>(is_v ? p.kv.v : p.kv.k) + page_head(p.kv, page, h);
    const float f = I8 ? (is_v ? p.kv.v_scale : p.kv.k_scale)[static_cast<size_t>(page) * nkv + h] : 1.0f;
    constexpr int kBatch = 4;  // loads of a thread that go out together
    if (is_v) {                // a thread has a dim's positions
        const int b0 = t0 / N, blocks = (t0 + n - 1) / N + 1 - b0;
        for (int i0 = threadIdx.x; i0 < blocks * hd; i0 += kBatch * kReadThreads) {
            piece x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u)  // (behind the last: the last again)
                x[u] = *reinterpret_cast<const piece*>(pool + (static_cast<size_t>(b0) * hd + min(i0 + u * kReadThreads, blocks * hd - 1)) * N);
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kReadThreads, b = i / hd, dim = i - b * hd;
                if (b >= blocks) break;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int j = (b0 + b) * N + e - t0;
                    if (j >= 0 && j < n) rows[j * width + dim] = paged_value<T>(static_cast<float>(x[u][e]), f);
                }
            }
        }
    } else {  // 16 bytes of a position's output
        constexpr int M = 16 / sizeof(T), kParts = N / M;
        typedef V part __attribute__((ext_vector_type(M)));
        typedef T quad __attribute__((ext_vector_type(M)));
        const int per = hd / M;
        for (int i0 = threadIdx.x; i0 < n * per; i0 += kBatch * kReadThreads) {
            part x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = min(i0 + u * kReadThreads, n * per - 1), j = i / per, q = i - j * per;
                x[u] = *reinterpret_cast<const part*>(pool + (static_cast<size_t>(q / kParts) * p.kv.page + t0 + j) * N + q % kParts * M);
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kReadThreads, j = i / per, q = i - j * per;
                if (j >= n) break;
                T* at = rows + j * width + q * M;
                quad y;
#pragma unroll
                for (int e = 0; e < M; ++e) y[e] = paged_value<T>(static_cast<float>(x[u][e]), f);
                if constexpr (VEC)
                    *reinterpret_cast<quad*>(at) = y;
                else
#pragma unroll
                    for (int e = 0; e < M; ++e) at[e] = y[e];
            }
        }
    }
}

hipError_t launch_paged_read(const PagedReadLaunch& p, hipStream_t s) {
    const dim3 grid(2 * p.kv.nkv, (p.step.max_rows + kReadRows - 2) / kReadRows + 1, p.step.seqs);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kReadThreads), 0, s, p); };
    auto by_type = [&](auto vec) {
        constexpr bool VEC = decltype(vec)::value;
        if (p.kv.i8)
            p.f16 ? go(paged_read_kernel<_Float16, true, VEC>) : go(paged_read_kernel<float, true, VEC>);
        else
            p.f16 ? go(paged_read_kernel<_Float16, false, VEC>) : go(paged_read_kernel<float, false, VEC>);
    };
    (reinterpret_cast<uintptr_t>(p.k_out) & 15u) == 0 ? by_type(std::true_type{}) : by_type(std::false_type{});
    return hipGetLastError();
}

}  // namespace xqhip
