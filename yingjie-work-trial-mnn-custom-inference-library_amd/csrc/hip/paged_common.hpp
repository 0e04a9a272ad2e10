// paged_common.hpp - what the kernels over paged caches share: the rows of a
// step and the pages of a sequence, every index that comes from device memory
// bounded before it is used.
#pragma once

#include "xqhip_common.hpp"
#include "xqhip_kernels.hpp"

namespace xqhip {

struct SeqRows {
    int row0, rows;  // first row of the step, rows (0: takes no part)
    int past;        // positions before the step, < 0: not a sequence
};

// rows of sequence s (wave-uniform s)
__device__ __forceinline__ SeqRows seq_rows(const PagedStep& st, int s) {
    const int a = st.row0[s], b = st.row0[s + 1], past = st.past[s];
    SeqRows r;
    r.row0 = max(0, min(a, st.rows));
    r.rows = min(max(0, max(0, min(b, st.rows)) - r.row0), st.max_rows);  // (b bounded by itself: any int32 less row0 may wrap)
    r.past = past;
    return r;
}

// The sequence that a row belongs to, by the whole wave: the sequences whose first row is not past it are counted.
// seqs: none (rows behind the last sequence).
__device__ __forceinline__ int seq_of_row(const PagedStep& st, int row) {
    const int lane = threadIdx.x & (kWave - 1);
    int n = 0;
    for (int b = 1; b <= st.seqs; b += kWave) {
        const int s = b + lane;
        n += __popcll(__builtin_amdgcn_ballot_w64(s <= st.seqs && st.row0[min(s, st.seqs)] <= row));
    }
    return n;
}

// sum over the lanes up to each, of the whole wave
__device__ __forceinline__ int wave_scan_int(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    const int a = __builtin_amdgcn_readlane(v, 15), b = a + __builtin_amdgcn_readlane(v, 31), c = b + __builtin_amdgcn_readlane(v, 47);
    const int row = (threadIdx.x & (kWave - 1)) >> 4;
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}

// positions that the table has room for
__device__ __forceinline__ int table_positions(const PagedStep& st, const PagedCache& kv) { return st.max_pages * kv.page; }

// the page of positions page * i .. of sequence s, -1: none
__device__ __forceinline__ int page_at(const PagedStep& st, const PagedCache& kv, int s, int i) {
    if (i < 0 || i >= st.max_pages) return -1;
    const int pg = st.table[static_cast<size_t>(s) * st.max_pages + i];
    return pg >= 0 && pg < kv.pages ? pg : -1;
}

// element offsets of (page, kv head, position in the page, dim) in k and v; E = elements of a 16-byte piece
__device__ __forceinline__ size_t page_head(const PagedCache& kv, int page, int h) {
    return (static_cast<size_t>(page) * kv.nkv + h) * kv.page * kv.head_dim;
}
template <int E>
__device__ __forceinline__ int k_offset(const PagedCache& kv, int pos, int dim) {
    return (dim / E * kv.page + pos) * E + dim % E;
}
template <int E>
__device__ __forceinline__ int v_offset(const PagedCache& kv, int pos, int dim) {
    return (pos / E * kv.head_dim + dim) * E + pos % E;
}

}  // namespace xqhip
