// paged_reach.cuh -- what a row of a paged attention sees when that is more
// than "its sequence's newest positions": groups of sequences that share their
// beginnings, and rows that are joined from two attentions over different
// positions.  Device helpers of paged_tiles.cu and paged_few.cu.
#pragma once

#include "paged.cuh"

namespace fo {

// The group that sequence `seq` belongs to; -1: none.
__device__ __forceinline__ int group_of(const fo_paged_reach &r, int seq) {
    if (r.n_groups == 0 || seq < r.group_start[0] || seq >= r.group_start[r.n_groups]) return -1;
    int lo = 0, hi = r.n_groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (r.group_start[mid] <= seq) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Positions that a sequence shares (those of its table at most), and the
// sequence whose pages hold them.
struct Shared {
    int len, leader;
};
__device__ __forceinline__ Shared shared_of(const fo_paged_reach &r, const fo_paged_batch &b, int page_size, int seq,
                                            unsigned *err) {
    const int g = group_of(r, seq);
    if (g < 0) return {0, seq};
    const int len = r.group_lens[g], leader = r.group_start[g];
    if (len < 0 || len > (int)b.table_stride * page_size || leader < 0 || leader >= (int)b.n_seqs) {
        atomicOr(err, FO_DEVERR_PAGED);
        return {0, seq};
    }
    return {len, leader};
}

// A group as a sequence of its own: all rows of its sequences, over the shared
// positions.  Number 0 stands for the sequences before the first group and
// n_groups + 1 for those behind the last, which share nothing.
struct Group {
    int first, n;  // rows
    int len;       // shared positions
    int leader;    // the sequence whose pages hold them
};
__device__ __forceinline__ Group load_group(const fo_paged_reach &r, const fo_paged_batch &b, int page_size, int number,
                                            unsigned *err) {
    const int g = number - 1, last = (int)b.n_seqs;
    const int b0 = g < 0 ? 0 : r.group_start[g], b1 = g < r.n_groups ? r.group_start[g + 1] : last;
    Group x = {0, 0, 0, b0};
    if (b0 < 0 || b1 < b0 || b1 > last) {
        atomicOr(err, FO_DEVERR_PAGED);
        x.leader = 0;
        return x;
    }
    if (b0 == b1) {
        x.leader = 0;
        return x;
    }
    const int r0 = b.row_start ? b.row_start[b0] : b0 * (int)b.max_rows;
    const int r1 = b.row_start ? b.row_start[b1] : b1 * (int)b.max_rows;
    if (r0 < 0 || r1 < r0 || r1 > (int)b.total_rows) {
        atomicOr(err, FO_DEVERR_PAGED);
        return x;
    }
    x.first = r0;
    x.n = r1 - r0;
    if (g < 0 || g >= r.n_groups) return x;
    x.len = r.group_lens[g];
    if (x.len < 0 || x.len > (int)b.table_stride * page_size) {
        atomicOr(err, FO_DEVERR_PAGED);
        x.len = 0;
    }
    return x;
}

// Sequence of a row when the sequences' row counts differ: the last one that
// starts at or before it.
__device__ __forceinline__ int sequence_of_row(const fo_paged_batch &b, int row) {
    int lo = 0, hi = (int)b.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.row_start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A row's position in its sequence; -1: it has none.
__device__ __forceinline__ int place_of_row(const fo_paged_batch &b, int page_size, int row, unsigned *err) {
    const int seq = b.row_start ? sequence_of_row(b, row) : (int)((unsigned)row / (unsigned)b.max_rows);
    const Sequence s = load_sequence(b, page_size, seq, err);
    const int r = row - s.first, p = s.len - s.n + r;
    return r < 0 || r >= s.n || p < 0 ? -1 : p;
}

constexpr float REACH_LOG2E = 1.4426950408889634f, REACH_LN2 = 0.6931471805599453f;

// A row's two unfinished parts: {maximum, sum} and the factors that bring each
// one's sums to the common maximum.
struct Joined {
    float m, l, f0, f1;
};
__device__ __forceinline__ Joined join_parts(float m0, float l0, float m1, float l1) {
    Joined j;
    j.m = fmaxf(m0, m1);
    const float shift = j.m == -INFINITY ? 0.0f : j.m;
    // (exp2 of a difference of at most 0, on the special function unit: within 2^-22.)
    j.f0 = exp2f(m0 - shift);
    j.f1 = exp2f(m1 - shift);
    j.l = l0 * j.f0 + l1 * j.f1;
    return j;
}
// 1 / (sum + the sink's term), 0 for a row that has seen nothing.
__device__ __forceinline__ float inverse_sum(float sink, float m, float l) {
    return l == 0.0f ? 0.0f : 1.0f / (l + exp2f(fmaf(sink, REACH_LOG2E, -m)));
}
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.0f ? -INFINITY : (m + log2f(l)) * REACH_LN2;
}

}  // namespace fo
