// paged_append.cuh -- appending keys and values to the paged 8-bit cache, the
// position rotation applied on the way (keys into the cache, queries into
// their own rows).
//
// The rows of one sequence that fall into one page are a segment: with m =
// max |x| over a segment's rows of a head (keys after rotation), the page's
// scale becomes max(old, m / 127) (or / 448), old counting only when the page
// already holds earlier positions; x is stored as rne(x / scale), and where
// the scale grew the earlier codes become rne(code * (old / new)).  A
// segment's rows are read once and kept in registers between the maximum and
// the codes.
//
// A segment's rows of one head's keys or values are a task.  With few rows a
// call (a decode step, drafts to verify) a task is a warp's, blocks behind
// the tasks' rotate the queries, and one launch does it all.  With many rows
// (prompts) a team of threads takes a task, 16 elements a thread, and goes
// through several heads of the segment with one read of its rotation table's
// entries, which are twice the size of a head's BF16 values; the next
// head's rows are on their way while this one's are encoded.
//
// A step is bound by its chain of loads (length, page, scale; rows): 64
// sequences x 1 row 3.4 us, of which a launch is 2.4.  Prompts are bound by
// instructions, 33 for each value appended to FP8 codes (with its rotation),
// next to HBM for the queries: a 6,544-row page, FP32, 21.4 us (4.1 TB/s; 28.5
// with the queries in a launch of their own); 24 ragged prompts of 49,000 rows,
// 8 heads of 128 and 32 of queries, BF16, 270 us (4.3 TB/s; the queries' launch
// alone, profiled, 134 us at 6.0).  A thread for each 16 values keeps them
// between the maximum and the codes; at the 64 registers that this leaves, every
// variant spills some (172 to 322 bytes of stores), which is part of those
// instructions.  Before heads shared a read of the
// rotation's table, and with a division for each code, the prompts took 505 us.
//
// With AXES (paged_append_axes.cu) a row's pairs have positions on several axes;
// the variants without are unchanged by it.  The 6,544-row page on three: 22.7 us.
#pragma once

#include "paged_rope.cuh"

#include <algorithm>

namespace fo {

constexpr int APPEND_FEW_THREADS = 256;
constexpr int APPEND_FEW_ROWS = 8;  // rows that a warp's task holds in registers

// A row's entries of the rotation's table: NaN outside it.
template <bool AXES>
struct RowEntries {
    const float2 *entries = nullptr;
    bool inside = true;
    AxisEntries on_axes;
    __device__ __forceinline__ void find(const fo_append_launch &a, int64_t row, int64_t position, bool first) {
        if constexpr (AXES) {
            if (!on_axes.read(a.axes, a.rope.positions, row) && first) atomicOr(a.err, FO_DEVERR_POSITION);
        } else {
            const int64_t p = a.rope.row_positions ? (int64_t)a.rope.row_positions[row] : position;
            inside = p >= 0 && p < a.rope.positions;
            if (!inside && first) atomicOr(a.err, FO_DEVERR_POSITION);
            entries = reinterpret_cast<const float2 *>(a.rope.table) + (inside ? p : 0) * (a.rope.rot_dim / 2);
        }
    }
    __device__ __forceinline__ float2 operator()(const fo_append_launch &a, int pair) const {
        if constexpr (AXES) return on_axes.entry(a.axes, a.rope, pair);
        else return inside ? load_entry(entries + pair) : make_float2(NAN, NAN);
    }
};

// Eight elements d .. d + 7 of a row, rotated when `rotate` is set.
template <typename T, bool VEC, bool AXES>
__device__ __forceinline__ void append_load(const fo_append_launch &a, const T *x, int d, const RowEntries<AXES> &entries,
                                            bool rotate, float *y) {
    float u[8];
    auto load = [&](int at, float *to) {
        if constexpr (VEC) {
            load8(x + at, to);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) to[e] = load1(x + at + e);
        }
    };
    load(d, u);
    const int rot = a.rope.rot_dim, h2 = rot / 2;
    if (!rotate || d >= rot) {
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = u[e];
        return;
    }
    auto entry = [&](int pair) { return entries(a, pair); };
    if (a.rope.layout == FO_ROPE_INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const bool turn = d + e < rot;
            const float2 cs = turn ? entry((d + e) / 2) : make_float2(1.0f, 0.0f);
            y[e] = turn ? rot_first(u[e], u[e + 1], cs) : u[e];
            y[e + 1] = turn ? rot_second(u[e], u[e + 1], cs) : u[e + 1];
        }
    } else if (h2 % 8 == 0) {
        // All eight are a pair's first elements, or all its second ones.
        float v[8];
        const bool first = d < h2;
        load(first ? d + h2 : d - h2, v);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float2 cs = entry(first ? d + e : d + e - h2);
            y[e] = first ? rot_first(u[e], v[e], cs) : rot_second(v[e], u[e], cs);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = d + e;
            y[e] = u[e];
            if (i < h2) y[e] = rot_first(u[e], load1(x + i + h2), entry(i));
            else if (i < rot) y[e] = rot_second(load1(x + i - h2), u[e], entry(i - h2));
        }
    }
}

// A segment: sequence `seq`'s rows in its j-th touched page.  (Positions and rows
// are below 2^31, pages a power of two: 64-bit divisions are kept out.  Segments
// are numbered with some to spare, whose pages may begin beyond 2^31.)
struct Segment {
    int seq, page, row0, p0;  // the sequence's page number, its first row here and that one's position
    int rows, begin;          // rows (none: nothing to do) and where in the page they begin
};
__device__ __forceinline__ Segment segment_at(const fo_append_launch &a, int seq, int j) {
    const int page = a.kv.page_size, shift = 31 - __clz(page);
    const Sequence s = load_sequence(a.batch, page, seq, a.err);
    const int len = s.len, from = max(len - s.n, 0);  // first position that is stored
    Segment g;
    g.seq = seq;
    g.page = (from >> shift) + j;
    const int64_t begins = (int64_t)g.page << shift;
    g.p0 = max(from, (int)min64(len, begins));
    const int p1 = (int)min64(len, begins + page);
    g.rows = s.n > 0 && p1 > g.p0 ? p1 - g.p0 : 0;
    g.begin = g.p0 & (page - 1);
    g.row0 = s.first + (g.p0 - (len - s.n));
    return g;
}

// A task's part of the pool.
struct Tile {
    uint8_t *codes;
    float *scale;
    bool valid;
};
template <int D>
__device__ __forceinline__ Tile tile_of(const fo_append_launch &a, const Segment &s, int head, bool value) {
    Tile t;
    const int64_t id = page_of(a.batch, a.kv.n_pages, s.seq, s.page, a.err, t.valid) * a.kv.n_kv_heads + head;
    t.scale = (value ? a.kv.v_scales : a.kv.k_scales) + id;
    t.codes = static_cast<uint8_t *>(value ? a.kv.v_codes : a.kv.k_codes) + id * a.kv.page_size * D;
    return t;
}

// The page's earlier codes, `begin` positions of them, against a larger scale.
template <int D, int FORMAT>
__device__ __forceinline__ void encode_again(uint8_t *codes, int begin, float ratio, int t, int threads) {
    uint4 *held = reinterpret_cast<uint4 *>(codes);
    for (int i = t; i < begin * (D / 16); i += threads) {
        uint4 w = held[i];
        uint32_t *ws = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float f[4];
            decode4<FORMAT>(ws[q], f);
            ws[q] = encode4<FORMAT>(__fmul_rn(f[0], ratio), __fmul_rn(f[1], ratio), __fmul_rn(f[2], ratio),
                                    __fmul_rn(f[3], ratio));
        }
        held[i] = w;
    }
}

// The largest finite magnitude of N values and `m`; `odd` if one is not finite.
template <int N>
__device__ __forceinline__ void note(const float *x, float &m, bool &odd) {
    float top = m, zero = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) {
        top = fmaxf(top, fabsf(x[e]));
        zero = fmaf(x[e], 0.0f, zero);  // NaN from a value that is not finite
    }
    if (zero != zero) {
        odd = true;
        top = m;
#pragma unroll
        for (int e = 0; e < N; e++)
            if (fabsf(x[e]) <= FLT_MAX) top = fmaxf(top, fabsf(x[e]));
    }
    m = top;
}

// A task of few rows by a warp.
template <int D, typename T, int FORMAT, bool VEC, bool AXES>
__device__ __forceinline__ void append_few(const fo_append_launch &a, const Segment &s, int head, bool value, int t) {
    constexpr int GROUPS = D / 8;            // groups of eight in a row
    constexpr int ROWS_STEP = 32 / GROUPS;   // rows a step covers
    constexpr int MAXIT = APPEND_FEW_ROWS / ROWS_STEP;
    const fo_rows &src = value ? a.v : a.k;
    const int d = (t % GROUPS) * 8, r0 = t / GROUPS;
    const bool rotate = a.rotate && !value;
    float x[MAXIT][8];
    float m = 0.0f;
    bool odd = false;  // a value that is not finite
#pragma unroll
    for (int it = 0; it < MAXIT; it++) {
        const int r = r0 + it * ROWS_STEP;
        if (r >= s.rows) continue;
        const T *xr = static_cast<const T *>(src.data) + (s.row0 + r) * src.row_stride + head * src.head_stride;
        RowEntries<AXES> entries;
        if (rotate) entries.find(a, s.row0 + r, s.p0 + r, d == 0);
        append_load<T, VEC, AXES>(a, xr, d, entries, rotate, x[it]);
        note<8>(x[it], m, odd);
    }
    // The page, looked up while the rows are on their way.
    const Tile tile = tile_of<D>(a, s, head, value);
    const float old = s.begin > 0 ? *tile.scale : 0.0f;
    m = warp_max(m);
    if (odd) atomicOr(a.err, FO_DEVERR_VALUE);
    if (!tile.valid) return;
    const float scale = fmaxf(old, __fdiv_rn(m, code_max(FORMAT)));
    if (scale > old && s.begin > 0) encode_again<D, FORMAT>(tile.codes, s.begin, __fdiv_rn(old, scale), t, 32);
    if (t == 0) *tile.scale = scale;
    const bool normal = scale >= 1e-30f;
    const float inverse = normal ? __frcp_rn(scale) : 0.0f;
#pragma unroll
    for (int it = 0; it < MAXIT; it++) {
        const int r = r0 + it * ROWS_STEP;
        if (r >= s.rows) continue;
        *reinterpret_cast<uint2 *>(tile.codes + (s.begin + r) * D + d) =
            encode8<FORMAT>(x[it], scale, inverse, odd || !normal);
    }
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

// Rows that may touch this many pages of a sequence.
__host__ __device__ inline int64_t segments_of(int64_t rows, int64_t page) {
    return rows <= 0 ? 0 : (rows + page - 2) / page + 1;
}

// The rotation of the queries: a row's position is its place in the cache
// unless positions are given; a row without such a place (a padded slot's, or of
// no sequence) is copied.
__device__ __forceinline__ int64_t position_of_row(const fo_append_launch &a, int64_t row, bool &padded) {
    padded = false;
    if (a.rope.row_positions) return (int64_t)a.rope.row_positions[row];
    const int seq = a.batch.row_start ? sequence_of_row(a.batch, (int)row) : (int)((unsigned)row / (unsigned)a.batch.max_rows);
    const Sequence s = load_sequence(a.batch, a.kv.page_size, seq, a.err);
    const int r = (int)row - s.first, p = s.len - s.n + r;
    padded = r < 0 || r >= s.n || p < 0;
    return padded ? -1 : p;
}
template <typename T, bool AXES>
__device__ __forceinline__ void rotate_queries(const fo_append_launch &a, int64_t block, bool half, bool vec) {
    auto position = [&](int64_t row, bool &padded) { return position_of_row(a, row, padded); };
    const int t = threadIdx.x;
    if (half)
        vec ? rope_block<T, true, true, AXES>(a.q, block, t, position)
            : rope_block<T, true, false, AXES>(a.q, block, t, position);
    else
        vec ? rope_block<T, false, true, AXES>(a.q, block, t, position)
            : rope_block<T, false, false, AXES>(a.q, block, t, position);
}

template <typename T, bool AXES>
__global__ void __launch_bounds__(ROPE_THREADS, 3) paged_rope_kernel(const __grid_constant__ fo_append_launch a, bool half,
                                                                     bool vec) {
    wait_for_prior_kernel();
    rotate_queries<T, AXES>(a, blockIdx.x, half, vec);
}

// Few rows a sequence: as many segments for each sequence as it can touch.
template <int D, typename T, int FORMAT, bool VEC, bool AXES>
__global__ void __launch_bounds__(APPEND_FEW_THREADS, 3)
    append_few_kernel(const __grid_constant__ fo_append_launch a, unsigned task_blocks, unsigned per_seq, bool q_half,
                      bool q_vec) {
    wait_for_prior_kernel();
    if (blockIdx.x >= task_blocks) {
        rotate_queries<T, AXES>(a, blockIdx.x - task_blocks, q_half, q_vec);
        return;
    }
    const unsigned heads2 = 2 * a.kv.n_kv_heads;
    const unsigned task = blockIdx.x * (APPEND_FEW_THREADS / 32) + (threadIdx.x >> 5), segment = task / heads2;
    const unsigned part = task - segment * heads2, seq = segment / per_seq;
    if (seq >= a.batch.n_seqs) return;
    const Segment s = segment_at(a, (int)seq, (int)(segment - seq * per_seq));
    if (s.rows > 0) append_few<D, T, FORMAT, VEC, AXES>(a, s, part >> 1, part & 1, threadIdx.x & 31);
}

// Many rows.  A block takes `heads` heads of a segment's keys or values, a team
// of page_size * D / 16 threads a head at a time.  A thread's 16 elements are
// two groups of eight: neighbours, or in the half layout the two elements of
// eight pairs (when rot_dim / 2 is a multiple of eight; LINED_UP is false for
// other half layouts).
// Segments are numbered per sequence; when row counts differ, sequence b's
// start at row_start[b] / page + 2 b, which leaves each at least rows / page +
// 2 numbers, enough for what it can touch, in total_rows / page + 2 n_seqs.
template <int D, typename T, int FORMAT, bool VEC, bool AXES, bool LINED_UP>
__global__ void __launch_bounds__(D == 64 ? 512 : 1024, D == 64 ? 2 : 1) append_many_kernel(
    const __grid_constant__ fo_append_launch a, unsigned task_blocks, unsigned per_seq, int heads, bool q_half, bool q_vec) {
    __shared__ float red[2][32];
    wait_for_prior_kernel();
    if (blockIdx.x >= task_blocks) {
        rotate_queries<T, AXES>(a, blockIdx.x - task_blocks, q_half, q_vec);
        return;
    }
    const int page = a.kv.page_size, n_heads = a.kv.n_kv_heads;
    const int chunks = (n_heads + heads - 1) / heads;
    const unsigned segment = blockIdx.x / (2 * chunks);
    const int part = (int)(blockIdx.x - segment * 2 * chunks);
    const bool value = part >= chunks;
    const int head0 = (part - (value ? chunks : 0)) * heads, head1 = min(head0 + heads, n_heads);
    int seq, j;
    if (per_seq > 0) {
        seq = (int)(segment / per_seq);
        j = (int)(segment - seq * per_seq);
    } else {
        const int shift = 31 - __clz(page);
        int lo = 0, hi = (int)a.batch.n_seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((a.batch.row_start[mid] >> shift) + 2 * mid <= (int)segment) lo = mid;
            else hi = mid - 1;
        }
        seq = lo;
        j = (int)segment - ((a.batch.row_start[seq] >> shift) + 2 * seq);
        if (j < 0) return;  // row_start out of order (the sequence's own check reports it)
    }
    const Segment s = segment_at(a, seq, j);
    if (s.rows == 0) return;
    const int team_shift = 31 - __clz(page * (D / 16)), team_size = 1 << team_shift, teams = blockDim.x >> team_shift;
    const int team = threadIdx.x >> team_shift, t = threadIdx.x & (team_size - 1);
    const int r = t / (D / 16), slot = t % (D / 16);
    const bool mine = r < s.rows;
    const fo_rows &src = value ? a.v : a.k;
    const bool rotate = a.rotate && !value;
    const int rot = a.rope.rot_dim, h2 = rot / 2;
    const bool half = rotate && a.rope.layout == FO_ROPE_HALF;
    const bool pair = LINED_UP && half && slot < rot / 16;
    const int d0 = pair ? 8 * slot : 16 * slot, d1 = pair ? d0 + h2 : d0 + 8;
    const T *row = static_cast<const T *>(src.data) + (s.row0 + (mine ? r : 0)) * src.row_stride;
    auto load = [&](int head, Raw8<T> (&to)[2]) {
        const T *x = row + head * src.head_stride;
        if constexpr (VEC) {
            to[0] = load_raw8(x + d0);
            to[1] = load_raw8(x + d1);
        } else {
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int e = 0; e < 8; e++) reinterpret_cast<T *>(to[g].w)[e] = x[(g ? d1 : d0) + e];
        }
    };
    // The next head's rows are asked for while there are registers for them.
    constexpr bool AHEAD = sizeof(T) == 2;
    Raw8<T> now[2], next[2];
    const int rounds = (heads + teams - 1) >> (31 - __clz(teams));
    if (AHEAD && mine && head0 + team < head1) load(head0 + team, now);
    RowEntries<AXES> entries;
    if (rotate && mine) entries.find(a, s.row0 + r, s.p0 + r, slot == 0);
    // Entries of the eight pairs, the same for every head: of (d0 + e, d1 + e), or
    // of (d0 + 2 e, d0 + 2 e + 1).
    float2 cs[8];
    const bool turned = rotate && mine && (!half || pair) && d0 < rot;
    if (turned) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const bool turn = pair || d0 + 2 * e < rot;
            cs[e] = turn ? entries(a, pair ? d0 + e : d0 / 2 + e) : make_float2(1.0f, 0.0f);
        }
    }
    bool valid;
    const int64_t id = page_of(a.batch, a.kv.n_pages, s.seq, s.page, a.err, valid) * n_heads;
    float *scales = (value ? a.kv.v_scales : a.kv.k_scales) + id;
    uint8_t *codes = static_cast<uint8_t *>(value ? a.kv.v_codes : a.kv.k_codes) + id * page * D;
    for (int round = 0; round < rounds; round++) {
        const int head = head0 + round * teams + team;
        const bool live = mine && head < head1;
        if (!AHEAD && live) load(head, now);
        const float old = s.begin > 0 && valid && head < head1 ? scales[head] : 0.0f;
        if (AHEAD && mine && head + teams < head1) load(head + teams, next);
        float y[16];
        float m = 0.0f;
        bool odd = false;
        if (live) {
            unpack8(now[0], y);
            unpack8(now[1], y + 8);
            if (pair) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float u = y[e], v = y[8 + e];
                    y[e] = rot_first(u, v, cs[e]);
                    y[8 + e] = rot_second(u, v, cs[e]);
                }
            } else if (turned) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float u = y[2 * e], v = y[2 * e + 1];
                    const bool turn = d0 + 2 * e < rot;
                    y[2 * e] = turn ? rot_first(u, v, cs[e]) : u;
                    y[2 * e + 1] = turn ? rot_second(u, v, cs[e]) : v;
                }
            }
            if constexpr (!LINED_UP) {
                const T *x = row + head * src.head_stride;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int i = d0 + e, p = i < h2 ? i : i - h2;
                    if (!rotate || i >= rot) continue;
                    const float2 c = entries(a, p);
                    y[e] = i < h2 ? rot_first(y[e], load1(x + i + h2), c) : rot_second(load1(x + i - h2), y[e], c);
                }
            }
            note<16>(y, m, odd);
        }
        m = warp_max(m);
        float *box = red[round & 1];
        if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = m;
        __syncthreads();
        const int warps = team_size / 32, lane = threadIdx.x & 31;
        m = warp_max(lane < warps ? box[team * warps + lane] : 0.0f);
        if (odd) atomicOr(a.err, FO_DEVERR_VALUE);
        if (valid && head < head1) {
            const float scale = fmaxf(old, __fdiv_rn(m, code_max(FORMAT)));
            uint8_t *at = codes + (int64_t)head * page * D;
            if (scale > old && s.begin > 0) encode_again<D, FORMAT>(at, s.begin, __fdiv_rn(old, scale), t, team_size);
            if (t == 0) scales[head] = scale;
            if (live) {
                const bool normal = scale >= 1e-30f;
                const float inverse = normal ? __frcp_rn(scale) : 0.0f;
                uint8_t *to = at + (s.begin + r) * D;
                const uint2 c0 = encode8<FORMAT>(y, scale, inverse, odd || !normal);
                const uint2 c1 = encode8<FORMAT>(y + 8, scale, inverse, odd || !normal);
                if (pair) {
                    *reinterpret_cast<uint2 *>(to + d0) = c0;
                    *reinterpret_cast<uint2 *>(to + d1) = c1;
                } else {
                    *reinterpret_cast<uint4 *>(to + d0) = make_uint4(c0.x, c0.y, c1.x, c1.y);
                }
            }
        }
        if constexpr (AHEAD) {
            now[0] = next[0];
            now[1] = next[1];
        }
    }
}

template <int D, typename T, int FORMAT, bool VEC, bool AXES>
cudaError_t launch_append(const fo_append_launch &in, cudaStream_t stream) {
    fo_append_launch a = in;
    const int64_t page = a.kv.page_size, heads2 = 2 * (int64_t)a.kv.n_kv_heads;
    bool q_vec = false;
    int64_t q_blocks = 0;  // each of ROPE_THREADS threads
    if (a.q.rows > 0) {
        q_vec = rope_shape(&a.q);
        const int64_t rows = ROPE_THREADS / a.q.block_x;
        q_blocks = (a.q.rows + rows - 1) / rows;
    }
    const bool q_half = a.rope.layout == FO_ROPE_HALF;
    if (a.batch.max_rows <= APPEND_FEW_ROWS) {
        const int64_t per_seq = segments_of(a.batch.max_rows, page), per_block = APPEND_FEW_THREADS / 32;
        const int64_t task_blocks = (per_seq * a.batch.n_seqs * heads2 + per_block - 1) / per_block;
        if (task_blocks + q_blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
        return launch(append_few_kernel<D, T, FORMAT, VEC, AXES>, dim3((unsigned)(task_blocks + q_blocks)),
                      dim3(APPEND_FEW_THREADS), 0, stream, a, (unsigned)task_blocks, (unsigned)per_seq, q_half, q_vec);
    }
    const int64_t per_seq = a.batch.row_start ? 0 : segments_of(a.batch.max_rows, page);
    const int64_t segments =
        a.batch.row_start ? a.batch.total_rows / page + 2 * a.batch.n_seqs : per_seq * a.batch.n_seqs;
    // Heads a block goes through: the more, the fewer reads of the rotation
    // table; but blocks enough for every SM.
    const int team = (int)page * (D / 16), threads = std::max(team, ROPE_THREADS);
    int heads = a.kv.n_kv_heads;
    auto blocks = [&](int64_t h) { return segments * 2 * ((a.kv.n_kv_heads + h - 1) / h); };
    while (heads > threads / team && blocks(heads) < 296) heads = (heads + 1) / 2;
    // The queries' blocks go along with tasks' blocks of their own size (a 6,544-row
    // FP32 page in 64-position pages: 28.5 us apart, 23.3 together, 21.4 now); next
    // to wider ones they would run at half their occupancy (24 ragged prompts: 281 us
    // apart, 334 together, 270 apart now).
    const bool together = threads == ROPE_THREADS;
    const int64_t grid = blocks(heads) + (together ? q_blocks : 0);
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
    const bool lined_up = !a.rotate || !q_half || a.rope.rot_dim % 16 == 0;
    cudaError_t e = launch(
        lined_up ? append_many_kernel<D, T, FORMAT, VEC, AXES, true> : append_many_kernel<D, T, FORMAT, VEC, AXES, false>,
        dim3((unsigned)grid), dim3(threads), 0, stream, a, (unsigned)blocks(heads), (unsigned)per_seq, heads, q_half, q_vec);
    if (e != cudaSuccess || together || q_blocks == 0) return e;
    return launch(paged_rope_kernel<T, AXES>, dim3((unsigned)q_blocks), dim3(ROPE_THREADS), 0, stream, a, q_half, q_vec);
}

template <int D, typename T, int FORMAT, bool AXES>
cudaError_t launch_append(const fo_append_launch &a, cudaStream_t stream) {
    const int64_t unit = sizeof(T) == 4 ? 4 : 8;  // elements in 16 bytes
    auto ok = [&](const fo_rows &r) {
        return (reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    return ok(a.k) && ok(a.v) ? launch_append<D, T, FORMAT, true, AXES>(a, stream)
                              : launch_append<D, T, FORMAT, false, AXES>(a, stream);
}

template <int D, typename T, bool AXES>
cudaError_t launch_append(const fo_append_launch &a, cudaStream_t stream) {
    return a.kv.format == FO_PAGED_I8 ? launch_append<D, T, FO_PAGED_I8, AXES>(a, stream)
                                      : launch_append<D, T, FO_PAGED_E4M3, AXES>(a, stream);
}

template <bool AXES>
cudaError_t launch_append(const fo_append_launch &a, cudaStream_t stream) {
    if (a.batch.total_rows <= 0) return cudaSuccess;
    const bool f32 = a.k.dtype == FO_DT_F32;
    if (a.kv.head_dim == 64)
        return f32 ? launch_append<64, float, AXES>(a, stream) : launch_append<64, uint16_t, AXES>(a, stream);
    return f32 ? launch_append<128, float, AXES>(a, stream) : launch_append<128, uint16_t, AXES>(a, stream);
}

}  // namespace fo
