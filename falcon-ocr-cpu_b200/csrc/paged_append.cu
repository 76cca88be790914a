// paged_append.cu -- appending keys and values to the paged 8-bit cache, the
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
// One task is (segment, KV head, keys | values).  A task of few rows is one
// warp's; of many rows (a prompt's), a whole block's.  Blocks behind the
// tasks rotate the queries.
#include "paged_rope.cuh"

#include <algorithm>

namespace fo {

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_FEW_ROWS = 8;  // rows that a warp's task holds in registers

// Maximum over a task's threads, a warp or the block.
template <int THREADS>
__device__ __forceinline__ float task_max(float m, float *red) {
    m = warp_max(m);
    if constexpr (THREADS > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        m = red[0];
#pragma unroll
        for (int w = 1; w < THREADS / 32; w++) m = fmaxf(m, red[w]);
    }
    return m;
}

// Eight elements d .. d + 7 of a row, rotated when `rotate` is set.
template <typename T, bool VEC>
__device__ __forceinline__ void append_load(const fo_append_launch &a, const T *x, int d, const float2 *entries,
                                            bool inside, bool rotate, float *y) {
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
    auto entry = [&](int pair) { return inside ? __ldg(entries + pair) : make_float2(NAN, NAN); };
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

// The segment of sequence `seq` in its j-th touched page, for KV head `head`
// of the keys or the values, by THREADS threads (t of them): MAXIT groups of
// eight elements each.
template <int D, typename T, int FORMAT, bool VEC, int THREADS, int MAXIT>
__device__ __forceinline__ void append_segment(const fo_append_launch &a, int64_t seq, int64_t j, int head, bool value,
                                               int t, float *red) {
    constexpr int GROUPS = D / 8;               // groups of eight in a row
    constexpr int ROWS_STEP = THREADS / GROUPS;  // rows a step covers
    const int page = a.kv.page_size;
    const Sequence s = load_sequence(a.batch, page, seq, a.err);
    const int64_t from = max64(s.len - s.n, 0);  // first position that is stored
    const int64_t pg = from / page + j;
    const int64_t p0 = max64(from, pg * page), p1 = min64(s.len, (pg + 1) * page);
    if (s.n == 0 || p0 >= p1) return;
    bool valid;
    const int64_t id = page_of(a.batch, a.kv.n_pages, seq, pg, a.err, valid);
    if (!valid) return;
    const int rows = (int)(p1 - p0), begin = (int)(p0 - pg * page);
    const int64_t row0 = s.first + (p0 - (s.len - s.n));
    const fo_rows &src = value ? a.v : a.k;
    const int64_t tile = id * a.kv.n_kv_heads + head;
    float *scale_at = (value ? a.kv.v_scales : a.kv.k_scales) + tile;
    uint8_t *codes = static_cast<uint8_t *>(value ? a.kv.v_codes : a.kv.k_codes) + tile * page * D;
    const float old = begin > 0 ? *scale_at : 0.0f;
    const int d = (t % GROUPS) * 8, r0 = t / GROUPS;
    const bool rotate = a.rotate && !value;
    float x[MAXIT][8];
    float m = 0.0f;
    bool odd = false;  // a value that is not finite
#pragma unroll
    for (int it = 0; it < MAXIT; it++) {
        const int r = r0 + it * ROWS_STEP;
        if (r >= rows) continue;
        const T *xr = static_cast<const T *>(src.data) + (row0 + r) * src.row_stride + head * src.head_stride;
        const float2 *entries = nullptr;
        bool inside = true;
        if (rotate) {
            const int64_t p = a.rope.row_positions ? (int64_t)__ldg(a.rope.row_positions + row0 + r) : p0 + r;
            inside = p >= 0 && p < a.rope.positions;
            if (!inside && d == 0) atomicOr(a.err, FO_DEVERR_POSITION);
            entries = reinterpret_cast<const float2 *>(a.rope.table) + (inside ? p : 0) * (a.rope.rot_dim / 2);
        }
        append_load<T, VEC>(a, xr, d, entries, inside, rotate, x[it]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = fabsf(x[it][e]);
            if (y <= FLT_MAX) m = fmaxf(m, y);
            else odd = true;
        }
    }
    m = task_max<THREADS>(m, red);
    if (odd) atomicOr(a.err, FO_DEVERR_VALUE);
    const float top = code_max(FORMAT);
    const float scale = fmaxf(old, __fdiv_rn(m, top));
    if (scale > old && begin > 0) {
        // The page's earlier codes against the larger scale.
        const float ratio = __fdiv_rn(old, scale);
        uint4 *held = reinterpret_cast<uint4 *>(codes);
        for (int i = t; i < begin * (D / 16); i += THREADS) {
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
    if (t == 0) *scale_at = scale;
#pragma unroll
    for (int it = 0; it < MAXIT; it++) {
        const int r = r0 + it * ROWS_STEP;
        if (r >= rows) continue;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = scaled(x[it][e], scale, top);
        const uint2 w = make_uint2(encode4<FORMAT>(y[0], y[1], y[2], y[3]), encode4<FORMAT>(y[4], y[5], y[6], y[7]));
        *reinterpret_cast<uint2 *>(codes + (begin + r) * D + d) = w;
    }
}

// Sequence of a row when the sequences' row counts differ: the last one that
// starts at or before it.
__device__ __forceinline__ int64_t sequence_of_row(const fo_paged_batch &b, int64_t row) {
    int64_t lo = 0, hi = b.n_seqs - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (__ldg(b.row_start + mid) <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Rows that may touch this many pages of a sequence.
__host__ __device__ inline int64_t segments_of(int64_t rows, int64_t page) {
    return rows <= 0 ? 0 : (rows + page - 2) / page + 1;
}

// Segments are numbered per sequence; when row counts differ and are large,
// sequence b's start at row_start[b] / page + 2 b, which leaves each at least
// rows / page + 2 numbers, enough for what it can touch, in total_rows / page
// + 2 n_seqs of them.
template <int D, typename T, int FORMAT, bool VEC, bool FEW>
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(const __grid_constant__ fo_append_launch a,
                                                                      int64_t task_blocks, int64_t segments,
                                                                      int64_t per_seq, bool q_half, bool q_vec) {
    __shared__ float red[APPEND_THREADS / 32];
    const int64_t page = a.kv.page_size;
    if (blockIdx.x >= task_blocks) {
        auto position = [&](int64_t row, bool &padded) {
            padded = false;
            if (a.rope.row_positions) return (int64_t)__ldg(a.rope.row_positions + row);
            const int64_t seq = a.batch.row_start ? sequence_of_row(a.batch, row) : row / a.batch.max_rows;
            const Sequence s = load_sequence(a.batch, (int)page, seq, a.err);
            const int64_t p = s.len - s.n + (row - s.first);
            padded = p < 0;
            return p;
        };
        const int64_t block = blockIdx.x - task_blocks;
        if (q_half) q_vec ? rope_block<T, true, true>(a.q, block, position) : rope_block<T, true, false>(a.q, block, position);
        else q_vec ? rope_block<T, false, true>(a.q, block, position) : rope_block<T, false, false>(a.q, block, position);
        return;
    }
    const int64_t heads2 = 2 * (int64_t)a.kv.n_kv_heads;
    const int64_t task = FEW ? blockIdx.x * (APPEND_THREADS / 32) + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t segment = task / heads2;
    const int part = (int)(task - segment * heads2);
    if (segment >= segments) return;
    int64_t seq, j;
    if (per_seq > 0) {
        seq = segment / per_seq;
        j = segment - seq * per_seq;
    } else {
        int64_t lo = 0, hi = a.batch.n_seqs - 1;
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) >> 1;
            if (__ldg(a.batch.row_start + mid) / page + 2 * mid <= segment) lo = mid;
            else hi = mid - 1;
        }
        seq = lo;
        j = segment - (__ldg(a.batch.row_start + seq) / page + 2 * seq);
        if (j < 0) return;  // row_start out of order (the sequence's own check reports it)
    }
    const int head = part >> 1;
    const bool value = part & 1;
    if constexpr (FEW)
        append_segment<D, T, FORMAT, VEC, 32, APPEND_FEW_ROWS * (D / 8) / 32>(a, seq, j, head, value, threadIdx.x & 31,
                                                                             red);
    else
        append_segment<D, T, FORMAT, VEC, APPEND_THREADS, 128 * (D / 8) / APPEND_THREADS>(a, seq, j, head, value,
                                                                                         threadIdx.x, red);
}

template <int D, typename T, int FORMAT, bool VEC>
cudaError_t launch_append(const fo_append_launch &in, cudaStream_t stream) {
    fo_append_launch a = in;
    const int64_t page = a.kv.page_size, heads2 = 2 * (int64_t)a.kv.n_kv_heads;
    const bool few = a.batch.max_rows <= APPEND_FEW_ROWS;
    // Few rows: every sequence has as many segments as it can touch.  Many
    // rows of one number: likewise.  Many of different numbers: numbered by
    // row_start.
    const bool numbered = !few && a.batch.row_start;
    const int64_t per_seq = numbered ? 0 : segments_of(a.batch.max_rows, page);
    const int64_t segments = numbered ? a.batch.total_rows / page + 2 * a.batch.n_seqs : per_seq * a.batch.n_seqs;
    const int64_t per_block = few ? APPEND_THREADS / 32 : 1;
    const int64_t task_blocks = (segments * heads2 + per_block - 1) / per_block;
    bool q_vec = false;
    int64_t q_blocks = 0;
    if (a.q.rows > 0) {
        q_vec = rope_shape(&a.q);
        const int64_t rows = ROPE_THREADS / a.q.block_x;
        q_blocks = (a.q.rows + rows - 1) / rows;
    }
    const int64_t grid = task_blocks + q_blocks;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
    const bool q_half = a.rope.layout == FO_ROPE_HALF;
    if (few)
        paged_append_kernel<D, T, FORMAT, VEC, true><<<(unsigned)grid, APPEND_THREADS, 0, stream>>>(
            a, task_blocks, segments, per_seq, q_half, q_vec);
    else
        paged_append_kernel<D, T, FORMAT, VEC, false><<<(unsigned)grid, APPEND_THREADS, 0, stream>>>(
            a, task_blocks, segments, per_seq, q_half, q_vec);
    return cudaGetLastError();
}

template <int D, typename T, int FORMAT>
cudaError_t launch_append(const fo_append_launch &a, cudaStream_t stream) {
    const int64_t unit = sizeof(T) == 4 ? 4 : 8;  // elements in 16 bytes
    auto ok = [&](const fo_rows &r) {
        return (reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    return ok(a.k) && ok(a.v) ? launch_append<D, T, FORMAT, true>(a, stream)
                              : launch_append<D, T, FORMAT, false>(a, stream);
}

template <int D, typename T>
cudaError_t launch_append(const fo_append_launch &a, cudaStream_t stream) {
    return a.kv.format == FO_PAGED_I8 ? launch_append<D, T, FO_PAGED_I8>(a, stream)
                                      : launch_append<D, T, FO_PAGED_E4M3>(a, stream);
}

}  // namespace fo

extern "C" cudaError_t fo_launch_paged_append(const fo_append_launch *a, cudaStream_t stream) {
    static_assert(fo::APPEND_THREADS == fo::ROPE_THREADS, "the queries' blocks have the tasks' width");
    if (a->batch.total_rows <= 0) return cudaSuccess;
    const bool f32 = a->k.dtype == FO_DT_F32;
    if (a->kv.head_dim == 64) return f32 ? fo::launch_append<64, float>(*a, stream) : fo::launch_append<64, uint16_t>(*a, stream);
    return f32 ? fo::launch_append<128, float>(*a, stream) : fo::launch_append<128, uint16_t>(*a, stream);
}
