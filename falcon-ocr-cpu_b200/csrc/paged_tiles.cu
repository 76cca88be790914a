// paged_tiles.cu -- attention of many query rows of a KV head over the paged
// 8-bit cache: prompts (over a window and first positions, or all of them), and
// the shared beginning of a group of sequences, once for all their rows.
//
// For a query row q that sees positions j: s_j = scale * kscale * (q . kcode_j),
// m = max s_j, out = sum_j e^(s_j - m) vscale vcode_j / (sum_j e^(s_j - m) +
// e^(sink - m)).  With 128 query rows and more to a KV head the products bound
// the call, so they belong on the 5th-generation tensor cores, in FP16 with FP32
// sums: FP16 holds every int8 and every e4m3 code, so nothing of the cache is
// rounded; a query row is taken relative to a power of two near its largest
// element (exact for BF16's 8 bits; FP32 rows as the sum of two FP16, 22 bits);
// a probability times its page's value scale, relative to the largest scale so
// far and times 2^10, is one FP16 (11 bits) or two, down to 2^-24 of the row's
// largest at full precision.  The sum of probabilities takes them unrounded.
//
// Work is a line of tiles of 128 positions, the tiles of a unit (128 or 256
// query rows of one KV head) adjacent; each of at most one block per SM takes an
// equal piece.  A block that holds a part of a unit leaves the rows' maxima, sums
// and outputs in scratch, which a second, small launch joins (by all SMs: joined
// by one of the unit's blocks, 8 units of 18 parts would wait for eight SMs'
// share of L2).
//
// In a block:
//   warp 12      walks the line: page numbers, scales, and bulk copies of the
//                codes into a ring, 8 KB a slot; announces the segments (a unit's
//                tiles in this block) to the other warps;
//   warps 8-11   codes to FP16, into swizzled operand tiles (two of keys, two of
//                values);
//   warps 13-14  an issuer for each stream, S_t = Q_t K^T and O_t += P_t V;
//   warp 15      keeps the bound of all other warps' waits;
//   warps 0-7    two softmax warpgroups, a thread to a query row: a segment's query
//                rows to FP16 operands, S from tensor memory, scales, mask,
//                exponentials, P back to tensor memory, and at the end of a
//                segment O.
// The two warpgroups are two streams: of a unit of more than 128 query rows each
// takes 128 of them over all tiles; of a smaller one, both take the same rows over
// every other tile, and join at the end, so a few rows still keep two tiles in
// flight.
// Tensor memory (512 columns): S_t at 128 t; heads of 64 and BF16 rows: O_t at
// 256 + 64 t, P_t at 384 + 64 t; else P_t in S_t's place and O_t at 256 + 128 t.
// Every wait is bounded; on a timeout the block unwinds, waits for its own copies
// and MMAs, frees tensor memory and reports through the error word.
//
// Measured (CUDA graph): a prompt of 6,544 rows in windows of 1,024 with 64 first
// positions, 2 query heads to each of 8 KV heads of 64, int8: 106 us, 0.15 of the
// measured FP16 peak; 16 ragged prompts of up to 4,096 rows, 4 query heads to each of
// 8 of 128, windows of 2,048 with 128, e4m3: 2,366 us, 0.36; 48 questions of up to 96
// rows to 4 documents of up to 9,001, the same heads: 657 us, 0.26; FP32 rows, the
// page's prompt 150 us, the ragged ones 5,302.  Of the
// prompt, profiled: 47.1 M warp instructions, 1.8 a cycle and SM, 92 % of the
// instructions found in the instruction cache.  With heads of 128 a pair of tiles
// takes 6,000 cycles, of which the products are 2,050: a stream waits 1,850 for its S,
// finds maxima in 1,100 and takes exponentials for 2,300, and as P lies in S's place
// the next S cannot be there before P V is done.  Heads of 64 have columns for both.
// Beginning with a unit takes 9,000 to 17,000 cycles.
#include "paged_reach.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace fo {
using namespace sm100;

constexpr int PT_TILE = 128;  // positions
constexpr int PT_SOFTMAX = 8, PT_CONVERTERS = 4;
constexpr int PT_PRODUCER = PT_SOFTMAX + PT_CONVERTERS, PT_ISSUER = PT_PRODUCER + 1;  // two issuers, and a warp that idles
constexpr int PT_THREADS = 512;
// Registers a thread: launched with 128, the softmax warpgroups' two take what
// the other two give up: 256 * 184 + 256 * 72 = 512 * 128.
constexpr int PT_LAUNCH_REGS = 128, PT_SOFTMAX_REGS = 184, PT_OTHER_REGS = 72;
static_assert(256 * PT_SOFTMAX_REGS + 256 * PT_OTHER_REGS == PT_THREADS * PT_LAUNCH_REGS, "register split");
constexpr int PT_SEGS = 8;    // segments announced at a time
constexpr int PT_METAS = 16;  // tiles whose scales are held: what the code ring and the operands can be ahead by, and more
constexpr uint32_t PT_SLOT = 8192, PT_PANEL = 16384;  // a slot of codes; 128 rows of 64 FP16
// What beginning with a unit costs, in tiles: its place in the line is so much longer.
// (Queries, first scores, output: 9,000 cycles, where a tile of 256 rows takes 4,500.
// With none, the blocks of a prompt's first, short units took twice as long as
// the others.)
constexpr int PT_START = 2;

// FP32 rows: tiles after which O is taken out of tensor memory and added to by ordinary
// FP32.  The tensor core's sums are truncated: a tile's sixteen additions leave 1e-7
// less of what is there (40 sequences over 16,384 positions came out 1.4e-5 too
// small; 1.0e-6 so), which BF16 rows, at half of that and 2^-9 of rounding, do not
// notice below millions of positions.
constexpr int PT_KEEP = 4;

// Exponent bits of a power of two above x (x from 2^-116 to 2^126; what is smaller
// is taken as that, relative to which FP16 holds less of it).
constexpr int PT_LOWEST = 12;
__device__ __forceinline__ int pt_above(float x) {
    return min(max((int)(__float_as_uint(x) >> 23 & 255u) + 1, PT_LOWEST), 253);
}

// A row's maximum moves only when a score passes it by more than 2^4 (the sum of
// both rounded down, so by no more beyond 2^25 either): P stays below 2^15, FP16's
// range.
constexpr float PT_SLACK = 4.0f;

template <int D, bool F32>
struct PtShape {
    static constexpr int TERMS = 1 + F32;  // FP16 terms of a query and of a probability
    static constexpr int Q_TILES = F32 && D == 128 ? 1 : 2;
    static constexpr int QUERIES = 128 * Q_TILES;
    static constexpr bool OWN_P = D == 64 && !F32;  // P has columns of its own, else S's
    static constexpr int PANELS = D / 64;
    static constexpr uint32_t OPERAND = PANELS * PT_PANEL;  // 128 rows of D FP16
    static constexpr uint32_t Q_BYTES = Q_TILES * TERMS * OPERAND;
    static constexpr int PARTS = D / 64;  // slots of a tile's keys, or values
    static constexpr int SLOTS = D == 64 ? 6 : 3;
    static constexpr uint32_t OFF_K = Q_BYTES, OFF_V = OFF_K + 2 * OPERAND, OFF_CODES = OFF_V + 2 * OPERAND;
    static constexpr uint32_t SMEM = OFF_CODES + SLOTS * PT_SLOT + 1024;
};

// A unit's tiles in this block, and the unit.
struct PtSegment {
    int n, base;     // tiles, and the first one's number in the block
    int pair, last;  // two query tiles; the block's last segment
    int head, first, q0, nq;  // KV head; the rows' first; the unit's queries [q0, q0 + nq) of them
    int p0, end, flat;        // position of the first row; end of what is seen; rows look their positions up
    int c1;                   // the last block that has tiles of the unit
    int part;                 // scratch of an unfinished unit's part, -1: the unit is whole
};

struct alignas(8) PtMeta {  // (its scales are read in pairs)
    float ks[8], vs[8];  // keys' and values' scales of each 16 positions' page
    int top;             // exponent bits of a power of two above the values' scales
    float least, most;   // the least of the keys' scales, 0: one is not a number above 0; and the largest
    int base;            // the tile's first position
    int from, to;        // positions [from, to) that rows may see of it
    unsigned pages;      // pages that were copied
};

template <int D, bool F32>
struct PtShared {
    using Shape = PtShape<D, F32>;
    uint64_t code_full[Shape::SLOTS], code_empty[Shape::SLOTS];
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t s_full[2], p_half[2], p_full[2], o_full[2];
    uint64_t q_full[2], q_both;  // a stream's queries are there; those of the first that the second uses too
    uint64_t seg_full[PT_SEGS], seg_free[PT_SEGS];
    uint64_t meta_full[PT_METAS];
    uint64_t x_full, x_free, done, ended;
    uint64_t turn[2][4];  // the exponentials of a stream's warp are done
    PtSegment seg[PT_SEGS];
    PtMeta meta[PT_METAS];
    int k_tile[2], v_tile[2];  // the tile that the operands are, or will be, of
    float xm[2][128], xl[2][128], xt[2][128], q_scale[128];
    int2 warp_sum[PT_THREADS / 32];
    int begin_item, begin_base, first_tile, last_tile, abort;
    uint32_t tmem;
};

// Waits for `phase` of `bar`, all lanes of a warp; false when the block gives up.  The bound
// is kept by a warp that does nothing else (the last one): when no tile has come
// along for FO_WAIT_NS it raises the flag.  (A clock in every wait is 60
// instructions each, of the few thousand that stay in the instruction cache.)
__device__ __forceinline__ bool pt_wait(uint64_t *bar, uint32_t phase, volatile int *abort_flag) {
    bool ok = true;
    while (!mbar_try_wait(bar, phase) && (ok = !*abort_flag)) {}
    return __all_sync(0xffffffffu, ok);
}

// ------------------------------------------------------------------ the line
// An item of the line: a unit of query rows of a sequence, for each KV head; or a
// group, all of its units of query rows, for each KV head.
struct PtItem {
    int seq;          // whose row of the page table
    int first, n;     // rows
    int p0, end;      // position of the first row; end of what is seen
    int low, t0, tf;  // first position seen behind the first ones; its tile; tiles of the first ones, which come before
    int shared, leader;  // positions in another sequence's pages, and that sequence
    int tiles, units;
    int q0;           // the unit's first query (a sequence's)
};

template <int QUERIES>
__device__ __forceinline__ PtItem pt_item(const fo_paged_tiles_launch &a, int index) {
    PtItem x;
    x.low = x.t0 = x.tf = x.q0 = x.p0 = x.shared = x.leader = 0;
    if (a.reach.over_groups) {
        const Group g = load_group(a.reach, a.batch, a.kv.page_size, index, a.err);
        x.seq = g.leader;
        x.first = g.first;
        x.n = g.n;
        x.end = g.len;
        x.tiles = max((int)(((unsigned)g.len + PT_TILE - 1) / PT_TILE), 1);
        x.units = (int)(((unsigned)(g.n * a.group) + QUERIES - 1) / QUERIES) * a.kv.n_kv_heads;
        return x;
    }
    int unit;  // of the sequence's
    if (a.q_units) {
        x.seq = index / a.q_units;
        unit = index - x.seq * a.q_units;
    } else {
        // The last sequence that begins at or before the number.
        auto begins = [&](int seq) { return (int)((long long)a.batch.row_start[seq] * a.group / QUERIES) + seq; };
        int lo = 0, hi = (int)a.batch.n_seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (begins(mid) <= index) lo = mid;
            else hi = mid - 1;
        }
        x.seq = lo;
        unit = index - begins(lo);
    }
    const Sequence s = load_sequence(a.batch, a.kv.page_size, x.seq, a.err);
    x.first = s.first;
    x.n = s.n;
    x.p0 = s.len - s.n;
    if (unit < 0 || (long long)unit * QUERIES >= (long long)s.n * a.group || s.n * a.group <= a.reach.few) {
        x.end = x.units = 0;
        x.tiles = 1;
        return x;
    }
    x.q0 = unit * QUERIES;
    const int queries = s.n * a.group - x.q0;
    x.units = a.kv.n_kv_heads;
    const int last = (x.q0 + min(queries, QUERIES) - 1) / a.group;
    const int from = max(x.p0 + x.q0 / a.group, 0);
    x.end = min(max(x.p0 + last + 1, 0), s.len);
    int first = a.reach.first;
    if (a.reach.n_groups > 0) {
        // The tile that the shared positions end in comes twice, for each sequence's part of it.
        const Shared g = shared_of(a.reach, a.batch, a.kv.page_size, x.seq, a.err);
        x.shared = x.low = first = g.len;
        x.leader = g.leader;
    } else {
        x.low = a.window > 0 ? max(from + 1 - a.window, 0) : 0;
    }
    x.t0 = x.low / PT_TILE;
    x.tf = (int)(((unsigned)min(first, x.end) + PT_TILE - 1) / PT_TILE);
    if (x.shared == 0) x.tf = min(x.tf, x.t0);
    if (a.reach.own_only) x.tf = 0;
    const int near = x.end > x.low ? (int)(((unsigned)x.end + PT_TILE - 1) / PT_TILE) - x.t0 : 0;
    x.tiles = max(near + x.tf, 1);
    return x;
}

// Sum of x over the block's earlier threads; `all` the whole block's.
template <typename Shared_>
__device__ __forceinline__ int2 pt_scan(int2 x, Shared_ &sh, int2 &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 sum = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum.x, o), v = __shfl_up_sync(0xffffffffu, sum.y, o);
        if (lane >= o) sum.x += u, sum.y += v;
    }
    __syncthreads();  // the last scan's sums have been read
    if (lane == 31) sh.warp_sum[warp] = sum;
    __syncthreads();
    int2 before = make_int2(sum.x - x.x, sum.y - x.y);
    all = make_int2(0, 0);
#pragma unroll 1
    for (int w = 0; w < PT_THREADS / 32; w++) {
        const int2 y = sh.warp_sum[w];
        if (w < warp) before.x += y.x, before.y += y.y;
        all.x += y.x, all.y += y.y;
    }
    return before;
}

// ------------------------------------------------------------------- numbers
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t m, uint32_t n, uint32_t b_mn_major) {
    return (1u << 4) | (b_mn_major << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ uint32_t pt_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pt_sub_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Four codes as four FP16 (exact).  int8: the byte of code + 128 under 1024's
// exponent is 1024 + code + 128.
template <int FORMAT>
__device__ __forceinline__ uint2 pt_widen(uint32_t w) {
    if constexpr (FORMAT == FO_PAGED_I8) {
        const uint32_t u = w ^ 0x80808080u;
        return make_uint2(pt_sub_f16x2(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u),
                          pt_sub_f16x2(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u));
    } else {
        return make_uint2(e4m3x2_f16x2(w & 0xFFFFu), e4m3x2_f16x2(w >> 16));
    }
}

// Writes 16 dimensions of a finished row.
template <typename T>
__device__ __forceinline__ void pt_store16(T *to, const float *v, bool vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 16; i += 8) store8(to + i, v + i);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) store1(to + i, v[i]);
    }
}

template <int D, int FORMAT, bool F32>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tiles_kernel(const __grid_constant__ fo_paged_tiles_launch a) {
    using Shape = PtShape<D, F32>;
    using T = typename std::conditional<F32, float, uint16_t>::type;
    constexpr int QUERIES = Shape::QUERIES, TERMS = Shape::TERMS, PANELS = Shape::PANELS, PARTS = Shape::PARTS;
    constexpr int SLOTS = Shape::SLOTS;
    constexpr bool OWN_P = Shape::OWN_P;
    extern __shared__ uint8_t pt_smem[];
    __shared__ PtShared<D, F32> sh;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pt_smem) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int *abort_flag = &sh.abort;

    if (warp == PT_ISSUER) {
        if (lane < SLOTS) mbar_init(&sh.code_full[lane], 1), mbar_init(&sh.code_empty[lane], PT_CONVERTERS);
        if (lane < 2) {
            mbar_init(&sh.k_full[lane], PT_CONVERTERS), mbar_init(&sh.v_full[lane], PT_CONVERTERS);
            mbar_init(&sh.k_empty[lane], 2), mbar_init(&sh.v_empty[lane], 2);
            mbar_init(&sh.s_full[lane], 1), mbar_init(&sh.o_full[lane], 1);
            mbar_init(&sh.p_full[lane], 4), mbar_init(&sh.q_full[lane], 4), mbar_init(&sh.p_half[lane], 4);
            sh.k_tile[lane] = sh.v_tile[lane] = -1;
        }
        if (lane < PT_SEGS) mbar_init(&sh.seg_full[lane], 1), mbar_init(&sh.seg_free[lane], PT_SOFTMAX + 2);
        if (lane < PT_METAS) mbar_init(&sh.meta_full[lane], 1);
        if (lane == 31) {
            mbar_init(&sh.x_full, PT_SOFTMAX), mbar_init(&sh.x_free, PT_SOFTMAX), mbar_init(&sh.done, 2);
            mbar_init(&sh.q_both, 4), mbar_init(&sh.ended, PT_THREADS / 32 - 1);
            for (int i = 0; i < 8; i++) mbar_init(&sh.turn[i & 1][i >> 1], 1);
            sh.abort = 0;
        }
        mbar_fence_init();
        __syncwarp();
        tmem_alloc(&sh.tmem, 512);
    }
    wait_for_prior_kernel();

    // This block's piece [begin, end) of the line, and where it begins.  (The
    // line is shorter than 2^31, checked on the host.)
    const int n_items = a.reach.over_groups ? a.reach.n_groups + 2
                        : a.q_units         ? (int)a.batch.n_seqs * a.q_units
                                            : (int)(a.batch.total_rows * a.group / QUERIES + a.batch.n_seqs);
    int per = 0, begin = 0, end = 0;
    // The line's length first, then the item that the piece begins in; with no more items than
    // threads at one go.
#pragma unroll 1
    for (bool known = false;;) {
        int2 all = make_int2(0, 0);  // length of the line, and tiles
#pragma unroll 1
        for (int first = 0; first < n_items; first += PT_THREADS) {
            int2 mine = make_int2(0, 0), chunk;
            PtItem x;
            if (first + tid < n_items) {
                // (Not every sequence whose rows are wrong is found by number.)
                if (!a.q_units && first + tid < (int)a.batch.n_seqs)
                    load_sequence(a.batch, a.kv.page_size, first + tid, a.err);
                x = pt_item<QUERIES>(a, first + tid);
                mine = make_int2((x.tiles + PT_START) * x.units, x.tiles * x.units);
            }
            int2 before = pt_scan(mine, sh, chunk);
            before.x += all.x, before.y += all.y;
            all.x += chunk.x, all.y += chunk.y;
            if (!known && n_items <= PT_THREADS) {
                known = true;
                per = max((int)((unsigned)(all.x + gridDim.x - 1) / gridDim.x), 2 + PT_START);
                begin = (int)min((long long)per * blockIdx.x, (long long)all.x);
                end = (int)min((long long)begin + per, (long long)all.x);
            }
            // Tiles before a place of the line in this thread's item.
            auto tiles = [&](int at, int unit) {
                return before.y + unit * x.tiles + max(at - before.x - unit * (x.tiles + PT_START) - PT_START, 0);
            };
            if (known && begin >= before.x && begin < before.x + mine.x) {
                sh.begin_item = first + tid;
                sh.begin_base = before.x;
                sh.first_tile = tiles(begin, (begin - before.x) / (x.tiles + PT_START));
            }
            if (known && end > before.x && end <= before.x + mine.x)
                sh.last_tile = tiles(end, (end - 1 - before.x) / (x.tiles + PT_START));
        }
        if (known) break;
        known = true;
        per = max((int)((unsigned)(all.x + gridDim.x - 1) / gridDim.x), 2 + PT_START);
        begin = (int)min((long long)per * blockIdx.x, (long long)all.x);
        end = (int)min((long long)begin + per, (long long)all.x);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int count = begin < end ? sh.last_tile - sh.first_tile : 0;
    if (count <= 0) {
        if (tid == 0) a.joins[8 * blockIdx.x] = 0;
        if (warp == PT_ISSUER) tmem_dealloc(tmem, 512);
        return;
    }

    if (warp < PT_SOFTMAX) {
        // -------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_SOFTMAX_REGS));
        const int t = warp >> 2, wq = warp & 3, r = tid & 127;
        const uint32_t at = tmem + ((uint32_t)(32 * wq) << 16);
        const uint32_t s_at = at + 128 * t, p_at = OWN_P ? at + 384 + 64 * t : s_at;
        auto o_at = [&](int stream) { return at + 256 + (OWN_P ? 64 : 128) * stream; };
        int turns = 0;  // tiles that this warp and the other stream's have taken turns at
        int c = 0, x_phase = 0, both_phase = 0;  // tiles of this stream so far; joins of both streams; queries of both
        bool ok = true;
        for (int s = 0; ok; s++) {
            ok = pt_wait(&sh.seg_full[s % PT_SEGS], (s / PT_SEGS) & 1, abort_flag);
            if (!ok) break;
            const PtSegment &seg = sh.seg[s % PT_SEGS];
            const int n = seg.n, base = seg.base, pair = seg.pair, last = seg.last;
            const int q = (pair ? 128 * t : 0) + r;  // of the unit's
            const bool live = (pair ? 128 * t : 0) + 32 * wq < seg.nq;
            // The row's queries, as operands, and what it sees.  (Rows that are none's see everything,
            // and are not kept.)
            const bool own = pair || t == 0 || n > 1;  // this stream has tiles
            const bool mine = q < seg.nq;
            float q_scale = 0.0f, sink = -INFINITY;
            int high = INT32_MAX, low = 0, h = 0;
            int64_t row = 0;
            if (mine) {
                const int qi = seg.q0 + q, row_of = qi / a.group;
                row = seg.first + row_of;
                h = seg.head * a.group + qi - row_of * a.group;
                if (a.sinks) sink = a.sinks[h];
                if (seg.flat) {
                    high = min(place_of_row(a.batch, a.kv.page_size, (int)row, a.err), seg.end - 1);
                } else {
                    high = max(seg.p0 + row_of, -1);
                    low = a.window > 0 ? max(high + 1 - a.window, 0) : 0;
                }
            }
            if (live && (pair || t == 0)) {
                // The warp's rows as they are into their places, 16 bytes to a lane and neighbouring
                // lanes in a row; then each thread its own row to FP16 operands there.  FP32 rows lie
                // where their two terms will be.
                constexpr int CHUNKS = D * (int)sizeof(T) / 16;
                uint8_t *rows = smem + t * TERMS * Shape::OPERAND + 32 * wq * 128;
                auto place = [&](int of, int chunk) {
                    return reinterpret_cast<uint4 *>(rows + (chunk >> 3) * PT_PANEL + of * 128 + (((chunk & 7) ^ (of & 7)) << 4));
                };
                const T *data = static_cast<const T *>(a.q.data);
                const long long at_q = row * a.q.row_stride + h * a.q.head_stride;
                constexpr int FLIGHT = 8;
#pragma unroll 1
                for (int x0 = 0; x0 < CHUNKS; x0 += FLIGHT) {
                    uint4 y[FLIGHT];
#pragma unroll
                    for (int x = 0; x < FLIGHT; x++) {
                        const int of = ((x0 + x) * 32 + lane) / CHUNKS, chunk = ((x0 + x) * 32 + lane) % CHUNKS;
                        const T *from = data + __shfl_sync(0xffffffffu, at_q, of) + chunk * (16 / (int)sizeof(T));
                        y[x] = make_uint4(0, 0, 0, 0);
                        if (q - lane + of >= seg.nq) continue;
                        if (a.q_vec) {
                            y[x] = *reinterpret_cast<const uint4 *>(from);
                        } else {
                            T z[16 / sizeof(T)];
#pragma unroll
                            for (int e = 0; e < 16 / (int)sizeof(T); e++) z[e] = from[e];
                            memcpy(&y[x], z, 16);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < FLIGHT; x++)
                        *place(((x0 + x) * 32 + lane) / CHUNKS, ((x0 + x) * 32 + lane) % CHUNKS) = y[x];
                }
                __syncwarp();
                // The largest magnitude, as bits, which are in its order (NaN above infinity): of FP32,
                // or of two BF16 at once.
                uint32_t most = 0;
                uint4 raw[F32 ? CHUNKS : 1];
#pragma unroll(F32 ? CHUNKS : 2)
                for (int x = 0; x < CHUNKS; x++) {
                    const uint4 w = *place(lane, x);
                    if constexpr (F32) {
                        raw[x] = w;
                        most = max(most, max(max(w.x & 0x7FFFFFFFu, w.y & 0x7FFFFFFFu),
                                             max(w.z & 0x7FFFFFFFu, w.w & 0x7FFFFFFFu)));
                    } else {
                        most = __vmaxu2(most, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu),
                                                       __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
                    }
                }
                if constexpr (!F32) most = max(most & 0xFFFFu, most >> 16) << 16;
                const bool finite = most < 0x7F800000u;
                // A power of two brings the largest element to [2^14, 2^15); 2^126 at most, which still
                // brings the least rows to where FP16 holds BF16's 8 bits.
                const int e = max((int)(most >> 23), 15);
                const float up = finite ? __uint_as_float((uint32_t)(268 - e) << 23) : 0.0f;
                q_scale = finite ? __uint_as_float((uint32_t)max(e - 14, 1) << 23) * a.scale * REACH_LOG2E : NAN;
                if constexpr (!F32) {
#pragma unroll 1
                    for (int x = 0; x < CHUNKS; x++) {
                        Raw8<T> w;
                        w.w[0] = *place(lane, x);
                        float y[8];
                        unpack8(w, y);
#pragma unroll
                        for (int e = 0; e < 8; e++) y[e] = finite ? y[e] * up : 0.0f;
                        *place(lane, x) = make_uint4(pt_f16x2(y[0], y[1]), pt_f16x2(y[2], y[3]), pt_f16x2(y[4], y[5]),
                                                     pt_f16x2(y[6], y[7]));
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < CHUNKS / 2; x++) {
                        const uint32_t w[8] = {raw[2 * x].x, raw[2 * x].y, raw[2 * x].z, raw[2 * x].w,
                                               raw[2 * x + 1].x, raw[2 * x + 1].y, raw[2 * x + 1].z, raw[2 * x + 1].w};
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float u = finite ? __uint_as_float(w[2 * e]) * up : 0.0f;
                            const float v = finite ? __uint_as_float(w[2 * e + 1]) * up : 0.0f;
                            hi[e] = pt_f16x2(u, v);
                            const float2 b = f16x2_f32x2(hi[e]);
                            lo[e] = pt_f16x2(u - b.x, v - b.y);
                        }
                        *place(lane, x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *place(lane, x + CHUNKS / 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                // Zeros, rows of no query and those that see nothing have scores of 0, or none, at any scale; at
                // this one they go the short way.
                if (most == 0 || high < 0) q_scale = 0x1p-30f;
                if (!pair) sh.q_scale[r] = q_scale;
                fence_proxy_async_smem();
            }
            __syncwarp();
            if (pair || t == 0) {
                if (lane == 0) {
                    mbar_arrive(&sh.q_full[t]);
                    if (!pair && n > 1) mbar_arrive(&sh.q_both);
                }
            } else if (own) {
                ok = pt_wait(&sh.q_both, both_phase, abort_flag);
                if (!ok) break;
                if (live) q_scale = sh.q_scale[r];
                if (lane == 0) mbar_arrive(&sh.q_full[t]);
            }
            if (!pair && n > 1) both_phase ^= 1;
            float m = -INFINITY, l = 0.0f;
            int top = PT_LOWEST;  // exponent bits of a power of two above the scales of the values that the row sees
            bool any = false;
            // FP32 rows: what was summed up to a few tiles ago is outside tensor memory, relative to
            // these.
            bool kept = false;
            float kept_m = 0.0f;
            int kept_top = 0;
            float4 *keep = reinterpret_cast<float4 *>(a.part_o) +
                           (int64_t)(2 * gridDim.x + blockIdx.x) * (D / 4) * FO_TILES_QUERIES + 128 * t + r;
            // O and the sums kept, into what is kept or (`back`) into O.
            auto move = [&](bool back) {
                const float f = !kept ? 0.0f
                                      : (m == -INFINITY ? 1.0f : ex2(kept_m - m)) *
                                            __uint_as_float((uint32_t)max(127 + kept_top - top, 0) << 23);
                tc_fence_after();
#pragma unroll 1
                for (int d = 0; d < D; d += 16) {
                    uint32_t o[16];
                    FO_TMEM_LD16(o_at(t) + d, o);
                    float4 y[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        y[e] = kept ? __ldcg(keep + (d / 4 + e) * FO_TILES_QUERIES) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        y[e].x = fmaf(y[e].x, f, __uint_as_float(o[4 * e]));
                        y[e].y = fmaf(y[e].y, f, __uint_as_float(o[4 * e + 1]));
                        y[e].z = fmaf(y[e].z, f, __uint_as_float(o[4 * e + 2]));
                        y[e].w = fmaf(y[e].w, f, __uint_as_float(o[4 * e + 3]));
                        if (!back) {
                            __stcg(keep + (d / 4 + e) * FO_TILES_QUERIES, y[e]);
                        } else {
                            o[4 * e] = __float_as_uint(y[e].x), o[4 * e + 1] = __float_as_uint(y[e].y);
                            o[4 * e + 2] = __float_as_uint(y[e].z), o[4 * e + 3] = __float_as_uint(y[e].w);
                        }
                    }
                    if (back) FO_TMEM_ST16(o_at(t) + d, o);
                }
                if (back) tmem_wait_st();
                kept = true;
                kept_m = m;
                kept_top = top;
            };
            // Turns, where both have queries.  (With P in columns of its own the streams do better without:
            // a page's prompt 106.6 us, with 110.1; heads of 128 the other way, 2,443 and 2,375.)
            const bool turning = !OWN_P && pair && 128 + 32 * wq < seg.nq;
            for (int i = pair ? 0 : t; i < n; i += pair ? 1 : 2, c++) {
                const int k = base + i;
                ok = pt_wait(&sh.s_full[t], c & 1, abort_flag);
                if (!ok) break;
                if (!live) {
                    // No query in this warp: whatever its lanes hold stays theirs.  (It arrives once
                    // for each tile as the others do, not for the next one before they have for this.)
                    if (any) ok = pt_wait(&sh.o_full[t], (c - 1) & 1, abort_flag);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive(&sh.p_half[t]), mbar_arrive(&sh.p_full[t]);
                    __syncwarp();
                    any = true;
                    continue;
                }
                ok = pt_wait(&sh.meta_full[k % PT_METAS], (k / PT_METAS) & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const PtMeta &meta = sh.meta[k % PT_METAS];
                const int tile = meta.base;
                int tile_top = meta.top;
                const int hi = min(high, meta.to - 1), lo = max(low, meta.from);
                // The scores' factors will multiply -infinity too, of which a product that underflows to 0
                // would make NaN; and scores that may pass 2^25 are rounded before their maximum is taken
                // from them, or what is left, exact, could be more than P has room for.  (Rows that are not
                // finite are NaN either way, and do not send the others round about, where their scores are
                // rounded once more.)
                constexpr float MOST = 0x1p25f / (0x1p15f * (FORMAT == FO_PAGED_I8 ? 128.0f : 448.0f) * D);
                const bool plain = __all_sync(0xffffffffu, !(meta.least * q_scale < FLT_MIN || meta.most * q_scale > MOST));
                const bool all = hi - tile >= PT_TILE - 1 && (lo <= tile || a.reach.first - tile >= PT_TILE);
                if (!__all_sync(0xffffffffu, plain && all)) {
                    // Scores of keys that the row does not see become -infinity in tensor memory, 32 keys
                    // at a time, where a row of the warp does not see them all.  (Code of every kind runs
                    // on an SM at once, and what does not stay in its instruction cache costs more than
                    // these round trips: 128 masks in line took 3,000 cycles.)  Scales that would make
                    // something else of -infinity are multiplied here.
                    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; };
                    tile_top = PT_LOWEST;
#pragma unroll 1
                    for (int w = 0; w < 4; w++) {
                        // Keys that the row sees, as bits.  (Differences that cannot wrap: every one is of
                        // numbers from -1 up.)
                        const int b = tile + 32 * w;
                        const uint32_t see = below(min(hi - b, 32) + 1) & (~below(lo - b) | below(a.reach.first - b));
                        if (see & 0x0000FFFFu) tile_top = max(tile_top, pt_above(meta.vs[2 * w]));
                        if (see & 0xFFFF0000u) tile_top = max(tile_top, pt_above(meta.vs[2 * w + 1]));
                        if (__all_sync(0xffffffffu, plain && see == 0xFFFFFFFFu)) continue;
                        uint32_t x[32];
                        FO_TMEM_LD32(s_at + 32 * w, x);
                        const float f0 = plain ? 1.0f : meta.ks[2 * w] * q_scale;
                        const float f1 = plain ? 1.0f : meta.ks[2 * w + 1] * q_scale;
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            const float y = __uint_as_float(x[e]) * (e < 16 ? f0 : f1);
                            x[e] = see >> e & 1 ? __float_as_uint(y) : 0xFF800000u;
                        }
                        FO_TMEM_ST32(s_at + 32 * w, x);
                        tmem_wait_st();
                    }
                }
                // What 32 keys of a row need: their scores' factors (log2 units), the largest score, and
                // the probabilities.
                // (Read before the scores are waited for.)
                auto factors = [&](int w) {
                    const float2 ks = *reinterpret_cast<const float2 *>(&meta.ks[2 * w]);
                    return plain ? make_float2(ks.x * q_scale, ks.y * q_scale) : make_float2(1.0f, 1.0f);
                };
                float mx = -INFINITY;
                auto largest = [&](const uint32_t *raw, float2 f) {
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                        for (int e = 16 * g; e < 16 * g + 16; e += 4) {
                            m0 = fmaxf(fmaxf(m0, __uint_as_float(raw[e])), __uint_as_float(raw[e + 1]));
                            m1 = fmaxf(fmaxf(m1, __uint_as_float(raw[e + 2])), __uint_as_float(raw[e + 3]));
                        }
                        mx = fmaxf(mx, fmaxf(m0, m1) * (g ? f.y : f.x));
                    }
                };
                // S is read twice, in short loops: what is run over and over has to stay in the instruction
                // cache (with the row in registers and all of it in line: 123 us for a page's prompt where
                // this takes 110, 2,621 for ragged prompts with heads of 128 against 2,375).
                uint32_t raw[64];
                FO_TMEM_LD32(s_at, raw);
#pragma unroll 1
                for (int w = 0; w < 4; w += 2) {
                    const float2 f0 = factors(w), f1 = factors(w + 1);
                    tmem_wait_ld();
                    FO_TMEM_LD32(s_at + 32 * w + 32, (raw + 32));
                    largest(raw, f0);
                    tmem_wait_ld();
                    FO_TMEM_LD32(s_at + (32 * w + 64) % 128, raw);  // (at last the first keys again)
                    largest(raw + 32, f1);
                }
                if (F32 && any && i / (pair ? 1 : 2) % PT_KEEP == 0) move(false);
                float factor = 1.0f;  // of what has been summed so far
                if (!any) {
                    m = mx;
                    top = tile_top;
                } else if (__any_sync(0xffffffffu, mx > __fadd_rd(m, PT_SLACK) || tile_top > top)) {
                    const float next = fmaxf(m, mx);
                    const float alpha = next == -INFINITY ? 1.0f : ex2(m - next);
                    l *= alpha;
                    // (Beyond 2^-126 what was summed is nothing next to what comes.)
                    factor = alpha * __uint_as_float((uint32_t)max(127 + top - max(top, tile_top), 0) << 23);
                    m = next;
                    top = max(top, tile_top);
                }
                const float shift = m == -INFINITY ? 0.0f : m;
                // P may be written, and O touched, once the PV before is complete.
                // (In S's place, S would not be there before.)
                if (any) {
                    if (OWN_P) ok = pt_wait(&sh.o_full[t], (c - 1) & 1, abort_flag);
                    if (!ok) break;
                    if (__any_sync(0xffffffffu, factor != 1.0f) && !(F32 && i / (pair ? 1 : 2) % PT_KEEP == 0)) {
                        tc_fence_after();
#pragma unroll 1
                        for (int d = 0; d < D; d += 16) {
                            uint32_t o[16];
                            FO_TMEM_LD16(o_at(t) + d, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                            FO_TMEM_ST16(o_at(t) + d, o);
                        }
                    }
                }
                // The two streams' warps of an SM's quarter take turns at the exponentials, which its special
                // function unit bounds; the one that is not at them does the rest.
                if (turning && (t == 1 || turns > 0)) {
                    ok = pt_wait(&sh.turn[t ^ 1][wq], (t == 1 ? turns : turns - 1) & 1, abort_flag);
                    if (!ok) break;
                }
                // Values' scales are taken times 2^10 / top; those of pages that the row does not see meet
                // zeros.
                const float inverse_top = __uint_as_float((uint32_t)(264 - top) << 23);
                float2 sum = make_float2(0.0f, 0.0f);
                auto values = [&](int w) {
                    const float2 vs = *reinterpret_cast<const float2 *>(&meta.vs[2 * w]);
                    return make_float2(fminf(vs.x * inverse_top, FLT_MAX), fminf(vs.y * inverse_top, FLT_MAX));
                };
                auto probabilities = [&](const uint32_t *raw, int w, float2 f, float2 vs) {
                    float2 p[16];
                    uint32_t term[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float g = e < 8 ? f.x : f.y, v = e < 8 ? vs.x : vs.y;
                        const float2 x = __ffma2_rn(make_float2(__uint_as_float(raw[2 * e]), __uint_as_float(raw[2 * e + 1])),
                                                    make_float2(g, g), make_float2(-shift, -shift));
                        p[e] = make_float2(ex2(x.x), ex2(x.y));
                        sum = __fadd2_rn(sum, p[e]);
                        p[e] = __fmul2_rn(p[e], make_float2(v, v));
                        term[e] = pt_f16x2(p[e].x, p[e].y);
                    }
                    FO_TMEM_ST16(p_at + 16 * TERMS * w, term);
                    if constexpr (F32) {
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float2 b = f16x2_f32x2(term[e]);
                            term[e] = pt_f16x2(p[e].x - b.x, p[e].y - b.y);
                        }
                        FO_TMEM_ST16(p_at + 16 * TERMS * w + 16, term);
                    }
                };
#pragma unroll 1
                for (int w = 0; w < 4; w += 2) {
                    const float2 f0 = factors(w), f1 = factors(w + 1), v0 = values(w), v1 = values(w + 1);
                    tmem_wait_ld();
                    FO_TMEM_LD32(s_at + 32 * w + 32, (raw + 32));
                    probabilities(raw, w, f0, v0);
                    if (w == 2) {
                        // The first half is multiplied while the second is computed.
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.p_half[t]);
                    }
                    tmem_wait_ld();
                    if (w == 0) FO_TMEM_LD32(s_at + 64, raw);
                    probabilities(raw + 32, w + 1, f1, v1);
                }
                l += sum.x + sum.y;
                if (turning) {
                    if (lane == 0) mbar_arrive(&sh.turn[t][wq]);
                    turns++;
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
                any = true;
            }
            if (!ok) break;
            // The segment's end.
            if (any) {
                ok = pt_wait(&sh.o_full[t], (c - 1) & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
            }
            if (F32 && live && kept) move(true);
            // O times f0, and where both streams have these rows the other's times f1.
            const float unit = __uint_as_float((uint32_t)(top - 10) << 23);  // of O
            float f0 = unit, f1 = 0.0f;
            int c0 = 0, c1 = D;  // this thread's dimensions
            bool has0 = any, has1 = false;
            int o_from = t;
            if (!pair) {
                sh.xm[t][r] = m;
                sh.xl[t][r] = l;
                sh.xt[t][r] = unit;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.x_full);
                ok = pt_wait(&sh.x_full, x_phase, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const Joined j = join_parts(sh.xm[0][r], sh.xl[0][r], sh.xm[1][r], sh.xl[1][r]);
                m = j.m;
                l = j.l;
                f0 = j.f0 * sh.xt[0][r];
                f1 = j.f1 * sh.xt[1][r];
                c0 = t * (D / 2);
                c1 = c0 + D / 2;
                has0 = true;
                has1 = n > 1;
                o_from = 0;
            }
            if (live) {
                const int part = seg.part;
                float inv = 0.0f, fp = 0.0f;
                const int64_t at_row = row * a.q.heads + h;
                if (mine && part < 0 && a.reach.raw_o) {
                    if (pair || t == 0) reinterpret_cast<float2 *>(a.reach.raw_ml)[at_row] = make_float2(m, l);
                } else if (mine && part < 0) {
                    if (a.reach.prior_o) {
                        const float2 prior = reinterpret_cast<const float2 *>(a.reach.prior_ml)[at_row];
                        const Joined j = join_parts(m, l, prior.x, prior.y);
                        m = j.m;
                        l = j.l;
                        f0 *= j.f0;
                        f1 *= j.f0;
                        fp = j.f1;
                    }
                    inv = inverse_sum(sink, m, l);
                    if (a.lse && (pair || t == 0)) a.lse[at_row] = log_sum(m, l);
                } else if (mine && (pair || t == 0)) {
                    reinterpret_cast<float2 *>(a.part_ml)[(int64_t)part * FO_TILES_QUERIES + q] = make_float2(m, l);
                }
                // Where the row's sums are, by the block that its unit begins in.
                if (mine && a.reach.parts_of && (pair || t == 0) && (part < 0 || part & 1))
                    reinterpret_cast<int2 *>(a.reach.parts_of)[at_row] = make_int2(part < 0 ? -1 : (int)blockIdx.x, seg.c1 | q << 16);
                T *out = static_cast<T *>(a.out.data) + row * a.out.row_stride + h * a.out.head_stride;
                // Finished rows of one stream, as most are, 32 dimensions at a time.
                const bool simple = !has1 && part < 0 && !a.reach.raw_o && !a.reach.prior_o && a.out_vec;
                if (simple) {
                    // BF16 rows of a pair by way of the queries' place, which this warp is done with, so
                    // that eight lanes write 128 bytes of a row.
                    const bool staged = !F32 && pair;
                    uint8_t *stage = smem + t * TERMS * Shape::OPERAND + 32 * wq * 128;
                    const float scale = f0 * inv;
#pragma unroll 1
                    for (int d = c0; d < c1; d += 32) {
                        uint32_t o[32];
                        float v[32];
                        FO_TMEM_LD32(o_at(o_from) + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = __uint_as_float(o[e]) * scale;
                        if (staged) {
#pragma unroll
                            for (int e = 0; e < 32; e += 8)
                                store8(reinterpret_cast<T *>(stage + (d >> 6) * PT_PANEL + lane * 128 +
                                                             ((((d + e) >> 3 & 7) ^ (lane & 7)) << 4)),
                                       v + e);
                        } else if (mine) {
#pragma unroll
                            for (int e = 0; e < 32; e += 8) store8(out + d + e, v + e);
                        }
                    }
                    if (staged) {
                        const long long at_out = row * a.out.row_stride + h * a.out.head_stride;
                        __syncwarp();
#pragma unroll 1
                        for (int x = 0; x < 8 * PANELS; x++) {
                            const int from = (x & 7) * 4 + (lane >> 3), chunk = lane & 7;  // of the warp's rows
                            const long long to = __shfl_sync(0xffffffffu, at_out, from);
                            const uint4 y = *reinterpret_cast<const uint4 *>(stage + (x >> 3) * PT_PANEL + from * 128 +
                                                                             ((chunk ^ (from & 7)) << 4));
                            if (q - lane + from < seg.nq)
                                *reinterpret_cast<uint4 *>(static_cast<T *>(a.out.data) + to + (x >> 3) * 64 + 8 * chunk) = y;
                        }
                        __syncwarp();
                    }
                }
#pragma unroll 1
                for (int d = simple ? c1 : c0; d < c1; d += 16) {
                    uint32_t o[16];
                    float v[16];
                    if (has0) {
                        FO_TMEM_LD16(o_at(o_from) + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = __uint_as_float(o[e]) * f0;
                    }
                    if (has1) {
                        FO_TMEM_LD16(o_at(1) + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = fmaf(__uint_as_float(o[e]), f1, v[e]);
                    }
                    if (!mine) continue;
                    if (part >= 0 || a.reach.raw_o) {
                        const int64_t step = part >= 0 ? FO_TILES_QUERIES : 1;
                        float4 *to = part >= 0 ? reinterpret_cast<float4 *>(a.part_o) +
                                                     ((int64_t)part * (D / 4) + d / 4) * FO_TILES_QUERIES + q
                                               : reinterpret_cast<float4 *>(a.reach.raw_o + at_row * D + d);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            __stcg(to + e * step, make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]));
                        continue;
                    }
                    if (a.reach.prior_o) {
                        const float4 *from = reinterpret_cast<const float4 *>(a.reach.prior_o + at_row * D + d);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float4 y = __ldcg(from + e);
                            v[4 * e] = fmaf(y.x, fp, v[4 * e]);
                            v[4 * e + 1] = fmaf(y.y, fp, v[4 * e + 1]);
                            v[4 * e + 2] = fmaf(y.z, fp, v[4 * e + 2]);
                            v[4 * e + 3] = fmaf(y.w, fp, v[4 * e + 3]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) v[e] *= inv;
                    pt_store16(out + d, v, a.out_vec);
                }
            }
            if (!pair) {
                // Neither stream goes on to write its O before the other has read it.
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.x_free);
                ok = pt_wait(&sh.x_free, x_phase, abort_flag);
                x_phase ^= 1;
                if (!ok) break;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.seg_free[s % PT_SEGS]);
            if (last) break;
        }
    } else if (warp < PT_PRODUCER) {
        // ----------------------------------------------------------- converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_OTHER_REGS));
        const int ct = tid - 32 * PT_SOFTMAX, log_page = 31 - __clz(a.kv.page_size);
        constexpr int CHUNKS = D / 16;  // 16-byte chunks of a row's codes
        int slot = 0, round = 0;
        bool ok = true;
        for (int k = 0; k < count && ok; k++) {
#pragma unroll 1
            for (int value = 0; value < 2; value++) {
                uint64_t *full = value ? &sh.v_full[k & 1] : &sh.k_full[k & 1];
                uint64_t *empty = value ? &sh.v_empty[k & 1] : &sh.k_empty[k & 1];
                uint8_t *to = smem + (value ? Shape::OFF_V : Shape::OFF_K) + (k & 1) * Shape::OPERAND;
                if (k > 1) ok = pt_wait(empty, (k / 2 - 1) & 1, abort_flag);
                if (!ok) break;
                if (ct == 0) *(volatile int *)(value ? &sh.v_tile[k & 1] : &sh.k_tile[k & 1]) = k;
#pragma unroll 1
                for (int h = 0; h < PARTS; h++) {
                    ok = pt_wait(&sh.code_full[slot], round & 1, abort_flag);
                    if (!ok) break;
                    const uint4 *from = reinterpret_cast<const uint4 *>(smem + Shape::OFF_CODES + slot * PT_SLOT);
                    const unsigned pages = sh.meta[k % PT_METAS].pages;
                    const int row_from = sh.meta[k % PT_METAS].from - sh.meta[k % PT_METAS].base;
                    const int row_to = sh.meta[k % PT_METAS].to - sh.meta[k % PT_METAS].base;
                    uint4 w[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) w[j] = from[j * 128 + ct];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int u = j * 128 + ct, row = h * (PT_TILE / PARTS) + u / CHUNKS, chunk = u % CHUNKS;
                        // Values that were not copied, or that no row sees, may be any bytes: an FP8 NaN
                        // times a probability of 0 would be NaN.
                        if (value && !(row >= row_from && row < row_to && (pages >> (row >> log_page) & 1)))
                            w[j] = make_uint4(0, 0, 0, 0);
                        const uint2 h0 = pt_widen<FORMAT>(w[j].x), h1 = pt_widen<FORMAT>(w[j].y);
                        const uint2 h2 = pt_widen<FORMAT>(w[j].z), h3 = pt_widen<FORMAT>(w[j].w);
                        uint8_t *line = to + (chunk >> 2) * PT_PANEL + row * 128;
                        const int c16 = 2 * (chunk & 3), odd = chunk >> 2;  // which half first: other banks for the panels
                        const uint4 lo = make_uint4(h0.x, h0.y, h1.x, h1.y), hi = make_uint4(h2.x, h2.y, h3.x, h3.y);
                        *reinterpret_cast<uint4 *>(line + (((c16 + odd) ^ (row & 7)) << 4)) = odd ? hi : lo;
                        *reinterpret_cast<uint4 *>(line + (((c16 + 1 - odd) ^ (row & 7)) << 4)) = odd ? lo : hi;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.code_empty[slot]);
                    if (++slot == SLOTS) slot = 0, round++;
                }
                if (!ok) break;
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_OTHER_REGS));
        if (warp == PT_PRODUCER) {
            // --------------------------------------------------------- producer
            const int page = a.kv.page_size, log_page = 31 - __clz(page), pages = max(PT_TILE >> log_page, 1);
            PtItem item;
            item.units = 0;
            int index = sh.begin_item - 1, unit = 0, tile = 0;
            int segs = 0, ahead = 0, left = 0, head = 0;
            int at_unit = 0;  // the unit's place in the line
            bool ok = true;
            if (lane == 0) a.joins[8 * blockIdx.x] = 0;
            struct Next {
                int base, from, to, head, id;  // the tile's positions [from, to) that rows may see
                float ks, vs;
                bool wanted, bad;  // rows see this lane's page; its number is outside the pool
            };
            auto fetch = [&]() {
                Next x;
                x.base = x.from = x.to = x.head = x.id = 0;
                x.ks = x.vs = 0.0f;
                x.wanted = x.bad = false;
                if (ahead >= count || !ok) return x;
                if (unit == item.units) {
                    do item = pt_item<QUERIES>(a, ++index);
                    while (item.units == 0 && index < n_items - 1);
                    unit = 0;
                    if (ahead == 0) {
                        at_unit = sh.begin_base;
                        unit = (begin - at_unit) / (item.tiles + PT_START);
                        at_unit += unit * (item.tiles + PT_START);
                        tile = max(begin - at_unit - PT_START, 0);
                    }
                }
                if (left == 0) {
                    // A new segment: the rest of the unit, or of the block's piece.
                    const int n = min(item.tiles - tile, count - ahead);
                    left = n;
                    const int heads = a.kv.n_kv_heads, q_unit = a.reach.over_groups ? unit / heads : 0;
                    head = unit - q_unit * heads;
                    if (segs >= PT_SEGS)
                        ok = pt_wait(&sh.seg_free[segs % PT_SEGS], (segs / PT_SEGS - 1) & 1, abort_flag);
                    if (!ok) return x;
                    if (lane == 0) {
                        PtSegment &g = sh.seg[segs % PT_SEGS];
                        g.n = n;
                        g.base = ahead;
                        g.head = head;
                        g.first = item.first;
                        g.q0 = item.q0 + q_unit * QUERIES;
                        g.nq = min(item.n * a.group - g.q0, QUERIES);
                        g.pair = Shape::Q_TILES == 2 && g.nq > 128;
                        g.last = ahead + n == count;
                        g.p0 = item.p0;
                        g.end = item.end;
                        g.flat = a.reach.over_groups;
                        g.part = -1;
                        g.c1 = 0;
                        if (n < item.tiles) {
                            const int from = at_unit + PT_START;
                            const int c0 = from / per, c1 = (from + item.tiles - 1) / per;
                            g.part = 2 * (int)blockIdx.x + (c0 == (int)blockIdx.x ? 1 : 0);
                            g.c1 = c1;
                            if (c0 == (int)blockIdx.x) {
                                int *j = a.joins + 8 * blockIdx.x;
                                j[1] = g.first;
                                j[2] = g.q0;
                                j[3] = g.head;
                                j[4] = c1;
                                j[0] = g.nq;
                            }
                        }
                        mbar_arrive(&sh.seg_full[segs % PT_SEGS]);
                    }
                    __syncwarp();
                    segs++;
                }
                const bool early = tile < item.tf;
                x.base = (early ? tile : item.t0 + tile - item.tf) * PT_TILE;
                x.head = head;
                // Of a shared beginning, the first tiles' positions are the leader's and end with it, and the others
                // begin behind it.
                x.from = item.shared > 0 && !early ? item.shared : 0;
                x.to = item.shared > 0 && early ? min(item.shared, item.end) : item.end;
                const int off = lane << log_page;
                if (lane < pages && off < x.to - x.base) {
                    const int begins = (x.base + off) >> log_page << log_page;  // of the page
                    const bool seen = item.shared > 0 ? early || page > item.shared - begins
                                                      : begins < a.reach.first || page > item.low - begins;
                    if (seen) {
                        x.wanted = true;
                        x.id = a.batch.page_table[(item.shared > 0 && early ? item.leader : item.seq) * a.batch.table_stride +
                                                  (begins >> log_page)];
                    }
                }
                ahead++;
                left--;
                if (++tile == item.tiles) {
                    tile = 0;
                    unit++;
                    at_unit += item.tiles + PT_START;
                }
                return x;
            };
            auto scales = [&](Next &x) {
                if (!x.wanted) return;
                x.bad = x.id < 0 || x.id >= a.kv.n_pages;
                if (x.bad) return;
                const int64_t at = (int64_t)x.id * a.kv.n_kv_heads + x.head;
                x.ks = a.kv.k_scales[at];
                x.vs = a.kv.v_scales[at];
            };
            int slot = 0, round = 0, issued = 0;
            Next now = {}, next = {}, later = {};
            // Page numbers two tiles ahead, scales one.
#pragma unroll 1
            for (int k = -2; k < count && ok; k++) {
                now = next;
                next = later;
                later = fetch();
                scales(next);
                if (k < 0) continue;
                if (!ok) break;
                if (round > 0) ok = pt_wait(&sh.code_empty[slot], (round - 1) & 1, abort_flag);
                if (!ok) break;
                // The tile's scales.  A page number outside the pool, or a scale that is not finite,
                // gives NaN to the rows that see the page, by their scores.
                const bool load = now.wanted && !now.bad;
                const bool sane = load && fabsf(now.ks) <= FLT_MAX && fabsf(now.vs) <= FLT_MAX;
                if (now.bad) atomicOr(a.err, FO_DEVERR_PAGED);
                // (That of a page that no row sees is never used.)
                const float ks = !now.wanted ? 1.0f : !sane ? NAN : now.ks, vs = sane ? now.vs : 0.0f;
                const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(vs))));
                PtMeta &meta = sh.meta[k % PT_METAS];
                const unsigned mask = __ballot_sync(0xffffffffu, load);
                // Eight entries of 16 positions each; a page larger than that has several.
                const int shift = log_page - 4;
                const float ks8 = __shfl_sync(0xffffffffu, ks, lane < 8 ? min(lane >> shift, 31) : 0);
                const float vs8 = __shfl_sync(0xffffffffu, vs, lane < 8 ? min(lane >> shift, 31) : 0);
                if (lane < 8) {
                    meta.ks[lane] = ks8;
                    meta.vs[lane] = vs8;
                }
                // (Numbers above 0 are in their bits' order.)
                const float least = __uint_as_float(__reduce_min_sync(0xffffffffu, ks > 0.0f ? __float_as_uint(ks) : 0u));
                const float largest =
                    __uint_as_float(__reduce_max_sync(0xffffffffu, now.wanted && ks > 0.0f ? __float_as_uint(ks) : 0u));
                if (lane == 8) meta.top = pt_above(most), meta.least = least, meta.most = largest;
                if (lane == 9) meta.base = now.base;
                if (lane == 10) meta.pages = mask;
                if (lane == 11) meta.from = now.from, meta.to = now.to;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.meta_full[k % PT_METAS]);
#pragma unroll 1
                for (int p = 0; p < 2 * PARTS; p++) {
                    if (p > 0 && round > 0) {
                        ok = pt_wait(&sh.code_empty[slot], (round - 1) & 1, abort_flag);
                        if (!ok) break;
                    }
                    // This slot's rows [h, h + 128 / PARTS) of the tile's.
                    constexpr int ROWS = PT_TILE / PARTS;
                    const int h = p % PARTS * ROWS, rows = min(page, ROWS);
                    const int at = page > ROWS ? 0 : (lane << log_page) - h;  // of this lane's page in the slot
                    const bool here = load && at >= 0 && at < ROWS;
                    const uint32_t n_here = __popc(__ballot_sync(0xffffffffu, here));
                    if (lane == 0) mbar_expect_tx(&sh.code_full[slot], n_here * (uint32_t)(rows * D));
                    __syncwarp();
                    if (here) {
                        const uint8_t *codes = static_cast<const uint8_t *>(p < PARTS ? a.kv.k_codes : a.kv.v_codes);
                        codes += (((int64_t)now.id * a.kv.n_kv_heads + now.head) * page + (page > ROWS ? h : 0)) * D;
                        bulk_g2s(smem + Shape::OFF_CODES + slot * PT_SLOT + at * D, codes, rows * D, &sh.code_full[slot]);
                    }
                    __syncwarp();
                    issued++;
                    if (++slot == SLOTS) slot = 0, round++;
                }
            }
            if (lane == 0) {
                // The copies in flight land before the block ends, also where another warp gave up.
                for (int i = max(issued - SLOTS, 0); i < issued; i++)
                    mbar_wait_drain(&sh.code_full[i % SLOTS], (i / SLOTS) & 1);
            }
        } else if (warp < PT_ISSUER + 2) {
            // ---------------------------------------------------------- issuers
            // A warp for each stream, whose code is the same and short (one for both, polling whatever
            // could be ready, fetched its long loop anew each time: up to 3,000 cycles from a P to its
            // MMA).  The whole warp runs the loop and its waits, so that addresses stay uniform; one
            // elected lane issues.
            const int t = warp - PT_ISSUER;
            const uint32_t base = smem_u32(smem);
            constexpr uint32_t ID_S = idesc_f16(128, 128, 0), ID_PV = idesc_f16(128, D, 1);
            const uint64_t dQ = sdesc_sw128(base, 16, 1024), dK = sdesc_sw128(base + Shape::OFF_K, 16, 1024);
            const uint64_t dV = sdesc_sw128(base + Shape::OFF_V, PT_PANEL, 1024);
            constexpr uint32_t OPERAND16 = Shape::OPERAND >> 4, PANEL16 = PT_PANEL >> 4;
            struct Tile {
                int k, pair;
                bool first;  // of its segment's in this stream, or since O was taken away
            };
            auto issue_s = [&](const Tile &x) {
                if (elect_one()) {
                    uint32_t more = 0;
#pragma unroll 1
                    for (int term = TERMS - 1; term >= 0; term--) {
                        const uint64_t q = dQ + ((x.pair ? t : 0) * TERMS + term) * OPERAND16;
                        const uint64_t b = dK + (x.k & 1) * OPERAND16;
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {
                            const uint32_t off = (kk >> 2) * PANEL16 + 2 * (kk & 3);
                            mma_bf16(tmem + 128 * t, q + off, b + off, ID_S, more);
                            more = 1;
                        }
                    }
                    mma_commit(&sh.s_full[t]);
                    // A tile that is this stream's alone is released for both.
                    mma_commit(&sh.k_empty[x.k & 1]);
                    if (!x.pair) mma_commit(&sh.k_empty[x.k & 1]);
                }
                __syncwarp();
            };
            // Half h of the keys.
            auto issue_pv = [&](const Tile &x, int h) {
                if (elect_one()) {
                    const uint32_t p = tmem + (OWN_P ? 384 + 64 * t : 128 * t), o = tmem + 256 + (OWN_P ? 64 : 128) * t;
                    const uint64_t b = dV + (x.k & 1) * OPERAND16;
#pragma unroll 1
                    for (int term = TERMS - 1; term >= 0; term--)  // the small terms while the sum is
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const int kk = 4 * h + y;
                            mma_bf16_ts(o, p + 16 * (term + TERMS * (kk >> 1)) + 8 * (kk & 1), b + kk * (2048 >> 4), ID_PV,
                                        term < TERMS - 1 || kk > 0 || !x.first);
                        }
                    if (h == 1) {
                        mma_commit(&sh.o_full[t]);
                        mma_commit(&sh.v_empty[x.k & 1]);
                        if (!x.pair) mma_commit(&sh.v_empty[x.k & 1]);
                    }
                }
                __syncwarp();
            };
            // Waits for tile k's operands.  A stream skips tiles that are the other's, and a parity wait
            // cannot tell a phase from the one two before; once the operands' tile number is k, the phase
            // before is over.
            auto there = [&](uint64_t *full, const int *number, int k) {
                for (;;) {
                    if (!pt_wait(full + (k & 1), (k >> 1) & 1, abort_flag)) return false;
                    if (__all_sync(0xffffffffu, *(const volatile int *)(number + (k & 1)) == k))
                        return pt_wait(full + (k & 1), (k >> 1) & 1, abort_flag);
                    if (__any_sync(0xffffffffu, *abort_flag)) return false;
                }
            };
            // The stream's place: the next tile of its own is i of segment seg.
            int seg = -1, i = 0, n = 0, first = 0, pair = 0, loads = 0;
            bool last = false, ok = true;
            // Goes on to the next segment with a tile of this stream's; false after the last one.
            auto enter = [&]() {
                while (i >= n) {
                    if (seg >= 0) {
                        if (lane == 0) mbar_arrive(&sh.seg_free[seg % PT_SEGS]);
                        __syncwarp();
                    }
                    if (last) return false;
                    seg++;
                    ok = pt_wait(&sh.seg_full[seg % PT_SEGS], (seg / PT_SEGS) & 1, abort_flag);
                    if (!ok) return false;
                    const PtSegment &g = sh.seg[seg % PT_SEGS];
                    n = g.n;
                    first = g.base;
                    pair = g.pair;
                    last = g.last;
                    i = pair ? 0 : t;
                }
                ok = pt_wait(&sh.q_full[t], loads & 1, abort_flag);
                loads++;
                return ok;
            };
            auto take = [&]() {
                const Tile x = {first + i, pair, F32 ? i / (pair ? 1 : 2) % PT_KEEP == 0 : i < (pair ? 1 : 2)};
                i += pair ? 1 : 2;
                return x;
            };
            bool more = enter();
            Tile now = {};
            if (more) {
                now = take();
                ok = there(sh.k_full, sh.k_tile, now.k);
                tc_fence_after();
                if (ok) issue_s(now);
            }
            for (int c = 0; more && ok; c++) {
                Tile next = {};
                bool issued = false;
                const bool same = i < n;  // the next tile is of the same segment
                if (same) next = take();
                ok = there(sh.v_full, sh.v_tile, now.k) && pt_wait(&sh.p_half[t], c & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                issue_pv(now, 0);
                ok = pt_wait(&sh.p_full[t], c & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                if (OWN_P && same) {
                    // S first, if its keys are there: it is what the softmax waits for next.
                    issued = __all_sync(0xffffffffu, *(volatile int *)&sh.k_tile[next.k & 1] == next.k &&
                                                         mbar_test(&sh.k_full[next.k & 1], (next.k >> 1) & 1));
                    if (issued) {
                        tc_fence_after();
                        issue_s(next);
                    }
                }
                issue_pv(now, 1);
                if (!issued) {
                    if (!same) {
                        more = enter();
                        if (!more) break;
                        next = take();
                    }
                    ok = there(sh.k_full, sh.k_tile, next.k);
                    if (ok && !OWN_P) ok = pt_wait(&sh.o_full[t], c & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(next);
                }
                now = next;
            }
            // Every issued MMA completes before tensor memory is released.
            if (elect_one()) mma_commit(&sh.done);
            __syncwarp();
            if (lane == 0) mbar_wait_drain(&sh.done, 0);
            __syncwarp();
        } else {
            // ---------------------------------------------------------- the bound
            uint64_t t0 = globaltimer();
            int seen = 0;
            while (!mbar_try_wait(&sh.ended, 0)) {
                __nanosleep(500);
                const int now = *(volatile int *)&sh.k_tile[0] + *(volatile int *)&sh.k_tile[1];
                if (now != seen) t0 = globaltimer();
                seen = now;
                if (globaltimer() - t0 <= FO_WAIT_NS) continue;
                *abort_flag = 1;
                if (lane == 0) atomicOr(a.err, FO_DEVERR_WAIT_TIMEOUT);
                break;
            }
            __syncwarp();
        }
    }
    if (warp < PT_THREADS / 32 - 1 && lane == 0) mbar_arrive(&sh.ended);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == PT_ISSUER) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------- the joining
// The parts of the unit that begins in block blockIdx.x and goes on in others, in
// the blocks' order: 32 of its queries, four dimensions to a thread.
constexpr int PJ_QUERIES = 32, PJ_THREADS = 256;
template <int D, bool F32>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const __grid_constant__ fo_paged_tiles_launch a) {
    using T = typename std::conditional<F32, float, uint16_t>::type;
    wait_for_prior_kernel();
    const int c0 = blockIdx.x;
    const int4 j0 = __ldcg(reinterpret_cast<const int4 *>(a.joins) + 2 * c0);
    const int nq = j0.x, q = blockIdx.y * PJ_QUERIES + (threadIdx.x & 31);
    if (blockIdx.y * PJ_QUERIES >= nq || q >= nq) return;
    const int first = j0.y, qi = j0.z + q, head = j0.w, c1 = __ldcg(a.joins + 8 * c0 + 4);
    const int r = qi / a.group, h = head * a.group + qi - r * a.group;
    const int64_t row = first + r, at_row = row * a.q.heads + h;
    const float2 *mls = reinterpret_cast<const float2 *>(a.part_ml);
    auto part = [&](int c) { return (int64_t)(2 * c + (c == c0 ? 1 : 0)); };
    float2 prior = make_float2(-INFINITY, 0.0f);
    if (a.reach.prior_o) prior = reinterpret_cast<const float2 *>(a.reach.prior_ml)[at_row];
    float m = prior.x;
#pragma unroll 4
    for (int c = c0; c <= c1; c++) m = fmaxf(m, __ldcg(mls + part(c) * FO_TILES_QUERIES + q).x);
    const float shift = m == -INFINITY ? 0.0f : m, fp = exp2f(prior.x - shift);
    constexpr int QUADS = D / 4, STEP = PJ_THREADS / 32, MINE = QUADS / STEP;
    const int quad0 = threadIdx.x >> 5;
    float l = prior.y * fp;
    float4 v[MINE];
#pragma unroll
    for (int i = 0; i < MINE; i++) {
        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.reach.prior_o) {
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(a.reach.prior_o + at_row * D) + quad0 + STEP * i);
            v[i] = make_float4(y.x * fp, y.y * fp, y.z * fp, y.w * fp);
        }
    }
#pragma unroll 4
    for (int c = c0; c <= c1; c++) {
        const float2 ml = __ldcg(mls + part(c) * FO_TILES_QUERIES + q);
        const float f = exp2f(ml.x - shift);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(a.part_o) +
                                    (part(c) * QUADS + quad0 + STEP * i) * FO_TILES_QUERIES + q);
            v[i] = make_float4(fmaf(y.x, f, v[i].x), fmaf(y.y, f, v[i].y), fmaf(y.z, f, v[i].z), fmaf(y.w, f, v[i].w));
        }
    }
    if (a.reach.raw_o) {
#pragma unroll
        for (int i = 0; i < MINE; i++)
            reinterpret_cast<float4 *>(a.reach.raw_o + at_row * D)[quad0 + STEP * i] = v[i];
        if (quad0 == 0) reinterpret_cast<float2 *>(a.reach.raw_ml)[at_row] = make_float2(m, l);
        return;
    }
    const float inv = inverse_sum(a.sinks ? a.sinks[h] : -INFINITY, m, l);
    T *out = static_cast<T *>(a.out.data) + row * a.out.row_stride + h * a.out.head_stride;
#pragma unroll
    for (int i = 0; i < MINE; i++) {
        T *to = out + 4 * (quad0 + STEP * i);
        const float4 y = make_float4(v[i].x * inv, v[i].y * inv, v[i].z * inv, v[i].w * inv);
        if (!a.out_vec) {
            store1(to, y.x);
            store1(to + 1, y.y);
            store1(to + 2, y.z);
            store1(to + 3, y.w);
        } else if constexpr (F32) {
            *reinterpret_cast<float4 *>(to) = y;
        } else {
            *reinterpret_cast<uint2 *>(to) = make_uint2(bf16_pair(y.x, y.y), bf16_pair(y.z, y.w));
        }
    }
    if (a.lse && quad0 == 0) a.lse[at_row] = log_sum(m, l);
}

template <int D, int FORMAT, bool F32>
cudaError_t launch_tiles(const fo_paged_tiles_launch &in, int sms, cudaStream_t stream) {
    fo_paged_tiles_launch a = in;
    using Shape = PtShape<D, F32>;
    static_assert(Shape::SMEM + sizeof(PtShared<D, F32>) <= 227 * 1024, "shared memory");
    auto *kernel = paged_tiles_kernel<D, FORMAT, F32>;
    // The attribute belongs to each device's context: set once per device.
    static std::atomic<unsigned long long> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
        if (e != cudaSuccess) return e;
        // The kernel's register split is only sound at the launch count that it
        // was written for.
        cudaFuncAttributes f;
        e = cudaFuncGetAttributes(&f, kernel);
        if (e != cudaSuccess) return e;
        if (f.numRegs != PT_LAUNCH_REGS) return cudaErrorInvalidConfiguration;
        configured.fetch_or(bit);
    }
    // No more blocks than the most tiles there can be for, two to a block.
    const int64_t table = (a.batch.table_stride * a.kv.page_size + PT_TILE - 1) / PT_TILE;
    a.q_units = (int)((a.batch.max_rows * a.group + Shape::QUERIES - 1) / Shape::QUERIES);
    // Ragged sequences of up to so many units: as many numbers for each, those behind a
    // sequence's rows for nothing.  Of more, a number is the rows before the sequence in
    // units, and the sequences before it: floor(first / Q) + b + floor(n / Q) + 1 is at most
    // the next one's floor((first + n) / Q) + b + 1, so they are in order, and there is
    // hardly one that is nothing's; finding the sequence takes a search.
    constexpr int MOST_UNITS = 4;
    if (a.batch.row_start && !a.reach.over_groups && a.q_units > MOST_UNITS) a.q_units = 0;
    const int64_t units = a.reach.over_groups
                              ? (a.batch.total_rows * a.group + Shape::QUERIES - 1) / Shape::QUERIES + a.reach.n_groups + 2
                          : a.q_units ? a.batch.n_seqs * a.q_units
                                      : a.batch.total_rows * a.group / Shape::QUERIES + a.batch.n_seqs;
    const int64_t most = units * a.kv.n_kv_heads * table;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(sms, (most + 1) / 2));
    cudaError_t e = launch(kernel, dim3(grid), dim3(PT_THREADS), Shape::SMEM, stream, a);
    if (e != cudaSuccess || grid == 1 || a.reach.parts_of) return e;
    return launch(paged_join_kernel<D, F32>, dim3(grid, Shape::QUERIES / PJ_QUERIES), dim3(PJ_THREADS), 0, stream, a);
}

template <int D>
cudaError_t launch_tiles(const fo_paged_tiles_launch &a, int sms, cudaStream_t stream) {
    if (a.q.dtype == FO_DT_F32)
        return a.kv.format == FO_PAGED_I8 ? launch_tiles<D, FO_PAGED_I8, true>(a, sms, stream)
                                          : launch_tiles<D, FO_PAGED_E4M3, true>(a, sms, stream);
    return a.kv.format == FO_PAGED_I8 ? launch_tiles<D, FO_PAGED_I8, false>(a, sms, stream)
                                      : launch_tiles<D, FO_PAGED_E4M3, false>(a, sms, stream);
}

}  // namespace fo

extern "C" cudaError_t fo_launch_paged_tiles(const fo_paged_tiles_launch *args, int sms, cudaStream_t stream) {
    fo_paged_tiles_launch a = *args;
    if (a.batch.total_rows <= 0) return cudaSuccess;
    a.group = a.q.heads / a.kv.n_kv_heads;
    auto aligned = [](const fo_rows &r) {
        const int64_t unit = r.dtype == FO_DT_F32 ? 4 : 8;  // elements in 16 bytes
        return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    a.q_vec = aligned(a.q);
    a.out_vec = aligned(a.out);
    return a.kv.head_dim == 64 ? fo::launch_tiles<64>(a, sms, stream) : fo::launch_tiles<128>(a, sms, stream);
}
