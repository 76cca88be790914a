// paged_attention.cu -- attention of a batch's query rows over a paged 8-bit
// KV cache.
//
// For a query row q at position p of its sequence, over the visible positions
// j: s_j = scale * kscale * (q . kcode_j), m = max s_j, out = sum_j e^(s_j - m)
// vscale vcode_j / (sum_j e^(s_j - m) + e^(sink - m)), kscale and vscale those
// of j's page.  Every key and value is read once for all query heads and rows
// of its KV head, so the call is bound by HBM: positions x KV heads x 2 D
// bytes.
//
// Work is a line of tiles, 16 KB of one KV head of one sequence (64 or 128
// positions; and one group of its queries, where there are more than a block
// holds), the tiles of a (sequence, KV head) adjacent.  Each of at most one block per SM
// takes an equal piece of the line, wherever sequences begin and end, so
// uneven lengths leave no SM behind and one long sequence is spread over all
// of them.  A block that holds only part of a (sequence, KV head) leaves its
// maximum, sum and output in scratch, and the last block of those that share
// it (a counter in scratch) joins the parts in order.
//
// In a block four producer warps walk the page table a step ahead and copy
// tiles into a ring in shared memory with TMA (swizzled, so that the reads
// below meet no bank conflicts); eight consumer warps, two to a tile, a half
// each, take tiles in turn, each with its own running maximum and sum, and are
// joined at a piece's end.  A
// consumer computes S^T = K Q^T and O^T += V^T P^T on m16n8k16 tensor
// instructions with the codes as the A operand: an int8 or FP8 code is an
// FP16 number exactly, and a scale multiplies a finished sum, so nothing of the
// cache is rounded.  The 5th-generation MMA reads its operands from shared
// memory or TMEM, which would cost every tile a trip back through shared
// memory after the conversion; a decode's few queries leave these instructions
// far from bounding the kernel.  A query is held as FP16 relative to a
// power of two near its largest element: BF16's 8 bits exactly, FP32 as the sum
// of two terms (22 bits) in neighbouring columns.  Probabilities are scaled
// by 2^10 so that FP16 holds those down to 2^-24 of the largest at full
// precision; BF16 rows round them to FP16's 11 bits, three more than the
// output has, FP32 rows carry a second term.  Sums, maxima and outputs are FP32.
#include "paged.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <atomic>
#include <cudaTypedefs.h>

namespace fo {

constexpr int PA_CONSUMERS = 8;  // consumer warps
constexpr int PA_PRODUCERS = 4;  // producer warps
constexpr int PA_STAGES = 12;    // tiles in the ring
// A parity wait cannot tell a barrier's phase from the one two before it.
// Every slot of the ring is filled by one producer warp only and emptied by
// one group of consumer warps only, each of which passes its phases one by one.
static_assert(PA_STAGES % PA_PRODUCERS == 0 && PA_STAGES % (PA_CONSUMERS / 2) == 0, "owners of the ring's slots");
constexpr int PA_THREADS = 32 * (PA_CONSUMERS + PA_PRODUCERS);
// Registers a thread: launched with 168 (65,536 over 384 threads), the
// producers' warpgroup gives up what the consumers' two take:
// 128 * 72 + 256 * 216 = 384 * 168.
constexpr int PA_LAUNCH_REGS = 168, PA_PRODUCER_REGS = 72, PA_CONSUMER_REGS = 216;
static_assert(128 * PA_PRODUCER_REGS + 256 * PA_CONSUMER_REGS == PA_THREADS * PA_LAUNCH_REGS, "register split");
constexpr float PA_P_BITS = 10.0f;  // probabilities are held times 2^10
constexpr float PA_LOG2E = 1.4426950408889634f, PA_LN2 = 0.6931471805599453f;

template <int D>
struct PaShape {
    static constexpr int TILE_BYTES = 8192;        // of keys, and of values
    static constexpr int TILE = TILE_BYTES / D;    // positions
    static constexpr int HALF = TILE / 2;          // a consumer warp's
    static constexpr int STAGE = 2 * TILE_BYTES;
    static constexpr int COMB_LD = 64 + 4;         // a column of the joining buffer (64 dimensions), in floats
    static constexpr int COMB = PA_CONSUMERS * 8 * COMB_LD * 4;
    static constexpr int SMEM = 1024 + PA_STAGES * STAGE + COMB;
};

// The row of eight that a fragment's row g stands for: such that a K
// fragment's and a V fragment's reads fall into different banks under the
// tile's swizzle (128-byte rows: 128-byte swizzle; 64-byte rows: 64-byte).
template <int D>
__device__ __forceinline__ int pa_key(int g) {
    if constexpr (D == 128) return g & 1 ? (g - 1) ^ 5 : g;
    return (0x65217430u >> (4 * g)) & 7;
}

__device__ __forceinline__ void pa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit elements, two per lane along a row, transposed.
__device__ __forceinline__ uint32_t pa_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pa_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Four codes as FP16 (exact): the low two and the high two.
template <int FORMAT>
__device__ __forceinline__ void pa_codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (FORMAT == FO_PAGED_I8) {
        // 1024 + (code + 128) has the code in its low bits; 1152 = 0x6480.
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
    } else {
        lo = e4m3x2_f16x2(w & 0xFFFFu);
        hi = e4m3x2_f16x2(w >> 16);
    }
}

// A sequence's share of the line of tiles.
struct PaWork {
    Sequence s;
    int low;     // first position that any of its rows sees
    int t0;      // its tile
    int tiles;   // per KV head and group of queries (one at least, so that rows that see nothing are written)
    int groups;  // groups of `queries` queries
};
template <int TILE>
__device__ __forceinline__ PaWork pa_work(const fo_paged_attention_launch &a, int64_t seq) {
    PaWork w;
    w.s = load_sequence(a.batch, a.kv.page_size, seq, a.err);
    const int64_t p0 = max64(w.s.len - w.s.n, 0);
    w.low = a.window > 0 ? (int)max64(p0 + 1 - a.window, 0) : 0;
    w.t0 = w.low / TILE;
    w.tiles = max((int)((w.s.len + TILE - 1) / TILE) - w.t0, 1);
    w.groups = (w.s.n * a.group + a.queries - 1) / a.queries;
    return w;
}

// A place in the line: a sequence, a unit of it (KV head, group of queries)
// and a tile of the unit.
template <int TILE>
struct PaCursor {
    PaWork w;
    int seq, unit, tile;
    __device__ __forceinline__ int head() const { return unit / w.groups; }
    __device__ __forceinline__ int group() const { return unit % w.groups; }
    __device__ __forceinline__ int left() const { return w.tiles - tile; }
    // Moves on by n tiles, at most to the unit's end.
    __device__ __forceinline__ void advance(const fo_paged_attention_launch &a, int n) {
        tile += n;
        if (tile < w.tiles) return;
        tile = 0;
        if (++unit < a.kv.n_kv_heads * w.groups) return;
        unit = 0;
        do {
            if (++seq >= a.batch.n_seqs) return;
            w = pa_work<TILE>(a, seq);
        } while (w.groups == 0);
    }
};

struct PaShared {
    uint64_t full[PA_STAGES], empty[PA_STAGES];
    float scales[PA_STAGES][16];  // keys' of a tile's pages, then values'
    float ml[PA_CONSUMERS][16][2];
    long long warp_sum[PA_THREADS / 32];
    long long begin_base;
    int begin_seq, abort, last;
};

// Sum of x over the block's earlier threads; `all` the whole block's.
__device__ __forceinline__ long long pa_scan(long long x, PaShared &sh, long long &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    __syncthreads();  // the last scan's sums have been read
    if (lane == 31) sh.warp_sum[warp] = incl;
    __syncthreads();
    long long before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < PA_THREADS / 32; w++) {
        if (w < warp) before += sh.warp_sum[w];
        all += sh.warp_sum[w];
    }
    return before + incl - x;
}

__device__ __forceinline__ void pa_consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * PA_CONSUMERS) : "memory"); }

template <int D, int FORMAT, int NT, int TERMS>
__global__ void __launch_bounds__(PA_THREADS, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                           const __grid_constant__ fo_paged_attention_launch a) {
    using Shape = PaShape<D>;
    constexpr int STAGES = PA_STAGES;
    constexpr int TILE = Shape::TILE, HALF = Shape::HALF;
    constexpr int STEPS = HALF / 16;       // m16 steps of a consumer's half
    constexpr int KW = D / 16;             // words of a K row per lane
    constexpr int VW = D / 32;             // words of a V row per lane
    constexpr int MT = D / 16;             // m16 tiles of the output's dimensions
    constexpr int QN = 8 / TERMS;          // queries of an n8 tile
    constexpr int WARP_QUERIES = NT * QN;  // queries of a consumer warp
    using T = typename std::conditional<TERMS == 2, float, uint16_t>::type;
    extern __shared__ uint8_t pa_smem[];
    __shared__ PaShared sh;
    uint8_t *tiles = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pa_smem) + 1023) & ~uintptr_t(1023));
    float *comb = reinterpret_cast<float *>(tiles + STAGES * Shape::STAGE);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int key_groups = PA_CONSUMERS / 2 / a.col_groups;

    // This block's piece [begin, end) of the line, and where it begins.
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) {
            sm100::mbar_init(&sh.full[i], 1);
            sm100::mbar_init(&sh.empty[i], 2 * a.col_groups);
        }
        sm100::mbar_fence_init();
        sh.abort = 0;
    }
    auto work_of = [&](int64_t seq) -> long long {
        if (seq >= a.batch.n_seqs) return 0;
        const PaWork w = pa_work<TILE>(a, seq);
        return (long long)w.tiles * w.groups * a.kv.n_kv_heads;
    };
    long long all, mine = work_of(tid);
    long long before = pa_scan(mine, sh, all);
    long long total = all, chunk = all;
    for (int64_t base = PA_THREADS; base < a.batch.n_seqs; base += PA_THREADS) {
        pa_scan(work_of(base + tid), sh, all);
        total += all;
    }
    const long long per = max((total + gridDim.x - 1) / gridDim.x, (long long)key_groups);
    const long long begin = per * blockIdx.x, end = min(begin + per, total);
    if (begin >= end) return;
    for (int64_t base = 0, sum = 0;;) {
        if (begin >= sum + before && begin < sum + before + mine) {
            sh.begin_seq = (int)base + tid;
            sh.begin_base = sum + before;
        }
        base += PA_THREADS;
        if (base >= a.batch.n_seqs) break;
        // Only batches wider than a block come here.
        sum += chunk;
        mine = work_of(base + tid);
        before = pa_scan(mine, sh, chunk);
    }
    __syncthreads();
    PaCursor<TILE> at;
    at.seq = sh.begin_seq;
    at.w = pa_work<TILE>(a, at.seq);
    long long base = sh.begin_base;  // the line's number of at's sequence's first tile
    {
        const int in = (int)(begin - base);
        at.unit = in / at.w.tiles;
        at.tile = in - at.unit * at.w.tiles;
    }
    const int count = (int)(end - begin);
    const int page = a.kv.page_size;
    const int pages = page >= TILE ? 1 : TILE / page;  // of a tile

    if (warp >= PA_CONSUMERS) {
        // ------------------------------------------------------------ producer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_PRODUCER_REGS));
        // Each producer warp issues every PA_PRODUCERS-th tile of the block's: one
        // warp's wait, expectation and two copies take about 500 cycles, more
        // than a tile's share of HBM's time.  Page numbers and scales are fetched
        // a batch of 32 pages at a time, the numbers two batches ahead of the
        // copies and the scales one.
        const int producer = warp - PA_CONSUMERS;
        const int per_batch = 32 / pages;
        const int j = lane % pages, off = lane / pages;
        struct Batch {
            int first, n;   // the block's tiles first, first + PA_PRODUCERS, ..: n of them
            int head, row;  // KV head, and this lane's page: its first row, its number (-1: none)
            int id;
            bool bad;
            float ks, vs;
        };
        int ahead = 0;  // tiles handed to batches
        bool more = true;
        auto fetch_id = [&]() {
            Batch b;
            b.id = -1;
            b.bad = false;
            b.row = 0;
            b.ks = b.vs = 0.0f;
            b.first = b.n = b.head = 0;
            const int span = min(min(PA_PRODUCERS * per_batch, at.left()), count - ahead);
            if (span <= 0) {
                more = false;
                return b;
            }
            const int skip = (producer - ahead % PA_PRODUCERS + PA_PRODUCERS) % PA_PRODUCERS;
            b.first = ahead + skip;
            b.n = (span - skip + PA_PRODUCERS - 1) / PA_PRODUCERS;
            b.head = at.head();
            // The first position that the page's copy holds.
            const int64_t pos = (int64_t)(at.w.t0 + at.tile + skip + PA_PRODUCERS * off) * TILE + j * page;
            const int64_t begins = pos / page * page;
            if (off < b.n && pos < at.w.s.len && begins + page > at.w.low) {
                b.id = __ldg(a.batch.page_table + at.seq * a.batch.table_stride + pos / page);
                b.row = (int)(pos - begins);
            }
            ahead += span;
            at.advance(a, span);
            return b;
        };
        auto fetch_scales = [&](Batch &b) {
            if (b.id == -1) return;
            b.bad = b.id < 0 || b.id >= a.kv.n_pages;
            if (b.bad) return;
            const int64_t tile = (int64_t)b.id * a.kv.n_kv_heads + b.head;
            b.ks = __ldg(a.kv.k_scales + tile);
            b.vs = __ldg(a.kv.v_scales + tile);
        };
        if (lane == 0) {
            sm100::tma_prefetch(&k_map);
            sm100::tma_prefetch(&v_map);
        }
        const uint64_t policy = sm100::l2_evict_first();
        const int rows = min(page, TILE);
        const uint32_t bytes = (uint32_t)rows * D;
        int last = -1;  // the last tile whose copies were issued
        bool ok = true;
        // The first page numbers are asked for together, the first scales while
        // the second numbers are on their way.
        Batch now = fetch_id(), next = fetch_id();
        fetch_scales(now);
        for (bool rest = true; rest && ok;) {
            rest = more;
            Batch later = fetch_id();
            fetch_scales(next);
            for (int i = 0; i < now.n; i++) {
                const int tile = now.first + PA_PRODUCERS * i, slot = tile % STAGES, round = tile / STAGES;
                if (round > 0 && !sm100::mbar_wait(&sh.empty[slot], (round - 1) & 1, &sh.abort, a.err)) {
                    ok = false;
                    break;
                }
                const bool here = off == i;
                const bool load = here && now.id != -1 && !now.bad;
                const uint32_t n_loads = __popc(__ballot_sync(0xffffffffu, load));
                if (lane == 0) {
                    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(
                                     sm100::smem_u32(&sh.full[slot])),
                                 "r"(n_loads * 2 * bytes)
                                 : "memory");
                }
                __syncwarp();
                if (load) {
                    uint8_t *kt = tiles + slot * Shape::STAGE + j * bytes, *vt = kt + Shape::TILE_BYTES;
                    const int row = now.head * page + now.row;
                    if (a.evict_first) {
                        sm100::tma_load_3d_hint(kt, &k_map, &sh.full[slot], 0, row, now.id, policy);
                        sm100::tma_load_3d_hint(vt, &v_map, &sh.full[slot], 0, row, now.id, policy);
                    } else {
                        sm100::tma_load_3d(kt, &k_map, &sh.full[slot], 0, row, now.id);
                        sm100::tma_load_3d(vt, &v_map, &sh.full[slot], 0, row, now.id);
                    }
                }
                if (here) {
                    // A page number outside the pool gives NaN; a page that no row
                    // sees has scales of 0.
                    sh.scales[slot][j] = now.bad ? NAN : now.ks;
                    sh.scales[slot][8 + j] = now.bad ? NAN : now.vs;
                    if (now.bad) atomicOr(a.err, FO_DEVERR_PAGED);
                }
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&sh.full[slot]);
                last = tile;
            }
            now = next;
            next = later;
        }
        if (!ok && lane == 0) {
            // A consumer gave up: the copies in flight land before the block ends.
            for (int i = last; i >= 0 && i > last - STAGES; i -= PA_PRODUCERS)
                sm100::mbar_wait_drain(&sh.full[i % STAGES], (i / STAGES) & 1);
        }
        return;
    }

    // ---------------------------------------------------------------- consumers
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_CONSUMER_REGS));
    const int g = lane >> 2, t = lane & 3;
    const int col_group = warp % a.col_groups, half = warp / a.col_groups % 2, key_group = warp / a.col_groups / 2;
    const int kg = pa_key<D>(g), kt0 = pa_key<D>(2 * t), kt1 = pa_key<D>(2 * t + 1);
    // Byte offsets of this lane's pieces of a K row and of its V rows.
    const int k_off = D == 128 ? kg * 128 + ((t ^ kg) << 4) : kg * 64 + ((t ^ (kg >> 1 & 3)) << 4);
    const int v_off0 = D == 128 ? kt0 * 128 + ((g ^ kt0) << 4) : kt0 * 64 + (((g >> 1) ^ (kt0 >> 1 & 3)) << 4) + (g & 1) * 8;
    const int v_off1 = D == 128 ? kt1 * 128 + ((g ^ kt1) << 4) : kt1 * 64 + (((g >> 1) ^ (kt1 >> 1 & 3)) << 4) + (g & 1) * 8;
    const int page_shift = 31 - __clz(min(page, TILE) / 16);  // log2 of the m16 steps of a page's part of a tile
    bool ok = true;

    for (int i = 0; i < count;) {
        const int n = min(at.left(), count - i);
        const Sequence &s = at.w.s;
        const int head = at.head(), q0 = at.group() * a.queries;
        const int n_queries = min(s.n * a.group - q0, a.queries);  // of this unit
        const int p_first = (int)(s.len - s.n);                    // position of the sequence's first row
        // The queries as B operands: column g of tile nt, elements 16 t .. 16 t
        // + 15 (and 64 more, of the second half).
        uint32_t qf[NT][KW][2];
        float q_scale[NT][2];  // of this lane's columns 2 t, 2 t + 1
        int q_pos[NT][2];
        auto query_of = [&](int nt, int col) { return col_group * WARP_QUERIES + nt * QN + (TERMS == 2 ? col >> 1 : col); };
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int qi = query_of(nt, g);
            float x[KW / 4][16];
            float top = 0.0f;
            if (qi < n_queries) {
                const int r = (q0 + qi) / a.group, hh = (q0 + qi) - r * a.group;
                const T *q = static_cast<const T *>(a.q.data) + (s.first + r) * a.q.row_stride +
                             (head * a.group + hh) * a.q.head_stride + 16 * t;
#pragma unroll
                for (int c = 0; c < KW / 4; c++) {
                    if (a.q_vec) {
                        load8(q + 64 * c, x[c]);
                        load8(q + 64 * c + 8, x[c] + 8);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) x[c][e] = load1(q + 64 * c + e);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(x[c][e]));
                }
            } else {
#pragma unroll
                for (int c = 0; c < KW / 4; c++)
#pragma unroll
                    for (int e = 0; e < 16; e++) x[c][e] = 0.0f;
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // A power of two near the largest element (1 for none, and within what
            // both it and its inverse can be).
            const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
            const float unit = __uint_as_float((uint32_t)(254 - e) << 23);
            const float back = __uint_as_float((uint32_t)e << 23) * a.scale * PA_LOG2E;
#pragma unroll
            for (int c = 0; c < KW / 4; c++)
#pragma unroll
                for (int w = 0; w < 4; w++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float y0 = x[c][4 * w + 2 * h] * unit, y1 = x[c][4 * w + 2 * h + 1] * unit;
                        uint32_t f = pa_f16x2(y0, y1);
                        if (TERMS == 2 && (g & 1)) {
                            const float2 z = f16x2_f32x2(f);
                            f = pa_f16x2(y0 - z.x, y1 - z.y);
                        }
                        qf[nt][4 * c + w][h] = f;
                    }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                q_scale[nt][h] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + h));
                const int qh = query_of(nt, 2 * t + h);
                q_pos[nt][h] = qh < n_queries ? p_first + (q0 + qh) / a.group : -1;
            }
        }
        float m[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int d = 0; d < MT; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[d][nt][e] = 0.0f;
        }
        // Tiles all of whose positions every row sees need no mask.
        const int p_last = p_first + s.n - 1;
        const int low_last = a.window > 0 ? max(p_last + 1 - (int)min64(a.window, INT32_MAX / 2), 0) : 0;

        int k = i + (key_group - i % key_groups + key_groups) % key_groups;
        for (; ok && k < i + n; k += key_groups) {
            const int slot = k % STAGES;
            // The first position of this warp's half.
            const int pos0 = (at.w.t0 + at.tile + (k - i)) * TILE + half * HALF;
            ok = sm100::mbar_wait(&sh.full[slot], (k / STAGES) & 1, &sh.abort, a.err);
            if (!ok) break;
            if (pos0 > p_last || pos0 + HALF <= at.w.low) {
                // No row sees any of it.
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&sh.empty[slot]);
                continue;
            }
            const uint8_t *kt = tiles + slot * Shape::STAGE + half * HALF * D;
            uint8_t *vt = tiles + slot * Shape::STAGE + Shape::TILE_BYTES + half * HALF * D;
            // S^T: rows = keys, columns = queries.
            float c[STEPS][NT][4];
#pragma unroll
            for (int mt = 0; mt < STEPS; mt++) {
                uint32_t kw[2][KW];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint8_t *row = kt + (16 * mt + 8 * h) * D;
                    *reinterpret_cast<uint4 *>(kw[h]) = *reinterpret_cast<const uint4 *>(row + k_off);
                    if constexpr (D == 128)
                        *reinterpret_cast<uint4 *>(kw[h] + 4) = *reinterpret_cast<const uint4 *>(row + (k_off ^ 64));
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) c[mt][nt][e] = 0.0f;
#pragma unroll
                for (int w = 0; w < KW; w++) {
                    uint32_t a0, a1, a2, a3;
                    pa_codes<FORMAT>(kw[0][w], a0, a2);
                    pa_codes<FORMAT>(kw[1][w], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) pa_mma(c[mt][nt], a0, a1, a2, a3, qf[nt][w][0], qf[nt][w][1]);
                }
            }
            const bool masked = pos0 + HALF - 1 > p_first || pos0 < low_last;
            // Scores, times log2 e; FP32 rows have a query's two terms in
            // neighbouring columns.
            float mx[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < STEPS; mt++) {
                const float ks = sh.scales[slot][(half * STEPS + mt) >> page_shift];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if constexpr (TERMS == 2) {
                        c[mt][nt][0] = c[mt][nt][1] = (c[mt][nt][0] + c[mt][nt][1]) * (ks * q_scale[nt][0]);
                        c[mt][nt][2] = c[mt][nt][3] = (c[mt][nt][2] + c[mt][nt][3]) * (ks * q_scale[nt][0]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) c[mt][nt][e] *= ks * q_scale[nt][e & 1];
                    }
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int pos = pos0 + 16 * mt + kg + (e >> 1) * 8, p = q_pos[nt][e & 1];
                            const bool seen = pos <= p && (a.window == 0 || pos > p - a.window);
                            if (!seen) c[mt][nt][e] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[nt][e & 1] = fmaxf(mx[nt][e & 1], c[mt][nt][e]);
                }
            }
            float alpha[NT][2];
            bool moved = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float x = mx[nt][h];
                    if (TERMS == 2 && h == 1) {
                        mx[nt][1] = mx[nt][0];
                        m[nt][1] = m[nt][0];
                        alpha[nt][1] = alpha[nt][0];
                        continue;
                    }
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = fmaxf(x, m[nt][h]);
                    moved |= x != m[nt][h];
                    // While nothing has been seen the maximum stays -infinity and
                    // every probability below is 0.
                    alpha[nt][h] = x == -INFINITY ? 1.0f : sm100::ex2(m[nt][h] - x);
                    m[nt][h] = x;
                    mx[nt][h] = x == -INFINITY ? 0.0f : x - PA_P_BITS;
                }
            if (TERMS == 2) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    mx[nt][1] = mx[nt][0];
                    m[nt][1] = m[nt][0];
                    alpha[nt][1] = alpha[nt][0];
                }
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) l[nt][h] *= alpha[nt][h];
#pragma unroll
                    for (int d = 0; d < MT; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[d][nt][e] *= alpha[nt][e & 1];
                }
            }
            // Probabilities, transposed into B operands: rows = keys of V.
            uint32_t pf[STEPS][NT][2];
#pragma unroll
            for (int mt = 0; mt < STEPS; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        uint32_t f;
                        if constexpr (TERMS == 2) {
                            const float p = sm100::ex2(c[mt][nt][2 * r] - mx[nt][0]);
                            l[nt][0] += p;
                            const uint32_t hi = pa_f16x2(p, 0.0f);
                            f = pa_f16x2(p, p - f16x2_f32x2(hi).x);
                        } else {
                            const float p0 = sm100::ex2(c[mt][nt][2 * r] - mx[nt][0]);
                            const float p1 = sm100::ex2(c[mt][nt][2 * r + 1] - mx[nt][1]);
                            l[nt][0] += p0;
                            l[nt][1] += p1;
                            f = pa_f16x2(p0, p1);
                        }
                        pf[mt][nt][r] = pa_transpose(f);
                    }
            if constexpr (FORMAT == FO_PAGED_E4M3) {
                // Rows beyond the sequence, or of pages that no row sees, may hold any
                // bytes: an FP8 NaN times a probability of 0 would be NaN.
                const int lo_row = max(at.w.low / page * page - pos0, 0), hi_row = (int)min64(s.len - pos0, HALF);
                if (lo_row > 0 || hi_row < HALF) {
                    for (int x = lane; x < HALF * D / 16; x += 32) {
                        const int row = x / (D / 16);
                        if (row < lo_row || row >= hi_row) reinterpret_cast<uint4 *>(vt)[x] = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
            }
            float acc[MT][NT][4];
#pragma unroll
            for (int d = 0; d < MT; d++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[d][nt][e] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < STEPS; kk++) {
                uint32_t va[VW], vb[VW], vc[VW], vd[VW];
                const uint8_t *row = vt + 16 * kk * D;
                if constexpr (D == 128) {
                    *reinterpret_cast<uint4 *>(va) = *reinterpret_cast<const uint4 *>(row + v_off0);
                    *reinterpret_cast<uint4 *>(vb) = *reinterpret_cast<const uint4 *>(row + v_off1);
                    *reinterpret_cast<uint4 *>(vc) = *reinterpret_cast<const uint4 *>(row + 8 * D + v_off0);
                    *reinterpret_cast<uint4 *>(vd) = *reinterpret_cast<const uint4 *>(row + 8 * D + v_off1);
                } else {
                    *reinterpret_cast<uint2 *>(va) = *reinterpret_cast<const uint2 *>(row + v_off0);
                    *reinterpret_cast<uint2 *>(vb) = *reinterpret_cast<const uint2 *>(row + v_off1);
                    *reinterpret_cast<uint2 *>(vc) = *reinterpret_cast<const uint2 *>(row + 8 * D + v_off0);
                    *reinterpret_cast<uint2 *>(vd) = *reinterpret_cast<const uint2 *>(row + 8 * D + v_off1);
                }
#pragma unroll
                for (int w = 0; w < VW; w++)
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        // Dimensions 4 w + 2 b, 4 w + 2 b + 1 of the lane's, two keys each.
                        uint32_t a0, a1, a2, a3;
                        pa_codes<FORMAT>(__byte_perm(va[w], vb[w], b ? 0x7362 : 0x5140), a0, a1);
                        pa_codes<FORMAT>(__byte_perm(vc[w], vd[w], b ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            pa_mma(acc[2 * w + b][nt], a0, a1, a2, a3, pf[kk][nt][0], pf[kk][nt][1]);
                    }
                if (kk == STEPS - 1 || ((half * STEPS + kk + 1) & ((1 << page_shift) - 1)) == 0) {
                    // The end of a page: its scale.
                    const float vs = sh.scales[slot][8 + ((half * STEPS + kk) >> page_shift)];
#pragma unroll
                    for (int d = 0; d < MT; d++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                o[d][nt][e] = fmaf(acc[d][nt][e], vs, o[d][nt][e]);
                                acc[d][nt][e] = 0.0f;
                            }
                }
            }
            if constexpr (FORMAT == FO_PAGED_E4M3) sm100::fence_proxy_async_smem();  // zeros before the next copy
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&sh.empty[slot]);
        }

        // Join the key groups' parts, an n8 tile at a time.
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float x = TERMS == 2 ? l[nt][0] : l[nt][h];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) {
                    sh.ml[warp][8 * nt + 2 * t + h][0] = ok ? m[nt][h] : NAN;
                    sh.ml[warp][8 * nt + 2 * t + h][1] = x;
                }
            }
        // The unit's tiles in the line, and the blocks that share it.
        const long long unit_begin = begin + i - at.tile, unit_end = unit_begin + at.w.tiles;
        const int c0 = (int)(unit_begin / per), c1 = (int)((unit_end - 1) / per);
        const int64_t part = 2 * (int64_t)blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0);
        auto write_out = [&](int qi, int quad, float4 v, float mm, float ll) {
            const int r = (q0 + qi) / a.group, h = head * a.group + (q0 + qi) - r * a.group;
            float sum = ll;
            if (a.sinks) sum += sm100::ex2(fmaf(__ldg(a.sinks + h), PA_LOG2E, PA_P_BITS - mm));
            const float inv = ll == 0.0f ? 0.0f : 1.0f / sum;
            T *out = static_cast<T *>(a.out.data) + (s.first + r) * a.out.row_stride + h * a.out.head_stride + 4 * quad;
            if (a.out_vec) {
                if constexpr (TERMS == 2)
                    *reinterpret_cast<float4 *>(out) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                else
                    *reinterpret_cast<uint2 *>(out) = make_uint2(bf16_pair(v.x * inv, v.y * inv), bf16_pair(v.z * inv, v.w * inv));
            } else {
                store1(out, v.x * inv);
                store1(out + 1, v.y * inv);
                store1(out + 2, v.z * inv);
                store1(out + 3, v.w * inv);
            }
            if (a.lse && quad == 0)
                a.lse[(s.first + r) * a.q.heads + h] = ll == 0.0f ? -INFINITY : (mm + log2f(ll) - PA_P_BITS) * PA_LN2;
        };
#pragma unroll
        for (int pass = 0; pass < NT * (D / 64); pass++) {
            // An n8 tile's columns, 64 dimensions of them.
            const int nt = pass / (D / 64), d64 = pass % (D / 64);
            if (D == 64 || g / 4 == d64) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float *col = comb + (warp * 8 + 2 * t + h) * Shape::COMB_LD + (D / 8) * g - 64 * d64;
#pragma unroll
                    for (int d = 0; d < MT; d += 2)
                        *reinterpret_cast<float4 *>(col + 2 * d) =
                            make_float4(o[d][nt][h], o[d][nt][2 + h], o[d + 1][nt][h], o[d + 1][nt][2 + h]);
                }
            }
            pa_consumers_sync();
            for (int x = tid; x < a.col_groups * QN * 16; x += 32 * PA_CONSUMERS) {
                const int quad = x % 16, cq = x / 16;
                const int cg = cq / QN, col = (cq - cg * QN) * TERMS;
                const int qi = query_of(nt, 0) + (cg - col_group) * WARP_QUERIES + col / TERMS;
                if (qi >= n_queries) continue;
                float mm = -INFINITY, ll = 0.0f;
                bool lost = false;
                for (int w = cg; w < PA_CONSUMERS; w += a.col_groups) {
                    const float mw = sh.ml[w][8 * nt + col][0];
                    lost |= mw != mw;
                    mm = fmaxf(mm, mw);
                }
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int w = cg; w < PA_CONSUMERS; w += a.col_groups) {
                    const float mw = sh.ml[w][8 * nt + col][0];
                    if (mw == -INFINITY) continue;
                    const float f = sm100::ex2(mw - mm);
                    ll = fmaf(sh.ml[w][8 * nt + col][1], f, ll);
                    const float *from = comb + (w * 8 + col) * Shape::COMB_LD + 4 * quad;
                    float4 u = *reinterpret_cast<const float4 *>(from);
                    if constexpr (TERMS == 2) {
                        const float4 u1 = *reinterpret_cast<const float4 *>(from + Shape::COMB_LD);
                        u = make_float4(u.x + u1.x, u.y + u1.y, u.z + u1.z, u.w + u1.w);
                    }
                    v = make_float4(fmaf(u.x, f, v.x), fmaf(u.y, f, v.y), fmaf(u.z, f, v.z), fmaf(u.w, f, v.w));
                }
                if (lost) ll = NAN;
                const int at_quad = 16 * d64 + quad;
                if (c0 == c1) {
                    write_out(qi, at_quad, v, mm, ll);
                } else {
                    *reinterpret_cast<float4 *>(a.part_o + (part * a.queries + qi) * D + 4 * at_quad) = v;
                    if (at_quad == 0)
                        *reinterpret_cast<float2 *>(a.part_ml + (part * a.queries + qi) * 2) = make_float2(mm, ll);
                }
            }
            pa_consumers_sync();
        }
        if (c0 != c1) {
            // The last block to come joins the parts in their order.
            if (tid == 0) {
                __threadfence();
                sh.last = atomicAdd(a.counters + c0, 1u) == (unsigned)(c1 - c0);
                if (sh.last) a.counters[c0] = 0;
                __threadfence();
            }
            pa_consumers_sync();
            if (sh.last) {
                for (int x = tid; x < n_queries * (D / 4); x += 32 * PA_CONSUMERS) {
                    const int quad = x % (D / 4), qi = x / (D / 4);
                    auto at_part = [&](int cta) { return ((2 * (int64_t)cta + (cta == c0 ? 1 : 0)) * a.queries + qi); };
                    float mm = -INFINITY, ll = 0.0f;
                    for (int cta = c0; cta <= c1; cta++)
                        mm = fmaxf(mm, __ldcg(reinterpret_cast<const float2 *>(a.part_ml) + at_part(cta)).x);
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int cta = c0; cta <= c1; cta++) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.part_ml) + at_part(cta));
                        const float4 u = __ldcg(reinterpret_cast<const float4 *>(a.part_o + at_part(cta) * D) + quad);
                        const float f = ml.x == -INFINITY ? 0.0f : sm100::ex2(ml.x - mm);
                        ll = fmaf(ml.y, f, ll);
                        v = make_float4(fmaf(u.x, f, v.x), fmaf(u.y, f, v.y), fmaf(u.z, f, v.z), fmaf(u.w, f, v.w));
                    }
                    write_out(qi, quad, v, mm, ll);
                }
            }
            pa_consumers_sync();
        }
        i += n;
        at.advance(a, n);
    }
}

PFN_cuTensorMapEncodeTiled_v12000 pa_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
    return fn;
}

// A pool's codes as rows of head_dim bytes, [pages][heads * page_size], copied
// a page's (or half of a 128-position page's) rows of one head at a time.
bool pa_map(CUtensorMap *map, const void *codes, const fo_paged_kv &kv) {
    auto fn = pa_encoder();
    if (!fn) return false;
    const cuuint64_t rows = (cuuint64_t)kv.n_kv_heads * kv.page_size;
    cuuint64_t dims[3] = {(cuuint64_t)kv.head_dim, rows, (cuuint64_t)kv.n_pages};
    cuuint64_t strides[2] = {(cuuint64_t)kv.head_dim, rows * kv.head_dim};
    cuuint32_t box[3] = {(cuuint32_t)kv.head_dim, (cuuint32_t)std::min<int>(kv.page_size, 8192 / kv.head_dim), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(codes), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, kv.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int FORMAT, int NT, int TERMS>
cudaError_t launch_attention(const fo_paged_attention_launch &a, unsigned grid, cudaStream_t stream) {
    auto *kernel = paged_attention_kernel<D, FORMAT, NT, TERMS>;
    // The attribute belongs to each device's context: set once per device.
    static std::atomic<unsigned long long> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PaShape<D>::SMEM);
        if (e != cudaSuccess) return e;
        // The kernel's register split is only sound at the launch count that it
        // was written for.
        cudaFuncAttributes f;
        e = cudaFuncGetAttributes(&f, kernel);
        if (e != cudaSuccess) return e;
        if (f.numRegs != PA_LAUNCH_REGS) return cudaErrorInvalidConfiguration;
        configured.fetch_or(bit);
    }
    CUtensorMap k_map, v_map;
    if (!pa_map(&k_map, a.kv.k_codes, a.kv) || !pa_map(&v_map, a.kv.v_codes, a.kv)) return cudaErrorNotSupported;
    kernel<<<grid, PA_THREADS, PaShape<D>::SMEM, stream>>>(k_map, v_map, a);
    return cudaGetLastError();
}

template <int D, int FORMAT>
cudaError_t launch_attention(const fo_paged_attention_launch &a, int nt, unsigned grid, cudaStream_t stream) {
    if (a.q.dtype == FO_DT_F32)
        return nt == 1 ? launch_attention<D, FORMAT, 1, 2>(a, grid, stream) : launch_attention<D, FORMAT, 2, 2>(a, grid, stream);
    return nt == 1 ? launch_attention<D, FORMAT, 1, 1>(a, grid, stream) : launch_attention<D, FORMAT, 2, 1>(a, grid, stream);
}

}  // namespace fo

extern "C" cudaError_t fo_launch_paged_attention(const fo_paged_attention_launch *args, int sms, cudaStream_t stream) {
    fo_paged_attention_launch a = *args;
    if (a.batch.total_rows <= 0) return cudaSuccess;
    a.group = a.q.heads / a.kv.n_kv_heads;
    // Columns of the products: a query's, times its terms.  A warp takes 8, or
    // 16; beyond that 2 or 4 warps share each tile; beyond that a (sequence, KV
    // head) is read once for each group of queries.
    const int terms = a.q.dtype == FO_DT_F32 ? 2 : 1;
    const int64_t columns = a.batch.max_rows * a.group * terms;
    const int nt = columns <= 8 ? 1 : 2;
    a.col_groups = columns <= 16 ? 1 : columns <= 32 ? 2 : 4;
    a.queries = 8 * nt * a.col_groups / terms;
    a.evict_first = columns <= 64;
    auto aligned = [](const fo_rows &r, int64_t bytes) {
        const int64_t unit = bytes / (r.dtype == FO_DT_F32 ? 4 : 2);
        return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    a.q_vec = aligned(a.q, 16);
    a.out_vec = aligned(a.out, terms == 2 ? 16 : 8);
    // No more blocks than the most tiles there can be for, one for each group
    // of consumer warps.
    const int64_t most = a.batch.n_seqs * a.kv.n_kv_heads * ((columns / terms + a.queries - 1) / a.queries) *
                         ((a.batch.table_stride * a.kv.page_size * a.kv.head_dim + 8191) / 8192);
    const int64_t groups = fo::PA_CONSUMERS / 2 / a.col_groups;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(sms, (most + groups - 1) / groups));
    if (a.kv.head_dim == 64)
        return a.kv.format == FO_PAGED_I8 ? fo::launch_attention<64, FO_PAGED_I8>(a, nt, grid, stream)
                                          : fo::launch_attention<64, FO_PAGED_E4M3>(a, nt, grid, stream);
    return a.kv.format == FO_PAGED_I8 ? fo::launch_attention<128, FO_PAGED_I8>(a, nt, grid, stream)
                                      : fo::launch_attention<128, FO_PAGED_E4M3>(a, nt, grid, stream);
}
