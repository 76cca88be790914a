// paged_attention.cuh -- attention of a batch's query rows over a paged 8-bit
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
// In a block two producer warps walk the page table a step ahead and copy
// tiles into a ring in shared memory with TMA (swizzled, so that the reads
// below meet no bank conflicts); twelve consumer warps, two to a tile, a half
// each, take tiles in turn, each with its own running maximum and sum; and two
// epilogue warps split the next (sequence, KV head)'s queries into operands
// while the consumers are at this one's, join the consumers' parts, and write
// or hand on the result, so that the consumers go from one to the next
// without waiting for any of that.
//
// The codes are the A operands of tensor instructions, keys as they lie, values
// through transposing shared-memory loads: a consumer computes S^T = K Q^T and
// O^T += V^T P^T.  Nothing of the cache is rounded; a scale multiplies a
// finished sum.
//   int8: m16n8k32 products of bytes with exact 32-bit sums, one for each byte
//   of a query and of a probability.  A query is a 23-bit integer relative to a
//   power of two near its largest element: within 2^-22 of that one, and exactly a
//   BF16 query's element where it is at least 2^-14 of the largest.  (16 bits for BF16
//   rows, one product of three fewer, take 282 us instead of 303 at 40 queries to a
//   KV head and 89 instead of 91 at two, but next to one large element the scores
//   lose what BF16 holds.)
//   A probability is an integer of 16 bits (BF16 rows, whose output has 8), or
//   23, relative to its half tile's largest.  Where a few keys are so large that
//   half or more of a query's lanes have none of 2^-8 of the largest (a text's
//   first tokens often take most of the softmax, with values near zero),
//   what the integers leave is multiplied too, in a second set of products: each
//   probability then keeps 8 bits, or 15, of its own down to 2^-24 of the largest.
//   (Looking for that takes 2 us of 93 where HBM bounds the call.)
//   e4m3: m16n8k16 products of FP16, which holds every e4m3 number.  (With
//   m16n8k32 products of e4m3, two terms to a query and three to a probability,
//   an earlier form took 124 us for 64 sequences of 7,500, and 97 with FP16,
//   although in isolation that instruction takes 4.3 cycles, this one 8.0.)  A
//   query is relative to a power of two near its largest element: BF16's 8 bits exactly, FP32 as the
//   sum of two FP16 (22 bits); a probability, times 2^10 so that FP16 holds
//   those down to 2^-24 of the largest at full precision, is one FP16 (11 bits)
//   or two.
// The 5th-generation MMA would want the few queries' side padded and every
// score and output moved through TMEM; at a decode's few columns these
// instructions take a small part of the time that HBM needs for a tile.
// Maxima, sums and outputs are FP32.
//
// Measured (CUDA graph): 64 sequences of 6,545 to 8,592 positions, 2 queries to
// each of 8 KV heads of 64, int8: 86 us, 5.7 TB/s, 0.89 of the measured copy
// bandwidth; 16 of 1,000 to 32,768, 4 queries, heads of 128, e4m3: 112 us, 6.0
// TB/s.  Earlier forms, 64 sequences of 7,500 in a stream of calls: one
// producer warp 165 us; four, with int8 converted to FP16 for m16n8k16 products,
// 110; products of the codes themselves, parts joined by the consumers, 103; by
// epilogue warps, 95.  With 40 queries to a KV head (10 of the 12 consumer warps
// at one tile) a tile takes some 7,200 warp instructions, at 36 % of the issue slots
// with the tensor pipe at 13 %: 304 us for 48 sequences in a window of 4,096, 1.2
// TB/s.  A call of one short sequence takes 9.7 us, a chain of launch, length, page
// number, tile and join.  Spills: 0 to 88 bytes of stores in a variant.
//
// With LOST (paged_attention_window.cu) a page whose number is outside the pool, or
// that has a scale that is not finite, makes NaN of the rows that see it and of no
// others; without, a page number does of all rows of its unit.  (A flag in the
// arguments in place of the variant: one short sequence 9.8 us for 9.6, a serving
// step 31.7 for 30.8.)  64 sequences in a window of 4,096, 2 query rows to each of
// 8 KV heads of 64, int8: 55 us either way.
// With REACH too (paged_attention_reach.cu) a row also sees a few first positions
// behind its window, whose tiles come before the window's in the line.  Those 64
// sequences with 16 first positions: 57.4 us against a floor of 41; a unit's change
// costs some 3 us and a unit here is short.
#pragma once

#include "paged.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <atomic>
#include <cudaTypedefs.h>

namespace fo {

constexpr int PA_CONSUMERS = 12;  // consumer warps
constexpr int PA_PRODUCERS = 2;   // producer warps
constexpr int PA_EPILOGUES = 2;   // epilogue warps
constexpr int PA_STAGES = 8;      // tiles in the ring
// A parity wait cannot tell a barrier's phase from the one two before it, so
// every slot is filled by one producer warp only, which passes the phases of
// its empty barrier one by one; a consumer, whose slots others use too, first
// sees the slot's tile number, which is written once the phase before the
// tile's own is over.
static_assert(PA_STAGES % PA_PRODUCERS == 0, "owners of the ring's slots");
constexpr int PA_THREADS = 32 * (PA_CONSUMERS + PA_PRODUCERS + PA_EPILOGUES);
// Registers a thread: launched with 128 (65,536 over 512 threads), the
// producers' and epilogues' warpgroup gives up what the consumers' three take:
// 128 * 104 + 384 * 136 = 512 * 128.
constexpr int PA_LAUNCH_REGS = 128, PA_OTHER_REGS = 104, PA_CONSUMER_REGS = 136;
static_assert(128 * PA_OTHER_REGS + 384 * PA_CONSUMER_REGS == PA_THREADS * PA_LAUNCH_REGS, "register split");
constexpr float PA_LOG2E = 1.4426950408889634f, PA_LN2 = 0.6931471805599453f;

template <int D, int FORMAT, bool F32>
struct PaShape {
    static constexpr int TILE_BYTES = 8192;        // of keys, and of values
    static constexpr int TILE = TILE_BYTES / D;    // positions
    static constexpr int HALF = TILE / 2;          // a consumer warp's
    static constexpr int STAGE = 2 * TILE_BYTES;
    static constexpr bool I8 = FORMAT == FO_PAGED_I8;
    static constexpr int QT = I8 ? 3 : 1 + F32;    // a query's terms
    static constexpr int PT = (I8 ? 2 : 1) + F32;  // a probability's
    static constexpr int KQ = I8 ? D / 32 : D / 16;          // k steps over a row's elements
    static constexpr int PART_LD = D + 4;          // a column of a consumer's part, in floats
    static constexpr int PARTS = PA_CONSUMERS * 8 * PART_LD * 4;
    static constexpr int REST = I8 ? PT * (HALF / 16) * 128 : 0;  // a warp's second set of probabilities
    static constexpr int Q_TILE = QT * KQ * 32 * 8;  // an n8 tile of queries as operands
    static constexpr int smem(int q_tiles) {
        return 1024 + PA_STAGES * STAGE + PARTS + PA_CONSUMERS * REST + q_tiles * Q_TILE;
    }
};

// The key of eight that a fragment's row g stands for: such that a K
// fragment's reads fall into different banks under the tile's swizzle (128-byte
// rows: 128-byte swizzle; 64-byte rows: 64-byte).  Rows 8 .. 15 of a fragment
// stand for the keys 8 + pa_key(g ^ 4), so that the eight rows of a V load do too.
template <int D>
__host__ __device__ constexpr int pa_key(int g) {
    return D == 128 ? g >> 1 | (g & 1) << 2 : g;
}

// Accumulators of int8 products start at 1.5 * 2^23's bits, so that read as
// floats they are 1.5 * 2^23 + sum (sums here stay below 2^22).
constexpr uint32_t PA_MAGIC = 0x4B400000u;
constexpr float PA_MAGIC_F = 12582912.0f;

// c += a b, a m16 x k32, b k32 x n8: int8 codes by signed or unsigned bytes.
template <bool SIGNED>
__device__ __forceinline__ void pa_imma(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    if constexpr (SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with FP16, k16.
__device__ __forceinline__ void pa_hmma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two 16 x 16 matrices of bytes, transposed: lanes 0 .. 15 give the addresses
// of the first one's rows, 16 .. 31 of the second's; r[0] and r[1] are its
// columns g and g + 8, rows 4 t .. 4 t + 3.
__device__ __forceinline__ void pa_load_transposed(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address));
}
// An 8 x 8 matrix of 16-bit elements, two per lane along a row, transposed.
__device__ __forceinline__ uint32_t pa_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// (The largest number in place of infinity: of maxima beyond 2^27, 2^10 less is
// rounded to 2^16 less, for which FP16 has no room.)
__device__ __forceinline__ uint32_t pa_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// A sequence's share of the line of tiles.
struct PaWork {
    Sequence s;
    int low;     // first position that any of its rows sees
    int t0;      // its tile
    int tiles;   // per KV head and group of queries (one at least, so that rows that see nothing are written)
    int groups;  // groups of `queries` queries
};
// Tiles of the first positions, which come before tile t0 in the line.
template <int TILE>
__device__ __forceinline__ int pa_early(const fo_paged_attention_launch &a, const PaWork &w) {
    return min((int)(((unsigned)min(a.reach.first, w.s.len) + TILE - 1) / TILE), w.t0);
}
// The tile of the sequence that is number i of a unit's.
template <int TILE, bool REACH>
__device__ __forceinline__ int pa_tile(const fo_paged_attention_launch &a, const PaWork &w, int i) {
    if constexpr (REACH) {
        const int early = pa_early<TILE>(a, w);
        if (i < early) return i;
        return w.t0 + i - early;
    }
    return w.t0 + i;
}
template <int TILE, bool REACH>
__device__ __forceinline__ PaWork pa_work(const fo_paged_attention_launch &a, int seq) {
    PaWork w;
    w.s = load_sequence(a.batch, a.kv.page_size, seq, a.err);
    const int p0 = max(w.s.len - w.s.n, 0);
    w.low = a.window > 0 ? max(p0 + 1 - a.window, 0) : 0;
    w.t0 = w.low / TILE;
    w.tiles = (int)(((unsigned)w.s.len + TILE - 1) / TILE) - w.t0;
    if constexpr (REACH) w.tiles += pa_early<TILE>(a, w);
    w.tiles = max(w.tiles, 1);
    const int queries = w.s.n * a.group;
    if (REACH && a.reach.few > 0 && queries > a.reach.few) {
        w.groups = 0;
        return w;
    }
    w.groups = queries <= a.queries ? queries > 0 : (queries + FO_PAGED_QUERIES - 1) / FO_PAGED_QUERIES;
    return w;
}

// A place in the line: a sequence, a unit of it (KV head, group of queries)
// and a tile of the unit.
template <int TILE, bool REACH>
struct PaCursor {
    PaWork w;
    int seq, unit, tile;
    __device__ __forceinline__ int head() const { return w.groups == 1 ? unit : unit / w.groups; }
    __device__ __forceinline__ int group() const { return w.groups == 1 ? 0 : unit % w.groups; }
    __device__ __forceinline__ int left() const { return w.tiles - tile; }
    // Moves on by n tiles, at most to the unit's end.
    __device__ __forceinline__ void advance(const fo_paged_attention_launch &a, int n) {
        tile += n;
        if (tile < w.tiles) return;
        tile = 0;
        if (++unit < a.kv.n_kv_heads * w.groups) return;
        unit = 0;
        do {
            if (++seq >= (int)a.batch.n_seqs) return;
            w = pa_work<TILE, REACH>(a, seq);
        } while (w.groups == 0);
    }
};

// Where a consumer warp is.  It waits in shared memory while the warp goes
// through a segment's tiles, which want its registers.
template <int TILE, bool REACH>
struct PaPlace {
    PaCursor<TILE, REACH> at;
    int begin, per;
};

struct PaShared {
    uint64_t full[PA_STAGES], empty[PA_STAGES];
    uint64_t q_full, q_free;        // a segment's queries are there; have been taken
    uint64_t part_full, part_free;  // its parts
    // Of a unit that other blocks share, at the block's last segment (1) or its
    // first one: its part is in scratch; whether this block joins them is known.
    uint64_t shared_ready[2], shared_go[2];
    int joins[2];
    float scales[PA_STAGES][16];    // keys' of a tile's pages, then values'
    int tile[PA_STAGES];            // the block's number of the tile in a slot
    float ml[PA_CONSUMERS][8][2];
    float q_scale[FO_PAGED_QUERIES];
    int q_pos[FO_PAGED_QUERIES];
    int2 warp_sum[PA_THREADS / 32];
    int begin_base, begin_seq, abort;
    int places[PA_CONSUMERS][12];  // a consumer warp's PaPlace
};

// Waits for the block's tile k in its slot; false when the block gave up.  The
// first wait may have been for the phase two before; the tile's number says
// that the one before is over, and the second wait is for the tile's own.
__device__ __forceinline__ bool pa_wait_tile(PaShared &sh, int slot, int k, unsigned *err) {
    const uint32_t phase = (k / PA_STAGES) & 1;
    uint64_t t0 = 0;
    for (uint32_t it = 1;; ++it) {
        if (!sm100::mbar_wait(&sh.full[slot], phase, &sh.abort, err)) return false;
        if (*(volatile int *)&sh.tile[slot] == k) return sm100::mbar_wait(&sh.full[slot], phase, &sh.abort, err);
        if ((it & 63) != 0) continue;
        if (*(volatile int *)&sh.abort) return false;
        if (t0 == 0) t0 = sm100::globaltimer();
        if (sm100::globaltimer() - t0 > FO_WAIT_NS) {
            *(volatile int *)&sh.abort = 1;
            atomicOr(err, FO_DEVERR_WAIT_TIMEOUT);
            return false;
        }
    }
}

// Sum of x over the block's earlier threads; `all` the whole block's.
__device__ __forceinline__ int2 pa_scan(int2 x, PaShared &sh, int2 &all) {
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
#pragma unroll 4
    for (int w = 0; w < PA_THREADS / 32; w++) {
        const int2 y = sh.warp_sum[w];
        if (w < warp) before.x += y.x, before.y += y.y;
        all.x += y.x, all.y += y.y;
    }
    return before;
}

// A unit's queries and the blocks [c0, c1] that share its tiles in the line.
struct PaUnit {
    int first;  // the sequence's first row
    int head, q0, n_queries, c0, c1;
    bool alone;
    // Scratch of block `cta`'s part (a block shares two units at most: the one it
    // begins in, and the one that begins in it).
    __device__ __forceinline__ int64_t part(const fo_paged_attention_launch &a, int cta, int qi) const {
        return (2 * (int64_t)cta + (cta == c0 ? 1 : 0)) * a.queries + qi;
    }
};
template <int TILE, bool REACH>
__device__ __forceinline__ PaUnit pa_unit(const fo_paged_attention_launch &a, const PaCursor<TILE, REACH> &at, int at_line,
                                          int n, int per) {
    PaUnit u;
    u.first = at.w.s.first;
    u.head = at.head();
    u.q0 = at.group() * a.queries;
    u.n_queries = min(at.w.s.n * a.group - u.q0, a.queries);
    u.alone = at.tile == 0 && n == at.w.tiles;
    u.c0 = u.c1 = blockIdx.x;
    if (!u.alone) {
        const int begin = at_line - at.tile;
        u.c0 = begin / per;
        u.c1 = (begin + at.w.tiles - 1) / per;
    }
    return u;
}

// Four dimensions of a query's output from their sum v, the sum ll of the
// probabilities and the maximum mm that both are relative to.
template <int D, bool F32>
__device__ __forceinline__ void pa_write(const fo_paged_attention_launch &a, const PaUnit &u, int qi, int quad, float4 v,
                                         float mm, float ll) {
    using T = typename std::conditional<F32, float, uint16_t>::type;
    const int q = u.q0 + qi, r = q / a.group, h = u.head * a.group + q - r * a.group;
    float sum = ll;
    if (a.sinks) sum += sm100::ex2(fmaf(a.sinks[h], PA_LOG2E, -mm));
    const float inv = ll == 0.0f ? 0.0f : 1.0f / sum;
    v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    T *out = static_cast<T *>(a.out.data) + (int64_t)(u.first + r) * a.out.row_stride + h * a.out.head_stride + 4 * quad;
    if (!a.out_vec) {
        store1(out, v.x);
        store1(out + 1, v.y);
        store1(out + 2, v.z);
        store1(out + 3, v.w);
    } else if constexpr (F32) {
        *reinterpret_cast<float4 *>(out) = v;
    } else {
        *reinterpret_cast<uint2 *>(out) = make_uint2(bf16_pair(v.x, v.y), bf16_pair(v.z, v.w));
    }
    if (a.lse && quad == 0) a.lse[(int64_t)(u.first + r) * a.q.heads + h] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * PA_LN2;
}

// The blocks' parts of a unit joined in their order, by warp `rank` of `warps`
// (all of them in the last block to come), a query at a time: the maxima and
// sums a block to a lane, then four dimensions to a lane.
template <int D, bool F32>
__device__ __forceinline__ void pa_join_blocks(const fo_paged_attention_launch &a, const PaUnit &u, int rank, int warps) {
    constexpr int QUADS = D / 4, SETS = 32 / QUADS;  // lanes that share a quad take every SETS-th block
    const int lane = threadIdx.x & 31, quad = lane % QUADS, set = lane / QUADS;
    const int n = u.c1 - u.c0 + 1;
    const float2 *mls = reinterpret_cast<const float2 *>(a.part_ml);
    for (int qi = rank; qi < u.n_queries; qi += warps) {
        float mm = -INFINITY;
        bool lost = false;
        for (int j = lane; j < n; j += 32) {
            const float2 ml = __ldcg(mls + u.part(a, u.c0 + j, qi));
            lost |= ml.y != ml.y;
            mm = fmaxf(mm, ml.x);
        }
        mm = warp_max(mm);
        lost = __any_sync(0xffffffffu, lost);
        float ll = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int j0 = 0; j0 < n; j0 += 32) {
            float f = 0.0f;
            if (j0 + lane < n) {
                const float2 ml = __ldcg(mls + u.part(a, u.c0 + j0 + lane, qi));
                if (ml.x != -INFINITY) f = sm100::ex2(ml.x - mm);
                ll = fmaf(ml.y, f, ll);
            }
            const int most = min(32, n - j0);
#pragma unroll 8
            for (int j = 0; j < most; j += SETS) {
                const float fj = __shfl_sync(0xffffffffu, f, j + set);
                if (j + set < most && fj != 0.0f) {
                    const float4 x =
                        __ldcg(reinterpret_cast<const float4 *>(a.part_o + u.part(a, u.c0 + j0 + j + set, qi) * D) + quad);
                    v = make_float4(fmaf(x.x, fj, v.x), fmaf(x.y, fj, v.y), fmaf(x.z, fj, v.z), fmaf(x.w, fj, v.w));
                }
            }
        }
        ll = warp_sum(ll);
        if constexpr (SETS == 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
        }
        if (set == 0) pa_write<D, F32>(a, u, qi, quad, v, mm, lost ? NAN : ll);
    }
}

// The epilogue warps: `me` of PA_EPILOGUES takes every PA_EPILOGUES-th n8 tile of
// queries to split into operands, and every such query to join and write.
template <int D, int FORMAT, bool F32, int TILE, bool REACH>
__device__ __forceinline__ void pa_epilogue(const fo_paged_attention_launch &a, PaShared &sh, PaCursor<TILE, REACH> at, int count,
                                            int begin, int per, int me, float *parts, uint2 *q_ops) {
    using Shape = PaShape<D, FORMAT, F32>;
    using T = typename std::conditional<F32, float, uint16_t>::type;
    constexpr bool I8 = FORMAT == FO_PAGED_I8;
    constexpr int QT = Shape::QT, KQ = Shape::KQ;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    // A unit's queries as B operands: column g of an n8 tile, this lane's elements
    // 16 t .. 16 t + 15 of each 64.
    auto split = [&](const PaCursor<TILE, REACH> &u) {
        const int q0 = u.group() * a.queries, head = u.head();
        const int n_queries = min(u.w.s.n * a.group - q0, a.queries);
        for (int tile = me; tile * 8 < n_queries; tile += PA_EPILOGUES) {
            const int qi = tile * 8 + g;
            const T *q = nullptr;
            int r = 0;
            if (qi < n_queries) {
                r = (q0 + qi) / a.group;
                q = static_cast<const T *>(a.q.data) + (int64_t)(u.w.s.first + r) * a.q.row_stride +
                    (head * a.group + (q0 + qi) - r * a.group) * a.q.head_stride + 16 * t;
            }
            // Read twice, 16 elements at a time: the largest first.
            auto load = [&](int c, float (&x)[16]) {
                if (!q) {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = 0.0f;
                } else if (a.q_vec) {
                    load8(q + 64 * c, x);
                    load8(q + 64 * c + 8, x + 8);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = load1(q + 64 * c + e);
                }
            };
            float top = 0.0f;
            bool finite = true;
#pragma unroll
            for (int c = 0; c < D / 64; c++) {
                float x[16];
                load(c, x);
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    top = fmaxf(top, fabsf(x[e]));
                    finite &= fabsf(x[e]) <= FLT_MAX;
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const unsigned all_finite = __ballot_sync(0xffffffffu, finite);
            // A power of two near the largest element brings it to [2^21, 2^22)
            // (int8) or [1, 2) (e4m3); in two factors, so that FP32's whole range
            // of exponents can be brought there.
            const int e = max((int)(__float_as_uint(top) >> 23), 1);
            const float up = I8 ? 2097152.0f : 1.0f;
            const float inv0 = __uint_as_float((uint32_t)(254 - (e + 1) / 2 - 63) << 23);
            const float inv1 = __uint_as_float((uint32_t)(254 - (e - (e + 1) / 2) - 64) << 23) * up;
            if (t == 0) {
                const bool good = (all_finite >> (lane & 28) & 15) == 15;
                sh.q_scale[qi] = good ? __uint_as_float((uint32_t)e << 23) / up * a.scale * PA_LOG2E : NAN;
                sh.q_pos[qi] = q ? u.w.s.len - u.w.s.n + r : -1;
            }
            uint2 *to = q_ops + tile * (Shape::Q_TILE / 8) + lane;
#pragma unroll 1
            for (int c = 0; c < D / 64; c++) {
                float x[16];
                load(c, x);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    // Elements 4 w .. 4 w + 3.
                    float y[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) y[i] = x[4 * w + i] * inv0 * inv1;
                    if constexpr (I8) {
                        // Step 2 c + w / 2, register w % 2.
                        uint32_t z[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) z[i] = (uint32_t)__float2int_rn(y[i]);
                        const uint32_t lo01 = __byte_perm(z[0], z[1], 0x5140), lo23 = __byte_perm(z[2], z[3], 0x5140);
                        const uint32_t hi01 = __byte_perm(z[0], z[1], 0x0062), hi23 = __byte_perm(z[2], z[3], 0x0062);
                        // The highest byte, which is signed, first.
                        const uint32_t f[3] = {__byte_perm(hi01, hi23, 0x5410), __byte_perm(lo01, lo23, 0x7632),
                                               __byte_perm(lo01, lo23, 0x5410)};
#pragma unroll
                        for (int i = 0; i < QT; i++)
                            reinterpret_cast<uint32_t *>(to + (i * KQ + 2 * c + w / 2) * 32)[w % 2] = f[i];
                    } else {
                        // Step 4 c + w.
#pragma unroll
                        for (int i = 0; i < QT; i++) {
                            const uint32_t f0 = pa_f16x2(y[0], y[1]), f1 = pa_f16x2(y[2], y[3]);
                            to[(i * KQ + 4 * c + w) * 32] = make_uint2(f0, f1);
                            const float2 b0 = f16x2_f32x2(f0), b1 = f16x2_f32x2(f1);
                            y[0] -= b0.x, y[1] -= b0.y, y[2] -= b1.x, y[3] -= b1.y;
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&sh.q_full);
    };

    PaCursor<TILE, REACH> next = at;
    int next_i = 0;
    split(next);
    for (int i = 0, segment = 0; i < count; segment++) {
        const int n = min(at.left(), count - i);
        // The next unit's queries.
        next_i += n;
        next.advance(a, n);
        if (next_i < count) {
            if (!sm100::mbar_wait(&sh.q_free, segment & 1, &sh.abort, a.err)) return;
            split(next);
        }
        const PaUnit u = pa_unit(a, at, begin + i, n, per);
        if (!sm100::mbar_wait(&sh.part_full, segment & 1, &sh.abort, a.err)) return;
        // The consumers' parts of one query, four dimensions at a time.
        for (int x = lane; x < (u.n_queries - me + PA_EPILOGUES - 1) / PA_EPILOGUES * (D / 4); x += 32) {
            const int quad = x % (D / 4), qi = x / (D / 4) * PA_EPILOGUES + me;
            const int cg = qi / 8, col = qi % 8;
            float mm = -INFINITY, ll = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            bool lost = false;
#pragma unroll 4
            for (int w = cg; w < PA_CONSUMERS; w += a.col_groups) {
                const float2 ml = *reinterpret_cast<const float2 *>(sh.ml[w][col]);
                lost |= ml.y != ml.y;
                mm = fmaxf(mm, ml.x);
            }
#pragma unroll 4
            for (int w = cg; w < PA_CONSUMERS; w += a.col_groups) {
                const float2 ml = *reinterpret_cast<const float2 *>(sh.ml[w][col]);
                if (ml.x == -INFINITY) continue;  // it has seen nothing, and left no output
                const float4 z = *reinterpret_cast<const float4 *>(parts + (w * 8 + col) * Shape::PART_LD + 4 * quad);
                const float f = sm100::ex2(ml.x - mm);
                ll = fmaf(ml.y, f, ll);
                v = make_float4(fmaf(z.x, f, v.x), fmaf(z.y, f, v.y), fmaf(z.z, f, v.z), fmaf(z.w, f, v.w));
            }
            if (lost) ll = NAN;
            if (u.alone) {
                pa_write<D, F32>(a, u, qi, quad, v, mm, ll);
            } else {
                const int64_t at_me = u.part(a, blockIdx.x, qi);
                __stcg(reinterpret_cast<float4 *>(a.part_o + at_me * D) + quad, v);
                if (quad == 0) __stcg(reinterpret_cast<float2 *>(a.part_ml) + at_me, make_float2(mm, ll));
            }
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&sh.part_free);
        if (!u.alone) {
            // The last block to come (the unit's counter says so) joins the parts: with
            // all its warps when this was its last segment, else with these two.
            const int last = i + n == count;
            __threadfence();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&sh.shared_ready[last]);
            if (me == 0) {
                if (!sm100::mbar_wait(&sh.shared_ready[last], 0, &sh.abort, a.err)) return;
                if (lane == 0) {
                    __threadfence();
                    const bool joins = atomicAdd(a.counters + u.c0, 1u) == (unsigned)(u.c1 - u.c0);
                    if (joins) a.counters[u.c0] = 0;
                    __threadfence();
                    sh.joins[last] = joins;
                    sm100::mbar_arrive(&sh.shared_go[last]);
                }
                __syncwarp();
            }
            if (!sm100::mbar_wait(&sh.shared_go[last], 0, &sh.abort, a.err)) return;
            if (sh.joins[last])
                pa_join_blocks<D, F32>(a, u, me, last ? PA_EPILOGUES + PA_CONSUMERS : PA_EPILOGUES);
        }
        i += n;
        at.advance(a, n);
    }
}

template <int D, int FORMAT, bool F32, bool REACH, bool LOST>
__global__ void __launch_bounds__(PA_THREADS, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                           const __grid_constant__ fo_paged_attention_launch a) {
    using Shape = PaShape<D, FORMAT, F32>;
    constexpr int STAGES = PA_STAGES;
    constexpr int TILE = Shape::TILE, HALF = Shape::HALF;
    constexpr int STEPS = HALF / 16;   // m16 steps of a consumer's half
    constexpr int KW = D / 16;         // words of a K row per lane
    constexpr int VS = HALF / 32;      // pairs of V loads over a half's keys, 32 keys each
    constexpr int MT = D / 16;         // m16 tiles of the output's dimensions
    constexpr bool I8 = FORMAT == FO_PAGED_I8;
    constexpr int QT = Shape::QT, PT = Shape::PT, KQ = Shape::KQ;
    // The queries' operands stay in registers where there is room, and are read
    // for each tile otherwise.
    constexpr bool Q_REGS = QT * KQ <= (I8 ? 6 : 8);
    extern __shared__ uint8_t pa_smem[];
    __shared__ PaShared sh;
    uint8_t *tiles = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pa_smem) + 1023) & ~uintptr_t(1023));
    float *parts = reinterpret_cast<float *>(tiles + STAGES * Shape::STAGE);
    uint32_t *rests = reinterpret_cast<uint32_t *>(tiles + STAGES * Shape::STAGE + Shape::PARTS);
    uint2 *q_ops = reinterpret_cast<uint2 *>(tiles + STAGES * Shape::STAGE + Shape::PARTS + PA_CONSUMERS * Shape::REST);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int key_groups = PA_CONSUMERS / 2 / a.col_groups;

    if (warp == PA_THREADS / 32 - 1) {
        if (lane < STAGES) {
            sm100::mbar_init(&sh.full[lane], 1);
            sm100::mbar_init(&sh.empty[lane], 2 * a.col_groups);
            sh.tile[lane] = -1;
        }
        if (lane == 8) sm100::mbar_init(&sh.q_full, PA_EPILOGUES), sm100::mbar_init(&sh.part_free, PA_EPILOGUES);
        if (lane == 9) sm100::mbar_init(&sh.q_free, PA_CONSUMERS), sm100::mbar_init(&sh.part_full, PA_CONSUMERS);
        if (lane == 10 || lane == 11) {
            sm100::mbar_init(&sh.shared_ready[lane - 10], PA_EPILOGUES);
            sm100::mbar_init(&sh.shared_go[lane - 10], 1);
        }
        sm100::mbar_fence_init();
        if (lane == 12) sh.abort = 0;
    }
    wait_for_prior_kernel();
    // This block's piece [begin, end) of the line, and where it begins.  (The
    // line's tiles are below 2^31, checked on the host.)
    // No more units than blocks, and short ones: a block for each, since handing a
    // part on to another block takes longer (about 4 us) than these tiles.
    const int n_seqs = (int)a.batch.n_seqs, few = 4 * key_groups;
    PaCursor<TILE, REACH> at;
    int per = 0, begin = 0, end, base;
    bool whole = false;
    auto work_of = [&](int seq, PaWork &w) {  // its tiles and units
        if (seq >= n_seqs) return make_int2(0, 0);
        w = pa_work<TILE, REACH>(a, seq);
        const int units = w.groups * a.kv.n_kv_heads;
        return make_int2(w.tiles * units, units);
    };
    if (n_seqs <= 32) {
        // Every warp for itself, a sequence to a lane.
        PaWork w = {};
        const int2 mine = work_of(lane, w);
        int2 sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum.x, o), v = __shfl_up_sync(0xffffffffu, sum.y, o);
            if (lane >= o) sum.x += u, sum.y += v;
        }
        const int2 all = make_int2(__shfl_sync(0xffffffffu, sum.x, 31), __shfl_sync(0xffffffffu, sum.y, 31));
        whole = a.whole_units && __all_sync(0xffffffffu, mine.y == 0 || w.tiles <= few);
        if (!whole) {
            per = max((int)((unsigned)(all.x + gridDim.x - 1) / gridDim.x), key_groups);
            begin = (int)min((long long)per * blockIdx.x, (long long)all.x);
        }
        end = whole ? all.y : (int)min((long long)begin + per, (long long)all.x);
        if (whole ? (int)blockIdx.x >= end : begin >= end) return;
        const int at_line = whole ? (int)blockIdx.x : begin, before = whole ? sum.y - mine.y : sum.x - mine.x;
        const int own = __ffs(__ballot_sync(0xffffffffu, at_line >= before && at_line < before + (whole ? mine.y : mine.x))) - 1;
        at.seq = own;
        base = __shfl_sync(0xffffffffu, before, own);
        at.w.s.first = __shfl_sync(0xffffffffu, w.s.first, own);
        at.w.s.len = __shfl_sync(0xffffffffu, w.s.len, own);
        at.w.s.n = __shfl_sync(0xffffffffu, w.s.n, own);
        at.w.low = __shfl_sync(0xffffffffu, w.low, own);
        at.w.t0 = __shfl_sync(0xffffffffu, w.t0, own);
        at.w.tiles = __shfl_sync(0xffffffffu, w.tiles, own);
        at.w.groups = __shfl_sync(0xffffffffu, w.groups, own);
        __syncthreads();  // the barriers are there
    } else {
        PaWork w = {};
        int2 all, mine = work_of(tid, w), before = pa_scan(mine, sh, all), chunk = all;
        whole = a.whole_units && __syncthreads_and(mine.y == 0 || w.tiles <= few);
        for (int first = PA_THREADS; first < n_seqs; first += PA_THREADS) {
            int2 more;
            pa_scan(work_of(first + tid, w), sh, more);
            all.x += more.x;
        }
        if (!whole) {
            per = max((int)((unsigned)(all.x + gridDim.x - 1) / gridDim.x), key_groups);
            begin = (int)min((long long)per * blockIdx.x, (long long)all.x);
        }
        end = whole ? all.y : (int)min((long long)begin + per, (long long)all.x);
        if (whole ? (int)blockIdx.x >= end : begin >= end) return;
        const int at_line = whole ? (int)blockIdx.x : begin;
        for (int first = 0, sum = 0;;) {
            const int from = sum + (whole ? before.y : before.x);
            if (at_line >= from && at_line < from + (whole ? mine.y : mine.x)) {
                sh.begin_seq = first + tid;
                sh.begin_base = from;
            }
            first += PA_THREADS;
            if (first >= n_seqs) break;
            // Only batches wider than a block come here.
            sum += chunk.x;
            mine = work_of(first + tid, w);
            before = pa_scan(mine, sh, chunk);
        }
        __syncthreads();
        at.seq = sh.begin_seq;
        base = sh.begin_base;
        at.w = pa_work<TILE, REACH>(a, at.seq);
    }
    if (whole) {
        at.unit = blockIdx.x - base;
        at.tile = 0;
        end = at.w.tiles;
    } else {
        at.unit = (begin - base) / at.w.tiles;
        at.tile = (begin - base) - at.unit * at.w.tiles;
    }
    const int count = end - begin;
    const int page = a.kv.page_size, log_page = 31 - __clz(page);
    const int pages = max(TILE >> log_page, 1);  // of a tile

    if (warp >= PA_CONSUMERS) {
        // ------------------------------------------------------------ producer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_OTHER_REGS));
        if (warp >= PA_CONSUMERS + PA_PRODUCERS) {
            pa_epilogue<D, FORMAT, F32, TILE, REACH>(a, sh, at, count, begin, per, warp - PA_CONSUMERS - PA_PRODUCERS, parts, q_ops);
            return;
        }
        // Each producer warp issues every PA_PRODUCERS-th tile of the block's: one
        // warp's wait, expectation and two copies take about 500 cycles, more
        // than a tile's share of HBM's time.  Page numbers and scales are fetched
        // a batch of 32 pages at a time, the numbers two batches ahead of the
        // copies and the scales one.
        const int producer = warp - PA_CONSUMERS;
        const int log_pages = 31 - __clz(pages), per_batch = 32 >> log_pages;
        const int j = lane & (pages - 1), off = lane >> log_pages;
        struct Batch {
            int first, n;   // the block's tiles first, first + PA_PRODUCERS, ..: n of them
            int head, row;  // KV head, and this lane's page: its first row, its number
            int id;
            bool wanted, bad;  // rows see it; they do and its number is outside the pool
            float ks, vs;
        };
        int ahead = 0;  // tiles handed to batches
        bool more = true;
        auto fetch_id = [&]() {
            Batch b;
            b.id = 0;
            b.wanted = b.bad = false;
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
            const int64_t pos =
                (int64_t)pa_tile<TILE, REACH>(a, at.w, at.tile + skip + PA_PRODUCERS * off) * TILE + (j << log_page);
            const int64_t begins = pos >> log_page << log_page;
            if (off < b.n && pos < at.w.s.len && (begins + page > at.w.low || (REACH && begins < a.reach.first))) {
                b.id = a.batch.page_table[at.seq * a.batch.table_stride + (pos >> log_page)];
                b.row = (int)(pos - begins);
                b.wanted = true;
            }
            ahead += span;
            at.advance(a, span);
            return b;
        };
        auto fetch_scales = [&](Batch &b) {
            if (!b.wanted) return;
            b.bad = b.id < 0 || b.id >= a.kv.n_pages;
            if (b.bad) return;
            const int64_t tile = (int64_t)b.id * a.kv.n_kv_heads + b.head;
            b.ks = a.kv.k_scales[tile];
            b.vs = a.kv.v_scales[tile];
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
                if (lane == 0) *(volatile int *)&sh.tile[slot] = tile;
                const bool here = off == i;
                const bool load = here && now.wanted && !now.bad;
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
                    if constexpr (LOST) {
                        // Like values that are not finite, by the scores: rows that do not see the page are
                        // not changed by it.
                        const bool lost = now.bad || !(fabsf(now.ks) <= FLT_MAX && fabsf(now.vs) <= FLT_MAX);
                        sh.scales[slot][j] = lost ? NAN : now.ks;
                        sh.scales[slot][8 + j] = lost ? 0.0f : now.vs;
                        if (FORMAT == FO_PAGED_E4M3 && now.bad) {  // (what is there may be NaN)
                            uint4 *vt = reinterpret_cast<uint4 *>(tiles + slot * Shape::STAGE + Shape::TILE_BYTES + j * bytes);
                            for (uint32_t x = 0; x < bytes / 16; x++) vt[x] = make_uint4(0, 0, 0, 0);
                            sm100::fence_proxy_async_smem();  // these before the next copy
                        }
                    } else {
                        sh.scales[slot][j] = now.bad ? NAN : now.ks;
                        sh.scales[slot][8 + j] = now.bad ? NAN : now.vs;
                    }
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
    // This lane's pieces of K rows g and g + 8 of a fragment, and its row of a V
    // load: row 4 t' + i of a 16 x 16 matrix is the key of the fragment's row 2 t'
    // + (i & 1) + 8 (i >> 1), as the probabilities' transposition leaves them.
    const int k0 = pa_key<D>(g), k1 = pa_key<D>(g ^ 4);
    const int k_off0 = k0 * D + ((D == 128 ? t ^ k0 : t ^ (k0 >> 1 & 3)) << 4);
    const int k_off1 = (8 + k1) * D + ((D == 128 ? t ^ k1 : t ^ (k1 >> 1 & 3)) << 4);
    const int v_pair = (lane >> 2 & 3) * 2 + (lane & 1), v_high = lane >> 1 & 1;
    const int v_key = pa_key<D>(v_high ? v_pair ^ 4 : v_pair);
    const int v_row = (lane >> 4) * 16 + v_high * 8 + v_key;
    const uint32_t v_base = v_row * D;
    const int v_swizzle = D == 128 ? v_key : v_key >> 1 & 3;
    const int page_shift = 31 - __clz(min(page, TILE) / 16);  // log2 of the m16 steps of a page's part of a tile

    const uint2 *q_from = q_ops + col_group * (Shape::Q_TILE / 8) + lane;
    uint32_t *rest = rests + warp * (Shape::REST / 4) + lane;

    using Place = PaPlace<TILE, REACH>;
    Place *place = reinterpret_cast<Place *>(sh.places[warp]);
    static_assert(sizeof(Place) == sizeof(sh.places[0]), "a place");
    if (lane == 0) *place = {at, begin, per};
    __syncwarp();

    for (int i = 0, segment = 0; i < count; segment++) {
        const PaCursor<TILE, REACH> here = place->at;
        const int n = min(here.left(), count - i);
        const int n_queries = min(here.w.s.n * a.group - here.group() * a.queries, a.queries);  // of this unit
        const int len = here.w.s.len, low = here.w.low;
        const int p_first = len - here.w.s.n;  // positions of the sequence's first row and of its last
        const int p_last = p_first + here.w.s.n - 1;
        const int tile0 = here.w.t0 + here.tile - i;
        // The queries as B operands.
        uint2 qf[Q_REGS ? QT * KQ : 1];
        float q_scale[2];  // of this lane's columns 2 t, 2 t + 1
        int q_pos[2];
        if (!sm100::mbar_wait(&sh.q_full, segment & 1, &sh.abort, a.err)) return;
        if constexpr (Q_REGS) {
#pragma unroll
            for (int x = 0; x < QT * KQ; x++) qf[x] = q_from[32 * x];
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            q_scale[h] = sh.q_scale[col_group * 8 + 2 * t + h];
            q_pos[h] = sh.q_pos[col_group * 8 + 2 * t + h];
        }
        if constexpr (Q_REGS) {
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&sh.q_free);
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[MT][4] = {};
        // Tiles all of whose positions every row sees need no mask.
        const int low_last = a.window > 0 ? max(p_last + 1 - a.window, 0) : 0;
        bool any = false;

        int k = i + (key_group - i % key_groups + key_groups) % key_groups;
        for (; k < i + n; k += key_groups) {
            const int slot = k % STAGES;
            // The first position of this warp's half.
            const int pos0 = (REACH ? pa_tile<TILE, true>(a, here.w, here.tile + k - i) : tile0 + k) * TILE + half * HALF;
            if (!pa_wait_tile(sh, slot, k, a.err)) return;
            // (Differences, since pos0 + HALF may be 2^31.)
            if (col_group * 8 >= n_queries || pos0 > p_last || (low - pos0 >= HALF && (!REACH || pos0 >= a.reach.first))) {
                // No row of this warp's sees any of it.
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&sh.empty[slot]);
                continue;
            }
            any = true;
            const uint8_t *kt = tiles + slot * Shape::STAGE + half * HALF * D;
            uint8_t *vt = tiles + slot * Shape::STAGE + Shape::TILE_BYTES + half * HALF * D;
            if constexpr (!I8) {
                // Rows beyond the sequence, or of pages that no row sees, may hold any
                // bytes: an FP8 NaN times a probability of 0 would be NaN.
                // (The first positions' pages are there, behind a window too.)
                const int lo_row = max((low >> log_page << log_page) - pos0, 0), hi_row = min(len - pos0, HALF);
                if (lo_row > 0 || hi_row < HALF) {
                    for (int x = lane; x < HALF * D / 16; x += 32) {
                        const int row = x / (D / 16);
                        const bool unseen = row < lo_row && (!REACH || (pos0 + row) >> log_page << log_page >= a.reach.first);
                        if (unseen || row >= hi_row) reinterpret_cast<uint4 *>(vt)[x] = make_uint4(0, 0, 0, 0);
                    }
                    sm100::fence_proxy_async_smem();  // these before the next copy
                    __syncwarp();
                }
            }
            // S^T: rows = keys, columns = queries; scores times log2 e.
            float c[STEPS][4], mx[2] = {-INFINITY, -INFINITY};
            const bool masked = p_first - pos0 < HALF - 1 || (pos0 < low_last && (!REACH || a.reach.first - pos0 < HALF));
            constexpr int AHEAD = D == 64 ? 2 : 1;  // as many steps at a time as there are registers for
#pragma unroll
            for (int m0 = 0; m0 < STEPS; m0 += AHEAD) {
                uint32_t kw[AHEAD][2][KW];
#pragma unroll
                for (int mt = 0; mt < AHEAD; mt++) {
                    const uint8_t *row = kt + 16 * (m0 + mt) * D;
                    *reinterpret_cast<uint4 *>(kw[mt][0]) = *reinterpret_cast<const uint4 *>(row + k_off0);
                    *reinterpret_cast<uint4 *>(kw[mt][1]) = *reinterpret_cast<const uint4 *>(row + k_off1);
                    if constexpr (D == 128) {
                        *reinterpret_cast<uint4 *>(kw[mt][0] + 4) = *reinterpret_cast<const uint4 *>(row + (k_off0 ^ 64));
                        *reinterpret_cast<uint4 *>(kw[mt][1] + 4) = *reinterpret_cast<const uint4 *>(row + (k_off1 ^ 64));
                    }
                }
                constexpr int A = I8 ? QT : 1;  // accumulators: int8's terms have their own
                typename std::conditional<I8, uint32_t, float>::type acc[AHEAD][A][4];
#pragma unroll
                for (int mt = 0; mt < AHEAD; mt++)
#pragma unroll
                    for (int x = 0; x < A; x++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[mt][x][e] = I8 ? PA_MAGIC : 0;
#pragma unroll
                for (int w = 0; w < KQ; w++) {
                    uint2 b[QT];
#pragma unroll
                    for (int x = 0; x < QT; x++) b[x] = Q_REGS ? qf[Q_REGS ? x * KQ + w : 0] : q_from[32 * (x * KQ + w)];
#pragma unroll
                    for (int mt = 0; mt < AHEAD; mt++) {
                        uint32_t f[4];
                        if constexpr (I8) {
                            f[0] = kw[mt][0][2 * w], f[1] = kw[mt][1][2 * w];
                            f[2] = kw[mt][0][2 * w + 1], f[3] = kw[mt][1][2 * w + 1];
                        } else {
                            f[0] = e4m3x2_f16x2(kw[mt][0][w] & 0xFFFFu), f[1] = e4m3x2_f16x2(kw[mt][1][w] & 0xFFFFu);
                            f[2] = e4m3x2_f16x2(kw[mt][0][w] >> 16), f[3] = e4m3x2_f16x2(kw[mt][1][w] >> 16);
                        }
#pragma unroll
                        for (int x = 0; x < QT; x++) {
                            if constexpr (!I8) pa_hmma(acc[mt][0], f[0], f[1], f[2], f[3], b[x].x, b[x].y);
                            else if (x == 0) pa_imma<true>(acc[mt][0], f[0], f[1], f[2], f[3], b[x].x, b[x].y);
                            else pa_imma<false>(acc[mt][x], f[0], f[1], f[2], f[3], b[x].x, b[x].y);
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < AHEAD; mt++) {
                    float (&sc)[4] = c[m0 + mt];
                    const float ks = sh.scales[slot][(half * STEPS + m0 + mt) >> page_shift];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (I8) {
                            sc[e] = __uint_as_float(acc[mt][A - 1][e]) - PA_MAGIC_F;
                            sc[e] = fmaf(__uint_as_float(acc[mt][A > 1 ? A - 2 : 0][e]) - PA_MAGIC_F, 256.0f, sc[e]);
                            sc[e] = fmaf(__uint_as_float(acc[mt][0][e]) - PA_MAGIC_F, 65536.0f, sc[e]);
                        } else {
                            sc[e] = acc[mt][0][e];
                        }
                        sc[e] *= ks * q_scale[e & 1];
                    }
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int pos = pos0 + 16 * (m0 + mt) + (e < 2 ? k0 : 8 + k1), p = q_pos[e & 1];
                            bool seen = pos <= p && (a.window == 0 || p - pos < a.window);
                            if constexpr (REACH) seen |= pos <= p && pos < a.reach.first;
                            if (!seen) sc[e] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e & 1] = fmaxf(mx[e & 1], sc[e]);
                }
            }
            // The values and their scales, and the slot is free.
            const uint32_t v_at = sm100::smem_u32(vt) + v_base;
            uint32_t va[MT][VS][4];
#pragma unroll
            for (int d = 0; d < MT; d++)
#pragma unroll
                for (int v = 0; v < VS; v++) pa_load_transposed(va[d][v], v_at + 32 * v * D + ((d ^ v_swizzle) << 4));
            float vs[STEPS];
#pragma unroll
            for (int x = 0; x < STEPS; x++) vs[x] = sh.scales[slot][8 + ((half * STEPS + x) >> page_shift)];
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&sh.empty[slot]);
            // The half's own maximum, which its probabilities are relative to, and
            // the running one: alpha brings the sums so far to it, beta the half's.
            constexpr float P_BITS = I8 ? 0.0f : 10.0f;  // e4m3: probabilities are held times 2^10
            float alpha[2], beta[2];
            bool moved = false;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float x = mx[h];
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                const float top = fmaxf(x, m[h]);
                // While nothing has been seen the maximum stays -infinity and every
                // probability is 0.
                alpha[h] = top == -INFINITY ? 1.0f : sm100::ex2(m[h] - top);
                beta[h] = x == -INFINITY ? 0.0f : sm100::ex2(x - top - P_BITS);
                moved |= top != m[h];
                m[h] = top;
                mx[h] = x == -INFINITY ? 0.0f : x - P_BITS;
            }
            // Probabilities' terms, transposed into B operands.
            // int8: [term][32 keys][16 of them], e4m3: [term][16 keys][8 of them].
            uint32_t pf[PT][STEPS * (I8 ? 1 : 2)];
            float sum0 = 0.0f, sum1 = 0.0f;
            // int8: 2^23 + p times its largest integer holds that integer's bytes.
            constexpr float TOP = F32 ? 8388607.0f : 65535.0f, BASE = 8388608.0f;
            auto bytes = [&](int mt, const uint2 &lower, const uint2 &upper) {  // rows 0 .. 7 of the m16 step, 8 .. 15
                const uint32_t lo0 = pa_transpose(__byte_perm(lower.x, lower.y, 0x5410));
                const uint32_t lo1 = pa_transpose(__byte_perm(upper.x, upper.y, 0x5410));
                pf[0][mt] = __byte_perm(lo0, lo1, 0x6420);
                pf[1 % PT][mt] = __byte_perm(lo0, lo1, 0x7531);
                if constexpr (F32)
                    pf[PT - 1][mt] = __byte_perm(pa_transpose(__byte_perm(lower.x, lower.y, 0x7632)),
                                                 pa_transpose(__byte_perm(upper.x, upper.y, 0x7632)), 0x6420);
            };
            auto probabilities = [&](int mt, int r) {
                const float2 p = make_float2(sm100::ex2(c[mt][2 * r] - mx[0]), sm100::ex2(c[mt][2 * r + 1] - mx[1]));
                sum0 += p.x;
                sum1 += p.y;
                return p;
            };
            if constexpr (!I8) {
#pragma unroll
                for (int mt = 0; mt < STEPS; mt++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const float2 p = probabilities(mt, r);
                        const uint32_t f = pa_f16x2(p.x, p.y);
                        pf[0][2 * mt + r] = pa_transpose(f);
                        if constexpr (F32) {
                            const float2 b = f16x2_f32x2(f);
                            pf[PT - 1][2 * mt + r] = pa_transpose(pa_f16x2(p.x - b.x, p.y - b.y));
                        }
                    }
            } else {
#pragma unroll
                for (int mt = 0; mt < STEPS; mt++) {
                    const float2 lower = probabilities(mt, 0), upper = probabilities(mt, 1);
                    bytes(mt, make_uint2(__float_as_uint(fmaf(lower.x, TOP, BASE)), __float_as_uint(fmaf(lower.y, TOP, BASE))),
                          make_uint2(__float_as_uint(fmaf(upper.x, TOP, BASE)), __float_as_uint(fmaf(upper.y, TOP, BASE))));
                }
            }
            // A lane whose probabilities sum to less than 2^-8 has none of that size.
            bool twice = false;
            if constexpr (I8) {
                constexpr float SMALL = 1.0f / 256.0f;
                if (__any_sync(0xffffffffu, fminf(sum0, sum1) < SMALL)) {
                    // Such lanes, among the eight of a query's that see any key.
                    const uint32_t mine = 0x11111111u << t;
                    auto few = [&](float sum) {
                        const int see = __popc(__ballot_sync(0xffffffffu, sum > 0.0f) & mine);
                        const int small = __popc(__ballot_sync(0xffffffffu, sum > 0.0f && sum < SMALL) & mine);
                        return small > 0 && 2 * small >= see;
                    };
                    const bool few0 = few(sum0), few1 = few(sum1);
                    twice = __any_sync(0xffffffffu, few0 || few1);
                    if (twice) {
                        // Again, rounded down; what that leaves, as another integer of as
                        // many bits, waits in shared memory for the products of the first.
                        auto whole = [&](const float2 &p) {
                            return make_uint2(__float_as_uint(__fmaf_rd(p.x, TOP, BASE)),
                                              __float_as_uint(__fmaf_rd(p.y, TOP, BASE)));
                        };
                        auto left = [&](const float2 &p, const uint2 &u) {
                            const float x = fmaf(p.x, TOP, BASE - __uint_as_float(u.x));
                            const float y = fmaf(p.y, TOP, BASE - __uint_as_float(u.y));
                            return make_uint2(__float_as_uint(fmaf(x, TOP, BASE)), __float_as_uint(fmaf(y, TOP, BASE)));
                        };
                        const float keep0 = sum0, keep1 = sum1;
#pragma unroll
                        for (int mt = 0; mt < STEPS; mt++) {
                            const float2 lower = probabilities(mt, 0), upper = probabilities(mt, 1);
                            const uint2 u0 = whole(lower), u1 = whole(upper);
                            bytes(mt, left(lower, u0), left(upper, u1));
#pragma unroll
                            for (int x = 0; x < PT; x++) rest[32 * (x * STEPS + mt)] = pf[x][mt];
                            bytes(mt, u0, u1);
                        }
                        sum0 = keep0;
                        sum1 = keep1;
                    }
                }
            }
            l[0] = fmaf(sum0, beta[0], l[0] * alpha[0]);
            l[1] = fmaf(sum1, beta[1], l[1] * alpha[1]);
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int d = 0; d < MT; d++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[d][e] *= alpha[e & 1];
            }
            // O^T: rows = dimensions, columns = queries; two m16 tiles of dimensions
            // at a time, each page's sum times its scale: the products over one
            // page's keys, the steps [from, to) of 16; WHOLE: all of the half's.
            auto page_sum = [&](auto whole, int from, int to, float scale) {
                constexpr bool WHOLE = decltype(whole)::value;
                const float f0 = scale * beta[0], f1 = scale * beta[1];
                constexpr int A = I8 ? PT : 1;
#pragma unroll
                for (int d2 = 0; d2 < MT; d2 += 2) {
                    typename std::conditional<I8, uint32_t, float>::type acc[2][A][4];
#pragma unroll
                    for (int d = 0; d < 2; d++)
#pragma unroll
                        for (int x = 0; x < A; x++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[d][x][e] = I8 ? PA_MAGIC : 0;
#pragma unroll
                    for (int v = 0; v < VS; v++) {
                        const bool first = WHOLE || (2 * v >= from && 2 * v < to);
                        const bool second = WHOLE || (2 * v + 1 >= from && 2 * v + 1 < to);
                        if constexpr (I8) {
                            if (!first && !second) continue;
#pragma unroll
                            for (int x = 0; x < PT; x++) {
                                const uint32_t b0 = first ? pf[x][2 * v] : 0u, b1 = second ? pf[x][2 * v + 1] : 0u;
#pragma unroll
                                for (int d = 0; d < 2; d++) {
                                    const uint32_t (&r)[4] = va[d2 + d][v];
                                    pa_imma<false>(acc[d][x], r[0], r[1], r[2], r[3], b0, b1);
                                }
                            }
                        } else {
#pragma unroll
                            for (int y = 0; y < 2; y++) {
                                if (!(y ? second : first)) continue;
#pragma unroll
                                for (int d = 0; d < 2; d++) {
                                    const uint32_t u0 = va[d2 + d][v][2 * y], u1 = va[d2 + d][v][2 * y + 1];
                                    const uint32_t a0 = e4m3x2_f16x2(u0 & 0xFFFFu), a1 = e4m3x2_f16x2(u1 & 0xFFFFu);
                                    const uint32_t a2 = e4m3x2_f16x2(u0 >> 16), a3 = e4m3x2_f16x2(u1 >> 16);
#pragma unroll
                                    for (int x = 0; x < PT; x++)
                                        pa_hmma(acc[d][0], a0, a1, a2, a3, pf[x][4 * v + 2 * y], pf[x][4 * v + 2 * y + 1]);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int d = 0; d < 2; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float sum;
                            if constexpr (I8) {
                                // Term 0 is the lowest byte.
                                sum = fmaf(__uint_as_float(acc[d][A > 1][e]) - PA_MAGIC_F, 256.0f,
                                           __uint_as_float(acc[d][0][e]) - PA_MAGIC_F);
                                if constexpr (F32)
                                    sum = fmaf(__uint_as_float(acc[d][A - 1][e]) - PA_MAGIC_F, 65536.0f, sum);
                            } else {
                                sum = acc[d][0][e];
                            }
                            o[d2 + d][e] = fmaf(sum, e & 1 ? f1 : f0, o[d2 + d][e]);
                        }
                }
            };
            for (bool again = twice;; again = false) {
                if constexpr (I8) beta[0] *= 1.0f / TOP, beta[1] *= 1.0f / TOP;
                if ((1 << page_shift) >= STEPS) {
                    page_sum(std::true_type{}, 0, STEPS, vs[0]);
                } else if (page_shift == 1) {
#pragma unroll
                    for (int from = 0; from < STEPS; from += 2) page_sum(std::false_type{}, from, from + 2, vs[from]);
                } else {
#pragma unroll
                    for (int from = 0; from < STEPS; from++) page_sum(std::false_type{}, from, from + 1, vs[from]);
                }
                if (!I8 || !again) break;
#pragma unroll
                for (int x = 0; x < PT; x++)
#pragma unroll
                    for (int mt = 0; mt < STEPS; mt++) pf[x][mt] = rest[32 * (x * STEPS + mt)];
            }
        }

        if constexpr (!Q_REGS) {
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&sh.q_free);
        }
        // This warp's part, for the epilogue warps to join.  A sum that is not a
        // number (a query that is not finite and saw a position, a page number
        // outside the pool) makes its query's output NaN.
        if (segment > 0 && !sm100::mbar_wait(&sh.part_free, (segment - 1) & 1, &sh.abort, a.err)) return;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float x = l[h];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            if (g == 0) {
                sh.ml[warp][2 * t + h][0] = m[h];
                sh.ml[warp][2 * t + h][1] = x;
            }
            if (any) {
                float *col = parts + (warp * 8 + 2 * t + h) * Shape::PART_LD + g;
#pragma unroll
                for (int d = 0; d < MT; d++) {
                    col[16 * d] = o[d][h];
                    col[16 * d + 8] = o[d][2 + h];
                }
            }
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&sh.part_full);
        Place was = *place;
        if (i + n == count && !(was.at.tile == 0 && n == was.at.w.tiles)) {
            if (!sm100::mbar_wait(&sh.shared_go[1], 0, &sh.abort, a.err)) return;
            if (sh.joins[1])
                pa_join_blocks<D, F32>(a, pa_unit(a, was.at, was.begin + i, n, was.per), PA_EPILOGUES + warp,
                                              PA_EPILOGUES + PA_CONSUMERS);
        }
        i += n;
        if (i >= count) break;
        was.at.advance(a, n);
        __syncwarp();
        if (lane == 0) place->at = was.at;
        __syncwarp();
    }
}

inline PFN_cuTensorMapEncodeTiled_v12000 pa_encoder() {
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
inline bool pa_map(CUtensorMap *map, const void *codes, const fo_paged_kv &kv) {
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

template <int D, int FORMAT, bool F32, bool REACH, bool LOST>
cudaError_t launch_attention(const fo_paged_attention_launch &a, unsigned grid, cudaStream_t stream) {
    auto *kernel = paged_attention_kernel<D, FORMAT, F32, REACH, LOST>;
    using Shape = PaShape<D, FORMAT, F32>;
    static_assert(Shape::smem(PA_CONSUMERS / 2) + sizeof(PaShared) <= 227 * 1024, "shared memory");
    // The attribute belongs to each device's context: set once per device.
    static std::atomic<unsigned long long> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             Shape::smem(PA_CONSUMERS / 2));
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
    return launch(kernel, dim3(grid), dim3(PA_THREADS), Shape::smem(a.queries / 8), stream, k_map, v_map, a);
}

template <int D, bool REACH, bool LOST>
cudaError_t launch_attention(const fo_paged_attention_launch &a, unsigned grid, cudaStream_t stream) {
    if (a.q.dtype == FO_DT_F32)
        return a.kv.format == FO_PAGED_I8 ? launch_attention<D, FO_PAGED_I8, true, REACH, LOST>(a, grid, stream)
                                          : launch_attention<D, FO_PAGED_E4M3, true, REACH, LOST>(a, grid, stream);
    return a.kv.format == FO_PAGED_I8 ? launch_attention<D, FO_PAGED_I8, false, REACH, LOST>(a, grid, stream)
                                      : launch_attention<D, FO_PAGED_E4M3, false, REACH, LOST>(a, grid, stream);
}

template <bool REACH, bool LOST>
cudaError_t launch_attention(const fo_paged_attention_launch &args, int sms, cudaStream_t stream) {
    fo_paged_attention_launch a = args;
    if (a.batch.total_rows <= 0) return cudaSuccess;
    a.group = a.q.heads / a.kv.n_kv_heads;
    // A warp takes the queries of one n8 tile; beyond that 2, 3 or 6 warps share
    // each half of a tile; beyond that a (sequence, KV head) is read once for
    // each group of queries.
    int64_t queries = a.batch.max_rows * a.group;
    if (REACH && a.reach.few > 0) queries = std::min<int64_t>(queries, a.reach.few);
    a.col_groups = queries <= 8 ? 1 : queries <= 16 ? 2 : queries <= 24 ? 3 : 6;
    a.queries = 8 * a.col_groups;
    a.evict_first = queries <= a.queries;
    auto aligned = [](const fo_rows &r, int64_t bytes) {
        const int64_t unit = bytes / (r.dtype == FO_DT_F32 ? 4 : 2);
        return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    a.q_vec = aligned(a.q, 16);
    a.out_vec = aligned(a.out, a.q.dtype == FO_DT_F32 ? 16 : 8);
    // No more blocks than the most tiles there can be for, one for each group
    // of consumer warps.
    const int64_t units = a.batch.n_seqs * a.kv.n_kv_heads * ((queries + a.queries - 1) / a.queries);
    const int64_t most = units * ((a.batch.table_stride * a.kv.page_size * a.kv.head_dim + 8191) / 8192 + REACH);
    const int64_t groups = PA_CONSUMERS / 2 / a.col_groups;
    a.whole_units = units <= sms && a.batch.n_seqs <= PA_THREADS;
    int64_t blocks = std::min<int64_t>(sms, (most + groups - 1) / groups);
    if (a.whole_units) blocks = std::max(blocks, units);
    const unsigned grid = (unsigned)std::max<int64_t>(1, blocks);
    if (most > INT32_MAX) return cudaErrorInvalidValue;
    return a.kv.head_dim == 64 ? launch_attention<64, REACH, LOST>(a, grid, stream)
                               : launch_attention<128, REACH, LOST>(a, grid, stream);
}

}  // namespace fo
