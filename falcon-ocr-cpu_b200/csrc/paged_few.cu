// paged_few.cu -- attention of few query rows where sequences share their
// beginnings: a group's rows over the shared positions, and each sequence's rows
// over its own positions behind them, joined with what the shared ones gave.
//
// For a query row q and the positions j that it sees of a range: s_j = scale *
// kscale * (q . kcode_j), and the sums of e^(s_j - m) and e^(s_j - m) vscale vcode_j.
// Such ranges are short and there are many (64 sequences' own 500 positions are 512
// units of 64 KB), so latency bounds them, and what a kernel does once for a unit:
// the units are spread as thinly as they go, eight or four warps to a block, 16 positions
// to a warp at a time, the blocks of a cluster sharing a unit where there are
// few, lanes' parts joined once at the end, by way of distributed shared memory.
// (paged_attention.cuh's kernel goes from unit to unit with blocks of sixteen
// warps, which is what long ranges want: 52 us for 64 uneven sequences of 1 to
// 1,024 positions where this one takes 27, profiled and cold.  In FP32 on CUDA
// cores this kernel took 36.)  Measured (CUDA graph, both parts): 8 readings of 6,544
// positions 20.5 us; 64 continuations of 16,384, the shared part by paged_tiles.cu,
// 50.2.
// Codes become FP16, which holds them exactly, in registers, where they lie as they
// are loaded: 16 adjacent dimensions of a key to a lane are four k steps of
// m16n8k16 products if the query's elements are taken in the same order, and of
// a value 8 dimensions of four positions are the B operands of eight products.
// S^T = K Q^T has keys in rows and queries in columns; the probabilities go
// through a transposition of 8 x 8 matrices to become P's rows.  A query, and a
// probability times its page's value scale, are one FP16 each, or two for FP32 rows:
// 11 or 22 bits of their own (paged_tiles.cu says relative to what).
#include "paged_reach.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace fo {

constexpr int PF_WARPS = 8, PF_THREADS = 32 * PF_WARPS;  // of a block at most
constexpr int PF_LOWEST = 12;       // exponent bits of the least power of two that scales are relative to
constexpr float PF_SLACK = 4.0f;    // log2: what a score may pass the maximum by before that moves (no more: rounded down)

__device__ __forceinline__ uint32_t pf_cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void pf_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Another block's shared memory, at this block's address.  (In order with the cluster's
// barriers, which are volatile too; ordinary loads may pass.)
__device__ __forceinline__ uint32_t pf_at(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 pf_remote2(const float *p, uint32_t rank) {
    float2 x;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(pf_at(p, rank)));
    return x;
}
__device__ __forceinline__ float4 pf_remote4(const float *p, uint32_t rank) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(pf_at(p, rank)));
    return x;
}
__device__ __forceinline__ void pf_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit elements, two per lane along a row, transposed.
__device__ __forceinline__ uint32_t pf_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pf_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Bytes 0 and 1 of a word as two FP16 codes (exact).  int8: the byte of code + 128
// under 1024's exponent is 1024 + code + 128.
template <int FORMAT>
__device__ __forceinline__ uint32_t pf_widen(uint32_t pair) {
    if constexpr (FORMAT == FO_PAGED_I8) {
        uint32_t r;
        asm("sub.rn.f16x2 %0, %1, %2;"
            : "=r"(r)
            : "r"(__byte_perm(pair ^ 0x8080u, 0x64646464u, 0x4140)), "r"(0x64806480u));
        return r;
    } else {
        return e4m3x2_f16x2(pair & 0xFFFFu);
    }
}

// Copies into shared memory: 16 bytes, none of them read and zeros written where `bytes`
// is 0, and 4.
__device__ __forceinline__ void pf_copy16(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pf_copy4(uint32_t to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// Steps of a warp that are on their way or computed, and later its part.
template <int D>
struct PfShape {
    static constexpr int STAGES = D == 64 ? 4 : 3;
    static constexpr int STAGE = 2 * 16 * D + 16;  // 16 positions' keys and values, and their page's scales
};
template <int D, int NT>
struct PfShared {
    float block_o[8 * NT][D], block_ml[8 * NT][2], ml[PF_WARPS][8 * NT][2];
    // [warps][STAGES * STAGE], a warp's part [8 * NT][D] in its own
};
template <int D, int NT>
__host__ __device__ constexpr int pf_smem(int warps) {
    return (int)sizeof(PfShared<D, NT>) + warps * PfShape<D>::STAGES * PfShape<D>::STAGE;
}

// NT: n8 tiles of queries.
template <int D, int FORMAT, bool F32, int NT>
__global__ void __launch_bounds__(PF_THREADS, F32 && NT == 2 ? 1 : 2)
    paged_few_kernel(const __grid_constant__ fo_paged_few_launch a) {
    using T = typename std::conditional<F32, float, uint16_t>::type;
    constexpr int TERMS = 1 + F32, HALVES = D / 64, KQ = 4 * HALVES;
    constexpr int STAGES = PfShape<D>::STAGES, STAGE = PfShape<D>::STAGE;
    static_assert(8 * NT * D * 4 <= STAGES * STAGE && sizeof(PfShared<D, NT>) % 16 == 0, "a warp's part");
    extern __shared__ __align__(16) uint8_t pf_memory[];
    PfShared<D, NT> &sh = *reinterpret_cast<PfShared<D, NT> *>(pf_memory);
    wait_for_prior_kernel();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t *stages = pf_memory + sizeof(PfShared<D, NT>) + warp * STAGES * STAGE;
    auto part_of = [&](int w) {
        return reinterpret_cast<float *>(pf_memory + sizeof(PfShared<D, NT>) + w * STAGES * STAGE);
    };
    const int heads = a.kv.n_kv_heads, page = a.kv.page_size, log_page = 31 - __clz(page);
    const int blocks = gridDim.y, rank = blocks > 1 ? (int)pf_cluster_rank() : 0;
    // The unit: rows [first, first + n) of a sequence or a group, positions [from, to), queries from q0 on.
    const int item = blockIdx.x / heads, head = blockIdx.x - item * heads, index = item / a.q_units;
    const int q0 = (item - index * a.q_units) * 8 * NT;
    int seq = index, first, n, len = 0, from = 0, to;
    if (a.reach.over_groups) {
        const Group x = load_group(a.reach, a.batch, page, index, a.err);
        seq = x.leader;
        first = x.first;
        n = x.n;
        to = x.len;
    } else {
        const Sequence x = load_sequence(a.batch, page, seq, a.err);
        first = x.first;
        n = x.n;
        to = len = x.len;
        from = min(shared_of(a.reach, a.batch, page, seq, a.err).len, to);
    }
    const int n_queries = min(n * a.group - q0, 8 * NT);
    if (n_queries <= 0) return;  // all of the cluster's blocks

    // Queries as B operands: column g of a tile, this lane's dimensions 16 t .. 16 t + 15 of each
    // 64.  Relative to a power of two that brings a query's largest element to [2^14, 2^15).
    uint32_t qf[NT][TERMS][KQ][2];
    float q_scale[NT][2];  // of this lane's columns 2 t, 2 t + 1
    int place[NT][2];      // the last position that they see
#pragma unroll
    for (int x = 0; x < NT; x++) {
        const int qi = q0 + 8 * x + g, r = qi / a.group;
        const bool mine = qi - q0 < n_queries;
        float y[HALVES][16], most = 0.0f;
        const T *row = static_cast<const T *>(a.q.data) + (int64_t)(first + (mine ? r : 0)) * a.q.row_stride +
                       (head * a.group + (mine ? qi - r * a.group : 0)) * a.q.head_stride + 16 * t;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            if (a.q_vec) {
                load8(row + 64 * h, y[h]);
                load8(row + 64 * h + 8, y[h] + 8);
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) y[h][e] = load1(row + 64 * h + e);
            }
        }
        bool finite = true;
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                most = fmaxf(most, fabsf(y[h][e]));
                finite &= fabsf(y[h][e]) <= FLT_MAX;
            }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        finite = (__ballot_sync(0xffffffffu, finite) >> (lane & 28) & 15) == 15;
        const int e = max((int)(__float_as_uint(most) >> 23), 15);
        const float up = finite ? __uint_as_float((uint32_t)(268 - e) << 23) : 0.0f;
        const float scale = finite ? __uint_as_float((uint32_t)max(e - 14, 1) << 23) * a.scale * REACH_LOG2E : NAN;
        int pos = -1;
        if (mine) pos = a.reach.over_groups ? min(place_of_row(a.batch, page, first + r, a.err), to - 1) : len - n + r;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            q_scale[x][h] = __shfl_sync(0xffffffffu, scale, 8 * t + 4 * h);
            place[x][h] = __shfl_sync(0xffffffffu, pos, 8 * t + 4 * h);
        }
#pragma unroll
        for (int w = 0; w < KQ; w++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float u = y[w / 4][4 * (w & 3) + 2 * h] * up, v = y[w / 4][4 * (w & 3) + 2 * h + 1] * up;
                if (!finite) u = v = 0.0f;
#pragma unroll
                for (int z = 0; z < TERMS; z++) {
                    qf[x][z][w][h] = pf_f16x2(u, v);
                    const float2 b = f16x2_f32x2(qf[x][z][w][h]);
                    u -= b.x;
                    v -= b.y;
                }
            }
    }

    float m[NT][2], l[NT][2], o[8 * HALVES][4];
    int top[NT][2];  // exponent bits of a power of two above the scales of the values that a query sees
#pragma unroll
    for (int x = 0; x < NT; x++)
#pragma unroll
        for (int h = 0; h < 2; h++) m[x][h] = -INFINITY, l[x][h] = 0.0f, top[x][h] = PF_LOWEST;
#pragma unroll
    for (int d = 0; d < 8 * HALVES; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[d][e] = 0.0f;

    // Steps of 16 positions, of one page, several on their way at once (one ahead, in registers,
    // left each step waiting 2,000 cycles for its own), and the page numbers of those after them.
    const int base = from & ~15, steps = to > from ? (to - base + 15) / 16 : 0, stride = a.warps * blocks;
    const int32_t *table = a.batch.page_table + seq * a.batch.table_stride;
    auto ask = [&](int at) { return at < steps ? table[((int64_t)base + 16 * (int64_t)at) >> log_page] : 0; };
    const uint32_t page_bytes = (uint32_t)(page * D), to_stages = (uint32_t)__cvta_generic_to_shared(stages) + 16 * lane;
    const uint8_t *my_k = static_cast<const uint8_t *>(a.kv.k_codes) + (int64_t)head * page_bytes + 16 * lane;
    const uint8_t *my_v = static_cast<const uint8_t *>(a.kv.v_codes) + (int64_t)head * page_bytes + 16 * lane;
    const float *my_scales = (lane & 1 ? a.kv.v_scales : a.kv.k_scales) + head;
    auto load = [&](int at, int id, int stage) {
        if (at < steps) {
            const uint32_t to_k = to_stages + stage * STAGE;
            const int pos = base + 16 * at;
            if (id >= 0 && id < a.kv.n_pages) {
                const int64_t codes = (int64_t)id * ((int64_t)heads * page_bytes) + (pos & (page - 1)) * D;
#pragma unroll
                for (int x = 0; x < D; x += 32) {
                    // Values that no row sees may be any bytes: an FP8 NaN times a probability of 0 would be NaN.
                    const int row = (x + lane) / (D / 16) + pos;
                    pf_copy16(to_k + 16 * x, my_k + codes + 16 * x, 16);
                    pf_copy16(to_k + 16 * D + 16 * x, my_v + codes + 16 * x, row >= from && row < to ? 16 : 0);
                }
                if (lane < 2) pf_copy4(to_k + 32 * D - 12 * lane, my_scales + (int64_t)id * heads);
            } else {
#pragma unroll
                for (int x = 0; x < 2 * D; x += 32) pf_copy16(to_k + 16 * x, my_k, 0);
                if (lane > 0) return;
                float *scales = reinterpret_cast<float *>(stages + stage * STAGE + 32 * D);

                // The rows that see the page get NaN, by their scores.
                atomicOr(a.err, FO_DEVERR_PAGED);
                scales[0] = NAN;
                scales[1] = 0.0f;
            }
        }
    };
    auto commit = []() { asm volatile("cp.async.commit_group;" ::: "memory"); };
    int i = warp * blocks + rank, ids[STAGES + 1];
#pragma unroll
    for (int x = 0; x <= STAGES; x++) ids[x] = ask(i + x * stride);
#pragma unroll
    for (int x = 0; x < STAGES - 1; x++) {
        load(i + x * stride, ids[x], x);
        commit();
    }
    int id0 = ids[STAGES - 1], id1 = ids[STAGES];
#pragma unroll 1
    for (int stage = 0; i < steps; i += stride) {
        load(i + (STAGES - 1) * stride, id0, stage == 0 ? STAGES - 1 : stage - 1);
        commit();
        id0 = id1;
        id1 = ask(i + (STAGES + 1) * stride);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const int pos = base + 16 * i;
        struct {
            uint4 k[HALVES][2];  // keys g and g + 8, dimensions 16 t ..
            uint2 v[HALVES][4];  // positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9, dimensions 8 g ..
            float ks, vs;
        } now;
        const uint8_t *at = stages + stage * STAGE;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            now.k[h][0] = *reinterpret_cast<const uint4 *>(at + g * D + 64 * h + 16 * t);
            now.k[h][1] = *reinterpret_cast<const uint4 *>(at + (g + 8) * D + 64 * h + 16 * t);
#pragma unroll
            for (int e = 0; e < 4; e++)
                now.v[h][e] = *reinterpret_cast<const uint2 *>(at + (16 + 2 * t + (e & 1) + 8 * (e >> 1)) * D + 64 * h + 8 * g);
        }
        now.ks = *reinterpret_cast<const float *>(at + 32 * D);
        now.vs = *reinterpret_cast<const float *>(at + 32 * D + 4);
        if (!(fabsf(now.ks) <= FLT_MAX && fabsf(now.vs) <= FLT_MAX)) now.ks = NAN, now.vs = 0.0f;
        __syncwarp();  // the stage may be written again
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        // Scores in log2 units: keys g and g + 8, columns 2 t and 2 t + 1 of a tile.
        float c[NT][4];
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) c[x][e] = 0.0f;
#pragma unroll
        for (int w = 0; w < KQ; w++) {
            const uint32_t k0 = (&now.k[w / 4][0].x)[w & 3], k1 = (&now.k[w / 4][1].x)[w & 3];
            const uint32_t a0 = pf_widen<FORMAT>(k0), a1 = pf_widen<FORMAT>(k1);
            const uint32_t a2 = pf_widen<FORMAT>(k0 >> 16), a3 = pf_widen<FORMAT>(k1 >> 16);
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int z = 0; z < TERMS; z++) pf_mma(c[x], a0, a1, a2, a3, qf[x][z][w][0], qf[x][z][w][1]);
        }
        const int step_top = min(max((int)(__float_as_uint(now.vs) >> 23 & 255u) + 1, PF_LOWEST), 253);
        bool moves = false;
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int p = pos + g + 8 * (e >> 1);
                const bool seen = p >= from && p <= place[x][e & 1];
                c[x][e] = seen ? c[x][e] * (now.ks * q_scale[x][e & 1]) : -INFINITY;
                moves |= c[x][e] > __fadd_rd(m[x][e & 1], PF_SLACK) || (seen && step_top > top[x][e & 1]);
            }
        if (__any_sync(0xffffffffu, moves)) {
            float factor[NT][2];
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float high = fmaxf(c[x][h], c[x][2 + h]);
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 4));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 8));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 16));
                    high = fmaxf(high, m[x][h]);
                    const float alpha = high == -INFINITY ? 1.0f : sm100::ex2(m[x][h] - high);
                    // (A step that the query sees any of is seen from its first position on.)
                    const int up = place[x][h] >= max(pos, from) ? max(top[x][h], step_top) : top[x][h];
                    factor[x][h] = alpha * __uint_as_float((uint32_t)max(127 + top[x][h] - up, 0) << 23);
                    l[x][h] *= alpha;
                    m[x][h] = high;
                    top[x][h] = up;
                }
#pragma unroll
            for (int x = 0; x < NT; x++) {
                // Row g of O is column g of the scores.
                const float f0 = __shfl_sync(0xffffffffu, factor[x][0], g >> 1);
                const float f1 = __shfl_sync(0xffffffffu, factor[x][1], g >> 1), f = g & 1 ? f1 : f0;
#pragma unroll
                for (int d = 0; d < 8 * HALVES; d++) o[d][2 * x] *= f, o[d][2 * x + 1] *= f;
            }
        }
        uint32_t p[TERMS][4] = {};  // A operands: queries in rows
#pragma unroll
        for (int x = 0; x < NT; x++) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float shift = m[x][e & 1] == -INFINITY ? 0.0f : m[x][e & 1];
                y[e] = sm100::ex2(c[x][e] - shift);
                l[x][e & 1] += y[e];
                const float v = now.vs * __uint_as_float((uint32_t)(264 - top[x][e & 1]) << 23);
                y[e] = y[e] == 0.0f ? 0.0f : y[e] * v;  // what is not seen adds nothing, whatever its scale is
            }
#pragma unroll
            for (int z = 0; z < TERMS; z++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t w = pf_f16x2(y[2 * h], y[2 * h + 1]);
                    const float2 b = f16x2_f32x2(w);
                    y[2 * h] -= b.x;
                    y[2 * h + 1] -= b.y;
                    p[z][x + 2 * h] = pf_transpose(w);
                }
        }
        // Dimension 8 n + j of a half is column n of its product j.  A step's products have a sum of their
        // own, added to the others' by ordinary FP32: the tensor core truncates its sums, which left
        // FP32 rows 2.3e-5 too small after 16,384 positions of a sequence's own and 2.0e-4 after
        // 131,072 (now 1e-6).  It costs 0 to 2 %, and the registers it frees gain 17 % with FP32 rows,
        // heads of 128 and up to 16,000 positions each (951 to 786 us).
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                auto pick = [&](int e) {
                    const uint32_t u = j < 4 ? now.v[h][e].x : now.v[h][e].y, v = j < 4 ? now.v[h][e + 1].x : now.v[h][e + 1].y;
                    return pf_widen<FORMAT>(__byte_perm(u, v, (j & 3) | ((j & 3) + 4) << 4));
                };
                const uint32_t b0 = pick(0), b1 = pick(2);
                float step[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int z = TERMS - 1; z >= 0; z--) pf_mma(step, p[z][0], p[z][1], p[z][2], p[z][3], b0, b1);
#pragma unroll
                for (int e = 0; e < 4; e++) o[8 * h + j][e] += step[e];
            }
    }

    // This warp's part, in place of its stages.
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    float *part = part_of(warp);
#pragma unroll
    for (int x = 0; x < NT; x++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], 4);
            l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], 8);
            l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], 16);
            if (g == 0) sh.ml[warp][8 * x + 2 * t + h][0] = m[x][h], sh.ml[warp][8 * x + 2 * t + h][1] = l[x][h];
        }
        const int t0 = __shfl_sync(0xffffffffu, top[x][0], g >> 1), t1 = __shfl_sync(0xffffffffu, top[x][1], g >> 1);
        const float unit = __uint_as_float((uint32_t)((g & 1 ? t1 : t0) - 10) << 23);
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *reinterpret_cast<float4 *>(part + (8 * x + g) * D + 64 * h + 8 * (2 * t + e) + j) =
                        make_float4(o[8 * h + j][2 * x + e] * unit, o[8 * h + j + 1][2 * x + e] * unit,
                                    o[8 * h + j + 2][2 * x + e] * unit, o[8 * h + j + 3][2 * x + e] * unit);
    }
    __syncthreads();
    // The block's warps.
#pragma unroll 1
    for (int y = threadIdx.x; y < n_queries * (D / 4); y += blockDim.x) {
        const int qi = y / (D / 4), quad = y % (D / 4);
        float high = -INFINITY, sum = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int w = 0; w < a.warps; w++) high = fmaxf(high, sh.ml[w][qi][0]);
        const float shift = high == -INFINITY ? 0.0f : high;
#pragma unroll 4
        for (int w = 0; w < a.warps; w++) {
            const float f = sm100::ex2(sh.ml[w][qi][0] - shift);
            const float4 z = *reinterpret_cast<const float4 *>(part_of(w) + qi * D + 4 * quad);
            sum = fmaf(sh.ml[w][qi][1], f, sum);
            v = make_float4(fmaf(z.x, f, v.x), fmaf(z.y, f, v.y), fmaf(z.z, f, v.z), fmaf(z.w, f, v.w));
        }
        *reinterpret_cast<float4 *>(&sh.block_o[qi][4 * quad]) = v;
        if (quad == 0) sh.block_ml[qi][0] = high, sh.block_ml[qi][1] = sum;
    }
    if (blocks > 1) pf_cluster_sync();
    else __syncthreads();
    // The cluster's blocks, and what the shared positions gave: four dimensions of a query at a time.
#pragma unroll 1
    for (int y = rank * blockDim.x + threadIdx.x; y < n_queries * (D / 4); y += blocks * blockDim.x) {
        const int qi = y / (D / 4), quad = y % (D / 4), r = (q0 + qi) / a.group, h = head * a.group + q0 + qi - r * a.group;
        const int64_t row = first + r, at_row = row * a.q.heads + h;
        float high = -INFINITY, sum = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](float pm, float pl, const float4 &z) {
            // Two parts, the one with the larger maximum as it is.
            const float up = fmaxf(high, pm), shift = up == -INFINITY ? 0.0f : up;
            const float f = sm100::ex2(pm - shift), keep = sm100::ex2(high - shift);
            sum = fmaf(pl, f, sum * keep);
            v = make_float4(fmaf(z.x, f, v.x * keep), fmaf(z.y, f, v.y * keep), fmaf(z.z, f, v.z * keep),
                            fmaf(z.w, f, v.w * keep));
            high = up;
        };
        // (Four blocks' at once: one after the other they took half of a call's time.)
#pragma unroll 1
        for (int c = 0; c < blocks; c += 4) {
            float2 ml[4];
            float4 z[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                ml[e] = pf_remote2(sh.block_ml[qi], min(c + e, blocks - 1));
                z[e] = pf_remote4(&sh.block_o[qi][4 * quad], min(c + e, blocks - 1));
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c + e < blocks) add(ml[e].x, ml[e].y, z[e]);
        }
        if (a.reach.raw_o) {
            reinterpret_cast<float4 *>(a.reach.raw_o + at_row * D)[quad] = v;
            if (quad == 0) reinterpret_cast<float2 *>(a.reach.raw_ml)[at_row] = make_float2(high, sum);
            continue;
        }
        // Of the shared positions, one finished sum, or parts of several blocks.  (Of a group that
        // was refused the latter are whatever was there.)
        int c0 = 0, c1 = -1, unit_q = 0;
        if (a.reach.parts_of) {
            const int2 parts = __ldcg(reinterpret_cast<const int2 *>(a.reach.parts_of) + at_row);
            const int last = parts.y & 0xFFFF, number = parts.y >> 16;
            if (parts.x >= 0 && parts.x <= last && last < a.parts && number >= 0 && number < FO_TILES_QUERIES)
                c0 = parts.x, c1 = last, unit_q = number;
        }
        if (c1 < 0) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.reach.prior_ml) + at_row);
            add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4 *>(a.reach.prior_o + at_row * D) + quad));
        }
#pragma unroll 6
        for (int c = c0; c <= c1; c++) {
            const int64_t part = 2 * c + (c == c0 ? 1 : 0);
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.part_ml) + part * FO_TILES_QUERIES + unit_q);
            add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4 *>(a.part_o) + (part * (D / 4) + quad) * FO_TILES_QUERIES +
                                   unit_q));
        }
        const float inv = inverse_sum(a.sinks ? a.sinks[h] : -INFINITY, high, sum);
        v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        T *out = static_cast<T *>(a.out.data) + row * a.out.row_stride + h * a.out.head_stride + 4 * quad;
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
        if (a.lse && quad == 0) a.lse[at_row] = log_sum(high, sum);
    }
    if (blocks > 1) pf_cluster_sync();  // no block's shared memory goes while another reads it
}

template <int D, int FORMAT, bool F32, int NT>
cudaError_t launch_few(const fo_paged_few_launch &in, int sms, cudaStream_t stream) {
    fo_paged_few_launch a = in;
    auto *kernel = paged_few_kernel<D, FORMAT, F32, NT>;
    constexpr int SMEM = pf_smem<D, NT>(PF_WARPS);
    {
        // The attributes belong to each device's context: set once per device.
        static std::atomic<unsigned long long> configured{0};
        int dev = 0;
        cudaGetDevice(&dev);
        const unsigned long long bit = 1ull << (dev & 63);
        if (!(configured.load() & bit)) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            configured.fetch_or(bit);
        }
    }
    // A group may have all rows of the call.
    const int64_t queries = (a.reach.over_groups ? a.batch.total_rows : a.batch.max_rows) * a.group;
    const int64_t items = a.reach.over_groups ? a.reach.n_groups + 2 : a.batch.n_seqs;
    a.q_units = (int)((queries + 8 * NT - 1) / (8 * NT));
    const int64_t units = items * a.q_units * a.kv.n_kv_heads;
    if (units > 0x7FFFFFFF) return cudaErrorInvalidValue;
    // Blocks that share a unit: as many as there are SMs for, two blocks of eight warps to an SM; and
    // with units enough, blocks of four warps, of which twice as many run at once.  (Of groups,
    // the two that stand for sequences outside them have next to nothing to do.)
    const int64_t busy = a.reach.over_groups ? (int64_t)a.reach.n_groups * a.kv.n_kv_heads : units;
    int blocks = 1;
    while (blocks < 8 && 2 * blocks * busy <= 2 * sms) blocks *= 2;
    // Sixteen, which want that many SMs next to each other, for no more units than there are such
    // neighbourhoods: 8 units over 6,544 positions 20.5 us with sixteen, 23.2 with eight; 16 units
    // 37.0 and 33.2.
    if (blocks == 8 && 16 * busy <= sms) blocks = 16;
    a.warps = busy > 2 * sms ? 4 : 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)units, (unsigned)blocks);
    cfg.blockDim = dim3(32 * a.warps);
    cfg.dynamicSmemBytes = pf_smem<D, NT>(a.warps);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = (unsigned)blocks;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int D, int FORMAT, bool F32>
cudaError_t launch_few(const fo_paged_few_launch &a, int sms, cudaStream_t stream) {
    const int64_t queries = (a.reach.over_groups ? a.batch.total_rows : a.batch.max_rows) * a.group;
    return queries <= 8 ? launch_few<D, FORMAT, F32, 1>(a, sms, stream) : launch_few<D, FORMAT, F32, 2>(a, sms, stream);
}

template <int D>
cudaError_t launch_few(const fo_paged_few_launch &a, int sms, cudaStream_t stream) {
    if (a.q.dtype == FO_DT_F32)
        return a.kv.format == FO_PAGED_I8 ? launch_few<D, FO_PAGED_I8, true>(a, sms, stream)
                                          : launch_few<D, FO_PAGED_E4M3, true>(a, sms, stream);
    return a.kv.format == FO_PAGED_I8 ? launch_few<D, FO_PAGED_I8, false>(a, sms, stream)
                                      : launch_few<D, FO_PAGED_E4M3, false>(a, sms, stream);
}

}  // namespace fo

extern "C" cudaError_t fo_launch_paged_few(const fo_paged_few_launch *args, int sms, cudaStream_t stream) {
    fo_paged_few_launch a = *args;
    if (a.batch.total_rows <= 0) return cudaSuccess;
    a.group = a.q.heads / a.kv.n_kv_heads;
    a.parts = sms;
    auto aligned = [](const fo_rows &r, int64_t bytes) {
        const int64_t unit = bytes / (r.dtype == FO_DT_F32 ? 4 : 2);
        return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    a.q_vec = aligned(a.q, 16);
    a.out_vec = aligned(a.out, a.q.dtype == FO_DT_F32 ? 16 : 8);
    return a.kv.head_dim == 64 ? fo::launch_few<64>(a, sms, stream) : fo::launch_few<128>(a, sms, stream);
}
