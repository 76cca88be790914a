// paged_own.cu -- the end of an attention of sequences that share their
// beginnings, where a KV head has few query rows of each: every sequence's own
// positions, behind the shared ones, joined with what another launch found over
// those (paged_attention_reach.cu, paged_tiles.cu).
//
// For a query row q over its sequence's positions j from the shared ones' end to
// its own place: s_j = scale * kscale * (q . kcode_j), and the sums of e^(s_j - m)
// and e^(s_j - m) vscale vcode_j in FP32.  Own parts are short and there are many:
// 64 sequences of 500 positions are 512 units of 64 KB.  What bounds them is
// latency, so the units are spread as thinly as they go: eight warps to a block,
// 32 (heads of 64) or 16 positions to a warp at a time, blocks of a cluster sharing a
// unit where there are few, and FP32 arithmetic on CUDA cores, which a few query
// rows leave far below their rate.  (The tensor-core kernel, whose blocks of
// sixteen warps go from unit to unit, takes 47 us for these, this one MEASURED.)
// A lane has 16 dimensions of a row: a load is 16 bytes of codes, a score a sum
// over 4 or 8 lanes, and a value goes to the lane's own outputs; each lane
// keeps a maximum of the rows that it has seen, and lanes, warps and blocks (by
// way of distributed shared memory) are joined once, at the end.
#include "paged_reach.cuh"

#include <algorithm>
#include <type_traits>

namespace fo {

constexpr int PO_WARPS = 8, PO_THREADS = 32 * PO_WARPS, PO_QUERIES = FO_PAGED_FEW;

__device__ __forceinline__ uint32_t po_cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void po_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of another block's shared memory, at this block's address.
__device__ __forceinline__ float po_remote(const float *p, uint32_t rank) {
    uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
    float x;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}"
                 : "=f"(x)
                 : "r"(at), "r"(rank)
                 : "memory");
    return x;
}

// QN queries to a warp.
template <int D, int FORMAT, bool F32, int QN>
__global__ void __launch_bounds__(PO_THREADS, QN == 4 ? 1 : 2)
    paged_own_kernel(const __grid_constant__ fo_paged_own_launch a) {
    using T = typename std::conditional<F32, float, uint16_t>::type;
    constexpr int LANES = D / 16, ROWS = 32 / LANES;  // lanes of a row, rows of a load
    constexpr int LOADS = 4, STEP = LOADS * ROWS;     // loads in flight; positions of a step
    __shared__ float part_o[PO_WARPS][QN][D], part_ml[PO_WARPS][QN][2];
    __shared__ float block_o[PO_QUERIES][D], block_ml[PO_QUERIES][2];
    wait_for_prior_kernel();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = a.kv.n_kv_heads, seq = blockIdx.x / heads, head = blockIdx.x - seq * heads;
    const int blocks = gridDim.y, rank = blocks > 1 ? (int)po_cluster_rank() : 0;
    const Sequence s = load_sequence(a.batch, a.kv.page_size, seq, a.err);
    const int n_queries = min(s.n * a.group, PO_QUERIES);
    if (n_queries == 0) return;  // all of the cluster's blocks
    const int from = min(shared_of(a.reach, a.batch, a.kv.page_size, seq, a.err).len, s.len);

    // This warp's queries, and which of the sequence's steps are its own.
    const int q0 = warp % a.q_warps * QN, split = warp / a.q_warps, splits = PO_WARPS / a.q_warps;
    const int d0 = lane % LANES * 16;
    float q[QN][16], scale[QN], m[QN], l[QN], o[QN][16];
    int place[QN];
#pragma unroll
    for (int x = 0; x < QN; x++) {
        const bool mine = q0 + x < n_queries;
        const int r = mine ? (q0 + x) / a.group : 0;
        place[x] = mine ? s.len - s.n + r : -1;
        const T *row = static_cast<const T *>(a.q.data) + (int64_t)(s.first + r) * a.q.row_stride +
                       (head * a.group + (mine ? q0 + x - r * a.group : 0)) * a.q.head_stride + d0;
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 16; e++) q[x][e] = 0.0f;
        if (mine) {
            if (a.q_vec) {
                load8(row, q[x]);
                load8(row + 8, q[x] + 8);
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) q[x][e] = load1(row + e);
            }
#pragma unroll
            for (int e = 0; e < 16; e++) finite &= fabsf(q[x][e]) <= FLT_MAX;
        }
        // A query that is not finite makes every score NaN.
        const unsigned all = __ballot_sync(0xffffffffu, finite), row_lanes = (1u << LANES) - 1u;
        scale[x] = (all >> (lane / LANES * LANES) & row_lanes) == row_lanes ? a.scale * REACH_LOG2E : NAN;
        m[x] = -INFINITY;
        l[x] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++) o[x][e] = 0.0f;
    }

    const int page = a.kv.page_size, log_page = 31 - __clz(page);
    const int base = from & ~(STEP - 1);  // (a load's rows are of one page)
    const int steps = s.len > from ? (s.len - base + STEP - 1) / STEP : 0, stride = splits * blocks;
    const uint8_t *k_codes = static_cast<const uint8_t *>(a.kv.k_codes), *v_codes = static_cast<const uint8_t *>(a.kv.v_codes);
    const int32_t *table = a.batch.page_table + seq * a.batch.table_stride;
    int ids[LOADS];
    auto ask = [&](int i) {  // the page numbers of a step's loads
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            const int64_t pos = (int64_t)base + (int64_t)i * STEP + u * ROWS;
            ids[u] = i < steps && pos < s.len && pos + ROWS > from ? table[pos >> log_page] : 0;
        }
    };
    int i = split * blocks + rank;
    ask(i);
#pragma unroll 1
    for (; i < steps; i += stride) {
        uint4 kw[LOADS], vw[LOADS];
        float ks[LOADS], vs[LOADS];
        const int pos0 = base + i * STEP + lane / LANES;
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            const int pos = pos0 + u * ROWS;
            const bool inside = pos >= from && pos < s.len;
            const bool valid = ids[u] >= 0 && ids[u] < a.kv.n_pages;
            if (inside && !valid) atomicOr(a.err, FO_DEVERR_PAGED);
            const int64_t tile = (int64_t)ids[u] * heads + head;
            ks[u] = inside && !valid ? NAN : 0.0f;
            vs[u] = 0.0f;
            kw[u] = vw[u] = make_uint4(0, 0, 0, 0);
            if (inside && valid) {
                const int64_t at = (tile * page + (pos & (page - 1))) * D + d0;
                kw[u] = *reinterpret_cast<const uint4 *>(k_codes + at);
                vw[u] = *reinterpret_cast<const uint4 *>(v_codes + at);
                ks[u] = a.kv.k_scales[tile];
                vs[u] = a.kv.v_scales[tile];
            }
        }
        ask(i + stride);
        float sc[LOADS][QN];
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            float k[16];
            decode4<FORMAT>(kw[u].x, k);
            decode4<FORMAT>(kw[u].y, k + 4);
            decode4<FORMAT>(kw[u].z, k + 8);
            decode4<FORMAT>(kw[u].w, k + 12);
#pragma unroll
            for (int x = 0; x < QN; x++) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) sum = fmaf(k[e], q[x][e], sum);
#pragma unroll
                for (int w = 1; w < LANES; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                const int pos = pos0 + u * ROWS;
                sc[u][x] = pos >= from && pos <= place[x] ? sum * (ks[u] * scale[x]) : -INFINITY;
            }
        }
#pragma unroll
        for (int x = 0; x < QN; x++) {
            float top = m[x];
#pragma unroll
            for (int u = 0; u < LOADS; u++) top = fmaxf(top, sc[u][x]);
            const float shift = top == -INFINITY ? 0.0f : top, alpha = exp2f(m[x] - shift);
            m[x] = top;
            l[x] *= alpha;
#pragma unroll
            for (int e = 0; e < 16; e++) o[x][e] *= alpha;
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                // (What is not seen adds nothing, whatever its scale is.)
                const float p = exp2f(sc[u][x] - shift);
                l[x] += p;
                sc[u][x] = p == 0.0f ? 0.0f : p * vs[u];
            }
        }
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            float v[16];
            decode4<FORMAT>(vw[u].x, v);
            decode4<FORMAT>(vw[u].y, v + 4);
            decode4<FORMAT>(vw[u].z, v + 8);
            decode4<FORMAT>(vw[u].w, v + 12);
#pragma unroll
            for (int x = 0; x < QN; x++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[x][e] = fmaf(v[e], sc[u][x], o[x][e]);
        }
    }

    // The lanes of a warp, which have different rows of the same dimensions.
#pragma unroll
    for (int x = 0; x < QN; x++) {
        float top = m[x];
#pragma unroll
        for (int w = LANES; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float f = exp2f(m[x] - (top == -INFINITY ? 0.0f : top));
        l[x] *= f;
#pragma unroll
        for (int e = 0; e < 16; e++) o[x][e] *= f;
#pragma unroll
        for (int w = LANES; w < 32; w <<= 1) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], w);
#pragma unroll
            for (int e = 0; e < 16; e++) o[x][e] += __shfl_xor_sync(0xffffffffu, o[x][e], w);
        }
        if (lane < LANES) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<float4 *>(&part_o[warp][x][d0 + e]) =
                    make_float4(o[x][e], o[x][e + 1], o[x][e + 2], o[x][e + 3]);
            if (lane == 0) part_ml[warp][x][0] = top, part_ml[warp][x][1] = l[x];
        }
    }
    __syncthreads();
    // The block's warps that have the same queries.
    for (int y = threadIdx.x; y < n_queries * D; y += PO_THREADS) {
        const int qi = y / D, d = y % D, x = qi % QN, w0 = qi / QN;
        float top = -INFINITY, sum = 0.0f, v = 0.0f;
        for (int w = w0; w < PO_WARPS; w += a.q_warps) top = fmaxf(top, part_ml[w][x][0]);
        const float shift = top == -INFINITY ? 0.0f : top;
        for (int w = w0; w < PO_WARPS; w += a.q_warps) {
            const float f = exp2f(part_ml[w][x][0] - shift);
            sum = fmaf(part_ml[w][x][1], f, sum);
            v = fmaf(part_o[w][x][d], f, v);
        }
        block_o[qi][d] = v;
        if (d == 0) block_ml[qi][0] = top, block_ml[qi][1] = sum;
    }
    if (blocks > 1) po_cluster_sync();
    else __syncthreads();
    // The cluster's blocks, and what the shared positions gave: four dimensions of a query at a time.
    for (int y = rank * PO_THREADS + threadIdx.x; y < n_queries * (D / 4); y += blocks * PO_THREADS) {
        const int qi = y / (D / 4), quad = y % (D / 4), r = qi / a.group, h = head * a.group + qi - r * a.group;
        const int64_t row = s.first + r, at_row = row * a.q.heads + h;
        // Either one finished sum, or parts of several blocks.
        int c0 = 0, c1 = -1, unit_q = 0;
        float top = -INFINITY;
        float2 prior = make_float2(-INFINITY, 0.0f);
        if (a.reach.parts_of) {
            const int2 parts = __ldcg(reinterpret_cast<const int2 *>(a.reach.parts_of) + at_row);
            // (Of a group that was refused they are whatever was there.)
            const int last = parts.y & 0xFFFF, number = parts.y >> 16;
            if (parts.x >= 0 && parts.x <= last && last < a.parts && number >= 0 && number < FO_TILES_QUERIES)
                c0 = parts.x, c1 = last, unit_q = number;
        }
        const bool whole = c1 < 0;
        if (whole) prior = __ldcg(reinterpret_cast<const float2 *>(a.reach.prior_ml) + at_row);
        const float2 *mls = reinterpret_cast<const float2 *>(a.part_ml);
        auto part = [&](int c) { return (int64_t)(2 * c + (c == c0 ? 1 : 0)); };
        for (int c = 0; c < blocks; c++)
            top = fmaxf(top, blocks > 1 ? po_remote(&block_ml[qi][0], c) : block_ml[qi][0]);
        top = fmaxf(top, prior.x);
#pragma unroll 4
        for (int c = c0; c <= c1; c++) top = fmaxf(top, __ldcg(mls + part(c) * FO_TILES_QUERIES + unit_q).x);
        const float shift = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](float pm, float pl, const float4 &z) {
            const float f = exp2f(pm - shift);
            sum = fmaf(pl, f, sum);
            v = make_float4(fmaf(z.x, f, v.x), fmaf(z.y, f, v.y), fmaf(z.z, f, v.z), fmaf(z.w, f, v.w));
        };
        if (whole) add(prior.x, prior.y, __ldcg(reinterpret_cast<const float4 *>(a.reach.prior_o + at_row * D) + quad));
#pragma unroll 4
        for (int c = c0; c <= c1; c++) {
            const float2 ml = __ldcg(mls + part(c) * FO_TILES_QUERIES + unit_q);
            add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4 *>(a.part_o) +
                                   (part(c) * (D / 4) + quad) * FO_TILES_QUERIES + unit_q));
        }
        for (int c = 0; c < blocks; c++) {
            const float *z = &block_o[qi][4 * quad];
            if (blocks > 1)
                add(po_remote(&block_ml[qi][0], c), po_remote(&block_ml[qi][1], c),
                    make_float4(po_remote(z, c), po_remote(z + 1, c), po_remote(z + 2, c), po_remote(z + 3, c)));
            else add(block_ml[qi][0], block_ml[qi][1], make_float4(z[0], z[1], z[2], z[3]));
        }
        const float inv = inverse_sum(a.sinks ? a.sinks[h] : -INFINITY, top, sum);
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
        if (a.lse && quad == 0) a.lse[at_row] = log_sum(top, sum);
    }
    if (blocks > 1) po_cluster_sync();  // no block's shared memory goes while another reads it
}

template <int D, int FORMAT, bool F32, int QN>
cudaError_t launch_own(const fo_paged_own_launch &in, int sms, cudaStream_t stream) {
    fo_paged_own_launch a = in;
    const int queries = (int)(a.batch.max_rows * a.group), warps = (queries + QN - 1) / QN;
    a.q_warps = warps <= 1 ? 1 : warps <= 2 ? 2 : 4;
    const int64_t units = a.batch.n_seqs * a.kv.n_kv_heads;
    if (units > 0x7FFFFFFF) return cudaErrorInvalidValue;
    // Blocks that share a unit: as many as there are SMs for, two blocks to an SM.
    int blocks = 1;
    while (blocks < 8 && 2 * blocks * units <= 2 * sms) blocks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)units, (unsigned)blocks);
    cfg.blockDim = dim3(PO_THREADS);
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
    return cudaLaunchKernelEx(&cfg, paged_own_kernel<D, FORMAT, F32, QN>, a);
}

template <int D, int FORMAT, bool F32>
cudaError_t launch_own(const fo_paged_own_launch &a, int sms, cudaStream_t stream) {
    const int64_t queries = a.batch.max_rows * a.group;
    return queries <= 1 ? launch_own<D, FORMAT, F32, 1>(a, sms, stream)
                        : queries <= 2 ? launch_own<D, FORMAT, F32, 2>(a, sms, stream)
                                       : launch_own<D, FORMAT, F32, 4>(a, sms, stream);
}

template <int D>
cudaError_t launch_own(const fo_paged_own_launch &a, int sms, cudaStream_t stream) {
    if (a.q.dtype == FO_DT_F32)
        return a.kv.format == FO_PAGED_I8 ? launch_own<D, FO_PAGED_I8, true>(a, sms, stream)
                                          : launch_own<D, FO_PAGED_E4M3, true>(a, sms, stream);
    return a.kv.format == FO_PAGED_I8 ? launch_own<D, FO_PAGED_I8, false>(a, sms, stream)
                                      : launch_own<D, FO_PAGED_E4M3, false>(a, sms, stream);
}

}  // namespace fo

extern "C" cudaError_t fo_launch_paged_own(const fo_paged_own_launch *args, int sms, cudaStream_t stream) {
    fo_paged_own_launch a = *args;
    if (a.batch.total_rows <= 0) return cudaSuccess;
    a.group = a.q.heads / a.kv.n_kv_heads;
    a.parts = sms;
    if (a.batch.max_rows * a.group > FO_PAGED_FEW) return cudaErrorInvalidValue;
    auto aligned = [](const fo_rows &r, int64_t bytes) {
        const int64_t unit = bytes / (r.dtype == FO_DT_F32 ? 4 : 2);
        return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    a.q_vec = aligned(a.q, 16);
    a.out_vec = aligned(a.out, a.q.dtype == FO_DT_F32 ? 16 : 8);
    return a.kv.head_dim == 64 ? fo::launch_own<64>(a, sms, stream) : fo::launch_own<128>(a, sms, stream);
}
