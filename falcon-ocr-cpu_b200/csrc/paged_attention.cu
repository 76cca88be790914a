// paged_attention.cu -- attention of a batch's query rows over a paged 8-bit
// KV cache.
//
// A first form: one block per (row, query head), a thread per position for
// the scores and a thread per output dimension for the values, the running
// maximum and sum of the softmax over chunks of 128 positions, all in FP32.
#include "paged.cuh"

namespace fo {

constexpr int PA_CHUNK = 128;

template <int D, typename T, int FORMAT>
__global__ void __launch_bounds__(PA_CHUNK) paged_attention_kernel(const __grid_constant__ fo_paged_attention_launch a) {
    __shared__ float qs[D], ps[PA_CHUNK], red[4];
    const int64_t seq = blockIdx.y;
    const int head = blockIdx.x, r = blockIdx.z, t = threadIdx.x;
    const int page = a.kv.page_size;
    const Sequence s = load_sequence(a.batch, page, seq, a.err);
    if (r >= s.n) return;
    const int64_t row = s.first + r, p = s.len - s.n + r;
    const T *q = static_cast<const T *>(a.q.data) + row * a.q.row_stride + head * a.q.head_stride;
    for (int d = t; d < D; d += PA_CHUNK) qs[d] = load1(q + d);
    __syncthreads();
    const int kvh = head / (a.q.heads / a.kv.n_kv_heads);
    const int64_t low = a.window > 0 ? max64(0, p + 1 - a.window) : 0;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int64_t c = low; c <= p; c += PA_CHUNK) {
        const int n = (int)min64(PA_CHUNK, p + 1 - c);
        float x = -INFINITY;
        bool valid;
        if (t < n) {
            const int64_t at = c + t;
            const int64_t tile = page_of(a.batch, a.kv.n_pages, seq, at / page, a.err, valid) * a.kv.n_kv_heads + kvh;
            const uint32_t *k = reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.kv.k_codes) +
                                                                   (tile * page + at % page) * D);
            float acc = 0.0f;
            for (int i = 0; i < D / 4; i++) {
                float f[4];
                decode4<FORMAT>(k[i], f);
                for (int e = 0; e < 4; e++) acc = fmaf(qs[4 * i + e], f[e], acc);
            }
            x = acc * a.kv.k_scales[tile] * a.scale;
        }
        float mx = warp_max(x);
        if ((t & 31) == 0) red[t >> 5] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = fmaxf(m, mx);
        const float alpha = expf(m - mn), w = t < n ? expf(x - mn) : 0.0f;
        ps[t] = w;
        const float sum = warp_sum(w);
        __syncthreads();
        if ((t & 31) == 0) red[t >> 5] = sum;
        __syncthreads();
        l = l * alpha + (red[0] + red[1]) + (red[2] + red[3]);
        m = mn;
        if (t < D) {
            o *= alpha;
            for (int i = 0; i < n; i++) {
                const int64_t at = c + i;
                const int64_t tile =
                    page_of(a.batch, a.kv.n_pages, seq, at / page, a.err, valid) * a.kv.n_kv_heads + kvh;
                const uint8_t *v = static_cast<const uint8_t *>(a.kv.v_codes) + (tile * page + at % page) * D;
                float f[4];
                decode4<FORMAT>(v[t], f);
                o = fmaf(ps[i] * a.kv.v_scales[tile], f[0], o);
            }
        }
        __syncthreads();
    }
    float total = l;
    if (a.sinks && l > 0.0f) total += expf(a.sinks[head] - m);
    T *out = static_cast<T *>(a.out.data) + row * a.out.row_stride + head * a.out.head_stride;
    if (t < D) store1(out + t, l > 0.0f ? o / total : 0.0f);
    if (a.lse && t == 0) a.lse[row * a.q.heads + head] = l > 0.0f ? m + logf(l) : -INFINITY;
}

}  // namespace fo

extern "C" cudaError_t fo_launch_paged_attention(const fo_paged_attention_launch *a, cudaStream_t stream) {
    if (a->batch.total_rows <= 0) return cudaSuccess;
    const dim3 grid((unsigned)a->q.heads, (unsigned)a->batch.n_seqs, (unsigned)a->batch.max_rows);
    auto go = [&](auto *kernel) { kernel<<<grid, fo::PA_CHUNK, 0, stream>>>(*a); };
    const bool i8 = a->kv.format == FO_PAGED_I8, f32 = a->q.dtype == FO_DT_F32;
    if (a->kv.head_dim == 64) {
        if (f32) i8 ? go(fo::paged_attention_kernel<64, float, 0>) : go(fo::paged_attention_kernel<64, float, 1>);
        else i8 ? go(fo::paged_attention_kernel<64, uint16_t, 0>) : go(fo::paged_attention_kernel<64, uint16_t, 1>);
    } else {
        if (f32) i8 ? go(fo::paged_attention_kernel<128, float, 0>) : go(fo::paged_attention_kernel<128, float, 1>);
        else i8 ? go(fo::paged_attention_kernel<128, uint16_t, 0>) : go(fo::paged_attention_kernel<128, uint16_t, 1>);
    }
    return cudaGetLastError();
}
