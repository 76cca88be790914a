// rope.cu -- rotary positions: the table of {cos, sin} by position, and the
// rotation of rows of heads (forward, or transposed for the gradient).
//
// Pair (a, b) of a row at position p becomes (a c - b s, b c + a s) with
// {c, s} = table[p][pair].  Every value is read once and written once and a
// table row serves all heads of a token, so the kernel is bound by HBM: a
// thread takes the same eight elements (or the same eight pairs, in the half
// layout) of two or four heads of one row, so its table entries are read
// once and all its loads are in flight together, asked for before the row's
// position is known.  Measured: 32,771 rows x 40 heads x 128 BF16 119 us (5.8
// TB/s, 0.90 of the measured copy bandwidth), 6,544 rows x 24 x 64 FP32 16.6 us
// (4.9 TB/s; a launch that does next to nothing takes 2.4 us), 8 rows 2.4 us.
#include "paged_rope.cuh"

namespace fo {

__global__ void __launch_bounds__(256) rope_table_kernel(float2 *table, int64_t positions, int pairs,
                                                         fo_rope_scaling s) {
    const int64_t n = positions * pairs;
    const double rot = 2.0 * pairs;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (int64_t)gridDim.x * blockDim.x) {
        const int64_t p = e / pairs;
        const int i = (int)(e - p * pairs);
        const double theta =
            s.scaling == FO_ROPE_NTK && pairs > 1 ? s.theta * pow(s.factor, rot / (rot - 2.0)) : s.theta;
        double f = pow(theta, -2.0 * i / rot), m = 1.0;
        if (s.scaling == FO_ROPE_LINEAR) f /= s.factor;
        if (s.scaling == FO_ROPE_YARN) {
            // Pair number at which a frequency turns beta times over the
            // original positions: rot ln(original / (2 pi beta)) / (2 ln theta).
            const double two_pi = 6.283185307179586;
            const double at_fast = rot * log(s.original_positions / (s.beta_fast * two_pi)) / (2.0 * log(s.theta));
            const double at_slow = rot * log(s.original_positions / (s.beta_slow * two_pi)) / (2.0 * log(s.theta));
            const double low = fmax(floor(at_fast), 0.0), high = fmin(ceil(at_slow), rot - 1.0);
            const double ramp = fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
            f = f / s.factor * ramp + f * (1.0 - ramp);
            m = s.attention_factor != 0.0 ? s.attention_factor : 0.1 * log(s.factor) + 1.0;
        }
        double sn, cs;
        sincos((double)p * f, &sn, &cs);
        table[e] = make_float2((float)(cs * m), (float)(sn * m));
    }
}

template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS, 3) rope_kernel(const __grid_constant__ fo_rope_launch a) {
    wait_for_prior_kernel();
    rope_block<T, HALF, VEC>(a, blockIdx.x, threadIdx.x, [&](int64_t row, bool &padded) {
        padded = false;
        return a.rope.row_positions ? (int64_t)a.rope.row_positions[row] : row;
    });
}

}  // namespace fo

extern "C" cudaError_t fo_launch_rope_table(float *table, int64_t positions, int32_t rot_dim,
                                            const fo_rope_scaling *scaling, cudaStream_t stream) {
    const int64_t n = positions * (rot_dim / 2);
    if (n <= 0) return cudaSuccess;
    const unsigned grid = (unsigned)fo::min64((n + 255) / 256, 148 * 16);
    fo::rope_table_kernel<<<grid, 256, 0, stream>>>(reinterpret_cast<float2 *>(table), positions, rot_dim / 2,
                                                    *scaling);
    return cudaGetLastError();
}

extern "C" cudaError_t fo_launch_rope(const fo_rope_launch *args, cudaStream_t stream) {
    if (args->rows <= 0 || args->x.heads <= 0) return cudaSuccess;
    fo_rope_launch a = *args;
    const bool vec = fo::rope_shape(&a);
    const int rows = fo::ROPE_THREADS / a.block_x;
    const unsigned grid = (unsigned)((a.rows + rows - 1) / rows), block = fo::ROPE_THREADS;
    const bool half = a.rope.layout == FO_ROPE_HALF;
    cudaError_t e = cudaSuccess;
    auto go = [&](auto *kernel) { e = fo::launch(kernel, grid, block, 0, stream, a); };
    if (a.x.dtype == FO_DT_F32) {
        if (half) vec ? go(fo::rope_kernel<float, true, true>) : go(fo::rope_kernel<float, true, false>);
        else vec ? go(fo::rope_kernel<float, false, true>) : go(fo::rope_kernel<float, false, false>);
    } else {
        if (half) vec ? go(fo::rope_kernel<uint16_t, true, true>) : go(fo::rope_kernel<uint16_t, true, false>);
        else vec ? go(fo::rope_kernel<uint16_t, false, true>) : go(fo::rope_kernel<uint16_t, false, false>);
    }
    return e;
}
