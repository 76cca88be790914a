// paged_append_axes.cu -- appending to the paged 8-bit cache, rows rotated by
// positions on several axes (the kernels: paged_append.cuh).
#include "paged_append.cuh"

extern "C" cudaError_t fo_launch_paged_append_axes(const fo_append_launch *a, cudaStream_t stream) {
    return fo::launch_append<true>(*a, stream);
}
