// paged_append.cu -- appending to the paged 8-bit cache, rows rotated by one
// position each (the kernels and what they measured: paged_append.cuh).  They
// overlap the one before them up to their wait_for_prior_kernel().
#include "paged_append.cuh"

extern "C" cudaError_t fo_launch_paged_append(const fo_append_launch *a, cudaStream_t stream) {
    return fo::launch_append<false>(*a, stream);
}
