// paged_attention.cu -- attention of a batch's query rows over a paged 8-bit KV
// cache: every position before the row's own, or the newest of them (the kernel
// and what it measured: paged_attention.cuh).  It overlaps the one before it up to
// its wait_for_prior_kernel().
#include "paged_attention.cuh"

extern "C" cudaError_t fo_launch_paged_attention(const fo_paged_attention_launch *args, int sms, cudaStream_t stream) {
    return fo::launch_attention<false, false>(*args, sms, stream);
}
