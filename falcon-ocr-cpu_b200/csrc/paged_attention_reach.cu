// paged_attention_reach.cu -- the paged attention's kernel where rows see a few
// first positions behind their window, or stand beside longer sequences that
// another kernel takes (paged_attention.cuh): the few query rows of decode steps.
#include "paged_attention.cuh"

extern "C" cudaError_t fo_launch_paged_attention_reach(const fo_paged_attention_launch *args, int sms,
                                                       cudaStream_t stream) {
    return fo::launch_attention<true, true>(*args, sms, stream);
}
