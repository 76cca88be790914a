// paged_attention_window.cu -- the paged attention's kernel for windows without
// first positions (paged_attention.cuh), where a lost page is lost to the rows that
// see it alone: few query rows of decode steps.
#include "paged_attention.cuh"

extern "C" cudaError_t fo_launch_paged_attention_window(const fo_paged_attention_launch *args, int sms,
                                                        cudaStream_t stream) {
    return fo::launch_attention<false, true>(*args, sms, stream);
}
