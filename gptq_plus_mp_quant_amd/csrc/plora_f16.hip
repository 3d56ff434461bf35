// Packed linears with low-rank adapters: fp16 tensors.
#include "plora_kernels.h"

template void rq_lora_down<__half>(const RqDownJobs<__half>&, void*, int, hipStream_t);
template void rq_lora_rows<__half>(const __half*, int, int64_t, const RqPacked&, int, const __half*, const RqLora<__half>&, const RqLow&, const void*, __half*, int64_t, hipStream_t);
template void rq_lora_grads<__half>(const RqLoraDx<__half>&, const __half*, int64_t, int, const __half*, int64_t, int, int, const RqLora<__half>&, const RqLow&, const RqLow&, __half*, __half*, hipStream_t);
