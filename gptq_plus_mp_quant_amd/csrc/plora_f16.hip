// Packed linears with low-rank adapters: fp16 tensors.
#include "plora_kernels.h"

template void rq_lora_down<__half>(const __half*, int, int64_t, int, bool, const RqLora<__half>&, const RqLow&, hipStream_t);
template void rq_lora_rows<__half>(const __half*, int, int64_t, const RqPacked&, int, const __half*, const RqLora<__half>&, const RqLow&, __half*, int64_t, hipStream_t);
template void rq_lora_dx<__half>(const float*, int, int64_t, int, int, const RqLora<__half>&, const RqLow&, __half*, int64_t, hipStream_t);
template void rq_lora_outer<__half>(const __half*, int64_t, int, const __half*, int64_t, int, int, const RqLora<__half>&, const RqLow&, const RqLow&, __half*, __half*, hipStream_t);
