// Packed linears with low-rank adapters: fp32 tensors.
#include "plora_kernels.h"

template void rq_lora_down<float>(const RqDownJobs<float>&, void*, int, hipStream_t);
template void rq_lora_rows<float>(const float*, int, int64_t, const RqPacked&, int, const float*, const RqLora<float>&, const RqLow&, const void*, float*, int64_t, hipStream_t);
template void rq_lora_grads<float>(const RqLoraDx<float>&, const float*, int64_t, int, const float*, int64_t, int, int, const RqLora<float>&, const RqLow&, const RqLow&, float*, float*, hipStream_t);
