// Packed linears with low-rank adapters: fp32 tensors.
#include "plora_kernels.h"

template void rq_lora_down<float>(const float*, int, int64_t, int, bool, const RqLora<float>&, const RqLow&, hipStream_t);
template void rq_lora_rows<float>(const float*, int, int64_t, const RqPacked&, int, const float*, const RqLora<float>&, const RqLow&, float*, int64_t, hipStream_t);
template void rq_lora_dx<float>(const float*, int, int64_t, int, int, const RqLora<float>&, const RqLow&, float*, int64_t, hipStream_t);
template void rq_lora_outer<float>(const float*, int64_t, int, const float*, int64_t, int, int, const RqLora<float>&, const RqLow&, const RqLow&, float*, float*, hipStream_t);
