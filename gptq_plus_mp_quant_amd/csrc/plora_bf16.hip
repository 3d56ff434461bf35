// Packed linears with low-rank adapters: bf16 tensors.
#include "plora_kernels.h"

template void rq_lora_down<__hip_bfloat16>(const RqDownJobs<__hip_bfloat16>&, void*, int, hipStream_t);
template void rq_lora_rows<__hip_bfloat16>(const __hip_bfloat16*, int, int64_t, const RqPacked&, int, const __hip_bfloat16*, const RqLora<__hip_bfloat16>&, const RqLow&, const void*, __hip_bfloat16*, int64_t, hipStream_t);
template void rq_lora_grads<__hip_bfloat16>(const RqLoraDx<__hip_bfloat16>&, const __hip_bfloat16*, int64_t, int, const __hip_bfloat16*, int64_t, int, int, const RqLora<__hip_bfloat16>&, const RqLow&, const RqLow&, __hip_bfloat16*, __hip_bfloat16*, hipStream_t);
