// The gated half of a packed feed-forward block: bf16 tensors.
#include "pgated_kernels.h"

template void rq_gated_rows<__hip_bfloat16>(const __hip_bfloat16*, void*, int, int64_t, const RqPacked&, int, const RqPacked&, int, int, float*, __hip_bfloat16*, int64_t, hipStream_t);
template void rq_gated_pre_grad<__hip_bfloat16>(const __hip_bfloat16*, int64_t, int, int, int, const float*, float*, hipStream_t);
template void rq_gated_join<__hip_bfloat16>(const float*, int, int, int, __hip_bfloat16*, int64_t, hipStream_t);
