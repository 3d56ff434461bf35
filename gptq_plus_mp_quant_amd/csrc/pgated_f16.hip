// The gated half of a packed feed-forward block: fp16 tensors.
#include "pgated_kernels.h"

template void rq_gated_rows<__half>(const __half*, void*, int, int64_t, const RqPacked&, int, const RqPacked&, int, int, float*, __half*, int64_t, hipStream_t);
template void rq_gated_pre_grad<__half>(const __half*, int64_t, int, int, int, const float*, float*, hipStream_t);
template void rq_gated_join<__half>(const float*, int, int, int, __half*, int64_t, hipStream_t);
