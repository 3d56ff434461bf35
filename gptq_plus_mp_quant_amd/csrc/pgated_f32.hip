// The gated half of a packed feed-forward block: fp32 tensors.
#include "pgated_kernels.h"

template void rq_gated_rows<float>(const float*, void*, int, int64_t, const RqPacked&, int, const RqPacked&, int, int, float*, float*, int64_t, hipStream_t);
template void rq_gated_pre_grad<float>(const float*, int64_t, int, int, int, const float*, float*, hipStream_t);
template void rq_gated_join<float>(const float*, int, int, int, float*, int64_t, hipStream_t);
