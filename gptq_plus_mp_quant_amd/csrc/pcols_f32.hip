// Gradients of products with packed weights: fp32 tensors.
#include "plinear_types.h"
#include "plinear_cols.h"

template void rq_linear_cols<float>(const float*, int, int64_t, const RqPacked&, int, float*, float*, int64_t, hipStream_t);
template void rq_lora_cols<float>(const float*, int, int64_t, const RqPacked&, int, const RqColSplit&, float*, const RqDownJobs<float>&, hipStream_t);
template void rq_cols_parts<float>(const float*, int, int64_t, const RqPacked&, int, const RqColSplit&, float*, hipStream_t);
