// Gradients of products with packed weights: fp16 tensors.
#include "plinear_types.h"
#include "plinear_cols.h"

template void rq_linear_cols<__half>(const __half*, int, int64_t, const RqPacked&, int, float*, __half*, int64_t, hipStream_t);
template void rq_lora_cols<__half>(const __half*, int, int64_t, const RqPacked&, int, const RqColSplit&, float*, const RqDownJobs<__half>&, hipStream_t);
