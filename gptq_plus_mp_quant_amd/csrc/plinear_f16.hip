// Products with packed weights: fp16 tensors.
#include "plinear_types.h"
#include "plinear_rows.h"

template void rq_linear_rows<__half>(const __half*, int, int64_t, const RqPacked&, int, const __half*, __half*, int64_t, hipStream_t);
