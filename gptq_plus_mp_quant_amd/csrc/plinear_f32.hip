// Products with packed weights: fp32 tensors.
#include "plinear_types.h"
#include "plinear_rows.h"
#include "plinear_cols.h"

template void rq_linear_rows<float>(const float*, int, int64_t, const RqPacked&, int, const float*, float*, int64_t, hipStream_t);
template void rq_linear_cols<float>(const float*, int, int64_t, const RqPacked&, int, float*, float*, int64_t, hipStream_t);
