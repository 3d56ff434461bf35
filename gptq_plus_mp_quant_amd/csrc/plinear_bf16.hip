// Products with packed weights: bf16 tensors.
#include "plinear_types.h"
#include "plinear_rows.h"
#include "plinear_cols.h"

template void rq_linear_rows<__hip_bfloat16>(const __hip_bfloat16*, int, int64_t, const RqPacked&, int, const __hip_bfloat16*, __hip_bfloat16*, int64_t, hipStream_t);
template void rq_linear_cols<__hip_bfloat16>(const __hip_bfloat16*, int, int64_t, const RqPacked&, int, float*, __hip_bfloat16*, int64_t, hipStream_t);
