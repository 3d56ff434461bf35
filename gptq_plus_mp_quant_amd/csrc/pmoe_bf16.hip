// The products of a mixture-of-experts layer: bf16 tensors.
#include "pmoe_kernels.h"

template void rq_moe_in<__hip_bfloat16>(const __hip_bfloat16*, int64_t, const RqExperts&, int, const RqExperts&, int, const RqMoe&, hipStream_t);
template void rq_moe_out<__hip_bfloat16>(const RqExperts&, int, const RqMoe&, __hip_bfloat16*, int64_t, hipStream_t);
