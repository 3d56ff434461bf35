// The products of a mixture-of-experts layer: fp32 tensors.
#include "pmoe_kernels.h"

template void rq_moe_in<float>(const float*, int64_t, const RqExperts&, int, const RqExperts&, int, const RqMoe&, hipStream_t);
template void rq_moe_out<float>(const RqExperts&, int, const RqMoe&, float*, int64_t, hipStream_t);
