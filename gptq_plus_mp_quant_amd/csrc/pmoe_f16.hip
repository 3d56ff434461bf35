// The products of a mixture-of-experts layer: fp16 tensors.
#include "pmoe_kernels.h"

template void rq_moe_in<__half>(const __half*, int64_t, const RqExperts&, int, const RqExperts&, int, const RqMoe&, hipStream_t);
template void rq_moe_out<__half>(const RqExperts&, int, const RqMoe&, __half*, int64_t, hipStream_t);
