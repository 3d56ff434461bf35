// Gradients through two packed weights at once, from fp32 gradients of their products.
#include "plinear_types.h"
#include "plinear_cols.h"

void rq_cols_parts2(const float* dy, int T, int64_t ldy, int64_t plane, const RqPacked& w0, const RqPacked& w1, int nbits,
                    const RqColSplit& sp, float* part, hipStream_t s) {
  cols_of<float, 2>(Cols<float>{dy, T, ldy, plane, &w1, sp, part, {}}, w0, nbits, s);
}
