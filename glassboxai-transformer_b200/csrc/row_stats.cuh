// row_stats.cuh -- parts of a row of logits joined into the whole row's
// statistics (verify.cu).  For the host too, where the tests run the tree that
// the kernel's lanes form.
#pragma once

#include <cuda_runtime.h>
#include <math.h>

namespace gbx {

// A part of a row: x its maximum, y the sum of 2^((v - x) c2) over it.  Of two
// parts the one with the larger maximum stays as it is and the other is brought
// to that maximum, so that neither the order of the arguments nor the way a
// compiler contracts a sum of products shows in a bit of the result: in a
// butterfly the two lanes of a pair call this with their arguments swapped, and
// every lane has to end with the same row.
template <class Exp2>
__host__ __device__ __forceinline__ float2 row_join(float2 a, float2 b, float c2, Exp2 exp2_of)
{
    const bool first = a.x >= b.x;
    const float2 hi = first ? a : b, lo = first ? b : a;
    const float down = hi.x == -INFINITY ? 0.0f : (lo.x - hi.x) * c2;   // nothing above -inf yet: both sums as they are
    return make_float2(fmaxf(a.x, b.x), fmaf(lo.y, exp2_of(down), hi.y));
}

}  // namespace gbx
