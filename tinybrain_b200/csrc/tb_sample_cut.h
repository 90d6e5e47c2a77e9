// tb_sample_cut.h -- where a row's weights end, for the device and the host (the
// tests compile it with the host's compiler).
#pragma once

#include <cmath>

#ifdef __CUDACC__
#define TB_CUT __host__ __device__ __forceinline__
#else
#define TB_CUT inline
#endif

namespace tb {

constexpr double kNoWeight = 700.0;  // nats below the maximum where weights end

// The lowest value with a weight at temperature T: the smallest float that lies no
// more than kNoWeight T below `top`.  Rounded up: the exponentials of the weights are
// made for no less, and half a step of a large `top` can be many times T.
TB_CUT float lowest_weighted(float top, float T) {
    const double end = (double)top - kNoWeight * (double)T;
#ifdef __CUDA_ARCH__
    return __double2float_ru(end);  // the same in one instruction
#else
    const float cut = (float)end;
    return (double)cut < end ? nextafterf(cut, INFINITY) : cut;
#endif
}

}  // namespace tb
