// Which points a block of the two-pass group norm takes; plain C++, for the kernels
// and for host programs.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define CPDE_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define CPDE_HOST_DEVICE inline
#endif

namespace cpde::ops {

// The points [lo, hi) of split `split` of `splits`, for lengths below 2^31 and up to
// 2^31 splits: their sum needs the 32nd bit.
CPDE_HOST_DEVICE void split_range(int32_t length, int32_t split, int32_t splits, int32_t& lo, int32_t& hi) {
    const int64_t per = (uint32_t(length) + uint32_t(splits) - 1) / uint32_t(splits);
    const int64_t first = split * per;
    lo = int32_t(first < length ? first : length);
    hi = int32_t(first + per < length ? first + per : length);
}

}  // namespace cpde::ops
