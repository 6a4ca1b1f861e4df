// Division by a number that a launch has in common, by one product: a number between 1 and 2^31, and quotients of
// anything below 2^31.  (Plain C++, so that a host test runs it.)
//
// With 2^(s-1) < d <= 2^s and m = floor(2^(31+s) / d) + 1 the product m d is past 2^(31+s) by at most d, so q m / 2^(31+s) is
// past q / d by at most q / 2^(31+s) < 2^-s <= 1 / d: not enough to reach the next whole number.  m has 32 bits.  (Division
// by invariant integers: T. Granlund and P. Montgomery, PLDI 1994.)
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define B200ALG_BOTH __host__ __device__ __forceinline__
#else
#define B200ALG_BOTH inline
#endif

namespace b200alg {

struct FastDivide {
    uint32_t d, m, shift;
    FastDivide() = default;
    explicit FastDivide(uint32_t divisor) : d(divisor), shift(31) {
        while (((uint64_t)d << 31) > (uint64_t)1 << shift) ++shift;
        m = (uint32_t)(((uint64_t)1 << shift) / d + 1);
    }
    B200ALG_BOTH uint32_t operator()(uint32_t q) const { return (uint32_t)((uint64_t)q * m >> shift); }
};

}  // namespace b200alg
