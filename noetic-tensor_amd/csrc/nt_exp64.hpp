// 2^t in f64 for the kernels whose sums decide tokens.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nt {
namespace {

constexpr double kLog2e64 = 1.4426950408889634074;

// 2^(d c) for d c <= 1000 within 2e-12 relative and 0 for d at least `low` below 0 (low c is -1100; a NaN gives 0 too: the
// callers look for those themselves). 2^n by v_ldexp_f64 with n = d c to the nearest whole number, taken by an fma
// onto 1.5 2^52, which leaves n in the low word, times 2^f for f in [-1/2, 1/2]: the polynomial that agrees with
// 2^f at the nine Chebyshev nodes of that interval (its largest relative error is 1.1e-12). An f64 instruction of
// any of these kinds takes 4.5 clocks a wave where an f32 fma takes 2.4 and v_exp_f32 8.2 (measured), so that a weight with
// its conversion, difference and addition is 72 clocks, against about 20 in f32.
__device__ __forceinline__ double exp2_64(double d, double c, double low) {
    d = fmax(d, low);
    const double y = fma(d, c, 0x1.8p52);
    const int n = int(uint32_t(uint64_t(__double_as_longlong(y))));
    const double f = fma(d, c, 0x1.8p52 - y);
    double p = 0x1.63d136366db24p-20;
    p = fma(p, f, 0x1.00dc4a532fb8ep-16);
    p = fma(p, f, 0x1.4308ac85aa947p-13);
    p = fma(p, f, 0x1.5d8745a728441p-10);
    p = fma(p, f, 0x1.3b2ab7181b755p-7);
    p = fma(p, f, 0x1.c6b08dd6fd234p-5);
    p = fma(p, f, 0x1.ebfbdff823cedp-3);
    p = fma(p, f, 0x1.62e42fef84cf0p-1);
    p = fma(p, f, 1.0);
    return __builtin_ldexp(p, n);
}

}  // namespace
}  // namespace nt
