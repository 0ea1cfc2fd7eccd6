// 2^t in f64 for the kernels whose sums decide tokens.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nt {
namespace {

// 2^t for t <= 1000 within 2e-14 relative; t below -1100 (and a NaN: the callers look for those
// themselves) gives 0. 2^n by v_ldexp_f64 with n = t to the nearest whole number, taken by the addition of
// 1.5 2^52, which leaves n in the sum's low word, times 2^f for f in [-1/2, 1/2]: the polynomial that
// agrees with 2^f at the ten Chebyshev nodes of that interval (its largest relative error is 1.8e-14). f64 fma, add
// and max run at the f32 rate here, 16 lanes a clock and SIMD, so that 16 instructions are 64 clocks a wave.
__device__ __forceinline__ double exp2_64(double t) {
    t = fmax(t, -1100.0);
    const double y = t + 0x1.8p52;
    const int n = int(uint32_t(uint64_t(__double_as_longlong(y))));
    const double f = t - (y - 0x1.8p52);
    double p = 0x1.b6571de2f2351p-24;
    p = fma(p, f, 0x1.63ef969a64d3cp-20);
    p = fma(p, f, 0x1.ffcb76789860fp-17);
    p = fma(p, f, 0x1.43088e257f341p-13);
    p = fma(p, f, 0x1.5d87fe908f88ap-10);
    p = fma(p, f, 0x1.3b2ab72b175eep-7);
    p = fma(p, f, 0x1.c6b08d7044119p-5);
    p = fma(p, f, 0x1.ebfbdff8149f2p-3);
    p = fma(p, f, 0x1.62e42fefa39f7p-1);
    p = fma(p, f, 0x1.000000000003dp+0);
    return __builtin_ldexp(p, n);
}

constexpr double kLog2e64 = 1.4426950408889634074;

}  // namespace
}  // namespace nt
