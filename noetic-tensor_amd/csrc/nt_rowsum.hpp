// A row's chunks loaded without a branch, and sums of 2^(v c) over its values v in f32 exponentials, one lane's share,
// with f64 totals.
#pragma once

#include "nt_exp64.hpp"
#include "nt_rows.hpp"

namespace nt {
namespace {

// A row's loads, none under a condition: with one, the compiler lets every load wait for the one before it, whose registers
// the other branch would write. AL (aligned_rows, row bytes below 2^31): non-temporal buffer loads, zeros past the row's
// end; f32 rows in two groups of four columns a lane, 256 apart, so that each instruction reads one contiguous kilobyte.
// Otherwise loads at the elements' own alignment, the row's last ones from 8 columns before its end, so that a lane there
// holds columns of its neighbour too; rows of under 8 columns by elements. Column j of lane l in chunk ch is col(); those
// that are not the lane's own (its neighbour's, or past the row) are in the row's last chunk only, where clean() gives them -inf.
template <int DT, int MK, bool AL>
struct RowLoad {
    static constexpr bool kSplit = AL && DT == NT_F32;
    static constexpr int kHalf = kChunk / 2;
    const void *x, *m;
    __amdgpu_buffer_rsrc_t xr, mr;
    int64_t V;
    int last;

    __device__ __forceinline__ RowLoad(const void *xrow, const void *mrow, int64_t V_, int nc) : x(xrow), m(mrow), V(V_), last(nc - 1) {
        if constexpr (AL) {
            xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(xrow), short(0), int(V) * Elem<DT>::kBytes, kBufferWord3);
            mr = xr;
            if constexpr (MK != NT_MASK_NONE)
                mr = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(mrow), short(0), int(V) * MaskWords<MK>::kBytes, kBufferWord3);
        }
    }
    static __device__ __forceinline__ int64_t own(int ch, int lane) { return int64_t(ch) * kChunk + lane * kEpl; }
    __device__ __forceinline__ int64_t first(int ch, int lane) const {
        const int64_t e0 = own(ch, lane);
        if constexpr (AL) return e0;
        else return V < kEpl ? e0 : (e0 + kEpl <= V ? e0 : V - kEpl);
    }
    __device__ __forceinline__ int64_t col(int ch, int lane, int j) const {
        if constexpr (kSplit) return int64_t(ch) * kChunk + lane * 4 + (j < 4 ? j : kHalf - 4 + j);
        else return first(ch, lane) + j;
    }
    // The raw words of chunk ch (in: the row has it; otherwise anything).
    __device__ __forceinline__ void load(Raw<DT, MK> &r, int ch, int lane, bool in = true) const {
        if constexpr (kSplit) {
            const int e0 = in ? ch * kChunk + lane * 4 : int(V);
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const auto a = __builtin_amdgcn_raw_buffer_load_b128(xr, (e0 + q * kHalf) * 4, 0, kCachePolicyNT);
#pragma unroll
                for (int i = 0; i < 4; i++) r.x[4 * q + i] = a[i];
                if constexpr (MK == NT_MASK_U8) {
                    r.m[q] = __builtin_amdgcn_raw_buffer_load_b32(mr, e0 + q * kHalf, 0, kCachePolicyNT);
                } else if constexpr (MK == NT_MASK_F32) {
                    const auto k = __builtin_amdgcn_raw_buffer_load_b128(mr, (e0 + q * kHalf) * 4, 0, kCachePolicyNT);
#pragma unroll
                    for (int i = 0; i < 4; i++) r.m[4 * q + i] = k[i];
                }
            }
        } else if constexpr (AL) {
            const int e0 = in ? int(own(ch, lane)) : int(V);
#pragma unroll
            for (int q = 0; q < Elem<DT>::kWords / 4; q++) {
                const auto a = __builtin_amdgcn_raw_buffer_load_b128(xr, e0 * Elem<DT>::kBytes + 16 * q, 0, kCachePolicyNT);
#pragma unroll
                for (int i = 0; i < 4; i++) r.x[4 * q + i] = a[i];
            }
            if constexpr (MK == NT_MASK_U8) {
                const auto k = __builtin_amdgcn_raw_buffer_load_b64(mr, e0, 0, kCachePolicyNT);
                r.m[0] = k[0];
                r.m[1] = k[1];
            } else if constexpr (MK == NT_MASK_F32) {
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const auto a = __builtin_amdgcn_raw_buffer_load_b128(mr, e0 * 4 + 16 * q, 0, kCachePolicyNT);
#pragma unroll
                    for (int i = 0; i < 4; i++) r.m[4 * q + i] = a[i];
                }
            }
        } else if (V < kEpl) {
            load_raw<DT, MK, false>(r, x, m, in ? own(ch, lane) : V, V);
        } else {
            const int64_t e = in ? first(ch, lane) : 0;
            if constexpr (DT == NT_F32) {
                const u32x4_f32 *q = reinterpret_cast<const u32x4_f32 *>(static_cast<const float *>(x) + e);
                const u32x4_f32 a = q[0], b = q[1];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    r.x[i] = a[i];
                    r.x[4 + i] = b[i];
                }
            } else {
                const u32x4_f16 a = *reinterpret_cast<const u32x4_f16 *>(static_cast<const uint16_t *>(x) + e);
#pragma unroll
                for (int i = 0; i < 4; i++) r.x[i] = a[i];
            }
            if constexpr (MK == NT_MASK_U8) {
                const u32x2_u8 k = *reinterpret_cast<const u32x2_u8 *>(static_cast<const uint8_t *>(m) + e);
                r.m[0] = k[0];
                r.m[1] = k[1];
            } else if constexpr (MK == NT_MASK_F32) {
                const u32x4_f32 *q = reinterpret_cast<const u32x4_f32 *>(static_cast<const float *>(m) + e);
                const u32x4_f32 a = q[0], b = q[1];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    r.m[i] = a[i];
                    r.m[4 + i] = b[i];
                }
            }
        }
    }
    // Whether column col(j) of the lane is its own.
    __device__ __forceinline__ bool mine(int ch, int lane, int j) const {
        const int64_t e = col(ch, lane, j);
        if constexpr (AL) return e < V;
        else return e >= own(ch, lane) && e < V;
    }
    template <class T>
    __device__ __forceinline__ void clean(T (&v)[kEpl], int ch, int lane) const {
        if (ch != last) return;
#pragma unroll
        for (int j = 0; j < kEpl; j++) v[j] = mine(ch, lane, j) ? v[j] : T(-INFINITY);
    }
};

// take(slot, chunk, next) for chunks c, c + step, .. below c1 with D of them loaded ahead by load(slot, chunk): take uses
// the slot's words and then loads `next` into it. The loop takes D chunks at a time with no condition between them, without
// which the compiler knows how many loads came after the one that it waits for (and else waits for all of them).
template <int D, class L, class F>
__device__ __forceinline__ void stream(int c, int step, int c1, L &&load, F &&take) {
    static_for<0, D>([&](auto k) { load(k, c + k.value * step); });
    for (; c + (D - 1) * step < c1; c += D * step)
        static_for<0, D>([&](auto k) { take(k, c + k.value * step, c + (k.value + D) * step); });
    static_for<0, D>([&](auto k) {
        const int ch = c + k.value * step;
        if (ch < c1) take(k, ch, c1);
    });
}

// A sum relative to the lane's reference: the first maximum it met, moved only where a later
// value lies 60 log2 units above it, so that most chunks cost a weight one fma, one exponential and one addition. The
// reference is kept as the f32 product -ref c that the fma adds, and what its rounding and c's leave of it goes
// into at(). Products past 2^20, whose f32 steps are no small part of a log2 unit, are taken by differences.
// A weight is within 2^-23 (the instruction) and |t| 2^-23 ln 2 of its argument t (the fma's rounding and
// c's); a NaN or +inf leaves a NaN in S.
struct LaneSums {
    double S = 0.0;
    float ref = -INFINITY, neg = 0.0f, lim = -INFINITY;

    // Takes `top`, not below the limit (a NaN among others), into the reference; whether weights go by the fma.
    __device__ __forceinline__ bool settle(float top, float c) {
        if (!(top < INFINITY)) {
            S = NAN;
            return true;
        }
        const float r = fmaxf(ref, top), now = -(r * c);
        const bool far = fabsf(now) > 0x1p20f;
        if (ref != -INFINITY) {
            const double was = lim == -INFINITY ? -double(ref) * double(c) : double(neg);
            S *= exp2_64((far ? -double(r) * double(c) : double(now)) - was, 1.0, -1100.0);
        }
        ref = r;
        neg = far ? 0.0f : now;  // (unused there, and maybe infinite: an excluded value's weight is 0 and no NaN)
        lim = far ? -INFINITY : fminf(r + 60.0f / c, FLT_MAX);  // (an infinity is past it at any temperature)
        return !far;
    }
    // Takes 8 values; their maximum.
    __device__ __forceinline__ float add(const float v[kEpl], float c) {
        float w[kEpl];
        const float top = max8_hw(v);
        bool fast = top <= lim;
        // (lanes without a token so far have none here either: their weights are 0)
        if (!fast && !(top == -INFINITY)) fast = settle(top, c);
        else fast = true;
        if (fast) {
#pragma unroll
            for (int j = 0; j < kEpl; j++) w[j] = exp2_hw(fmaf(v[j], c, neg));
        } else {
#pragma unroll
            for (int j = 0; j < kEpl; j++) w[j] = exp2_hw((v[j] - ref) * c);
        }
        S += double(tree8(w));
        return top;
    }
    // The value whose weight is 1 (c: what c32 is the f32 of); -inf where the lane met no token.
    __device__ __forceinline__ double at(double c, float c32) const {
        if (ref == -INFINITY || lim == -INFINITY) return double(ref);
        return -(double(neg) + double(ref) * (double(c32) - c)) / c;
    }
};

// The same over f64 values z of unit scale (tempered logits under an additive mask, which may lower a row so far that an f32 step is
// no small part of their differences): the exponentials' arguments are f64 differences from the reference, rounded to f32,
// and the reference is moved where a value lies 16 above it. A weight is within 2^-23 and |t| 3 2^-24 ln 2. What f32 would round to an
// infinity (kPast on) is one: excluded, or a NaN in S.
struct FarSum {
    static constexpr double kPast = 0x1.ffffffp127, kNothing = -0x1.fffffefffffffp127;  // (the next one to -kPast)
    double S = 0.0, ref = kNothing;

    __device__ __forceinline__ void add(const double z[kEpl], double low) {
        float d[kEpl];
#pragma unroll
        for (int j = 0; j < kEpl; j++) d[j] = float(z[j] - ref);
        if (!(max8_hw(d) <= 16.0f)) {
            double high = z[0];
#pragma unroll
            for (int j = 1; j < kEpl; j++) high = fmax(high, z[j]);
            if (high < kPast) {
                S *= exp2_64(ref - high, kLog2e64, low);
                ref = high;
#pragma unroll
                for (int j = 0; j < kEpl; j++) d[j] = float(z[j] - ref);
            } else {
                S = NAN;
            }
        }
#pragma unroll
        for (int j = 0; j < kEpl; j++) d[j] = exp2_hw(d[j] * kLog2e);
        S += double(tree8(d));
    }
    // The z whose weight is 1; -inf where the lane met no token.
    __device__ __forceinline__ double at(double, float) const { return ref == kNothing ? -INFINITY : ref; }
};

__device__ __forceinline__ double wave_max_d(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, kWave));
    return v;
}

// S relative to a, moved to the reference `to` (at least a); low: -1100 / c.
__device__ __forceinline__ double moved(double S, double a, double to, double c, double low) {
    return a == -INFINITY || a == to ? S : S * exp2_64(a - to, c, low);
}

// A temperature whose scale of the exponentials, log2(e) / T, f32 holds: T itself one of its normal numbers.
inline int check_scale(double T) {
    if (T >= double(FLT_MIN) && T <= double(FLT_MAX)) return 0;
    char buf[128];
    std::snprintf(buf, sizeof buf, "tempered_logits: temperature %g (%s)", T,
                  T > 0.0 && std::isfinite(T) ? "must be a normal f32" : "must be positive");
    return fail(NT_E_ARG, buf);
}

}  // namespace
}  // namespace nt
