// 8-bit rows and their product: a row (a token's activations, an output channel's weights) held as integers
// q = round(x / s) with one f32 scale s = max |x| / 127, and C = (qa qb^T) sa sb on the matrix cores.
//
// The reference has no 8-bit type; these stand beside its cast and its reduced-precision product
// (src/tensor/gpu/mod.rs:142-144, 157-162), as MatmulPrecision::Half's bf16 operands do
// (src/tensor/precision.rs:4-8).
//
// Quantizing: the quotient's nearest integer, ties to even, of the exact x / s, so that the integers depend on
// no rounding of the quotient: r = round(x (1/s)) is at most one off next to a border, and the remainder
// x - r s, exact in one fma, says which side x is on. Bounded by HBM: the values in, a byte each out (4096 x 4096 bf16
// there and back 25 us of 21 at a copy's rate, 4.73 TB/s; 1024 x 50304 f32 by columns 147 of 109).
//
// The product: v_mfma_i32_32x32x32_i8 sums exactly in 32 bits (k up to 131071 keeps |sum| under 2^31), so the
// only roundings are the sum's to f32, the two scales' products and the output type's. Up to four tokens are bound by the
// weight's bytes (1 x 128256 x 4096: 98 us with the token's own 8 bits, 5.4 TB/s), a decode batch by the same and the
// rounds of tiles (64 x 50304 x 4096: 53 us, 4.0 TB/s), a prompt by the matrix cores (4096 x 16384 x 4096: 257 us,
// 2.1 POP/s, a large library product's rate here).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "../../include/noetic_ops.h"
#include "nt_internal.hpp"
#include "nt_plan.hpp"
#include "nt_tile.hpp"

namespace nt {
namespace {

using namespace tile;

typedef u32x4 u32x4u __attribute__((aligned(1)));

template <int T>
__device__ __forceinline__ float load_f32(const void *p, int64_t i) {
    if constexpr (T == NT_F32) return static_cast<const float *>(p)[i];
    else if constexpr (T == NT_BF16) return __builtin_bit_cast(float, uint32_t(static_cast<const uint16_t *>(p)[i]) << 16);
    else return float(static_cast<const _Float16 *>(p)[i]);
}

// A row's scale from its largest magnitude, NaN where it holds a NaN or an infinity.
__device__ __forceinline__ float scale_of(float amax, bool finite) { return finite ? amax / 127.0f : NAN; }

// The 8-bit value of x at scale s; `inv` is 1 / s rounded. A row of zeros (s 0) is zeros, as is one whose scale
// is NaN. Scales under 2^-100, whose reciprocal or products may leave f32, take the quotient in f64, which is
// as exact here: |x / s - (n + 1/2)| is 0 or over 2^-33.
__device__ __forceinline__ int quantized(float x, float s, float inv) {
    if (!(s >= 0x1p-100f)) {
        if (!(s > 0.0f)) return 0;
        const double r = rint(double(x) / double(s));
        return int(fmin(fmax(r, -127.0), 127.0));  // (a subnormal scale's own rounding may pass 127)
    }
    float r = rintf(x * inv);
    const float d = 2.0f * fmaf(-r, s, x);  // twice the exact remainder
    const bool odd = (int(r) & 1) != 0;
    if (d > s || (d == s && odd)) r += 1.0f;
    else if (-d > s || (-d == s && odd)) r -= 1.0f;
    return int(r);
}

// Four of them as bytes of a word. x (1/s) + 1.5 2^23 rounds to the integer in one fma and leaves it in the low
// byte; only where some remainder reaches half the scale (a value next to a border) are the four taken again as
// above. (5 operations a value instead of 15: 4096 x 4096 bf16 rows 19.2 -> 16.5 us.)
__device__ __forceinline__ uint32_t quantized4(const float (&x)[4], float s, float inv) {
    constexpr float kMagic = 12582912.0f;
    uint32_t b[4];
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float t = fmaf(x[e], inv, kMagic);
        b[e] = __builtin_bit_cast(uint32_t, t);
        most = fmaxf(most, fabsf(fmaf(-(t - kMagic), s, x[e])));
    }
    if (!(s >= 0x1p-100f) || most * 2.0f >= s)
#pragma unroll
        for (int e = 0; e < 4; e++) b[e] = uint32_t(quantized(x[e], s, inv));
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u),
                                 0x05040100u);
}

// Eight neighbouring values, at the elements' own alignment.
template <int T>
__device__ __forceinline__ void load8(const void *p, int64_t i, float (&x)[8]) {
    if constexpr (T == NT_F32) {
        __builtin_memcpy(x, static_cast<const float *>(p) + i, 32);
    } else {
        uint16_t h[8];
        __builtin_memcpy(h, static_cast<const uint16_t *>(p) + i, 16);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (T == NT_BF16) x[e] = __builtin_bit_cast(float, uint32_t(h[e]) << 16);
            else x[e] = float(__builtin_bit_cast(_Float16, h[e]));
        }
    }
}

// THREADS threads a row, ROWS rows a workgroup: a wave a row while that leaves a lane at most 8 chunks of eight
// values (4096 columns) and gives every CU a row, else 256 threads a row. A lane's first KEEP chunks stay in registers between the two passes; past those
// (16384 columns) the row is read again, from the caches.
template <int T, int THREADS, int KEEP>
__global__ __launch_bounds__(256) void k_quantize_rows(const void *xv, int64_t rows, int64_t cols, int64_t ld, int8_t *q,
                                                       float *scale) {
    constexpr int ROWS = 256 / THREADS;
    __shared__ float s_max[4];
    __shared__ int s_bad[4];
    const int t = threadIdx.x % THREADS;
    const int64_t row = blockIdx.x * int64_t(ROWS) + threadIdx.x / THREADS;
    if (ROWS > 1 && row >= rows) return;
    const int64_t at = row * ld, chunks = cols / 8;
    float x[KEEP][8];
    float m = 0.0f;
    bool bad = false;
    auto see = [&](float v) {
        const float a = fabsf(v);
        bad |= !(a < INFINITY);
        m = fmaxf(m, a);
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const int64_t c = t + int64_t(k) * THREADS;
        if (c < chunks) {
            load8<T>(xv, at + c * 8, x[k]);
#pragma unroll
            for (int e = 0; e < 8; e++) see(x[k][e]);
        }
    }
    for (int64_t c = t + int64_t(KEEP) * THREADS; c < chunks; c += THREADS) {
        float y[8];
        load8<T>(xv, at + c * 8, y);
#pragma unroll
        for (int e = 0; e < 8; e++) see(y[e]);
    }
    if (chunks * 8 + t < cols && t < 8) see(load_f32<T>(xv, at + chunks * 8 + t));
#pragma unroll
    for (int d = 32; d; d /= 2) m = fmaxf(m, __shfl_xor(m, d, 64));
    bool any = __any(bad);
    if constexpr (THREADS > 64) {
        if (t % 64 == 0) s_max[t / 64] = m, s_bad[t / 64] = any;
        __syncthreads();
        m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        any = s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
    }
    const float s = scale_of(m, !any), inv = 1.0f / s;
    if (t == 0) scale[row] = s;
    int8_t *o = q + row * cols;
    auto put = [&](int64_t c, const float (&v)[8]) {
        const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
        const uint32_t w[2] = {quantized4(a, s, inv), quantized4(b, s, inv)};
        __builtin_memcpy(o + c * 8, w, 8);
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const int64_t c = t + int64_t(k) * THREADS;
        if (c < chunks) put(c, x[k]);
    }
    for (int64_t c = t + int64_t(KEEP) * THREADS; c < chunks; c += THREADS) {
        float y[8];
        load8<T>(xv, at + c * 8, y);
        put(c, y);
    }
    if (chunks * 8 + t < cols && t < 8) o[chunks * 8 + t] = int8_t(quantized(load_f32<T>(xv, at + chunks * 8 + t), s, inv));
}

// (a launch holds fewer than 2^32 threads: 2^23 rows at a time)
template <int T>
int launch_rows(const uint8_t *x, int64_t rows, int64_t cols, int64_t ld, int8_t *q, float *scale) {
    constexpr int64_t kMost = int64_t(1) << 23, kSize = T == NT_F32 ? 4 : 2;
    for (int64_t r = 0; r < rows; r += kMost) {
        const int64_t n = std::min(kMost, rows - r);
        const uint8_t *from = x + r * ld * kSize;
        int8_t *to = q + r * cols;
        if (cols <= 4096 && rows >= 1024)
            k_quantize_rows<T, 64, 8><<<dim3(unsigned(ceil_div(n, 4))), dim3(256), 0, ctx().stream>>>(from, n, cols, ld, to, scale + r);
        else
            k_quantize_rows<T, 256, 8><<<dim3(unsigned(n)), dim3(256), 0, ctx().stream>>>(from, n, cols, ld, to, scale + r);
        if (int rc = launched("k_quantize_rows")) return rc;
    }
    return 0;
}

// Rows that are the columns of x [n, ld]. A workgroup takes W of them and `per` rows of x, a thread four neighbouring ones
// (16 bytes of f32, 8 of a 16-bit type) in four rows of x at a time: a word of each of its columns. Bounded by HBM and
// the last-level cache: x is read for the magnitudes and again for the values, which do not fit on the chip: 1024 x 50304
// f32 takes 73 us where that cache holds x, 89 cold (its bytes once, at a copy's rate: 54).
template <int T, int W>
struct Columns {
    const void *x;
    int64_t cols, n, ld, c;
    int have;

    __device__ __forceinline__ Columns(const void *x, int64_t cols, int64_t n, int64_t ld, int64_t c)
        : x(x), cols(cols), n(n), ld(ld), c(c), have(cols - c >= 4 ? 4 : (cols > c ? int(cols - c) : 0)) {}

    // rows k .. k + 3 of x
    __device__ __forceinline__ void load(int64_t k, float (&v)[4][4]) const {
#pragma unroll
        for (int u = 0; u < 4; u++) v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.0f;
        if (have == 4 && k + 4 <= n) {
            if constexpr (T == NT_F32) {
#pragma unroll
                for (int u = 0; u < 4; u++) __builtin_memcpy(v[u], static_cast<const float *>(x) + (k + u) * ld + c, 16);
            } else {
                uint16_t h[4][4];
#pragma unroll
                for (int u = 0; u < 4; u++) __builtin_memcpy(h[u], static_cast<const uint16_t *>(x) + (k + u) * ld + c, 8);
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (T == NT_BF16) v[u][e] = __builtin_bit_cast(float, uint32_t(h[u][e]) << 16);
                        else v[u][e] = float(__builtin_bit_cast(_Float16, h[u][e]));
                    }
            }
            return;
        }
        for (int u = 0; u < 4; u++)
            for (int e = 0; e < 4; e++)
                if (e < have && k + u < n) v[u][e] = load_f32<T>(x, (k + u) * ld + c + e);
    }

    // The largest magnitude of each column over rows r0 .. r1 - 1 as the bits of an f32, which order as their values do,
    // infinities and NaN at the end; the workgroup's, in s_top[0].
    __device__ __forceinline__ void top(int64_t r0, int64_t r1, uint32_t (&s_top)[32][W]) const {
        const int g = threadIdx.x / (W / 4), lc = threadIdx.x % (W / 4) * 4;
        uint32_t m[4] = {0, 0, 0, 0};
        for (int64_t k0 = r0; k0 < r1; k0 += 256) {
            float v[2][4][4];
            load(k0 + 4 * g, v[0]);
            load(k0 + 128 + 4 * g, v[1]);
#pragma unroll
            for (int w = 0; w < 2; w++)
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) m[e] = max(m[e], __builtin_bit_cast(uint32_t, v[w][u][e]) & 0x7fffffffu);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) s_top[g][lc + e] = m[e];
        __syncthreads();
        if (threadIdx.x < W) {
            uint32_t t = 0;
            for (int k = 0; k < 32; k++) t = max(t, s_top[k][threadIdx.x]);
            s_top[0][threadIdx.x] = t;
        }
    }
};

// The largest magnitudes of `per` rows (a multiple of 256), [parts, cols].
template <int T, int W>
__global__ __launch_bounds__(W * 8) void k_column_tops(const void *x, int64_t cols, int64_t n, int64_t ld, int64_t per,
                                                       uint32_t *tops) {
    __shared__ uint32_t s_top[32][W];
    const int64_t c0 = int64_t(blockIdx.x) * W, r0 = blockIdx.y * per;
    const Columns<T, W> at(x, cols, n, ld, c0 + threadIdx.x % (W / 4) * 4);
    at.top(r0, min(n, r0 + per), s_top);
    if (threadIdx.x < W && c0 + threadIdx.x < cols) tops[blockIdx.y * cols + c0 + threadIdx.x] = s_top[0][threadIdx.x];
}

// `tops` null: all of n, whose second reading comes from the caches where they hold it. The words go out through LDS, 128
// values of a column side by side.
template <int T, int W>
__global__ __launch_bounds__(W * 8) void k_quantize_columns(const void *x, int64_t cols, int64_t n, int64_t ld, int64_t per,
                                                            const uint32_t *tops, int parts, int8_t *q, float *scale) {
    __shared__ uint32_t s_top[32][W];
    __shared__ float s_scale[W];
    __shared__ uint32_t tile[W][33];  // [column][words of 4 rows of x]
    const int t = threadIdx.x, g = t / (W / 4), lc = (t % (W / 4)) * 4;
    const int64_t c0 = int64_t(blockIdx.x) * W, r0 = blockIdx.y * per, r1 = min(n, r0 + per);
    const Columns<T, W> at(x, cols, n, ld, c0 + lc);
    float v[4][4];
    if (tops) {
        at.load(r0 + 4 * g, v);
        uint32_t m = 0;
        const int64_t c = c0 + t % W;
        if (c < cols)
            for (int k = t / W; k < parts; k += 8) m = max(m, tops[k * cols + c]);
        s_top[t / W][t % W] = m;
        __syncthreads();
        if (t < W)
            for (int k = 1; k < 8; k++) m = max(m, s_top[k][t]);
        if (t < W) s_top[0][t] = m;
    } else {
        at.top(0, n, s_top);
        at.load(4 * g, v);
    }
    if (t < W) {
        const float top = __builtin_bit_cast(float, s_top[0][t]), s = scale_of(top, top < INFINITY);
        s_scale[t] = s;
        if (c0 + t < cols && blockIdx.y == 0) scale[c0 + t] = s;
    }
    __syncthreads();
    float s[4], inv[4];
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = s_scale[lc + e], inv[e] = 1.0f / s[e];
    for (int64_t k0 = r0; k0 < r1; k0 += 128) {  // 128 rows of x at a time, the next ones' loads ahead
        float next[4][4];
        at.load(k0 + 128 + 4 * g, next);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a[4] = {v[0][e], v[1][e], v[2][e], v[3][e]};
            tile[lc + e][g] = quantized4(a, s[e], inv[e]);
        }
        __syncthreads();
        // 8 threads a column, 16 bytes each
        const int col = t / 8, b = (t % 8) * 16;
        const int64_t left = n - k0 - b;
        if (c0 + col < cols && left > 0) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = tile[col][b / 4 + e];
            int8_t *o = q + (c0 + col) * n + k0 + b;
            if (left >= 16) __builtin_memcpy(o, w, 16);
            else
                for (int e = 0; e < 16; e++)
                    if (e < left) o[e] = int8_t(w[e / 4] >> (8 * (e % 4)));
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[u][e] = next[u][e];
    }
}

template <int T>
int launch_columns(const uint8_t *x, int64_t cols, int64_t n, int64_t ld, int8_t *q, float *scale) {
    constexpr int64_t kMost = int64_t(1) << 28, kSize = T == NT_F32 ? 4 : 2, W = 64;
    const int64_t blocks = ceil_div(cols, W);
    int64_t per = n, parts = 1;
    void *tops = nullptr;
    // Fewer workgroups than CUs: the rows of x in parts, two workgroups a CU, the magnitudes in a launch of their own (us,
    // f32, whole and in parts: 4096 x 12576 144 and 108, 4096 x 4096 60 and 39, 11008 x 92 236 and 16; but 1024 x 16384,
    // as many as there are CUs, 32 and 38).
    if (blocks < 256 && n > 256) {
        per = round_up(ceil_div(n, ceil_div(512, blocks)), 256);
        parts = ceil_div(n, per);
    }
    if (parts > 1) {
        if (int rc = scratch_alloc(size_t(parts * cols * 4), &tops)) return rc;
        k_column_tops<T, W><<<dim3(unsigned(blocks), unsigned(parts)), dim3(W * 8), 0, ctx().stream>>>(
            x, cols, n, ld, per, static_cast<uint32_t *>(tops));
        int rc = launched("k_column_tops");
        if (!rc) {
            k_quantize_columns<T, W><<<dim3(unsigned(blocks), unsigned(parts)), dim3(W * 8), 0, ctx().stream>>>(
                x, cols, n, ld, per, static_cast<uint32_t *>(tops), int(parts), q, scale);
            rc = launched("k_quantize_columns");
        }
        const int rf = scratch_release(tops);
        return rc ? rc : rf;
    }
    for (int64_t c = 0; c < cols; c += kMost) {
        const int64_t w = std::min(kMost, cols - c);
        k_quantize_columns<T, W><<<dim3(unsigned(ceil_div(w, W))), dim3(W * 8), 0, ctx().stream>>>(x + c * kSize, w, n, ld, n, nullptr, 0,
                                                                                                  q + c * n, scale + c);
        if (int rc = launched("k_quantize_columns")) return rc;
    }
    return 0;
}

// A thread takes eight neighbouring values at a time, of one row or, where rows are not whole chunks, of two or more.
template <int T>
__global__ __launch_bounds__(256) void k_dequantize(const int8_t *q, const float *scale, int64_t rows, int64_t cols, void *out) {
    const int64_t total = rows * cols, chunks = total / 8;
    const bool whole = cols % 8 == 0;
    auto value = [](int8_t b, float s) {
        float x = float(b) * s;
        asm("" : "+v"(x));  // (rounded to f32 first for every type: the f16 product is not made one instruction)
        return x;
    };
    auto put = [&](int64_t i, float x) {
        if constexpr (T == NT_F32) static_cast<float *>(out)[i] = x;
        else if constexpr (T == NT_BF16) static_cast<uint16_t *>(out)[i] = uint16_t(pair16<Bf16>(x, 0.0f));
        else static_cast<uint16_t *>(out)[i] = uint16_t(pair16<F16>(x, 0.0f));
    };
    for (int64_t c = blockIdx.x * int64_t(256) + threadIdx.x; c < chunks; c += int64_t(gridDim.x) * 256) {
        const int64_t i = c * 8;
        int8_t b[8];
        __builtin_memcpy(b, q + i, 8);
        // (a 32-bit quotient where it does: an index division of 64 bits costs more than the chunk)
        const int64_t r = total <= 0xffffffffu ? int64_t(uint32_t(i) / uint32_t(cols)) : i / cols;
        float x[8];
        if (whole) {
            const float s = scale[r];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = value(b[e], s);
        } else {
            int64_t row = r, left = cols - (i - r * cols);
            float s = scale[row];
            for (int e = 0; e < 8; e++) {
                if (left == 0) s = scale[++row], left = cols;
                x[e] = value(b[e], s);
                left--;
            }
        }
        if constexpr (T == NT_F32) {
            __builtin_memcpy(static_cast<float *>(out) + i, x, 32);
        } else {
            typedef typename std::conditional<T == NT_BF16, Bf16, F16>::type E;
            const uint32_t w[4] = {pair16<E>(x[0], x[1]), pair16<E>(x[2], x[3]), pair16<E>(x[4], x[5]), pair16<E>(x[6], x[7])};
            __builtin_memcpy(static_cast<uint16_t *>(out) + i, w, 16);
        }
    }
    if (blockIdx.x == 0 && chunks * 8 + threadIdx.x < total) {
        const int64_t i = chunks * 8 + threadIdx.x;
        put(i, value(q[i], scale[i / cols]));
    }
}

// Bytes of rows into rows of `ldo` (a multiple of 16) bytes, zeros from `cols` on.
__global__ __launch_bounds__(256) void k_pad_bytes(const uint8_t *src, int64_t rows, int64_t cols, int64_t ld, uint8_t *out,
                                                   int64_t ldo) {
    const int64_t per = ldo / 16, total = rows * per;
    for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i / per, c = (i - r * per) * 16;
        const uint8_t *s = src + r * ld + c;
        union {
            u32x4 v;
            uint8_t b[16];
        } x;
        if (c + 16 <= cols) x.v = *reinterpret_cast<const u32x4u *>(s);
        else
            for (int e = 0; e < 16; e++) x.b[e] = c + e < cols ? s[e] : uint8_t(0);
        *reinterpret_cast<u32x4 *>(out + r * ldo + c) = x.v;
    }
}

struct Int8P {
    const uint8_t *a, *b;
    int64_t lda, ldb, m, n, kb;
    uint32_t tm, tn;
    const float *sa, *sb;
    void *out;
    int64_t ldo;
    int64_t per;   // bytes of k of a split
    int32_t *slab; // [splits][m][n] integer sums, or null: the outputs themselves
};

constexpr int kSlab = -1;  // OUT: the integer sums of a split of k

template <class S, int OUT>
__global__ __launch_bounds__(S::kThreads, 1) void k_int8_tiles(Int8P p) {
    constexpr int TM = S::TM, TN = S::TN, WM = S::WM, WN = S::WN;
    typedef Tile<I8, TM, TN, WM, WN, false, false> T;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int im, in;
    tile_of(blockIdx.x, p.tm, p.tn, im, in);
    const int64_t m0 = int64_t(im) * T::BM, n0 = int64_t(in) * T::BN;
    const int64_t k0 = blockIdx.y * p.per, kb = p.kb - k0 < p.per ? p.kb - k0 : p.per;
    // One row of tiles: each from a stage of k of its own on (the sums are exact in any order). Weight rows a power of two
    // of bytes apart fall on the same HBM channels where every tile reads the same k at once: 64 x 50304 x 4096 59 -> 53 us.
    // With more rows of tiles those of a column share its panel, and stay together.
    const int first = p.tm == 1 && kb > 0 ? 2 * (in % int((kb + 127) / 128)) : 0;
    T t;
    t.run(lds, Operand{p.a + m0 * p.lda + k0, p.lda, p.m - m0, kb}, Operand{p.b + n0 * p.ldb + k0, p.ldb, p.n - n0, kb}, kb, wave,
          lane, first);
    const int wm = wave / WN, wn = wave % WN;
    constexpr bool kWide = OUT == NT_F32 || OUT == kSlab;
    typedef typename std::conditional<kWide, u32x4, u32x2>::type V;
    typedef typename std::conditional<OUT == NT_F16, F16, Bf16>::type E;
    constexpr int kSize = kWide ? 4 : 2;
    static_assert(store_bytes<TN>(kSize) * WM * WN <= T::kLds, "the blocks fit");
    const int64_t col0 = n0 + 32 * TN * wn;
    if constexpr (OUT == kSlab) {
        if (col0 >= p.n) return;
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int64_t row0 = m0 + 32 * (TM * wm + i);
            if (row0 >= p.m) break;
            V v[4 * TN];
#pragma unroll
            for (int q = 0; q < 4 * TN; q++) {
                const int x[4] = {t.acc[i][q / 4][4 * (q % 4)], t.acc[i][q / 4][4 * (q % 4) + 1], t.acc[i][q / 4][4 * (q % 4) + 2],
                                  t.acc[i][q / 4][4 * (q % 4) + 3]};
                v[q] = V{uint32_t(x[0]), uint32_t(x[1]), uint32_t(x[2]), uint32_t(x[3])};
            }
            store_block<TN>(lds + wave * store_bytes<TN>(4), v, lane,
                            reinterpret_cast<uint8_t *>(p.slab + (int64_t(blockIdx.y) * p.m + row0) * p.n + col0), p.n * 4,
                            p.m - row0 < 32 ? int(p.m - row0) : 32, p.n - col0 < 32 * TN ? int(p.n - col0) * 4 : 128 * TN);
        }
        return;
    } else {
    // (every scale before the first store, which the compiler takes to change them)
    float sb[4 * TN][4];
#pragma unroll
    for (int q = 0; q < 4 * TN; q++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int64_t col = col0 + 8 * q + 4 * (lane / 32) + e;
            sb[q][e] = p.sb[col < p.n ? col : p.n - 1];
        }
    float sa[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t row = m0 + 32 * (TM * wm + i) + lane % 32;
        sa[i] = p.sa[row < p.m ? row : p.m - 1];
    }
    if (col0 >= p.n) return;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t row0 = m0 + 32 * (TM * wm + i);
        if (row0 >= p.m) break;
        V v[4 * TN];
#pragma unroll
        for (int q = 0; q < 4 * TN; q++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = float(t.acc[i][q / 4][4 * (q % 4) + e]) * sa[i] * sb[q][e];
            if constexpr (OUT == NT_F32) v[q] = V{__builtin_bit_cast(uint32_t, x[0]), __builtin_bit_cast(uint32_t, x[1]),
                                                  __builtin_bit_cast(uint32_t, x[2]), __builtin_bit_cast(uint32_t, x[3])};
            else v[q] = V{pair16<E>(x[0], x[1]), pair16<E>(x[2], x[3])};
        }
        const int64_t rows = p.m - row0, bytes = (p.n - col0) * kSize;
        store_block<TN>(lds + wave * store_bytes<TN>(kSize), v, lane,
                        static_cast<uint8_t *>(p.out) + (row0 * p.ldo + col0) * kSize, p.ldo * kSize,
                        rows < 32 ? int(rows) : 32, bytes < 32 * TN * kSize ? int(bytes) : 32 * TN * kSize);
    }
    }
}

template <int T>
__device__ __forceinline__ void put(void *out, int64_t at, float x) {
    if constexpr (T == NT_F32) static_cast<float *>(out)[at] = x;
    else if constexpr (T == NT_BF16) static_cast<uint16_t *>(out)[at] = uint16_t(pair16<Bf16>(x, 0.0f));
    else static_cast<uint16_t *>(out)[at] = uint16_t(pair16<F16>(x, 0.0f));
}

// The splits' sums (integers: their order does not matter), scaled and rounded.
template <int OUT>
__global__ __launch_bounds__(256) void k_int8_fold(Int8P p, int splits) {
    const int64_t total = p.m * p.n;
    for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i / p.n, c = i - r * p.n;
        int sum = 0;
        int z = 0;
        for (; z + 8 <= splits; z += 8) {  // (eight loads in flight)
            int v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = p.slab[(z + k) * total + i];
#pragma unroll
            for (int k = 0; k < 8; k++) sum += v[k];
        }
        for (; z < splits; z++) sum += p.slab[z * total + i];
        put<OUT>(p.out, r * p.ldo + c, float(sum) * p.sa[r] * p.sb[c]);
    }
}

// Up to four rows of a: the weight's stream from HBM is all there is. A wave takes eight rows of b, a KiB of each at a time
// (a load's lanes side by side: whole lines), against the same KiB of a, by four-byte dot products in the vector
// units; the lanes' sums are exchanged at the end, so that each ends with one of 64 (eight rows by up to eight). A row of
// 128256 x 4096 weights: 131 us by tiles of 64 rows, 91 to 96 so. (Five to eight rows' dots take longer than the bytes.)
template <int M, int OUT>
__global__ __launch_bounds__(256) void k_int8_few(Int8P p) {
    constexpr int NR = 8;
    const int lane = threadIdx.x & 63;
    const int64_t n0 = (int64_t(blockIdx.x) * 4 + threadIdx.x / 64) * NR;
    if (n0 >= p.n) return;
    const uint8_t *row[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) row[r] = p.b + (n0 + r < p.n ? n0 + r : p.n - 1) * p.ldb;
    int acc[NR][M];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int i = 0; i < M; i++) acc[r][i] = 0;
    auto dots = [&](int64_t at, bool in) {
        u32x4 w[NR], a[M];
#pragma unroll
        for (int r = 0; r < NR; r++) w[r] = u32x4{0, 0, 0, 0};
        if (in) {
#pragma unroll
            for (int r = 0; r < NR; r++) w[r] = *reinterpret_cast<const u32x4 *>(row[r] + at);
        }
#pragma unroll
        for (int i = 0; i < M; i++) a[i] = in ? *reinterpret_cast<const u32x4 *>(p.a + i * p.lda + at) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int i = 0; i < M; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[r][i] = __builtin_amdgcn_sdot4(int(w[r][e]), int(a[i][e]), acc[r][i], false);
    };
    int64_t at = lane * 16;
    for (; at - lane * 16 + 1024 <= p.kb; at += 1024) dots(at, true);
    if (at - lane * 16 < p.kb) dots(at, at < p.kb);
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int i = 0; i < M; i++)
#pragma unroll
            for (int d = 32; d; d /= 2) acc[r][i] += __shfl_xor(acc[r][i], d, 64);
    const int r = lane % NR, i = lane / NR;
    if (i >= M || n0 + r >= p.n) return;
    int sum = 0;
#pragma unroll
    for (int rr = 0; rr < NR; rr++)
#pragma unroll
        for (int ii = 0; ii < M; ii++)
            if (rr == r && ii == i) sum = acc[rr][ii];
    const float x = float(sum) * p.sa[i] * p.sb[n0 + r];
    put<OUT>(p.out, i * p.ldo + n0 + r, x);
}

template <int M, int OUT>
int launch_few(const Int8P &p) {
    k_int8_few<M, OUT><<<dim3(unsigned(ceil_div(p.n, 32))), dim3(256), 0, ctx().stream>>>(p);
    return launched("k_int8_few");
}

template <class S, int OUT>
int launch_tiles(Int8P p, int64_t splits) {
    p.tm = uint32_t(ceil_div(p.m, S::kRows)), p.tn = uint32_t(ceil_div(p.n, S::kCols));
    k_int8_tiles<S, OUT><<<dim3(p.tm * p.tn, unsigned(splits)), dim3(S::kThreads), 0, ctx().stream>>>(p);
    return launched("k_int8_tiles");
}

template <int OUT>
int by_size(const Int8P &p, const Plan &s) {
    switch (s.size) {
        case Size::kSmall: return launch_tiles<Small, OUT>(p, s.splits);
        case Size::kMedium: return launch_tiles<Medium, OUT>(p, s.splits);
        default: return launch_tiles<Large, OUT>(p, s.splits);
    }
}

// Up to four rows row by row, else by tiles (`s`); a split k's sums through slabs.
template <int OUT>
int tiles(const Int8P &p, const Plan &s) {
    switch (p.m) {
        case 1: return launch_few<1, OUT>(p);
        case 2: return launch_few<2, OUT>(p);
        case 3: return launch_few<3, OUT>(p);
        case 4: return launch_few<4, OUT>(p);
        default: break;
    }
    if (!p.slab) return by_size<OUT>(p, s);
    if (int rc = by_size<kSlab>(p, s)) return rc;
    k_int8_fold<OUT><<<dim3(unsigned(std::min<int64_t>(ceil_div(p.m * p.n, 256), 8192))), dim3(256), 0, ctx().stream>>>(
        p, int(s.splits));
    return launched("k_int8_fold");
}

int pad_rows(const int8_t *src, int64_t rows, int64_t cols, int64_t ld, uint8_t *out, int64_t ldo) {
    const int64_t n = rows * (ldo / 16);
    hipLaunchKernelGGL(k_pad_bytes, dim3(unsigned(std::min<int64_t>(ceil_div(n, 256), 8192))), dim3(256), 0, ctx().stream,
                       reinterpret_cast<const uint8_t *>(src), rows, cols, ld, out, ldo);
    return launched("k_pad_bytes");
}

bool aligned(const void *p, int64_t cols, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 16 == 0 && cols % 16 == 0;
}

// Scratch of 1 MiB and more is refused under stream capture, as the training readout's is (rl_readout_train.hip).
int fits_capture(const char *who, int64_t need) {
    bool cap = false;
    if (need < (int64_t(1) << 20)) return 0;
    if (int rc = stream_capturing(&cap)) return rc;
    return cap ? fail(NT_E_UNSUPPORTED, std::string(who) + ": " + std::to_string(need) + " bytes of scratch under stream capture (under 1 MiB)")
               : 0;
}

constexpr int64_t kMaxK = 131071, kMaxLd = int64_t(1) << 22;

int product(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb, int64_t m, int64_t n,
            int64_t k, int32_t dtype, void *out, int64_t ldo) {
    const bool ad = k == 0 || aligned(a, k, lda), bd = k == 0 || aligned(b, k, ldb);  // (no k: nothing is read)
    const int64_t kp = round_up(k, 16);
    const Plan s = plan(m, n, kp, true);
    const int64_t abytes = ad ? 0 : round_up(m * kp, 256), bbytes = bd ? 0 : round_up(n * kp, 256);
    const bool slabs = m > 4 && s.splits > 1;
    const int64_t need = abytes + bbytes + (slabs ? s.splits * m * n * 4 : 0);
    void *ws = nullptr;
    if (int rc = fits_capture("matmul_int8", need)) return rc;
    if (need > 0)
        if (int rc = scratch_alloc(size_t(need), &ws)) return rc;
    uint8_t *pa = static_cast<uint8_t *>(ws), *pb = pa + abytes;
    Int8P p{reinterpret_cast<const uint8_t *>(a), reinterpret_cast<const uint8_t *>(b), lda, ldb, m, n, kp, 0, 0, sa, sb, out,
            ldo, s.per, slabs ? reinterpret_cast<int32_t *>(pb + bbytes) : nullptr};
    int rc = 0;
    if (!ad) {
        rc = pad_rows(a, m, k, lda, pa, kp);
        p.a = pa, p.lda = kp;
    }
    if (!rc && !bd) {
        rc = pad_rows(b, n, k, ldb, pb, kp);
        p.b = pb, p.ldb = kp;
    }
    if (!rc) {
        rc = dtype == NT_F32 ? tiles<NT_F32>(p, s) : dtype == NT_BF16 ? tiles<NT_BF16>(p, s) : tiles<NT_F16>(p, s);
    }
    const int rf = scratch_release(ws);
    return rc ? rc : rf;
}

bool float_type(int32_t t) { return t == NT_F32 || t == NT_BF16 || t == NT_F16; }
int size_of(int32_t t) { return t == NT_F32 ? 4 : 2; }

// A view as rows of its last dimension: {rows, columns, strides of both}, if its leading dimensions fold into
// one stride.
struct Rows {
    int64_t rows, cols, row_stride, col_stride;
};
bool as_rows(const NtLayout *l, Rows *o) {
    const int r = l->rank;
    o->rows = 1, o->cols = l->shape[r - 1], o->col_stride = l->strides[r - 1], o->row_stride = 0;
    for (int d = r - 2; d >= 0; d--) {
        if (l->shape[d] == 1) continue;
        if (o->rows == 1) o->row_stride = l->strides[d];
        else if (l->strides[d] != o->row_stride * o->rows) return false;
        o->rows *= l->shape[d];
    }
    return true;
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int nt_hip_quantize_int8(const void *x, const NtLayout *xl, int32_t dtype, int8_t *q, float *scale) {
    const char *who = "quantize_int8";
    if (!xl || xl->rank < 1 || xl->rank > NT_MAX_RANK) return fail(NT_E_ARG, std::string(who) + ": a view of rank 1 to 8");
    if (!float_type(dtype)) return fail(NT_E_ARG, std::string(who) + ": dtype " + std::to_string(dtype) + " (f32, bf16 or f16)");
    int64_t total = 1;
    for (int d = 0; d < xl->rank; d++) {
        if (xl->shape[d] < 0 || xl->strides[d] < 0 || xl->offset < 0)
            return fail(NT_E_ARG, std::string(who) + ": negative shape, stride or offset");
        if (__builtin_mul_overflow(total, xl->shape[d], &total) || total > (int64_t(1) << 40))
            return fail(NT_E_ARG, std::string(who) + ": more than 2^40 values");
    }
    int64_t rows = 1;  // (of no columns there may be any number: as many scales)
    for (int d = 0; d + 1 < xl->rank; d++)
        if (__builtin_mul_overflow(rows, xl->shape[d], &rows) || rows > (int64_t(1) << 40))
            return fail(NT_E_ARG, std::string(who) + ": more than 2^40 rows");
    const int64_t cols = xl->shape[xl->rank - 1];
    if (rows > 0 && (!scale || (total > 0 && (!x || !q))))
        return fail(NT_E_ARG, std::string(who) + ": null buffer");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    if (rows == 0) return 0;
    Rows v;
    void *ws = nullptr;
    const uint8_t *src = static_cast<const uint8_t *>(x) + xl->offset * size_of(dtype);
    const bool folds = as_rows(xl, &v);
    const bool columns = folds && v.rows > 1 && v.cols > 1 && v.row_stride == 1 && v.col_stride != 1;
    if (!columns && !(folds && (v.col_stride == 1 || v.cols == 1))) {  // any other view: its values in order first
        if (int rc = fits_capture(who, total * size_of(dtype))) return rc;
        if (int rc = scratch_alloc(size_t(total) * size_of(dtype), &ws)) return rc;
        lk.unlock();
        int rc = nt_hip_copy(x, xl, size_of(dtype), ws);
        if (int re = enter(&lk)) return rc ? rc : re;
        if (rc) {
            (void)scratch_release(ws);
            return rc;
        }
        src = static_cast<const uint8_t *>(ws);
        v = Rows{rows, cols, cols, 1};
    }
    auto launch = [&](auto type) {
        constexpr int T = decltype(type)::value;
        return columns ? launch_columns<T>(src, v.rows, v.cols, v.col_stride, q, scale)
                       : launch_rows<T>(src, v.rows, v.cols, v.row_stride, q, scale);
    };
    const int rc = dtype == NT_F32 ? launch(std::integral_constant<int, NT_F32>{})
                   : dtype == NT_BF16 ? launch(std::integral_constant<int, NT_BF16>{})
                                      : launch(std::integral_constant<int, NT_F16>{});
    const int rf = scratch_release(ws);
    return rc ? rc : rf;
}

int nt_hip_dequantize_int8(const int8_t *q, const float *scale, int64_t rows, int64_t cols, int32_t dtype, void *out) {
    const char *who = "dequantize_int8";
    if (!float_type(dtype)) return fail(NT_E_ARG, std::string(who) + ": dtype " + std::to_string(dtype) + " (f32, bf16 or f16)");
    if (rows < 0 || cols < 0 || (cols > 0 && rows > (int64_t(1) << 40) / cols))
        return fail(NT_E_ARG, std::string(who) + ": " + std::to_string(rows) + " rows of " + std::to_string(cols));
    if (rows * cols > 0 && (!q || !scale || !out)) return fail(NT_E_ARG, std::string(who) + ": null buffer");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    if (rows * cols == 0) return 0;
    const dim3 grid(unsigned(std::min<int64_t>(ceil_div(rows * cols, 2048), 16384)));
    if (dtype == NT_F32) hipLaunchKernelGGL(k_dequantize<NT_F32>, grid, dim3(256), 0, ctx().stream, q, scale, rows, cols, out);
    else if (dtype == NT_BF16) hipLaunchKernelGGL(k_dequantize<NT_BF16>, grid, dim3(256), 0, ctx().stream, q, scale, rows, cols, out);
    else hipLaunchKernelGGL(k_dequantize<NT_F16>, grid, dim3(256), 0, ctx().stream, q, scale, rows, cols, out);
    return launched("k_dequantize");
}

int nt_hip_matmul_int8(const int8_t *a, int64_t lda, const float *a_scale, const int8_t *b, int64_t ldb, const float *b_scale,
                       int64_t m, int64_t n, int64_t k, int32_t dtype, void *out, int64_t ldo) {
    const char *who = "matmul_int8";
    if (!float_type(dtype)) return fail(NT_E_ARG, std::string(who) + ": dtype " + std::to_string(dtype) + " (f32, bf16 or f16)");
    if (m < 0 || n < 0 || k < 0 || m > (1 << 24) || n > (1 << 24) || k > kMaxK || lda < k || ldb < k || ldo < n || lda > kMaxLd ||
        ldb > kMaxLd || ceil_div(m, 256) * ceil_div(n, 256) >= (1 << 23))
        return fail(NT_E_ARG, std::string(who) + ": [" + std::to_string(m) + ", " + std::to_string(k) + "] x [" + std::to_string(n) +
                                  ", " + std::to_string(k) + "], row strides " + std::to_string(lda) + ", " +
                                  std::to_string(ldb) + ", " + std::to_string(ldo) +
                                  " (m and n at most 2^24 and 2^39 outputs, k at most 131071, strides at least the row, "
                                  "the operands' at most 2^22)");
    if (m > 0 && n > 0 && (!a_scale || !b_scale || !out || (k > 0 && (!a || !b))))
        return fail(NT_E_ARG, std::string(who) + ": null buffer");
    if (reinterpret_cast<uintptr_t>(out) % size_of(dtype)) return fail(NT_E_ARG, std::string(who) + ": unaligned out");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    if (m == 0 || n == 0) return 0;
    return product(a, lda, a_scale, b, ldb, b_scale, m, n, k, dtype, out, ldo);
}

}  // extern "C"
