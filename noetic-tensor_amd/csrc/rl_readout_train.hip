// The training readout: token log-probabilities, entropies and log-sum-exps of logits x = H W from the
// hidden states, and their gradients with respect to H and W, the logits never kept.
//
// The reference multiplies (the decoder's head, src/nn/decoder.rs:272,286; linear.rs:1-3), keeps [rows, V]
// logits, and differentiates log_softmax, gather and categorical_entropy on them (activation.rs:30-42,
// rl.rs:134-141, 405-414). Here, with z = x / T + mask:
//
//  Forward: k_readout_stats computes a tile of x on the matrix cores (nt_tile.hpp) and reduces it where it
//  stands: per row and block of columns the reference, the largest value (x, or z in f32 where an additive mask makes
//  it), and the sums of w = 2^d and, for the entropy, w d over the differences d from it in units of ln 2 (f32: at
//  most 128 terms). Differences first, products after: logits of any size, or a bias of -1e9 in every column, lose no
//  more than their own f32 rounding. k_readout_merge joins a row's blocks in f64:
//    lse = ln sum e^z, logp = z[token] - lse, entropy = lse - sum p z.
//
//  Backward: p = e^(z - base - rest), of the forward's two parts of the log-sum-exp, the difference from the base taken
//  first, comes from the logits computed once more, piece by piece of the vocabulary, so that
//    G = dL/dx = (g_logp (onehot - p) - g_entropy p (ln p + entropy)) / T
//  is held for one piece at a time, in the operands' 16-bit type: three products per piece, x = H W,
//  dW = G^T H (the piece's rows of it, whole) and dH += G W^T (f32 sums over the pieces). 8 rows V dim
//  operations with the forward's, against 6 where the logits are kept: the least there is without them.
//
//  Rounding: G is rounded on the way (2^-9 of itself for bf16, 2^-12 for f16, as the gradients are when they are
//  written), and for f16 the rows of H below; every sum is f32. A row's entry at its token is most of G, and its rounding
//  would show in the gradients as their own does, so what it left goes into them, times the row of H into dW as a stage
//  more of its product (LeftRows) and times the token's row of W into dH as its sums are folded: the error is the written
//  values' own, 0.0017 of the norm for bf16, where it was 0.0023 (2048 x 4096 x 50304 +1%, 4096 x 4096 x
//  128256 +0.8%). A DV weight's columns are read for it up to 512 rows; more rows of dH are scaled for it (kColumnRows).
//  For f16, whose range G would leave, a row of G is held in units of 2^(e - 14), 2^e over |g_logp| + 16 |g_entropy|
//  (p |ln p + entropy| is under 14 for a vocabulary of 2^20), and for dW the row of H is scaled by 2^e and the one power
//  of two that puts the largest value of all scaled rows under 2^15: what rows far below the largest lose to f16's
//  smallest steps is 2^-40 of that value, less than the smallest step of a gradient that holds the largest row's.
//
//  Bound by the matrix cores for many rows, and those by power: 4096 x 4096 x 128256 bf16 is scored in 3.3 ms (1.3
//  PFLOP/s at a clock near 1.5 GHz; a library product alone 2.99) and scored and differentiated in 13.5 to 13.8 ms (1.25
//  to 1.27 at its 8 R V dim). Few rows are bound by the weight's bytes and the launches: 64 x 1024 x 32000 scored in 27 us
//  (of 14 at a copy's rate), 128 rows differentiated with it in 113 (28).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "../../include/noetic_hip.h"
#include "nt_internal.hpp"
#include "nt_plan.hpp"
#include "nt_tile.hpp"

namespace nt {
namespace {

using namespace tile;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLog2eD = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

typedef u32x4 u32x4u __attribute__((aligned(1)));
typedef f32x16 f32x16_t;

// The mask of a readout call: none, a u8 keep-mask or an additive f32 one, a row per logits row (ld > 0) or
// one for all (ld 0), from the piece's first column on.
struct MaskP {
    const uint8_t *u8;
    const float *f32;
    int64_t ld;
};

// A wave's block of the mask, 32 rows by 32 TN columns, through LDS: whole 16-byte pieces of its rows in (a lane's
// own four columns of 32 rows would be 16 scattered loads), a lane's four columns of its row out. Columns past the
// vocabulary's `n`, whose logits are 0 (nt_tile.hpp), count as excluded.
template <int TN>
struct MaskBlock {
    static constexpr int kU8 = 32 * TN + 16, kF32 = 128 * TN + 16;  // bytes of a row in LDS
    static constexpr int kLds = 32 * kF32, kShared = 128 * TN;  // (of 32 rows, and of one that all share)
    // Rows row0 .. row0 + rows - 1 of the mask (a row that all share, ld 0, once, before the first block).
    static __device__ __forceinline__ void in(uint8_t *lds, const MaskP &m, int64_t row0, int rows, int col, int n, int lane,
                                              bool first) {
        if (m.ld == 0) {
            if (!first || lane >= 8 * TN) return;
            const int c = lane * 4;
            if (m.u8) {
                uint32_t k = 0;
                for (int e = 0; e < 4; e++)
                    if (col + c + e < n) k |= uint32_t(m.u8[col + c + e]) << (8 * e);
                *reinterpret_cast<uint32_t *>(lds + c) = k;
            } else {
                float f[4];
                for (int e = 0; e < 4; e++) f[e] = col + c + e < n ? m.f32[col + c + e] : -INFINITY;
                __builtin_memcpy(lds + c * 4, f, 16);
            }
            return;
        }
        if (m.u8) {
            constexpr int kPer = 2 * TN, kRows = 64 / kPer, kLoads = 32 / kRows;
            const int c = (lane % kPer) * 16, left = n - col - c;
            u32x4 v[kLoads];
#pragma unroll
            for (int g = 0; g < kLoads; g++) {
                const int r = g * kRows + lane / kPer;
                const uint8_t *s = m.u8 + (row0 + (r < rows ? r : rows - 1)) * m.ld + col + c;
                v[g] = u32x4{0, 0, 0, 0};
                if (left >= 16) v[g] = *reinterpret_cast<const u32x4u *>(s);
                else
                    for (int e = 0; e < left; e++) v[g][e / 4] |= uint32_t(s[e]) << (8 * (e % 4));
            }
#pragma unroll
            for (int g = 0; g < kLoads; g++)
                *reinterpret_cast<u32x4 *>(lds + (g * kRows + lane / kPer) * kU8 + c) = v[g];
        } else {
            constexpr int kPer = 8 * TN, kRows = 64 / kPer, kLoads = 32 / kRows, kBatch = 8;
            const int c = (lane % kPer) * 4, left = n - col - c;
#pragma unroll
            for (int b = 0; b < kLoads; b += kBatch) {
                float v[kBatch][4];
#pragma unroll
                for (int g = 0; g < kBatch; g++) {
                    const int r = (b + g) * kRows + lane / kPer;
                    const float *s = m.f32 + (row0 + (r < rows ? r : rows - 1)) * m.ld + col + c;
                    if (left >= 4) __builtin_memcpy(v[g], s, 16);
                    else
                        for (int e = 0; e < 4; e++) v[g][e] = e < left ? s[e] : -INFINITY;
                }
#pragma unroll
                for (int g = 0; g < kBatch; g++) __builtin_memcpy(lds + ((b + g) * kRows + lane / kPer) * kF32 + c * 4, v[g], 16);
            }
        }
    }
    // x's values under it: -inf where a keep-mask excludes; z = x / T + mask in f32 under an additive one (`invt`: 1 / T)
    static __device__ __forceinline__ void out(const uint8_t *lds, const MaskP &m, float invt, int lane, float (&x)[4 * TN][4]) {
        const int r = m.ld == 0 ? 0 : lane % 32, h = lane / 32;
        if (m.u8) {
#pragma unroll
            for (int q = 0; q < 4 * TN; q++) {
                const uint32_t k = *reinterpret_cast<const uint32_t *>(lds + r * kU8 + 8 * q + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; e++) x[q][e] = (k >> (8 * e)) & 0xffu ? x[q][e] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4 * TN; q++) {
                float f[4];
                __builtin_memcpy(f, lds + r * kF32 + 32 * q + 16 * h, 16);
#pragma unroll
                for (int e = 0; e < 4; e++) x[q][e] = x[q][e] * invt + f[e];
            }
        }
    }
};

// Without a mask: the columns past the vocabulary's end, `left` columns from this lane's first.
template <int Q>
__device__ __forceinline__ void ended(float (&x)[Q][4], int left) {
#pragma unroll
    for (int q = 0; q < Q; q++) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[q][e] = 8 * q + e < left ? x[q][e] : -INFINITY;
        __builtin_amdgcn_sched_barrier(0);  // (or every comparison is made at once, into more registers than there are)
    }
}

// A piece of the vocabulary: x[r, v] = sum_k H(r, k) W(v, k) for `n` columns from v0 on.
struct PieceP {
    const uint8_t *h;  // k-contiguous [rows, ldh bytes]
    const uint8_t *w;  // the piece's rows [n, ldw bytes] (VD) or columns of [dim, ldw bytes] (DV)
    int64_t ldh, ldw, wwidth;  // wwidth: bytes of a row of the piece (a multiple of 16)
    int64_t rows, kbytes, dim;
    int n;
    int64_t v0;
    uint32_t tm, tn;
    float c, invt;     // log2(e) / T (under an additive mask log2(e)), 1 / T
    MaskP mask;
    const int32_t *tokens;
    // forward
    float *ref, *sum, *esum;  // [block][rows_p]: the largest value, the sums relative to it
    int64_t rows_p, block0;   // rows padded for those, the piece's first block
    float *xtok;              // [rows] the token's raw logit
    // backward
    const float4 *coef;       // [rows] {the largest value (+inf: nothing flows), a, b, the token's term}
    uint8_t *g;               // [rows, ldg bytes], of which gbytes are written: zeros past n
    int64_t ldg, gbytes;
    float *left;              // [rows] what the rounding of G's entry at the row's token left (first: see CoefP)
    float *turn;              // [rows] what makes up for it in the row of dH (1: nothing), or null
};

template <class T, bool BTR>
__device__ __forceinline__ Operand weight_rows(const PieceP &p, int in) {
    const int64_t n0 = int64_t(in) * T::BN;
    if constexpr (BTR) return Operand{p.w + n0 * 2, p.ldw, p.dim, p.wwidth - n0 * 2};
    else return Operand{p.w + n0 * p.ldw, p.ldw, p.n - n0, p.kbytes};
}

template <class E, class S, bool BTR, bool ENT, bool MASK>
__global__ __launch_bounds__(S::kThreads, 1) void k_readout_stats(PieceP p) {
    constexpr int TM = S::TM, TN = S::TN, WM = S::WM, WN = S::WN;
    typedef Tile<E, TM, TN, WM, WN, false, BTR> T;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int im, in;
    tile_of(blockIdx.x, p.tm, p.tn, im, in);
    T t;
    t.run(lds, Operand{p.h + int64_t(im) * T::BM * p.ldh, p.ldh, p.rows - int64_t(im) * T::BM, p.kbytes},
          weight_rows<T, BTR>(p, in), p.kbytes, wave, lane);
    const int wm = wave / WN, wn = wave % WN;
    const int col0 = in * T::BN + 32 * TN * wn + 4 * (lane / 32);
    static_assert(MaskBlock<TN>::kLds * WM * WN <= T::kLds, "the mask's blocks fit");
    uint8_t *const mlds = lds + wave * MaskBlock<TN>::kLds;
    const int64_t block = p.block0 + int64_t(in) * WN + wn;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t row = int64_t(im) * T::BM + 32 * (TM * wm + i) + lane % 32;
        const bool live = row < p.rows;
        const int64_t r = live ? row : 0;
        // the token's logit, if it is one of this lane's columns (of 32 rows few have it among the wave's)
        const int64_t tok = p.tokens[r] - p.v0 - col0;
        const bool mine = live && tok >= 0 && tok < 32 * TN && (tok & 4) == 0 && tok + col0 < p.n;
        if (__any(mine)) {
            float xt = 0.0f;
#pragma unroll
            for (int q = 0; q < 4 * TN; q++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (tok == 8 * q + e) xt = t.acc[i][q / 4][4 * (q % 4) + e];
            if (mine) p.xtok[row] = xt;
        }
        float x[4 * TN][4];
#pragma unroll
        for (int q = 0; q < 4 * TN; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[q][e] = t.acc[i][q / 4][4 * (q % 4) + e];
        if constexpr (MASK) {
            const int64_t row0 = row - lane % 32;
            if (row0 < p.rows)
                MaskBlock<TN>::in(mlds, p.mask, row0, p.rows - row0 < 32 ? int(p.rows - row0) : 32, in * T::BN + 32 * TN * wn, p.n, lane, i == 0);
            wave_exchange();
            MaskBlock<TN>::out(mlds, p.mask, p.invt, lane, x);
            wave_exchange();
        } else if (in * T::BN + T::BN > p.n) {
            ended(x, p.n - col0);
        }
        float m = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4 * TN; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) m = fmaxf(m, x[q][e]);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float ref = m == -INFINITY ? 0.0f : m;
        float s = 0.0f, es = 0.0f;
#pragma unroll
        for (int q = 0; q < 4 * TN; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = (x[q][e] - ref) * p.c, w = __builtin_amdgcn_exp2f(d);
                s += w;
                if constexpr (ENT) es += w > 0.0f ? w * d : 0.0f;
            }
        s += __shfl_xor(s, 32, 64);
        if constexpr (ENT) es += __shfl_xor(es, 32, 64);
        if (live && lane < 32) {
            p.ref[block * p.rows_p + row] = m;
            p.sum[block * p.rows_p + row] = s;
            if constexpr (ENT) p.esum[block * p.rows_p + row] = es;
        }
    }
}

struct MergeP {
    const float *ref, *sum, *esum;
    int64_t rows, rows_p;
    int blocks;
    int64_t vocab;
    const float *xtok;
    const int32_t *tokens;
    MaskP mask;
    double tau;
    float c, invt;
    float *logp, *entropy, *base, *rest;
    uint8_t *status;
};

// A workgroup joins the blocks of 32 rows, 32 threads a row, in f64 and in the same order always: a thread its
// blocks by eights (loads in flight together), each eight against its own maximum.
__global__ __launch_bounds__(1024) void k_readout_merge(MergeP p) {
    constexpr int kSegs = 32, kBatch = 8;
    __shared__ float sm[kSegs][32];
    __shared__ double ss[kSegs][32], st[kSegs][32];
    const int lr = threadIdx.x % 32, seg = threadIdx.x / 32;
    const int64_t row = int64_t(blockIdx.x) * 32 + lr;
    const bool live = row < p.rows;
    float m = -INFINITY;  // the maximum so far, s and t in its units
    double s = 0.0, t = 0.0;
    for (int b0 = seg; b0 < p.blocks; b0 += kBatch * kSegs) {
        float r[kBatch], q[kBatch], e[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            const int b = b0 + k * kSegs;
            const bool in = b < p.blocks && live;
            r[k] = in ? p.ref[b * p.rows_p + row] : -INFINITY;
            q[k] = in ? p.sum[b * p.rows_p + row] : 0.0f;
            e[k] = in && p.esum ? p.esum[b * p.rows_p + row] : 0.0f;
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kBatch; k++) top = fmaxf(top, r[k]);
        const float base = top == -INFINITY ? 0.0f : top;
        if (m > -INFINITY) {
            const float d = (m - base) * p.c;
            const double f = double(__builtin_amdgcn_exp2f(d));
            t = f * (t + double(d) * s);
            s *= f;
        }
        m = top;
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            // (a block with nothing allowed has ref -inf and sum 0; with NaNs alone, sum NaN)
            if (r[k] == -INFINITY && q[k] == 0.0f) continue;
            const float d = (r[k] - base) * p.c;
            const double f = r[k] == -INFINITY ? 1.0 : double(__builtin_amdgcn_exp2f(d));
            s += f * double(q[k]);
            t += f * (double(e[k]) + double(d) * double(q[k]));
        }
    }
    sm[seg][lr] = m;
    ss[seg][lr] = s;
    st[seg][lr] = t;
    __syncthreads();
    if (seg != 0 || !live) return;
    for (int k = 0; k < kSegs; k++) m = fmaxf(m, sm[k][lr]);
    s = t = 0.0;
    for (int k = 0; k < kSegs; k++) {
        const double q = ss[k][lr];
        if (sm[k][lr] == -INFINITY) {
            s += q;  // 0, or NaN
            continue;
        }
        const float d = (sm[k][lr] - m) * p.c;
        const double f = double(__builtin_amdgcn_exp2f(d));
        s += f * q;
        t += f * (st[k][lr] + double(d) * q);
    }
    const int64_t tok = p.tokens[row];
    const bool bad = tok < 0 || tok >= p.vocab;
    // The largest z and, relative to it, the log of the sum: apart, since under a large bias in every column (a mask of
    // the type's lowest value) the sum's last bits are not the logits'.
    const double zmax = p.mask.f32 ? double(m) : double(m) / p.tau, lns = kLn2 * log2(s);
    const float base = float(zmax);
    const bool none = base == -INFINITY && s == s;  // (or every value below what z holds)
    const bool ok = !none && s > 0.0 && s < INFINITY && base < INFINITY;
    uint8_t status = ok ? NT_ROW_OK : (none ? NT_ROW_NO_TOKEN : NT_ROW_NAN);
    if (p.base) p.base[row] = ok ? base : (none ? -INFINITY : NAN);
    if (p.rest) p.rest[row] = ok ? float((zmax - double(base)) + lns) : (none ? 0.0f : NAN);
    if (p.entropy) p.entropy[row] = ok ? float(lns - kLn2 * t / s) : NAN;
    float lp = NAN;
    if (ok && !bad) {
        double z = double(p.xtok[row]) / p.tau;
        if (p.mask.u8 && !p.mask.u8[row * p.mask.ld + tok]) z = -INFINITY;
        else if (p.mask.f32) z = double(p.xtok[row] * p.invt + p.mask.f32[row * p.mask.ld + tok]);  // (as its column's value)
        lp = float((z - zmax) - lns);
    }
    p.logp[row] = lp;
    if (ok && bad) status = NT_ROW_BAD_TOKEN;
    p.status[row] = status;
}

// ---------------------------------------------------------------------------------- backward

struct CoefP {
    const float *base, *rest, *entropy, *g_logp, *g_entropy;
    const int32_t *tokens;
    int64_t rows, vocab;
    double tau;
    int f32mask, f16;
    float4 *coef;
    float *left;   // [rows] 0 where nothing flows; else 8 |g_entropy| in G's units until G is there
    float *turn;   // [rows] ones here, or null
    unsigned coefs;  // workgroups; those behind them list the tokens
    int2 *place;   // [vocab / 256] a bucket's first entry in `listed`, and how many
    uint32_t *listed;  // [rows] row << 8 | token % 256
    float *up;     // [rows] f16: 2^e, what a row of G was divided by (0: nothing flows)
    int *top;      // [1] f16: cleared here, for k_readout_top
};

constexpr int kNoTop = -(1 << 30);

// The rows whose token is in 256 columns of the vocabulary, `bucket`, in their order, but for those that nothing flows
// through (a batch's padding may hold one token many times): a workgroup goes through all the tokens, a wave through
// consecutive ones, once to count them and those of the buckets in front, whose places they may not fill, once to
// write them.
constexpr int kBucket = 256;
__device__ __forceinline__ bool nothing_flows(double gl, double ge, float base) { return (gl == 0.0 && ge == 0.0) || base == -INFINITY; }
__device__ __forceinline__ void list_tokens(const CoefP &p, int bucket) {
    __shared__ int s_hits[16], s_less[16];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t per = ((p.rows + 15) / 16 + 63) / 64 * 64, first = wave * per < p.rows ? wave * per : p.rows;
    const int64_t last = first + per < p.rows ? first + per : p.rows;
    const uint32_t from = uint32_t(bucket) * kBucket;
    auto token = [&](int64_t r) { return r < last ? uint32_t(p.tokens[r]) : ~0u; };
    auto listed = [&](int64_t r, uint32_t t) {
        return t < p.vocab && t - from < uint32_t(kBucket) &&
               !nothing_flows(p.g_logp ? p.g_logp[r] : 0.0, p.g_entropy ? p.g_entropy[r] : 0.0, p.base[r]);
    };
    int hits = 0, less = 0;
    for (int64_t r = first + lane; r - lane < last; r += 512) {
        uint32_t t[8];
#pragma unroll
        for (int u = 0; u < 8; u++) t[u] = token(r + 64 * u);  // (eight loads in flight)
#pragma unroll
        for (int u = 0; u < 8; u++) {
            hits += __popcll(__ballot(listed(r + 64 * u, t[u])));
            less += __popcll(__ballot(t[u] < from));
        }
    }
    if (lane == 0) s_hits[wave] = hits, s_less[wave] = less;
    __syncthreads();
    int start = 0, all = 0, at = 0;
    for (int w = 0; w < 16; w++) {
        start += s_less[w];
        if (w == wave) at = all;
        all += s_hits[w];
    }
    if (threadIdx.x == 0) p.place[bucket] = int2{start, all};
    if (hits == 0) return;
    at += start;
    for (int64_t r = first + lane; r - lane < last; r += 64) {
        const uint32_t t = token(r);
        const bool hit = listed(r, t);
        const uint64_t m = __ballot(hit);
        if (hit) p.listed[at + __popcll(m & ((uint64_t(1) << lane) - 1))] = uint32_t(r) << 8 | (t - from);
        at += __popcll(m);
    }
}

// What a row's upstream gradients make of it: with l = (value - largest) c, so that p = 2^l q, q = e^-rest, and ln p =
// l ln 2 - rest, G = 2^l (a + b l) + the token's term.
__global__ __launch_bounds__(1024) void k_readout_coef(CoefP p) {
    if (blockIdx.x >= p.coefs) return list_tokens(p, int(blockIdx.x - p.coefs));
    if (p.f16 && blockIdx.x == 0 && threadIdx.x == 0) *p.top = kNoTop;
    for (int64_t r = blockIdx.x * int64_t(1024) + threadIdx.x; r < p.rows; r += int64_t(p.coefs) * 1024) {
        const int64_t tok = p.tokens[r];
        double gl = p.g_logp ? double(p.g_logp[r]) : 0.0;
        if (tok < 0 || tok >= p.vocab) gl = 0.0;
        const double ge = p.g_entropy ? double(p.g_entropy[r]) : 0.0;
        const double h = p.g_entropy ? double(p.entropy[r]) : 0.0;
        // the largest value as the columns have it: z's (an additive mask), or x's, whose rounding goes to the rest
        const float base = p.base[r], top_x = p.f32mask ? base : float(double(base) * p.tau);
        const double rest = double(p.rest[r]) + (p.f32mask ? 0.0 : double(base) - double(top_x) / p.tau), q = exp(-rest);
        const bool dead = nothing_flows(gl, ge, base);
        double unit = 1.0;  // f16: G's unit, a power of two
        float up = 0.0f;
        if (p.f16 && !dead) {
            const double size = fabs(gl) + 16.0 * fabs(ge);
            int e = 0;
            if (size > 0.0 && size < INFINITY) {
                (void)frexp(size, &e);  // size < 2^e
                e = e < -126 ? -126 : (e > 126 ? 126 : e);
            }
            up = ldexpf(1.0f, e);
            unit = ldexp(1.0, 14 - e);
        } else if (!p.f16) {
            unit = 1.0 / p.tau;
        }
        if (p.f16) p.up[r] = up;
        const bool term = !dead && tok >= 0 && tok < p.vocab;
        p.left[r] = term ? float(8.0 * fabs(ge) * unit) : 0.0f;
        if (p.turn) p.turn[r] = 1.0f;
        const float a = float(-(gl + ge * (h - rest)) * q * unit), b = float(-ge * kLn2 * q * unit);
        p.coef[r] = dead ? float4{INFINITY, 0.0f, 0.0f, 0.0f} : float4{top_x, a, b, float(gl * unit)};
    }
}

// Of a normal power of two.
__device__ __forceinline__ int exponent(float p) { return int(__builtin_bit_cast(uint32_t, p) >> 23) - 127; }

// f16: the exponent that the largest |h| 2^e of all rows is under, a wave a row. (A maximum of integers: the same in any
// order. Infinities and NaNs do not count.)
__global__ __launch_bounds__(256) void k_readout_top(const uint16_t *h, int64_t rows, int64_t cols, int64_t ld, const float *up,
                                                     int *top) {
    const int lane = threadIdx.x % 64;
    const int64_t row = blockIdx.x * int64_t(4) + threadIdx.x / 64;
    if (row >= rows || up[row] == 0.0f) return;
    uint32_t most = 0;  // (magnitudes order as their bits do)
    auto see = [&](uint32_t b) {
        b &= 0x7fffu;
        if (b < 0x7c00u && b > most) most = b;
    };
    const uint16_t *s = h + row * ld;
    for (int64_t c = lane * 8; c < cols; c += 512) {
        if (c + 8 <= cols) {
            const u32x4 v = *reinterpret_cast<const u32x4u *>(s + c);
#pragma unroll
            for (int e = 0; e < 4; e++) see(v[e]), see(v[e] >> 16);
        } else {
            for (int e = 0; c + e < cols; e++) see(s[c + e]);
        }
    }
#pragma unroll
    for (int d = 32; d; d /= 2) most = max(most, uint32_t(__shfl_xor(int(most), d, 64)));
    if (lane == 0 && most > 0) {
        int e;  // |h| < 2^e
        (void)frexpf(float(__builtin_bit_cast(_Float16, uint16_t(most))), &e);
        atomicMax(top, e + exponent(up[row]));
    }
}

// What f16 rows of H are scaled by besides their own 2^e, and its inverse for dW.
__device__ __forceinline__ int lift(const int *top) { return 15 - (*top == kNoTop ? 0 : *top); }

// Rows of 16-bit values into rows of `ldo` bytes, zeros from `cols` to their end: an operand that is not laid
// out as the copies need it. With `coef`, the rows that nothing flows through are zeros (whatever they hold, a
// NaN too, stays out of dW) and with `up`, f16 rows are scaled by up 2^lift, a power of two.
__global__ __launch_bounds__(256) void k_readout_rows(const uint16_t *src, int64_t rows, int64_t cols, int64_t ld,
                                                      uint8_t *out, int64_t ldo, const float4 *coef, const float *up,
                                                      const int *top) {
    const int64_t per = ldo / 16, total = rows * per;
    for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i / per, c = (i - r * per) * 8;
        const uint16_t *s = src + r * ld + c;
        union {
            u32x4 v;
            uint16_t h[8];
            _Float16 f[8];
        } x;
        x.v = u32x4{0, 0, 0, 0};
        if (!coef || coef[r].x != INFINITY) {
            if (c + 8 <= cols) x.v = *reinterpret_cast<const u32x4u *>(s);
            else
                for (int e = 0; e < 8; e++) x.h[e] = c + e < cols ? s[e] : uint16_t(0);
            if (up) {
                const int l = exponent(up[r]) + lift(top);  // (f32 need not hold 2^l)
#pragma unroll
                for (int e = 0; e < 8; e++) x.f[e] = _Float16(ldexpf(float(x.f[e]), l));
            }
        }
        *reinterpret_cast<u32x4 *>(out + r * ldo + c * 2) = x.v;
    }
}

template <class E>
__device__ __forceinline__ float widened(uint32_t h) {
    if constexpr (std::is_same<E, Bf16>::value) return __builtin_bit_cast(float, h << 16);
    else return float(__builtin_bit_cast(_Float16, uint16_t(h)));
}

// A piece's G.
template <class E, class S, bool BTR, bool MASK>
__global__ __launch_bounds__(S::kThreads, 1) void k_readout_g(PieceP p) {
    constexpr int TM = S::TM, TN = S::TN, WM = S::WM, WN = S::WN;
    typedef Tile<E, TM, TN, WM, WN, false, BTR> T;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int im, in;
    tile_of(blockIdx.x, p.tm, p.tn, im, in);
    T t;
    t.run(lds, Operand{p.h + int64_t(im) * T::BM * p.ldh, p.ldh, p.rows - int64_t(im) * T::BM, p.kbytes},
          weight_rows<T, BTR>(p, in), p.kbytes, wave, lane);
    const int wm = wave / WN, wn = wave % WN;
    const int col0 = in * T::BN + 32 * TN * wn + 4 * (lane / 32);
    const int64_t bytes = p.gbytes - (in * T::BN + 32 * TN * wn) * 2;
    // (a mask's 32 rows are read before G's block is written over them; a row that all share stays in front of it)
    constexpr int kShared = MASK ? MaskBlock<TN>::kShared : 0, kMask = MASK ? MaskBlock<TN>::kLds : 0;
    constexpr int kStore = kShared + store_bytes<TN>(2), kWave = kStore > kMask ? kStore : kMask;
    static_assert(kWave * WM * WN <= T::kLds && kWave % 16 == 0, "the blocks fit");
    uint8_t *const mlds = lds + wave * kWave, *const slds = mlds + kShared;
    float4 coef[TM];
    int tok[TM];  // the token's column from this lane's first, or -1
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t row = int64_t(im) * T::BM + 32 * (TM * wm + i) + lane % 32, r = row < p.rows ? row : p.rows - 1;
        coef[i] = p.coef[r];
        const int64_t at = p.tokens[r] - p.v0;
        tok[i] = at >= 0 && at < p.n && row < p.rows ? int(at) - col0 : -1;
    }
    if (bytes <= 0) return;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t row0 = int64_t(im) * T::BM + 32 * (TM * wm + i);
        if (row0 >= p.rows) break;
        const float4 k = coef[i];
        const bool dead = k.x == INFINITY;
        // (of 32 rows few have their token among this wave's columns)
        const bool mine = __any(tok[i] >= 0 && tok[i] < 32 * TN);
        float at_token = 0.0f, held = 0.0f;  // the row's entry at its token, and as it is written
        u32x2 v[4 * TN];
        float x[4 * TN][4];
#pragma unroll
        for (int q = 0; q < 4 * TN; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[q][e] = t.acc[i][q / 4][4 * (q % 4) + e];
        if constexpr (MASK) {
            MaskBlock<TN>::in(mlds, p.mask, row0, p.rows - row0 < 32 ? int(p.rows - row0) : 32, in * T::BN + 32 * TN * wn, p.n, lane, i == 0);
            wave_exchange();
            MaskBlock<TN>::out(mlds, p.mask, p.invt, lane, x);
            wave_exchange();
        } else if (in * T::BN + T::BN > p.n) {
            ended(x, p.n - col0);
        }
#pragma unroll
        for (int q = 0; q < 4 * TN; q++) {
            float g[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float l = (x[q][e] - k.x) * p.c, w = __builtin_amdgcn_exp2f(l);
                g[e] = w * fmaf(k.z, fmaxf(l, -200.0f), k.y);  // (p 0: 0, and a NaN stays in w)
            }
            if (mine)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (tok[i] == 8 * q + e) at_token = g[e] += k.w;
            v[q] = dead ? u32x2{0, 0} : u32x2{pair16<E>(g[0], g[1]), pair16<E>(g[2], g[3])};
            if (mine)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (tok[i] == 8 * q + e) held = widened<E>((e < 2 ? v[q].x : v[q].y) >> (16 * (e % 2)) & 0xffffu);
        }
        if (mine && tok[i] >= 0 && tok[i] < 32 * TN && (tok[i] & 4) == 0 && !dead) {
            const int64_t r = row0 + lane % 32;
            const float left = at_token - held;
            if (p.turn && fabsf(held) > p.left[r] && fabsf(left) <= 0x1p-8f * fabsf(held)) p.turn[r] = at_token / held;
            p.left[r] = left;
        }
        const int rows = p.rows - row0 < 32 ? int(p.rows - row0) : 32, have = bytes < 64 * TN ? int(bytes) : 64 * TN;
        uint8_t *o = p.g + row0 * p.ldg + (in * T::BN + 32 * TN * wn) * 2;
        store_block<TN>(slds, v, lane, o, p.ldg, rows, have);
    }
}

// C[m, n] = sum_k A(m, k) B(n, k) over the k of split z: into the gradient itself (16-bit, scaled), or into
// the split's f32 slab, set or added to.
struct GradP {
    const uint8_t *a, *b;
    int64_t lda, ldb, wa, wb; // strides, and bytes of a row of a transposed operand (a multiple of 16)
    int64_t m, n, k;          // k in elements (a k-contiguous operand's row is padded with zeros to 16 bytes)
    int64_t per;              // k of a split, a multiple of 32
    uint32_t tm, tn;
    uint16_t *out;            // [m, ldo] or null
    int64_t ldo;
    float *slab;              // [splits][m][n] f32
    int add;
    const float *row_scale;   // f16: [m] or null
    const float *turn;        // [m] or null: another scale of the rows (dH)
    const int *top;           // f16: [1] or null
    float fixed;
    // dW: what the rounding of G left of the tokens' entries
    const float *left;        // [k]
    const int2 *place;        // the rows of each 256 tokens
    const uint32_t *listed;
    int64_t v0;               // the vocabulary's first row of the output (VD) or column (DV)
    bool dv;
};

// dW's share of what the rounding of G left of each row's entry at its token, left[r] H(r, .) to the token's row of dW
// (column, DV), as more k of the product: 32 of the rows whose token is in the tile's bucket at a time, one side of a stage
// their rows of H, the other zeros but for each row's left (rounded to the operands' type: 2^-9 of what G's rounding
// left) at its token. (Few rows have their token in a tile: of 4096, 8 in 256 columns of 128256, one stage beside 128.)
template <class S>
struct LeftRows {
    static_assert(S::kRows <= kBucket && S::kCols <= kBucket, "a tile in a bucket");
    int2 place;
    int in;       // the tile's first column in its bucket
    uint32_t e;   // this lane's of the first 64 rows, and what is left (0: none)
    float left;

    __device__ __forceinline__ void entry(const GradP &p, int j, uint32_t &e, float &left) const {
        e = j < place.y ? p.listed[place.x + j] : 0u;
        left = j < place.y ? p.left[e >> 8] : 0.0f;
    }
    // In front of the product (its latency beside the product's).
    __device__ __forceinline__ void init(const GradP &p, int64_t m0, int64_t n0, int lane) {
        const int64_t v = p.v0 + (p.dv ? n0 : m0);
        place = p.place[v / kBucket];
        in = int(v % kBucket);
        entry(p, lane, e, left);
    }
    // One operand's panel of a stage (nt_tile.hpp), B columns: H's rows of lane j0 + k's entries, or the lefts.
    template <int B>
    __device__ __forceinline__ void rows(uint8_t *panel, const uint8_t *h, int64_t ldh, int64_t wh, uint32_t e, int j0) const {
        typedef Side<B, S::WM * S::WN, true> P;
        constexpr int kPer = 2 * B / 16;  // chunks of 16 bytes a row
        for (int x = threadIdx.x; x < 32 * kPer; x += S::kThreads) {
            const int k = x / kPer, at = x % kPer * 16;
            const int64_t r = uint32_t(__shfl(int(e), j0 + k, 64)) >> 8;
            u32x4 v = {0, 0, 0, 0};
            if (at < wh) v = *reinterpret_cast<const u32x4 *>(h + r * ldh + at);
            *reinterpret_cast<u32x4 *>(panel + P::at(k, at)) = v;
        }
    }
    template <class E, int B>
    __device__ __forceinline__ void tokens(uint8_t *panel, uint32_t e, float left, int j0, int lane) const {
        typedef Side<B, S::WM * S::WN, true> P;
        for (int x = threadIdx.x; x < 4 * B; x += S::kThreads) *reinterpret_cast<u32x4 *>(panel + x * 16) = u32x4{0, 0, 0, 0};
        __syncthreads();
        const uint32_t c = (e & 255u) - uint32_t(in);
        if (threadIdx.x < 64 && lane - j0 >= 0 && lane - j0 < 32 && left != 0.0f && c < uint32_t(B))
            *reinterpret_cast<uint16_t *>(panel + P::at(lane - j0, int(c) * 2)) = uint16_t(pair16<E>(left, 0.0f));
    }
    template <class E, class T>
    __device__ __forceinline__ void add(T &t, uint8_t *lds, const GradP &p, int64_t m0, int64_t n0, int wave, int lane) {
        constexpr int BM = T::BM, BN = T::BN;
        uint8_t *const a = lds, *const b = lds + T::SideA::kBytes;
        for (int j = 0; j < place.y; j += 32) {
            if (j > 0 && j % 64 == 0) entry(p, j + lane, e, left);
            const int j0 = j % 64;
            if (p.dv) {
                rows<BM>(a, p.a + m0 * 2, p.lda, p.wa - m0 * 2, e, j0);
                tokens<E, BN>(b, e, left, j0, lane);
            } else {
                rows<BN>(b, p.b + n0 * 2, p.ldb, p.wb - n0 * 2, e, j0);
                tokens<E, BM>(a, e, left, j0, lane);
            }
            __syncthreads();
            t.stage(lds, wave, lane);
            __syncthreads();
        }
    }
};

// (Two waves a SIMD, 256 registers each, or the smaller tiles' second workgroup waits: dW 128 x 1024 x 32000 54 -> 30 us.)
template <class E, class S, bool ATR, bool BTR>
__global__ __launch_bounds__(S::kThreads, S::TM == 1 ? 2 : 1) void k_readout_grad(GradP p) {
    constexpr int TM = S::TM, TN = S::TN, WM = S::WM, WN = S::WN;
    typedef Tile<E, TM, TN, WM, WN, ATR, BTR> T;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int im, in;
    tile_of(blockIdx.x, p.tm, p.tn, im, in);
    const int64_t k0 = blockIdx.y * p.per, left = p.k - k0 < p.per ? p.k - k0 : p.per;
    const int64_t kn = left > 0 ? left : 0;  // (a shorter last piece may leave a split nothing: zeros)
    const int64_t m0 = int64_t(im) * T::BM, n0 = int64_t(in) * T::BN;
    const int64_t kb = (kn * 2 + 15) / 16 * 16;
    const Operand a = ATR ? Operand{p.a + k0 * p.lda + m0 * 2, p.lda, kn, p.wa - m0 * 2}
                          : Operand{p.a + m0 * p.lda + k0 * 2, p.lda, p.m - m0, kb};
    const Operand b = BTR ? Operand{p.b + k0 * p.ldb + n0 * 2, p.ldb, kn, p.wb - n0 * 2}
                          : Operand{p.b + n0 * p.ldb + k0 * 2, p.ldb, p.n - n0, kb};
    constexpr bool kDW = ATR && BTR;
    LeftRows<S> lefts;
    if (kDW) lefts.init(p, m0, n0, lane);
    T t;
    t.run(lds, a, b, kb, wave, lane);
    if constexpr (kDW)
        if (blockIdx.y == 0) lefts.template add<E>(t, lds, p, m0, n0, wave, lane);
    const int wm = wave / WN, wn = wave % WN;
    const float whole = p.top ? ldexpf(p.fixed, -lift(p.top)) : p.fixed;
    const int64_t col0 = n0 + 32 * TN * wn;
    if (col0 >= p.n) return;
    float f[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t row = m0 + 32 * (TM * wm + i) + lane % 32;
        const int64_t r = row < p.m ? row : p.m - 1;
        f[i] = p.row_scale ? p.row_scale[r] * whole : whole;
        if (!kDW && p.turn) f[i] *= p.turn[r];
    }
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t row0 = m0 + 32 * (TM * wm + i);
        if (row0 >= p.m) break;
        const int rows = p.m - row0 < 32 ? int(p.m - row0) : 32;
        const int cols = p.n - col0 < 32 * TN ? int(p.n - col0) : 32 * TN;
        if (p.out) {
            u32x2 v[4 * TN];
#pragma unroll
            for (int q = 0; q < 4 * TN; q++) {
                v[q] = u32x2{pair16<E>(t.acc[i][q / 4][4 * (q % 4)] * f[i], t.acc[i][q / 4][4 * (q % 4) + 1] * f[i]),
                             pair16<E>(t.acc[i][q / 4][4 * (q % 4) + 2] * f[i], t.acc[i][q / 4][4 * (q % 4) + 3] * f[i])};
            }
            store_block<TN>(lds + wave * store_bytes<TN>(2), v, lane, reinterpret_cast<uint8_t *>(p.out + row0 * p.ldo + col0),
                            p.ldo * 2, rows, cols * 2);
            continue;
        }
        float *o = p.slab + (int64_t(blockIdx.y) * p.m + row0) * p.n + col0;
        float c[4 * TN][4];
#pragma unroll
        for (int q = 0; q < 4 * TN; q++) c[q][0] = c[q][1] = c[q][2] = c[q][3] = 0.0f;
        if (p.add) {  // (every load before the first store)
#pragma unroll
            for (int q = 0; q < 4 * TN; q++) {
                const int r = lane % 32, at = 8 * q + 4 * (lane / 32), have = r < rows ? cols - at : 0;
                const float *s = o + int64_t(r) * p.n + at;
                if (have >= 4) __builtin_memcpy(c[q], s, 16);
                else
                    for (int e = 0; e < 4; e++)
                        if (e < have) c[q][e] = s[e];
            }
        }
        u32x4 v[4 * TN];
#pragma unroll
        for (int q = 0; q < 4 * TN; q++) {
#pragma unroll
            for (int e = 0; e < 4; e++) c[q][e] += t.acc[i][q / 4][4 * (q % 4) + e];
            __builtin_memcpy(&v[q], c[q], 16);
        }
        store_block<TN>(lds + wave * store_bytes<TN>(4), v, lane, reinterpret_cast<uint8_t *>(o), p.n * 4, rows, cols * 4);
    }
}

// The slabs' sum in their order, scaled and rounded; with `left`, first each row's times the token's row of W (a column
// of it, DV).
struct LeftP {
    const float *left;      // [m] or null
    const int32_t *tokens;  // [m]
    const uint16_t *w;
    int64_t ldw;
    int dv;
};

// Rows up to which a DV weight's columns are read for it: a column's every value is a line of its own, and for 2048 rows of
// dim 4096 (V 50304) they took 90 us of 2930. A row of dH of more is scaled instead, by the exact entry over the rounded
// one: its token's part is then right, and the others' off by that factor, within 2^-9 of 1 (bf16; f16 2^-12). Without an
// entropy's gradient the others are no larger than the token's (a row of G sums to zero, so their part is the token's entry
// times a mean of W's columns); with one the row is scaled where its token's entry is over 8 |g_entropy|, which the other
// entries' norm by p (ln p + entropy), sqrt(max p Var ln p) at the most, is under up to vocabularies of 2^20.
constexpr int64_t kColumnRows = 512;

template <class E>
__global__ __launch_bounds__(256) void k_readout_fold(const float *slab, int splits, int64_t m, int64_t n, LeftP p, uint16_t *out,
                                                      int64_t ldo, const float *row_scale, const float *turn, const int *top,
                                                      float fixed) {
    const int64_t per = (n + 3) / 4, total = m * per;
    for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i / per, c = (i - r * per) * 4;
        const int have = n - c >= 4 ? 4 : int(n - c);
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float left = p.left ? p.left[r] : 0.0f;
        if (left != 0.0f) {
            const uint16_t *w = p.w + (p.dv ? c * p.ldw + p.tokens[r] : p.tokens[r] * p.ldw + c);
            for (int e = 0; e < have; e++) x[e] = left * widened<E>(w[p.dv ? e * p.ldw : e]);
        }
        auto at = [&](int z) { return slab + (z * m + r) * n + c; };
        int z = 0;
        if (have == 4)
            for (; z + 8 <= splits; z += 8) {  // (eight loads in flight)
                float v[8][4];
#pragma unroll
                for (int k = 0; k < 8; k++) __builtin_memcpy(v[k], at(z + k), 16);
#pragma unroll
                for (int k = 0; k < 8; k++)
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] += v[k][e];
            }
        for (; z < splits; z++)
            for (int e = 0; e < have; e++) x[e] += at(z)[e];
        float f = top ? ldexpf(fixed, -lift(top)) : fixed;
        if (row_scale) f *= row_scale[r];
        if (turn) f *= turn[r];
        uint16_t *o = out + r * ldo + c;
        const uint32_t w[2] = {pair16<E>(x[0] * f, x[1] * f), pair16<E>(x[2] * f, x[3] * f)};
        if (have == 4) __builtin_memcpy(o, w, 8);
        else
            for (int e = 0; e < have; e++) o[e] = uint16_t(w[e / 2] >> (16 * (e % 2)));
    }
}

// ---------------------------------------------------------------------------------- host

// Scratch of one call: sizes are asked for first, then allocated, the large ones each by itself (the library keeps
// blocks of up to 128 MiB for the next call; a larger one is the device pool's, and its allocation may wait for the
// stream), then the places.
struct Scratch {
    static constexpr int kMost = 16;
    static constexpr size_t kAlone = size_t(1) << 20;
    size_t size[kMost], together = 0;
    void *place[kMost], *shared = nullptr;
    int n = 0;
    int add(int64_t bytes) {
        size[n] = (size_t(bytes) + 255) & ~size_t(255);
        place[n] = nullptr;
        if (size[n] < kAlone) together += size[n];
        return n++;
    }
    // `large`: the call takes 256 x 256 tiles. Under stream capture such a call, and one with 1 MiB of scratch, is refused: a
    // captured step of 2100 x 512 x 32768 faulted in its replays, for a cause not found, where it runs as it should
    // outside of a graph; captured steps of smaller tiles whose scratch is one block replay rightly.
    int allocate(const char *who, bool large) {
        bool cap = false;
        if (int rc = stream_capturing(&cap)) return rc;
        large |= together >= kAlone;
        for (int i = 0; i < n; i++) large |= size[i] >= kAlone;
        if (cap && large)
            return fail(NT_E_UNSUPPORTED, std::string(who) + ": too large for stream capture (256 x 256 tiles, or scratch of 1 MiB "
                                                             "and more)");
        if (int rc = scratch_alloc(together, &shared)) return rc;
        uint8_t *at = static_cast<uint8_t *>(shared);
        for (int i = 0; i < n; i++) {
            if (size[i] >= kAlone) {
                if (int rc = scratch_alloc(size[i], &place[i])) return rc;
            } else {
                place[i] = at;
                at += size[i];
            }
        }
        return 0;
    }
    template <class P>
    P *at(int i) const {
        return static_cast<P *>(place[i]);
    }
    ~Scratch() {
        for (int i = 0; i < n; i++)
            if (size[i] >= kAlone && place[i]) (void)scratch_release(place[i]);
        if (shared) (void)scratch_release(shared);
    }
};

constexpr int64_t kMaxDim = 65536, kMaxVocab = 1 << 20, kMaxRows = 1 << 24;

// What both entries check of the operands. `dv`: the weight is [dim, vocab].
int check(const char *who, const void *hidden, const void *weight, int32_t dtype, int32_t layout, int64_t rows, int64_t vocab,
          int64_t dim, int64_t ldh, int64_t ldw, int32_t mask_kind, const void *mask, int64_t mask_ld, double tau,
          const int32_t *tokens) {
    if (dtype != NT_BF16 && dtype != NT_F16)
        return fail(NT_E_ARG, std::string(who) + ": dtype " + std::to_string(dtype) + " (NT_BF16 or NT_F16)");
    if (layout != NT_READOUT_W_DV && layout != NT_READOUT_W_VD)
        return fail(NT_E_ARG, std::string(who) + ": layout " + std::to_string(layout) + " (NT_READOUT_W_DV or _VD)");
    const int64_t wrow = layout == NT_READOUT_W_DV ? vocab : dim;
    if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab || dim < 1 || dim > kMaxDim || ldh < dim || ldw < wrow ||
        ldh > (int64_t(1) << 21) || ldw > (int64_t(1) << 21))
        return fail(NT_E_ARG, std::string(who) + ": rows " + std::to_string(rows) + " (at most 2^24), vocab " +
                                  std::to_string(vocab) + " (1 to 2^20), dim " + std::to_string(dim) +
                                  " (1 to 65536), ldh " + std::to_string(ldh) + ", ldw " + std::to_string(ldw) +
                                  " (at least the row, at most 2^21)");
    if (mask_kind != NT_MASK_NONE && mask_kind != NT_MASK_U8 && mask_kind != NT_MASK_F32)
        return fail(NT_E_ARG, std::string(who) + ": mask kind " + std::to_string(mask_kind));
    if ((mask_kind == NT_MASK_NONE) != (mask == nullptr))
        return fail(NT_E_ARG, std::string(who) + ": mask kind and mask pointer disagree");
    if (mask && mask_ld != 0 && mask_ld < vocab)
        return fail(NT_E_ARG, std::string(who) + ": mask_ld " + std::to_string(mask_ld) + " (0, or at least vocab)");
    if (mask_kind == NT_MASK_F32 && reinterpret_cast<uintptr_t>(mask) % 4)
        return fail(NT_E_ARG, std::string(who) + ": unaligned mask");
    if (!(tau > 0.0) || !std::isfinite(tau) || !(float(kLog2eD / tau) > 0.0f) || std::isinf(float(kLog2eD / tau)))
        return fail(NT_E_ARG, "tempered_logits: temperature " + std::to_string(tau) + " (must be positive)");
    if (rows > 0 && (!hidden || !weight || !tokens || reinterpret_cast<uintptr_t>(hidden) % 2 ||
                     reinterpret_cast<uintptr_t>(weight) % 2))
        return fail(NT_E_ARG, std::string(who) + ": null or unaligned hidden or weight, or null tokens");
    return 0;
}

bool aligned(const void *p, int64_t cols, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && cols % 8 == 0;
}

int copy_rows(const void *src, int64_t rows, int64_t cols, int64_t ld, uint8_t *out, int64_t ldo, const float4 *coef,
              const float *up, const int *top) {
    const int64_t n = rows * (ldo / 16);
    hipLaunchKernelGGL(k_readout_rows, dim3(unsigned(std::min<int64_t>(ceil_div(n, 256), 8192))), dim3(256), 0,
                       ctx().stream, static_cast<const uint16_t *>(src), rows, cols, ld, out, ldo, coef, up, top);
    return launched("k_readout_rows");
}

// A piece of the weight as the copies need it: in place, or copied into `buf` where it is not aligned.
int piece_weight(const void *weight, bool dv, bool direct, int64_t v0, int64_t n, int64_t dim, int64_t ldw, uint8_t *buf,
                 PieceP *p) {
    const uint16_t *s = static_cast<const uint16_t *>(weight) + (dv ? v0 : v0 * ldw);
    p->wwidth = round_up(dv ? n : dim, 8) * 2;
    if (direct) {
        p->w = reinterpret_cast<const uint8_t *>(s);
        p->ldw = ldw * 2;
        return 0;
    }
    p->w = buf;
    p->ldw = p->wwidth;
    return copy_rows(s, dv ? dim : n, dv ? n : dim, ldw, buf, p->ldw, nullptr, nullptr, nullptr);
}

MaskP mask_at(int32_t kind, const void *mask, int64_t ld, int64_t v0) {
    MaskP m{nullptr, nullptr, ld};
    if (kind == NT_MASK_U8) m.u8 = static_cast<const uint8_t *>(mask) + v0;
    if (kind == NT_MASK_F32) m.f32 = static_cast<const float *>(mask) + v0;
    return m;
}

constexpr int kBlockCols = 128;  // columns of a forward block: a wave's of a 256-column tile
constexpr int kTile = 256;

// The vocabulary's pieces: whole tiles, `cols` of them at most.
int64_t piece_cols(int64_t vocab, int64_t cols) {
    const int64_t most = std::max<int64_t>(kTile, cols / kTile * kTile);
    const int64_t pieces = ceil_div(vocab, most);
    return std::min(round_up(ceil_div(vocab, pieces), kTile), round_up(vocab, kTile));
}

// Columns c0 .. c0 + n - 1 of a piece (c0 a multiple of 256).
PieceP part_of(const PieceP &p, bool dv, int64_t c0, int64_t n) {
    PieceP q = p;
    q.w += dv ? c0 * 2 : c0 * p.ldw;
    q.wwidth -= dv ? c0 * 2 : 0;
    q.n = int(n);
    q.v0 += c0;
    q.block0 += c0 / 128;
    q.g += c0 * 2;
    q.gbytes = c0 + n < p.n ? n * 2 : p.gbytes - c0 * 2;
    if (p.mask.u8) q.mask.u8 += c0;
    if (p.mask.f32) q.mask.f32 += c0;
    return q;
}

template <class E, class S, bool BTR>
int launch_stats(PieceP p, bool ent) {
    p.tm = uint32_t(ceil_div(p.rows, S::kRows));
    p.tn = uint32_t(ceil_div(p.n, S::kCols));
    const dim3 grid(p.tm * p.tn), block(S::kThreads);
    hipStream_t st = ctx().stream;
    if (p.mask.u8 || p.mask.f32) {
        if (ent) k_readout_stats<E, S, BTR, true, true><<<grid, block, 0, st>>>(p);
        else k_readout_stats<E, S, BTR, false, true><<<grid, block, 0, st>>>(p);
    } else {
        if (ent) k_readout_stats<E, S, BTR, true, false><<<grid, block, 0, st>>>(p);
        else k_readout_stats<E, S, BTR, false, false><<<grid, block, 0, st>>>(p);
    }
    return launched("k_readout_stats");
}

template <class E, bool BTR>
int stats(const PieceP &p, bool ent) {
    if (const int64_t c = whole_rounds(p.rows, p.n, p.kbytes)) {
        if (int rc = launch_stats<E, Large, BTR>(part_of(p, BTR, 0, c), ent)) return rc;
        return stats<E, BTR>(part_of(p, BTR, c, p.n - c), ent);
    }
    switch (plan(p.rows, p.n, p.kbytes, false).size) {
        case Size::kSmall: return launch_stats<E, Small, BTR>(p, ent);
        case Size::kMedium: return launch_stats<E, Medium, BTR>(p, ent);
        default: return launch_stats<E, Large, BTR>(p, ent);
    }
}

template <class E, class S, bool BTR>
int launch_g(PieceP p) {
    p.tm = uint32_t(ceil_div(p.rows, S::kRows));
    p.tn = uint32_t(ceil_div(p.n, S::kCols));
    const dim3 grid(p.tm * p.tn), block(S::kThreads);
    if (p.mask.u8 || p.mask.f32) k_readout_g<E, S, BTR, true><<<grid, block, 0, ctx().stream>>>(p);
    else k_readout_g<E, S, BTR, false><<<grid, block, 0, ctx().stream>>>(p);
    return launched("k_readout_g");
}

template <class E, bool BTR>
int g_piece(const PieceP &p) {
    if (const int64_t c = whole_rounds(p.rows, p.n, p.kbytes)) {
        if (int rc = launch_g<E, Large, BTR>(part_of(p, BTR, 0, c))) return rc;
        return g_piece<E, BTR>(part_of(p, BTR, c, p.n - c));
    }
    switch (plan(p.rows, p.n, p.kbytes, false).size) {
        case Size::kSmall: return launch_g<E, Small, BTR>(p);
        case Size::kMedium: return launch_g<E, Medium, BTR>(p);
        default: return launch_g<E, Large, BTR>(p);
    }
}

int forward(const NtRlReadoutStatsArgs *a) {
    const bool dv = a->layout == NT_READOUT_W_DV;
    const int64_t R = a->rows, V = a->vocab, d = a->dim, kp = round_up(d, 8);
    const bool hdirect = aligned(a->hidden, d, a->ldh);
    const bool wdirect = aligned(a->weight, dv ? V : d, a->ldw);
    // one launch for the whole vocabulary, but for a copied weight (pieces of 128 MiB) and more than 2^20 large tiles (a
    // launch holds fewer than 2^32 threads: 2^23 small ones of 128)
    int64_t most = (int64_t(1) << 20) / ceil_div(R, kTile) * kTile;
    if (!wdirect) most = std::min(most, (int64_t(1) << 26) / kp);
    const int64_t cols = piece_cols(V, most);
    const int64_t blocks = ceil_div(V, kTile) * 2, rows_p = round_up(R, 32);  // (a large tile writes whole ones)
    Scratch s;
    const int o_h = s.add(hdirect ? 0 : R * kp * 2);
    const int o_w = s.add(wdirect ? 0 : (dv ? d * cols : cols * kp) * 2);
    const int o_ref = s.add(blocks * rows_p * 4), o_sum = s.add(blocks * rows_p * 4);
    const int o_es = s.add(a->entropy ? blocks * rows_p * 4 : 0), o_x = s.add(R * 4);
    if (int rc = s.allocate("nt_hip_rl_readout_score_stats", plan(R, std::min(cols, V), kp * 2, false).size == Size::kLarge)) return rc;
    PieceP p{};
    p.h = static_cast<const uint8_t *>(a->hidden);
    p.ldh = a->ldh * 2;
    if (!hdirect) {
        if (int rc = copy_rows(a->hidden, R, d, a->ldh, s.at<uint8_t>(o_h), kp * 2, nullptr, nullptr, nullptr)) return rc;
        p.h = s.at<uint8_t>(o_h);
        p.ldh = kp * 2;
    }
    p.rows = R;
    p.dim = d;
    p.kbytes = kp * 2;
    p.c = a->mask_kind == NT_MASK_F32 ? kLog2e : float(kLog2eD / a->temperature);
    p.invt = float(1.0 / a->temperature);
    p.tokens = a->tokens;
    p.ref = s.at<float>(o_ref);
    p.sum = s.at<float>(o_sum);
    p.esum = a->entropy ? s.at<float>(o_es) : nullptr;
    p.rows_p = rows_p;
    p.xtok = s.at<float>(o_x);
    for (int64_t v0 = 0; v0 < V; v0 += cols) {
        const int64_t n = std::min(cols, V - v0);
        if (int rc = piece_weight(a->weight, dv, wdirect, v0, n, d, a->ldw, s.at<uint8_t>(o_w), &p)) return rc;
        p.n = int(n);
        p.v0 = v0;
        p.block0 = v0 / kBlockCols;
        p.mask = mask_at(a->mask_kind, a->mask, a->mask_ld, v0);
        const bool bf16 = a->dtype == NT_BF16, ent = a->entropy != nullptr;
        const int rc = dv ? (bf16 ? stats<Bf16, true>(p, ent) : stats<F16, true>(p, ent))
                          : (bf16 ? stats<Bf16, false>(p, ent) : stats<F16, false>(p, ent));
        if (rc) return rc;
    }
    MergeP q{};
    q.ref = p.ref;
    q.sum = p.sum;
    q.esum = p.esum;
    q.rows = R;
    q.rows_p = rows_p;
    q.blocks = int(ceil_div(V, kBlockCols));
    q.vocab = V;
    q.xtok = p.xtok;
    q.tokens = a->tokens;
    q.mask = mask_at(a->mask_kind, a->mask, a->mask_ld, 0);
    q.tau = a->temperature;
    q.c = p.c;
    q.invt = p.invt;
    q.logp = a->logp;
    q.entropy = a->entropy;
    q.base = a->lse_base;
    q.rest = a->lse_rest;
    q.status = a->status;
    hipLaunchKernelGGL(k_readout_merge, dim3(unsigned(ceil_div(R, 32))), dim3(1024), 0, ctx().stream, q);
    return launched("k_readout_merge");
}

template <class E>
int fold(const GradP &p, int64_t splits, uint16_t *out, const LeftP &left = {}) {
    const int64_t n = p.m * ceil_div(p.n, 4);
    hipLaunchKernelGGL(k_readout_fold<E>, dim3(unsigned(std::min<int64_t>(ceil_div(n, 256), 8192))), dim3(256), 0,
                       ctx().stream, p.slab, int(splits), p.m, p.n, left, out, p.ldo, p.row_scale, p.turn, p.top, p.fixed);
    return launched("k_readout_fold");
}

template <class E, class S, bool ATR, bool BTR>
int launch_product(GradP p, const Plan &s) {
    p.per = s.per / 2;
    p.tm = uint32_t(ceil_div(p.m, S::kRows));
    p.tn = uint32_t(ceil_div(p.n, S::kCols));
    k_readout_grad<E, S, ATR, BTR><<<dim3(p.tm * p.tn, unsigned(s.splits)), dim3(S::kThreads), 0, ctx().stream>>>(p);
    return launched("k_readout_grad");
}

template <class E, bool ATR, bool BTR>
int product(const GradP &p, const Plan &s) {
    switch (s.size) {
        case Size::kSmall: return launch_product<E, Small, ATR, BTR>(p, s);
        case Size::kMedium: return launch_product<E, Medium, ATR, BTR>(p, s);
        default: return launch_product<E, Large, ATR, BTR>(p, s);
    }
}

// One piece of the vocabulary: its G, its rows of dW, its share of dH.
struct BackP {
    const NtRlReadoutStatsGradArgs *a;
    PieceP p;
    Plan sh, sw;
    bool hslab, hleft;
    const int2 *place;
    const uint32_t *listed;
    const uint8_t *hs;  // the scaled hidden states, [rows, ldhs bytes]
    int64_t ldhs;
    float *slab_h, *slab_w;
    const float *up;
    const int *top;
    float fixed;
    bool last;
};

template <class E, bool DV>
int piece(const BackP &b) {
    const NtRlReadoutStatsGradArgs *a = b.a;
    const PieceP &p = b.p;
    if (int rc = g_piece<E, DV>(p)) return rc;
    if (a->grad_weight) {
        GradP w{};
        w.a = DV ? b.hs : p.g;
        w.lda = w.wa = DV ? b.ldhs : p.ldg;
        w.b = DV ? p.g : b.hs;
        w.ldb = w.wb = DV ? p.ldg : b.ldhs;
        w.m = DV ? p.dim : p.n;
        w.n = DV ? p.n : p.dim;
        w.k = p.rows;
        w.left = p.left;
        w.place = b.place;
        w.listed = b.listed;
        w.v0 = p.v0;
        w.dv = DV;
        uint16_t *out = static_cast<uint16_t *>(a->grad_weight) + (DV ? p.v0 : p.v0 * a->grad_weight_ld);
        w.ldo = a->grad_weight_ld;
        w.out = b.sw.splits > 1 ? nullptr : out;
        w.slab = b.slab_w;
        w.top = b.top;
        w.fixed = b.fixed;
        const int64_t c = b.sw.splits > 1 ? 0 : whole_rounds(DV ? w.m : w.n, DV ? w.n : w.m, w.k * 2);
        if (c) {  // whole rounds of the vocabulary's side, and its rest
            GradP first = w, rest = w;
            (DV ? first.n : first.m) = c;
            (DV ? rest.n : rest.m) -= c;
            (DV ? rest.b : rest.a) += c * 2;
            (DV ? rest.wb : rest.wa) -= c * 2;
            rest.out += DV ? c : c * rest.ldo;
            rest.v0 += c;
            if (int rc = launch_product<E, Large, true, true>(first, b.sw)) return rc;
            if (int rc = product<E, true, true>(rest, plan(rest.m, rest.n, rest.k * 2, false))) return rc;
        } else if (int rc = product<E, true, true>(w, b.sw)) {
            return rc;
        }
        if (b.sw.splits > 1)
            if (int rc = fold<E>(w, b.sw.splits, out)) return rc;
    }
    if (a->grad_hidden) {
        GradP h{};
        h.a = p.g;
        h.lda = p.ldg;
        h.b = p.w;
        h.ldb = p.ldw;
        h.wb = p.wwidth;
        h.m = p.rows;
        h.n = p.dim;
        h.k = p.n;
        h.ldo = a->grad_hidden_ld;
        uint16_t *out = static_cast<uint16_t *>(a->grad_hidden);
        h.out = b.hslab ? nullptr : out;
        h.slab = b.slab_h;
        h.add = p.v0 > 0;
        h.row_scale = b.up;
        h.turn = p.turn;
        h.fixed = b.fixed;
        if (int rc = product<E, false, !DV>(h, b.sh)) return rc;
        if (b.hslab && b.last) {
            const LeftP left{b.hleft ? p.left : nullptr, p.tokens, static_cast<const uint16_t *>(a->weight), a->ldw, DV};
            if (int rc = fold<E>(h, b.sh.splits, out, left)) return rc;
        }
    }
    return 0;
}

int backward(const NtRlReadoutStatsGradArgs *a) {
    const bool dv = a->layout == NT_READOUT_W_DV, f16 = a->dtype == NT_F16;
    const int64_t R = a->rows, V = a->vocab, d = a->dim, kp = round_up(d, 8);
    if (R == 0) {  // a sum over no rows
        GradP w{};
        w.m = dv ? d : V;
        w.n = dv ? V : d;
        w.ldo = a->grad_weight_ld;
        return a->grad_weight ? fold<Bf16>(w, 0, static_cast<uint16_t *>(a->grad_weight)) : 0;
    }
    const bool hdirect = aligned(a->hidden, d, a->ldh);
    const bool wdirect = aligned(a->weight, dv ? V : d, a->ldw);
    // G of a piece takes at most 512 MiB, a copied piece of the weight 128 MiB. (Pieces of 128 MiB of G, which the
    // memory-side cache would hold between the products, lost: dH's sums are read and written for each piece. 4096 x
    // 4096 x 128256 13.8 against 13.5 ms.)
    int64_t most = (int64_t(1) << 28) / R;
    if (!wdirect) most = std::min(most, (int64_t(1) << 26) / kp);
    const int64_t cols = piece_cols(V, most);
    // dH: [rows, dim], k the piece's columns; dW: [vocab, dim] or [dim, vocab], k the rows
    const int64_t width = std::min(cols, V);
    const Plan sh = plan(R, d, round_up(width, 8) * 2, true);
    const Plan sw = dv ? plan(d, width, R * 2, true) : plan(width, d, R * 2, true);
    const bool hleft = !dv || R <= kColumnRows, hslab = hleft || sh.splits > 1 || cols < V;
    Scratch s;
    const int o_h = s.add(hdirect ? 0 : R * kp * 2), o_hs = s.add(a->grad_weight ? R * kp * 2 : 0);
    const int o_w = s.add(wdirect ? 0 : (dv ? d * cols : cols * kp) * 2);
    const int o_coef = s.add(R * 16), o_left = s.add(R * 4), o_up = s.add(f16 ? R * 4 : 0), o_top = s.add(f16 ? 4 : 0);
    const int64_t buckets = a->grad_weight ? ceil_div(V, kBucket) : 0;
    const int o_turn = s.add(a->grad_hidden && !hleft ? R * 4 : 0);
    const int o_place = s.add(buckets * 8), o_listed = s.add(buckets ? R * 4 : 0);
    const int o_g = s.add(R * cols * 2);
    const int o_sh = s.add(a->grad_hidden && hslab ? sh.splits * R * d * 4 : 0);
    const int o_sw = s.add(a->grad_weight && sw.splits > 1 ? sw.splits * std::min(cols, V) * d * 4 : 0);
    const bool large = plan(R, width, kp * 2, false).size == Size::kLarge || (a->grad_hidden && sh.size == Size::kLarge) ||
                       (a->grad_weight && sw.size == Size::kLarge);
    if (int rc = s.allocate("nt_hip_rl_readout_score_backward", large)) return rc;
    const float *up = f16 ? s.at<float>(o_up) : nullptr;
    int *top = f16 ? s.at<int>(o_top) : nullptr;
    const float fixed = f16 ? float(ldexp(1.0, -14) / a->temperature) : 1.0f;
    CoefP c{};
    c.base = a->lse_base;
    c.rest = a->lse_rest;
    c.entropy = a->entropy;
    c.g_logp = a->g_logp;
    c.g_entropy = a->g_entropy;
    c.tokens = a->tokens;
    c.rows = R;
    c.vocab = V;
    c.tau = a->temperature;
    c.f32mask = a->mask_kind == NT_MASK_F32;
    c.f16 = f16;
    c.coef = s.at<float4>(o_coef);
    c.left = s.at<float>(o_left);
    c.turn = a->grad_hidden && !hleft ? s.at<float>(o_turn) : nullptr;
    c.up = f16 ? s.at<float>(o_up) : nullptr;
    c.top = top;
    c.coefs = unsigned(std::min<int64_t>(ceil_div(R, 1024), 256));
    c.place = s.at<int2>(o_place);
    c.listed = s.at<uint32_t>(o_listed);
    hipLaunchKernelGGL(k_readout_coef, dim3(c.coefs + unsigned(buckets)), dim3(1024), 0, ctx().stream, c);
    if (int rc = launched("k_readout_coef")) return rc;
    if (a->grad_weight && f16) {
        hipLaunchKernelGGL(k_readout_top, dim3(unsigned(ceil_div(R, 4))), dim3(256), 0, ctx().stream,
                           static_cast<const uint16_t *>(a->hidden), R, d, a->ldh, up, top);
        if (int rc = launched("k_readout_top")) return rc;
    }
    if (a->grad_weight)
        if (int rc = copy_rows(a->hidden, R, d, a->ldh, s.at<uint8_t>(o_hs), kp * 2, c.coef, up, top)) return rc;
    PieceP p{};
    p.h = static_cast<const uint8_t *>(a->hidden);
    p.ldh = a->ldh * 2;
    if (!hdirect) {
        if (int rc = copy_rows(a->hidden, R, d, a->ldh, s.at<uint8_t>(o_h), kp * 2, nullptr, nullptr, nullptr)) return rc;
        p.h = s.at<uint8_t>(o_h);
        p.ldh = kp * 2;
    }
    p.rows = R;
    p.dim = d;
    p.kbytes = kp * 2;
    p.c = a->mask_kind == NT_MASK_F32 ? kLog2e : float(kLog2eD / a->temperature);
    p.invt = float(1.0 / a->temperature);
    p.tokens = a->tokens;
    p.coef = c.coef;
    p.g = s.at<uint8_t>(o_g);
    p.left = c.left;
    p.turn = c.turn;
    for (int64_t v0 = 0; v0 < V; v0 += cols) {
        const int64_t n = std::min(cols, V - v0);
        if (int rc = piece_weight(a->weight, dv, wdirect, v0, n, d, a->ldw, s.at<uint8_t>(o_w), &p)) return rc;
        p.n = int(n);
        p.v0 = v0;
        p.ldg = p.gbytes = round_up(n, 8) * 2;
        p.mask = mask_at(a->mask_kind, a->mask, a->mask_ld, v0);
        BackP b{a, p, sh, sw, hslab, hleft, c.place, c.listed, s.at<uint8_t>(o_hs), kp * 2, s.at<float>(o_sh), s.at<float>(o_sw),
                up, top, fixed, v0 + cols >= V};
        const int rc = dv ? (f16 ? piece<F16, true>(b) : piece<Bf16, true>(b)) : (f16 ? piece<F16, false>(b) : piece<Bf16, false>(b));
        if (rc) return rc;
    }
    return 0;
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_hip_rl_readout_score_stats(const NtRlReadoutStatsArgs *a) {
    const char *who = "nt_hip_rl_readout_score_stats";
    if (!a) return fail(NT_E_ARG, std::string(who) + ": null args");
    if (int rc = check(who, a->hidden, a->weight, a->dtype, a->layout, a->rows, a->vocab, a->dim, a->ldh, a->ldw, a->mask_kind,
                       a->mask, a->mask_ld, a->temperature, a->tokens))
        return rc;
    if (a->rows > 0 && (!a->logp || !a->status)) return fail(NT_E_ARG, std::string(who) + ": null logp or status");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    return a->rows == 0 ? 0 : forward(a);
}

extern "C" int nt_hip_rl_readout_score_backward(const NtRlReadoutStatsGradArgs *a) {
    const char *who = "nt_hip_rl_readout_score_backward";
    if (!a) return fail(NT_E_ARG, std::string(who) + ": null args");
    if (int rc = check(who, a->hidden, a->weight, a->dtype, a->layout, a->rows, a->vocab, a->dim, a->ldh, a->ldw, a->mask_kind,
                       a->mask, a->mask_ld, a->temperature, a->tokens))
        return rc;
    if (!a->grad_hidden && !a->grad_weight) return fail(NT_E_ARG, std::string(who) + ": no gradient asked for");
    const int64_t wrow = a->layout == NT_READOUT_W_DV ? a->vocab : a->dim;
    if ((a->grad_hidden && (a->grad_hidden_ld < a->dim || reinterpret_cast<uintptr_t>(a->grad_hidden) % 2)) ||
        (a->grad_weight && (a->grad_weight_ld < wrow || reinterpret_cast<uintptr_t>(a->grad_weight) % 2)))
        return fail(NT_E_ARG, std::string(who) + ": a gradient's row stride is under its row, or it is unaligned");
    if (a->rows > 0 && (!a->lse_base || !a->lse_rest || (a->g_entropy && !a->entropy)))
        return fail(NT_E_ARG, std::string(who) + ": null lse_base or lse_rest, or g_entropy without the entropy");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    return backward(a);
}
