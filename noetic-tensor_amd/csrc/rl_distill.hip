// nt_hip_rl_distill and nt_hip_rl_distill_backward: a row's divergence from a teacher's listed tokens, and its
// gradient.
//
// Forward: a workgroup (several a row where rows are few) streams the logits once. A bitmap in LDS, a bit a column,
// says which columns the list holds, and finds an id listed twice: the stream sums what is off the list, relative to a
// maximum off the list (next to that of a listed token its exponentials could all be 0, and the whole less the listed
// part would lose what is left to the rounding of the whole), and the listed ones join it in f64. Exponentials of the
// stream are f32, a lane's sum f64 (LaneSums). HBM bounds it: 4096 x 128256 bf16 163 us, 6.4 TB/s. With an additive mask z is f64
// throughout, as it is for the listed tokens (FarSum).
// A divergence is a small difference of large sums, so it is taken as one of its second order: with
// d = ln q - ln w, sum w (-d) = sum w (e^d - 1 - d) over a whole distribution (sum q = sum w = 1), whose terms
// are all positive and whose derivative by an error of ln q, sum (q - w), vanishes. The f32
// exponentials' error then does not reach it.
//
// Backward: every column's gradient is its exponential times one factor of the row, both relative to a maximum off the list
// (relative to a listed token's the exponentials could be 0 and the factor past f32), written as it streams
// by; then the listed ones, in f64 and rounded once, are written over it (after a barrier, by the same workgroup).
// 4096 x 128256 bf16, one row in 16 without an upstream gradient: 408 us, 5.0 TB/s of reads and writes, where a plain copy reaches 4.7.
#include <algorithm>

#include "nt_exp64.hpp"
#include "nt_rows.hpp"
#include "nt_rowsum.hpp"

namespace nt {
namespace {

constexpr int kDistillThreads = 256;
constexpr int kDistillWaves = kDistillThreads / kWave;
constexpr int kDistillAhead = 4;              // chunks a wave loads ahead
constexpr int kMaxListed = 1024;
constexpr int kMapChunks = 512;               // chunks a workgroup's bitmap covers: 2^18 columns, 32 KiB

struct DistillRec {
    double R, a;     // sum over the piece's columns off the list, relative to a (-inf: none is allowed)
    int64_t bad;     // an id outside the vocabulary, or one listed twice
};

struct DistillP {
    const void *x, *mask;
    int64_t V, ld;
    MaskMap mm;
    double c, low;      // exponent scale of a value: log2(e) / T (none, u8) or log2(e) (f32 mask); -1100 / c
    float c32;
    double inv_t;       // 1 / T
    double unit;        // z of one unit of value: 1 / T, or 1 with an f32 mask
    int nc, segs, per;
    int k, tail;
    const int32_t *ids;
    const float *teacher;
    float *loss;
    double *stats;
    uint8_t *status;
    DistillRec *rec;    // segs > 1
    // backward
    const float *g;
    void *grad;
    int64_t gld;
};

// A tempered logit under an additive mask. In f64: a mask may lower a whole row so far (-1e9) that an f32 step is no small part
// of its logits' differences, and the sums and the listed tokens have to be of the same values.
__device__ __forceinline__ double tempered64(const DistillP &p, float x, float m) { return fma(double(x), p.inv_t, double(m)); }

// The value of one listed token (see c) in f64, -inf where it is excluded.
template <int DT, int MK>
__device__ __forceinline__ double listed_value(const DistillP &p, const void *xrow, const void *mrow, int64_t v) {
    float x;
    if constexpr (DT == NT_F32) x = static_cast<const float *>(xrow)[v];
    else x = widen16<DT>(uint32_t(static_cast<const uint16_t *>(xrow)[v]));
    if constexpr (MK == NT_MASK_U8) {
        if (static_cast<const uint8_t *>(mrow)[v] == 0) return -INFINITY;
    } else if constexpr (MK == NT_MASK_F32) {
        const double z = tempered64(p, x, static_cast<const float *>(mrow)[v]);
        return fabs(z) < FarSum::kPast ? z : z * INFINITY;  // (past f32, as in the sums: infinite; a NaN stays one)
    }
    return double(x);
}

// A sum over the workgroup in f64; every thread gets it. `s` holds a value per wave.
__device__ __forceinline__ double group_sum_d(double v, double *s) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) s[threadIdx.x / kWave] = v;
    __syncthreads();
    double t = s[0];
    for (int w = 1; w < kDistillWaves; w++) t += s[w];
    return t;
}

// A maximum over the workgroup, likewise.
__device__ __forceinline__ double group_max_d(double v, double *s) {
    v = wave_max_d(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) s[threadIdx.x / kWave] = v;
    __syncthreads();
    double t = s[0];
    for (int w = 1; w < kDistillWaves; w++) t = fmax(t, s[w]);
    return t;
}

// Two f32 in eight bytes.
__device__ __forceinline__ double two_floats(float a, float b) {
    return __longlong_as_double(int64_t((uint64_t(__float_as_uint(a)) << 32) | __float_as_uint(b)));
}
__device__ __forceinline__ float first_float(double v) { return __uint_as_float(uint32_t(uint64_t(__double_as_longlong(v)) >> 32)); }
__device__ __forceinline__ float second_float(double v) { return __uint_as_float(uint32_t(uint64_t(__double_as_longlong(v)))); }

// A row's loss, statistics and status from its merged sums. The whole workgroup.
template <int DT, int MK>
__device__ void distill_finish(const DistillP &p, int64_t row, const DistillRec &r, double *s) {
    const void *xrow = static_cast<const char *>(p.x) + row * p.ld * Elem<DT>::kBytes;
    const void *mrow = nullptr;
    if constexpr (MK != NT_MASK_NONE) mrow = static_cast<const char *>(p.mask) + mask_row_at(p.mm, row) * MaskWords<MK>::kBytes;
    const int32_t *ids = p.ids + row * p.k;
    const float *teacher = p.teacher + row * p.k;
    // What a weight's logarithm is less: the largest, a teacher's f32, and the logarithm of the sum relative to it, apart (of
    // logits that a mask lowered far enough their sum would keep the first alone).
    double most = 0.0, ln_norm = 0.0;
    if (p.tail == NT_TAIL_RENORMALIZE) {
        double t = 0.0;
        most = -INFINITY;
        for (int j = threadIdx.x; j < p.k; j += kDistillThreads) most = ids[j] >= 0 ? fmax(most, double(teacher[j])) : most;
        most = group_max_d(most, s);
        for (int j = threadIdx.x; j < p.k; j += kDistillThreads)
            if (ids[j] >= 0) t += exp(double(teacher[j]) - most);
        ln_norm = log(group_sum_d(t, s));
    }
    // the listed tokens' values (a thread's are kDistillThreads apart), and with their sum the whole row's
    constexpr int kEach = kMaxListed / kDistillThreads;
    double v[kEach], a = r.a, listed = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const int j = i * kDistillThreads + int(threadIdx.x), id = j < p.k ? ids[j] : -1;
        v[i] = id >= 0 && id < p.V ? listed_value<DT, MK>(p, xrow, mrow, id) : -INFINITY;
        a = fmax(a, v[i]);
    }
    a = group_max_d(a, s);
#pragma unroll
    for (int i = 0; i < kEach; i++)
        if (v[i] != -INFINITY) listed += exp((v[i] - a) * p.unit);  // (a NaN, or +inf less itself: a NaN)
    const double S = moved(r.R, r.a, a, p.c, p.low) + group_sum_d(listed, s), ln_s = log(S);
    int st = NT_ROW_OK;
    if (!(S == S)) st = NT_ROW_NAN;
    else if (a == -INFINITY) st = NT_ROW_NO_TOKEN;
    else if (r.bad) st = NT_ROW_BAD_TOKEN;
    double loss = 0.0, mass = 0.0, rest = 0.0;
    if (st == NT_ROW_OK) {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int j = i * kDistillThreads + int(threadIdx.x);
            if (j >= p.k || ids[j] < 0) continue;
            const double lw = (double(teacher[j]) - most) - ln_norm, w = exp(lw);
            const double lq = (v[i] - a) * p.unit - ln_s, d = lq - lw;
            mass += w;
            if (p.tail != NT_TAIL_REST) {
                if (!(w == 0.0)) loss -= w * d;
            } else if (w == 0.0) {
                loss += exp(lq);
            } else {
                loss += fabs(d) < 1.0 ? w * (expm1(d) - d) : exp(lq) - w - w * d;
            }
        }
    }
    loss = group_sum_d(loss, s);
    mass = group_sum_d(mass, s);
    if (threadIdx.x != 0) return;
    double total = mass;
    if (p.tail == NT_TAIL_REST) {
        rest = mass < 1.0 ? 1.0 - mass : 0.0;
        const double lq = r.a == -INFINITY ? -INFINITY : log(r.R) + (r.a - a) * p.unit - ln_s, q = exp(lq);
        total = mass < 1.0 ? 1.0 : mass;
        if (rest > 0.0 && r.a != -INFINITY) {
            const double d = lq - log(rest);
            loss += fabs(d) < 1.0 ? rest * (expm1(d) - d) : q - rest - rest * d;
        } else {
            // (an outcome of one side alone: the terms' sum is then over other masses than 1 and 1)
            loss += q - rest;
        }
        loss += total - 1.0;
    }
    p.loss[row] = st == NT_ROW_OK ? float(loss) : NAN;
    p.status[row] = uint8_t(st);
    double *o = p.stats + row * NT_DISTILL_STATS;
    // For the backward, off the list: the base of its exponentials (a value that f32 holds but under an additive mask), and the
    // factor of one, total q_off / R - rest / R with R relative to the base. On it: the reference of q, and total over the sum relative to that.
    const bool off = r.a != -INFINITY;
    const double held = MK == NT_MASK_F32 ? r.a : double(float(fmin(fmax(r.a, -double(FLT_MAX)), double(FLT_MAX))));
    const double base = off ? held : 0.0;
    const double factor = off ? (total * exp((r.a - a) * p.unit) / S - rest / r.R) * exp2((base - r.a) * p.c) : 0.0;
    o[0] = base;
    o[1] = two_floats(st == NT_ROW_OK ? float(factor) : NAN, float(most));
    o[2] = a;
    o[3] = st == NT_ROW_OK ? total / S : NAN;
    o[4] = ln_norm;
}

template <int DT, int MK, bool AL>
__global__ __launch_bounds__(kDistillThreads) void k_distill(DistillP p) {
    extern __shared__ uint32_t map[];
    __shared__ double red[kDistillWaves];
    __shared__ DistillRec ws[kDistillWaves];
    __shared__ int bad;
    const int64_t row = blockIdx.x / unsigned(p.segs);
    const int seg = int(blockIdx.x % unsigned(p.segs));
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const void *xrow = static_cast<const char *>(p.x) + row * p.ld * Elem<DT>::kBytes;
    const void *mrow = nullptr;
    if constexpr (MK != NT_MASK_NONE) mrow = static_cast<const char *>(p.mask) + mask_row_at(p.mm, row) * MaskWords<MK>::kBytes;
    const int c0 = seg * p.per, c1 = min(p.nc, c0 + p.per);

    for (int i = threadIdx.x; i < (c1 - c0) * (kChunk / 32); i += kDistillThreads) map[i] = 0;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < p.k; j += kDistillThreads) {
        const int32_t id = p.ids[row * p.k + j];
        if (id < -1 || id >= p.V) {
            bad = 1;
        } else if (id >= c0 * kChunk && id - c0 * kChunk < (c1 - c0) * kChunk) {
            const uint32_t at = uint32_t(id - c0 * kChunk), bit = 1u << (at % 32);
            if (atomicOr(&map[at / 32], bit) & bit) bad = 1;
        }
    }
    __syncthreads();
    const uint8_t *bytes = reinterpret_cast<const uint8_t *>(map);

    const RowLoad<DT, MK, AL> in(xrow, mrow, p.V, p.nc);
    std::conditional_t<MK == NT_MASK_F32, FarSum, LaneSums> sum;
    Raw<DT, MK> raw[kDistillAhead];
    auto load = [&](auto i, int ch) { in.load(raw[i.value], ch, lane, ch < c1); };
    stream<kDistillAhead>(c0 + wave, kDistillWaves, c1, load, [&](auto i, int ch, int next) {
        std::conditional_t<MK == NT_MASK_F32, double, float> v[kEpl];
        if constexpr (MK == NT_MASK_F32) {
#pragma unroll
            for (int j = 0; j < kEpl; j++) v[j] = tempered64(p, logit<DT>(raw[i.value].x, j), __uint_as_float(raw[i.value].m[j]));
        } else {
            decode_e<DT, MK, kEpl>(raw[i.value].x, raw[i.value].m, v, 1.0f, true);
        }
        in.clean(v, ch, lane);
        load(i, next);
        // bit j for column j
        uint32_t on;
        if constexpr (decltype(in)::kSplit) {
            const int at = (ch - c0) * kWave + lane / 2, shift = 4 * (lane & 1);
            on = ((bytes[at] >> shift) & 15u) | (((bytes[at + kWave / 2] >> shift) & 15u) << 4);
        } else {
            // (past the row's end a lane's own columns come after its neighbour's)
            on = uint32_t(bytes[(ch - c0) * kWave + lane]) << (AL ? 0 : min(int64_t(8), in.own(ch, lane) - in.first(ch, lane)));
        }
        if (__ballot(on != 0) != 0) {
#pragma unroll
            for (int j = 0; j < kEpl; j++) v[j] = (on >> j) & 1u ? -INFINITY : v[j];
        }
        if constexpr (MK == NT_MASK_F32) sum.add(v, p.low);
        else sum.add(v, p.c32);
    });
    const double at = sum.at(p.c, p.c32), top = wave_max_d(at);
    const double R = wave_sum_d(moved(sum.S, at, top, p.c, p.low));
    if (lane == 0) ws[wave] = DistillRec{R, top, 0};
    __syncthreads();
    DistillRec r{0.0, ws[0].a, bad};
    for (int w = 1; w < kDistillWaves; w++) r.a = fmax(r.a, ws[w].a);
    for (int w = 0; w < kDistillWaves; w++) r.R += moved(ws[w].R, ws[w].a, r.a, p.c, p.low);
    if (p.segs > 1) {
        if (threadIdx.x == 0) p.rec[row * p.segs + seg] = r;
        return;
    }
    distill_finish<DT, MK>(p, row, r, red);
}

// The rows of a launch with several workgroups a row.
template <int DT, int MK>
__global__ __launch_bounds__(kDistillThreads) void k_distill_finish(DistillP p) {
    __shared__ double red[kDistillWaves];
    const int64_t row = blockIdx.x;
    const DistillRec *rec = p.rec + row * p.segs;
    DistillRec r{0.0, -INFINITY, 0};
    for (int g = 0; g < p.segs; g++) {
        r.a = fmax(r.a, rec[g].a);
        r.bad |= rec[g].bad;
    }
    for (int g = 0; g < p.segs; g++) r.R += moved(rec[g].R, rec[g].a, r.a, p.c, p.low);
    distill_finish<DT, MK>(p, row, r, red);
}

// Two gradients in a 16-bit dtype, a in the low half, to nearest even.
template <int GDT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (GDT == NT_BF16) {
        uint32_t r;
        asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
        return r;
    } else {
        return uint32_t(__builtin_bit_cast(uint16_t, _Float16(a))) | (uint32_t(__builtin_bit_cast(uint16_t, _Float16(b))) << 16);
    }
}

template <int GDT>
__device__ __forceinline__ void store1(void *grow, int64_t e, float o) {
    if constexpr (GDT == NT_F32) static_cast<float *>(grow)[e] = o;
    else static_cast<uint16_t *>(grow)[e] = uint16_t(pack2<GDT>(o, o));
}

// 8 gradients at column e0; AL: 16-byte aligned, all inside the row.
template <int GDT, bool AL>
__device__ __forceinline__ void store8(void *grow, int64_t e0, int64_t V, const float *o) {
    if (e0 >= V) return;
    if (AL || e0 + kEpl <= V) {
        if constexpr (GDT == NT_F32) {
            auto *d = reinterpret_cast<u32x4_f32 *>(static_cast<float *>(grow) + e0);
            if constexpr (AL) {
                auto *q = reinterpret_cast<v4u *>(d);
                __builtin_nontemporal_store(v4u{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])}, q);
                __builtin_nontemporal_store(v4u{__float_as_uint(o[4]), __float_as_uint(o[5]), __float_as_uint(o[6]), __float_as_uint(o[7])}, q + 1);
            } else {
                d[0] = u32x4_f32{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])};
                d[1] = u32x4_f32{__float_as_uint(o[4]), __float_as_uint(o[5]), __float_as_uint(o[6]), __float_as_uint(o[7])};
            }
        } else {
            const uint32_t w0 = pack2<GDT>(o[0], o[1]), w1 = pack2<GDT>(o[2], o[3]), w2 = pack2<GDT>(o[4], o[5]), w3 = pack2<GDT>(o[6], o[7]);
            if constexpr (AL) __builtin_nontemporal_store(v4u{w0, w1, w2, w3}, reinterpret_cast<v4u *>(static_cast<uint16_t *>(grow) + e0));
            else *reinterpret_cast<u32x4_f16 *>(static_cast<uint16_t *>(grow) + e0) = u32x4_f16{w0, w1, w2, w3};
        }
        return;
    }
    for (int j = 0; j < kEpl && e0 + j < V; j++) store1<GDT>(grow, e0 + j, o[j]);
}

// 4 gradients at column e, aligned, all inside the row or none.
template <int GDT>
__device__ __forceinline__ void store4(void *grow, int64_t e, int64_t V, const float *o) {
    if (e >= V) return;
    if constexpr (GDT == NT_F32) {
        __builtin_nontemporal_store(v4u{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])},
                                    reinterpret_cast<v4u *>(static_cast<float *>(grow) + e));
    } else {
        typedef uint32_t v2u __attribute__((ext_vector_type(2)));
        __builtin_nontemporal_store(v2u{pack2<GDT>(o[0], o[1]), pack2<GDT>(o[2], o[3])},
                                    reinterpret_cast<v2u *>(static_cast<uint16_t *>(grow) + e));
    }
}

template <int DT, int MK, int GDT, bool AL>
__global__ __launch_bounds__(kDistillThreads) void k_distill_grad(DistillP p) {
    const int64_t row = blockIdx.x / unsigned(p.segs);
    const int seg = int(blockIdx.x % unsigned(p.segs));
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const void *xrow = static_cast<const char *>(p.x) + row * p.ld * Elem<DT>::kBytes;
    const void *mrow = nullptr;
    if constexpr (MK != NT_MASK_NONE) mrow = static_cast<const char *>(p.mask) + mask_row_at(p.mm, row) * MaskWords<MK>::kBytes;
    void *grow = static_cast<char *>(p.grad) + row * p.gld * (GDT == NT_F32 ? 4 : 2);
    const int c0 = seg * p.per, c1 = min(p.nc, c0 + p.per);
    const float g = p.g[row];
    if (g == 0.0f) {
        const float zero[kEpl] = {};
        for (int ch = c0 + wave; ch < c1; ch += kDistillWaves) store8<GDT, AL>(grow, int64_t(ch) * kChunk + lane * kEpl, p.V, zero);
        return;
    }
    const double *st = p.stats + row * NT_DISTILL_STATS;
    const double scale = double(g) * p.inv_t;
    const double far = st[0];
    const float base = float(far), factor = float(scale * double(first_float(st[1])));
    const double most = double(second_float(st[1]));
    const RowLoad<DT, MK, AL> in(xrow, mrow, p.V, p.nc);
    Raw<DT, MK> raw[kDistillAhead];
    auto load = [&](auto i, int ch) { in.load(raw[i.value], ch, lane, ch < c1); };
    stream<kDistillAhead>(c0 + wave, kDistillWaves, c1, load, [&](auto i, int ch, int next) {
        float v[kEpl], o[kEpl];
        if constexpr (MK == NT_MASK_F32) {
#pragma unroll
            for (int j = 0; j < kEpl; j++)
                v[j] = float(tempered64(p, logit<DT>(raw[i.value].x, j), __uint_as_float(raw[i.value].m[j])) - far);
        } else {
            decode_e<DT, MK, kEpl>(raw[i.value].x, raw[i.value].m, v, 1.0f, true);
#pragma unroll
            for (int j = 0; j < kEpl; j++) v[j] -= base;
        }
        load(i, next);
#pragma unroll
        for (int j = 0; j < kEpl; j++) o[j] = fmaf(exp2_hw(v[j] * p.c32), factor, 0.0f);
        if constexpr (decltype(in)::kSplit) {
            store4<GDT>(grow, in.col(ch, lane, 0), p.V, o);
            store4<GDT>(grow, in.col(ch, lane, 4), p.V, o + 4);
        } else if (AL || in.first(ch, lane) == in.own(ch, lane)) {
            store8<GDT, AL>(grow, in.own(ch, lane), p.V, o);
        } else {
            for (int j = 0; j < kEpl; j++)
                if (in.mine(ch, lane, j)) store1<GDT>(grow, in.first(ch, lane) + j, o[j]);
        }
    });
    // the listed columns of this piece, over what was just written there
    wait_vmcnt<0>();
    __syncthreads();
    for (int j = threadIdx.x; j < p.k; j += kDistillThreads) {
        const int64_t id = p.ids[row * p.k + j];
        if (id < int64_t(c0) * kChunk || id >= int64_t(c1) * kChunk || id >= p.V) continue;
        const double w = exp((double(p.teacher[row * p.k + j]) - most) - st[4]);
        const double q = exp((listed_value<DT, MK>(p, xrow, mrow, id) - st[2]) * p.unit) * st[3];  // (times the total)
        const double o = scale * (q - w);
        if constexpr (GDT == NT_F32) {
            static_cast<float *>(grow)[id] = float(o);
        } else if constexpr (GDT == NT_F16) {
            static_cast<uint16_t *>(grow)[id] = __builtin_bit_cast(uint16_t, _Float16(o));
        } else {
            // (to f32 with the last bit odd where that was not exact, so that the second rounding is the only one)
            float f = float(o);
            if (double(f) != o && f == f) {
                const uint32_t b = __float_as_uint(f);
                const bool past = fabs(double(f)) > fabs(o);
                f = __uint_as_float((past ? b - 1 : b) | 1u);
            }
            static_cast<uint16_t *>(grow)[id] = uint16_t(pack2<GDT>(f, f));
        }
    }
}

// Pieces of a row for `rows` rows of nc chunks: up to `groups` workgroups, of `least` chunks or more and at most kMapChunks.
void cut_rows(int64_t rows, int nc, int64_t groups, int least, int *segs, int *per) {
    const int64_t few = std::max<int64_t>(1, std::min<int64_t>(groups / std::max<int64_t>(rows, 1), nc / least));
    *per = int(std::min<int64_t>(kMapChunks, (nc + few - 1) / few));
    *segs = (nc + *per - 1) / *per;
}

int distill_check(const char *who, int64_t rows, int64_t vocab, int64_t k, double temperature) {
    if (int rc = check_scale(temperature)) return rc;
    if (k < 1 || k > kMaxListed)
        return fail(NT_E_ARG, std::string(who) + ": " + std::to_string(k) + " listed tokens a row (1 to " + std::to_string(kMaxListed) + ")");
    // (a launch holds fewer than 2^32 threads; columns are counted in 32 bits)
    if (vocab > 0x7fffffffLL - 16 * kChunk || rows > 0xffffffLL || rows * ((vocab + (int64_t(1) << 18) - 1) >> 18) > 0xffffffLL)
        return fail(NT_E_ARG, std::string(who) + ": rows past 2^24 (of 2^18 columns) or vocab past 2^31");
    return 0;
}

template <class F>
void by_dtype(int dtype, int mk, F &&f) {
    auto by_mk = [&](auto dt) {
        if (mk == NT_MASK_U8) f(dt, std::integral_constant<int, NT_MASK_U8>{});
        else if (mk == NT_MASK_F32) f(dt, std::integral_constant<int, NT_MASK_F32>{});
        else f(dt, std::integral_constant<int, NT_MASK_NONE>{});
    };
    if (dtype == NT_F32) by_mk(std::integral_constant<int, NT_F32>{});
    else if (dtype == NT_BF16) by_mk(std::integral_constant<int, NT_BF16>{});
    else by_mk(std::integral_constant<int, NT_F16>{});
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int nt_hip_rl_distill(const NtRlDistillArgs *a) {
    const char *who = "nt_hip_rl_distill";
    if (!a) return fail(NT_E_ARG, std::string(who) + ": null args");
    if (int rc = check_rows(a->rows, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, a->mask_ld, who)) return rc;
    MaskMap mm;
    if (int rc = mask_map(a->mask_rows, a->rows, a->vocab, a->mask_kind, a->mask_ld, who, &mm)) return rc;
    if (int rc = distill_check(who, a->rows, a->vocab, a->k, a->temperature)) return rc;
    if (a->tail < NT_TAIL_REST || a->tail > NT_TAIL_RENORMALIZE)
        return fail(NT_E_ARG, std::string(who) + ": tail " + std::to_string(a->tail));
    if (!a->logits || !a->ids || !a->teacher_logp || !a->loss || !a->stats || !a->status)
        return fail(NT_E_ARG, std::string(who) + ": null logits, ids, teacher_logp or outputs");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    if (a->rows == 0) return 0;
    DistillP p{};
    p.x = a->logits;
    p.mask = a->mask;
    p.V = a->vocab;
    p.ld = a->ld;
    p.mm = mm;
    p.c = a->mask_kind == NT_MASK_F32 ? kLog2e64 : kLog2e64 / a->temperature;
    p.c32 = float(p.c);
    p.low = -1100.0 / p.c;
    p.inv_t = 1.0 / a->temperature;
    p.unit = a->mask_kind == NT_MASK_F32 ? 1.0 : p.inv_t;
    p.nc = int((a->vocab + kChunk - 1) / kChunk);
    // (the finishing launch is worth 120 chunks: 128 rows of 32000 bf16 16.4 us in one piece, 18.9 in two; 1 of 128256 19.7 and 19.1)
    cut_rows(a->rows, p.nc, 512, 120, &p.segs, &p.per);
    p.k = int(a->k);
    p.tail = a->tail;
    p.ids = a->ids;
    p.teacher = a->teacher_logp;
    p.loss = a->loss;
    p.stats = a->stats;
    p.status = a->status;
    void *ws = nullptr;
    if (p.segs > 1) {
        const size_t need = sizeof(DistillRec) * size_t(a->rows) * size_t(p.segs);
        bool cap = false;
        if (int rc = stream_capturing(&cap)) return rc;
        if (cap && need >= size_t(1) << 20)
            return fail(NT_E_UNSUPPORTED, std::string(who) + ": a workspace of " + std::to_string(need) +
                                              " bytes under stream capture (less than 1 MiB)");
        if (int rc = scratch_alloc(need, &ws)) return rc;
        p.rec = static_cast<DistillRec *>(ws);
    }
    const bool al = aligned_rows(a->logits, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, mm) && a->vocab * 4 <= 0x7fffffffLL;
    hipStream_t s = ctx().stream;
    by_dtype(a->dtype, a->mask_kind, [&](auto dt, auto mk) {
        constexpr int DT = decltype(dt)::value, MK = decltype(mk)::value;
        const dim3 grid(unsigned(a->rows * p.segs));
        const size_t lds = size_t(p.per) * (kChunk / 8);
        if (al) hipLaunchKernelGGL((k_distill<DT, MK, true>), grid, dim3(kDistillThreads), lds, s, p);
        else hipLaunchKernelGGL((k_distill<DT, MK, false>), grid, dim3(kDistillThreads), lds, s, p);
        if (p.segs > 1) hipLaunchKernelGGL((k_distill_finish<DT, MK>), dim3(unsigned(a->rows)), dim3(kDistillThreads), 0, s, p);
    });
    const int rc = launched(who);
    const int rc2 = scratch_release(ws);
    return rc ? rc : rc2;
}

int nt_hip_rl_distill_backward(const NtRlDistillGradArgs *a) {
    const char *who = "nt_hip_rl_distill_backward";
    if (!a) return fail(NT_E_ARG, std::string(who) + ": null args");
    if (int rc = check_rows(a->rows, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, a->mask_ld, who)) return rc;
    MaskMap mm;
    if (int rc = mask_map(a->mask_rows, a->rows, a->vocab, a->mask_kind, a->mask_ld, who, &mm)) return rc;
    if (int rc = distill_check(who, a->rows, a->vocab, a->k, a->temperature)) return rc;
    if (!a->logits || !a->ids || !a->teacher_logp || !a->stats || !a->g_loss || !a->grad)
        return fail(NT_E_ARG, std::string(who) + ": null logits, ids, teacher_logp, stats, g_loss or grad");
    if (a->grad_dtype != NT_F32 && a->grad_dtype != NT_BF16 && a->grad_dtype != NT_F16)
        return fail(NT_E_ARG, std::string(who) + ": grad dtype " + std::to_string(a->grad_dtype));
    if (a->grad_ld < a->vocab) return fail(NT_E_ARG, std::string(who) + ": grad_ld < vocab");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    if (a->rows == 0) return 0;
    DistillP p{};
    p.x = a->logits;
    p.mask = a->mask;
    p.V = a->vocab;
    p.ld = a->ld;
    p.mm = mm;
    p.c = a->mask_kind == NT_MASK_F32 ? kLog2e64 : kLog2e64 / a->temperature;
    p.c32 = float(p.c);
    p.low = -1100.0 / p.c;
    p.inv_t = 1.0 / a->temperature;
    p.unit = a->mask_kind == NT_MASK_F32 ? 1.0 : p.inv_t;
    p.nc = int((a->vocab + kChunk - 1) / kChunk);
    cut_rows(a->rows, p.nc, 4096, kDistillWaves, &p.segs, &p.per);
    p.k = int(a->k);
    p.ids = a->ids;
    p.teacher = a->teacher_logp;
    p.stats = const_cast<double *>(a->stats);
    p.g = a->g_loss;
    p.grad = a->grad;
    p.gld = a->grad_ld;
    const bool al = aligned_rows(a->logits, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, mm) && a->vocab * 4 <= 0x7fffffffLL &&
                    a->grad_ld % kEpl == 0 && reinterpret_cast<uintptr_t>(a->grad) % 16 == 0;
    hipStream_t s = ctx().stream;
    by_dtype(a->dtype, a->mask_kind, [&](auto dt, auto mk) {
        constexpr int DT = decltype(dt)::value, MK = decltype(mk)::value;
        const dim3 grid(unsigned(a->rows * p.segs));
        auto launch = [&](auto gdt) {
            constexpr int GDT = decltype(gdt)::value;
            if (al) hipLaunchKernelGGL((k_distill_grad<DT, MK, GDT, true>), grid, dim3(kDistillThreads), 0, s, p);
            else hipLaunchKernelGGL((k_distill_grad<DT, MK, GDT, false>), grid, dim3(kDistillThreads), 0, s, p);
        };
        if (a->grad_dtype == NT_F32) launch(std::integral_constant<int, NT_F32>{});
        else if (a->grad_dtype == NT_BF16) launch(std::integral_constant<int, NT_BF16>{});
        else launch(std::integral_constant<int, NT_F16>{});
    });
    return launched(who);
}

}  // extern "C"
