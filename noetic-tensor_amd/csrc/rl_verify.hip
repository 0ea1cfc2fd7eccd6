// nt_hip_rl_verify_drafted: drafted tokens against the target's distribution, and the token drawn in place of the
// first one refused.
//
// Which tokens come out is decided by comparisons of a uniform with sums over the vocabulary, and a flat row of
// 128256 tokens has one every 8e-6 of the unit interval: sums within 1e-7, as f32 exponentials give, would put one
// draw in a hundred on a token's neighbour. The row that a token is drawn from is therefore summed in f64 with f64
// exponentials (exp2_64), and so is every row where there are few. Of many rows, f32 exponentials say whether
// a draft is accepted, unless u q / p lies within their error of 1 (one draft in 50000): such a row is summed
// again in f64.
//
//  * k_verify_rows: the log-sum-exps of a position's target row and draft row, in one pass over both (and
//    their mask, read once for the two). Few positions: several workgroups each, in f64 (kWide). Many: one each
//    (kNarrow), bound by the rows' bytes; they go by position first and sequence second, each judges its
//    draft, and one whose sequence has had a draft refused before it leaves at once (what it would compute is not
//    used, so whether it saw the refusal in time changes no result).
//  * k_verify_sums (kNarrow): the first refused position, any row that was too close to call, and the f64
//    log-sum-exps of the rows at that position, over several workgroups a sequence.
//  * k_verify_draw: r = max(p - q, 0) of that position summed by chunks of 512 columns, over several workgroups.
//  * k_verify_pick: one wave a sequence finds the chunk that holds u sum r, and in it the token.
#include <algorithm>

#include "nt_exp64.hpp"
#include "nt_rows.hpp"

namespace nt {
namespace {

constexpr int kRowThreads = 512;              // k_verify_rows
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kDrawThreads = 256;             // k_verify_sums, k_verify_draw
constexpr int kDrawWaves = kDrawThreads / kWave;
constexpr int kMaxDrafts = 127;
constexpr int kVerifySegs = 64;               // workgroups a position or a drawn row, at most (one lane each)
// How k_verify_rows sums: in f64, in f32 (see judge), or in f32 with the first largest value.
enum { kWide, kNarrow, kGreedy };
// What f32 sums may be off in a draft's log2 ratio: each of the two log-sum-exps by 6e-6 (exponentials within 2^-23 and
// |t| 3 2^-24 ln 2 of arguments t, |t| < 24 where it matters; the lanes' references move a few times), and with an additive
// mask, whose values are f32 tempered logits, by half an f32 step of the largest of each.
constexpr double kClose32 = 2e-5;

// What a workgroup found in its piece of a position's rows: sums S relative to the reference a (value space,
// as decoded below), of the target and of the drafter; greedy: the target's first largest value and its place.
struct VerifyRec {
    double S, Sd;
    float a, ad;
    int32_t at;
    float top;
};

// What becomes of a position, from its sums: accepted, drawn from, too close for f32, or a row status that ends
// the sequence (kBad + NT_ROW_*).
enum { kAccept = 0, kDraw = 1, kTooClose = 2, kBad = 3 };
struct Verdict {
    int what;
    int32_t at;     // greedy: the first largest
    double lp, lq;  // log-sum-exps in log2 units (lq 0 without draft logits)
    double logp;    // ln p of the draft
};

// What is drawn from at a sequence's last position: p's and q's log-sum-exps (log2 units) and how.
enum { kDrawNone = -1, kDrawTarget = 0, kDrawRest = 1, kDrawOthers = 2 };
struct VerifyPick {
    double lp, lq;
    int32_t pos, mode;
};

struct VerifyP {
    const void *x, *y, *mask;
    int64_t V, ld, ldy;
    MaskMap mm;
    double c, cd;             // log2(e) / T of the target and the drafter
    double inv_t, inv_td;     // 1 / T
    float cap, capd;          // 2^500 in value units
    float s32, sd32;          // log2 units of one unit of value
    int nc;                   // chunks of a row
    int seqs, K;
    int segs, per;            // workgroups a position, chunks each
    int dsegs, dper;          // workgroups a drawn row, chunks each
    const int32_t *tokens, *lengths;
    const double *u;
    int32_t *ids, *accepted;
    float *logp;
    uint8_t *status;
    VerifyRec *rec;           // [seqs][K + 1][segs], or of the drawn rows [seqs][dsegs]
    Verdict *verdict;         // one workgroup a position: [seqs][K + 1]
    double *sums;             // [seqs][nc]
    VerifyPick *pick;         // [seqs]
    int32_t *first;           // one workgroup a position: [seqs] the first one known to be refused
};

// The larger, a NaN if there is one.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max8_nan(const float v[kEpl]) {
    return max_nan(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])), max_nan(max_nan(v[4], v[5]), max_nan(v[6], v[7])));
}

// One lane's logits and what stands for them: value v (a logit, -inf where a u8 mask excludes it; with an
// additive mask the f32 nearest to the tempered logit, kGreedy: the f32 sum), and in f64 the exponent
// v c - A, of an additive mask x c + m log2(e) - A.
template <int DT, int MK, int HOW>
struct Lane8 {
    float v[kEpl];
    float x[MK == NT_MASK_F32 ? kEpl : 1], m[MK == NT_MASK_F32 ? kEpl : 1];

    __device__ __forceinline__ void decode(const uint32_t *xw, const uint32_t *mw, double inv_t) {
        if constexpr (MK == NT_MASK_F32) {
#pragma unroll
            for (int j = 0; j < kEpl; j++) {
                x[j] = logit<DT>(xw, j);
                m[j] = __uint_as_float(mw[j]);
                v[j] = HOW == kGreedy ? x[j] + m[j] : float(fma(double(x[j]), inv_t, double(m[j])));
            }
        } else {
            decode_words<DT, MK>(xw, mw, v, 1.0f, true);
        }
    }
    __device__ __forceinline__ double arg(int j, double c, double neg_a) const {
        if constexpr (MK == NT_MASK_F32) return fma(double(x[j]), c, fma(double(m[j]), kLog2e64, neg_a));
        else return fma(double(v[j]), c, neg_a);
    }
};

// The log2 units of one unit of value.
template <int MK>
__device__ __forceinline__ double value_scale(double c) {
    return MK == NT_MASK_F32 ? kLog2e64 : c;
}

// A lane's f64 sum of 2^(arg) relative to its reference: the first maximum it met, moved only where a later logit lies
// 2^500 above it, which f64 holds and logits hardly reach.
struct LaneSum {
    double S = 0.0, neg_a = 0.0;
    float ref = -INFINITY, lim = -INFINITY;

    template <int DT, int MK, int H>
    __device__ __forceinline__ void add(const Lane8<DT, MK, H> &l, double c, float cap) {
        const float top = max8_nan(l.v);
        if (!(top <= lim)) {
            if (top < INFINITY) {
                const double s = value_scale<MK>(c);
                if (ref != -INFINITY) S *= exp2_64((double(ref) - double(top)) * s);
                ref = top;
                lim = top + cap;
                neg_a = -double(ref) * s;
            } else {
                S = NAN;
            }
        }
        double w[kEpl];
#pragma unroll
        for (int j = 0; j < kEpl; j++) w[j] = exp2_64(l.arg(j, c, neg_a));
        S += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    }
};

// The same of f32 exponentials, relative to the lane's maximum so far. A NaN or +inf leaves a NaN.
struct LaneSum32 {
    double S = 0.0;
    float ref = -INFINITY;

    __device__ __forceinline__ void add(const float v[kEpl], float scale) {
        const float top = fmaxf(ref, max8(v)), sh = top == -INFINITY ? 0.0f : top;
        float w[kEpl];
#pragma unroll
        for (int j = 0; j < kEpl; j++) w[j] = exp2_hw((v[j] - sh) * scale);
        S = fma(S, double(exp2_hw((ref - sh) * scale)), double(tree8(w)));
        ref = top;
    }
};

// S relative to a, moved to the reference at (at least a).
__device__ __forceinline__ double moved(double S, float a, float at, double scale) {
    return a == -INFINITY || a == at ? S : S * exp2_64((double(a) - double(at)) * scale);
}

// The tempered logit of one token in log2 units, -inf where it is excluded.
template <int DT, int MK>
__device__ __forceinline__ double token_arg(const void *xrow, const void *mrow, int64_t v, double c) {
    float x;
    if constexpr (DT == NT_F32) x = static_cast<const float *>(xrow)[v];
    else x = widen16<DT>(uint32_t(static_cast<const uint16_t *>(xrow)[v]));
    if constexpr (MK == NT_MASK_U8) {
        if (static_cast<const uint8_t *>(mrow)[v] == 0) return -INFINITY;
    } else if constexpr (MK == NT_MASK_F32) {
        return fma(double(x), c, double(static_cast<const float *>(mrow)[v]) * kLog2e64);
    }
    return double(x) * c;
}

template <int DT, int MK>
struct VerifyRows {
    const void *x, *y, *m;
    __device__ __forceinline__ VerifyRows(const VerifyP &p, int64_t s, int64_t t) {
        const int64_t row = s * (p.K + 1) + t;
        x = static_cast<const char *>(p.x) + row * p.ld * Elem<DT>::kBytes;
        y = p.y && t < p.K ? static_cast<const char *>(p.y) + (s * p.K + t) * p.ldy * Elem<DT>::kBytes : nullptr;
        m = nullptr;
        if constexpr (MK != NT_MASK_NONE)
            m = static_cast<const char *>(p.mask) + mask_row_at(p.mm, row) * MaskWords<MK>::kBytes;
    }
};

__device__ __forceinline__ int drafts_of(const VerifyP &p, int64_t s) { return p.lengths ? p.lengths[s] : p.K; }

// Position t of a sequence of n drafts, from its merged sums.
template <int DT, int MK, int HOW>
__device__ __forceinline__ Verdict judge(const VerifyP &p, int64_t s, int t, int n, const VerifyRec &r) {
    Verdict d{kDraw, r.at, 0.0, 0.0, 0.0};
    const VerifyRows<DT, MK> rows(p, s, t);
    if (!(r.S == r.S)) {
        d.what = kBad + NT_ROW_NAN;
        return d;
    }
    if (r.a == -INFINITY) {
        d.what = kBad + NT_ROW_NO_TOKEN;
        return d;
    }
    d.lp = double(r.a) * value_scale<MK>(p.c) + log2(r.S);
    if (t >= n) return d;
    const int32_t tok = p.tokens[s * p.K + t];
    if (tok < 0 || tok >= p.V) {
        d.what = kBad + NT_ROW_BAD_TOKEN;
        return d;
    }
    const double l = token_arg<DT, MK>(rows.x, rows.m, tok, p.c) - d.lp;
    d.logp = l * kLn2;
    if constexpr (HOW == kGreedy) {
        d.what = r.at == tok ? kAccept : kDraw;
        return d;
    }
    double lq = 0.0;
    if (rows.y) {
        if (!(r.Sd == r.Sd)) {
            d.what = kBad + NT_ROW_NAN;
            return d;
        }
        if (r.ad == -INFINITY) {
            d.what = kBad + NT_ROW_NO_TOKEN;
            return d;
        }
        d.lq = double(r.ad) * value_scale<MK>(p.cd) + log2(r.Sd);
        lq = token_arg<DT, MK>(rows.y, rows.m, tok, p.cd) - d.lq;
    }
    // u q < p: a draft that the drafter gives nothing is accepted where the target gives it something, and one
    // that the target gives nothing never is (inf - inf compares false)
    const double u = p.u[s * (p.K + 1) + t];
    d.what = u < exp2(l - lq) ? kAccept : kDraw;
    if constexpr (HOW == kNarrow) {
        const double near = kClose32 + (MK == NT_MASK_F32 ? 0x1p-23 * kLog2e64 * (fabs(double(r.a)) + (rows.y ? fabs(double(r.ad)) : 0.0)) : 0.0);
        if (fabs(log2(u) - (l - lq)) < near) d.what = kTooClose;
    }
    return d;
}

// A wave's sums from its lanes'.
template <int MK, class L>
__device__ __forceinline__ VerifyRec wave_rec(const VerifyP &p, const L &x, const L &y) {
    VerifyRec r{0.0, 0.0, -INFINITY, -INFINITY, 0, 0.0f};
    r.a = wave_max(x.ref);
    r.S = wave_sum_d(moved(x.S, x.ref, r.a, value_scale<MK>(p.c)));
    r.ad = wave_max(y.ref);
    r.Sd = wave_sum_d(moved(y.S, y.ref, r.ad, value_scale<MK>(p.cd)));
    return r;
}

// The waves' sums in order.
template <int MK, int WAVES>
__device__ __forceinline__ VerifyRec waves_rec(const VerifyP &p, const VerifyRec *ws) {
    VerifyRec r = ws[0];
    for (int w = 1; w < WAVES; w++) {
        r.a = fmaxf(r.a, ws[w].a);
        r.ad = fmaxf(r.ad, ws[w].ad);
        if (ws[w].top > r.top || (ws[w].top == r.top && ws[w].at < r.at)) {
            r.top = ws[w].top;
            r.at = ws[w].at;
        }
    }
    r.S = r.Sd = 0.0;
    for (int w = 0; w < WAVES; w++) {
        r.S += moved(ws[w].S, ws[w].a, r.a, value_scale<MK>(p.c));
        r.Sd += moved(ws[w].Sd, ws[w].ad, r.ad, value_scale<MK>(p.cd));
    }
    return r;
}

// Chunks c, c + step, .. below c1 of a position's rows (BOTH: and the drafter's) into the lane's sums.
template <int DT, int MK, bool AL, int HOW, class L>
__device__ __forceinline__ void add_rows(const VerifyP &p, const VerifyRows<DT, MK> &rows, bool both, int c, int step, int c1,
                                         int lane, L &sx, L &sy, float *top, int32_t *at) {
    Raw<DT, MK> rx[2];
    Raw<DT, NT_MASK_NONE> ry[2];
    auto load = [&](int k, int ch) {
        if (ch >= c1) return;
        const int64_t e0 = int64_t(ch) * kChunk + lane * kEpl;
        load_raw<DT, MK, AL>(rx[k], rows.x, rows.m, e0, p.V);
        if (both) load_raw<DT, NT_MASK_NONE, AL>(ry[k], rows.y, nullptr, e0, p.V);
    };
    auto take = [&](int k, int ch, int next) {
        Lane8<DT, MK, HOW> lx, ly;
        lx.decode(rx[k].x, rx[k].m, p.inv_t);
        if (both) ly.decode(ry[k].x, rx[k].m, p.inv_td);
        load(k, next);
        if constexpr (HOW == kGreedy) {
#pragma unroll
            for (int j = 0; j < kEpl; j++) {
                const bool up = lx.v[j] > *top;
                *top = up ? lx.v[j] : *top;
                *at = up ? ch * kChunk + lane * kEpl + j : *at;
            }
        }
        if constexpr (HOW == kWide) {
            sx.add(lx, p.c, p.cap);
            if (both) sy.add(ly, p.cd, p.capd);
        } else {
            sx.add(lx.v, p.s32);
            if (both) sy.add(ly.v, p.sd32);
        }
    };
    load(0, c);
    load(1, c + step);
    for (; c < c1; c += 2 * step) {
        take(0, c, c + 2 * step);
        if (c + step < c1) take(1, c + step, c + 3 * step);
    }
}

template <int HOW>
using Sum = std::conditional_t<HOW == kWide, LaneSum, LaneSum32>;

template <int DT, int MK, bool AL, int HOW>
__global__ __launch_bounds__(kRowThreads) void k_verify_rows(VerifyP p) {
    __shared__ VerifyRec ws[kRowWaves];
    __shared__ int leave;
    const unsigned per_t = unsigned(p.seqs) * unsigned(p.segs);
    const int t = int(blockIdx.x / per_t);
    const unsigned b = blockIdx.x % per_t;
    const int64_t s = b / unsigned(p.segs);
    const int seg = int(b % unsigned(p.segs));
    const int n = drafts_of(p, s);
    if (n < 0 || n > p.K || t > n) return;
    if (p.first) {
        if (threadIdx.x == 0)
            leave = __hip_atomic_load(&p.first[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) < t;
        __syncthreads();
        if (leave) return;
    }
    const VerifyRows<DT, MK> rows(p, s, t);
    const bool both = HOW != kGreedy && rows.y != nullptr && t < n;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const int c1 = min(p.nc, (seg + 1) * p.per);
    Sum<HOW> sx, sy;
    float top = -INFINITY;
    int32_t at = 0x7fffffff;
    add_rows<DT, MK, AL, HOW>(p, rows, both, seg * p.per + wave, kRowWaves, c1, lane, sx, sy, &top, &at);
    VerifyRec r = wave_rec<MK>(p, sx, sy);
    if constexpr (HOW == kGreedy) {
        r.top = wave_max(top);
        r.at = wave_min_i(top == r.top ? at : 0x7fffffff);
    }
    if (lane == 0) ws[wave] = r;
    __syncthreads();
    if (threadIdx.x != 0) return;
    r = waves_rec<MK, kRowWaves>(p, ws);
    if (!p.first) {
        p.rec[(s * (p.K + 1) + t) * p.segs + seg] = r;
        return;
    }
    const Verdict d = judge<DT, MK, HOW>(p, s, t, n, r);
    p.verdict[s * (p.K + 1) + t] = d;
    if (d.what != kAccept && d.what != kTooClose)
        __hip_atomic_fetch_min(&p.first[s], t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A sequence whose length is none: refused. One workgroup.
__device__ __forceinline__ void refuse_length(const VerifyP &p, int64_t s) {
    const int K1 = p.K + 1;
    for (int t = threadIdx.x; t < K1; t += blockDim.x) {
        p.ids[s * K1 + t] = -1;
        if (p.logp) p.logp[s * K1 + t] = t == 0 ? NAN : 0.0f;
    }
    if (threadIdx.x == 0) {
        p.accepted[s] = 0;
        p.status[s] = uint8_t(NT_ROW_BAD_TOKEN);
        p.pick[s].mode = kDrawNone;
    }
}

// What a sequence ends with at position a, of verdict d.
template <bool GREEDY>
__device__ __forceinline__ VerifyPick pick_of(const VerifyP &p, const Verdict &d, int a, int n) {
    VerifyPick k{d.lp, d.lq, a, kDrawNone};
    if (d.what < kBad && !GREEDY) k.mode = a == n ? kDrawTarget : (p.y ? kDrawRest : kDrawOthers);
    return k;
}

// The sequence's outputs but for the drawn token (k_verify_pick's), from its verdicts up to a. One workgroup.
template <int DT, int MK, bool GREEDY>
__device__ __forceinline__ void write_kept(const VerifyP &p, int64_t s, const Verdict *vs, const VerifyPick &k) {
    const int K1 = p.K + 1, a = k.pos;
    const Verdict &d = vs[a];
    for (int t = threadIdx.x; t < K1; t += blockDim.x) {
        if (t == a && k.mode != kDrawNone) continue;
        float lp = 0.0f;
        int32_t id = -1;
        if (t < a) {
            id = p.tokens[s * p.K + t];
            lp = float(vs[t].logp);
        } else if (t == a) {
            lp = NAN;
            if (GREEDY && d.what < kBad) {
                const VerifyRows<DT, MK> rows(p, s, a);
                id = d.at;
                lp = float((token_arg<DT, MK>(rows.x, rows.m, id, p.c) - d.lp) * kLn2);
            }
        }
        p.ids[s * K1 + t] = id;
        if (p.logp) p.logp[s * K1 + t] = lp;
    }
    if (threadIdx.x == 0) {
        p.accepted[s] = a;
        p.status[s] = uint8_t(d.what < kBad ? NT_ROW_OK : d.what - kBad);
        if constexpr (!GREEDY) p.pick[s] = k;
    }
}

// One workgroup a position: a sequence's verdicts into vs, those too close to call (not greedy) summed in f64,
// and its last position.
template <int DT, int MK, bool AL, bool GREEDY>
__device__ __forceinline__ int settle(const VerifyP &p, int64_t s, int n, Verdict *vs, VerifyRec *ws) {
    const int upto = min(n, p.first[s]), lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    for (int t = threadIdx.x; t <= upto; t += kDrawThreads) vs[t] = p.verdict[s * (p.K + 1) + t];
    __syncthreads();
    int a = 0;
    for (;; a++) {
        if constexpr (!GREEDY) {
            if (vs[a].what == kTooClose) {
                const VerifyRows<DT, MK> rows(p, s, a);
                LaneSum sx, sy;
                add_rows<DT, MK, AL, kWide>(p, rows, rows.y != nullptr, wave, kDrawWaves, p.nc, lane, sx, sy, nullptr, nullptr);
                const VerifyRec r = wave_rec<MK>(p, sx, sy);
                if (lane == 0) ws[wave] = r;
                __syncthreads();
                const Verdict d = judge<DT, MK, kWide>(p, s, a, n, waves_rec<MK, kDrawWaves>(p, ws));
                if (threadIdx.x == 0) vs[a] = d;
                __syncthreads();
            }
        }
        // (the last of them is no accepted one: position n never is, nor the first one refused)
        if (a == upto || vs[a].what != kAccept) return a;
    }
}

template <int DT, int MK, bool AL>
__global__ __launch_bounds__(kDrawThreads) void k_verify_sums(VerifyP p) {
    __shared__ Verdict vs[kMaxDrafts + 1];
    __shared__ VerifyRec ws[kDrawWaves];
    const int64_t s = blockIdx.x / unsigned(p.dsegs);
    const int seg = int(blockIdx.x % unsigned(p.dsegs));
    const int n = drafts_of(p, s);
    if (n < 0 || n > p.K) {
        if (seg == 0) refuse_length(p, s);
        return;
    }
    const int a = settle<DT, MK, AL, false>(p, s, n, vs, ws);
    const VerifyPick k = pick_of<false>(p, vs[a], a, n);
    if (seg == 0) write_kept<DT, MK, false>(p, s, vs, k);
    if (k.mode == kDrawNone) return;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const VerifyRows<DT, MK> rows(p, s, a);
    LaneSum sx, sy;
    add_rows<DT, MK, AL, kWide>(p, rows, k.mode == kDrawRest, seg * p.dper + wave, kDrawWaves, min(p.nc, (seg + 1) * p.dper), lane,
                                sx, sy, nullptr, nullptr);
    __syncthreads();
    const VerifyRec r = wave_rec<MK>(p, sx, sy);
    if (lane == 0) ws[wave] = r;
    __syncthreads();
    if (threadIdx.x == 0) p.rec[s * p.dsegs + seg] = waves_rec<MK, kDrawWaves>(p, ws);
}

// One wave: the sums of `segs` pieces.
template <int MK>
__device__ __forceinline__ VerifyRec merge_recs(const VerifyP &p, const VerifyRec *rec, int segs, int lane) {
    VerifyRec r{0.0, 0.0, -INFINITY, -INFINITY, 0x7fffffff, -INFINITY};
    if (lane < segs) r = rec[lane];
    VerifyRec f;
    f.a = wave_max(r.a);
    f.ad = wave_max(r.ad);
    f.S = wave_sum_d(moved(r.S, r.a, f.a, value_scale<MK>(p.c)));
    f.Sd = wave_sum_d(moved(r.Sd, r.ad, f.ad, value_scale<MK>(p.cd)));
    f.top = wave_max(r.top);
    f.at = wave_min_i(r.top == f.top ? r.at : 0x7fffffff);
    return f;
}

// r of one lane's 8 columns of a chunk.
template <int DT, int MK>
__device__ __forceinline__ void rest8(const VerifyP &p, const VerifyPick &k, int32_t tok, const Raw<DT, MK> &rx,
                                      const Raw<DT, NT_MASK_NONE> &ry, int64_t e0, double r[kEpl]) {
    Lane8<DT, MK, kWide> l;
    l.decode(rx.x, rx.m, p.inv_t);
#pragma unroll
    for (int j = 0; j < kEpl; j++) r[j] = exp2_64(l.arg(j, p.c, -k.lp));
    if (k.mode == kDrawRest) {
        l.decode(ry.x, rx.m, p.inv_td);
#pragma unroll
        for (int j = 0; j < kEpl; j++) r[j] = fmax(r[j] - exp2_64(l.arg(j, p.cd, -k.lq)), 0.0);
    } else if (k.mode == kDrawOthers) {
#pragma unroll
        for (int j = 0; j < kEpl; j++) r[j] = e0 + j == tok ? 0.0 : r[j];
    }
}

template <int DT, int MK, bool AL>
__device__ __forceinline__ void load_rest(const VerifyP &p, const VerifyRows<DT, MK> &rows, int mode, int ch, int lane,
                                          Raw<DT, MK> &rx, Raw<DT, NT_MASK_NONE> &ry) {
    const int64_t e0 = int64_t(ch) * kChunk + lane * kEpl;
    load_raw<DT, MK, AL>(rx, rows.x, rows.m, e0, p.V);
    if (mode == kDrawRest) load_raw<DT, NT_MASK_NONE, AL>(ry, rows.y, nullptr, e0, p.V);
}

__device__ __forceinline__ double sum8(const double r[kEpl]) {
    return ((((((r[0] + r[1]) + r[2]) + r[3]) + r[4]) + r[5]) + r[6]) + r[7];
}

template <int DT, int MK, bool AL, bool GREEDY>
__global__ __launch_bounds__(kDrawThreads) void k_verify_draw(VerifyP p) {
    __shared__ Verdict vs[kMaxDrafts + 1];
    __shared__ VerifyRec ws[kDrawWaves];
    const int64_t s = blockIdx.x / unsigned(p.dsegs);
    const int seg = int(blockIdx.x % unsigned(p.dsegs));
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const int n = drafts_of(p, s);
    VerifyPick k;
    if (!GREEDY && p.first) {
        // k_verify_sums has settled the sequence
        k = p.pick[s];
        if (k.mode == kDrawNone) return;
        const VerifyRec r = merge_recs<MK>(p, p.rec + s * p.dsegs, p.dsegs, lane);
        k.lp = double(r.a) * value_scale<MK>(p.c) + log2(r.S);
        if (k.mode == kDrawRest) k.lq = double(r.ad) * value_scale<MK>(p.cd) + log2(r.Sd);
    } else {
        if (n < 0 || n > p.K) {
            if (seg == 0) refuse_length(p, s);
            return;
        }
        int a = 0;
        if (p.first) {
            a = settle<DT, MK, AL, true>(p, s, n, vs, ws);
        } else {
            for (int t = wave; t <= n; t += kDrawWaves) {
                const VerifyRec r = merge_recs<MK>(p, p.rec + (s * (p.K + 1) + t) * p.segs, p.segs, lane);
                const Verdict d = judge<DT, MK, GREEDY ? kGreedy : kWide>(p, s, t, n, r);
                if (lane == 0) vs[t] = d;
            }
            __syncthreads();
            while (a < n && vs[a].what == kAccept) a++;
        }
        k = pick_of<GREEDY>(p, vs[a], a, n);
        if (seg == 0) write_kept<DT, MK, GREEDY>(p, s, vs, k);
        if (GREEDY || k.mode == kDrawNone) return;
    }
    const int a = k.pos;
    const VerifyRows<DT, MK> rows(p, s, a);
    const int32_t tok = k.mode == kDrawOthers ? p.tokens[s * p.K + a] : -1;
    const int c1 = min(p.nc, (seg + 1) * p.dper);
    int c = seg * p.dper + wave;
    Raw<DT, MK> rx, nx;
    Raw<DT, NT_MASK_NONE> ry, ny;
    if (c < c1) load_rest<DT, MK, AL>(p, rows, k.mode, c, lane, rx, ry);
    for (; c < c1; c += kDrawWaves) {
        if (c + kDrawWaves < c1) load_rest<DT, MK, AL>(p, rows, k.mode, c + kDrawWaves, lane, nx, ny);
        double r[kEpl];
        rest8<DT, MK>(p, k, tok, rx, ry, int64_t(c) * kChunk + lane * kEpl, r);
        const double sum = wave_scan_dpp(sum8(r));
        if (lane == kWave - 1) p.sums[s * p.nc + c] = sum;
        rx = nx;
        ry = ny;
    }
}

// The chunk sums' total; each lane holds the same.
__device__ __forceinline__ double sums_total(const double *sums, int nc, int lane) {
    double total = 0.0;
    for (int c0 = 0; c0 < nc; c0 += kWave)
        total += readlane_d(wave_scan_dpp(c0 + lane < nc ? sums[c0 + lane] : 0.0), kWave - 1);
    return total;
}

template <int DT, int MK, bool AL>
__global__ __launch_bounds__(kWave) void k_verify_pick(VerifyP p) {
    const int64_t s = blockIdx.x;
    const int lane = threadIdx.x;
    VerifyPick k = p.pick[s];
    if (k.mode == kDrawNone) return;
    if (p.first) {
        const VerifyRec r = merge_recs<MK>(p, p.rec + s * p.dsegs, p.dsegs, lane);
        k.lp = double(r.a) * value_scale<MK>(p.c) + log2(r.S);
        if (k.mode == kDrawRest) k.lq = double(r.ad) * value_scale<MK>(p.cd) + log2(r.Sd);
    }
    const VerifyRows<DT, MK> rows(p, s, k.pos);
    const int32_t tok = k.mode == kDrawOthers ? p.tokens[s * p.K + k.pos] : -1;
    double *sums = p.sums + s * p.nc;
    Raw<DT, MK> rx;
    Raw<DT, NT_MASK_NONE> ry;
    double r[kEpl];
    double total = sums_total(sums, p.nc, lane);
    if (!(total > 0.0)) {
        // refused, and yet p is nowhere above q (a uniform of 1 against a draft of equal p and q): p itself
        k.mode = kDrawTarget;
        for (int c = 0; c < p.nc; c++) {
            load_rest<DT, MK, AL>(p, rows, k.mode, c, lane, rx, ry);
            rest8<DT, MK>(p, k, tok, rx, ry, int64_t(c) * kChunk + lane * kEpl, r);
            const double sum = wave_scan_dpp(sum8(r));
            if (lane == kWave - 1) sums[c] = sum;
        }
        __threadfence_block();
        total = sums_total(sums, p.nc, lane);
    }
    const double want = p.u[s * (p.K + 1) + p.K] * total;
    // the first chunk whose running sum passes `want`; if none does, the last that holds anything
    double run = 0.0, before = 0.0;
    int chunk = -1, last = 0;
    for (int c0 = 0; c0 < p.nc && chunk < 0; c0 += kWave) {
        const double v = c0 + lane < p.nc ? sums[c0 + lane] : 0.0;
        const double cum = run + wave_scan_dpp(v);
        const int f = first_lane(__ballot(c0 + lane < p.nc && cum > want));
        const int l = last_lane(__ballot(v > 0.0));
        if (l >= 0) last = c0 + l;
        if (f >= 0) {
            chunk = c0 + f;
            before = f > 0 ? readlane_d(cum, f - 1) : run;
        }
        run = readlane_d(cum, kWave - 1);
    }
    const bool crossed = chunk >= 0;
    if (!crossed) chunk = last;
    const int64_t e0 = int64_t(chunk) * kChunk + lane * kEpl;
    load_rest<DT, MK, AL>(p, rows, k.mode, chunk, lane, rx, ry);
    rest8<DT, MK>(p, k, tok, rx, ry, e0, r);
    const double mine = sum8(r);
    double cum = before + (wave_scan_dpp(mine) - mine);
    int here = -1, some = -1;
#pragma unroll
    for (int j = 0; j < kEpl; j++) {
        cum += r[j];
        if (here < 0 && crossed && r[j] > 0.0 && cum > want) here = j;
        if (r[j] > 0.0) some = j;
    }
    const int f = first_lane(__ballot(here >= 0));
    const int l = f >= 0 ? f : last_lane(__ballot(some >= 0));
    if (lane == l) {
        const int64_t v = e0 + (f >= 0 ? here : some);
        p.ids[s * (p.K + 1) + k.pos] = int32_t(v);
        if (p.logp)
            p.logp[s * (p.K + 1) + k.pos] = float((token_arg<DT, MK>(rows.x, rows.m, v, p.c) - k.lp) * kLn2);
    }
}

__global__ void k_verify_init(int32_t *first, int n) {
    const int i = int(blockIdx.x * blockDim.x + threadIdx.x);
    if (i < n) first[i] = 0x7fffffff;
}

template <int DT, int MK, bool AL>
void verify_launch(const VerifyP &p, bool greedy, hipStream_t s) {
    if (p.first)
        hipLaunchKernelGGL(k_verify_init, dim3(unsigned((p.seqs + 255) / 256)), dim3(256), 0, s, p.first, p.seqs);
    const dim3 rows(unsigned(int64_t(p.seqs) * (p.K + 1) * p.segs)), draw(unsigned(p.seqs * p.dsegs));
    if (greedy) {
        hipLaunchKernelGGL((k_verify_rows<DT, MK, AL, kGreedy>), rows, dim3(kRowThreads), 0, s, p);
        hipLaunchKernelGGL((k_verify_draw<DT, MK, AL, true>), draw, dim3(kDrawThreads), 0, s, p);
        return;
    }
    if (p.first) {
        hipLaunchKernelGGL((k_verify_rows<DT, MK, AL, kNarrow>), rows, dim3(kRowThreads), 0, s, p);
        hipLaunchKernelGGL((k_verify_sums<DT, MK, AL>), draw, dim3(kDrawThreads), 0, s, p);
    } else {
        hipLaunchKernelGGL((k_verify_rows<DT, MK, AL, kWide>), rows, dim3(kRowThreads), 0, s, p);
    }
    hipLaunchKernelGGL((k_verify_draw<DT, MK, AL, false>), draw, dim3(kDrawThreads), 0, s, p);
    hipLaunchKernelGGL((k_verify_pick<DT, MK, AL>), dim3(unsigned(p.seqs)), dim3(kWave), 0, s, p);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_hip_rl_verify_drafted(const NtRlVerifyArgs *a) {
    const char *who = "nt_hip_rl_verify_drafted";
    if (!a) return fail(NT_E_ARG, std::string(who) + ": null args");
    const int64_t seqs = a->seqs, K = a->drafted;
    // (a launch holds fewer than 2^32 threads, a position 1024)
    if (seqs < 0 || K < 0 || K > kMaxDrafts || seqs > 0x3fffffLL / (K + 1))
        return fail(NT_E_ARG, std::string(who) + ": " + std::to_string(seqs) + " sequences of " + std::to_string(K) +
                                  " drafts (0 to " + std::to_string(kMaxDrafts) + ", fewer than 2^22 positions)");
    const int64_t rows = seqs * (K + 1);
    if (int rc = check_rows(rows, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, a->mask_ld, who)) return rc;
    MaskMap mm;
    if (int rc = mask_map(a->mask_rows, rows, a->vocab, a->mask_kind, a->mask_ld, who, &mm)) return rc;
    if (!(a->temperature >= 0.0) || !std::isfinite(a->temperature))
        return fail(NT_E_ARG, "verify_drafted: temperature " + std::to_string(a->temperature) + " (must be ≥ 0)");
    const bool greedy = a->temperature == 0.0, draft = !greedy && a->draft_logits && K > 0;
    if (draft && (!(a->draft_temperature > 0.0) || !std::isfinite(a->draft_temperature)))
        return fail(NT_E_ARG, "verify_drafted: draft temperature " + std::to_string(a->draft_temperature) + " (must be positive)");
    if (draft && a->draft_ld < a->vocab) return fail(NT_E_ARG, std::string(who) + ": draft_ld < vocab");
    if (a->vocab > 0x7fffffffLL - kChunk) return fail(NT_E_ARG, std::string(who) + ": vocab past 2^31");
    if (!a->logits || !a->ids || !a->accepted || !a->status || (K > 0 && !a->tokens) || (!greedy && !a->uniforms))
        return fail(NT_E_ARG, std::string(who) + ": null logits, tokens, uniforms or outputs");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    if (seqs == 0) return 0;

    VerifyP p{};
    p.x = a->logits;
    p.y = draft ? a->draft_logits : nullptr;
    p.mask = a->mask;
    p.V = a->vocab;
    p.ld = a->ld;
    p.ldy = a->draft_ld;
    p.mm = mm;
    const double T = greedy ? 1.0 : a->temperature, Td = draft ? a->draft_temperature : 1.0;
    p.c = kLog2e64 / T;
    p.cd = kLog2e64 / Td;
    p.inv_t = 1.0 / T;
    p.inv_td = 1.0 / Td;
    const bool added = a->mask_kind == NT_MASK_F32;
    p.cap = float(500.0 / (added ? kLog2e64 : p.c));
    p.capd = float(500.0 / (added ? kLog2e64 : p.cd));
    p.s32 = added ? kLog2e : float(p.c);
    p.sd32 = added ? kLog2e : float(p.cd);
    p.nc = int((a->vocab + kChunk - 1) / kChunk);
    p.seqs = int(seqs);
    p.K = int(K);
    // One workgroup a position where the positions alone fill the chip's 256 CUs, so that a refusal can spare the
    // later ones; otherwise about two a CU, each of a chunk per wave or more.
    const bool one = rows >= 256;
    p.segs = one ? 1
                 : int(std::min<int64_t>({int64_t(kVerifySegs), (512 + rows - 1) / rows,
                                          (p.nc + kRowWaves - 1) / kRowWaves}));
    p.per = (p.nc + p.segs - 1) / p.segs;
    p.segs = (p.nc + p.per - 1) / p.per;
    // The drawn rows: about 1024 workgroups, each of a chunk per wave or more.
    p.dsegs = greedy ? 1 : int(std::max<int64_t>(1, std::min<int64_t>({1024 / seqs, int64_t(kVerifySegs), (p.nc + kDrawWaves - 1) / kDrawWaves})));
    p.dper = (p.nc + p.dsegs - 1) / p.dsegs;
    p.dsegs = (p.nc + p.dper - 1) / p.dper;
    p.tokens = a->tokens;
    p.lengths = a->lengths;
    p.u = a->uniforms;
    p.ids = a->ids;
    p.accepted = a->accepted;
    p.logp = a->logp;
    p.status = a->status;

    const auto round = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t recs = round(sizeof(VerifyRec) * size_t(one ? seqs * p.dsegs : rows * p.segs));
    const size_t verdicts = one ? round(sizeof(Verdict) * size_t(rows)) : 0;
    const size_t sums = greedy ? 0 : round(sizeof(double) * size_t(seqs) * size_t(p.nc));
    const size_t picks = round(sizeof(VerifyPick) * size_t(seqs)), firsts = one ? round(sizeof(int32_t) * size_t(seqs)) : 0;
    const size_t need = recs + verdicts + sums + picks + firsts;
    bool cap = false;
    if (int rc = stream_capturing(&cap)) return rc;
    if (cap && need >= size_t(1) << 20)
        return fail(NT_E_UNSUPPORTED, std::string(who) + ": a workspace of " + std::to_string(need) +
                                          " bytes under stream capture (less than 1 MiB)");
    void *ws = nullptr;
    if (int rc = scratch_alloc(need, &ws)) return rc;
    char *at = static_cast<char *>(ws);
    p.rec = reinterpret_cast<VerifyRec *>(at);
    p.verdict = reinterpret_cast<Verdict *>(at + recs);
    p.sums = reinterpret_cast<double *>(at + recs + verdicts);
    p.pick = reinterpret_cast<VerifyPick *>(at + recs + verdicts + sums);
    if (one) p.first = reinterpret_cast<int32_t *>(at + recs + verdicts + sums + picks);

    bool al = aligned_rows(a->logits, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, mm);
    if (draft) al = al && a->draft_ld % kEpl == 0 && reinterpret_cast<uintptr_t>(a->draft_logits) % 16 == 0;
    hipStream_t s = ctx().stream;
    auto by_al = [&](auto dt, auto mk) {
        constexpr int DT = decltype(dt)::value, MK = decltype(mk)::value;
        if (al) verify_launch<DT, MK, true>(p, greedy, s);
        else verify_launch<DT, MK, false>(p, greedy, s);
    };
    auto by_mk = [&](auto dt) {
        if (a->mask_kind == NT_MASK_U8) by_al(dt, std::integral_constant<int, NT_MASK_U8>{});
        else if (a->mask_kind == NT_MASK_F32) by_al(dt, std::integral_constant<int, NT_MASK_F32>{});
        else by_al(dt, std::integral_constant<int, NT_MASK_NONE>{});
    };
    if (a->dtype == NT_F32) by_mk(std::integral_constant<int, NT_F32>{});
    else if (a->dtype == NT_BF16) by_mk(std::integral_constant<int, NT_BF16>{});
    else by_mk(std::integral_constant<int, NT_F16>{});
    const int rc = launched(who);
    const int rc2 = scratch_release(ws);
    return rc ? rc : rc2;
}
