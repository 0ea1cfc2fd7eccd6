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
//  * k_verify_draw: the first refused position (any row that was too close to call summed in f64), and in one f64 pass
//    over the rows there, by several workgroups a sequence, their sums and what r = max(p - q, 0) needs of
//    them: per chunk of 512 columns the sums of both over the columns with p > q. Which those are is known before the
//    sums are, from the sums of k_verify_rows, but for columns where p / q lies too near 1; a chunk that has such a
//    column is left to the next kernel, and all are where those sums turn out to be further off.
//  * k_verify_pick: the chunks' sums of r, then the chunk that holds u sum r, and in it the token.
//
// 256 sequences of 7 drafts over 128256 bf16: 110, 58 and 8 to 16 us of them; the first is bound by HBM, the second by
// f64 exponentials (two a column, 40 us of instructions).
#include <algorithm>

#include "nt_exp64.hpp"
#include "nt_rows.hpp"
#include "nt_rowsum.hpp"

namespace nt {
namespace {

constexpr int kRowThreads = 512;              // k_verify_rows
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kDrawThreads = 256;             // k_verify_draw, k_verify_pick
constexpr int kDrawWaves = kDrawThreads / kWave;
constexpr int kMaxDrafts = 127;
constexpr int kAhead = 4;                     // chunks loaded ahead of f32 sums
constexpr int kVerifySegs = 64;               // workgroups a position or a drawn row, at most (one lane each)
// How k_verify_rows sums: in f64, in f32 (see judge), or in f32 with the first largest value.
enum { kWide, kNarrow, kGreedy };
// What f32 sums may be off in a log2 ratio of p and q: each of the two log-sum-exps by 6e-6 (of an argument t, up to 60 where a
// reference trails its lane's largest value: half a step of it 1.9e-6, the rounding of c 60 2^-24 = 3.6e-6; the instruction and trees of 8
// 0.5e-6; under an additive mask f64 differences of up to 23 above theirs, 4.6e-6). f64 sums: 1e-11.
constexpr double kClose32 = 2e-5;
// How near 1 a column's p / q is left to k_verify_pick: far more than f64 sums are off, and more than f32 sums of these rows
// usually are (1e-7; with a wider one, equal 16-bit differences of many columns fall into it: one row in 200 at kClose32).
constexpr double kNear64 = 1e-9, kNear32 = 1e-6;

// What a workgroup found in its piece of a position's rows: sums S relative to the reference a (in tempered logits,
// or with no additive mask logits), of the target and of the drafter; greedy: the target's first largest value and its place.
struct VerifyRec {
    double S, Sd, a, ad;
    int32_t at;
    float top;
};

// What becomes of a position, from its sums: accepted, drawn from, too close for f32, or a row status that ends
// the sequence (kBad + NT_ROW_*).
enum { kAccept = 0, kDraw = 1, kTooClose = 2, kBad = 3 };
struct Verdict {
    int what;
    int32_t at;            // greedy: the first largest; otherwise whether the sums are f64
    double a, ls, ad, lsd; // the log-sum-exps: references and log2 of the sums (drafter's 0 without its logits)
    double logp;           // ln p of the draft
};

// What is drawn from at a sequence's last position: references of p and q (their sums are k_verify_draw's) and how, and the
// ratio of the sums that k_verify_draw went by, with how far it may be off.
enum { kDrawNone = -1, kDrawTarget = 0, kDrawRest = 1, kDrawOthers = 2 };
struct VerifyPick {
    double a, ad, ratio, near;
    int32_t pos, mode;
};

struct VerifyP {
    const void *x, *y, *mask;
    int64_t V, ld, ldy;
    MaskMap mm;
    double inv_t, inv_td;     // 1 / T of the target and the drafter
    double c, cd;             // log2 units of one unit of value: log2(e) / T, with an additive mask log2(e)
    double low, lowd;         // -1100 / c
    float cap, capd;          // 500 / c
    float c32, cd32;
    int nc;                   // chunks of a row
    int seqs, K;
    int segs, per;            // workgroups a position, chunks each
    int dsegs, dper;          // workgroups a drawn row, chunks each
    const int32_t *tokens, *lengths;
    const double *u;
    int32_t *ids, *accepted;
    float *logp;
    uint8_t *status;
    VerifyRec *rec;           // several workgroups a position: [seqs][K + 1][segs]
    Verdict *verdict;         // one: [seqs][K + 1]
    int32_t *first;           //      [seqs] the first position known to be refused
    double2 *total;           // [seqs][dsegs] the drawn rows' sums
    double2 *sums;            // [seqs][nc] of their chunks: of P - ratio Q, and of Q, where that is above 0 (y NaN: left)
    VerifyPick *pick;         // [seqs]
};

// The larger, a NaN if there is one.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max8_nan(const float v[kEpl]) {
    return max_nan(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])), max_nan(max_nan(v[4], v[5]), max_nan(v[6], v[7])));
}

// One lane's 8 values: a logit, -inf where a u8 mask excludes it; with an additive mask the tempered logit in f64
// (v: the f32 nearest to it, infinite past f32, which FarSum sees to; kGreedy: the f32 sum).
template <int DT, int MK, int HOW>
struct Lane8 {
    static constexpr bool kTwo = MK == NT_MASK_F32 && HOW != kGreedy;
    float v[kEpl];
    double z[kTwo ? kEpl : 1];

    __device__ __forceinline__ void decode(const uint32_t *xw, const uint32_t *mw, double inv_t) {
        if constexpr (MK == NT_MASK_F32) {
#pragma unroll
            for (int j = 0; j < kEpl; j++) {
                const float x = logit<DT>(xw, j), m = __uint_as_float(mw[j]);
                if constexpr (HOW == kGreedy) {
                    v[j] = x + m;
                } else {
                    const double t = fma(double(x), inv_t, double(m));
                    if constexpr (kTwo) z[j] = t;
                    v[j] = float(t);
                }
            }
        } else {
            decode_e<DT, MK, kEpl>(xw, mw, v, 1.0f, true);
        }
    }
    template <class R>
    __device__ __forceinline__ void clean(const R &row, int ch, int lane) {
        if constexpr (kTwo && HOW == kNarrow) {
            row.clean(z, ch, lane);
        } else {
            row.clean(v, ch, lane);
            if constexpr (kTwo) {
#pragma unroll
                for (int j = 0; j < kEpl; j++) z[j] = v[j] == -INFINITY ? -INFINITY : z[j];
            }
        }
    }
    __device__ __forceinline__ double at(int j) const {
        if constexpr (kTwo) return z[j];
        else return double(v[j]);
    }
};

__device__ __forceinline__ double sum8(const double r[kEpl]) {
    return ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
}

// A lane's f64 sum relative to its reference: the first maximum it met, moved only where a later value lies 2^500 above
// it, which f64 holds and logits hardly reach. A NaN or +inf leaves a NaN.
struct LaneSum {
    double S = 0.0, ref = -INFINITY;
    float lim = -INFINITY;

    template <class L>
    __device__ __forceinline__ void add(const L &l, double c, double low, float cap) {
        const float top = max8_nan(l.v);
        double high = double(top);
        bool over = !(top <= lim);
        if constexpr (L::kTwo) {  // (an f32 step may be more than 2^500: in f64)
            high = l.z[0];
#pragma unroll
            for (int j = 1; j < kEpl; j++) high = fmax(high, l.z[j]);
            over = high > ref + double(cap) || !(top < INFINITY);
        }
        if (over) {
            if (top < INFINITY) {
                if (ref != -INFINITY) S *= exp2_64(ref - high, c, low);
                ref = high;
                lim = fminf(top + cap, FLT_MAX);
            } else {
                S = NAN;
            }
        }
        double w[kEpl];
#pragma unroll
        for (int j = 0; j < kEpl; j++) w[j] = exp2_64(l.at(j) - ref, c, low);
        S += sum8(w);
    }
    __device__ __forceinline__ double at(double, float) const { return ref; }
};

// The value of one token (see Lane8), -inf where it is excluded. Greedy under an additive mask: the f32 sum, as the row's sums
// take it (where a mask lowers a whole row, its rounding is no small part of the differences).
template <int DT, int MK, bool GREEDY>
__device__ __forceinline__ double token_value(const void *xrow, const void *mrow, int64_t v, double inv_t) {
    float x;
    if constexpr (DT == NT_F32) x = static_cast<const float *>(xrow)[v];
    else x = widen16<DT>(uint32_t(static_cast<const uint16_t *>(xrow)[v]));
    if constexpr (MK == NT_MASK_U8) {
        if (static_cast<const uint8_t *>(mrow)[v] == 0) return -INFINITY;
    } else if constexpr (MK == NT_MASK_F32) {
        const float m = static_cast<const float *>(mrow)[v];
        if constexpr (GREEDY) return double(x + m);
        else return fma(double(x), inv_t, double(m));
    }
    return double(x);
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

// The draft at position t < n, its values and its uniform, loaded before the sums are known.
struct Draft {
    int32_t tok = -1;
    double x = 0.0, y = 0.0, u = 0.0;

    template <int DT, int MK, bool GREEDY>
    __device__ __forceinline__ void load(const VerifyP &p, const VerifyRows<DT, MK> &rows, int64_t s, int t, int n) {
        if (t >= n) return;
        tok = p.tokens[s * p.K + t];
        if constexpr (!GREEDY) u = p.u[s * (p.K + 1) + t];
        if (tok < 0 || tok >= p.V) return;
        x = token_value<DT, MK, GREEDY>(rows.x, rows.m, tok, p.inv_t);
        if (rows.y) y = token_value<DT, MK, GREEDY>(rows.y, rows.m, tok, p.inv_td);
    }
};

// Position t of a sequence of n drafts, from its merged sums.
template <int DT, int MK, int HOW>
__device__ __forceinline__ Verdict judge(const VerifyP &p, const VerifyRows<DT, MK> &rows, const Draft &w, int t, int n, const VerifyRec &r) {
    Verdict d{kDraw, HOW == kGreedy ? r.at : HOW == kWide, r.a, 0.0, 0.0, 0.0, 0.0};
    if (!(r.S == r.S)) {
        d.what = kBad + NT_ROW_NAN;
        return d;
    }
    if (r.a == -INFINITY) {
        d.what = kBad + NT_ROW_NO_TOKEN;
        return d;
    }
    d.ls = log2(r.S);
    if (t >= n) return d;
    if (w.tok < 0 || w.tok >= p.V) {
        d.what = kBad + NT_ROW_BAD_TOKEN;
        return d;
    }
    const double l = (w.x - r.a) * p.c - d.ls;
    d.logp = l * kLn2;
    if constexpr (HOW == kGreedy) {
        d.what = r.at == w.tok ? kAccept : kDraw;
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
        d.ad = r.ad;
        d.lsd = log2(r.Sd);
        lq = (w.y - r.ad) * p.cd - d.lsd;
    }
    // u q < p: a draft that the drafter gives nothing is accepted where the target gives it something, and one
    // that the target gives nothing never is (inf - inf compares false)
    d.what = w.u < exp2(l - lq) ? kAccept : kDraw;
    if constexpr (HOW == kNarrow) {
        if (fabs(log2(w.u) - (l - lq)) < kClose32) d.what = kTooClose;
    }
    return d;
}

// A wave's sums from its lanes'.
template <class L>
__device__ __forceinline__ VerifyRec wave_rec(const VerifyP &p, const L &x, const L &y) {
    VerifyRec r{0.0, 0.0, -INFINITY, -INFINITY, 0, 0.0f};
    const double a = x.at(p.c, p.c32), ad = y.at(p.cd, p.cd32);
    r.a = wave_max_d(a);
    r.S = wave_sum_d(moved(x.S, a, r.a, p.c, p.low));
    r.ad = wave_max_d(ad);
    r.Sd = wave_sum_d(moved(y.S, ad, r.ad, p.cd, p.lowd));
    return r;
}

// One wave: the sums of `segs` pieces.
__device__ __forceinline__ VerifyRec merge_recs(const VerifyP &p, const VerifyRec *rec, int segs, int lane) {
    VerifyRec r{0.0, 0.0, -INFINITY, -INFINITY, 0x7fffffff, -INFINITY};
    if (lane < segs) r = rec[lane];
    VerifyRec f;
    f.a = wave_max_d(r.a);
    f.ad = wave_max_d(r.ad);
    f.S = wave_sum_d(moved(r.S, r.a, f.a, p.c, p.low));
    f.Sd = wave_sum_d(moved(r.Sd, r.ad, f.ad, p.cd, p.lowd));
    f.top = wave_max(r.top);
    f.at = wave_min_i(r.top == f.top ? r.at : 0x7fffffff);
    return f;
}

// f(chunk, target's values, drafter's values) for chunks c, c + step, .. below c1 of a position's rows (both: the
// drafter's are read).
template <int DT, int MK, bool AL, int HOW, class F>
__device__ __forceinline__ void over_rows(const VerifyP &p, const VerifyRows<DT, MK> &rows, bool both, int c, int step, int c1,
                                          int lane, F &&f) {
    constexpr int D = HOW == kWide ? 2 : kAhead;
    Raw<DT, MK> rx[D];
    Raw<DT, NT_MASK_NONE> ry[D];
    const RowLoad<DT, MK, AL> x(rows.x, rows.m, p.V, p.nc);
    const RowLoad<DT, NT_MASK_NONE, AL> y(rows.y, nullptr, p.V, p.nc);
    auto load = [&](auto k, int ch) {
        x.load(rx[k.value], ch, lane, ch < c1);
        if (both) y.load(ry[k.value], ch, lane, ch < c1);
    };
    stream<D>(c, step, c1, load, [&](auto k, int ch, int next) {
        Lane8<DT, MK, HOW> lx, ly;
        lx.decode(rx[k.value].x, rx[k.value].m, p.inv_t);
        lx.clean(x, ch, lane);
        if (both) {
            ly.decode(ry[k.value].x, rx[k.value].m, p.inv_td);
            ly.clean(y, ch, lane);
        }
        load(k, next);
        f(ch, lx, ly);
    });
}

// The lanes' sums of a position's rows.
template <int DT, int MK, bool AL, int HOW, class L>
__device__ __forceinline__ void add_rows(const VerifyP &p, const VerifyRows<DT, MK> &rows, bool both, int c, int step, int c1,
                                         int lane, L &sx, L &sy, float *top, int32_t *at) {
    over_rows<DT, MK, AL, HOW>(p, rows, both, c, step, c1, lane, [&](int ch, const auto &lx, const auto &ly) {
        if constexpr (HOW == kGreedy) {
            const RowLoad<DT, MK, AL> row(rows.x, rows.m, p.V, p.nc);
#pragma unroll
            for (int j = 0; j < kEpl; j++) {
                const bool up = lx.v[j] > *top;
                *top = up ? lx.v[j] : *top;
                *at = up ? int32_t(row.col(ch, lane, j)) : *at;
            }
        }
        if constexpr (HOW == kWide) {
            sx.add(lx, p.c, p.low, p.cap);
            if (both) sy.add(ly, p.cd, p.lowd, p.capd);
        } else if constexpr (std::is_same_v<L, FarSum>) {
            sx.add(lx.z, p.low);
            if (both) sy.add(ly.z, p.lowd);
        } else {
            sx.add(lx.v, p.c32);
            if (both) sy.add(ly.v, p.cd32);
        }
    });
}

template <int HOW, int MK>
using Sum = std::conditional_t<HOW == kWide, LaneSum, std::conditional_t<HOW == kNarrow && MK == NT_MASK_F32, FarSum, LaneSums>>;

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
    Draft w;
    if (p.first) w.load<DT, MK, HOW == kGreedy>(p, rows, s, t, n);
    Sum<HOW, MK> sx, sy;
    float top = -INFINITY;
    int32_t at = 0x7fffffff;
    add_rows<DT, MK, AL, HOW>(p, rows, both, seg * p.per + wave, kRowWaves, c1, lane, sx, sy, &top, &at);
    VerifyRec r = wave_rec(p, sx, sy);
    if constexpr (HOW == kGreedy) {
        r.top = wave_max(top);
        r.at = wave_min_i(top == r.top ? at : 0x7fffffff);
    }
    if (lane == 0) ws[wave] = r;
    __syncthreads();
    if (wave != 0) return;
    r = merge_recs(p, ws, kRowWaves, lane);
    if (!p.first) {
        if (lane == 0) p.rec[(s * (p.K + 1) + t) * p.segs + seg] = r;
        return;
    }
    if (lane != 0) return;
    const Verdict d = judge<DT, MK, HOW>(p, rows, w, t, n, r);
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

// The sequence's verdicts into vs, and its last position. One workgroup.
template <int DT, int MK, bool AL, bool GREEDY>
__device__ __forceinline__ int settle(const VerifyP &p, int64_t s, int n, Verdict *vs, VerifyRec *ws) {
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    int upto = n;
    if (p.first) {
        upto = min(n, p.first[s]);
        for (int t = threadIdx.x; t <= upto; t += kDrawThreads) vs[t] = p.verdict[s * (p.K + 1) + t];
    } else {
        for (int t = wave; t <= n; t += kDrawWaves) {
            const VerifyRows<DT, MK> rows(p, s, t);
            Draft w;
            w.load<DT, MK, GREEDY>(p, rows, s, t, n);
            const VerifyRec r = merge_recs(p, p.rec + (s * (p.K + 1) + t) * p.segs, p.segs, lane);
            const Verdict d = judge<DT, MK, GREEDY ? kGreedy : kWide>(p, rows, w, t, n, r);
            if (lane == 0) vs[t] = d;
        }
    }
    __syncthreads();
    for (int a = 0;; a++) {
        if constexpr (!GREEDY) {
            if (vs[a].what == kTooClose) {
                const VerifyRows<DT, MK> rows(p, s, a);
                LaneSum sx, sy;
                add_rows<DT, MK, AL, kWide>(p, rows, rows.y != nullptr, wave, kDrawWaves, p.nc, lane, sx, sy, nullptr, nullptr);
                const VerifyRec r = wave_rec(p, sx, sy);
                if (lane == 0) ws[wave] = r;
                __syncthreads();
                Draft w;
                w.load<DT, MK, false>(p, rows, s, a, n);
                const Verdict d = judge<DT, MK, kWide>(p, rows, w, a, n, merge_recs(p, ws, kDrawWaves, lane));
                if (threadIdx.x == 0) vs[a] = d;
                __syncthreads();
            }
        }
        // (the last of them is no accepted one: position n never is, nor the first one refused)
        if (a == upto || vs[a].what != kAccept) return a;
    }
}

template <int DT, int MK, bool AL, bool GREEDY>
__global__ __launch_bounds__(kDrawThreads, 4) void k_verify_draw(VerifyP p) {
    __shared__ Verdict vs[kMaxDrafts + 1];
    __shared__ VerifyRec ws[kDrawWaves];
    const int64_t s = blockIdx.x / unsigned(p.dsegs);
    const int seg = int(blockIdx.x % unsigned(p.dsegs));
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const int n = drafts_of(p, s), K1 = p.K + 1;
    if (n < 0 || n > p.K) {
        if (seg == 0) refuse_length(p, s);
        return;
    }
    const int a = settle<DT, MK, AL, GREEDY>(p, s, n, vs, ws);
    const Verdict d = vs[a];
    const VerifyRows<DT, MK> rows(p, s, a);
    const double ratio = exp2(d.ls - d.lsd), near = d.at ? kNear64 : kNear32;
    int mode = kDrawNone;
    if (d.what < kBad && !GREEDY) mode = a == n ? kDrawTarget : (p.y ? kDrawRest : kDrawOthers);
    if (seg == 0) {
        // what is kept, but for the drawn token (k_verify_pick's)
        for (int t = threadIdx.x; t < K1; t += kDrawThreads) {
            if (t == a && mode != kDrawNone) continue;
            float lp = 0.0f;
            int32_t id = -1;
            if (t < a) {
                id = p.tokens[s * p.K + t];
                lp = float(vs[t].logp);
            } else if (t == a) {
                lp = NAN;
                if (GREEDY && d.what < kBad) {
                    id = d.at;
                    lp = float(((token_value<DT, MK, true>(rows.x, rows.m, id, p.inv_t) - d.a) * p.c - d.ls) * kLn2);
                }
            }
            p.ids[s * K1 + t] = id;
            if (p.logp) p.logp[s * K1 + t] = lp;
        }
        if (threadIdx.x == 0) {
            p.accepted[s] = a;
            p.status[s] = uint8_t(d.what < kBad ? NT_ROW_OK : d.what - kBad);
            if constexpr (!GREEDY) p.pick[s] = VerifyPick{d.a, d.ad, ratio, near, a, mode};
        }
    }
    if (GREEDY || mode == kDrawNone) return;

    // p and q are P = 2^((x - a) c) and Q = 2^((y - ad) cd) over their sums, r = max(P - ratio Q, 0) over P's with the ratio of
    // the sums
    const int32_t tok = mode == kDrawOthers ? p.tokens[s * p.K + a] : -1;
    double2 total{0.0, 0.0};
    over_rows<DT, MK, AL, kWide>(p, rows, mode == kDrawRest, seg * p.dper + wave, kDrawWaves, min(p.nc, (seg + 1) * p.dper), lane,
                                 [&](int ch, const auto &lx, const auto &ly) {
        double P[kEpl];
#pragma unroll
        for (int j = 0; j < kEpl; j++) P[j] = exp2_64(lx.at(j) - d.a, p.c, p.low);
        total.x += sum8(P);
        bool left = false;
        double q = 0.0;
        if (mode == kDrawRest) {
            double Q[kEpl];
#pragma unroll
            for (int j = 0; j < kEpl; j++) Q[j] = exp2_64(ly.at(j) - d.ad, p.cd, p.lowd);
            total.y += sum8(Q);
#pragma unroll
            for (int j = 0; j < kEpl; j++) {
                const double over = fma(-ratio, Q[j], P[j]);
                left = left || fabs(over) < P[j] * near;
                P[j] = fmax(over, 0.0);
                Q[j] = over > 0.0 ? Q[j] : 0.0;
            }
            q = wave_sum_d(sum8(Q));
        } else if (mode == kDrawOthers) {
            const RowLoad<DT, MK, AL> row(rows.x, rows.m, p.V, p.nc);
#pragma unroll
            for (int j = 0; j < kEpl; j++) P[j] = row.col(ch, lane, j) == tok ? 0.0 : P[j];
        }
        const double x = wave_sum_d(sum8(P));
        if (__ballot(left)) q = NAN;
        if (lane == 0) p.sums[s * p.nc + ch] = double2{x, q};
    });
    total.x = wave_sum_d(total.x);
    total.y = wave_sum_d(total.y);
    __syncthreads();
    if (lane == 0) {
        ws[wave].S = total.x;
        ws[wave].Sd = total.y;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kDrawWaves; w++) {
            total.x += ws[w].S;
            total.y += ws[w].Sd;
        }
        p.total[s * p.dsegs + seg] = total;
    }
}

// r of one lane's 8 columns: p = 2^((x - a) c) / sums.x less q.
template <int DT, int MK, bool AL>
__device__ __forceinline__ void rest8(const VerifyP &p, const VerifyRows<DT, MK> &rows, const VerifyPick &k, double2 inv, int32_t tok,
                                      int64_t e0, double r[kEpl]) {
    Raw<DT, MK> rx;
    Raw<DT, NT_MASK_NONE> ry;
    load_raw<DT, MK, AL>(rx, rows.x, rows.m, e0, p.V);
    if (k.mode == kDrawRest) load_raw<DT, NT_MASK_NONE, AL>(ry, rows.y, nullptr, e0, p.V);
    Lane8<DT, MK, kWide> l;
    l.decode(rx.x, rx.m, p.inv_t);
#pragma unroll
    for (int j = 0; j < kEpl; j++) r[j] = exp2_64(l.at(j) - k.a, p.c, p.low) * inv.x;
    if (k.mode == kDrawRest) {
        l.decode(ry.x, rx.m, p.inv_td);
#pragma unroll
        for (int j = 0; j < kEpl; j++) r[j] = fmax(r[j] - exp2_64(l.at(j) - k.ad, p.cd, p.lowd) * inv.y, 0.0);
    } else if (k.mode == kDrawOthers) {
#pragma unroll
        for (int j = 0; j < kEpl; j++) r[j] = e0 + j == tok ? 0.0 : r[j];
    }
}

// The chunk sums' total; each lane holds the same.
__device__ __forceinline__ double sums_total(const double2 *sums, int nc, int lane) {
    double total = 0.0;
    for (int c0 = 0; c0 < nc; c0 += kWave)
        total += readlane_d(wave_scan_dpp(c0 + lane < nc ? sums[c0 + lane].x : 0.0), kWave - 1);
    return total;
}

template <int DT, int MK, bool AL>
__global__ __launch_bounds__(kDrawThreads) void k_verify_pick(VerifyP p) {
    const int64_t s = blockIdx.x;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    VerifyPick k = p.pick[s];
    if (k.mode == kDrawNone) return;
    const VerifyRows<DT, MK> rows(p, s, k.pos);
    const int32_t tok = k.mode == kDrawOthers ? p.tokens[s * p.K + k.pos] : -1;
    double2 *sums = p.sums + s * p.nc, whole{0.0, 0.0};
    if (lane < p.dsegs) whole = p.total[s * p.dsegs + lane];
    whole.x = wave_sum_d(whole.x);
    whole.y = wave_sum_d(whole.y);
    const double2 inv{1.0 / whole.x, k.mode == kDrawRest ? 1.0 / whole.y : 0.0};
    // (P - ratio Q of the right ratio, whole.x / whole.y)
    const double more = k.mode == kDrawRest ? k.ratio - whole.x / whole.y : 0.0;
    const bool all = fabs(more) > 0.5 * k.near * k.ratio;
    double r[kEpl];
    // r of each chunk, 64 of them a wave at a time; those that were left are computed here
    for (int c0 = wave * kWave; c0 < p.nc; c0 += kDrawWaves * kWave) {
        double2 v{0.0, 0.0};
        if (c0 + lane < p.nc) v = sums[c0 + lane];
        double sum = fmax((v.x + more * v.y) * inv.x, 0.0);
        for (uint64_t left = __ballot(c0 + lane < p.nc && (all || !(v.y == v.y))); left; left &= left - 1) {
            const int i = __builtin_ctzll(left);
            rest8<DT, MK, AL>(p, rows, k, inv, tok, int64_t(c0 + i) * kChunk + lane * kEpl, r);
            const double one = wave_sum_d(sum8(r));
            if (lane == i) sum = one;
        }
        if (c0 + lane < p.nc) sums[c0 + lane].x = sum;
    }
    __syncthreads();
    if (wave != 0) return;
    double total = sums_total(sums, p.nc, lane);
    if (!(total > 0.0)) {
        // refused, and yet p is nowhere above q (a uniform of 1 against a draft of equal p and q): p itself
        k.mode = kDrawTarget;
        for (int c = 0; c < p.nc; c++) {
            rest8<DT, MK, AL>(p, rows, k, inv, -1, int64_t(c) * kChunk + lane * kEpl, r);
            const double sum = wave_sum_d(sum8(r));
            if (lane == 0) sums[c].x = sum;
        }
        __threadfence_block();
        total = sums_total(sums, p.nc, lane);
    }
    const double want = p.u[s * (p.K + 1) + p.K] * total;
    // the first chunk whose running sum passes `want`; if none does, the last that holds anything
    double run = 0.0, before = 0.0;
    int chunk = -1, last = 0;
    for (int c0 = 0; c0 < p.nc && chunk < 0; c0 += kWave) {
        const double v = c0 + lane < p.nc ? sums[c0 + lane].x : 0.0;
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
    rest8<DT, MK, AL>(p, rows, k, inv, tok, e0, r);
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
            p.logp[s * (p.K + 1) + k.pos] =
                float(((token_value<DT, MK, false>(rows.x, rows.m, v, p.inv_t) - k.a) * p.c - log2(whole.x)) * kLn2);
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
    } else {
        hipLaunchKernelGGL((k_verify_rows<DT, MK, AL, kWide>), rows, dim3(kRowThreads), 0, s, p);
    }
    hipLaunchKernelGGL((k_verify_draw<DT, MK, AL, false>), draw, dim3(kDrawThreads), 0, s, p);
    hipLaunchKernelGGL((k_verify_pick<DT, MK, AL>), dim3(unsigned(p.seqs)), dim3(kDrawThreads), 0, s, p);
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
    p.inv_t = 1.0 / T;
    p.inv_td = 1.0 / Td;
    const bool added = a->mask_kind == NT_MASK_F32;
    p.c = added ? kLog2e64 : kLog2e64 / T;
    p.cd = added ? kLog2e64 : kLog2e64 / Td;
    p.low = -1100.0 / p.c;
    p.lowd = -1100.0 / p.cd;
    p.cap = float(std::min(500.0 / p.c, 1e38));  // (an infinity is past it at any temperature)
    p.capd = float(std::min(500.0 / p.cd, 1e38));
    p.c32 = float(p.c);
    p.cd32 = float(p.cd);
    p.nc = int((a->vocab + kChunk - 1) / kChunk);
    p.seqs = int(seqs);
    p.K = int(K);
    // One workgroup a position where the positions alone fill the chip's 256 CUs, so that a refusal can spare the
    // later ones; otherwise about two a CU, each of a chunk per wave or more. (3 drafts, in several and in one: 128 positions of
    // 32000 bf16 29.9 and 32.2 us, of 128256 47.6 and 44.3; 256 positions 35.9 and 32.7, 70.5 and 54.6; 512 of 128256 117 and
    // 87.) A temperature whose scale f32 does not hold goes the f64 way too.
    const auto held = [](double c) { return c >= double(FLT_MIN) && c <= double(FLT_MAX); };
    const bool one = rows >= 256 && held(p.c) && held(p.cd);
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
    const size_t recs = one ? 0 : round(sizeof(VerifyRec) * size_t(rows) * size_t(p.segs));
    const size_t verdicts = one ? round(sizeof(Verdict) * size_t(rows)) : 0;
    const size_t firsts = one ? round(sizeof(int32_t) * size_t(seqs)) : 0;
    const size_t totals = greedy ? 0 : round(sizeof(double2) * size_t(seqs) * size_t(p.dsegs));
    const size_t sums = greedy ? 0 : round(sizeof(double2) * size_t(seqs) * size_t(p.nc));
    const size_t picks = round(sizeof(VerifyPick) * size_t(seqs));
    const size_t need = recs + verdicts + firsts + totals + sums + picks;
    bool cap = false;
    if (int rc = stream_capturing(&cap)) return rc;
    if (cap && need >= size_t(1) << 20)
        return fail(NT_E_UNSUPPORTED, std::string(who) + ": a workspace of " + std::to_string(need) +
                                          " bytes under stream capture (less than 1 MiB)");
    void *ws = nullptr;
    if (int rc = scratch_alloc(need, &ws)) return rc;
    char *at = static_cast<char *>(ws);
    p.rec = reinterpret_cast<VerifyRec *>(at);
    p.verdict = reinterpret_cast<Verdict *>(at += recs);
    if (one) p.first = reinterpret_cast<int32_t *>(at + verdicts);
    p.total = reinterpret_cast<double2 *>(at += verdicts + firsts);
    p.sums = reinterpret_cast<double2 *>(at += totals);
    p.pick = reinterpret_cast<VerifyPick *>(at + sums);

    bool al = aligned_rows(a->logits, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, mm) && a->vocab * 4 <= 0x7fffffffLL;
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
