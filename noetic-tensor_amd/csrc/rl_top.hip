// nt_hip_rl_top_logprobs: the k most likely tokens of each row and their log-probabilities, in one pass.
//
// A workgroup streams its row (or, where rows are few, a piece of one) in tiles that its registers hold. It keeps
// a list of candidates in LDS and a threshold that the k-th largest so far is known to reach, and a tile adds the few
// elements above it; the same registers give the tile's part of the log-sum-exp. The first threshold comes from
// the largest value of each lane's groups of eight: k groups that reach it are k elements that do. A value is
// compared as 64 bits, the f32 made an ordered integer over the complement of its column, so that no two are equal and ties
// go to the lowest column. When the list grows past kKeep, a threshold between the k-th and the 2k-th of it is
// found by bisection and the rest dropped; where many values are equal or the row rises (a tile may then
// bring more than the list holds), the tile goes in by groups and the list is cut to its k largest exactly.
// At the end a candidate's place is the number of candidates above it.
//
// What bounds it: the row's bytes, and for the log-sum-exp f32 exponentials as the scorer takes them.
#include <algorithm>

#include "nt_rows.hpp"

namespace nt {
namespace {

constexpr int kTopThreads = 256;
constexpr int kTopWaves = kTopThreads / kWave;
constexpr int kList = 4096;          // candidates in LDS (a full group of a tile over kMaxK fits: 1024 + 2048)
constexpr int kKeep = 1024;          // the list is cut when it is longer (or longer than 2 k)
constexpr int kMaxK = 1024;
constexpr int kTopSegs = 64;         // pieces of a row, at most

// A piece's part of the row's log-sum-exp: S relative to a; n candidates follow.
struct TopRec {
    double S;
    float a;
    int32_t n;
};

struct TopP {
    const void *x, *mask;
    int64_t V, ld;
    MaskMap mm;
    float c;            // exponent scale of a value: log2(e) / T (none, u8) or log2(e) (f32 mask)
    float tau;
    int tau_one;
    double inv_t;       // value -> z: 1 / T, or 1 with an f32 mask
    int k;
    int nc;             // chunks of a row
    int segs, per;      // pieces of a row, chunks each
    int32_t *ids;
    float *logp;
    uint8_t *status;
    TopRec *rec;        // segs > 1: [rows][segs]
    uint64_t *cand;     // segs > 1: [rows][segs][2 k]
};

// An f32 as an integer of the same order (-0 and +0 alike), and back.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kNone = 0x007fffffu;  // ordered(-inf): an excluded token's, never a candidate

// LDS of a workgroup.
struct TopS {
    uint64_t list[kList];
    uint64_t least;          // a candidate is above it
    uint32_t sums[2][kTopWaves];
    int count;
    double S[kTopWaves];
    float a[kTopWaves];
};

// The sum over the workgroup of a count that each lane's wave already agrees on (one barrier: two buffers in turn).
__device__ __forceinline__ uint32_t group_sum(TopS &s, uint32_t wave_count, int turn) {
    if ((threadIdx.x & (kWave - 1)) == 0) s.sums[turn & 1][threadIdx.x / kWave] = wave_count;
    __syncthreads();
    uint32_t n = 0;
#pragma unroll
    for (int w = 0; w < kTopWaves; w++) n += s.sums[turn & 1][w];
    return n;
}

// The largest found t such that at least k of the workgroup's N keys a lane are t or more, as soon as no more than
// `most` are (bit by bit from the top; exact when it reaches the last). 0 where fewer than k are above `floor`
// (floor: what a lane holds in place of nothing).
template <class T, int N>
__device__ __forceinline__ T kth_bound(TopS &s, const T (&key)[N], int k, int most) {
    T t = 0;
    int turn = 0;
    for (int bit = int(sizeof(T)) * 8 - 1; bit >= 0; bit--) {
        const T up = t | (T(1) << bit);
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < N; i++) n += uint32_t(__popcll(__ballot(key[i] >= up)));
        n = group_sum(s, n, turn++);
        if (int(n) >= k) {
            t = up;
            if (int(n) <= most) break;
        }
    }
    __syncthreads();  // (the sums' buffers are free again)
    return t;
}

// Keep of the list what is `bound` or more. Every thread holds its entries (list[i * 256 + thread]) in `mine`.
template <int N>
__device__ __forceinline__ void keep_from(TopS &s, const uint64_t (&mine)[N], uint64_t bound) {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const bool in = mine[i] >= bound && mine[i] != 0;
        const uint64_t b = __ballot(in);
        if (b == 0) continue;
        int at = 0;
        if ((threadIdx.x & (kWave - 1)) == unsigned(__builtin_ctzll(b))) at = atomicAdd(&s.count, int(__popcll(b)));
        at = __builtin_amdgcn_readlane(at, __builtin_ctzll(b));
        if (in) s.list[at + __popcll(b & ((uint64_t(1) << (threadIdx.x & (kWave - 1))) - 1))] = mine[i];
    }
    __syncthreads();
}

// Cut the list of `count` > k to at most max(2 k, ..) entries that hold its k largest (`exact`: to those k), and
// raise the threshold to it.
__device__ __attribute__((noinline)) void cut_list(TopS &s, int count, int k, bool exact) {
    constexpr int N = kList / kTopThreads;
    uint64_t mine[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int at = i * kTopThreads + int(threadIdx.x);
        mine[i] = at < count ? s.list[at] : 0;
    }
    uint64_t bound = 0;
    if (!exact) {
        uint32_t hi[N];
#pragma unroll
        for (int i = 0; i < N; i++) hi[i] = uint32_t(mine[i] >> 32);
        bound = uint64_t(kth_bound<uint32_t, N>(s, hi, k, 2 * k)) << 32;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < N; i++) n += uint32_t(__popcll(__ballot(mine[i] >= bound)));
        n = group_sum(s, n, 0);
        __syncthreads();
        exact = int(n) > 2 * k;  // (equal values: by their columns too)
    }
    if (exact) bound = kth_bound<uint64_t, N>(s, mine, k, k);
    keep_from<N>(s, mine, bound);
    if (threadIdx.x == 0 && bound > 0 && bound - 1 > s.least) s.least = bound - 1;
    __syncthreads();
}

// The row's tokens from the list and its log-sum-exp (base in z, rest ln of the sum). Every thread.
__device__ __forceinline__ void top_finish(TopS &s, const TopP &p, int64_t row, double S, float a) {
    int32_t *ids = p.ids + row * p.k;
    float *logp = p.logp + row * p.k;
    int st = NT_ROW_OK;
    if (!(S == S)) st = NT_ROW_NAN;
    else if (a == -INFINITY) st = NT_ROW_NO_TOKEN;
    if (threadIdx.x == 0) p.status[row] = uint8_t(st);
    int n = s.count;
    if (n > kKeep) {
        cut_list(s, n, p.k, false);
        n = s.count;
    }
    if (st != NT_ROW_OK) n = 0;
    const double lse = double(a) * p.inv_t + log(S);
    for (int i = threadIdx.x; i < n; i += kTopThreads) {
        const uint64_t key = s.list[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += s.list[j] > key;
        if (rank < p.k) {
            ids[rank] = int32_t(~uint32_t(key));
            logp[rank] = float(double(unordered(uint32_t(key >> 32))) * p.inv_t - lse);
        }
    }
    for (int i = n + threadIdx.x; i < p.k; i += kTopThreads) {
        ids[i] = -1;
        logp[i] = st == NT_ROW_OK ? -INFINITY : NAN;
    }
}

// A workgroup's waves' sums.
__device__ __forceinline__ void waves_sum(const TopS &s, float c, double *S, float *a) {
    float m = s.a[0];
    for (int w = 1; w < kTopWaves; w++) m = fmaxf(m, s.a[w]);
    double t = 0.0;
    for (int w = 0; w < kTopWaves; w++)
        t += s.a[w] == -INFINITY ? s.S[w] : s.S[w] * exp2((double(s.a[w]) - double(m)) * double(c));
    *S = t;
    *a = m;
}

template <int DT, int MK, bool AL>
__global__ __launch_bounds__(kTopThreads) void k_top(TopP p) {
    // a tile: NC chunks a wave, held as 16-bit logits with the u8 mask folded in, or as f32 values
    constexpr bool HALF = DT != NT_F32 && MK != NT_MASK_F32;
    constexpr int NC = HALF ? 8 : 4, W = HALF ? 4 : 8, HDT = HALF ? DT : NT_F32;
    __shared__ TopS s;
    const int64_t row = blockIdx.x / unsigned(p.segs);
    const int seg = int(blockIdx.x % unsigned(p.segs));
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const void *xrow = static_cast<const char *>(p.x) + row * p.ld * Elem<DT>::kBytes;
    const void *mrow = nullptr;
    if constexpr (MK != NT_MASK_NONE) mrow = static_cast<const char *>(p.mask) + mask_row_at(p.mm, row) * MaskWords<MK>::kBytes;
    const bool tau_one = p.tau_one != 0;
    const int c1 = min(p.nc, (seg + 1) * p.per);
    if (threadIdx.x == 0) {
        s.count = 0;
        s.least = (uint64_t(kNone) << 32) | 0xffffffffu;
    }
    __syncthreads();
    double S = 0.0;
    float a = -INFINITY;
    bool bounded = false;  // (the list has a threshold of its own)
    for (int t0 = seg * p.per; t0 < c1; t0 += NC * kTopWaves) {
        Raw<DT, MK> raw[NC];
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const int ch = t0 + i * kTopWaves + wave;
            load_raw<DT, MK, AL>(raw[i], xrow, mrow, ch < c1 ? int64_t(ch) * kChunk + lane * kEpl : p.V, p.V);
        }
        uint32_t held[NC][W];
        float gm[NC];
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NC; i++) {
            float v[kEpl];
            decode<DT, MK>(raw[i], v, p.tau, tau_one);
#pragma unroll
            for (int j = 0; j < W; j++) held[i][j] = HALF ? raw[i].x[j] : __float_as_uint(v[j]);
            if constexpr (HALF && MK == NT_MASK_U8) fold_values<DT>(held[i], v);
            gm[i] = max8(v);
            m = fmaxf(m, gm[i]);
        }
        // the log-sum-exp's part, relative to the larger of the wave's maximum so far and the tile's
        m = fmaxf(wave_max(m), a);
        const float sh = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; i++) {
            float w[kEpl];
#pragma unroll
            for (int j = 0; j < kEpl; j++) w[j] = exp2_hw((logit<HDT>(held[i], j) - sh) * p.c);
            sum += tree8(w);
        }
        if (a != m && a != -INFINITY) S *= exp2((double(a) - double(m)) * double(p.c));
        S += wave_sum_d(double(sum));
        a = m;

        // the threshold, once k groups' maxima give one
        auto bound_by_groups = [&]() {
            uint32_t g[NC];
#pragma unroll
            for (int i = 0; i < NC; i++) g[i] = ordered(gm[i]);
            const uint32_t b = kth_bound<uint32_t, NC>(s, g, p.k, 2 * p.k);
            if (threadIdx.x == 0 && b > kNone && (uint64_t(b) << 32) - 1 > s.least) s.least = (uint64_t(b) << 32) - 1;
            __syncthreads();
            return b > kNone;
        };
        // the elements of chunks i0 .. i1 - 1 above the threshold, as far as the list holds them
        auto append = [&](int i0, int i1) {
            const uint64_t least = s.least;
            const float lf = unordered(uint32_t(least >> 32));
#pragma unroll
            for (int i = 0; i < NC; i++) {
                if (i < i0 || i >= i1 || __ballot(gm[i] >= lf) == 0) continue;
                const uint32_t e0 = uint32_t(t0 + i * kTopWaves + wave) * kChunk + lane * kEpl;
#pragma unroll
                for (int j = 0; j < kEpl; j++) {
                    const float v = logit<HDT>(held[i], j);
                    const uint64_t key = (uint64_t(ordered(v)) << 32) | uint32_t(~(e0 + j));
                    const bool in = v >= lf && key > least;
                    const uint64_t b = __ballot(in);
                    if (b == 0) continue;
                    int at = 0;
                    if (lane == int(__builtin_ctzll(b))) at = atomicAdd(&s.count, int(__popcll(b)));
                    at = __builtin_amdgcn_readlane(at, __builtin_ctzll(b)) + int(__popcll(b & ((uint64_t(1) << lane) - 1)));
                    if (in && at < kList) s.list[at] = key;
                }
            }
        };
        if (!bounded) bounded = bound_by_groups();
        const int before = s.count;
        __syncthreads();
        append(0, NC);
        __syncthreads();
        int n = s.count;
        __syncthreads();
        if (n > kList) {
            // more than the list holds: once more with the tile's own threshold, and if that does not help in groups
            if (threadIdx.x == 0) s.count = before;
            __syncthreads();
            bounded = bound_by_groups() || bounded;
            append(0, NC);
            __syncthreads();
            n = s.count;
            __syncthreads();
            if (n > kList) {
                if (threadIdx.x == 0) s.count = before;
                n = before;
                __syncthreads();
                for (int i = 0; i < NC; i++) {
                    if (n > p.k) cut_list(s, n, p.k, true);
                    append(i, i + 1);
                    __syncthreads();
                    n = s.count;
                    __syncthreads();
                }
            }
        }
        if (n > max(kKeep, 2 * p.k)) {
            cut_list(s, n, p.k, false);
            bounded = true;
        }
    }
    if (lane == 0) {
        s.S[wave] = S;
        s.a[wave] = a;
    }
    __syncthreads();
    waves_sum(s, p.c, &S, &a);
    if (p.segs == 1) {
        top_finish(s, p, row, S, a);
        return;
    }
    int n = s.count;
    if (n > 2 * p.k) {
        cut_list(s, n, p.k, false);
        n = s.count;
    }
    const int64_t at = row * p.segs + seg;
    for (int i = threadIdx.x; i < n; i += kTopThreads) p.cand[at * 2 * p.k + i] = s.list[i];
    if (threadIdx.x == 0) p.rec[at] = TopRec{S, a, n};
}

// The rows of a launch with several workgroups a row.
__global__ __launch_bounds__(kTopThreads) void k_top_finish(TopP p) {
    __shared__ TopS s;
    const int64_t row = blockIdx.x;
    const TopRec *rec = p.rec + row * p.segs;
    if (threadIdx.x == 0) {
        s.count = 0;
        s.least = 0;
    }
    float a = -INFINITY;
    for (int g = 0; g < p.segs; g++) a = fmaxf(a, rec[g].a);
    double S = 0.0;
    for (int g = 0; g < p.segs; g++)
        S += rec[g].a == -INFINITY ? rec[g].S : rec[g].S * exp2((double(rec[g].a) - double(a)) * double(p.c));
    int n = 0;
    __syncthreads();
    for (int g = 0; g < p.segs; g++) {
        const int more = rec[g].n;
        if (n + more > kList) {
            cut_list(s, n, p.k, true);
            n = s.count;
            __syncthreads();
        }
        for (int i = threadIdx.x; i < more; i += kTopThreads) s.list[n + i] = p.cand[(row * p.segs + g) * 2 * p.k + i];
        n += more;
        __syncthreads();
        if (threadIdx.x == 0) s.count = n;
        __syncthreads();
    }
    top_finish(s, p, row, S, a);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" int nt_hip_rl_top_logprobs(const NtRlTopArgs *a) {
    const char *who = "nt_hip_rl_top_logprobs";
    if (!a) return fail(NT_E_ARG, std::string(who) + ": null args");
    if (int rc = check_rows(a->rows, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, a->mask_ld, who)) return rc;
    MaskMap mm;
    if (int rc = mask_map(a->mask_rows, a->rows, a->vocab, a->mask_kind, a->mask_ld, who, &mm)) return rc;
    if (!(a->temperature > 0.0) || !std::isfinite(a->temperature))
        return fail(NT_E_ARG, "tempered_logits: temperature " + std::to_string(a->temperature) + " (must be positive)");
    if (a->k < 1 || a->k > kMaxK || a->k > a->vocab)
        return fail(NT_E_ARG, "top_logprobs: k " + std::to_string(a->k) + " of " + std::to_string(a->vocab) +
                                  " tokens (1 to min(vocab, " + std::to_string(kMaxK) + "))");
    // (a launch holds fewer than 2^32 threads; columns are counted in 32 bits)
    if (a->vocab > 0x7fffffffLL - 16 * kChunk || a->rows > 0xffffffLL)
        return fail(NT_E_ARG, std::string(who) + ": rows past 2^24 or vocab past 2^31");
    if (!a->logits || !a->ids || !a->logp || !a->status) return fail(NT_E_ARG, std::string(who) + ": null logits or outputs");
    std::unique_lock<std::mutex> lk;
    if (int rc = enter(&lk)) return rc;
    if (a->rows == 0) return 0;
    TopP p{};
    p.x = a->logits;
    p.mask = a->mask;
    p.V = a->vocab;
    p.ld = a->ld;
    p.mm = mm;
    p.tau = float(a->temperature);
    p.tau_one = a->temperature == 1.0;
    const bool added = a->mask_kind == NT_MASK_F32;
    p.c = added || p.tau_one ? kLog2e : float(double(kLog2e) / a->temperature);
    p.inv_t = added ? 1.0 : 1.0 / a->temperature;
    p.k = int(a->k);
    p.nc = int((a->vocab + kChunk - 1) / kChunk);
    // About 1024 workgroups, each of a chunk per wave or more.
    p.segs = int(std::max<int64_t>(1, std::min<int64_t>({1024 / a->rows, int64_t(kTopSegs), (p.nc + kTopWaves - 1) / kTopWaves})));
    p.per = (p.nc + p.segs - 1) / p.segs;
    p.segs = (p.nc + p.per - 1) / p.per;
    p.ids = a->ids;
    p.logp = a->logp;
    p.status = a->status;
    void *ws = nullptr;
    if (p.segs > 1) {
        const size_t n = size_t(a->rows) * size_t(p.segs), recs = n * sizeof(TopRec), need = recs + n * 16 * size_t(p.k);
        bool cap = false;
        if (int rc = stream_capturing(&cap)) return rc;
        if (cap && need >= size_t(1) << 20)
            return fail(NT_E_UNSUPPORTED, std::string(who) + ": a workspace of " + std::to_string(need) +
                                              " bytes under stream capture (less than 1 MiB)");
        if (int rc = scratch_alloc(need, &ws)) return rc;
        p.rec = static_cast<TopRec *>(ws);
        p.cand = reinterpret_cast<uint64_t *>(static_cast<char *>(ws) + recs);
    }
    const bool al = aligned_rows(a->logits, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, mm);
    hipStream_t s = ctx().stream;
    const dim3 grid(unsigned(a->rows * p.segs));
    auto by_al = [&](auto dt, auto mk) {
        constexpr int DT = decltype(dt)::value, MK = decltype(mk)::value;
        if (al) hipLaunchKernelGGL((k_top<DT, MK, true>), grid, dim3(kTopThreads), 0, s, p);
        else hipLaunchKernelGGL((k_top<DT, MK, false>), grid, dim3(kTopThreads), 0, s, p);
    };
    auto by_mk = [&](auto dt) {
        if (a->mask_kind == NT_MASK_U8) by_al(dt, std::integral_constant<int, NT_MASK_U8>{});
        else if (a->mask_kind == NT_MASK_F32) by_al(dt, std::integral_constant<int, NT_MASK_F32>{});
        else by_al(dt, std::integral_constant<int, NT_MASK_NONE>{});
    };
    if (a->dtype == NT_F32) by_mk(std::integral_constant<int, NT_F32>{});
    else if (a->dtype == NT_BF16) by_mk(std::integral_constant<int, NT_BF16>{});
    else by_mk(std::integral_constant<int, NT_F16>{});
    if (p.segs > 1) hipLaunchKernelGGL(k_top_finish, dim3(unsigned(a->rows)), dim3(kTopThreads), 0, s, p);
    const int rc = launched(who);
    const int rc2 = scratch_release(ws);
    return rc ? rc : rc2;
}
