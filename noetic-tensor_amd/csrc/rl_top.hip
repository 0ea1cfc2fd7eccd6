// nt_hip_rl_top_logprobs: the k most likely tokens of each row and their log-probabilities, in one pass.
//
// A workgroup streams its row (or, where rows are few, a piece of one) once, and takes from it the log-sum-exp and the
// largest value of each group of columns: a lane's columns in a sixteenth of the row.
// With t the k-th largest of those maxima (joined to 256, 512 or 1024 for few k), k groups reach t, so k columns do, and the columns
// that reach it lie in groups whose maximum does: those few groups are read again, from the caches, and hardly more than k
// columns (1.4 k at the most) go on a list in LDS. A column's place is the number of listed ones above it.
// Values are compared as 64 bits, the f32 made an ordered integer over the complement of its column, so that
// no two are equal and ties go to the lowest column. Where the list does not hold what reaches t (many equal
// values), the row goes through it in order, a few hundred columns at a time, and it is cut to its k
// largest whenever it fills.
//
// What bounds it: the row's bytes (64 of 4096 x 50304 bf16: 86 us, 4.8 TB/s), and after each row's stream some 8 us of
// counting, reading again and placing, which other workgroups' streams hide where there are rounds of them.
#include <algorithm>

#include "nt_rows.hpp"
#include "nt_rowsum.hpp"

namespace nt {
namespace {

constexpr int kTopThreads = 256;
constexpr int kTopWaves = kTopThreads / kWave;
constexpr int kMaxK = 1024;
constexpr int kFewK = 256;           
constexpr int kTopSegs = 64;         // pieces of a row, at most
constexpr int kTopAhead = 4;         // chunks a wave loads ahead

// The two forms, k up to kFewK and past it: G groups a lane, the list's length, and the chunks that go through it at a time in order.
template <bool BIG>
struct TopForm {
    static constexpr int G = 16, kList = BIG ? 4096 : 1024, kRound = BIG ? 4 : 1;
    static_assert((BIG ? kMaxK : kFewK) + kRound * kChunk <= kList, "a cut list and a round more");
};

// A piece's part of the row's log-sum-exp: S relative to a; n candidates follow.
struct TopRec {
    double S, a;
    int64_t n;
};

struct TopP {
    const void *x, *mask;
    int64_t V, ld;
    MaskMap mm;
    double c, low;      // exponent scale of a value: log2(e) / T (none, u8) or log2(e) (f32 mask); -1100 / c
    float c32, tau;
    int tau_one;
    double inv_t;       // value -> z: 1 / T, or 1 with an f32 mask
    int k;
    int nc;             // chunks of a row
    int segs, per;      // pieces of a row, chunks each
    int32_t *ids;
    float *logp;
    uint8_t *status;
    TopRec *rec;        // segs > 1: [rows][segs]
    uint64_t *cand;     // segs > 1: [rows][segs][cand_of(k)]
};

// How many candidates a piece hands on, at most.
__host__ __device__ __forceinline__ int cand_of(int k) { return k + k / 4 + 32; }

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
template <bool BIG>
struct TopS {
    uint64_t list[TopForm<BIG>::kList];
    float gmax[TopForm<BIG>::G * kTopThreads];  // the groups' maxima
    uint64_t sums[2][kTopWaves];
    int count, groups;
    double S[kTopWaves], a[kTopWaves];
};

// The largest found t such that at least k of the workgroup's N keys a lane are t or more, as soon as no more than
// `most` are (two bits at a time from the top; exact when it reaches the last). 0 where there are not k keys but 0.
template <class T, int N, bool BIG>
__device__ __forceinline__ T kth_bound(TopS<BIG> &s, const T (&key)[N], int k, int most) {
    T t = 0;
    int turn = 0;
    for (int bit = int(sizeof(T)) * 8 - 2; bit >= 0; bit -= 2) {
        // (three counts of at most 2^10 x 4 waves in a word)
        uint64_t n = 0;
#pragma unroll
        for (int d = 1; d < 4; d++) {
            const T up = t | (T(d) << bit);
            uint32_t one = 0;
#pragma unroll
            for (int i = 0; i < N; i++) one += uint32_t(__popcll(__ballot(key[i] >= up)));
            n |= uint64_t(one) << (16 * d);
        }
        if ((threadIdx.x & (kWave - 1)) == 0) s.sums[turn & 1][threadIdx.x / kWave] = n;
        __syncthreads();
        n = 0;
#pragma unroll
        for (int w = 0; w < kTopWaves; w++) n += s.sums[turn & 1][w];
        turn++;
        int d = 3;
        while (d > 0 && int((n >> (16 * d)) & 0xffff) < k) d--;
        t |= T(d) << bit;
        if (d > 0 && int((n >> (16 * d)) & 0xffff) <= most) break;
    }
    __syncthreads();  // (the sums' buffers are free again)
    return t;
}

// Cut the list of `n` entries to its k largest; the k-th of them. The whole workgroup.
template <bool BIG>
__device__ __forceinline__ uint64_t cut_list(TopS<BIG> &s, int n, int k) {
    constexpr int N = TopForm<BIG>::kList / kTopThreads;
    uint64_t mine[N];
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int at = i * kTopThreads + int(threadIdx.x);
        mine[i] = at < n ? s.list[at] : 0;
    }
    const uint64_t bound = kth_bound<uint64_t, N, BIG>(s, mine, k, k);
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const bool in = mine[i] >= bound && mine[i] != 0;
        const uint64_t b = __ballot(in);
        if (b == 0) continue;
        int at = 0;
        if (lane == int(__builtin_ctzll(b))) at = atomicAdd(&s.count, int(__popcll(b)));
        at = __builtin_amdgcn_readlane(at, __builtin_ctzll(b));
        if (in) s.list[at + __popcll(b & ((uint64_t(1) << lane) - 1))] = mine[i];
    }
    __syncthreads();
    return bound;
}

// The row's tokens from the list of n and its log-sum-exp. Every thread.
template <bool BIG>
__device__ __forceinline__ void top_finish(TopS<BIG> &s, const TopP &p, int64_t row, int n, double S, double a) {
    int32_t *ids = p.ids + row * p.k;
    float *logp = p.logp + row * p.k;
    int st = NT_ROW_OK;
    if (!(S == S)) st = NT_ROW_NAN;
    else if (a == -INFINITY) st = NT_ROW_NO_TOKEN;
    if (threadIdx.x == 0) p.status[row] = uint8_t(st);
    if (st != NT_ROW_OK) n = 0;
    const double ln_s = log(S);
    for (int i = threadIdx.x; i < n; i += kTopThreads) {
        const uint64_t key = s.list[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) rank += s.list[j] > key;
        if (rank < p.k) {
            ids[rank] = int32_t(~uint32_t(key));
            logp[rank] = float((double(unordered(uint32_t(key >> 32))) - a) * p.inv_t - ln_s);
        }
    }
    for (int i = n + threadIdx.x; i < p.k; i += kTopThreads) {
        ids[i] = -1;
        logp[i] = st == NT_ROW_OK ? -INFINITY : NAN;
    }
}

// Sums relative to a of the lanes' own, over the wave.
__device__ __forceinline__ void wave_merge(const TopP &p, double &S, double &a) {
    const double m = wave_max_d(a);
    S = wave_sum_d(moved(S, a, m, p.c, p.low));
    a = m;
}

template <int DT, int MK, bool AL, bool BIG>
__global__ __launch_bounds__(kTopThreads) void k_top(TopP p) {
    using F = TopForm<BIG>;
    __shared__ TopS<BIG> s;
    const int64_t row = blockIdx.x / unsigned(p.segs);
    const int seg = int(blockIdx.x % unsigned(p.segs));
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / kWave));
    const void *xrow = static_cast<const char *>(p.x) + row * p.ld * Elem<DT>::kBytes;
    const void *mrow = nullptr;
    if constexpr (MK != NT_MASK_NONE) mrow = static_cast<const char *>(p.mask) + mask_row_at(p.mm, row) * MaskWords<MK>::kBytes;
    const RowLoad<DT, MK, AL> in(xrow, mrow, p.V, p.nc);
    const bool tau_one = p.tau_one != 0;
    const int c0 = seg * p.per, c1 = min(p.nc, c0 + p.per);
    // the wave's chunks are c0 + wave + 4 j; group q of a lane has j in [q cpg, q cpg + cpg)
    const int J = (c1 - c0 + kTopWaves - 1) / kTopWaves, cpg = (J + F::G - 1) / F::G;
    if (threadIdx.x == 0) s.count = s.groups = 0;
    LaneSums sum;
    float gm = -INFINITY;
    int q = 0, left = cpg;
    Raw<DT, MK> raw[kTopAhead];
    auto load = [&](auto i, int ch) { in.load(raw[i.value], ch, lane, ch < c1); };
    stream<kTopAhead>(c0 + wave, kTopWaves, c1, load, [&](auto i, int ch, int next) {
        float v[kEpl];
        decode_e<DT, MK, kEpl>(raw[i.value].x, raw[i.value].m, v, p.tau, tau_one);
        in.clean(v, ch, lane);
        load(i, next);
        const float top = sum.add(v, p.c32);
        gm = max3_hw(gm, top, top);
        if (--left == 0) {
            s.gmax[q++ * kTopThreads + threadIdx.x] = gm;
            gm = -INFINITY;
            left = cpg;
        }
    });
    for (; q < F::G; q++) {
        s.gmax[q * kTopThreads + threadIdx.x] = gm;
        gm = -INFINITY;
    }
    double S = sum.S, a = sum.at(p.c, p.c32);
    wave_merge(p, S, a);
    if (lane == 0) {
        s.S[wave] = S;
        s.a[wave] = a;
    }
    // the threshold: what is on the list is above `least`. Of the largest of all a lane's groups where there are four lanes for
    // each of the k, of pairs or fours of them else: k of those reach it too, and they are fewer to count.
    uint32_t g[F::G];
#pragma unroll
    for (int i = 0; i < F::G; i++) g[i] = ordered(s.gmax[i * kTopThreads + threadIdx.x]);  // (this thread's own)
    const auto of_groups = [&](auto n) {
        constexpr int N = decltype(n)::value;
        uint32_t h[N];
#pragma unroll
        for (int i = 0; i < N; i++) h[i] = g[i];
#pragma unroll
        for (int i = N; i < F::G; i++) h[i % N] = max(h[i % N], g[i]);
        return kth_bound<uint32_t, N, BIG>(s, h, p.k, p.k + p.k / 8 + 16);
    };
    uint32_t bound;
    if constexpr (BIG) bound = of_groups(std::integral_constant<int, F::G>{});
    else if (p.k <= 64) bound = of_groups(std::integral_constant<int, 1>{});
    else if (p.k <= 128) bound = of_groups(std::integral_constant<int, 2>{});
    else bound = of_groups(std::integral_constant<int, 4>{});
    if (bound <= kNone) bound = kNone + 1;
    const float lf = unordered(bound);
    uint64_t least = (uint64_t(bound) << 32) - 1;
    // the groups that reach it, their numbers where their maxima were
    uint16_t *group = reinterpret_cast<uint16_t *>(s.gmax);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < F::G; q++) {
        const bool in = g[q] >= bound;
        const uint64_t b = __ballot(in);
        if (b == 0) continue;
        int at = 0;
        if (lane == int(__builtin_ctzll(b))) at = atomicAdd(&s.groups, int(__popcll(b)));
        at = __builtin_amdgcn_readlane(at, __builtin_ctzll(b));
        if (in) group[at + __popcll(b & ((uint64_t(1) << lane) - 1))] = uint16_t(q * kTopThreads + threadIdx.x);
    }
    __syncthreads();
    // v and its column, if it goes on the list: where, or kList and more where that is full
    auto append = [&](float v, int64_t e) {
        const uint64_t key = (uint64_t(ordered(v)) << 32) | uint32_t(~uint32_t(e));
        if (!(v >= lf) || v == -INFINITY || key <= least) return;
        const int at = atomicAdd(&s.count, 1);
        if (at < F::kList) s.list[at] = key;
    };
    // (four of their chunks a thread at a time: each costs a load's latency otherwise, 11 us of a row of 151936 f32)
    const int items = s.groups * cpg;
    constexpr int kItems = 4;
    for (int t0 = threadIdx.x; t0 < items; t0 += kItems * kTopThreads) {
        Raw<DT, MK> part[kItems];
        int at[kItems], of[kItems];
#pragma unroll
        for (int i = 0; i < kItems; i++) {
            const int it = min(t0 + i * kTopThreads, items - 1), id = group[it / cpg], thread = id % kTopThreads;
            const int j = id / kTopThreads * cpg + it % cpg, ch = c0 + thread / kWave + j * kTopWaves;
            const bool some = t0 + i * kTopThreads < items && j < J && ch < c1;
            at[i] = some ? ch : -1;
            of[i] = thread % kWave;
            in.load(part[i], some ? ch : c0, of[i]);
        }
#pragma unroll
        for (int i = 0; i < kItems; i++) {
            // (other threads are adding to the count: a look at it, which only ends work early)
            if (at[i] < 0 || __hip_atomic_load(&s.count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) > F::kList) continue;
            float v[kEpl];
            decode_e<DT, MK, kEpl>(part[i].x, part[i].m, v, p.tau, tau_one);
            in.clean(v, at[i], of[i]);
#pragma unroll
            for (int e = 0; e < kEpl; e++) append(v[e], in.col(at[i], of[i], e));
        }
    }
    __syncthreads();
    int n = s.count;
    __syncthreads();
    if (n > F::kList) {
        // too many reach it (equal values): in the columns' order, the list cut whenever a round might not fit
        if (threadIdx.x == 0) s.count = 0;
        n = 0;
        __syncthreads();
        for (int t0 = c0; t0 < c1; t0 += F::kRound) {
            if (n > F::kList - F::kRound * kChunk) {
                least = cut_list(s, n, p.k);
                __syncthreads();
            }
            if (wave < F::kRound && t0 + wave < c1) {
                const int64_t e0 = int64_t(t0 + wave) * kChunk + lane * kEpl;
                Raw<DT, MK> raw;
                float v[kEpl];
                load_raw<DT, MK, AL>(raw, xrow, mrow, e0, p.V);
                decode_e<DT, MK, kEpl>(raw.x, raw.m, v, p.tau, tau_one);
#pragma unroll
                for (int e = 0; e < kEpl; e++) append(v[e], e0 + e);
            }
            __syncthreads();
            n = s.count;
            __syncthreads();
        }
    }
    // (placing 512 entries costs less than cutting them)
    if (n > (p.segs > 1 ? cand_of(p.k) : max(2 * p.k, 512))) {
        cut_list(s, n, p.k);
        n = p.k;
    }
    a = s.a[0];
    for (int w = 1; w < kTopWaves; w++) a = fmax(a, s.a[w]);
    S = 0.0;
    for (int w = 0; w < kTopWaves; w++) S += moved(s.S[w], s.a[w], a, p.c, p.low);
    if (p.segs == 1) {
        top_finish(s, p, row, n, S, a);
        return;
    }
    const int64_t at = row * p.segs + seg;
    for (int i = threadIdx.x; i < n; i += kTopThreads) p.cand[at * cand_of(p.k) + i] = s.list[i];
    if (threadIdx.x == 0) p.rec[at] = TopRec{S, a, n};
}

// The rows of a launch with several workgroups a row.
template <bool BIG>
__global__ __launch_bounds__(kTopThreads) void k_top_finish(TopP p) {
    using F = TopForm<BIG>;
    __shared__ TopS<BIG> s;
    __shared__ int first[kTopSegs + 1];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const TopRec *rec = p.rec + row * p.segs;
    // (every wave the same: a piece a lane)
    TopRec r{0.0, -INFINITY, 0};
    if (lane < p.segs) r = rec[lane];
    double S = r.S, a = r.a;
    wave_merge(p, S, a);
    int before = int(r.n);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int m = __shfl_up(before, o, kWave);
        if (lane >= o) before += m;
    }
    if (wave == 0) first[lane + 1] = before;
    if (threadIdx.x == 0) first[0] = s.count = 0;
    __syncthreads();
    const int stride = cand_of(p.k);
    const uint64_t *cand = p.cand + row * p.segs * stride;
    const int all = first[kTopSegs];
    int n;
    if (all <= F::kList) {
        for (int g = wave; g < p.segs; g += kTopWaves)
            for (int i = lane; i < first[g + 1] - first[g]; i += kWave) s.list[first[g] + i] = cand[g * stride + i];
        n = all;
        __syncthreads();
    } else {
        // a round of the list's free places at a time
        n = 0;
        for (int g = 0; g < p.segs; g++) {
            const int more = first[g + 1] - first[g];
            for (int i0 = 0; i0 < more;) {
                if (n == F::kList) {
                    cut_list(s, n, p.k);
                    n = p.k;
                    __syncthreads();
                }
                const int take = min(more - i0, F::kList - n);
                for (int i = threadIdx.x; i < take; i += kTopThreads) s.list[n + i] = cand[g * stride + i0 + i];
                n += take;
                i0 += take;
                __syncthreads();
            }
        }
    }
    if (n > max(2 * p.k, 512)) {
        cut_list(s, n, p.k);
        n = p.k;
    }
    top_finish(s, p, row, n, S, a);
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
    if (int rc = check_scale(a->temperature)) return rc;
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
    p.c = added ? kLog2e64 : kLog2e64 / a->temperature;
    p.c32 = float(p.c);
    p.low = -1100.0 / p.c;
    p.inv_t = added ? 1.0 : 1.0 / a->temperature;
    p.k = int(a->k);
    p.nc = int((a->vocab + kChunk - 1) / kChunk);
    // Up to 512 workgroups, each of 120 chunks or more (the finishing launch is worth about as many: 1 row of 50257 bf16 16.7 us in
    // one piece, 23.3 in four; 64 of 128256 24.2 in one, 22.9 in two, 31 in four), and no more of a row than what they hand on (k
    // and a quarter and 16 each) can be placed together.
    p.segs = int(std::max<int64_t>(1, std::min<int64_t>({512 / a->rows, int64_t(kTopSegs), int64_t(p.nc / 120),
                                                         (p.k > kFewK ? 4096 : 512) / (p.k + p.k / 4 + 16)})));
    p.per = (p.nc + p.segs - 1) / p.segs;
    p.segs = (p.nc + p.per - 1) / p.per;
    p.ids = a->ids;
    p.logp = a->logp;
    p.status = a->status;
    void *ws = nullptr;
    if (p.segs > 1) {
        const size_t n = size_t(a->rows) * size_t(p.segs), recs = n * sizeof(TopRec), need = recs + n * 8 * size_t(cand_of(p.k));
        bool cap = false;
        if (int rc = stream_capturing(&cap)) return rc;
        if (cap && need >= size_t(1) << 20)
            return fail(NT_E_UNSUPPORTED, std::string(who) + ": a workspace of " + std::to_string(need) +
                                              " bytes under stream capture (less than 1 MiB)");
        if (int rc = scratch_alloc(need, &ws)) return rc;
        p.rec = static_cast<TopRec *>(ws);
        p.cand = reinterpret_cast<uint64_t *>(static_cast<char *>(ws) + recs);
    }
    const bool al = aligned_rows(a->logits, a->vocab, a->ld, a->dtype, a->mask_kind, a->mask, mm) && a->vocab * 4 <= 0x7fffffffLL;
    hipStream_t s = ctx().stream;
    const dim3 grid(unsigned(a->rows * p.segs));
    auto by_al = [&](auto dt, auto mk) {
        constexpr int DT = decltype(dt)::value, MK = decltype(mk)::value;
        auto by_k = [&](auto big) {
            constexpr bool BIG = decltype(big)::value;
            if (al) hipLaunchKernelGGL((k_top<DT, MK, true, BIG>), grid, dim3(kTopThreads), 0, s, p);
            else hipLaunchKernelGGL((k_top<DT, MK, false, BIG>), grid, dim3(kTopThreads), 0, s, p);
            if (p.segs > 1) hipLaunchKernelGGL(k_top_finish<BIG>, dim3(unsigned(a->rows)), dim3(kTopThreads), 0, s, p);
        };
        if (p.k > kFewK) by_k(std::true_type{});
        else by_k(std::false_type{});
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
