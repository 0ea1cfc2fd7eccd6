// A matrix product's output tile on the matrix cores of gfx950, from operands in their natural row-major
// layouts: acc[m][n] = sum_k A(m, k) B(n, k), 16-bit floats with f32 sums or 8-bit integers with 32-bit
// ones. Shared by the training readout (rl_readout_train.hip) and the 8-bit product (int8.hip).
//
// An operand is k-contiguous (row m at base + m ld, its k bytes side by side) or, for 16-bit types,
// transposed (TR: row k at base + k ld, its m side by side), so that a product and both of its gradients
// read the same tensors: logits = H W^T, dH = G W, dW = G^T H, none of them copied or transposed first.
//
// A workgroup of WM x WN waves owns a (32 TM WM) x (32 TN WN) tile, a wave 32 TM x 32 TN of it as TM x TN MFMA
// tiles of 32 x 32. k goes by stages of 64 bytes of a row (32 k of a 16-bit type, 64 of an 8-bit one): both
// operands' panels are copied by the load unit straight into LDS.
//
// LDS: a k-contiguous panel is [row][64 bytes], the four 16-byte chunks of row r at chunk c ^ (r / 4 % 4); a
// transposed one is [32 k][2 B bytes], row k's 64-byte units at u ^ f(k). So the reads below (one 16-byte
// chunk of 32 rows, or 4 k of 32 columns by ds_read_b64_tr_b16) touch every bank once per pass. The load
// unit writes LDS lane by lane, so it is the global address of each lane that is permuted.
//
// Rows past the operand's last, k past its end, whole stages past it and a transposed operand's columns past its last
// (what is behind a row, a NaN too, would pass an additive mask's -inf) read as zeros through the buffer resource's
// range and touch no memory; a row's bytes count is a multiple of 16 (callers pad).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

namespace nt {
namespace tile {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void *lds_ptr;

// The element types: one MFMA takes 16 bytes of k of 32 rows from each half of the wave.
struct Bf16 {
    typedef f32x16 Acc;
    static __device__ __forceinline__ Acc mfma(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};
struct F16 {
    typedef f32x16 Acc;
    static __device__ __forceinline__ Acc mfma(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
};
struct I8 {
    typedef i32x16 Acc;
    static __device__ __forceinline__ Acc mfma(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0,
                                                     0);
    }
};

// One operand of a tile: its first row (k-contiguous) or column (TR), the byte stride between rows, the rows
// there are (k-contiguous: of the operand's own; TR: of k) from there, and their bytes from there (a multiple
// of 16; k-contiguous: the bytes of k). Nothing past the last row's last byte is read.
struct Operand {
    const uint8_t *base;
    int64_t ld;
    int64_t rows;
    int64_t width;
};

constexpr int kWord3 = 0x00020000;
constexpr int kStageK = 64;  // bytes of a k-contiguous row per stage; a transposed operand's 32 rows

template <int... I, class F>
__device__ __forceinline__ void unrolled(std::integer_sequence<int, I...>, F &&f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F &&f) {
    unrolled(std::make_integer_sequence<int, N>{}, f);
}

// One operand's side of a tile of B rows (or columns, TR): its copies into LDS and its fragment reads.
template <int B, int NW, bool TR>
struct Side {
    static constexpr int kCopies = B / 16 / NW;  // of 1 KiB, per wave and stage
    static constexpr int kBytes = B * kStageK;   // of a stage
    static constexpr int kAddr = TR ? 4 : 2;
    static_assert(B % (16 * NW) == 0, "whole copies per wave");
    uint32_t voff[kCopies];  // this lane's source bytes from the stage's base
    int chunk;               // k-contiguous: this lane's 16-byte chunk of the stage
    const uint8_t *base;
    int64_t ld, rows, width;
    uint32_t addr[kAddr];

    static __device__ __forceinline__ int swz(int k) { return B == 64 ? (k >> 1) & 1 : k & 3; }

    // Where byte `at` of row k of a stage lies (TR).
    static __device__ __forceinline__ int at(int k, int at) { return k * 2 * B + ((at / 64) ^ swz(k)) * 64 + at % 64; }

    __device__ __forceinline__ void init(const Operand &o, int wave, int lane, int first_tile) {
        base = o.base, ld = o.ld, width = o.width;
        rows = !TR && o.rows > B ? B : o.rows;
#pragma unroll
        for (int q = 0; q < kCopies; q++) {
            const int slot = wave * kCopies + q;
            if constexpr (!TR) {
                const int row = 16 * slot + lane / 4;
                chunk = (lane % 4) ^ ((row >> 2) & 3);
                voff[q] = uint32_t(row * ld) + chunk * 16;
            } else {
                constexpr int kRow = 2 * B;  // bytes of a row in LDS
                const int k = (1024 / kRow) * slot + lane * 16 / kRow;
                const int at = ((lane % (kRow / 16)) ^ (swz(k) << 2)) * 16;
                voff[q] = at < width ? uint32_t(k * ld) + at : 0x80000000u;
            }
        }
        if constexpr (!TR)
            src[0] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), short(0), int((rows - 1) * ld + width), kWord3);
        reads(lane, first_tile);
    }
    // Where the fragments of this lane lie in a stage, from tile `first_tile` of 32 rows on.
    __device__ __forceinline__ void reads(int lane, int first_tile) {
        if constexpr (!TR) {
            const int row = 32 * first_tile + lane % 32, s = (row >> 2) & 3;
            addr[0] = row * kStageK + ((lane / 32) ^ s) * 16;
            addr[1] = row * kStageK + ((2 + lane / 32) ^ s) * 16;
        } else {
            const int k = 8 * (lane / 32) + (lane % 16) / 4;  // + 16 j + 4 e, which do not change swz(k)
#pragma unroll
            for (int i = 0; i < 4; i++)
                addr[i] = k * 2 * B + ((first_tile + i) ^ swz(k)) * 64 + ((lane / 16) % 2) * 32 + (lane % 4) * 8;
        }
    }

    // The copies of stages `t` (even) and t + 1: begin(t), then each by the half it belongs to, into `lds` (this
    // operand's part of that stage's buffer).
    __amdgpu_buffer_rsrc_t src[TR ? 2 : 1];
    uint32_t koff[2];
    __device__ __forceinline__ void begin(int t) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if constexpr (!TR) {
                // a chunk past the row's end is pushed past the range
                const uint32_t k0 = (t + h) * kStageK;
                koff[h] = int64_t(k0) + chunk * 16 < width ? k0 : 0x80000000u;
            } else {
                const int64_t k0 = int64_t(t + h) * 32, left = rows - k0;
                const int64_t bytes = left <= 0 ? 0 : (left < 32 ? left - 1 : 31) * ld + width;
                src[h] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base + (left <= 0 ? 0 : k0 * ld)), short(0),
                                                           int(bytes), kWord3);
            }
        }
    }
    template <int Q, int H>
    __device__ __forceinline__ void copy(uint8_t *lds, int wave) const {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(src[TR ? H : 0], (lds_ptr)(lds + (wave * kCopies + Q) * 1024), 16,
                                                 TR ? voff[Q] : voff[Q] + koff[H], 0, 0, 0);
    }

    // The fragments of one k half of a stage: T tiles of 32 rows, by one read each (k-contiguous) or two (TR).
    static constexpr int kReads = TR ? 2 : 1;
    typedef typename std::conditional<TR, u32x2, u32x4>::type Part;

    // Read R of half J (`at`: the stage's LDS address plus this operand's), issued only: the register is in
    // flight until landed() below.
    template <int R, int J>
    __device__ __forceinline__ void issue(uint32_t at, Part &d) const {
        if constexpr (!TR)
            asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(d) : "v"(at + addr[J]), "i"(R * 32 * kStageK) : "memory");
        else
            asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2"
                         : "=v"(d)
                         : "v"(at + addr[R / 2]), "i"(J * 32 * B + (R % 2) * 8 * B)
                         : "memory");
    }
    template <int N>
    static __device__ __forceinline__ u32x4 fragment(const Part (&f)[N], int i) {
        if constexpr (!TR) return f[i];
        else return u32x4{f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y};
    }
};

// The wait for every LDS read issued, and each register taken through it: nothing that uses one can be placed
// before, and none is free while its read is in flight.
template <class P, int N, class Q, int M>
__device__ __forceinline__ void landed(P (&a)[N], Q (&b)[M]) {
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a[0]) : : "memory");
#pragma unroll
    for (int i = 1; i < N; i++) asm volatile("" : "+v"(a[i]) : : "memory");
#pragma unroll
    for (int i = 0; i < M; i++) asm volatile("" : "+v"(b[i]) : : "memory");
}

// The tile. Lane l of wave (wm, wn) holds in acc[i][j][v] the output of row 32 (TM wm + i) + l % 32 at column
// 32 (TN wn + j) + 8 (v / 4) + 4 (l / 32) + v % 4: B is the MFMA's first operand, so that a lane's values are
// of one row and by four of neighbouring columns.
template <class E, int TM, int TN, int WM, int WN, bool ATR, bool BTR, int PAIRS = 2>
struct Tile {
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    typedef Side<BM, kWaves, ATR> SideA;
    typedef Side<BN, kWaves, BTR> SideB;
    static constexpr int kStageBytes = SideA::kBytes + SideB::kBytes;
    static constexpr int kStages = 2 * PAIRS + 1;
    static constexpr int kLds = kStages * kStageBytes;
    static constexpr int kCopies = SideA::kCopies + SideB::kCopies;  // of a wave per stage
    static constexpr int kPair = 2 * kCopies;
    static constexpr int part(int q) { return kPair * q / 4; }
    static constexpr int kReadsA = TM * SideA::kReads, kReadsB = TN * SideB::kReads;
    static_assert(PAIRS >= 2 && kLds <= 163840 && (PAIRS - 2) * kPair + part(3) < 64, "LDS, and vmcnt's range");
    typename E::Acc acc[TM][TN];

    struct Frags {
        typename SideA::Part a[kReadsA];
        typename SideB::Part b[kReadsB];
    };

    // acc = the product over `kb` bytes of k (of a k-contiguous row; 2 bytes a row of a transposed operand).
    //
    // Stage t sits in buffer t % kStages; its two k halves are steps of TM TN MFMAs. One wave runs on each SIMD, so
    // whatever is not an MFMA is placed between two of them, where it runs while the first executes: in a
    // stage's first step the reads of its second half, in its second step those of the next stage's first.
    // Stages go in pairs, whose copies are issued side by side: a k-contiguous row's two 64 bytes are one
    // cache line, and an L1 of 32 KiB does not keep it from one stage to the next (4096 x 4096 x 128256 scored
    // in 4188 us with single stages). From an even stage t on the pair t + 2 PAIRS goes into the buffers of t - 1 and
    // t, which every wave has read by the barrier in front, a quarter of its copies in each of four steps: the
    // load unit takes about 24 cycles for a copy of 1 KiB, and a wave whose copy has to wait issues no MFMAs.
    //
    // The stages are taken from stage `first` (even) on, those in front of it last.
    __device__ __forceinline__ void run(uint8_t *lds, const Operand &a, const Operand &b, int64_t kb, int wave, int lane,
                                        int first = 0) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass, which drops the body, cannot emit its lambdas' asm)
        SideA sa;
        SideB sb;
        const int wm = wave / WN, wn = wave % WN;
        sa.init(a, wave, lane, TM * wm);
        sb.init(b, wave, lane, TN * wn);
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[i][j][v] = 0;
        const int n = int((kb + kStageK - 1) / kStageK);
        const int n2 = (n + 1) / 2 * 2;
        auto turn = [&](int t) {
            if (t >= n2) return t;
            const int u = t + first;
            return u >= n2 ? u - n2 : u;
        };
        const uint32_t at = uint32_t((uintptr_t)(lds_ptr)(lds));
        Frags x, y;
        unrolled<PAIRS - 1>([&](auto u) {
            uint8_t *to = lds + 2 * u * kStageBytes;
            sa.begin(turn(2 * u));
            sb.begin(turn(2 * u));
            unrolled<kPair>([&](auto o) { copy<o>(sa, sb, to, to + kStageBytes, wave); });
        });
        uint32_t even = (2 * PAIRS - 2) * kStageBytes, odd = even + kStageBytes;  // the buffers of the pair being copied
        sa.begin(turn(2 * PAIRS - 2));
        sb.begin(turn(2 * PAIRS - 2));
        unrolled<part(3)>([&](auto o) { copy<o>(sa, sb, lds + even, lds + odd, wave); });
        wait_copies<(PAIRS - 2) * kPair + part(3)>();
        asm volatile("s_barrier" ::: "memory");
        unrolled<kReadsA>([&](auto r) { sa.template issue<r, 0>(at, x.a[r]); });
        unrolled<kReadsB>([&](auto r) { sb.template issue<r, 0>(at + SideA::kBytes, x.b[r]); });
        landed(x.a, x.b);
        uint32_t b0 = 0;  // stage t's buffer
        auto after = [](uint32_t o) { return o + kStageBytes == kLds ? 0u : o + kStageBytes; };
        for (int t = 0; t < n; t += 2) {
            const uint32_t b1 = after(b0), b2 = after(b1);
            step<0, part(3), kPair>(sa, sb, x, y, at + b0, lds + even, lds + odd, wave);
            landed(y.a, y.b);
            asm volatile("s_barrier" ::: "memory");  // every wave has read stage t
            sa.begin(turn(t + 2 * PAIRS));
            sb.begin(turn(t + 2 * PAIRS));
            even = after(odd);  // (stage t - 1's)
            odd = b0;
            step<1, 0, part(1)>(sa, sb, y, x, at + b1, lds + even, lds + odd, wave);
            landed(x.a, x.b);
            step<0, part(1), part(2)>(sa, sb, x, y, at + b1, lds + even, lds + odd, wave);
            landed(y.a, y.b);
            wait_copies<(PAIRS - 2) * kPair + part(2)>();  // the pair t + 2
            asm volatile("s_barrier" ::: "memory");
            step<1, part(2), part(3)>(sa, sb, y, x, at + b2, lds + even, lds + odd, wave);
            landed(x.a, x.b);
            b0 = b2;
        }
        // every copy has landed, and every wave is past its last read, before the caller uses the LDS; said so that the
        // compiler knows it too, which else waits for all memory operations, stores among them, wherever a caller's loop or
        // branch reads the LDS
        wait_copies<0>();
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        asm volatile("s_barrier" ::: "memory");
#endif
    }

    // acc += the product over one more stage, which the caller has put in the first buffer (in front of a barrier).
    __device__ __forceinline__ void stage(uint8_t *lds, int wave, int lane) {
#ifdef __HIP_DEVICE_COMPILE__  // (as in run)
        SideA sa;
        SideB sb;
        sa.reads(lane, TM * (wave / WN));
        sb.reads(lane, TN * (wave % WN));
        const uint32_t at = uint32_t((uintptr_t)(lds_ptr)(lds));
        unrolled<2>([&](auto j) {
            Frags x;
            unrolled<kReadsA>([&](auto r) { sa.template issue<r, j>(at, x.a[r]); });
            unrolled<kReadsB>([&](auto r) { sb.template issue<r, j>(at + SideA::kBytes, x.b[r]); });
            landed(x.a, x.b);
            unrolled<TM * TN>([&](auto m) {
                constexpr int I = decltype(m)::value / TN, K = decltype(m)::value % TN;
                acc[I][K] = E::mfma(SideB::fragment(x.b, K), SideA::fragment(x.a, I), acc[I][K]);
            });
        });
#endif
    }

private:
    template <int N>
    static __device__ __forceinline__ void wait_copies() {
        asm volatile("s_waitcnt vmcnt(%0)" : : "i"(N) : "memory");
    }

    // Copy O of a pair of stages: both halves of one copy side by side.
    template <int O>
    static __device__ __forceinline__ void copy(const SideA &sa, const SideB &sb, uint8_t *even, uint8_t *odd, int wave) {
        constexpr int Q = O / 2, H = O % 2;
        uint8_t *to = H ? odd : even;
        if constexpr (Q < SideA::kCopies) sa.template copy<Q, H>(to, wave);
        else sb.template copy<Q - SideA::kCopies, H>(to + SideA::kBytes, wave);
    }

    // A step's MFMAs on `f`, between them the reads of half 1 - J at `at` into `g`, by the last but four of them
    // so that they land meanwhile, and copies FROM .. TO - 1 of the pair into its buffers, evenly.
    template <int J, int FROM, int TO>
    __device__ __forceinline__ void step(const SideA &sa, const SideB &sb, const Frags &f, Frags &g, uint32_t at, uint8_t *even,
                                         uint8_t *odd, int wave) {
        constexpr int kMfmas = TM * TN, kReads = kReadsA + kReadsB;
        unrolled<kMfmas>([&](auto m_c) {
            constexpr int M = decltype(m_c)::value, I = M / TN, K = M % TN;
            acc[I][K] = E::mfma(SideB::fragment(f.b, K), SideA::fragment(f.a, I), acc[I][K]);
            __builtin_amdgcn_sched_barrier(0);
            constexpr int kSpread = kMfmas > 4 ? kMfmas - 4 : kMfmas;
            constexpr int kFrom = M * kReads / kSpread < kReads ? M * kReads / kSpread : kReads;
            constexpr int kTo = (M + 1) * kReads / kSpread < kReads ? (M + 1) * kReads / kSpread : kReads;
            unrolled<kTo - kFrom>([&](auto o_c) {
                constexpr int O = kFrom + decltype(o_c)::value;
                if constexpr (O < kReadsB) sb.template issue<O, 1 - J>(at + SideA::kBytes, g.b[O]);
                else sa.template issue<O - kReadsB, 1 - J>(at, g.a[O - kReadsB]);
                __builtin_amdgcn_sched_barrier(0);
            });
            constexpr int cFrom = FROM + M * (TO - FROM) / kMfmas, cTo = FROM + (M + 1) * (TO - FROM) / kMfmas;
            unrolled<cTo - cFrom>([&](auto o_c) {
                copy<cFrom + decltype(o_c)::value>(sa, sb, even, odd, wave);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
    }
};

// The output tile of a workgroup: tiles in groups of 8 row tiles by all column tiles, column after column,
// the workgroups of one XCD (the hardware deals them out in turn) side by side in that order, so that the
// tiles an XCD works on at once share panels in its L2.
__device__ __forceinline__ void tile_of(uint32_t wg, uint32_t tm, uint32_t tn, int &im, int &in) {
    const uint32_t n = tm * tn, per = n / 8, rest = n % 8;
    const uint32_t x = wg % 8, y = wg / 8;
    const uint32_t p = x * per + (x < rest ? x : rest) + y;
    const uint32_t group = p / (8 * tn), gm = tm - group * 8 < 8 ? tm - group * 8 : 8;
    const uint32_t q = p - group * 8 * tn;
    im = int(group * 8 + q % gm);
    in = int(q / gm);
}

// Two f32 values rounded to nearest even into 16 bits, `lo` in the low half.
template <class E>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
    if constexpr (std::is_same<E, Bf16>::value) {
        uint32_t r;
        asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(lo), "v"(hi));
        return r;
    } else {
        return __builtin_bit_cast(uint32_t, f16x2{_Float16(lo), _Float16(hi)});
    }
}

// Between the lanes' stores into a wave's own LDS and other lanes' loads from it, and between those loads and the next
// stores: the LDS takes a wave's accesses in their order, and the compiler, for which a lane's own accesses are all there
// is, keeps them on their sides of this. No instruction.
__device__ __forceinline__ void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wave's 32 x 32 TN block of the output as whole cache lines: the tile's layout gives a lane four neighbouring
// columns of a row, 32 rows a store, so that a line would be written eight bytes at a time. Through LDS (wave
// `lds`: 32 rows of 32 TN values, the caller's barrier in front) a store's lanes cover whole rows of the block. In
// LDS, row r's 16-byte chunk c is at c ^ (r % 16), 16-bit values with their chunk's halves swapped in rows
// 16 .. 31: writes and reads free of bank conflicts.
// V: u32x2 (four 16-bit values) or u32x4 (four 32-bit ones); v[4 j + a] is columns 32 j + 8 a + 4 (lane / 32) ...
// `out`: the block's first value, rows ldo bytes apart; `rows` and `bytes` of the block are stored.
template <int TN, class V>
__device__ __forceinline__ void store_block(uint8_t *lds, const V (&v)[4 * TN], int lane, uint8_t *out, int64_t ldo,
                                            int rows, int bytes) {
    constexpr bool kHalf = sizeof(V) == 8;
    constexpr int kRow = 32 * TN * int(sizeof(V)) / 4, kPer = kRow / 16, kAt = 64 / kPer;  // chunks a row, rows a store
    static_assert(kPer >= 16 && kPer <= 64, "chunks of a row");
    const int r = lane % 32, h = lane / 32;
#pragma unroll
    for (int q = 0; q < 4 * TN; q++) {
        if constexpr (kHalf)
            *reinterpret_cast<u32x2 *>(lds + r * kRow + (q ^ (r % 16)) * 16 + (h ^ (r / 16)) * 8) = v[q];
        else
            *reinterpret_cast<u32x4 *>(lds + r * kRow + ((2 * q + h) ^ (r % 16)) * 16) = v[q];
    }
    wave_exchange();
    const int c = lane % kPer;
#pragma unroll
    for (int g = 0; g < 32 / kAt; g++) {
        const int row = g * kAt + lane / kPer;
        u32x4 x = *reinterpret_cast<const u32x4 *>(lds + row * kRow + (c ^ (row % 16)) * 16);
        if (kHalf && row >= 16) x = u32x4{x.z, x.w, x.x, x.y};
        if (row >= rows) continue;
        uint8_t *o = out + row * ldo + c * 16;
        const int left = bytes - c * 16;
        if (left >= 16) __builtin_memcpy(o, &x, 16);
        else {
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            if constexpr (kHalf) {
                for (int e = 0; e < 8; e++)
                    if (2 * e < left) reinterpret_cast<uint16_t *>(o)[e] = uint16_t(w[e / 2] >> (16 * (e % 2)));
            } else {
                for (int e = 0; e < 4; e++)
                    if (4 * e < left) reinterpret_cast<uint32_t *>(o)[e] = w[e];
            }
        }
    }
    wave_exchange();
}
// The LDS a wave's blocks take.
template <int TN>
constexpr int store_bytes(int value_bytes) {
    return 32 * 32 * TN * value_bytes;
}

}  // namespace tile
}  // namespace nt
