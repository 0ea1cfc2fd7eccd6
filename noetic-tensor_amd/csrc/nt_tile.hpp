// A matrix product's output tile on the matrix cores of gfx950, from operands in their natural row-major
// layouts: acc[m][n] = sum_k A(m, k) B(n, k), 16-bit floats with f32 sums or 8-bit integers with 32-bit
// ones. Shared by the training readout (rl_readout_train.hip) and the 8-bit product (int8.hip).
//
// An operand is k-contiguous (row m at base + m ld, its k bytes side by side) or, for 16-bit types,
// transposed (TR: row k at base + k ld, its m side by side), so that a product and both of its gradients
// read the same tensors: logits = H W^T, dH = G W, dW = G^T H, none of them copied or transposed first.
//
// A workgroup of four waves owns a (32 TM WM) x (32 TN WN) tile, a wave 32 TM x 32 TN of it as TM x TN MFMA
// tiles of 32 x 32. k goes by stages of 64 bytes of a row (32 k of a 16-bit type, 64 of an 8-bit one): both
// operands' panels are copied by the load unit straight into LDS.
//
// LDS: a k-contiguous panel is [row][64 bytes], the four 16-byte chunks of row r at chunk c ^ (r / 4 % 4); a
// transposed one is [32 k][2 B bytes], row k's 64-byte units at u ^ f(k). So the reads below (one 16-byte
// chunk of 32 rows, or 4 k of 32 columns by ds_read_b64_tr_b16) touch every bank once per pass. The load
// unit writes LDS lane by lane, so it is the global address of each lane that is permuted.
//
// Rows past the operand's last, k past its end and whole stages past it read as zeros through the buffer
// resource's range and touch no memory; a k-contiguous row's bytes count is a multiple of 16 (callers pad).
// A transposed operand's columns past its last hold the next row's values: they reach only output columns
// that are not stored.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

namespace nt {
namespace tile {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
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
                voff[q] = uint32_t(k * ld) + ((lane % (kRow / 16)) ^ (swz(k) << 2)) * 16;
            }
        }
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

    // The copies of stage `t` into `lds` (this operand's part of the stage's buffer).
    __device__ __forceinline__ void copy(uint8_t *lds, int t, int wave) const {
        if constexpr (!TR) {
            // a chunk past the row's end is pushed past the range
            const int64_t last = (rows - 1) * ld + width;
            const __amdgpu_buffer_rsrc_t r =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), short(0), int(last), kWord3);
            const uint32_t k0 = t * kStageK;
            const uint32_t koff = int64_t(k0) + chunk * 16 < width ? k0 : 0x80000000u;
#pragma unroll
            for (int q = 0; q < kCopies; q++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + (wave * kCopies + q) * 1024), 16,
                                                         voff[q] + koff, 0, 0, 0);
        } else {
            const int64_t left = rows - int64_t(t) * 32;
            const int64_t bytes = left <= 0 ? 0 : (left < 32 ? left - 1 : 31) * ld + width;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint8_t *>(base + (left <= 0 ? 0 : int64_t(t) * 32 * ld)), short(0), int(bytes), kWord3);
#pragma unroll
            for (int q = 0; q < kCopies; q++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + (wave * kCopies + q) * 1024), 16, voff[q], 0,
                                                         0, 0);
        }
    }

    // Fragment i of k half j of a stage (`at`: the stage's LDS address plus this operand's), waited for.
    template <int I, int J>
    __device__ __forceinline__ u32x4 read(uint32_t at) const {
        if constexpr (!TR) {
            u32x4 d;
            asm volatile("ds_read_b128 %0, %1 offset:%2\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(d)
                         : "v"(at + addr[J]), "i"(I * 32 * kStageK)
                         : "memory");
            return d;
        } else {
            static_assert(I < 4, "addr");
            u32x2 d, e;
            asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4\n\t"
                         "s_waitcnt lgkmcnt(0)"
                         : "=&v"(d), "=&v"(e)
                         : "v"(at + addr[I]), "i"(J * 32 * B), "i"(J * 32 * B + 8 * B)
                         : "memory");
            return u32x4{d.x, d.y, e.x, e.y};
        }
    }
};

// The tile. Lane l of wave (wm, wn) holds in acc[i][j][v] the output of row 32 (TM wm + i) + l % 32 at column
// 32 (TN wn + j) + 8 (v / 4) + 4 (l / 32) + v % 4: B is the MFMA's first operand, so that a lane's values are
// of one row and by four of neighbouring columns.
template <class E, int TM, int TN, int WM, int WN, bool ATR, bool BTR>
struct Tile {
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    typedef Side<BM, kWaves, ATR> SideA;
    typedef Side<BN, kWaves, BTR> SideB;
    static constexpr int kStageBytes = SideA::kBytes + SideB::kBytes;
    static constexpr int kStages = 2;
    static constexpr int kLds = kStages * kStageBytes;
    typename E::Acc acc[TM][TN];

    // acc = the product over `kb` bytes of k (of a k-contiguous row; 2 bytes a row of a transposed operand)
    __device__ __forceinline__ void run(uint8_t *lds, const Operand &a, const Operand &b, int64_t kb, int wave, int lane) {
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
        sa.copy(lds, 0, wave);
        sb.copy(lds + SideA::kBytes, 0, wave);
        const uint32_t at = uint32_t((uintptr_t)(lds_ptr)(lds));
        for (int t = 0; t < n; t++) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            uint8_t *next = lds + ((t + 1) % kStages) * kStageBytes;
            sa.copy(next, t + 1, wave);
            sb.copy(next + SideA::kBytes, t + 1, wave);
            const uint32_t now = at + (t % kStages) * kStageBytes;
            unrolled<2>([&](auto j_c) {
                constexpr int J = decltype(j_c)::value;
                u32x4 fa[TM], fb[TN];
                unrolled<TM>([&](auto i_c) { fa[i_c] = sa.template read<i_c, J>(now); });
                unrolled<TN>([&](auto i_c) { fb[i_c] = sb.template read<i_c, J>(now + SideA::kBytes); });
#pragma unroll
                for (int i = 0; i < TM; i++)
#pragma unroll
                    for (int k = 0; k < TN; k++) acc[i][k] = E::mfma(fb[k], fa[i], acc[i][k]);
            });
        }
        // every copy has landed, and every wave is past its last read, before the caller uses the LDS
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#endif
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
        const uint16_t a = __builtin_bit_cast(uint16_t, _Float16(lo)), b = __builtin_bit_cast(uint16_t, _Float16(hi));
        return uint32_t(a) | (uint32_t(b) << 16);
    }
}

}  // namespace tile
}  // namespace nt
