// A workgroup's tile of a matrix product, for kernels that go on with the sums
// in registers (cross_entropy.hip, orthogonal.hip).
//
// The tile has kM "rows" and kN "columns": out(m, n) = sum over k of A(m, k) B(n, k),
// with FP32 sums.  Four waves share it, two by two.  Operands are 16-bit matrices in
// memory either by rows (a row's k adjacent) or by columns (a k's rows adjacent);
// both go to LDS as they lie, 32 of k at a time, straight from memory and three
// steps deep, so that the loads of two steps are on their way while one is
// multiplied.  Operands by columns are turned by gfx950's transposed LDS reads.
//
// Two such workgroups fit a compute unit (72 KB of LDS, 128 sums per lane at 256 x
// 128), so that one's epilogue runs under the other's products.
//
// A 32x32x16 instruction leaves lane l with column l & 31 and rows 8 g + 4 (l >> 5) + i
// (register 4 g + i): four adjacent rows of a column lie in one lane.
#pragma once

#include "attention_core.h"

namespace lct {

enum class Lie { kRows, kColumns };

// One operand's tile of kTile rows by 32 of k: how it comes to LDS and how an
// instruction's 32 rows by 16 of k are read from there.
//
// By rows: 4 chunks of 16 bytes per row, permuted by the row's bits 1 and 2, so that 8
// rows read at one chunk lie in different 16-byte columns of the 128 bytes of a clock.
// By columns: a line of kTile values per k, permuted by swizzle() as the attention
// kernels' tiles are.
template <Lie kLie, int kTile, int kStep, int kThreads>
struct Operand {
    static constexpr int kValues = kTile * kStep;
    static constexpr int kCount = kValues * 2 / (kThreads * 16);
    static constexpr int kChunks = kLie == Lie::kRows ? kStep / 8 : kTile / 8;
    static_assert(kCount >= 1);

    const uint16_t *base;     // the tile's first row, k = 0
    int64_t stride;           // of a row (kRows) or of k (kColumns)
    int32_t valid;            // rows that there are
    uint32_t offset[kCount];

    static __device__ __forceinline__ int permuted(int line, int chunk) {
        return chunk ^ (kLie == Lie::kColumns ? swizzle(line) : kStep == 32 ? (line >> 1) & 3 : line & 7);
    }

    __device__ __forceinline__ void prepare(const void *matrix, int64_t stride_, int64_t first,
                                            int64_t rows) {
        stride = stride_;
        valid = static_cast<int32_t>(rows - first < kTile ? rows - first : kTile);
        base = static_cast<const uint16_t *>(matrix)
               + (kLie == Lie::kRows ? first * stride : first);
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int slot = i * kThreads + threadIdx.x;
            const int line = slot / kChunks, chunk = permuted(line, slot % kChunks);
            offset[i] = static_cast<uint32_t>(line) * static_cast<uint32_t>(stride) * 2u
                        + static_cast<uint32_t>(chunk) * 16u;
            if (kLie == Lie::kColumns && chunk * 8 >= valid) offset[i] = kOutOfRange;
        }
    }

    // k .. k + 31 of `depth`; zeros past it and past the last row.
    __device__ __forceinline__ void issue(int32_t k, int32_t depth, uint16_t *tile) const {
        const int32_t left = depth - k;
        const int32_t lines = kLie == Lie::kRows ? valid : min(left, kStep);
        // (A row's last chunk is whole: what it holds past `depth` meets zeros of the
        // other operand.)
        const int32_t last = kLie == Lie::kRows ? (left + 7) & ~7 : valid;
        const __amdgpu_buffer_rsrc_t rsrc =
            make_rsrc(base + (kLie == Lie::kRows ? k : k * stride),
                      left > 0 ? (static_cast<uint32_t>(lines - 1) * static_cast<uint32_t>(stride)
                                  + static_cast<uint32_t>(last))
                                     * 2u
                               : 0u);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        const bool whole = kLie == Lie::kColumns || left >= kStep;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            uint32_t at = offset[i];
            if (!whole) {
                const int slot = i * kThreads + threadIdx.x;
                if (permuted(slot / kChunks, slot % kChunks) * 8 >= left) at = kOutOfRange;
            }
            load_to_lds(rsrc, tile + (i * (kThreads / kWave) + wave) * 512, at);
        }
    }

    // Rows 32 n .. + 31, values 16 step .. + 15 of k.
    static __device__ __forceinline__ u32x4 read(const uint16_t *tile, int n, int step) {
        const int lane = wave_lane();
        if constexpr (kLie == Lie::kRows) {
            const int row = lane & 31;
            const int chunk = permuted(row, 2 * step + (lane >> 5));
            return *reinterpret_cast<const u32x4 *>(tile + (32 * n + row) * kStep
                                                    + chunk * 8);
        } else {
            const int line = 8 * (lane >> 5) + ((lane & 15) >> 2);
            const int chunk = 4 * n + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
            const uint16_t *at = tile + (16 * step + line) * kTile + (lane & 1) * 4;
            const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4 *)(at + permuted(line, chunk) * 8));
            const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4 *)(at + 4 * kTile
                                                            + permuted(line + 4, chunk) * 8));
            const u32x2 lo = __builtin_bit_cast(u32x2, a), hi = __builtin_bit_cast(u32x2, b);
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
    }
    static constexpr int kReads = kLie == Lie::kRows ? 1 : 2;
};

// A barrier behind which all waves' LDS reads are done, and all their loads but the last
// `kLeft` of each.
template <int kLeft>
__device__ __forceinline__ void loads_barrier() {
    static_assert(kLeft < 64);
    __builtin_amdgcn_s_waitcnt((kLeft & 15) | (kLeft >> 4) << 14 | 0x70);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <bool kHalf, Lie kLieA, Lie kLieB, int kM_, int kN_, int kWavesM, int kWavesN, int kStep,
          int kStages>
struct Product {
    static constexpr int kM = kM_, kN = kN_, kThreads = 64 * kWavesM * kWavesN;
    using A = Operand<kLieA, kM, kStep, kThreads>;
    using B = Operand<kLieB, kN, kStep, kThreads>;
    static constexpr int kWaveM = kM / kWavesM, kWaveN = kN / kWavesN;
    static constexpr int kRowTiles = kWaveM / 32, kColumnTiles = kWaveN / 32;
    static constexpr int kStage = A::kValues + B::kValues;   // values of LDS

    f32x16 sum[kRowTiles][kColumnTiles];

    static __device__ __forceinline__ int wave() {
        return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    }
    // The first row and column of this wave's part of the tile.
    static __device__ __forceinline__ int first_row() { return (wave() % kWavesM) * kWaveM; }
    static __device__ __forceinline__ int first_column() { return (wave() / kWavesM) * kWaveN; }

    __device__ __forceinline__ void multiply(const uint16_t *stage) {
        const uint16_t *a_tile = stage, *b_tile = stage + A::kValues;
        const int row_tile = first_row() / 32, column_tile = first_column() / 32;
#pragma unroll
        for (int s = 0; s < kStep / 16; ++s) {
            u32x4 b[kColumnTiles];
#pragma unroll
            for (int n = 0; n < kColumnTiles; ++n) b[n] = B::read(b_tile, column_tile + n, s);
#pragma unroll
            for (int m = 0; m < kRowTiles; ++m) {
                const u32x4 a = A::read(a_tile, row_tile + m, s);
#pragma unroll
                for (int n = 0; n < kColumnTiles; ++n)
                    sum[m][n] = Element<kHalf>::multiply(a, b[n], sum[m][n]);
            }
        }
    }

    // All of `depth`; the stages are free afterwards.
    __device__ __forceinline__ void run(const A &a, const B &b, int32_t depth,
                                        uint16_t *const (&stages)[kStages]) {
        constexpr int kLoads = A::kCount + B::kCount;
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m)
#pragma unroll
            for (int n = 0; n < kColumnTiles; ++n) sum[m][n] = f32x16{};
        const auto load = [&](int32_t k, uint16_t *stage) __attribute__((always_inline)) {
            a.issue(k, depth, stage);
            b.issue(k, depth, stage + A::kValues);
        };
#pragma unroll
        for (int s = 0; s + 1 < kStages; ++s) load(s * kStep, stages[s]);
        for (int32_t k = 0; k < depth; k += kStages * kStep) {
#pragma unroll
            for (int s = 0; s < kStages; ++s) {
                // Behind the barrier all have the stage's loads, and have read the stage
                // that is loaded next.
                loads_barrier<kLoads * (kStages - 2)>();
                load(k + (s + kStages - 1) * kStep, stages[(s + kStages - 1) % kStages]);
                multiply(stages[s]);
            }
        }
        // Loads of steps past the end are still on their way.
        loads_barrier<0>();
    }
};

}  // namespace lct
