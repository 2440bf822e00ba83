// A workgroup's tile of a matrix product, for kernels that go on with the sums
// in registers (cross_entropy.hip, orthogonal.hip).
//
// The tile has kM "rows" and kN "columns": out(m, n) = sum over k of A(m, k) B(n, k),
// with FP32 sums.  Operands are 16-bit matrices in memory either by rows (a row's k
// adjacent) or by columns (a k's rows adjacent); both go to LDS as they lie, kStep of k at a
// time, straight from memory and kStages steps deep.  Operands by columns are turned by
// gfx950's transposed LDS reads.  A wave reads the next 16 of k from LDS while it multiplies
// these; the barrier of a step lies between the two, under products.
//
// A 32x32x16 instruction leaves lane l with column l & 31 and rows 8 g + 4 (l >> 5) + i
// (register 4 g + i): four adjacent rows of a column lie in one lane.
#pragma once

#include "attention_core.h"

namespace lct {

enum class Lie { kRows, kColumns };

// One operand's tile of kTile rows by kStep of k: how it comes to LDS and how an
// instruction's 32 rows by 16 of k are read from there.
//
// LDS returns 256 bytes a clock: the chunks of 16 bytes that 16 rows are read at (by
// rows), and the 64 bytes of each of 4 lines (by columns, a line of kTile values per k), are
// permuted so that they lie in different ones of its 16 columns (counted: no conflicts).
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
        if constexpr (kLie == Lie::kRows)
            return chunk ^ (kStep == 32 ? (line >> 2) & 3 : (line >> 1) & 7);
        else    // (every second line of 128 or 384 bytes is 128 further as it is)
            return chunk ^ (kTile % 128 ? (line & 2) << 1 : (line & 3) << 2);
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

    // k .. k + kStep - 1 of `depth`; zeros past it and past the last row.
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

    // Where this lane reads the fragments of 32 rows from `first_row` on by 16 of k, in a
    // tile: places that differ by more than a constant.  (Held in registers that the
    // compiler does not look into: left alone, it finds constant addresses in some, whose
    // reads it then takes for ones of any stage and lets wait for all loads.)
    static constexpr int kPlaces = kLie == Lie::kRows ? kStep / 16 : 4;   // kColumns: of 4 n
    struct Places {
        int at[kPlaces];
    };
    static __device__ __forceinline__ Places places(int first_row) {
        const int lane = wave_lane();
        Places p;
        if constexpr (kLie == Lie::kRows) {
            const int row = lane & 31;
#pragma unroll
            for (int s = 0; s < kPlaces; ++s)
                p.at[s] = (first_row + row) * kStep + permuted(row, 2 * s + (lane >> 5)) * 8;
        } else {
            const int line = 8 * (lane >> 5) + ((lane & 15) >> 2);
            const int chunk = first_row / 8 + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
#pragma unroll
            for (int n = 0; n < kPlaces; ++n)
                p.at[n] = line * kTile + permuted(line, chunk + 4 * n) * 8 + (lane & 1) * 4;
        }
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) asm("" : "+v"(p.at[i]));
        return p;
    }

    // Fragment n, k 16 step .. + 15.
    static __device__ __forceinline__ u32x4 read(const uint16_t *tile, const Places &p, int n,
                                                 int step) {
        if constexpr (kLie == Lie::kRows) {
            return *reinterpret_cast<const u32x4 *>(tile + p.at[step] + 32 * n * kStep);
        } else {
            // (The permutation moves chunks within 16 of them.)
            const uint16_t *at = tile + p.at[n & 3] + (n & ~3) * 32 + 16 * step * kTile;
            const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4 *)(at));
            const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4 *)(at + 4 * kTile));
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

template <bool kHalf, Lie kLieA, Lie kLieB, int kM_, int kN_, int kWavesM_, int kWavesN, int kStep,
          int kStages_>
struct Product {
    static constexpr int kM = kM_, kN = kN_, kThreads = kWave * kWavesM_ * kWavesN;
    static constexpr int kStages = kStages_, kWavesM = kWavesM_;
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

    struct Fragments {
        u32x4 a[kRowTiles], b[kColumnTiles];
    };
    static constexpr int kFragmentReads = kRowTiles * A::kReads + kColumnTiles * B::kReads;

    static __device__ __forceinline__ void read(Fragments &f, const uint16_t *stage,
                                                const typename A::Places &a,
                                                const typename B::Places &b, int s) {
#pragma unroll
        for (int n = 0; n < kColumnTiles; ++n) f.b[n] = B::read(stage + A::kValues, b, n, s);
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m) f.a[m] = A::read(stage, a, m, s);
    }
    __device__ __forceinline__ void multiply(const Fragments &f) {
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m)
#pragma unroll
            for (int n = 0; n < kColumnTiles; ++n)
                sum[m][n] = Element<kHalf>::multiply(f.a[m], f.b[n], sum[m][n]);
    }

    // The sums' first values: start(m, n) gives 16 registers' of a 32 x 32 tile.
    template <class Start>
    __device__ __forceinline__ void begin(Start start) {
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m)
#pragma unroll
            for (int n = 0; n < kColumnTiles; ++n) sum[m][n] = start(m, n);
    }
    __device__ __forceinline__ void begin() {
        begin([](int, int) { return f32x16{}; });
    }

    // Adds all of `depth` to the sums; the stages are free afterwards.
    __device__ __forceinline__ void run(const A &a, const B &b, int32_t depth,
                                        uint16_t *s0, uint16_t *s1, uint16_t *s2, uint16_t *s3) {
        uint16_t *const stages[4] = {s0, s1, s2, s3};
        constexpr int kLoads = A::kCount + B::kCount, kParts = kStep / 16;
        const auto load = [&](int32_t k, uint16_t *stage) __attribute__((always_inline)) {
            a.issue(k, depth, stage);
            b.issue(k, depth, stage + A::kValues);
        };
#pragma unroll
        for (int s = 0; s < kStages; ++s) load(s * kStep, stages[s]);
        loads_barrier<kLoads * (kStages - 1)>();
        // Two sets of fragments: one is read while the other is multiplied.
        const typename A::Places at_a = A::places(first_row());
        const typename B::Places at_b = B::places(first_column());
        Fragments f[2];
        read(f[0], stages[0], at_a, at_b, 0);
        for (int32_t k = 0; k < depth; k += kStages * kStep) {
#pragma unroll
            for (int s = 0; s < kStages; ++s) {
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    const int now = (s * kParts + part) & 1;
                    if (part + 1 < kParts) {
                        read(f[now ^ 1], stages[s], at_a, at_b, part + 1);
                    } else {
                        // Behind the barrier all have the next stage's loads, and have read
                        // this one, which is loaded for the step after the others.
                        loads_barrier<kLoads * (kStages - 2)>();
                        load(k + (s + kStages) * kStep, stages[s]);
                        read(f[now ^ 1], stages[(s + 1) % kStages], at_a, at_b, 0);
                    }
                    multiply(f[now]);
                    __builtin_amdgcn_sched_group_barrier(kLdsReadGroup, kFragmentReads, 0);
                    __builtin_amdgcn_sched_group_barrier(kMatrixGroup, kRowTiles * kColumnTiles, 0);
                }
            }
        }
        // Loads of steps past the end are still on their way.
        loads_barrier<0>();
    }
};

// The stages' LDS of product P, as run()'s last arguments.  (Arrays of their own: the compiler
// then knows which loads a read has to wait for.)
#define LCT_PRODUCT_STAGES(P)                                                                  \
    __shared__ __attribute__((aligned(1024))) uint16_t stage0[P::kStage];                      \
    __shared__ __attribute__((aligned(1024))) uint16_t stage1[P::kStage];                      \
    __shared__ __attribute__((aligned(1024))) uint16_t stage2[P::kStages > 2 ? P::kStage : 8]; \
    __shared__ __attribute__((aligned(1024))) uint16_t stage3[P::kStages > 3 ? P::kStage : 8]

// What one wave wrote to LDS can be read by its other lanes.
__device__ __forceinline__ void wave_fence() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// 16 bytes a lane of a tile's kLines lines of kChunks pieces: lane l's of access i are those of
// slot 64 i + l.  What is past the `lines` lines of `length` values (a multiple of 8) that
// the matrix has from the tile on reads as zeros and is not written.
template <int kLines, int kChunks>
struct Lines {
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t pitch;      // bytes
    int32_t length;

    __device__ __forceinline__ Lines(const uint16_t *base, int64_t stride, int32_t lines,
                                     int32_t length_)
        : pitch(static_cast<uint32_t>(stride) * 2u), length(length_) {
        // (Of the tile alone: 32 bits hold its size.)
        length = min(length, kChunks * 8);
        rsrc = make_rsrc(base, lines > 0 && length > 0
                                   ? static_cast<uint32_t>(min(lines, kLines) - 1) * pitch
                                         + static_cast<uint32_t>(length) * 2u
                                   : 0u);
    }
    __device__ __forceinline__ uint32_t at(int first, int slot) const {
        const int chunk = slot % kChunks;
        return chunk * 8 < length ? static_cast<uint32_t>(first + slot / kChunks) * pitch
                                        + static_cast<uint32_t>(chunk) * 16u
                                  : kOutOfRange;
    }
    __device__ __forceinline__ u32x4 load(int first, int slot) const {
        return __builtin_bit_cast(u32x4,
                                  __builtin_amdgcn_raw_buffer_load_b128(rsrc, at(first, slot), 0, 0));
    }
    __device__ __forceinline__ void store(u32x4 v, int first, int slot) const {
        store_b128<0>(__builtin_bit_cast(uint4, v), rsrc, at(first, slot));
    }
};

// A wave's tile (rows m, columns n; pair(m, n, r) gives two adjacent rows' values) to memory
// with a column's rows next to each other: 8 bytes a lane into LDS of the wave's own
// (kTurnValues<P>), 16 bytes a lane out of it, so that a column's rows are stored together.
// `rows`: how many there are from the wave's first on, a multiple of 8.
template <class P>
constexpr int kTurnValues = 32 * (P::kWaveM + 8);

template <class P, class Pair>
__device__ __forceinline__ void store_columns(uint16_t *out, int64_t stride, int32_t columns,
                                              int32_t rows, uint16_t *mine, Pair pair) {
    constexpr int kPitch = P::kWaveM + 8, kChunks = P::kWaveM / 8;
    const int lane = wave_lane();
    const Lines<P::kWaveN, kChunks> lines(out, stride, columns, rows);
    uint16_t *at = mine + (lane & 31) * kPitch + (lane >> 5) * 4;
#pragma unroll
    for (int n = 0; n < P::kColumnTiles; ++n) {
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<u32x2 *>(at + 32 * m + 8 * g) =
                    u32x2{pair(m, n, 4 * g), pair(m, n, 4 * g + 2)};
        wave_fence();
#pragma unroll
        for (int i = 0; i < 32 * kChunks / kWave; ++i) {
            const int slot = i * kWave + lane;
            lines.store(*reinterpret_cast<const u32x4 *>(mine + slot / kChunks * kPitch
                                                         + slot % kChunks * 8),
                        32 * n, slot);
        }
        wave_fence();
    }
}

// The other way: take(m, n, r, pair) gets each two adjacent rows' values, zeros where there
// are none.
template <class P, class Take>
__device__ __forceinline__ void load_columns(const uint16_t *from, int64_t stride, int32_t columns,
                                             int32_t rows, uint16_t *mine, Take take) {
    constexpr int kPitch = P::kWaveM + 8, kChunks = P::kWaveM / 8;
    constexpr int kCount = 32 * kChunks / kWave;
    const int lane = wave_lane();
    const Lines<P::kWaveN, kChunks> lines(from, stride, columns, rows);
    const uint16_t *at = mine + (lane & 31) * kPitch + (lane >> 5) * 4;
#pragma unroll
    for (int n = 0; n < P::kColumnTiles; ++n) {
        u32x4 v[kCount];
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] = lines.load(32 * n, i * kWave + lane);
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int slot = i * kWave + lane;
            *reinterpret_cast<u32x4 *>(mine + slot / kChunks * kPitch + slot % kChunks * 8) = v[i];
        }
        wave_fence();
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const u32x2 pairs = *reinterpret_cast<const u32x2 *>(at + 32 * m + 8 * g);
                take(m, n, 4 * g, pairs[0]);
                take(m, n, 4 * g + 2, pairs[1]);
            }
        wave_fence();
    }
}

// A wave's tile to memory with a row's columns next to each other, 32 rows at a time.
// `columns`: how many there are from the wave's first on, a multiple of 8.
template <class P, class Pair>
__device__ __forceinline__ void store_rows(uint16_t *out, int64_t stride, int32_t rows,
                                           int32_t columns, uint16_t *mine, Pair pair) {
    constexpr int kPitch = P::kWaveN + 8, kChunks = P::kWaveN / 8;
    static_assert(32 * kPitch <= kTurnValues<P>);
    const int lane = wave_lane();
    const Lines<P::kWaveM, kChunks> lines(out, stride, rows, columns);
    // Of two rows' values of two adjacent lanes: the even one takes the first row's, the
    // odd one the second's.
    const uint32_t select = lane & 1 ? 0x03020706u : 0x05040100u;
    uint16_t *at = mine + (4 * (lane >> 5) + (lane & 1)) * kPitch + (lane & 30);
#pragma unroll
    for (int m = 0; m < P::kRowTiles; ++m) {
#pragma unroll
        for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const uint32_t own = pair(m, n, r);
                const uint32_t other = __builtin_amdgcn_mov_dpp(own, 0xB1, 0xF, 0xF, true);
                *reinterpret_cast<uint32_t *>(at + (8 * (r / 4) + r % 4) * kPitch + 32 * n) =
                    __builtin_amdgcn_perm(other, own, select);
            }
        wave_fence();
#pragma unroll
        for (int i = 0; i < 32 * kChunks / kWave; ++i) {
            const int slot = i * kWave + lane;
            lines.store(*reinterpret_cast<const u32x4 *>(mine + slot / kChunks * kPitch
                                                         + slot % kChunks * 8),
                        32 * m, slot);
        }
        wave_fence();
    }
}

// That LDS: in the stages, which a finished run() leaves free.
template <class P>
__device__ __forceinline__ uint16_t *turn_values(uint16_t *s0, uint16_t *s1, uint16_t *s2,
                                                 uint16_t *s3) {
    constexpr int kWaves = P::kThreads / kWave, kPer = (kWaves + P::kStages - 1) / P::kStages;
    static_assert(kPer * kTurnValues<P> <= P::kStage);
    const int wave = P::wave(), stage = wave / kPer;
    uint16_t *base = stage == 0 ? s0 : s1;
    if constexpr (2 * kPer < kWaves) base = stage < 2 ? base : stage == 2 ? s2 : s3;
    return base + wave % kPer * kTurnValues<P>;
}

}  // namespace lct
