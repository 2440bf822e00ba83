// What the attention kernels share: 32 x 32 matrix tiles of BF16 or FP16 with
// FP32 sums, their operands in LDS, and which keys a query sees.
//
// Tiles.  A 32x32x16 matrix instruction takes, per lane, 8 consecutive values of
// its summed axis (lane & 31: the row or column, lane >> 5: which half of the
// 16), and leaves lane l with column l & 31 and rows 8 g + 4 (l >> 5) + i
// (register 4 g + i).  The kernels compute the scores with the axis that the
// next product sums over in the rows, so a lane's 16 scores are, two groups g at
// a time, already the next instruction's operand: the summed axis is then taken
// in the order 8 (j / 4) + 4 (l >> 5) + j % 4, and the other operand is read in
// that order too.  No score moves between lanes.
//
// LDS tiles hold rows of 64 or 128 values (kPitch; narrower heads padded with
// zeros by the loads' range check).  Each row's 16-byte chunks are permuted by
// an exclusive or with swizzle(row), a permutation of 0..7 over 8 rows that
// also keeps 4 rows' chunk pairs apart: rows read by 8 lanes at one chunk, and
// transposed reads of 4 rows by 32 bytes, lie in different 16-byte columns of
// the 128 bytes that LDS returns in a clock.
#pragma once

#include <type_traits>

#include "lct_device.h"

namespace lct {

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using i16x4 = __attribute__((ext_vector_type(4))) short;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;

// The two 16-bit types: the matrix instruction and the rounding of a pair.
template <bool kHalf>
struct Element {
    static __device__ __forceinline__ f32x16 multiply(u32x4 a, u32x4 b, f32x16 c) {
        if constexpr (kHalf)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                          __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                           __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                           0);
    }
    static __device__ __forceinline__ uint32_t round_pair(float x, float y) {
        const f32x2 v = {x, y};
        if constexpr (kHalf)
            return __builtin_bit_cast(
                uint32_t,
                __builtin_convertvector(v, __attribute__((ext_vector_type(2))) _Float16));
        else
            return __builtin_bit_cast(
                uint32_t, __builtin_convertvector(v, __attribute__((ext_vector_type(2))) __bf16));
    }
    static __device__ __forceinline__ float low(uint32_t pair) {
        if constexpr (kHalf)
            return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(pair)));
        else
            return __uint_as_float(pair << 16);
    }
    static __device__ __forceinline__ float high(uint32_t pair) {
        if constexpr (kHalf)
            return low(pair >> 16);
        else
            return __uint_as_float(pair & 0xFFFF0000u);
    }
};

// How far (log2) a running maximum may lag.  In FP16 the weights are held 2^kHalfLift
// larger, up to 2^15: one below 2^-25 of the largest would be lost, and a cache has
// enough keys for those to count.
constexpr float kRescale = 8.0f, kHalfLift = 7.0f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Both halves of a wave: f(lane's value, the value of the lane 32 further).
__device__ __forceinline__ float across_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float across_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

constexpr int kAttentionThreads = 256;
constexpr int kAttentionWaves = kAttentionThreads / kWave;

template <int kDim>
constexpr int kPitchOf = kDim <= 64 ? 64 : 128;

__device__ __forceinline__ int swizzle(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

// 16 bytes per lane from rsrc + offset to adjacent 16 bytes at `lds`.  (A plain
// function: in a template the host's pass checks the builtin's size against
// the host's target.)
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, uint16_t *lds,
                                            uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rsrc, (__attribute__((address_space(3))) void *)lds, 16, offset, 0, 0, 0);
}

// The loads of an LDS tile of kRows rows, kPitch values each, by a workgroup:
// wave w's load i fills the 1024 bytes at (i * waves + w) * 1024, and lane l's
// 16 bytes of them hold the chunk that belongs there.  Chunks past the head's
// width get an offset that the range check rejects (LDS receives zeros).
template <int kRows, int kPitch, int kThreads = kAttentionThreads>
struct TileLoads {
    static constexpr int kCount = kRows * kPitch * 2 / (kThreads * 16);
    uint32_t offset[kCount];

    __device__ __forceinline__ void prepare(int64_t row_stride, int32_t dim) {
        constexpr int kChunks = kPitch / 8;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int slot = i * kThreads + threadIdx.x;
            const int row = slot / kChunks;
            const int chunk = (slot % kChunks) ^ swizzle(row);
            offset[i] = chunk * 8 < dim
                            ? static_cast<uint32_t>(row * row_stride * 2 + chunk * 16)
                            : kOutOfRange;
        }
    }

    // Rows [0, rows) from `base`; zeros for the others.
    __device__ __forceinline__ void issue(const uint16_t *base, int32_t rows, int64_t row_stride,
                                          int32_t dim, uint16_t *tile) const {
        // Below 2^31 bytes: 32 bits hold the product.
        const int32_t valid = min(rows, kRows);
        const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(
            base, valid > 0 ? (static_cast<uint32_t>(valid - 1) * static_cast<uint32_t>(row_stride)
                               + static_cast<uint32_t>(dim))
                                  * 2u
                            : 0u);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
#pragma unroll
        for (int i = 0; i < kCount; ++i)
            load_to_lds(rsrc, tile + (i * (kThreads / kWave) + wave) * 512, offset[i]);
    }
};

// Operand rows 32 n + (lane & 31), values 16 step + 8 (lane >> 5) .. + 7.
template <int kPitch>
__device__ __forceinline__ u32x4 read_rows(const uint16_t *tile, int n, int step) {
    const int lane = wave_lane(), row = lane & 31;
    const int chunk = (2 * step + (lane >> 5)) ^ swizzle(row);
    return *reinterpret_cast<const u32x4 *>(tile + (32 * n + row) * kPitch + chunk * 8);
}

// Operand rows are the tile's columns 32 column + (lane & 31); the summed axis
// is its rows `first` .. + 15 in the order at the top of this file.
template <int kPitch>
__device__ __forceinline__ u32x4 read_columns(const uint16_t *tile, int first, int column) {
    const int lane = wave_lane();
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int chunk = (4 * column + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ swizzle(row);
    const uint16_t *at = tile + (first + row) * kPitch + chunk * 8 + (lane & 1) * 4;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4 *)(at));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4 *)(at + 8 * kPitch));
    const u32x2 lo = __builtin_bit_cast(u32x2, a), hi = __builtin_bit_cast(u32x2, b);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// The order of the matrix products since the last branch and of the LDS reads that
// feed them: kFirst reads, then a product and the next kReads reads in turn.  (Left
// alone, the compiler reads an operand just before its product, which then waits
// for LDS.)
constexpr int kMatrixGroup = 0x008, kLdsReadGroup = 0x100;    // sched_group_barrier's masks
template <int kProducts, int kReads, int kFirst>
__device__ __forceinline__ void read_ahead() {
    constexpr int kLeft = kProducts - kFirst / kReads;
    __builtin_amdgcn_sched_group_barrier(kLdsReadGroup, kFirst, 0);
#pragma unroll
    for (int i = 0; i < kLeft; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMatrixGroup, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kLdsReadGroup, kReads, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMatrixGroup, kFirst / kReads, 0);
}

// Two groups (8 registers) of a tile of scores as the next operand.
template <bool kHalf>
__device__ __forceinline__ u32x4 as_operand(const f32x16 &s, int pair) {
    u32x4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        out[j] = Element<kHalf>::round_pair(s[8 * pair + 2 * j], s[8 * pair + 2 * j + 1]);
    return out;
}

// Row `row` of a [.., token, channel] matrix as the operand of `step`, straight
// from memory; zeros past the last row and past the head's width.
__device__ __forceinline__ u32x4 load_operand(const uint16_t *base, int64_t row_stride, int32_t row,
                                              int32_t rows, int32_t dim, int step) {
    const int32_t channel = 16 * step + 8 * (wave_lane() >> 5);
    u32x4 out = {0u, 0u, 0u, 0u};
    if (row < rows && channel < dim)
        out = *reinterpret_cast<const u32x4 *>(base + row * row_stride + channel);
    return out;
}

// Query i stands at position i + keys - queries; it sees key j where j <= its
// position, j and it lie below the sequence's length, and j is among the last
// `window` keys up to it or among the first `sinks`.
struct Sight {
    int32_t limit;    // one past the last visible key; 0: none
    int32_t low;      // first key of the window
    int32_t sinks;    // and the keys below this
    __device__ __forceinline__ bool operator()(int32_t key) const {
        return key < limit && (key >= low || key < sinks);
    }
};

// What a lane's query sees of a tile of scores, by its place in the registers:
// register 4 g + i of rows 32 n .. holds key first + 32 n + 8 g + 4 half + i.
// The gap from that key to the query's position must lie between 0 and the
// window, one unsigned comparison (a query that sees nothing is at a position
// before all keys); tiles with sinks (uniform: few) need two more.
struct TileSight {
    int32_t gap;            // position - key of register 0
    uint32_t reach;
    int32_t sinks;          // sinks from register 0's key on, 0 where the tile has none
    __device__ __forceinline__ TileSight(const lct_attention &a, int32_t position, int32_t first) {
        const int32_t key = first + 4 * (wave_lane() >> 5);
        gap = position - key;
        reach = a.window > 0 ? static_cast<uint32_t>(a.window) : 0x40000000u;
        sinks = a.window > 0 && first < a.sinks ? a.sinks - key : 0;
    }
    // `offset`: 32 n + 8 g + i.
    __device__ __forceinline__ bool operator()(int32_t offset) const {
        return static_cast<uint32_t>(gap - offset) < reach;
    }
    __device__ __forceinline__ bool with_sinks(int32_t offset) const {
        return (*this)(offset) || (offset < sinks && offset <= gap);
    }
    template <class Keep>
    __device__ __forceinline__ void each(int32_t first, int32_t base, int32_t total_sinks,
                                         Keep keep) const {
        if (first < total_sinks) {
#pragma unroll
            for (int r = 0; r < 16; ++r) keep(r, with_sinks(base + 8 * (r / 4) + r % 4));
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) keep(r, (*this)(base + 8 * (r / 4) + r % 4));
        }
    }
};

// Before every key: where a query that sees none stands.
constexpr int32_t kNowhere = -(1 << 30);

// Keys a sequence has, within the tensor's.
__device__ __forceinline__ int32_t sequence_length(const lct_attention &a, int32_t b) {
    return a.lengths == nullptr ? a.keys : max(0, min(a.lengths[b], a.keys));
}

__device__ __forceinline__ Sight sight_of(const lct_attention &a, int32_t position,
                                          int32_t length) {
    Sight s;
    s.limit = position >= 0 && position < length ? position + 1 : 0;
    s.low = a.window > 0 ? position - a.window + 1 : 0;
    s.sinks = a.window > 0 ? a.sinks : 0;
    return s;
}

// The tiles of kTile keys that queries at positions first..last see: those of
// the sinks, then those of the window.
struct KeyTiles {
    int32_t sink_tiles, start, count, end;
    __device__ __forceinline__ KeyTiles(const lct_attention &a, int32_t first, int32_t last,
                                        int32_t length, int32_t tile) {
        end = first < length ? min(last + 1, length) : 0;
        const int32_t low = a.window > 0 ? max(0, max(first, 0) - a.window + 1) : 0;
        const int32_t sinks = a.window > 0 ? min(min(a.sinks, low), end) : 0;
        sink_tiles = end > 0 ? (sinks + tile - 1) / tile : 0;
        start = max(low / tile, sink_tiles) * tile;
        count = sink_tiles + (end > start ? (end - start + tile - 1) / tile : 0);
    }
    __device__ __forceinline__ int32_t first_key(int32_t t, int32_t tile) const {
        return t < sink_tiles ? t * tile : start + (t - sink_tiles) * tile;
    }
};

// Workgroups are handed to the 8 XCDs in turn, each with an L2 of its own: the
// items (all of a head next to each other) are dealt out in 8 runs, so that a
// head's workgroups share one L2.  Returns items or more past the last one.
__device__ __forceinline__ int64_t xcd_item(int64_t items, uint32_t place) {
    const int64_t per = (items + 7) / 8;
    return (place & 7) * per + (place >> 3);
}
__host__ __device__ inline int64_t xcd_grid(int64_t items) { return (items + 7) / 8 * 8; }

constexpr int64_t kMaxAttentionItems = int64_t{1} << 23;   // 256 threads each: below 2^32

// What every entry point asks of its tensors (attention.hip).
int32_t check_attention(const lct_attention *a);
// Joins the parts of a->queries' keys into a.out and, unless NULL, a.lse.
int32_t join_parts(const lct_attention &a, int32_t splits, const float *parts, hipStream_t stream);

// Calls launch(integral_constant<head width in registers>).
template <class Launch>
void by_width(int32_t dim, Launch launch) {
    if (dim <= 32) launch(std::integral_constant<int, 32>{});
    else if (dim <= 64) launch(std::integral_constant<int, 64>{});
    else if (dim <= 96) launch(std::integral_constant<int, 96>{});
    else launch(std::integral_constant<int, 128>{});
}

}  // namespace lct
