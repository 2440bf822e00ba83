// Attention with a sliding window and sinks, forward and backward.
//
// Follows LCT/components/layers.py:225-305, whose causal attention is a library's.
// out = softmax(scale q k^T) v over the keys that a query sees: the last `window`
// up to its own and the first `sinks` (attention_core.h).  Only tiles that some
// query of a workgroup sees are loaded, a wave skips those that none of its own
// sees, and those that all of them see are computed without masks.
#include <algorithm>
#include <type_traits>

#include "attention_core.h"

namespace lct {
namespace {

constexpr int kQueryTile = 128;      // queries of a workgroup, 32 per wave
constexpr int kKeyTile = 64;         // keys per step
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHalfWeights = 256.0f;
constexpr int32_t kFewKeys = 64;     // rows of up to so many keys get an exact delta
constexpr int32_t kMaxTokens = 1 << 30;

// lse's and delta's values per head: whole query tiles, the last one's extra
// rows among them.
__host__ __device__ __forceinline__ int64_t lse_pitch(int32_t queries) {
    return (int64_t{queries} + kQueryTile - 1) / kQueryTile * kQueryTile;
}

// A lane's share of one row (4 of each 8 channels), times `factor`.
template <bool kHalf, int kColumns>
__device__ __forceinline__ void store_row(uint16_t *dst, const f32x16 (&x)[kColumns], float factor,
                                          int32_t dim) {
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int32_t channel = 32 * c + 8 * g + 4 * (wave_lane() >> 5);
            if (channel >= dim) continue;
            u32x2 pairs;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                pairs[i] = Element<kHalf>::round_pair(x[c][4 * g + 2 * i] * factor,
                                                      x[c][4 * g + 2 * i + 1] * factor);
            *reinterpret_cast<u32x2 *>(dst + channel) = pairs;
        }
}

// ---- infinities and NaN in masked places
//
// A masked weight is an exact zero, but the matrix instructions multiply it, and
// zero times an infinity or a NaN is a NaN: values that a query does not see
// reach it where they share a tile with some that it does.  Padding is loaded
// as zeros; for the rest a wave looks at its sums when they are done, and where
// one is not finite it computes its rows again, key by key, from what they see
// alone: 100 cycles per pair, and only then.

// Whether a sum of the wave is an infinity or a NaN.
template <int kCount>
__device__ __forceinline__ bool not_finite(const f32x16 (&x)[kCount]) {
    float probe = 0.0f;
#pragma unroll
    for (int c = 0; c < kCount; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) probe = __builtin_fmaf(x[c][r], 0.0f, probe);
    return __any(!(probe == 0.0f));
}

// One row's two channels of this lane; zeros past the head's width.
__device__ __forceinline__ uint32_t lane_pair(const uint16_t *row, int32_t dim) {
    const int32_t channel = 2 * wave_lane();
    return channel < dim ? *reinterpret_cast<const uint32_t *>(row + channel) : 0u;
}

template <bool kHalf>
__device__ __forceinline__ float row_product(uint32_t a, uint32_t b) {
    using E = Element<kHalf>;
    float sum = E::low(a) * E::low(b) + E::high(a) * E::high(b);
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, kWave);
    return sum;
}

__device__ __forceinline__ float of_lane(float v, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// A workgroup has 128 queries of a head, a wave 32 of them, and walks its key
// tiles once: scores with the keys in their rows (a lane's 32 scores of a tile are
// one query's, so its maximum and sum need one exchange between two lanes), the
// running maximum and sum of the softmax per lane, and the product with the
// values.  The next tile's keys and values are on their way to LDS meanwhile.
//
// The maximum may lag by 2^kRescale before the sums are scaled to a new one: all
// are FP32, so the weights' larger values cost no precision, and after the first
// tiles the 32 to 128 products are rarely due.  The weights are rounded to the
// tensors' type for the product (BF16 2^-9, FP16 2^-12 of each weight); their sum is
// taken before.
//
// Matrix instructions, LDS reads (one fragment per instruction) and the softmax's
// vector instructions take about 512, 512 and 450 clocks of a SIMD per 32 x 32
// scores at heads of 128, at 1.9 to 2.0 GHz under this load; the two waves of a
// SIMD overlap them in part (matrix instructions busy half of the time).  1500 to
// 1580 us for 8191 queries after 8192 keys, 32 heads of 128 over 8 (1045 to 1100
// TFLOP/s; 1580 where 1525 with the compiler's order of LDS reads in place of
// read_ahead; in FP16 1680 to 1750); 485 to 500 us for 1 x 16384, 16 heads over 4,
// window 4096 (960 to 990); 22 to 23 us for 8 x 1024, 12 heads of 64, window 256, whose
// few steps per wave leave it to latency (while a CU has work, 0.56 of the launch,
// its vector units are 0.55 busy, its matrix units 0.21).  Tried at the first of these,
// then 1525: 32-key halves of a tile with the second half's scores issued between the
// first's exponentials 1650 us; matrix phases at a higher wave priority 1560; column
// reads without the wait that the compiler puts before them 1645; 64 queries per wave,
// which halve the LDS reads but leave one wave per SIMD, 2020 with the instructions
// interleaved by hand; 8 waves per workgroup, 4 in their products while the other 4
// are in their softmax, 1605.
template <bool kHalf, int kDim, bool kSplit>
__global__ __launch_bounds__(kAttentionThreads, 2) void attention_forward_kernel(
    lct_attention a, int32_t tiles, int32_t splits, float *__restrict__ parts) {
    constexpr int kPitch = kPitchOf<kDim>;
    constexpr int kSteps = kDim / 16, kColumns = kDim / 32;
    __shared__ __attribute__((aligned(1024))) uint16_t k_even[kKeyTile * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t v_even[kKeyTile * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t k_odd[kKeyTile * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t v_odd[kKeyTile * kPitch];

    const int64_t per_head = int64_t{tiles} * splits;
    const int64_t item = xcd_item(per_head * a.batch * a.heads, blockIdx.x);
    if (item >= per_head * a.batch * a.heads) return;
    const int32_t bh = static_cast<int32_t>(item / per_head);
    const int32_t part = static_cast<int32_t>(item % per_head);
    const int32_t b = bh / a.heads, h = bh % a.heads, kv = h / (a.heads / a.kv_heads);
    // The last queries see the most keys: they go first.
    const int32_t tile = tiles - 1 - part / splits, split = part % splits;

    const int lane = wave_lane(), half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int32_t shift = a.keys - a.queries;
    const int32_t length = sequence_length(a, b);
    const int32_t first = tile * kQueryTile;
    const int32_t last = min(first + kQueryTile, a.queries) - 1;
    const KeyTiles all(a, first + shift, last + shift, length, kKeyTile);
    const int32_t per_split = (all.count + splits - 1) / splits;
    const int32_t begin = split * per_split, end = min(all.count, begin + per_split);

    // This wave's queries, one per lane (twice): q, and what each sees.
    const int32_t wave_first = first + 32 * wave;
    const int32_t row = wave_first + (lane & 31);
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + b * a.q_stride[0] + h * a.q_stride[1];
    u32x4 q_operand[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
        q_operand[s] = load_operand(q, a.q_stride[2], row, a.queries, a.head_dim, s);
    const int32_t position =
        row < a.queries && row + shift >= 0 && row + shift < length ? row + shift : kNowhere;
    const int32_t tile_sinks = a.window > 0 ? a.sinks : 0;
    const int32_t low_position = wave_first + shift;
    const int32_t high_position = min(wave_first + 31, a.queries - 1) + shift;

    const uint16_t *k = static_cast<const uint16_t *>(a.k) + b * a.k_stride[0] + kv * a.k_stride[1];
    const uint16_t *v = static_cast<const uint16_t *>(a.v) + b * a.v_stride[0] + kv * a.v_stride[1];
    TileLoads<kKeyTile, kPitch> k_loads, v_loads;
    k_loads.prepare(a.k_stride[2], a.head_dim);
    v_loads.prepare(a.v_stride[2], a.head_dim);
    const auto load = [&](int32_t t, uint16_t *keys, uint16_t *values)
                          __attribute__((always_inline)) {
        const int32_t key = all.first_key(t, kKeyTile);
        k_loads.issue(k + key * a.k_stride[2], length - key, a.k_stride[2], a.head_dim, keys);
        v_loads.issue(v + key * a.v_stride[2], length - key, a.v_stride[2], a.head_dim, values);
    };

    const float factor = a.scale * kLog2e;
    f32x16 out[kColumns];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) out[c] = f32x16{};
    float most = -INFINITY;     // the scores' running maximum, or up to kRescale below
    float shifted = 0.0f;       // its product with factor, 0 while no key was seen
    float total = 0.0f;         // this lane's keys' weights

    const auto step = [&](int32_t t, const uint16_t *keys, const uint16_t *values)
                          __attribute__((always_inline)) {
        const int32_t key = all.first_key(t, kKeyTile);
        const bool seen_by_some =
            key <= high_position
            && (a.window == 0 || key + kKeyTile > low_position - a.window + 1 || key < a.sinks);
        if (!seen_by_some) return;
        const bool seen_by_all =
            key + kKeyTile - 1 <= low_position && high_position < length
            && (a.window == 0 || high_position - key < a.window || key + kKeyTile <= a.sinks);
        f32x16 s[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n] = f32x16{};
#pragma unroll
            for (int d = 0; d < kSteps; ++d)
                s[n] = Element<kHalf>::multiply(read_rows<kPitch>(keys, n, d), q_operand[d], s[n]);
        }
        read_ahead<2 * kSteps, 1, 2>();
        if (!seen_by_all) {
            const TileSight sight(a, position, key);
#pragma unroll
            for (int n = 0; n < 2; ++n)
                sight.each(key, 32 * n, tile_sinks,
                           [&](int r, bool seen) { s[n][r] = seen ? s[n][r] : -INFINITY; });
        }
        float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(fmaxf(top, s[0][r]), s[1][r]);
        top = across_max(top);
        if (__any(top * factor > most * factor + kRescale)) {
            const float next = fmaxf(most, top);
            const float scaled = next == -INFINITY ? 0.0f : next * factor;
            const float change = exp2_fast(most * factor - scaled);
            most = next;
            shifted = scaled - (kHalf ? kHalfLift : 0.0f);
            total *= change;
#pragma unroll
            for (int c = 0; c < kColumns; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) out[c][r] *= change;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[n][r] = exp2_fast(__builtin_fmaf(s[n][r], factor, -shifted));
                total += s[n][r];
            }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const u32x4 weights = as_operand<kHalf>(s[n], p);
#pragma unroll
                for (int c = 0; c < kColumns; ++c)
                    out[c] = Element<kHalf>::multiply(
                        read_columns<kPitch>(values, 32 * n + 16 * p, c), weights, out[c]);
            }
        read_ahead<4 * kColumns, 2, 6>();
    };

    if (begin < end) load(begin, k_even, v_even);
    for (int32_t t = begin; t < end; t += 2) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 1 < end) load(t + 1, k_odd, v_odd);
        step(t, k_even, v_even);
        if (t + 1 >= end) break;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 2 < end) load(t + 2, k_even, v_even);
        step(t + 1, k_odd, v_odd);
    }

    total = across_sum(total);
    if (not_finite(out)) {
        const int32_t channel = 2 * lane;
        for (int r = 0; r < 32; ++r) {
            const int32_t at = wave_first + r;
            if (at >= a.queries) break;
            const Sight seen = sight_of(a, at + shift, length);
            const uint32_t q_pair = lane_pair(q + at * a.q_stride[2], a.head_dim);
            float largest = -INFINITY, base = 0.0f, sum = 0.0f, x = 0.0f, y = 0.0f;
            for (int32_t t = begin; t < end; ++t) {
                const int32_t key = all.first_key(t, kKeyTile);
                for (int32_t j = key; j < key + kKeyTile; ++j) {
                    if (!seen(j)) continue;
                    const uint32_t v_pair = lane_pair(v + j * a.v_stride[2], a.head_dim);
                    const float score =
                        factor
                        * row_product<kHalf>(q_pair, lane_pair(k + j * a.k_stride[2], a.head_dim));
                    largest = fmaxf(largest, score);
                    const float next = largest == -INFINITY ? 0.0f : largest;
                    const float change = sum == 0.0f ? 0.0f : exp2_fast(base - next);
                    const float weight = exp2_fast(score - next);
                    base = next;
                    x = (sum == 0.0f ? 0.0f : x * change) + weight * Element<kHalf>::low(v_pair);
                    y = (sum == 0.0f ? 0.0f : y * change) + weight * Element<kHalf>::high(v_pair);
                    sum = sum * change + weight;
                }
            }
            if constexpr (kSplit) {
                float *part_out =
                    parts + ((int64_t{bh} * splits + split) * a.queries + at) * (a.head_dim + 2);
                if (channel < a.head_dim)
                    *reinterpret_cast<f32x2 *>(part_out + channel) = f32x2{x, y};
                if (lane == 0) *reinterpret_cast<f32x2 *>(part_out + a.head_dim) = f32x2{base, sum};
            } else {
                const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
                if (channel < a.head_dim)
                    *reinterpret_cast<uint32_t *>(
                        static_cast<uint16_t *>(a.out) + b * a.out_stride[0] + h * a.out_stride[1]
                        + at * a.out_stride[2] + channel) =
                        Element<kHalf>::round_pair(x * inverse, y * inverse);
                if (a.lse != nullptr && lane == 0)
                    a.lse[int64_t{bh} * lse_pitch(a.queries) + at] =
                        sum == 0.0f ? INFINITY : base + __log2f(sum);
            }
        }
        if (!kSplit && a.lse != nullptr && half == 0 && row >= a.queries)
            a.lse[int64_t{bh} * lse_pitch(a.queries) + row] = INFINITY;
        return;
    }
    if constexpr (kSplit) {
        if (row >= a.queries) return;
        float *part_out =
            parts + ((int64_t{bh} * splits + split) * a.queries + row) * (a.head_dim + 2);
#pragma unroll
        for (int c = 0; c < kColumns; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int32_t channel = 32 * c + 8 * g + 4 * half;
                if (channel >= a.head_dim) continue;
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    *reinterpret_cast<f32x2 *>(part_out + channel + i) =
                        f32x2{out[c][4 * g + i], out[c][4 * g + i + 1]};
            }
        if (half == 0)
            *reinterpret_cast<f32x2 *>(part_out + a.head_dim) = f32x2{shifted, total};
        return;
    }
    // Rows past the last query have no output but a place in lse.
    if (a.lse != nullptr && half == 0)
        a.lse[int64_t{bh} * lse_pitch(a.queries) + row] =
            total == 0.0f || row >= a.queries ? INFINITY : shifted + __log2f(total);
    if (row >= a.queries) return;
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t *dst = static_cast<uint16_t *>(a.out) + b * a.out_stride[0] + h * a.out_stride[1]
                    + row * a.out_stride[2];
    store_row<kHalf, kColumns>(dst, out, inverse, a.head_dim);
}

// Joins the parts of a query's keys: sum of 2^(shift - largest) out, over the
// same sum of the weights.  A workgroup per query, two channels per lane, a
// quarter of the parts per wave; lane s holds part s's shift and weight, so the
// parts' loads do not wait for each other (64 queries of 16 parts: 5.5 us; a wave
// per query that read part after part: 18).
template <bool kHalf>
__global__ __launch_bounds__(kAttentionThreads) void attention_join_kernel(
    lct_attention a, int64_t pitch, int32_t splits, const float *__restrict__ parts) {
    static_assert(LCT_MAX_ATTENTION_SPLITS <= kWave, "a lane per part");
    __shared__ f32x2 sums[kAttentionWaves][kWave];
    const int64_t item = blockIdx.x;
    const int32_t bh = static_cast<int32_t>(item / pitch), row = static_cast<int32_t>(item % pitch);
    const int lane = wave_lane(), wave = threadIdx.x / kWave;
    if (row >= a.queries) {
        if (threadIdx.x == 0) a.lse[item] = INFINITY;
        return;
    }
    const int32_t width = a.head_dim + 2, channel = 2 * lane;
    const float *part = parts + (int64_t{bh} * splits * a.queries + row) * width;
    const int64_t step = int64_t{a.queries} * width;
    f32x2 stats = {0.0f, 0.0f};
    if (lane < splits) stats = *reinterpret_cast<const f32x2 *>(part + lane * step + a.head_dim);
    float largest = stats[1] != 0.0f ? stats[0] : -INFINITY;
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d, kWave));
    const float weight = stats[1] != 0.0f ? exp2_fast(stats[0] - largest) : 0.0f;
    float total = weight * stats[1];
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) total += __shfl_xor(total, d, kWave);
    f32x2 sum = {0.0f, 0.0f};
    if (channel < a.head_dim) {
#pragma unroll 4
        for (int32_t s = wave; s < splits; s += kAttentionWaves) {
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), s));
            const f32x2 o = *reinterpret_cast<const f32x2 *>(part + s * step + channel);
            // A part that saw nothing has no sums.
            if (w != 0.0f) sum += w * o;
        }
    }
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave != 0) return;
    if (a.lse != nullptr && lane == 0)
        a.lse[item] = total == 0.0f ? INFINITY : largest + __log2f(total);
    if (channel >= a.head_dim) return;
#pragma unroll
    for (int w = 1; w < kAttentionWaves; ++w) sum += sums[w][lane];
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t *dst = static_cast<uint16_t *>(a.out) + (bh / a.heads) * a.out_stride[0]
                    + (bh % a.heads) * a.out_stride[1] + row * a.out_stride[2];
    *reinterpret_cast<uint32_t *>(dst + channel) =
        Element<kHalf>::round_pair(sum[0] * inverse, sum[1] * inverse);
}

// ---- backward
//
// With P = 2^(factor s - lse), dP = dO v^T and delta = sum(dO out):
// dS = P (dP - delta), dq = scale dS k, dk = scale dS^T q, dv = P^T dO.  Two
// kernels, one per side that is summed over, each of which computes the scores
// again: seven products in place of five, but no sum is shared between
// workgroups, so results do not depend on timing.

// dS is the product of a weight and an incoming gradient, often far below FP16's
// normal numbers (and now and then above its largest): 4096 keys under gradients of
// 1e-4 left a fifth of them zero.  In FP16 a lane, whose sums are of one query or
// key, holds them and each dS times a power of two that begins at 2^60 (FP16's
// least products are 2^-48) and goes down to put the largest dS so far between 2^8
// and 2^15.  What is 2^22 smaller is still rounded to FP16's 11 bits.  A lane's
// maximum of 16 numbers per 32 x 32 scores: at 1 x 16384, 16 heads of 128 over 4,
// window 4096, dq takes 720 us where it took 690, dk and dv 1230 as before; at 8 x
// 1024, 12 heads of 64, window 256, 32.8 for 29.7 and 41.4 for 40.3.
constexpr float kHalfPower = 60.0f, kHalfFirst = 0x1p60f;
constexpr float kHalfMost = 0x1p15f;

template <int kColumns>
__device__ __forceinline__ void multiply_all(f32x16 (&x)[kColumns], float factor) {
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[c][r] *= factor;
}

// Multiplies `ds` and `sums` by a power of two, lowered(factor), where `ds` is too large.
template <int kColumns, class Lowered>
__device__ __forceinline__ void lower_half(f32x16 &ds, f32x16 (&sums)[kColumns], Lowered lowered) {
    float top = fmaxf(fabsf(ds[0]), fabsf(ds[1]));
#pragma unroll
    for (int r = 2; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
    if (!__any(top > kHalfMost)) return;
    top = across_max(top);                   // of both lanes that share the sums
    const float factor =
        top > kHalfMost ? __uint_as_float((262u << 23) - (__float_as_uint(top) & 0x7F800000u))
                        : 1.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= factor;
    multiply_all(sums, factor);
    lowered(factor);
}

// A wave's 32 queries, the keys in tiles of 64: as in the forward kernel, with dP
// beside the scores (its sums begin at -delta) and the keys' columns for the last
// product.  delta is taken from the operands on their way in, and stored for the
// other kernel.  650 to 670 us for 1 x 16384, 16 heads of 128 over 4, window 4096 (1080
// to 1110 TFLOP/s; 690 with the compiler's order of LDS reads), 29 to 30 us for 8 x
// 1024, 12 heads of 64, window 256, three waves per SIMD (in FP16 32.8; two waves 38.5),
// by latency: CUs have work in 0.63 of it, vector units then 0.42 busy, matrix 0.23.
template <bool kHalf, int kDim>
__global__ __launch_bounds__(kAttentionThreads, kDim > 64 ? 2 : 3) void attention_dq_kernel(
    lct_attention a, lct_attention_gradients d, int32_t tiles) {
    constexpr int kPitch = kPitchOf<kDim>;
    constexpr int kSteps = kDim / 16, kColumns = kDim / 32;
    __shared__ __attribute__((aligned(1024))) uint16_t k_even[kKeyTile * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t v_even[kKeyTile * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t k_odd[kKeyTile * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t v_odd[kKeyTile * kPitch];

    const int64_t items = int64_t{tiles} * a.batch * a.heads;
    const int64_t item = xcd_item(items, blockIdx.x);
    if (item >= items) return;
    const int32_t bh = static_cast<int32_t>(item / tiles);
    const int32_t b = bh / a.heads, h = bh % a.heads, kv = h / (a.heads / a.kv_heads);
    const int32_t tile = tiles - 1 - static_cast<int32_t>(item % tiles);

    const int lane = wave_lane(), half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int32_t shift = a.keys - a.queries;
    const int32_t length = sequence_length(a, b);
    const int32_t first = tile * kQueryTile;
    const int32_t last = min(first + kQueryTile, a.queries) - 1;
    const KeyTiles all(a, first + shift, last + shift, length, kKeyTile);

    const int32_t wave_first = first + 32 * wave;
    const int32_t row = wave_first + (lane & 31);
    const int32_t position =
        row < a.queries && row + shift >= 0 && row + shift < length ? row + shift : kNowhere;
    const int32_t tile_sinks = a.window > 0 ? a.sinks : 0;
    const int32_t low_position = wave_first + shift;
    const int32_t high_position = min(wave_first + 31, a.queries - 1) + shift;
    // Queries that see nothing take part as zeros.
    const int32_t rows = position != kNowhere ? a.queries : 0;

    u32x4 q_operand[kSteps], g_operand[kSteps];
    float delta = 0.0f;
    {
        const uint16_t *q =
            static_cast<const uint16_t *>(a.q) + b * a.q_stride[0] + h * a.q_stride[1];
        const uint16_t *g = static_cast<const uint16_t *>(d.grad) + b * d.grad_stride[0]
                            + h * d.grad_stride[1];
        const uint16_t *o =
            static_cast<const uint16_t *>(a.out) + b * a.out_stride[0] + h * a.out_stride[1];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q_operand[s] = load_operand(q, a.q_stride[2], row, rows, a.head_dim, s);
            g_operand[s] = load_operand(g, d.grad_stride[2], row, rows, a.head_dim, s);
            const u32x4 out = load_operand(o, a.out_stride[2], row, rows, a.head_dim, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                delta += Element<kHalf>::low(g_operand[s][i]) * Element<kHalf>::low(out[i]);
                delta += Element<kHalf>::high(g_operand[s][i]) * Element<kHalf>::high(out[i]);
            }
        }
    }
    delta = across_sum(delta);
    const int64_t at = int64_t{bh} * lse_pitch(a.queries) + row;

    const uint16_t *k = static_cast<const uint16_t *>(a.k) + b * a.k_stride[0] + kv * a.k_stride[1];
    const uint16_t *v = static_cast<const uint16_t *>(a.v) + b * a.v_stride[0] + kv * a.v_stride[1];
    TileLoads<kKeyTile, kPitch> k_loads, v_loads;
    k_loads.prepare(a.k_stride[2], a.head_dim);
    v_loads.prepare(a.v_stride[2], a.head_dim);
    const auto load = [&](int32_t t, uint16_t *keys, uint16_t *values)
                          __attribute__((always_inline)) {
        const int32_t key = all.first_key(t, kKeyTile);
        k_loads.issue(k + key * a.k_stride[2], length - key, a.k_stride[2], a.head_dim, keys);
        v_loads.issue(v + key * a.v_stride[2], length - key, a.v_stride[2], a.head_dim, values);
    };

    const float factor = a.scale * kLog2e;
    f32x16 dq[kColumns];
    float base = -a.lse[at]; // what exponents begin at; in FP16 with dS's power of two
    float rest = 0.0f;       // this lane's keys' sum of dS
    const auto step = [&](auto sums, int32_t t, const uint16_t *keys, const uint16_t *values)
                          __attribute__((always_inline)) {
        const int32_t key = all.first_key(t, kKeyTile);
        const bool seen_by_some =
            key <= high_position
            && (a.window == 0 || key + kKeyTile > low_position - a.window + 1 || key < a.sinks);
        if (!seen_by_some) return;
        const bool seen_by_all =
            key + kKeyTile - 1 <= low_position && high_position < length
            && (a.window == 0 || high_position - key < a.window || key + kKeyTile <= a.sinks);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f32x16 s{}, e;
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = -delta;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                s = Element<kHalf>::multiply(read_rows<kPitch>(keys, n, i), q_operand[i], s);
                e = Element<kHalf>::multiply(read_rows<kPitch>(values, n, i), g_operand[i], e);
            }
            read_ahead<2 * kSteps, 1, 4>();
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[r] = exp2_fast(__builtin_fmaf(s[r], factor, base)) * e[r];
            if (!seen_by_all)
                TileSight(a, position, key).each(
                    key, 32 * n, tile_sinks,
                    [&](int r, bool seen) { s[r] = seen ? s[r] : 0.0f; });
            if constexpr (decltype(sums)::value) {
#pragma unroll
                for (int r = 0; r < 16; ++r) rest += s[r];
            } else {
                if constexpr (kHalf)
                    lower_half(s, dq, [&](float factor) {
                        base += static_cast<float>(
                            static_cast<int32_t>(__float_as_uint(factor) >> 23) - 127);
                    });
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const u32x4 ds = as_operand<kHalf>(s, p);
#pragma unroll
                    for (int c = 0; c < kColumns; ++c)
                        dq[c] = Element<kHalf>::multiply(
                            read_columns<kPitch>(keys, 32 * n + 16 * p, c), ds, dq[c]);
                }
                read_ahead<2 * kColumns, 2, 6>();
            }
        }
    };

    const auto walk = [&](auto sums) __attribute__((always_inline)) {
        if (all.count > 0) load(0, k_even, v_even);
        for (int32_t t = 0; t < all.count; t += 2) {
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (t + 1 < all.count) load(t + 1, k_odd, v_odd);
            step(sums, t, k_even, v_even);
            if (t + 1 >= all.count) break;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (t + 2 < all.count) load(t + 2, k_even, v_even);
            step(sums, t + 1, k_odd, v_odd);
        }
    };
    // A row's dS sum to zero: what they sum to is what the rounding of `out` left in
    // delta.  Where rows see few keys, that reaches dq and dk as much as the rounding
    // of dS does (their error against FP64 is 1.48 and 1.47 times that of one
    // rounding without this, 1.43 and 1.42 with it, at 515 tokens under a window of
    // 127; rows of 16 keys and less make the difference), so it is taken out first.
    // Where the window makes all rows such ones, every workgroup walks twice: 26.4 us
    // at 8 x 1024, 12 heads of 64, window 64, for 21.9 at window 65.
    const bool few = first + shift < kFewKeys
                     || (a.window > 0 && a.window <= kFewKeys && a.sinks <= kFewKeys - a.window);
    if (few) {
        walk(std::true_type{});
        delta += across_sum(rest);
        __syncthreads();                 // all have read the tiles of this pass
    }
    if (half == 0) d.delta[at] = delta;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) dq[c] = f32x16{};
    if constexpr (kHalf) base += kHalfPower;
    walk(std::false_type{});
    if constexpr (kHalf) {
        // A row that sees nothing has no power, and zeros.
        const float power = base + a.lse[at];
        multiply_all(dq, power == power ? exp2_fast(-power) : 1.0f);
    }
    if (not_finite(dq)) {
        const int32_t channel = 2 * lane;
        const uint16_t *q =
            static_cast<const uint16_t *>(a.q) + b * a.q_stride[0] + h * a.q_stride[1];
        const uint16_t *g = static_cast<const uint16_t *>(d.grad) + b * d.grad_stride[0]
                            + h * d.grad_stride[1];
        for (int r = 0; r < 32; ++r) {
            const int32_t at = wave_first + r;
            if (at >= a.queries) break;
            const Sight seen = sight_of(a, at + shift, length);
            const uint32_t q_pair = lane_pair(q + at * a.q_stride[2], a.head_dim);
            const uint32_t g_pair = lane_pair(g + at * d.grad_stride[2], a.head_dim);
            const float row_lse = a.lse[int64_t{bh} * lse_pitch(a.queries) + at];
            const float row_delta = of_lane(delta, r);
            float x = 0.0f, y = 0.0f;
            for (int32_t t = 0; t < all.count; ++t) {
                const int32_t key = all.first_key(t, kKeyTile);
                for (int32_t j = key; j < key + kKeyTile; ++j) {
                    if (!seen(j)) continue;
                    const uint32_t k_pair = lane_pair(k + j * a.k_stride[2], a.head_dim);
                    const float score = row_product<kHalf>(q_pair, k_pair);
                    const float dp = row_product<kHalf>(
                        g_pair, lane_pair(v + j * a.v_stride[2], a.head_dim));
                    const float ds =
                        exp2_fast(__builtin_fmaf(score, factor, -row_lse)) * (dp - row_delta);
                    x += ds * Element<kHalf>::low(k_pair);
                    y += ds * Element<kHalf>::high(k_pair);
                }
            }
            if (channel < a.head_dim)
                *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(d.dq) + b * d.dq_stride[0]
                                              + h * d.dq_stride[1] + at * d.dq_stride[2]
                                              + channel) =
                    Element<kHalf>::round_pair(x * a.scale, y * a.scale);
        }
        return;
    }
    if (row >= a.queries) return;
    uint16_t *dst = static_cast<uint16_t *>(d.dq) + b * d.dq_stride[0] + h * d.dq_stride[1]
                    + row * d.dq_stride[2];
    store_row<kHalf, kColumns>(dst, dq, a.scale, a.head_dim);
}

// From a part of a key block's gradients in the workspace to the next.  A power of
// two, of which all parts of a key lie a multiple apart, would put them on the same
// channels of the memory: the sum of 61 parts of 256 keys of 4 heads of 128 took 39
// us, and takes 15; of 9 parts of 128 keys 9 and 5.7.
__host__ __device__ __forceinline__ int64_t part_pitch(int32_t per_block, int32_t dim) {
    return int64_t{2} * per_block * dim + LCT_ATTENTION_PART_GAP;
}

// How a key block's queries are shared: blocks that hold sinks are seen by all
// later queries and have parts of their own number.  A kind of one part stores its
// gradients itself and has no place in the workspace.
struct KeyBlocks {
    int32_t blocks, sink_blocks, splits, sink_splits;
    __host__ __device__ __forceinline__ int64_t sink_parts() const {
        return int64_t{sink_blocks} * sink_splits;
    }
    __host__ __device__ __forceinline__ int64_t other_parts() const {
        return int64_t{blocks - sink_blocks} * splits;
    }
    __host__ __device__ __forceinline__ int64_t stored_sink_parts() const {
        return sink_splits > 1 ? sink_parts() : 0;
    }
    // Of a head, in the workspace.
    __host__ __device__ __forceinline__ int64_t stored_parts() const {
        return stored_sink_parts() + (splits > 1 ? other_parts() : 0);
    }
    // Of a block of several parts.
    __host__ __device__ __forceinline__ int64_t first_part(int32_t block) const {
        return block < sink_blocks ? int64_t{block} * sink_splits
                                   : stored_sink_parts() + int64_t{block - sink_blocks} * splits;
    }
    // One past the last block that may have several.
    __host__ __device__ __forceinline__ int32_t end_of_parts() const {
        return splits > 1 ? blocks : sink_blocks;
    }
    __host__ __device__ __forceinline__ int32_t parts_of(int32_t block) const {
        return block < sink_blocks ? sink_splits : splits;
    }
};

constexpr int kQueryStep = 64;       // queries per step

// Keys of a workgroup of the kernel below.
__host__ __device__ constexpr int key_block(int dim) { return dim > 64 ? 256 : 128; }

// A wave's 32 keys, the queries (of all heads that share them) in tiles of 64;
// S and dP have the queries in their rows, so that P and dS are the operands of
// dv and dk, whose other operands are the columns of the tiles that S and dP read
// by rows.
//
// Four products per tile, each fragment of LDS read for one of them: LDS (128
// bytes a clock, what four SIMDs' matrix instructions use) and the matrix
// instructions are busy alike.  Heads wider than 64 hold 128 registers of sums and
// 32 of the keys' operands; the values' stay in LDS (64 KB for 256 keys, read
// again for each tile), so that two waves share a SIMD.  1060 to 1200 us for 1 x 16384,
// 16 heads of 128 over 4, window 4096 (800 to 910 TFLOP/s; 1110 where 1080 with the
// compiler's order of LDS reads; 0.16 of it the end, when the workgroups of the last
// keys, which fewer queries see, are done: parts of equal work would cost as much to
// add); 64 keys per wave at one wave per SIMD, which read half as much: 1420; 32 with
// all operands in registers at one wave per SIMD: 2200.  8 x 1024, 12 heads of 64,
// window 256: 38 to 39 us at three waves per SIMD (two: 42), by latency: CUs have work
// in 0.65 of it, vector units then 0.34 busy, matrix 0.19.
template <bool kHalf, int kDim>
__global__ __launch_bounds__(key_block(kDim) * 2, kDim > 64 ? 2 : 3) void attention_dkdv_kernel(
    lct_attention a, lct_attention_gradients d, KeyBlocks blocks, float *__restrict__ parts) {
    constexpr int kPitch = kPitchOf<kDim>;
    constexpr int kSteps = kDim / 16, kColumns = kDim / 32;
    constexpr int kKeyBlock = key_block(kDim), kWaveKeys = 32, kThreads = kKeyBlock * 2;
    __shared__ __attribute__((aligned(1024))) uint16_t q_even[kQueryStep * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t g_even[kQueryStep * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t q_odd[kQueryStep * kPitch];
    __shared__ __attribute__((aligned(1024))) uint16_t g_odd[kQueryStep * kPitch];
    __shared__ __attribute__((aligned(1024))) float stats_even[2 * kQueryStep];
    __shared__ __attribute__((aligned(1024))) float stats_odd[2 * kQueryStep];
    // Wide heads leave no registers for the values' operands beside the sums.
    constexpr bool kStaged = kDim > 64;
    __shared__ __attribute__((aligned(1024))) uint16_t v_block[kStaged ? kKeyBlock * kPitch : 512];

    // The blocks without sinks, then those with: each kind dealt out over the
    // XCDs by itself, since their parts are of unequal length.
    const int64_t heads = int64_t{a.batch} * a.kv_heads;
    const int64_t other_items = blocks.other_parts() * heads;
    const uint32_t other_grid = static_cast<uint32_t>(xcd_grid(other_items));
    const bool sinks = blockIdx.x >= other_grid;
    const int64_t items = sinks ? blocks.sink_parts() * heads : other_items;
    const int64_t item = xcd_item(items, sinks ? blockIdx.x - other_grid : blockIdx.x);
    if (item >= items) return;
    const int64_t per_head = sinks ? blocks.sink_parts() : blocks.other_parts();
    const int32_t bkv = static_cast<int32_t>(item / per_head);
    const int32_t b = bkv / a.kv_heads, kv = bkv % a.kv_heads, group = a.heads / a.kv_heads;
    const int32_t part = static_cast<int32_t>(item % per_head);
    const int32_t splits = sinks ? blocks.sink_splits : blocks.splits;
    const int32_t block = (sinks ? 0 : blocks.sink_blocks) + part / splits, split = part % splits;

    const int lane = wave_lane(), half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int32_t shift = a.keys - a.queries;
    const int32_t length = sequence_length(a, b);
    const int32_t first = block * kKeyBlock;
    // Positions that see some of the block's keys, and their queries' tiles.
    const int32_t last_key = min(first + kKeyBlock, length) - 1;
    const int32_t last_position =
        last_key < first                            ? -1
        : a.window == 0 || first < a.sinks          ? length - 1
        : last_key > length - a.window              ? length - 1
                                                    : last_key + a.window - 1;
    const int32_t live = min(a.queries, length - shift);     // queries below the length
    const int32_t low = max(0, first - shift), high = min(live, last_position + 1 - shift);
    const int32_t low_tile = low / kQueryStep;
    const int32_t per_query_head =
        high > low ? (high + kQueryStep - 1) / kQueryStep - low_tile : 0;
    const int32_t steps = per_query_head * group;
    const int32_t per_split = (steps + splits - 1) / splits;
    const int32_t begin = split * per_split, end = min(steps, begin + per_split);

    const int32_t wave_first = first + kWaveKeys * wave;
    const uint16_t *k = static_cast<const uint16_t *>(a.k) + b * a.k_stride[0] + kv * a.k_stride[1];
    const uint16_t *v = static_cast<const uint16_t *>(a.v) + b * a.v_stride[0] + kv * a.v_stride[1];
    const int32_t key = wave_first + (lane & 31);
    u32x4 k_operand[kSteps], v_operand[kStaged ? 1 : kSteps];
    if constexpr (kStaged) {
        TileLoads<kQueryStep, kPitch, kThreads> v_loads;
        v_loads.prepare(a.v_stride[2], a.head_dim);
#pragma unroll
        for (int i = 0; i < kKeyBlock; i += kQueryStep)
            v_loads.issue(v + (first + i) * a.v_stride[2], length - first - i, a.v_stride[2],
                          a.head_dim, v_block + i * kPitch);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        k_operand[s] = load_operand(k, a.k_stride[2], key, length, a.head_dim, s);
        if constexpr (!kStaged)
            v_operand[s] = load_operand(v, a.v_stride[2], key, length, a.head_dim, s);
    }

    TileLoads<kQueryStep, kPitch, kThreads> q_loads, g_loads;
    q_loads.prepare(a.q_stride[2], a.head_dim);
    g_loads.prepare(d.grad_stride[2], a.head_dim);
    // The step that is loaded next: its head and its tile of queries.
    int32_t next_head = kv * group, next_tile = low_tile;
    if (begin < end) {
        next_head += begin / per_query_head;
        next_tile += begin % per_query_head;
    }
    int32_t here_tile = next_tile;           // the tile of the step that is computed next
    const auto load = [&](uint16_t *q_tile, uint16_t *g_tile, float *stats)
                          __attribute__((always_inline)) {
        const int32_t h = next_head, query = next_tile * kQueryStep;
        q_loads.issue(static_cast<const uint16_t *>(a.q) + b * a.q_stride[0] + h * a.q_stride[1]
                          + query * a.q_stride[2],
                      live - query, a.q_stride[2], a.head_dim, q_tile);
        g_loads.issue(static_cast<const uint16_t *>(d.grad) + b * d.grad_stride[0]
                          + h * d.grad_stride[1] + query * d.grad_stride[2],
                      live - query, d.grad_stride[2], a.head_dim, g_tile);
        if (wave < 2) {
            const float *from = (wave == 0 ? a.lse : d.delta)
                                + (int64_t{b} * a.heads + h) * lse_pitch(a.queries) + query;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                make_rsrc(from, kQueryStep * 4),
                (__attribute__((address_space(3))) void *)(stats + wave * kQueryStep), 4, lane * 4,
                0, 0, 0);
        }
        if (++next_tile == low_tile + per_query_head) {
            next_tile = low_tile;
            ++next_head;
        }
    };

    const float factor = a.scale * kLog2e;
    const uint32_t reach =
        a.window == 0 || key < a.sinks ? kMaxTokens : static_cast<uint32_t>(a.window);
    f32x16 dk[kColumns], dv[kColumns];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) dk[c] = dv[c] = f32x16{};
    float up = kHalfFirst;   // of dS and dk in FP16

    // 32 of the step's queries, at `position`; `all`: each sees all the wave's keys.
    const auto rows = [&](int n, bool all, int32_t position, const uint16_t *q_tile,
                          const uint16_t *g_tile, const float *stats)
                          __attribute__((always_inline)) {
        f32x16 s{}, e;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 delta = *reinterpret_cast<const f32x4 *>(stats + kQueryStep + 32 * n + 8 * g
                                                                 + 4 * half);
#pragma unroll
            for (int i = 0; i < 4; ++i) e[4 * g + i] = -delta[i];
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            s = Element<kHalf>::multiply(read_rows<kPitch>(q_tile, n, i), k_operand[i], s);
            const u32x4 v_rows =
                kStaged ? read_rows<kPitch>(v_block, wave, i) : v_operand[kStaged ? 0 : i];
            e = Element<kHalf>::multiply(read_rows<kPitch>(g_tile, n, i), v_rows, e);
        }
        if constexpr (kStaged) {
            // delta's reads and 4 more, then 3 reads for every 2 products.
            __builtin_amdgcn_sched_group_barrier(kLdsReadGroup, 8, 0);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                __builtin_amdgcn_sched_group_barrier(kMatrixGroup, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kLdsReadGroup, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kMatrixGroup, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kLdsReadGroup, 2, 0);
            }
        }
        if (!all) {
            // Position - key: from 0 to below what the key's place allows; rows past
            // the sequence are few tiles' (uniform).
            const int32_t at = position + 4 * half;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int32_t c = 8 * (r / 4) + r % 4;
                s[r] = static_cast<uint32_t>(at - key + c) < reach ? s[r] : -INFINITY;
            }
            if (position + 31 >= length) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[r] = at < length - (8 * (r / 4) + r % 4) ? s[r] : -INFINITY;
            }
        }
        // In FP16 the weights of long rows lie below the normal numbers: they are
        // held 2^8 larger until the sums of dv are stored.
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 lse = *reinterpret_cast<const f32x4 *>(stats + 32 * n + 8 * g + 4 * half);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * g + i;
                s[r] = exp2_fast(__builtin_fmaf(s[r], factor, -lse[i]));
                e[r] *= kHalf ? s[r] * up : s[r];
                if (kHalf) s[r] *= kHalfWeights;
            }
        }
        if constexpr (kHalf) {
            lower_half(e, dk, [&](float factor) { up *= factor; });
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const u32x4 weights = as_operand<kHalf>(s, p), ds = as_operand<kHalf>(e, p);
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                dv[c] = Element<kHalf>::multiply(
                    read_columns<kPitch>(g_tile, 32 * n + 16 * p, c), weights, dv[c]);
                dk[c] = Element<kHalf>::multiply(
                    read_columns<kPitch>(q_tile, 32 * n + 16 * p, c), ds, dk[c]);
            }
        }
        if constexpr (kStaged) read_ahead<4 * kColumns, 2, 4>();
    };
    const auto step = [&](const uint16_t *q_tile, const uint16_t *g_tile, const float *stats)
                          __attribute__((always_inline)) {
        const int32_t position = here_tile * kQueryStep + shift;
        if (++here_tile == low_tile + per_query_head) here_tile = low_tile;
        const int32_t last_here = position + kQueryStep - 1, wave_last = wave_first + kWaveKeys - 1;
        const bool all =
            wave_last <= position && last_here < length
            && (a.window == 0 || last_here - wave_first < a.window || wave_last < a.sinks);
#pragma unroll 1
        for (int n = 0; n < 2; ++n) {
            const int32_t here = position + 32 * n;
            if (all
                || (here + 31 >= wave_first
                    && (a.window == 0 || here - wave_last < a.window || wave_first < a.sinks)))
                rows(n, all, here, q_tile, g_tile, stats);
        }
    };

    if (begin < end) load(q_even, g_even, stats_even);
    for (int32_t t = begin; t < end; t += 2) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 1 < end) load(q_odd, g_odd, stats_odd);
        step(q_even, g_even, stats_even);
        if (t + 1 >= end) break;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 2 < end) load(q_even, g_even, stats_even);
        step(q_odd, g_odd, stats_odd);
    }

    float *part_out =             // read where there are several parts
        splits == 1 ? nullptr
                    : parts
                          + (bkv * blocks.stored_parts() + blocks.first_part(block) + split)
                                * part_pitch(kKeyBlock, a.head_dim);
    if constexpr (kHalf) multiply_all(dk, 1.0f / up);
    if (not_finite(dk) || not_finite(dv)) {
        const int32_t channel = 2 * lane;
        for (int32_t j = wave_first; j < min(wave_first + kWaveKeys, a.keys); ++j) {
            float kx = 0.0f, ky = 0.0f, vx = 0.0f, vy = 0.0f;
            const bool there = j < length;
            const uint32_t k_pair = there ? lane_pair(k + j * a.k_stride[2], a.head_dim) : 0u;
            const uint32_t v_pair = there ? lane_pair(v + j * a.v_stride[2], a.head_dim) : 0u;
            for (int32_t t = begin; t < end; ++t) {
                const int32_t h = kv * group + t / per_query_head;
                const int32_t query = (low_tile + t % per_query_head) * kQueryStep;
                const uint16_t *q =
                    static_cast<const uint16_t *>(a.q) + b * a.q_stride[0] + h * a.q_stride[1];
                const uint16_t *g = static_cast<const uint16_t *>(d.grad) + b * d.grad_stride[0]
                                    + h * d.grad_stride[1];
                const int64_t stats = (int64_t{b} * a.heads + h) * lse_pitch(a.queries);
                for (int32_t i = query; i < min(query + kQueryStep, live); ++i) {
                    if (!sight_of(a, i + shift, length)(j)) continue;
                    const uint32_t q_pair = lane_pair(q + i * a.q_stride[2], a.head_dim);
                    const uint32_t g_pair = lane_pair(g + i * d.grad_stride[2], a.head_dim);
                    const float weight = exp2_fast(__builtin_fmaf(
                        row_product<kHalf>(q_pair, k_pair), factor, -a.lse[stats + i]));
                    const float ds =
                        weight * (row_product<kHalf>(g_pair, v_pair) - d.delta[stats + i]);
                    vx += weight * Element<kHalf>::low(g_pair);
                    vy += weight * Element<kHalf>::high(g_pair);
                    kx += ds * Element<kHalf>::low(q_pair);
                    ky += ds * Element<kHalf>::high(q_pair);
                }
            }
            if (channel >= a.head_dim) continue;
            if (splits > 1) {
                float *dst = part_out + int64_t{j - first} * a.head_dim + channel;
                *reinterpret_cast<f32x2 *>(dst) = f32x2{kx * a.scale, ky * a.scale};
                *reinterpret_cast<f32x2 *>(dst + kKeyBlock * a.head_dim) = f32x2{vx, vy};
                continue;
            }
            *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(d.dk) + b * d.dk_stride[0]
                                          + kv * d.dk_stride[1] + j * d.dk_stride[2] + channel) =
                Element<kHalf>::round_pair(kx * a.scale, ky * a.scale);
            *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(d.dv) + b * d.dv_stride[0]
                                          + kv * d.dv_stride[1] + j * d.dv_stride[2] + channel) =
                Element<kHalf>::round_pair(vx, vy);
        }
        return;
    }
    const float dv_scale = kHalf ? 1.0f / kHalfWeights : 1.0f;
    if (key >= a.keys) return;
    if (splits == 1) {
        store_row<kHalf, kColumns>(static_cast<uint16_t *>(d.dk) + b * d.dk_stride[0]
                                       + kv * d.dk_stride[1] + key * d.dk_stride[2],
                                   dk, a.scale, a.head_dim);
        store_row<kHalf, kColumns>(static_cast<uint16_t *>(d.dv) + b * d.dv_stride[0]
                                       + kv * d.dv_stride[1] + key * d.dv_stride[2],
                                   dv, dv_scale, a.head_dim);
        return;
    }
    float *dst = part_out + int64_t{key - first} * a.head_dim;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int32_t channel = 32 * c + 8 * g + 4 * half;
            if (channel >= a.head_dim) continue;
            f32x4 x, y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = dk[c][4 * g + i] * a.scale;
                y[i] = dv[c][4 * g + i] * dv_scale;
            }
            *reinterpret_cast<f32x4 *>(dst + channel) = x;
            *reinterpret_cast<f32x4 *>(dst + kKeyBlock * a.head_dim + channel) = y;
        }
}

// Adds the parts of the blocks from `first_block` on that have several, in
// their order.  Four channels of one key per thread.
template <bool kHalf>
__global__ __launch_bounds__(kAttentionThreads) void attention_sum_parts_kernel(
    lct_attention a, lct_attention_gradients d, KeyBlocks blocks, const float *__restrict__ parts,
    int32_t end_block) {
    const int32_t quads = a.head_dim / 4, per_block = key_block(a.head_dim);
    const int64_t item = int64_t{blockIdx.x} * kAttentionThreads + threadIdx.x;
    const int32_t channel = 4 * static_cast<int32_t>(item % quads);
    const int64_t keys = min(int64_t{a.keys}, int64_t{end_block} * per_block);
    const int32_t key = static_cast<int32_t>(item / quads % keys);
    const int64_t bkv = item / quads / keys;
    if (bkv >= int64_t{a.batch} * a.kv_heads) return;
    const int32_t block = key / per_block;
    const int32_t count = blocks.parts_of(block);
    if (count == 1) return;
    const int64_t step = part_pitch(per_block, a.head_dim);
    const float *src = parts + (bkv * blocks.stored_parts() + blocks.first_part(block)) * step
                       + int64_t{key % per_block} * a.head_dim + channel;
    f32x4 x{}, y{};
#pragma unroll 8
    for (int32_t s = 0; s < count; ++s) {
        x += *reinterpret_cast<const f32x4 *>(src + s * step);
        y += *reinterpret_cast<const f32x4 *>(src + s * step + per_block * a.head_dim);
    }
    const int64_t b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
    u32x2 dk, dv;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        dk[i] = Element<kHalf>::round_pair(x[2 * i], x[2 * i + 1]);
        dv[i] = Element<kHalf>::round_pair(y[2 * i], y[2 * i + 1]);
    }
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(d.dk) + b * d.dk_stride[0]
                               + kv * d.dk_stride[1] + key * d.dk_stride[2] + channel) = dk;
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(d.dv) + b * d.dv_stride[0]
                               + kv * d.dv_stride[1] + key * d.dv_stride[2] + channel) = dv;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool strides_ok(const int64_t (&stride)[3]) {
    for (const int64_t s : stride)
        if (s < 0 || (s & 7) != 0) return false;
    return stride[2] < (int64_t{1} << 24);
}


}  // namespace

int32_t check_attention(const lct_attention *a) {
    if (!a || !a->q || !a->k || !a->v || !a->out) return LCT_E_NULL;
    if (a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads != 0
        || a->queries <= 0 || a->keys <= 0 || a->queries > kMaxTokens || a->keys > kMaxTokens
        || a->head_dim <= 0 || a->head_dim > LCT_MAX_HEAD_DIM || (a->head_dim & 7) != 0
        || int64_t{a->batch} * a->heads > kMaxAttentionItems)
        return LCT_E_SIZE;
    if (a->window < 0 || a->window > kMaxTokens || a->sinks < 0 || a->sinks > kMaxTokens
        || !(a->scale > 0.0f) || !(a->scale < INFINITY) || !strides_ok(a->q_stride)
        || !strides_ok(a->k_stride) || !strides_ok(a->v_stride) || !strides_ok(a->out_stride)
        || !aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)
        || !aligned16(a->lse))
        return LCT_E_ARG;
    return LCT_OK;
}

int32_t join_parts(const lct_attention &a, int32_t splits, const float *parts,
                   hipStream_t stream) {
    const int64_t pitch = a.lse != nullptr ? lse_pitch(a.queries) : a.queries;
    const uint32_t grid = static_cast<uint32_t>(int64_t{a.batch} * a.heads * pitch);
    if (a.fp16)
        attention_join_kernel<true>
            <<<grid, kAttentionThreads, 0, stream>>>(a, pitch, splits, parts);
    else
        attention_join_kernel<false>
            <<<grid, kAttentionThreads, 0, stream>>>(a, pitch, splits, parts);
    return static_cast<int32_t>(hipGetLastError());
}

namespace {

template <bool kHalf>
int32_t forward(const lct_attention &a, int32_t splits, float *workspace, hipStream_t stream) {
    const int32_t tiles = (a.queries + kQueryTile - 1) / kQueryTile;
    const int64_t items = int64_t{tiles} * splits * a.batch * a.heads;
    if (items > kMaxAttentionItems) return LCT_E_SIZE;
    const uint32_t grid = static_cast<uint32_t>(xcd_grid(items));
    by_width(a.head_dim, [&](auto width) {
        constexpr int kDim = decltype(width)::value;
        if (splits > 1)
            attention_forward_kernel<kHalf, kDim, true>
                <<<grid, kAttentionThreads, 0, stream>>>(a, tiles, splits, workspace);
        else
            attention_forward_kernel<kHalf, kDim, false>
                <<<grid, kAttentionThreads, 0, stream>>>(a, tiles, splits, workspace);
    });
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || splits == 1) return static_cast<int32_t>(err);
    return join_parts(a, splits, workspace, stream);
}

// Workgroups of the launch that adds parts: four channels of a key per thread.
int64_t sum_groups(const lct_attention &a, const KeyBlocks &blocks) {
    const int64_t keys =
        std::min<int64_t>(a.keys, int64_t{blocks.end_of_parts()} * key_block(a.head_dim));
    const int64_t threads = keys * (a.head_dim / 4) * a.batch * a.kv_heads;
    return (threads + kAttentionThreads - 1) / kAttentionThreads;
}

template <bool kHalf>
int32_t backward(const lct_attention &a, const lct_attention_gradients &d, const KeyBlocks &blocks,
                 float *workspace, hipStream_t stream) {
    const int32_t tiles = (a.queries + kQueryTile - 1) / kQueryTile;
    const int64_t items = int64_t{tiles} * a.batch * a.heads;
    const int64_t heads = int64_t{a.batch} * a.kv_heads;
    const uint32_t parts = static_cast<uint32_t>(xcd_grid(blocks.other_parts() * heads)
                                                 + xcd_grid(blocks.sink_parts() * heads));
    by_width(a.head_dim, [&](auto width) {
        constexpr int kDim = decltype(width)::value;
        attention_dq_kernel<kHalf, kDim>
            <<<static_cast<uint32_t>(xcd_grid(items)), kAttentionThreads, 0, stream>>>(a, d, tiles);
        attention_dkdv_kernel<kHalf, kDim>
            <<<parts, 2 * key_block(kDim), 0, stream>>>(a, d, blocks, workspace);
    });
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return static_cast<int32_t>(err);
    if (blocks.stored_parts() == 0) return LCT_OK;
    attention_sum_parts_kernel<kHalf>
        <<<static_cast<uint32_t>(sum_groups(a, blocks)), kAttentionThreads, 0, stream>>>(
            a, d, blocks, workspace, blocks.end_of_parts());
    return static_cast<int32_t>(hipGetLastError());
}

}  // namespace
}  // namespace lct

using namespace lct;

extern "C" int32_t lct_attention_forward(const lct_attention *a, int32_t splits, float *workspace,
                                         int64_t workspace_floats, hipStream_t stream) {
    if (const int32_t code = check_attention(a); code != LCT_OK) return code;
    if (splits <= 0 || splits > LCT_MAX_ATTENTION_SPLITS) return LCT_E_ARG;
    if (splits > 1) {
        if (!workspace) return LCT_E_NULL;
        if (workspace_floats / (a->head_dim + 2) / splits / a->queries
            < int64_t{a->batch} * a->heads)
            return LCT_E_SIZE;
        if ((reinterpret_cast<uintptr_t>(workspace) & 7) != 0) return LCT_E_ARG;
        if (int64_t{a->batch} * a->heads * lse_pitch(a->queries) > kMaxAttentionItems)
            return LCT_E_SIZE;
    }
    return a->fp16 ? forward<true>(*a, splits, workspace, stream)
                   : forward<false>(*a, splits, workspace, stream);
}

extern "C" int32_t lct_attention_backward(const lct_attention *a, const lct_attention_gradients *d,
                                          int32_t splits, int32_t sink_splits, float *workspace,
                                          int64_t workspace_floats, hipStream_t stream) {
    if (const int32_t code = check_attention(a); code != LCT_OK) return code;
    if (!d || !a->lse || !d->grad || !d->dq || !d->dk || !d->dv || !d->delta) return LCT_E_NULL;
    if (splits <= 0 || splits > LCT_MAX_ATTENTION_SPLITS || sink_splits <= 0
        || sink_splits > LCT_MAX_ATTENTION_SPLITS || !strides_ok(d->grad_stride)
        || !strides_ok(d->dq_stride) || !strides_ok(d->dk_stride) || !strides_ok(d->dv_stride)
        || !aligned16(d->grad) || !aligned16(d->dq) || !aligned16(d->dk) || !aligned16(d->dv)
        || !aligned16(d->delta) || !aligned16(workspace))
        return LCT_E_ARG;
    KeyBlocks blocks;
    const int32_t per_block = key_block(a->head_dim);
    blocks.blocks = (a->keys + per_block - 1) / per_block;
    blocks.sink_blocks =
        a->window > 0 ? (std::min(a->sinks, a->keys) + per_block - 1) / per_block : 0;
    blocks.splits = splits;
    blocks.sink_splits = sink_splits;
    const int64_t heads = int64_t{a->batch} * a->kv_heads;
    if ((blocks.sink_parts() + blocks.other_parts()) * heads > kMaxAttentionItems
        || int64_t{(a->queries + kQueryTile - 1) / kQueryTile} * a->batch * a->heads
               > kMaxAttentionItems
        || (blocks.stored_parts() > 0 && sum_groups(*a, blocks) > kMaxAttentionItems))
        return LCT_E_SIZE;
    if (blocks.stored_parts() > 0) {
        if (!workspace) return LCT_E_NULL;
        if (workspace_floats < blocks.stored_parts() * heads * part_pitch(per_block, a->head_dim))
            return LCT_E_SIZE;
    }
    return a->fp16 ? backward<true>(*a, *d, blocks, workspace, stream)
                   : backward<false>(*a, *d, blocks, workspace, stream);
}
