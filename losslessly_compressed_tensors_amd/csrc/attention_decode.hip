// One query per sequence against its cache of keys and values, with a sliding
// window and sinks.
//
// A workgroup takes a key head (16 of its query heads at most, the columns of
// 16x16x32 matrix instructions) and a share of the visible keys; its 4 waves
// take tiles of 32 keys in turn, each by itself, with the next tile's loads in
// registers.  Keys go from memory straight into operands; values pass through
// the wave's own LDS rows for the transposed read.  As in attention_core.h a
// lane's scores are the next product's operand: lane l holds keys 4 (l >> 4) + i
// and 16 more of query l & 15, and the values are read in that order.
//
// Bound by the read of the keys and values that the query sees: 5.8 TB/s for 64
// sequences under a window of 4096 (32 heads of 128 over 8, 187 us), 6.6 TB/s for 4
// of up to 131072 keys (263 to 272 us, and 6 for the join of 42 parts), where a plain
// read reaches 6.9.  The loads are issued whether or not there is a next tile, by
// range-checked resources: with branches around them the wait for one tile also
// waited for the next (200 and 322 us).  One sequence of 257 keys: 5.1 us, a
// launch's latency and three tiles'.
#include <algorithm>
#include <type_traits>

#include "attention_core.h"

namespace lct {
namespace {

constexpr int kDecodeKeys = 32;      // keys per tile
constexpr int kQueries = 16;         // query heads per workgroup
constexpr float kLog2e = 1.4426950408889634f;

// Keys and values of more bytes than half the memory side's cache (256 MiB) are
// read past it: 263 us in place of 292 for 4 sequences of up to 131072 keys, 188
// for 192 at 64 of 4100 (1.7 and 1.1 GB); 6.3 for 6.0 at one of 257, which
// stays in it.
constexpr int kStreaming = 2;
constexpr int64_t kCacheBytes = int64_t{128} << 20;

template <bool kHalf>
__device__ __forceinline__ f32x4 multiply16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (kHalf)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Over the four lanes l & 15 + 16 i.
__device__ __forceinline__ float quarters_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return across_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return across_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

template <bool kHalf, int kDim, bool kSplit, int kCache>
__global__ __launch_bounds__(kAttentionThreads, 2) void attention_decode_kernel(
    lct_attention a, int32_t splits, float *__restrict__ parts) {
    constexpr int kPitch = kPitchOf<kDim>;
    constexpr int kSteps = kDim / 32, kColumns = kDim / 16;
    constexpr int kChunks = kPitch / 8;                        // 16-byte chunks of an LDS row
    constexpr int kValueLoads = kDecodeKeys * kChunks / kWave;
    constexpr int kMergePitch = kDim + 4;
    constexpr int kValueBytes = kAttentionWaves * kDecodeKeys * kPitch * 2;
    constexpr int kMergeBytes = kAttentionWaves * kQueries * kMergePitch * 4;
    __shared__ __attribute__((aligned(1024))) char
        shared[kValueBytes > kMergeBytes ? kValueBytes : kMergeBytes];

    const int lane = wave_lane(), column = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int32_t group = a.heads / a.kv_heads;
    const int32_t chunks = (group + kQueries - 1) / kQueries;
    const int64_t item = blockIdx.x;
    const int32_t split = static_cast<int32_t>(item % splits);
    const int64_t rest = item / splits;
    const int32_t chunk = static_cast<int32_t>(rest % chunks);
    const int32_t kv = static_cast<int32_t>(rest / chunks % a.kv_heads);
    const int32_t b = static_cast<int32_t>(rest / chunks / a.kv_heads);

    const int32_t length = sequence_length(a, b);
    const KeyTiles all(a, length - 1, length - 1, length, kDecodeKeys);
    const Sight sight = sight_of(a, length - 1, length);
    const int32_t per_split = (all.count + splits - 1) / splits;
    const int32_t begin = split * per_split, end = min(all.count, begin + per_split);

    const int32_t in_group = chunk * kQueries + column;
    const int32_t h = kv * group + in_group;
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + b * a.q_stride[0] + h * a.q_stride[1];
    const uint16_t *k = static_cast<const uint16_t *>(a.k) + b * a.k_stride[0] + kv * a.k_stride[1];
    const uint16_t *v = static_cast<const uint16_t *>(a.v) + b * a.v_stride[0] + kv * a.v_stride[1];
    u32x4 q_operand[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int32_t channel = 32 * s + 8 * quarter;
        q_operand[s] = u32x4{0u, 0u, 0u, 0u};
        if (in_group < group && channel < a.head_dim)
            q_operand[s] = *reinterpret_cast<const u32x4 *>(q + channel);
    }

    struct Tile {
        u32x4 k[2][kSteps], v[kValueLoads];
    };
    // This lane's places in a tile; past the head's width, one that the range
    // check rejects.  So are keys past the sequence: both load zeros.
    uint32_t k_place[2][kSteps], v_place[kValueLoads];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int32_t channel = 32 * s + 8 * quarter;
            k_place[n][s] = channel < a.head_dim ? static_cast<uint32_t>(
                                (16 * n + column) * a.k_stride[2] + channel) * 2u
                                                 : kOutOfRange;
        }
#pragma unroll
    for (int i = 0; i < kValueLoads; ++i) {
        const int slot = i * kWave + lane, channel = slot % kChunks * 8;
        v_place[i] = channel < a.head_dim ? static_cast<uint32_t>(
                         slot / kChunks * a.v_stride[2] + channel) * 2u
                                          : kOutOfRange;
    }
    const auto load = [&](int32_t t, Tile &tile) __attribute__((always_inline)) {
        const int32_t first = all.first_key(t, kDecodeKeys);
        const int32_t rows = min(length - first, kDecodeKeys) - 1;
        // Past the last tile nothing is in range.  The loads are issued all the
        // same, so that the wait for the tile before leaves them in flight.
        const auto records = [&](int64_t stride) {
            return t < end ? static_cast<uint32_t>(rows * stride + a.head_dim) * 2u : 0u;
        };
        const __amdgpu_buffer_rsrc_t k_rows =
            make_rsrc(k + first * a.k_stride[2], records(a.k_stride[2]));
        const __amdgpu_buffer_rsrc_t v_rows =
            make_rsrc(v + first * a.v_stride[2], records(a.v_stride[2]));
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                tile.k[n][s] = __builtin_bit_cast(
                    u32x4, __builtin_amdgcn_raw_buffer_load_b128(k_rows, k_place[n][s], 0,
                                                                 kCache));
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i)
            tile.v[i] = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(v_rows, v_place[i], 0, kCache));
    };

    const float factor = a.scale * kLog2e;
    uint16_t *values = reinterpret_cast<uint16_t *>(shared) + wave * kDecodeKeys * kPitch;
    f32x4 out[kColumns];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) out[c] = f32x4{};
    float most = -INFINITY, shifted = 0.0f, total = 0.0f;

    const auto step = [&](int32_t t, Tile &tile) __attribute__((always_inline)) {
        const int32_t first = all.first_key(t, kDecodeKeys);
        const bool seen_by_all = first + kDecodeKeys <= length
                                 && (first >= sight.low || first + kDecodeKeys <= sight.sinks);
        // What the query does not see may be anything: its values become zeros.
        if (!seen_by_all) {
#pragma unroll
            for (int i = 0; i < kValueLoads; ++i)
                if (!sight(first + (i * kWave + lane) / kChunks))
                    tile.v[i] = u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i) {
            const int slot = i * kWave + lane;
            const int row = slot / kChunks, at = (slot % kChunks) ^ swizzle(row);
            *reinterpret_cast<u32x4 *>(values + row * kPitch + at * 8) = tile.v[i];
        }
        f32x4 s[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n] = f32x4{};
#pragma unroll
            for (int d = 0; d < kSteps; ++d)
                s[n] = multiply16<kHalf>(tile.k[n][d], q_operand[d], s[n]);
        }
        if (!seen_by_all) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[n][i] = sight(first + 16 * n + 4 * quarter + i) ? s[n][i] : -INFINITY;
        }
        float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) top = fmaxf(fmaxf(top, s[0][i]), s[1][i]);
        top = quarters_max(top);
        if (__any(top * factor > most * factor + kRescale)) {
            const float next = fmaxf(most, top);
            const float scaled = next == -INFINITY ? 0.0f : next * factor;
            const float change = exp2_fast(most * factor - scaled);
            most = next;
            shifted = scaled - (kHalf ? kHalfLift : 0.0f);
            total *= change;
#pragma unroll
            for (int c = 0; c < kColumns; ++c) out[c] *= change;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][i] = exp2_fast(__builtin_fmaf(s[n][i], factor, -shifted));
                total += s[n][i];
            }
        u32x4 weights;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                weights[2 * n + i] = Element<kHalf>::round_pair(s[n][2 * i], s[n][2 * i + 1]);
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
            const int row = 4 * quarter + ((lane & 15) >> 2);
            const int at = (2 * c + ((lane >> 1) & 1)) ^ swizzle(row);
            const uint16_t *from = values + row * kPitch + at * 8 + (lane & 1) * 4;
            const u32x2 low = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (__attribute__((address_space(3))) i16x4 *)(from)));
            const u32x2 high = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (__attribute__((address_space(3))) i16x4 *)(from + 16 * kPitch)));
            out[c] = multiply16<kHalf>(u32x4{low[0], low[1], high[0], high[1]}, weights, out[c]);
        }
    };

    // The wave's own LDS rows: its operations on them run in order.
    Tile even, odd;
    int32_t t = begin + wave;
    load(t, even);
    for (; t < end; t += 2 * kAttentionWaves) {
        load(t + kAttentionWaves, odd);
        step(t, even);
        if (t + kAttentionWaves >= end) break;
        load(t + 2 * kAttentionWaves, even);
        step(t + kAttentionWaves, odd);
    }
    total = quarters_sum(total);

    // The waves' parts meet in LDS, in wave order.
    __syncthreads();
    float *merge = reinterpret_cast<float *>(shared);
    float *mine = merge + (wave * kQueries + column) * kMergePitch;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
        *reinterpret_cast<f32x4 *>(mine + 16 * c + 4 * quarter) = out[c];
    if (quarter == 0) *reinterpret_cast<f32x2 *>(mine + kDim) = f32x2{shifted, total};
    __syncthreads();
    const int32_t pairs = a.head_dim / 2;
    const int32_t rows = min(kQueries, group - chunk * kQueries);
    for (int32_t i = threadIdx.x; i < rows * pairs; i += kAttentionThreads) {
        const int32_t row = i / pairs, channel = 2 * (i % pairs);
        float largest = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttentionWaves; ++w) {
            const float *from = merge + (w * kQueries + row) * kMergePitch + kDim;
            if (from[1] != 0.0f) largest = fmaxf(largest, from[0]);
        }
        float sum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttentionWaves; ++w) {
            const float *from = merge + (w * kQueries + row) * kMergePitch;
            if (from[kDim + 1] == 0.0f) continue;
            const float weight = exp2_fast(from[kDim] - largest);
            sum += weight * from[kDim + 1];
            x += weight * from[channel];
            y += weight * from[channel + 1];
        }
        const int32_t head = kv * group + chunk * kQueries + row;
        if constexpr (kSplit) {
            float *part = parts
                          + ((int64_t{b} * a.heads + head) * splits + split) * (a.head_dim + 2);
            *reinterpret_cast<f32x2 *>(part + channel) = f32x2{x, y};
            if (channel == 0) *reinterpret_cast<f32x2 *>(part + a.head_dim) = f32x2{largest, sum};
        } else {
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint16_t *dst = static_cast<uint16_t *>(a.out) + b * a.out_stride[0]
                            + head * a.out_stride[1];
            *reinterpret_cast<uint32_t *>(dst + channel) =
                Element<kHalf>::round_pair(x * inverse, y * inverse);
        }
    }
}

template <bool kHalf>
int32_t decode(const lct_attention &a, int32_t splits, float *workspace, hipStream_t stream) {
    const int64_t chunks = (a.heads / a.kv_heads + kQueries - 1) / kQueries;
    const uint32_t grid = static_cast<uint32_t>(chunks * a.kv_heads * a.batch * splits);
    const auto launch = [&](auto width, auto split, auto cache) {
        attention_decode_kernel<kHalf, decltype(width)::value, decltype(split)::value,
                                decltype(cache)::value>
            <<<grid, kAttentionThreads, 0, stream>>>(a, splits, workspace);
    };
    const int64_t seen =
        a.window > 0 ? std::min<int64_t>(a.keys, int64_t{a.window} + a.sinks) : a.keys;
    const bool stream_once = 4 * seen * a.batch * a.kv_heads * a.head_dim > kCacheBytes;
    by_width(a.head_dim, [&](auto width) {
        if (splits > 1 && stream_once)
            launch(width, std::true_type{}, std::integral_constant<int, kStreaming>{});
        else if (splits > 1)
            launch(width, std::true_type{}, std::integral_constant<int, 0>{});
        else if (stream_once)
            launch(width, std::false_type{}, std::integral_constant<int, kStreaming>{});
        else
            launch(width, std::false_type{}, std::integral_constant<int, 0>{});
    });
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || splits == 1) return static_cast<int32_t>(err);
    return join_parts(a, splits, workspace, stream);
}

}  // namespace
}  // namespace lct

using namespace lct;

extern "C" int32_t lct_attention_decode(const lct_attention *a, int32_t splits, float *workspace,
                                        int64_t workspace_floats, hipStream_t stream) {
    if (const int32_t code = check_attention(a); code != LCT_OK) return code;
    if (a->queries != 1 || a->lse != nullptr || splits <= 0 || splits > LCT_MAX_ATTENTION_SPLITS)
        return LCT_E_ARG;
    if (int64_t{a->batch} * a->heads * splits > kMaxAttentionItems) return LCT_E_SIZE;
    if (splits > 1) {
        if (!workspace) return LCT_E_NULL;
        if (workspace_floats / (a->head_dim + 2) / splits < int64_t{a->batch} * a->heads)
            return LCT_E_SIZE;
        if ((reinterpret_cast<uintptr_t>(workspace) & 7) != 0) return LCT_E_ARG;
    }
    return a->fp16 ? decode<true>(*a, splits, workspace, stream)
                   : decode<false>(*a, splits, workspace, stream);
}
