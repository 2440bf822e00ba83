// Softmax cross entropy of a projection onto a vocabulary, and its gradients, in
// pieces of the vocabulary: the logits are never kept.
//
// Follows examples/nanogpt/train_gpt_lct.py:88-140, whose head keeps a chunk of
// tokens' logits.  With z = x W^T + bias and, under a soft cap s, l = z / sqrt(1 + (z /
// s)^2) (else l = z):
//     loss = log(sum_v exp(l_v)) - l_t = log(1 + sum_{v != t} exp(l_v - l_t)),
//     dz_v = g (exp(l_v) / sum - [v = t]) (1 + (z / s)^2)^(-3/2),
//     dx = dz W,  dW = dz^T x,  dbias = the columns' sums of dz.
// dz is rounded to 16 bits for its products, as far off as their results' own rounding: the
// gradients end up to 1.25 times as far from those in 64 bits as ones rounded once.  Multiplying
// what the rounding leaves too would double both products (1.26 of 2.6 ms of 8192 x 50304 x 768).
// Of up to 128 tokens, whose products wait for memory in any case, that is done: there a few
// large values carry the results.
// The second form of the loss keeps its precision where the target is likely:
// the target is left out of the sums, and its own gradient is exp(-loss) - 1.
//
// Tokens that do not count (target ignore_index) are not multiplied: `rows` lists the
// others, the products run over those, and what an ignored token's x holds reaches
// nothing.
#include <algorithm>

#include "product_core.h"

namespace lct {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// dz in FP16 is held 2^14 larger: |dz| <= 1, and a probability is lost below 2^-38.
constexpr float kHalfGradient = 16384.0f;
// Where |z / s| may be squared in FP32; the cap is reached far below.
constexpr float kCapped = 1e18f;

// The tiles, two workgroups per compute unit.  Of operands by rows a step of 32 of k asks L2
// for 64 bytes a row, and L2's requests bound the tile (counted: 0.83 of one per clock and
// channel): a step is 64.  By columns a line is 256 or 512 bytes anyhow, and three steps of 32
// leave the larger tile.  us of a step of 8192 x 50304 x 768 | 1013 x 50257 x 1024 | 16384 x
// 100352 x 2048 with these: 2760 | 409 | 21608; logits by 256 x 128, three steps of 32: 2937 |
// 439 | 23543; by 128 x 128, two of 64: 3065 | 439 | 22403.
constexpr int kLogitRows = LCT_CROSS_ENTROPY_BIAS_TOKENS;
template <bool kHalf>
using LogitProduct = Product<kHalf, Lie::kRows, Lie::kRows, kLogitRows, 128, 2, 2, 64, 2>;
// Deep products: us of a call with this | the tile above, of 8192 tokens 50176 x 768 612 | 582,
// x 1024 758 | 748, x 1536 1066 | 1104, x 2048 1377 | 1439, 32000 x 4096 1703 | 1809; of 2048
// tokens 50176 x 1536 306 | 298, 32000 x 4096 449 | 491; of 512 128 | 172; of 256 110 | 108, and
// 131072 x 2048 151 | 176.  One workgroup per compute unit, whose end no other's products hide.
// The rule goes by channels alone, of more than 128 tokens: 1536 channels lose 3 % of 8192 tokens
// by it and gain 3 % of 2048, and 4096 channels lose 2 % of 256.
constexpr int32_t kDeep = 2048;
template <bool kHalf>
using DeepProduct = Product<kHalf, Lie::kRows, Lie::kRows, 256, 256, 4, 2, 64, 2>;
// A few tokens, the vocabulary's rows streamed four steps ahead.  us of a call with this | the
// wide tile: 50304 x 768, 1 token 26.2 | 26.3, 16 25.0 | 26.7, 32 24.9 | 27.2; 32000 x 4096, 1
// token 64.8 | 80.3, 32 65.8 | 80.5.  The latter is 4.1 TB/s; of the former 14.6 us are the
// kernel's (5.3 TB/s).
constexpr int kFewTokens = 32;
template <bool kHalf>
using FewProduct = Product<kHalf, Lie::kRows, Lie::kRows, 128, kFewTokens, 4, 1, 64, 4>;
// Of up to 128 tokens, with dz in two numbers (kExact), and of more: us of a step of 8192 x 50304
// x 768 | 1013 x 50257 x 1024 | 16384 x 100352 x 2048 with 256 x 256 2737 | 402 | 21059, with the
// smaller tile 2763 | 405 | 21708 (both with parts chosen for the latter).
template <bool kHalf, Lie kLieB, bool kExact>
using GradientProduct =
    std::conditional_t<kExact, Product<kHalf, Lie::kColumns, kLieB, 256, 128, 2, 2, 32, 3>,
                       Product<kHalf, Lie::kColumns, kLieB, 256, 256, 2, 4, 32, 4>>;
template <bool kHalf, bool kExact>
using HiddenProduct = GradientProduct<kHalf, Lie::kColumns, kExact>;
template <bool kHalf, bool kExact>
using WeightProduct = GradientProduct<kHalf, Lie::kRows, kExact>;

// The counted tokens, as prepare_kernel found them.
struct Counted {
    const int32_t *count;      // how many
    const int32_t *rows;       // int32[count]: which tokens
    const int32_t *targets;    // their targets, -1 for none of the vocabulary
    const float *lse, *losses, *factor;   // backward: of those
    const float *scale;        // backward: what gradients are multiplied by at the end
    const void *gathered;      // their x, where not all count
};

__device__ __forceinline__ const void *hidden_of(const lct_cross_entropy &c, const Counted &t,
                                                 int32_t count, int64_t *stride) {
    const bool all = count == c.tokens;
    *stride = all ? c.x_stride : c.dim;
    return all ? c.x : t.gathered;
}

__device__ __forceinline__ int64_t target_of(const lct_cross_entropy &c, int64_t n) {
    return c.targets_64 ? static_cast<const int64_t *>(c.targets)[n]
                        : static_cast<const int32_t *>(c.targets)[n];
}

// The counted tokens' x next to each other, 16 bytes a thread, where not all count.
__device__ __forceinline__ void gather(const lct_cross_entropy &c, int32_t count,
                                       const int32_t *rows, void *out, int64_t first,
                                       int64_t step) {
    if (count == c.tokens) return;
    const int32_t chunks = c.dim / 8;
    for (int64_t at = first; at < int64_t{count} * chunks; at += step) {
        const int32_t i = static_cast<int32_t>(at / chunks);
        const int32_t chunk = static_cast<int32_t>(at % chunks);
        static_cast<u32x4 *>(out)[at] = *reinterpret_cast<const u32x4 *>(
            static_cast<const uint16_t *>(c.x) + rows[i] * c.x_stride + chunk * 8);
    }
}

__global__ __launch_bounds__(256) void gather_kernel(lct_cross_entropy c, Counted t, void *out) {
    gather(c, *t.count, t.rows, out, int64_t{blockIdx.x} * 256 + threadIdx.x,
           int64_t{gridDim.x} * 256);
}

// 16-byte pieces of x up to which the one workgroup of prepare_kernel gathers itself.  us of a
// call of 300 tokens with that | a launch of its own: 64 channels (2400 pieces) 23.0 | 26.1, 256
// (9600) 23.2 | 26.0, 768 (28800) 33.6 | 26.5; of 1000 tokens of 256 (32000) 31.3 | 26.2.
constexpr int64_t kGatherHere = 8192;

// ---- the counted tokens, in order

constexpr int kPrepareThreads = 1024, kPrepareEach = 16;
constexpr int kGroups = kPrepareThreads / kWave * kPrepareEach;

__device__ __forceinline__ float block_max(float v, float *scratch) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, kWave));
    if (wave_lane() == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < kPrepareThreads / kWave; ++w) v = fmaxf(v, scratch[w]);
    __syncthreads();
    return v;
}

// One workgroup.  Forward (grad NULL): which tokens count, and lse and losses of the
// others.  Backward: also the factor of each token's dz and what all gradients are
// multiplied by at the end: a token's incoming gradient over the power of two above the
// largest, and that power, so that dz lies within [-1, 1] whatever the incoming gradients
// are.  (All infinite or NaN ones go to their tokens' factors.)
struct PrepareGradients {
    const float *grad;       // NULL: forward
    int32_t per_token, mean;
};

__global__ __launch_bounds__(kPrepareThreads) void prepare_kernel(lct_cross_entropy c, Counted t,
                                                                  PrepareGradients g, float *lse,
                                                                  float *losses, void *gathered) {
    auto *const rows = const_cast<int32_t *>(t.rows);
    auto *const targets = const_cast<int32_t *>(t.targets);
    const float *const grad = g.grad;
    __shared__ float scratch[kPrepareThreads / kWave];
    __shared__ int32_t counts[kGroups], ends[kGroups / kWave];
    float largest = 0.0f;
    if (grad != nullptr && g.per_token)
        for (int32_t n = threadIdx.x; n < c.tokens; n += kPrepareThreads)
            if (target_of(c, n) != c.ignore_index) {
                const float of = fabsf(grad[n]);
                if (of < INFINITY) largest = fmaxf(largest, of);
            }
    float power = 1.0f;
    if (grad != nullptr && g.per_token) {
        largest = block_max(largest, scratch);
        // 2^e >= largest, within FP32's normal numbers.
        if (largest > 0.0f) power = ldexpf(1.0f, min(max(ilogbf(largest) + 1, -126), 127));
    }
    const float hold = c.fp16 ? kHalfGradient : 1.0f;
    // Sixteen tokens a thread, their loads in flight together, between the workgroup's
    // meetings.
    int32_t done = 0;
    for (int64_t first = 0; first < c.tokens; first += kPrepareThreads * kPrepareEach) {
        int64_t target[kPrepareEach];
#pragma unroll
        for (int k = 0; k < kPrepareEach; ++k) {
            const int64_t n = first + k * kPrepareThreads + threadIdx.x;
            target[k] = n < c.tokens ? target_of(c, n) : c.ignore_index;
        }
#pragma unroll
        for (int k = 0; k < kPrepareEach; ++k) {
            const uint64_t counted = __ballot(target[k] != c.ignore_index);
            if (wave_lane() == 0)
                counts[k * (kPrepareThreads / kWave) + threadIdx.x / kWave] = __popcll(counted);
        }
        __syncthreads();
        // Where each wave's group begins, by the first four waves.
        int32_t own = 0, inclusive = 0;
        if (threadIdx.x < kGroups) {
            own = counts[threadIdx.x];
            inclusive = wave_inclusive_scan(own);
            if (wave_lane() == kWave - 1) ends[threadIdx.x / kWave] = inclusive;
        }
        __syncthreads();
        int32_t total = 0;
#pragma unroll
        for (int w = 0; w < kGroups / kWave; ++w) {
            if (threadIdx.x < kGroups && w < static_cast<int>(threadIdx.x / kWave))
                inclusive += ends[w];
            total += ends[w];
        }
        if (threadIdx.x < kGroups) counts[threadIdx.x] = done + inclusive - own;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPrepareEach; ++k) {
            const int64_t n = first + k * kPrepareThreads + threadIdx.x;
            if (n >= c.tokens) continue;
            const bool counted = target[k] != c.ignore_index;
            const uint64_t before = __ballot(counted) & ((uint64_t{1} << wave_lane()) - 1);
            if (counted) {
                const int32_t i = counts[k * (kPrepareThreads / kWave) + threadIdx.x / kWave]
                                  + __popcll(before);
                const bool inside = target[k] >= 0 && target[k] < c.vocab;
                rows[i] = static_cast<int32_t>(n);
                targets[i] = inside ? static_cast<int32_t>(target[k]) : -1;
                if (grad != nullptr) {
                    const_cast<float *>(t.lse)[i] = lse[n];
                    const_cast<float *>(t.losses)[i] = losses[n];
                    const float factor = g.per_token ? grad[n] / power : 1.0f;
                    const_cast<float *>(t.factor)[i] = inside ? factor * hold : NAN;
                }
            } else if (grad == nullptr) {
                lse[n] = 0.0f;
                losses[n] = 0.0f;
            }
        }
        done += total;
        __syncthreads();
    }
    if (gathered != nullptr)      // (behind the last barrier above: the rows are written)
        gather(c, done, rows, gathered, threadIdx.x, kPrepareThreads);
    if (threadIdx.x == 0) {
        *const_cast<int32_t *>(t.count) = done;
        if (grad != nullptr) {
            const float tokens = g.mean ? fmaxf(1.0f, done) : 1.0f;
            *const_cast<float *>(t.scale) = (g.per_token ? power : *grad / tokens) / hold;
        }
    }
}

// ---- forward

// The sums under way of one token over part of the vocabulary, the target left out:
// the largest logit and the sum of exponentials from there, in powers of two.
struct Part {
    float most, total;
};

__device__ __forceinline__ Part joined(Part a, Part b) {
    const float most = fmaxf(a.most, b.most);
    const float base = most == -INFINITY ? 0.0f : most;
    return {most, a.total * exp2_fast(a.most - base) + b.total * exp2_fast(b.most - base)};
}

// l = z root(z), root(z) = (1 + (z / s)^2)^(-1/2).
struct Cap {
    float cap, inverse;
    __device__ __forceinline__ float root(float z) const {
        const float u = z * inverse;
        return __builtin_amdgcn_rsqf(__builtin_fmaf(u, u, 1.0f));
    }
    // z, or the largest of its sign that root() takes; NaN stays.
    __device__ __forceinline__ float within(float z) const {
        const float most = kCapped * cap;
        return fabsf(z) > most ? copysignf(most, z) : z;
    }
};

// Whether some |z| of the wave's is larger than root() takes: then all go through within().
template <class P>
__device__ __forceinline__ bool far_of(const P &p, const Cap &cap) {
    float largest = 0.0f;
#pragma unroll
    for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
        for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) largest = fmaxf(largest, fabsf(p.sum[m][n][r]));
    return __any(largest > kCapped * cap.cap);
}

// P::kM of the vocabulary (rows, in a lane's registers) by P::kN tokens (columns, a lane
// each): a token's maximum and sum need one exchange between two lanes.
//
// Bound by the matrix instructions: 2 * tokens * vocab * dim operations, and the exponentials
// behind them.  14746 x 100352 x 2048: 5.0 to 5.2 ms, 1210 to 1170 TFLOP/s (matrix instructions
// busy 0.66 of the time, at the power limit's 1.74 GHz); 4095 x 32000 x 4096: 0.83 to 0.97 ms, 1290
// to 1100 (0.69, 1.6 GHz); 8192 x 50304 x 768, capped: 623 to 730 us, 1010 to 870 (12 steps a tile;
// 0.54, 1.78 GHz).
template <class P, bool kCap, bool kBias>
__global__ __launch_bounds__(P::kThreads, P::kThreads == 256 ? 2 : 1) void logits_kernel(
    lct_cross_entropy c, Counted t, int32_t vocab_tiles, int32_t token_tiles,
    Part *__restrict__ parts) {
    LCT_PRODUCT_STAGES(P);
    const int32_t count = t.count == nullptr ? c.tokens : *t.count;
    const int64_t item = xcd_item(int64_t{vocab_tiles} * token_tiles, blockIdx.x);
    if (item >= int64_t{vocab_tiles} * token_tiles) return;
    // Eight vocabulary tiles against all tokens, then the next eight.
    const int32_t group = static_cast<int32_t>(item / (8 * int64_t{token_tiles}));
    const int32_t in_group = static_cast<int32_t>(item % (8 * int64_t{token_tiles}));
    const int32_t width = min(8, vocab_tiles - 8 * group);
    const int32_t vocab_tile = 8 * group + in_group % width, token_tile = in_group / width;
    if (int64_t{token_tile} * P::kN >= count) return;

    int64_t x_stride = c.x_stride;
    const void *x = c.x;
    if (t.count != nullptr) x = hidden_of(c, t, count, &x_stride);
    typename P::A a;
    typename P::B b;
    a.prepare(c.weight, c.weight_stride, int64_t{vocab_tile} * P::kM, c.vocab);
    b.prepare(x, x_stride, int64_t{token_tile} * P::kN, count);
    const int half = wave_lane() >> 5;
    const int32_t first = vocab_tile * P::kM + P::first_row();
    P p;
    if constexpr (kBias) {
        const __amdgpu_buffer_rsrc_t bias = make_rsrc(c.bias, static_cast<uint32_t>(c.vocab) * 4u);
        p.begin([&](int m, int) {
            f32x16 v;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                v[r] = __builtin_bit_cast(
                    float, __builtin_amdgcn_raw_buffer_load_b32(
                               bias, (first + 32 * m + 8 * (r / 4) + 4 * half + r % 4) * 4, 0, 0));
            return v;
        });
    } else {
        p.begin();
    }
    p.run(a, b, c.dim, stage0, stage1, stage2, stage3);
    if constexpr (kCap) {
        const Cap cap{c.softcap, 1.0f / c.softcap};
        if (far_of(p, cap)) {
#pragma unroll
            for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
                for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) p.sum[m][n][r] = cap.within(p.sum[m][n][r]);
        }
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) p.sum[m][n][r] *= cap.root(p.sum[m][n][r]);
    }
    if (first + P::kWaveM > c.vocab) {
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (first + 32 * m + 8 * (r / 4) + 4 * half + r % 4 >= c.vocab)
                        p.sum[m][n][r] = -INFINITY;
    }
    const int32_t entries = P::kWavesM * vocab_tiles;
#pragma unroll
    for (int n = 0; n < P::kColumnTiles; ++n) {
        const int32_t token = token_tile * P::kN + p.first_column() + 32 * n + (wave_lane() & 31);
        int32_t target = -1;
        if (token < count) {
            if (t.count != nullptr) target = t.targets[token];
            else target = static_cast<int32_t>(std::min<int64_t>(
                     std::max<int64_t>(target_of(c, token), -1), c.vocab));
        }
        target -= first;
        if (__any(target >= 0 && target < P::kWaveM)) {
#pragma unroll
            for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * m + 8 * (r / 4) + 4 * half + r % 4 == target)
                        p.sum[m][n][r] = -INFINITY;
        }
        float most = p.sum[0][n][0];
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) most = fmaxf(most, p.sum[m][n][r]);
        most = across_max(most) * kLog2e;
        const float base = most == -INFINITY ? 0.0f : most;
        float total = 0.0f;
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                total += exp2_fast(__builtin_fmaf(p.sum[m][n][r], kLog2e, -base));
        total = across_sum(total);
        if (half == 0 && token < count)
            parts[int64_t{token} * entries + P::kWavesM * vocab_tile + p.wave() % P::kWavesM] =
                Part{most, total};
    }
}

// kWaves join one token's parts and compute its target's logit: the loss and lse (in powers
// of two).  Reads the parts once, in flight together: 8192 x 526 in 16.3 us, 2.1 TB/s.
template <bool kHalf, int kWaves>
__global__ __launch_bounds__(256) void join_kernel(lct_cross_entropy c, Counted t, int32_t entries,
                                                   const Part *__restrict__ parts,
                                                   float *__restrict__ lse,
                                                   float *__restrict__ losses) {
    using E = Element<kHalf>;
    constexpr int kStep = kWaves * kWave, kAtOnce = 4;
    __shared__ Part others[4];
    __shared__ float products[4];
    const int32_t count = t.count == nullptr ? c.tokens : *t.count;
    const int32_t i = blockIdx.x * (4 / kWaves) + threadIdx.x / kStep;
    if (i >= count) return;
    const int lane = wave_lane(), place = threadIdx.x % kStep;
    const int32_t n = t.count == nullptr ? i : t.rows[i];
    const int64_t target = target_of(c, n);
    if (target == c.ignore_index) {
        if (place == 0) lse[n] = losses[n] = 0.0f;
        return;
    }
    const bool inside = target >= 0 && target < c.vocab;
    Part part{-INFINITY, 0.0f};
    for (int32_t first = place; first < entries; first += kAtOnce * kStep) {
        Part of[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int32_t e = first + k * kStep;
            of[k] = e < entries ? parts[int64_t{i} * entries + e] : Part{-INFINITY, 0.0f};
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) part = joined(part, of[k]);
    }
    float logit = 0.0f;
    if (inside) {
        const uint16_t *x = static_cast<const uint16_t *>(c.x) + n * c.x_stride;
        const uint16_t *w = static_cast<const uint16_t *>(c.weight) + target * c.weight_stride;
        for (int32_t d = 8 * place; d < c.dim; d += 8 * kStep) {
            const u32x4 p = *reinterpret_cast<const u32x4 *>(x + d);
            const u32x4 q = *reinterpret_cast<const u32x4 *>(w + d);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                logit = __builtin_fmaf(E::low(p[k]), E::low(q[k]), logit);
                logit = __builtin_fmaf(E::high(p[k]), E::high(q[k]), logit);
            }
        }
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
        logit += __shfl_xor(logit, d, kWave);
        part = joined(part,
                      Part{__shfl_xor(part.most, d, kWave), __shfl_xor(part.total, d, kWave)});
    }
    if constexpr (kWaves > 1) {
        if (lane == 0) {
            others[threadIdx.x / kWave] = part;
            products[threadIdx.x / kWave] = logit;
        }
        __syncthreads();
        if (threadIdx.x >= kWave) return;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            part = joined(part, others[w]);
            logit += products[w];
        }
    }
    if (lane != 0) return;
    if (!inside) {
        lse[n] = losses[n] = NAN;
        return;
    }
    if (c.bias != nullptr) logit += c.bias[target];
    if (c.softcap > 0.0f) {
        const Cap cap{c.softcap, 1.0f / c.softcap};
        logit = cap.within(logit);
        const float u = logit * cap.inverse;
        logit = logit / sqrtf(__builtin_fmaf(u, u, 1.0f));
    }
    // The others' weight over the target's, or that one's inverse.
    const float own = logit * kLog2e;
    const float above = part.most - own + log2f(part.total);
    const float rest = log1pf(above > 0.0f ? exp2f(-above) : part.total * exp2f(part.most - own));
    float loss = above > 0.0f ? __builtin_fmaf(above, kLn2, rest) : rest;
    float sum = above > 0.0f ? part.most + log2f(part.total) + rest * kLog2e : own + rest * kLog2e;
    if (part.total == 0.0f || logit == INFINITY) {    // no others, or nothing but the target
        loss = logit - logit;
        sum = own + loss;
    }
    losses[n] = loss;
    lse[n] = sum;
}

// The losses' sum or mean; one workgroup, in a fixed order.
__global__ __launch_bounds__(kPrepareThreads) void total_kernel(lct_cross_entropy c,
                                                                const float *__restrict__ losses,
                                                                int32_t mean, float *out) {
    __shared__ double sums[kPrepareThreads / kWave];
    __shared__ int32_t counts[kPrepareThreads / kWave];
    double sum = 0.0;
    int32_t count = 0;
    for (int32_t n = threadIdx.x; n < c.tokens; n += kPrepareThreads) {
        sum += losses[n];
        count += target_of(c, n) != c.ignore_index;
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
        sum += __shfl_xor(sum, d, kWave);
        count += __shfl_xor(count, d, kWave);
    }
    if (wave_lane() == 0) {
        sums[threadIdx.x / kWave] = sum;
        counts[threadIdx.x / kWave] = count;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kPrepareThreads / kWave; ++w) {
        sum += sums[w];
        count += counts[w];
    }
    *out = static_cast<float>(mean ? sum / max(1, count) : sum);
}

// ---- backward

// dz of P::kM tokens (rows) by P::kN of a piece of the vocabulary (columns, a lane each), the
// logits computed again: written by columns, [vocabulary][token], which both products
// that follow read, and its sums over these tokens.
//
// As the logits' kernel, and 2 bytes written a logit: a quarter of 8192 x 50304 x 768, capped,
// 194 to 220 us, 820 to 720 TFLOP/s (matrix instructions busy 0.39 of the time, at 2.0 GHz; the
// epilogue's exponential, root and stores take as long as the 12 steps); a thirteenth of 14746
// x 100352 x 2048 462 to 475 us, 1010 to 980.  The parts a workgroup works in, of both on a compute unit,
// overlap: starting half of them late, or stores past the caches, changed nothing.
template <class P, bool kHalf, bool kCap, bool kBias>
__global__ __launch_bounds__(P::kThreads, 2) void gradient_kernel(
    lct_cross_entropy c, Counted t, int32_t first_vocab, int32_t piece, int32_t vocab_tiles,
    int32_t token_tiles, uint16_t *dz, uint16_t *dz_rest, int64_t dz_stride, float *bias_parts) {
    LCT_PRODUCT_STAGES(P);
    const int32_t count = *t.count;
    const int64_t item = xcd_item(int64_t{vocab_tiles} * token_tiles, blockIdx.x);
    if (item >= int64_t{vocab_tiles} * token_tiles) return;
    const int32_t group = static_cast<int32_t>(item / (8 * int64_t{vocab_tiles}));
    const int32_t in_group = static_cast<int32_t>(item % (8 * int64_t{vocab_tiles}));
    const int32_t width = min(8, token_tiles - 8 * group);
    const int32_t token_tile = 8 * group + in_group % width, vocab_tile = in_group / width;
    if (int64_t{token_tile} * P::kM >= count) return;

    int64_t x_stride;
    const void *x = hidden_of(c, t, count, &x_stride);
    const int32_t last_vocab = first_vocab + piece;
    typename P::A a;
    typename P::B b;
    a.prepare(x, x_stride, int64_t{token_tile} * P::kM, count);
    b.prepare(c.weight, c.weight_stride, first_vocab + int64_t{vocab_tile} * P::kN, last_vocab);
    // Of each token, with its factor f: lse - log2 |f|, so that the exponential from there is
    // |f| times the probability, f's sign, the target and dz there.  Tokens past the last:
    // zeros.
    static_assert(P::kM <= P::kThreads);
    float4 own{INFINITY, 1.0f, __int_as_float(-1), 0.0f};
    {
        const int32_t i = token_tile * P::kM + threadIdx.x;
        if (threadIdx.x < P::kM && i < count) {
            const float f = t.factor[i];
            own = float4{t.lse[i] - log2f(fabsf(f)), copysignf(1.0f, f),
                         __int_as_float(t.targets[i]), t.losses[i]};
            own.w = f * expm1f(-own.w);
        }
    }
    const int lane = wave_lane(), half = lane >> 5;
    const int32_t first = first_vocab + vocab_tile * P::kN + P::first_column();
    P p;
    if constexpr (kBias) {
        float bias[P::kColumnTiles];
#pragma unroll
        for (int n = 0; n < P::kColumnTiles; ++n) {
            const int32_t column = first + 32 * n + (lane & 31);
            bias[n] = column < last_vocab ? c.bias[column] : 0.0f;
        }
        p.begin([&](int, int n) { return f32x16{} + bias[n]; });
    } else {
        p.begin();
    }
    p.run(a, b, c.dim, stage0, stage1, stage2, stage3);

    auto *row_values = reinterpret_cast<float4 *>(stage0);
    if (threadIdx.x < P::kM) row_values[threadIdx.x] = own;
    __syncthreads();
    const Cap cap{c.softcap, 1.0f / c.softcap};
    if constexpr (kCap) {
        if (far_of(p, cap)) {
#pragma unroll
            for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
                for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) p.sum[m][n][r] = cap.within(p.sum[m][n][r]);
        }
    }
    float column_sum[P::kColumnTiles] = {};
#pragma unroll
    for (int m = 0; m < P::kRowTiles; ++m) {
        const float4 *values = row_values + p.first_row() + 32 * m;
        const float4 mine = values[lane & 31];
        const int32_t target = __float_as_int(mine.z) - first;
        // Rare: a target, a negative factor, tokens past the last.
        const bool some = __any((target >= 0 && target < P::kWaveN) || mine.y < 0.0f
                                || token_tile * P::kM + p.first_row() + 32 * m + 31 >= count);
        const auto each = [&](auto rare) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 8 * (r / 4) + 4 * half + r % 4;
                const float4 v = values[row];
                const int32_t at = __float_as_int(v.z) - first - (lane & 31);
                const bool none = token_tile * P::kM + p.first_row() + 32 * m + row >= count;
#pragma unroll
                for (int n = 0; n < P::kColumnTiles; ++n) {
                    float z = p.sum[m][n][r], slope = 1.0f;
                    if constexpr (kCap) {
                        const float root = cap.root(z);
                        z *= root;
                        slope = root * root * root;
                    }
                    float d = exp2_fast(__builtin_fmaf(z, kLog2e, -v.x));
                    if constexpr (decltype(rare)::value) {
                        d = at == 32 * n ? v.w : d * v.y;
                        d = none ? 0.0f : d;
                    }
                    p.sum[m][n][r] = kCap ? d * slope : d;
                }
            }
        };
        if (some) each(std::true_type{});
        else each(std::false_type{});
#pragma unroll
        for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) column_sum[n] += p.sum[m][n][r];
    }
    __syncthreads();     // the LDS of row_values is written again
    if (first + P::kWaveN > last_vocab) {
#pragma unroll
        for (int n = 0; n < P::kColumnTiles; ++n)
            if (first + 32 * n + (lane & 31) >= last_vocab) {
#pragma unroll
                for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
                    for (int r = 0; r < 16; ++r) p.sum[m][n][r] = 0.0f;
            }
    }
    if (bias_parts != nullptr) {
#pragma unroll
        for (int n = 0; n < P::kColumnTiles; ++n) {
            const float sum = across_sum(column_sum[n]);
            const int32_t column = first + 32 * n + (lane & 31);
            if (half == 0 && column < last_vocab)
                bias_parts[(int64_t{token_tile} * P::kWavesM + p.wave() % P::kWavesM) * c.vocab
                           + column] = sum;
        }
    }
    if (dz == nullptr) return;
    const int32_t column = vocab_tile * P::kN + p.first_column();
    const int32_t row = token_tile * P::kM + p.first_row();
    using E = Element<kHalf>;
    uint16_t *const mine = turn_values<P>(stage0, stage1, stage2, stage3);
    const int64_t at = column * dz_stride + row;
    const int32_t rows = static_cast<int32_t>(dz_stride) - row;
    store_columns<P>(dz + at, dz_stride, piece - column, rows, mine, [&](int m, int n, int r) {
        return E::round_pair(p.sum[m][n][r], p.sum[m][n][r + 1]);
    });
    if (dz_rest == nullptr) return;
    store_columns<P>(dz_rest + at, dz_stride, piece - column, rows, mine, [&](int m, int n, int r) {
        const float a = p.sum[m][n][r], b = p.sum[m][n][r + 1];
        const uint32_t pair = E::round_pair(a, b);
        return E::round_pair(a - E::low(pair), b - E::high(pair));
    });
}

// What both products of a piece with dz need.
struct PieceProducts {
    int32_t first_vocab, piece, splits, dim_tiles, token_tiles, vocab_tiles;
    const uint16_t *dz, *dz_rest;     // dz_rest: what dz's rounding leaves, or NULL
    int64_t dz_stride;
    float *hidden_parts;
    uint16_t *grad_weight;
};

// dx of a piece of the vocabulary, or of one of its parts: channels (rows) by tokens
// (columns), added to the earlier pieces' in FP32.
template <bool kHalf, bool kExact>
__device__ __forceinline__ void hidden_gradient(const lct_cross_entropy &c, int32_t count,
                                                const PieceProducts &q, int64_t item,
                                                uint16_t *stage0, uint16_t *stage1,
                                                uint16_t *stage2, uint16_t *stage3) {
    using P = HiddenProduct<kHalf, kExact>;
    const int32_t dim_tile = static_cast<int32_t>(item % q.dim_tiles);
    const int32_t token_tile = static_cast<int32_t>(item / q.dim_tiles % q.token_tiles);
    const int32_t split = static_cast<int32_t>(item / q.dim_tiles / q.token_tiles);
    if (int64_t{token_tile} * P::kN >= count) return;
    const int32_t per = ((q.piece + q.splits - 1) / q.splits + 31) / 32 * 32;
    const int32_t begin = min(q.piece, split * per), end = min(q.piece, begin + per);
    typename P::A a;
    typename P::B b;
    a.prepare(static_cast<const uint16_t *>(c.weight) + (q.first_vocab + begin) * c.weight_stride,
              c.weight_stride, int64_t{dim_tile} * P::kM, c.dim);
    const int64_t tokens = (int64_t{count} + 7) / 8 * 8;
    b.prepare(q.dz + begin * q.dz_stride, q.dz_stride, int64_t{token_tile} * P::kN, tokens);
    P p;
    p.begin();
    p.run(a, b, end - begin, stage0, stage1, stage2, stage3);
    if constexpr (kExact) {
        b.prepare(q.dz_rest + begin * q.dz_stride, q.dz_stride, int64_t{token_tile} * P::kN,
                  tokens);
        p.run(a, b, end - begin, stage0, stage1, stage2, stage3);
    }

    const int lane = wave_lane();
#pragma unroll
    for (int n = 0; n < P::kColumnTiles; ++n) {
        const int32_t token = token_tile * P::kN + p.first_column() + 32 * n + (lane & 31);
        if (token >= count) continue;
        float *out = q.hidden_parts + (int64_t{split} * c.tokens + token) * c.dim;
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int32_t d =
                    dim_tile * P::kM + p.first_row() + 32 * m + 8 * g + 4 * (lane >> 5);
                if (d >= c.dim) continue;
                f32x4 v{p.sum[m][n][4 * g], p.sum[m][n][4 * g + 1], p.sum[m][n][4 * g + 2],
                        p.sum[m][n][4 * g + 3]};
                if (q.first_vocab > 0) v += *reinterpret_cast<const f32x4 *>(out + d);
                *reinterpret_cast<f32x4 *>(out + d) = v;
            }
    }
}

// dW of a piece: channels (rows) by vocabulary (columns).
template <bool kHalf, bool kExact>
__device__ __forceinline__ void weight_gradient(const lct_cross_entropy &c, const Counted &t,
                                                int32_t count, const PieceProducts &q,
                                                int64_t item, uint16_t *stage0, uint16_t *stage1,
                                                uint16_t *stage2, uint16_t *stage3) {
    using P = WeightProduct<kHalf, kExact>;
    const int32_t dim_tile = static_cast<int32_t>(item % q.dim_tiles);
    const int32_t vocab_tile = static_cast<int32_t>(item / q.dim_tiles);
    int64_t x_stride;
    const void *x = hidden_of(c, t, count, &x_stride);
    typename P::A a;
    typename P::B b;
    a.prepare(x, x_stride, int64_t{dim_tile} * P::kM, c.dim);
    b.prepare(q.dz, q.dz_stride, int64_t{vocab_tile} * P::kN, q.piece);
    P p;
    p.begin();
    // Tokens past the last: zeros of dz (up to 7) against zeros of x.
    p.run(a, b, count, stage0, stage1, stage2, stage3);
    if constexpr (kExact) {
        b.prepare(q.dz_rest, q.dz_stride, int64_t{vocab_tile} * P::kN, q.piece);
        p.run(a, b, count, stage0, stage1, stage2, stage3);
    }

    const float scale = *t.scale;
    const int32_t column = vocab_tile * P::kN + p.first_column();
    const int32_t row = dim_tile * P::kM + p.first_row();
    store_columns<P>(q.grad_weight + (int64_t{q.first_vocab} + column) * c.dim + row, c.dim,
                     q.piece - column, c.dim - row, turn_values<P>(stage0, stage1, stage2, stage3),
                     [&](int m, int n, int r) {
                         return Element<kHalf>::round_pair(p.sum[m][n][r] * scale,
                                                           p.sum[m][n][r + 1] * scale);
                     });
}

// Both, one launch: neither has as many tiles as fill the compute units evenly.
//
// Bound by the matrix instructions: a quarter of 8192 x 50304 x 768 314 to 322 us, 1010 to 980
// TFLOP/s (96 tiles 400 steps deep and 150 of 256 fill the compute units to three quarters: busy
// 0.66 of the time, matrix instructions 0.50, at 1.93 GHz); a thirteenth of 14746 x 100352 x 2048
// 794 to 820 us, 1180 to 1140 (0.86, 0.63, 1.77 GHz).
template <bool kHalf, bool kExact>
__global__ __launch_bounds__(kExact ? 256 : 512, kExact ? 2 : 1) void products_kernel(
    lct_cross_entropy c, Counted t, PieceProducts q, uint32_t weight_grid) {
    using P = HiddenProduct<kHalf, kExact>;
    static_assert(P::kThreads == (kExact ? 256 : 512)
                  && P::kThreads == WeightProduct<kHalf, kExact>::kThreads);
    static_assert(P::kStage == WeightProduct<kHalf, kExact>::kStage
                  && P::kStages == WeightProduct<kHalf, kExact>::kStages);
    LCT_PRODUCT_STAGES(P);
    const int32_t count = *t.count;
    if (blockIdx.x < weight_grid) {
        const int64_t items = int64_t{q.dim_tiles} * q.vocab_tiles;
        const int64_t item = xcd_item(items, blockIdx.x);
        if (item < items)
            weight_gradient<kHalf, kExact>(c, t, count, q, item, stage0, stage1, stage2, stage3);
    } else {
        const int64_t items = int64_t{q.dim_tiles} * q.token_tiles * q.splits;
        const int64_t item = xcd_item(items, blockIdx.x - weight_grid);
        if (item < items)
            hidden_gradient<kHalf, kExact>(c, count, q, item, stage0, stage1, stage2, stage3);
    }
}

// dx from its parts, 8 values a thread; zeros for tokens that do not count.
template <bool kHalf>
__device__ __forceinline__ void join_hidden(const lct_cross_entropy &c, const Counted &t,
                                            int32_t splits, const float *__restrict__ parts,
                                            uint16_t *__restrict__ grad_x, int64_t first,
                                            int64_t step) {
    using E = Element<kHalf>;
    const int32_t count = *t.count, chunks = c.dim / 8;
    const float scale = *t.scale;
    for (int64_t at = first; at < int64_t{count} * chunks; at += step) {
        const int32_t i = static_cast<int32_t>(at / chunks);
        const int32_t d = static_cast<int32_t>(at % chunks) * 8;
        f32x4 lo{}, hi{};
        for (int32_t s = 0; s < splits; ++s) {
            const float *from = parts + (int64_t{s} * c.tokens + i) * c.dim + d;
            lo += *reinterpret_cast<const f32x4 *>(from);
            hi += *reinterpret_cast<const f32x4 *>(from + 4);
        }
        lo *= scale;
        hi *= scale;
        *reinterpret_cast<u32x4 *>(grad_x + int64_t{t.rows[i]} * c.dim + d) =
            u32x4{E::round_pair(lo[0], lo[1]), E::round_pair(lo[2], lo[3]),
                  E::round_pair(hi[0], hi[1]), E::round_pair(hi[2], hi[3])};
    }
    if (count == c.tokens) return;
    for (int64_t at = first; at < int64_t{c.tokens} * chunks; at += step)
        if (target_of(c, at / chunks) == c.ignore_index)
            *reinterpret_cast<u32x4 *>(grad_x + at * 8) = u32x4{0u, 0u, 0u, 0u};
}

// The bias's gradient: 64 of the vocabulary, their parts (one per `rows` / 2 tokens) among the
// four waves.
__device__ __forceinline__ void join_bias(const lct_cross_entropy &c, const Counted &t,
                                          int32_t rows, const float *__restrict__ parts,
                                          float *__restrict__ grad_bias, int32_t block) {
    __shared__ float sums[4][kWave];
    const int32_t v = block * kWave + wave_lane(), wave = threadIdx.x / kWave;
    const int32_t all = 2 * ((*t.count + rows - 1) / rows);
    float sum = 0.0f;
    if (v < c.vocab)
        for (int32_t i = wave; i < all; i += 4) sum += parts[int64_t{i} * c.vocab + v];
    sums[wave][wave_lane()] = sum;
    __syncthreads();
    if (wave == 0 && v < c.vocab)
        grad_bias[v] = (sum + sums[1][wave_lane()] + (sums[2][wave_lane()] + sums[3][wave_lane()]))
                       * *t.scale;
}

template <bool kHalf>
__global__ __launch_bounds__(256) void join_gradients_kernel(lct_cross_entropy c, Counted t,
                                                             int32_t splits, const float *hidden,
                                                             uint16_t *grad_x, int32_t rows,
                                                             const float *bias, float *grad_bias,
                                                             uint32_t bias_grid) {
    if (blockIdx.x < bias_grid)
        join_bias(c, t, rows, bias, grad_bias, blockIdx.x);
    else
        join_hidden<kHalf>(c, t, splits, hidden, grad_x,
                           int64_t{blockIdx.x - bias_grid} * 256 + threadIdx.x,
                           int64_t{gridDim.x - bias_grid} * 256);
}

// ---- entry points

bool aligned(const void *p, uintptr_t bytes) { return !(reinterpret_cast<uintptr_t>(p) % bytes); }

int32_t check(const lct_cross_entropy *c) {
    if (c == nullptr || c->x == nullptr || c->weight == nullptr || c->targets == nullptr)
        return LCT_E_NULL;
    // Tiles are addressed by 32-bit byte offsets: 256 rows of up to 2^22 values.  A launch has
    // fewer than 2^32 threads, 256 for 192 x 128 logits.
    if (c->tokens < 1 || c->tokens > LCT_MAX_CROSS_ENTROPY_TOKENS || c->vocab < 1
        || c->vocab > LCT_MAX_CROSS_ENTROPY_VOCAB || c->dim < 8 || c->dim % 8
        || c->dim > LCT_MAX_CROSS_ENTROPY_DIM
        || int64_t{c->tokens} * c->vocab > LCT_MAX_CROSS_ENTROPY_LOGITS)
        return LCT_E_SIZE;
    if (c->x_stride < c->dim || c->x_stride % 8 || c->x_stride > LCT_MAX_CROSS_ENTROPY_DIM
        || c->weight_stride < c->dim || c->weight_stride % 8
        || c->weight_stride > LCT_MAX_CROSS_ENTROPY_DIM || !aligned(c->x, 16)
        || !aligned(c->weight, 16) || !aligned(c->bias, 4)
        || !aligned(c->targets, c->targets_64 ? 8 : 4) || !(c->softcap >= 0.0f)
        || !(c->softcap < 1e19f) || (c->softcap > 0.0f && c->softcap < 1e-19f))
        return LCT_E_ARG;
    return 0;
}

int32_t tiles_of(int64_t n, int32_t tile) { return static_cast<int32_t>((n + tile - 1) / tile); }

constexpr int32_t kMaxStrideGrid = 1 << 16;
constexpr int64_t kMaxItems = int64_t{1} << 22;    // 512 threads each: below 2^32
// Tokens up to which four waves join one's parts.  us of a call with four | one: 50304 x 768, 64
// tokens 26.2 | 27.9, 256 35.3 | 36.9, 1024 91.4 | 92.4, 2048 159.2 | 158.7, 4096 297.1 | 294.6.
constexpr int32_t kWideJoin = 1024;

uint32_t chunk_grid_of(const lct_cross_entropy &c) {
    return static_cast<uint32_t>(
        std::min<int64_t>(kMaxStrideGrid, (int64_t{c.tokens} * (c.dim / 8) + 255) / 256));
}

void prepare(const lct_cross_entropy &c, const Counted &t, void *gathered,
             const PrepareGradients &g, float *lse, float *losses, hipStream_t stream) {
    const bool here = int64_t{c.tokens} * (c.dim / 8) <= kGatherHere;
    prepare_kernel<<<1, kPrepareThreads, 0, stream>>>(c, t, g, lse, losses,
                                                      here ? gathered : nullptr);
    if (!here) gather_kernel<<<chunk_grid_of(c), 256, 0, stream>>>(c, t, gathered);
}

template <class T>
struct Type {
    using type = T;
};

template <class Launch>
void by_form(const lct_cross_entropy &c, Launch launch) {
    const auto with = [&](auto half) {
        const auto capped = [&](auto cap) {
            if (c.bias != nullptr) launch(half, cap, std::true_type{});
            else launch(half, cap, std::false_type{});
        };
        if (c.softcap > 0.0f) capped(std::true_type{});
        else capped(std::false_type{});
    };
    if (c.fp16) with(std::true_type{});
    else with(std::false_type{});
}

}  // namespace
}  // namespace lct

using namespace lct;

extern "C" int32_t lct_cross_entropy_forward(const lct_cross_entropy *c, int32_t *index,
                                             int64_t index_size, void *gathered,
                                             int64_t gathered_size, float *parts,
                                             int64_t part_floats, float *lse, float *losses,
                                             float *total, int32_t mean, hipStream_t stream) {
    if (const int32_t bad = check(c)) return bad;
    if (parts == nullptr || lse == nullptr || losses == nullptr) return LCT_E_NULL;
    // (Up to 128 tokens would leave half of a deep tile without any.)
    const bool few = c->tokens <= kFewTokens, deep = c->dim >= kDeep && c->tokens > 128;
    const int32_t vocab_tiles = tiles_of(c->vocab, few ? 128 : deep ? 256 : kLogitRows);
    const int32_t token_tiles = tiles_of(c->tokens, few ? kFewTokens : deep ? 256 : 128);
    const int32_t entries = (few || deep ? 4 : 2) * vocab_tiles;
    if (part_floats < int64_t{2} * entries * c->tokens || !aligned(parts, 8)) return LCT_E_SIZE;
    Counted t{};
    if (index != nullptr) {
        if (gathered == nullptr) return LCT_E_NULL;
        if (index_size < 1 + 2 * int64_t{c->tokens}
            || gathered_size < int64_t{c->tokens} * c->dim || !aligned(gathered, 16))
            return LCT_E_SIZE;
        t.count = index;
        t.rows = index + 1;
        t.targets = index + 1 + c->tokens;
        t.gathered = gathered;
        prepare(*c, t, gathered, PrepareGradients{}, lse, losses, stream);
    }
    const uint32_t grid = static_cast<uint32_t>(xcd_grid(int64_t{vocab_tiles} * token_tiles));
    auto *of = reinterpret_cast<Part *>(parts);
    by_form(*c, [&](auto half, auto cap, auto bias) {
        constexpr bool kHalf = decltype(half)::value;
        const auto with = [&](auto product) {
            using P = typename decltype(product)::type;
            logits_kernel<P, decltype(cap)::value, decltype(bias)::value>
                <<<grid, P::kThreads, 0, stream>>>(*c, t, vocab_tiles, token_tiles, of);
        };
        if (few) with(Type<FewProduct<kHalf>>{});
        else if (deep) with(Type<DeepProduct<kHalf>>{});
        else with(Type<LogitProduct<kHalf>>{});
    });
    const bool wide = c->tokens <= kWideJoin;
    const uint32_t joins = static_cast<uint32_t>(wide ? c->tokens : (c->tokens + 3) / 4);
    const auto join = [&](auto half) {
        constexpr bool kHalf = decltype(half)::value;
        if (wide)
            join_kernel<kHalf, 4><<<joins, 256, 0, stream>>>(*c, t, entries, of, lse, losses);
        else
            join_kernel<kHalf, 1><<<joins, 256, 0, stream>>>(*c, t, entries, of, lse, losses);
    };
    if (c->fp16) join(std::true_type{});
    else join(std::false_type{});
    if (total != nullptr)
        total_kernel<<<1, kPrepareThreads, 0, stream>>>(*c, losses, mean, total);
    return static_cast<int32_t>(hipGetLastError());
}

extern "C" int32_t lct_cross_entropy_backward(const lct_cross_entropy *c,
                                              const lct_cross_entropy_gradients *d,
                                              hipStream_t stream) {
    if (const int32_t bad = check(c)) return bad;
    if (d == nullptr || d->grad == nullptr || d->lse == nullptr || d->losses == nullptr
        || d->index == nullptr || d->values == nullptr || d->gathered == nullptr)
        return LCT_E_NULL;
    const bool products = d->grad_x != nullptr || d->grad_weight != nullptr;
    if ((products && d->dz == nullptr) || (d->grad_x != nullptr && d->hidden_parts == nullptr)
        || (d->grad_bias != nullptr && (d->bias_parts == nullptr || c->bias == nullptr)))
        return LCT_E_NULL;
    const int64_t tokens = c->tokens, pitch = (tokens + 7) / 8 * 8;
    const bool exact = tokens <= LCT_CROSS_ENTROPY_EXACT_TOKENS;
    const int32_t token_tiles = tiles_of(tokens, kLogitRows);
    if (d->piece < 1 || d->piece % 128 || d->splits < 1 || d->splits > LCT_MAX_CROSS_ENTROPY_SPLITS
        || d->index_size < 1 + 2 * tokens || d->value_floats < 1 + 3 * tokens
        || d->gathered_size < tokens * c->dim
        || (products && d->dz_size < std::min(d->piece, c->vocab) * pitch * (exact ? 2 : 1))
        || (d->grad_x != nullptr && d->hidden_floats < d->splits * tokens * c->dim)
        || (d->grad_bias != nullptr
            && d->bias_floats < int64_t{2} * token_tiles * c->vocab))
        return LCT_E_SIZE;
    if (!aligned(d->gathered, 16) || !aligned(d->dz, 16) || !aligned(d->hidden_parts, 16)
        || !aligned(d->grad_x, 16) || !aligned(d->grad_weight, 16))
        return LCT_E_ARG;
    const int32_t tile = exact ? 128 : 256;    // of tokens and of the vocabulary
    const int32_t dim_tiles = tiles_of(c->dim, 256), hidden_tiles = tiles_of(tokens, tile);
    if (int64_t{dim_tiles} * (int64_t{hidden_tiles} * d->splits
                              + tiles_of(std::min(d->piece, c->vocab), tile)) > kMaxItems)
        return LCT_E_SIZE;
    Counted t{};
    int32_t *rows = d->index + 1, *targets = rows + tokens;
    float *lse = d->values + 1, *losses = lse + tokens, *factor = losses + tokens;
    t.count = d->index;
    t.rows = rows;
    t.targets = targets;
    t.scale = d->values;
    t.lse = lse;
    t.losses = losses;
    t.factor = factor;
    t.gathered = d->gathered;
    prepare(*c, t, d->gathered, PrepareGradients{d->grad, d->grad_per_token, d->mean},
            const_cast<float *>(d->lse), const_cast<float *>(d->losses), stream);
    const uint32_t chunk_grid = chunk_grid_of(*c);
    auto *dz = static_cast<uint16_t *>(d->dz);
    uint16_t *const rest = exact && dz != nullptr ? dz + std::min(d->piece, c->vocab) * pitch
                                                  : nullptr;
    for (int32_t first = 0; first < c->vocab; first += d->piece) {
        const int32_t piece = std::min(d->piece, c->vocab - first);
        const int32_t vocab_tiles = tiles_of(piece, 128);
        const uint32_t grid = static_cast<uint32_t>(xcd_grid(int64_t{vocab_tiles} * token_tiles));
        by_form(*c, [&](auto half, auto cap, auto bias) {
            gradient_kernel<LogitProduct<decltype(half)::value>, decltype(half)::value,
                            decltype(cap)::value, decltype(bias)::value>
                <<<grid, 256, 0, stream>>>(*c, t, first, piece, vocab_tiles, token_tiles,
                                           products ? dz : nullptr, products ? rest : nullptr,
                                           pitch,
                                           d->grad_bias != nullptr ? d->bias_parts : nullptr);
        });
        if (!products) continue;
        const int32_t weight_tiles = tiles_of(piece, tile);
        const PieceProducts q{first,        piece,        d->splits, dim_tiles,
                              hidden_tiles, weight_tiles, dz,        rest,
                              pitch,        d->hidden_parts,
                              static_cast<uint16_t *>(d->grad_weight)};
        const uint32_t weight_grid =
            d->grad_weight == nullptr
                ? 0
                : static_cast<uint32_t>(xcd_grid(int64_t{dim_tiles} * weight_tiles));
        const uint32_t hidden_grid =
            d->grad_x == nullptr
                ? 0
                : static_cast<uint32_t>(xcd_grid(int64_t{dim_tiles} * hidden_tiles * d->splits));
        const auto multiply = [&](auto half, auto both) {
            constexpr bool kHalf = decltype(half)::value, kBoth = decltype(both)::value;
            products_kernel<kHalf, kBoth>
                <<<weight_grid + hidden_grid, HiddenProduct<kHalf, kBoth>::kThreads, 0, stream>>>(
                    *c, t, q, weight_grid);
        };
        const auto with = [&](auto half) {
            if (exact) multiply(half, std::true_type{});
            else multiply(half, std::false_type{});
        };
        if (c->fp16) with(std::true_type{});
        else with(std::false_type{});
    }
    const uint32_t bias_grid =
        d->grad_bias != nullptr ? static_cast<uint32_t>(tiles_of(c->vocab, kWave)) : 0;
    const uint32_t hidden_grid = d->grad_x != nullptr ? chunk_grid : 0;
    if (bias_grid + hidden_grid > 0) {
        auto *out = static_cast<uint16_t *>(d->grad_x);
        if (c->fp16)
            join_gradients_kernel<true><<<bias_grid + hidden_grid, 256, 0, stream>>>(
                *c, t, d->splits, d->hidden_parts, out, kLogitRows, d->bias_parts, d->grad_bias,
                bias_grid);
        else
            join_gradients_kernel<false><<<bias_grid + hidden_grid, 256, 0, stream>>>(
                *c, t, d->splits, d->hidden_parts, out, kLogitRows, d->bias_parts, d->grad_bias,
                bias_grid);
    }
    return static_cast<int32_t>(hipGetLastError());
}
