// Dropout from a counter-based generator, with the residual's addition:
// out = residual + (kept ? x factor : 0).
//
// Eight values share one draw of Philox-4x32 with ten rounds (J. Salmon, M.
// Moraes, R. Dror and D. Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// 2011), at counter (index / 8, offset) under the key `seed`; a value is kept
// where its 16 bits are at least `below`.  The mask is a function of these
// alone: it is never stored, and the gradient's pass draws it again.
//
// Bound by memory where the launch is not what counts (the ten rounds' products
// take about half of the time that the values' bytes do): a thread has one draw.
#include <type_traits>

#include "attention_core.h"

namespace lct {
namespace {

constexpr int kThreads = 256;
// With the residual, tensors of more bytes than the memory side's cache are read
// and written past the caches: 121 us in place of 139 at 16383 x 8192 BF16 (6.7
// TB/s), 6.3 to 8.0 | 7.4 to 7.6 at 8192 x 768.  Without (83 us at 16383 x 8192,
// 6.5 TB/s), it makes no difference.
constexpr int64_t kCacheBytes = int64_t{256} << 20;

// The four words of counter (index, offset).
__device__ __forceinline__ u32x4 philox(uint64_t index, uint64_t offset, uint64_t seed) {
    uint32_t a = static_cast<uint32_t>(index), b = static_cast<uint32_t>(index >> 32);
    uint32_t c = static_cast<uint32_t>(offset), d = static_cast<uint32_t>(offset >> 32);
    uint32_t low = static_cast<uint32_t>(seed), high = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t x = uint64_t{a} * 0xD2511F53u, y = uint64_t{c} * 0xCD9E8D57u;
        a = static_cast<uint32_t>(y >> 32) ^ b ^ low;
        b = static_cast<uint32_t>(y);
        c = static_cast<uint32_t>(x >> 32) ^ d ^ high;
        d = static_cast<uint32_t>(x);
        low += 0x9E3779B9u;
        high += 0xBB67AE85u;
    }
    return u32x4{a, b, c, d};
}

// 16 bytes; kOnce: past the caches.
template <bool kOnce>
__device__ __forceinline__ u32x4 load16(const void *p) {
    if constexpr (kOnce) return __builtin_nontemporal_load(static_cast<const u32x4 *>(p));
    else return *static_cast<const u32x4 *>(p);
}
template <bool kOnce>
__device__ __forceinline__ void store16(u32x4 v, void *p) {
    if constexpr (kOnce) __builtin_nontemporal_store(v, static_cast<u32x4 *>(p));
    else *static_cast<u32x4 *>(p) = v;
}

template <int kType, bool kOnce>
struct Eight;      // eight values as FP32, from and to memory

template <bool kHalf, bool kOnce>
struct EightHalves {
    u32x4 v;
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        v = load16<kOnce>(static_cast<const uint16_t *>(p) + i);
    }
    __device__ __forceinline__ void load_some(const void *p, int64_t i, int count) {
        v = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count)
                v[j / 2] |= uint32_t{static_cast<const uint16_t *>(p)[i + j]} << (16 * (j & 1));
    }
    __device__ __forceinline__ float get(int j) const {
        return j & 1 ? Element<kHalf>::high(v[j / 2]) : Element<kHalf>::low(v[j / 2]);
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = Element<kHalf>::round_pair(x[2 * j], x[2 * j + 1]);
    }
    __device__ __forceinline__ void store(void *p, int64_t i) const {
        store16<kOnce>(v, static_cast<uint16_t *>(p) + i);
    }
    __device__ __forceinline__ void store_some(void *p, int64_t i, int count) const {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count)
                static_cast<uint16_t *>(p)[i + j] =
                    static_cast<uint16_t>(v[j / 2] >> (16 * (j & 1)));
    }
};
template <bool kOnce>
struct Eight<LCT_BF16, kOnce> : EightHalves<false, kOnce> {};
template <bool kOnce>
struct Eight<LCT_FP16, kOnce> : EightHalves<true, kOnce> {};
template <bool kOnce>
struct Eight<LCT_FP32, kOnce> {
    f32x4 v[2];
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        const float *src = static_cast<const float *>(p) + i;
        v[0] = __builtin_bit_cast(f32x4, load16<kOnce>(src));
        v[1] = __builtin_bit_cast(f32x4, load16<kOnce>(src + 4));
    }
    __device__ __forceinline__ void load_some(const void *p, int64_t i, int count) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j / 4][j & 3] = 0.0f;
            if (j < count) v[j / 4][j & 3] = static_cast<const float *>(p)[i + j];
        }
    }
    __device__ __forceinline__ float get(int j) const { return v[j / 4][j & 3]; }
    __device__ __forceinline__ void set(const float (&x)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j / 4][j & 3] = x[j];
    }
    __device__ __forceinline__ void store(void *p, int64_t i) const {
        float *dst = static_cast<float *>(p) + i;
        store16<kOnce>(__builtin_bit_cast(u32x4, v[0]), dst);
        store16<kOnce>(__builtin_bit_cast(u32x4, v[1]), dst + 4);
    }
    __device__ __forceinline__ void store_some(void *p, int64_t i, int count) const {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) static_cast<float *>(p)[i + j] = v[j / 4][j & 3];
    }
};

template <int kType, bool kResidual, bool kOnce>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const void *__restrict__ x,
                                                           const void *__restrict__ residual,
                                                           void *__restrict__ out, int64_t n,
                                                           uint32_t below, float factor,
                                                           uint64_t seed, uint64_t offset,
                                                           const int64_t *__restrict__ more) {
    const int64_t group = int64_t{blockIdx.x} * kThreads + threadIdx.x, i = group * 8;
    if (i >= n) return;
    if (more != nullptr) offset += static_cast<uint64_t>(*more);
    const bool whole = i + 8 <= n;
    const int count = whole ? 8 : static_cast<int>(n - i);
    Eight<kType, kOnce> values, base;
    if (whole) {
        values.load(x, i);
        if (kResidual) base.load(residual, i);
    } else {
        values.load_some(x, i, count);
        if (kResidual) base.load_some(residual, i, count);
    }
    const u32x4 words = philox(static_cast<uint64_t>(group), offset, seed);
    float result[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t bits = j & 1 ? words[j / 2] >> 16 : words[j / 2] & 0xFFFFu;
        // A select, not a product: an infinity or NaN that is dropped is gone.
        if (kResidual)
            result[j] = bits >= below ? __builtin_fmaf(values.get(j), factor, base.get(j))
                                      : base.get(j);
        else
            result[j] = bits >= below ? values.get(j) * factor : 0.0f;
    }
    values.set(result);
    if (whole) values.store(out, i);
    else values.store_some(out, i, count);
}

template <int kType>
int32_t launch(const void *x, const void *residual, void *out, int64_t n, uint32_t below,
               float factor, uint64_t seed, uint64_t offset, const int64_t *more,
               hipStream_t stream) {
    const uint32_t grid = static_cast<uint32_t>((n + kThreads * 8 - 1) / (kThreads * 8));
    const auto run = [&](auto with, auto once) {
        dropout_kernel<kType, decltype(with)::value, decltype(once)::value>
            <<<grid, kThreads, 0, stream>>>(x, residual, out, n, below, factor, seed, offset, more);
    };
    constexpr int64_t kSize = kType == LCT_FP32 ? 4 : 2;
    if (residual == nullptr) run(std::false_type{}, std::false_type{});
    else if (3 * n * kSize <= kCacheBytes) run(std::true_type{}, std::false_type{});
    else run(std::true_type{}, std::true_type{});
    return static_cast<int32_t>(hipGetLastError());
}

}  // namespace
}  // namespace lct

using namespace lct;

extern "C" int32_t lct_dropout(const void *x, const void *residual, void *out, int64_t n,
                               int32_t type, int32_t below, uint64_t seed, uint64_t offset,
                               const int64_t *offset_more, hipStream_t stream) {
    if (!x || !out) return LCT_E_NULL;
    if (n <= 0 || n > (int64_t{1} << 35) - 2048) return LCT_E_SIZE;
    if (below < 0 || below > 65536
        || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual)
             | reinterpret_cast<uintptr_t>(out))
            & 15) != 0
        || (reinterpret_cast<uintptr_t>(offset_more) & 7) != 0)
        return LCT_E_ARG;
    // The inverse of the chance of being kept, so that the mean stays.
    const float factor = below < 65536 ? 65536.0f / static_cast<float>(65536 - below) : 0.0f;
    switch (type) {
    case LCT_BF16:
        return launch<LCT_BF16>(x, residual, out, n, below, factor, seed, offset, offset_more,
                                stream);
    case LCT_FP16:
        return launch<LCT_FP16>(x, residual, out, n, below, factor, seed, offset, offset_more,
                                stream);
    case LCT_FP32:
        return launch<LCT_FP32>(x, residual, out, n, below, factor, seed, offset, offset_more,
                                stream);
    default: return LCT_E_ARG;
    }
}
