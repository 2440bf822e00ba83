// Rotary positions of queries and keys, and a new token's way into the caches.
//
// A pair (x, y) of channels at position p turns by the angle p f of its
// frequency: (x cos - y sin, y cos + x sin), times a magnitude.  Frequencies are
// fractions of a turn per position in 64-bit fixed point, so the product with
// the position wraps modulo one turn exactly: no table bounds the context.  A
// position p multiplies the frequency's rounding, 2^-65 of a turn; for any that 32
// bits hold the product is less than the angle's rounding to FP32 in [-1/2, 1/2].
//
// Follows examples/nanogpt/train_gpt_lct.py:150-165 (whose rotation has the
// other sense: negative frequencies).
#include <algorithm>

#include "attention_core.h"

namespace lct {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = LCT_MAX_ROTARY_DIM / 2;
constexpr int kMaxTokens = 16;       // tokens of a workgroup

template <int kType>
struct Value;
template <>
struct Value<LCT_BF16> {
    using Bits = uint16_t;
    static __device__ __forceinline__ float load(Bits b) { return bf16_to_float(b); }
    static __device__ __forceinline__ Bits store(float x) {
        return __builtin_bit_cast(Bits, static_cast<__bf16>(x));
    }
};
template <>
struct Value<LCT_FP16> {
    using Bits = uint16_t;
    static __device__ __forceinline__ float load(Bits b) {
        return static_cast<float>(__builtin_bit_cast(_Float16, b));
    }
    static __device__ __forceinline__ Bits store(float x) {
        return __builtin_bit_cast(Bits, static_cast<_Float16>(x));
    }
};
template <>
struct Value<LCT_FP32> {
    using Bits = uint32_t;
    static __device__ __forceinline__ float load(Bits b) { return __uint_as_float(b); }
    static __device__ __forceinline__ Bits store(float x) { return __float_as_uint(x); }
};

// How the (token, head, unit) items of a workgroup's tokens are counted: units
// of kVector adjacent channels (with those half the rotated part further on in
// the half layout), pairs first, then the channels that are only copied.
struct Counts {
    int32_t per_group;      // tokens of a workgroup
    int32_t pair_units, units, per_token;
    uint32_t units_inverse, per_token_inverse;   // ceil(2^32 / .), 0 for 1, 1 for all
};

__device__ __forceinline__ int32_t divide(int32_t x, uint32_t inverse) {
    return inverse == 0u ? x : static_cast<int32_t>(__umulhi(static_cast<uint32_t>(x), inverse));
}

__device__ __forceinline__ int64_t position_of(const lct_rotary &r, int64_t b, int64_t t) {
    int64_t p = r.start + (r.positions == nullptr || r.position_stride[1] == 0 ? t : 0);
    if (r.positions != nullptr)
        p += r.positions[b * r.position_stride[0] + t * r.position_stride[1]];
    return p;
}

// Where a token's q, k and v are and go (elements; k's and v's place -1: nowhere).
struct Places {
    int64_t position, in[3], out[3];
};

// A workgroup takes a few tokens: it computes their angles' sines and cosines
// once, into LDS, for all of their heads, while its first units are on their way,
// then moves its units, kAhead of a thread's in flight.  Bound by memory: 127 us
// for 32767 tokens of 40 heads of 128 in FP16, half of each turned (5.3 TB/s; one
// unit at a time with the token's place computed for each: 195), 10.3 us for 8 x
// 1024 tokens of 24 heads of 64 (the angles before the first loads: 10.9), 4.3 us
// for one token of 64 sequences, most of it the launch.
template <int kType, int kVector, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rotary_kernel(lct_rotary r, Counts n) {
    using V = Value<kType>;
    using Bits = typename V::Bits;
    struct alignas(sizeof(Bits) * kVector) Pack {
        Bits v[kVector];
    };
    constexpr int kAhead = 4;
    __shared__ f32x2 turn[kMaxTokens * kMaxPairs];
    __shared__ Places places[kMaxTokens];
    const int64_t tokens = int64_t{r.batch} * r.tokens;
    const int64_t first = int64_t{blockIdx.x} * n.per_group;
    const int32_t here = static_cast<int32_t>(min(int64_t{n.per_group}, tokens - first));
    const int32_t pairs = r.rotary_dim / 2;
    if (static_cast<int32_t>(threadIdx.x) < here) {
        static_assert(kMaxTokens <= kThreads, "a thread per token");
        const int64_t token = first + threadIdx.x, b = token / r.tokens, t = token % r.tokens;
        const int64_t p = position_of(r, b, t);
        Places &at = places[threadIdx.x];
        at.position = p;
        at.in[0] = b * r.q_in_stride[0] + t * r.q_in_stride[1];
        at.in[1] = b * r.k_in_stride[0] + t * r.k_in_stride[1];
        at.in[2] = b * r.v_in_stride[0] + t * r.v_in_stride[1];
        at.out[0] = b * r.q_out_stride[0] + t * r.q_out_stride[1];
        const int64_t to = r.capacity > 0 ? p : t;
        const bool kept = r.capacity == 0 || (p >= 0 && p < r.capacity);
        at.out[1] = kept ? b * r.k_out_stride[0] + to * r.k_out_stride[1] : -1;
        at.out[2] = kept ? b * r.v_out_stride[0] + to * r.v_out_stride[1] : -1;
    }
    __syncthreads();

    const int32_t items = here * n.per_token;
    Pack x[kAhead], y[kAhead];
    Bits *dst[kAhead];           // null: nothing to store
    int32_t angles[kAhead];      // first of the unit's in `turn`, or -1: a copy
    int32_t gap[kAhead];         // from x's channels to y's, or 0: no y
    const auto load = [&](int32_t base) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            dst[u] = nullptr;
            angles[u] = -1;
            const int32_t i = base + u * kThreads;
            if (i >= items) continue;
            const int32_t token = divide(i, n.per_token_inverse);
            const int32_t in_token = i - token * n.per_token;
            int32_t head = divide(in_token, n.units_inverse);
            const int32_t unit = in_token - head * n.units;
            // q's heads, then k's, then v's.
            const bool is_q = head < r.heads;
            if (!is_q) head -= r.heads;
            const bool is_k = !is_q && head < r.kv_heads;
            if (!is_q && !is_k) head -= r.kv_heads;
            const auto pick = [&](auto q, auto k, auto v) { return is_q ? q : is_k ? k : v; };
            const int which = pick(0, 1, 2);
            const int64_t to = places[token].out[which];
            if (to < 0) continue;
            const int32_t in_head = static_cast<int32_t>(
                pick(r.q_in_stride[2], r.k_in_stride[2], r.v_in_stride[2]));
            const int32_t out_head = static_cast<int32_t>(
                pick(r.q_out_stride[2], r.k_out_stride[2], r.v_out_stride[2]));
            int32_t c = unit * kVector;
            gap[u] = 0;
            if (unit >= n.pair_units) {              // channels past the rotated part
                c = r.rotary_dim + (unit - n.pair_units) * kVector;
            } else if (!kInterleaved) {
                angles[u] = token * pairs + c;
                gap[u] = pairs;
            } else if (kVector > 1) {
                angles[u] = token * pairs + c / 2;
            } else {
                c = 2 * unit;
                angles[u] = token * pairs + unit;
                gap[u] = 1;
            }
            if (which == 2) angles[u] = -1;
            const Bits *src = static_cast<const Bits *>(pick(r.q_in, r.k_in, r.v_in))
                              + places[token].in[which] + int64_t{head} * in_head + c;
            dst[u] = static_cast<Bits *>(pick(r.q_out, r.k_out, r.v_out)) + to
                     + int64_t{head} * out_head + c;
            x[u] = *reinterpret_cast<const Pack *>(src);
            if (gap[u] != 0) y[u] = *reinterpret_cast<const Pack *>(src + gap[u]);
        }
    };
    const auto store = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (dst[u] == nullptr) continue;
            if constexpr (kInterleaved && kVector > 1) {
                if (angles[u] >= 0) {
#pragma unroll
                    for (int j = 0; j < kVector; j += 2) {
                        const f32x2 a = turn[angles[u] + j / 2];
                        const float v = V::load(x[u].v[j]), w = V::load(x[u].v[j + 1]);
                        x[u].v[j] = V::store(v * a[0] - w * a[1]);
                        x[u].v[j + 1] = V::store(w * a[0] + v * a[1]);
                    }
                }
                *reinterpret_cast<Pack *>(dst[u]) = x[u];
                continue;
            }
            if (angles[u] >= 0) {
#pragma unroll
                for (int j = 0; j < kVector; ++j) {
                    const f32x2 a = turn[angles[u] + j];
                    const float v = V::load(x[u].v[j]), w = V::load(y[u].v[j]);
                    x[u].v[j] = V::store(v * a[0] - w * a[1]);
                    y[u].v[j] = V::store(w * a[0] + v * a[1]);
                }
            }
            *reinterpret_cast<Pack *>(dst[u]) = x[u];
            if (gap[u] != 0) *reinterpret_cast<Pack *>(dst[u] + gap[u]) = y[u];
        }
    };

    load(threadIdx.x);
    for (int32_t i = threadIdx.x; i < here * pairs; i += kThreads) {
        const int32_t token = i / pairs;
        const int64_t angle =
            static_cast<int64_t>(static_cast<uint64_t>(places[token].position)
                                 * static_cast<uint64_t>(r.turns[i - token * pairs]));
        float sine, cosine;
        sincospif(static_cast<float>(angle) * 0x1p-63f, &sine, &cosine);
        turn[i] = f32x2{cosine * r.magnitude, (r.inverse ? -sine : sine) * r.magnitude};
    }
    __syncthreads();
    for (int32_t base = threadIdx.x; base < items;) {
        store();
        base += kAhead * kThreads;
        if (base < items) load(base);
    }
}

// x / d is the high half of x ceil(2^32 / d) where x d is up to 2^32: for the items
// of several tokens, up to 2^16, and for those of one (3 x 4096 heads of 128 units).
constexpr int32_t kMaxItems = 1 << 16;

uint32_t inverse_of(int32_t x) {
    return static_cast<uint32_t>(((uint64_t{1} << 32) + x - 1) / x);
}

bool multiples(const int64_t (&stride)[3], int32_t of) {
    return stride[0] % of == 0 && stride[1] % of == 0 && stride[2] % of == 0;
}

bool heads_near(const int64_t (&stride)[3]) {
    return stride[2] >= 0 && stride[2] <= INT32_MAX;
}

bool aligned_to(const void *p, uintptr_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

template <int kType, int kVector>
int32_t launch(const lct_rotary &r, hipStream_t stream) {
    const int32_t pairs = r.rotary_dim / 2;
    Counts n;
    n.pair_units = r.interleaved && kVector > 1 ? r.rotary_dim / kVector : pairs / kVector;
    n.units = n.pair_units + (r.head_dim - r.rotary_dim) / kVector;
    n.per_token = (r.heads + (r.k_in ? r.kv_heads : 0) + (r.v_in ? r.kv_heads : 0)) * n.units;
    const int64_t tokens = int64_t{r.batch} * r.tokens;
    // Whole rounds of the threads' units (to a tenth), while there are workgroups
    // for every compute unit.
    const int64_t most = std::min<int64_t>(
        {kMaxTokens, kMaxItems / n.per_token, std::max<int64_t>(1, tokens / 1024)});
    constexpr int64_t kRound = 4 * kThreads;
    n.per_group = 1;
    double best = 0.0;
    for (int64_t per = 1; per <= most; ++per) {
        const int64_t units = per * n.per_token;
        const double used = static_cast<double>(units)
                            / static_cast<double>((units + kRound - 1) / kRound * kRound);
        if (used > best + 1e-9) {
            best = used;
            n.per_group = static_cast<int32_t>(per);
        }
        if (best >= 0.9) break;
    }
    n.units_inverse = inverse_of(n.units);
    // Of one token all items are: more than kMaxItems may be its own.
    n.per_token_inverse = n.per_group == 1 ? 1u : inverse_of(n.per_token);
    const int64_t grid = (tokens + n.per_group - 1) / n.per_group;
    if (grid >= int64_t{1} << 24) return LCT_E_SIZE;
    if (r.interleaved)
        rotary_kernel<kType, kVector, true>
            <<<static_cast<uint32_t>(grid), kThreads, 0, stream>>>(r, n);
    else
        rotary_kernel<kType, kVector, false>
            <<<static_cast<uint32_t>(grid), kThreads, 0, stream>>>(r, n);
    return static_cast<int32_t>(hipGetLastError());
}

template <int kType>
int32_t by_vector(const lct_rotary &r, hipStream_t stream) {
    constexpr int kVector = 16 / sizeof(typename Value<kType>::Bits);
    const int32_t pairs = r.rotary_dim / 2;
    bool wide = (r.interleaved ? r.rotary_dim : pairs) % kVector == 0 && r.head_dim % kVector == 0
                && r.rotary_dim % kVector == 0;
    const auto fits = [&](const void *in, void *out, const int64_t (&is)[3],
                          const int64_t (&os)[3]) {
        return in == nullptr
               || (aligned_to(in, 16) && aligned_to(out, 16) && multiples(is, kVector)
                   && multiples(os, kVector));
    };
    wide = wide && fits(r.q_in, r.q_out, r.q_in_stride, r.q_out_stride)
           && fits(r.k_in, r.k_out, r.k_in_stride, r.k_out_stride)
           && fits(r.v_in, r.v_out, r.v_in_stride, r.v_out_stride);
    return wide ? launch<kType, kVector>(r, stream) : launch<kType, 1>(r, stream);
}

}  // namespace
}  // namespace lct

using namespace lct;

extern "C" int32_t lct_rotate(const lct_rotary *r, hipStream_t stream) {
    if (!r || !r->q_in || !r->q_out || !r->turns || (r->k_in && !r->k_out)
        || (r->v_in && (!r->v_out || !r->k_in)))
        return LCT_E_NULL;
    if (r->batch <= 0 || r->tokens <= 0 || r->heads <= 0 || (r->k_in && r->kv_heads <= 0)
        || r->head_dim <= 0 || r->head_dim > LCT_MAX_ROTARY_DIM || r->rotary_dim <= 0
        || r->rotary_dim > r->head_dim || (r->rotary_dim & 1) != 0 || r->capacity < 0
        || r->heads > 4096 || r->kv_heads > 4096)
        return LCT_E_SIZE;
    const uintptr_t size = r->type == LCT_FP32 ? 4 : 2;
    if (!aligned_to(r->q_in, size) || !aligned_to(r->q_out, size) || !aligned_to(r->k_in, size)
        || !aligned_to(r->k_out, size) || !aligned_to(r->v_in, size) || !aligned_to(r->v_out, size)
        || (r->v_in && r->capacity <= 0) || !heads_near(r->q_in_stride)
        || !heads_near(r->k_in_stride) || !heads_near(r->v_in_stride)
        || !heads_near(r->q_out_stride) || !heads_near(r->k_out_stride)
        || !heads_near(r->v_out_stride))
        return LCT_E_ARG;
    switch (r->type) {
    case LCT_BF16: return by_vector<LCT_BF16>(*r, stream);
    case LCT_FP16: return by_vector<LCT_FP16>(*r, stream);
    case LCT_FP32: return by_vector<LCT_FP32>(*r, stream);
    default: return LCT_E_ARG;
    }
}
