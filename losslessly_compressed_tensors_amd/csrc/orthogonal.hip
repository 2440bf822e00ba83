// Muon's orthogonalisation: a Newton-Schulz iteration on a batch of matrices.
//
// Follows the trainer's optimizer (LCT/components/sparse_utils.py:71-86), in the arithmetic
// of components/sparse_utils.py: with X = G / (|G| + eps), transposed where that makes it
// wide (rows <= columns),
//     A = X X^T,  P = b A + c A A,  X <- a X + P X,    (a, b, c) = (2, -3/2, 1/2).
//
// Three products a step, each a launch over all matrices: A and P are symmetric, so
// tiles above the diagonal are not computed but written from below it.
//
// X is held in 32 bits, as the sum of two FP16 numbers, the second at 2^11 times the first's
// power of two: 23 bits, rounded 1.5 times as far off as FP32 (root mean square), and what is
// below FP16's range in the first number is in the second's.  The products take the first
// of them, and A and P in FP16, all at fixed powers of two.  Small singular directions only
// double in the early steps.  What rounds X itself adds noise in all directions, and the
// steps that follow double that too: with X in 16 bits, 12 steps of a matrix whose
// singular values fall off as 1/i end 0.1 (BF16) or 0.01 (FP16) of the norm away.  P X is
// small in the small directions on either side, so that rounding P's and X's operands
// there is harmless: 4e-4.  Near the end, where P is -1, each step leaves what its operands'
// rounding took from X: 2e-4 sqrt(steps) of the norm after many.  No value exceeds 1 by more
// than roundings, so FP16's range suffices and its three more bits are free.
#include <algorithm>

#include "product_core.h"

namespace lct {
namespace {

constexpr float kA = 2.0f, kB = -1.5f, kC = 0.5f;
// The operands' powers of two: X within 1 + 2^-8 (2^10 of 65504), A likewise, |P| <= 1.2.
constexpr float kHoldX = 1024.0f, kHoldA = 4096.0f;
// X's second number, over the first's: at most half a step of that, 2^-12 of 2^10.
constexpr float kHoldRest = 2048.0f;

using Half = Element<true>;

// ---- from G, and to the result where it has no rows of whole 16-byte pieces

constexpr int kTile = 64;

__device__ __forceinline__ float element(const lct_orthogonal &o, int64_t at) {
    if (o.type == LCT_FP32) return static_cast<const float *>(o.input)[at];
    const uint16_t v = static_cast<const uint16_t *>(o.input)[at];
    return o.type == LCT_FP16 ? Half::low(v) : Element<false>::low(v);
}

// Eight values of a matrix, the wide orientation's (i, j) and the next seven along the
// dimension whose elements are adjacent (rows if `turned`); zeros past the end.
__device__ __forceinline__ void eight(const lct_orthogonal &o, int32_t matrix, int32_t i,
                                      int32_t j, bool turned, float (&v)[8]) {
    const int64_t at = matrix * o.stride[0] + i * o.stride[1] + j * o.stride[2];
    const int64_t step = turned ? o.stride[1] : o.stride[2];
    const bool inside = turned ? j < o.cols : i < o.rows;
    const int32_t left = inside ? (turned ? o.rows - i : o.cols - j) : 0;
    const int32_t size = o.type == LCT_FP32 ? 4 : 2;
    const char *from = static_cast<const char *>(o.input) + at * size;
    if (left >= 8 && step == 1 && reinterpret_cast<uintptr_t>(from) % 16 == 0) {
        u32x4 p = *reinterpret_cast<const u32x4 *>(from);
        if (o.type == LCT_FP32) {
            const u32x4 q = *reinterpret_cast<const u32x4 *>(from + 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = __uint_as_float(p[k]);
                v[4 + k] = __uint_as_float(q[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = o.type == LCT_FP16 ? Half::low(p[k]) : Element<false>::low(p[k]);
                v[2 * k + 1] = o.type == LCT_FP16 ? Half::high(p[k]) : Element<false>::high(p[k]);
            }
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < left ? element(o, at + k * step) : 0.0f;
}

// kCount of them, at place(k, &i, &j): where all are whole and aligned, the loads in flight
// together.
template <int kCount, class Place>
__device__ __forceinline__ void load_eights(const lct_orthogonal &o, int32_t matrix, bool turned,
                                            float (&v)[kCount][8], Place place) {
    const int32_t size = o.type == LCT_FP32 ? 4 : 2, piece = 16 / size;
    const int64_t line = turned ? o.stride[2] : o.stride[1];
    const bool whole = (turned ? o.stride[1] : o.stride[2]) == 1 && line % piece == 0
                       && o.stride[0] % piece == 0 && (turned ? o.rows : o.cols) % 8 == 0
                       && reinterpret_cast<uintptr_t>(o.input) % 16 == 0;
    if (!whole) {
#pragma unroll
        for (int k = 0; k < kCount; ++k) {
            int i, j;
            place(k, &i, &j);
            eight(o, matrix, i, j, turned, v[k]);
        }
        return;
    }
    const char *const from = static_cast<const char *>(o.input) + matrix * o.stride[0] * size;
    u32x4 raw[kCount], more[kCount];
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
        int i, j;
        place(k, &i, &j);
        const bool inside = i < o.rows && j < o.cols;
        const char *at = from + (inside ? (i * o.stride[1] + j * o.stride[2]) * size : 0);
        raw[k] = *reinterpret_cast<const u32x4 *>(at);
        if (o.type == LCT_FP32) more[k] = *reinterpret_cast<const u32x4 *>(at + 16);
    }
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
        int i, j;
        place(k, &i, &j);
        const bool inside = i < o.rows && j < o.cols;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const uint32_t pair = raw[k][n / 2];
            float of;
            if (o.type == LCT_FP32)
                of = __uint_as_float(n < 4 ? raw[k][n % 4] : more[k][n % 4]);
            else if (o.type == LCT_FP16)
                of = n % 2 ? Half::high(pair) : Half::low(pair);
            else
                of = n % 2 ? Element<false>::high(pair) : Element<false>::low(pair);
            v[k][n] = inside ? of : 0.0f;
        }
    }
}

__device__ __forceinline__ bool is_turned(const lct_orthogonal &o) {
    return o.stride[2] != 1 && o.stride[1] == 1;
}

// The sum of squares of a part of a matrix, in FP64: of FP32's and BF16's largest, too.
__global__ __launch_bounds__(256) void norm_kernel(lct_orthogonal o, int32_t parts, double *out) {
    __shared__ double sums[4];
    const int32_t matrix = blockIdx.x / parts, part = blockIdx.x % parts;
    const int32_t across = (o.cols + kTile - 1) / kTile;
    const int64_t tiles = int64_t{(o.rows + kTile - 1) / kTile} * across;
    const bool turned = is_turned(o);
    double sum = 0.0;
    for (int64_t t = part; t < tiles; t += parts) {
        const int32_t i0 = static_cast<int32_t>(t / across) * kTile;
        const int32_t j0 = static_cast<int32_t>(t % across) * kTile;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int line = 32 * k + threadIdx.x / 8, chunk = threadIdx.x % 8 * 8;
            float v[8];
            eight(o, matrix, i0 + (turned ? chunk : line), j0 + (turned ? line : chunk), turned, v);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const double x = v[n];
                sum += x * x;
            }
        }
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, kWave);
    if (wave_lane() == 0) sums[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) out[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// X's second number of two adjacent values, whose first ones are `pair`.
__device__ __forceinline__ uint32_t rest(float x, float y, uint32_t pair) {
    return Half::round_pair((x - Half::low(pair)) * kHoldRest, (y - Half::high(pair)) * kHoldRest);
}

// 2^10 X of both numbers.
__device__ __forceinline__ float both(float first, float second) {
    return __builtin_fmaf(1.0f / kHoldRest, second, first);
}

// X from G, in rows of whole 16-byte pieces; zeros in what both dimensions are widened by.
__global__ __launch_bounds__(256) void start_kernel(lct_orthogonal o, int32_t parts,
                                                    const double *__restrict__ norms,
                                                    int32_t rows, int32_t cols, uint16_t *x,
                                                    uint16_t *x_rest) {
    __shared__ float tile[kTile][kTile + 1];
    __shared__ double sums[4];
    const int32_t across = (cols + kTile - 1) / kTile, down = (rows + kTile - 1) / kTile;
    const int32_t matrix = blockIdx.x / (across * down), t = blockIdx.x % (across * down);
    double sum = 0.0;
    for (int32_t k = threadIdx.x; k < parts; k += 256) sum += norms[int64_t{matrix} * parts + k];
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, kWave);
    if (wave_lane() == 0) sums[threadIdx.x / kWave] = sum;
    const int32_t i0 = t / across * kTile, j0 = t % across * kTile;
    const bool turned = is_turned(o);
    __syncthreads();
    const double inverse = 1.0 / (sqrt(sums[0] + sums[1] + sums[2] + sums[3]) + o.eps);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int line = 32 * k + threadIdx.x / 8, chunk = threadIdx.x % 8 * 8;
        float v[8];
        eight(o, matrix, i0 + (turned ? chunk : line), j0 + (turned ? line : chunk), turned, v);
#pragma unroll
        for (int n = 0; n < 8; ++n)
            tile[turned ? chunk + n : line][turned ? line : chunk + n] =
                static_cast<float>(v[n] * inverse);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = 32 * k + threadIdx.x / 8, j = threadIdx.x % 8 * 8;
        if (i0 + i >= rows || j0 + j >= cols) continue;
        u32x4 first, second;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float a = tile[i][j + 2 * n] * kHoldX, b = tile[i][j + 2 * n + 1] * kHoldX;
            first[n] = Half::round_pair(a, b);
            second[n] = rest(a, b, first[n]);
        }
        const int64_t at = (int64_t{matrix} * rows + i0 + i) * cols + j0 + j;
        *reinterpret_cast<u32x4 *>(x + at) = first;
        *reinterpret_cast<u32x4 *>(x_rest + at) = second;
    }
}

// scale X to an `out` of any strides.
__global__ __launch_bounds__(256) void finish_kernel(lct_orthogonal o, int32_t rows, int32_t cols,
                                                     const uint16_t *x, const uint16_t *x_rest) {
    __shared__ uint16_t tile[kTile][kTile + 2];
    const int32_t across = (o.cols + kTile - 1) / kTile, down = (o.rows + kTile - 1) / kTile;
    const int32_t matrix = blockIdx.x / (across * down), t = blockIdx.x % (across * down);
    const int32_t i0 = t / across * kTile, j0 = t % across * kTile;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = 32 * k + threadIdx.x / 8, j = threadIdx.x % 8 * 8;
        if (i0 + i >= rows || j0 + j >= cols) continue;
        const int64_t at = (int64_t{matrix} * rows + i0 + i) * cols + j0 + j;
        const u32x4 p = *reinterpret_cast<const u32x4 *>(x + at);
        const u32x4 q = *reinterpret_cast<const u32x4 *>(x_rest + at);
        const float factor = o.scale * (1.0f / kHoldX);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint32_t pair =
                Element<false>::round_pair(both(Half::low(p[n]), Half::low(q[n])) * factor,
                                           both(Half::high(p[n]), Half::high(q[n])) * factor);
            tile[i][j + 2 * n] = static_cast<uint16_t>(pair);
            tile[i][j + 2 * n + 1] = static_cast<uint16_t>(pair >> 16);
        }
    }
    __syncthreads();
    const bool turned = o.out_stride[2] != 1;
    for (int k = threadIdx.x / kTile; k < kTile; k += 4) {
        const int i = turned ? threadIdx.x % kTile : k, j = turned ? k : threadIdx.x % kTile;
        if (i0 + i < o.rows && j0 + j < o.cols)
            static_cast<uint16_t *>(o.out)[matrix * o.out_stride[0] + (i0 + i) * o.out_stride[1]
                                           + (j0 + j) * o.out_stride[2]] = tile[i][j];
    }
}

// ---- small matrices: all steps by one workgroup
//
// X as operand, A and P lie in LDS, X itself in FP32 in the registers that the update's
// products leave it in: a wave has 32 x 32 tiles of it, columns in a lane's registers.  Rows are
// 80 bytes off a multiple of 256, so that neither 16 rows' chunks nor 4 lines' 64 bytes meet
// in a clock of LDS.

constexpr int kSmallRows = LCT_ORTHOGONAL_SMALL_ROWS, kSmallCols = LCT_ORTHOGONAL_SMALL_COLS;
constexpr int kSmallPad = 40;

template <int kPitch>
__device__ __forceinline__ u32x4 small_rows(const uint16_t *from, int block, int step) {
    const int lane = wave_lane();
    return *reinterpret_cast<const u32x4 *>(from + (32 * block + (lane & 31)) * kPitch + 16 * step
                                            + 8 * (lane >> 5));
}

template <int kPitch>
__device__ __forceinline__ u32x4 small_columns(const uint16_t *from, int block, int step) {
    const int lane = wave_lane();
    const uint16_t *at = from + (16 * step + 8 * (lane >> 5) + ((lane & 15) >> 2)) * kPitch
                         + 32 * block + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4 *)(at));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4 *)(at + 4 * kPitch));
    const u32x2 lo = __builtin_bit_cast(u32x2, a), hi = __builtin_bit_cast(u32x2, b);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// A tile's four adjacent values of a lane, as FP16, to (row, column) of a matrix in LDS.
template <int kPitch>
__device__ __forceinline__ void small_store(uint16_t *to, int row_block, int column_block,
                                            const f32x16 &v, float factor) {
    uint16_t *at = to + (32 * row_block + (wave_lane() & 31)) * kPitch + 32 * column_block
                   + 4 * (wave_lane() >> 5);
#pragma unroll
    for (int g = 0; g < 4; ++g)
        *reinterpret_cast<u32x2 *>(at + 8 * g) =
            u32x2{Half::round_pair(v[4 * g] * factor, v[4 * g + 1] * factor),
                  Half::round_pair(v[4 * g + 2] * factor, v[4 * g + 3] * factor)};
}

// kTiles tiles, blocks `first` .. of the right operand's rows against the left one's fragments:
// the next step's are read while one is multiplied.
template <int kTiles, class Left, class Right>
__device__ __forceinline__ void small_product(f32x16 (&sum)[kTiles], int steps, Left left,
                                              Right right) {
    u32x4 a = left(0), b[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        sum[t] = f32x16{};
        b[t] = right(t, 0);
    }
    for (int k = 0; k < steps; ++k) {
        const int next = min(k + 1, steps - 1);
        const u32x4 next_a = left(next);
        u32x4 next_b[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) next_b[t] = right(t, next);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) sum[t] = Half::multiply(a, b[t], sum[t]);
        // (The reads stay in this round: the compiler would move them to their use.)
        a = next_a;
        asm volatile("" : "+v"(a));
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            b[t] = next_b[t];
            asm volatile("" : "+v"(b[t]));
        }
    }
}

template <int kRows, int kCols, int kWaves>
__global__ __launch_bounds__(kWaves *kWave) void small_kernel(lct_orthogonal o) {
    constexpr int kThreads = kWaves * kWave, kRowBlocks = kRows / 32;
    constexpr int kTiles = kRowBlocks * (kCols / 32) / kWaves;
    // (More waves than squares: the last have none.)
    constexpr int kSquares =
        kRowBlocks * kRowBlocks < kWaves ? 1 : kRowBlocks * kRowBlocks / kWaves;
    constexpr int kPitch = kCols + kSmallPad, kSquarePitch = kRows + kSmallPad;
    static_assert(kTiles <= kRowBlocks && kSquares <= kRowBlocks);
    // At the start, X's second number lies where A and P will.
    constexpr int kSquareValues = kRows * kSquarePitch;
    constexpr int kRest = kRows * kPitch > 2 * kSquareValues ? kRows * kPitch : 2 * kSquareValues;
    __shared__ __attribute__((aligned(16))) uint16_t operand[kRows * kPitch];
    __shared__ __attribute__((aligned(16))) uint16_t squares[kRest];
    __shared__ double sums[kWaves];
    uint16_t *const gram = squares, *const poly = squares + kSquareValues;
    const int lane = wave_lane();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int32_t matrix = blockIdx.x;
    // Blocks of 32 and steps of 16 that the matrices reach into.
    const int row_blocks = (o.rows + 31) / 32, column_blocks = (o.cols + 31) / 32;
    const int row_steps = (o.rows + 15) / 16, column_steps = (o.cols + 15) / 16;

    // X's place in the registers that it is loaded to: pieces of eight along the dimension
    // whose elements are adjacent.
    constexpr int kPieces = kRows * kCols / 8 / kThreads;
    float v[kPieces][8];
    const bool turned = is_turned(o);
    const auto place = [&](int k, auto by_rows, int *i, int *j) __attribute__((always_inline)) {
        constexpr int kAcross = decltype(by_rows)::value ? kRows / 8 : kCols / 8;
        const int slot = k * kThreads + threadIdx.x, line = slot / kAcross;
        const int chunk = slot % kAcross * 8;
        *i = decltype(by_rows)::value ? chunk : line;
        *j = decltype(by_rows)::value ? line : chunk;
    };
    const auto load = [&](auto by_rows) __attribute__((always_inline)) {
        load_eights<kPieces>(o, matrix, decltype(by_rows)::value, v,
                             [&](int k, int *i, int *j) { place(k, by_rows, i, j); });
    };
    if (turned) load(std::true_type{});
    else load(std::false_type{});
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kPieces; ++k)
#pragma unroll
        for (int n = 0; n < 8; ++n) sum += static_cast<double>(v[k][n]) * v[k][n];
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, kWave);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kWaves; ++w) sum += sums[w];
    const double inverse = 1.0 / (sqrt(sum) + o.eps);
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
        u32x4 first, second;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float a = static_cast<float>(v[k][2 * n] * inverse) * kHoldX;
            const float b = static_cast<float>(v[k][2 * n + 1] * inverse) * kHoldX;
            first[n] = Half::round_pair(a, b);
            second[n] = rest(a, b, first[n]);
        }
        int i, j;
        if (!turned) {
            place(k, std::false_type{}, &i, &j);
            *reinterpret_cast<u32x4 *>(operand + i * kPitch + j) = first;
            *reinterpret_cast<u32x4 *>(squares + i * kPitch + j) = second;
        } else {
            place(k, std::true_type{}, &i, &j);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int at = (i + n) * kPitch + j;
                operand[at] = static_cast<uint16_t>(first[n / 2] >> (n % 2 * 16));
                squares[at] = static_cast<uint16_t>(second[n / 2] >> (n % 2 * 16));
            }
        }
    }
    __syncthreads();

    // A wave's tiles are of one block of columns, whose fragment they share.
    const int column = wave * kTiles / kRowBlocks, first = wave * kTiles % kRowBlocks;
    const int square_column = wave * kSquares / kRowBlocks;
    const int square_first = wave * kSquares % kRowBlocks;
    const bool has = column < column_blocks;
    const bool has_square = square_column < row_blocks && square_first < row_blocks;
    f32x16 x[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        const int at = (32 * (first + t) + (lane & 31)) * kPitch + 32 * column + 4 * (lane >> 5);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const u32x2 p = *reinterpret_cast<const u32x2 *>(operand + at + 8 * g);
            const u32x2 q = *reinterpret_cast<const u32x2 *>(squares + at + 8 * g);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                x[t][4 * g + 2 * r] = both(Half::low(p[r]), Half::low(q[r])) * (1.0f / kHoldX);
                x[t][4 * g + 2 * r + 1] =
                    both(Half::high(p[r]), Half::high(q[r])) * (1.0f / kHoldX);
            }
        }
    }
    __syncthreads();

    for (int32_t s = 0; s < o.steps; ++s) {
        if (has_square) {
            f32x16 a[kSquares];
            small_product<kSquares>(
                a, column_steps,
                [&](int k) { return small_rows<kPitch>(operand, square_column, k); },
                [&](int t, int k) { return small_rows<kPitch>(operand, square_first + t, k); });
#pragma unroll
            for (int t = 0; t < kSquares; ++t)
                small_store<kSquarePitch>(gram, square_first + t, square_column, a[t],
                                          kHoldA / (kHoldX * kHoldX));
        }
        __syncthreads();
        if (has_square) {
            f32x16 p[kSquares];
            small_product<kSquares>(
                p, row_steps,
                [&](int k) { return small_rows<kSquarePitch>(gram, square_column, k); },
                [&](int t, int k) { return small_rows<kSquarePitch>(gram, square_first + t, k); });
#pragma unroll
            for (int t = 0; t < kSquares; ++t) {
                const uint16_t *own = gram + (32 * (square_first + t) + (lane & 31)) * kSquarePitch
                                      + 32 * square_column + 4 * (lane >> 5);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const u32x2 pairs = *reinterpret_cast<const u32x2 *>(own + 8 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        p[t][4 * g + r] = __builtin_fmaf(
                            kC / kHoldA, p[t][4 * g + r],
                            kB * (r % 2 ? Half::high(pairs[r / 2]) : Half::low(pairs[r / 2])));
                }
                small_store<kSquarePitch>(poly, square_first + t, square_column, p[t], 1.0f);
            }
        }
        __syncthreads();
        if (has) {
            f32x16 v[kTiles];
            small_product<kTiles>(
                v, row_steps, [&](int k) { return small_columns<kPitch>(operand, column, k); },
                [&](int t, int k) { return small_rows<kSquarePitch>(poly, first + t, k); });
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    x[t][r] = __builtin_fmaf(1.0f / (kHoldA * kHoldX), v[t][r], kA * x[t][r]);
        }
        __syncthreads();     // all have read the operand
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
            small_store<kPitch>(operand, first + t, column, x[t], kHoldX);
        __syncthreads();
    }

    // The result through LDS, to lie as it is written.
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        uint16_t *at = operand + (32 * (first + t) + (lane & 31)) * kPitch + 32 * column
                       + 4 * (lane >> 5);
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<u32x2 *>(at + 8 * g) =
                u32x2{Element<false>::round_pair(x[t][4 * g] * o.scale, x[t][4 * g + 1] * o.scale),
                      Element<false>::round_pair(x[t][4 * g + 2] * o.scale,
                                                 x[t][4 * g + 3] * o.scale)};
    }
    __syncthreads();
    auto *const out = static_cast<uint16_t *>(o.out) + matrix * o.out_stride[0];
    const bool out_turned = o.out_stride[2] != 1;
    const int64_t step = out_turned ? o.out_stride[1] : 1;
    const int64_t line_step = out_turned ? o.out_stride[2] : o.out_stride[1];
    const bool whole = step == 1 && line_step % 8 == 0 && o.out_stride[0] % 8 == 0
                       && reinterpret_cast<uintptr_t>(o.out) % 16 == 0;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
        int i, j;
        u32x4 of{};
        if (!out_turned) {
            place(k, std::false_type{}, &i, &j);
            of = *reinterpret_cast<const u32x4 *>(operand + i * kPitch + j);
        } else {
            place(k, std::true_type{}, &i, &j);
#pragma unroll
            for (int n = 0; n < 8; ++n)
                of[n / 2] |= static_cast<uint32_t>(operand[(i + n) * kPitch + j]) << (n % 2 * 16);
        }
        if (i >= o.rows || j >= o.cols) continue;
        uint16_t *to = out + i * o.out_stride[1] + j * o.out_stride[2];
        const int32_t left = out_turned ? o.rows - i : o.cols - j;
        if (whole && left >= 8) {
            *reinterpret_cast<u32x4 *>(to) = of;
        } else {
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (n < left) to[n * step] = static_cast<uint16_t>(of[n / 2] >> (n % 2 * 16));
        }
    }
}

// The smallest that holds the matrices.  Bound by the steps' order: three products, each with
// its barriers and its reads of LDS, of one compute unit.  Up to 256 of them run at once: 8 of
// 96 x 160, 5 steps, 30.6 us (of which 12 without a step), where the launches for larger
// matrices took 68; one of 64 x 64, 12 steps: 25 us.
void small(const lct_orthogonal &o, hipStream_t stream) {
    const uint32_t count = static_cast<uint32_t>(o.count);
    if (o.rows <= 64 && o.cols <= 64) small_kernel<64, 64, 4><<<count, 256, 0, stream>>>(o);
    else if (o.rows <= 64 && o.cols <= 128)
        small_kernel<64, 128, 4><<<count, 256, 0, stream>>>(o);
    else if (o.rows <= 64) small_kernel<64, 256, 8><<<count, 512, 0, stream>>>(o);
    else if (o.cols <= 128) small_kernel<128, 128, 8><<<count, 512, 0, stream>>>(o);
    else small_kernel<128, 256, 8><<<count, 512, 0, stream>>>(o);
}

// ---- products

// Tile t of the lower triangle's, row by row.
__device__ __forceinline__ void lower_tile(int32_t t, int32_t *i, int32_t *j) {
    int32_t row = static_cast<int32_t>(sqrtf(2.0f * static_cast<float>(t)));
    while (row * (row + 1) / 2 > t) --row;
    while ((row + 1) * (row + 2) / 2 <= t) ++row;
    *i = row;
    *j = t - row * (row + 1) / 2;
}

// out = factor L R + share (E + F): a symmetric product (of X and itself, or of two polynomials
// of one symmetric matrix, which commute) of operands by rows, and up to kMore of the
// matrices E and F.  `size`: rows of the result.
struct SymmetricTerms {
    const uint16_t *left, *right, *more[2];
    uint16_t *out;
    float factor, share;
};

// What becomes of tile (i, j)'s sums.
template <class P, int kMore>
__device__ __forceinline__ void finish_symmetric(P &p, const SymmetricTerms &s, int32_t matrix,
                                                 int32_t i, int32_t j, int32_t size,
                                                 uint16_t *mine) {
    const int32_t row = i * P::kM + p.first_row(), column = j * P::kN + p.first_column();
    const int64_t first = int64_t{matrix} * size * size;
#pragma unroll
    for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
        for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) p.sum[m][n][r] *= s.factor;
#pragma unroll
    for (int e = 0; e < kMore; ++e)
        // Its value at (row, column) is that at (column, row).
        load_columns<P>(s.more[e] + first + int64_t{column} * size + row, size, size - column,
                        size - row, mine,
                        [&](int m, int n, int r, uint32_t own) __attribute__((always_inline)) {
                            p.sum[m][n][r] =
                                __builtin_fmaf(s.share, Half::low(own), p.sum[m][n][r]);
                            p.sum[m][n][r + 1] =
                                __builtin_fmaf(s.share, Half::high(own), p.sum[m][n][r + 1]);
                        });
    const auto pair = [&](int m, int n, int r) __attribute__((always_inline)) {
        return Half::round_pair(p.sum[m][n][r], p.sum[m][n][r + 1]);
    };
    store_columns<P>(s.out + first + int64_t{column} * size + row, size, size - column, size - row,
                     mine, pair);
    if (i != j)
        store_rows<P>(s.out + first + int64_t{row} * size + column, size, size - row, size - column,
                      mine, pair);
}

// Tiles that run at once; the depth from which on the last of them, where they are at most
// half as many, are split; a part's least depth; parts (that symmetric_join_kernel loads at
// once).  us with 1 | 2 | 4 | 8 | 16 parts at most: 4096 x 11008 (528 tiles) 3203 | 2892 | 2777 |
// 2779 | 2804; 4096 x 4096 1707 | 1572 | 1520 | 1545 | 1546; 16 x 4096 x 1024 (576 tiles) 1424 |
// 1372 | 1359 | 1370 | 1371; 4 x 2048 x 8192 (544) 2304 | 2134 | 2077 | 2067 | 2106.
constexpr int32_t kSlots = 512, kSplitDepth = LCT_ORTHOGONAL_SPLIT_DEPTH, kPartDepth = 512;
constexpr int32_t kMostSplits = 4;

// The first `whole` tiles by a workgroup each, the others, which would leave most compute
// units without one, by `splits` of them with a part of the depth each: their sums go to
// `parts` as they lie in the registers, and symmetric_join_kernel goes on with them.
struct SymmetricShare {
    int32_t tiles, whole, splits;
    uint32_t whole_grid;
    f32x4 *parts;
};

template <class P>
constexpr int kPartPieces = P::kRowTiles * P::kColumnTiles * 4;

// Bound by the matrix instructions, and by what a tile's beginning and end cost beside few steps:
// 48 x 768 x 768 (1008 tiles of 128 x 128, 12 steps of 64) 42.5 us, 600 TFLOP/s over the 21 of 36
// tiles that are computed; 4096 x 4096 by 11008 212 us, 900.  One of 768 x 768 (78 tiles of 64 x
// 64): 6.4 us, the latency of 12 steps and of a launch.
template <class P, int kMore>
__global__ __launch_bounds__(P::kThreads, 2) void symmetric_kernel(SymmetricTerms s,
                                                                   SymmetricShare share,
                                                                   int32_t size, int32_t depth) {
    static_assert(P::kM == P::kN);
    LCT_PRODUCT_STAGES(P);
    int64_t item;
    int32_t begin = 0, end = depth;
    const bool part = blockIdx.x >= share.whole_grid;
    if (part) {
        const int32_t t = blockIdx.x - share.whole_grid;
        const int32_t per = ((depth + share.splits - 1) / share.splits + 63) / 64 * 64;
        item = share.whole + t / share.splits;
        begin = min(depth, t % share.splits * per);
        end = min(depth, begin + per);
    } else {
        item = xcd_item(share.whole, blockIdx.x);
        if (item >= share.whole) return;
    }
    const int32_t matrix = static_cast<int32_t>(item / share.tiles);
    int32_t i, j;
    lower_tile(static_cast<int32_t>(item % share.tiles), &i, &j);
    const int64_t of = int64_t{matrix} * size * depth + begin;
    typename P::A a;
    typename P::B b;
    a.prepare(s.left + of, depth, int64_t{i} * P::kM, size);
    b.prepare(s.right + of, depth, int64_t{j} * P::kN, size);
    P p;
    p.begin();
    p.run(a, b, end - begin, stage0, stage1, stage2, stage3);
    if (part) {
        f32x4 *to = share.parts
                    + int64_t{blockIdx.x - share.whole_grid} * kPartPieces<P> * P::kThreads
                    + threadIdx.x;
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int n = 0; n < P::kColumnTiles; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    to[((m * P::kColumnTiles + n) * 4 + g) * P::kThreads] =
                        f32x4{p.sum[m][n][4 * g], p.sum[m][n][4 * g + 1], p.sum[m][n][4 * g + 2],
                              p.sum[m][n][4 * g + 3]};
        return;
    }
    finish_symmetric<P, kMore>(p, s, matrix, i, j, size,
                               turn_values<P>(stage0, stage1, stage2, stage3));
}

// The parts of a tile, added in order.
template <class P, int kMore>
__global__ __launch_bounds__(P::kThreads, 1) void symmetric_join_kernel(SymmetricTerms s,
                                                                     SymmetricShare share,
                                                                     int32_t size) {
    __shared__ __attribute__((aligned(16))) uint16_t turn[P::kThreads / kWave * kTurnValues<P>];
    const int64_t item = share.whole + blockIdx.x;
    const int32_t matrix = static_cast<int32_t>(item / share.tiles);
    int32_t i, j;
    lower_tile(static_cast<int32_t>(item % share.tiles), &i, &j);
    P p;
    p.begin();
    // All parts' loads in flight together.
    constexpr int kPieces = kPartPieces<P>;
    const f32x4 *const from =
        share.parts + int64_t{blockIdx.x} * share.splits * kPieces * P::kThreads + threadIdx.x;
    f32x4 v[kMostSplits][kPieces];
#pragma unroll
    for (int k = 0; k < kMostSplits; ++k)
#pragma unroll
        for (int q = 0; q < kPieces; ++q)
            v[k][q] = from[(int64_t{min(k, share.splits - 1)} * kPieces + q) * P::kThreads];
#pragma unroll
    for (int k = 0; k < kMostSplits; ++k)
        if (k < share.splits)
#pragma unroll
            for (int q = 0; q < kPieces; ++q)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    p.sum[q / 4 / P::kColumnTiles][q / 4 % P::kColumnTiles][4 * (q % 4) + r] +=
                        v[k][q][r];
    finish_symmetric<P, kMore>(p, s, matrix, i, j, size, turn + P::wave() * kTurnValues<P>);
}

// X <- share X + S X: P::kM columns of X (rows of the tile) by P::kN rows of X (columns, a lane
// each).  The last step writes the result, scaled, in BF16 and G's orientation, if its
// rows are whole 16-byte pieces.
//
// Bound by the products and by X's way in and out (4 bytes a value each way, through LDS), which
// a tile's waves do one after the other: 48 x 768 x 768 82 to 84 us, 530 TFLOP/s; 4096 x 4096 by
// 11008 395 to 411 us, 935 to 900; 16 x 1024 x 4096 219 us, 620.
template <class P, bool kLast>
__global__ __launch_bounds__(P::kThreads, P::kThreads == 256 ? 2 : 1) void update_kernel(
    const uint16_t *poly, const uint16_t *x, int32_t count, int32_t rows, int32_t cols,
    int32_t row_tiles, int32_t column_tiles, float share, uint16_t *x_rest, uint16_t *next,
    lct_orthogonal o) {
    LCT_PRODUCT_STAGES(P);
    const int64_t tiles = int64_t{row_tiles} * column_tiles;
    const int64_t item = xcd_item(count * tiles, blockIdx.x);
    if (item >= count * tiles) return;
    const int32_t matrix = static_cast<int32_t>(item / tiles);
    const int32_t j = static_cast<int32_t>(item % tiles) / row_tiles;
    const int32_t i = static_cast<int32_t>(item % tiles) % row_tiles;
    const int64_t first = int64_t{matrix} * rows * cols;
    typename P::A a;
    typename P::B b;
    a.prepare(x + first, cols, int64_t{j} * P::kM, cols);
    b.prepare(poly + int64_t{matrix} * rows * rows, rows, int64_t{i} * P::kN, rows);
    P p;
    p.begin();
    p.run(a, b, rows, stage0, stage1, stage2, stage3);

    const int32_t column = j * P::kM + p.first_row(), row = i * P::kN + p.first_column();
    const int64_t at = first + int64_t{row} * cols + column;
    uint16_t *mine = turn_values<P>(stage0, stage1, stage2, stage3);
    // 2^10 X: the sums are 2^22 S X.
    load_columns<P>(x + at, cols, rows - row, cols - column, mine,
                    [&](int m, int n, int r, uint32_t old) __attribute__((always_inline)) {
                        p.sum[m][n][r] = __builtin_fmaf(1.0f / kHoldA, p.sum[m][n][r],
                                                        share * Half::low(old));
                        p.sum[m][n][r + 1] = __builtin_fmaf(1.0f / kHoldA, p.sum[m][n][r + 1],
                                                            share * Half::high(old));
                    });
    const float share_rest = share * (1.0f / kHoldRest);
    load_columns<P>(x_rest + at, cols, rows - row, cols - column, mine,
                    [&](int m, int n, int r, uint32_t old) __attribute__((always_inline)) {
                        p.sum[m][n][r] = __builtin_fmaf(share_rest, Half::low(old), p.sum[m][n][r]);
                        p.sum[m][n][r + 1] =
                            __builtin_fmaf(share_rest, Half::high(old), p.sum[m][n][r + 1]);
                    });
    if constexpr (kLast) {
        const float factor = o.scale * (1.0f / kHoldX);
        const auto pair = [&](int m, int n, int r) __attribute__((always_inline)) {
            return Element<false>::round_pair(p.sum[m][n][r] * factor, p.sum[m][n][r + 1] * factor);
        };
        uint16_t *out = static_cast<uint16_t *>(o.out) + matrix * o.out_stride[0];
        if (o.out_stride[2] == 1)
            store_columns<P>(out + row * o.out_stride[1] + column, o.out_stride[1], o.rows - row,
                             o.cols - column, mine, pair);
        else
            store_rows<P>(out + column * o.out_stride[2] + row, o.out_stride[2], o.cols - column,
                          o.rows - row, mine, pair);
    } else {
        store_columns<P>(next + at, cols, rows - row, cols - column, mine,
                         [&](int m, int n, int r) __attribute__((always_inline)) {
                             return Half::round_pair(p.sum[m][n][r], p.sum[m][n][r + 1]);
                         });
        store_columns<P>(x_rest + at, cols, rows - row, cols - column, mine,
                         [&](int m, int n, int r) __attribute__((always_inline)) {
                             const float u = p.sum[m][n][r], v = p.sum[m][n][r + 1];
                             return rest(u, v, Half::round_pair(u, v));
                         });
    }
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// ---- tiles, by how many there are for the 256 compute units
//
// us of 5 or 12 steps, with tiles of 64 x 64 | 128 x 128 (and, of the update, 256 x 128 | 256 x
// 256) in all products, two workgroups per compute unit but of the last.  The products by
// 128 x 128 have, of one 768 x 768, 21 lower tiles and 36 in the update: 110 | 185; of 3:
// 282 | 439; of 6 (126, 216): 405 with an update by 128 385 | 447; of 4 x 1024 x 1024 (144,
// 256): 234 | 238; of 12 x 768 x 768 (252, 432): 589 | 537 | 557; of 48 (1008, 1728): 2188
// | 1807 | 1779 | 1814; of 4096 x 4096 (528, 1024): 2380 | 1780 | 1698 | 1680; of 4096 x
// 11008: | 3347 | 3217 | 3112.
template <int kSize>
using Symmetric =
    Product<true, Lie::kRows, Lie::kRows, kSize, kSize, 2, 2, 64, kSize == 64 ? 4 : 2>;
template <int kM, int kN, int kWavesN, int kStep, int kStages>
using Update = Product<true, Lie::kColumns, Lie::kRows, kM, kN, 2, kWavesN, kStep, kStages>;
constexpr int64_t kFewTiles = 160, kManyTiles = 800;   // of 128 x 128
constexpr int32_t kLongDepth = 1024;

struct Iteration {
    int32_t count, rows, cols;
    uint16_t *x, *next, *x_rest, *square[3];
    hipStream_t stream;
    f32x4 *parts;

    // Tiles of 128 x 128.
    int64_t lower_tiles() const {
        const int64_t blocks = (rows + 127) / 128;
        return count * (blocks * (blocks + 1) / 2);
    }
    int64_t all_tiles() const {
        return count * int64_t{(rows + 127) / 128} * ((cols + 127) / 128);
    }

    template <int kSize, int kMore>
    void launch_symmetric(const SymmetricTerms &s, int32_t depth) const {
        using P = Symmetric<kSize>;
        const int32_t blocks = (rows + kSize - 1) / kSize, tiles = blocks * (blocks + 1) / 2;
        const int32_t all = count * tiles, rest = all % kSlots;
        SymmetricShare share{tiles, all, 1, 0, parts};
        if (kSize == 128 && depth >= kSplitDepth && rest > 0 && rest <= kSlots / 2) {
            share.whole = all - rest;
            share.splits = std::min(std::min(kSlots / rest, depth / kPartDepth), kMostSplits);
        }
        share.whole_grid = static_cast<uint32_t>(xcd_grid(share.whole));
        const int32_t split = all - share.whole;
        symmetric_kernel<P, kMore>
            <<<share.whole_grid + split * share.splits, P::kThreads, 0, stream>>>(s, share, rows,
                                                                                 depth);
        if constexpr (kSize == 128)
            if (split > 0)
                symmetric_join_kernel<P, kMore><<<split, P::kThreads, 0, stream>>>(s, share, rows);
    }
    void symmetric(const SymmetricTerms &s, int32_t depth) const {
        const auto with = [&](auto more) {
            if (lower_tiles() < kFewTiles) launch_symmetric<64, decltype(more)::value>(s, depth);
            else launch_symmetric<128, decltype(more)::value>(s, depth);
        };
        if (s.more[1] != nullptr) with(std::integral_constant<int, 2>{});
        else if (s.more[0] != nullptr) with(std::integral_constant<int, 1>{});
        else with(std::integral_constant<int, 0>{});
    }
    // out = A = X X^T.
    void gram(uint16_t *out) const {
        symmetric({x, x, {nullptr, nullptr}, out, kHoldA / (kHoldX * kHoldX), 0.0f}, cols);
    }
    // out = b A + c A A.
    void poly(const uint16_t *a, uint16_t *out) const {
        symmetric({a, a, {a, nullptr}, out, kC / kHoldA, kB}, rows);
    }
    // out = a (E + F) + L R.
    void sum(const uint16_t *l, const uint16_t *r, const uint16_t *e, const uint16_t *f,
             uint16_t *out) const {
        symmetric({l, r, {e, f}, out, 1.0f / kHoldA, kA}, rows);
    }
    template <class P, bool kLast>
    void launch_update(const uint16_t *s, float share, const lct_orthogonal &o) const {
        const int32_t row_tiles = (rows + P::kN - 1) / P::kN;
        const int32_t column_tiles = (cols + P::kM - 1) / P::kM;
        const int64_t items = int64_t{count} * row_tiles * column_tiles;
        update_kernel<P, kLast><<<static_cast<uint32_t>(xcd_grid(items)), P::kThreads, 0, stream>>>(
            s, x, count, rows, cols, row_tiles, column_tiles, share, x_rest, next, o);
    }
    // X <- share X + S X.
    void update(const uint16_t *s, float share, bool last, const lct_orthogonal &o) {
        const auto with = [&](auto which) {
            using P = typename decltype(which)::type;
            if (last) launch_update<P, true>(s, share, o);
            else launch_update<P, false>(s, share, o);
        };
        const int64_t tiles = all_tiles();
        if (tiles < kFewTiles) with(Type<Update<64, 64, 2, 64, 4>>{});
        else if (tiles < kManyTiles) with(Type<Update<128, 128, 2, 64, 2>>{});
        else if (rows < kLongDepth) with(Type<Update<256, 128, 2, 32, 3>>{});
        else with(Type<Update<256, 256, 4, 32, 4>>{});
        std::swap(x, next);
    }
    template <class T>
    struct Type {
        using type = T;
    };
};

}  // namespace
}  // namespace lct

using namespace lct;

extern "C" int32_t lct_orthogonalize(const lct_orthogonal *o, void *workspace,
                                     int64_t workspace_bytes, hipStream_t stream) {
    if (o == nullptr || o->input == nullptr || o->out == nullptr) return LCT_E_NULL;
    if (o->count < 1 || o->rows < 1 || o->cols < o->rows
        || o->cols > LCT_MAX_ORTHOGONAL_DIM || o->steps < 0)
        return LCT_E_SIZE;
    if (o->type < LCT_BF16 || o->type > LCT_FP32) return LCT_E_ARG;
    if (o->rows <= kSmallRows && o->cols <= kSmallCols) {
        if (o->count >= LCT_MAX_ORTHOGONAL_TILES) return LCT_E_SIZE;
        small(*o, stream);
        return static_cast<int32_t>(hipGetLastError());
    }
    if (workspace == nullptr) return LCT_E_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return LCT_E_ARG;
    const int64_t rows = up8(o->rows), cols = up8(o->cols), count = o->count;
    const int64_t values = count * rows * cols, square = count * rows * rows;
    const int64_t tiles = ((rows + 63) / 64) * ((cols + 63) / 64);
    // A launch has fewer than 2^32 threads; no product's tile is smaller than 64 x 64.
    if (count * tiles >= LCT_MAX_ORTHOGONAL_TILES) return LCT_E_SIZE;
    const int32_t parts =
        static_cast<int32_t>(std::min<int64_t>(LCT_ORTHOGONAL_NORM_PARTS, (tiles + 3) / 4));
    // Norms, X's first number as it is and to be, its second, and three square matrices.
    const int64_t norm_bytes = count * LCT_ORTHOGONAL_NORM_PARTS * 8;
    // (Parts of up to kSlots tiles.)
    const int64_t part_bytes = cols >= kSplitDepth ? LCT_ORTHOGONAL_SPLIT_BYTES : 0;
    if (workspace_bytes < norm_bytes + part_bytes + 6 * (values + square)) return LCT_E_SIZE;
    auto *norms = static_cast<double *>(workspace);
    char *const after = static_cast<char *>(workspace) + norm_bytes;
    auto *x = reinterpret_cast<uint16_t *>(after + part_bytes);
    uint16_t *const squares = x + 3 * values;
    Iteration it{static_cast<int32_t>(count),
                 static_cast<int32_t>(rows),
                 static_cast<int32_t>(cols),
                 x,
                 x + values,
                 x + 2 * values,
                 {squares, squares + square, squares + 2 * square},
                 stream,
                 reinterpret_cast<f32x4 *>(after)};
    norm_kernel<<<static_cast<uint32_t>(count * parts), 256, 0, stream>>>(*o, parts, norms);
    start_kernel<<<static_cast<uint32_t>(count * tiles), 256, 0, stream>>>(
        *o, parts, norms, it.rows, it.cols, it.x, it.x_rest);
    const int inner = o->out_stride[2] == 1 ? 2 : 1;
    const int64_t length = inner == 2 ? o->cols : o->rows, line = o->out_stride[3 - inner];
    // (A tile's lines are addressed by 32-bit byte offsets: finish_kernel has no such limit.)
    const bool whole = o->out_stride[inner] == 1 && length % 8 == 0 && line % 8 == 0
                       && line >= length && line <= LCT_MAX_ORTHOGONAL_DIM
                       && o->out_stride[0] % 8 == 0
                       && reinterpret_cast<uintptr_t>(o->out) % 16 == 0;
    // Two steps at once have 3 products with X, of rows^2 cols each, in place of 6 and 5 in
    // place of 2 of rows^3, the symmetric ones by half.  us of 12 or 5 steps one | two at a time:
    // 48 x 768 x 768 1765 | 1858; 16 x 4096 x 1024 1907 | 1409; 4096 x 11008 3955 | 3217; of few
    // tiles, which cost their launches, 768 x 768 138 | 138.
    const bool pairs = 2 * cols >= 3 * rows && it.all_tiles() >= kFewTiles;
    for (int32_t s = 0; s < o->steps;) {
        uint16_t *const m = it.square[0], *const p = it.square[1], *const r = it.square[2];
        it.gram(m);
        it.poly(m, p);
        if (pairs && s + 2 <= o->steps) {
            // Two steps at once, X <- (a + P') (a + P) X: the second's A' = (a + P) A (a + P).
            it.sum(p, m, m, nullptr, r);
            it.sum(p, r, r, nullptr, m);
            it.poly(m, r);
            it.sum(r, p, r, p, m);
            s += 2;
            it.update(m, kA * kA, s == o->steps && whole, *o);
        } else {
            s += 1;
            it.update(p, kA, s == o->steps && whole, *o);
        }
    }
    if (o->steps == 0 || !whole)
        finish_kernel<<<static_cast<uint32_t>(count * tiles), 256, 0, stream>>>(
            *o, it.rows, it.cols, it.x, it.x_rest);
    return static_cast<int32_t>(hipGetLastError());
}
