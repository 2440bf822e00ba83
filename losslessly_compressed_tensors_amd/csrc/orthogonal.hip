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
// X is kept in FP32, its operands, A and P in FP16 at fixed powers of two.  Small singular
// directions only double in the early steps.  What rounds X itself adds noise in all
// directions, and the steps that follow double that too: with X in 16 bits, 12
// steps of a matrix whose singular values fall off as 1/i end 0.1 (BF16) or 0.01 (FP16)
// of the norm away.  P X is small in the small directions on either side, so that
// rounding P's and X's operands there is harmless: 4e-4.  No value exceeds 1 by
// more than roundings, so FP16's range suffices and its three more bits are free.
#include <algorithm>

#include "product_core.h"

namespace lct {
namespace {

constexpr float kA = 2.0f, kB = -1.5f, kC = 0.5f;
// The operands' powers of two: X within 1 + 2^-8 (2^10 of 65504), A likewise, |P| <= 1.2.
constexpr float kHoldX = 1024.0f, kHoldA = 4096.0f;

using GramProduct = Product<true, Lie::kRows, Lie::kRows, 256, 128, 2, 2, 32, 3>;
using UpdateProduct = Product<true, Lie::kColumns, Lie::kRows, 256, 128, 2, 2, 32, 3>;

constexpr int kTile = 64;
constexpr int kMaxNormParts = LCT_ORTHOGONAL_NORM_PARTS;

__device__ __forceinline__ float element(const lct_orthogonal &o, int64_t at) {
    if (o.type == LCT_FP32) return static_cast<const float *>(o.input)[at];
    const uint16_t v = static_cast<const uint16_t *>(o.input)[at];
    return o.type == LCT_FP16 ? Element<true>::low(v) : Element<false>::low(v);
}

// A matrix's row i, column j as the wide orientation has them.
__device__ __forceinline__ int64_t place(const lct_orthogonal &o, int32_t matrix, int32_t i,
                                         int32_t j) {
    return matrix * o.stride[0] + i * o.stride[1] + j * o.stride[2];
}

// The sum of squares of a part of a matrix, in FP64: of FP32's and BF16's largest, too.
__global__ __launch_bounds__(256) void norm_kernel(lct_orthogonal o, int32_t parts, double *out) {
    __shared__ double sums[4];
    const int32_t matrix = blockIdx.x / parts, part = blockIdx.x % parts;
    const int32_t across = (o.cols + kTile - 1) / kTile;
    const int64_t tiles = int64_t{(o.rows + kTile - 1) / kTile} * across;
    // Lanes along the dimension whose elements are adjacent.
    const bool turned = o.stride[2] != 1 && o.stride[1] == 1;
    const int32_t x = threadIdx.x % kTile, y = threadIdx.x / kTile;
    double sum = 0.0;
    for (int64_t t = part; t < tiles; t += parts) {
        const int32_t i0 = static_cast<int32_t>(t / across) * kTile;
        const int32_t j0 = static_cast<int32_t>(t % across) * kTile;
        for (int32_t k = y; k < kTile; k += 4) {
            const int32_t i = i0 + (turned ? x : k), j = j0 + (turned ? k : x);
            if (i < o.rows && j < o.cols) {
                const double v = element(o, place(o, matrix, i, j));
                sum += v * v;
            }
        }
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, kWave);
    if (wave_lane() == 0) sums[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) out[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// X from G, in FP32 and as operand, in rows of whole 16-byte pieces; zeros in what both
// dimensions are widened by.
__global__ __launch_bounds__(256) void start_kernel(lct_orthogonal o, int32_t parts,
                                                    const double *__restrict__ norms,
                                                    int32_t rows, int32_t cols, float *x,
                                                    uint16_t *operand) {
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
    const bool turned = o.stride[2] != 1 && o.stride[1] == 1;
    const int32_t a = threadIdx.x % kTile, b = threadIdx.x / kTile;
    __syncthreads();
    const double inverse = 1.0 / (sqrt(sums[0] + sums[1] + sums[2] + sums[3]) + o.eps);
    for (int32_t k = b; k < kTile; k += 4) {
        const int32_t i = turned ? a : k, j = turned ? k : a;
        float v = 0.0f;
        if (i0 + i < o.rows && j0 + j < o.cols)
            v = static_cast<float>(element(o, place(o, matrix, i0 + i, j0 + j)) * inverse);
        tile[i][j] = v;
    }
    __syncthreads();
    for (int32_t k = b; k < kTile; k += 4) {
        if (i0 + k >= rows || j0 + a >= cols) continue;
        const int64_t at = (int64_t{matrix} * rows + i0 + k) * cols + j0 + a;
        const float v = tile[k][a];
        x[at] = v;
        operand[at] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v * kHoldX));
    }
}

// Tile `t` of those of a symmetric matrix that touch its lower triangle: 256 rows (block
// i) by 128 columns (block j <= 2 i + 1), i's 2 i + 2 tiles in turn.
__device__ __forceinline__ void lower_tile(int32_t t, int32_t *i, int32_t *j) {
    int32_t row = static_cast<int32_t>(sqrtf(static_cast<float>(t)));
    while (row * (row + 1) > t) --row;
    while ((row + 1) * (row + 2) <= t) ++row;
    *i = row;
    *j = t - row * (row + 1);
}
__host__ __device__ inline int32_t lower_tiles(int32_t rows) {
    const int32_t down = (rows + 255) / 256;
    // The last block's second column block may be past the end.
    return down * (down + 1) - ((rows + 127) / 128 < 2 * down ? 1 : 0);
}

// A symmetric product of an operand by rows with itself: A (kPoly false; from X) or P
// (from A).  `size`: rows of the result.
template <bool kPoly>
__global__ __launch_bounds__(256, 2) void symmetric_kernel(const uint16_t *operand, int32_t count,
                                                           int32_t size, int32_t depth,
                                                           int32_t tiles, uint16_t *out) {
    using P = GramProduct;
    LCT_PRODUCT_STAGES(P);
    const int64_t item = xcd_item(int64_t{count} * tiles, blockIdx.x);
    if (item >= int64_t{count} * tiles) return;
    const int32_t matrix = static_cast<int32_t>(item / tiles);
    int32_t i, j;
    lower_tile(static_cast<int32_t>(item % tiles), &i, &j);
    const uint16_t *from = operand + int64_t{matrix} * size * depth;
    out += int64_t{matrix} * size * size;
    P::A a;
    P::B b;
    a.prepare(from, depth, int64_t{i} * P::kM, size);
    b.prepare(from, depth, int64_t{j} * P::kN, size);
    P p;
    p.begin();
    p.run(a, b, depth, stage0, stage1, stage2, stage3);

    const int lane = wave_lane(), half = lane >> 5;
    // A block on the diagonal is computed whole, by its two tiles.
    const bool mirror = j < 2 * i;
#pragma unroll
    for (int n = 0; n < P::kColumnTiles; ++n) {
        const int32_t column = j * P::kN + p.first_column() + 32 * n + (lane & 31);
        if (column >= size) continue;
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int32_t row = i * P::kM + p.first_row() + 32 * m + 8 * g + 4 * half;
                if (row >= size) continue;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = p.sum[m][n][4 * g + r];
                if constexpr (kPoly) {
                    const u32x2 own =
                        *reinterpret_cast<const u32x2 *>(from + int64_t{column} * depth + row);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float of = r % 2 ? Element<true>::high(own[r / 2])
                                               : Element<true>::low(own[r / 2]);
                        v[r] = __builtin_fmaf(kC / kHoldA, v[r], kB * of);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] *= kHoldA / (kHoldX * kHoldX);
                }
                const u32x2 pairs = {Element<true>::round_pair(v[0], v[1]),
                                     Element<true>::round_pair(v[2], v[3])};
                *reinterpret_cast<u32x2 *>(out + int64_t{column} * size + row) = pairs;
                if (mirror) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        out[int64_t{row + r} * size + column] =
                            static_cast<uint16_t>(pairs[r / 2] >> (r % 2 * 16));
                }
            }
    }
}

// X <- a X + P X: 256 columns of X (rows of the tile) by 128 rows of X (columns, a lane
// each).  The last step writes the result, scaled, in BF16 and G's orientation.
template <bool kLast>
__global__ __launch_bounds__(256, 2) void update_kernel(const uint16_t *poly,
                                                        const uint16_t *operand, int32_t count,
                                                        int32_t rows, int32_t cols,
                                                        int32_t row_tiles, int32_t column_tiles,
                                                        float *x, uint16_t *next, float scale,
                                                        lct_orthogonal o) {
    using P = UpdateProduct;
    LCT_PRODUCT_STAGES(P);
    const int64_t tiles = int64_t{row_tiles} * column_tiles;
    const int64_t item = xcd_item(count * tiles, blockIdx.x);
    if (item >= count * tiles) return;
    const int32_t matrix = static_cast<int32_t>(item / tiles);
    const int32_t j = static_cast<int32_t>(item % tiles) / row_tiles;
    const int32_t i = static_cast<int32_t>(item % tiles) % row_tiles;
    const int64_t first = int64_t{matrix} * rows * cols;
    P::A a;
    P::B b;
    a.prepare(operand + first, cols, int64_t{j} * P::kM, cols);
    b.prepare(poly + int64_t{matrix} * rows * rows, rows, int64_t{i} * P::kN, rows);
    P p;
    p.begin();
    p.run(a, b, rows, stage0, stage1, stage2, stage3);

    const int lane = wave_lane(), half = lane >> 5;
#pragma unroll
    for (int n = 0; n < P::kColumnTiles; ++n) {
        const int32_t row = i * P::kN + p.first_column() + 32 * n + (lane & 31);
        if (row >= rows) continue;
#pragma unroll
        for (int m = 0; m < P::kRowTiles; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int32_t column = j * P::kM + p.first_row() + 32 * m + 8 * g + 4 * half;
                if (column >= cols) continue;
                const int64_t at = first + int64_t{row} * cols + column;
                const f32x4 old = *reinterpret_cast<const f32x4 *>(x + at);
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    v[r] = __builtin_fmaf(1.0f / (kHoldA * kHoldX), p.sum[m][n][4 * g + r],
                                          kA * old[r]);
                if constexpr (kLast) {
                    if (row >= o.rows) continue;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (column + r < o.cols)
                            static_cast<uint16_t *>(o.out)[matrix * o.out_stride[0]
                                                           + row * o.out_stride[1]
                                                           + (column + r) * o.out_stride[2]] =
                                static_cast<uint16_t>(
                                    Element<false>::round_pair(v[r] * scale, 0.0f));
                } else {
                    *reinterpret_cast<f32x4 *>(x + at) = v;
                    *reinterpret_cast<u32x2 *>(next + at) =
                        u32x2{Element<true>::round_pair(v[0] * kHoldX, v[1] * kHoldX),
                              Element<true>::round_pair(v[2] * kHoldX, v[3] * kHoldX)};
                }
            }
    }
}

// No steps: the scaled start.
__global__ __launch_bounds__(256) void copy_kernel(lct_orthogonal o, int32_t rows, int32_t cols,
                                                   const float *x) {
    const int64_t all = int64_t{o.count} * o.rows * o.cols;
    for (int64_t at = int64_t{blockIdx.x} * 256 + threadIdx.x; at < all;
         at += int64_t{gridDim.x} * 256) {
        const int32_t j = static_cast<int32_t>(at % o.cols);
        const int64_t rest = at / o.cols;
        const int32_t i = static_cast<int32_t>(rest % o.rows);
        const int64_t matrix = rest / o.rows;
        static_cast<uint16_t *>(o.out)[matrix * o.out_stride[0] + i * o.out_stride[1]
                                       + j * o.out_stride[2]] =
            static_cast<uint16_t>(Element<false>::round_pair(
                x[(matrix * rows + i) * cols + j] * o.scale, 0.0f));
    }
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

}  // namespace
}  // namespace lct

using namespace lct;

extern "C" int32_t lct_orthogonalize(const lct_orthogonal *o, void *workspace,
                                     int64_t workspace_bytes, hipStream_t stream) {
    if (o == nullptr || o->input == nullptr || o->out == nullptr || workspace == nullptr)
        return LCT_E_NULL;
    if (o->count < 1 || o->rows < 1 || o->cols < o->rows
        || o->cols > LCT_MAX_ORTHOGONAL_DIM || o->steps < 0)
        return LCT_E_SIZE;
    if (o->type < LCT_BF16 || o->type > LCT_FP32 || reinterpret_cast<uintptr_t>(workspace) % 16)
        return LCT_E_ARG;
    const int64_t rows = up8(o->rows), cols = up8(o->cols), count = o->count;
    const int64_t values = count * rows * cols, square = count * rows * rows;
    const int32_t tiles64 =
        static_cast<int32_t>(((o->rows + 63) / 64) * int64_t{(o->cols + 63) / 64});
    const int32_t parts = std::min(kMaxNormParts, (tiles64 + 3) / 4);
    const int64_t starts = count * ((rows + 63) / 64) * ((cols + 63) / 64);
    const int64_t updates = count * ((rows + 127) / 128) * ((cols + 255) / 256);
    const int32_t lower = lower_tiles(static_cast<int32_t>(rows));
    if (starts >= 1 << 23 || updates >= 1 << 23 || count * lower >= 1 << 23) return LCT_E_SIZE;
    // Norms, X, two operands of X, A and P.
    const int64_t norm_bytes = (count * kMaxNormParts * 8 + 15) / 16 * 16;
    if (workspace_bytes < norm_bytes + values * 8 + square * 4) return LCT_E_SIZE;
    auto *norms = static_cast<double *>(workspace);
    auto *x = reinterpret_cast<float *>(static_cast<char *>(workspace) + norm_bytes);
    auto *operand = reinterpret_cast<uint16_t *>(x + values);
    uint16_t *next = operand + values, *gram = next + values, *poly = gram + square;

    norm_kernel<<<static_cast<uint32_t>(count * parts), 256, 0, stream>>>(*o, parts, norms);
    start_kernel<<<static_cast<uint32_t>(starts), 256, 0, stream>>>(
        *o, parts, norms, static_cast<int32_t>(rows), static_cast<int32_t>(cols), x, operand);
    if (o->steps == 0)
        copy_kernel<<<1024, 256, 0, stream>>>(*o, static_cast<int32_t>(rows),
                                              static_cast<int32_t>(cols), x);
    const int32_t r = static_cast<int32_t>(rows), c = static_cast<int32_t>(cols);
    const int32_t n = static_cast<int32_t>(count);
    for (int32_t s = 0; s < o->steps; ++s) {
        const uint32_t half = static_cast<uint32_t>(xcd_grid(count * lower));
        symmetric_kernel<false><<<half, 256, 0, stream>>>(operand, n, r, c, lower, gram);
        symmetric_kernel<true><<<half, 256, 0, stream>>>(gram, n, r, r, lower, poly);
        const uint32_t grid = static_cast<uint32_t>(xcd_grid(updates));
        if (s + 1 < o->steps)
            update_kernel<false><<<grid, 256, 0, stream>>>(poly, operand, n, r, c, (r + 127) / 128,
                                                           (c + 255) / 256, x, next, o->scale, *o);
        else
            update_kernel<true><<<grid, 256, 0, stream>>>(poly, operand, n, r, c, (r + 127) / 128,
                                                          (c + 255) / 256, x, next, o->scale, *o);
        std::swap(operand, next);
    }
    return static_cast<int32_t>(hipGetLastError());
}
