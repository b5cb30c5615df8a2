// Softmax cross entropy of a linear layer's logits that are never kept.
//
// For each row t of x [rows, width], with z = x W + b [classes]:
//   loss_t = log(sum_v exp(z_v)) - z_target,
//   dz_v   = share_t (exp(z_v) / sum - [v = target]),
//   dx = dz W^T, dW = x^T dz, db = the sum over rows of dz.
// A row whose target is no class number is left out: its loss and its part of
// every gradient are zero, whatever x holds there. The share of a row is its
// upstream gradient, or one over the number of rows that count (the mean loss).
//
// Rows are taken in pieces: the logits of a piece live in a workspace until
// their gradients are used.
#include "halves_product.hpp"
#include "reduce_common.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>

namespace vchip {
namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kLowest = -__builtin_huge_valf();

// The class a target names, or -1.
__device__ inline int64_t class_of(float target, int64_t classes) {
    if (!(target >= 0.0f && target < float(classes))) return -1;
    const int64_t c = int64_t(target);
    return float(c) == target ? c : -1;
}

constexpr int kCountThreads = 1024;

// share[0] = one over the number of rows that count, or zero.
__global__ __launch_bounds__(kCountThreads) void count_kernel(const float* __restrict__ targets, int64_t rows, int64_t classes,
                                                              float* __restrict__ share) {
    __shared__ double lds[kCountThreads / 64];
    double n = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += kCountThreads) n += class_of(targets[r], classes) >= 0 ? 1.0 : 0.0;
    n = red::block_sum(n, lds);
    if (threadIdx.x == 0) share[0] = n > 0.0 ? float(1.0 / n) : 0.0f;
}

// mean[0] = share[0] times the sum of the losses.
__global__ __launch_bounds__(kCountThreads) void mean_kernel(const float* __restrict__ losses, int64_t rows,
                                                             const float* __restrict__ share, float* __restrict__ mean) {
    __shared__ double lds[kCountThreads / 64];
    double s = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += kCountThreads) s += double(losses[r]);
    s = red::block_sum(s, lds);
    if (threadIdx.x == 0) mean[0] = float(s * double(share[0]));
}

// A copy of x whose left out rows are zeros: zero times what they hold would not be zero for an infinity or a NaN.
__global__ __launch_bounds__(256) void counted_rows_kernel(const float* __restrict__ x, const float* __restrict__ targets,
                                                           float* __restrict__ out, int64_t rows, int64_t width,
                                                           int64_t classes) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const bool counted = class_of(targets[r], classes) >= 0;
        for (int64_t c = threadIdx.x; c < width; c += 256) out[r * width + c] = counted ? x[r * width + c] : 0.0f;
    }
}

constexpr int kRowThreads = 256;

__device__ inline float workgroup_max(float v, float* lds) {
    const int lane = red::lane_id();
    const auto larger = [](float a, float b) { return fmaxf(a, b); };
    v = larger(v, red::partner<0>(v, lane));
    v = larger(v, red::partner<1>(v, lane));
    v = larger(v, red::partner<2>(v, lane));
    v = larger(v, red::partner<3>(v, lane));
    v = larger(v, red::partner<4>(v, lane));
    v = larger(v, red::partner<5>(v, lane));
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    float m = lds[0];
    for (int w = 1; w < kRowThreads / 64; ++w) m = fmaxf(m, lds[w]);
    return m;
}

// A workgroup a row: its loss from the logits z (without the bias), and, where Gradient, z becomes dz.
template <bool Gradient>
__global__ __launch_bounds__(kRowThreads) void logits_kernel(float* __restrict__ z, const float* __restrict__ bias,
                                                             const float* __restrict__ targets, const float* __restrict__ shares,
                                                             bool one_share, int64_t rows, int64_t classes,
                                                             float* __restrict__ losses) {
    __shared__ double sums[kRowThreads / 64];
    __shared__ float most[kRowThreads / 64];
    __shared__ double total_of_row;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        __syncthreads();
        float* const row = z + r * classes;
        const int64_t target = class_of(targets[r], classes);
        if (target < 0) {
            if (losses && threadIdx.x == 0) losses[r] = 0.0f;
            if constexpr (Gradient)
                for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) row[c] = 0.0f;
            continue;
        }
        const auto value = [&](int64_t c) { return bias ? row[c] + bias[c] : row[c]; };
        float m = kLowest;
        for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) m = fmaxf(m, value(c));
        m = workgroup_max(m, most);
        double s = 0.0;
        for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) s += double(expf(value(c) - m));
        s = red::block_sum(s, sums);
        if (threadIdx.x == 0) total_of_row = s;
        __syncthreads();
        s = total_of_row;
        const float at = value(target) - m;
        if (losses && threadIdx.x == 0) losses[r] = float(log(s) - double(at));
        if constexpr (Gradient) {
            const float share = one_share ? shares[0] : shares[r], scale = float(double(share) / s);
            const double own = double(expf(at));
            __syncthreads();  // every thread has read the target's logit
            for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) {
                const float e = expf(value(c) - m);
                // The others' sum in double: one minus a share near one would leave no bits.
                row[c] = c == target ? float(-double(share) * ((s - own) / s)) : e * scale;
            }
        }
    }
}


// ---- large products: packed halves -----------------------------------------------------
//
// The three products of a piece read packed operands (halves_product.hpp), each made once:
//   z^T = W^T x^T  from the columns of W and the rows of x, along the features,
//   dx  = dz W^T   from the rows of dz and of W, along the classes,
//   dW  = x^T dz   from the columns of x and of dz, along the rows of the piece.
// The logits are made transposed: a thread of the product then holds 64 classes of a token, whose maximum and sum need no
// exchange but one, and the largest gradient of a class is that of a row in memory.

using halves::half;
using halves::h8;

constexpr int kPackThreads = 256, kPackRows = 32, kPackColumns = 128;
constexpr float kLog2e = 1.44269504f;

__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A matrix of floats whose left out rows are zeros.
struct Plain {
    const float* values;
    const float* targets;  // null: every row counts
    int64_t rows, columns, classes;
    const uint32_t *row_most, *column_most;  // the largest magnitudes, as bits
    __device__ inline bool row_counts(int64_t r) const { return r < rows && (!targets || class_of(targets[r], classes) >= 0); }
    // Eight values of a row from column c, a multiple of eight.
    __device__ inline void load(int64_t r, bool counts, int64_t c, float (&v)[8]) const {
        const float* const at = values + r * columns + c;
        if (counts && c + 8 <= columns) {
            const f4u lo = *reinterpret_cast<const f4u*>(at), hi = *reinterpret_cast<const f4u*>(at + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = lo[i];
                v[4 + i] = hi[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = counts && c + i < columns ? at[i] : 0.0f;
        }
    }
    struct Columns {
        __device__ inline float along_row(float v, int) const { return v; }
    };
    __device__ inline Columns hold(int64_t) const { return {}; }
    __device__ inline void load(int64_t r, bool counts, int64_t c, const Columns&, float (&v)[8]) const { load(r, counts, c, v); }
    __device__ inline uint32_t row_bits(int64_t r) const { return r < rows ? row_most[r] : 0u; }
    __device__ inline uint32_t column_bits(int64_t c) const { return c < columns ? column_most[c] : 0u; }
};

// What a token's gradients are made of, from its logits' statistics.
struct Token {
    float most, scale;  // exp(z - most) * scale is the share of a class
    float others;       // the share of all classes but the target's, which is minus the target's gradient
    int target;         // -1: left out
};

// dz^T [classes, tokens], for shares of one, of the logits z^T. Along a class (a row) times the tokens' shares.
struct Gradients {
    const float* logits;
    int64_t stride;
    const Token* tokens;
    const float* shares;
    bool one_share;
    int64_t rows, columns;  // classes, tokens
    const uint32_t* row_most;
    __device__ inline bool row_counts(int64_t r) const { return r < rows; }
    static __device__ inline float of(float z, int64_t r, const Token& t) {
        if (t.target < 0) return 0.0f;
        return t.target == int(r) ? -t.others : exp_of(z - t.most) * t.scale;
    }
    struct Columns {
        Token token[8];
        float share[8];
        __device__ inline float along_row(float v, int i) const { return v * share[i]; }
    };
    __device__ inline Columns hold(int64_t c) const {
        Columns held;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            held.token[i] = c + i < columns ? tokens[c + i] : Token{0.0f, 0.0f, 0.0f, -1};
            held.share[i] = held.token[i].target < 0 ? 0.0f : shares[one_share ? 0 : c + i];
        }
        return held;
    }
    // The stride is a multiple of 256, and whole rows are there to read.
    __device__ inline void load(int64_t r, bool counts, int64_t c, const Columns& held, float (&v)[8]) const {
        const float* const at = logits + r * stride + c;
        const red::f4 none{0.0f, 0.0f, 0.0f, 0.0f}, lo = counts ? red::ld4(at) : none, hi = counts ? red::ld4(at + 4) : none;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = counts ? of(i < 4 ? lo[i % 4] : hi[i % 4], r, held.token[i]) : 0.0f;
    }
    __device__ inline uint32_t row_bits(int64_t r) const { return r < rows ? row_most[r] : 0u; }
    __device__ inline uint32_t column_bits(int64_t c) const {
        return c < columns ? __builtin_bit_cast(uint32_t, tokens[c].others) : 0u;
    }
};

// Packs a matrix by its rows (along columns, row_lines a row) and by its columns (along rows, column_lines a column); either may
// be null. A workgroup takes 32 rows and 128 columns, past the ends zeros.
template <class Source>
__global__ __launch_bounds__(kPackThreads) void pack_kernel(Source from, half* __restrict__ by_row, int row_lines,
                                                            half* __restrict__ by_column, int column_lines, int across) {
    __shared__ float tile[kPackRows][kPackColumns + 4];
    const int64_t block = block_id();
    const int64_t row0 = block / across * kPackRows, column0 = block % across * kPackColumns;
    // Sixteen threads read 512 neighbouring bytes of a row.
    const int c = 8 * (threadIdx.x % 16);
    const int64_t column = column0 + c;
    const auto held = from.hold(column);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = threadIdx.x / 16 + 16 * j;
        const int64_t row = row0 + r;
        float v[8], scaled[8];
        from.load(row, from.row_counts(row), column, held, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            tile[r][c + i] = v[i];
            scaled[i] = held.along_row(v[i], i);
        }
        if (by_row && column / 32 < row_lines) {
            h8 first, second;
            halves::split8(scaled, halves::exponent_of(from.row_bits(row)), first, second);
            half* const to = by_row + (row * row_lines + column / 32) * 64 + column % 32 * 2;
            *reinterpret_cast<h8*>(to) = first;
            *reinterpret_cast<h8*>(to + 8) = second;
        }
    }
    if (!by_column) return;
    __syncthreads();
    const int64_t line = row0 / 32;
    if (line >= column_lines) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int at = threadIdx.x / 4 + 64 * j, g = threadIdx.x % 4;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[8 * g + i][at];
        h8 first, second;
        halves::split8(v, halves::exponent_of(from.column_bits(column0 + at)), first, second);
        half* const to = by_column + ((column0 + at) * column_lines + line) * 64 + 16 * g;
        *reinterpret_cast<h8*>(to) = first;
        *reinterpret_cast<h8*>(to + 8) = second;
    }
}

constexpr int kMostRows = 64, kMostColumns = 256;

// The largest finite magnitudes of a matrix's rows and columns, as bits, into arrays of zeros: bits of positive floats are
// ordered as the floats are, so the order of the atomics does not matter. A workgroup takes 64 rows and 256 columns.
__global__ __launch_bounds__(256) void most_kernel(const float* __restrict__ values, const float* __restrict__ targets,
                                                   int64_t rows, int64_t columns, int64_t classes, int across,
                                                   uint32_t* __restrict__ row_most, uint32_t* __restrict__ column_most) {
    __shared__ uint32_t of_column[4][kMostColumns];
    const int64_t block = block_id();
    const int64_t row0 = block / across * kMostRows, column0 = block % across * kMostColumns;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = column0 + 4 * lane;
    uint32_t most[4] = {0, 0, 0, 0};
    for (int j = 0; j < kMostRows / 4; ++j) {
        const int64_t r = row0 + wave + 4 * j;
        if (r >= rows) break;  // the same in the whole wavefront
        if (targets && class_of(targets[r], classes) < 0) continue;
        uint32_t row = 0;
        f4u v{0.0f, 0.0f, 0.0f, 0.0f};
        if (c + 4 <= columns) {
            v = *reinterpret_cast<const f4u*>(values + r * columns + c);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = c + e < columns ? values[r * columns + c + e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t bits = __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu;
            bits = bits < 0x7F800000u ? bits : 0u;
            most[e] = max(most[e], bits);
            row = max(row, bits);
        }
        if (row_most) {
            row = max(row, red::partner<0>(row, lane));
            row = max(row, red::partner<1>(row, lane));
            row = max(row, red::partner<2>(row, lane));
            row = max(row, red::partner<3>(row, lane));
            row = max(row, red::partner<4>(row, lane));
            row = max(row, red::partner<5>(row, lane));
            if (lane == 0) atomicMax(&row_most[r], row);
        }
    }
    if (!column_most) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) of_column[wave][4 * lane + e] = most[e];
    __syncthreads();
    const int64_t column = column0 + threadIdx.x;
    uint32_t all = of_column[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < 4; ++w) all = max(all, of_column[w][threadIdx.x]);
    if (column < columns && all) atomicMax(&column_most[column], all);
}

// The largest |dz share| of each class, as bits, into zeros; and, where Sums, of every 512 tokens the class's sum of them, into
// sums [token groups][classes]. A wavefront holds 512 tokens and takes 16 classes. The largest without its exponential: of
// the exponents' maximum one is taken at the end.
constexpr int kGroupTokens = 512, kGroupClasses = 16;
template <bool Sums>
__global__ __launch_bounds__(64) void class_most_kernel(Gradients from, uint32_t* __restrict__ most, double* __restrict__ sums,
                                                        int groups) {
    const int lane = threadIdx.x;
    const int64_t block = block_id(), group = block % groups;
    const int64_t c0 = group * kGroupTokens + 8 * lane, v0 = block / groups * kGroupClasses;
    const bool inside = c0 < from.stride;
    const Gradients::Columns held = from.hold(c0);
    float offset[8], own[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float share = __builtin_amdgcn_logf(fabsf(held.share[i]));
        offset[i] = __builtin_amdgcn_logf(held.token[i].scale) + share;
        own[i] = __builtin_amdgcn_logf(held.token[i].others) + share;
    }
    for (int k = 0; k < kGroupClasses; ++k) {
        const int64_t v = v0 + k;
        if (v >= from.rows) break;
        const float* const at = from.logits + v * from.stride + c0;
        const red::f4 none{0.0f, 0.0f, 0.0f, 0.0f}, lo = inside ? red::ld4(at) : none, hi = inside ? red::ld4(at + 4) : none;
        float top = kLowest;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = i < 4 ? lo[i % 4] : hi[i % 4];
            const Token& t = held.token[i];
            if (t.target >= 0) top = fmaxf(top, t.target == int(v) ? own[i] : __builtin_fmaf(z - t.most, kLog2e, offset[i]));
            if constexpr (Sums) sum += double(Gradients::of(z, v, t) * held.share[i]);
        }
        top = fmaxf(top, red::partner<0>(top, lane));
        top = fmaxf(top, red::partner<1>(top, lane));
        top = fmaxf(top, red::partner<2>(top, lane));
        top = fmaxf(top, red::partner<3>(top, lane));
        top = fmaxf(top, red::partner<4>(top, lane));
        top = fmaxf(top, red::partner<5>(top, lane));
        if constexpr (Sums) sum = red::wave_sum(sum);
        if (lane == 0) {
            const uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_amdgcn_exp2f(top));
            if (bits && bits < 0x7F800000u) atomicMax(&most[v], bits);
            if constexpr (Sums) sums[group * from.rows + v] = sum;
        }
    }
}

// ---- the products -----------------------------------------------------------------------

// z^T: scaled back, with the bias, stored if wanted; and of each 128 classes of a token the maximum, the sum of the exponentials
// over it, and the target's logit.
struct Logits {
    const uint32_t *class_most, *token_most;
    const float *bias, *targets;
    float *out, *most, *sum, *at_target;
    int64_t classes, tokens, stride;
    __device__ inline void operator()(halves::Tile& tile, int m, int n) const {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        const int64_t v0 = int64_t(m) * halves::kTile, t0 = int64_t(n) * halves::kTile + 64 * (wave % 4) + lane % 32;
        const int left = int(min(classes - v0, int64_t(halves::kTile)));  // classes of this tile
        const int row0 = 128 * (wave / 4) + 4 * (lane / 32);
        float top[2], others[2];
        int e_token[2], target[2];  // the target's row in this tile
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            top[b] = kLowest;
            others[b] = 0.0f;
            const int64_t t = t0 + 32 * b;
            e_token[b] = t < tokens ? halves::exponent_of(token_most[t]) : 0;
            const int64_t own = t < tokens ? class_of(targets[t], classes) - v0 : -1;
            target[b] = own >= 0 && own < halves::kTile ? int(own) : -1;
        }
        const uint32_t* bits = class_most + v0 + row0;  // padded to whole tiles
        const float* of_bias = bias + v0 + row0;
        float* to = out + (v0 + row0) * stride + t0;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            int e[16];
            // Of 32 rows at a time: the addresses and exponents of all do not fit the registers.
            asm volatile("" : "+v"(bits), "+v"(to), "+v"(of_bias));
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint4 of = *reinterpret_cast<const uint4*>(bits + 8 * g);
                e[4 * g] = halves::exponent_of(of.x);
                e[4 * g + 1] = halves::exponent_of(of.y);
                e[4 * g + 2] = halves::exponent_of(of.z);
                e[4 * g + 3] = halves::exponent_of(of.w);
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float z[16], high = top[b];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = row0 + 32 * a + 8 * (i / 4) + i % 4;
                    z[i] = __builtin_amdgcn_ldexpf(tile.acc[a][b][i], -(e[i] + e_token[b]));
                    if (r < left) {
                        if (bias) z[i] += of_bias[8 * (i / 4) + i % 4];
                        if (out) to[(8 * (i / 4) + i % 4) * stride + 32 * b] = z[i];
                        if (r == target[b]) at_target[t0 + 32 * b] = z[i];
                    } else {
                        z[i] = kLowest;
                    }
                    high = z[i] > high ? z[i] : high;
                }
                // Sums without the target's exponential: beside a share near one the others' would lose their bits. The
                // maximum is no NaN; where all are minus infinity the exponentials over zero are zeros (or NaN).
                const float over = high == kLowest ? 0.0f : high;
                others[b] *= top[b] == high ? 1.0f : exp_of(top[b] - high);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = row0 + 32 * a + 8 * (i / 4) + i % 4;
                    others[b] += r == target[b] ? 0.0f : exp_of(z[i] - over);
                }
                top[b] = high;
            }
            bits += 32;
            of_bias += 32;
            to += 32 * stride;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t t = t0 + 32 * b;
            const float both = fmaxf(top[b], red::partner<5>(top[b], lane));
            float mine = top[b] == both ? others[b] : others[b] * exp_of(top[b] - both);
            mine += red::partner<5>(mine, lane);
            if (lane < 32) {
                most[(2 * int64_t(m) + wave / 4) * stride + t] = both;
                sum[(2 * int64_t(m) + wave / 4) * stride + t] = mine;
            }
        }
    }
};

// The statistics of a piece's tokens from those of every 128 classes, and the losses. A token's parts are shared by four
// threads, wavefront w taking every fourth.
__global__ __launch_bounds__(256) void token_kernel(const float* __restrict__ most, const float* __restrict__ sum,
                                                    const float* __restrict__ at_target, const float* __restrict__ targets,
                                                    int parts, int64_t stride, int64_t tokens, int64_t classes,
                                                    Token* __restrict__ out, float* __restrict__ losses) {
    __shared__ float tops[4][64];
    __shared__ double totals[4][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t t = int64_t(blockIdx.x) * 64 + lane;  // below the stride
    float top = kLowest;
    for (int p = wave; p < parts; p += 4) top = fmaxf(top, most[p * stride + t]);
    tops[wave][lane] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0][lane], tops[1][lane]), fmaxf(tops[2][lane], tops[3][lane]));
    double others = 0.0;
    for (int p = wave; p < parts; p += 4) {
        const float m = most[p * stride + t];
        others += double(sum[p * stride + t]) * (m == top ? 1.0 : double(exp_of(m - top)));
    }
    totals[wave][lane] = others;
    __syncthreads();
    if (wave != 0 || t >= tokens) return;
    const int64_t target = class_of(targets[t], classes);
    if (target < 0) {
        if (out) out[t] = Token{0.0f, 0.0f, 0.0f, -1};
        if (losses) losses[t] = 0.0f;
        return;
    }
    others = ((totals[0][lane] + totals[1][lane]) + totals[2][lane]) + totals[3][lane];
    const float at = at_target[t] - top;
    const double total = others + double(expf(at));
    if (losses) losses[t] = float(log(total) - double(at));
    if (out) out[t] = Token{top, float(1.0 / total), float(others / total), int(target)};
}

// dx [tokens, width], times the tokens' shares.
struct InputGradient {
    const Token* of_token;
    const uint32_t* feature_most;
    const float* shares;
    bool one_share;
    float* out;
    int64_t tokens, width;
    __device__ inline void operator()(halves::Tile& tile, int m, int n) const {
        tile.each4([&](int r, int c, float(&v)[4]) {
            const int64_t t = int64_t(m) * halves::kTile + r, d = int64_t(n) * halves::kTile + c;
            if (d >= width) return;
            const int e = halves::exponent_of(feature_most[d]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (t + i >= tokens) continue;
                const Token token = of_token[t + i];
                const float share = token.target < 0 ? 0.0f : shares[one_share ? 0 : t + i];
                const int others = halves::exponent_of(__builtin_bit_cast(uint32_t, token.others));
                out[(t + i) * width + d] = token.target < 0 ? 0.0f : __builtin_amdgcn_ldexpf(v[i], -(e + others)) * share;
            }
        });
    }
};

// dW [width, classes], added to what is there for all pieces but the first.
struct WeightGradient {
    const uint32_t *feature_most, *class_most;
    float* out;
    int64_t width, classes;
    bool add;
    __device__ inline void operator()(halves::Tile& tile, int m, int n) const {
        tile.each4([&](int r, int c, float(&v)[4]) {
            const int64_t d = int64_t(m) * halves::kTile + r, k = int64_t(n) * halves::kTile + c;
            if (k >= classes) return;
            const int e = halves::exponent_of(class_most[k]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (d + i >= width) continue;
                float* const to = out + (d + i) * classes + k;
                const float g = __builtin_amdgcn_ldexpf(v[i], -(e + halves::exponent_of(feature_most[d + i])));
                *to = add ? *to + g : g;
            }
        });
    }
};

// How many of a split tile's parts are there, zero between launches (which follow each other on one stream).
constexpr int kMostSplit = 1024;
__device__ unsigned g_parts_done[kMostSplit];

template <class Epilogue>
__global__ __launch_bounds__(halves::kThreads) void product_kernel(const half* __restrict__ a, const half* __restrict__ b,
                                                                   halves::Tiles tiles, float* __restrict__ partial,
                                                                   Epilogue epilogue) {
    extern __shared__ __attribute__((aligned(128))) char lds[];
    __shared__ bool last;
    const halves::Place at = halves::place_of(tiles, blockIdx.x);
    const int parts = at.split ? tiles.parts : 1;
    const int begin = int(int64_t(tiles.lines) * at.part / parts), end = int(int64_t(tiles.lines) * (at.part + 1) / parts);
    const int64_t of_row = int64_t(tiles.lines) * (halves::kLineBytes / 2);
    halves::Tile tile;
    tile.clear();
    tile.accumulate(a + at.m * halves::kTile * of_row, b + at.n * halves::kTile * of_row, tiles.lines, begin, end, lds);
    if (at.split) {
        const int rest = (int(blockIdx.x) - tiles.whole) % tiles.rest;
        if (!tile.join(at.part, parts, partial + int64_t(rest) * parts * halves::Tile::kValues * halves::kThreads, &g_parts_done[rest],
                       last))
            return;
    }
    epilogue(tile, at.m, at.n);
}

void run(int status) {
    if (status != VC_HIP_OK) fail(status, vc_hip_last_error());
}

struct Call {
    const float *x, *weight, *bias, *targets;
    size_t rows, width, classes;
};

void check_call(const char* op, const Call& c) {
    const std::string name(op);
    if (c.width == 0 || c.classes == 0) fail(VC_HIP_ERR_INVALID_ARGUMENT, name + ": no features or no classes");
    if (c.classes > (size_t(1) << 24)) fail(VC_HIP_ERR_OVERFLOW, name + ": float32 class numbers reach 2^24 classes");
    if (c.width > (size_t(1) << 24) || c.rows >= (size_t(1) << 31)) fail(VC_HIP_ERR_OVERFLOW, name + ": too many rows or features");
    if (c.rows && (!c.x || !c.weight || !c.targets)) fail(VC_HIP_ERR_INVALID_ARGUMENT, name + ": null pointer");
}

// Logits of a piece: 2^28 of them, 1 GiB.
size_t rows_of_piece(const Call& c) { return std::max<size_t>(1, std::min(c.rows, (size_t(1) << 28) / c.classes)); }

void product(const float* a, const float* b, float* c, size_t m, size_t k, size_t n, bool trans_a, bool trans_b) {
    const size_t none = 0;
    run(vc_hip_matmul(a, b, c, m, k, n, &none, &none, 1, trans_a, trans_b));
}

void forward(Device& d, const Call& c, float* losses) {
    const size_t piece = rows_of_piece(c);
    Scratch logits(piece * c.classes * sizeof(float));
    for (size_t r = 0; r < c.rows; r += piece) {
        const size_t n = std::min(piece, c.rows - r);
        product(c.x + r * c.width, c.weight, logits.as<float>(), n, c.width, c.classes, false, false);
        launch(logits_kernel<false>, dim3(grid_1d(n, 1, 16u * unsigned(d.cu_count))), dim3(kRowThreads), 0, d.stream,
               logits.as<float>(), c.bias, c.targets + r, nullptr, false, int64_t(n), int64_t(c.classes), losses + r);
        after_launch("linear_cross_entropy rows");
    }
}

void gradient(Device& d, const Call& c, const float* shares, bool one_share, float* losses, float* grad_x, float* grad_weight,
              float* grad_bias) {
    const size_t piece = rows_of_piece(c), pieces = (c.rows + piece - 1) / piece;
    Scratch logits(piece * c.classes * sizeof(float));
    Scratch rows(grad_weight ? piece * c.width * sizeof(float) : 4);
    Scratch more(pieces > 1 ? std::max(grad_weight ? c.width * c.classes : 0, c.classes) * sizeof(float) : 4);
    for (size_t r = 0; r < c.rows; r += piece) {
        const size_t n = std::min(piece, c.rows - r);
        const float* const x = c.x + r * c.width;
        float* const z = logits.as<float>();
        product(x, c.weight, z, n, c.width, c.classes, false, false);
        launch(logits_kernel<true>, dim3(grid_1d(n, 1, 16u * unsigned(d.cu_count))), dim3(kRowThreads), 0, d.stream, z, c.bias,
               c.targets + r, one_share ? shares : shares + r, one_share, int64_t(n), int64_t(c.classes),
               losses ? losses + r : nullptr);
        after_launch("linear_cross_entropy rows");
        if (grad_x) product(z, c.weight, grad_x + r * c.width, n, c.classes, c.width, false, true);
        if (grad_weight) {
            launch(counted_rows_kernel, dim3(grid_1d(n, 1, 16u * unsigned(d.cu_count))), dim3(256), 0, d.stream, x, c.targets + r,
                   rows.as<float>(), int64_t(n), int64_t(c.width), int64_t(c.classes));
            after_launch("linear_cross_entropy counted rows");
            product(rows.as<float>(), z, r ? more.as<float>() : grad_weight, c.width, n, c.classes, true, false);
            if (r) run(vc_hip_axpy(grad_weight, more.as<float>(), c.width * c.classes, 1.0f));
        }
        if (grad_bias) {
            run(vc_hip_reduce_axis(z, r ? more.as<float>() : grad_bias, 1, n, c.classes, VC_REDUCE_SUM));
            if (r) run(vc_hip_axpy(grad_bias, more.as<float>(), c.classes, 1.0f));
        }
    }
}

template <class Epilogue>
void packed_product(Device& d, const half* a, const half* b, int64_t rows_a, int64_t rows_b, int64_t lines, const Epilogue& epilogue) {
    const halves::Tiles tiles = halves::tiles_of(rows_a, rows_b, lines, d.cu_count);
    if (tiles.rest > kMostSplit) fail(VC_HIP_ERR_RUNTIME, "linear_cross_entropy: more split tiles than counters");
    Scratch partial(tiles.rest ? size_t(tiles.rest) * tiles.parts * halves::Tile::kValues * halves::kThreads * sizeof(float) : 4);
    static const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(product_kernel<Epilogue>),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, halves::Tile::kLds);
    check_hip(allowed, "hipFuncSetAttribute");
    launch(product_kernel<Epilogue>, dim3(unsigned(tiles.blocks())), dim3(halves::kThreads), uint32_t(halves::Tile::kLds), d.stream, a, b,
           tiles, partial.as<float>(), epilogue);
    after_launch("linear_cross_entropy product");
}

int64_t whole_tiles(int64_t n) { return (n + halves::kTile - 1) / halves::kTile * halves::kTile; }
int64_t lines_of(int64_t n) { return (n + halves::kSlice - 1) / halves::kSlice; }
// A packed matrix of `rows` rows of `depth` values.
size_t packed_bytes(int64_t rows, int64_t depth) { return size_t(whole_tiles(rows)) * size_t(lines_of(depth)) * halves::kLineBytes; }

template <class Source>
void pack(Device& d, const Source& from, half* by_row, half* by_column) {
    const int64_t down = (by_row ? whole_tiles(from.rows) : lines_of(from.rows) * 32) / kPackRows;
    const int64_t across = whole_tiles(from.columns) / kPackColumns;
    launch(pack_kernel<Source>, grid_2d(size_t(down * across)), dim3(kPackThreads), 0, d.stream, from, by_row, int(lines_of(from.columns)),
           by_column, int(lines_of(from.rows)), int(across));
    after_launch("linear_cross_entropy pack");
}

void largest(Device& d, const float* values, const float* targets, size_t rows, size_t columns, size_t classes, uint32_t* row_most,
             uint32_t* column_most) {
    const size_t down = (rows + kMostRows - 1) / kMostRows, across = (columns + kMostColumns - 1) / kMostColumns;
    launch(most_kernel, grid_2d(down * across), dim3(256), 0, d.stream, values, targets, int64_t(rows), int64_t(columns),
           int64_t(classes), int(across), row_most, column_most);
    after_launch("linear_cross_entropy largest");
}

// The packed route. losses or, of a gradient, any output may be null; a call without gradients has no shares.
void packed(Device& d, const Call& c, const float* shares, bool one_share, float* losses, float* grad_x, float* grad_weight,
            float* grad_bias) {
    const bool gradient = grad_x || grad_weight || grad_bias;
    const int64_t width = int64_t(c.width), classes = int64_t(c.classes), rows = int64_t(c.rows);
    const int64_t most_rows = gradient ? std::max<int64_t>(1, (int64_t(1) << 28) / classes / halves::kTile) * halves::kTile : 65536;
    const int64_t pieces = (rows + most_rows - 1) / most_rows;
    const int64_t piece = std::min(most_rows, whole_tiles((rows + pieces - 1) / pieces));
    const int64_t parts = 2 * whole_tiles(classes) / halves::kTile;
    const int64_t groups = (piece + kGroupTokens - 1) / kGroupTokens;

    // The largest magnitudes: of W's rows and columns, of x's rows and columns, of a piece's classes.
    const int64_t n_width = whole_tiles(width), n_classes = whole_tiles(classes), n_rows = whole_tiles(rows);
    const int64_t n_most = 2 * n_width + n_classes + n_rows + (gradient ? pieces * n_classes : 0);
    Scratch most(size_t(n_most) * sizeof(uint32_t));
    run(vc_hip_fill(most.as<float>(), size_t(n_most), 0.0f));
    uint32_t *const w_rows = most.as<uint32_t>(), *const x_columns = w_rows + n_width, *const w_columns = x_columns + n_width;
    uint32_t *const x_rows = w_columns + n_classes, *const z_classes = x_rows + n_rows;
    largest(d, c.weight, nullptr, c.width, c.classes, c.classes, grad_x ? w_rows : nullptr, w_columns);
    largest(d, c.x, c.targets, c.rows, c.width, c.classes, x_rows, grad_weight ? x_columns : nullptr);

    Scratch wt(packed_bytes(classes, width)), w(grad_x ? packed_bytes(width, classes) : 4);
    pack(d, Plain{c.weight, nullptr, width, classes, classes, w_rows, w_columns}, grad_x ? w.as<half>() : nullptr, wt.as<half>());

    Scratch x(packed_bytes(piece, width)), xt(grad_weight ? packed_bytes(width, piece) : 4);
    Scratch logits(gradient ? size_t(classes * piece) * sizeof(float) : 4);
    Scratch zt(grad_weight ? packed_bytes(classes, piece) : 4), z(grad_x ? packed_bytes(piece, classes) : 4);
    Scratch statistics(size_t(2 * parts + 1) * size_t(piece) * sizeof(float)), tokens(size_t(piece) * sizeof(Token));
    Scratch sums(grad_bias ? size_t(pieces * groups * classes) * sizeof(double) : 4);
    float *const part_most = statistics.as<float>(), *const part_sum = part_most + parts * piece, *const at_target = part_sum + parts * piece;
    int64_t sum_rows = 0;

    for (int64_t p = 0, first = 0; p < pieces && first < rows; ++p, first += piece) {
        const int64_t n = std::min(piece, rows - first);
        const float *const targets = c.targets + first, *const own_shares = one_share ? shares : shares + first;
        uint32_t* const class_most = z_classes + p * n_classes;
        pack(d, Plain{c.x + first * width, targets, n, width, classes, x_rows + first, x_columns}, x.as<half>(),
             grad_weight ? xt.as<half>() : nullptr);
        packed_product(d, wt.as<half>(), x.as<half>(), classes, n, lines_of(width),
                       Logits{w_columns, x_rows + first, c.bias, targets, gradient ? logits.as<float>() : nullptr, part_most, part_sum,
                              at_target, classes, n, piece});
        launch(token_kernel, dim3(unsigned((n + 63) / 64)), dim3(256), 0, d.stream, part_most, part_sum, at_target, targets, int(parts),
               piece, n, classes, gradient ? tokens.as<Token>() : nullptr, losses ? losses + first : nullptr);
        after_launch("linear_cross_entropy tokens");
        if (!gradient) continue;
        const Gradients from{logits.as<float>(), piece, tokens.as<Token>(), own_shares, one_share, classes, n, class_most};
        const int64_t own_groups = (n + kGroupTokens - 1) / kGroupTokens;
        if (grad_weight || grad_bias) {
            const dim3 grid = grid_2d(size_t(own_groups * ((classes + kGroupClasses - 1) / kGroupClasses)));
            if (grad_bias)
                launch(class_most_kernel<true>, grid, dim3(64), 0, d.stream, from, class_most, sums.as<double>() + sum_rows * classes,
                       int(own_groups));
            else
                launch(class_most_kernel<false>, grid, dim3(64), 0, d.stream, from, class_most, nullptr, int(own_groups));
            after_launch("linear_cross_entropy classes");
            sum_rows += own_groups;
        }
        if (grad_x || grad_weight) pack(d, from, grad_weight ? zt.as<half>() : nullptr, grad_x ? z.as<half>() : nullptr);
        if (grad_x)
            packed_product(d, z.as<half>(), w.as<half>(), n, width, lines_of(classes),
                           InputGradient{tokens.as<Token>(), w_rows, own_shares, one_share, grad_x + first * width, n, width});
        if (grad_weight)
            packed_product(d, xt.as<half>(), zt.as<half>(), width, classes, lines_of(n),
                           WeightGradient{x_columns, class_most, grad_weight, width, classes, p > 0});
    }
    if (grad_bias) {
        launch(red::column_partials_kernel, dim3(unsigned((classes + 63) / 64)), dim3(64 * red::kCombineWaves), 0, d.stream,
               sums.as<double>(), sum_rows, classes, grad_bias);
        after_launch("linear_cross_entropy bias");
    }
}

bool takes_packed(const Call& c) {
    return double(c.rows) * double(c.width) * double(c.classes) >= double(1 << 28) && c.classes < (size_t(1) << 21) &&
           c.width < (size_t(1) << 21);
}

void count(Device& d, const Call& c, float* share) {
    launch(count_kernel, dim3(1), dim3(kCountThreads), 0, d.stream, c.targets, int64_t(c.rows), int64_t(c.classes), share);
    after_launch("linear_cross_entropy count");
}
void mean_of(Device& d, const Call& c, const float* losses, const float* share, float* mean) {
    launch(mean_kernel, dim3(1), dim3(kCountThreads), 0, d.stream, losses, int64_t(c.rows), share, mean);
    after_launch("linear_cross_entropy mean");
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_linear_xent_forward(const float* x, const float* weight, const float* bias, const float* targets, size_t rows,
                               size_t width, size_t classes, float* losses, float* mean) {
    return guard([&] {
        Device& d = require_device();
        const Call c{x, weight, bias, targets, rows, width, classes};
        check_call("linear_cross_entropy", c);
        if (rows == 0) {
            if (mean) run(vc_hip_fill(mean, 1, 0.0f));
            return;
        }
        if (!losses && !mean) return;
        const double products = 2.0 * double(rows) * double(width) * double(classes);
        Profiled p("linear_cross_entropy", products, 4.0 * double(width) * double(rows + classes));
        std::unique_ptr<Scratch> own;
        if (!losses) {
            own = std::make_unique<Scratch>(rows * sizeof(float));
            losses = own->as<float>();
        }
        if (takes_packed(c)) packed(d, c, nullptr, true, losses, nullptr, nullptr, nullptr);
        else forward(d, c, losses);
        if (mean) {
            Scratch share(sizeof(float));
            count(d, c, share.as<float>());
            mean_of(d, c, losses, share.as<float>(), mean);
        }
        p.done();
    });
}

int vc_hip_linear_xent_gradient(const float* x, const float* weight, const float* bias, const float* targets,
                                const float* shares, size_t rows, size_t width, size_t classes, float* mean, float* grad_x,
                                float* grad_weight, float* grad_bias) {
    return guard([&] {
        Device& d = require_device();
        const Call c{x, weight, bias, targets, rows, width, classes};
        check_call("linear_cross_entropy", c);
        if (shares && mean) fail(VC_HIP_ERR_INVALID_ARGUMENT, "linear_cross_entropy: the mean has shares of its own");
        if (rows == 0) {
            if (mean) run(vc_hip_fill(mean, 1, 0.0f));
            if (grad_weight) run(vc_hip_fill(grad_weight, width * classes, 0.0f));
            if (grad_bias) run(vc_hip_fill(grad_bias, classes, 0.0f));
            return;
        }
        const double products = 2.0 * double(rows) * double(width) * double(classes);
        Profiled p("linear_cross_entropy_gradient", products * (1.0 + (grad_x != nullptr) + (grad_weight != nullptr)),
                   8.0 * double(width) * double(rows + classes));
        Scratch share(sizeof(float)), losses(mean ? rows * sizeof(float) : 4);
        if (!shares) count(d, c, share.as<float>());
        const auto route = takes_packed(c) ? packed : gradient;
        route(d, c, shares ? shares : share.as<float>(), !shares, mean ? losses.as<float>() : nullptr, grad_x, grad_weight,
              grad_bias);
        if (mean) mean_of(d, c, losses.as<float>(), share.as<float>(), mean);
        p.done();
    });
}

}  // extern "C"
