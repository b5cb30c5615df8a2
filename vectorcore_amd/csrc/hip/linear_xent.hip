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
// All of them keep float32's precision: an error is one of a few roundings of the
// terms of the sum that it is in, whatever the operands' other values; packed, the
// gradients of a class do so down to 2^-82 of the largest upstream gradient.
//
// Rows are taken in pieces: the logits of a piece live in a workspace until
// their gradients are used. Three routes, by sizes alone:
// - up to 16 rows of many classes without gradients read W once and keep no
//   logits; bound by HBM (1 row, 1024 x 50000: 37 us of 205 MB, 5.5 TB/s, and 4 us
//   to join);
// - small or thin calls take float32 products and a kernel of the rows; bound by
//   launches (256 rows, 256 x 10 with gradients: 25 us in five);
// - others take packed products, bound by matrix instructions: 8192 rows, 1024 x
//   50000, of which 7373 count, with gradients 6.75 ms: 2.05 (the logits, 369
//   TFLOP/s), 1.81 and 1.90 (their gradients' products), 0.99 (the gradients, 4.4
//   GB at 4.4 TB/s), 0.3 for all others. 1536 rows that count without: 0.55 ms,
//   of which the logits 0.47. Where the operands' rows hold values too unlike for
//   two half-precision parts, three parts: 11.6 and 0.84 ms.
#include "halves_product.hpp"
#include "reduce_common.hpp"
#include "thirds_product.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

namespace vchip {
namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kLowest = -__builtin_huge_valf(), kLog2e = 1.44269504f;

// Off by roundings of x and one of the result, as the argument itself is.
__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// The class a target names, or -1.
__device__ inline int64_t class_of(float target, int64_t classes) {
    if (!(target >= 0.0f && target < float(classes))) return -1;
    const int64_t c = int64_t(target);
    return float(c) == target ? c : -1;
}

constexpr int kCountThreads = 1024, kCountRows = 4;  // rows of a thread and turn

// The rows that count: how many (counted), one over it or zero (share), and which, in order (place, or null), for the packed
// route with the largest finite magnitude of their shares (most, or null). losses: zeros for the others, or null. cleared: n_cleared
// words of zeros, by the workgroups behind the first.
__global__ __launch_bounds__(kCountThreads) void count_kernel(const float* __restrict__ targets, const float* __restrict__ shares,
                                                              int64_t rows, int64_t classes, int* __restrict__ counted,
                                                              float* __restrict__ share, int* __restrict__ place,
                                                              uint32_t* __restrict__ most, float* __restrict__ losses,
                                                              uint32_t* __restrict__ cleared, int64_t n_cleared) {
    if (blockIdx.x > 0) {
        const int64_t step = int64_t(gridDim.x - 1) * kCountThreads;
        for (int64_t i = int64_t(blockIdx.x - 1) * kCountThreads + threadIdx.x; i < n_cleared; i += step) cleared[i] = 0u;
        return;
    }
    __shared__ int of_wave[kCountThreads / 64];
    __shared__ uint32_t most_of_wave[kCountThreads / 64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int before = 0;
    uint32_t high = 0;
    for (int64_t r0 = 0; r0 < rows; r0 += kCountThreads * kCountRows) {
        const int64_t first = r0 + int64_t(threadIdx.x) * kCountRows;
        int flags = 0;
#pragma unroll
        for (int i = 0; i < kCountRows; ++i) {
            const int64_t r = first + i;
            if (r >= rows) continue;
            if (class_of(targets[r], classes) >= 0) {
                flags |= 1 << i;
                if (most && shares) {
                    const uint32_t bits = __builtin_bit_cast(uint32_t, shares[r]) & 0x7FFFFFFFu;
                    high = max(high, bits < 0x7F800000u ? bits : 0u);
                }
            } else if (losses) {
                losses[r] = 0.0f;
            }
        }
        const int own = __popc(flags);
        int upto = own;  // of this wavefront's lanes up to this one
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int other = __shfl_up(upto, d, 64);
            if (lane >= d) upto += other;
        }
        if (lane == 63) of_wave[wave] = upto;
        __syncthreads();
        int all = 0, at = before + upto - own;
        for (int w = 0; w < kCountThreads / 64; ++w) {
            if (w < wave) at += of_wave[w];
            all += of_wave[w];
        }
        if (place) {
#pragma unroll
            for (int i = 0; i < kCountRows; ++i)
                if (flags >> i & 1) place[at++] = int(first + i);
        }
        before += all;
        __syncthreads();
    }
    if (most) {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) high = max(high, uint32_t(__shfl_xor(int(high), d, 64)));
        if (lane == 0) most_of_wave[wave] = high;
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    const float one = before > 0 ? float(1.0 / double(before)) : 0.0f;
    if (counted) counted[0] = before;
    share[0] = one;
    if (!most) return;
    if (!shares) {
        most[0] = __builtin_bit_cast(uint32_t, one);
        return;
    }
    for (int w = 1; w < kCountThreads / 64; ++w) high = max(high, most_of_wave[w]);
    most[0] = max(high, most_of_wave[0]);
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

template <int Threads>
__device__ inline float workgroup_max(float v, float* lds) {
    const int lane = red::lane_id();
    v = fmaxf(v, red::partner<0>(v, lane));
    v = fmaxf(v, red::partner<1>(v, lane));
    v = fmaxf(v, red::partner<2>(v, lane));
    v = fmaxf(v, red::partner<3>(v, lane));
    v = fmaxf(v, red::partner<4>(v, lane));
    v = fmaxf(v, red::partner<5>(v, lane));
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    float m = lds[0];
    for (int w = 1; w < Threads / 64; ++w) m = fmaxf(m, lds[w]);
    return m;
}

// What the rows' kernel makes beside dz. losses, x and mean: each may be null.
struct RowOutputs {
    float* losses;    // of each row
    const float* x;   // [rows, width], of which counted_x gets a copy whose left out rows are zeros: zero times what they hold
    float* counted_x; // would not be zero for an infinity or a NaN
    int64_t width;
    float* mean;      // the mean loss of all rows
    double* partial;  // one of each workgroup
};

// Rows that each workgroup counts by itself: a launch less, but rows times rows reads. (Train steps of 1024 rows, 256 x 1000: 46 us,
// 53 with a launch that counts; of 4096, 128 x 128: 51 and 41.)
constexpr int kCountedHere = 1024;

// A workgroup a row: its loss from the logits z (without the bias), and, where Gradient, z becomes dz. Held: the row, of at most
// 4 Threads Held values, is read once and stays in registers; 0: read for the maximum, the sum and the gradient. Bound by the
// loads' latency: 468 rows of 26655 with gradients 35 us (of 100 MB; 57 with one load of a thread in flight), 19 rows of 52907
// 21 (47); 256 rows of 10, one wavefront each, 8.6.
// shares: of each row, or of all (one_share), or null: one over the number of rows that count, which each workgroup finds itself.
template <int Threads, int Held, bool Gradient>
__global__ __launch_bounds__(Threads) void logits_kernel(float* __restrict__ z, const float* __restrict__ bias,
                                                         const float* __restrict__ targets, const float* __restrict__ shares,
                                                         bool one_share, int64_t rows, int64_t classes, RowOutputs out) {
    __shared__ double sums[Threads / 64];
    __shared__ float most[Threads / 64];
    __shared__ double total_of_row;
    float one = 0.0f;
    if (!shares && (Gradient || out.mean)) {
        double n = 0.0;
        for (int64_t r = threadIdx.x; r < rows; r += Threads) n += class_of(targets[r], classes) >= 0 ? 1.0 : 0.0;
        n = red::block_sum(n, sums);
        if (threadIdx.x == 0) total_of_row = n;
        __syncthreads();
        n = total_of_row;
        one = n > 0.0 ? float(1.0 / n) : 0.0f;
    } else if (shares && one_share) {
        one = shares[0];
    }
    double lost = 0.0;  // in thread 0
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        __syncthreads();
        float* const row = z + r * classes;
        const int64_t target = class_of(targets[r], classes);
        if (Gradient && out.x)
            for (int64_t c = threadIdx.x; c < out.width; c += Threads)
                out.counted_x[r * out.width + c] = target >= 0 ? out.x[r * out.width + c] : 0.0f;
        if (target < 0) {
            if (out.losses && threadIdx.x == 0) out.losses[r] = 0.0f;
            if constexpr (Gradient)
                for (int64_t c = threadIdx.x; c < classes; c += Threads) row[c] = 0.0f;
            continue;
        }
        const auto value = [&](int64_t c) { return bias ? row[c] + bias[c] : row[c]; };
        const float at = value(target);
        // f(class, logit), four loads of four logits in flight; what f makes of them is written back if `keep`.
        const auto each = [&](auto&& f, bool keep = false) {
            constexpr int kLoads = 4;
            for (int64_t c0 = 4 * int64_t(threadIdx.x); c0 < classes; c0 += 4 * Threads * kLoads) {
                f4u x[kLoads], more[kLoads];
#pragma unroll
                for (int u = 0; u < kLoads; ++u) {
                    const int64_t c = c0 + 4 * Threads * u;
                    if (c + 3 < classes) {
                        x[u] = *reinterpret_cast<const f4u*>(row + c);
                        if (bias) more[u] = *reinterpret_cast<const f4u*>(bias + c);
                    }
                }
#pragma unroll
                for (int u = 0; u < kLoads; ++u) {
                    const int64_t c = c0 + 4 * Threads * u;
                    if (c + 3 < classes) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float y = bias ? x[u][e] + more[u][e] : x[u][e];
                            f(c + e, y);
                            x[u][e] = y;
                        }
                        if (keep) *reinterpret_cast<f4u*>(row + c) = x[u];
                    } else {
                        for (int64_t l = c; l < classes; ++l) {
                            float y = value(l);
                            f(l, y);
                            if (keep) row[l] = y;
                        }
                    }
                }
            }
        };
        f4u v[Held > 0 ? Held : 1];
        float m = kLowest;
        if constexpr (Held > 0) {
#pragma unroll
            for (int u = 0; u < Held; ++u) {
                const int64_t c = 4 * int64_t(threadIdx.x) + 4 * Threads * u;
                if (c + 3 < classes) {
                    v[u] = *reinterpret_cast<const f4u*>(row + c);
                    if (bias) {
                        const f4u more = *reinterpret_cast<const f4u*>(bias + c);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[u][e] += more[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][e] = c + e < classes ? value(c + e) : kLowest;
                }
            }
#pragma unroll
            for (int u = 0; u < Held; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, v[u][e]);
        } else {
            each([&](int64_t, float& x) { m = fmaxf(m, x); });
        }
        m = workgroup_max<Threads>(m, most);
        double s = 0.0;
        if constexpr (Held > 0) {
#pragma unroll
            for (int u = 0; u < Held; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool there = 4 * int64_t(threadIdx.x) + 4 * Threads * u + e < classes;
                    v[u][e] = there ? exp_of(v[u][e] - m) : 0.0f;
                    s += double(v[u][e]);
                }
        } else {
            each([&](int64_t, float& x) { s += double(exp_of(x - m)); });
        }
        s = red::block_sum(s, sums);
        if (threadIdx.x == 0) total_of_row = s;
        __syncthreads();  // and every thread has read the target's logit
        s = total_of_row;
        const double loss = log(s) - double(at - m);
        if (threadIdx.x == 0) {
            if (out.losses) out.losses[r] = float(loss);
            lost += loss;
        }
        if constexpr (Gradient) {
            const float share = !shares || one_share ? one : shares[r], scale = float(double(share) / s);
            // The others' sum in double: one minus a share near one would leave no bits.
            const float own = float(-double(share) * ((s - double(exp_of(at - m))) / s));
            if constexpr (Held > 0) {
#pragma unroll
                for (int u = 0; u < Held; ++u) {
                    const int64_t c = 4 * int64_t(threadIdx.x) + 4 * Threads * u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][e] = c + e == target ? own : v[u][e] * scale;
                    if (c + 3 < classes) {
                        *reinterpret_cast<f4u*>(row + c) = v[u];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < classes) row[c + e] = v[u][e];
                    }
                }
            } else {
                each([&](int64_t c, float& x) { x = c == target ? own : exp_of(x - m) * scale; }, true);
            }
        }
    }
    if (!out.mean || threadIdx.x >= 64) return;
    if (!red::count_in(lost, out.partial)) return;
    const double total = red::finish_partials(out.partial);
    if (threadIdx.x == 0) out.mean[0] = float(total * double(one));
}

// ---- large products: packed halves -----------------------------------------------------
//
// The rows that count are taken together, so that the others cost nothing. The three products of a piece of them read packed
// operands (halves_product.hpp), each made once:
//   z^T = W^T x^T  from the columns of W and the rows of x, along the features,
//   dx  = dz W^T   from the rows of dz and of W, along the classes,
//   dW  = x^T dz   from the columns of x and of dz, along the tokens of the piece.
// The logits are made transposed: a thread of the product then holds 64 classes of a token, whose maximum and sum need no
// exchange but one, and a class's gradients, packed along the tokens, take the place of its logits.
//
// A class's gradients may be small at every token (a rare class) and are scaled by a power of two of their own, for each block
// of 256 tokens that of the largest in it: the product's sums change their unit with the block.

using halves::half;
using halves::h8;

// How far the rows of the packed operands hold values unlike each other, in sixteenths of a bit: the most by which a row's largest
// exponent lies above the mean of its values' (zeros aside), for the rows of x and the columns of W (along the features), the
// rows of W (along the classes) and the columns of x (along the tokens). Also the largest exponents of x and W, and whether
// either holds an infinity or a NaN.
//
// Two half-precision parts keep 22 bits of a value or 2^-38 of its row's largest. The latter takes 2^-37 n X Y at most from a sum of
// n products, X and Y being both rows' largest. The sum of the products' magnitudes is at least n times the product of both rows'
// geometric means: where the largest lie 15 bits above those together (13 by the exponents, each of which leaves a bit open), less
// than 2^-22 of the sum's own terms is lost. Or n X Y <= 2^13: then it is 2^-24, what an exponential rounds by in any case. In the
// products of the logits' gradients that operand loses 2^-38 of a token's (of W: a class's) largest gradient at every class (token),
// for 2^17 of them 2^-21 of it times the other row's mean, and ten bits keep what the other row loses below 2^-26 of its mean.
// Calls beyond take three bfloat16 parts (thirds_product.hpp), which keep every value's 24 bits: a feature of 1e9 whose weights are
// 1e-9 costs time, not the logits.
struct Unlike {
    int x_rows, w_columns, w_rows, x_columns, x_most, w_most, not_finite;
    // width_bits: of the next power of two.
    __device__ inline bool thirds(int width_bits) const {
        const bool alike = x_rows + w_columns <= 13 * 16, small = x_most + w_most - 2 * kExponents + width_bits <= 13;
        return not_finite || !(alike || small) || w_rows > 10 * 16 || x_columns > 10 * 16;
    }
    static constexpr int kExponents = 149;  // of a finite value's exponent, for positive numbers
};
__device__ inline int exponent_over(float finite) { return __builtin_amdgcn_frexp_expf(finite) + Unlike::kExponents; }

// Which form the packed operands of a call have.
struct Form {
    const Unlike* unlike;
    int width_bits;
    __device__ inline bool thirds() const { return unlike->thirds(width_bits); }
};

constexpr int kPackThreads = 256, kPackRows = 32, kPackColumns = 128;
constexpr int kBlockTokens = 256, kBlockLines = kBlockTokens / halves::kSlice;

// A piece of the rows that count: rows place[first] .. of the call, as many as there are, at most `most`.
struct Piece {
    const int *counted, *place;
    int64_t first, most;
    __device__ inline int64_t tokens() const { return max(int64_t(0), min(most, int64_t(counted[0]) - first)); }
    __device__ inline int64_t row(int64_t t) const { return place[first + t]; }
};

// A matrix of floats [rows, columns], packed by its rows (along columns, row_lines a row) and by its columns (along rows,
// column_lines a column); either may be without memory. of.place: the matrix's rows are the piece's; else `rows` of them in order. The
// largest magnitudes are those of the whole matrix's rows and columns. exponents, filled: or null; of each column its exponent,
// and bias (or zero), minus infinity for the columns that fill the last tile. A workgroup takes 32 rows and 128 columns, past
// the ends zeros.
struct Packing {
    const float* values;
    Piece of;
    int64_t rows, columns;
    const uint32_t *row_most, *column_most;
    thirds::Operand by_row, by_column;
    int row_lines, column_lines, down, across;
    const float* bias;
    int* exponents;
    float* filled;
    size_t blocks() const { return size_t(down) * size_t(across); }
};

// Of two matrices in one launch, or of one (the second has no blocks).
__global__ __launch_bounds__(kPackThreads) void pack_kernel(Packing one, Packing two, Form form) {
    __shared__ float tile[kPackRows][kPackColumns + 4];
    int64_t block = block_id();
    const int64_t in_one = int64_t(one.down) * one.across;
    const bool first_one = block < in_one;
    if (!first_one) block -= in_one;
    const Packing p = first_one ? one : two;
    const int down = p.down, across = p.across, row_lines = p.row_lines, column_lines = p.column_lines;
    if (across == 0) return;
    const int64_t row0 = block / across * kPackRows, column0 = block % across * kPackColumns;
    if (block / across >= down) return;
    const Piece of = p.of;
    int64_t rows = p.rows;
    const int64_t columns = p.columns;
    const float* __restrict__ values = p.values;
    const uint32_t *const row_most = p.row_most, *const column_most = p.column_most;
    half* __restrict__ by_row = p.by_row.first;
    half* __restrict__ by_column = p.by_column.first;
    if (of.place) {
        rows = of.tokens();
        if (row0 >= (rows + halves::kTile - 1) / halves::kTile * halves::kTile) return;
    }
    if (p.exponents && row0 == 0 && threadIdx.x < kPackColumns) {
        const int64_t v = column0 + threadIdx.x;
        p.exponents[v] = v < columns ? halves::exponent_of(column_most[v]) : 0;
        p.filled[v] = v >= columns ? kLowest : p.bias ? p.bias[v] : 0.0f;
    }
    const bool thirds = form.thirds();
    // Sixteen threads read 512 neighbouring bytes of a row.
    const int c = 8 * (threadIdx.x % 16);
    const int64_t column = column0 + c;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = threadIdx.x / 16 + 16 * j;
        const bool there = row0 + r < rows;
        const int64_t row = there && of.place ? of.row(row0 + r) : row0 + r;
        const float* const at = values + row * columns + column;
        float v[8];
        if (there && column + 8 <= columns) {
            const f4u lo = *reinterpret_cast<const f4u*>(at), hi = *reinterpret_cast<const f4u*>(at + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = lo[i];
                v[4 + i] = hi[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = there && column + i < columns ? at[i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) tile[r][c + i] = v[i];
        if (!thirds && by_row && column / 32 < row_lines) {
            h8 first, second;
            halves::split8(v, there ? halves::exponent_of(row_most[row]) : 0, first, second);
            half* const to = by_row + ((row0 + r) * row_lines + column / 32) * 64 + column % 32;
            *reinterpret_cast<h8*>(to) = first;
            *reinterpret_cast<h8*>(to + 32) = second;
        }
    }
    if (!by_column && !thirds) return;
    __syncthreads();
    const int64_t line = row0 / 32;
    if (thirds) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = threadIdx.x % 32, g = threadIdx.x / 32 + 8 * j;
            if (by_row && (column0 + 8 * g) / 32 < row_lines) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = tile[r][8 * g + i];
                const bool there = row0 + r < rows;
                const int64_t row = there && of.place ? of.row(row0 + r) : row0 + r;
                thirds::store8(p.by_row, row_lines, row0 + r, column0 / 8 + g, v, there ? halves::exponent_of(row_most[row]) : 0);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int at = threadIdx.x % 128, g = threadIdx.x / 128 + 2 * j;
            if (by_column && line < column_lines) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = tile[8 * g + i][at];
                thirds::store8(p.by_column, column_lines, column0 + at, row0 / 8 + g, v,
                               column0 + at < columns ? halves::exponent_of(column_most[column0 + at]) : 0);
            }
        }
        return;
    }
    if (line >= column_lines) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int at = threadIdx.x / 4 + 64 * j, g = threadIdx.x % 4;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[8 * g + i][at];
        h8 first, second;
        halves::split8(v, column0 + at < columns ? halves::exponent_of(column_most[column0 + at]) : 0, first, second);
        half* const to = by_column + ((column0 + at) * column_lines + line) * 64 + 8 * g;
        *reinterpret_cast<h8*>(to) = first;
        *reinterpret_cast<h8*>(to + 32) = second;
    }
}

constexpr int kMostRows = 64, kMostColumns = 256, kCountShift = 36;
constexpr size_t kMostCounted = size_t(1) << 27;  // values of a row or column: their exponents' sum stays below 2^36

// The largest finite magnitudes of a matrix's rows and columns, as bits, and how many finite values are no zeros, times 2^36, plus
// their exponents' sum, into arrays of zeros: bits of positive floats are ordered as the floats are, and whole numbers are added,
// so the order of the atomics does not matter. Rows that targets (or null) leave out have no part; cleared (or null) gets zeros for
// them. A workgroup takes 64 rows and 256 columns.
struct Largest {
    const float *values, *targets;
    int64_t rows, columns;
    int down, across;
    uint32_t *row_most, *column_most;
    unsigned long long *row_sum, *column_sum;
    float* cleared;
    size_t blocks() const { return size_t(down) * size_t(across); }
};

// Over the wavefront, for 2^(Step + 1) rows at a time of which every lane holds a part: lane l gets row l % 16 of sixteen. Each
// exchange leaves a lane and its partner half of the rows each.
template <int Step, int N, class Op>
__device__ inline uint32_t lanes_rows(const uint32_t (&part)[N], int lane, Op op) {
    static_assert(N == 2 << Step);
    const bool upper = lane >> Step & 1;
    uint32_t kept[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const uint32_t mine = upper ? part[N / 2 + i] : part[i], other = upper ? part[i] : part[N / 2 + i];
        kept[i] = op(mine, red::partner<Step>(other, lane));
    }
    if constexpr (Step > 0) {
        return lanes_rows<Step - 1>(kept, lane, op);
    } else {
        uint32_t all = op(kept[0], red::partner<4>(kept[0], lane));
        return op(all, red::partner<5>(all, lane));
    }
}

// Of two matrices in one launch.
__global__ __launch_bounds__(256) void most_kernel(Largest one, Largest two, int64_t classes, Unlike* __restrict__ unlike) {
    __shared__ uint32_t of_column[4][kMostColumns], sum_of_column[4][kMostColumns];
    int64_t block = block_id();
    const int64_t in_one = int64_t(one.down) * one.across;
    const bool first_one = block < in_one;
    if (!first_one) block -= in_one;
    const Largest p = first_one ? one : two;
    if (block / p.across >= p.down) return;
    const int64_t rows = p.rows, columns = p.columns;
    const int64_t row0 = block / p.across * kMostRows, column0 = block % p.across * kMostColumns;
    const float *__restrict__ values = p.values, *__restrict__ targets = p.targets;
    uint32_t* const column_most = p.column_most;
    float* __restrict__ cleared = p.cleared;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = column0 + 4 * lane;
    constexpr int kRows = kMostRows / 4;  // of a wavefront
    const int64_t first = row0 + kRows * wave, own = first + lane;
    const bool inside = lane < kRows && own < rows;
    const uint64_t there = __ballot(inside), counted = __ballot(inside && (!targets || class_of(targets[own], classes) >= 0));
    f4u v[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const float* const at = values + (first + j) * columns + c;
        v[j] = f4u{0.0f, 0.0f, 0.0f, 0.0f};
        if (counted >> j & 1) {
            if (c + 4 <= columns) {
                v[j] = *reinterpret_cast<const f4u*>(at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] = c + e < columns ? at[e] : 0.0f;
            }
        } else if (cleared && (there >> j & 1)) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < columns) cleared[(first + j) * columns + c + e] = 0.0f;
        }
    }
    // Sums of at most 256 values: their number times 2^20 and their exponents'.
    uint32_t most[4] = {0, 0, 0, 0}, sums[4] = {0, 0, 0, 0}, row_most[kRows], row_sums[kRows];
    bool not_finite = false;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        row_most[j] = row_sums[j] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float value = v[j][e];  // a bit cast of a vector's element itself takes the first one
            uint32_t bits = __builtin_bit_cast(uint32_t, value) & 0x7FFFFFFFu;
            not_finite |= bits >= 0x7F800000u;
            bits = bits < 0x7F800000u ? bits : 0u;
            const uint32_t exponent = bits ? (1u << 20) + uint32_t(exponent_over(value)) : 0u;
            most[e] = max(most[e], bits);
            sums[e] += exponent;
            row_most[j] = max(row_most[j], bits);
            row_sums[j] += exponent;
        }
        asm volatile("" : "+v"(row_most[j]), "+v"(row_sums[j]));  // a row at a time: what is made of all of them needs more registers
#pragma unroll
        for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(most[e]), "+v"(sums[e]));
    }
    uint32_t of_row = 0, sum_of_row = 0;
    if (p.row_most) {  // lane j of the first sixteen: of the wavefront's row j
        of_row = lanes_rows<3>(row_most, lane, [](uint32_t a, uint32_t b) { return max(a, b); });
        sum_of_row = lanes_rows<3>(row_sums, lane, [](uint32_t a, uint32_t b) { return a + b; });
        if (lane >= kRows) of_row = 0;
    }
    if (__ballot(not_finite) && lane == 0) unlike->not_finite = 1;  // whoever writes it, and whenever, it is one
    const auto add = [](uint32_t* most, unsigned long long* sums, uint32_t largest, uint32_t sum) {
        if (!largest) return;
        atomicMax(most, largest);
        atomicAdd(sums, (unsigned long long)(sum >> 20) << kCountShift | (sum & 0xFFFFFu));
    };
    add(&p.row_most[own], &p.row_sum[own], of_row, sum_of_row);  // a row past the end has none
    if (!column_most) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        of_column[wave][4 * lane + e] = most[e];
        sum_of_column[wave][4 * lane + e] = sums[e];
    }
    __syncthreads();
    const int64_t column = column0 + threadIdx.x;
    uint32_t all = of_column[0][threadIdx.x], sum = sum_of_column[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        all = max(all, of_column[w][threadIdx.x]);
        sum += sum_of_column[w][threadIdx.x];
    }
    if (column < columns) add(&column_most[column], &p.column_sum[column], all, sum);
}

// The most unlike rows, of maxima and sums in the order W's columns (whole_classes of them), W's rows (width), x's columns
// (width), x's rows, which are blockIdx.y in this order; what most_kernel was not asked for is zeros.
__global__ __launch_bounds__(256) void unlike_kernel(const uint32_t* __restrict__ most, const unsigned long long* __restrict__ sums,
                                                     int64_t whole_classes, int64_t width, int64_t rows, Unlike* __restrict__ unlike) {
    __shared__ int of_wave[4][2];
    const int group = blockIdx.y, lane = threadIdx.x % 64;
    const int64_t first = group == 0 ? 0 : whole_classes + (group - 1) * width, n = group == 0 ? whole_classes : group == 3 ? rows : width;
    if (int64_t(blockIdx.x) * 256 >= n) return;
    int found[2] = {0, 0};  // the gap, the exponent
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        const unsigned long long of = sums[first + i];
        const float values = float(of >> kCountShift);
        if (values == 0.0f) continue;
        const int exponent = exponent_over(__builtin_bit_cast(float, most[first + i]));
        // The mean is off by 2^-14 at most, a sixteenth is the unit.
        const float mean = float(of & ((1ull << kCountShift) - 1)) / values;
        found[0] = max(found[0], int(ceilf((float(exponent) - mean) * 16.0f + 0.01f)));
        found[1] = max(found[1], exponent);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int v = found[i];
        v = max(v, red::partner<0>(v, lane));
        v = max(v, red::partner<1>(v, lane));
        v = max(v, red::partner<2>(v, lane));
        v = max(v, red::partner<3>(v, lane));
        v = max(v, red::partner<4>(v, lane));
        v = max(v, red::partner<5>(v, lane));
        if (lane == 0) of_wave[threadIdx.x / 64][i] = v;
    }
    __syncthreads();
    if (threadIdx.x >= 2) return;
    int* const gap = group == 0 ? &unlike->w_columns : group == 1 ? &unlike->w_rows : group == 2 ? &unlike->x_columns : &unlike->x_rows;
    int* const to = threadIdx.x == 0 ? gap : group == 0 ? &unlike->w_most : group == 3 ? &unlike->x_most : nullptr;
    if (!to) return;
    const int v = max(max(of_wave[0][threadIdx.x], of_wave[1][threadIdx.x]), max(of_wave[2][threadIdx.x], of_wave[3][threadIdx.x]));
    // Most workgroups find nothing more: a look costs less than the atomic.
    if (v > __hip_atomic_load(to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(to, v);
}

// What a token's gradients are made of, from its logits' statistics.
struct Token {
    float most, scale;  // exp(z - most) * scale is the share of a class
    float others;       // the share of all classes but the target's, which is minus the target's gradient
    int target;
};

// The exponent of a class's gradients in a block of tokens: that of the largest, but no unit is smaller than 2^-82 of the one
// that the largest of all could have, so that sums of larger units, 2^44 at most, stay finite in it. A block without any has the
// smallest, in which no sum loses bits.
__device__ inline int class_exponent(uint32_t most, uint32_t most_share) {
    const int smallest = halves::exponent_of(most_share) + 82;
    return most == 0 ? smallest : min(halves::exponent_of(most), smallest);
}

constexpr int kGradientStride = kBlockTokens + 2;  // four threads that read eight classes of a token each meet different banks

// The gradients dz^T of a piece from its logits z^T [classes, stride]: times the tokens' shares, packed along the tokens, in
// their place (three parts: into by_class, in the unit of the largest share); and for shares of one packed along the classes, by_token.
// Either may be without memory. most [blocks][whole classes]: the largest of
// each class, as bits. Sums: of each class, into sums [blocks][classes]. A workgroup takes 32 classes and a block of tokens;
// four lanes of a wavefront read a line of the logits, and then write it.
template <bool Sums>
__global__ __launch_bounds__(256) void gradients_kernel(float* logits, int64_t stride, Piece piece, const Token* __restrict__ tokens,
                                                        const float* __restrict__ shares, const uint32_t* __restrict__ most_share,
                                                        int64_t classes, int64_t whole_classes, uint32_t* __restrict__ most,
                                                        thirds::Operand by_token, thirds::Operand by_class, int lines,
                                                        double* __restrict__ sums, int blocks, Form form) {
    __shared__ float tile[32][kGradientStride];
    const int64_t id = block_id(), block = id % blocks, v0 = id / blocks * 32;
    if (v0 >= classes) return;
    const int64_t t0 = block * kBlockTokens, n = piece.tokens();
    if (t0 >= n) {
        if constexpr (Sums)
            if (threadIdx.x < 32 && v0 + threadIdx.x < classes) sums[block * classes + v0 + threadIdx.x] = 0.0;
        return;
    }
    const int lane = threadIdx.x % 64, c = 8 * (threadIdx.x % 32);
    float* const at = logits + (v0 + threadIdx.x / 32) * stride + t0 + c;
    red::f4 z[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (v0 + threadIdx.x / 32 + 8 * j < classes) {
            z[j][0] = red::ld4(at + 8 * j * stride);
            z[j][1] = red::ld4(at + 8 * j * stride + 4);
        }
    Token token[8];
    float share[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        token[i] = t0 + c + i < n ? tokens[t0 + c + i] : Token{0.0f, 0.0f, 0.0f, -1};
        share[i] = t0 + c + i < n ? shares[t0 + c + i] : 0.0f;
    }
    const uint32_t top = most_share[0];
    const bool thirds = form.thirds();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = threadIdx.x / 32 + 8 * j;
        const int v = int(v0) + r;
        const bool there = v < classes;
        float d[8];
        uint32_t high = 0;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = exp_of(z[j][i / 4][i % 4] - token[i].most) * token[i].scale;
            const float g = token[i].target == v ? -token[i].others : e;
            const bool counts = there && token[i].target >= 0;
            tile[r][c + i] = counts ? g : 0.0f;
            d[i] = counts ? g * share[i] : 0.0f;
            const uint32_t bits = __builtin_bit_cast(uint32_t, d[i]) & 0x7FFFFFFFu;
            high = max(high, bits < 0x7F800000u ? bits : 0u);
            if constexpr (Sums) sum += double(d[i]);
        }
        high = max(high, red::partner<0>(high, lane));
        high = max(high, red::partner<1>(high, lane));
        high = max(high, red::partner<2>(high, lane));
        high = max(high, red::partner<3>(high, lane));
        high = max(high, red::partner<4>(high, lane));
        if constexpr (Sums) {
            sum += red::partner<0>(sum, lane);
            sum += red::partner<1>(sum, lane);
            sum += red::partner<2>(sum, lane);
            sum += red::partner<3>(sum, lane);
            sum += red::partner<4>(sum, lane);
        }
        if (!there) continue;
        if (thirds) {
            if (by_class.first) thirds::store8(by_class, int(stride / halves::kSlice), v, (t0 + c) / 8, d, halves::exponent_of(top));
        } else {
            h8 first, second;
            halves::split8(d, class_exponent(high, top), first, second);
            half* const to = reinterpret_cast<half*>(at - c % 32 + 8 * j * stride) + c % 32;
            *reinterpret_cast<h8*>(to) = first;
            *reinterpret_cast<h8*>(to + 32) = second;
        }
        if (threadIdx.x % 32 == 0) {
            most[block * whole_classes + v] = high;
            if constexpr (Sums) sums[block * classes + v] = sum;
        }
    }
    if (!by_token.first) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        // Three parts of neighbouring tokens lie next to each other, of two parts those of neighbouring classes.
        const int t = thirds ? int(threadIdx.x) : threadIdx.x / 4 + 64 * j, g = thirds ? j : threadIdx.x % 4;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[8 * g + i][t];
        const uint32_t others = t0 + t < n ? __builtin_bit_cast(uint32_t, tokens[t0 + t].others) : 0u;
        if (thirds) {
            thirds::store8(by_token, lines, t0 + t, v0 / 8 + g, v, halves::exponent_of(others));
            continue;
        }
        h8 first, second;
        halves::split8(v, halves::exponent_of(others), first, second);
        half* const to = by_token.first + ((t0 + t) * lines + v0 / 32) * 64 + 8 * g;
        *reinterpret_cast<h8*>(to) = first;
        *reinterpret_cast<h8*>(to + 32) = second;
    }
}

// ---- the products -----------------------------------------------------------------------

// z^T: scaled back, with the bias, stored for a gradient (Store); and of each 128 classes of a token the maximum, the sum of the
// exponentials over it but the target's, and the target's logit. exponents, bias and out reach to the end of the last tile.
//
// A sum that holds an infinity or a NaN is lost to the parts (infinity minus infinity): it is made again value by value, so a
// class whose weight is minus infinity has no chance, as in the other routes.
template <bool Store>
struct Logits {
    static constexpr bool kElementwise = false, kUnits = false;
    Piece piece;
    const int* exponents;
    const uint32_t* row_most;
    const float *bias, *targets;
    float *out, *most, *sum, *at_target;
    int64_t classes, stride;
    int lines;
    const float *x, *weight;
    int64_t width;
    Form form;
    __device__ inline int64_t rows_a() const { return classes; }
    __device__ inline int64_t rows_b() const { return piece.tokens(); }
    __device__ inline int depth() const { return lines; }
    __device__ inline bool idle() const { return false; }
    // Class v's logit of token t, without the bias.
    __device__ inline float again(int64_t v, int64_t t) const {
        const float *const row = x + piece.row(t) * width, *column = weight + v;
        float s = 0.0f;
        int64_t k = 0;
        for (; k + 8 <= width && s == s; k += 8) {
            float a[8], b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[i] = row[k + i];
                b[i] = column[(k + i) * classes];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s = __builtin_fmaf(a[i], b[i], s);
        }
        if (s != s) return s;
        for (; k < width; ++k) s = __builtin_fmaf(row[k], column[k * classes], s);
        return s;
    }
    // Sums of three parts that are lost, again, in place: of finite values none is, and again() gives an infinity or a NaN, which
    // no scale changes. Apart from the rest, whose registers it would take (253, 203).
    template <int Blocks>
    __device__ inline void restore(halves::f16v (&acc)[4][Blocks], int m, int n, int wave, int first) const {
        const auto finite = [](float v) { return fabsf(v) < __builtin_huge_valf(); };
        const int lane = threadIdx.x % 64;
        const int64_t v0 = int64_t(m) * halves::kTile + 128 * (wave / 4) + 4 * (lane / 32);
        const int64_t t0 = int64_t(n) * halves::kTile + 64 * (wave % 4) + 32 * first + lane % 32, tokens = piece.tokens();
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < Blocks; ++b) {
                bool lost = false;
#pragma unroll
                for (int i = 0; i < 16; ++i) lost |= !finite(acc[a][b][i]);
                if (!lost) continue;
#pragma unroll 1
                for (int l = 0; l < 16; ++l) {
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum = l == i ? acc[a][b][i] : sum;
                    if (finite(sum)) continue;
                    const int64_t v = v0 + 32 * a + 8 * (l / 4) + l % 4, t = t0 + 32 * b;
                    sum = v < classes && t < tokens ? again(v, t) : 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[a][b][i] = l == i ? sum : acc[a][b][i];
                }
            }
    }
    // Of wave `wave` of a tile: its blocks of 32 columns from block `first`.
    template <int Blocks>
    __device__ inline void operator()(const halves::f16v (&acc)[4][Blocks], int m, int n, int wave, int first) const {
        const int lane = threadIdx.x % 64, column = 64 * (wave % 4) + 32 * first + lane % 32;
        const int64_t v0 = int64_t(m) * halves::kTile, t0 = int64_t(n) * halves::kTile + column;
        const int64_t tokens = piece.tokens();
        const int row0 = 128 * (wave / 4) + 4 * (lane / 32);
        float top[Blocks], others[Blocks];
        int e_token[Blocks], target[Blocks];  // the target's row in this tile
#pragma unroll
        for (int b = 0; b < Blocks; ++b) {
            top[b] = kLowest;
            others[b] = 0.0f;
            const int64_t t = t0 + 32 * b;
            const int64_t row = t < tokens ? piece.row(t) : 0;
            e_token[b] = t < tokens ? halves::exponent_of(row_most[row]) : 0;
            const int64_t own = t < tokens ? class_of(targets[row], classes) - v0 : -1;
            target[b] = own >= 0 && own < halves::kTile ? int(own) : -1;
        }
        const int* const of_class = exponents + v0;
        const float* const of_bias = bias + v0;
        // A row of the tile is a scalar offset: 256 rows of at most 2^16 floats stay within a buffer's 31 bits.
        const __amdgpu_buffer_rsrc_t rows =
            __builtin_amdgcn_make_buffer_rsrc(out + v0 * stride + int64_t(n) * halves::kTile, short(0), 0x7FFFFFFE, 0x00020000);
        const uint32_t row_bytes = uint32_t(stride) * 4u, at = uint32_t(row0) * row_bytes + uint32_t(column) * 4u;
#pragma unroll
        for (int a = 0; a < 4; ++a) {       // 32 rows of the tile, 16 of this thread's, at a time:
            asm volatile("" ::: "memory");  // the exponents of all do not fit the registers
            const int r0 = 32 * a;
            int e[16];
            float add[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int4 of = *reinterpret_cast<const int4*>(of_class + row0 + r0 + 8 * g);
                const red::f4 more = red::ld4(of_bias + row0 + r0 + 8 * g);
                e[4 * g] = of.x;
                e[4 * g + 1] = of.y;
                e[4 * g + 2] = of.z;
                e[4 * g + 3] = of.w;
#pragma unroll
                for (int i = 0; i < 4; ++i) add[4 * g + i] = more[i];
            }
#pragma unroll
            for (int b = 0; b < Blocks; ++b) {
                int own = target[b] - row0 - r0;  // the target's among these rows, if it is
                float z[16], high = top[b], found = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 8 * (i / 4) + i % 4;
                    z[i] = __builtin_amdgcn_ldexpf(acc[a][b][i], -(e[i] + e_token[b])) + add[i];
                    if constexpr (Store)
                        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, z[i]), rows, at + 128u * b,
                                                              uint32_t(r0 + r) * row_bytes, 0);
                    found = own == r ? z[i] : found;
                    high = z[i] > high ? z[i] : high;
                }
                if (own >= 0 && own < 32 && (own & 4) == 0) at_target[t0 + 32 * b] = found;
                asm volatile("" : "+v"(own));  // the comparisons are cheaper made twice than kept
                // Sums without the target's exponential: beside a share near one the others' would lose their bits. The
                // maximum is no NaN; where all are minus infinity the exponentials over zero are zeros (or NaN).
                const float over = high == kLowest ? 0.0f : high;
                others[b] *= top[b] == high ? 1.0f : exp_of(top[b] - high);
#pragma unroll
                for (int i = 0; i < 16; ++i) others[b] += own == 8 * (i / 4) + i % 4 ? 0.0f : exp_of(z[i] - over);
                top[b] = high;
                asm volatile("" : "+v"(others[b]));  // here, not behind all the rows, whose logits would have to be kept
            }
        }
#pragma unroll
        for (int b = 0; b < Blocks; ++b) {
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

// The statistics of a piece's tokens from those of every 128 classes, their shares in a row, and their losses. A workgroup takes
// 64 tokens, wavefront w every sixteenth part.
constexpr int kTokenWaves = 16;
__global__ __launch_bounds__(64 * kTokenWaves) void token_kernel(Piece piece, const float* __restrict__ most,
                                                                 const float* __restrict__ sum, const float* __restrict__ at_target,
                                                                 const float* __restrict__ targets, int parts, int64_t stride,
                                                                 int64_t classes, const float* __restrict__ shares, bool one_share,
                                                                 Token* __restrict__ out, float* __restrict__ own_shares,
                                                                 float* __restrict__ losses) {
    __shared__ float tops[kTokenWaves][64];
    __shared__ double totals[kTokenWaves][64];
    const int64_t n = piece.tokens();
    if (int64_t(blockIdx.x) * 64 >= n) return;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t t = int64_t(blockIdx.x) * 64 + lane;  // below the stride
    float top = kLowest;
#pragma unroll 8
    for (int p = wave; p < parts; p += kTokenWaves) top = fmaxf(top, most[p * stride + t]);
    tops[wave][lane] = top;
    __syncthreads();
    for (int w = 0; w < kTokenWaves; ++w) top = fmaxf(top, tops[w][lane]);
    double others = 0.0;
#pragma unroll 8
    for (int p = wave; p < parts; p += kTokenWaves) {
        const float m = most[p * stride + t];
        others += double(sum[p * stride + t]) * (m == top ? 1.0 : double(exp_of(m - top)));
    }
    totals[wave][lane] = others;
    __syncthreads();
    if (wave != 0 || t >= n) return;
    for (int w = 1; w < kTokenWaves; ++w) others += totals[w][lane];
    const int64_t row = piece.row(t);
    const float at = at_target[t] - top;
    const double total = others + double(expf(at));
    if (losses) losses[row] = float(log(total) - double(at));
    if (!out) return;
    out[t] = Token{top, float(1.0 / total), float(others / total), int(class_of(targets[row], classes))};
    own_shares[t] = shares[one_share ? 0 : row];
}

// total[c] = what the pieces before left there, but for the first one, plus the piece's blocks; out: of the last one, or null.
__global__ __launch_bounds__(64 * red::kCombineWaves) void bias_kernel(const double* __restrict__ sums, int64_t blocks, int64_t classes,
                                                                       bool first, double* __restrict__ total, float* __restrict__ out) {
    __shared__ double of_wave[red::kCombineWaves][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = int64_t(blockIdx.x) * 64 + lane;
    double acc[1] = {0.0};
    if (c < classes) red::combine_waves<1>(sums, blocks, classes, c, wave, 0, acc);
    of_wave[wave][lane] = acc[0];
    __syncthreads();
    if (wave != 0 || c >= classes) return;
    double sum = of_wave[0][lane];
    for (int w = 1; w < red::kCombineWaves; ++w) sum += of_wave[w][lane];
    if (!first) sum += total[c];
    if (out) out[c] = float(sum);
    else total[c] = sum;
}

// dx [rows, width], times the tokens' shares.
struct InputGradient {
    static constexpr bool kElementwise = true, kUnits = false;
    Piece piece;
    const Token* of_token;
    const uint32_t* feature_most;
    const float* shares;
    float* out;
    int64_t width;
    int lines;
    __device__ inline int64_t rows_a() const { return piece.tokens(); }
    __device__ inline int64_t rows_b() const { return width; }
    __device__ inline int depth() const { return lines; }
    __device__ inline bool idle() const { return false; }
    __device__ inline void store(int m, int n, int r, int c, const float (&v)[4]) const {
        const int64_t t = int64_t(m) * halves::kTile + r, d = int64_t(n) * halves::kTile + c, tokens = piece.tokens();
        if (d >= width) return;
        const int e = halves::exponent_of(feature_most[d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (t + i >= tokens) continue;
            const int others = halves::exponent_of(__builtin_bit_cast(uint32_t, of_token[t + i].others));
            out[piece.row(t + i) * width + d] = __builtin_amdgcn_ldexpf(v[i], -(e + others)) * shares[t + i];
        }
    }
};

// dW [width, classes], added to what is there for all pieces but the first.
struct WeightGradient {
    static constexpr bool kElementwise = true, kUnits = true;
    Piece piece;
    const uint32_t *feature_most, *class_most, *most_share;
    float* out;
    int64_t width, classes, whole_classes;
    bool add;
    __device__ inline int64_t rows_a() const { return width; }
    __device__ inline int64_t rows_b() const { return classes; }
    __device__ inline int depth() const { return int((piece.tokens() + halves::kSlice - 1) / halves::kSlice); }
    __device__ inline bool idle() const { return add && piece.tokens() == 0; }
    __device__ inline void store(int m, int n, int r, int c, const float (&v)[4]) const {
        const int64_t d = int64_t(m) * halves::kTile + r, k = int64_t(n) * halves::kTile + c;
        if (k >= classes) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (d + i >= width) continue;
            float* const to = out + (d + i) * classes + k;
            const float g = __builtin_amdgcn_ldexpf(v[i], -halves::exponent_of(feature_most[d + i]));
            *to = add ? *to + g : g;
        }
    }
};

// lines: a row's of either operand, of which depth() are multiplied; b_thirds: b, if that is in three parts. The parts of split tiles
// go to partial, for join_kernel.
template <class Of>
__global__ __launch_bounds__(halves::kThreads) void product_kernel(thirds::Operand a, const half* __restrict__ b,
                                                                   thirds::Operand b_thirds, int lines, int places,
                                                                   float* __restrict__ partial, Of of, Form form) {
    extern __shared__ __attribute__((aligned(128))) char lds[];
    if (of.idle()) return;
    const int depth = of.depth();
    const halves::Tiles tiles = halves::tiles_of(of.rows_a(), of.rows_b(), depth, places);
    if (int(blockIdx.x) >= tiles.whole + tiles.rest * tiles.parts) return;
    const halves::Place at = halves::place_of(tiles, blockIdx.x);
    int begin = 0, end = depth;
    if (at.part >= 0) {  // in whole blocks of tokens, as a class's unit changes with them
        const int units = (depth + kBlockLines - 1) / kBlockLines;
        begin = int(int64_t(units) * at.part / tiles.parts) * kBlockLines;
        end = min(depth, int(int64_t(units) * (at.part + 1) / tiles.parts) * kBlockLines);
    }
    const int64_t of_tile = int64_t(lines) * halves::kTile * (halves::kLineBytes / 2);
    halves::Tile tile;
    tile.clear();
    if (form.thirds()) {
        thirds::accumulate(tile, thirds::tile_of(a, at.m, lines), thirds::tile_of(b_thirds, at.n, lines), begin, end, lds);
        if constexpr (!Of::kElementwise)
            if (at.part < 0) of.restore(tile.acc, at.m, at.n, int(threadIdx.x / 64), 0);
        if constexpr (Of::kUnits) {
            const int by = -halves::exponent_of(of.most_share[0]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i) tile.acc[r][j][i] = __builtin_amdgcn_ldexpf(tile.acc[r][j][i], by);
        }
    } else if constexpr (Of::kUnits) {
        // A thread's two columns of the tile, which are classes, and the exponents of their units.
        const uint32_t* const most = of.class_most + int64_t(at.n) * halves::kTile + 64 * (threadIdx.x / 64 % 4) + threadIdx.x % 32;
        const uint32_t top = of.most_share[0];
        const auto unit = [&](int s, int column) { return class_exponent(most[s / kBlockLines * of.whole_classes + 32 * column], top); };
        int now[2], next[2];  // the sums end in units of one
#pragma unroll
        for (int j = 0; j < 2; ++j) now[j] = begin < end ? unit(begin, j) : 0;
        tile.accumulate<kBlockLines>(
            a.first + at.m * of_tile, b + at.n * of_tile, lines, begin, end, lds,
            [&](int s) {
#pragma unroll
                for (int j = 0; j < 2; ++j) next[j] = s + kBlockLines < end ? unit(s + kBlockLines, j) : 0;
            },
            [&](int) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int by = next[j] - now[j];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int i = 0; i < 16; ++i) tile.acc[r][j][i] = __builtin_amdgcn_ldexpf(tile.acc[r][j][i], by);
                    now[j] = next[j];
                }
            });
    } else {
        tile.accumulate<0>(a.first + at.m * of_tile, b + at.n * of_tile, lines, begin, end, lds, [](int) {}, [](int) {});
    }
    if (at.part >= 0)
        tile.store_part(partial + int64_t(at.rest * tiles.parts + at.part) * halves::Tile::kValues * halves::kThreads);
    else if constexpr (Of::kElementwise)
        tile.each4([&](int r, int c, float(&v)[4]) { of.store(at.m, at.n, r, c, v); });
    else
        of(tile.acc, at.m, at.n, int(threadIdx.x / 64), 0);
}

// The split tiles of a product: a workgroup for four values of every thread, of results that are stored value by value, or for one
// of the two blocks of 32 columns of two waves. (48 tiles of five parts of the logits: 20 us, 35 with a workgroup for a tile.)
template <class Of>
constexpr int kJoinThreads = Of::kElementwise ? halves::kThreads : 128;
template <class Of>
constexpr int kJoinShares = Of::kElementwise ? halves::Tile::kValues / 4 : 2 * halves::kThreads / kJoinThreads<Of>;

template <class Of>
__global__ __launch_bounds__(kJoinThreads<Of>) void join_kernel(int places, const float* __restrict__ partial, Of of) {
    if (of.idle()) return;
    const halves::Tiles tiles = halves::tiles_of(of.rows_a(), of.rows_b(), of.depth(), places);
    for (int u = blockIdx.x; u < tiles.rest * kJoinShares<Of>; u += gridDim.x) {
        const int rest = u / kJoinShares<Of>, share = u % kJoinShares<Of>;
        const halves::Place at = halves::tile_at(tiles, tiles.whole + rest);
        const float* const from = partial + int64_t(rest * tiles.parts) * halves::Tile::kValues * halves::kThreads;
        if constexpr (Of::kElementwise) {
            halves::Tile::each_part(from, tiles.parts, share, [&](int r, int c, const float(&v)[4]) { of.store(at.m, at.n, r, c, v); });
        } else {
            const int thread = share / 2 * kJoinThreads<Of> + int(threadIdx.x);
            halves::f16v acc[4][1];
            halves::Tile::load_parts(from, tiles.parts, thread, share % 2, acc);
            if (of.form.thirds()) of.restore(acc, at.m, at.n, thread / 64, share % 2);
            of(acc, at.m, at.n, thread / 64, share % 2);
        }
    }
}

// ---- a few rows without gradients: the weights are read once -----------------------------
//
// Bound by reading W. A workgroup takes 128 classes, its wavefronts 16 features in turn, with their loads of 512 bytes in flight;
// what its rows' logits come to there is left as in the packed route, and joined by a second launch.

constexpr int kRowThreads = 256, kFewMost = 16, kFewWaves = 8, kFewClasses = 128, kFewLoads = 16;
constexpr int kFewFeatures = kFewWaves * kFewLoads;  // of a workgroup's turn

template <int Rows>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(const float* __restrict__ x, const float* __restrict__ weight,
                                                                  const float* __restrict__ bias, const float* __restrict__ targets,
                                                                  int rows, int64_t width, int64_t classes, float* __restrict__ most,
                                                                  float* __restrict__ sum, float* __restrict__ at_target) {
    __shared__ float part[kFewWaves][Rows][kFewClasses];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t v0 = int64_t(blockIdx.x) * kFewClasses, v = v0 + 2 * lane;
    // A pair past the end is read from the last two classes (or the only one twice) and never used.
    const int64_t first = min(v, classes - 1), second = min(v + 1, classes - 1);
    const bool pair = second == first + 1;
    float acc[Rows][2] = {};
    const auto add = [&](int64_t k, float a, float b) {
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            const float own = x[int64_t(min(r, rows - 1)) * width + k];
            acc[r][0] = __builtin_fmaf(own, a, acc[r][0]);
            acc[r][1] = __builtin_fmaf(own, b, acc[r][1]);
        }
    };
    typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));
    for (int64_t k = kFewLoads * wave; k < width; k += kFewFeatures) {
        if (k + kFewLoads <= width) {
            f2u w[kFewLoads];
#pragma unroll
            for (int u = 0; u < kFewLoads; ++u) {
                const float* const at = weight + (k + u) * classes;
                if (pair) w[u] = *reinterpret_cast<const f2u*>(at + first);
                else w[u] = f2u{at[first], at[second]};
            }
#pragma unroll
            for (int u = 0; u < kFewLoads; ++u) add(k + u, w[u][0], w[u][1]);
        } else {
            for (int64_t l = k; l < width; ++l) add(l, weight[l * classes + first], weight[l * classes + second]);
        }
    }
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        part[wave][r][2 * lane] = acc[r][0];
        part[wave][r][2 * lane + 1] = acc[r][1];
    }
    __syncthreads();
    for (int r = wave; r < rows; r += kFewWaves) {
        const int64_t target = class_of(targets[r], classes);
        float z[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = lane + 64 * i;
            z[i] = part[0][r][c];
#pragma unroll
            for (int w = 1; w < kFewWaves; ++w) z[i] += part[w][r][c];
            const bool there = v0 + c < classes;
            if (bias && there) z[i] += bias[v0 + c];
            if (!there) z[i] = kLowest;
            if (there && v0 + c == target) at_target[r] = z[i];
        }
        float top = z[0] > kLowest ? z[0] : kLowest;
        top = z[1] > top ? z[1] : top;
        const auto larger = [](float a, float b) { return b > a ? b : a; };
        top = larger(top, red::partner<0>(top, lane));
        top = larger(top, red::partner<1>(top, lane));
        top = larger(top, red::partner<2>(top, lane));
        top = larger(top, red::partner<3>(top, lane));
        top = larger(top, red::partner<4>(top, lane));
        top = larger(top, red::partner<5>(top, lane));
        const float over = top == kLowest ? 0.0f : top;
        float others = v0 + lane == target ? 0.0f : exp_of(z[0] - over);
        others += v0 + lane + 64 == target ? 0.0f : exp_of(z[1] - over);
        others += red::partner<0>(others, lane);
        others += red::partner<1>(others, lane);
        others += red::partner<2>(others, lane);
        others += red::partner<3>(others, lane);
        others += red::partner<4>(others, lane);
        others += red::partner<5>(others, lane);
        if (lane == 0) {
            most[int64_t(r) * gridDim.x + blockIdx.x] = top;
            sum[int64_t(r) * gridDim.x + blockIdx.x] = others;
        }
    }
}

// A workgroup a row.
__global__ __launch_bounds__(kRowThreads) void few_join_kernel(const float* __restrict__ most, const float* __restrict__ sum,
                                                               const float* __restrict__ at_target, const float* __restrict__ targets,
                                                               int parts, int64_t classes, float* __restrict__ losses) {
    __shared__ float tops[kRowThreads / 64];
    __shared__ double sums[kRowThreads / 64];
    const int64_t r = blockIdx.x;
    if (class_of(targets[r], classes) < 0) {
        if (threadIdx.x == 0) losses[r] = 0.0f;
        return;
    }
    float top = kLowest;
    for (int p = threadIdx.x; p < parts; p += kRowThreads) top = fmaxf(top, most[r * parts + p]);
    top = workgroup_max<kRowThreads>(top, tops);
    double others = 0.0;
    for (int p = threadIdx.x; p < parts; p += kRowThreads) {
        const float m = most[r * parts + p];
        others += double(sum[r * parts + p]) * (m == top ? 1.0 : double(exp_of(m - top)));
    }
    others = red::block_sum(others, sums);
    if (threadIdx.x != 0) return;
    const float at = at_target[r] - top;
    losses[r] = float(log(others + double(expf(at))) - double(at));
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

// Logits of a piece: 2^26 of them, 256 MiB.
size_t rows_of_piece(const Call& c) { return std::max<size_t>(1, std::min(c.rows, (size_t(1) << 26) / c.classes)); }

void product(const float* a, const float* b, float* c, size_t m, size_t k, size_t n, bool trans_a, bool trans_b) {
    const size_t none = 0;
    run(vc_hip_matmul(a, b, c, m, k, n, &none, &none, 1, trans_a, trans_b));
}

// Rows of a piece in whole. out's pointers are the piece's.
template <bool Gradient>
void rows_of(Device& d, float* z, const Call& c, const float* targets, const float* shares, bool one_share, size_t n, const RowOutputs& out) {
    // One workgroup a row is at most what the finishing count takes.
    const dim3 grid(unsigned(std::min<size_t>(n, std::min<size_t>(red::kMaxFinishBlocks, 16 * size_t(d.cu_count)))));
    const auto go = [&](auto kernel, int threads) {
        launch(kernel, grid, dim3(unsigned(threads)), 0, d.stream, z, c.bias, targets, shares, one_share, int64_t(n), int64_t(c.classes), out);
    };
    if (c.classes <= 256) go(logits_kernel<64, 1, Gradient>, 64);
    else if (c.classes <= 1024) go(logits_kernel<256, 1, Gradient>, 256);
    else if (c.classes <= 4096) go(logits_kernel<256, 4, Gradient>, 256);
    else if (c.classes <= 8192) go(logits_kernel<1024, 2, Gradient>, 1024);
    else go(logits_kernel<1024, 0, Gradient>, 1024);
    after_launch("linear_cross_entropy rows");
}

void count(Device& d, const Call& c, const float* shares, int* counted, float* share, int* place, uint32_t* most, float* losses,
           uint32_t* cleared = nullptr, int64_t n_cleared = 0) {
    const unsigned clearing = n_cleared > 0 ? grid_1d(size_t(n_cleared), kCountThreads, 64) : 0;
    launch(count_kernel, dim3(1 + clearing), dim3(kCountThreads), 0, d.stream, c.targets, shares, int64_t(c.rows), int64_t(c.classes),
           counted, share, place, most, losses, cleared, n_cleared);
    after_launch("linear_cross_entropy count");
}
void mean_of(Device& d, const Call& c, const float* losses, const float* share, float* mean) {
    launch(mean_kernel, dim3(1), dim3(kCountThreads), 0, d.stream, losses, int64_t(c.rows), share, mean);
    after_launch("linear_cross_entropy mean");
}

// The route of float32 products: logits, rows, and the gradients' two products. losses, mean and the gradients: any of them.
// shares: of each row, or null for those of the mean.
void direct(Device& d, const Call& c, const float* shares, float* losses, float* mean, float* grad_x, float* grad_weight,
            float* grad_bias) {
    const bool gradient = grad_x || grad_weight || grad_bias;
    const size_t piece = rows_of_piece(c), pieces = (c.rows + piece - 1) / piece;
    const bool counted_here = pieces == 1 && c.rows <= kCountedHere, added_here = mean && pieces == 1;
    const bool own_losses = mean && !added_here && !losses;  // the mean adds up the rows' losses, which the caller may want too
    Scratch share(sizeof(float)), losses_of_mean(own_losses ? c.rows * sizeof(float) : 4);
    Scratch partial(added_here ? red::kMaxFinishBlocks * sizeof(double) : 4);
    const bool count_first = !shares && (gradient || mean) && !counted_here;
    if (count_first) count(d, c, nullptr, nullptr, share.as<float>(), nullptr, nullptr, nullptr);
    if (own_losses) losses = losses_of_mean.as<float>();
    Scratch logits(piece * c.classes * sizeof(float)), rows(grad_weight ? piece * c.width * sizeof(float) : 4);
    Scratch more(pieces > 1 && gradient ? std::max(grad_weight ? c.width * c.classes : 0, c.classes) * sizeof(float) : 4);
    for (size_t r = 0; r < c.rows; r += piece) {
        const size_t n = std::min(piece, c.rows - r);
        const float* const x = c.x + r * c.width;
        float* const z = logits.as<float>();
        product(x, c.weight, z, n, c.width, c.classes, false, false);
        const RowOutputs out{losses ? losses + r : nullptr, grad_weight ? x : nullptr, rows.as<float>(), int64_t(c.width),
                             added_here ? mean : nullptr, partial.as<double>()};
        const float* const own = shares ? shares + r : count_first ? share.as<float>() : nullptr;
        if (!gradient) {
            rows_of<false>(d, z, c, c.targets + r, own, !shares, n, out);
            continue;
        }
        rows_of<true>(d, z, c, c.targets + r, own, !shares, n, out);
        if (grad_x) product(z, c.weight, grad_x + r * c.width, n, c.classes, c.width, false, true);
        if (grad_weight) {
            product(rows.as<float>(), z, r ? more.as<float>() : grad_weight, c.width, n, c.classes, true, false);
            if (r) run(vc_hip_axpy(grad_weight, more.as<float>(), c.width * c.classes, 1.0f));
        }
        if (grad_bias) {
            run(vc_hip_reduce_axis(z, r ? more.as<float>() : grad_bias, 1, n, c.classes, VC_REDUCE_SUM));
            if (r) run(vc_hip_axpy(grad_bias, more.as<float>(), c.classes, 1.0f));
        }
    }
    if (mean && !added_here) mean_of(d, c, losses, share.as<float>(), mean);
}

int64_t whole_tiles(int64_t n) { return (n + halves::kTile - 1) / halves::kTile * halves::kTile; }
int64_t lines_of(int64_t n) { return (n + halves::kSlice - 1) / halves::kSlice; }
// Memory of a packed matrix of `rows` rows of `depth` values, if it is wanted. The third parts lie apart, so that two parts lie as
// if there were none (in one buffer of 1.5 times the size, 256 rows, 1024 x 50000 took 6 us more to pack and 11 to multiply).
struct Packed {
    Scratch first, third;
    bool wanted;
    static size_t third_bytes(int64_t rows, int64_t depth) {
        return size_t(whole_tiles(rows) / halves::kTile) * size_t(thirds::third_bytes(int(lines_of(depth))));
    }
    Packed(int64_t rows, int64_t depth, bool want)
        : first(want ? 2 * third_bytes(rows, depth) : 4), third(want ? third_bytes(rows, depth) : 4), wanted(want) {}
    thirds::Operand operand() const { return wanted ? thirds::Operand{first.as<half>(), third.as<half>()} : thirds::Operand{nullptr, nullptr}; }
};

// A product of at most these rows; partial: room for one split tile a CU.
template <class Of>
void product_of(Device& d, const thirds::Operand& a, const half* b, const thirds::Operand& b_thirds, int64_t rows_a, int64_t rows_b,
                int64_t lines, float* partial, const Of& of, const Form& form) {
    constexpr int kLds = std::max(halves::Tile::kLds, thirds::kLds);
    const int64_t blocks = halves::most_blocks(rows_a, rows_b, d.cu_count);
    if (blocks > int64_t(1) << 22) fail(VC_HIP_ERR_OVERFLOW, "linear_cross_entropy: too many tiles");
    static const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(product_kernel<Of>),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    check_hip(allowed, "hipFuncSetAttribute");
    launch(product_kernel<Of>, dim3(unsigned(blocks)), dim3(halves::kThreads), uint32_t(kLds), d.stream, a, b, b_thirds, int(lines),
           d.cu_count, partial, of, form);
    after_launch("linear_cross_entropy product");
    if (lines < halves::kLeastSplit) return;
    launch(join_kernel<Of>, dim3(unsigned(d.cu_count) * (Of::kElementwise ? 4u : 8u)), dim3(kJoinThreads<Of>), 0, d.stream, d.cu_count,
           static_cast<const float*>(partial), of);
    after_launch("linear_cross_entropy join");
}

Packing packing(const float* values, const Piece& of, int64_t rows, int64_t columns, const uint32_t* row_most,
                const uint32_t* column_most, const thirds::Operand& by_row, const thirds::Operand& by_column) {
    const int64_t down = (by_row.first ? whole_tiles(rows) : lines_of(rows) * 32) / kPackRows, across = whole_tiles(columns) / kPackColumns;
    return Packing{values, of, rows, columns, row_most, column_most, by_row, by_column, int(lines_of(columns)), int(lines_of(rows)),
                   int(down), int(across), nullptr, nullptr, nullptr};
}
void pack(Device& d, const Packing& one, const Packing& two, const Form& form) {
    launch(pack_kernel, grid_2d(one.blocks() + two.blocks()), dim3(kPackThreads), 0, d.stream, one, two, form);
    after_launch("linear_cross_entropy pack");
}

// sums - most: of the arrays' sums and maxima, which lie in the same order.
Largest largest(const float* values, const float* targets, size_t rows, size_t columns, uint32_t* most, unsigned long long* sums,
                uint32_t* row_most, uint32_t* column_most, float* cleared) {
    const auto sums_of = [&](uint32_t* of) { return of ? sums + (of - most) : nullptr; };
    return Largest{values, targets, int64_t(rows), int64_t(columns), int((rows + kMostRows - 1) / kMostRows),
                   int((columns + kMostColumns - 1) / kMostColumns), row_most, column_most, sums_of(row_most), sums_of(column_most), cleared};
}

// The packed route. shares: of each row, or null for those of the mean, which goes to share[0]. losses and, of a gradient, any
// output may be null.
//
// A piece's logits take 4 bytes a value, their packed gradients 6 for each of x and W: 2 GiB and 6 GiB at most, of 288.
void packed(Device& d, const Call& c, const float* shares, float* share, float* losses, float* grad_x, float* grad_weight,
            float* grad_bias) {
    const bool gradient = grad_x || grad_weight || grad_bias;
    const int64_t width = int64_t(c.width), classes = int64_t(c.classes), rows = int64_t(c.rows);
    const int64_t whole_classes = whole_tiles(classes);
    const int64_t fitting = gradient ? (int64_t(1) << 29) / whole_classes / halves::kTile * halves::kTile : 65536;  // classes < 2^21
    const int64_t most_rows = std::min<int64_t>(fitting, 65536), pieces = (rows + most_rows - 1) / most_rows;
    const int64_t piece = whole_tiles((rows + pieces - 1) / pieces);
    const int64_t parts = 2 * whole_classes / halves::kTile, blocks = piece / kBlockTokens;

    // Of W's rows and columns and x's rows and columns the sums of exponents and the largest magnitudes, behind what they come to,
    // and the largest of the shares.
    const int64_t n_most = 2 * width + whole_classes + rows, cleared = 8 + 3 * n_most;  // words
    static_assert(sizeof(Unlike) <= 8 * sizeof(uint32_t));
    Scratch most(size_t(cleared + 1) * sizeof(uint32_t)), numbers(size_t(rows + 1) * sizeof(int));
    Unlike* const unlike = most.as<Unlike>();
    auto* const exponent_sums = reinterpret_cast<unsigned long long*>(most.as<uint32_t>() + 8);
    uint32_t* const maxima = most.as<uint32_t>() + 8 + 2 * n_most;
    uint32_t *const w_columns = maxima, *const w_rows = w_columns + whole_classes, *const x_columns = w_rows + width;
    uint32_t *const x_rows = x_columns + width, *const most_share = x_rows + rows;
    int *const counted = numbers.as<int>(), *const place = counted + 1;
    count(d, c, shares, counted, share, place, gradient ? most_share : nullptr, losses, most.as<uint32_t>(), cleared);
    const Largest of_w = largest(c.weight, nullptr, c.width, c.classes, maxima, exponent_sums, grad_x ? w_rows : nullptr, w_columns,
                                 nullptr);
    const Largest of_x = largest(c.x, c.targets, c.rows, c.width, maxima, exponent_sums, x_rows, grad_weight ? x_columns : nullptr,
                                 grad_x);
    launch(most_kernel, grid_2d(of_w.blocks() + of_x.blocks()), dim3(256), 0, d.stream, of_w, of_x, classes, unlike);
    after_launch("linear_cross_entropy largest");
    launch(unlike_kernel, dim3(grid_1d(size_t(std::max({whole_classes, width, rows})), 256, 256), 4), dim3(256), 0, d.stream, static_cast<const uint32_t*>(maxima),
           static_cast<const unsigned long long*>(exponent_sums), whole_classes, width, rows, unlike);
    after_launch("linear_cross_entropy unlike");
    int width_bits = 0;
    while ((int64_t(1) << width_bits) < width) ++width_bits;
    const Form form{unlike, width_bits};
    Scratch of_class(size_t(2 * whole_classes) * sizeof(float));
    int* const exponents = of_class.as<int>();
    float* const bias = of_class.as<float>() + whole_classes;

    const Packed wt(classes, width, true), w(width, classes, grad_x);
    Packing of_weight = packing(c.weight, Piece{}, width, classes, w_rows, w_columns, w.operand(), wt.operand());
    of_weight.bias = c.bias;
    of_weight.exponents = exponents;
    of_weight.filled = bias;

    const Packed x(piece, width, true), xt(width, piece, grad_weight), z(piece, classes, grad_x);
    const Packed zt(classes, piece, grad_weight);  // three parts: two take the place of the logits
    Scratch logits(gradient ? size_t(whole_classes * piece) * sizeof(float) : 4);
    Scratch statistics(size_t(2 * parts + 2) * size_t(piece) * sizeof(float)), tokens(size_t(piece) * sizeof(Token));
    Scratch class_most(gradient ? size_t(blocks * whole_classes) * sizeof(uint32_t) : 4);
    Scratch sums(grad_bias ? size_t((blocks + 1) * classes) * sizeof(double) : 4);
    double* const bias_total = sums.as<double>() + blocks * classes;
    Scratch partial(size_t(d.cu_count) * halves::Tile::kValues * halves::kThreads * sizeof(float));
    float *const part_most = statistics.as<float>(), *const part_sum = part_most + parts * piece;
    float *const at_target = part_sum + parts * piece, *const own_shares = at_target + piece;

    for (int64_t p = 0; p < pieces; ++p) {
        const Piece of{counted, place, p * piece, piece};
        const Packing of_rows = packing(c.x, of, piece, width, x_rows, x_columns, x.operand(), xt.operand());
        pack(d, of_rows, p == 0 ? of_weight : Packing{}, form);
        const auto z_of = [&](auto store) {
            product_of(d, wt.operand(), x.operand().first, x.operand(), classes, piece, lines_of(width), partial.as<float>(),
                       Logits<store()>{of, exponents, x_rows, bias, c.targets, logits.as<float>(), part_most, part_sum, at_target, classes,
                                       piece, int(lines_of(width)), c.x, c.weight, width, form},
                       form);
        };
        gradient ? z_of(std::true_type{}) : z_of(std::false_type{});
        launch(token_kernel, dim3(unsigned(piece / 64)), dim3(64 * kTokenWaves), 0, d.stream, of, part_most, part_sum, at_target, c.targets,
               int(parts), piece, classes, shares ? shares : share, !shares, gradient ? tokens.as<Token>() : nullptr, own_shares, losses);
        after_launch("linear_cross_entropy tokens");
        if (!gradient) continue;
        const auto gradients = grad_bias ? gradients_kernel<true> : gradients_kernel<false>;
        launch(gradients, grid_2d(size_t(blocks * lines_of(classes))), dim3(256), 0, d.stream, logits.as<float>(), piece, of,
               tokens.as<Token>(), own_shares, most_share, classes, whole_classes, class_most.as<uint32_t>(),
               z.operand(), zt.operand(), int(lines_of(classes)),
               sums.as<double>(), int(blocks), form);
        after_launch("linear_cross_entropy gradients");
        if (grad_bias) {
            launch(bias_kernel, dim3(unsigned((classes + 63) / 64)), dim3(64 * red::kCombineWaves), 0, d.stream,
                   static_cast<const double*>(sums.as<double>()), blocks, classes, p == 0, bias_total, p + 1 == pieces ? grad_bias : nullptr);
            after_launch("linear_cross_entropy bias");
        }
        if (grad_x)
            product_of(d, z.operand(), w.operand().first, w.operand(), piece, width, lines_of(classes), partial.as<float>(),
                       InputGradient{of, tokens.as<Token>(), w_rows, own_shares, grad_x, width, int(lines_of(classes))}, form);
        if (grad_weight)
            product_of(d, xt.operand(), logits.as<half>(), zt.operand(), width, classes, piece / halves::kSlice, partial.as<float>(),
                       WeightGradient{of, x_columns, class_most.as<uint32_t>(), most_share, grad_weight, width, classes, whole_classes,
                                      p > 0},
                       form);
    }
}

void few_rows(Device& d, const Call& c, float* losses) {
    const size_t parts = (c.classes + kFewClasses - 1) / kFewClasses;
    Scratch statistics((2 * parts + 1) * c.rows * sizeof(float));
    float *const most = statistics.as<float>(), *const sum = most + parts * c.rows, *const at_target = sum + parts * c.rows;
    const auto kernel = c.rows == 1   ? few_rows_kernel<1>
                        : c.rows == 2 ? few_rows_kernel<2>
                        : c.rows <= 4 ? few_rows_kernel<4>
                        : c.rows <= 8 ? few_rows_kernel<8>
                                      : few_rows_kernel<16>;
    launch(kernel, dim3(unsigned(parts)), dim3(64 * kFewWaves), 0, d.stream, c.x, c.weight, c.bias, c.targets, int(c.rows),
           int64_t(c.width), int64_t(c.classes), most, sum, at_target);
    after_launch("linear_cross_entropy few rows");
    launch(few_join_kernel, dim3(unsigned(c.rows)), dim3(kRowThreads), 0, d.stream, most, sum, at_target, c.targets, int(parts),
           int64_t(c.classes), losses);
    after_launch("linear_cross_entropy few rows");
}

// Whether reading the weight once for a few rows pays, by estimates of this route's time and that of float32 products in us. A
// workgroup walks all features of its 128 classes, 128 features in 1.6 us or more, so few classes leave most CUs idle for long.
// Measured, this route and products: 1 row, 1024 x 50000: 39, 56 us; 1024 x 16000: 16, 21; 1024 x 4000: 18, 13; 4096 x 10: 51, 10;
// 65536 x 10: 740, 19. 8 rows, 1024 x 50000: 44, 57; 512 x 16000: 15.7, 16.0; 128 x 400: 8.9, 9.7; 2048 x 1000: 41, 11. 16 rows,
// 512 x 50000: 37, 39; 1024 x 50000: 62, 57; 16 x 128: 9.8, 8.2.
bool takes_few(const Device& d, const Call& c) {
    if (c.rows > kFewMost) return false;
    const double rows = double(c.rows), bytes = 4.0 * double(c.width) * double(c.classes);
    const double groups = double((c.classes + kFewClasses - 1) / kFewClasses), turns = double((c.width + kFewFeatures - 1) / kFewFeatures);
    const double few = 5.5 + std::max(bytes / 5.5e6, turns * (1.6 + 0.009 * rows * rows) * std::max(1.0, groups / double(d.cu_count)));
    return few < 0.9 * (9.0 + bytes / 5.0e6 + 1.2e-4 * double(c.classes));
}

// A packed product's time in us, of `tiles` tiles of `lines` lines on `places` CUs, by what tiles_of makes of it.
double product_time(int64_t tiles, int64_t lines, int64_t places) {
    const int64_t rest = tiles % places;
    const double line = 2.5;
    double time = 4.0 + line * double(lines) * double(tiles / places);
    if (rest == 0) return time;
    const int64_t parts = lines >= halves::kLeastSplit ? std::min(places / rest, lines / 8) : 1;
    const bool split = parts > 1 && 50 * lines * (parts - 1) > parts * (100 + 2 * rest * parts);
    return time + line * double(lines) / double(split ? parts : 1) + (split ? 16.0 : 0.0);
}

// Whether packing pays: by estimates of both routes' times in us, for the gradients that are wanted. Measured (estimated), direct
// and packed, in us: losses alone of 128 rows, 1024 x 50000: 163 (144), 220 (217); of 256: 259 (279), 222 (217); 999, 515 x 10007:
// 162 (181), 79 (88); 4096, 256 x 1000: 43 (36), 51 (57); 2135, 1719 x 466: 51 (63), 81 (81). Train steps of 128 rows, 1024 x 50000:
// 460 (423), 567 (490); of 256: 773 (827), 612 (553); 2048, 1024 x 1024: 162 (152), 149 (183); 2135, 1719 x 466: 163 (180), 202
// (189); 1590, 1518 x 1016: 211 (250), 166 (185); 3145, 18 x 25838: 489 (519), 629 (626), with a bias, a tenth of the rows left out,
// 659 (673), 592 (626); 4096, 96 x 10000: 386 (429), 366 (364); 16384, 256 x 1000: 283 (333), 234 (224). The gradient of x alone, 256
// rows, 1024 x 50000: 522 (558), 424 (398); of the weight alone, 4096, 96 x 10000: 283 (293), 226 (257); of the bias alone, 4096, 96
// x 10000: 246 (234), 157 (145); 2048, 512 x 2048: 78 (75), 82 (91); 8192, 1024 x 5000: 885 (958), 384 (363).
bool takes_packed(const Device& d, const Call& c, bool of_x, bool of_weight, bool of_bias) {
    if (c.classes >= (size_t(1) << 21) || c.width >= (size_t(1) << 21)) return false;  // a load's offset has 31 bits
    if (c.rows >= kMostCounted) return false;
    const bool gradient = of_x || of_weight || of_bias, aligned = c.width % 4 == 0 && c.classes % 4 == 0;
    const double n = double(c.rows), weights = double(c.width) * double(c.classes), logits = n * double(c.classes);
    const double products = 1.0 + of_x + of_weight;
    const double direct = (gradient ? 20.0 : 10.0) + 2e-6 * products * n * weights / (aligned ? 105.0 : 66.0) +
                          (1.5e-6 * products + (of_bias ? 1.9e-6 : 0.0)) * logits;
    const int64_t rows = whole_tiles(int64_t(c.rows)) / halves::kTile, features = whole_tiles(int64_t(c.width)) / halves::kTile;
    const int64_t classes = whole_tiles(int64_t(c.classes)) / halves::kTile;
    double packed = 30.0 + (0.9e-6 + 1.1e-6 * products) * (weights + n * double(c.width)) +
                    product_time(classes * rows, lines_of(int64_t(c.width)), d.cu_count);
    if (gradient) packed += 4.0 * products + (1.2e-6 + 0.8e-6 * products) * logits;
    if (of_x) packed += product_time(rows * features, lines_of(int64_t(c.classes)), d.cu_count);
    if (of_weight) packed += product_time(features * classes, lines_of(int64_t(c.rows)), d.cu_count);
    return direct > packed;
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
        const bool few = takes_few(d, c);
        if (!few && !takes_packed(d, c, false, false, false)) {
            direct(d, c, nullptr, losses, mean, nullptr, nullptr, nullptr);
        } else {
            Scratch own(losses ? 4 : rows * sizeof(float)), share(sizeof(float));
            if (!losses) losses = own.as<float>();
            if (few) {
                few_rows(d, c, losses);
                if (mean) count(d, c, nullptr, nullptr, share.as<float>(), nullptr, nullptr, nullptr);
            } else {
                packed(d, c, nullptr, share.as<float>(), losses, nullptr, nullptr, nullptr);
            }
            if (mean) mean_of(d, c, losses, share.as<float>(), mean);
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
        if (takes_packed(d, c, grad_x, grad_weight, grad_bias)) {
            Scratch share(sizeof(float)), losses(mean ? rows * sizeof(float) : 4);
            packed(d, c, shares, share.as<float>(), mean ? losses.as<float>() : nullptr, grad_x, grad_weight, grad_bias);
            if (mean) mean_of(d, c, losses.as<float>(), share.as<float>(), mean);
        } else {
            direct(d, c, shares, nullptr, mean, grad_x, grad_weight, grad_bias);
        }
        p.done();
    });
}

}  // extern "C"
