// Orthogonalised momentum updates of weight matrices.
//
// With U = U S V^T the singular value decomposition of an update, the step is
// U V^T, approached without one: X = U / ||U|| and, `steps` times,
//   X <- a X + (b G + c G G) X,   G = X X^T (or X <- a X + X (b G + c G G), G = X^T X for a tall X),
// which maps every singular value s to a s + b s^3 + c s^5, at most 1.21. An
// iteration is three products over the longer side n and the shorter m: G and
// P = b G + c G G, symmetric, of which the tiles on and above the diagonal are
// computed and stored twice, and a X + P X: m m n + m m m + 2 m m n operations.
//
// All values stay near one by construction (|x| <= 1.21, |g| <= 1.5, |p| <= 3; G and
// P are held around an identity from some iteration on, see Quintic),
// so the products run as three half-precision products of two parts each
// (packed_product.hpp), on values scaled by 2^14 in memory: below 2^15.6 they are
// in half precision's range, and a part below its smallest step is 2^-38 of one.
// The error relative to the norm, which is what the iteration keeps of its input, is
// no larger than that of float32 products (test_muon_precision.py), at half of it for
// most shapes. The scale is a power of two and costs nothing.
//
// Every iterate is written twice, as X (of X and X^T the one with the shorter
// side first) and transposed, as the products read it along the shared side.
//
// All matrices of a call run in the same launches, three an iteration: a train
// step's matrices fill the chip together, and small ones share the latency.
//
// Bound by the matrix instructions where matrices are large: 1024 x 4096, 4096 x
// 4096 and 4096 x 1000 take 453 us for the last product of an iteration (340
// TFLOP/s), 277 for G (279) and 232 for P (305), of 408 TFLOP/s that a third of
// the library's half-precision rate would be; the update and the first split
// are 88 and 80 us (4.3 TB/s). Small ones are bound by the latency of a launch and its
// first loads: 784 x 256 and 256 x 10 take 25 us an iteration.
#include "packed_product.hpp"
#include "reduce_common.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

namespace vchip {
namespace {

constexpr float kScale = 16384.0f;

// a, b and c of an iteration around G = H + shift: a X + (b G + c G G) X is
// (a + b shift + c shift^2) X + ((b + 2 c shift) H + c H H) X. The first iterations
// bring singular values up from far below one, and G holds them best. In later ones
// most are near one, where a X and P X cancel to a fifth, and a rounding of P
// counts five times; with shift 1 nothing cancels and P is small. So is H's
// diagonal, beside whose squares the matrix instructions cut the other products of
// a sum short, always to one side (G G: 2 ulp of each diagonal element). 26 x 3266,
// error relative to the norm: 2.4e-6 with shift 0 throughout, 8.3e-7 so.
constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;
struct Quintic {
    float a, b, c, shift;
};
__device__ inline Quintic quintic_of(bool shifted) {
    return shifted ? Quintic{float(kA + kB + kC), float(kB + 2.0 * kC), float(kC), 1.0f} : Quintic{float(kA), float(kB), float(kC), 0.0f};
}
// The first iteration with shift 1: where equal singular values, 1 / sqrt(shorter)
// at first, have passed sqrt(1/2), the third at the latest, which the largest of
// unlike ones reach by then.
int turn_of(int64_t shorter) {
    double s = 1.0 / std::sqrt(double(shorter));
    int step = 0;
    for (; step < 2 && s * s < 0.5; ++step) s *= kA + s * s * (kB + s * s * kC);
    return step;
}
constexpr int kNormBlocks = 1024;  // partial sums of squares of a matrix, at most
constexpr int kAtOnce = 12;       // matrices (or batches of equal ones) of a launch
constexpr int kMostSplit = 2048;  // tiles of a launch whose sums are split
using packed::place;
using packed::half;

// `count` matrices [rows, cols].
struct Matrix {
    const float* grad;
    float *momentum, *param;  // null for a plain iterate
    float *update, *out;      // what is orthogonalised; the plain iterate's result
    half *x, *xt, *y, *yt;    // the scaled iterate [shorter, longer] and its transpose; the next one
    half *gram, *poly;        // [shorter, shorter]
    double* partials;
    int64_t rows, cols, shorter, longer;  // the sides are padded to whole tiles
    int count, blocks, turn;  // turn: of the iterations, see turn_of
    float rate;
    // Of the launch: the first workgroup (or die's); the tiles from `from`; parts of each one's sum; split tiles and parts before.
    int first, from, tiles, splits, counters, parts;

    __host__ __device__ int64_t elements() const { return rows * cols; }
    __host__ __device__ bool wide() const { return rows <= cols; }
};
struct Batch {
    Matrix of[kAtOnce + 1];  // of a product: also the tiles of the last round
    int n;
};

__device__ inline int find(const Batch& batch, int block) {
    int i = 0;
    while (i + 1 < batch.n && block >= batch.of[i + 1].first) ++i;
    return i;
}

// x = g + mu * m after m = mu * m + g, or x = g; the squares of x are summed in
// double, a partial for each workgroup, in a fixed order.
__global__ __launch_bounds__(256) void update_kernel(Batch batch, float mu) {
    __shared__ double sums[4];
    const Matrix& m = batch.of[find(batch, blockIdx.x)];
    const int block = (blockIdx.x - m.first) % m.blocks, z = (blockIdx.x - m.first) / m.blocks;
    const int64_t count = m.elements(), base = z * count;
    const float* const grad = m.grad + base;
    float *const momentum = m.momentum ? m.momentum + base : nullptr, *const x = m.update + base;
    double sum = 0.0;
    for (int64_t i = int64_t(block) * 256 + threadIdx.x; i < count; i += int64_t(m.blocks) * 256) {
        float v = grad[i];
        if (momentum) {
            const float next = momentum[i] * mu + v;
            momentum[i] = next;
            v = v + mu * next;
        }
        x[i] = v;
        sum += double(v) * double(v);
    }
    sum = red::wave_sum(sum);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) m.partials[z * m.blocks + block] = sums[0] + sums[1] + sums[2] + sums[3];
}

// 1 / ||update|| (0 for zeros), by the whole workgroup.
__device__ inline double inverse_norm(const Matrix& m, int z) {
    __shared__ double sums[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < m.blocks; i += 256) sum += m.partials[z * m.blocks + i];
    sum = red::wave_sum(sum);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    const double norm = sqrt(sums[0] + sums[1] + sums[2] + sums[3]);
    return norm == 0.0 ? 0.0 : 1.0 / norm;
}

// The first iterate without a step: out = update / ||update||.
__global__ __launch_bounds__(256) void normalise_kernel(Batch batch) {
    const Matrix& m = batch.of[find(batch, blockIdx.x)];
    const int block = (blockIdx.x - m.first) % m.blocks, z = (blockIdx.x - m.first) / m.blocks;
    const double factor = inverse_norm(m, z);
    const int64_t count = m.elements();
    for (int64_t i = int64_t(block) * 256 + threadIdx.x; i < count; i += int64_t(m.blocks) * 256)
        m.out[z * count + i] = float(double(m.update[z * count + i]) * factor);
}

// x = kScale * update / ||update|| and its transpose, a 64 x 64 tile of both a workgroup.
__global__ __launch_bounds__(256) void pack_kernel(Batch batch) {
    __shared__ float tile[64][65];  // [shorter][longer]
    const Matrix& m = batch.of[find(batch, blockIdx.x)];
    const int64_t across = m.longer / 64, tiles = across * (m.shorter / 64);
    const int64_t id = int(blockIdx.x) - m.first, z = id / tiles;
    const int64_t s0 = id % tiles / across * 64, l0 = id % across * 64;
    const float* const from = m.update + z * m.elements();
    const bool wide = m.wide();
    float line[16];  // of the update, read before the norm is known
#pragma unroll
    for (int n = 0; n < 16; ++n) {
        const int64_t row = (wide ? s0 : l0) + threadIdx.x / 64 + 4 * n, col = (wide ? l0 : s0) + threadIdx.x % 64;
        line[n] = row < m.rows && col < m.cols ? from[row * m.cols + col] : 0.0f;
    }
    const double factor = double(kScale) * inverse_norm(m, int(z));
#pragma unroll
    for (int n = 0; n < 16; ++n) {
        const float v = float(double(line[n]) * factor);
        const int i = threadIdx.x / 64 + 4 * n;
        if (wide) tile[i][threadIdx.x % 64] = v;
        else tile[threadIdx.x % 64][i] = v;
    }
    __syncthreads();
    half *const x = m.x + z * 2 * m.shorter * m.longer, *const xt = m.xt + z * 2 * m.shorter * m.longer;
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int row = i / 16, k = i % 16 * 4;
        float v[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = tile[row][k + e];
            w[e] = tile[k + e][row];
        }
        packed::store4(x + place(s0 + row, l0 + k, m.longer), v);
        packed::store4(xt + place(l0 + row, s0 + k, m.shorter), w);
    }
}

// ---- small matrices -----------------------------------------------------------------
// Up to 64 by 256 or 32 by 512: a workgroup takes a matrix through the whole call in LDS, in
// 32 x 32 tiles on the float32 matrix instructions, whose lane l holds row (of A)
// or column (of B) l % 32 at k = l / 32. Which k meet is free as long as both
// sides agree, so a lane reads four neighbouring ones at once.
//
// Five iterations, this and in tiles: 10 x 7 20 and 67 us, 64 x 64 39 and 72, 64 x
// 256 80 and 83; 300 of 64 x 128 97 and 261. Bound by the chain of three products
// and barriers on one CU; only for calls of such matrices alone, as next to larger
// ones the tiles of small ones cost nothing.

constexpr size_t kMostSteps = 64;  // of one launch
constexpr int kShort = 64, kLong = 256, kSquareStride = kShort + 4;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

__device__ inline f16v multiply4(f4 a, f4 b, f16v c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
// C += A B^T of 32 rows each, over k in [begin, end), multiples of 8.
__device__ inline f16v multiply_rows(const float* a, const float* b, int stride, int begin, int end, f16v c) {
    const int lane = red::lane_id(), at = lane % 32 * stride + lane / 32 * 4;
#pragma unroll 2
    for (int k = begin; k < end; k += 8)
        c = multiply4(*reinterpret_cast<const f4*>(a + at + k), *reinterpret_cast<const f4*>(b + at + k), c);
    return c;
}
// f(row, column, value) of a tile's values.
template <class F>
__device__ inline void each_value(const f16v& c, F&& f) {
    const int lane = red::lane_id();
#pragma unroll
    for (int e = 0; e < 16; ++e) f(e / 4 * 8 + lane / 32 * 4 + e % 4, lane % 32, c[e]);
}

__global__ __launch_bounds__(256) void small_kernel(Batch batch, float mu, float keep, int steps) {
    __shared__ __align__(16) float x[kShort * (kLong + 4)], g[kShort * kSquareStride], q[kShort * kSquareStride];
    __shared__ double sums[4];
    const Matrix& m = batch.of[find(batch, blockIdx.x)];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int rows = int(m.rows), cols = int(m.cols), count = rows * cols;
    const bool wide = m.wide();
    const int tall_tiles = ((wide ? rows : cols) + 31) / 32, long_tiles = ((wide ? cols : rows) + 31) / 32;
    const int stride = tall_tiles == 2 ? kLong + 4 : 2 * kLong + 4;  // rows of 16-byte groups that meet different banks
    const int64_t base = int64_t(int(blockIdx.x) - m.first) * count;
    for (int i = threadIdx.x; i < tall_tiles * 32 * stride; i += 256) x[i] = 0.0f;
    __syncthreads();
    const auto at = [&](int i) {
        const int row = i / cols, col = i - row * cols;
        return wide ? row * stride + col : col * stride + row;
    };
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += 256) {
        float v = m.grad[base + i];
        if (m.momentum) {
            const float next = m.momentum[base + i] * mu + v;
            m.momentum[base + i] = next;
            v = v + mu * next;
        }
        x[at(i)] = v;
        sum += double(v) * double(v);
    }
    sum = red::wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    const double norm = sqrt(sums[0] + sums[1] + sums[2] + sums[3]), factor = norm == 0.0 ? 0.0 : 1.0 / norm;
    for (int i = threadIdx.x; i < tall_tiles * 32 * stride; i += 256) x[i] = float(double(x[i]) * factor);
    __syncthreads();
    const f16v zero = {};
    const int i0 = tall_tiles == 2 ? wave / 2 * 32 : 0, j0 = tall_tiles == 2 ? wave % 2 * 32 : 0;  // this wave's tile
    for (int step = 0; step < steps; ++step) {
        const Quintic f = quintic_of(step >= m.turn);
        // H; a single tile's k is shared out to the waves.
        if (tall_tiles == 2) {
            each_value(multiply_rows(x + i0 * stride, x + j0 * stride, stride, 0, 32 * long_tiles, zero),
                       [&](int r, int c, float v) { g[(i0 + r) * kSquareStride + j0 + c] = v - (i0 + r == j0 + c ? f.shift : 0.0f); });
        } else {
            each_value(multiply_rows(x, x, stride, 8 * long_tiles * wave, 8 * long_tiles * (wave + 1), zero),
                       [&](int r, int c, float v) { q[wave * 1024 + r * 32 + c] = v; });
            __syncthreads();
            for (int i = threadIdx.x; i < 1024; i += 256) {
                const float* const part = q + i;
                g[i / 32 * kSquareStride + i % 32] =
                    (part[0] + part[1024]) + (part[2 * 1024] + part[3 * 1024]) - (i / 32 == i % 32 ? f.shift : 0.0f);
            }
        }
        __syncthreads();
        // Q = a I + b H + c H H
        if (tall_tiles == 2 || wave == 0)
            each_value(multiply_rows(g + i0 * kSquareStride, g + j0 * kSquareStride, kSquareStride, 0, 32 * tall_tiles, zero),
                       [&](int r, int c, float v) {
                           const int place = (i0 + r) * kSquareStride + j0 + c;
                           q[place] = f.b * g[place] + f.c * v + (i0 + r == j0 + c ? f.a : 0.0f);
                       });
        __syncthreads();
        // X = Q X, whole columns a wave
        for (int t = wave; t < long_tiles; t += 4) {
            f16v upper = zero, lower = zero;
            for (int k = 0; k < 32 * tall_tiles; k += 8) {
                const int k0 = k + lane / 32 * 4, column = 32 * t + lane % 32;
                f4 b;
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = x[(k0 + e) * stride + column];
                upper = multiply4(*reinterpret_cast<const f4*>(q + lane % 32 * kSquareStride + k0), b, upper);
                if (tall_tiles == 2)
                    lower = multiply4(*reinterpret_cast<const f4*>(q + (32 + lane % 32) * kSquareStride + k0), b, lower);
            }
            each_value(upper, [&](int r, int c, float v) { x[r * stride + 32 * t + c] = v; });
            if (tall_tiles == 2) each_value(lower, [&](int r, int c, float v) { x[(32 + r) * stride + 32 * t + c] = v; });
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < count; i += 256) {
        if (m.param) m.param[base + i] = keep * m.param[base + i] - m.rate * x[at(i)];
        else m.out[base + i] = x[at(i)];
    }
}

bool small(const Matrix& m) {
    const int64_t shorter = std::min(m.rows, m.cols);
    return shorter <= kShort && std::max(m.rows, m.cols) <= (shorter <= 32 ? 2 * kLong : kLong);
}

// ---- matrices in tiles --------------------------------------------------------------

enum class Kind { Gram, Poly, Apply };

// Counts of the parts of a tile's sum that are done; zero between launches,
// which the library's stream never overlaps.
__device__ unsigned g_tile_done[kMostSplit];

// A tile of G, P or the next X. last: the next X leaves the scale, to `out` or
// into the parameter.
template <Kind K, int BT, int Stages>
__global__ __launch_bounds__(packed::kThreads, 2) void product_kernel(Batch batch, int step, bool last, float keep, float* partial) {
    using Tile = packed::Tile<BT, Stages>;
    __shared__ __align__(16) char lds[Tile::kLds];
    __shared__ bool finisher;
    // Each of the chip's eight dies, which workgroups go to in turn, gets neighbouring tiles of every matrix,
    // whose operands its cache then serves (an iteration of the large matrices above 1013 to 990 us). Shares of
    // the whole batch instead gave dies matrices of unlike depth, and the last product took a quarter longer.
    const Matrix& m = batch.of[find(batch, int(blockIdx.x) / 8)];
    const bool shifted = step >= m.turn;  // (read with the rest of m)
    const int row_tiles = int(m.shorter / BT), column_tiles = K == Kind::Apply ? int(m.longer / BT) : row_tiles;
    const int tiles = K == Kind::Apply ? row_tiles * column_tiles : row_tiles * (row_tiles + 1) / 2;
    const int blocks = m.tiles * m.splits, share = (blocks + 7) / 8;
    int id = int(blockIdx.x) % 8 * share + int(blockIdx.x) / 8 - m.first;
    if (id >= blocks) return;
    const int part = id % m.splits;
    id /= m.splits;
    const int tile_id = id + m.from;
    const int64_t z = tile_id / tiles;
    // Strips of eight rows, column by column, of the tiles with i <= j where the product is symmetric.
    int rest = tile_id % tiles, i = 0, j = 0, high = 0;
    for (;;) {
        high = min(8, row_tiles - i);
        const int triangle = K == Kind::Apply ? 0 : high * (high + 1) / 2, from = K == Kind::Apply ? 0 : i + high;
        const int strip = triangle + high * (column_tiles - from);
        if (rest >= strip) {
            rest -= strip;
            i += high;
            continue;
        }
        if (rest < triangle) {
            j = i;
            for (int n = 1; rest >= n; ++n, ++j) rest -= n;
            i += rest;
        } else {
            rest -= triangle;
            j = from + rest / high;
            i += rest % high;
        }
        break;
    }
    const int64_t m0 = int64_t(i) * BT, n0 = int64_t(j) * BT;
    const int64_t whole = z * 2 * m.shorter * m.longer, square = z * 2 * m.shorter * m.shorter;
    const int64_t depth = K == Kind::Gram ? m.longer : m.shorter, slices = depth / packed::kSlice;
    // The squares are their own transposes.
    const half* const a = K == Kind::Gram ? m.x + whole : (K == Kind::Poly ? m.gram : m.poly) + square;
    const half* const b = K == Kind::Gram ? a : K == Kind::Poly ? a : m.xt + whole;
    Tile tile;
    tile.clear();
    tile.template accumulate<K == Kind::Gram>(a + m0 * 2 * depth, b + n0 * 2 * depth, depth, slices * part / m.splits, slices * (part + 1) / m.splits, lds);

    if (m.splits > 1) {
        // The part that counts in last adds all of them in order.
        constexpr int kValues = BT * BT / packed::kThreads;
        float* const mine = partial + (int64_t(m.parts) + int64_t(id) * m.splits) * BT * BT + threadIdx.x;
        int at = 0;
        tile.each4([&](int, int, float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                __hip_atomic_store(&mine[(int64_t(part) * kValues + at++) * packed::kThreads], v[e], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        });
        red::wait_stores_visible();
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned* const done = &g_tile_done[m.counters + id];
            finisher = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == unsigned(m.splits);
            if (finisher) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!finisher) return;
        tile.clear();
        for (int q = 0; q < m.splits; ++q) {
            at = 0;
            tile.each4([&](int, int, float (&v)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] += __hip_atomic_load(&mine[(int64_t(q) * kValues + at++) * packed::kThreads], __ATOMIC_RELAXED,
                                              __HIP_MEMORY_SCOPE_AGENT);
            });
        }
    }

    const float unit = 1.0f / kScale;
    const Quintic f = quintic_of(shifted);
    if constexpr (K == Kind::Apply) {
        tile.mix(f.a, m.x + whole, unit, m0, n0, m.longer);
        if (!last) {
            tile.store(m.y + whole, m0, n0, m.longer);
            tile.store_transposed(m.yt + whole, m0, n0, m.shorter, lds);
            return;
        }
        const bool wide = m.wide();
        float *const out = m.out ? m.out + z * m.elements() : nullptr, *const param = m.param ? m.param + z * m.elements() : nullptr;
        const int64_t rows = wide ? m.rows : m.cols, cols = wide ? m.cols : m.rows;  // without the padding
        tile.each4([&](int r, int c, float (&v)[4]) {
            const int64_t row = m0 + r, col = n0 + c;
            if (col >= cols) return;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (row + e >= rows) return;
                const int64_t at = wide ? (row + e) * cols + col : col * rows + row + e;
                if (param) param[at] = keep * param[at] - m.rate * (v[e] * unit);
                else out[at] = v[e] * unit;
            }
        });
    } else {
        half* const out = (K == Kind::Gram ? m.gram : m.poly) + square;
        if constexpr (K == Kind::Poly) {
            tile.mix(f.b, m.gram + square, f.c * unit, m0, n0, m.shorter);
        } else {
            tile.each4([&](int r, int c, float (&v)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = v[e] * unit - (i == j && r + e == c ? f.shift * kScale : 0.0f);
            });
        }
        tile.store(out, m0, n0, m.shorter);
        if (i != j) tile.store_transposed(out, m0, n0, m.shorter, lds);
    }
}

// Numbers the workgroups of a launch.
template <class F>
int64_t assign(Batch& batch, F&& workgroups) {
    int64_t first = 0;
    for (int i = 0; i < batch.n; ++i) {
        batch.of[i].first = int(first);
        first += workgroups(batch.of[i]);
        if (first >= int64_t(1) << 31) fail(VC_HIP_ERR_OVERFLOW, "orthogonalise: too many tiles");
    }
    return first;
}

int64_t tiles_of(Kind kind, const Matrix& m, int64_t bt) {
    const int64_t t = m.shorter / bt;
    return m.count * (kind == Kind::Apply ? t * (m.longer / bt) : t * (t + 1) / 2);
}

// Where tiles are few, sums are split into parts of at least eight slices (1024 x
// 4096: 519 us, 817 with whole sums). More stages in flight where a CU has one
// workgroup at most (1024 x 1024: 284 us, 348 with two stages; 2048 x 2048, with
// more workgroups than that: 775 with two stages, 907 with four).
//
// A CU has two workgroups with tiles of 128. Where the last round of them would
// leave half of the places empty, its sums are split as well, and its tiles are
// the last of the matrix with the most. (The matrices above, whose G and P have 600
// tiles for 512 places: both products 532 to 504 us an iteration, P alone 264 to
// 233; twice as many parts of the last round, or more, gained no more.)
template <Kind K, int BT>
void product(Device& d, Batch batch, int step, bool last = false, float keep = 0.0f) {
    const auto slices = [](const Matrix& m) { return (K == Kind::Gram ? m.longer : m.shorter) / packed::kSlice; };
    int64_t tiles = 0, most = 0;
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        const int64_t own = tiles_of(K, m, BT);
        if (own >= int64_t(1) << 28) fail(VC_HIP_ERR_OVERFLOW, "orthogonalise: too many tiles");
        m.from = 0;
        m.tiles = int(own);
        tiles += own;
        if (own > batch.of[most].tiles) most = i;
    }
    const int64_t wanted = tiles > kMostSplit ? 1 : std::max<int64_t>(1, d.cu_count / tiles);
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        m.splits = int(std::max<int64_t>(1, std::min(wanted, slices(m) / 8)));
    }
    const int64_t places = 2 * d.cu_count, over = tiles % places;
    if (BT == 128 && tiles > places && over && over <= places / 2 && batch.of[most].tiles > over && over <= kMostSplit) {
        batch.of[most].tiles -= int(over);
        Matrix& end = batch.of[batch.n++];
        end = batch.of[most];
        end.from = batch.of[most].tiles;
        end.tiles = int(over);
        end.splits = int(std::max<int64_t>(1, std::min(d.cu_count / over, slices(end) / 8)));
    }
    int64_t counters = 0, parts = 0, blocks = 0;
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        m.counters = int(counters);
        m.parts = int(parts);
        if (m.splits > 1) {
            counters += m.tiles;
            parts += int64_t(m.tiles) * m.splits;
        }
        blocks += int64_t(m.tiles) * m.splits;
        if (blocks >= int64_t(1) << 30) fail(VC_HIP_ERR_OVERFLOW, "orthogonalise: too many tiles");
    }
    const int64_t shares = assign(batch, [](const Matrix& m) { return (int64_t(m.tiles) * m.splits + 7) / 8; });
    Scratch partial(parts ? size_t(parts) * BT * BT * sizeof(float) : 4);
    const dim3 grid{unsigned(8 * shares)}, threads{packed::kThreads};
    if (blocks <= d.cu_count)
        launch(product_kernel<K, BT, 4>, grid, threads, 0, d.stream, batch, step, last, keep, partial.as<float>());
    else
        launch(product_kernel<K, BT, 2>, grid, threads, 0, d.stream, batch, step, last, keep, partial.as<float>());
    after_launch("orthogonalise product");
}

// Whether tiles of 128 give three of four CUs work, parts of a sum at least 1024
// deep counted; four tiles of 64 read twice what one of 128 reads. Five
// iterations, every product by tiles of 128 and of 64: 1024 x 1024 412 and 285
// us, 2048 x 2048 869 and 814 (775 with 128 in the last product alone, as here),
// 2816 x 2816 1535 and 1773, 4096 x 4096 4508 and 5087.
bool wide_tiles(const Device& d, const Batch& batch, Kind kind) {
    int64_t tiles = 0, blocks = 0;
    for (int i = 0; i < batch.n; ++i) tiles += tiles_of(kind, batch.of[i], 128);
    const int64_t wanted = std::max<int64_t>(1, d.cu_count / tiles);
    for (int i = 0; i < batch.n; ++i) {
        const Matrix& m = batch.of[i];
        const int64_t depth = kind == Kind::Gram ? m.longer : m.shorter;
        blocks += tiles_of(kind, m, 128) * std::max<int64_t>(1, std::min(wanted, depth / 1024));
    }
    return blocks >= d.cu_count * 3 / 4;
}

// The iterates of a batch; x and its successor take turns.
void run(Device& d, Batch& batch, float mu, float keep, size_t steps) {
    for (int i = 0; i < batch.n; ++i) batch.of[i].turn = turn_of(std::min(batch.of[i].rows, batch.of[i].cols));
    if (steps > 0 && steps <= kMostSteps && std::all_of(batch.of, batch.of + batch.n, small)) {
        const int64_t matrices = assign(batch, [](const Matrix& m) { return int64_t(m.count); });
        launch(small_kernel, dim3(unsigned(matrices)), dim3(256), 0, d.stream, batch, mu, keep, int(steps));
        after_launch("orthogonalise small");
        return;
    }
    const auto pad = [&](int64_t to) {
        for (int i = 0; i < batch.n; ++i) {
            Matrix& m = batch.of[i];
            m.shorter = (std::min(m.rows, m.cols) + to - 1) / to * to;
            m.longer = (std::max(m.rows, m.cols) + to - 1) / to * to;
        }
    };
    pad(128);
    const bool wide_gram = wide_tiles(d, batch, Kind::Gram), wide_poly = wide_tiles(d, batch, Kind::Poly);
    const bool wide_apply = wide_tiles(d, batch, Kind::Apply);
    if (!wide_gram && !wide_poly && !wide_apply) pad(64);
    int64_t partials = 0, squares = 0, wholes = 0;
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        m.blocks = int(grid_1d(size_t(m.elements()), 1024, kNormBlocks));
        partials += int64_t(m.count) * m.blocks;
        squares += m.count * m.shorter * m.shorter;
        wholes += m.count * m.shorter * m.longer;
    }
    // Four bytes a value; the update lies where the second iterate will.
    Scratch sums(partials * sizeof(double)), x(wholes * 4), xt(wholes * 4), y(wholes * 4), yt(wholes * 4), gram(squares * 4),
        poly(squares * 4);
    partials = squares = wholes = 0;
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        m.x = x.as<half>() + 2 * wholes;
        m.xt = xt.as<half>() + 2 * wholes;
        m.y = y.as<half>() + 2 * wholes;
        m.yt = yt.as<half>() + 2 * wholes;
        m.update = y.as<float>() + wholes;
        m.gram = gram.as<half>() + 2 * squares;
        m.poly = poly.as<half>() + 2 * squares;
        m.partials = sums.as<double>() + partials;
        partials += int64_t(m.count) * m.blocks;
        squares += m.count * m.shorter * m.shorter;
        wholes += m.count * m.shorter * m.longer;
    }
    int64_t blocks = assign(batch, [](const Matrix& m) { return int64_t(m.count) * m.blocks; });
    launch(update_kernel, dim3(unsigned(blocks)), dim3(256), 0, d.stream, batch, mu);
    after_launch("muon update");
    if (steps == 0) {
        launch(normalise_kernel, dim3(unsigned(blocks)), dim3(256), 0, d.stream, batch);
        after_launch("orthogonalise");
        return;
    }
    blocks = assign(batch, [](const Matrix& m) { return m.count * (m.shorter / 64) * (m.longer / 64); });
    launch(pack_kernel, dim3(unsigned(blocks)), dim3(256), 0, d.stream, batch);
    after_launch("orthogonalise pack");
    for (size_t i = 0; i < steps; ++i) {
        const bool last = i + 1 == steps;
        const int step = int(std::min<size_t>(i, 2));  // all later ones are like the third
        wide_gram ? product<Kind::Gram, 128>(d, batch, step) : product<Kind::Gram, 64>(d, batch, step);
        wide_poly ? product<Kind::Poly, 128>(d, batch, step) : product<Kind::Poly, 64>(d, batch, step);
        wide_apply ? product<Kind::Apply, 128>(d, batch, step, last, keep) : product<Kind::Apply, 64>(d, batch, step, last, keep);
        for (int k = 0; k < batch.n; ++k) {
            std::swap(batch.of[k].x, batch.of[k].y);
            std::swap(batch.of[k].xt, batch.of[k].yt);
        }
    }
}

void check_matrix(size_t count, size_t rows, size_t cols) {
    const size_t most = size_t(1) << 21;  // 128 rows of parts stay within a buffer load's 31-bit offsets
    if (count > 65535) fail(VC_HIP_ERR_INVALID_ARGUMENT, "orthogonalise: at most 65535 matrices");
    if (rows > most || cols > most) fail(VC_HIP_ERR_OVERFLOW, "orthogonalise: matrix too large");
}

double flops(const Matrix& m, size_t steps) {
    const double s = double(std::min(m.rows, m.cols)), l = double(std::max(m.rows, m.cols));
    return double(m.count) * double(steps) * (3.0 * s * s * l + s * s * s);
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_orthogonalise(const float* in, size_t count, size_t rows, size_t cols, size_t steps, float* out) {
    return guard([&] {
        Device& d = require_device();
        check_matrix(count, rows, cols);
        if (count == 0 || rows == 0 || cols == 0) return;
        if (!in || !out) fail(VC_HIP_ERR_INVALID_ARGUMENT, "orthogonalise: null pointer");
        Batch batch{};
        batch.n = 1;
        Matrix& m = batch.of[0];
        m.grad = in;
        m.out = out;
        m.rows = int64_t(rows);
        m.cols = int64_t(cols);
        m.count = int(count);
        Profiled p("orthogonalise", flops(m, steps), 8.0 * count * rows * cols);
        run(d, batch, 0.0f, 0.0f, steps);
        p.done();
    });
}

int vc_hip_muon_step(const vc_hip_muon_item* items, size_t n_items, float rate, float mu, float decay, size_t steps) {
    return guard([&] {
        Device& d = require_device();
        if (n_items && !items) fail(VC_HIP_ERR_INVALID_ARGUMENT, "muon_step: null items");
        if (steps == 0) fail(VC_HIP_ERR_INVALID_ARGUMENT, "muon_step: no steps");
        for (size_t i = 0; i < n_items; ++i) {
            const vc_hip_muon_item& it = items[i];
            check_matrix(it.count, it.rows, it.cols);
            if (it.count * it.rows * it.cols && (!it.param || !it.momentum || !it.grad))
                fail(VC_HIP_ERR_INVALID_ARGUMENT, "muon_step: null pointer");
        }
        size_t next = 0;
        while (next < n_items) {
            Batch batch{};
            double work = 0.0, bytes = 0.0;
            for (; next < n_items && batch.n < kAtOnce; ++next) {
                const vc_hip_muon_item& it = items[next];
                if (it.count * it.rows * it.cols == 0) continue;
                Matrix& m = batch.of[batch.n++];
                m.grad = it.grad;
                m.momentum = it.momentum;
                m.param = it.param;
                m.rows = int64_t(it.rows);
                m.cols = int64_t(it.cols);
                m.count = int(it.count);
                m.rate = rate * float(std::sqrt(std::max(1.0, double(it.cols) / double(it.rows))));
                work += flops(m, steps);
                bytes += 20.0 * it.count * it.rows * it.cols;
            }
            if (batch.n == 0) break;
            Profiled p("muon_step", work, bytes);
            run(d, batch, mu, 1.0f - rate * decay, steps);
            p.done();
        }
    });
}

}  // extern "C"
