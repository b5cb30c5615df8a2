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
// All values stay near one by construction (|x| <= 1.21, |g| <= 1.5, |p| <= 3),
// so the products run as three half-precision products of two parts each
// (split_product.hpp), on values scaled by 2^14 in memory: below 2^15.6 they are
// in half precision's range, and a part below its smallest step is 2^-38 of one.
// The error is that of a float32 product relative to the norm, which is what the
// iteration keeps of its input. The scale is a power of two and costs nothing.
//
// All matrices of a call run in the same launches, three an iteration: a train
// step's matrices fill the chip together, and small ones share the latency.
#include "reduce_common.hpp"
#include "split_product.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

namespace vchip {
namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScale = 16384.0f;
constexpr int kNormBlocks = 64;   // partial sums of squares of a matrix
constexpr int kAtOnce = 12;       // matrices (or batches of equal ones) of a launch
constexpr int kMostSplit = 2048;  // tiles of a launch whose sums are split
using S = split::Fp16x2;

// `count` matrices [rows, cols].
struct Matrix {
    const float* grad;
    float *momentum, *param;     // null for a plain iterate
    float *x, *y, *gram, *poly;  // scaled: the iterate, its successor; both squares
    double* partials;
    int64_t rows, cols;
    int count, blocks;
    float rate;
    int first, splits, counters;  // of the launch: the first workgroup, parts of each tile's sum, its first count

    __host__ __device__ int64_t elements() const { return rows * cols; }
    __host__ __device__ bool wide() const { return rows <= cols; }
    __host__ __device__ int64_t shorter() const { return rows <= cols ? rows : cols; }
    __host__ __device__ int64_t longer() const { return rows <= cols ? cols : rows; }
};
struct Batch {
    Matrix of[kAtOnce];
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
    float *const momentum = m.momentum ? m.momentum + base : nullptr, *const x = m.x + base;
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

// x becomes scale * x / ||x||.
__global__ __launch_bounds__(256) void normalise_kernel(Batch batch, float scale) {
    const Matrix& m = batch.of[find(batch, blockIdx.x)];
    const int block = (blockIdx.x - m.first) % m.blocks, z = (blockIdx.x - m.first) / m.blocks;
    double sum = 0.0;
    for (int i = 0; i < m.blocks; ++i) sum += m.partials[z * m.blocks + i];
    const double norm = sqrt(sum), factor = norm == 0.0 ? 0.0 : double(scale) / norm;
    const int64_t count = m.elements();
    float* const x = m.x + z * count;
    for (int64_t i = int64_t(block) * 256 + threadIdx.x; i < count; i += int64_t(m.blocks) * 256)
        x[i] = float(double(x[i]) * factor);
}

enum class Kind { Gram, Poly, Apply };

// Counts of the parts of a tile's sum that are done; zero between launches,
// which the library's stream never overlaps.
__device__ unsigned g_tile_done[kMostSplit];

// A tile of G, P or the next X. last: the next X leaves the scale, to y or into
// the parameter.
template <Kind K, int BT>
__global__ __launch_bounds__(split::kThreads, K == Kind::Apply && BT == 128 ? 2 : 3) void product_kernel(Batch batch, bool last, float keep, float* partial) {
    __shared__ split::Slice<S, BT> as, bs;
    __shared__ bool finisher;
    const Matrix& m = batch.of[find(batch, blockIdx.x)];
    const int64_t rows = K == Kind::Apply ? m.rows : m.shorter(), cols = K == Kind::Apply ? m.cols : m.shorter();
    const int64_t depth = K == Kind::Gram ? m.longer() : m.shorter();
    const int row_tiles = int((rows + BT - 1) / BT), column_tiles = int((cols + BT - 1) / BT);
    const int tiles = K == Kind::Apply ? row_tiles * column_tiles : row_tiles * (row_tiles + 1) / 2;
    int id = int(blockIdx.x) - m.first;
    const int part = id % m.splits;
    id /= m.splits;
    const int z = id / tiles, tile_id = id % tiles;
    int i = tile_id / column_tiles, j = tile_id % column_tiles;
    if constexpr (K != Kind::Apply) {  // the tile_id-th with i <= j
        i = 0;
        j = tile_id;
        while (j >= row_tiles - i) {
            j -= row_tiles - i;
            ++i;
        }
        j += i;
    }
    const int64_t m0 = int64_t(i) * BT, n0 = int64_t(j) * BT;
    const float* const x = m.x + z * m.elements();
    const int64_t square = z * m.shorter() * m.shorter();
    // This part's slices of k.
    const int64_t slices = (depth + split::kSliceK - 1) / split::kSliceK;
    const int64_t begin = slices * part / m.splits * split::kSliceK;
    const int64_t end = min(depth, slices * (part + 1) / m.splits * split::kSliceK);

    split::Tile<S, BT, BT> tile;
    tile.clear();
    const auto run = [&](auto& a, auto& b, auto&& load_a, auto&& load_b) {
        load_a(begin);
        load_b(begin);
        for (int64_t k = begin; k < end; k += split::kSliceK) {
            a.store(as);
            b.store(bs);
            __syncthreads();
            if (k + split::kSliceK < end) {
                load_a(k + split::kSliceK);
                load_b(k + split::kSliceK);
            }
            tile.multiply(as, bs);
            __syncthreads();
        }
    };
    using Along = split::AlongK<BT>;
    using Across = split::AcrossK<BT>;
    const auto along = [&](const float* from, int64_t first, int64_t many, int64_t ld, const float* (&p)[Along::kChunks]) {
#pragma unroll
        for (int c = 0; c < Along::kChunks; ++c) p[c] = from + min(first + Along::row(c), many - 1) * ld;
    };
    const auto across = [&](int64_t first, int64_t many, unsigned (&at)[Across::kChunks]) {
#pragma unroll
        for (int c = 0; c < Across::kChunks; ++c) at[c] = unsigned(min(int64_t(Across::row(c)), many - 1 - first));
    };
    const auto line_of = [](const float* from, int64_t ld) {
        return [=](int64_t k) {
            const float* const line = from + k * ld;
            return [=](int) { return line; };
        };
    };
    if (K == Kind::Poly || (K == Kind::Gram && m.wide()) || (K == Kind::Apply && !m.wide())) {
        // The squares are their own transposes.
        const float* const fa = K == Kind::Poly ? m.gram + square : x;
        const float* const fb = K == Kind::Gram ? x : (K == Kind::Poly ? m.gram : m.poly) + square;
        const int64_t lda = K == Kind::Poly ? m.shorter() : m.cols, ldb = K == Kind::Gram ? m.cols : m.shorter();
        Along a, b;
        const float *pa[Along::kChunks], *pb[Along::kChunks];
        along(fa, m0, rows, lda, pa);
        along(fb, n0, cols, ldb, pb);
        run(a, b, [&](int64_t k) { a.load(pa, k, end); }, [&](int64_t k) { b.load(pb, k, end); });
    } else if constexpr (K == Kind::Gram) {
        Across a, b;
        unsigned at_a[Across::kChunks], at_b[Across::kChunks];
        across(m0, rows, at_a);
        across(n0, cols, at_b);
        run(a, b, [&](int64_t k) { a.load(at_a, k, end, line_of(x + m0, m.cols)); },
            [&](int64_t k) { b.load(at_b, k, end, line_of(x + n0, m.cols)); });
    } else if constexpr (K == Kind::Apply) {
        Along a;
        Across b;
        const float* pa[Along::kChunks];
        unsigned at_b[Across::kChunks];
        along(m.poly + square, m0, rows, m.shorter(), pa);
        across(n0, cols, at_b);
        run(a, b, [&](int64_t k) { a.load(pa, k, end); }, [&](int64_t k) { b.load(at_b, k, end, line_of(x + n0, m.cols)); });
    }

    if (m.splits > 1) {
        // The part that counts in last adds all of them in order.
        constexpr int kValues = BT * BT / split::kThreads;
        float* const mine = partial + (int64_t(blockIdx.x) - part) * BT * BT + threadIdx.x;
        int at = 0;
        tile.each([&](int, int, float& v) {
            __hip_atomic_store(&mine[(int64_t(part) * kValues + at++) * split::kThreads], v, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        });
        red::wait_stores_visible();
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned* const done = &g_tile_done[(int(blockIdx.x) - m.first) / m.splits + m.counters];
            finisher = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == unsigned(m.splits);
            if (finisher) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!finisher) return;
        tile.clear();
        for (int q = 0; q < m.splits; ++q) {
            at = 0;
            tile.each([&](int, int, float& v) {
                v += __hip_atomic_load(&mine[(int64_t(q) * kValues + at++) * split::kThreads], __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
            });
        }
    }

    const float unit = 1.0f / kScale;
    if constexpr (K == Kind::Apply) {
        float* const out = m.y + z * m.elements();
        float* const param = m.param ? m.param + z * m.elements() : nullptr;
        tile.each([&](int r, int c, float& v) {
            const int64_t row = m0 + r, col = n0 + c;
            if (row >= rows || col >= cols) return;
            const int64_t at = row * cols + col;
            const float next = kA * x[at] + v * unit;
            if (!last) out[at] = next;
            else if (param) param[at] = keep * param[at] - m.rate * (next * unit);
            else out[at] = next * unit;
        });
    } else {
        float* const out = (K == Kind::Gram ? m.gram : m.poly) + square;
        tile.each([&](int r, int c, float& v) {
            const int64_t row = m0 + r, col = n0 + c;
            if (row >= rows || col >= cols) return;
            v *= unit;
            if constexpr (K == Kind::Poly) v = kB * m.gram[square + row * cols + col] + kC * v;
            out[row * cols + col] = v;
            if (i != j) out[col * cols + row] = v;
        });
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
    if (kind == Kind::Apply) return m.count * ((m.rows + bt - 1) / bt) * ((m.cols + bt - 1) / bt);
    const int64_t t = (m.shorter() + bt - 1) / bt;
    return m.count * (t * (t + 1) / 2);
}
int64_t all_tiles(Kind kind, const Batch& batch, int64_t bt) {
    int64_t tiles = 0;
    for (int i = 0; i < batch.n; ++i) tiles += tiles_of(kind, batch.of[i], bt);
    return tiles;
}

// Where tiles are few, sums are split into parts of at least four slices.
template <Kind K, int BT>
void product_tiles(Device& d, Batch& batch, bool last, float keep) {
    const int64_t tiles = all_tiles(K, batch, BT);
    const int64_t wanted = tiles > kMostSplit ? 1 : std::max<int64_t>(1, 2 * d.cu_count / std::max<int64_t>(1, tiles));
    int64_t counters = 0;
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        const int64_t slices = ((K == Kind::Gram ? m.longer() : m.shorter()) + split::kSliceK - 1) / split::kSliceK;
        m.splits = int(std::max<int64_t>(1, std::min(wanted, slices / 4)));
        m.counters = int(counters);
        counters += tiles_of(K, m, BT);
    }
    const int64_t blocks = assign(batch, [](const Matrix& m) { return tiles_of(K, m, BT) * m.splits; });
    Scratch partial(wanted > 1 ? size_t(blocks) * BT * BT * sizeof(float) : 4);
    launch(product_kernel<K, BT>, dim3(unsigned(blocks)), dim3(split::kThreads), 0, d.stream, batch, last, keep,
           partial.as<float>());
    after_launch("orthogonalise product");
}

// Tiles of 128 where they give every other CU work, else of 64.
template <Kind K>
void product(Device& d, Batch& batch, bool last = false, float keep = 0.0f) {
    if (all_tiles(K, batch, 128) >= d.cu_count / 2) product_tiles<K, 128>(d, batch, last, keep);
    else product_tiles<K, 64>(d, batch, last, keep);
}

// The iterates of a batch; x and its successor take turns.
void run(Device& d, Batch& batch, float mu, float keep, size_t steps) {
    int64_t partials = 0, squares = 0, elements = 0;
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        m.blocks = int(grid_1d(size_t(m.elements()), 2048, kNormBlocks));
        partials += int64_t(m.count) * m.blocks;
        squares += m.count * m.shorter() * m.shorter();
        elements += m.count * m.elements();
    }
    Scratch sums(partials * sizeof(double)), first(elements * sizeof(float)), second(elements * sizeof(float)),
        gram(squares * sizeof(float)), poly(squares * sizeof(float));
    std::vector<float*> out(batch.n);
    partials = squares = elements = 0;
    for (int i = 0; i < batch.n; ++i) {
        Matrix& m = batch.of[i];
        out[i] = m.y;
        m.x = steps == 0 ? out[i] : first.as<float>() + elements;
        m.y = second.as<float>() + elements;
        m.gram = gram.as<float>() + squares;
        m.poly = poly.as<float>() + squares;
        m.partials = sums.as<double>() + partials;
        partials += int64_t(m.count) * m.blocks;
        squares += m.count * m.shorter() * m.shorter();
        elements += m.count * m.elements();
    }
    const auto pass = [&](auto kernel, float value) {
        const int64_t blocks = assign(batch, [](const Matrix& m) { return int64_t(m.count) * m.blocks; });
        launch(kernel, dim3(unsigned(blocks)), dim3(256), 0, d.stream, batch, value);
        after_launch("orthogonalise");
    };
    pass(update_kernel, mu);
    pass(normalise_kernel, steps == 0 ? 1.0f : kScale);
    for (size_t i = 0; i < steps; ++i) {
        const bool last = i + 1 == steps;
        if (last)
            for (int k = 0; k < batch.n; ++k) batch.of[k].y = out[k];
        product<Kind::Gram>(d, batch);
        product<Kind::Poly>(d, batch);
        product<Kind::Apply>(d, batch, last, keep);
        for (int k = 0; k < batch.n; ++k) std::swap(batch.of[k].x, batch.of[k].y);
    }
}

void check_matrix(size_t count, size_t rows, size_t cols) {
    const size_t most = size_t(1) << 30;
    if (count > 65535) fail(VC_HIP_ERR_INVALID_ARGUMENT, "orthogonalise: at most 65535 matrices");
    if (rows > most || cols > most) fail(VC_HIP_ERR_OVERFLOW, "orthogonalise: matrix too large");
}

double flops(const Matrix& m, size_t steps) {
    const double s = double(m.shorter()), l = double(m.longer());
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
        m.y = out;
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
