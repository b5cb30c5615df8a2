// A mixture of experts: the plan that sorts a batch's picks by expert, the
// products of each expert's rows with its matrices and their gradients, and
// the weighted sum of a token's picks.
#include "reduce_common.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <string>

namespace vchip {
namespace {

using red::kWave;

constexpr size_t kMaxExperts = 1024;

// ---- the plan ---------------------------------------------------------------------
// A counting sort that keeps equal experts in pick order. Chunks of picks are
// counted by one launch; a second one adds up the counts before each chunk and
// places the picks, a wavefront finding the lanes of equal experts by ballots.
// Up to one round of picks a single workgroup does both.

constexpr int kPlanBlock = 512, kPlanWaves = kPlanBlock / kWave;
constexpr size_t kPlanChunks = 128;

// The group of an entry: its expert, or `experts` where it is none.
__device__ inline int group_of(float entry, int experts) {
    return entry >= 0.0f && entry < float(experts) && entry == truncf(entry) ? int(entry) : experts;
}

__global__ __launch_bounds__(kPlanBlock) void plan_count_kernel(const float* __restrict__ chosen, int rows, int chunk,
                                                                int experts, int* __restrict__ counts) {
    extern __shared__ int lds[];
    for (int e = threadIdx.x; e <= experts; e += kPlanBlock) lds[e] = 0;
    __syncthreads();
    const int begin = blockIdx.x * chunk, end = min(rows, begin + chunk);
    for (int p = begin + int(threadIdx.x); p < end; p += kPlanBlock) atomicAdd(&lds[group_of(chosen[p], experts)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += kPlanBlock) counts[blockIdx.x * (experts + 1) + e] = lds[e];
}

// counts: of every chunk, or null for one chunk counted here.
__global__ __launch_bounds__(kPlanBlock) void plan_place_kernel(const float* __restrict__ chosen, int rows, int chunk,
                                                                int experts, const int* __restrict__ counts,
                                                                int* __restrict__ offsets, int* __restrict__ order,
                                                                int* __restrict__ place) {
    extern __shared__ int lds[];
    const int groups = experts + 1, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    int* const next = lds;                 // the chunk's next row of each group
    int* const total = lds + groups;       // all rows of each group, then their sum before it
    int* const found = lds + 2 * groups;   // [wave][group] of the round
    const int begin = blockIdx.x * chunk, end = min(rows, begin + chunk);
    for (int e = tid; e < groups; e += kPlanBlock) {
        int before = 0, all = 0;
        if (counts)
            for (int c = 0; c < int(gridDim.x); ++c) {
                const int n = counts[c * groups + e];
                if (c < int(blockIdx.x)) before += n;
                all += n;
            }
        next[e] = before;
        total[e] = all;
    }
    __syncthreads();
    if (!counts) {
        for (int p = begin + tid; p < end; p += kPlanBlock) atomicAdd(&total[group_of(chosen[p], experts)], 1);
        __syncthreads();
    }
    if (wave == 0) {
        int sum = 0;  // before this lane's groups
        for (int base = 0; base < groups; base += kWave) {
            const int e = base + lane, n = e < groups ? total[e] : 0;
            int upto = n;
            for (int d = 1; d < kWave; d <<= 1) {
                const int v = __shfl_up(upto, d);
                if (lane >= d) upto += v;
            }
            if (e < groups) total[e] = sum + upto - n;
            sum += __shfl(upto, kWave - 1);
        }
    }
    __syncthreads();
    for (int e = tid; e < groups; e += kPlanBlock) {
        next[e] += total[e];
        if (blockIdx.x == 0) offsets[e] = total[e];
    }
    if (blockIdx.x == 0 && tid == 0) offsets[groups] = rows;
    const int bits = 32 - __clz(groups);
    for (int round = begin; round < end; round += kPlanBlock) {
        for (int i = tid; i < kPlanWaves * groups; i += kPlanBlock) found[i] = 0;
        __syncthreads();
        const int p = round + tid;
        const int e = p < end ? group_of(chosen[p], experts) : groups;
        uint64_t same = ~0ull;
        for (int b = 0; b < bits; ++b) {
            const uint64_t ones = __ballot(e >> b & 1);
            same &= e >> b & 1 ? ones : ~ones;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (p < end && rank == 0) found[wave * groups + e] = __popcll(same);
        __syncthreads();
        if (p < end) {
            int row = next[e] + rank;
            for (int w = 0; w < wave; ++w) row += found[w * groups + e];
            order[row] = p;
            place[p] = row;
        }
        __syncthreads();
        for (int g = tid; g < groups; g += kPlanBlock)
            for (int w = 0; w < kPlanWaves; ++w) next[g] += found[w * groups + g];
        __syncthreads();
    }
}

size_t plan_chunk(size_t rows) {
    const size_t rounds = (rows + kPlanBlock - 1) / kPlanBlock;
    return (rounds + kPlanChunks - 1) / kPlanChunks * kPlanBlock;
}
size_t plan_chunks(size_t rows) {
    const size_t chunk = plan_chunk(rows);
    return chunk ? (rows + chunk - 1) / chunk : 0;
}

void check_plan_sizes(size_t tokens, size_t top_k, size_t experts) {
    if (experts == 0 || experts > kMaxExperts)
        fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert plan: between 1 and 1024 experts are supported, got " + std::to_string(experts));
    if (top_k == 0) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert plan: a token needs a pick");
    if (tokens >= (size_t(1) << 31) / top_k) fail(VC_HIP_ERR_OVERFLOW, "expert plan: too many picks for int32 rows");
}

struct Plan {
    size_t tokens, top_k, experts, rows;
    const int *offsets, *order, *place;
};

Plan plan_of(const vc_hip_expert_plan* plan) {
    if (!plan || (!plan->words && plan->tokens)) fail(VC_HIP_ERR_INVALID_ARGUMENT, "null expert plan");
    check_plan_sizes(plan->tokens, plan->top_k, plan->experts);
    const size_t rows = plan->tokens * plan->top_k;
    const int* words = plan->words;
    return Plan{plan->tokens, plan->top_k, plan->experts, rows, words, words + plan->experts + 2, words + plan->experts + 2 + rows};
}

// ---- products -----------------------------------------------------------------------
// 64 x 64 tiles of C by 256 threads, 4 x 4 each, k through LDS 16 at a time.

constexpr int kTile = 64, kSlice = 16;

// A's element (row i of the tile, k) and B's (k, column j) as each kind of product stores them.
struct ProductArgs {
    const float *a, *b, *a2, *b2;
    float* c;
    const int *offsets, *order;
    int experts, top_k;     // top_k: of a gathered A, 0 where A lies in row order
    int64_t width, columns;  // of each expert's matrix [width, columns]
};

// Which of the tiles of kTile rows, counted group by group, this is.
__device__ inline bool find_rows(const int* offsets, int groups, int tile, int& group, int& begin, int& end) {
    for (int e = 0; e < groups; ++e) {
        const int lo = offsets[e], hi = offsets[e + 1], tiles = (hi - lo + kTile - 1) / kTile;
        if (tile < tiles) {
            group = e;
            begin = lo + tile * kTile;
            end = min(hi, begin + kTile);
            return true;
        }
        tile -= tiles;
    }
    return false;
}

enum class Product { Forward, Input, Weight };

template <Product P>
__global__ __launch_bounds__(256) void product_kernel(ProductArgs p) {
    __shared__ float as[kSlice][kTile + 4], bs[kSlice][kTile + 4];
    const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
    int group = blockIdx.z, begin = 0, end = 0;
    int64_t m0 = 0;
    const int64_t n0 = int64_t(blockIdx.x) * kTile, n = P == Product::Input ? p.width : p.columns;
    int64_t depth;
    if constexpr (P == Product::Weight) {
        begin = p.offsets[group];
        end = p.offsets[group + 1];
        m0 = int64_t(blockIdx.y) * kTile;
        depth = end - begin;
    } else {
        if (!find_rows(p.offsets, p.experts + 1, blockIdx.y, group, begin, end)) return;
        depth = P == Product::Input ? p.columns : p.width;
    }
    float acc[4][4] = {};
    for (int pass = 0; pass < (P == Product::Input && p.a2 ? 2 : 1); ++pass) {
        const float* const a = pass ? p.a2 : p.a;
        const float* const w = (pass ? p.b2 : p.b) + (P == Product::Weight ? 0 : int64_t(group) * p.width * p.columns);
        if (P != Product::Weight && group == p.experts) break;  // dropped picks: zero rows
        for (int64_t k0 = 0; k0 < depth; k0 += kSlice) {
            for (int i = tid; i < kSlice * kTile; i += 256) {
                float av = 0.0f, bv = 0.0f;
                if constexpr (P == Product::Weight) {
                    const int kk = i / kTile, x = i % kTile;
                    const int64_t r = begin + k0 + kk;
                    if (r < end) {
                        const int64_t row = p.top_k ? p.order[r] / p.top_k : r;
                        if (m0 + x < p.width) av = a[row * p.width + m0 + x];
                        if (n0 + x < n) bv = w[r * p.columns + n0 + x];
                    }
                    as[kk][x] = av;
                    bs[kk][x] = bv;
                } else {
                    const int x = i / kSlice, kk = i % kSlice;
                    const int64_t r = begin + x;
                    if (r < end && k0 + kk < depth) {
                        const int64_t row = p.top_k ? p.order[r] / p.top_k : r;
                        av = a[row * depth + k0 + kk];
                    }
                    as[kk][x] = av;
                    if constexpr (P == Product::Input) {
                        if (n0 + x < n && k0 + kk < depth) bv = w[(n0 + x) * p.columns + k0 + kk];
                        bs[kk][x] = bv;
                    } else {
                        const int bk = i / kTile, bx = i % kTile;
                        if (n0 + bx < n && k0 + bk < depth) bv = w[(k0 + bk) * p.columns + n0 + bx];
                        bs[bk][bx] = bv;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < kSlice; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[kk][ty + 16 * i], bs[kk][tx + 16 * j], acc[i][j]);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t col = n0 + tx + 16 * j;
            if (col >= n) continue;
            if constexpr (P == Product::Weight) {
                const int64_t row = m0 + ty + 16 * i;
                if (row < p.width) p.c[(int64_t(group) * p.width + row) * n + col] = acc[i][j];
            } else {
                const int64_t row = begin + ty + 16 * i;
                if (row < end) p.c[row * n + col] = acc[i][j];
            }
        }
}

unsigned tiles_of(size_t n) { return unsigned((n + kTile - 1) / kTile); }

void row_product(Device& d, const Plan& plan, bool input, ProductArgs p) {
    const unsigned row_tiles = unsigned(plan.rows / kTile + plan.experts + 1);
    if (input)
        launch(product_kernel<Product::Input>, dim3(tiles_of(p.width), row_tiles), dim3(256), 0, d.stream, p);
    else
        launch(product_kernel<Product::Forward>, dim3(tiles_of(p.columns), row_tiles), dim3(256), 0, d.stream, p);
    after_launch("expert product");
}

// ---- the gated unit -------------------------------------------------------------------

__device__ inline float sigmoid(float x) {
    const float e = expf(-fabsf(x));
    return (x >= 0.0f ? 1.0f : e) / (1.0f + e);
}

__global__ __launch_bounds__(256) void gate_kernel(const float* __restrict__ g, const float* __restrict__ u, int64_t count,
                                                   float* __restrict__ out) {
    const int64_t stride = int64_t(gridDim.x) * 256;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += stride) out[i] = g[i] * sigmoid(g[i]) * u[i];
}

// d silu(g) = s (1 + g (1 - s)) with s = sigmoid(g).
__global__ __launch_bounds__(256) void gate_backward_kernel(const float* __restrict__ grad, const float* __restrict__ g,
                                                            const float* __restrict__ u, int64_t count,
                                                            float* __restrict__ dg, float* __restrict__ du) {
    const int64_t stride = int64_t(gridDim.x) * 256;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += stride) {
        const float s = sigmoid(g[i]);
        du[i] = grad[i] * (g[i] * s);
        dg[i] = grad[i] * u[i] * (s * (1.0f + g[i] * (1.0f - s)));
    }
}

// ---- a token's picks ------------------------------------------------------------------

__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ rows, const float* __restrict__ weights,
                                                      const int* __restrict__ place, const int* __restrict__ offsets,
                                                      int experts, int64_t tokens, int top_k, int64_t width,
                                                      float* __restrict__ out) {
    const int kept = offsets[experts];  // rows of dropped picks come after
    for (int64_t t = blockIdx.y; t < tokens; t += gridDim.y)
        for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < width; i += int64_t(gridDim.x) * 256) {
            float sum = 0.0f;
            for (int j = 0; j < top_k; ++j) {
                const int64_t r = place[t * top_k + j];
                if (r >= kept) continue;
                const float v = rows[r * width + i];
                sum = weights ? fmaf(weights[t * top_k + j], v, sum) : sum + v;
            }
            out[t * width + i] = sum;
        }
}

// A wavefront per pick.
__global__ __launch_bounds__(256) void combine_backward_kernel(const float* __restrict__ grad, const float* __restrict__ rows,
                                                               const float* __restrict__ weights,
                                                               const int* __restrict__ place, const int* __restrict__ offsets,
                                                               int experts, int64_t picks, int top_k, int64_t width,
                                                               float* __restrict__ grad_rows,
                                                               float* __restrict__ grad_weights) {
    const int lane = threadIdx.x % kWave, kept = offsets[experts];
    const int64_t p = int64_t(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (p >= picks) return;
    const int64_t r = place[p];
    const float* const g = grad + p / top_k * width;
    const bool dropped = r >= kept;
    const float w = weights && !dropped ? weights[p] : 0.0f;
    double dot = 0.0;
    for (int64_t i = lane; i < width; i += kWave) {
        const float v = g[i];
        if (grad_weights && !dropped) dot += double(v) * double(rows[r * width + i]);
        if (grad_rows) grad_rows[r * width + i] = dropped ? 0.0f : w * v;
    }
    if (grad_weights) {
        dot = red::wave_sum(dot);
        if (lane == 0) grad_weights[p] = float(dot);
    }
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_expert_plan_words(size_t tokens, size_t top_k, size_t experts, size_t* words) {
    return guard([&] {
        if (!words) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert plan: null output");
        check_plan_sizes(tokens, top_k, experts);
        const size_t rows = tokens * top_k;
        *words = experts + 2 + 2 * rows + plan_chunks(rows) * (experts + 1);
    });
}

int vc_hip_expert_plan_build(const float* chosen, size_t tokens, size_t top_k, size_t experts, int32_t* words) {
    return guard([&] {
        Device& d = require_device();
        check_plan_sizes(tokens, top_k, experts);
        const size_t rows = tokens * top_k, chunks = plan_chunks(rows), chunk = plan_chunk(rows);
        if (!words || (rows && !chosen)) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert plan: null pointer");
        int* const order = words + experts + 2;
        int* const counts = order + 2 * rows;
        Profiled p("expert_plan", 0.0, 12.0 * rows);
        const uint32_t lds = uint32_t((2 + kPlanWaves) * (experts + 1) * sizeof(int));
        if (chunks > 1) {
            launch(plan_count_kernel, dim3(unsigned(chunks)), dim3(kPlanBlock), uint32_t((experts + 1) * sizeof(int)), d.stream,
                   chosen, int(rows), int(chunk), int(experts), counts);
            after_launch("expert plan counts");
        }
        launch(plan_place_kernel, dim3(unsigned(std::max<size_t>(chunks, 1))), dim3(kPlanBlock), lds, d.stream, chosen,
               int(rows), int(chunk), int(experts), static_cast<const int*>(chunks > 1 ? counts : nullptr), words, order,
               order + rows);
        after_launch("expert plan");
        p.done();
    });
}

int vc_hip_expert_linear_forward(const float* x, const float* w, const vc_hip_expert_plan* plan, size_t width,
                                 size_t columns, int ordered, float* out) {
    return guard([&] {
        Device& d = require_device();
        const Plan q = plan_of(plan);
        if (q.rows == 0 || columns == 0) return;
        if (!out || (width && (!x || !w))) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_linear: null pointer");
        Profiled p("expert_linear", 2.0 * q.rows * width * columns, 4.0 * (q.rows * (width + columns) + q.experts * width * columns));
        row_product(d, q, false,
                    ProductArgs{x, w, nullptr, nullptr, out, q.offsets, q.order, int(q.experts), ordered ? 0 : int(q.top_k),
                                int64_t(width), int64_t(columns)});
        p.done();
    });
}

int vc_hip_expert_gated_forward(const float* x, const float* gate, const float* up, const vc_hip_expert_plan* plan,
                                size_t width, size_t columns, int ordered, float* out, float* save_gate, float* save_up) {
    return guard([&] {
        Device& d = require_device();
        const Plan q = plan_of(plan);
        if (!save_gate != !save_up) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_gated: both saved products or neither");
        if (q.rows == 0 || columns == 0) return;
        if (!out || (width && (!x || !gate || !up))) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_gated: null pointer");
        Profiled p("expert_gated", 4.0 * q.rows * width * columns,
                   4.0 * (q.rows * (width + (save_gate ? 3.0 : 1.0) * columns) + 2.0 * q.experts * width * columns));
        const size_t count = q.rows * columns;
        Scratch scratch(save_gate ? 4 : 2 * count * sizeof(float));
        float* const g = save_gate ? save_gate : scratch.as<float>();
        float* const u = save_up ? save_up : scratch.as<float>() + count;
        ProductArgs args{x, gate, nullptr, nullptr, g, q.offsets, q.order, int(q.experts), ordered ? 0 : int(q.top_k),
                         int64_t(width), int64_t(columns)};
        row_product(d, q, false, args);
        args.b = up;
        args.c = u;
        row_product(d, q, false, args);
        launch(gate_kernel, dim3(grid_1d(count, 256, 8192)), dim3(256), 0, d.stream, static_cast<const float*>(g),
               static_cast<const float*>(u), int64_t(count), out);
        after_launch("expert_gated");
        p.done();
    });
}

int vc_hip_expert_gated_backward(const float* grad, const float* saved_gate, const float* saved_up, size_t count,
                                 float* grad_gate, float* grad_up) {
    return guard([&] {
        Device& d = require_device();
        if (count == 0) return;
        if (!grad || !saved_gate || !saved_up || !grad_gate || !grad_up)
            fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_gated_backward: null pointer");
        Profiled p("expert_gated_backward", 10.0 * count, 20.0 * count);
        launch(gate_backward_kernel, dim3(grid_1d(count, 256, 8192)), dim3(256), 0, d.stream, grad, saved_gate, saved_up,
               int64_t(count), grad_gate, grad_up);
        after_launch("expert_gated_backward");
        p.done();
    });
}

int vc_hip_expert_linear_backward_input(const float* grad, const float* w, const float* grad2, const float* w2,
                                        const vc_hip_expert_plan* plan, size_t width, size_t columns, float* grad_rows) {
    return guard([&] {
        Device& d = require_device();
        const Plan q = plan_of(plan);
        if (!grad2 != !w2) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_linear_backward_input: half of a second product");
        if (q.rows == 0 || width == 0) return;
        if (!grad_rows || (columns && (!grad || !w))) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_linear_backward_input: null pointer");
        const double products = grad2 ? 2.0 : 1.0;
        Profiled p("expert_backward_input", products * 2.0 * q.rows * width * columns,
                   4.0 * (q.rows * (width + products * columns) + products * q.experts * width * columns));
        row_product(d, q, true,
                    ProductArgs{grad, w, grad2, w2, grad_rows, q.offsets, q.order, int(q.experts), 0, int64_t(width),
                                int64_t(columns)});
        p.done();
    });
}

int vc_hip_expert_linear_backward_weight(const float* x, const float* grad, const vc_hip_expert_plan* plan, size_t width,
                                         size_t columns, int ordered, float* grad_w) {
    return guard([&] {
        Device& d = require_device();
        const Plan q = plan_of(plan);
        if (width == 0 || columns == 0) return;
        if (!grad_w || (q.rows && (!x || !grad))) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_linear_backward_weight: null pointer");
        if (width > size_t(kTile) * 65535) fail(VC_HIP_ERR_OVERFLOW, "expert_linear_backward_weight: too many rows");
        Profiled p("expert_backward_weight", 2.0 * q.rows * width * columns,
                   4.0 * (q.rows * (width + columns) + q.experts * width * columns));
        launch(product_kernel<Product::Weight>, dim3(tiles_of(columns), tiles_of(width), unsigned(q.experts)), dim3(256), 0,
               d.stream,
               ProductArgs{x, grad, nullptr, nullptr, grad_w, q.offsets, q.order, int(q.experts), ordered ? 0 : int(q.top_k),
                           int64_t(width), int64_t(columns)});
        after_launch("expert_backward_weight");
        p.done();
    });
}

int vc_hip_expert_combine_forward(const float* rows, const float* weights, const vc_hip_expert_plan* plan, size_t width,
                                  float* out) {
    return guard([&] {
        Device& d = require_device();
        const Plan q = plan_of(plan);
        if (q.tokens == 0 || width == 0) return;
        if (!rows || !out) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_combine: null pointer");
        Profiled p("expert_combine", 2.0 * q.rows * width, 4.0 * (q.rows + q.tokens) * width);
        launch(combine_kernel, dim3(grid_1d(width, 256, 64), unsigned(std::min<size_t>(q.tokens, 65535))), dim3(256), 0, d.stream,
               rows, weights, q.place, q.offsets, int(q.experts), int64_t(q.tokens), int(q.top_k), int64_t(width), out);
        after_launch("expert_combine");
        p.done();
    });
}

int vc_hip_expert_combine_backward(const float* grad, const float* rows, const float* weights,
                                   const vc_hip_expert_plan* plan, size_t width, float* grad_rows, float* grad_weights) {
    return guard([&] {
        Device& d = require_device();
        const Plan q = plan_of(plan);
        if (q.tokens == 0 || (!grad_rows && !grad_weights)) return;
        if (width && (!grad || (grad_rows && !weights) || (grad_weights && !rows)))
            fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_combine_backward: null pointer");
        Profiled p("expert_combine_backward", 3.0 * q.rows * width, 4.0 * (q.tokens + 2.0 * q.rows) * width);
        launch(combine_backward_kernel, dim3(unsigned((q.rows + 3) / 4)), dim3(256), 0, d.stream, grad, rows, weights, q.place,
               q.offsets, int(q.experts), int64_t(q.rows), int(q.top_k), int64_t(width), grad_rows, grad_weights);
        after_launch("expert_combine_backward");
        p.done();
    });
}

}  // extern "C"
