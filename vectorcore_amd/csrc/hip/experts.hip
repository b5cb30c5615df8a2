// A mixture of experts: the plan that sorts a batch's picks by expert, the
// products of each expert's rows with its matrices and their gradients, and
// the weighted sum of a token's picks.
#include "reduce_common.hpp"
#include "split_product.hpp"
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
// Up to one round of picks a single workgroup does both. Picks are numbered
// without a sign, as the last chunk and the last round may end behind 2^31.

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
    const unsigned begin = blockIdx.x * unsigned(chunk), end = min(unsigned(rows), begin + unsigned(chunk));
    for (unsigned p = begin + threadIdx.x; p < end; p += kPlanBlock) atomicAdd(&lds[group_of(chosen[p], experts)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += kPlanBlock) counts[blockIdx.x * (experts + 1) + e] = lds[e];
}

// counts: of every chunk, or null for one chunk counted here.
__global__ __launch_bounds__(kPlanBlock) void plan_place_kernel(const float* __restrict__ chosen, int rows, int chunk,
                                                                int experts, const int* __restrict__ counts,
                                                                int top_k, int* __restrict__ offsets, int* __restrict__ token,
                                                                int* __restrict__ place) {
    extern __shared__ int lds[];
    const int groups = experts + 1, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    int* const next = lds;                 // the chunk's next row of each group
    int* const total = lds + groups;       // all rows of each group, then their sum before it
    int* const found = lds + 2 * groups;   // [wave][group] of the round
    const unsigned begin = blockIdx.x * unsigned(chunk), end = min(unsigned(rows), begin + unsigned(chunk));
    for (int e = tid; e < groups; e += kPlanBlock) {
        int before = 0, all = 0;
        if (counts)
#pragma unroll 8
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
        for (unsigned p = begin + tid; p < end; p += kPlanBlock) atomicAdd(&total[group_of(chosen[p], experts)], 1);
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
    for (unsigned round = begin; round < end; round += kPlanBlock) {
        for (int i = tid; i < kPlanWaves * groups; i += kPlanBlock) found[i] = 0;
        __syncthreads();
        const unsigned p = round + tid;
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
            token[row] = int(p / unsigned(top_k));
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
    const int *offsets, *token, *place;
};

Plan plan_of(const vc_hip_expert_plan* plan) {
    if (!plan || (!plan->words && plan->tokens)) fail(VC_HIP_ERR_INVALID_ARGUMENT, "null expert plan");
    check_plan_sizes(plan->tokens, plan->top_k, plan->experts);
    const size_t rows = plan->tokens * plan->top_k;
    const int* words = plan->words;
    return Plan{plan->tokens, plan->top_k, plan->experts, rows, words, words + plan->experts + 2, words + plan->experts + 2 + rows};
}

// ---- products -----------------------------------------------------------------------
// Tiles of 64 or 128 rows of one group (split_product.hpp). Bound by the matrix
// instructions and, beside them, by the vector instructions that split operands:
// 16384 rows of 8 experts, 1024 x 4096, reach 177 TFLOP/s in the gated unit, 154 in
// the plain product, 170 to the rows and 170 to the weights, of 215 that a sixth of
// the library's bfloat16 rate would be. 49152 rows of 64 experts, 1024 x 512: 154,
// 151, 162 and 119, as sums of 768 rows leave prologues and stores a larger share.
//
// A sum that is not finite (an infinity or NaN among its operands, or a value that
// rounds to an infinity) is computed again by its lane, term after term: right, but
// slow where there are many. A training pass of the first batch: 8.0 ms, 174 with
// one token of NaN (all of its experts' gradients are), 388 with one such weight
// and 628 with one such expert.

using S = split::Bf16x3;

struct ProductArgs {
    const float *a, *b, *a2, *b2;
    float *c, *c2, *c3;
    const int *offsets, *token;  // token: of each row of a gathered A, null where A lies in row order
    int experts;
    int64_t width, columns;  // of each expert's matrix [width, columns]
    // Tiles of 64: parts of each tile's sum, workgroup w the part w / (grid / parts).
    int parts = 1;
    float* partial = nullptr;
    int down = 1;  // of a weight's tiles: rectangles above each other, 8 / down side by side
};

struct RowTile {
    int group, begin, end;  // rows of one group
    int64_t column;         // tile of columns
    bool live;
    int64_t id;  // of a live tile among all
};

constexpr int64_t kSplitTiles = 4096;        // whose sums are split, at most
__device__ unsigned g_tile_done[kSplitTiles];  // parts done; zero between launches, which never overlap

// A part's k, in whole slices.
struct Range {
    int64_t begin, end;
};
__device__ inline Range part_of(int64_t depth, int part, int parts) {
    if (parts == 1) return {0, depth};
    const int64_t slices = (depth + split::kSliceK - 1) / split::kSliceK;
    return {slices * part / parts * split::kSliceK, min(depth, slices * (part + 1) / parts * split::kSliceK)};
}

// The tile-th of the groups' tiles of Rows rows.
template <int Rows>
__device__ inline RowTile find_rows(const int* __restrict__ offsets, int groups, int tile, int64_t column) {
    const int lane = threadIdx.x % kWave;
    RowTile t{0, 0, 0, column, false, 0};
    for (int base = 0; base < groups; base += kWave) {
        const int e = base + lane;
        const int lo = e < groups ? offsets[e] : 0, hi = e < groups ? offsets[e + 1] : 0;
        const int n = (hi - lo + Rows - 1) / Rows;
        int upto = n;
        for (int d = 1; d < kWave; d <<= 1) {
            const int v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        const uint64_t past = __ballot(upto > tile);
        if (past) {
            const int at = __builtin_ctzll(past);
            t.live = true;
            t.group = base + at;
            t.begin = __shfl(lo, at) + (tile - __shfl(upto - n, at)) * Rows;
            t.end = min(__shfl(hi, at), t.begin + Rows);
            break;
        }
        tile -= __shfl(upto, kWave - 1);
    }
    t.group = __builtin_amdgcn_readfirstlane(t.group);
    t.begin = __builtin_amdgcn_readfirstlane(t.begin);
    t.end = __builtin_amdgcn_readfirstlane(t.end);
    return t;
}

// The tile of this workgroup. Row tiles are numbered group by group and taken
// eight at a time, those of a column together; each of the chip's eight dies
// (workgroups go to them in turn) gets neighbouring ones, which read the same
// operands through its cache.
template <int BM>
__device__ inline RowTile find_tile(const int* __restrict__ offsets, int groups, int64_t column_tiles, unsigned block) {
    const int lane = threadIdx.x % kWave;
    int all = 0;
    for (int base = 0; base < groups; base += kWave) {
        const int e = base + lane;
        const int n = e < groups ? (offsets[e + 1] - offsets[e] + BM - 1) / BM : 0;
        int sum = n;
        for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
        all += sum;
    }
    const int64_t total = all * column_tiles, share = (total + 7) / 8;
    const int64_t id = block % 8 * share + block / 8;
    if (block / 8 >= share || id >= total) return RowTile{0, 0, 0, 0, false, 0};
    const int64_t strip = id / (8 * column_tiles), place = id % (8 * column_tiles), high = min(int64_t(8), all - 8 * strip);
    RowTile t = find_rows<BM>(offsets, groups, int(8 * strip + place % high), place / high);
    t.id = id;
    return t;
}

__device__ inline float sigmoid(float x) {
    const float e = expf(-fabsf(x));
    return (x >= 0.0f ? 1.0f : e) / (1.0f + e);
}

// Slices on their way of tiles of `rows` rows.
constexpr int ahead(int rows) { return rows == 128 ? 1 : 3; }

// C[r] = x_r @ w[group], or silu(x_r @ gate) * (x_r @ up): there a tile holds
// 64 columns of both products, so that a thread holds both values of an element.
template <bool Gated, int BM>
__global__ __launch_bounds__(split::kThreads, Gated && BM == 128 ? 3 : 2) void forward_kernel(ProductArgs p) {
    constexpr int BN = Gated ? 128 : BM, kColumns = Gated ? BN / 2 : BN;
    __shared__ split::Slice<S, BM> as;
    __shared__ split::Slice<S, BN> bs;
    const int parts = BM == 64 ? p.parts : 1, tiles = int(gridDim.x) / parts, part = int(blockIdx.x) / tiles;
    const RowTile t = find_tile<BM>(p.offsets, p.experts + 1, (p.columns + kColumns - 1) / kColumns, blockIdx.x % tiles);
    if (!t.live) return;
    const int64_t n0 = t.column * kColumns;
    split::Tile<S, BM, BN> tile;
    tile.clear();
    const int64_t matrix = int64_t(t.group) * p.width * p.columns;
    const auto source = [&](int r) { return p.a + int64_t(p.token ? p.token[r] : r) * p.width; };
    if (t.group < p.experts) {
        using A = split::AlongK<BM>;
        using B = split::AcrossK<BN>;
        const Range range = part_of(p.width, part, parts);
        const float* pa[A::kChunks];
        unsigned at[B::kChunks];
#pragma unroll
        for (int j = 0; j < A::kChunks; ++j) pa[j] = source(min(t.begin + A::row(j), t.end - 1));
#pragma unroll
        for (int j = 0; j < B::kChunks; ++j)
            at[j] = unsigned(min(int64_t(Gated ? B::row(0) : B::row(j)), p.columns - 1 - n0));
        const float *const w = p.b + matrix + n0, *const w2 = Gated ? p.b2 + matrix + n0 : w;
        const auto line = [&](int64_t k) {
            const int64_t at_k = k * p.columns;
            return [=](int j) { return (j ? w2 : w) + at_k; };
        };
        split::accumulate<ahead(BM), A, B>(
            tile, as, bs, range.begin, range.end,
            [&](A& a, B& b, int64_t k) {
                a.load(pa, k);
                b.load(at, k, line);
            },
            [&](A& a, B& b, int64_t k) {
                a.load_rest(pa, k, p.width);
                b.load_rest(at, k, p.width, line);
            });
    }
    if constexpr (BM == 64) {
        __shared__ bool last;
        if (parts > 1 && !split::join(tile, part, parts, p.partial + t.id * parts * (BM * BN), &g_tile_done[t.id], last)) return;
    }
    // A lost sum, value by value.
    const auto again = [&](const float* w, int r, int64_t col) {
        const float* const x = source(r);
        float sum = 0.0f;
        for (int64_t k = 0; k < p.width; ++k) sum = fmaf(x[k], w[matrix + k * p.columns + col], sum);
        return sum;
    };
    if constexpr (Gated) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        const int64_t col = n0 + wave % 2 * 32 + lane % 32;
        if (col >= p.columns) return;
#pragma unroll
        for (int m = 0; m < tile.kM; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = t.begin + wave / 2 * (BM / 2) + 32 * m + 8 * (i / 4) + 4 * (lane / 32) + i % 4;
                if (r >= t.end) continue;
                float g = tile.acc[m][0][i], u = tile.acc[m][1][i];
                if (!split::finite(g)) g = again(p.b, r, col);
                if (!split::finite(u)) u = again(p.b2, r, col);
                const int64_t at = int64_t(r) * p.columns + col;
                p.c[at] = g * sigmoid(g) * u;
                if (p.c2) {
                    p.c2[at] = g;
                    p.c3[at] = u;
                }
            }
    } else {
        if (tile.lost() && t.group < p.experts)
            tile.each([&](int m, int n, float& v) {
                const int r = t.begin + m;
                const int64_t col = n0 + n;
                if (!split::finite(v) && r < t.end && col < p.columns) v = again(p.b, r, col);
            });
        tile.each([&](int m, int n, float v) {
            const int r = t.begin + m;
            const int64_t col = n0 + n;
            if (r < t.end && col < p.columns) p.c[int64_t(r) * p.columns + col] = v;
        });
    }
}

// C[r] = a[r] @ b[group]^T (+ a2[r] @ b2[group]^T).
template <int BM>
__global__ __launch_bounds__(split::kThreads, BM == 128 ? 3 : 2) void input_kernel(ProductArgs p) {
    __shared__ split::Slice<S, BM> as, bs;
    const int parts = BM == 64 ? p.parts : 1, tiles = int(gridDim.x) / parts, part = int(blockIdx.x) / tiles;
    const RowTile t = find_tile<BM>(p.offsets, p.experts + 1, (p.width + BM - 1) / BM, blockIdx.x % tiles);
    if (!t.live) return;
    const int64_t n0 = t.column * BM, matrix = int64_t(t.group) * p.width * p.columns;
    split::Tile<S, BM, BM> tile;
    tile.clear();
    const int products = p.a2 ? 2 : 1;
    const Range range = part_of(p.columns, part, parts);
    if (t.group < p.experts) {
        for (int product = 0; product < products; ++product) {
            const float *const from = product ? p.a2 : p.a, *const w = (product ? p.b2 : p.b) + matrix;
            using A = split::AlongK<BM>;
            const float *pa[A::kChunks], *pb[A::kChunks];
#pragma unroll
            for (int j = 0; j < A::kChunks; ++j) pa[j] = from + int64_t(min(t.begin + A::row(j), t.end - 1)) * p.columns;
#pragma unroll
            for (int j = 0; j < A::kChunks; ++j) pb[j] = w + min(n0 + A::row(j), p.width - 1) * p.columns;
            split::accumulate<ahead(BM), A, A>(
                tile, as, bs, range.begin, range.end,
                [&](A& a, A& b, int64_t k) {
                    a.load(pa, k);
                    b.load(pb, k);
                },
                [&](A& a, A& b, int64_t k) {
                    a.load_rest(pa, k, p.columns);
                    b.load_rest(pb, k, p.columns);
                });
        }
    }
    if constexpr (BM == 64) {
        __shared__ bool last;
        if (parts > 1 && !split::join(tile, part, parts, p.partial + t.id * parts * (BM * BM), &g_tile_done[t.id], last)) return;
    }
    if (tile.lost() && t.group < p.experts)  // sums again, value by value
        tile.each([&](int m, int n, float& v) {
            const int64_t r = t.begin + m, col = n0 + n;
            if (split::finite(v) || r >= t.end || col >= p.width) return;
            v = 0.0f;
            for (int product = 0; product < products; ++product) {
                const float *const x = (product ? p.a2 : p.a) + r * p.columns;
                const float *const w = (product ? p.b2 : p.b) + matrix + col * p.columns;
                for (int64_t k = 0; k < p.columns; ++k) v = fmaf(x[k], w[k], v);
            }
        });
    tile.each([&](int m, int n, float v) {
        const int64_t r = t.begin + m, col = n0 + n;
        if (r < t.end && col < p.width) p.c[r * p.width + col] = v;
    });
}

// C[e] = sum over e's rows of x_r^T b[r]. Every die takes a rectangle of each
// expert's tiles (experts differ in their rows): that of `down` by `across`.
template <int BM, int BN>
__global__ __launch_bounds__(split::kThreads, 2) void weight_kernel(ProductArgs p) {
    __shared__ split::Slice<S, BM> as;
    __shared__ split::Slice<S, BN> bs;
    const int64_t row_tiles = (p.width + BM - 1) / BM, column_tiles = (p.columns + BN - 1) / BN;
    const int64_t total = row_tiles * column_tiles, high = (row_tiles + p.down - 1) / p.down;
    const int64_t wide = (column_tiles + 8 / p.down - 1) / (8 / p.down), share = high * wide;
    const int parts = BM == 64 ? p.parts : 1, blocks = int(gridDim.x) / parts, part = int(blockIdx.x) / blocks;
    const int block = int(blockIdx.x) % blocks, unit = int(block / 8 / share), group = unit % p.experts;
    const float* const grad = unit < p.experts ? p.b : p.b2;
    float* const out = unit < p.experts ? p.c : p.c2;
    const int place = (block + unit) % 8;  // of the rectangle: those that are not whole go round the dies
    const int64_t row = place % p.down * high + block / 8 % share % high;
    const int64_t column = place / p.down * wide + block / 8 % share / high, id = row * column_tiles + column;
    if (row >= row_tiles || column >= column_tiles) return;
    const int64_t m0 = row * BM, n0 = column * BN;
    const int begin = p.offsets[group], depth = p.offsets[group + 1] - begin;
    const auto source = [&](int64_t r) { return int64_t(p.token ? p.token[r] : r) * p.width; };
    split::Tile<S, BM, BN> tile;
    tile.clear();
    using A = split::AcrossK<BM>;
    using B = split::AcrossK<BN>;
    unsigned at_a[A::kChunks], at_b[B::kChunks];
#pragma unroll
    for (int j = 0; j < A::kChunks; ++j) at_a[j] = unsigned(min(int64_t(A::row(j)), p.width - 1 - m0));
#pragma unroll
    for (int j = 0; j < B::kChunks; ++j) at_b[j] = unsigned(min(int64_t(B::row(j)), p.columns - 1 - n0));
    const auto line_a = [&](int64_t k) {
        const float* const line = p.a + m0 + source(begin + k);
        return [=](int) { return line; };
    };
    const auto line_b = [&](int64_t k) {
        const float* const line = grad + n0 + (begin + k) * p.columns;
        return [=](int) { return line; };
    };
    const Range range = part_of(depth, part, parts);
    split::accumulate<ahead(BM), A, B>(
        tile, as, bs, range.begin, range.end,
        [&](A& a, B& b, int64_t k) {
            a.load(at_a, k, line_a);
            b.load(at_b, k, line_b);
        },
        [&](A& a, B& b, int64_t k) {
            a.load_rest(at_a, k, depth, line_a);
            b.load_rest(at_b, k, depth, line_b);
        });
    if constexpr (BM == 64) {
        __shared__ bool last;
        const int64_t at = unit * total + id;
        if (parts > 1 && !split::join(tile, part, parts, p.partial + at * parts * (BM * BN), &g_tile_done[at], last)) return;
    }
    if (tile.lost())  // sums again, value by value
        tile.each([&](int m, int n, float& v) {
            const int64_t row = m0 + m, col = n0 + n;
            if (split::finite(v) || row >= p.width || col >= p.columns) return;
            v = 0.0f;
            for (int r = begin; r < begin + depth; ++r) v = fmaf(p.a[source(r) + row], grad[int64_t(r) * p.columns + col], v);
        });
    tile.each([&](int m, int n, float v) {
        const int64_t row = m0 + m, col = n0 + n;
        if (row < p.width && col < p.columns) out[(int64_t(group) * p.width + row) * p.columns + col] = v;
    });
}

// ---- few rows of each expert ----------------------------------------------------------
// Bound by reading the weights, which every expert's rows need once: a workgroup
// takes up to four rows of an expert, a tile of columns and a part of k. Each
// lane reads four columns of eight k at a time, and each weight goes into as many
// fused multiply-adds as there are rows; x is read from LDS. A wave reads whole
// 1 KiB lines of 256 columns, or, where few rows reach few experts, 256-byte
// lines of 64 columns at four places of k: the parts of k are then fewer and
// longer. The sums of the waves' k are added in LDS, those of workgroups by the
// one that counts in last, in order.
//
// Forward pass of 30 experts of 1024 x 1024, this and tiles of 64 rows: 4 rows an
// expert on average 91 and 129 us, 8 rows 129 and 126, 16 rows 154 and 130. One
// token of 2 of 16 experts, 1024 x 4096: 19.9 us for the two products of the gated
// unit (67 MB, 3.4 TB/s) and 14.1 for the third; 16 tokens that reach some 42 of 64
// experts, 1024 x 512: 36.8 and 21.0 us (174 and 87 MB, 4.7 and 4.1 TB/s). The
// average decides, as the host does not know the load. An uneven one costs no more:
// 384 rows of 64 experts, 1024 x 512, take 90 and 35 us evenly, 45 and 19 on six
// experts, 41 and 19 on one, whose weights the caches serve after the first rows.

constexpr int kThinRows = 4, kThinDepth = 512, kThinTiles = 4096;
constexpr size_t kThinMost = 6;  // rows of an expert on average

__device__ unsigned g_thin_done[kThinTiles];  // parts done of a tile; zero between launches

// out: of column threadIdx.x of the tile.
template <int Matrices, int Rows, int Columns>
__device__ inline void thin_sums(const ProductArgs& p, const RowTile& t, int64_t begin, int64_t end, float (*xs)[kThinDepth],
                                 float* sums, float (&out)[Rows][Matrices]) {
    constexpr int kPlaces = 256 / Columns, kLanes = kWave / kPlaces;  // places of k in a wave, lanes of each
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t n0 = t.column * Columns, col = n0 + 4 * (lane % kLanes);
    const int64_t matrix = int64_t(t.group) * p.width * p.columns;
    const int inside = int(min(int64_t(4), p.columns - col));  // of this lane's columns
    split::f4u acc[Rows][Matrices];
#pragma unroll
    for (int r = 0; r < Rows; ++r)
#pragma unroll
        for (int m = 0; m < Matrices; ++m) acc[r][m] = split::f4u{0, 0, 0, 0};
    for (int64_t k0 = begin; k0 < end; k0 += kThinDepth) {
        const int depth = int(min(int64_t(kThinDepth), end - k0)), padded = (depth + 7) / 8 * 8;
        for (int r = 0; r < Rows; ++r) {
            const int row = min(t.begin + r, t.end - 1);
            const float* const x = p.a + int64_t(p.token ? p.token[row] : row) * p.width + k0;
            for (int k = threadIdx.x; k < padded; k += 256) xs[r][k] = k < depth ? x[k] : 0.0f;
        }
        __syncthreads();
        for (int k = 8 * (kPlaces * wave + lane / kLanes); k < depth; k += 32 * kPlaces) {
            split::f4u w[Matrices][8];
            const unsigned at = unsigned(k) * unsigned(p.columns) + unsigned(col - n0);
#pragma unroll
            for (int m = 0; m < Matrices; ++m) {
                const float* const from = (m ? p.b2 : p.b) + matrix + k0 * p.columns + n0;  // uniform
                if (k + 8 <= depth && n0 + Columns <= p.columns) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[m][i] = *reinterpret_cast<const split::f4u*>(from + i * p.columns + at);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) w[m][i][c] = k + i < depth && c < inside ? (from + i * p.columns)[at + c] : 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < Rows; ++r)
#pragma unroll
                for (int m = 0; m < Matrices; ++m)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[r][m][c] = fmaf(xs[r][k + i], w[m][i][c], acc[r][m][c]);
        }
        __syncthreads();
    }
    const int place = wave * kPlaces + lane / kLanes;
#pragma unroll
    for (int r = 0; r < Rows; ++r)
#pragma unroll
        for (int m = 0; m < Matrices; ++m) {
#pragma unroll
            for (int c = 0; c < 4; ++c) sums[place * Columns + 4 * (lane % kLanes) + c] = acc[r][m][c];
            __syncthreads();
            float sum = 0.0f;
#pragma unroll
            for (int q = 0; q < 4 * kPlaces; ++q) sum += sums[q * Columns + threadIdx.x % Columns];
            out[r][m] = sum;
            __syncthreads();
        }
}

template <bool Gated, int Rows, int Columns>
__device__ inline void thin_tile(const ProductArgs& p, const RowTile& t, int part, int splits, int64_t tile, float* partial,
                                 float (*xs)[kThinDepth], float* sums, bool& finisher) {
    constexpr int kMatrices = Gated ? 2 : 1;
    const int64_t groups = (p.width + 7) / 8;
    const int64_t begin = min(p.width, groups * part / splits * 8), end = min(p.width, groups * (part + 1) / splits * 8);
    float out[Rows][kMatrices];
    thin_sums<kMatrices, Rows, Columns>(p, t, begin, end, xs, sums, out);
    const bool mine = threadIdx.x < Columns;
    if (splits > 1) {
        constexpr int kValues = Rows * kMatrices;
        float* const parts = partial + tile * splits * (kThinRows * kMatrices * Columns) + threadIdx.x % Columns;
        if (mine) {
#pragma unroll
            for (int v = 0; v < kValues; ++v)
                __hip_atomic_store(&parts[(part * kValues + v) * Columns], out[v / kMatrices][v % kMatrices], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        }
        red::wait_stores_visible();
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned* const done = &g_thin_done[tile];
            finisher = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == unsigned(splits);
            if (finisher) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!finisher) return;
#pragma unroll
        for (int v = 0; v < kValues; ++v) {
            float sum = 0.0f;
            for (int q = 0; q < splits; q += 8) {
                float ahead[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    ahead[i] = __hip_atomic_load(&parts[(min(q + i, splits - 1) * kValues + v) * Columns], __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (q + i < splits) sum += ahead[i];
            }
            out[v / kMatrices][v % kMatrices] = sum;
        }
    }
    const int64_t col = t.column * Columns + threadIdx.x;
    if (!mine || col >= p.columns) return;
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        if (t.begin + r >= t.end) break;
        const int64_t at = int64_t(t.begin + r) * p.columns + col;
        if constexpr (Gated) {
            const float g = out[r][0], u = out[r][1];
            p.c[at] = g * sigmoid(g) * u;
            if (p.c2) {
                p.c2[at] = g;
                p.c3[at] = u;
            }
        } else {
            p.c[at] = out[r][0];
        }
    }
}

// Workgroups in the order of rows, columns, parts of k.
template <bool Gated, int Columns>
__global__ __launch_bounds__(256, Gated ? 2 : 3) void thin_kernel(ProductArgs p, int splits, float* partial) {
    __shared__ float xs[kThinRows][kThinDepth], sums[1024];
    __shared__ bool finisher;
    const int64_t column_tiles = (p.columns + Columns - 1) / Columns;
    const int part = int(blockIdx.x % splits);
    const int64_t tile = blockIdx.x / splits;
    const RowTile t = find_rows<kThinRows>(p.offsets, p.experts + 1, int(tile / column_tiles), tile % column_tiles);
    if (!t.live) return;
    if (t.group == p.experts) {  // dropped picks: zero rows
        const int64_t col = t.column * Columns + threadIdx.x;
        if (part || threadIdx.x >= Columns || col >= p.columns) return;
        for (int64_t r = t.begin; r < t.end; ++r) {
            p.c[r * p.columns + col] = 0.0f;
            if (Gated && p.c2) p.c2[r * p.columns + col] = p.c3[r * p.columns + col] = 0.0f;
        }
        return;
    }
    const int rows = t.end - t.begin;
    if (rows == 1) thin_tile<Gated, 1, Columns>(p, t, part, splits, tile, partial, xs, sums, finisher);
    else if (rows == 2) thin_tile<Gated, 2, Columns>(p, t, part, splits, tile, partial, xs, sums, finisher);
    else thin_tile<Gated, 4, Columns>(p, t, part, splits, tile, partial, xs, sums, finisher);
}

int64_t tiles_of(size_t n, int tile) { return int64_t((n + tile - 1) / tile); }

// A grid for `tiles` tiles at most, in whole rounds of the eight dies.
dim3 tile_grid(int64_t tiles) {
    const int64_t blocks = (tiles + 7) / 8 * 8;
    if (blocks > int64_t(kMostBlocks)) fail(VC_HIP_ERR_OVERFLOW, "expert product: too many tiles");
    return dim3(unsigned(blocks));
}
// Row tiles by column tiles at most.
int64_t tiles_at_most(const Plan& plan, int rows, size_t width, int columns) {
    return int64_t(plan.rows / rows + plan.experts + 1) * tiles_of(width, columns);
}

// Parts of a sum over `depth` for `tiles` tiles of 64, at least four slices each,
// for four workgroups on every CU, and the memory for `values` of every tile and
// part. (Training passes, this, two workgroups with eight slices, and six with
// four: 256 tokens of 8 experts 1024 x 1024 207, 231 and 206 us; 999 of 5 experts
// 131 x 515 144, 151 and 142; 2048 of 4 experts 512 x 512 184, 193 and 200.)
struct Parts {
    int64_t parts;
    Scratch partial;
    Parts(Device& d, int64_t tiles, int64_t depth, int64_t values)
        : parts(tiles > kSplitTiles ? 1 : std::max<int64_t>(1, std::min(4 * d.cu_count / std::max<int64_t>(1, tiles), depth / 128))),
          partial(parts > 1 ? size_t(tiles * parts * values) * sizeof(float) : 4) {}
    ProductArgs operator()(ProductArgs args) const {
        args.parts = int(parts);
        args.partial = partial.as<float>();
        return args;
    }
};
dim3 operator*(dim3 grid, int64_t parts) {
    if (grid.x * parts > int64_t(kMostBlocks)) fail(VC_HIP_ERR_OVERFLOW, "expert product: too many tiles");
    return dim3(unsigned(grid.x * parts));
}

// Whether tiles of 128 rows give every CU one; otherwise tiles of 64 halve or
// quarter what each of them computes. A training pass of 8 experts, 1024 x 1024,
// two a token, by tiles of 128 and of 64: 256 tokens 453 and 312 us, 1024 tokens
// 555 and 505, 2048 tokens 800 and 799, 4096 tokens 1278 and 1327.
bool enough(Device& d, int64_t tiles) { return tiles >= d.cu_count; }

// (A lane's place in kThinDepth lines is a 32-bit offset.)
bool thin(const Plan& plan, size_t columns) { return plan.rows <= kThinMost * plan.experts && columns <= size_t(1) << 20; }

// Parts of k, of 64 to 128 at least, for three workgroups on every CU; narrow
// tiles of columns where wide ones would leave that to more than six parts.
template <bool Gated, int Columns>
void launch_thin(Device& d, int64_t rows, const ProductArgs& args) {
    const int64_t tiles = rows * tiles_of(size_t(args.columns), Columns), wanted = (3 * d.cu_count + tiles - 1) / tiles;
    const int64_t splits = tiles > kThinTiles ? 1 : std::max<int64_t>(1, std::min(wanted, args.width / (Columns == 64 ? 128 : 64)));
    if (tiles * splits > int64_t(kMostBlocks)) fail(VC_HIP_ERR_OVERFLOW, "expert product: too many tiles");
    Scratch partial(splits > 1 ? size_t(tiles * splits) * kThinRows * Columns * (Gated ? 2 : 1) * sizeof(float) : 4);
    launch(thin_kernel<Gated, Columns>, dim3(unsigned(tiles * splits)), dim3(256), 0, d.stream, args, int(splits),
           partial.as<float>());
}
template <bool Gated>
void launch_thin(Device& d, const Plan& plan, const ProductArgs& args) {
    const int64_t rows = std::min<int64_t>(plan.rows, int64_t(plan.rows / kThinRows + plan.experts + 1));
    if (2 * rows * tiles_of(size_t(args.columns), 256) < d.cu_count) launch_thin<Gated, 64>(d, rows, args);
    else launch_thin<Gated, 256>(d, rows, args);
}

// ---- the gated unit -------------------------------------------------------------------

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

// Bound by HBM: four columns a lane, the rows of four picks on their way. A row's
// last four columns may lie in two lanes' reach; both store the same. Blocks are
// as many lanes wide as a row needs. (49152 rows of 1024: 39.8 us, 5.9 TB/s; a
// column a lane and a row at a time 75. The gradients below: 77.9 and 106 us.)
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ rows, const float* __restrict__ weights,
                                                      const int* __restrict__ place, const int* __restrict__ offsets,
                                                      int experts, int64_t tokens, int top_k, int64_t width,
                                                      float* __restrict__ out) {
    const int kept = offsets[experts];  // rows of dropped picks come after
    const int64_t chunk = 4 * (int64_t(blockIdx.x) * blockDim.x + threadIdx.x);
    if (chunk >= width) return;
    const bool whole = width >= 4;
    const int64_t i = whole ? min(chunk, width - 4) : 0;
    const int some = int(min(width, int64_t(4)));
    for (int64_t t = int64_t(blockIdx.y) * blockDim.y + threadIdx.y; t < tokens; t += int64_t(gridDim.y) * blockDim.y) {
        split::f4u sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int j0 = 0; j0 < top_k; j0 += 4) {
            split::f4u v[4];
            float w[4];
            int at[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) at[j] = j0 + j < top_k ? place[t * top_k + j0 + j] : kept;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = split::f4u{0.0f, 0.0f, 0.0f, 0.0f};
                w[j] = 0.0f;
                if (at[j] < kept) {
                    const float* const from = rows + at[j] * width + i;
                    if (whole) v[j] = *reinterpret_cast<const split::f4u*>(from);
                    else
                        for (int e = 0; e < some; ++e) v[j][e] = from[e];
                    w[j] = weights ? weights[t * top_k + j0 + j] : 1.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(w[j], v[j][e], sum[e]);
        }
        if (whole) *reinterpret_cast<split::f4u*>(out + t * width + i) = sum;
        else
            for (int e = 0; e < some; ++e) out[t * width + e] = sum[e];
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
    const int64_t p = block_id() * 4 + threadIdx.x / kWave;
    if (p >= picks) return;
    const int64_t r = place[p];
    const float* const g = grad + p / top_k * width;
    const bool dropped = r >= kept;
    const float w = weights && !dropped ? weights[p] : 0.0f;
    double dot = 0.0;
    const float* const from = rows + r * width;
    float* const to = grad_rows + r * width;
    int64_t i = 4 * lane;
#pragma unroll 4
    for (; i + 4 <= width; i += 4 * kWave) {
        const split::f4u v = *reinterpret_cast<const split::f4u*>(g + i);
        if (grad_weights && !dropped) {
            const split::f4u z = *reinterpret_cast<const split::f4u*>(from + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) dot += double(v[e]) * double(z[e]);
        }
        if (grad_rows) {
            split::f4u d;
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = dropped ? 0.0f : w * v[e];
            *reinterpret_cast<split::f4u*>(to + i) = d;
        }
    }
    for (; i < width; ++i) {  // of the one lane whose four columns end outside
        const float v = g[i];
        if (grad_weights && !dropped) dot += double(v) * double(from[i]);
        if (grad_rows) to[i] = dropped ? 0.0f : w * v;
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
        int* const token = words + experts + 2;
        int* const counts = token + 2 * rows;
        Profiled p("expert_plan", 0.0, 12.0 * rows);
        const uint32_t lds = uint32_t((2 + kPlanWaves) * (experts + 1) * sizeof(int));
        if (chunks > 1) {
            launch(plan_count_kernel, dim3(unsigned(chunks)), dim3(kPlanBlock), uint32_t((experts + 1) * sizeof(int)), d.stream,
                   chosen, int(rows), int(chunk), int(experts), counts);
            after_launch("expert plan counts");
        }
        launch(plan_place_kernel, dim3(unsigned(std::max<size_t>(chunks, 1))), dim3(kPlanBlock), lds, d.stream, chosen,
               int(rows), int(chunk), int(experts), static_cast<const int*>(chunks > 1 ? counts : nullptr),
               int(top_k), words, token, token + rows);
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
        const ProductArgs args{x, w, nullptr, nullptr, out, nullptr, nullptr, q.offsets, ordered ? nullptr : q.token,
                               int(q.experts), int64_t(width), int64_t(columns)};
        const dim3 threads(split::kThreads);
        if (thin(q, columns))
            launch_thin<false>(d, q, args);
        else if (enough(d, int64_t(q.rows / 128) * tiles_of(columns, 128)))
            launch(forward_kernel<false, 128>, tile_grid(tiles_at_most(q, 128, columns, 128)), threads, 0, d.stream, args);
        else {
            const int64_t tiles = tiles_at_most(q, 64, columns, 64);
            const Parts parts(d, tiles, args.width, 64 * 64);
            launch(forward_kernel<false, 64>, tile_grid(tiles) * parts.parts, threads, 0, d.stream, parts(args));
        }
        after_launch("expert_linear");
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
        const ProductArgs args{x, gate, nullptr, up, out, save_gate, save_up, q.offsets, ordered ? nullptr : q.token,
                               int(q.experts), int64_t(width), int64_t(columns)};
        const dim3 threads(split::kThreads);
        if (thin(q, columns))
            launch_thin<true>(d, q, args);
        else if (enough(d, int64_t(q.rows / 128) * tiles_of(columns, 64)))
            launch(forward_kernel<true, 128>, tile_grid(tiles_at_most(q, 128, columns, 64)), threads, 0, d.stream, args);
        else {
            const int64_t tiles = tiles_at_most(q, 64, columns, 64);
            const Parts parts(d, tiles, args.width, 64 * 128);
            launch(forward_kernel<true, 64>, tile_grid(tiles) * parts.parts, threads, 0, d.stream, parts(args));
        }
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
        const ProductArgs args{grad, w, grad2, w2, grad_rows, nullptr, nullptr, q.offsets, nullptr, int(q.experts),
                               int64_t(width), int64_t(columns)};
        const dim3 threads(split::kThreads);
        if (enough(d, int64_t(q.rows / 128) * tiles_of(width, 128)))
            launch(input_kernel<128>, tile_grid(tiles_at_most(q, 128, width, 128)), threads, 0, d.stream, args);
        else {
            const int64_t tiles = tiles_at_most(q, 64, width, 64);
            const Parts parts(d, tiles, args.columns, 64 * 64);
            launch(input_kernel<64>, tile_grid(tiles) * parts.parts, threads, 0, d.stream, parts(args));
        }
        after_launch("expert_backward_input");
        p.done();
    });
}

int vc_hip_expert_linear_backward_weight(const float* x, const float* grad, const float* grad2,
                                         const vc_hip_expert_plan* plan, size_t width, size_t columns, int ordered,
                                         float* grad_w, float* grad_w2) {
    return guard([&] {
        Device& d = require_device();
        const Plan q = plan_of(plan);
        if (!grad_w2 != !grad2) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_linear_backward_weight: half of a second product");
        if (width == 0 || columns == 0) return;
        if (!grad_w || (q.rows && (!x || !grad))) fail(VC_HIP_ERR_INVALID_ARGUMENT, "expert_linear_backward_weight: null pointer");
        if (q.rows == 0) {  // zeros, without the plan's words, which no token needs
            for (float* const out : {grad_w, grad_w2})
                if (out)
                    if (const int status = vc_hip_fill(out, q.experts * width * columns, 0.0f)) fail(status, vc_hip_last_error());
            return;
        }
        const int64_t products = grad2 ? 2 : 1;
        Profiled p("expert_backward_weight", products * 2.0 * q.rows * width * columns,
                   4.0 * (q.rows * (width + products * columns) + products * q.experts * width * columns));
        const ProductArgs args{x, grad, nullptr, grad2, grad_w, grad_w2, nullptr, q.offsets, ordered ? nullptr : q.token,
                               int(q.experts), int64_t(width), int64_t(columns)};
        // 256 columns a tile where they fill the chip: x is then split half as often. (8 experts, 1024 x 4096 over 16384
        // rows: 809 us, with 128 columns 935. The products of rows gain nothing, as fewer tiles fit the CUs less evenly.)
        const auto run = [&](auto bm, auto bn, ProductArgs a, int64_t parts) {
            // The rectangles that read the least.
            const int64_t rows = tiles_of(width, bm()), cols = tiles_of(columns, bn());
            int64_t least = 0, share = 0;
            for (int down = 1; down <= 8; down *= 2) {
                const int64_t high = (rows + down - 1) / down, wide = (cols + 8 / down - 1) / (8 / down);
                const int64_t reads = high * wide * 1024 + high * bm() + wide * bn();  // tiles first: rounding up adds empty ones
                if (share == 0 || reads < least) {
                    least = reads;
                    share = high * wide;
                    a.down = down;
                }
            }
            launch(weight_kernel<bm(), bn()>, tile_grid(products * int64_t(q.experts) * share * 8) * parts, dim3(split::kThreads),
                   0, d.stream, a);
        };
        using std::integral_constant;
        const int64_t row_tiles = products * int64_t(q.experts) * tiles_of(width, 128);
        if (row_tiles * tiles_of(columns, 256) >= 2 * d.cu_count) {
            run(integral_constant<int, 128>(), integral_constant<int, 256>(), args, 1);
        } else if (enough(d, row_tiles * tiles_of(columns, 128))) {
            run(integral_constant<int, 128>(), integral_constant<int, 128>(), args, 1);
        } else {
            const int64_t tiles = products * int64_t(q.experts) * tiles_of(width, 64) * tiles_of(columns, 64);
            const Parts parts(d, tiles, int64_t(q.rows / q.experts), 64 * 64);
            run(integral_constant<int, 64>(), integral_constant<int, 64>(), parts(args), parts.parts);
        }
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
        unsigned lanes = 1;
        while (lanes < 256 && 4 * lanes < width) lanes *= 2;
        const unsigned tokens = 256 / lanes;
        const size_t across = (width + 4 * lanes - 1) / (4 * lanes);
        if (across > kMostBlocks) fail(VC_HIP_ERR_OVERFLOW, "expert_combine: rows too long");
        launch(combine_kernel, dim3(unsigned(across), unsigned(std::min<size_t>((q.tokens + tokens - 1) / tokens, 65535))),
               dim3(lanes, tokens), 0, d.stream,
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
        launch(combine_backward_kernel, grid_2d((q.rows + 3) / 4), dim3(256), 0, d.stream, grad, rows, weights, q.place,
               q.offsets, int(q.experts), int64_t(q.rows), int(q.top_k), int64_t(width), grad_rows, grad_weights);
        after_launch("expert_combine_backward");
        p.done();
    });
}

}  // extern "C"
