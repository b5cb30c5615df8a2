// Products C = A B^T of float32 values near one on the half-precision matrix
// instructions, with operands that were split when they were written.
//
// x = x1 + x2 with half-precision parts, 22 bits of x; of the four products x2 y2
// (2^-22 of the largest) is left out. Three instructions of 32 cycles take the
// place of eight of 64 (V_MFMA_F32_32X32X2_F32). Half precision ends at 65504 and
// steps by 2^-24 at zero: the caller scales its values into that range.
//
// A matrix is stored as its parts: 32 neighbouring values of a row are one
// 128-byte line, their first parts, then their second ones. An operand is k
// contiguous, its rows and k padded with zeros to whole tiles, so a slice of 32 k
// goes to LDS by loads that write there directly, a line in eight 16-byte chunks,
// without a vector instruction. (Vector instructions do not run beside matrix
// instructions: two waves a SIMD that issue both took the sum of their times.)
#pragma once

#include "reduce_common.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vchip {
namespace packed {

constexpr int kThreads = 256, kSlice = 32, kLine = 64;  // halves of a line

typedef _Float16 half;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// Element (row, k) of a matrix with rows of `depth` values (a multiple of 32).
__host__ __device__ inline int64_t place(int64_t row, int64_t k, int64_t depth) {
    return row * 2 * depth + k / kSlice * kLine + k % kSlice;
}

// What a value is stored as: its parts in the low and the high half.
__device__ inline uint32_t parts(float v) {
    const _Float16 first = _Float16(v), second = _Float16(v - float(first));
    return uint32_t(__builtin_bit_cast(uint16_t, first)) | uint32_t(__builtin_bit_cast(uint16_t, second)) << 16;
}

// Four values along k, k a multiple of 4.
__device__ inline void store4(_Float16* to, const float (&v)[4]) {
    h4 first, second;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        first[i] = _Float16(v[i]);
        second[i] = _Float16(v[i] - float(first[i]));
    }
    *reinterpret_cast<h4*>(to) = first;
    *reinterpret_cast<h4*>(to + kSlice) = second;
}
// s_waitcnt that leaves `loads` vector memory operations in flight.
template <int Loads>
__device__ inline void wait_loads() {
    __builtin_amdgcn_s_waitcnt((Loads & 15) | (Loads >> 4) << 14 | 0x0F70);
}

// A tile of BT x BT by four waves, each a quarter in 32 x 32 blocks.
template <int BT, int Stages>
struct Tile {
    static constexpr int kBlocks = BT / 64;       // of a wave, each way
    static constexpr int kLoads = BT / 32;        // of a wave, operand and slice
    static constexpr int kStage = 2 * BT * 128;   // bytes
    static constexpr int kLds = Stages * kStage;
    f16v acc[kBlocks][kBlocks];

    __device__ inline void clear() {
#pragma unroll
        for (int a = 0; a < kBlocks; ++a)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
    }

    // One load: 64 chunks of 16 bytes, lane l's to byte 16 l of the wave's part
    // of the stage. Inline assembly, as the compiler would wait for every load in
    // flight before LDS reads that it cannot tell apart; what a stage's loads
    // have written is waited for before the barrier that hands it on.
    template <int At>
    static __device__ inline void load_one(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t uniform, uint32_t lds) {
        asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :
                     : "s"(lds), "v"(off), "s"(rs), "s"(uniform), "i"(At)
                     : "memory", "m0", "scc");
    }
    template <int Q, int At>
    static __device__ inline void load_rows(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t step, uint32_t lds) {
        if constexpr (Q < kLoads) {
            load_one<At + 4096 * Q>(rs, off, Q * step, lds);
            load_rows<Q + 1, At>(rs, off, step, lds);
        }
    }

    // acc += the products of k slices [begin, end) of BT rows of each operand;
    // a, b: their first rows; depth: k of a whole row. lds: kLds bytes.
    //
    // Row r's chunk c (first parts 0 to 3, second 4 to 7) lies in slot c ^ (r / 2 % 8)
    // of its 128 bytes: 16 rows of a fragment then meet different banks. Slice
    // s + Stages - 1 is requested while slice s is multiplied. Apart: the products
    // with a second part have sums of their own, so that the large sums round a third
    // as often (of G's diagonal over 416 k: 1.8 x 2^-24 of it, 4.0 in one sum; five
    // iterations of 31 matrices of 26 x 3266: 1.3e-6 of the norm, 2.5e-6).
    template <bool Apart>
    __device__ inline void accumulate(const _Float16* a, const _Float16* b, int64_t depth, int64_t begin, int64_t end, char* lds) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        const uint32_t row_bytes = uint32_t(depth) * 4u;
        const uint32_t off = uint32_t(8 * wave + lane / 8) * row_bytes + uint32_t((lane % 8) ^ (4 * (wave % 2) + lane / 16)) * 16u;
        const uint32_t to = __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)lds)) + 1024u * uint32_t(wave));
        const auto request = [&](int64_t s, int stage) {
            const int64_t at = min(s, end - 1) * kLine;
            const uint32_t dst = to + uint32_t(stage) * kStage;
            load_rows<0, 0>(__builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16*>(a + at), short(0), 0x7FFFFFFE, 0x00020000), off,
                            32u * row_bytes, dst);
            load_rows<0, BT * 128>(__builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16*>(b + at), short(0), 0x7FFFFFFE, 0x00020000),
                                   off, 32u * row_bytes, dst);
        };
        const int half = lane / 32, swizzle = lane / 2 % 8;
        const int row_a = wave / 2 * (BT / 2) + lane % 32, row_b = BT + wave % 2 * (BT / 2) + lane % 32;
        f16v small[Apart ? kBlocks : 1][Apart ? kBlocks : 1] = {};  // of the products with a second part
        const auto multiply = [&](int stage) {
            const char* const from = lds + stage * kStage;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                h8 x[kBlocks][2], y[kBlocks][2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int slot = ((4 * q + 2 * t + half) ^ swizzle) * 16;
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i) {
                        x[i][q] = *reinterpret_cast<const h8*>(from + (row_a + 32 * i) * 128 + slot);
                        y[i][q] = *reinterpret_cast<const h8*>(from + (row_b + 32 * i) * 128 + slot);
                    }
                }
#pragma unroll
                for (int p = 0; p < 3; ++p)  // the small products first
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                        for (int j = 0; j < kBlocks; ++j) {
                            f16v& sum = Apart && p < 2 ? small[Apart ? i : 0][Apart ? j : 0] : acc[i][j];
                            sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i][p == 1], y[j][p == 0], sum, 0, 0, 0);
                        }
            }
        };
#pragma unroll
        for (int s = 0; s < Stages - 1; ++s) request(begin + s, s);
        int stage = 0;
        for (int64_t s = begin; s < end; ++s) {
            wait_loads<2 * kLoads * (Stages - 2)>();
            __syncthreads();  // slice s is there, and slice s - 1 has been read
            request(s + Stages - 1, stage == 0 ? Stages - 1 : stage - 1);
            multiply(stage);
            stage = stage == Stages - 1 ? 0 : stage + 1;
        }
        wait_loads<0>();  // no load may land in LDS that others use by then
        if constexpr (Apart) {
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int j = 0; j < kBlocks; ++j) acc[i][j] += small[i][j];
        }
    }

    // f(row, column, v) for four values in neighbouring rows of a column.
    template <class F>
    __device__ inline void each4(F&& f) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
#pragma unroll
        for (int a = 0; a < kBlocks; ++a)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = acc[a][b][4 * g + i];
                    f(wave / 2 * (BT / 2) + 32 * a + 8 * g + 4 * (lane / 32), wave % 2 * (BT / 2) + 32 * b + lane % 32, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[a][b][4 * g + i] = v[i];
                }
    }

    // This thread's place of the tile from element (m0, n0) of a matrix: 32 lanes hold a line, the even ones first parts and
    // the odd ones second parts of two neighbours. f(place, value) for each value.
    template <class P, class F>
    __device__ inline void each_place(P* matrix, int64_t m0, int64_t n0, int64_t depth, F&& f) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        P* const line = matrix + place(m0 + wave / 2 * (BT / 2) + 4 * (lane / 32), n0 + wave % 2 * (BT / 2), depth) +
                        lane % 2 * kSlice + lane % 32 / 2 * 2;
#pragma unroll
        for (int a = 0; a < kBlocks; ++a)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float v = acc[a][b][i];
                    f(line + (32 * a + 8 * (i / 4) + i % 4) * 2 * depth + b * kLine, v);
                    acc[a][b][i] = v;
                }
    }
    // Two neighbours' parts, of one kind each, to one's parts of both kinds, and back.
    static __device__ inline uint32_t exchange(uint32_t mine) {
        const int lane = red::lane_id();
        return __builtin_amdgcn_perm(red::partner<0>(mine, lane), mine, lane % 2 ? 0x03020706u : 0x05040100u);
    }
    __device__ inline void store(half* to, int64_t m0, int64_t n0, int64_t depth) {
        each_place(to, m0, n0, depth, [](half* at, float& v) { *reinterpret_cast<uint32_t*>(at) = exchange(parts(v)); });
    }
    // tile = a * matrix + b * tile.
    __device__ inline void mix(float a, const half* matrix, float b, int64_t m0, int64_t n0, int64_t depth) {
        each_place(matrix, m0, n0, depth, [&](const half* at, float& v) {
            const uint32_t both = exchange(*reinterpret_cast<const uint32_t*>(at));
            const float x = float(__builtin_bit_cast(half, uint16_t(both))) + float(__builtin_bit_cast(half, uint16_t(both >> 16)));
            v = a * x + b * v;
        });
    }
    // The tile transposed: its element (row, column) becomes (n0 + column, m0 + row). A wave collects 32 rows of it in LDS,
    // a line of each column, and writes whole lines. lds: of the finished accumulate().
    __device__ inline void store_transposed(half* to, int64_t m0, int64_t n0, int64_t depth, char* lds) {
        constexpr int kColumns = BT / 2, kStride = 128 + 16;  // of a wave; bytes, so that neighbours meet other banks
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        static_assert(4 * kColumns * kStride <= kLds, "the waves' lines exceed the stages");
        char* const mine = lds + wave * kColumns * kStride;
        __syncthreads();  // no wave reads the stages any more
#pragma unroll
        for (int a = 0; a < kBlocks; ++a) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = acc[a][b][4 * g + i];
                    store4(reinterpret_cast<half*>(mine + (32 * b + lane % 32) * kStride) + 8 * g + 4 * (lane / 32), v);
                }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            half* const line = to + place(n0 + wave % 2 * kColumns, m0 + wave / 2 * (BT / 2) + 32 * a, depth);
#pragma unroll
            for (int c = 0; c < kColumns; c += 8)
                *reinterpret_cast<h8*>(line + (c + lane / 8) * 2 * depth + lane % 8 * 8) =
                    *reinterpret_cast<const h8*>(mine + (c + lane / 8) * kStride + lane % 8 * 16);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }
};

}  // namespace packed
}  // namespace vchip
