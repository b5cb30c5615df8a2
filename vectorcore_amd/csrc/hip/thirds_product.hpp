// Products C = A B^T of float32 values at float32's precision whatever the values,
// on the tiles of halves_product.hpp: the form for operands whose rows hold values
// too unlike for two half-precision parts.
//
// A value, scaled by a power of two of its row, is the sum of three bfloat16 parts,
// each the rounding of what the earlier ones leave: all 24 bits of every value down
// to 2^-123 of its row's largest. Of the nine products of two values' parts those
// below 2^-26 of the largest are left out; six instructions for three. A part of an
// infinity or a NaN is an infinity or a NaN, and so is every sum that it is in.
//
// An operand is stored as the matrix instructions read it: of each 256 rows and 16
// k one block of 16 KiB, [part][k / 8][row][8], of the first two parts, which take
// the place of the two half parts, and one of 8 KiB of the third parts elsewhere. A
// slice of either operand is then two runs of memory, of which every wave loads 1
// KiB at a time straight to LDS, and a fragment is read without bank conflicts.
//
// Bound by the matrix instructions: 7373 x 1024 by 50000 long sums take 3.25 ms (232
// TFLOP/s of float32 products, 1393 of bfloat16 ones), two half parts 1.81.
#pragma once

#include "halves_product.hpp"

namespace vchip {
namespace thirds {

using halves::kThreads;
using halves::kTile;

constexpr int kSlice = 16, kParts = 3, kPart = 2 * kTile * 16;  // bytes of a part of a block
constexpr int kStages = 3, kLds = kStages * 2 * kParts * kPart;

typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2v __attribute__((ext_vector_type(2)));

// A packed operand: its first parts, which hold both half parts otherwise, and its third ones.
struct Operand {
    halves::half *first, *third;
};

// Of rows of `lines` times 32 k: the eight from 8 k8 of a row, scaled by 2^e.
__device__ inline void store8(const Operand& to, int lines, int64_t row, int64_t k8, const float (&v)[8], int e) {
    f2v rest[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rest[i] = f2v{__builtin_amdgcn_ldexpf(v[2 * i], e), __builtin_amdgcn_ldexpf(v[2 * i + 1], e)};
    const int64_t block = (row / kTile) * (2 * int64_t(lines)) + k8 / 2, in = k8 % 2 * kTile + row % kTile;
    b8* const first = reinterpret_cast<b8*>(to.first) + block * (4 * kTile) + in;
    b8* const third = reinterpret_cast<b8*>(to.third) + block * (2 * kTile) + in;
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
        b8 out;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const b2 part = __builtin_convertvector(rest[i], b2);
            out[2 * i] = part[0];
            out[2 * i + 1] = part[1];
            rest[i][0] -= float(part[0]);
            rest[i][1] -= float(part[1]);
        }
        if (p < 2) first[2 * p * kTile] = out;
        else *third = out;
    }
}

// Bytes of the third parts of an operand's tile; its first two take twice that, as much as its half parts.
__host__ __device__ inline int64_t third_bytes(int lines) { return 2 * int64_t(lines) * kPart; }
__device__ inline Operand tile_of(const Operand& of, int64_t tile, int lines) {
    return Operand{of.first + tile * third_bytes(lines), of.third + tile * third_bytes(lines) / 2};  // two bytes each
}

template <int At>
__device__ inline void load_block(__amdgpu_buffer_rsrc_t first, __amdgpu_buffer_rsrc_t third, uint32_t off, uint32_t lds) {
    halves::Tile::load_one<At>(first, off, 0, lds);
    halves::Tile::load_one<At + kPart>(first, off, kPart, lds);
    halves::Tile::load_one<At + 2 * kPart>(third, off, 0, lds);
}

// tile += the products of lines [begin, end) of a tile of either operand. lds: kLds bytes. Two slices are on their way while one
// is multiplied: a slice takes about 3000 cycles, as one of the halves' does.
__device__ inline void accumulate(halves::Tile& tile, const Operand& a, const Operand& b, int begin, int end, char* lds) {
    if (end <= begin) return;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const uint32_t off = 1024u * uint32_t(wave) + 16u * uint32_t(lane);
    const uint32_t to =
        __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>((halves::lds_ptr_t)lds)) + 1024u * uint32_t(wave));
    const int first = 2 * begin, last = 2 * end - 1;
    const auto from = [](halves::half* parts, int64_t s, int bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(parts) + s * bytes, short(0), bytes, 0x00020000);
    };
    constexpr int kOperand = kParts * kPart;  // bytes in a stage
    const auto request = [&](int s, int stage) {
        const uint32_t dst = to + uint32_t(stage) * (2 * kOperand);
        load_block<0>(from(a.first, s, 2 * kPart), from(a.third, s, kPart), off, dst);
        load_block<kOperand>(from(b.first, s, 2 * kPart), from(b.third, s, kPart), off, dst);
    };
    const int at_a = lane / 32 * (kTile * 16) + (128 * (wave / 4) + lane % 32) * 16;
    const int at_b = kOperand + lane / 32 * (kTile * 16) + (64 * (wave % 4) + lane % 32) * 16;
    constexpr int kA[6] = {0, 2, 1, 0, 1, 0}, kB[6] = {2, 0, 1, 1, 0, 0};  // the small products first
    const auto multiply = [&](int stage) {
        const char* const at = lds + stage * (2 * kOperand);
        b8 y[2][kParts];
#pragma unroll
        for (int q = 0; q < kParts; ++q)
#pragma unroll
            for (int j = 0; j < 2; ++j) y[j][q] = *reinterpret_cast<const b8*>(at + at_b + (2 * q * kTile + 32 * j) * 16);
#pragma unroll
        for (int h = 0; h < 4; h += 2) {
            b8 x[2][kParts];
#pragma unroll
            for (int q = 0; q < kParts; ++q)
#pragma unroll
                for (int i = 0; i < 2; ++i) x[i][q] = *reinterpret_cast<const b8*>(at + at_a + (2 * q * kTile + 32 * (h + i)) * 16);
#pragma unroll
            for (int p = 0; p < 6; ++p)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        tile.acc[h + i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[i][kA[p]], y[j][kB[p]], tile.acc[h + i][j], 0, 0, 0);
        }
    };
    request(first, 0);
    request(min(first + 1, last), 1);
    int stage = 0;
    for (int s = first; s <= last; ++s) {
        halves::wait_loads<6>();  // all but the next slice's
        __syncthreads();          // slice s is there, and slice s - 1 has been read
        request(min(s + 2, last), stage == 0 ? 2 : stage - 1);
        multiply(stage);
        stage = stage == 2 ? 0 : stage + 1;
    }
    halves::wait_loads<0>();  // no load may land in LDS that others use by then
}

}  // namespace thirds
}  // namespace vchip
