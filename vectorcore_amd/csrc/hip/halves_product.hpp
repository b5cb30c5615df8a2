// Products C = A B^T of float32 values on the half-precision matrix instructions,
// for operands that are used whole and once: each is packed into memory first.
//
// A value is scaled by a power of two of its row and split, x 2^e = x1 + x2, with
// half-precision parts. e brings the row's largest magnitude to 2^13 .. 2^14, so a
// value keeps 22 bits or an error of 2^-38 of the largest, whichever is more. Of
// the four products of two values' parts x2 y2 (2^-22 of the largest) is left out.
// Three instructions of 32 cycles take the place of eight of 64 of the float32
// matrix instruction. For operands whose rows hold values that are finite and not
// too unlike each other; for others thirds_product.hpp.
//
// 32 neighbouring values of a row are one 128-byte line, their first parts, then
// their second ones: four threads that hold eight values each then write 64
// neighbouring bytes at a time. Rows are padded to 256 and lines to whole ones with
// zeros, so the loads of a tile need no check and go straight to LDS.
//
// Bound by the matrix instructions and the card's power: 7373 x 1024 by 50000 long
// sums takes 1.83 ms (413 TFLOP/s of float32 products, 1239 of half-precision
// ones, where the library's large half-precision product reaches 1286). There the
// instructions are busy for 68% of the cycles at a clock of 1.73 GHz of 2.4, so
// fewer stalls give a lower clock: 256 x 128 tiles with two workgroups a CU took
// 11% more time, four waves of 128 x 128 34%, four stages of half a slice, and
// fragments read ahead over the barrier, the same.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vchip {
namespace halves {

constexpr int kThreads = 512, kTile = 256, kSlice = 32, kLineBytes = 128;

typedef _Float16 half;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// The exponent that brings a largest magnitude, as a float's bits, to 2^13 .. 2^14.
__device__ inline int exponent_of(uint32_t bits) {
    return bits == 0 ? 0 : 14 - __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, bits));
}

// The chunks of eight values along k, scaled by 2^e.
__device__ inline void split8(const float (&v)[8], int e, h8& first, h8& second) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = __builtin_amdgcn_ldexpf(v[i], e);
        first[i] = half(x);
        second[i] = half(x - float(first[i]));
    }
}

// s_waitcnt that leaves `loads` vector memory operations in flight.
template <int Loads>
__device__ inline void wait_loads() {
    __builtin_amdgcn_s_waitcnt((Loads & 15) | (Loads >> 4) << 14 | 0x0F70);
}

// A tile of 256 x 256 by eight waves, wave w rows 128 (w / 4) .. and columns 64 (w % 4) .. in 32 x 32 blocks. Two waves a SIMD
// and one workgroup a CU: a 16-deep step of a wave reads 12 KiB of LDS for 24 instructions, and a slice of 32 k (64 KiB of
// loads) takes about 3000 cycles, which covers the loads of the next.
struct Tile {
    static constexpr int kStage = 2 * kTile * kLineBytes, kLds = 2 * kStage, kValues = 128;
    f16v acc[4][2];

    __device__ inline void clear() {
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
    }

    // One load: 64 chunks of 16 bytes, lane l's to byte 16 l of the wave's part of the stage. Inline assembly, as the compiler
    // would wait for every load in flight before LDS reads that it cannot tell apart; what a stage's loads have written is
    // waited for before the barrier that hands it on.
    template <int At>
    static __device__ inline void load_one(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t uniform, uint32_t lds) {
        asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :
                     : "s"(lds), "v"(off), "s"(rs), "s"(uniform), "i"(At)
                     : "memory", "m0", "scc");
    }
    template <int At>
    static __device__ inline void load_rows(const half* from, uint32_t off, uint32_t step, uint32_t lds) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<half*>(from), short(0), 0x7FFFFFFE, 0x00020000);
        load_one<At>(rs, off, 0, lds);
        load_one<At + 8192>(rs, off, step, lds);
        load_one<At + 16384>(rs, off, 2 * step, lds);
        load_one<At + 24576>(rs, off, 3 * step, lds);
    }

    // acc += the products of lines [begin, end) of 256 rows of each operand; a, b: their first rows; lines: of a row, at
    // most 2^16 (a load's offset has 31 bits). lds: kLds bytes. Row r's chunk c lies in slot c ^ (r / 2 % 8) of its 128 bytes:
    // the rows of a fragment then meet different banks.
    // Run lines at a time (0: all), from a multiple of that many, before(s) and after(s) around those from s.
    template <int Run, class Before, class After>
    __device__ inline void accumulate(const half* a, const half* b, int lines, int begin, int end, char* lds, Before&& before, After&& after) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        const uint32_t row_bytes = uint32_t(lines) * kLineBytes;
        const uint32_t off = uint32_t(8 * wave + lane / 8) * row_bytes + uint32_t((lane % 8) ^ (4 * (wave % 2) + lane / 16)) * 16u;
        const uint32_t to = __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)lds)) + 1024u * uint32_t(wave));
        const auto request = [&](int s, int stage) {
            const int64_t at = int64_t(s) * (kLineBytes / 2);
            const uint32_t dst = to + uint32_t(stage) * kStage;
            load_rows<0>(a + at, off, 64u * row_bytes, dst);
            load_rows<kTile * kLineBytes>(b + at, off, 64u * row_bytes, dst);
        };
        const int row_a = 128 * (wave / 4) + lane % 32, row_b = kTile + 64 * (wave % 4) + lane % 32;
        const int half_wave = lane / 32, swizzle = lane / 2 % 8;
        const auto multiply = [&](int stage) {
            const char* const from = lds + stage * kStage;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                h8 x[4][2], y[2][2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int slot = ((4 * q + 2 * t + half_wave) ^ swizzle) * 16;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i][q] = *reinterpret_cast<const h8*>(from + (row_a + 32 * i) * kLineBytes + slot);
#pragma unroll
                    for (int j = 0; j < 2; ++j) y[j][q] = *reinterpret_cast<const h8*>(from + (row_b + 32 * j) * kLineBytes + slot);
                }
#pragma unroll
                for (int p = 0; p < 3; ++p)  // the small products first
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i][p == 1], y[j][p == 0], acc[i][j], 0, 0, 0);
            }
        };
        if (end <= begin) return;
        request(begin, 0);
        int stage = 0;
        const auto slice = [&](int s) {
            wait_loads<0>();
            __syncthreads();  // slice s is there, and slice s - 1 has been read
            request(min(s + 1, end - 1), stage ^ 1);
            multiply(stage);
            stage ^= 1;
        };
        if constexpr (Run == 0) {
            for (int s = begin; s < end; ++s) slice(s);
        } else {
            for (int first = begin; first < end; first += Run) {
                const int last = min(end, first + Run);
                before(first);
                for (int s = first; s < last; ++s) slice(s);
                after(first);
            }
        }
        wait_loads<0>();  // no load may land in LDS that others use by then
    }

    // f(row, column, v) for the four values of neighbouring rows of a column; f may change them.
    template <class F>
    __device__ inline void each4(F&& f) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    asm volatile("" ::: "memory");  // addresses and loads of one group at a time: all do not fit the registers
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = acc[a][b][4 * g + i];
                    f(128 * (wave / 4) + 32 * a + 8 * g + 4 * (lane / 32), 64 * (wave % 4) + 32 * b + lane % 32, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[a][b][4 * g + i] = v[i];
                }
    }

    // Of a tile whose sums are split: this part's, kValues values of every thread.
    __device__ inline void store_part(float* partial) const {
        float* to = partial + threadIdx.x;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                asm volatile("" : "+v"(to)::"memory");
#pragma unroll
                for (int i = 0; i < 16; ++i) to[i * kThreads] = acc[a][b][i];
                to += 16 * kThreads;
            }
    }
    // The sum of all parts, in their order, of a thread's values in column block b; four parts' loads of 16 values in flight.
    static __device__ inline void load_parts(const float* partial, int parts, int thread, int b, f16v (&sum)[4][1]) {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const float* from = partial + (2 * a + b) * 16 * kThreads + thread;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[a][0][i] = 0.0f;
            for (int p = 0; p < parts; p += 4) {
                float v[4][16];
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        v[q][i] = p + q < parts ? from[(int64_t(p + q) * kValues + i) * kThreads] : 0.0f;
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[a][0][i] += v[q][i];
            }
        }
    }
    // The same for four values alone: group q of 32 of a thread, f(row, column, v).
    template <class F>
    static __device__ inline void each_part(const float* partial, int parts, int q, F&& f) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int p = 0; p < parts; p += 4) {
            float w[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[u][i] = p + u < parts ? partial[(int64_t(p + u) * kValues + 4 * q + i) * kThreads + threadIdx.x] : 0.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += w[u][i];
        }
        const int block = q / 4, g = q % 4;
        f(128 * (wave / 4) + 32 * (block / 2) + 8 * g + 4 * (lane / 32), 64 * (wave % 4) + 32 * (block % 2) + lane % 32, v);
    }
};

// The tiles of a product: `whole` workgroups compute one each, the others' sums are split over `parts` each, so that the last
// round of workgroups fills the CUs. Where that gains: a line takes 2.5 us, and a part is written and read again in 0.1 us of all
// CUs' time, by a launch of 5 us. (120 tiles of 29 lines: 83 us, 44 in halves and 18 to join them.)
constexpr int kLeastSplit = 24;  // lines
struct Tiles {
    int down, across;  // tiles of A's and of B's rows
    int whole, rest, parts;
};
__device__ inline Tiles tiles_of(int64_t rows_a, int64_t rows_b, int lines, int places) {
    Tiles t{int((rows_a + kTile - 1) / kTile), int((rows_b + kTile - 1) / kTile), 0, 0, 1};
    const int all = t.down * t.across, rest = all % places;
    if (rest && lines >= kLeastSplit) {
        const int parts = min(places / rest, lines / 8);
        if (50 * int64_t(lines) * (parts - 1) > parts * (100 + 2 * int64_t(rest) * parts)) {  // in twentieths of 1 us
            t.rest = rest;
            t.parts = parts;
        }
    }
    t.whole = all - t.rest;
    return t;
}
// At least as many workgroups as tiles_of asks for, of these rows or fewer.
inline int64_t most_blocks(int64_t rows_a, int64_t rows_b, int64_t places) {
    const int64_t all = ((rows_a + kTile - 1) / kTile) * ((rows_b + kTile - 1) / kTile);
    return (all + places - 1) / places * places;
}

// Which tile a workgroup computes. Neighbouring workgroups go to the eight XCDs in turn: each XCD takes a run of the order, in
// which eight tiles of A's rows by all of B's follow each other, so what its 32 CUs read at a time is shared in its L2.
struct Place {
    int m, n;
    int rest, part;  // of a split tile: which, and which of its parts; else -1
};
__device__ inline Place tile_at(const Tiles& t, int id) {
    const int run = 8 * t.across, first = id / run * 8, high = min(8, t.down - first), in = id % run;
    return Place{first + in % high, in / high, -1, -1};
}
// block < t.whole + t.rest * t.parts
__device__ inline Place place_of(const Tiles& t, int block) {
    if (block < t.whole) {
        const int each = t.whole / 8, over = t.whole % 8, xcd = block % 8;
        return tile_at(t, xcd * each + min(xcd, over) + block / 8);
    }
    const int rest = (block - t.whole) % t.rest;
    Place p = tile_at(t, t.whole + rest);
    p.rest = rest;
    p.part = (block - t.whole) / t.rest;
    return p;
}

}  // namespace halves
}  // namespace vchip
