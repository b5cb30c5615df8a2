// Matrix products of float32 operands on the 16-bit matrix instructions, at
// float32's precision.
//
// Every value is written as a sum of three bfloat16 numbers, x = x1 + x2 + x3,
// each the rounding of what the earlier ones leave: |x2| <= 2^-9 |x|, |x3| <=
// 2^-18 |x|, and the parts' 24 bits hold all of x. Of the nine products of two
// values' parts those below 2^-26 of the largest (x2 y3, x3 y2, x3 y3) are left
// out. bfloat16 has float32's exponents, so values of 2^-110 (8e-34) or more may
// meet any others; its least step is 2^-133, by half of which a smaller value may
// be off (2^-120 by 2^-14 of itself), which shows where it meets one above 2^80.
// The six
// others are exact and summed in float32 by the matrix instructions, whose
// 16-deep sums round less often than a float32 chain does: six instructions of
// 32 cycles take the place of eight of 64 (V_MFMA_F32_32X32X2_F32).
//
// A workgroup of four waves computes a BM x BN tile of C, each wave a quarter
// of it in 32 x 32 blocks, k in slices of 32. A thread loads its share of a
// slice into registers while the slice before it is multiplied, splits it, and
// stores the parts in LDS as the matrix instructions read them: [part][k / 8]
// [row][8], so a fragment is one 16-byte read per lane and a transposed operand
// costs nothing more than a k-contiguous one.
#pragma once

#include "reduce_common.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vchip {
namespace split {

constexpr int kThreads = 256, kSliceK = 32, kGroups = kSliceK / 8;

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f2v __attribute__((ext_vector_type(2)));

struct Bf16x3 {
    static constexpr int kParts = 3, kProducts = 6;
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    // Parts of A and B of each product, the smallest products first.
    static constexpr int kA[6] = {0, 2, 1, 0, 1, 0}, kB[6] = {2, 0, 1, 1, 0, 0};
    static __device__ inline f16v multiply(v8 a, v8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
// The parts of eight values, packed.
template <class S>
__device__ inline void split8(const float (&v)[8], typename S::v8 (&out)[S::kParts]) {
    f2v rest[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rest[i] = f2v{v[2 * i], v[2 * i + 1]};
#pragma unroll
    for (int p = 0; p < S::kParts; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const typename S::v2 part = __builtin_convertvector(rest[i], typename S::v2);
            out[p][2 * i] = part[0];
            out[p][2 * i + 1] = part[1];
            if (p + 1 < S::kParts) {
                rest[i][0] -= float(part[0]);
                rest[i][1] -= float(part[1]);
            }
        }
    }
}

// The LDS image of Rows rows of an operand's slice. A k-group's rows are two
// 16-byte slots longer than they need to be: eight threads that store the four
// groups of two rows then meet different banks.
template <class S, int Rows>
struct Slice {
    static constexpr int kStride = Rows + 2;
    typename S::v8 at[S::kParts][kGroups][kStride];
};

// ---- operands: what one thread loads of a slice, and where it stores it -----------

// k contiguous: element (row, k) at pointer(row)[k]. Thread t holds k-group
// t % 4 of rows t / 4 + 64 j, so four threads read 128 contiguous bytes.
template <int Rows>
struct AlongK {
    static constexpr int kChunks = Rows / 64;
    float v[kChunks][8];

    // p: the chunks' rows at k = 0. A row past the operand's end may be any
    // row of it: what it gives is never stored.
    __device__ inline void load(const float* const (&p)[kChunks], int64_t k0) {
        const int64_t k = k0 + 8 * (threadIdx.x % kGroups);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const f4u lo = *reinterpret_cast<const f4u*>(p[j] + k), hi = *reinterpret_cast<const f4u*>(p[j] + k + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[j][i] = lo[i];
                v[j][4 + i] = hi[i];
            }
        }
    }
    // Zeros for the slice's first `n` k.
    __device__ inline void drop(int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool stays = 8 * int(threadIdx.x % kGroups) + i >= n;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) v[j][i] = stays ? v[j][i] : 0.0f;
        }
    }
    // A slice of which k < depth are there.
    __device__ inline void load_rest(const float* const (&p)[kChunks], int64_t k0, int64_t depth) {
        const int64_t k = k0 + 8 * (threadIdx.x % kGroups);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = k + i < depth ? p[j][k + i] : 0.0f;
    }
    template <class S>
    __device__ inline void store(Slice<S, Rows>& lds) const {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            typename S::v8 parts[S::kParts];
            split8<S>(v[j], parts);
#pragma unroll
            for (int q = 0; q < S::kParts; ++q) lds.at[q][threadIdx.x % kGroups][threadIdx.x / kGroups + 64 * j] = parts[q];
        }
    }
    static __device__ inline int row(int j) { return threadIdx.x / kGroups + 64 * j; }
};

// Rows contiguous: element (row, k) at line(k)[row]. Wave w holds k-group w,
// lane l rows l + 64 j: a wave reads 256 contiguous bytes of each k, whatever
// the rows' alignment, and stores to neighbouring slots.
template <int Rows>
struct AcrossK {
    static constexpr int kChunks = Rows / 64;
    float v[kChunks][8];

    // line(k): the line of k < depth, uniform in the wave. at: the chunks' places in a line; a row past the operand's
    // end may be any place of it: what it gives is never stored.
    template <class Line>
    __device__ inline void load(const unsigned (&at)[kChunks], int64_t k0, Line&& line) {
        const int64_t k = k0 + 8 * __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto from = line(k + i);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) v[j][i] = from(j)[at[j]];
        }
    }
    __device__ inline void drop(int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool stays = 8 * int(threadIdx.x / 64) + i >= n;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) v[j][i] = stays ? v[j][i] : 0.0f;
        }
    }
    template <class Line>
    __device__ inline void load_rest(const unsigned (&at)[kChunks], int64_t k0, int64_t depth, Line&& line) {
        const int64_t k = k0 + 8 * __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool inside = k + i < depth;
            const auto from = line(inside ? k + i : 0);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) v[j][i] = inside ? from(j)[at[j]] : 0.0f;
        }
    }
    template <class S>
    __device__ inline void store(Slice<S, Rows>& lds) const {
        const int group = threadIdx.x / 64, lane = threadIdx.x % 64;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            typename S::v8 parts[S::kParts];
            split8<S>(v[j], parts);
#pragma unroll
            for (int q = 0; q < S::kParts; ++q) lds.at[q][group][lane + 64 * j] = parts[q];
        }
    }
    static __device__ inline int row(int j) { return threadIdx.x % 64 + 64 * j; }
};

// Is a sum of products lost to an infinity, a NaN or a value that rounds to an
// infinity in 16 bits? Its parts give NaN or an infinity then.
__device__ inline bool finite(float x) { return fabsf(x) < __builtin_huge_valf(); }

// ---- the tile -----------------------------------------------------------------------

// Wave w computes rows BM / 2 (w / 2) .. and, of every 64 columns, the half w % 2.
template <class S, int BM, int BN>
struct Tile {
    static constexpr int kM = BM / 64, kN = BN / 64;  // 32 x 32 blocks of a wave
    static constexpr int kValues = 16 * kM * kN;      // of a thread
    f16v acc[kM][kN];

    __device__ inline void clear() {
#pragma unroll
        for (int a = 0; a < kM; ++a)
#pragma unroll
            for (int b = 0; b < kN; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
    }

    // k-groups k and k + 1 of a slice.
    __device__ inline void multiply(const Slice<S, BM>& as, const Slice<S, BN>& bs, int k) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        const int m0 = wave / 2 * (BM / 2) + lane % 32, n0 = wave % 2 * 32 + lane % 32;
        {
            typename S::v8 a[kM][S::kParts];
#pragma unroll
            for (int q = 0; q < S::kParts; ++q)
#pragma unroll
                for (int i = 0; i < kM; ++i) a[i][q] = as.at[q][k + lane / 32][m0 + 32 * i];
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                typename S::v8 b[S::kParts];
#pragma unroll
                for (int q = 0; q < S::kParts; ++q) b[q] = bs.at[q][k + lane / 32][n0 + 64 * j];
#pragma unroll
                for (int p = 0; p < S::kProducts; ++p)
#pragma unroll
                    for (int i = 0; i < kM; ++i) acc[i][j] = S::multiply(a[i][S::kA[p]], b[S::kB[p]], acc[i][j]);
            }
        }
    }

    // Is one of this thread's values not finite? See finite().
    __device__ inline bool lost() const {
        bool any = false;
#pragma unroll
        for (int a = 0; a < kM; ++a)
#pragma unroll
            for (int b = 0; b < kN; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) any |= !finite(acc[a][b][i]);
        return any;
    }

    // f(row, column, value) for each value this thread holds; f may change it.
    template <class F>
    __device__ inline void each(F&& f) {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
#pragma unroll
        for (int a = 0; a < kM; ++a)
#pragma unroll
            for (int b = 0; b < kN; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float v = acc[a][b][i];
                    f(wave / 2 * (BM / 2) + 32 * a + 8 * (i / 4) + 4 * (lane / 32) + i % 4, wave % 2 * 32 + 64 * b + lane % 32, v);
                    acc[a][b][i] = v;
                }
    }
};

// The products of k in [begin, end) onto a tile. load(a, b, k) reads the slice
// from k, rest(a, b, k) the last one, of which end - k are there. Ahead register
// sets hold slices that are on their way: one where other workgroups of the CU
// hide the wait, more for grids that leave a CU one or two.
//
// With one, the last slice ends at `end`, whatever the sum's length, so that it is
// read like the others, and what it shares with the slice before it is dropped (a
// training pass of 49152 rows of 64 experts, 1024 x 512, each with some other count:
// 3388 us, 3444 with a last slice read value by value). With more this
// gained nothing (2100 rows of 20 experts, 90 x 150: 105 and 100 us).
template <int Ahead, class A, class B, class T, class SA, class SB, class Load, class Rest>
__device__ inline void accumulate(T& tile, SA& as, SB& bs, int64_t begin, int64_t end, Load&& load, Rest&& rest) {
    A a[Ahead];
    B b[Ahead];
    if (end <= begin) return;
    const auto multiply = [&](const A& x, const B& y, auto&& next) {
        x.store(as);
        y.store(bs);
        __syncthreads();
        next();
        tile.multiply(as, bs, 0);
        tile.multiply(as, bs, 2);
        __syncthreads();
    };
    if constexpr (Ahead == 1) {
        const bool less = end < kSliceK;  // begin is a multiple of a slice
        const int slices = int((end - begin + kSliceK - 1) / kSliceK);
        const int shared = less ? 0 : int(begin + int64_t(slices) * kSliceK - end);
        const auto at = [&](int s) { return min(begin + int64_t(s) * kSliceK, end - kSliceK); };
        if (less) rest(a[0], b[0], begin);
        else load(a[0], b[0], at(0));
        for (int s = 0; s < slices; ++s) {
            if (s + 1 == slices && shared) {
                a[0].drop(shared);
                b[0].drop(shared);
            }
            multiply(a[0], b[0], [&] {
                if (s + 1 < slices) load(a[0], b[0], at(s + 1));
            });
        }
    } else {
        const int full = int((end - begin) / kSliceK);
        // Always the same number of loads on their way (past the end the last slice is read again), so that the compiler
        // waits for just those it needs.
        const auto at = [&](int s) { return begin + int64_t(min(s, full - 1)) * kSliceK; };
        if (full > 0) {
#pragma unroll
            for (int i = 0; i < Ahead; ++i) load(a[i], b[i], at(i));
        }
        for (int s = 0; s < full; s += Ahead) {
#pragma unroll
            for (int i = 0; i < Ahead; ++i) {
                if (s + i >= full) break;
                multiply(a[i], b[i], [&] { load(a[i], b[i], at(s + i + Ahead)); });
            }
        }
        if (begin + int64_t(full) * kSliceK < end) {
            rest(a[0], b[0], begin + int64_t(full) * kSliceK);
            multiply(a[0], b[0], [] {});
        }
    }
}

// One of `parts` workgroups that each hold a part of a tile's sums: false for
// all but the one that counts in last on `done` (zero before and after), which
// adds the parts in their order. partial: of this tile, parts * kValues values
// of every thread.
template <class T>
__device__ inline bool join(T& tile, int part, int parts, float* partial, unsigned* done, bool& last) {
    float* const mine = partial + threadIdx.x;
    int at = 0;
    tile.each([&](int, int, float& v) {
        __hip_atomic_store(&mine[(part * T::kValues + at++) * kThreads], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    });
    red::wait_stores_visible();
    __syncthreads();
    if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == unsigned(parts);
        if (last) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return false;
    tile.clear();
    for (int q = 0; q < parts; ++q) {
        at = 0;
        tile.each([&](int, int, float& v) {
            v += __hip_atomic_load(&mine[(q * T::kValues + at++) * kThreads], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        });
    }
    return true;
}

}  // namespace split
}  // namespace vchip
