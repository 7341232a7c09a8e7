// int8_gemm.hip -- the launches of the 8-bit product, for the C ABI in include/ridge_int8.h.

#include "int8_gemm.hpp"
#include "int8_launch.hpp"
#include "ridge_int8.h"

#include <hip/hip_runtime.h>

namespace {

using ridge::Int8Operands;
using ridge::Int8Sizes;

// How a product runs, by number: tiles of C as one workgroup each, or (kFew) small ones
// whose K a workgroup's waves share.
using ridge::Tile128x128;
using ridge::Tile256x128;
using ridge::Tile256x256;
using Pair128x128 = ridge::Int8Traits<128, 128, 128, 32, 64, 2>;   // two workgroups a CU
using Tile64x128 = ridge::Int8Traits<64, 128, 128, 32, 32, 3>;
using Tile64x64 = ridge::Int8Traits<64, 64, 128, 16, 32, 4>;
using Few16x16 = ridge::Int8FewTraits<1, 1, 8, 2>;
using Few32x16 = ridge::Int8FewTraits<2, 1, 8, 2>;
using Few32x32 = ridge::Int8FewTraits<2, 2, 8, 2>;

constexpr int kCUs = ridge::kInt8CUs;
constexpr int kForms = 9, kFirstFew = 6;
struct FormCost {
    int rows, cols;
    int call, tile, perK;   // 10 ns: c, a and 1000 b of the time c + n (a + b K)
};
// With n the tiles of the busiest CU, the time of a launch is about c + n (a + b K): within 8
// to 14% by form (one standard deviation, the larger forms up to 13% too long on average) of
// 620 products of 1 to 8192 rows, 74 to 16384 columns and K of 75 to 16384, of whole and odd
// sizes, each timed in every form. By it the choice was 0.6% slower on average than the
// fastest form timed, 16% in the worst case (2216 x 4158 x 256). For 16 x 16 tiles b = 0.43
// instead of 0.31 changes 42 of those choices, 31 of them for the worse, by 4% on average (2 x
// 8576 x 2520 7.3 us instead of 5.6), though some gain (8 x 12288 x 4096 9.6 instead of 10.2).
// 256 x 256 tiles count their last round by its parts (int8Rounds). What the forms are for,
// us 256x256 | 256x128 | 128x128 | its pair | 64x128 | 64x64 | few 16x16 | 32x16 | 32x32:
//   4096 x 4096 x 4096   52.3 | 58.8 | 75.0 | 61.9 | 80.8 | 98.3 | - | - | -
//   2319 x 1792 x 6784   64.1 | 33.8 | 49.1 | 37.8 | 45.6 | 48.8 | - | - | -
//   2048 x 2048 x 2048   25.2 | 16.0 | 11.6 | 13.6 | 13.0 | 15.6 | 86 | 93 | 59
//   3873 x 4263 x 175    21.5 | 21.8 | 23.6 | 17.2 | 21.5 | 29.6 | - | - | -
//   149 x 8886 x 6784    64.0 | 30.7 | 23.9 | 32.2 | 18.0 | 20.5 | 54 | 54 | 38
//   48 x 8192 x 4096     39.9 | 20.1 | 15.7 | 20.6 | 12.0 | 8.3 | 13.3 | 15.9 | 11.2
//   1 x 4096 x 4096      39.7 | 19.9 | 15.6 | 20.1 | 11.3 | 7.5 | 5.0 | 5.2 | 5.6
//   300 x 300 x 8192     75.1 | 38.2 | 27.3 | 38.0 | 19.6 | 12.9 | 8.7 | 7.1 | 8.5
//   792 x 256 x 3468     45.7 | 28.3 | 18.8 | 23.3 | 15.0 | 11.1 | 9.6 | 9.6 | 7.9
constexpr FormCost kForm[kForms] = {
    {256, 256, 0, 750, 856},  {256, 128, 0, 680, 455}, {128, 128, 50, 400, 327},
    {128, 128, 190, 220, 372}, {64, 128, 200, 150, 223}, {64, 64, 210, 120, 136},
    {16, 16, 170, 70, 31},    {32, 16, 100, 170, 52},  {32, 32, 80, 200, 73},
};

// A grid's work-items fit 32 bits, its tiles the kernels' divisions, and neither gains more
// than a round by parts.
constexpr int64_t kMostTiles = (1 << 23) - 1024;

int64_t tilesOf(int form, int64_t M, int64_t N) {
    const FormCost& f = kForm[form];
    return ((M + f.rows - 1) / f.rows) * ((N + f.cols - 1) / f.cols);
}

int chooseForm(const Int8Sizes& z, bool packed) {
    int best = 0;
    int64_t least = INT64_MAX;
    // Small tiles of all sizes take the arguments of small ones only.
    for (int i = 0; i < (packed ? kForms : kFirstFew); ++i) {
        const FormCost& f = kForm[i];
        const int64_t tiles = tilesOf(i, z.M, z.N);
        if (i > 0 && tiles >= kMostTiles) continue;
        auto rounds = [&](const FormCost& of, int64_t n) { return n * (of.tile + (int64_t)of.perK * z.K / 1000); };
        int64_t cost = f.call + rounds(f, (tiles + kCUs - 1) / kCUs);
        if (i == 0 && tiles < kMostTiles) {
            const ridge::Int8Rounds r = ridge::int8Rounds((int)tiles);
            if (r.parts > 1) cost = rounds(f, r.whole / kCUs) + rounds(kForm[r.parts == 2 ? 1 : 2], 1);
        }
        if (cost < least) best = i, least = cost;
    }
    return best;
}

// A C of more than this whose rows are whole cache lines is stored past the caches: it would
// push the operands out of them. us, cached | past the caches, forms 0, 1 and 3: 8192 x
// 8192 x 128 51.3 | 45.3, 52.2 | 42.0, 47.1 | 39.3; x 1024 91.1 | 84.0, 115.9 | 88.5, 111.0 |
// 88.6; x 8192 424 | 420. Lines that two tiles share lose by it (8192 x 8191 x 512 66.8 |
// 78.8), and so does a smaller C (4096 x 8192 x 1024 40.7 | 44.2).
constexpr int64_t kStreamBytes = (int64_t)64 << 20;

template <typename Out>
bool streams(const Int8Operands& p, const Int8Sizes& z) {
    return (int64_t)z.M * z.N * (int64_t)sizeof(Out) > kStreamBytes && z.ldc * (int64_t)sizeof(Out) % 128 == 0 &&
           (uintptr_t)p.C % 128 == 0;
}

template <typename T, typename Out, bool PINGPONG, bool PACKED, bool STREAM = false>
hipError_t launchTiles(const Int8Operands& p, const Int8Sizes& z, int64_t tiles, hipStream_t stream) {
    return ridge::launchKernel(ridge::int8GemmKernel<T, Out, PINGPONG, PACKED, STREAM>, (unsigned)tiles, T::kThreads,
                               stream, ridge::int8Args<PACKED>(p, z));
}

template <typename Out, bool PACKED, bool STREAM>
hipError_t launchRounds(const Int8Operands& p, const Int8Sizes& z, int64_t tiles, hipStream_t stream) {
    return ridge::launchKernel(ridge::int8RoundsKernel<Out, PACKED, STREAM>,
                               (unsigned)ridge::int8Rounds((int)tiles).blocks, Tile256x256::kThreads, stream,
                               ridge::int8Args<PACKED>(p, z));
}

template <typename T, typename Out>
hipError_t launchFew(const Int8Operands& p, const Int8Sizes& z, int64_t tiles, hipStream_t stream) {
    return ridge::launchKernel(ridge::int8FewKernel<T, Out>, (unsigned)tiles, T::kThreads, stream,
                               ridge::int8Args<true>(p, z));
}

template <typename Out, bool PACKED>
hipError_t launchForm(int form, const Int8Operands& p, const Int8Sizes& z, hipStream_t s) {
    const int64_t tiles = tilesOf(form, z.M, z.N);
    if (tiles >= kMostTiles) return hipErrorInvalidValue;
    if (streams<Out>(p, z)) {   // the other forms hardly ever have a C of that size
        switch (form) {
            case 0: return launchRounds<Out, PACKED, true>(p, z, tiles, s);
            case 1: return launchTiles<Tile256x128, Out, true, PACKED, true>(p, z, tiles, s);
            case 3: return launchTiles<Pair128x128, Out, false, PACKED, true>(p, z, tiles, s);
        }
    }
    switch (form) {
        case 0: return launchRounds<Out, PACKED, false>(p, z, tiles, s);
        case 1: return launchTiles<Tile256x128, Out, true, PACKED>(p, z, tiles, s);
        case 2: return launchTiles<Tile128x128, Out, false, PACKED>(p, z, tiles, s);
        case 3: return launchTiles<Pair128x128, Out, false, PACKED>(p, z, tiles, s);
        case 4: return launchTiles<Tile64x128, Out, false, PACKED>(p, z, tiles, s);
        case 5: return launchTiles<Tile64x64, Out, false, PACKED>(p, z, tiles, s);
    }
    if constexpr (PACKED) {
        switch (form) {
            case 6: return launchFew<Few16x16, Out>(p, z, tiles, s);
            case 7: return launchFew<Few32x16, Out>(p, z, tiles, s);
            case 8: return launchFew<Few32x32, Out>(p, z, tiles, s);
        }
    }
    return hipErrorInvalidValue;
}

template <typename Out>
hipError_t launchGemm(const Int8Operands& p, const Int8Sizes& z, hipStream_t stream) {
    const bool packed = ridge::int8ArgsFit(z);
    const int form = chooseForm(z, packed);
    return packed ? launchForm<Out, true>(form, p, z, stream) : launchForm<Out, false>(form, p, z, stream);
}

constexpr int64_t kMostRows = INT32_MAX - 255;   // whole tiles of them still fit 31 bits

bool aligned(const void* p, size_t to) { return p != nullptr && ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

extern "C" int64_t ridge_int8_row_stride(int64_t cols) {
    const int64_t to = cols > 512 ? 128 : 16;
    return (cols + to - 1) / to * to;
}

extern "C" int ridge_int8_gemm(const int8_t* A, int64_t lda, const float* scaleA, const int8_t* B, int64_t ldb,
                               const float* scaleB, const void* bias, void* C, int64_t ldc, int type, int64_t M,
                               int64_t N, int64_t K, void* stream) {
    if (type != RIDGE_F16 && type != RIDGE_BF16 && type != RIDGE_F32) return hipErrorInvalidValue;
    if (M < 0 || N < 0 || K < 1 || K > RIDGE_INT8_MAX_K) return hipErrorInvalidValue;
    if (M == 0 || N == 0) return hipSuccess;
    const size_t size = type == RIDGE_F32 ? 4 : 2;
    if (M > kMostRows || N > kMostRows || lda < K || ldb < K || lda % 16 || ldb % 16 || lda >= (1 << 23) ||
        ldb >= (1 << 23) || ldc < N || !aligned(A, 16) || !aligned(B, 16) || !aligned(scaleA, 4) ||
        !aligned(scaleB, 4) || !aligned(C, size) || ((uintptr_t)bias & (size - 1)))
        return hipErrorInvalidValue;
    const Int8Operands p = {A, B, scaleA, scaleB, bias, C};
    const Int8Sizes z = {(int)M, (int)N, (int)K, (int)lda, (int)ldb, ldc};
    switch (type) {
        case RIDGE_F16: return launchGemm<_Float16>(p, z, (hipStream_t)stream);
        case RIDGE_BF16: return launchGemm<__bf16>(p, z, (hipStream_t)stream);
        default: return launchGemm<float>(p, z, (hipStream_t)stream);
    }
}

extern "C" int ridge_int8_gemm_form(int64_t M, int64_t N, int64_t K) {
    if (M < 1 || N < 1 || K < 1 || M > kMostRows || N > kMostRows || K > RIDGE_INT8_MAX_K) return -1;
    const int ld = (int)ridge_int8_row_stride(K);
    const Int8Sizes z = {(int)M, (int)N, (int)K, ld, ld, N};
    const int form = chooseForm(z, ridge::int8ArgsFit(z));
    return tilesOf(form, M, N) < kMostTiles ? form : -1;
}
