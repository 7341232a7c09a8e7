// int8_gemm.hip -- the launches of the 8-bit product, for the C ABI in include/ridge_int8.h.

#include "int8_gemm.hpp"
#include "ridge_int8.h"

#include <hip/hip_runtime.h>

namespace {

using ridge::Int8Args;

constexpr int kCUs = 256;   // of an MI355X

template <typename T, typename Out, bool PINGPONG>
hipError_t launchTiles(Int8Args args, hipStream_t stream) {
    const int64_t tilesM = ridge::int8TilesM<T>(args.M), tilesN = ridge::int8TilesN<T>(args.N);
    if (tilesM * tilesN > (int64_t)UINT32_MAX / T::kThreads) return hipErrorInvalidValue;
    args.order = ridge::tileOrder<T::BM, T::BN, ridge::kInt8GroupM>((int)tilesM * T::BM, (int)tilesN * T::BN);
    ridge::int8GemmKernel<T, Out, PINGPONG><<<dim3((unsigned)(tilesM * tilesN)), dim3(T::kThreads), 0, stream>>>(args);
    return hipGetLastError();
}

template <typename T, typename Out>
hipError_t launchFew(const Int8Args& args, hipStream_t stream) {
    const unsigned blocks = (unsigned)((args.N + 16 * T::TN - 1) / (16 * T::TN));
    ridge::int8FewKernel<T, Out><<<dim3(blocks), dim3(T::kThreads), 0, stream>>>(ridge::fewArgs(args));
    return hipGetLastError();
}

// The tiles, eight wavefronts each, and what a CU takes for one of each with the chip
// full, in 2.5 ns a 64 k (measured at K = 4096).
using Tile256x256 = ridge::Int8Traits<256, 256, 128, 128, 64, 2>;
using Tile256x128 = ridge::Int8Traits<256, 128, 128, 64, 64, 3>;   // ping-pong: 5% faster than uniform
using Tile128x128 = ridge::Int8Traits<128, 128, 128, 32, 64, 3>;
using Tile64x128 = ridge::Int8Traits<64, 128, 128, 32, 32, 3>;
using Tile64x64 = ridge::Int8Traits<64, 64, 128, 16, 32, 4>;
constexpr int kTiles = 5;
constexpr int kTileRows[kTiles] = {256, 256, 128, 64, 64};
constexpr int kTileCols[kTiles] = {256, 128, 128, 128, 64};
constexpr int64_t kTileCost[kTiles] = {470, 280, 175, 107, 73};

// The tile whose grid keeps the busiest CU shortest, the larger one where two are alike. A
// smaller tile moves more operand bytes for its products, a larger one leaves CUs idle on
// a small grid. Measured at K = 4096, us, 256x256 | 256x128 | 128x128 | 64x128 | 64x64:
// 256 x 4096 40 | 22.6 | 17.5 | 12.1 | 9.0; 512 x 4096 40 | 22.9 | 17.8 | 13.2 | 14.5;
// 1024 x 4096 40 | 23.5 | 20.1 | 21.8 | 26.8; 2048 x 4096 43 | 30.9 | 40 | 42 | 51;
// 4096 x 4096 53 | 61 | 77 | 81 | 101.
int chooseTile(int64_t M, int64_t N) {
    int best = 0;
    int64_t least = INT64_MAX;
    for (int t = 0; t < kTiles; ++t) {
        const int64_t tiles = ((M + kTileRows[t] - 1) / kTileRows[t]) * ((N + kTileCols[t] - 1) / kTileCols[t]);
        const int64_t cost = (tiles + kCUs - 1) / kCUs * kTileCost[t];
        if (cost < least) best = t, least = cost;
    }
    return best;
}

template <typename Out>
hipError_t launchGemm(const Int8Args& args, hipStream_t stream) {
    // Few tokens and no more channels than one workgroup of 16 a CU takes: a 64 x 64 tile
    // would leave three CUs in four idle. us, few | 64 x 64 tiles, K = 4096: 1 x 4096 4.9 |
    // 7.4, 20 x 4096 5.7 | 7.6, 64 x 4096 8.3 | 8.2; 64 x 2000 x 8000 11.5 | 16.8; 1 x 1000
    // x 16384 7.1 | 20.5. With twice the channels the tiles are as fast: 16 x 8192 8.2 | 7.8.
    static_assert(ridge::kFewMostN == 16 * kCUs, "a workgroup of 16 channels on each CU");
    if (args.N <= ridge::kFewMostN && args.ldc <= UINT32_MAX) {
        if (args.M <= 16) return launchFew<ridge::Int8FewTraits<1, 1, 16, 2>, Out>(args, stream);
        if (args.M <= 32) return launchFew<ridge::Int8FewTraits<2, 1, 8, 2>, Out>(args, stream);
        if (args.M <= ridge::kFewMostM) return launchFew<ridge::Int8FewTraits<4, 1, 8, 2>, Out>(args, stream);
    }
    switch (chooseTile(args.M, args.N)) {
        case 0: return launchTiles<Tile256x256, Out, false>(args, stream);
        case 1: return launchTiles<Tile256x128, Out, true>(args, stream);
        case 2: return launchTiles<Tile128x128, Out, false>(args, stream);
        case 3: return launchTiles<Tile64x128, Out, false>(args, stream);
        default: return launchTiles<Tile64x64, Out, false>(args, stream);
    }
}

bool aligned(const void* p, size_t to) { return p != nullptr && ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

extern "C" int ridge_int8_gemm(const int8_t* A, int64_t lda, const float* scaleA, const int8_t* B, int64_t ldb,
                               const float* scaleB, const void* bias, void* C, int64_t ldc, int type, int64_t M,
                               int64_t N, int64_t K, void* stream) {
    if (type != RIDGE_F16 && type != RIDGE_BF16 && type != RIDGE_F32) return hipErrorInvalidValue;
    if (M < 0 || N < 0 || K < 1 || K > RIDGE_INT8_MAX_K) return hipErrorInvalidValue;
    if (M == 0 || N == 0) return hipSuccess;
    const size_t size = type == RIDGE_F32 ? 4 : 2;
    constexpr int64_t kMostRows = INT32_MAX - 255;   // whole tiles of them still fit 31 bits
    if (M > kMostRows || N > kMostRows || lda < K || ldb < K || lda % 16 || ldb % 16 || lda >= (1 << 23) ||
        ldb >= (1 << 23) || ldc < N || !aligned(A, 16) || !aligned(B, 16) || !aligned(scaleA, 4) ||
        !aligned(scaleB, 4) || !aligned(C, size) || ((uintptr_t)bias & (size - 1)))
        return hipErrorInvalidValue;
    const Int8Args args = {A,        B,        scaleA, scaleB, bias,   C, (int)lda, (int)ldb, ldc, (int)M,
                           (int)N, (int)K, {}};
    switch (type) {
        case RIDGE_F16: return launchGemm<_Float16>(args, (hipStream_t)stream);
        case RIDGE_BF16: return launchGemm<__bf16>(args, (hipStream_t)stream);
        default: return launchGemm<float>(args, (hipStream_t)stream);
    }
}
