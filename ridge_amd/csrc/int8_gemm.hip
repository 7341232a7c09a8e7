// int8_gemm.hip -- the launches of the 8-bit product, for the C ABI in include/ridge_int8.h.

#include "int8_gemm.hpp"
#include "ridge_int8.h"

#include <hip/hip_runtime.h>

namespace {

using ridge::Int8Args;

template <typename T, typename Out>
hipError_t launchTiles(Int8Args args, hipStream_t stream) {
    const int64_t tilesM = ridge::int8TilesM<T>(args.M), tilesN = ridge::int8TilesN<T>(args.N);
    if (tilesM * tilesN > (int64_t)UINT32_MAX / T::kThreads) return hipErrorInvalidValue;
    args.order = ridge::tileOrder<T::BM, T::BN, ridge::kInt8GroupM>((int)tilesM * T::BM, (int)tilesN * T::BN);
    ridge::int8GemmKernel<T, Out><<<dim3((unsigned)(tilesM * tilesN)), dim3(T::kThreads), 0, stream>>>(args);
    return hipGetLastError();
}

template <typename Out>
hipError_t launchGemm(const Int8Args& args, hipStream_t stream) {
    return launchTiles<ridge::Int8Traits<128, 128, 128, 32, 64, 3>, Out>(args, stream);
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
