// attention_common.hpp -- what the launches around the 8-bit cache share: the checks of their
// sizes and the walk of waves over the heads of tokens.
#pragma once

#include "int8_launch.hpp"
#include "int8_values.hpp"
#include "ridge_attention.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace ridge {

constexpr int kWave = 64;
constexpr int kBlock = 256;
constexpr int kWavesPerBlock = kBlock / kWave;
constexpr int64_t kMostBlocks = 1 << 20;  // of a grid: its blocks walk what is behind them

inline bool isType(int type) { return type == RIDGE_F16 || type == RIDGE_BF16 || type == RIDGE_F32; }
inline size_t sizeOf(int type) { return type == RIDGE_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t to) { return p != nullptr && ((uintptr_t)p & (to - 1)) == 0; }

// Heads that a kernel may walk: an address of their type where there are any, strides that are
// none below 0.
inline bool headsFit(const ridge_attention_heads_t* h, int type, int64_t tokens) {
    return h != nullptr && h->heads >= 0 && h->heads <= 65535 && h->token >= 0 && h->head >= 0 &&
           (h->heads == 0 || tokens == 0 || aligned(h->at, sizeOf(type)));
}

inline bool cacheFits(const ridge_attention_cache_t* c) {
    if (c == nullptr || !aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->kScale, 16) || !aligned(c->vScale, 16))
        return false;
    for (int64_t stride : {c->pageStride, c->headStride, c->tokenStride})
        if (stride < 0 || stride % 16) return false;
    for (int64_t stride : {c->scalePage, c->scaleHead})
        if (stride < 0 || stride % 4) return false;
    // A block of 16 rows is reached by 32-bit offsets.
    return c->tokenStride < (int64_t)1 << 27 && c->dim >= 1 && c->dim <= RIDGE_ATTENTION_MAX_DIM && c->heads >= 1 && c->heads <= 65535 && c->pageSize >= 16 &&
           c->pageSize % 16 == 0 && c->pages >= 1 && c->pages <= RIDGE_ATTENTION_MAX_SLOTS / c->pageSize;
}

// f's answer for a value of the code's type.
template <typename F>
hipError_t typed(int type, F&& f) {
    switch (type) {
        case RIDGE_F16: return f((_Float16)0);
        case RIDGE_BF16: return f((__bf16)0);
        default: return f(0.0f);
    }
}

// A kernel's tokens are cut into `chunks` parts each, a wave a part. Calls f(token, part) for each
// part of this wave. There are fewer than 2^32 - kMostBlocks * kWavesPerBlock of them.
template <typename F>
__device__ __forceinline__ void walkParts(uint32_t tokens, uint32_t chunks, F&& f) {
    const uint32_t parts = tokens * chunks, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    for (uint32_t i = blockIdx.x * kWavesPerBlock + wave; i < parts; i += (uint32_t)kMostBlocks * kWavesPerBlock) {
        const uint32_t token = i / chunks;
        f((int64_t)token, (int)(i - token * chunks));
    }
}

// The cut: `each` of a token's `rounds` go to a part, so that there are about as many parts as
// waves run at a time (32 on each CU), and whole tokens where there are more tokens than that.
struct Cut {
    int each, chunks;
    unsigned blocks;
    Cut(int64_t tokens, int64_t rounds) {
        constexpr int64_t kWavesWanted = 8192;
        each = (int)std::clamp<int64_t>(tokens * rounds / kWavesWanted, 1, rounds);
        chunks = (int)((rounds + each - 1) / each);
        blocks = (unsigned)std::min((tokens * chunks + kWavesPerBlock - 1) / kWavesPerBlock, kMostBlocks);
    }
};

// Maximum over the LANES lanes (a power of two) of a row.
template <int LANES>
__device__ __forceinline__ uint32_t mostOf(uint32_t top) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    return top;
}

template <int LANES>
__device__ __forceinline__ float sumOf(float sum) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) sum += __shfl_xor(sum, d);
    return sum;
}

}  // namespace ridge
