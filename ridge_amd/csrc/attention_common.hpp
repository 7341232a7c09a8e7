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
#include <type_traits>

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

// A number that is the same for all lanes, read past the vector unit.
__device__ __forceinline__ int32_t uniformLoad(const int32_t* at) {
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)at;
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

// What op makes of the values of the LANES lanes (a power of two) of a row, in all of them: within 16
// lanes by exchanges that are part of an instruction, behind that by swaps of registers' halves.
template <int LANES, typename T, typename Op>
__device__ __forceinline__ T overLanes(T v, Op op) {
    auto moved = [](T x, auto control) {
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(control)::value, 15, 15, true));
    };
    auto both = [&](auto halves) {   // an element of a vector has no address for a cast of its bits
        const unsigned a = halves[0], b = halves[1];
        return op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
    };
    if constexpr (LANES >= 2) v = op(v, moved(v, std::integral_constant<int, 0xb1>()));    // lanes 1 0 3 2
    if constexpr (LANES >= 4) v = op(v, moved(v, std::integral_constant<int, 0x4e>()));    // lanes 2 3 0 1
    if constexpr (LANES >= 8) v = op(v, moved(v, std::integral_constant<int, 0x141>()));   // 8 lanes mirrored
    if constexpr (LANES >= 16) v = op(v, moved(v, std::integral_constant<int, 0x140>()));  // 16 lanes mirrored
    const auto bits = [&] { return __builtin_bit_cast(unsigned, v); };
    if constexpr (LANES >= 32) v = both(__builtin_amdgcn_permlane16_swap(bits(), bits(), false, false));
    if constexpr (LANES >= 64) v = both(__builtin_amdgcn_permlane32_swap(bits(), bits(), false, false));
    return v;
}

template <int LANES>
__device__ __forceinline__ uint32_t mostOf(uint32_t top) {
    return overLanes<LANES>(top, [](uint32_t a, uint32_t b) { return max(a, b); });
}

template <int LANES>
__device__ __forceinline__ float sumOf(float sum) {
    return overLanes<LANES>(sum, [](float a, float b) { return a + b; });
}

}  // namespace ridge
