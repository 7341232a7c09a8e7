// attention_cache.hip -- rows written to the 8-bit cache and read back, for the C ABI in
// include/ridge_attention.h.
//
// A row (a token's key or value of one head) is held by the lanes that its columns fill, 8
// values each: one read of it, its largest magnitude by exchanges between those lanes, and
// the rounding that every 8-bit row of the framework has. Memory bounds both directions.

#include "attention_common.hpp"

namespace {

using ridge::kBlock;
using ridge::kWave;

constexpr int kVec = 8;   // columns of a lane

struct CacheArgs {
    ridge_attention_cache_t cache;
    const int32_t* slots;
    void* k;
    void* v;
    int64_t kToken, kHead, vToken, vHead;
    int32_t tokens, each, chunks;   // a wave's heads at a time and the parts that a token's are cut into
};

// n values of a head at once, the last few of its columns one at a time.
template <typename T>
__device__ __forceinline__ void loadPart(const T* at, int n, float (&x)[kVec]) {
    if (n >= kVec) return ridge::loadRow<false>(at, x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = e < n ? (float)at[e] : 0.0f;
}

template <bool STREAM, typename T>
__device__ __forceinline__ void storePart(T* at, int n, const float (&x)[kVec]) {
    if (n >= kVec) return ridge::storeRow<STREAM>(at, x);
#pragma unroll
    for (int e = 0; e < kVec; ++e)
        if (e < n) at[e] = (T)x[e];
}

// Calls f(token, its slot, head) for each head whose key and value this lane has a part of.
template <int LANES, typename F>
__device__ __forceinline__ void walk(const CacheArgs& a, F&& f) {
    constexpr int kHeads = kWave / LANES;
    ridge::walkParts(a.tokens, a.chunks, [&](int64_t token, int part) {
        const int32_t slot = ridge::uniformLoad(a.slots + token);
        const int from = part * a.each * kHeads + (int)(threadIdx.x % kWave) / LANES;
        for (int i = 0; i < a.each; ++i) {
            const int head = from + i * kHeads;
            if (head < a.cache.heads) f(token, slot, head);
        }
    });
}

// Where a slot's row of a head and its scale are, from the beginning of k or v.
struct Place {
    int64_t row, scale;
    __device__ Place(const ridge_attention_cache_t& c, int32_t slot, int head) {
        const int32_t page = slot / c.pageSize, at = slot - page * c.pageSize;
        row = page * c.pageStride + head * c.headStride + at * c.tokenStride;
        scale = page * c.scalePage + head * c.scaleHead + at;
    }
};

__device__ __forceinline__ bool holds(const ridge_attention_cache_t& c, int32_t slot) {
    return slot >= 0 && slot / c.pageSize < c.pages;
}

// x / 127, rounded correctly: the product with the reciprocal, corrected by its exact remainder. Three
// instructions where a division takes ten. (Infinities become NaNs.)
__device__ __forceinline__ float by127(float x) {
    constexpr float kInverse = 1.0f / 127.0f;
    const float q = x * kInverse;
    return fmaf(fmaf(-127.0f, q, x), kInverse, q);
}

// A row's 8 bits out of this lane's part of it, and its scale: as ridge::stepOf has them for a row that
// nothing multiplies, with two divisions by 127 instead of three of any numbers. The vector ALU bounds
// the writing (16384 x 8 x 128 in bfloat16 25.1 us with stepOf and a lift of every row).
template <int LANES>
__device__ __forceinline__ void storeRow8(float (&x)[kVec], int n, int8_t* at, float* scaleAt) {
    uint32_t top = 0;
#pragma unroll
    for (float value : x) top = max(top, ridge::magnitude(value));
    const float most = __uint_as_float(ridge::mostOf<LANES>(top));
    const bool small = most < ridge::kSmallRow;
    const float lifted = small ? most * ridge::kLift : most;
    ridge::Step step;
    step.whole = by127(lifted);
    step.rest = by127(fmaf(-127.0f, step.whole, lifted));
    float scale = most <= FLT_MAX ? step.whole : most;
    if (__builtin_amdgcn_ballot_w64(small)) {   // few waves have such a row
        scale = small ? step.whole / ridge::kLift : scale;
        if (scale < FLT_MIN) {
            scale = FLT_MIN;
            step.whole = FLT_MIN * ridge::kLift, step.rest = 0.0f;
        }
#pragma unroll
        for (float& value : x) value *= small ? ridge::kLift : 1.0f;
    }
    step.inverse = 1.0f / step.whole;
    if (n >= kVec) {
        ridge::storeRounded(at, x, step);
    } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const float one[1] = {x[e]};
            if (e < n) ridge::storeRounded(at + e, one, step);
        }
    }
    if (threadIdx.x % LANES == 0) *scaleAt = scale;
}

template <typename T, int LANES>
__global__ __launch_bounds__(kBlock) void writeKernel(CacheArgs a) {
    const int col = threadIdx.x % LANES * kVec, n = a.cache.dim - col;
    walk<LANES>(a, [&](int64_t token, int32_t slot, int head) {
        float k[kVec] = {}, v[kVec] = {};   // on their way beside the slot
        if (n > 0) {
            loadPart((const T*)a.k + token * a.kToken + head * a.kHead + col, n, k);
            loadPart((const T*)a.v + token * a.vToken + head * a.vHead + col, n, v);
        }
        if (!holds(a.cache, slot)) return;
        const Place to(a.cache, slot, head);
        storeRow8<LANES>(k, n, a.cache.k + to.row + col, a.cache.kScale + to.scale);
        storeRow8<LANES>(v, n, a.cache.v + to.row + col, a.cache.vScale + to.scale);
    });
}

// STREAM: the values past the caches.
template <typename T, int LANES, bool STREAM>
__global__ __launch_bounds__(kBlock) void readKernel(CacheArgs a) {
    typedef signed char Bytes __attribute__((ext_vector_type(kVec), aligned(8)));
    const int col = threadIdx.x % LANES * kVec, n = a.cache.dim - col;
    walk<LANES>(a, [&](int64_t token, int32_t slot, int head) {
        if (n <= 0) return;
        float k[kVec], v[kVec];
        if (holds(a.cache, slot)) {
            const Place from(a.cache, slot, head);
            const Bytes kb = *(const Bytes*)(a.cache.k + from.row + col);   // rows are readable to 16
            const Bytes vb = *(const Bytes*)(a.cache.v + from.row + col);
            const float kScale = a.cache.kScale[from.scale], vScale = a.cache.vScale[from.scale];
#pragma unroll
            for (int e = 0; e < kVec; ++e) k[e] = (float)kb[e] * kScale, v[e] = (float)vb[e] * vScale;
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) k[e] = v[e] = slot < 0 ? 0.0f : NAN;
        }
        storePart<STREAM>((T*)a.k + token * a.kToken + head * a.kHead + col, n, k);
        storePart<STREAM>((T*)a.v + token * a.vToken + head * a.vHead + col, n, v);
    });
}

template <typename Kernel>
hipError_t launchRows(Kernel kernel, CacheArgs a, int lanes, hipStream_t stream) {
    const int rows = kWave / lanes;
    const ridge::Cut cut(a.tokens, (a.cache.heads + rows - 1) / rows);
    a.each = cut.each, a.chunks = cut.chunks;
    return ridge::launchKernel(kernel, cut.blocks, kBlock, stream, a);
}

// Values of this size in all, and more, are written past the caches (us of 32768 x 8 x 128 in
// bfloat16, cached | past them: 42.5 | 33.4). Rows are read and written through them.
constexpr int64_t kStreamBytes = (int64_t)64 << 20;

template <typename T, int LANES>
hipError_t launchLanes(const CacheArgs& a, bool write, hipStream_t s) {
    if (write) return launchRows(writeKernel<T, LANES>, a, LANES, s);
    const bool streams = 2 * (int64_t)a.tokens * a.cache.heads * a.cache.dim * (int64_t)sizeof(T) >= kStreamBytes;
    return launchRows(streams ? readKernel<T, LANES, true> : readKernel<T, LANES, false>, a, LANES, s);
}

template <typename T>
hipError_t launchTyped(const CacheArgs& a, bool write, hipStream_t s) {
    if (a.cache.dim <= 8 * kVec) return launchLanes<T, 8>(a, write, s);
    if (a.cache.dim <= 16 * kVec) return launchLanes<T, 16>(a, write, s);
    return launchLanes<T, 32>(a, write, s);
}

hipError_t launchCache(const ridge_attention_cache_t* cache, const int32_t* slots, const ridge_attention_heads_t* k,
                       const ridge_attention_heads_t* v, int type, int64_t tokens, bool write, void* stream) {
    if (!ridge::isType(type) || !ridge::cacheFits(cache) || !ridge::headsFit(k, type, tokens) || !ridge::headsFit(v, type, tokens) ||
        k->heads != cache->heads || v->heads != cache->heads || tokens < 0 || tokens > INT32_MAX)
        return hipErrorInvalidValue;
    if (tokens == 0) return hipSuccess;
    if (!ridge::aligned(slots, 4)) return hipErrorInvalidValue;
    const CacheArgs a = {*cache, slots, k->at, v->at, k->token, k->head, v->token, v->head, (int32_t)tokens, 0, 0};
    return ridge::typed(type, [&](auto element) { return launchTyped<decltype(element)>(a, write, (hipStream_t)stream); });
}

}  // namespace

extern "C" int ridge_attention_write(const ridge_attention_cache_t* cache, const int32_t* slots,
                                     const ridge_attention_heads_t* k, const ridge_attention_heads_t* v, int type,
                                     int64_t tokens, void* stream) {
    return launchCache(cache, slots, k, v, type, tokens, true, stream);
}

extern "C" int ridge_attention_read(const ridge_attention_cache_t* cache, const int32_t* slots,
                                    const ridge_attention_heads_t* k, const ridge_attention_heads_t* v, int type,
                                    int64_t tokens, void* stream) {
    return launchCache(cache, slots, k, v, type, tokens, false, stream);
}
