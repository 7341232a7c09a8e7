// attention_attend.hip -- the attention of each sequence's newest token over the 8-bit cache,
// for the C ABI in include/ridge_attention.h.
//
//   s_t = scale (q . k_t) kScale_t,  p_t = exp(s_t - max s),  out = sum p_t vScale_t v_t / sum p_t
//
// in one pass over the cache: a wave a query head, four columns a lane, with the running
// maximum and sum of the softmax. Sums are taken over 64 tokens and then of those: added one by
// one to a sum of 1, probabilities under 2^-24 would be lost however many there are.

#include "attention_common.hpp"

namespace {

using ridge::kBlock;
using ridge::kMostBlocks;
using ridge::kWave;
using ridge::kWavesPerBlock;

struct AttendArgs {
    ridge_attention_cache_t cache;
    const void* q;
    void* out;
    float* lse;
    const int32_t* pages;
    const int32_t* lengths;
    int64_t qToken, qHead, outToken, outHead, pagesStride, pagesEach, window;
    int32_t batch, heads;
    float scale;   // times log2(e): exponentials are powers of two
};

template <typename T>
__global__ __launch_bounds__(kBlock) void attendKernel(AttendArgs a) {
    constexpr int kVec = 4;
    typedef signed char Bytes __attribute__((ext_vector_type(kVec), aligned(4)));
    const ridge_attention_cache_t& c = a.cache;
    const int lane = threadIdx.x % kWave, col = lane * kVec;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const bool holds = col < c.dim;   // rows are readable to 16 bytes
    for (uint32_t i = blockIdx.x * kWavesPerBlock + wave; i < (uint32_t)(a.batch * a.heads); i += kMostBlocks * kWavesPerBlock) {
        const int64_t b = i / a.heads;
        const int head = (int)(i - b * a.heads), kvHead = head / (a.heads / c.heads);
        const int32_t length = a.lengths[b];
        const bool bad = length < 0 || length > a.pagesEach * c.pageSize;
        const T* const q = (const T*)a.q + b * a.qToken + head * a.qHead;
        float x[kVec], o[kVec] = {}, top = -INFINITY, sum = 0.0f, some[kVec] = {}, someSum = 0.0f;
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = col + e < c.dim ? (float)q[col + e] * a.scale : 0.0f;
        for (int32_t t = a.window ? (int32_t)max(length - a.window, (int64_t)0) : 0; !bad && t < length; ++t) {
            const int32_t page = a.pages[b * a.pagesStride + t / c.pageSize];
            const int at = (int)(t % c.pageSize);
            const bool there = (uint32_t)page < (uint64_t)c.pages;
            const int64_t row = (there ? page : 0) * c.pageStride + kvHead * c.headStride + at * c.tokenStride + col;
            const int64_t scaleAt = (there ? page : 0) * c.scalePage + kvHead * c.scaleHead + at;
            const Bytes k = holds ? *(const Bytes*)(c.k + row) : Bytes(0), v = holds ? *(const Bytes*)(c.v + row) : Bytes(0);
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < kVec; ++e) s = fmaf(x[e], (float)k[e], s);
            s = there ? ridge::sumOf<kWave>(s) * c.kScale[scaleAt] : NAN;
            const float most = fmaxf(top, s), least = most == -INFINITY ? 0.0f : most;
            const float keep = __builtin_amdgcn_exp2f(top - least), p = __builtin_amdgcn_exp2f(s - least);
            const float pv = p * c.vScale[scaleAt];
            top = most;
            const bool last = t % 64 == 63 || t + 1 == length;
            someSum = fmaf(someSum, keep, p);
            sum = fmaf(sum, keep, last ? someSum : 0.0f);
            someSum = last ? 0.0f : someSum;
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                some[e] = fmaf(some[e], keep, pv * (float)v[e]);
                o[e] = fmaf(o[e], keep, last ? some[e] : 0.0f);
                some[e] = last ? 0.0f : some[e];
            }
        }
        const bool none = length == 0;
        T* const out = (T*)a.out + b * a.outToken + head * a.outHead;
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            if (col + e < c.dim) out[col + e] = (T)(bad ? NAN : none ? 0.0f : o[e] / sum);
        if (lane == 0 && a.lse) a.lse[i] = bad ? NAN : none ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
    }
}

}  // namespace

extern "C" int64_t ridge_attention_workspace(int64_t batch, int32_t heads, int32_t kvHeads, int32_t dim, int64_t pagesEach,
                                             int32_t pageSize) {
    if (batch < 0 || kvHeads < 1 || heads < 0 || heads > 65535 || batch > INT32_MAX / std::max(heads, 1) || heads % kvHeads || dim < 1 ||
        dim > RIDGE_ATTENTION_MAX_DIM || pageSize < 16 || pageSize % 16 || pagesEach < 0 ||
        pagesEach > RIDGE_ATTENTION_MAX_SLOTS / pageSize)
        return -1;
    return 0;
}

extern "C" int ridge_attention_attend(const ridge_attention_heads_t* q, const ridge_attention_cache_t* cache,
                                      const int32_t* pages, int64_t pagesStride, int64_t pagesEach, const int32_t* lengths,
                                      float scale, int64_t window, const ridge_attention_heads_t* out, float* lse, int type,
                                      int64_t batch, void* workspace, int64_t workspaceBytes, void* stream) {
    if (!ridge::isType(type) || !ridge::cacheFits(cache) || !ridge::headsFit(q, type, batch) || !ridge::headsFit(out, type, batch) ||
        q->heads != out->heads || !(std::fabs(scale) <= FLT_MAX / 2) || window < 0 || pagesStride < 0)
        return hipErrorInvalidValue;
    const int64_t wanted =
        ridge_attention_workspace(batch, q->heads, cache->heads, cache->dim, pagesEach, cache->pageSize);
    if (wanted < 0) return hipErrorInvalidValue;
    if (batch == 0 || q->heads == 0) return hipSuccess;
    if (workspaceBytes < wanted || (wanted && !ridge::aligned(workspace, 16)) || (pagesEach && !ridge::aligned(pages, 4)) ||
        !ridge::aligned(lengths, 4) || (lse && !ridge::aligned(lse, 4)))
        return hipErrorInvalidValue;
    AttendArgs a = {};
    a.cache = *cache, a.q = q->at, a.out = out->at, a.lse = lse, a.pages = pages, a.lengths = lengths;
    a.qToken = q->token, a.qHead = q->head, a.outToken = out->token, a.outHead = out->head;
    a.pagesStride = pagesStride, a.pagesEach = pagesEach, a.window = window, a.batch = (int32_t)batch, a.heads = q->heads;
    a.scale = (float)(scale * 1.4426950408889634);
    const int64_t blocks = std::min((batch * q->heads + kWavesPerBlock - 1) / kWavesPerBlock, kMostBlocks);
    return ridge::typed(type, [&](auto element) {
        return ridge::launchKernel(attendKernel<decltype(element)>, (unsigned)blocks, kBlock, (hipStream_t)stream, a);
    });
}
