// attention_rope.hip -- the norm and the rotation of query and key heads in one pass, for the C
// ABI in include/ridge_attention.h.
//
//   y = x / sqrt(mean(x^2) + eps) * w,   y1' = y1 c - y2 s,   y2' = y2 c + y1 s
//
// for each pair of columns of each head of each token. Memory bounds it: each value is read
// once and written once, and a token's cosines and sines are read once for all of its heads.
// A lane holds both columns of its pairs, so the rotation needs no exchange between lanes and
// the norm one reduction over the few lanes of a head.

#include "attention_common.hpp"

namespace {

using ridge::kBlock;
using ridge::kWave;
using ridge::loadRow;
using ridge::storeRow;

struct RopeArgs {
    const void* q;
    const void* k;
    void* qOut;
    void* kOut;
    const void* qWeight;
    const void* kWeight;
    const float* table;
    const int32_t* positions;
    int64_t qToken, qHead, kToken, kHead, qOutToken, qOutHead, kOutToken, kOutHead, positionStride;
    int32_t tokens, qHeads, kHeads, tableRows, tableStride, pairs, dim;
    int32_t each, chunks;        // heads of a wave at a time and the parts that a token's heads are cut into
    int32_t axes, end0, end1, end2;    // the ends of the pairs of axes 0, 1 and 2
    int32_t interleaved;
    float eps;
};

// A token's rows of the table, one for each axis: their offsets, or kNowhere for a position outside it.
// They are the same for all lanes of a wave. A table is less than 4 GiB.
constexpr uint32_t kNowhere = 0xffffffff;
struct Rows {
    uint32_t at[RIDGE_ATTENTION_MAX_AXES];
    __device__ Rows(const RopeArgs& a, int64_t token) {
#pragma unroll
        for (int i = 0; i < RIDGE_ATTENTION_MAX_AXES; ++i) {
            const uint32_t position = (uint32_t)ridge::uniformLoad(a.positions + token * a.positionStride + min(i, a.axes - 1));
            at[i] = position < (uint32_t)a.tableRows ? position * (uint32_t)a.tableStride : kNowhere;
        }
    }
    // The cosines of a pair, sines behind them; `there`: whether its position is in the table, whose
    // first row it is otherwise.
    __device__ __forceinline__ const float* of(const RopeArgs& a, int pair, bool& there) const {
        const uint32_t row = pair < a.end0 ? at[0] : pair < a.end1 ? at[1] : pair < a.end2 ? at[2] : at[3];
        there = row != kNowhere;
        return a.table + ((there ? row : 0) + (uint32_t)pair);
    }
};

// A head's sum of squares past the range of f32 would make the root 0 and the head silently so.
__device__ __forceinline__ float rootOf(float squares, const RopeArgs& a) {
    return squares <= FLT_MAX ? 1.0f / sqrtf(squares / (float)a.dim + a.eps) : NAN;
}

// One head of a token, as its operands and results.
template <typename T, typename W>
struct Head {
    const T* x;
    T* out;
    const W* weight;
    __device__ Head(const RopeArgs& a, int64_t token, int head) {
        const bool isQ = head < a.qHeads;
        const int h = isQ ? head : head - a.qHeads;
        x = isQ ? (const T*)a.q + token * a.qToken + h * a.qHead : (const T*)a.k + token * a.kToken + h * a.kHead;
        out = isQ ? (T*)a.qOut + token * a.qOutToken + h * a.qOutHead : (T*)a.kOut + token * a.kOutToken + h * a.kOutHead;
        weight = (const W*)(isQ ? a.qWeight : a.kWeight);
    }
};

template <bool STREAM, typename Vec, typename T>
__device__ __forceinline__ Vec loadVec(const T* at) {
    if constexpr (STREAM) return __builtin_nontemporal_load((const Vec*)at);
    return *(const Vec*)at;
}

// V pairs a lane, LANES lanes a head: what vectors of V elements hold whole of. The columns that
// keep their values follow the pairs, two vectors a lane as well. STREAM: past the caches. MIXED: a
// section may end inside a vector of pairs.
template <typename T, typename W, int V, int LANES, bool INTERLEAVED, bool STREAM, bool MIXED>
__global__ __launch_bounds__(kBlock) void ropeKernel(RopeArgs a) {
    typedef typename ridge::Memory<T, V>::Vec Vec;
    constexpr int kHeads = kWave / LANES;
    const int lane = threadIdx.x % LANES;
    const int turning = a.pairs / V, still = (a.dim - 2 * a.pairs) / V;   // vectors of pairs, and of other columns
    const bool turns = lane < turning;
    const int pair = lane * V, rest = 2 * (lane - turning);
    const int first = turns ? (INTERLEAVED ? 2 * pair : pair) : 2 * a.pairs + rest * V;
    const int second = turns ? (INTERLEAVED ? 2 * pair + V : a.pairs + pair) : first + V;
    const bool hasFirst = turns || rest < still, hasSecond = turns || rest + 1 < still;
    const int heads = a.qHeads + a.kHeads;
    ridge::walkParts(a.tokens, a.chunks, [&](int64_t token, int part) {
        const int from = part * a.each * kHeads + (int)(threadIdx.x % kWave) / LANES;
        // Each head's columns are on their way while the one before it is turned, the first one's with
        // the rotation.
        Vec next[2] = {};
        auto load = [&](int head) {
            const T* const x = Head<T, W>(a, token, head).x;
            if (hasFirst) next[0] = loadVec<STREAM, Vec>(x + first);
            if (hasSecond) next[1] = loadVec<STREAM, Vec>(x + second);
        };
        if (from < heads) load(from);
        const Rows rows(a, token);
        float c[V], s[V];
        if (turns) {
            bool there;
            if constexpr (!MIXED) {   // a vector's pairs are of one axis
                const float* const row = rows.of(a, pair, there);
                loadRow<false>(row, c);
                loadRow<false>(row + a.pairs, s);
#pragma unroll
                for (int e = 0; e < V; ++e) c[e] = there ? c[e] : NAN;
            } else {
                int begin = pair;
                asm volatile("" : "+v"(begin));   // the comparisons of a vector's pairs are not held from token to token
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float* const row = rows.of(a, begin + e, there);
                    c[e] = there ? row[0] : NAN, s[e] = row[a.pairs];
                }
            }
        }
        for (int i = 0; i < a.each; ++i) {
            const int head = from + i * kHeads;
            if (head >= heads) return;
            const Head<T, W> h(a, token, head);
            float x[2][V];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) x[j][e] = (float)next[j][e];
            if (i + 1 < a.each && head + kHeads < heads) load(head + kHeads);
            if (h.weight) {
                float squares = 0.0f;
#pragma unroll
                for (int e = 0; e < V; ++e) squares = fmaf(x[0][e], x[0][e], fmaf(x[1][e], x[1][e], squares));
                const float root = rootOf(ridge::sumOf<LANES>(squares), a);
                float w[2][V] = {};
                if (hasFirst) loadRow<false>(h.weight + first, w[0]);
                if (hasSecond) loadRow<false>(h.weight + second, w[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) x[j][e] = x[j][e] * root * w[j][e];
            }
            if (turns) {
                // The lane's pairs: of x[0] and x[1], or of each other column of both.
                constexpr int kBehind = INTERLEAVED && V > 1 ? 1 : V;
                float* const flat = x[0];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float &y1 = flat[kBehind == 1 ? 2 * e : e], &y2 = flat[(kBehind == 1 ? 2 * e : e) + kBehind];
                    const float turned = fmaf(y1, c[e], -(y2 * s[e]));
                    y2 = fmaf(y2, c[e], y1 * s[e]);
                    y1 = turned;
                }
            }
            if (hasFirst) storeRow<STREAM>(h.out + first, x[0]);
            if (hasSecond) storeRow<STREAM>(h.out + second, x[1]);
        }
    });
}

// More than 64 odd pairs and columns: a wave a head, a column a lane at a time. A column's partner
// is read again; every read is before the first write, so that a head may be turned in place.
template <typename T, typename W>
__global__ __launch_bounds__(kBlock) void ropeAnyKernel(RopeArgs a) {
    constexpr int kMost = RIDGE_ATTENTION_MAX_DIM / kWave;
    const int heads = a.qHeads + a.kHeads;
    ridge::walkParts(a.tokens, a.chunks, [&](int64_t token, int part) {
        const int from = part * a.each;
        for (int head = from; head < min(heads, from + a.each); ++head) {
            const Head<T, W> h(a, token, head);
            int lane = threadIdx.x % kWave;
            asm volatile("" : "+v"(lane));   // nor are comparisons of columns held here
            float x[kMost], other[kMost], squares = 0.0f;
            auto partnerOf = [&](int col) { return a.interleaved ? col ^ 1 : col < a.pairs ? col + a.pairs : col - a.pairs; };
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                const int col = lane + i * kWave;
                x[i] = col < a.dim ? (float)h.x[col] : 0.0f;
                other[i] = col < 2 * a.pairs ? (float)h.x[partnerOf(col)] : 0.0f;
                squares = fmaf(x[i], x[i], squares);
            }
            const float root = h.weight ? rootOf(ridge::sumOf<kWave>(squares), a) : 1.0f;
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                const int col = lane + i * kWave;
                if (col >= a.dim) break;
                float y = h.weight ? x[i] * root * (float)h.weight[col] : x[i];
                if (col < 2 * a.pairs) {
                    const int partner = partnerOf(col);
                    const float z = h.weight ? other[i] * root * (float)h.weight[partner] : other[i];
                    const Rows rows(a, token);
                    const bool isFirst = col < partner;
                    const int pair = a.interleaved ? col / 2 : min(col, partner);
                    bool there;
                    const float* const row = rows.of(a, pair, there);
                    const float c = there ? row[0] : NAN, s = row[a.pairs];
                    y = isFirst ? fmaf(y, c, -(z * s)) : fmaf(y, c, z * s);
                }
                h.out[col] = (T)y;
            }
        }
    });
}

// The cosines and sines stay in a wave's registers for the heads of its part.
template <typename Kernel>
hipError_t launchRope(Kernel kernel, RopeArgs a, int perWave, hipStream_t stream) {
    const ridge::Cut cut(a.tokens, (a.qHeads + a.kHeads + perWave - 1) / perWave);
    a.each = cut.each, a.chunks = cut.chunks;
    return ridge::launchKernel(kernel, cut.blocks, kBlock, stream, a);
}

template <typename T, typename W, int V, int LANES, bool STREAM, bool MIXED>
hipError_t launchLanes(const RopeArgs& a, hipStream_t stream) {
    return a.interleaved ? launchRope(ropeKernel<T, W, V, LANES, true, STREAM, MIXED>, a, kWave / LANES, stream)
                         : launchRope(ropeKernel<T, W, V, LANES, false, STREAM, MIXED>, a, kWave / LANES, stream);
}

template <typename T, typename W, int V, int LANES>
hipError_t launchLanes(const RopeArgs& a, bool streams, hipStream_t stream) {
    const bool mixed = a.end0 % V || a.end1 % V || a.end2 % V;
    if constexpr (V > 1)
        if (mixed) return launchLanes<T, W, V, LANES, false, true>(a, stream);
    if constexpr (V * sizeof(T) == 16)
        if (streams) return launchLanes<T, W, V, LANES, true, false>(a, stream);
    return launchLanes<T, W, V, LANES, false, false>(a, stream);
}

// Heads of this size in all, and more, are read and written past the caches: what the attention of
// a prompt reads next would not find them there.
constexpr int64_t kStreamBytes = (int64_t)64 << 20;

// The widest vectors that pairs and columns are whole ones of, up to 16 bytes a lane and load.
template <typename T, typename W>
hipError_t launchTyped(const RopeArgs& a, hipStream_t stream) {
    constexpr int kWide = 16 / sizeof(T);
    const int rest = a.dim - 2 * a.pairs;
    int v = kWide;
    while (v > 1 && (a.pairs % v || rest % v)) v /= 2;
    const int lanes = a.pairs / v + (rest / v + 1) / 2;
    const bool streams = (int64_t)a.tokens * (a.qHeads + a.kHeads) * a.dim * (int64_t)sizeof(T) >= kStreamBytes;
    if constexpr (kWide == 8) {   // 256 columns are 16 lanes
        if (v == 8 && lanes <= 4) return launchLanes<T, W, 8, 4>(a, streams, stream);
        if (v == 8 && lanes <= 8) return launchLanes<T, W, 8, 8>(a, streams, stream);
        if (v == 8) return launchLanes<T, W, 8, 16>(a, streams, stream);
    }
    if (v == 4 && lanes <= 16) return launchLanes<T, W, 4, 16>(a, streams, stream);
    if (v == 4) return launchLanes<T, W, 4, 32>(a, streams, stream);
    if (v == 2 && lanes <= 32) return launchLanes<T, W, 2, 32>(a, streams, stream);
    if (v == 2) return launchLanes<T, W, 2, 64>(a, streams, stream);
    return lanes <= 64 ? launchLanes<T, W, 1, 64>(a, streams, stream) : launchRope(ropeAnyKernel<T, W>, a, 1, stream);
}

}  // namespace

extern "C" int ridge_attention_norm_rope(const ridge_attention_heads_t* q, const ridge_attention_heads_t* k, int type,
                                         const void* qWeight, const void* kWeight, int weightType, float eps,
                                         const ridge_attention_rotation_t* rotation, const ridge_attention_heads_t* qOut,
                                         const ridge_attention_heads_t* kOut, int64_t tokens, int32_t dim, void* stream) {
    using ridge::aligned, ridge::headsFit, ridge::sizeOf;
    if (!ridge::isType(type) || tokens < 0 || tokens > INT32_MAX || dim < 1 || dim > RIDGE_ATTENTION_MAX_DIM ||
        rotation == nullptr || !(eps > 0.0f && eps <= FLT_MAX))
        return hipErrorInvalidValue;
    if ((qWeight || kWeight) && weightType != type && weightType != RIDGE_F32) return hipErrorInvalidValue;
    for (const void* weight : {qWeight, kWeight})
        if (weight && !aligned(weight, sizeOf(weightType))) return hipErrorInvalidValue;
    const ridge_attention_rotation_t& r = *rotation;
    if (r.pairs < 1 || r.pairs > dim / 2 || r.axes < 1 || r.axes > RIDGE_ATTENTION_MAX_AXES || r.tableRows < 1 ||
        r.tableRows > INT32_MAX || r.tableStride < 2 * r.pairs || r.tableStride >= (1ll << 30) / r.tableRows || r.positionStride < 0 || !aligned(r.table, 4))
        return hipErrorInvalidValue;
    int ends[RIDGE_ATTENTION_MAX_AXES], end = 0;
    for (int i = 0; i < RIDGE_ATTENTION_MAX_AXES; ++i) {
        if (i < r.axes && (r.sections[i] < 0 || r.sections[i] > r.pairs - end)) return hipErrorInvalidValue;
        end += i < r.axes ? r.sections[i] : 0;
        ends[i] = i + 1 < r.axes ? end : r.pairs;
    }
    if (end != r.pairs) return hipErrorInvalidValue;
    if (!headsFit(q, type, tokens) || !headsFit(k, type, tokens) || !headsFit(qOut, type, tokens) || !headsFit(kOut, type, tokens) ||
        q->heads != qOut->heads || k->heads != kOut->heads)
        return hipErrorInvalidValue;
    if (tokens == 0 || q->heads + k->heads == 0) return hipSuccess;
    if (!aligned(r.positions, 4)) return hipErrorInvalidValue;
    RopeArgs a = {};
    a.q = q->at, a.k = k->at, a.qOut = qOut->at, a.kOut = kOut->at, a.qWeight = qWeight, a.kWeight = kWeight;
    a.table = r.table, a.positions = r.positions;
    a.qToken = q->token, a.qHead = q->head, a.kToken = k->token, a.kHead = k->head;
    a.qOutToken = qOut->token, a.qOutHead = qOut->head, a.kOutToken = kOut->token, a.kOutHead = kOut->head;
    a.tableStride = (int32_t)r.tableStride, a.positionStride = r.positionStride, a.tokens = (int32_t)tokens;
    a.qHeads = q->heads, a.kHeads = k->heads, a.tableRows = (int32_t)r.tableRows, a.pairs = r.pairs, a.dim = dim;
    a.end0 = ends[0], a.end1 = ends[1], a.end2 = ends[2], a.interleaved = r.interleaved != 0, a.eps = eps, a.axes = r.axes;
    hipStream_t s = (hipStream_t)stream;
    return ridge::typed(type, [&](auto element) {
        typedef decltype(element) T;
        if (weightType == RIDGE_F32 && (qWeight || kWeight)) return launchTyped<T, float>(a, s);
        return launchTyped<T, T>(a, s);
    });
}
