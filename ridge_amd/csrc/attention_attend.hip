// attention_attend.hip -- the attention of each sequence's newest token over the 8-bit cache,
// for the C ABI in include/ridge_attention.h.
//
//   s_t = scale (q . k_t) kScale_t,  p_t = exp(s_t - max s),  out = sum p_t vScale_t v_t / sum p_t
//
// in one pass over the cache, whose bytes bound it: a workgroup takes one key head of a part of a
// sequence, its four waves 32 tokens at a time in turn, and each wave keeps the running maximum
// and sum of the softmax and the weighted values of up to 16 query heads that share the key head.
// Both products are matrix instructions (16 x 16 x 32, f16): 8-bit whole numbers are exact in f16,
// a query in 16 bits is too (of f32, and of p, two f16 parts are taken), and sums are f32.
//
// No operand goes through LDS or moves between lanes. The scores are computed transposed, keys as
// rows and heads as columns, so that a lane ends with 4 tokens of each 16 for one head; those are
// the k's that the second product, values as rows (transposed too) and heads as columns, wants
// from that lane, if the tokens of k = 8 g + 4 a + r are 16 a + 4 g + r. So a lane loads the values of
// those tokens and no others, and the running maximum's factor is its own head's everywhere.
//
// A sequence is cut into parts by its own length alone, so that its result does not depend on the
// others; a second launch joins the parts where there may be more than one.

#include "attention_common.hpp"

namespace {

using ridge::kBlock;
using ridge::kMostBlocks;
using ridge::kWave;
using ridge::kWavesPerBlock;

typedef _Float16 Half8 __attribute__((ext_vector_type(8)));
typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
typedef float Float4 __attribute__((ext_vector_type(4)));
typedef uint32_t Word4 __attribute__((ext_vector_type(4)));

constexpr int kHeadTile = 16;    // query heads of a workgroup
constexpr int kTile = 32;        // tokens of a wave at a time
constexpr int kRound = kTile * kWavesPerBlock;
constexpr int kLeastPart = 512;  // tokens of a part
constexpr int kMostParts = 64;   // of a sequence: longer ones have longer parts

struct AttendArgs {
    const int8_t* k;
    const int8_t* v;
    const float* kScale;
    const float* vScale;
    const void* q;
    void* out;
    float* lse;
    const int32_t* pages;
    const int32_t* lengths;
    float* parts;          // sums [batch * heads * mostParts][dim], then maxima and sums of p
    int64_t pageStride, headStride, scalePage, scaleHead;
    int64_t qToken, qHead, outToken, outHead, pagesStride;
    uint64_t pageMagic;    // (block * pageMagic) >> pageShift is block / blocks of a page
    uint32_t tokenStride, pageShift, pageBlocks, pages_;
    int32_t capacity, window, batch, heads, kvHeads, dim, tiles, mostParts;
    float scale;           // times log2(e): exponentials are powers of two
};

// What a sequence's length says: its tokens [begin, end), cut from `base` on into `parts` of
// `each`, whole rounds of a workgroup.
struct Range {
    int32_t begin, end, base, each, parts;
    bool bad;
    __host__ __device__ Range(int32_t length, int32_t capacity, int32_t window) {
        bad = length < 0 || length > capacity;
        end = bad ? 0 : length;
        begin = window && end > window ? end - window : 0;
        base = begin / 16 * 16;
        const int32_t n = end - base;
        each = n <= kLeastPart * kMostParts ? kLeastPart
                                            : (int32_t)(((int64_t)n + kMostParts * kRound - 1) / (kMostParts * kRound)) * kRound;
        parts = (int32_t)(((int64_t)n + each - 1) / each);
    }
};

__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// A whole number of the program's that is the same for all lanes, read past the vector unit.
__device__ __forceinline__ int32_t uniformLoad(const int32_t* at) {
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)at;
}

// Largest over the four lanes of a head (lane, lane ^ 16, lane ^ 32 and both).
__device__ __forceinline__ float most4(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum4(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// 2^n for n in -126 .. 127.
__device__ __forceinline__ float power2(int n) { return __int_as_float((n + 127) << 23); }
__device__ __forceinline__ int exponentOf(float v) { return (int)(__float_as_uint(v) >> 23 & 255) - 127; }

// Two f16 of the whole numbers in bytes `lo` of low and `hi` of high (biased by 128), times 2^-9:
// the byte as a f16 below the normal ones is its 2^-24th, which the product lifts and the sum unbiases.
__device__ __forceinline__ Half2 halves(uint32_t high, uint32_t low, int hi, int lo) {
    const uint32_t both = __builtin_amdgcn_perm(high, low, 0x0c000c00u | (uint32_t)(4 + hi) << 16 | (uint32_t)lo);
    const Half2 lift = {(_Float16)32768.0f, (_Float16)32768.0f}, bias = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_elementwise_fma(__builtin_bit_cast(Half2, both), lift, bias);
}
constexpr int kByteExponent = -9;

// Two values in f16, and what they leave. The compiler may convert a product with one rounding at one
// place and with two at another: the empty statement has the remainder taken of what was in fact
// rounded (without it a few heads in 1000 had a p off by 2^-11).
__device__ __forceinline__ void split(float a, float b, Half2& high, float& restA, float& restB) {
    uint32_t both = __builtin_bit_cast(uint32_t, Half2{(_Float16)a, (_Float16)b});
    asm("" : "+v"(both));
    high = __builtin_bit_cast(Half2, both);
    restA = a - (float)high.x;
    restB = b - (float)high.y;
}

__device__ __forceinline__ Half8 join(Half2 a, Half2 b, Half2 c, Half2 d) {
    return Half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Where a wave's 32 tokens are: two blocks of 16, each in one page. The same for all its lanes.
struct Place {
    int64_t rows[2], scales[2];   // from the beginning of k or v and of their scales
    bool there[2];                // whether the page is one of the cache's: else it is the first one instead
};

// 32 tokens' operands of a lane. COLS: a head's columns, padded.
template <int COLS>
struct Tile {
    static constexpr int kChunks = COLS / 16;      // 16-byte chunks of a key
    static constexpr int kKeys = COLS / 64;        // of them that a lane's scores take from each token
    static constexpr int kLoads = kChunks / 2;     // of a lane for 32 keys
    static constexpr int kWords = COLS / 64;       // words of a value that a lane loads
    Word4 k[kLoads];
    uint32_t v[2][4][kWords];
    Float4 kScale[2], vScale[2];
};

template <int COLS>
__device__ __forceinline__ void loadWords(uint32_t (&to)[COLS / 64], const int8_t* at) {
    typedef uint32_t Words __attribute__((ext_vector_type(COLS / 64)));
    if constexpr (COLS == 64) {
        to[0] = __builtin_nontemporal_load((const uint32_t*)at);
    } else {
        const Words w = __builtin_nontemporal_load((const Words*)at);
#pragma unroll
        for (int i = 0; i < COLS / 64; ++i) to[i] = w[i];
    }
}

// One workgroup's part of a sequence: 16 query heads over [from, to) of its tokens.
template <typename T, int COLS>
struct Part {
    static constexpr int kKeys = Tile<COLS>::kKeys;
    static constexpr int kBytes = COLS / 16;       // of a value that a lane loads, and sums of 16 columns that it holds 4 of
    static constexpr bool kSplitQ = sizeof(T) == 4;
    const AttendArgs& a;
    const int lane = threadIdx.x % kWave, at = lane % 16, group = lane / 16;
    Half8 q[kKeys][2], qLow[kSplitQ ? kKeys : 1][2];
    float qScale;                                  // of scores, in powers of two
    Float4 sum[kBytes];                            // of value columns kBytes (4 group + r) + i, for head `at`
    float top = -INFINITY, total = 0.0f;           // the largest score, and this lane's part of the sum of p
    float unit = 0.0f, lift = 0.0f;                // a power of two above every value's scale so far, and 2^15 / unit
    int exponent = 0;                              // of unit

    __device__ Part(const AttendArgs& a) : a(a) {}

    // The query's fragments: 8 columns from 64 i + 16 group + 8 j on, of head `at`, whose columns are in
    // LDS. Of bf16 and f32 the head is scaled by a power of two so that its largest column is 2^14
    // to 2^15.
    __device__ void loadQuery(const float* row) {
        float x[kKeys][2][8];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[i][j][e] = row[64 * i + 16 * group + 8 * j + e];
                    most = fmaxf(most, fabsf(x[i][j][e]));
                }
        float up = 1.0f;
        int down = 0;
        if constexpr (!std::is_same_v<T, _Float16>) {
            const int n = max(-96, exponentOf(most4(most)) - 14);
            up = n < -96 ? 1.0f : power2(-n);
            down = n;
        }
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    Half2 high;
                    float rest[2];
                    split(x[i][j][e] * up, x[i][j][e + 1] * up, high, rest[0], rest[1]);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        q[i][j][e + n] = high[n];
                        if constexpr (kSplitQ) qLow[i][j][e + n] = (_Float16)rest[n];
                    }
                }
        qScale = ldexpf(a.scale, down - kByteExponent);
    }

    // The 32 tokens from t on; blocks behind `lastBlock` are that one, which is masked.
    __device__ __forceinline__ Place find(int32_t t, int32_t lastBlock, const int32_t* pages) const {
        Place place;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t block = min(t / 16 + b, lastBlock);
            const uint32_t page = (uint32_t)((block * a.pageMagic) >> a.pageShift), in = (block - page * a.pageBlocks) * 16;
            const uint32_t p = uniformLoad(pages + page);
            place.there[b] = p < a.pages_;
            place.rows[b] = (int64_t)(place.there[b] ? p : 0) * a.pageStride + (int64_t)in * a.tokenStride;
            place.scales[b] = (int64_t)(place.there[b] ? p : 0) * a.scalePage + in;
        }
        return place;
    }

    // Whole keys, a chunk a lane: 64 / kChunks of them at once, which are whole cache lines. Of 64
    // columns a lane's chunk is the one that its scores take.
    __device__ __forceinline__ void loadKeys(Tile<COLS>& tile, const Place& place, const int8_t* k, const float* scales) const {
        constexpr int kChunks = Tile<COLS>::kChunks, kRows = kWave / kChunks;
        const uint32_t chunk = 16 * (kThroughLds ? lane % kChunks : group);
        const uint32_t offset = (kThroughLds ? lane / kChunks : at) * a.tokenStride + (chunk < dim16() ? chunk : 0);
#pragma unroll
        for (int n = 0; n < Tile<COLS>::kLoads; ++n) {
            const int row = n * kRows;
            tile.k[n] = __builtin_nontemporal_load((const Word4*)(k + place.rows[row / 16] + row % 16 * (int64_t)a.tokenStride + offset));
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            tile.kScale[b] = *(const Float4*)(scales + place.scales[b] + 4 * group);
            if (!place.there[b]) tile.kScale[b] = NAN;
        }
    }

    __device__ __forceinline__ void loadValues(Tile<COLS>& tile, const Place& place, const int8_t* v, const float* scales) const {
        const uint32_t col = kBytes * at, offset = 4 * group * a.tokenStride + (col < dim16() ? col : 0);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int r = 0; r < 4; ++r) loadWords<COLS>(tile.v[b][r], v + place.rows[b] + r * (int64_t)a.tokenStride + offset);
            tile.vScale[b] = *(const Float4*)(scales + place.scales[b] + 4 * group);
        }
    }

    __device__ __forceinline__ uint32_t dim16() const { return (a.dim + 15) & ~15; }

    // Keys go through LDS of the wave's own, from whole rows to the 16 bytes of a token that a lane's
    // scores take; chunks of a row are swapped so that neither side meets another lane's bank.
    static constexpr bool kThroughLds = COLS > 64;
    __device__ static __forceinline__ int swap(int row) { return COLS == 128 ? row / 2 % 8 : row % 16; }
    __device__ __forceinline__ void putKeys(const Tile<COLS>& tile, Word4* lds) const {
        constexpr int kChunks = Tile<COLS>::kChunks, kRows = kWave / kChunks;
#pragma unroll
        for (int n = 0; n < Tile<COLS>::kLoads; ++n) {
            const int row = n * kRows + lane / kChunks;
            lds[row * kChunks + (lane % kChunks ^ swap(row))] = tile.k[n];
        }
    }
    __device__ __forceinline__ void getKeys(Word4 (&k)[2][kKeys], const Word4* lds) const {
        constexpr int kChunks = Tile<COLS>::kChunks;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < kKeys; ++i) k[b][i] = lds[(16 * b + at) * kChunks + ((4 * i + group) ^ swap(16 * b + at))];
    }

    // The scores of 32 tokens.
    __device__ __forceinline__ void score(const Word4 (&k)[2][kKeys], const Float4 (&kScale)[2], float (&s)[2][4]) const {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            Float4 score = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                const Word4 w = k[b][i] ^ 0x80808080u;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t x = w[2 * j], y = w[2 * j + 1];
                    const Half8 keys = join(halves(x, x, 1, 0), halves(x, x, 3, 2), halves(y, y, 1, 0), halves(y, y, 3, 2));
                    score = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, q[i][j], score, 0, 0, 0);
                    if constexpr (kSplitQ) score = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, qLow[i][j], score, 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[b][r] = score[r] * kScale[b][r] * qScale;
        }
    }

    // Adds the tokens t .. t + 31 with their scores; those outside [begin, end) count nothing.
    __device__ __forceinline__ void add(Tile<COLS>& tile, float (&s)[2][4], int32_t t, int32_t begin, int32_t end) {
        if (t < begin || t + kTile > end) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int32_t token = t + 16 * b + 4 * group + r;
                    const bool counts = token >= begin && token < end;
                    s[b][r] = counts ? s[b][r] : -INFINITY;
                    tile.vScale[b][r] = counts ? tile.vScale[b][r] : 0.0f;
                }
        }
        float most = s[0][0], scale = fabsf(tile.vScale[0][0]);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) most = fmaxf(most, s[b][r]), scale = fmaxf(scale, fabsf(tile.vScale[b][r]));
        // Few tiles have a new maximum or a new largest scale: the sums are rescaled in a branch.
        if (__builtin_amdgcn_ballot_w64(most > top || scale > unit)) {
            const float next = fmaxf(top, most4(most));
            float factor = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - next);
            top = next;
            total *= factor;
#pragma unroll
            for (int d = 1; d < kWave; d *= 2) scale = fmaxf(scale, __shfl_xor(scale, d));
            if (scale > unit) {
                const int now = min(127, max(-112, exponentOf(scale) + 1));
                factor = unit == 0.0f ? 0.0f : ldexpf(factor, exponent - now);
                exponent = now;
                unit = power2(now);
                lift = power2(15 - now);
            }
#pragma unroll
            for (int i = 0; i < kBytes; ++i) sum[i] *= factor;
        }
        const float from = top == -INFINITY ? 0.0f : top;
        Half8 high, low;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                float weight[2], rest[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float p = __builtin_amdgcn_exp2f(s[b][r + n] - from);
                    total += p;
                    weight[n] = p * (tile.vScale[b][r + n] * lift);
                }
                Half2 both;
                split(weight[0], weight[1], both, rest[0], rest[1]);
#pragma unroll
                for (int n = 0; n < 2; ++n) high[4 * b + r + n] = both[n], low[4 * b + r + n] = (_Float16)rest[n];
            }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < Tile<COLS>::kWords; ++i) tile.v[b][r][i] ^= 0x80808080u;
#pragma unroll
        for (int i = 0; i < kBytes; ++i) {
            auto pair = [&](int b, int r) { return halves(tile.v[b][r + 1][i / 4], tile.v[b][r][i / 4], i % 4, i % 4); };
            const Half8 values = join(pair(0, 0), pair(0, 2), pair(1, 0), pair(1, 2));
            sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values, high, sum[i], 0, 0, 0);
            sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values, low, sum[i], 0, 0, 0);
        }
    }
};

// Result (b, head): 16 bits or f32 of `value` columns.
template <typename T>
__device__ __forceinline__ void storeOut(const AttendArgs& a, int64_t b, int head, int col, float value) {
    ((T*)a.out)[b * a.outToken + head * a.outHead + col] = (T)value;
}

__device__ __forceinline__ float logSum(float top, float total) {
    return (top + __builtin_amdgcn_logf(total)) * 0.69314718055994531f;
}

// Waves of a SIMD, by what their registers leave room for.
template <typename T>
constexpr int wavesOf(int cols) {
    return cols == 64 ? 4 : cols == 128 ? (sizeof(T) == 4 ? 2 : 3) : sizeof(T) == 4 ? 1 : 2;
}

template <typename T, int COLS>
__global__ __launch_bounds__(kBlock, wavesOf<T>(COLS)) void attendKernel(AttendArgs a) {
    constexpr int kBytes = COLS / 16;
    __shared__ float tops[kWavesPerBlock][kHeadTile], totals[kWavesPerBlock][kHeadTile];
    __shared__ union {
        float sums[kWavesPerBlock][kHeadTile][COLS + 4];
        Word4 keys[kWavesPerBlock][kTile * Tile<COLS>::kChunks];
    } lds;
    auto& sums = lds.sums;
    const int wave = uniform(threadIdx.x / kWave), shared = a.heads / a.kvHeads;
    const int part = blockIdx.x, kvHead = blockIdx.y / a.tiles, tile16 = blockIdx.y - kvHead * a.tiles;
    const int64_t b = blockIdx.z;
    const Range range(uniformLoad(a.lengths + b), a.capacity, a.window);
    const int first = kvHead * shared + tile16 * kHeadTile, count = min(kHeadTile, shared - tile16 * kHeadTile);
    if (range.parts == 0) {   // no tokens, or a length outside the cache
        if (part) return;
        for (int c = threadIdx.x; c < count * a.dim; c += kBlock)
            storeOut<T>(a, b, first + c / a.dim, c % a.dim, range.bad ? NAN : 0.0f);
        if (a.lse && threadIdx.x < count) a.lse[b * a.heads + first + threadIdx.x] = range.bad ? NAN : -INFINITY;
        return;
    }
    if (part >= range.parts) return;
    const int32_t from = range.base + part * range.each, to = min(range.end, from + range.each);
    const int32_t* const pages = a.pages + b * a.pagesStride;
    const int8_t *const k = a.k + kvHead * a.headStride, *const v = a.v + kvHead * a.headStride;
    const float *const kScale = a.kScale + kvHead * a.scaleHead, *const vScale = a.vScale + kvHead * a.scaleHead;
    const int32_t lastBlock = (to - 1) / 16;
    Part<T, COLS> p(a);
    Tile<COLS> tile;
    int32_t t = from + wave * kTile;
    Place place;
    if (t < to) {
        place = p.find(t, lastBlock, pages);
        p.loadKeys(tile, place, k, kScale);
        p.loadValues(tile, place, v, vScale);
    }
    // The heads' queries, in f32, with zeros behind them.
    const T* const q = (const T*)a.q + b * a.qToken + first * a.qHead;
    for (int c = threadIdx.x; c < kHeadTile * COLS; c += kBlock) {
        const int h = c / COLS, col = c % COLS;
        sums[0][h][col] = h < count && col < a.dim ? (float)q[h * a.qHead + col] : 0.0f;
    }
    __syncthreads();
    p.loadQuery(sums[0][p.at]);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kBytes; ++j) p.sum[j] = 0.0f;
    Word4* const keys = lds.keys[wave];
    while (t < to) {
        // The next tokens' keys are on their way while these are weighed, their values behind that.
        const int32_t next = t + kRound;
        if (next < to) place = p.find(next, lastBlock, pages);
        Word4 own[2][Tile<COLS>::kKeys];
        const Float4 scales[2] = {tile.kScale[0], tile.kScale[1]};
        if constexpr (Part<T, COLS>::kThroughLds) {
            p.putKeys(tile, keys);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) own[h][0] = tile.k[h];
        }
        if (next < to) p.loadKeys(tile, place, k, kScale);
        if constexpr (Part<T, COLS>::kThroughLds) p.getKeys(own, keys);
        float s[2][4];
        p.score(own, scales, s);
        p.add(tile, s, t, range.begin, to);
        if (next < to) p.loadValues(tile, place, v, vScale);
        t = next;
    }
    __syncthreads();   // the keys' LDS becomes the sums'
    // The waves' sums, each times what its maximum is below the largest by, are added in their order.
    p.total = sum4(p.total);
    if (p.group == 0) tops[wave][p.at] = p.top, totals[wave][p.at] = p.total;
    __syncthreads();
    float top = tops[0][p.at];
#pragma unroll
    for (int w = 1; w < kWavesPerBlock; ++w) top = fmaxf(top, tops[w][p.at]);
    const float below = top == -INFINITY ? 0.0f : top;
    const float factor = __builtin_amdgcn_exp2f(p.top - below) * (p.unit == 0.0f ? 0.0f : 1.0f);
    if (p.at < count) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < kBytes; ++j)
                sums[wave][p.at][kBytes * (4 * p.group + r) + j] =
                    ldexpf(p.sum[j][r] * factor, p.exponent - 15 - kByteExponent);
    }
    __syncthreads();
    const bool alone = range.parts == 1;
    for (int c = threadIdx.x; c < count * COLS; c += kBlock) {
        const int h = c / COLS, col = c % COLS;
        float most = tops[0][h], value = 0.0f, total = 0.0f;
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, tops[w][h]);
        const float least = most == -INFINITY ? 0.0f : most;
#pragma unroll
        for (int w = 0; w < kWavesPerBlock; ++w) {
            value += sums[w][h][col];
            total = fmaf(totals[w][h], __builtin_amdgcn_exp2f(tops[w][h] - least), total);
        }
        const int64_t row = b * a.heads + first + h;
        if (alone) {
            if (col < a.dim) storeOut<T>(a, b, first + h, col, value / total);
            if (col == 0 && a.lse) a.lse[row] = logSum(most, total);
        } else {
            const int64_t place = row * a.mostParts + part, places = (int64_t)a.batch * a.heads * a.mostParts;
            if (col < a.dim) a.parts[place * a.dim + col] = value;
            if (col == 0) {
                a.parts[places * a.dim + 2 * place] = most;
                a.parts[places * a.dim + 2 * place + 1] = total;
            }
        }
    }
}

// One workgroup a result: its parts' sums, each times what its maximum is below the largest by. The
// waves take the parts in turn.
template <typename T>
__global__ __launch_bounds__(kBlock) void joinKernel(AttendArgs a) {
    constexpr int kMost = RIDGE_ATTENTION_MAX_DIM / kWave;
    __shared__ float sums[kWavesPerBlock][RIDGE_ATTENTION_MAX_DIM];
    const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
    const uint32_t rows = (uint32_t)a.batch * a.heads;
    for (uint32_t row = blockIdx.x; row < rows; row += kMostBlocks) {
        const int64_t b = row / a.heads;
        const int head = row % a.heads;
        const Range range(uniformLoad(a.lengths + b), a.capacity, a.window);
        if (range.parts <= 1) continue;
        const int64_t place = (int64_t)row * a.mostParts, places = (int64_t)rows * a.mostParts;
        const float* const ends = a.parts + places * a.dim + 2 * place;
        const float top = lane < range.parts ? ends[2 * lane] : -INFINITY;
        float most = top;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        const float least = most == -INFINITY ? 0.0f : most;
        const float weight = lane < range.parts ? __builtin_amdgcn_exp2f(top - least) : 0.0f;
        const float total = ridge::sumOf<kWave>(lane < range.parts ? weight * ends[2 * lane + 1] : 0.0f);
        float x[kMost] = {};
        for (int p = wave; p < range.parts; p += kWavesPerBlock) {
            const float w = __shfl(weight, p);
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                const int col = lane + i * kWave;
                if (col < a.dim) x[i] = fmaf(w, a.parts[(place + p) * a.dim + col], x[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kMost; ++i) sums[wave][lane + i * kWave] = x[i];
        __syncthreads();
        const int col = threadIdx.x;
        float value = 0.0f;
#pragma unroll
        for (int w = 0; w < kWavesPerBlock; ++w) value += sums[w][col];
        if (col < a.dim) storeOut<T>(a, b, head, col, value / total);
        if (col == 0 && a.lse) a.lse[row] = logSum(most, total);
        __syncthreads();
    }
}

// The most parts that any sequence of these pages has.
int mostPartsOf(int64_t capacity, int64_t window) {
    const int64_t most = window && window + 15 < capacity ? window + 15 : capacity;
    return (int)std::clamp<int64_t>((most + kLeastPart - 1) / kLeastPart, 1, kMostParts);
}

// A grid has 65535 blocks at the most along its second and third directions.
constexpr int64_t kMostBatch = 65535;

template <typename T>
hipError_t launchTyped(AttendArgs a, hipStream_t stream) {
    const int64_t batch = a.batch;
    for (int64_t from = 0; from < batch; from += kMostBatch) {
        a.batch = (int32_t)std::min(batch - from, kMostBatch);
        const dim3 grid((unsigned)a.mostParts, (unsigned)(a.kvHeads * a.tiles), (unsigned)a.batch);
        hipError_t rc = a.dim <= 64    ? ridge::launchKernel(attendKernel<T, 64>, grid, kBlock, stream, a)
                        : a.dim <= 128 ? ridge::launchKernel(attendKernel<T, 128>, grid, kBlock, stream, a)
                                       : ridge::launchKernel(attendKernel<T, 256>, grid, kBlock, stream, a);
        if (rc == hipSuccess && a.mostParts > 1)
            rc = ridge::launchKernel(joinKernel<T>, (unsigned)std::min<int64_t>((int64_t)a.batch * a.heads, kMostBlocks), kBlock,
                                     stream, a);
        if (rc != hipSuccess) return rc;
        a.q = (const T*)a.q + kMostBatch * a.qToken, a.out = (T*)a.out + kMostBatch * a.outToken;
        a.pages += kMostBatch * a.pagesStride, a.lengths += kMostBatch;
        if (a.lse) a.lse += kMostBatch * a.heads;
    }
    return hipSuccess;
}

}  // namespace

extern "C" int64_t ridge_attention_workspace(int64_t batch, int32_t heads, int32_t kvHeads, int32_t dim, int64_t pagesEach,
                                             int32_t pageSize) {
    if (batch < 0 || kvHeads < 1 || heads < 0 || heads > 65535 || heads % kvHeads || dim < 1 ||
        dim > RIDGE_ATTENTION_MAX_DIM || pageSize < 16 || pageSize % 16 || pagesEach < 0 ||
        pagesEach > RIDGE_ATTENTION_MAX_SLOTS / pageSize)
        return -1;
    // Items, and their tiles of heads with them, are counted in 32 bits.
    if (batch > (INT32_MAX - 8 * 65536) / kMostParts / std::max(heads, 1)) return -1;
    const int parts = mostPartsOf(pagesEach * pageSize, 0);
    return parts == 1 ? 0 : batch * heads * parts * (dim + 2) * 4;
}

extern "C" int ridge_attention_attend(const ridge_attention_heads_t* q, const ridge_attention_cache_t* cache,
                                      const int32_t* pages, int64_t pagesStride, int64_t pagesEach, const int32_t* lengths,
                                      float scale, int64_t window, const ridge_attention_heads_t* out, float* lse, int type,
                                      int64_t batch, void* workspace, int64_t workspaceBytes, void* stream) {
    if (!ridge::isType(type) || !ridge::cacheFits(cache) || !ridge::headsFit(q, type, batch) ||
        !ridge::headsFit(out, type, batch) || q->heads != out->heads || !(std::fabs(scale) <= FLT_MAX / 2) || window < 0 ||
        pagesStride < 0)
        return hipErrorInvalidValue;
    const int64_t wanted =
        ridge_attention_workspace(batch, q->heads, cache->heads, cache->dim, pagesEach, cache->pageSize);
    if (wanted < 0) return hipErrorInvalidValue;
    if (batch == 0 || q->heads == 0) return hipSuccess;
    if (workspaceBytes < wanted || (wanted && !ridge::aligned(workspace, 16)) || (pagesEach && !ridge::aligned(pages, 4)) ||
        !ridge::aligned(lengths, 4) || (lse && !ridge::aligned(lse, 4)))
        return hipErrorInvalidValue;
    const int64_t capacity = pagesEach * cache->pageSize;
    AttendArgs a = {};
    a.k = cache->k, a.v = cache->v, a.kScale = cache->kScale, a.vScale = cache->vScale;
    a.q = q->at, a.out = out->at, a.lse = lse, a.pages = pages, a.lengths = lengths, a.parts = (float*)workspace;
    a.pageStride = cache->pageStride, a.headStride = cache->headStride, a.tokenStride = (uint32_t)cache->tokenStride;
    a.scalePage = cache->scalePage, a.scaleHead = cache->scaleHead;
    a.qToken = q->token, a.qHead = q->head, a.outToken = out->token, a.outHead = out->head, a.pagesStride = pagesStride;
    // Blocks are fewer than 2^27: with as many bits and the divisor's the quotient is exact.
    a.pageBlocks = (uint32_t)cache->pageSize / 16;
    a.pageShift = 27;
    while ((1u << (a.pageShift - 27)) < a.pageBlocks) ++a.pageShift;
    a.pageMagic = ((1ull << a.pageShift) + a.pageBlocks - 1) / a.pageBlocks;
    a.pages_ = (uint32_t)cache->pages, a.capacity = (int32_t)capacity;
    a.window = window >= capacity ? 0 : (int32_t)window, a.batch = (int32_t)batch, a.heads = q->heads;
    a.kvHeads = cache->heads, a.dim = cache->dim, a.tiles = (a.heads / a.kvHeads + kHeadTile - 1) / kHeadTile;
    a.mostParts = mostPartsOf(capacity, a.window);
    a.scale = (float)(scale * 1.4426950408889634);
    return ridge::typed(type, [&](auto element) { return launchTyped<decltype(element)>(a, (hipStream_t)stream); });
}
