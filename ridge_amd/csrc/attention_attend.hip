// attention_attend.hip -- the attention of each sequence's newest token over the 8-bit cache,
// for the C ABI in include/ridge_attention.h.
//
//   s_t = scale (q . k_t) kScale_t,  p_t = exp(s_t - max s),  out = sum p_t vScale_t v_t / sum p_t
//
// in one pass over the cache, whose bytes bound it: a workgroup takes one key head of a part of a
// sequence, its four waves 32 tokens at a time in turn, and each wave keeps the running maximum
// and sum of the softmax and the weighted values of up to 16 query heads that share the key head.
// Both products are matrix instructions (16 x 16 x 32) with sums in f32, and no operand of them is rounded:
// 8-bit whole numbers are exact in bf16 and f16. A query of f16 or bf16 is of its own type, one of f32 three
// parts of bf16, and so is p vScale, which has 24 bits and any size. In one or two parts of f16 (64 x 16384
// tokens 269 us for 275, in f32 286 for 305) a query's columns 2^-32 of its largest lost their bits,
// and values beside a far larger one, whatever its p.
//
// No value and no probability goes through LDS or moves between lanes (keys of more than 64 columns do, so
// that a load covers whole cache lines). The scores are computed transposed, keys as rows and heads as
// columns, so that a lane ends with 4 tokens of each 16 for one head; those are the k's that the
// second product, values as rows (transposed too) and heads as columns, wants from that lane, if the tokens
// of k = 8 g + 4 a + r are 16 a + 4 g + r. So a lane loads the values of those tokens and no others, and the
// running maximum's factor is its own head's everywhere.
//
// Work is shared evenly: the rounds (128 tokens) of all sequences' key heads, one behind the other, are
// cut into one equal share for each workgroup that runs at a time, whatever the sequences' lengths.
// A sequence's head that a share's border cuts has its pieces joined by a second launch.

#include "attention_common.hpp"

namespace {

using ridge::kBlock;
using ridge::kWave;
using ridge::kWavesPerBlock;
using ridge::uniformLoad;

typedef _Float16 Half8 __attribute__((ext_vector_type(8)));
typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
typedef __bf16 Brain8 __attribute__((ext_vector_type(8)));
typedef float Float4 __attribute__((ext_vector_type(4)));
typedef uint32_t Word4 __attribute__((ext_vector_type(4)));

constexpr int kHeadTile = 16;    // query heads of a workgroup
constexpr int kTile = 32;        // tokens of a wave at a time
constexpr int kRound = kTile * kWavesPerBlock;

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
    float* pieces;         // of cut heads: Piece::of
    int4* ends;            // of each key head and tile, or of each workgroup, whichever are fewer: what of it is to join
    int64_t pageStride, headStride, scalePage, scaleHead;
    int64_t qToken, qHead, outToken, outHead, pagesStride;
    uint32_t tokenStride, pageCount, pageBlocks;   // blocks: of 16 tokens, of a page
    uint32_t pageMagic, pageShift;                 // block / pageBlocks is 16 block times pageMagic, shifted by 32 + pageShift
    int32_t capacity, window, batch, heads, kvHeads, dim, tiles, tileHeads;   // tileHeads: the most of a tile
    int32_t shared, byHead;   // query heads of a key head; whether `ends` are the heads'
    float scale;           // times log2(e), as exponentials are powers of two, and times 2^-scaleExponent: 1 to 2
    int32_t scaleExponent;
};

// What a sequence's length says: its tokens [begin, end), and the rounds of a workgroup from `base` on
// that hold them.
struct Range {
    int32_t begin, end, base;
    uint32_t rounds;
    bool bad;
    __device__ Range(int32_t length, int32_t capacity, int32_t window) {
        bad = length < 0 || length > capacity;
        end = bad ? 0 : length;
        begin = window && end > window ? end - window : 0;
        base = begin / 16 * 16;
        rounds = (uint32_t)(end - base + kRound - 1) / kRound;
    }
    // One of no tokens has a round too: its results are written.
    __device__ uint32_t share() const { return max(rounds, 1u); }
};

// A cut head's piece that a workgroup has computed: its first one, or its last. For each query head the
// sums of its columns, and then what they and the sum of p are relative to, and this.
struct Piece {
    float* at;
    __device__ Piece(const AttendArgs& a, int index) : at(a.pieces + (int64_t)index * a.tileHeads * (a.dim + 2)) {}
    __device__ static int of(uint32_t block, bool first) { return 2 * block + !first; }
    __device__ float* sums(const AttendArgs& a, int head) const { return at + head * a.dim; }
    __device__ float* ends(const AttendArgs& a, int head) const { return at + a.tileHeads * a.dim + 2 * head; }
};

__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// Largest and sum over the four lanes of a head: this one, lane ^ 16, lane ^ 32 and both.
__device__ __forceinline__ float most4(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 2^n for n in -126 .. 127.
__device__ __forceinline__ float power2(int n) { return __int_as_float((n + 127) << 23); }
__device__ __forceinline__ int exponentOf(float v) { return (int)(__float_as_uint(v) >> 23 & 255) - 127; }

// Two f16 of the whole numbers in bytes `lo` of low and `hi` of high (biased by 128), times 2^-9, in 5
// instructions for 4 where bf16 takes 6:
// the byte as a f16 below the normal ones is its 2^-24th, which the product lifts and the sum unbiases.
__device__ __forceinline__ Half2 halves(uint32_t high, uint32_t low, int hi, int lo) {
    const uint32_t both = __builtin_amdgcn_perm(high, low, 0x0c000c00u | (uint32_t)(4 + hi) << 16 | (uint32_t)lo);
    const Half2 lift = {(_Float16)32768.0f, (_Float16)32768.0f}, bias = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_elementwise_fma(__builtin_bit_cast(Half2, both), lift, bias);
}

__device__ __forceinline__ Half8 join(Half2 a, Half2 b, Half2 c, Half2 d) {
    return Half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The upper halves of two floats: as bf16 they are the floats but for their last 16 bits.
__device__ __forceinline__ uint32_t tops(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// Two bf16 of the whole numbers in bytes i of a and j of b.
__device__ __forceinline__ uint32_t wholes(uint32_t a, int i, uint32_t b, int j) {
    return tops((float)(int8_t)(a >> 8 * i), (float)(int8_t)(b >> 8 * j));
}
// What a float's upper half leaves: exact, so that three halves in turn are all of its 24 bits. (Not
// joined with a product that the float is: that would be the remainder of another number.)
__device__ __forceinline__ float restOf(float v) {
#pragma clang fp contract(off)
    return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}

// Where a wave's 32 tokens are: two blocks of 16, each in one page. The same for all its lanes.
struct Blocks {
    uint32_t page[2], in[2];   // the cache's page, and the first token in it
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

// Loads past the caches (bit 1): a key or value is read once by a workgroup, and its cache line whole by one
// load. (More than 16 query heads of a key head are several workgroups' work, each of which reads it.)
constexpr int kStream = 2;

// Memory from `at` on, for offsets of 32 bits: no lane computes an address.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t memory(const void* at) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, 0xffffffff, 0x00027000);
}

template <int n>
__device__ __forceinline__ void loadWords(uint32_t (&to)[n], __amdgpu_buffer_rsrc_t from, uint32_t lane, uint32_t all) {
    if constexpr (n == 1) {
        to[0] = __builtin_amdgcn_raw_buffer_load_b32(from, lane, all, kStream);
    } else if constexpr (n == 2) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(from, lane, all, kStream);
        to[0] = w[0], to[1] = w[1];
    } else {
        const auto w = __builtin_amdgcn_raw_buffer_load_b128(from, lane, all, kStream);
#pragma unroll
        for (int i = 0; i < n; ++i) to[i] = w[i];
    }
}

// One wave's tokens of a part of a sequence, for 16 query heads. Probabilities are relative,
// 2^(score - from), 1 for the largest score; the sum of them goes by nothing else. The sums of values are
// of scales times 2^-exponent, which is 0 but where the largest scale so far is far from one:
// they have room for 2^31 tokens of any scale, and the three parts of p times a scale of FLT_MIN are
// normal numbers as well.
template <typename T, int COLS>
struct Part {
    static constexpr int kKeys = Tile<COLS>::kKeys;
    static constexpr int kBytes = COLS / 16;       // of a value that a lane loads, and sums of 16 columns that it holds 4 of
    static constexpr bool kHalf = std::is_same_v<T, _Float16>;
    static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;   // of a query: bf16, or f16 where it is that
    static constexpr int kByteExponent = kHalf ? -9 : 0;    // of keys
    static constexpr int kSmall = -40, kLarge = 39;                    // exponents,
    static constexpr float kMostSmall = 0x1p-40f, kMostPlain = 0x1p88f;   // of scales up to this, and past that
    typedef typename ridge::Memory<T, 8>::Vec Vec;

    const AttendArgs& a;
    const int lane, at = lane % 16, group = lane / 16;
    Word4 q[kParts][kKeys][2];
    float qScale;                                  // of scores, to powers of two
    Float4 sum[kBytes];                            // of value columns kBytes (4 group + r) + i, for head `at`
    float top, from, total;                        // the largest score, and this lane's part of the sum of p
    float most;                                    // of scales that the exponent is for
    int exponent;                                  // of the sums; the same for all lanes

    __device__ Part(const AttendArgs& a, int lane) : a(a), lane(lane) {}

    __device__ __forceinline__ void clear() {
        top = from = -INFINITY, total = 0.0f, exponent = kSmall, most = kMostSmall;
#pragma unroll
        for (int j = 0; j < kBytes; ++j) sum[j] = 0.0f;
    }

    // The query's columns that this lane multiplies: 8 from 64 i + 16 group + 8 j on, of head `at`.
    struct Query {
        Vec x[kKeys][2];
    };
    __device__ __forceinline__ void loadQuery(Query& query, const T* row) const {
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = 64 * i + 16 * group + 8 * j;
                if (a.dim % 8 == 0) {
                    query.x[i][j] = *(const Vec*)(row + (col < a.dim ? col : 0));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const T x = row[min(col + e, a.dim - 1)];
                        query.x[i][j][e] = col + e < a.dim ? x : (T)0;
                    }
                }
            }
    }

    // Its fragments, in bf16 or f16 without a rounding: the query times a power of two that makes the largest
    // column of a bf16 or f32 head about 2^14, and that keeps qScale a normal number, whatever the scale
    // (of f16 it is 1 but for scales below 2^-135, beside which small columns lose bits). A
    // negative scale turns the query, so that the largest score has the largest p.
    __device__ __forceinline__ void setQuery(const Query& query) {
        float x[kKeys][2][8];
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool has = 64 * i + 16 * group + 8 * j < a.dim;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][j][e] = has ? (float)query.x[i][j][e] : 0.0f;
            }
        int down = 0;
        if constexpr (!kHalf) {
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < kKeys; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[i][j][e]));
            const int exponent = exponentOf(most4(most));
            down = max(-96, exponent - 14);
            down = max(min(down, 126 - a.scaleExponent), exponent - 104);
        }
        down = max(down, -126 + kByteExponent - a.scaleExponent);
        // Never 0, as a masked score of -inf stays one: of a scale of 0 the query is.
        qScale = fmaxf(ldexpf(fabsf(a.scale), a.scaleExponent + down - kByteExponent), FLT_MIN);
        const float up = a.scale == 0.0f ? 0.0f : copysignf(power2(-down), a.scale);
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    float u = x[i][j][e] * up, w = x[i][j][e + 1] * up;
                    if constexpr (kHalf) {
                        q[0][i][j][e / 2] = __builtin_bit_cast(uint32_t, Half2{(_Float16)u, (_Float16)w});
                    } else {
#pragma unroll
                        for (int n = 0; n < kParts; ++n) {
                            q[n][i][j][e / 2] = tops(u, w);
                            u = restOf(u), w = restOf(w);
                        }
                    }
                }
    }

    // The blocks of the 32 tokens from t on; those behind `lastBlock` are that one, which is masked.
    __device__ __forceinline__ Blocks find(int32_t t, uint32_t lastBlock, const int32_t* pages) const {
        Blocks blocks;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t block = min((uint32_t)t / 16 + b, lastBlock);
            const uint32_t page = __umulhi(block * 16, a.pageMagic) >> a.pageShift;
            blocks.page[b] = uniformLoad(pages + page);
            blocks.in[b] = (block - page * a.pageBlocks) * 16;
        }
        return blocks;
    }
    // A page outside the cache is read as its first one.
    __device__ __forceinline__ bool there(const Blocks& blocks, int b) const { return blocks.page[b] < a.pageCount; }
    __device__ __forceinline__ int64_t rowsOf(const Blocks& blocks, int b) const {
        return (there(blocks, b) ? blocks.page[b] * a.pageStride : 0) + (int64_t)blocks.in[b] * a.tokenStride;
    }
    __device__ __forceinline__ const float* scalesOf(const float* scales, const Blocks& blocks, int b) const {
        return scales + (there(blocks, b) ? blocks.page[b] * a.scalePage : 0) + blocks.in[b];
    }
    __device__ __forceinline__ uint32_t within(uint32_t col) const { return col < (uint32_t)((a.dim + 15) & ~15) ? col : 0; }

    // Whole keys, a chunk a lane: 64 / kChunks of them at once, which are whole cache lines. Of 64
    // columns a lane's chunk is the one that its scores take. A page outside the cache makes NaNs.
    __device__ __forceinline__ void loadKeys(Tile<COLS>& tile, const Blocks& blocks, const int8_t* k, const float* scales) const {
        constexpr int kChunks = Tile<COLS>::kChunks, kRows = kWave / kChunks, kEach = Tile<COLS>::kLoads / 2;
        const uint32_t row = kThroughLds ? lane / kChunks : at, chunk = 16 * (kThroughLds ? lane % kChunks : group);
        const uint32_t offset = row * a.tokenStride + within(chunk);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const auto from = memory(k + rowsOf(blocks, b));
#pragma unroll
            for (int n = 0; n < kEach; ++n)
                tile.k[b * kEach + n] = __builtin_bit_cast(
                    Word4, __builtin_amdgcn_raw_buffer_load_b128(from, offset, n * kRows * a.tokenStride, kStream));
            tile.kScale[b] = *(const Float4*)(scalesOf(scales, blocks, b) + 4 * group);
            if (!there(blocks, b)) tile.kScale[b] = NAN;
        }
    }

    __device__ __forceinline__ void loadValues(Tile<COLS>& tile, const Blocks& blocks, const int8_t* v, const float* scales) const {
        const uint32_t offset = 4 * group * a.tokenStride + within(kBytes * at);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const auto from = memory(v + rowsOf(blocks, b));
#pragma unroll
            for (int r = 0; r < 4; ++r) loadWords(tile.v[b][r], from, offset, r * a.tokenStride);
            tile.vScale[b] = *(const Float4*)(scalesOf(scales, blocks, b) + 4 * group);
        }
    }

    // Keys go through LDS of the wave's own, from whole rows to the 16 bytes of a token that a lane's
    // scores take; chunks of a row are swapped so that neither side meets another lane's bank. A wave's
    // accesses of LDS are done in their order, so the lanes wait for nothing: the compiler alone is told, before
    // a lane reads what another one wrote and before it writes where another one read.
    static constexpr bool kThroughLds = COLS > 64;
    __device__ static __forceinline__ void handOver() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
    }
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

    // The scores of 32 tokens, still to be multiplied by qScale.
    __device__ __forceinline__ void score(const Word4 (&k)[2][kKeys], const Float4 (&kScale)[2], float (&s)[2][4]) const {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            Float4 score = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (kHalf) {
                        const uint32_t x = k[b][i][2 * j] ^ 0x80808080u, y = k[b][i][2 * j + 1] ^ 0x80808080u;
                        const Half8 keys = join(halves(x, x, 1, 0), halves(x, x, 3, 2), halves(y, y, 1, 0), halves(y, y, 3, 2));
                        score = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, __builtin_bit_cast(Half8, q[0][i][j]), score, 0, 0, 0);
                    } else {
                        const uint32_t x = k[b][i][2 * j], y = k[b][i][2 * j + 1];
                        const Word4 keys = {wholes(x, 0, x, 1), wholes(x, 2, x, 3), wholes(y, 0, y, 1), wholes(y, 2, y, 3)};
#pragma unroll
                        for (int n = 0; n < kParts; ++n)
                            score = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Brain8, keys),
                                                                            __builtin_bit_cast(Brain8, q[n][i][j]), score, 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[b][r] = score[r] * kScale[b][r];
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
        float highest = s[0][0], scale = fabsf(tile.vScale[0][0]);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) highest = fmaxf(highest, s[b][r]), scale = fmaxf(scale, fabsf(tile.vScale[b][r]));
        // Few tiles have a new maximum or a scale that wants another exponent: the sums are rescaled in a branch.
        if (__builtin_amdgcn_ballot_w64(highest > top || scale > most)) {
            const int before = exponent;
            if (__builtin_amdgcn_ballot_w64(scale > most)) {   // the 16 heads' lanes have the same tokens
                const bool large = __builtin_amdgcn_ballot_w64(scale > kMostPlain);
                exponent = large ? kLarge : 0, most = large ? INFINITY : kMostPlain;
            }
            const bool none = top == -INFINITY;
            top = fmaxf(top, most4(highest));
            const float now = top == -INFINITY ? -INFINITY : top * qScale;
            const float factor = none ? 0.0f : __builtin_amdgcn_exp2f(from - now), down = factor * power2(before - exponent);
            from = now;
            total *= factor;
#pragma unroll
            for (int i = 0; i < kBytes; ++i) sum[i] *= down;
        }
        if (exponent) {
            const float down = power2(-exponent);
#pragma unroll
            for (int b = 0; b < 2; ++b) tile.vScale[b] *= down;
        }
        const float least = top == -INFINITY ? 0.0f : from;
        Word4 high, middle, low;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                float weight[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[b][r + n], qScale, -least));
                    total += p;
                    weight[n] = p * tile.vScale[b][r + n];
                }
                const int at = 2 * b + r / 2;
                high[at] = tops(weight[0], weight[1]);
                for (float& w : weight) w = restOf(w);
                middle[at] = tops(weight[0], weight[1]);
                for (float& w : weight) w = restOf(w);
                low[at] = tops(weight[0], weight[1]);
            }
#pragma unroll
        for (int i = 0; i < kBytes; ++i) {
            auto pair = [&](int b, int r) { return wholes(tile.v[b][r][i / 4], i % 4, tile.v[b][r + 1][i / 4], i % 4); };
            const Word4 values = {pair(0, 0), pair(0, 2), pair(1, 0), pair(1, 2)};
            for (const Word4& part : {high, middle, low})
                sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Brain8, values),
                                                                 __builtin_bit_cast(Brain8, part), sum[i], 0, 0, 0);
        }
    }
};

// The launch's arguments, read again, so that what follows holds no registers before it.
__device__ __forceinline__ const AttendArgs& again() {
    typedef const __attribute__((address_space(4))) AttendArgs Constant;
    uintptr_t at = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const AttendArgs*)(Constant*)at;
}

// Result (b, head): 16 bits or f32 of `value` columns.
template <typename T>
__device__ __forceinline__ void storeOut(const AttendArgs& a, int64_t b, int head, int col, float value) {
    ((T*)a.out)[b * a.outToken + head * a.outHead + col] = (T)value;
}

__device__ __forceinline__ float logSum(float from, float total) {
    return (from + __builtin_amdgcn_logf(total)) * 0.69314718055994531f;
}

// Waves of a SIMD, by what their registers leave room for.
template <typename T>
constexpr int wavesOf(int cols) {
    return cols == 64 ? 4 : cols == 128 ? (sizeof(T) == 4 ? 2 : 3) : sizeof(T) == 4 ? 1 : 2;
}

// What a workgroup computes: rounds that follow each other, in the order of sequences and heads.
struct Share {
    uint32_t size, first, left;   // rounds of every workgroup, before this one's, and of it
    int32_t b, y;                 // where they begin: the sequence, the key head and 16 of its query heads,
    uint32_t round;               // and the round
    int32_t length;               // of that sequence
};

// An even share of all rounds, found from the sequences' lengths, 64 at a time.
__device__ __forceinline__ Share shareOf(const AttendArgs& a, uint32_t block, uint32_t blocks) {
    const int lane = threadIdx.x % kWave, heads = a.kvHeads * a.tiles;
    int32_t length = 0;
    auto load = [&](int from) {
        if (from + lane >= a.batch) return 0u;
        length = a.lengths[from + lane];
        return Range(length, a.capacity, a.window).share();
    };
    auto sum = [&](uint32_t v) {   // of this lane and those before it: in rows of 16 lanes, then rows
        auto from = [&](auto control, auto rows) {
            return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(control)::value, decltype(rows)::value, 15, false);
        };
        typedef std::integral_constant<int, 15> All;
        v += from(std::integral_constant<int, 0x111>(), All());   // 1, 2, 4 and 8 lanes before
        v += from(std::integral_constant<int, 0x112>(), All());
        v += from(std::integral_constant<int, 0x114>(), All());
        v += from(std::integral_constant<int, 0x118>(), All());
        v += from(std::integral_constant<int, 0x142>(), std::integral_constant<int, 10>());   // the row's last before
        v += from(std::integral_constant<int, 0x143>(), std::integral_constant<int, 12>());   // lane 31
        return v;
    };
    auto lastOf = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1); };
    uint32_t total = 0, before = sum(load(0));
    for (int from = 0;;) {
        total += lastOf(before);
        if ((from += kWave) >= a.batch) break;
        before = sum(load(from));
    }
    total *= heads;
    Share share = {};
    share.size = (total + blocks - 1) / blocks;
    share.first = block * share.size;
    if (share.first >= total) return share;
    share.left = min(share.size, total - share.first);
    const uint32_t sought = share.first / heads;
    uint32_t passed = 0;
    int from = 0;
    if (a.batch > kWave) before = sum(load(0));
    while (true) {
        const uint32_t here = lastOf(before);
        if (passed + here > sought) break;
        passed += here;
        from += kWave;
        before = sum(load(from));
    }
    const int behind = uniform(__builtin_ctzll(__builtin_amdgcn_ballot_w64(passed + before > sought)));
    if (behind) passed += (uint32_t)__builtin_amdgcn_readlane((int)before, behind - 1);
    share.b = from + behind;
    const uint32_t in = share.first - passed * heads;
    share.length = __builtin_amdgcn_readlane(length, behind);
    const uint32_t each = Range(share.length, a.capacity, a.window).share();
    share.y = uniform(in / each);
    share.round = uniform(in - share.y * each);
    return share;
}

// EVEN: workgroups share all rounds; else each has one sequence's head.
template <typename T, int COLS, bool EVEN>
__global__ __launch_bounds__(kBlock, wavesOf<T>(COLS)) void attendKernel(AttendArgs args) {
    constexpr int kBytes = COLS / 16;
    __shared__ float froms[kWavesPerBlock][kHeadTile], totals[kWavesPerBlock][kHeadTile];
    __shared__ union {
        float sums[kWavesPerBlock][kHeadTile][COLS + 4];
        Word4 keys[kWavesPerBlock][kTile * Tile<COLS>::kChunks];
    } lds;
    const uint32_t block = EVEN ? blockIdx.x : 0;
    Share share = {};
    if constexpr (EVEN) {
        share = shareOf(again(), block, gridDim.x);
        if (share.left == 0) {
            if (threadIdx.x == 0 && !again().byHead) again().ends[block] = {1, 0, 0, 0};
            return;
        }
    } else {
        share.left = 1, share.b = blockIdx.z, share.y = blockIdx.y;
        share.length = uniformLoad(args.lengths + share.b);
    }
    bool isFirst = true;
    do {
        AttendArgs const& a = EVEN ? again() : args;
        int thread = threadIdx.x;
        if constexpr (EVEN) asm volatile("" : "+v"(thread));   // so that nothing is held from one head to the next
        const int wave = uniform(thread / kWave), y = share.y, kvHead = a.tiles == 1 ? y : y / a.tiles;
        const int tile16 = y - kvHead * a.tiles, first = kvHead * a.shared + tile16 * kHeadTile;
        const int count = min(kHeadTile, a.shared - tile16 * kHeadTile);
        const int64_t b = share.b;
        Part<T, COLS> p(a, thread % kWave);
        const Range range(share.length, a.capacity, a.window);
        const uint32_t rounds = EVEN ? min(share.left, range.share() - share.round) : range.share();
        const bool cut = EVEN && rounds != range.share(), ending = share.round + rounds == range.share();
        int32_t t = range.base + (int32_t)share.round * kRound;
        const int32_t to = (int32_t)min((int64_t)range.end, t + (int64_t)rounds * kRound);
        const uint32_t lastBlock = (uint32_t)max(to - 1, 0) / 16;
        t += wave * kTile;
        // Pages are looked up two tiles ahead, keys loaded one ahead, and values behind their predecessors.
        const int32_t* const pages = a.pages + b * a.pagesStride;
        Blocks blocks = {};
        if (range.rounds) blocks = p.find(t, lastBlock, pages);
        typename Part<T, COLS>::Query query;
        p.loadQuery(query, (const T*)a.q + b * a.qToken + (first + min(p.at, count - 1)) * a.qHead);
        if (EVEN && thread == 0 && (a.byHead ? ending : isFirst)) {
            // A head's pieces: where it begins, its workgroup's first or last one, and from there on first ones.
            int4 ends = {1, 0, 0, 0};
            if (share.round && ending) {
                const uint32_t begins = share.first - share.round, in = begins / share.size;
                ends = {Piece::of(in, begins == in * share.size), Piece::of(block, true), (int)(b * a.heads + first), count};
            }
            a.ends[a.byHead ? b * a.kvHeads * a.tiles + y : block] = ends;
        }
        const int piece = EVEN ? Piece::of(block, isFirst) : 0;
        isFirst = false;
        share.left -= EVEN ? rounds : 1;
        share.round = 0;
        if (++share.y == a.kvHeads * a.tiles) {
            share.y = 0, ++share.b;
            if (EVEN && share.left) share.length = uniformLoad(a.lengths + share.b);
        }
        if (range.rounds == 0) {   // no tokens, or a length outside the cache
            for (int c = thread; c < count * a.dim; c += kBlock)
                storeOut<T>(a, b, first + c / a.dim, c % a.dim, range.bad ? NAN : 0.0f);
            if (a.lse && thread < count) a.lse[b * a.heads + first + thread] = range.bad ? NAN : -INFINITY;
            continue;
        }
        const int8_t *const k = a.k + kvHead * a.headStride, *const v = a.v + kvHead * a.headStride;
        const float *const kScale = a.kScale + kvHead * a.scaleHead, *const vScale = a.vScale + kvHead * a.scaleHead;
        Tile<COLS> tile = {};
        if (t < to) {
            p.loadKeys(tile, blocks, k, kScale);
            p.loadValues(tile, blocks, v, vScale);
        }
        blocks = p.find(t + kRound, lastBlock, pages);
        p.setQuery(query);
        Word4* const keys = lds.keys[wave];
        p.clear();
        while (t < to) {
            const int32_t next = t + kRound;
            Word4 own[2][Tile<COLS>::kKeys];
            const Float4 scales[2] = {tile.kScale[0], tile.kScale[1]};
            if constexpr (Part<T, COLS>::kThroughLds) {
                p.putKeys(tile, keys);
                p.handOver();
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) own[h][0] = tile.k[h];
            }
            const Blocks ahead = p.find(next + kRound, lastBlock, pages);
            if (next < to) p.loadKeys(tile, blocks, k, kScale);
            if constexpr (Part<T, COLS>::kThroughLds) {
                p.getKeys(own, keys);
                p.handOver();
            }
            float s[2][4];
            p.score(own, scales, s);
            p.add(tile, s, t, range.begin, to);
            if (next < to) p.loadValues(tile, blocks, v, vScale);
            blocks = ahead;
            t = next;
        }
        // The waves' sums, from the largest `from` on, are added in their order.
        // With the exponent in both, the sum of p is relative to what the sums are. (Where one wave has scales up
        // to 2^-40 alone and another one scales past 2^88, a p below 2^-47 of the largest may so count nothing.)
        p.total = sum4(p.total) * power2(-p.exponent);
        p.from += (float)p.exponent;
        if (p.group == 0) froms[wave][p.at] = p.from, totals[wave][p.at] = p.total;
        __syncthreads();   // and the keys' LDS becomes the sums'
        float most = froms[0][p.at];
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, froms[w][p.at]);
        const float factor = __builtin_amdgcn_exp2f(p.from - (most == -INFINITY ? 0.0f : most));
        if (p.at < count) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < kBytes; ++j) lds.sums[wave][p.at][kBytes * (4 * p.group + r) + j] = p.sum[j][r] * factor;
        }
        __syncthreads();
        const AttendArgs& e = again();
        for (int c = thread; c < count * COLS; c += kBlock) {
            const int h = c / COLS, col = c % COLS;
            float most = froms[0][h], value = 0.0f, total = 0.0f;
#pragma unroll
            for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, froms[w][h]);
#pragma unroll
            for (int w = 0; w < kWavesPerBlock; ++w) {
                value += lds.sums[w][h][col];
                total = fmaf(totals[w][h], __builtin_amdgcn_exp2f(froms[w][h] - (most == -INFINITY ? 0.0f : most)), total);
            }
            const int64_t row = b * e.heads + first + h;
            if (!cut) {
                if (col < e.dim) storeOut<T>(e, b, first + h, col, value / total);
                if (col == 0 && e.lse) e.lse[row] = logSum(most, total);
            } else {
                const Piece to(e, piece);
                if (col < e.dim) to.sums(e, h)[col] = value;
                if (col == 0) to.ends(e, h)[0] = most, to.ends(e, h)[1] = total;
            }
        }
        if constexpr (EVEN) __syncthreads();   // before the next head's keys
    } while (EVEN && share.left > 0);
}

// One workgroup for each query head of each key head that has pieces. The waves take them in turn, each
// with its own running maximum; what all lanes share is read past the vector unit.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void joinKernel(AttendArgs a) {
    constexpr int kMost = RIDGE_ATTENTION_MAX_DIM / kWave, kAtOnce = 4;
    __shared__ float sums[WAVES][RIDGE_ATTENTION_MAX_DIM], froms[WAVES], totals[WAVES];
    const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), h = blockIdx.y;
    const int32_t* const ends = (const int32_t*)(a.ends + blockIdx.x);
    const int begin = uniformLoad(ends), last = uniformLoad(ends + 1), row = uniformLoad(ends + 2) + h;
    if (begin > last || h >= uniformLoad(ends + 3)) return;
    const int block = begin / 2, pieces = last / 2 - block + 1;
    float x[kMost] = {}, top = -INFINITY, total = 0.0f;
    for (int i = wave; i < pieces; i += WAVES * kAtOnce) {
        float part[kAtOnce][kMost], from[kAtOnce], sum[kAtOnce], now = top;
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const int p = i + n * WAVES;
            from[n] = -INFINITY, sum[n] = 0.0f;
#pragma unroll
            for (int j = 0; j < kMost; ++j) part[n][j] = 0.0f;
            if (p < pieces) {
                const Piece piece(a, p == 0 ? begin : 2 * (block + p));
                from[n] = __int_as_float(uniformLoad((const int32_t*)piece.ends(a, h)));
                sum[n] = __int_as_float(uniformLoad((const int32_t*)piece.ends(a, h) + 1));
#pragma unroll
                for (int j = 0; j < kMost; ++j)
                    if (j * kWave < a.dim) part[n][j] = piece.sums(a, h)[min(lane + j * kWave, a.dim - 1)];
            }
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) now = fmaxf(now, from[n]);
        const float least = now == -INFINITY ? 0.0f : now, keep = __builtin_amdgcn_exp2f(top - least);
        top = now;
        total *= keep;
#pragma unroll
        for (int j = 0; j < kMost; ++j) x[j] *= keep;
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const float weight = __builtin_amdgcn_exp2f(from[n] - least);
            total = fmaf(weight, sum[n], total);
#pragma unroll
            for (int j = 0; j < kMost; ++j) x[j] = fmaf(weight, part[n][j], x[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < kMost; ++j) sums[wave][lane + j * kWave] = x[j];
    if (lane == 0) froms[wave] = top, totals[wave] = total;
    __syncthreads();
    const int col = threadIdx.x;
    if (col >= a.dim) return;
    float most = froms[0], value = 0.0f, all = 0.0f;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) most = fmaxf(most, froms[w]);
    const float least = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float weight = __builtin_amdgcn_exp2f(froms[w] - least);
        value = fmaf(weight, sums[w][col], value);
        all = fmaf(weight, totals[w], all);
    }
    storeOut<T>(a, row / a.heads, row % a.heads, col, value / all);
    if (col == 0 && a.lse) a.lse[row] = logSum(most, all);
}

// Workgroups that run at a time, by columns and the type's bytes.
int residentOf(int dim, size_t bytes) {
    const int cols = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    return 256 * (bytes == 4 ? wavesOf<float>(cols) : wavesOf<_Float16>(cols)) * 4 / kWavesPerBlock;
}

// Whether each key head (and tile) has a workgroup, which needs no second launch, instead of an even
// share of all rounds. us of sequences of one length, each their own | shared, 8 key heads of 128:
//   1 x 512 10.1 | 9.7, 1 x 768 13 | 10, 16 x 1024 20 | 15, 32 x 1024 22 | 25, 64 x 1024 28 | 37,
//   32 x 2048 38 | 37, 64 x 2048 50 | 58, 128 x 4096 185 | 193;
// of lengths from a quarter on: 32 x 1024 21 | 21, 64 x 2048 40 | 46, 128 x 4096 140 | 130. What one long
// sequence among short ones costs alone (2.2 us for each 128 tokens) bounds the lengths. Up to 512 tokens a
// result depends on no other sequence.
bool eachItsOwn(int64_t batch, int64_t heads, int64_t capacity) {
    return capacity <= 512 || (capacity <= 1024 && batch * heads >= 256) || (capacity <= 2048 && batch * heads >= 512);
}

// A grid has 65535 blocks at the most along its second and third directions.
constexpr int64_t kMostBatch = 65535;

template <typename T>
hipError_t launchTyped(AttendArgs a, hipStream_t stream) {
    const int64_t batch = a.batch;
    const bool even = a.pieces != nullptr;
    const unsigned blocks = residentOf(a.dim, sizeof(T));
    if (even) {   // at a multiple of 16 bytes behind the pieces
        a.ends = (int4*)(a.pieces + ((int64_t)2 * blocks * a.tileHeads * (a.dim + 2) + 3) / 4 * 4);
    }
    for (int64_t from = 0; from < batch; from += kMostBatch) {
        a.batch = (int32_t)std::min(batch - from, kMostBatch);
        const int64_t heads = (int64_t)a.batch * a.kvHeads * a.tiles;
        a.byHead = heads < blocks;
        const dim3 grid = even ? dim3(blocks) : dim3(1, (unsigned)(a.kvHeads * a.tiles), (unsigned)a.batch);
        auto launch = [&](auto direct, auto evenly) { return ridge::launchKernel(even ? evenly : direct, grid, kBlock, stream, a); };
        hipError_t rc = a.dim <= 64    ? launch(attendKernel<T, 64, false>, attendKernel<T, 64, true>)
                        : a.dim <= 128 ? launch(attendKernel<T, 128, false>, attendKernel<T, 128, true>)
                                       : launch(attendKernel<T, 256, false>, attendKernel<T, 256, true>);
        if (rc == hipSuccess && even) {
            // Few heads have many pieces each: us of 8 heads of 93, 4 waves | 16: 9.3 | 4.4.
            const bool few = heads * a.tileHeads <= 256;
            const dim3 each((unsigned)std::min<int64_t>(heads, blocks), (unsigned)a.tileHeads);
            rc = few ? ridge::launchKernel(joinKernel<T, 16>, each, 16 * kWave, stream, a)
                     : ridge::launchKernel(joinKernel<T, 4>, each, 4 * kWave, stream, a);
        }
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
    // Rounds of all heads are counted in 32 bits.
    const int64_t capacity = pagesEach * pageSize, rounds = capacity / kRound + 2;
    if (batch > INT32_MAX / std::max(heads, 1) / rounds) return -1;
    const int64_t shared = heads / kvHeads, tiles = (shared + kHeadTile - 1) / kHeadTile;
    if (eachItsOwn(batch, kvHeads * tiles, capacity)) return 0;
    // Two pieces of each workgroup, and what ends in it.
    const int64_t blocks = residentOf(dim, 2), tileHeads = std::clamp<int64_t>(shared, 1, kHeadTile);
    return blocks * (2 * tileHeads * (dim + 2) * 4 + 16);
}

extern "C" int ridge_attention_attend(const ridge_attention_heads_t* q, const ridge_attention_cache_t* cache,
                                      const int32_t* pages, int64_t pagesStride, int64_t pagesEach, const int32_t* lengths,
                                      float scale, int64_t window, const ridge_attention_heads_t* out, float* lse, int type,
                                      int64_t batch, void* workspace, int64_t workspaceBytes, void* stream) {
    if (!ridge::isType(type) || !ridge::cacheFits(cache) || !ridge::headsFit(q, type, batch) ||
        !ridge::headsFit(out, type, batch) || q->heads != out->heads || !(std::fabs(scale) <= FLT_MAX / 2) || window < 0 ||
        pagesStride < 0 || (type == RIDGE_F16 && std::fabs(scale) > 0x1p118f))
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
    a.q = q->at, a.out = out->at, a.lse = lse, a.pages = pages, a.lengths = lengths, a.pieces = nullptr;
    a.pageStride = cache->pageStride, a.headStride = cache->headStride, a.tokenStride = (uint32_t)cache->tokenStride;
    a.scalePage = cache->scalePage, a.scaleHead = cache->scaleHead;
    a.qToken = q->token, a.qHead = q->head, a.outToken = out->token, a.outHead = out->head, a.pagesStride = pagesStride;
    // Blocks are fewer than 2^27: with 28 bits more than the divisor's the quotient is exact.
    a.pageBlocks = (uint32_t)cache->pageSize / 16;
    while ((1u << a.pageShift) < a.pageBlocks) ++a.pageShift;
    a.pageMagic = (uint32_t)(((1ull << (28 + a.pageShift)) + a.pageBlocks - 1) / a.pageBlocks);
    a.pageCount = (uint32_t)cache->pages, a.capacity = (int32_t)capacity;
    a.window = window >= capacity ? 0 : (int32_t)window, a.batch = (int32_t)batch, a.heads = q->heads;
    a.kvHeads = cache->heads, a.dim = cache->dim, a.tiles = (a.heads / a.kvHeads + kHeadTile - 1) / kHeadTile;
    a.shared = a.heads / a.kvHeads, a.tileHeads = std::min(kHeadTile, a.shared);
    const int64_t longest = a.window ? std::min(capacity, (int64_t)a.window + 15) : capacity;   // whole blocks of 16
    if (!eachItsOwn(batch, (int64_t)a.kvHeads * a.tiles, longest)) a.pieces = (float*)workspace;
    const double wide = scale * 1.4426950408889634;
    a.scaleExponent = scale == 0.0f ? 0 : std::ilogb(wide), a.scale = (float)std::scalbn(wide, -a.scaleExponent);
    return ridge::typed(type, [&](auto element) { return launchTyped<decltype(element)>(a, (hipStream_t)stream); });
}
