// int8_gemm.hpp -- matrix product of 8-bit rows for gfx950 (MI355X): 32-bit integer sums
// on the matrix pipes, one scale for each row of A and of B in the epilogue.
//
//   C[m, n] = (sum over k of A[m, k] B[n, k]) scaleA[m] scaleB[n] + bias[n]
//
// A (M x K) and B (N x K) both have k along memory. v_mfma_i32_16x16x64_i8 takes 16
// consecutive k of one row a lane (16 bytes, lane group g = lane / 16 holding k = 16 g ..
// 16 g + 15), which is byte for byte the operand layout of the FP16 instruction of half
// the K: a tile's rows are loaded straight into LDS in 16-byte chunks, swizzled
// (swizzleRows), and both fragments are single ds_read_b128s. With B's fragment in the
// first operand lane l holds C[m0 + l % 16][n0 + 4 (l / 16) + r] in element r.
//
// Any M, N and K: a row past the end of A or B is replaced by the last one (its products
// are not stored), and of the last K tile's chunks those past the end by the last chunk;
// what A's fragments hold behind K is cleared before it is multiplied, so what is read of
// B there does not matter.
#pragma once

#include "gemm_mfma.hpp"

namespace ridge {

typedef int int4_t __attribute__((ext_vector_type(4)));

constexpr int kInt8MfmaK = 64;   // k of one instruction

// A launch's arguments. They are written to device memory before it, 64 bytes at a time:
// a second write would cost up to 0.5 us of the host's time, which is what the shortest
// products wait for. So where sizes allow (int8ArgsFit) they are packed into one: strides, multiples
// of 16 below 2^23, in 19 bits each, K in 17, M and N in 16, ldc in 32.
struct Int8Operands {
    const int8_t* A;
    const int8_t* B;
    const float* scaleA;
    const float* scaleB;
    const void* bias;
    void* C;
};

struct Int8Sizes {
    int M, N, K, lda, ldb;
    int64_t ldc;
};

template <bool PACKED>
struct Int8Args;
template <>
struct Int8Args<true> {
    Int8Operands p;
    uint64_t stridesAndK, rest;
    __host__ __device__ __forceinline__ Int8Sizes sizes() const {
        return {(int)(rest & 0xffff),
                (int)(rest >> 16 & 0xffff),
                (int)(stridesAndK >> 38),
                (int)(stridesAndK & 0x7ffff) * 16,
                (int)(stridesAndK >> 19 & 0x7ffff) * 16,
                (int64_t)(rest >> 32)};
    }
};
template <>
struct Int8Args<false> {
    Int8Operands p;
    Int8Sizes s;
    __host__ __device__ __forceinline__ Int8Sizes sizes() const { return s; }
};
static_assert(sizeof(Int8Args<true>) <= 64, "arguments of one write");

inline bool int8ArgsFit(const Int8Sizes& s) { return s.M <= 0xffff && s.N <= 0xffff && s.ldc <= 0xffffffffll; }

template <bool PACKED>
inline Int8Args<PACKED> int8Args(const Int8Operands& p, const Int8Sizes& s) {
    if constexpr (PACKED) {
        return {p, (uint64_t)(s.lda / 16) | (uint64_t)(s.ldb / 16) << 19 | (uint64_t)s.K << 38,
                (uint64_t)s.M | (uint64_t)s.N << 16 | (uint64_t)s.ldc << 32};
    } else {
        return {p, s};
    }
}

// Where chunk q = 8 row + c of a tile whose rows are 8 chunks lies in LDS (an involution). LDS
// serves a fragment's read 16 lanes at a time, lanes {0-3, 12-15, 20-27} and {4-11, 16-19,
// 28-31} of each half of the wave: 16 rows of the tile, half of them at one chunk and half at
// the next, which have to lie in 16 different 16-byte slots of a 256-byte line. The mask
// repeats every 16 rows, so fragments 16 rows apart are a constant distance apart. (Counted
// conflicts: none.)
constexpr int kChunksPerRow = 8;
__device__ __forceinline__ int swizzleRows(int q) { return q ^ (q / 16) % kChunksPerRow; }

// BK counts bytes, which are elements.
template <int BM_, int BN_, int BK_, int WM_, int WN_, int STAGES_>
struct Int8Traits {
    static constexpr int BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_, kStages = STAGES_;
    static constexpr int kWavesN = BN / WN;
    static constexpr int kWaves = (BM / WM) * kWavesN;
    static constexpr int kThreads = kWaves * kWaveSize;
    static constexpr int TM = WM / kMfmaM;
    static constexpr int TN = WN / kMfmaN;
    static constexpr int KS = BK / kInt8MfmaK;
    static constexpr int CPR = BK / 16;   // 16-byte chunks of a tile's row
    static constexpr int kBytesA = BM * BK;
    static constexpr int kBytesB = BN * BK;
    static constexpr int kRegionA = kStages * kBytesA;   // LDS: A's stages, then B's
    static constexpr int kRing = kStages * (kBytesA + kBytesB);
    static constexpr int kLdsBytes = kRing + 4 * (BM + BN);   // and the tile's scales
    static constexpr int kPerWaveA = kBytesA / 1024 / kWaves;   // 1 KiB loads of a wave
    static constexpr int kPerWaveB = kBytesB / 1024 / kWaves;
    static constexpr int kLoadsPerTile = kPerWaveA + kPerWaveB;

    static_assert(BM % WM == 0 && BN % WN == 0 && WM % kMfmaM == 0 && WN % kMfmaN == 0, "tiles must nest");
    static_assert(CPR == kChunksPerRow, "the swizzle is derived for rows of 8 chunks");
    static_assert(kBytesA % (1024 * kWaves) == 0 && kBytesB % (1024 * kWaves) == 0, "loads must split over the waves");
    static_assert((kStages - 1) * kLoadsPerTile < 64, "in-flight loads exceed the vmcnt counter");
    static_assert(kLdsBytes <= 163840, "LDS is 160 KiB per workgroup on gfx950");
};

// Direct-to-LDS 4-byte load (globalLoadLds16's sibling): lane t's 4 bytes at base + offset
// land at ldsAddr + 4 t.
__device__ __forceinline__ void globalLoadLds4(const void* base, uint32_t offset, uint32_t ldsAddr) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(base), "{m0}"(ldsAddr) : "memory");
}

// The lane's number, counted anew: kept through the K loop it costs a register that the
// 256 x 256 x 128 tile has not got.
__device__ __forceinline__ int laneAgain() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(lane));
    return lane;
}

// A mask of the first `bytes` of 16 bytes (none for fewer than 1, all for 16 and more).
__device__ __forceinline__ int4_t firstBytes(int bytes) {
    int4_t mask;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int n = min(max(bytes - 4 * d, 0), 4);
        mask[d] = n == 4 ? -1 : (1 << (8 * n)) - 1;
    }
    return mask;
}

// A C element from its sum. The sum is exact and is rounded to f32's 24 bits here: a
// relative 2^-24, far below what the result's type keeps.
__device__ __forceinline__ float scaledSum(int sum, float a, float b, float bias) {
    return fmaf((float)sum * a, b, bias);
}

// One tile of C: its loads, fragments, products and epilogue.
template <typename T, typename Out>
struct Int8Block {
    static constexpr int TM = T::TM, TN = T::TN, KS = T::KS, CPR = T::CPR;

    const Int8Operands p;
    const Int8Sizes z;
    const char* lds;
    uint32_t ldsBase;
    int lane, wave, waveM, waveN;
    int blockRow, blockCol;
    const char* gA;
    const char* gB;
    uint32_t offA[T::kPerWaveA];   // lane byte offsets of this wave's loads
    uint32_t offB[T::kPerWaveB];
    int rdA[KS], rdB[KS];          // fragment byte offsets of the wave's first 16 rows
    int4_t acc[TM][TN];
    int numK, numFull;             // K tiles, and those that K fills

    __device__ __forceinline__ Int8Block(const char* ldsArray, const Int8Operands& operands, const Int8Sizes& a,
                                            int row, int col)
        : p(operands), z(a) {
        lds = ldsArray;
        ldsBase = ldsAddress(ldsArray);
        lane = threadIdx.x % kWaveSize;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
        waveM = wave / T::kWavesN;
        waveN = wave % T::kWavesN;
        blockRow = row;
        blockCol = col;
        gA = (const char*)p.A + (int64_t)row * a.lda;
        gB = (const char*)p.B + (int64_t)col * a.ldb;
        numFull = a.K / T::BK;
        numK = numFull + (a.K % T::BK != 0);
#pragma unroll
        for (int i = 0; i < T::kPerWaveA; ++i) offA[i] = offset(chunkOf(i), a.lda, a.M - 1 - row);
#pragma unroll
        for (int i = 0; i < T::kPerWaveB; ++i) offB[i] = offset(chunkOf(i), a.ldb, a.N - 1 - col);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = 4 * ks + lane / 16;
            rdA[ks] = swizzleRows((waveM * T::WM + lane % 16) * CPR + c) * 16;
            rdB[ks] = T::kRegionA + swizzleRows((waveN * T::WN + lane % 16) * CPR + c) * 16;
        }
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) acc[tm][tn] = int4_t{0, 0, 0, 0};
    }

    // The scales of the tile's rows and columns on their way to LDS, 64 a wave load: the
    // oldest loads of the wave, landed when its first K tile has. Issued before issueTile.
    __device__ __forceinline__ void issueScales() const {
        static_assert((T::BM + T::BN) / 64 <= T::kWaves && T::BM % 64 == 0 && T::BN % 64 == 0, "one load a wave");
        const uint32_t to = ldsBase + T::kRing + wave * 256;
        const int at = wave * 64 + lane;
        if (wave < T::BM / 64) {
            globalLoadLds4(p.scaleA + blockRow, 4u * (uint32_t)min(at, z.M - 1 - blockRow), to);
        } else if (wave < (T::BM + T::BN) / 64) {
            globalLoadLds4(p.scaleB + blockCol, 4u * (uint32_t)min(at - T::BM, z.N - 1 - blockCol), to);
        }
    }

    // The chunk of a tile that this lane's share of the wave's load i fetches.
    __device__ __forceinline__ int chunkOf(int i) const {
        return swizzleRows((i * T::kWaves + wave) * 64 + lane);
    }

    // Byte offset of a load's chunk from the tile's first row. Strides are below 2^23 and
    // tiles have at most 256 rows: offsets fit 32 bits.
    static __device__ __forceinline__ uint32_t offset(int chunk, int ld, int lastRow) {
        return (uint32_t)min(chunk / CPR, lastRow) * (uint32_t)ld + (uint32_t)(chunk % CPR) * 16u;
    }

    // Refills LDS stage `stage` with K tile kTile (this wave's share). WHOLE: K is known to
    // fill it; else a chunk behind K's last one is replaced by that.
    template <bool WHOLE>
    __device__ __forceinline__ void issueTile(int kTile, int stage) const {
        const char* srcA = gA + (int64_t)kTile * T::BK;
        const char* srcB = gB + (int64_t)kTile * T::BK;
        const uint32_t dstA = ldsBase + stage * T::kBytesA;
        const uint32_t dstB = ldsBase + T::kRegionA + stage * T::kBytesB;
        const int last = WHOLE || kTile < numFull ? CPR - 1 : (z.K - 1) / 16 - kTile * CPR;
        auto past = [&](int i) {
            if constexpr (WHOLE) return 0u;
            const int chunk = swizzleRows((i * T::kWaves + wave) * 64 + laneAgain()) % CPR;
            return (uint32_t)max(chunk - last, 0) * 16u;
        };
#pragma unroll
        for (int i = 0; i < T::kPerWaveA; ++i)
            globalLoadLds16(srcA, offA[i] - past(i), dstA + (i * T::kWaves + wave) * 1024);
#pragma unroll
        for (int i = 0; i < T::kPerWaveB; ++i)
            globalLoadLds16(srcB, offB[i] - past(i), dstB + (i * T::kWaves + wave) * 1024);
    }

    template <int STAGE>
    __device__ __forceinline__ void readFrags(int ks, int4_t (&a)[TM], int4_t (&b)[TN]) const {
        const RIDGE_LDS_AS char* l = (const RIDGE_LDS_AS char*)(lds);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
            a[tm] = *(const RIDGE_LDS_AS int4_t*)(l + rdA[ks] + STAGE * T::kBytesA + tm * 16 * T::BK);
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
            b[tn] = *(const RIDGE_LDS_AS int4_t*)(l + rdB[ks] + STAGE * T::kBytesB + tn * 16 * T::BK);
    }

    // Clears what A's fragments of K tile kTile hold behind K.
    __device__ __forceinline__ void clearBehind(int kTile, int ks, int4_t (&a)[TM]) const {
        const int4_t mask = firstBytes(z.K - (kTile * T::BK + ks * kInt8MfmaK + 16 * (laneAgain() / 16)));
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) a[tm] &= mask;
    }

    __device__ __forceinline__ void mfmaStep(const int4_t (&a)[TM], const int4_t (&b)[TN]) {
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int tm = (tn & 1) ? TM - 1 - i : i;
                acc[tm][tn] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[tn], a[tm], acc[tm][tn], 0, 0, 0);
            }
    }

    // Epilogue of one wave through a private LDS region, 16 rows a pass: a lane's four
    // columns are scaled, rounded and written there, and read back row by row, so that
    // every store but a row's last is 16 bytes a lane. A wave's LDS instructions run in
    // order, so only the compiler has to be kept from moving them; the next pass is
    // computed while the read-backs are on their way. Every wave has to be past its last
    // read of the ring. (256 x 256 tiles, 4096 cubed: 10.7k cycles with a wait on either
    // side of the region and the scales read from memory at the end, 6.9k so.)
    static constexpr int kChunks = T::WN * (int)sizeof(Out) / 16;   // 16-byte chunks of a region's row
    static constexpr int kRegionBytes = 16 * T::WN * (int)sizeof(Out);
    static constexpr int kPer = 16 / (int)sizeof(Out);              // elements of a chunk
    static constexpr int kReads = 16 * kChunks / 64;                // read-backs of a pass
    static_assert(T::kWaves * kRegionBytes <= T::kRing && 16 * kChunks % 64 == 0, "epilogue regions must fit the ring");
    typedef Out Quad __attribute__((ext_vector_type(4)));
    typedef Out Chunk __attribute__((ext_vector_type(kPer)));
    typedef Out Placed __attribute__((ext_vector_type(kPer), aligned(sizeof(Out))));

    // STREAM: past the caches.
    template <bool STREAM>
    __device__ __forceinline__ void store() const {
        RIDGE_LDS_AS char* region = (RIDGE_LDS_AS char*)(const_cast<char*>(lds)) + wave * kRegionBytes;
        const RIDGE_LDS_AS float* scales = (const RIDGE_LDS_AS float*)((const RIDGE_LDS_AS char*)(lds) + T::kRing);
        auto swz = [](int row, int chunk) { return chunk ^ ((row * kChunks / 16) % kChunks); };
        const int lane = laneAgain();
        const int g = lane / 16, r16 = lane % 16;
        const int row0 = blockRow + waveM * T::WM, col0 = blockCol + waveN * T::WN;
        float4_t sb[TN], add[TN];
#pragma unroll
        for (int tn = 0; tn < TN; ++tn) {
            sb[tn] = *(const RIDGE_LDS_AS float4_t*)(scales + T::BM + waveN * T::WN + tn * 16 + 4 * g);
            add[tn] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        if (p.bias != nullptr) {
            const Out* bias = (const Out*)p.bias;
#pragma unroll
            for (int tn = 0; tn < TN; ++tn)
#pragma unroll
                for (int e = 0; e < 4; ++e) add[tn][e] = (float)bias[min(col0 + tn * 16 + 4 * g + e, z.N - 1)];
        }
        Quad quads[TN];
        auto compute = [&](int tm) {
            const float sa = scales[waveM * T::WM + 16 * tm + r16];
#pragma unroll
            for (int tn = 0; tn < TN; ++tn)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    quads[tn][e] = (Out)scaledSum(acc[tm][tn][e], sa, sb[tn][e], add[tn][e]);
        };
        compute(0);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) {
                const int at = tn * 16 + 4 * g;
                *(RIDGE_LDS_AS Quad*)(region + (r16 * kChunks + swz(r16, at / kPer)) * 16 +
                                      (at % kPer) * sizeof(Out)) = quads[tn];
            }
            asm volatile("" ::: "memory");
            Chunk v[kReads];
#pragma unroll
            for (int j = 0; j < kReads; ++j) {
                const int q = j * 64 + lane;
                v[j] = *(const RIDGE_LDS_AS Chunk*)(region + (q / kChunks * kChunks + swz(q / kChunks, q % kChunks)) * 16);
            }
            asm volatile("" ::: "memory");
            if (tm + 1 < TM) compute(tm + 1);
#pragma unroll
            for (int j = 0; j < kReads; ++j) {
                const int q = j * 64 + lane;
                const int row = row0 + 16 * tm + q / kChunks, col = col0 + q % kChunks * kPer;
                if (row < z.M && col < z.N) {
                    Out* dst = (Out*)p.C + (int64_t)row * z.ldc + col;
                    if (col + kPer <= z.N) {
                        if constexpr (STREAM) {
                            __builtin_nontemporal_store(*(const Placed*)&v[j], (Placed*)dst);
                        } else {
                            *(Placed*)dst = v[j];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < kPer; ++e)
                            if (col + e < z.N) dst[e] = v[j][e];
                    }
                }
            }
        }
    }
};

// Scheduling hint for a k-step of the uniform loop: one LDS read behind every second
// product, so that the next step's reads hide under this step. (256 x 256 x 128, cycles of
// the K loop at 4096 cubed: none 93.6k, one read a product 82.9k, one in two 82.4k, one in
// four 89.4k.)
template <int TM, int TN>
__device__ __forceinline__ void interleaveReads() {
    constexpr int kMfmas = TM * TN, kReads = TM + TN;
#pragma unroll
    for (int i = 0; i < kMfmas / 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        if (i < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    if (kReads > kMfmas / 2) __builtin_amdgcn_sched_group_barrier(0x100, kReads - kMfmas / 2, 0);
}

// Every wavefront runs the same phase at the same time: fragments are double-buffered
// across k-steps, and the tile boundary sits inside the last k-step of a tile. Once tile
// kt + 1 has landed and every wave is past its reads of tile kt, the freed stage is
// refilled with tile kt + STAGES and tile kt + 1's first fragments are read while tile
// kt's last products run.
template <typename T, typename Blk>
__device__ __forceinline__ void int8UniformLoop(Blk& blk) {
    constexpr int STAGES = T::kStages;
    constexpr int KS = T::KS;
    constexpr int L = T::kLoadsPerTile;
    const int numK = blk.numK, numFull = blk.numFull;

    blk.issueScales();
    staticFor<STAGES>([&](auto sC) {
        if (sC.value < numK) blk.template issueTile<false>(sC.value, sC.value);
    });
    if (numK >= STAGES) {
        waitVmcnt<(STAGES - 1) * L>();
    } else {
        waitVmcnt<0>();
    }
    barrierLds();

    int4_t fa[2][T::TM], fb[2][T::TN];
    blk.template readFrags<0>(0, fa[0], fb[0]);
    // A pass covers whole turns of the ring with an even number of k-steps, so that
    // every stage and buffer number is a constant. Passes whose every refill tile exists
    // and is filled by K run first, without the tests.
    constexpr int U = (STAGES * KS) % 2 == 0 ? STAGES : 2 * STAGES;
    auto pass = [&](int kt0, auto steadyC) {
        constexpr bool steady = steadyC.value;
        staticFor<U>([&](auto iC) {
            constexpr int i = iC.value;
            constexpr int s = i % STAGES;
            constexpr int sNext = (s + 1) % STAGES;
            const int kt = kt0 + i;
            if (steady || kt < numK) {
                staticFor<KS>([&](auto ksC) {
                    constexpr int ks = ksC.value;
                    constexpr int cur = (i * KS + ks) & 1;
                    if constexpr (ks + 1 < KS) {
                        blk.template readFrags<s>(ks + 1, fa[cur ^ 1], fb[cur ^ 1]);
                    } else if (steady || kt + 1 < numK) {
                        if (steady || kt + STAGES - 1 < numK) {
                            waitVmcnt<(STAGES - 2) * L>();
                        } else {
                            waitVmcnt<0>();
                        }
                        barrierLds();
                        if (steady || kt + STAGES < numK) blk.template issueTile<steady>(kt + STAGES, s);
                        blk.template readFrags<sNext>(0, fa[cur ^ 1], fb[cur ^ 1]);
                    }
                    if (!steady && kt >= numFull) blk.clearBehind(kt, ks, fa[cur]);
                    blk.mfmaStep(fa[cur], fb[cur]);
                    interleaveReads<T::TM, T::TN>();
                });
            }
        });
    };
    int kt0 = 0;
    for (; kt0 + U - 1 + STAGES < numFull; kt0 += U) pass(kt0, std::true_type{});
    for (; kt0 < numK; kt0 += U) pass(kt0, std::false_type{});
    barrierLds();
}

// Ping-pong schedule for eight wavefronts, two on a SIMD: waves 0-3 and 4-7 alternate a
// memory phase (refill the stage freed by tile kt - 1 with tile kt + STAGES - 1, read all
// of tile kt's fragments) with a matrix phase (all its products), one barrier apart, so
// that one wave's products cover the other's LDS and global traffic. Group 0 reads tile t
// in phase 2 t, group 1 in phase 2 t + 1.
//  * A stage is refilled after both groups have read it: tile t + STAGES - 1 goes where
//    tile t - 1 was and is issued in phase 2 t or 2 t + 1.
//  * Tile t + 1 is in LDS before the barrier of phases 2 t + 1 | 2 t + 2: group 0 comes to
//    it behind its matrix phase and group 1 behind its memory phase, and each first waits
//    until only tiles t + 2 .. t + STAGES - 1 of its own loads are outstanding.
template <typename T, typename Blk>
__device__ __forceinline__ void int8PingPongLoop(Blk& blk) {
    static_assert(T::kWaves == 8 && T::kStages >= 3, "two groups of four waves, and a refill ahead of two tiles");
    constexpr int STAGES = T::kStages;
    constexpr int KS = T::KS;
    constexpr int L = T::kLoadsPerTile;
    const int numK = blk.numK, numFull = blk.numFull;

    blk.issueScales();
    staticFor<STAGES - 1>([&](auto sC) {
        if (sC.value < numK) blk.template issueTile<false>(sC.value, sC.value);
    });
    if (numK >= STAGES - 1) {
        waitVmcnt<(STAGES - 2) * L>();
    } else {
        waitVmcnt<0>();
    }
    barrierLds();

    // STEADY: the refill tile kt + STAGES - 1 exists and K fills it.
    auto tileBody = [&](auto sC, auto groupC, int kt, auto steadyC) {
        constexpr int s = sC.value;
        constexpr int sRefill = (s + STAGES - 1) % STAGES;
        constexpr int group = groupC.value;
        constexpr bool steady = steadyC.value;
        const bool refill = steady || kt + STAGES - 1 < numK;
        if (refill) blk.template issueTile<steady>(kt + STAGES - 1, sRefill);
        int4_t fa[KS][T::TM], fb[KS][T::TN];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) blk.template readFrags<s>(ks, fa[ks], fb[ks]);
        auto wait = [&] {
            if (refill) waitVmcnt<(STAGES - 2) * L>();
            else waitVmcnt<0>();
        };
        if constexpr (group == 1) wait();
        phaseBarrier();
        if (!steady && kt >= numFull) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) blk.clearBehind(kt, ks, fa[ks]);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) blk.mfmaStep(fa[ks], fb[ks]);
        if constexpr (group == 0) wait();
        phaseBarrier();
    };
    auto runGroup = [&](auto groupC) {
        if constexpr (groupC.value == 1) barrierLds();
        int kt0 = 0;
        for (; kt0 + 2 * STAGES - 2 < numFull; kt0 += STAGES)
            staticFor<STAGES>([&](auto sC) { tileBody(sC, groupC, kt0 + sC.value, std::true_type{}); });
        for (; kt0 < numK; kt0 += STAGES)
            staticFor<STAGES>([&](auto sC) {
                if (kt0 + sC.value < numK) tileBody(sC, groupC, kt0 + sC.value, std::false_type{});
            });
        // Matches group 1's at the start: behind it every wave is past its last read.
        if constexpr (groupC.value == 0) barrierLds();
    };
    if (blk.wave / 4 == 0) {
        runGroup(std::integral_constant<int, 0>{});
    } else {
        runGroup(std::integral_constant<int, 1>{});
    }
}

constexpr int kInt8GroupM = 8;

template <typename T>
__host__ __device__ inline int int8TilesM(int M) {
    return (M + T::BM - 1) / T::BM;
}
template <typename T>
__host__ __device__ inline int int8TilesN(int N) {
    return (N + T::BN - 1) / T::BN;
}

// n / d for n below 2^24, by f32's reciprocal and a correction: a uniform value.
__device__ __forceinline__ DivMod divideSmall(uint32_t n, uint32_t d) {
    uint32_t q = (uint32_t)__builtin_amdgcn_readfirstlane((int)((float)n * __builtin_amdgcn_rcpf((float)d)));
    int r = (int)(n - q * d);
    if (r < 0) {
        --q;
        r += (int)d;
    } else if (r >= (int)d) {
        ++q;
        r -= (int)d;
    }
    return {q, (uint32_t)r};
}

// tileOf's order (groups of kInt8GroupM tile rows, column by column) without its
// arguments: fewer than 2^23 tiles, which the launch sees to.
template <typename T>
__device__ __forceinline__ void int8TileOf(int id, int tilesM, int tilesN, int& row, int& col) {
    const DivMod group = divideSmall((uint32_t)id, (uint32_t)(kInt8GroupM * tilesN));
    const int first = (int)group.quot * kInt8GroupM;
    const DivMod in = divideSmall(group.rem, (uint32_t)min(tilesM - first, kInt8GroupM));
    row = (first + (int)in.rem) * T::BM;
    col = (int)in.quot * T::BN;
}

template <typename T, typename Out, bool PINGPONG, bool PACKED, bool STREAM>
__global__ __launch_bounds__(T::kThreads)
void int8GemmKernel(Int8Args<PACKED> args) {
    __shared__ __attribute__((aligned(1024))) char lds[T::kLdsBytes];
    const Int8Sizes z = args.sizes();
    const int tilesM = int8TilesM<T>(z.M), tilesN = int8TilesN<T>(z.N);
    int row, col;
    int8TileOf<T>(xcdRemap(blockIdx.x, tilesM * tilesN), tilesM, tilesN, row, col);
    Int8Block<T, Out> blk(lds, args.p, z, row, col);
    if constexpr (PINGPONG) {
        int8PingPongLoop<T>(blk);
    } else {
        int8UniformLoop<T>(blk);
    }
    blk.template store<STREAM>();
}

using Tile256x256 = Int8Traits<256, 256, 128, 128, 64, 2>;
using Tile256x128 = Int8Traits<256, 128, 128, 64, 64, 3>;   // ping-pong
using Tile128x128 = Int8Traits<128, 128, 128, 32, 64, 3>;

// Grids of 256 x 256 tiles: whole rounds of them on the chip's CUs, and what is left of
// more than a round cut into as many parts as still fit one: a last round of few tiles
// would leave most CUs idle. us, the fastest form without parts | with them: 4001 x 4103 x
// 2065 (272 tiles) 55.6 | 41.5, 5888 x 5888 x 1664 (529) 70.6 | 59.4, 6144 x 4096 x 2048
// (384) 58.2 | 51.4, 7663 x 5248 x 3712 (630) 129.6 | 121.4.
constexpr int kInt8CUs = 256;
struct Int8Rounds {
    int whole, parts, blocks;   // tiles in whole rounds; parts of each other tile; workgroups
};
__host__ __device__ inline Int8Rounds int8Rounds(int tiles) {
    const int left = tiles > kInt8CUs ? tiles % kInt8CUs : 0;
    const int parts = left == 0 || left > kInt8CUs / 2 ? 1 : left > kInt8CUs / 4 ? 2 : 4;
    const int whole = parts == 1 ? tiles : tiles - left;
    return {whole, parts, whole + (tiles - whole) * parts};
}

template <typename Out, bool PACKED, bool STREAM>
__global__ __launch_bounds__(Tile256x256::kThreads)
void int8RoundsKernel(Int8Args<PACKED> args) {
    using T = Tile256x256;
    static_assert(T::kThreads == Tile256x128::kThreads && T::kThreads == Tile128x128::kThreads, "parts of one launch");
    constexpr int kLds = T::kLdsBytes > Tile256x128::kLdsBytes ? T::kLdsBytes : Tile256x128::kLdsBytes;
    static_assert(kLds >= Tile128x128::kLdsBytes, "the parts share the tile's LDS");
    __shared__ __attribute__((aligned(1024))) char lds[kLds];
    const Int8Sizes z = args.sizes();
    const int tilesM = int8TilesM<T>(z.M), tilesN = int8TilesN<T>(z.N);
    const Int8Rounds r = int8Rounds(tilesM * tilesN);
    int row, col;
    if ((int)blockIdx.x < r.whole) {
        int8TileOf<T>(xcdRemap(blockIdx.x, r.whole), tilesM, tilesN, row, col);
        Int8Block<T, Out> blk(lds, args.p, z, row, col);
        int8UniformLoop<T>(blk);
        blk.template store<STREAM>();
        return;
    }
    const int id = xcdRemap(blockIdx.x - r.whole, r.blocks - r.whole);
    int8TileOf<T>(r.whole + id / r.parts, tilesM, tilesN, row, col);
    if (r.parts == 4) {
        row += id % 4 / 2 * 128;
        col += id % 2 * 128;
        if (row >= z.M || col >= z.N) return;   // a part of an edge tile that has nothing of C
        Int8Block<Tile128x128, Out> blk(lds, args.p, z, row, col);
        int8UniformLoop<Tile128x128>(blk);
        blk.template store<STREAM>();
    } else {
        col += id % 2 * 128;
        if (col >= z.N) return;
        Int8Block<Tile256x128, Out> blk(lds, args.p, z, row, col);
        int8PingPongLoop<Tile256x128>(blk);
        blk.template store<STREAM>();
    }
}

// ---------------------------------------------------------------------------
// Few tokens, or few tiles: 16 TM x 16 TN of C a workgroup, whose WAVES wavefronts share K.
//
// Wave w takes the 128-byte pieces w, w + WAVES, ... of every row, so that the workgroup
// reads its rows front to back. A wave streams its pieces through a ring of its own in LDS
// (eight lanes load a row's 128 bytes, one fragment read takes 16 rows: straight to
// registers the 16 lanes of a load would be 16 rows apart) and waits for nothing but its
// own loads: there is no barrier before the end, where the sums meet. They are 32-bit
// integers, whose order does not matter.
// ---------------------------------------------------------------------------
template <int TM_, int TN_, int WAVES_, int STAGES_>
struct Int8FewTraits {
    static constexpr int TM = TM_, TN = TN_, kWaves = WAVES_, kStages = STAGES_;
    static constexpr int kThreads = kWaves * kWaveSize;
    static constexpr int kPiece = 128;                       // bytes of a row a wave takes at once
    static constexpr int CPR = kPiece / 16;
    static_assert(CPR == kChunksPerRow, "the swizzle is derived for rows of 8 chunks");
    static constexpr int KS = kPiece / kInt8MfmaK;
    static constexpr int kTiles = TM * TN;                   // 16 x 16 tiles of C
    static constexpr int kPieceBytes = 16 * (TM + TN) * kPiece;
    static constexpr int kLoads = kPieceBytes / 1024;        // of a wave for a piece
    static constexpr int kWaveBytes = kStages * kPieceBytes;
    static constexpr int kLdsBytes = kWaves * kWaveBytes;
    static_assert(kLdsBytes <= 163840, "LDS is 160 KiB per workgroup on gfx950");
    static_assert((kStages - 1) * kLoads < 64, "in-flight loads exceed the vmcnt counter");
    static_assert(kTiles * 1024 <= kWaveBytes, "a wave's sums replace its ring");
};

template <typename T, typename Out>
__global__ __launch_bounds__(T::kThreads)
void int8FewKernel(Int8Args<true> args) {
    const Int8Operands p = args.p;
    const Int8Sizes z = args.sizes();
    constexpr int TM = T::TM, TN = T::TN, KS = T::KS, CPR = T::CPR, STAGES = T::kStages, L = T::kLoads;
    __shared__ __attribute__((aligned(1024))) char lds[T::kLdsBytes];
    const int lane = threadIdx.x % kWaveSize;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    // Workgroups of the same channels are neighbours on one XCD: they read the same rows of B.
    const int rowBlocks = (z.M + 16 * TM - 1) / (16 * TM), colBlocks = (z.N + 16 * TN - 1) / (16 * TN);
    const DivMod block = divideSmall((uint32_t)xcdRemap(blockIdx.x, rowBlocks * colBlocks), (uint32_t)rowBlocks);
    const int row0 = (int)block.rem * 16 * TM, col0 = (int)block.quot * 16 * TN;
    const int r16 = lane % 16, g = lane / 16;

    // A piece in LDS: 16 TN rows of B, then 16 TM rows of A. Load i fills eight of them.
    const char* gA = (const char*)p.A + (int64_t)row0 * z.lda;
    const char* gB = (const char*)p.B + (int64_t)col0 * z.ldb;
    uint32_t off[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int q = swizzleRows(64 * i + lane), row = q / CPR;
        off[i] = (uint32_t)(q % CPR) * 16u + (i < 2 * TN ? (uint32_t)min(row, z.N - 1 - col0) * (uint32_t)z.ldb
                                                         : (uint32_t)min(row - 16 * TN, z.M - 1 - row0) * (uint32_t)z.lda);
    }
    const uint32_t ring = ldsAddress(lds) + wave * T::kWaveBytes;
    const int pieces = (z.K + T::kPiece - 1) / T::kPiece;
    auto issue = [&](int piece, int stage) {
        const int64_t at = (int64_t)piece * T::kPiece;
        // How far behind the last chunk of K this lane's chunk is.
        const int last = min((z.K - 1) / 16 - piece * CPR, CPR - 1);
        auto past = [&](int i) { return (uint32_t)max(swizzleRows(64 * i + lane) % CPR - last, 0) * 16u; };
#pragma unroll
        for (int i = 0; i < L; ++i)
            globalLoadLds16((i < 2 * TN ? gB : gA) + at, off[i] - past(i),
                            ring + stage * T::kPieceBytes + i * 1024);
    };
    int4_t acc[TM][TN];
#pragma unroll
    for (int tm = 0; tm < TM; ++tm)
#pragma unroll
        for (int tn = 0; tn < TN; ++tn) acc[tm][tn] = int4_t{0, 0, 0, 0};

    const int mine = (pieces - wave + T::kWaves - 1) / T::kWaves;   // this wave's pieces; none or less: 0
    const RIDGE_LDS_AS char* const own = (const RIDGE_LDS_AS char*)(lds) + wave * T::kWaveBytes;
    const int rd = swizzleRows(r16 * CPR + g) * 16;             // k-step 0; step ks flips chunk bit 2
    staticFor<STAGES>([&](auto sC) {
        if (sC.value < mine) issue(wave + sC.value * T::kWaves, sC.value);
    });
    for (int i0 = 0; i0 < mine; i0 += STAGES) {
        staticFor<STAGES>([&](auto sC) {
            constexpr int s = sC.value;
            const int i = i0 + s;
            if (i < mine) {
                if (i + STAGES - 1 < mine) {
                    waitVmcnt<(STAGES - 1) * L>();
                } else {
                    waitVmcnt<0>();
                }
                int4_t a[KS][TM], b[KS][TN];
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const RIDGE_LDS_AS char* at = own + s * T::kPieceBytes + (rd ^ (ks * 64));
#pragma unroll
                    for (int tn = 0; tn < TN; ++tn) b[ks][tn] = *(const RIDGE_LDS_AS int4_t*)(at + tn * 2048);
#pragma unroll
                    for (int tm = 0; tm < TM; ++tm) a[ks][tm] = *(const RIDGE_LDS_AS int4_t*)(at + (TN + tm) * 2048);
                }
                const int piece = wave + i * T::kWaves;
                // The stage has been read before it is filled again.
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (i + STAGES < mine) issue(piece + STAGES * T::kWaves, s);
                if (piece * T::kPiece + T::kPiece > z.K) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const int4_t mask = firstBytes(z.K - (piece * T::kPiece + ks * kInt8MfmaK + 16 * g));
#pragma unroll
                        for (int tm = 0; tm < TM; ++tm) a[ks][tm] &= mask;
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
                        for (int tm = 0; tm < TM; ++tm)
                            acc[tm][tn] =
                                __builtin_amdgcn_mfma_i32_16x16x64_i8(b[ks][tn], a[ks][tm], acc[tm][tn], 0, 0, 0);
            }
        });
    }

    int4_t* sums = (int4_t*)(lds + wave * T::kWaveBytes);
#pragma unroll
    for (int tm = 0; tm < TM; ++tm)
#pragma unroll
        for (int tn = 0; tn < TN; ++tn) sums[(tm * TN + tn) * kWaveSize + lane] = acc[tm][tn];
    __syncthreads();
    // Wave w finishes the tiles w, w + WAVES, ...: lane l has token 16 tm + l % 16 and the
    // four channels from 16 tn + 4 (l / 16) on.
    for (int t = wave; t < T::kTiles; t += T::kWaves) {
        int4_t total = int4_t{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < T::kWaves; ++w)
            total += *(const int4_t*)(lds + w * T::kWaveBytes + (t * kWaveSize + lane) * 16);
        const int row = row0 + 16 * (t / TN) + r16, col = col0 + 16 * (t % TN) + 4 * g;
        if (row < z.M) {
            const float sa = p.scaleA[row];
            Out* dst = (Out*)p.C + (int64_t)row * z.ldc + col;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (col + e < z.N) {
                    const float add = p.bias ? (float)((const Out*)p.bias)[col + e] : 0.0f;
                    dst[e] = (Out)scaledSum(total[e], sa, p.scaleB[col + e], add);
                }
            }
        }
    }
}

}  // namespace ridge
