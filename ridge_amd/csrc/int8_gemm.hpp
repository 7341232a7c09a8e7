// int8_gemm.hpp -- matrix product of 8-bit rows for gfx950 (MI355X): 32-bit integer sums
// on the matrix pipes, one scale for each row of A and of B in the epilogue.
//
//   C[m, n] = (sum over k of A[m, k] B[n, k]) scaleA[m] scaleB[n] + bias[n]
//
// A (M x K) and B (N x K) both have k along memory. v_mfma_i32_16x16x64_i8 takes 16
// consecutive k of one row a lane (16 bytes, lane group g = lane / 16 holding k = 16 g ..
// 16 g + 15), which is byte for byte the operand layout of the FP16 instruction of half
// the K: a tile's rows are loaded straight into LDS in 16-byte chunks, swizzled (swizzleRows), and
// both fragments are single ds_read_b128s. With B's
// fragment in the first operand lane l holds C[m0 + l % 16][n0 + 4 (l / 16) + r] in
// element r.
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

struct Int8Args {
    const int8_t* A;
    const int8_t* B;
    const float* scaleA;
    const float* scaleB;
    const void* bias;
    void* C;
    int lda, ldb;
    int64_t ldc;
    int M, N, K;
    TileOrder order;   // of ceil(M / BM) x ceil(N / BN) tiles
};

// Where chunk q = row * CPR + c of a tile lies in LDS (an involution). A fragment's read
// has 16 lanes read one chunk of 16 consecutive rows, 256 bytes that LDS serves at once
// where they lie in 16 different 16-byte slots of a 256-byte line: 16 / CPR rows share
// such a line, and the mask gives the groups of rows that do different slots. It repeats
// every 16 rows, so fragments 16 rows apart are a constant distance apart.
template <int CPR>
__device__ __forceinline__ int swizzleRows(int q) {
    return q ^ ((q / 16) % CPR);
}

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
    static constexpr int kLdsBytes = kStages * (kBytesA + kBytesB);
    static constexpr int kPerWaveA = kBytesA / 1024 / kWaves;   // 1 KiB loads of a wave
    static constexpr int kPerWaveB = kBytesB / 1024 / kWaves;
    static constexpr int kLoadsPerTile = kPerWaveA + kPerWaveB;

    static_assert(BM % WM == 0 && BN % WN == 0 && WM % kMfmaM == 0 && WN % kMfmaN == 0, "tiles must nest");
    static_assert(BK == 64 || BK == 128 || BK == 256, "the swizzle is derived for rows of 4, 8 and 16 chunks");
    static_assert(kBytesA % (1024 * kWaves) == 0 && kBytesB % (1024 * kWaves) == 0, "loads must split over the waves");
    static_assert((kStages - 1) * kLoadsPerTile < 64, "in-flight loads exceed the vmcnt counter");
    static_assert(kLdsBytes <= 163840, "LDS is 160 KiB per workgroup on gfx950");
};

// A C element from its sum. The sum is exact and is rounded to f32's 24 bits here: a
// relative 2^-24, far below what the result's type keeps.
__device__ __forceinline__ float scaledSum(int sum, float a, float b, float bias) {
    return fmaf((float)sum * a, b, bias);
}

template <typename T, typename Out>
struct Int8Block {
    static constexpr int TM = T::TM, TN = T::TN, KS = T::KS, CPR = T::CPR;

    const Int8Args& args;
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

    __device__ __forceinline__ Int8Block(const char* ldsArray, const Int8Args& a, int row, int col) : args(a) {
        lds = ldsArray;
        ldsBase = ldsAddress(ldsArray);
        lane = threadIdx.x % kWaveSize;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
        waveM = wave / T::kWavesN;
        waveN = wave % T::kWavesN;
        blockRow = row;
        blockCol = col;
        gA = (const char*)a.A + (int64_t)row * a.lda;
        gB = (const char*)a.B + (int64_t)col * a.ldb;
        numFull = a.K / T::BK;
        numK = numFull + (a.K % T::BK != 0);
#pragma unroll
        for (int i = 0; i < T::kPerWaveA; ++i) offA[i] = offset(chunkOf(i), a.lda, a.M - 1 - row);
#pragma unroll
        for (int i = 0; i < T::kPerWaveB; ++i) offB[i] = offset(chunkOf(i), a.ldb, a.N - 1 - col);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            rdA[ks] = swizzleRows<CPR>((waveM * T::WM + lane % 16) * CPR + 4 * ks + lane / 16) * 16;
            rdB[ks] = T::kRegionA + swizzleRows<CPR>((waveN * T::WN + lane % 16) * CPR + 4 * ks + lane / 16) * 16;
        }
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) acc[tm][tn] = int4_t{0, 0, 0, 0};
    }

    // The chunk of a tile that this lane's share of the wave's load i fetches.
    __device__ __forceinline__ int chunkOf(int i) const {
        return swizzleRows<CPR>((i * T::kWaves + wave) * 64 + lane);
    }

    // Strides are below 2^23 and tiles have at most 256 rows, so offsets fit 32 bits.
    static __device__ __forceinline__ uint32_t offset(int chunk, int ld, int lastRow) {
        return (uint32_t)min(chunk / CPR, lastRow) * (uint32_t)ld + (uint32_t)(chunk % CPR) * 16u;
    }

    // Refills LDS stage `stage` with K tile kTile (this wave's share). `whole`: the tile
    // is known to be one that K fills.
    template <bool WHOLE>
    __device__ __forceinline__ void issueTile(int kTile, int stage) const {
        const char* srcA = gA + (int64_t)kTile * T::BK;
        const char* srcB = gB + (int64_t)kTile * T::BK;
        const uint32_t dstA = ldsBase + stage * T::kBytesA;
        const uint32_t dstB = ldsBase + T::kRegionA + stage * T::kBytesB;
        // How far behind the last chunk of K each lane's chunk is.
        const int last = WHOLE || kTile < numFull ? CPR - 1 : (args.K - 1) / 16 - kTile * CPR;
        auto past = [&](int i) { return WHOLE ? 0u : (uint32_t)max(chunkOf(i) % CPR - last, 0) * 16u; };
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
        const int left = args.K - (kTile * T::BK + ks * kInt8MfmaK + 16 * (lane / 16));
        int4_t mask;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int bytes = min(max(left - 4 * d, 0), 4);
            mask[d] = bytes == 4 ? -1 : (1 << (8 * bytes)) - 1;
        }
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
    // every store but a row's last is 16 bytes a lane. Every wave has to be past its last
    // read of the ring.
    static constexpr int kChunks = T::WN * (int)sizeof(Out) / 16;   // 16-byte chunks of a region's row
    static constexpr int kRegionBytes = 16 * T::WN * (int)sizeof(Out);
    static constexpr int kPer = 16 / (int)sizeof(Out);              // elements of a chunk
    static_assert(T::kWaves * kRegionBytes <= T::kLdsBytes, "epilogue regions must fit the ring");

    __device__ __forceinline__ void store() const {
        typedef Out Quad __attribute__((ext_vector_type(4)));
        typedef Out Chunk __attribute__((ext_vector_type(kPer)));
        typedef Out Placed __attribute__((ext_vector_type(kPer), aligned(sizeof(Out))));
        RIDGE_LDS_AS char* region = (RIDGE_LDS_AS char*)(const_cast<char*>(lds)) + wave * kRegionBytes;
        auto swz = [](int row, int chunk) { return chunk ^ ((row * kChunks / 16) % kChunks); };
        const int g = lane / 16, r16 = lane % 16;
        const int row0 = blockRow + waveM * T::WM, col0 = blockCol + waveN * T::WN;
        const Out* bias = (const Out*)args.bias;
        float sb[TN][4], add[TN][4];
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = min(col0 + tn * 16 + 4 * g + e, args.N - 1);
                sb[tn][e] = args.scaleB[col];
                add[tn][e] = bias ? (float)bias[col] : 0.0f;
            }
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const float sa = args.scaleA[min(row0 + 16 * tm + r16, args.M - 1)];
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) {
                Quad v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (Out)scaledSum(acc[tm][tn][e], sa, sb[tn][e], add[tn][e]);
                const int at = tn * 16 + 4 * g;
                *(RIDGE_LDS_AS Quad*)(region + (r16 * kChunks + swz(r16, at / kPer)) * 16 +
                                      (at % kPer) * sizeof(Out)) = v;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int j = 0; j < 16 * kChunks / 64; ++j) {
                const int q = j * 64 + lane, r = q / kChunks, c = q % kChunks;
                const Chunk v = *(const RIDGE_LDS_AS Chunk*)(region + (r * kChunks + swz(r, c)) * 16);
                const int row = row0 + 16 * tm + r, col = col0 + c * kPer;
                if (row < args.M && col < args.N) {
                    Out* dst = (Out*)args.C + (int64_t)row * args.ldc + col;
                    if (col + kPer <= args.N) {
                        *(Placed*)dst = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < kPer; ++e)
                            if (col + e < args.N) dst[e] = v[e];
                    }
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
};

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
                });
            }
        });
    };
    int kt0 = 0;
    for (; kt0 + U - 1 + STAGES < numFull; kt0 += U) pass(kt0, std::true_type{});
    for (; kt0 < numK; kt0 += U) pass(kt0, std::false_type{});
    barrierLds();
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

template <typename T, typename Out>
__global__ __launch_bounds__(T::kThreads)
void int8GemmKernel(Int8Args args) {
    __shared__ __attribute__((aligned(1024))) char lds[T::kLdsBytes];
    const int tilesM = int8TilesM<T>(args.M), tilesN = int8TilesN<T>(args.N);
    int row, col;
    tileOf<T::BM, T::BN, kInt8GroupM>(xcdRemap(blockIdx.x, tilesM * tilesN), tilesM * T::BM, tilesN * T::BN,
                                      args.order, row, col);
    Int8Block<T, Out> blk(lds, args, row, col);
    int8UniformLoop<T>(blk);
    blk.store();
}

}  // namespace ridge
