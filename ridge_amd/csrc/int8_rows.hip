// int8_rows.hip -- the operators that make 8-bit rows (quantize, silu_mul, rms_norm) and
// the one that reads them back, for the C ABI in include/ridge_int8.h.
//
// All three makers are one kernel around a different source of a row's f32 values: read
// the row once, hold its values in registers, reduce the largest magnitude (and, for the
// norm, the sum of squares) over the row's threads, round and write. Memory bounds them
// (16384 x 8192: the norm 5.4 TB/s, quantize 5.9): every input byte is read once and every
// output byte written once, in 16-byte and 8-byte pieces a lane. The gated activation is
// bound by its arithmetic, 33 vector instructions an element (4096 x 16384 77 us).
//
// A norm needs one reduction, not two: the sum of squares and the largest |s w| are taken
// together, because the reciprocal root that multiplies a whole row moves out of the
// maximum, and out of the quotients that are rounded.

#include "int8_launch.hpp"
#include "int8_values.hpp"
#include "ridge_int8.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace {

constexpr int kWave = 64;
constexpr int kVec = 8;  // elements a lane loads at once: 16 bytes of a 16-bit type

using ridge::kLift;
using ridge::kSmallRow;
using ridge::loadRow;
using ridge::magnitude;
using ridge::Step;
using ridge::stepOf;
using ridge::storeRounded;
using ridge::storeRow;

typedef signed char Bytes8 __attribute__((ext_vector_type(kVec), aligned(8)));

// A value that all lanes of the wave have, in a scalar register (a wave is never of two rows).
// It saves the norm, and rows read twice, a wave a SIMD (16384 x 8192 with dequantize 242 us
// without it, 226 with it); the gated kernels of 4 vectors lose one by it.
__device__ __forceinline__ float uniform(float v) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

// A launch's arguments. They are written to device memory before it, 64 bytes at a time:
// a kernel that takes more waits for a second write, up to 0.5 us a call (a norm of 2 x 4096
// in a sequence 3.5 us, of rows apart 3.8 to 3.9). What a kernel takes beyond these counts too: it must not ask for its
// grid's size.
struct RowArgs {
    const void* x;
    int8_t* q;
    float* scale;
    int64_t ldx, strideQ;
    int rows, cols;
    __device__ int64_t ldq() const { return strideQ; }
};

// The norm's, with its 16- and 32-bit matrices contiguous (the common case, which fits) or
// with strides of their own.
template <bool DENSE>
struct NormArgs;
template <>
struct NormArgs<true> {
    const void* x;
    int8_t* q;
    float* scale;
    const void* residual;
    const void* weight;
    void* residualOut;
    int rows, cols;
    float eps;
    uint32_t strideQ16;   // in 16 bytes
    __device__ int64_t ldq() const { return (int64_t)strideQ16 * 16; }
    __device__ int64_t ldxOf() const { return cols; }
    __device__ int64_t ldResidualOf() const { return cols; }
    __device__ int64_t ldResidualOutOf() const { return cols; }
};
static_assert(sizeof(RowArgs) <= 64 && sizeof(NormArgs<true>) <= 64, "arguments of one write");
template <>
struct NormArgs<false> {
    const void* x;
    int8_t* q;
    float* scale;
    const void* residual;
    const void* weight;
    void* residualOut;
    int rows, cols;
    float eps;
    int64_t ldx, strideQ, ldResidual, ldResidualOut;
    __device__ int64_t ldq() const { return strideQ; }
    __device__ int64_t ldxOf() const { return ldx; }
    __device__ int64_t ldResidualOf() const { return ldResidual; }
    __device__ int64_t ldResidualOutOf() const { return ldResidualOut; }
};

// e^x as 2^power times what is returned, the argument reduced as Cody and Waite do: x log2(e)
// in two f32 parts, the power the whole number next to it, and what is left for the
// exponential's instruction. Its steps are not to be contracted: high - n in one step with its
// product would hold the part that low adds.
__device__ __forceinline__ float exponentialParts(float x, int& power) {
#pragma clang fp contract(off)
    constexpr float kLog2e = 1.44269504088896341f, kRest = (float)(1.44269504088896341 - (double)kLog2e);
    const float high = x * kLog2e;
    const float low = fmaf(x, kRest, fmaf(x, kLog2e, -high));
    const float n = rintf(high);
    power = (int)n;
    return __builtin_amdgcn_exp2f((high - n) + low);
}

// e^x within a unit, as expf is (the same bits for every x below 1e30), of fewer instructions:
// the ends of the range are one clamp, behind which 2^power makes infinities and zeros by
// itself, and a NaN need not come out of it (it comes out of the gate's product).
__device__ __forceinline__ float exponential(float x) {
    int power;
    const float fraction = exponentialParts(__builtin_amdgcn_fmed3f(x, -128.0f, 128.0f), power);
    return ldexpf(fraction, power);
}

// v / d for d from 1 to e^85 and a little more, rounded correctly: Newton's step on the
// reciprocal, the product, and its exact remainder's correction. Six instructions, where a
// division of any two numbers takes ten and bounded the gated activation. Larger divisors'
// reciprocals leave the normal numbers.
constexpr float kFarGate = -85.0f, kFarDivisor = 8.2e36f;   // e^85 is 8.22e36
__device__ __forceinline__ float quotient(float v, float d) {
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.0f), r, r);
    const float q = v * r;
    return fmaf(fmaf(-d, q, v), r, q);
}

// silu(g) u for g under kFarGate, where the divisor 1 + e^-g is e^-g to f32, or infinite:
// g e^g u, computed without a number that leaves the range before the result does.
// Within 3 units. (u of less than 2^-62, which may lose bits, make nothing but zeros.)
__device__ __forceinline__ float farProduct(float g, float u) {
    int power;
    const float fraction = exponentialParts(fmaxf(g, -256.0f), power);
    return ldexpf(g * (g < -256.0f ? 0.0f : fraction) * (u * 0x1p-64f), power + 64);
}

// Sources of a row's values: load() gives n of them from column col on, and adds what the
// norm sums up.
template <typename T, bool STREAM>
struct Plain {
    typedef RowArgs Args;
    static constexpr bool kNorm = false, kStream = STREAM;
    const T* x;
    __device__ Plain(const Args& a, int64_t row) : x((const T*)a.x + row * a.ldx) {}
    template <int n>
    __device__ void load(int col, float (&v)[n], float&, bool) const {
        loadRow<STREAM>(x + col, v);
    }
};

template <typename T, bool STREAM>
struct Gated {
    typedef RowArgs Args;
    static constexpr bool kNorm = false, kStream = STREAM;
    const T* x;
    int cols;
    __device__ Gated(const Args& a, int64_t row) : x((const T*)a.x + row * a.ldx), cols(a.cols) {}
    template <int n>
    __device__ void load(int col, float (&v)[n], float&, bool) const {
        float u[n];
        loadRow<STREAM>(x + col, v);
        loadRow<STREAM>(x + cols + col, u);
        float d[n], g[n], most = 0.0f;
#pragma unroll
        for (int e = 0; e < n; ++e) {
            d[e] = 1.0f + exponential(-v[e]);
            most = fmaxf(most, d[e]);
            g[e] = v[e];
            v[e] = quotient(g[e], d[e]);
        }
#pragma unroll
        for (int e = 0; e < n; ++e) v[e] *= u[e];
        // Few waves have a far gate; the whole wave turns off for one, which keeps the others'
        // loop free of exec masks (4096 x 16384 with dequantize 98.7 us, 104 us without).
        if (__builtin_amdgcn_ballot_w64(most > kFarDivisor)) {
#pragma unroll
            for (int e = 0; e < n; ++e) {
                const float far = farProduct(g[e], u[e]);
                v[e] = g[e] < kFarGate ? far : v[e];
            }
        }
    }
};

// The residual's sum leaves with the row's last reading, so that it may replace x or the
// residual.
template <typename T, typename W, bool STREAM, bool DENSE>
struct Normed {
    typedef NormArgs<DENSE> Args;
    static constexpr bool kNorm = true, kStream = STREAM;
    const T* x;
    const T* residual;
    const W* weight;
    T* out;
    __device__ Normed(const Args& a, int64_t row)
        : x((const T*)a.x + row * a.ldxOf()),
          residual(a.residual ? (const T*)a.residual + row * a.ldResidualOf() : nullptr),
          weight((const W*)a.weight),
          out(a.residualOut ? (T*)a.residualOut + row * a.ldResidualOutOf() : nullptr) {}
    template <int n>
    __device__ void load(int col, float (&v)[n], float& squares, bool last) const {
        float w[n];
        loadRow<STREAM>(x + col, v);
        if (residual) {
            float r[n];
            loadRow<STREAM>(residual + col, r);
#pragma unroll
            for (int e = 0; e < n; ++e) v[e] += r[e];
            if (last) storeRow<STREAM>(out + col, v);
        }
        loadRow<false>(weight + col, w);
#pragma unroll
        for (int e = 0; e < n; ++e) {
            squares = fmaf(v[e], v[e], squares);
            v[e] *= w[e];
        }
    }
};

// Sum and maximum over the kThreads threads of a row, in an order that depends on
// nothing but kThreads.
template <int kThreads, bool kSum>
__device__ __forceinline__ void reduceRow(float& sum, uint32_t& top) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d /= 2) {
        if (kSum) sum += __shfl_xor(sum, d);
        top = max(top, (uint32_t)__shfl_xor((int)top, d));
    }
    if constexpr (kThreads > kWave) {
        constexpr int kWaves = kThreads / kWave;
        __shared__ float sums[kWaves];
        __shared__ uint32_t tops[kWaves];
        if (threadIdx.x % kWave == 0) {
            sums[threadIdx.x / kWave] = sum;
            tops[threadIdx.x / kWave] = top;
        }
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            if (kSum) sum += sums[i];
            top = max(top, tops[i]);
        }
        __syncthreads();  // the next row's partial results go to the same places
    }
}

constexpr int64_t kMostBlocks = 1 << 20;  // of a grid: its blocks walk the rows behind them

// One row a kThreads threads. kVecs vectors a thread hold the row; with kVecs = 0 a row
// of any length is read twice.
template <typename Source, int kThreads, int kVecs>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads)
void makeRowsKernel(typename Source::Args a) {
    constexpr int kBlock = kThreads < 256 ? 256 : kThreads;
    constexpr int kRowsPerBlock = kBlock / kThreads;
    constexpr bool kHeld = kVecs > 0;
    constexpr bool kScalar = Source::kNorm || !kHeld;   // a row's results in scalar registers
    const int lane = threadIdx.x % kThreads;
    const int whole = a.cols / kVec * kVec;    // columns of whole vectors
    const int single = whole + lane;           // and this lane's behind them
    for (int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + threadIdx.x / kThreads; row < a.rows;
         row += kMostBlocks * kRowsPerBlock) {
        const Source source(a, row);
        float v[kHeld ? kVecs : 1][kVec], one[1];
        float squares = 0.0f;
        uint32_t top = 0;
        // Calls f(column, values) for each of this lane's parts of the row.
        auto parts = [&](auto&& f) {
            if constexpr (kHeld) {
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    const int col = (i * kThreads + lane) * kVec;
                    if (col < whole) f(col, v[i]);
                }
            } else {
                for (int col = lane * kVec; col < whole; col += kThreads * kVec) f(col, v[0]);
            }
            if (single < a.cols) f(single, one);
        };
        parts([&](int col, auto& values) {
            source.load(col, values, squares, kHeld);
            for (float value : values) top = max(top, magnitude(value));
        });
        reduceRow<kThreads, Source::kNorm>(squares, top);
        float root = 1.0f;
        if constexpr (Source::kNorm) {
            // A sum past the range of f32 would make the root 0 and the row silently so.
            root = squares <= FLT_MAX ? 1.0f / sqrtf(squares / (float)a.cols + a.eps) : NAN;
        }
        const float most = kScalar ? uniform(__uint_as_float(top)) : __uint_as_float(top);
        const bool small = most < kSmallRow;
        float scale;
        Step step = stepOf(most, root, scale);
        if constexpr (kScalar) step = {uniform(step.whole), uniform(step.rest), uniform(step.inverse)};
        if (lane == 0) a.scale[row] = scale;
        int8_t* const q = a.q + row * a.ldq();
        auto lift = [&](int, auto& values) {
            for (float& value : values) value *= kLift;
        };
        if (kHeld && small) parts(lift);
        parts([&](int col, auto& values) {
            if constexpr (!kHeld) {
                source.load(col, values, squares, true);
                if (small) lift(col, values);
            }
            storeRounded(q + col, values, step);
        });
    }
}

constexpr int kDequantizeThreads = 256;

template <typename T, bool STREAM>
__global__ __launch_bounds__(kDequantizeThreads)
void dequantizeKernel(const int8_t* q, int64_t ldq, const float* scale, T* out, int64_t ldOut, int rows, int cols,
                      int pieces) {
    const int64_t total = (int64_t)rows * pieces;
    for (int64_t i = blockIdx.x; i < total; i += kMostBlocks) {
        const int row = (int)(i / pieces);
        const int col = ((int)(i % pieces) * kDequantizeThreads + (int)threadIdx.x) * kVec;
        if (col >= cols) continue;
        const Bytes8 b = *(const Bytes8*)(q + row * ldq + col);  // rows are readable to a multiple of 16
        const float s = scale[row];
        float v[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] = (float)b[e] * s;
        T* const at = out + row * ldOut + col;
        if (col + kVec <= cols) {
            storeRow<STREAM>(at, v);
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (col + e < cols) at[e] = (T)v[e];
        }
    }
}

// 16- and 32-bit matrices of this size and more are read and written past the caches: who
// comes next would not find them there, and the 8-bit rows, which the next product reads,
// stay. us, cached | past the caches, the norm of bfloat16 and a reader of its rows: 16384 x
// 8192 249 | 220, 4096 x 16384 137 | 123, 2048 x 4096 18.5 | 22.3.
constexpr int64_t kStreamBytes = (int64_t)64 << 20;

template <typename Source, int kThreads, int kVecs>
hipError_t launchRows(const typename Source::Args& a, hipStream_t stream) {
    constexpr int kBlock = kThreads < 256 ? 256 : kThreads;
    constexpr int kRowsPerBlock = kBlock / kThreads;
    const int64_t blocks = std::min<int64_t>((a.rows + (int64_t)kRowsPerBlock - 1) / kRowsPerBlock, kMostBlocks);
    return ridge::launchKernel(makeRowsKernel<Source, kThreads, kVecs>, (unsigned)blocks, kBlock, stream, a);
}

// The threads of a row, by its length: as many as hold it in at most four vectors each. A
// norm's 1024 threads have not got the registers for that: it reads rows of more than
// 16384 columns twice. Few rows leave CUs to spare and take more threads and fewer vectors
// each, which also is less code to run through once: us in a graph, silu of float16 as for
// many rows | so: 13 x 2048 4.4 | 3.0, 4 x 8192 4.6 | 4.1, 500 x 8192 7.6 | 7.4; but 600 x 8192
// 9.3 | 9.7, 4000 x 4096 18.9 | 22.9, 8000 x 600 10.5 | 13.7. Not the norm, whose sum would be added up in another order: a row's result must
// not depend on how many rows there are.
constexpr int kFewRows = 512;
template <typename Source>
hipError_t launchByLength(const typename Source::Args& a, hipStream_t stream) {
    if (a.cols <= 64 * kVec) return launchRows<Source, 64, 1>(a, stream);
    if constexpr (!Source::kNorm && !Source::kStream) {   // no few rows of these lengths are that large
        if (a.rows <= kFewRows && a.cols <= 256 * kVec) return launchRows<Source, 256, 1>(a, stream);
        if (a.rows <= kFewRows && a.cols <= 512 * kVec * 2) return launchRows<Source, 512, 2>(a, stream);
    }
    if (a.cols <= 64 * kVec * 4) return launchRows<Source, 64, 4>(a, stream);
    if (a.cols <= 256 * kVec * 4) return launchRows<Source, 256, 4>(a, stream);
    if (a.cols <= 512 * kVec * 4) return launchRows<Source, 512, 4>(a, stream);
    if constexpr (!Source::kNorm) {
        if (a.cols <= 1024 * kVec * 4) return launchRows<Source, 1024, 4>(a, stream);
    }
    return launchRows<Source, 1024, 0>(a, stream);
}

bool isType(int type) { return type == RIDGE_F16 || type == RIDGE_BF16 || type == RIDGE_F32; }

bool aligned(const void* p, size_t to) { return p != nullptr && ((uintptr_t)p & (to - 1)) == 0; }

size_t sizeOf(int type) { return type == RIDGE_F32 ? 4 : 2; }

// What every maker of rows asks for: sizes within 31 bits, strides of at least a row,
// and 8-bit rows at multiples of 16 bytes.
bool rowsFit(const void* x, int64_t ldx, int64_t width, int type, const int8_t* q, int64_t ldq, const float* scale,
             int64_t rows, int64_t cols) {
    return isType(type) && rows <= INT32_MAX && cols > 0 && width <= INT32_MAX - 65536 && ldx >= width &&
           ldq >= cols && ldq % 16 == 0 && aligned(x, sizeOf(type)) && aligned(q, 16) && aligned(scale, 4);
}

bool streams(int64_t rows, int64_t cols, int type) { return rows * cols >= kStreamBytes / (int64_t)sizeOf(type); }

template <template <typename, bool> class Source, typename T>
hipError_t launchPlain(const RowArgs& a, bool stream, hipStream_t s) {
    return stream ? launchByLength<Source<T, true>>(a, s) : launchByLength<Source<T, false>>(a, s);
}

template <template <typename, bool> class Source>
hipError_t launchTyped(const RowArgs& a, int type, bool stream, hipStream_t s) {
    switch (type) {
        case RIDGE_F16: return launchPlain<Source, _Float16>(a, stream, s);
        case RIDGE_BF16: return launchPlain<Source, __bf16>(a, stream, s);
        default: return launchPlain<Source, float>(a, stream, s);
    }
}

template <typename T, typename W>
hipError_t launchNorm(const NormArgs<false>& a, bool stream, hipStream_t s) {
    if (stream) return launchByLength<Normed<T, W, true, false>>(a, s);
    const NormArgs<true> d = {a.x, a.q, a.scale, a.residual, a.weight, a.residualOut, a.rows, a.cols, a.eps,
                              (uint32_t)(a.strideQ / 16)};
    const bool dense = a.rows == 1 || (a.ldx == a.cols && a.strideQ / 16 <= UINT32_MAX &&
                                       (!a.residual || (a.ldResidual == a.cols && a.ldResidualOut == a.cols)));
    return dense ? launchByLength<Normed<T, W, false, true>>(d, s) : launchByLength<Normed<T, W, false, false>>(a, s);
}

template <typename T>
hipError_t launchDequantize(const int8_t* q, int64_t ldq, const float* scale, void* out, int64_t ldOut, int rows,
                            int cols, bool stream, hipStream_t s) {
    const int pieces = (int)(((int64_t)cols + kDequantizeThreads * kVec - 1) / (kDequantizeThreads * kVec));
    const unsigned blocks = (unsigned)std::min<int64_t>((int64_t)rows * pieces, kMostBlocks);
    return ridge::launchKernel(stream ? dequantizeKernel<T, true> : dequantizeKernel<T, false>, blocks,
                               kDequantizeThreads, s, q, ldq, scale, (T*)out, ldOut, rows, cols, pieces);
}

}  // namespace

extern "C" int ridge_int8_quantize(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale,
                                   int64_t rows, int64_t cols, void* stream) {
    if (rows == 0 && cols > 0 && isType(type)) return hipSuccess;
    if (rows < 0 || !rowsFit(x, ldx, cols, type, q, ldq, scale, rows, cols)) return hipErrorInvalidValue;
    const RowArgs a = {x, q, scale, ldx, ldq, (int)rows, (int)cols};
    return launchTyped<Plain>(a, type, streams(rows, cols, type), (hipStream_t)stream);
}

extern "C" int ridge_int8_silu_mul(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale,
                                   int64_t rows, int64_t cols, void* stream) {
    if (rows == 0 && cols > 0 && isType(type)) return hipSuccess;
    if (rows < 0 || cols > INT32_MAX / 2 || !rowsFit(x, ldx, 2 * cols, type, q, ldq, scale, rows, cols))
        return hipErrorInvalidValue;
    const RowArgs a = {x, q, scale, ldx, ldq, (int)rows, (int)cols};
    return launchTyped<Gated>(a, type, streams(rows, 2 * cols, type), (hipStream_t)stream);
}

extern "C" int ridge_int8_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldResidual,
                                   const void* weight, int weightType, float eps, int type, void* residualOut,
                                   int64_t ldResidualOut, int8_t* q, int64_t ldq, float* scale, int64_t rows,
                                   int64_t cols, void* stream) {
    if (!isType(type) || (weightType != type && weightType != RIDGE_F32) || !(eps > 0.0f && eps <= FLT_MAX) ||
        (residual == nullptr) != (residualOut == nullptr))
        return hipErrorInvalidValue;
    if (rows == 0 && cols > 0) return hipSuccess;
    if (rows < 0 || !rowsFit(x, ldx, cols, type, q, ldq, scale, rows, cols) || !aligned(weight, sizeOf(weightType)))
        return hipErrorInvalidValue;
    if (residual && (!aligned(residual, sizeOf(type)) || !aligned(residualOut, sizeOf(type)) || ldResidual < cols ||
                     ldResidualOut < cols))
        return hipErrorInvalidValue;
    const NormArgs<false> a = {x,         q,         scale, residual, weight, residualOut, (int)rows,
                               (int)cols, eps,       ldx,   ldq,      ldResidual, ldResidualOut};
    const bool past = streams(rows, cols, type);
    hipStream_t s = (hipStream_t)stream;
    switch (type) {
        case RIDGE_F16:
            return weightType == type ? launchNorm<_Float16, _Float16>(a, past, s) : launchNorm<_Float16, float>(a, past, s);
        case RIDGE_BF16:
            return weightType == type ? launchNorm<__bf16, __bf16>(a, past, s) : launchNorm<__bf16, float>(a, past, s);
        default: return launchNorm<float, float>(a, past, s);
    }
}

extern "C" int ridge_int8_dequantize(const int8_t* q, int64_t ldq, const float* scale, void* out, int64_t ldOut,
                                     int type, int64_t rows, int64_t cols, void* stream) {
    if (rows == 0 && cols > 0 && isType(type)) return hipSuccess;
    if (rows < 0 || !rowsFit(out, ldOut, cols, type, q, ldq, scale, rows, cols)) return hipErrorInvalidValue;
    const bool past = streams(rows, cols, type);
    const int r = (int)rows, c = (int)cols;
    hipStream_t s = (hipStream_t)stream;
    switch (type) {
        case RIDGE_F16: return launchDequantize<_Float16>(q, ldq, scale, out, ldOut, r, c, past, s);
        case RIDGE_BF16: return launchDequantize<__bf16>(q, ldq, scale, out, ldOut, r, c, past, s);
        default: return launchDequantize<float>(q, ldq, scale, out, ldOut, r, c, past, s);
    }
}
