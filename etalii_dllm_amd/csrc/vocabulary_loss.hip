// The loss over the vocabulary from the last hidden states, and its gradients, without keeping the logits.
//
//   x = scale h.w     z = cap tanh(x / cap)     lse = log sum exp z     loss = lse - z[target]
//   g = (exp(z - lse) - onehot) dloss scale (1 - tanh^2)     dh = g W     dW = g^T h
//
// Only rows that count (a target inside the vocabulary) are worked on: they are listed first, and their hidden states gathered
// into whole 16-byte chunks, zeroes behind.
//
// Float32 values are multiplied as pairs of float16, three products: 22 bits and more of each value, off by 2^-39 of the largest at
// most: hidden states are scaled by the power of two that brings their row's largest value to the top of float16's range, weights
// by that of kScaleRows of them. Probabilities, times 2^14, are off by 2^-39 at most whatever their size, which leaves those of
// 2^-17 their 22 bits, those of 1e-8 12 and those below 2^-39 none: a power of two for each of the vocabulary, from its largest
// probability, would take the logits twice. (Three bfloat16 parts, six products, hold values of any size and take twice as long:
// gradients of 1020 rows, 49152 x 576, 1.6 ms.)
//
// Forward: tiles of logits on the matrix cores, vocabulary by rows, so that a lane owns a row of the batch; a tile leaves each
// row's largest logit and sum of exponentials of 128 of the vocabulary, which a last launch joins in a fixed order. The target's
// logit is formed where the rows are gathered, and goes into the sum as it is.
//
// Backward, a piece of the vocabulary at a time: the logits again, whose epilogue stores the softmax's part of g in the product's
// type; then its products with the weights and with the hidden states. (For that rounding dW's rows of tokens that are no target
// are off by 1.3 to 1.4 times their own. Up to kPairedRows rows, whose products wait for the weights' bytes, have what it leaves
// too, as further rows of the softmax, beside the hidden states once more: 37 rows, 151936 x 896, 265 to 286 us.) dh is added up in
// float32 over units of the vocabulary that go by its size alone, whatever the batch, so a row's bits are its own. The target's
// element c = expm1(z - lse) ... stays out of the 16-bit products: p - 1 is what is left of two near numbers where the model is
// sure, and with a uniform dloss its rounding would not average out. c W[target] is added to dh in float32, and the sums of c h by
// target (token_rows.h) to dW in the epilogue.
//
// Bound and measured. 8192 rows, 151936 x 1536 in bfloat16, forward 3.5 ms: 1090 TFLOP/s, matrix cores 52% busy at 1.7 GHz, to which
// power lowers the clock; gradients 11.5 ms: the logits again and their epilogue 0.43 ms for 16384 of the vocabulary (890
// TFLOP/s, matrix cores 43% busy, vector units 26%), both products 0.76 (1090). 1020 rows, 49152 x 576 in float32, gradients 0.69 ms,
// three products for each: 250 TFLOP/s of float32's. 37 rows, 151936 x 896 in bfloat16, forward 68 us: the weights once, 49 us
// (5.5 TB/s), and two launches. Weights that have to be packed first cost their reading and writing.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "dllm_hip.h"
#include "element.h"
#include "softcap.h"
#include "tile_product.h"
#include "token_rows.h"
#include "workspace.h"

using namespace dllm_hip;

namespace {

constexpr int64_t kPackPiece = 16384;  // of the vocabulary: weights packed at once, where they are
constexpr int kStatRows = 128;        // of the vocabulary: one maximum and sum
constexpr int64_t kFewRows = 256;
constexpr size_t kPieceBytes = size_t{1} << 28;
constexpr int64_t kStrideSlack = 64;  // elements between the softmax's rows: their stride is no power of two, which would meet on few channels
constexpr int kHalfShift = 14;  // float16 holds the softmax's part of g times 2^14, relative to the row's weight
constexpr int kTop = 15;        // pairs of float16 hold values up to 2^15
constexpr int64_t kScaleRows = 2048;  // of the vocabulary, that share a scale

// What the products read of a type: kLossPlanes parts of a value.
template <typename T>
struct LossProduct {
    using Part = T;
};
template <>
struct LossProduct<float> {
    using Part = _Float16;
};
template <typename T>
using LossPart = typename LossProduct<T>::Part;
template <typename T>
constexpr int kLossPlanes = sizeof(T) == 4 ? 2 : 1;
template <typename T>
constexpr bool kHalfParts = __is_same(LossPart<T>, _Float16);
template <typename T>
constexpr bool kScaled = sizeof(T) == 4;

constexpr int64_t kPairedRows = 64;
inline bool paired_rows(int64_t rows, int64_t dtype) { return rows <= kPairedRows && dtype != kFloat32; }

// Bytes of a row of n values.
template <typename T>
constexpr int64_t row_bytes(int64_t n) {
    return static_cast<int64_t>(round_up(n, kRowMultiple<kLossPlanes<T>>)) * 2 * kLossPlanes<T>;
}

// Float32 values as they are, 8 from column c on; a row takes as many bytes as one of pairs.
__device__ __forceinline__ void store_as_they_are(char* row, int64_t c, const float (&v)[8]) {
    float4* const to = reinterpret_cast<float4*>(row + c * 4);
    to[0] = {v[0], v[1], v[2], v[3]}, to[1] = {v[4], v[5], v[6], v[7]};
}

// 8 values of a row from column c on
template <typename T>
__device__ __forceinline__ void store_parts(char* row, int64_t c, const float (&v)[8]) {
    store_eight<LossPart<T>, kLossPlanes<T>>(row + value_at<kLossPlanes<T>>(c), v);
}

struct LossShape {
    int64_t rows, vocabulary, dim, padded, row;  // padded: dim in whole chunks; row: bytes of a packed one
    int64_t hidden_stride, dhidden_stride;
    float scale, softcap;
};

// ---- which rows count ----

// list[0 .. count): the rows whose target is inside, ascending; zeroes for the others.
__global__ __launch_bounds__(1024) void keep_rows_kernel(const int64_t* __restrict__ targets, int64_t n, int64_t vocabulary,
                                                         uint32_t* __restrict__ list, uint32_t* __restrict__ count, float* __restrict__ loss,
                                                         float* __restrict__ lse) {
    __shared__ uint32_t of_wave[16];
    const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
    uint32_t before = 0;
    for (int64_t base = 0; base < n; base += 1024) {
        const int64_t i = base + threadIdx.x;
        const bool inside = i < n && targets[i] >= 0 && targets[i] < vocabulary;
        const uint64_t mask = __ballot(inside);
        if (lane == 0) of_wave[wave] = __popcll(mask);
        __syncthreads();
        uint32_t at = before;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) at += of_wave[w];
            before += of_wave[w];
        }
        if (inside) list[at + __popcll(mask & ((uint64_t{1} << lane) - 1))] = static_cast<uint32_t>(i);
        if (i < n && !inside) {
            if (loss) loss[i] = 0.0f;
            if (lse) lse[i] = 0.0f;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *count = before;
}

// ---- packing ----

// The least e with |x| < 2^e for the float32 of these bits, x >= 0; 0 for zero.
__device__ __forceinline__ int exponent_of(int32_t bits) {
    int e = 0;
    if (bits != 0) frexpf(__builtin_bit_cast(float, bits), &e);
    return e;
}

// The bits of x's size, which grow with it; zero for what is not finite.
__device__ __forceinline__ uint32_t size_bits(float x) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
    return bits < 0x7f800000u ? bits : 0;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), s)));
    return v;
}

// The bits of the largest size of each kScaleRows rows, which are -1 before. (A maximum, so the order does not matter.)
constexpr int kSizeRows = 64;
template <int kWidth>
__global__ __launch_bounds__(256) void unit_sizes_kernel(const float* __restrict__ src, int64_t rows, int64_t dim, int32_t* __restrict__ sizes) {
    __shared__ uint32_t of_wave[4];
    const int64_t first = block_id() * kSizeRows;
    if (first >= rows) return;
    const int64_t n = min(rows - first, static_cast<int64_t>(kSizeRows)) * dim / kWidth;
    const float* const from = src + first * dim;
    uint32_t top = 0;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        float v[kWidth];
        load_as_float<float, kWidth>(from + i * kWidth, v);
#pragma unroll
        for (int e = 0; e < kWidth; ++e) top = max(top, size_bits(v[e]));
    }
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0)
        atomicMax(sizes + first / kScaleRows, static_cast<int>(max(max(of_wave[0], of_wave[1]), max(of_wave[2], of_wave[3]))));
}

// 8 elements of a row from column d on, zeroes past dim. kWhole: the row is whole 16-byte chunks.
template <typename T, bool kWhole>
__device__ __forceinline__ void load_eight(const T* row, int64_t d, int64_t dim, float (&v)[8]) {
    if constexpr (kWhole) {
#pragma unroll
        for (int p = 0; p < 8; p += kChunk<T>) {
            float w[kChunk<T>];
            load_as_float<T, kChunk<T>>(row + d + p, w);
#pragma unroll
            for (int e = 0; e < kChunk<T>; ++e) v[p + e] = w[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = d + e < dim ? static_cast<float>(row[d + e]) : 0.0f;
    }
}

// What scales a row by a power of two: nothing (kAsTheyAre: and float32 stays that), the size of its unit (weights), or its part in dW
// (hidden states): factor's exponent from the largest of that and the row's, so that the largest values are below 2^kTop; zero for none.
enum PackScale { kNoScale, kAsTheyAre, kUnitScale, kWeightScale };
constexpr int kNoWeight = -1000;      // the exponent of a factor of zero
constexpr int kExponentBase = 1000;  // the largest exponent is held with this added, -1 before any

struct PackArgs {
    const uint32_t *list, *count;
    int64_t n, dim, stride, chunks, row;
    const int32_t *exponent, *largest, *sizes;
    bool twice;  // the rows once more behind the last one
};

// Row list[j] (j itself without a list) of src as chunks of 8 values' parts.
template <typename T, bool kWhole, PackScale kScale>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ src, char* __restrict__ dst, PackArgs a) {
    const int64_t i = block_id() * 256 + threadIdx.x;
    const int64_t j = i / a.chunks, c = i - j * a.chunks;
    const int64_t n = a.count ? static_cast<int64_t>(*a.count) : a.n;
    if (j >= n) return;
    float v[8];
    load_eight<T, kWhole>(src + (a.list ? static_cast<int64_t>(a.list[j]) : j) * a.stride, c * 8, a.dim, v);
    if constexpr (kScale == kAsTheyAre) return store_as_they_are(dst + j * a.row, c * 8, v);
    if constexpr (kScale != kNoScale) {
        int by;
        if constexpr (kScale == kUnitScale) {
            by = kTop - exponent_of(a.sizes[j / kScaleRows]);
        } else {
            const int e = a.exponent[j];
            by = e == kNoWeight ? 2 * kNoWeight : e - (*a.largest - kExponentBase) + kTop;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], by);
    }
    store_parts<T>(dst + j * a.row, c * 8, v);
    if (kScale == kWeightScale && a.twice) store_parts<T>(dst + (n + j) * a.row, c * 8, v);
}

template <typename T, PackScale kScale>
int launch_pack(const T* src, char* dst, const PackArgs& args, hipStream_t stream) {
    PackArgs a = args;
    a.row = row_bytes<T>(a.dim);
    a.chunks = static_cast<int64_t>(ceil_div(a.dim, 8));
    const bool whole = a.dim % 8 == 0 && a.stride % kChunk<T> == 0 && aligned_to(src, 16);
    const dim3 grid = grid_of(ceil_div(a.n * a.chunks, 256));
    if (whole)
        pack_kernel<T, true, kScale><<<grid, 256, 0, stream>>>(src, dst, a);
    else
        pack_kernel<T, false, kScale><<<grid, 256, 0, stream>>>(src, dst, a);
    return check_launch("vocabulary_loss packing");
}

// ---- logits ----

// A logit from its product, and the cap's derivative.
struct Cap {
    float scale, softcap, in;
    __device__ __forceinline__ explicit Cap(const LossShape& s) : scale(s.scale), softcap(s.softcap), in(0.0f) {
        if (softcap != 0.0f) in = scale / softcap;
    }
    template <bool kCapped>
    __device__ __forceinline__ float logit(float x, float& derivative) const {
        derivative = 1.0f;
        if constexpr (!kCapped) return x * scale;
        return softcap * tanh_of_any_size(x * in, derivative);
    }
};

// ---- the listed rows ----

// What a row's gradient is formed from, by its place in the list.
struct RowTerms {
    float *lse, *factor;
    int32_t* target;
    int32_t* exponent;      // float16 parts: factor holds the weight's mantissa, this the power of two left out
    int32_t* row_exponent;  // float32: of the hidden states
};

struct RowsArgs {
    LossShape s;
    uint32_t *list, *count;  // kFind: written here
    char* packed;
    bool twice;  // packed: the rows once more behind the last one
    int32_t* row_exponent;  // float32: NULL: the values as they are
    // the forward's
    const int64_t* targets;
    float* at_target;  // by the place in the list
    // kFind
    float *loss_out, *lse_out;
    int32_t* sizes;  // set to -1
    int64_t units;
    // the backward's
    TokenOrder order;
    const float *lse, *dloss;
    RowTerms terms;
    float* coefficient;  // by row
    int32_t* largest;    // float16 parts: kExponentBase and the largest exponent of a factor and its row together
};

// factor = mantissa 2^exponent, mantissa in [1, 2)
__device__ __forceinline__ void take_apart(float factor, float& mantissa, int& exponent) {
    int e = 0;
    mantissa = factor;
    if (factor != 0.0f && isfinite(factor)) mantissa = 2.0f * frexpf(factor, &e), e -= 1;
    exponent = factor == 0.0f ? kNoWeight : e;
}

enum RowsOf { kListed, kFind, kBackward };
template <RowsOf kOf>
constexpr int kRowsThreads = kOf == kFind ? 1024 : 256;
constexpr int64_t kFindRows = 16384;  // the most that every workgroup counts through for itself

// A wave to a listed row: its hidden state in parts, and its target's logit, from a product in float32 added up by 64 lanes; of the
// backward, the target's element and what the softmax's epilogue reads. kFind: the workgroup lists its 16 rows itself, by counting the rows before them.
template <typename T, bool kWhole, bool kCapped, RowsOf kOf>
__global__ __launch_bounds__(kRowsThreads<kOf>) void rows_kernel(const T* __restrict__ hidden, const T* __restrict__ weight, RowsArgs a) {
    constexpr int kThreads = kRowsThreads<kOf>, kWaves = kThreads / kWave;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), lane = static_cast<int>(threadIdx.x) & 63;
    const int64_t first = block_id() * kWaves;
    int64_t j = first + wave, row;
    if constexpr (kOf == kFind) {
        const auto counts = [&](int64_t i) {
            const int64_t t = i < a.s.rows ? a.targets[i] : -1;
            return t >= 0 && t < a.s.vocabulary;
        };
        int64_t before = 0;
        for (int64_t base = 0; base < first; base += kThreads) before += __syncthreads_count(base + threadIdx.x < first && counts(base + threadIdx.x));
        const uint64_t mask = __ballot(lane < kWaves && counts(first + lane));
        if (block_id() == 0)
            for (int64_t i = threadIdx.x; i < a.units; i += kThreads) a.sizes[i] = -1;
        if (first >= a.s.rows) return;
        if (first + kWaves >= a.s.rows && threadIdx.x == 0) *a.count = static_cast<uint32_t>(before + __popcll(mask));
        row = first + wave;
        if (!(mask >> wave & 1)) {
            if (row < a.s.rows && lane == 0) {
                if (a.loss_out) a.loss_out[row] = 0.0f;
                if (a.lse_out) a.lse_out[row] = 0.0f;
            }
            return;
        }
        j = before + __popcll(mask & ((uint64_t{1} << wave) - 1));
        if (lane == 0) a.list[j] = static_cast<uint32_t>(row);
    } else {
        if (j >= static_cast<int64_t>(*a.count)) return;
        row = a.list[j];
    }
    const T* const h = hidden + row * a.s.hidden_stride;
    const int64_t target = kOf == kBackward ? static_cast<int64_t>(a.order.token[j]) : a.targets[row];
    const T* const w = weight + target * a.s.dim;
    uint32_t size = 0;  // of the row's largest value
    int exponent = 0;
    const bool scaled = kScaled<T> && a.row_exponent;
    if (scaled) {
        for (int64_t d = lane; d < a.s.dim; d += kWave) size = max(size, size_bits(h[d]));
        size = wave_max(size);
        exponent = exponent_of(static_cast<int32_t>(size));
        if (lane == 0) a.row_exponent[j] = exponent;
    }
    float x = 0.0f;
    for (int64_t d = lane * 8; d < a.s.padded; d += kWave * 8) {
        float v[8], u[8];
        load_eight<T, kWhole>(h, d, a.s.dim, v);
        load_eight<T, kWhole>(w, d, a.s.dim, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fmaf(v[e], u[e], x);
        if constexpr (kOf == kBackward && kHalfParts<T> && !kScaled<T>) {
#pragma unroll
            for (int e = 0; e < 8; ++e) size = max(size, size_bits(v[e]));
        }
        if constexpr (kScaled<T>) {
            if (!scaled) {
                store_as_they_are(a.packed + j * a.s.row, d, v);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], kTop - exponent);
        }
        store_parts<T>(a.packed + j * a.s.row, d, v);
        if (kOf == kBackward && !kHalfParts<T> && a.twice) store_parts<T>(a.packed + (*a.count + j) * a.s.row, d, v);
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) x += __shfl_xor(x, s);
    if constexpr (kOf == kBackward && kHalfParts<T> && !kScaled<T>) {
        size = wave_max(size);
        exponent = exponent_of(static_cast<int32_t>(size));
    }
    if (lane != 0) return;
    float derivative;
    const float z = Cap(a.s).logit<kCapped>(x, derivative);
    if constexpr (kOf != kBackward) {
        a.at_target[j] = z;
    } else {
        const float lse = a.lse[row], factor = a.dloss[row] * a.s.scale;
        a.coefficient[row] = expm1f(z - lse) * derivative * factor;
        a.terms.lse[j] = lse;
        a.terms.target[j] = static_cast<int32_t>(target);
        if constexpr (kHalfParts<T>) {
            float mantissa;
            int e;
            take_apart(factor, mantissa, e);
            a.terms.factor[j] = ldexpf(mantissa, kHalfShift);
            a.terms.exponent[j] = e;
            // a row of zeroes is zeroes by any power, and does not take the others' bits. (A maximum, so the order does not matter.)
            if (e != kNoWeight && size != 0) atomicMax(a.largest, e + exponent + kExponentBase);
        } else {
            a.terms.factor[j] = factor;
        }
    }
}

template <typename T, RowsOf kOf>
int launch_rows(const T* hidden, const T* weight, const RowsArgs& a, hipStream_t stream) {
    constexpr int kThreads = kRowsThreads<kOf>;
    const dim3 grid = grid_of(ceil_div(a.s.rows, kThreads / kWave));
    const bool whole = a.s.dim % 8 == 0 && a.s.hidden_stride % kChunk<T> == 0 && aligned_to(hidden, 16) && aligned_to(weight, 16);
    const bool capped = a.s.softcap != 0.0f;
    if (whole && capped)
        rows_kernel<T, true, true, kOf><<<grid, kThreads, 0, stream>>>(hidden, weight, a);
    else if (whole)
        rows_kernel<T, true, false, kOf><<<grid, kThreads, 0, stream>>>(hidden, weight, a);
    else if (capped)
        rows_kernel<T, false, true, kOf><<<grid, kThreads, 0, stream>>>(hidden, weight, a);
    else
        rows_kernel<T, false, false, kOf><<<grid, kThreads, 0, stream>>>(hidden, weight, a);
    return check_launch("vocabulary_loss rows");
}

// ---- tiles ----

// The products' tiles by the number of rows. 256 x 256 by eight waves, one workgroup to a CU; 128 x 128 by four, two to a CU, where
// the large ones would leave CUs without work or pad much; and for up to 64 rows, whose products wait for the weights'
// bytes, tiles of 64 rows. The forward's waves hold kStatRows of the vocabulary in all of them. (The gradients' large tiles of float32 spill
// three registers, outside their loop over k.)
//
// Float32's forward of up to kFewRows rows multiplies the values as they are (DirectTile): packing the weights reads them
// twice and stores them, which takes as long as the float32 products of some 250 rows (3 rows, 151936 x 1536: 257 us instead of 1240).
template <typename T, bool kAColumns, bool kBColumns, int kM, int kN, int kWavesM, int kWavesN, int kStages = 2>
using Product64 = TileProduct<LossPart<T>, kLossPlanes<T>, kM, kN, kWavesM, kWavesN, kAColumns, kBColumns, kStages>;

template <typename T>
struct LargeTiles {
    using Forward = Product64<T, false, false, 256, 256, 2, 4>;
    using Logits = Product64<T, false, false, 256, 256, 2, 4>;
    using Hidden = Product64<T, false, true, 256, 256, 2, 4>;
    using Weight = Product64<T, true, true, 256, 256, 2, 4>;
};
template <typename T>
struct MiddleTiles {
    using Forward = Product64<T, false, false, 256, 128, 2, 4>;  // of 16-bit types, as SmallTiles'
    using Logits = Product64<T, false, false, 128, 128, 2, 2>;
    using Hidden = Product64<T, false, true, 128, 128, 2, 2>;
    using Weight = Product64<T, true, true, 128, 128, 2, 2>;
};
template <typename T>
struct SmallTiles {
    using Forward = Product64<T, false, false, 128, 64, 1, 2>;
    using Logits = Product64<T, false, false, 64, 256, 1, 4>;
    using Hidden = Product64<T, false, true, 64, 64, 2, 2, 4>;
    using Weight = Product64<T, true, true, 128, 128, 2, 2>;
};

template <int kN, int kWavesM, int kWavesN>
using DirectTile = TileProduct<float, 1, kStatRows * kWavesM, kN, kWavesM, kWavesN, false, false>;

// Tiles of the rows that count, of those that the launch has for all rows. The others' workgroups come last and end, so that every XCD
// has as much to do (2047 rows of which 1228 count, 256000 x 2304: dh's tiles took 2.7 ms instead of 2.0 where four XCDs had them).
template <int kSize>
__device__ __forceinline__ int64_t tiles_that_count(int64_t count, int64_t tiles) {
    return min(tiles, (count + kSize - 1) / kSize);
}

// ---- forward ----

struct Stat {
    float top, sum;  // sum of exp(z - top); top -infinity: none
};

__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
    const float top = fmaxf(a.top, b.top), base = top == -INFINITY ? 0.0f : top;
    return {top, a.sum * __builtin_amdgcn_exp2f((a.top - base) * kLog2E) + b.sum * __builtin_amdgcn_exp2f((b.top - base) * kLog2E)};
}

struct ForwardArgs {
    LossShape s;
    Operand weight, hidden;
    int64_t k;      // values of a row that are read
    int64_t first;  // of the piece, in the vocabulary; weight.count: of the piece
    const uint32_t *list, *count;
    const int64_t* targets;
    Stat* stats;  // [unit of kStatRows][rows]
    const float* at_target;  // by the place in the list
    const int32_t* exponent;  // float32: by the place in the list
    const int32_t* sizes;     // float32: of the piece, by kScaleRows
};

template <typename T, bool kCapped, typename Tile>
__global__ __launch_bounds__(Tile::kThreads) void forward_kernel(ForwardArgs a, int64_t m_tiles, int64_t n_tiles) {
    static_assert(Tile::kWaveM == kStatRows);
    constexpr bool kScales = sizeof(T) != sizeof(typename Tile::Part);
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    const int64_t count = *a.count;
    int64_t m, n;
    n_tiles = tiles_that_count<Tile::kN>(count, n_tiles);
    if (block_id() >= m_tiles * n_tiles) return;
    tile_of(block_id(), m_tiles, n_tiles, m, n);
    typename Tile::Sums acc;
    Tile::run(a.weight, a.hidden, m * Tile::kM, n * Tile::kN, a.weight.count, count, a.k, 0, 0, (LdsByte*)lds, acc);
    const int64_t m0 = m * Tile::kM + Tile::wave_m(), n0 = n * Tile::kN + Tile::wave_n();
    if (m0 >= a.weight.count) return;
    const int64_t unit = (a.first + m0) / kStatRows;
    const int valid = static_cast<int>(min(a.weight.count - m0, static_cast<int64_t>(kStatRows)));
    const Cap cap(a.s);
    static_assert(kScaleRows % Tile::kM == 0);
    const int weight_exponent = kScales ? exponent_of(a.sizes[m * Tile::kM / kScaleRows]) - 2 * kTop : 0;
#pragma unroll
    for (int j = 0; j < Tile::kBlocksN; ++j) {
        const int64_t row = n0 + 32 * j + lane_column();
        const int by = kScales ? weight_exponent + a.exponent[min(row, count - 1)] : 0;
        const int target = row < count ? static_cast<int>(a.targets[a.list[row]] - a.first - m0) : -1;
        const bool any = __ballot(target >= 0 && target < kStatRows) != 0;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < Tile::kBlocksM; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float unused, x = acc[i][j][r];
                if constexpr (kScales) x = ldexpf(x, by);
                acc[i][j][r] = cap.logit<kCapped>(x, unused);
            }
            __builtin_amdgcn_sched_barrier(0);  // one block's values at a time: all of them do not fit the registers
        }
        if (valid < kStatRows) {
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 32 * i + block_row(r) < valid ? acc[i][j][r] : -INFINITY;
        }
        if (any) {
            // the sum has the target's logit as the loss subtracts it: what is left where the model is sure is then not their rounding
            const float known = a.at_target[min(row, count - 1)];
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 32 * i + block_row(r) == target ? known : acc[i][j][r];
        }
#pragma unroll
        for (int i = 0; i < Tile::kBlocksM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][j][r]);
        top = fmaxf(top, other_half(top));
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < Tile::kBlocksM; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f((acc[i][j][r] - base) * kLog2E);
            __builtin_amdgcn_sched_barrier(0);
        }
        sum += other_half(sum);
        if (row < count && lane_half() == 0) a.stats[unit * a.s.rows + row] = {top, sum};
    }
}

// Joins a row's statistics: 64 threads take every 64th unit, then the threads' in a fixed tree. 16 rows to a workgroup read whole lines
// (8192 rows, 151936 of the vocabulary: 51 us with 4); where rows are few, more workgroups of 4 do.
template <int kJoinRows>
__global__ __launch_bounds__(64 * kJoinRows) void join_stats_kernel(const Stat* __restrict__ stats, const float* __restrict__ at_target, int64_t units,
                                                         int64_t rows, const uint32_t* __restrict__ list, const uint32_t* __restrict__ count,
                                                         float* __restrict__ loss, float* __restrict__ lse) {
    __shared__ Stat of[64][kJoinRows];
    const int64_t n = *count, first = block_id() * kJoinRows;
    if (first >= n) return;
    const int part = static_cast<int>(threadIdx.x) / kJoinRows, which = static_cast<int>(threadIdx.x) % kJoinRows;
    const int64_t row = min(first + which, n - 1);
    Stat s = {-INFINITY, 0.0f};
    constexpr int kAhead = 8;
    for (int64_t u = part; u < units; u += 64 * kAhead) {
        Stat v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = u + 64 * k < units ? stats[(u + 64 * k) * rows + row] : Stat{-INFINITY, 0.0f};
#pragma unroll
        for (int k = 0; k < kAhead; ++k) s = join(s, v[k]);
    }
    of[part][which] = s;
    for (int step = 32; step > 0; step >>= 1) {
        __syncthreads();
        if (part < step) of[part][which] = s = join(s, of[part + step][which]);
    }
    if (part == 0 && first + which < n) {
        const float rest = kLn2 * __builtin_amdgcn_logf(s.sum);
        if (lse) lse[list[row]] = s.top + rest;
        if (loss) loss[list[row]] = s.top - at_target[row] + rest;  // the large numbers' difference first, which is exact where they are near
    }
}

// ---- backward ----

struct SoftmaxArgs {
    LossShape s;
    Operand hidden, weight;
    int64_t first;  // of the piece, in the vocabulary
    const uint32_t* count;
    RowTerms terms;
    char* out;  // [rows][piece] parts; kPaired: behind the last row what their rounding left, by the same rows
    int64_t out_stride;
    const int32_t* sizes;  // float32: of the piece, by kScaleRows
};

// The softmax's part of g, zero past the vocabulary's end and at the targets.
template <typename T, bool kCapped, bool kPaired, typename Tile>
__global__ __launch_bounds__(Tile::kThreads) void softmax_kernel(SoftmaxArgs a, int64_t m_tiles, int64_t n_tiles) {
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    const int64_t count = *a.count;
    int64_t m, n;
    m_tiles = tiles_that_count<Tile::kM>(count, m_tiles);
    if (block_id() >= m_tiles * n_tiles) return;
    tile_of(block_id(), m_tiles, n_tiles, m, n);
    typename Tile::Sums acc;
    Tile::run(a.hidden, a.weight, m * Tile::kM, n * Tile::kN, count, a.weight.count, a.s.padded, 0, 0, (LdsByte*)lds, acc);
    const int64_t m0 = m * Tile::kM + Tile::wave_m(), n0 = n * Tile::kN + Tile::wave_n();
    const Cap cap(a.s);
    struct Row {
        float lse, factor;
        int32_t target, by;
    };
    static_assert(kScaleRows % Tile::kN == 0);
    const int weight_exponent = kScaled<T> ? exponent_of(a.sizes[n * Tile::kN / kScaleRows]) - 2 * kTop : 0;
    const auto load = [&](int in_row, int) {
        const int64_t row = min(m0 + in_row, count - 1);
        return Row{a.terms.lse[row], a.terms.factor[row], a.terms.target[row], kScaled<T> ? weight_exponent + a.terms.row_exponent[row] : 0};
    };
    by_rows<Tile>(acc, (LdsByte*)lds, load, [&](int in_row, int in_column, float (&v)[8], const Row& of) {
        const int64_t row = m0 + in_row, column = n0 + in_column;
        if (row >= count) return;
        const int64_t target = of.target - a.first - column, left = a.weight.count - column;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float derivative;
            if constexpr (kScaled<T>) v[e] = ldexpf(v[e], of.by);
            const float z = cap.logit<kCapped>(v[e], derivative);
            float p = __builtin_amdgcn_exp2f((z - of.lse) * kLog2E) * of.factor;
            if constexpr (kCapped) p *= derivative;
            // float32's rounding first, in every kernel: a product that float16 alone takes would be rounded to that at once, and
            // kPaired takes it in float32 too
            if constexpr (__is_same(T, _Float16)) asm("" : "+v"(p));
            v[e] = e >= left || e == target ? 0.0f : p;
        }
        store_parts<T>(a.out + row * a.out_stride, column, v);
        if constexpr (kPaired) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] -= static_cast<float>(static_cast<T>(v[e]));
            store_parts<T>(a.out + (count + row) * a.out_stride, column, v);
        }
    });
}

// The products of a piece's softmax: with the weights, for dh, and with the hidden states, for dW, in one launch. Their tiles fill
// the CUs' rounds together (8192 rows, 16384 of the vocabulary, 1536 dimensions: 192 and 384 tiles, the first twice as long), and the longer ones begin.
struct GradientArgs {
    Operand softmax, weight, hidden;  // softmax.batch, weight.batch: a unit
    const uint32_t* count;
    int64_t dim, first, width, unit;  // first and width: of the piece
    // dh
    int64_t m_tiles, n_tiles;  // none without dh
    bool begin;  // the total begins here
    float *total, *part;  // [row], [unit][row] of those that count
    // dW
    int64_t weight_m_tiles, weight_n_tiles;
    const float* sums;       // the targets' part, by the index in `at`
    const int32_t* at;       // by token, -1: none
    const int32_t* largest;  // float16 parts: the power of two left out
    const int32_t* sizes;    // float32: of the piece, by kScaleRows, which are whole units
    bool accumulate;
    bool whole;  // dW's rows are whole 16-byte chunks
};

// Whether a tile of dh adds the piece's units to the total itself; else each unit has a part. With tiles for most CUs that saves the
// parts' way through memory; with fewer, the others would wait for them (8192 rows, 151936 x 1536, of which 3277 count: 78
// tiles; 5.8 ms in turn, 5.0 with parts). Parts are kPartFloats at most: to write and read more takes as long as the tiles in turn, beside
// dW's (12287 of the vocabulary: 1000 rows of 2900, 0.26 GiB of parts, 0.54 ms and 0.76 in turn; 2000 of 2304, 0.41 GiB, 0.64 and 0.53; 2458 of
// 2304, 0.51 GiB, 0.76 and 0.77). The additions and their order are the same.
template <typename Tile>
constexpr int64_t kTurnTiles = Tile::kM == 256 ? 160 : 320;
constexpr int64_t kPartFloats = int64_t{96} << 20;
template <typename Tile>
__host__ __device__ __forceinline__ bool in_turn(int64_t rows, int64_t dim, int64_t n_tiles, int64_t units) {
    return units == 1 || (rows + Tile::kM - 1) / Tile::kM * n_tiles >= kTurnTiles<Tile> || rows * dim * units > kPartFloats;
}

template <typename T, typename Tile>
__device__ __forceinline__ void hidden_tile(const GradientArgs& a, int64_t id, int64_t m_tiles, int64_t units, LdsByte* lds) {
    const int64_t count = *a.count, each = m_tiles * a.n_tiles;
    const bool turns = in_turn<Tile>(count, a.dim, a.n_tiles, units);
    const int64_t only = turns ? 0 : id / each, end = turns ? units : only + 1;
    int64_t m, n;
    tile_of(id - only * each, m_tiles, a.n_tiles, m, n);
    const int64_t m0 = m * Tile::kM + Tile::wave_m(), n0 = n * Tile::kN + Tile::wave_n();
    float* const out = turns ? a.total : a.part + only * count * a.dim;
    for (int64_t unit = only; unit < end; ++unit) {
        typename Tile::Sums acc;
        Tile::run(a.softmax, a.weight, m * Tile::kM, n * Tile::kN, count, a.dim, min(a.unit, a.width - unit * a.unit), unit, unit, lds, acc);
        const bool store = !turns || (a.begin && unit == 0);
        const int by = kScaled<T> ? exponent_of(a.sizes[unit * a.unit / kScaleRows]) - kTop : 0;
        struct Old {
            float4 v[2];
        };
        const bool fours = a.dim % 4 == 0;
        const auto load = [&](int in_row, int in_column) {
            const int64_t row = m0 + in_row, column = n0 + in_column;
            Old old = {};
            if (fours && !store && row < count) {
                const float* const from = out + row * a.dim + column;
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    if (column + 4 * q < a.dim) old.v[q] = *reinterpret_cast<const float4*>(from + 4 * q);
            }
            return old;
        };
        by_rows<Tile>(acc, lds, load, [&](int in_row, int in_column, float (&v)[8], const Old& old) {
            const int64_t row = m0 + in_row, column = n0 + in_column;
            if (row >= count) return;
            float* const to = out + row * a.dim + column;
            if constexpr (kScaled<T>) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], by);
            }
            if (fours) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if (column + 4 * q >= a.dim) continue;
                    float4 w = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    if (!store) w = make_float4(old.v[q].x + w.x, old.v[q].y + w.y, old.v[q].z + w.z, old.v[q].w + w.w);
                    *reinterpret_cast<float4*>(to + 4 * q) = w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (column + e < a.dim) to[e] = store ? v[e] : to[e] + v[e];
            }
        });
        if (unit + 1 < end) __syncthreads();  // the next unit's copies go where these rows were
    }
}

template <typename T, bool kPaired, typename Tile>
__device__ __forceinline__ void weight_tile(T* __restrict__ dweight, const GradientArgs& a, int64_t id, LdsByte* lds) {
    int64_t m, n;
    tile_of(id, a.weight_m_tiles, a.weight_n_tiles, m, n);
    typename Tile::Sums acc;
    Tile::run(a.softmax, a.hidden, m * Tile::kM, n * Tile::kN, a.width, a.dim, static_cast<int64_t>(*a.count) * (kPaired ? 2 : 1), 0, 0, lds, acc);
    const int64_t m0 = m * Tile::kM + Tile::wave_m(), n0 = n * Tile::kN + Tile::wave_n();
    const int by = kHalfParts<T> ? *a.largest - kExponentBase - kHalfShift - kTop : 0;
    struct Old {
        int32_t at;
        Pack<T, 8> v;
    };
    const auto load = [&](int in_row, int in_column) {
        const int64_t row = m0 + in_row, column = n0 + in_column;
        Old old = {-1, {}};
        if (row < a.width && column < a.dim) {
            old.at = a.at[a.first + row];
            if (a.accumulate && a.whole) old.v = *reinterpret_cast<const Pack<T, 8>*>(dweight + (a.first + row) * a.dim + column);
        }
        return old;
    };
    by_rows<Tile>(acc, lds, load, [&](int in_row, int in_column, float (&v)[8], const Old& old) {
        const int64_t row = m0 + in_row, column = n0 + in_column;
        if (row >= a.width || column >= a.dim) return;
        const int64_t at = old.at;
        T* const out = dweight + (a.first + row) * a.dim + column;
        if constexpr (kHalfParts<T>) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], by);
        }
        if (a.whole) {
            if (at >= 0) {
                float w[8];
                load_as_float<float, 8>(a.sums + at * a.dim + column, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += w[e];
            }
            if (a.accumulate) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += static_cast<float>(old.v.v[e]);
            }
            store_from_float<T, 8>(out, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (column + e >= a.dim) break;
                if (at >= 0) v[e] += a.sums[at * a.dim + column + e];
                if (a.accumulate) v[e] += static_cast<float>(out[e]);
                out[e] = static_cast<T>(v[e]);
            }
        }
    });
}

template <typename T, bool kPaired, typename HiddenTile, typename WeightTile>
__global__ __launch_bounds__(HiddenTile::kThreads) void gradient_kernel(T* __restrict__ dweight, GradientArgs a) {
    static_assert(HiddenTile::kThreads == WeightTile::kThreads);
    __shared__ __attribute__((aligned(1024))) char lds[HiddenTile::kLds > WeightTile::kLds ? HiddenTile::kLds : WeightTile::kLds];
    const int64_t id = block_id(), count = *a.count, m_tiles = tiles_that_count<HiddenTile::kM>(count, a.m_tiles), units = (a.width + a.unit - 1) / a.unit;
    const int64_t each = m_tiles * a.n_tiles, hidden_tiles = in_turn<HiddenTile>(count, a.dim, a.n_tiles, units) ? each : each * units;
    if (id < hidden_tiles)
        hidden_tile<T, HiddenTile>(a, id, m_tiles, units, (LdsByte*)lds);
    else if (id < hidden_tiles + a.weight_m_tiles * a.weight_n_tiles)
        weight_tile<T, kPaired, WeightTile>(dweight, a, id - hidden_tiles, (LdsByte*)lds);
}

// total (+)= the units' parts, in their order, where there are parts
template <typename HiddenTile>
__global__ __launch_bounds__(256) void add_parts_kernel(const float* __restrict__ part, float* __restrict__ total, const uint32_t* __restrict__ count,
                                                        int64_t dim, int64_t n_tiles, int units, bool begin) {
    const int64_t n = static_cast<int64_t>(*count) * dim;
    if (in_turn<HiddenTile>(*count, dim, n_tiles, units)) return;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        float v = begin ? part[i] : total[i] + part[i];
        for (int u = 1; u < units; ++u) v += part[u * n + i];
        total[i] = v;
    }
}

struct FinishArgs {
    LossShape s;
    TokenOrder order;
    RowTerms terms;
    const float *total, *coefficient;
    int64_t parts;  // total: so many units' parts, added here
};

template <typename T>
__global__ __launch_bounds__(256) void finish_hidden_kernel(const T* __restrict__ weight, T* __restrict__ dhidden, FinishArgs a) {
    const int64_t j = block_id(), count = *a.order.kept;
    if (j >= a.s.rows) return;
    const int64_t row = a.order.position[j];
    T* const out = dhidden + row * a.s.dhidden_stride;
    if (j >= count) {
        for (int64_t d = threadIdx.x; d < a.s.dim; d += 256) out[d] = static_cast<T>(0.0f);
        return;
    }
    const T* const w = weight + static_cast<int64_t>(a.order.token[j]) * a.s.dim;
    const float c = a.coefficient[row];
    const int by = kHalfParts<T> ? a.terms.exponent[j] - kHalfShift : 0;
    for (int64_t d = threadIdx.x; d < a.s.dim; d += 256) {
        float v = a.total[j * a.s.dim + d];
        constexpr int kAhead = 8;
        for (int64_t u = 1; u < a.parts; u += kAhead) {
            float w[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) w[k] = u + k < a.parts ? a.total[((u + k) * count + j) * a.s.dim + d] : 0.0f;
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (u + k < a.parts) v += w[k];
        }
        if constexpr (kHalfParts<T>) v = ldexpf(v, by);
        out[d] = static_cast<T>(fmaf(c, static_cast<float>(w[d]), v));
    }
}

// ---- workspaces ----

int check_shape(const dllm_hip_vocabulary_loss_shape* sh) {
    DLLM_REQUIRE(sh != nullptr, "null shape");
    DLLM_REQUIRE(sh->dtype >= 0 && sh->dtype <= 2, "dtype must be float32 (0), bfloat16 (1) or float16 (2)");
    DLLM_REQUIRE(sh->rows >= 0 && sh->rows < kMaxSortTokens, "rows must be in [0, 2^27)");
    DLLM_REQUIRE(sh->vocabulary >= 1 && sh->vocabulary < (int64_t{1} << 31), "vocabulary must be in [1, 2^31)");
    DLLM_REQUIRE(sh->dim >= 1 && sh->dim <= (1 << 16), "dim must be in [1, 2^16]");
    DLLM_REQUIRE(sh->rows * sh->vocabulary < (int64_t{1} << 48), "rows * vocabulary must be below 2^48");
    // in float32 the scale, the cap and their quotient are then ordinary numbers
    DLLM_REQUIRE(sh->softcap == 0.0 || (sh->softcap >= 0x1p-64 && sh->softcap <= 0x1p64), "softcap must be 0 or in [2^-64, 2^64]");
    DLLM_REQUIRE(sh->scale >= 0x1p-60 && sh->scale <= 0x1p60, "scale must be in [2^-60, 2^60]");
    for (const int64_t s : {sh->hidden_stride, sh->dhidden_stride})
        DLLM_REQUIRE(s == 0 || (s >= sh->dim && s < (int64_t{1} << 32)), "a row stride must be 0 or at least dim, below 2^32");
    return kOk;
}

LossShape loss_shape(const dllm_hip_vocabulary_loss_shape& sh) {
    LossShape s{};
    s.rows = sh.rows, s.vocabulary = sh.vocabulary, s.dim = sh.dim;
    s.padded = static_cast<int64_t>(round_up(sh.dim, 8));
    s.row = sh.dtype == kFloat32 ? row_bytes<float>(sh.dim) : row_bytes<_Float16>(sh.dim);
    s.hidden_stride = sh.hidden_stride ? sh.hidden_stride : sh.dim;
    s.dhidden_stride = sh.dhidden_stride ? sh.dhidden_stride : sh.dim;
    s.scale = static_cast<float>(sh.scale), s.softcap = static_cast<float>(sh.softcap);
    return s;
}

int planes_of(int64_t dtype) { return dtype == kFloat32 ? 2 : 1; }

// Of the vocabulary: one addition to dh. It goes by the vocabulary and type alone, so that a row's bits are its own. Shorter units are
// more workgroups where rows are few and more additions where they are many (94 rows, 5568 x 57: 81 us with 4096); float32's take
// three times as long and share a scale.
int64_t unit_of(const LossShape& s, int64_t dtype) {
    const int64_t most = dtype == kFloat32 ? kScaleRows : s.vocabulary > 65536 ? 8192 : 4096;
    int64_t unit = 512;
    while (unit < most && unit * 24 <= s.vocabulary) unit *= 2;  // a dozen at least
    return unit;
}

// Units of the backward's piece: as many as keep its softmax, and half of its packed weights, within kPieceBytes, at least one.
int64_t piece_units(const LossShape& s, int64_t dtype) {
    const int64_t unit = unit_of(s, dtype);
    const int64_t rows = paired_rows(s.rows, dtype) ? 2 * s.rows : s.rows;
    const size_t bytes = static_cast<size_t>(std::max(rows, s.padded / 2)) * unit * 2 * planes_of(dtype);
    // float32's pieces are whole scales, so that those do not go by the rows either
    const int64_t together = dtype == kFloat32 ? kScaleRows / unit : 1, groups = static_cast<int64_t>(kPieceBytes / std::max<size_t>(bytes, 1)) / together;
    const int64_t all = static_cast<int64_t>(ceil_div(s.vocabulary, unit * together));
    return std::clamp<int64_t>(groups, 1, all) * together;
}

struct LossLayout {
    size_t hidden, scaled, weight, list, stats, at_target, row_exponent, sizes;  // forward, sizes of both
    size_t terms, softmax, part, total, sums, sum_parts, at, coefficient;       // backward
    int64_t unit, units;
    size_t bytes;
    LossLayout(const LossShape& s, int64_t dtype, bool backward) {
        const size_t rows = static_cast<size_t>(s.rows), planes = planes_of(dtype), dim = static_cast<size_t>(s.dim);
        unit = unit_of(s, dtype), units = piece_units(s, dtype);
        const size_t piece = backward ? std::min<size_t>(units * unit, s.vocabulary) : std::min<size_t>(kPackPiece, s.vocabulary);
        const size_t times = backward && paired_rows(s.rows, dtype) ? 2 : 1;
        hidden = rows * s.row * (dtype == kBFloat16 ? times : 1);
        scaled = backward && dtype != kBFloat16 ? rows * s.row * times : 0;
        weight = piece * s.row;
        list = backward ? 0 : rows;
        stats = backward ? 0 : ceil_div(s.vocabulary, kStatRows) * rows;
        at_target = backward ? 0 : rows;
        row_exponent = dtype == kFloat32 ? rows : 0;
        sizes = dtype == kFloat32 ? ceil_div(s.vocabulary, kScaleRows) : 0;
        terms = backward ? round_up(rows, 256) : 0;
        softmax = backward ? rows * (units * unit + kStrideSlack) * planes * times : 0;
        part = backward && units > 1 ? std::min<size_t>(units * rows * dim, kPartFloats) : 0;
        total = backward ? rows * dim : 0;
        sums = total;
        sum_parts = backward ? token_sums_part_floats(s.rows, s.dim) : 0;
        at = backward ? s.vocabulary : 0;
        coefficient = backward ? rows : 0;
        Layout l;
        l.add<char>(hidden);
        l.add<char>(scaled);
        l.add<char>(weight);
        l.add<uint32_t>(list);
        l.add<uint32_t>(1);
        l.add<Stat>(stats);
        l.add<float>(at_target);
        l.add<int32_t>(row_exponent);
        l.add<int32_t>(1 + sizes + at);  // filled with -1 at once
        if (backward) {
            add_token_order(l, s.rows);
            for (int i = 0; i < 4; ++i) l.add<float>(terms);
            l.add<uint16_t>(softmax);
            for (const size_t n : {part, total, sums, sum_parts, coefficient}) l.add<float>(n);
        }
        bytes = l.bytes;
    }
};

template <typename T>
struct Buffers {
    char *hidden, *scaled, *weight;
    uint32_t *list, *count;
    Stat* stats;
    float* at_target;
    int32_t* row_exponent;
    int32_t *largest, *sizes, *at;
    TokenOrder order;
    RowTerms terms;
    char* softmax;
    float *part, *total, *sums, *sum_parts, *coefficient;
    Buffers(const LossLayout& l, const LossShape& s, bool backward, void* workspace, size_t bytes) {
        Carve c(workspace, bytes);
        hidden = c.take<char>(l.hidden);
        scaled = c.take<char>(l.scaled);
        weight = c.take<char>(l.weight);
        list = c.take<uint32_t>(l.list);
        count = c.take<uint32_t>(1);
        stats = c.take<Stat>(l.stats);
        at_target = c.take<float>(l.at_target);
        row_exponent = c.take<int32_t>(l.row_exponent);
        largest = c.take<int32_t>(1 + l.sizes + l.at);
        sizes = largest + 1, at = sizes + l.sizes;
        if (!backward) return;
        order = take_token_order(c, s.rows);
        terms.lse = c.take<float>(l.terms);
        terms.factor = c.take<float>(l.terms);
        terms.target = c.take<int32_t>(l.terms);
        terms.exponent = c.take<int32_t>(l.terms);
        terms.row_exponent = row_exponent;
        softmax = reinterpret_cast<char*>(c.take<uint16_t>(l.softmax));
        part = c.take<float>(l.part);
        total = c.take<float>(l.total);
        sums = c.take<float>(l.sums);
        sum_parts = c.take<float>(l.sum_parts);
        coefficient = c.take<float>(l.coefficient);
    }
};

// Whether the weights are read where they are. as_they_are: values, not pairs.
template <typename T>
bool weights_direct(const LossShape& s, const T* weight, bool as_they_are) {
    return as_they_are && s.dim % kChunk<T> == 0 && aligned_to(weight, 16);
}

// The weights of a piece as an operand: where they are, or packed. sizes: of the piece.
template <typename T>
int weight_operand(const LossShape& s, const T* weight, bool as_they_are, char* packed, int32_t* sizes, int64_t first, int64_t n, Operand& op,
                   hipStream_t stream) {
    op.count = n;
    op.batch = 0;
    op.stride = s.row;
    if (weights_direct(s, weight, as_they_are)) {
        op.stride = s.dim * static_cast<int64_t>(sizeof(T));
        op.base = reinterpret_cast<const char*>(weight + first * s.dim);
        return kOk;
    }
    op.base = packed;
    PackArgs p{};
    p.n = n, p.dim = s.dim, p.stride = s.dim, p.sizes = sizes;
    if constexpr (kScaled<T>) {
        if (as_they_are) return launch_pack<T, kAsTheyAre>(weight + first * s.dim, packed, p, stream);
        const float* const from = weight + first * s.dim;
        if (s.dim % 4 == 0 && aligned_to(from, 16))
            unit_sizes_kernel<4><<<grid_of(ceil_div(n, kSizeRows)), 256, 0, stream>>>(from, n, s.dim, sizes);
        else
            unit_sizes_kernel<1><<<grid_of(ceil_div(n, kSizeRows)), 256, 0, stream>>>(from, n, s.dim, sizes);
        return launch_pack<T, kUnitScale>(weight + first * s.dim, packed, p, stream);
    } else {
        return launch_pack<T, kNoScale>(weight + first * s.dim, packed, p, stream);
    }
}

template <typename T>
RowsArgs rows_args(const LossShape& s, const Buffers<T>& b) {
    RowsArgs a{};
    a.s = s, a.packed = b.hidden, a.row_exponent = b.row_exponent;
    return a;
}

Operand hidden_operand(const LossShape& s, const char* packed) { return {packed, s.row, 0, s.rows}; }

template <typename T, typename Tile>
void launch_forward(const ForwardArgs& a, hipStream_t stream) {
    const int64_t m = ceil_div(a.weight.count, Tile::kM), n = ceil_div(a.s.rows, Tile::kN);
    if (a.s.softcap != 0.0f)
        forward_kernel<T, true, Tile><<<grid_of(m * n), Tile::kThreads, 0, stream>>>(a, m, n);
    else
        forward_kernel<T, false, Tile><<<grid_of(m * n), Tile::kThreads, 0, stream>>>(a, m, n);
}

template <typename T>
int run_forward(const LossShape& s, int64_t dtype, const T* hidden, const T* weight, const int64_t* targets, float* loss, float* lse,
                void* workspace, size_t bytes, hipStream_t stream) {
    const LossLayout layout(s, dtype, false);
    const Buffers<T> b(layout, s, false, workspace, bytes);
    const bool few = kScaled<T> && s.rows <= kFewRows, direct = weights_direct(s, weight, !kScaled<T> || few);
    RowsArgs r = rows_args<T>(s, b);
    r.list = b.list, r.count = b.count, r.targets = targets, r.at_target = b.at_target;
    if (few) r.row_exponent = nullptr;
    if (s.rows <= kFindRows) {
        r.loss_out = loss, r.lse_out = lse, r.sizes = b.sizes, r.units = layout.sizes;
        DLLM_TRY((launch_rows<T, kFind>(hidden, weight, r, stream)));
    } else {
        keep_rows_kernel<<<1, 1024, 0, stream>>>(targets, s.rows, s.vocabulary, b.list, b.count, loss, lse);
        if (kScaled<T>) DLLM_TRY(fill_words(b.sizes, layout.sizes * 4, ~uint32_t{0}, stream));
        DLLM_TRY((launch_rows<T, kListed>(hidden, weight, r, stream)));
    }
    const int64_t piece = direct ? s.vocabulary : kPackPiece;
    for (int64_t first = 0; first < s.vocabulary; first += piece) {
        ForwardArgs a{};
        a.s = s, a.hidden = hidden_operand(s, b.hidden), a.k = direct ? s.dim : s.padded;
        a.sizes = b.sizes + first / kScaleRows, a.exponent = b.row_exponent;
        DLLM_TRY(weight_operand<T>(s, weight, !kScaled<T> || few, b.weight, b.sizes + first / kScaleRows, first,
                                   std::min(piece, s.vocabulary - first), a.weight, stream));
        a.first = first, a.list = b.list, a.count = b.count, a.targets = targets, a.stats = b.stats, a.at_target = b.at_target;
        if constexpr (kScaled<T>) {
            if (s.rows <= 32)
                launch_forward<T, DirectTile<32, 1, 1>>(a, stream);
            else if (s.rows <= 64)
                launch_forward<T, DirectTile<64, 1, 2>>(a, stream);
            else if (s.rows <= kFewRows)
                launch_forward<T, DirectTile<128, 2, 4>>(a, stream);
            else
                launch_forward<T, typename LargeTiles<T>::Forward>(a, stream);
        } else {
            if (s.rows <= 64)
                launch_forward<T, typename SmallTiles<T>::Forward>(a, stream);
            else if (s.rows <= 128)
                launch_forward<T, typename MiddleTiles<T>::Forward>(a, stream);
            else
                launch_forward<T, typename LargeTiles<T>::Forward>(a, stream);
        }
    }
    const auto join_rows = [&](auto rows) {
        constexpr int kJoinRows = decltype(rows)::value;
        join_stats_kernel<kJoinRows><<<grid_of(ceil_div(s.rows, kJoinRows)), 64 * kJoinRows, 0, stream>>>(
            b.stats, b.at_target, static_cast<int64_t>(ceil_div(s.vocabulary, kStatRows)), s.rows, b.list, b.count, loss, lse);
    };
    if (s.rows >= 4096)
        join_rows(std::integral_constant<int, 16>{});
    else
        join_rows(std::integral_constant<int, 4>{});
    return check_launch("vocabulary_loss");
}

// Whether 256 x 256 tiles take less time for a piece's products than 128 x 128 ones: a large tile takes as long as four small ones at
// two to a CU would, or a little less, so rounds and padding decide. It goes by all rows: how many count is not known here.
bool large_tiles(const LossShape& s, const LossLayout& l) {
    const auto time = [&](int64_t size, int64_t slots, double round) {
        const int64_t width = std::min(l.units * l.unit, s.vocabulary);
        const int64_t m = ceil_div(s.rows, size), n = ceil_div(width, size), d = ceil_div(s.dim, size);
        const double logits = std::ceil(static_cast<double>(m * n) / slots) * s.dim;
        const double products = std::max(std::ceil(static_cast<double>(m * d * l.units) * l.unit + static_cast<double>(n * d) * s.rows) / slots,
                                         static_cast<double>(l.unit));
        return (logits + products) * round;
    };
    return time(256, 256, 4.0) <= time(128, 512, 2.1);
}

template <typename T, typename Tiles>
int run_pieces(const LossShape& s, const Buffers<T>& b, const LossLayout& layout, const T* weight, bool dhidden, T* dweight, bool accumulate,
               int64_t& parts, hipStream_t stream) {
    using Logits = typename Tiles::Logits;
    using Hidden = typename Tiles::Hidden;
    using Weight = typename Tiles::Weight;
    constexpr bool kPaired = std::is_same_v<Tiles, SmallTiles<T>> && !kScaled<T>;
    const int64_t piece = layout.units * layout.unit;
    for (int64_t first = 0; first < s.vocabulary; first += piece) {
        SoftmaxArgs a{};
        a.s = s, a.hidden = hidden_operand(s, b.hidden);
        a.sizes = b.sizes + first / kScaleRows;
        DLLM_TRY(weight_operand<T>(s, weight, !kScaled<T>, b.weight, b.sizes + first / kScaleRows, first, std::min(piece, s.vocabulary - first), a.weight, stream));
        a.first = first, a.count = b.order.kept, a.terms = b.terms, a.out = b.softmax;
        a.out_stride = row_bytes<T>(piece + kStrideSlack);
        const int64_t width = a.weight.count, m = ceil_div(s.rows, Logits::kM), n = ceil_div(width, Logits::kN);
        if (s.softcap != 0.0f)
            softmax_kernel<T, true, kPaired, Logits><<<grid_of(m * n), Logits::kThreads, 0, stream>>>(a, m, n);
        else
            softmax_kernel<T, false, kPaired, Logits><<<grid_of(m * n), Logits::kThreads, 0, stream>>>(a, m, n);
        GradientArgs g{};
        g.softmax = Operand{b.softmax, a.out_stride, value_at<kLossPlanes<T>>(layout.unit), s.rows};
        g.weight = a.weight, g.weight.batch = layout.unit * a.weight.stride;
        g.hidden = hidden_operand(s, kHalfParts<T> ? b.scaled : b.hidden);
        g.sizes = a.sizes, g.count = b.order.kept, g.dim = s.dim, g.first = first, g.width = width, g.unit = layout.unit;
        const int64_t units = ceil_div(width, layout.unit);
        int64_t hidden_blocks = 0;
        bool add_parts = false;
        if (dhidden) {
            g.m_tiles = ceil_div(s.rows, Hidden::kM), g.n_tiles = ceil_div(s.dim, Hidden::kN);
            // (how many tiles there are is known where the rows that count are: either way's workgroups)
            const int64_t tiles = g.m_tiles * g.n_tiles;
            hidden_blocks = units == 1 ? tiles : std::max(tiles, std::min(tiles, kTurnTiles<Hidden> - 1) * units);
            add_parts = units > 1;
            if (add_parts && !in_turn<Hidden>(s.rows, s.dim, g.n_tiles, units) && piece >= s.vocabulary) parts = units, add_parts = false;  // one piece's: at the end
            g.begin = first == 0, g.total = b.total, g.part = b.part;
        }
        if (dweight) {
            g.weight_m_tiles = ceil_div(width, Weight::kM), g.weight_n_tiles = ceil_div(s.dim, Weight::kN);
            g.sums = b.sums, g.at = b.at, g.largest = b.largest, g.accumulate = accumulate;
            g.whole = s.dim % 8 == 0 && aligned_to(dweight, 16);
        }
        gradient_kernel<T, kPaired, Hidden, Weight><<<grid_of(hidden_blocks + g.weight_m_tiles * g.weight_n_tiles), Hidden::kThreads, 0, stream>>>(dweight, g);
        if (add_parts)
            add_parts_kernel<Hidden><<<static_cast<unsigned>(std::min<size_t>(ceil_div(s.rows * s.dim, 256), 4096)), 256, 0, stream>>>(
                b.part, b.total, b.order.kept, s.dim, g.n_tiles, static_cast<int>(units), first == 0);
    }
    return check_launch("vocabulary_loss_backward");
}

template <typename T>
int run_backward(const LossShape& s, int64_t dtype, const T* hidden, const T* weight, const int64_t* targets, const float* lse,
                 const float* dloss, T* dhidden, T* dweight, bool accumulate, void* workspace, size_t bytes, hipStream_t stream) {
    const LossLayout layout(s, dtype, true);
    const Buffers<T> b(layout, s, true, workspace, bytes);
    // -1 everywhere: until the rows and weights say how large they are, and the sums where they are
    DLLM_TRY(sort_tokens(targets, s.rows, s.vocabulary, b.order, b.largest, (1 + layout.sizes + (dweight ? layout.at : 0)) * 4, ~uint32_t{0}, stream));
    RowsArgs r = rows_args<T>(s, b);
    r.list = b.order.position, r.count = b.order.kept, r.order = b.order, r.lse = lse, r.dloss = dloss, r.terms = b.terms;
    r.coefficient = b.coefficient, r.largest = b.largest, r.twice = paired_rows(s.rows, dtype);
    DLLM_TRY((launch_rows<T, kBackward>(hidden, weight, r, stream)));
    if constexpr (kHalfParts<T>) {
        PackArgs p{};
        p.list = b.order.position, p.count = b.order.kept, p.n = s.rows, p.dim = s.dim, p.stride = s.hidden_stride;
        p.exponent = b.terms.exponent, p.largest = b.largest, p.twice = paired_rows(s.rows, dtype);
        if (dweight) DLLM_TRY((launch_pack<T, kWeightScale>(hidden, b.scaled, p, stream)));
    }
    if (dweight) {
        TokenSums sums{};
        sums.order = b.order, sums.n = s.rows, sums.vocabulary = s.vocabulary, sums.dim = s.dim, sums.stride = s.hidden_stride;
        sums.rows = hidden, sums.coefficient = b.coefficient, sums.scale = 1.0f, sums.part = b.sum_parts, sums.sums = b.sums, sums.first = b.at;
        DLLM_TRY(launch_token_sums(sums, dtype, stream));
    }
    int64_t parts = 1;
    const auto pieces = [&](auto tiles) {
        return run_pieces<T, decltype(tiles)>(s, b, layout, weight, dhidden != nullptr, dweight, accumulate, parts, stream);
    };
    if (s.rows <= kPairedRows)
        DLLM_TRY(pieces(SmallTiles<T>{}));
    else if (large_tiles(s, layout))
        DLLM_TRY(pieces(LargeTiles<T>{}));
    else
        DLLM_TRY(pieces(MiddleTiles<T>{}));
    if (dhidden) {
        FinishArgs f{s, b.order, b.terms, b.total, b.coefficient, 1};
        if (parts > 1) f.total = b.part, f.parts = parts;
        finish_hidden_kernel<T><<<grid_of(s.rows), 256, 0, stream>>>(weight, dhidden, f);
    }
    return check_launch("vocabulary_loss_backward");
}

}  // namespace

extern "C" {

size_t dllm_hip_vocabulary_loss_workspace(const dllm_hip_vocabulary_loss_shape* sh) {
    return check_shape(sh) == kOk ? LossLayout(loss_shape(*sh), sh->dtype, false).bytes : 0;
}

int dllm_hip_vocabulary_loss(const dllm_hip_vocabulary_loss_shape* sh, const void* hidden, const void* weight, const int64_t* targets,
                             float* loss, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    DLLM_TRY(check_shape(sh));
    if (sh->rows == 0 || (!loss && !lse)) return kOk;
    DLLM_REQUIRE(hidden && weight && targets, "null hidden, weight or targets");
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(hidden, size) && aligned_to(weight, size) && aligned_to(targets, 8) && aligned_to(loss, 4) && aligned_to(lse, 4),
                 "pointers must be aligned to the element");
    const LossShape s = loss_shape(*sh);
    DLLM_REQUIRE(workspace && workspace_bytes >= LossLayout(s, sh->dtype, false).bytes, "workspace too small for vocabulary_loss");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    const auto run = [&](auto type) {
        using T = decltype(type);
        return run_forward<T>(s, sh->dtype, static_cast<const T*>(hidden), static_cast<const T*>(weight), targets, loss, lse, workspace,
                              workspace_bytes, static_cast<hipStream_t>(stream));
    };
    switch (sh->dtype) {
        case kFloat32: return run(float{});
        case kBFloat16: return run(__bf16{});
        default: return run(_Float16{});
    }
}

size_t dllm_hip_vocabulary_loss_backward_workspace(const dllm_hip_vocabulary_loss_shape* sh) {
    return check_shape(sh) == kOk ? LossLayout(loss_shape(*sh), sh->dtype, true).bytes : 0;
}

int dllm_hip_vocabulary_loss_backward(const dllm_hip_vocabulary_loss_shape* sh, const void* hidden, const void* weight,
                                      const int64_t* targets, const float* lse, const float* dloss, void* dhidden, void* dweight,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    DLLM_TRY(check_shape(sh));
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(dhidden, size) && aligned_to(dweight, size), "pointers must be aligned to the element");
    if (!dhidden && !dweight) return kOk;
    if (sh->rows == 0) {
        const size_t table = static_cast<size_t>(sh->vocabulary) * sh->dim * size;
        return dweight && !sh->accumulate ? fill_words(dweight, table, 0, static_cast<hipStream_t>(stream)) : static_cast<int>(kOk);
    }
    DLLM_REQUIRE(hidden && weight && targets && lse && dloss, "null hidden, weight, targets, lse or dloss");
    DLLM_REQUIRE(aligned_to(hidden, size) && aligned_to(weight, size) && aligned_to(targets, 8) && aligned_to(lse, 4) && aligned_to(dloss, 4),
                 "pointers must be aligned to the element");
    const LossShape s = loss_shape(*sh);
    DLLM_REQUIRE(workspace && workspace_bytes >= LossLayout(s, sh->dtype, true).bytes, "workspace too small for vocabulary_loss_backward");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    const auto run = [&](auto type) {
        using T = decltype(type);
        return run_backward<T>(s, sh->dtype, static_cast<const T*>(hidden), static_cast<const T*>(weight), targets, lse, dloss,
                               static_cast<T*>(dhidden), static_cast<T*>(dweight), sh->accumulate != 0, workspace, workspace_bytes,
                               static_cast<hipStream_t>(stream));
    };
    switch (sh->dtype) {
        case kFloat32: return run(float{});
        case kBFloat16: return run(__bf16{});
        default: return run(_Float16{});
    }
}

}  // extern "C"
