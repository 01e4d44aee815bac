// Orthogonalised updates by Newton-Schulz products.
//
//   X = x / (|x| + eps);  steps times  A = X X^T,  B = b A + c A A,  X = a X + B X;  out = scale X
//
// on the m x n matrix with m <= n (the transposed one where rows exceed columns: X p(X^T X) = p(X X^T) X). The singular values alone
// change, each by the polynomial a s + b s^3 + c s^5; small ones grow by a in every step, so what a rounding of X adds in the
// directions of small singular values grows with them. X is therefore held to 22 bits and more, as a pair of float16, and what
// the products of 16-bit updates read is its first part: an error of theirs is relative to the term b A X + c A A X, which for
// small singular values is far smaller than a X.
//
// The products' operands are float16 (bfloat16's 8 bits would cost results two of theirs): one part of 11 bits for bfloat16
// updates, whose own 8 bits are coarser than what that adds: after five steps results are off by 1.00 (896 x 4864) to 1.2 times (70
// x 500) what their rounding alone is, 1.7e-3 in the 2-norm, where a few directions are strong as in a momentum; by 1.4 to 1.5
// times where all singular values are alike, which then are near one two steps earlier. Pairs of 22 bits, three products, for
// float32 and float16 ones, and for small matrices, whose few singular values average no rounding out (2 x 76: 2.5e-3 with one
// part). With singular values near one the term is as large as a X, and its error stays: calls of more than five steps multiply
// pairs from the fifth on (256 x 1024, six steps: 1.3 times with one part, 1.00 so; ten steps 2.3 and 1.01), at 1.9 times the time
// of such a step (24 of 896 x 4864, six steps: 3.33 to 4.28 ms; from the third step on singular values that are all alike would
// have 1.00 too, instead of 1.4 to 1.6 and 2.1 after ten steps, for another 1 ms).
//
// All values are bounded by the singular values, which stay near one, so fixed powers of two keep them in float16's range: X times
// 2^4 sqrt(n), A and B times 2^8.
//
// A and A A are symmetric: only tiles on and above the diagonal are formed, and stored twice. Where they are few and long, X X^T is
// formed in segments of its n columns at once, whose sums a launch of its own adds in order; where there are matrices enough, a
// workgroup takes the segments in turn and adds them in the same order, so a matrix has the same bits alone and among others.
//
// Bound and measured, bfloat16. 24 matrices of 896 x 4864, a step 560 us: X X^T 190 (560 TFLOP/s of the half that is formed; 672
// tiles of 128 are 1.3 rounds of the two that each CU holds), A A 42, X's new values 327, whose products alone take 220 and
// whose 834 MB alone 158: the two are hardly at once, though two workgroups share a CU (starting one of them later, or
// reading X ahead of the products, gave nothing). One of 8960 x 1536, a step 112 us: 34 and 9 for its sums of segments, 18, 67.
// Small ones (192 x 576 in float32, 135 us) are 17 launches of 4 to 15 us, each one workgroup's way through k.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "dllm_hip.h"
#include "element.h"
#include "tile_product.h"
#include "workspace.h"

using namespace dllm_hip;

namespace {

constexpr int kThreads = 256;
constexpr int64_t kNormElements = 1 << 12;  // at least, whose squares a workgroup adds
constexpr int64_t kNormParts = 512;         // at most, of a matrix
constexpr int kMaxSteps = 64;
constexpr float kGramScale = 0x1p8f;

// Parts of a value that the products read: of a type and a smaller side m.
constexpr int64_t kFewSingularValues = 64;
inline int product_planes(int64_t dtype, int64_t m) { return dtype == kBFloat16 && m > kFewSingularValues ? 1 : 2; }

// The step from which on all multiply pairs.
constexpr int64_t kCoarseSteps = 4;
inline int64_t pairs_from(const dllm_hip_orthogonalize_shape& sh) {
    if (product_planes(sh.dtype, std::min(sh.rows, sh.cols)) == 2) return 0;
    return sh.steps > kCoarseSteps + 1 ? kCoarseSteps : sh.steps;
}

using Half = _Float16;
using Half8 = Half __attribute__((ext_vector_type(8)));

struct Matrices {
    int64_t batch, m, n, m_padded, n_padded;  // padded to whole chunks
    bool turned;                              // m is the columns of x
    int64_t in_stride, in_batch, out_stride, out_batch;
    float x_scale;  // of X's planes
    double eps;
    float out_scale;
};

// Where X's values are. kPl 2: pairs as the products read them; kPl 1: the products read the first parts, the second ones are
// `rest` further.
template <int kPl>
struct Places {
    int64_t row, rest;  // bytes
    __host__ __device__ Places(const Matrices& s) : row(s.n_padded * 2 * kPl), rest(kPl == 2 ? kSecond : s.batch * s.m * s.n_padded * 2) {}
    __device__ __forceinline__ int64_t at(const Matrices& s, int64_t matrix, int64_t i, int64_t j) const {
        return (matrix * s.m + i) * row + value_at<kPl>(j);
    }
};

// 8 values as pairs, the second parts `rest` bytes further
__device__ __forceinline__ void store_pairs(char* to, int64_t rest, const float (&v)[8]) {
    Half8 first, second;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        first[e] = static_cast<Half>(v[e]);
        second[e] = static_cast<Half>(v[e] - static_cast<float>(first[e]));
    }
    *reinterpret_cast<Half8*>(to) = first;
    *reinterpret_cast<Half8*>(to + rest) = second;
}

// ---- norm and start ----

__device__ __forceinline__ double add_over_threads(double v) {
    __shared__ double of_wave[kThreads / kWave];
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) v += __shfl_xor(v, i);
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kThreads / kWave; ++w) v += of_wave[w];
    return v;
}

// The sum of squares of `rows_each` rows, in double: the squares of float32 and bfloat16 values are more than float32 holds.
template <typename T, int kWidth>
__global__ __launch_bounds__(kThreads) void squares_kernel(const T* __restrict__ x, double* __restrict__ part, int64_t rows, int64_t cols,
                                                           int64_t rows_each, int64_t parts, Matrices s) {
    if (block_id() >= parts * s.batch) return;
    const int64_t matrix = block_id() / parts, first = (block_id() - matrix * parts) * rows_each;
    const int64_t chunks = cols / kWidth, items = (min(first + rows_each, rows) - first) * chunks;
    const T* const from = x + matrix * s.in_batch + first * s.in_stride;
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < items; i += kThreads) {
        const int64_t r = i / chunks;
        float v[kWidth];
        load_as_float<T, kWidth>(from + r * s.in_stride + (i - r * chunks) * kWidth, v);
#pragma unroll
        for (int e = 0; e < kWidth; ++e) sum = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), sum);
    }
    sum = add_over_threads(sum);
    if (threadIdx.x == 0) part[block_id()] = sum;
}

// 64 x 64 of X: from x, or from its transposed. kWide: x's rows are whole chunks of 8.
template <typename T, bool kWide, int kPl>
__global__ __launch_bounds__(kThreads) void start_kernel(const T* __restrict__ x, const double* __restrict__ part, int64_t parts,
                                                         char* __restrict__ out, int64_t m_tiles, int64_t n_tiles, Matrices s) {
    __shared__ float tile[64][65];
    if (block_id() >= m_tiles * n_tiles * s.batch) return;
    const int64_t matrix = block_id() / (m_tiles * n_tiles), in_matrix = block_id() - matrix * m_tiles * n_tiles;
    const int64_t i0 = in_matrix / n_tiles * 64, j0 = in_matrix % n_tiles * 64;
    double squares = 0.0;
    for (int64_t p = threadIdx.x; p < parts; p += kThreads) squares += part[matrix * parts + p];
    const double norm = sqrt(add_over_threads(squares)) + s.eps;
    // the quotient's rounding is of X as a whole, which the steps forgive; a norm below float32's range, or above it, is not
    // (zeroes beside an eps whose inverse is none are zeroes)
    const double inverse = norm > 0.0 ? fmin(1.0 / norm, 0x1p1023) : NAN;
    const T* const from = x + matrix * s.in_batch;
    // rows and columns of x
    const int64_t r0 = s.turned ? j0 : i0, c0 = s.turned ? i0 : j0, rows = s.turned ? s.n : s.m, cols = s.turned ? s.m : s.n;
#pragma unroll
    for (int e = threadIdx.x; e < 64 * 8; e += kThreads) {
        const int r = e >> 3, c = (e & 7) * 8;
        float v[8] = {};
        if (r0 + r < rows) {
            const T* const at = from + (r0 + r) * s.in_stride + c0 + c;
            if constexpr (kWide) {
                if (c0 + c < cols) {
#pragma unroll
                    for (int q = 0; q < 8; q += kChunk<T>) {
                        float w[kChunk<T>];
                        load_as_float<T, kChunk<T>>(at + q, w);
#pragma unroll
                        for (int u = 0; u < kChunk<T>; ++u) v[q + u] = w[u];
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (c0 + c + u < cols) v[u] = static_cast<float>(at[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float w = static_cast<float>(static_cast<double>(v[u]) * inverse) * s.x_scale;
            if (s.turned)
                tile[c + u][r] = w;
            else
                tile[r][c + u] = w;
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = threadIdx.x; e < 64 * 8; e += kThreads) {
        const int64_t i = i0 + (e >> 3), j = j0 + (e & 7) * 8;
        if (i >= s.m || j >= s.n_padded) continue;
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = tile[e >> 3][(e & 7) * 8 + u];
        const Places<kPl> places(s);
        store_pairs(out + places.at(s, matrix, i, j), places.rest, v);
    }
}

// steps 0: out = scale X
template <typename T, int kPl>
__global__ __launch_bounds__(kThreads) void no_steps_kernel(const char* __restrict__ x, T* __restrict__ out, Matrices s) {
    const Places<kPl> places(s);
    const int64_t rows = s.turned ? s.n : s.m, cols = s.turned ? s.m : s.n, matrix = blockIdx.y;
    for (int64_t e = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; e < rows * cols; e += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t r = e / cols, c = e - r * cols, i = s.turned ? c : r, j = s.turned ? r : c;
        const char* const at = x + places.at(s, matrix, i, j);
        const float v = static_cast<float>(*reinterpret_cast<const Half*>(at)) + static_cast<float>(*reinterpret_cast<const Half*>(at + places.rest));
        out[matrix * s.out_batch + r * s.out_stride + c] = static_cast<T>(v * (s.out_scale / s.x_scale));
    }
}

// ---- products ----

// Index -> tile on or above the diagonal.
__device__ __forceinline__ void triangle_of(int64_t t, int64_t& m, int64_t& n) {
    n = static_cast<int64_t>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
    while (n * (n + 1) / 2 > t) --n;
    while ((n + 1) * (n + 2) / 2 <= t) ++n;
    m = t - n * (n + 1) / 2;
}

struct GramArgs {
    Matrices s;
    Operand of;  // both sides
    int64_t k, segment, segments;  // of k
    char* out;
    float factor;       // of the product
    const char* first;  // with it, plus first_factor times this
    float first_factor;
    float* part;  // [matrix][segment][m][m_padded]: a workgroup forms one segment; NULL: all in turn
};

// The values [first, end) of 8 alone.
template <int kPl>
__device__ __forceinline__ void store_some(char* out, const float (&v)[8], int64_t first, int64_t end) {
    if (first <= 0 && end >= 8) {
        store_eight<Half, kPl>(out, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (e < first || e >= end) continue;
        float left = v[e];
#pragma unroll
        for (int p = 0; p < kPl; ++p) {
            const Half part = static_cast<Half>(left);
            *reinterpret_cast<Half*>(out + p * kSecond + e * 2) = part;
            left -= static_cast<float>(part);
        }
    }
}

// 8 values' parts, of what a result is added to.
template <int kParts>
struct Held {
    Half8 part[kParts];
};

template <int kParts>
__device__ __forceinline__ Held<kParts> hold(const char* from, int64_t rest, bool inside) {
    Held<kParts> h;
#pragma unroll
    for (int p = 0; p < kParts; ++p) h.part[p] = inside ? *reinterpret_cast<const Half8*>(from + p * rest) : Half8{};
    return h;
}

template <int kParts>
__device__ __forceinline__ float held_value(const Held<kParts>& h, int e) {
    float v = 0.0f;
#pragma unroll
    for (int p = kParts - 1; p >= 0; --p) v += static_cast<float>(h.part[p][e]);
    return v;
}

// (i, j) of a symmetric matrix
template <int kPl>
__device__ __forceinline__ int64_t gram_at(const Matrices& s, int64_t matrix, int64_t i, int64_t j) {
    return (matrix * s.m + i) * s.m_padded * 2 * kPl + value_at<kPl>(j);
}

template <int kPl>
__device__ __forceinline__ Held<kPl> hold_gram(const GramArgs& a, int64_t matrix, int64_t i, int64_t j) {
    return hold<kPl>(a.first + gram_at<kPl>(a.s, matrix, i, j), kSecond, a.first && i < a.s.m && j < a.s.m_padded);
}

// 8 values of row i from column j on, finished; zero in the padding. What is left of the diagonal is stored from the right of it
// (mirror_gram): pairs' products are added in another order there, and which tiles cross the diagonal goes by their size.
template <int kPl>
__device__ __forceinline__ void finish_gram(const GramArgs& a, int64_t matrix, int64_t i, int64_t j, float (&v)[8], const Held<kPl>& first) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] *= a.factor;
        if (a.first) v[e] = fmaf(a.first_factor, held_value(first, e), v[e]);
        if (i >= a.s.m || j + e >= a.s.m) v[e] = 0.0f;
    }
    if (i < a.s.m && j < a.s.m_padded) store_some<kPl>(a.out + gram_at<kPl>(a.s, matrix, i, j), v, i - j, 8);
}

// 8 values of column j from row i on, finished, to the row and columns across the diagonal
template <int kPl>
__device__ __forceinline__ void mirror_gram(const GramArgs& a, int64_t matrix, int64_t i, int64_t j, const float (&v)[8]) {
    if (j < a.s.m && i < a.s.m_padded) store_some<kPl>(a.out + gram_at<kPl>(a.s, matrix, j, i), v, 0, j - i);
}

template <int kPl, typename Tile>
__global__ __launch_bounds__(Tile::kThreads) void gram_kernel(GramArgs a, int64_t tiles) {
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    const int64_t each = tiles * (tiles + 1) / 2, at_once = a.part ? a.segments : 1, total = each * a.s.batch * at_once;
    if (block_id() >= total) return;
    int64_t id, one, m, n;
    tile_of(block_id(), total, 1, id, one);
    const int64_t matrix = id / (each * at_once), in_matrix = id - matrix * each * at_once, only = in_matrix / each;
    triangle_of(in_matrix - only * each, m, n);
    const int64_t i0 = m * Tile::kM + Tile::wave_m(), j0 = n * Tile::kN + Tile::wave_n();
    typename Tile::Sums acc;
    if (a.part) {
        Operand of = a.of;
        of.base += value_at<kPl>(only * a.segment);
        Tile::run(of, of, m * Tile::kM, n * Tile::kN, a.s.m, a.s.m, min(a.segment, a.k - only * a.segment), matrix, matrix, (LdsByte*)lds, acc);
        float* const part = a.part + (matrix * a.segments + only) * a.s.m * a.s.m_padded;
        by_rows<Tile>(acc, (LdsByte*)lds, [](int, int) { return Nothing{}; }, [&](int row, int column, float (&v)[8], Nothing) {
            const int64_t i = i0 + row, j = j0 + column;
            if (i < a.s.m && j < a.s.m_padded) store_from_float<float, 8>(part + i * a.s.m_padded + j, v);
        });
        return;
    }
    Tile::template run<true>(a.of, a.of, m * Tile::kM, n * Tile::kN, a.s.m, a.s.m, a.k, matrix, matrix, (LdsByte*)lds, acc, a.segment);
    by_rows_and_columns<Tile>(
        acc, (LdsByte*)lds, true, [&](int row, int column) { return hold_gram<kPl>(a, matrix, i0 + row, j0 + column); },
        [&](int row, int column, float (&v)[8], const Held<kPl>& first) { finish_gram<kPl>(a, matrix, i0 + row, j0 + column, v, first); },
        [&](int row, int column, float (&v)[8]) { mirror_gram<kPl>(a, matrix, i0 + row, j0 + column, v); });
}

// Adds the segments' parts in order: 64 x 64 on or above the diagonal, of the `tiles` tiles of kTile that the parts were formed in.
template <int kPl, int kTile>
__global__ __launch_bounds__(kThreads) void join_segments_kernel(GramArgs a, int64_t tiles) {
    constexpr int kSub = kTile / 64;
    __shared__ float tile[64][65];
    const int64_t each = tiles * (tiles + 1) / 2 * kSub * kSub;
    if (block_id() >= each * a.s.batch) return;
    const int64_t matrix = block_id() / each, id = block_id() - matrix * each;
    const int sub = static_cast<int>(id % (kSub * kSub));
    int64_t m, n;
    triangle_of(id / (kSub * kSub), m, n);
    const int64_t i0 = m * kTile + sub / kSub * 64, j0 = n * kTile + sub % kSub * 64;
    const int64_t next = a.s.m * a.s.m_padded;
#pragma unroll
    for (int e = threadIdx.x; e < 64 * 8; e += kThreads) {
        const int64_t i = i0 + (e >> 3), j = j0 + (e & 7) * 8;
        float v[8] = {};
        if (i < a.s.m && j < a.s.m_padded) {
            const float* from = a.part + matrix * a.segments * next + i * a.s.m_padded + j;
            load_as_float<float, 8>(from, v);
            for (int64_t which = 1; which < a.segments; ++which) {
                float w[8];
                load_as_float<float, 8>(from + which * next, w);
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] += w[u];
            }
        }
        finish_gram<kPl>(a, matrix, i, j, v, hold_gram<kPl>(a, matrix, i, j));
#pragma unroll
        for (int u = 0; u < 8; ++u) tile[(e & 7) * 8 + u][e >> 3] = v[u];
    }
    __syncthreads();
#pragma unroll
    for (int e = threadIdx.x; e < 64 * 8; e += kThreads) {
        const int64_t j = j0 + (e >> 3), i = i0 + (e & 7) * 8;
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = tile[e >> 3][(e & 7) * 8 + u];
        mirror_gram<kPl>(a, matrix, i, j, v);
    }
}

struct UpdateArgs {
    Matrices s;
    Operand left, x;
    const char* from;  // X
    char* to;          // the new X; NULL in the last step
    float keep, factor;
    bool whole;  // the result's rows are whole chunks of 8
};

template <typename T>
__device__ __forceinline__ void store_result(T* to, int64_t left, bool whole, const float (&v)[8]) {
    if (whole) {
        if (left <= 0) return;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            store_from_float<T, 8>(to, v);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) to[e] = static_cast<T>(v[e]);
    }
}

// kTo: the new X's parts, of the products that read it next.
template <typename T, int kPl, int kTo, typename Tile>
__global__ __launch_bounds__(Tile::kThreads) void update_kernel(T* __restrict__ result, UpdateArgs a, int64_t m_tiles, int64_t n_tiles) {
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    if (block_id() >= m_tiles * n_tiles * a.s.batch) return;
    int64_t m, n;
    tile_of(block_id(), m_tiles, n_tiles * a.s.batch, m, n);
    const int64_t matrix = n / n_tiles;
    n -= matrix * n_tiles;
    typename Tile::Sums acc;
    Tile::run(a.left, a.x, m * Tile::kM, n * Tile::kN, a.s.m, a.s.n_padded, a.s.m, matrix, matrix, (LdsByte*)lds, acc);
    const int64_t i0 = m * Tile::kM + Tile::wave_m(), j0 = n * Tile::kN + Tile::wave_n();
    T* const out = result + matrix * a.s.out_batch;
    const Places<kPl> places(a.s);
    const Places<kTo> next(a.s);
    by_rows_and_columns<Tile>(
        acc, (LdsByte*)lds, !a.to && a.s.turned,
        [&](int row, int column) {
            const int64_t i = i0 + row, j = j0 + column;
            return hold<2>(a.from + places.at(a.s, matrix, i, j), places.rest, i < a.s.m && j < a.s.n_padded);
        },
        [&](int row, int column, float (&v)[8], const Held<2>& x) {
            const int64_t i = i0 + row, j = j0 + column;
            if (i >= a.s.m || j >= a.s.n_padded) return;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(a.keep, held_value(x, e), v[e] * a.factor);
            if (a.to)
                store_pairs(a.to + next.at(a.s, matrix, i, j), next.rest, v);
            else if (!a.s.turned)
                store_result(out + i * a.s.out_stride + j, a.s.n - j, a.whole, v);
        },
        [&](int row, int column, float (&v)[8]) {
            const int64_t i = i0 + row, j = j0 + column;
            if (j < a.s.n) store_result(out + j * a.s.out_stride + i, a.s.m - i, a.whole, v);
        });
}

// ---- the call ----

template <int kPl, int kSize, int kStages>
using GramTile = TileProduct<Half, kPl, kSize, kSize, 2, 2, false, false, kStages>;
template <int kPl, int kSize, int kStages>
using UpdateTile = TileProduct<Half, kPl, kSize, kSize, 2, kSize == 256 ? 4 : 2, false, true, kStages>;

Matrices matrices_of(const dllm_hip_orthogonalize_shape& sh) {
    Matrices s;
    s.batch = sh.batch;
    s.turned = sh.rows > sh.cols;
    s.m = std::min(sh.rows, sh.cols), s.n = std::max(sh.rows, sh.cols);
    const size_t multiple = pairs_from(sh) == sh.steps && sh.steps > 0 ? kRowMultiple<1> : kRowMultiple<2>;
    s.m_padded = static_cast<int64_t>(round_up(s.m, multiple)), s.n_padded = static_cast<int64_t>(round_up(s.n, multiple));
    s.in_stride = sh.x_stride ? sh.x_stride : sh.cols;
    s.out_stride = sh.out_stride ? sh.out_stride : sh.cols;
    s.in_batch = sh.x_batch_stride ? sh.x_batch_stride : sh.rows * s.in_stride;
    s.out_batch = sh.out_batch_stride ? sh.out_batch_stride : sh.rows * s.out_stride;
    s.x_scale = static_cast<float>(std::ldexp(1.0, 4 + static_cast<int>(std::log2(static_cast<double>(s.n)) / 2)));
    s.eps = sh.eps;
    s.out_scale = static_cast<float>(sh.scale);
    return s;
}

int64_t triangle(const Matrices& s, int64_t size) {
    const int64_t t = ceil_div(s.m, size);
    return t * (t + 1) / 2;
}

// Of k: what one matrix's tiles of 128 need to be about 512 workgroups, at least 1024 k each. It goes by the matrix's size alone.
int64_t segment_of(const Matrices& s, int64_t k) {
    const int64_t segments = std::clamp<int64_t>(512 / triangle(s, 128), 1, std::max<int64_t>(k / 1024, 1));
    return static_cast<int64_t>(round_up(ceil_div(k, segments), 64));
}

// Segments are formed at once where the matrices' tiles do not fill the CUs.
bool segments_at_once(const Matrices& s, int64_t k) { return segment_of(s, k) < k && triangle(s, 128) * s.batch < 384; }

int64_t norm_rows(const dllm_hip_orthogonalize_shape& sh) {
    return std::max<int64_t>({kNormElements / sh.cols, static_cast<int64_t>(ceil_div(sh.rows, kNormParts)), 1});
}

struct UpdateLayout {
    size_t norm, planes, gram, part, bytes;
    UpdateLayout(const dllm_hip_orthogonalize_shape& sh, const Matrices& s) {
        norm = static_cast<size_t>(s.batch) * ceil_div(sh.rows, norm_rows(sh));
        planes = 2 * static_cast<size_t>(s.batch) * s.m * s.n_padded;
        gram = static_cast<size_t>(pairs_from(sh) < sh.steps ? 2 : 1) * s.batch * s.m * s.m_padded;
        part = 0;
        for (const int64_t k : {s.n_padded, s.m})
            if (segments_at_once(s, k)) part = std::max(part, static_cast<size_t>(s.batch) * ceil_div(k, segment_of(s, k)) * s.m * s.m_padded);
        Layout l;
        l.add<double>(norm);
        for (const size_t n : {planes, planes, gram, gram}) l.add<Half>(n);
        l.add<float>(part);
        bytes = l.bytes;
    }
};

struct UpdateBuffers {
    double* norm;
    char *x[2], *gram, *left;
    float* part;
};

template <int kPl, typename Tile>
void launch_gram_tiles(const GramArgs& g, bool at_once, hipStream_t stream) {
    constexpr int kSize = Tile::kM;
    const int64_t tiles = ceil_div(g.s.m, kSize), all = triangle(g.s, kSize) * g.s.batch;
    gram_kernel<kPl, Tile><<<grid_of(all * (at_once ? g.segments : 1)), Tile::kThreads, 0, stream>>>(g, tiles);
    if (at_once) join_segments_kernel<kPl, kSize><<<grid_of(all * (kSize / 64) * (kSize / 64)), kThreads, 0, stream>>>(g, tiles);
}

// Tiles of 128 where they are enough for the CUs, else of 64 with more of their copies under way: a lone workgroup on a CU waits for
// them. (192 x 576 in float32: 16 us for X X^T with four stages of 64 x 64 tiles, 29 with two of 128 x 128.)
template <int kPl>
void launch_gram(GramArgs g, float* part, hipStream_t stream) {
    g.segment = segment_of(g.s, g.k), g.segments = ceil_div(g.k, g.segment);
    const bool at_once = segments_at_once(g.s, g.k);
    g.part = at_once ? part : nullptr;
    const int64_t blocks = triangle(g.s, 128) * g.s.batch * (at_once ? g.segments : 1);
    if (blocks >= 200) {
        launch_gram_tiles<kPl, GramTile<kPl, 128, 2>>(g, at_once, stream);
    } else if (triangle(g.s, 64) * g.s.batch * (at_once ? g.segments : 1) > 256) {
        launch_gram_tiles<kPl, GramTile<kPl, 64, 4>>(g, at_once, stream);
    } else {
        launch_gram_tiles<kPl, GramTile<kPl, 64, 8>>(g, at_once, stream);
    }
}

template <typename T, int kPl, int kTo, typename Tile>
void launch_update(const UpdateArgs& u, T* out, hipStream_t stream) {
    const int64_t m = ceil_div(u.s.m, Tile::kM), n = ceil_div(u.s.n, Tile::kN);
    update_kernel<T, kPl, kTo, Tile><<<grid_of(m * n * u.s.batch), Tile::kThreads, 0, stream>>>(out, u, m, n);
}

template <typename T, int kPl, int kTo>
int launch_step(const Matrices& s, const UpdateBuffers& b, const double* c, int from, bool last, T* out, hipStream_t stream) {
    const int64_t row = s.n_padded * 2 * kPl, gram_row = s.m_padded * 2 * kPl;
    const Operand x{b.x[from], row, s.m * row, s.m};
    GramArgs g{};
    g.s = s, g.of = x, g.k = s.n_padded, g.out = b.gram, g.factor = kGramScale / (s.x_scale * s.x_scale);
    launch_gram<kPl>(g, b.part, stream);
    const Operand gram{b.gram, gram_row, s.m * gram_row, s.m};
    g.of = gram, g.k = s.m, g.out = b.left, g.factor = static_cast<float>(c[2]) / kGramScale, g.first = b.gram, g.first_factor = static_cast<float>(c[1]);
    launch_gram<kPl>(g, b.part, stream);
    UpdateArgs u{};
    u.s = s, u.left = gram, u.left.base = b.left, u.x = x;
    u.from = b.x[from], u.to = last ? nullptr : b.x[1 - from];
    // the last step's result leaves X's scale
    const float unit = last ? s.out_scale / s.x_scale : 1.0f;
    u.keep = static_cast<float>(c[0]) * unit, u.factor = unit / kGramScale;
    const int64_t length = s.turned ? s.m : s.n;
    u.whole = length % 8 == 0 && s.out_stride % 8 == 0 && s.out_batch % 8 == 0 && aligned_to(out, 16);
    const int64_t large = ceil_div(s.m, 256) * ceil_div(s.n, 256) * s.batch, middle = ceil_div(s.m, 128) * ceil_div(s.n, 128) * s.batch;
    if (middle < 256 && ceil_div(s.m, 64) * ceil_div(s.n, 64) * s.batch <= 256)
        launch_update<T, kPl, kTo, UpdateTile<kPl, 64, 8>>(u, out, stream);
    else if (middle < 256)
        launch_update<T, kPl, kTo, UpdateTile<kPl, 64, 4>>(u, out, stream);
    else if (ceil_div(large, 256) * 2 <= ceil_div(middle, 512))
        launch_update<T, kPl, kTo, UpdateTile<kPl, 256, 2>>(u, out, stream);
    else
        launch_update<T, kPl, kTo, UpdateTile<kPl, 128, 2>>(u, out, stream);
    return check_launch("orthogonalize");
}

template <typename T, int kPl>
int run_planes(const dllm_hip_orthogonalize_shape& sh, const Matrices& s, const double* coefficients, const T* x, T* out, const UpdateBuffers& b,
               hipStream_t stream) {
    const int64_t parts = ceil_div(sh.rows, norm_rows(sh));
    constexpr int kWide = kChunk<T>;
    const bool chunks = sh.cols % kWide == 0 && s.in_stride % kWide == 0 && s.in_batch % kWide == 0 && aligned_to(x, 16);
    if (chunks)
        squares_kernel<T, kWide><<<grid_of(parts * s.batch), kThreads, 0, stream>>>(x, b.norm, sh.rows, sh.cols, norm_rows(sh), parts, s);
    else
        squares_kernel<T, 1><<<grid_of(parts * s.batch), kThreads, 0, stream>>>(x, b.norm, sh.rows, sh.cols, norm_rows(sh), parts, s);
    const int64_t m_tiles = ceil_div(s.m, 64), n_tiles = ceil_div(s.n_padded, 64);
    if (chunks && sh.cols % 8 == 0)
        start_kernel<T, true, kPl><<<grid_of(m_tiles * n_tiles * s.batch), kThreads, 0, stream>>>(x, b.norm, parts, b.x[0], m_tiles, n_tiles, s);
    else
        start_kernel<T, false, kPl><<<grid_of(m_tiles * n_tiles * s.batch), kThreads, 0, stream>>>(x, b.norm, parts, b.x[0], m_tiles, n_tiles, s);
    if (sh.steps == 0) {
        const size_t blocks = std::min<size_t>(ceil_div(s.m * s.n, kThreads), 4096);
        no_steps_kernel<T, kPl><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(s.batch)), kThreads, 0, stream>>>(b.x[0], out, s);
        return check_launch("orthogonalize");
    }
    static constexpr double kQuintic[3] = {3.4445, -4.7750, 2.0315};
    for (int64_t i = 0; i < sh.steps; ++i) {
        const double* const c = coefficients ? coefficients + 3 * i : kQuintic;
        const int from = static_cast<int>(i % 2);
        const bool last = i == sh.steps - 1;
        if constexpr (kPl == 1) {
            if (i >= pairs_from(sh)) {
                DLLM_TRY((launch_step<T, 2, 2>(s, b, c, from, last, out, stream)));
                continue;
            }
            if (!last && i + 1 == pairs_from(sh)) {
                DLLM_TRY((launch_step<T, 1, 2>(s, b, c, from, last, out, stream)));
                continue;
            }
        }
        DLLM_TRY((launch_step<T, kPl, kPl>(s, b, c, from, last, out, stream)));
    }
    return kOk;
}

template <typename T>
int run(const dllm_hip_orthogonalize_shape& sh, const Matrices& s, const double* coefficients, const void* x, void* out, const UpdateBuffers& b,
        hipStream_t stream) {
    if constexpr (__is_same(T, __bf16))
        if (product_planes(sh.dtype, s.m) == 1)
            return run_planes<T, 1>(sh, s, coefficients, static_cast<const T*>(x), static_cast<T*>(out), b, stream);
    return run_planes<T, 2>(sh, s, coefficients, static_cast<const T*>(x), static_cast<T*>(out), b, stream);
}

int check_shape(const dllm_hip_orthogonalize_shape* sh) {
    DLLM_REQUIRE(sh != nullptr, "null shape");
    DLLM_REQUIRE(sh->dtype >= 0 && sh->dtype <= 2, "dtype must be float32 (0), bfloat16 (1) or float16 (2)");
    DLLM_REQUIRE(sh->batch >= 0 && sh->batch <= 65535, "batch must be in [0, 65535]");
    DLLM_REQUIRE(sh->rows >= 1 && sh->rows <= (1 << 16) && sh->cols >= 1 && sh->cols <= (1 << 16), "rows and cols must be in [1, 2^16]");
    DLLM_REQUIRE(sh->steps >= 0 && sh->steps <= kMaxSteps, "steps must be in [0, 64]");
    DLLM_REQUIRE(sh->eps >= 0.0 && std::isfinite(sh->eps), "eps must be finite and not negative");
    DLLM_REQUIRE(std::isfinite(static_cast<float>(sh->scale)), "scale must be finite in float32");
    const int64_t strides[2][2] = {{sh->x_stride, sh->x_batch_stride}, {sh->out_stride, sh->out_batch_stride}};
    for (const auto& s : strides) {
        DLLM_REQUIRE(s[0] == 0 || s[0] >= sh->cols, "a row stride must be 0 or at least cols");
        const int64_t row = s[0] ? s[0] : sh->cols;
        DLLM_REQUIRE(row < (int64_t{1} << 32), "a row stride must be below 2^32");
        DLLM_REQUIRE(s[1] == 0 || (s[1] >= (sh->rows - 1) * row + sh->cols && s[1] < (int64_t{1} << 47)),
                     "a batch stride must be 0 or at least a matrix, below 2^47");
    }
    // (the workspace of more is no size that a GPU has)
    DLLM_REQUIRE(sh->batch * sh->rows * sh->cols < (int64_t{1} << 40), "too many matrices for one call");
    return kOk;
}

}  // namespace

extern "C" {

size_t dllm_hip_orthogonalize_workspace(const dllm_hip_orthogonalize_shape* sh) {
    return check_shape(sh) == kOk ? UpdateLayout(*sh, matrices_of(*sh)).bytes : 0;
}

int dllm_hip_orthogonalize(const dllm_hip_orthogonalize_shape* sh, const double* coefficients, const void* x, void* out, void* workspace,
                           size_t workspace_bytes, void* stream) {
    DLLM_TRY(check_shape(sh));
    if (sh->batch == 0) return kOk;
    DLLM_REQUIRE(x && out, "null x or out");
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(x, size) && aligned_to(out, size), "pointers must be aligned to the element");
    if (coefficients)
        for (int64_t i = 0; i < 3 * sh->steps; ++i)
            DLLM_REQUIRE(std::isfinite(static_cast<float>(coefficients[i])), "coefficients must be finite in float32");
    const Matrices s = matrices_of(*sh);
    DLLM_REQUIRE(x != out || (s.in_stride == s.out_stride && s.in_batch == s.out_batch), "in place needs equal strides");
    const UpdateLayout layout(*sh, s);
    DLLM_REQUIRE(workspace && workspace_bytes >= layout.bytes, "workspace too small for orthogonalize");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    Carve c(workspace, workspace_bytes);
    UpdateBuffers b;
    b.norm = c.take<double>(layout.norm);
    for (char*& p : b.x) p = reinterpret_cast<char*>(c.take<Half>(layout.planes));
    b.gram = reinterpret_cast<char*>(c.take<Half>(layout.gram));
    b.left = reinterpret_cast<char*>(c.take<Half>(layout.gram));
    b.part = c.take<float>(layout.part);
    auto st = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return run<float>(*sh, s, coefficients, x, out, b, st);
        case kBFloat16: return run<__bf16>(*sh, s, coefficients, x, out, b, st);
        default: return run<_Float16>(*sh, s, coefficients, x, out, b, st);
    }
}

}  // extern "C"
