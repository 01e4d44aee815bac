// Orthogonalised updates by Newton-Schulz products.
//
//   X = x / (|x| + eps);  steps times  A = X X^T,  B = b A + c A A,  X = a X + B X;  out = scale X
//
// on the m x n matrix with m <= n (the transposed one where rows exceed columns: X p(X^T X) = p(X X^T) X). The singular values alone
// change, each by the polynomial a s + b s^3 + c s^5; small ones grow by a in every step, so what a rounding of X adds in the
// directions of small singular values grows with them. X is therefore held in float32, and what the products read is rounded
// from it: an error of theirs is relative to the term b A X + c A A X, which for small singular values is far smaller than a X.
//
// The products' operands are float16, one plane for 16-bit updates (11 bits; bfloat16's 8 would cost its results two bits) and two
// for float32 ones (22 bits, three products). All values are bounded by the singular values, which stay near one, so fixed
// powers of two keep them in float16's range: X times 2^4 sqrt(n), A and B times 2^8.
//
// A and A A are symmetric: only tiles on and above the diagonal are formed, and stored twice.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "dllm_hip.h"
#include "element.h"
#include "tile_product.h"
#include "workspace.h"

using namespace dllm_hip;

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormParts = 64;  // workgroups that add up a matrix's squares
constexpr int kMaxSteps = 64;
constexpr float kGramScale = 0x1p8f;

template <typename T>
constexpr int kUpdatePlanes = sizeof(T) == 4 ? 2 : 1;

using Half = _Float16;

struct Matrices {
    int64_t batch, m, n, m_padded, n_padded;  // padded to whole chunks
    bool turned;                              // m is the columns of x
    int64_t in_stride, in_batch, out_stride, out_batch;
    float x_scale;  // of X's planes
    double eps;
    float out_scale;
};

// ---- norm and start ----

template <typename T>
__global__ __launch_bounds__(kNormThreads) void squares_kernel(const T* __restrict__ x, double* __restrict__ part, int64_t rows, int64_t cols,
                                                               Matrices s) {
    __shared__ double of_wave[kNormThreads / kWave];
    const T* const matrix = x + static_cast<int64_t>(blockIdx.y) * s.in_batch;
    double sum = 0.0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (int64_t c = threadIdx.x; c < cols; c += kNormThreads) {
            const double v = static_cast<double>(static_cast<float>(matrix[r * s.in_stride + c]));
            sum = fma(v, v, sum);
        }
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) sum += __shfl_xor(sum, i);
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kNormThreads / kWave; ++w) sum += of_wave[w];
        part[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = sum;
    }
}

// v as planes of float16 parts
template <int kPl>
__device__ __forceinline__ void split_half(float v, Half (&parts)[kPl]) {
#pragma unroll
    for (int p = 0; p < kPl; ++p) {
        parts[p] = static_cast<Half>(v);
        v -= static_cast<float>(parts[p]);
    }
}

// 64 x 64 of X: from x, or from its transposed.
template <typename T>
__global__ __launch_bounds__(256) void start_kernel(const T* __restrict__ x, const double* __restrict__ part, int parts, float* __restrict__ held,
                                                    Half* __restrict__ planes, int64_t plane, Matrices s) {
    constexpr int kPl = kUpdatePlanes<T>;
    __shared__ float tile[64][65];
    const int64_t matrix = blockIdx.z, i0 = static_cast<int64_t>(blockIdx.y) * 64, j0 = static_cast<int64_t>(blockIdx.x) * 64;
    double squares = 0.0;
    for (int p = 0; p < parts; ++p) squares += part[matrix * parts + p];
    const double norm = sqrt(squares) + s.eps;
    const T* const from = x + matrix * s.in_batch;
    for (int e = threadIdx.x; e < 64 * 64; e += 256) {
        const int slow = e >> 6, fast = e & 63;
        const int64_t i = i0 + (s.turned ? fast : slow), j = j0 + (s.turned ? slow : fast);
        float v = 0.0f;
        if (i < s.m && j < s.n)
            v = static_cast<float>(static_cast<double>(static_cast<float>(from[s.turned ? j * s.in_stride + i : i * s.in_stride + j])) / norm);
        tile[s.turned ? fast : slow][s.turned ? slow : fast] = v;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 64 * 64; e += 256) {
        const int64_t i = i0 + (e >> 6), j = j0 + (e & 63);
        if (i >= s.m || j >= s.n_padded) continue;
        const float v = tile[e >> 6][e & 63];
        const int64_t at = (matrix * s.m + i) * s.n_padded + j;
        held[at] = v;
        Half parts16[kPl];
        split_half<kPl>(v * s.x_scale, parts16);
#pragma unroll
        for (int p = 0; p < kPl; ++p) planes[p * plane + at] = parts16[p];
    }
}

// steps 0: out = scale X
template <typename T>
__global__ __launch_bounds__(256) void no_steps_kernel(const float* __restrict__ held, T* __restrict__ out, Matrices s) {
    const int64_t rows = s.turned ? s.n : s.m, cols = s.turned ? s.m : s.n, matrix = blockIdx.y;
    for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < rows * cols; e += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = e / cols, c = e - r * cols, i = s.turned ? c : r, j = s.turned ? r : c;
        out[matrix * s.out_batch + r * s.out_stride + c] = static_cast<T>(held[(matrix * s.m + i) * s.n_padded + j] * s.out_scale);
    }
}

// ---- products ----

// Workgroup id -> matrix and tile on or above the diagonal, an XCD's tiles contiguous.
__device__ __forceinline__ void triangle_of(int64_t id, int64_t tiles, int64_t batch, int64_t& matrix, int64_t& m, int64_t& n) {
    const int64_t each = tiles * (tiles + 1) / 2;
    int64_t one, t;
    tile_of(id, each * batch, 1, t, one);
    matrix = t / each;
    t -= matrix * each;
    n = static_cast<int64_t>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
    while (n * (n + 1) / 2 > t) --n;
    while ((n + 1) * (n + 2) / 2 <= t) ++n;
    m = t - n * (n + 1) / 2;
}

struct GramArgs {
    Matrices s;
    Operand of;  // both sides
    int64_t k;
    Half* out;
    int64_t out_plane;
    float factor;       // of the product
    const Half* first;  // with it, plus first_factor times this
    float first_factor;
};

// value at (i, j) of a symmetric matrix and, above the diagonal's tiles, at (j, i); zero in the padding
template <int kPl>
__device__ __forceinline__ void store_plane_values(Half* out, int64_t plane, int64_t at, float v) {
    Half parts[kPl];
    split_half<kPl>(v, parts);
#pragma unroll
    for (int p = 0; p < kPl; ++p) out[p * plane + at] = parts[p];
}

template <typename T, typename Tile>
__global__ __launch_bounds__(Tile::kThreads) void gram_kernel(GramArgs a, int64_t tiles) {
    constexpr int kPl = kUpdatePlanes<T>;
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    int64_t matrix, m, n;
    triangle_of(blockIdx.x, tiles, a.s.batch, matrix, m, n);
    typename Tile::Sums acc;
    Tile::run(a.of, a.of, m * Tile::kM, n * Tile::kN, a.s.m, a.s.m, a.k, matrix, matrix, (LdsByte*)lds, acc);
    const int64_t i0 = m * Tile::kM + Tile::wave_m(), j0 = n * Tile::kN + Tile::wave_n(), base = matrix * a.s.m * a.s.m_padded;
    Half* const out = a.out + base;
#pragma unroll
    for (int bi = 0; bi < Tile::kBlocksM; ++bi)
#pragma unroll
        for (int bj = 0; bj < Tile::kBlocksN; ++bj) {
            const int64_t j = j0 + 32 * bj + lane_column();
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t i = i0 + 32 * bi + block_row(r), at = i * a.s.m_padded + j;
                const bool inside = i < a.s.m && j < a.s.m;
                float v = inside ? acc[bi][bj][r] * a.factor : 0.0f;
                if (a.first && inside) {
                    float w = 0.0f;
#pragma unroll
                    for (int p = kPl - 1; p >= 0; --p) w += static_cast<float>(a.first[base + p * a.out_plane + at]);
                    v = fmaf(a.first_factor, w, v);
                }
                if (i < a.s.m && j < a.s.m_padded) store_plane_values<kPl>(out, a.out_plane, at, v);
                if (m != n && j < a.s.m && i < a.s.m_padded) store_plane_values<kPl>(out, a.out_plane, j * a.s.m_padded + i, v);
            }
        }
}

struct UpdateArgs {
    Matrices s;
    Operand left, x;
    float* held;
    Half* planes;  // of the new X; NULL in the last step
    int64_t plane;
    float keep, factor;
};

template <typename T, typename Tile>
__global__ __launch_bounds__(Tile::kThreads) void update_kernel(T* __restrict__ result, UpdateArgs a, int64_t m_tiles, int64_t n_tiles) {
    constexpr int kPl = kUpdatePlanes<T>;
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    int64_t m, n;
    tile_of(blockIdx.x, m_tiles, n_tiles * a.s.batch, m, n);
    const int64_t matrix = n / n_tiles;
    n -= matrix * n_tiles;
    typename Tile::Sums acc;
    Tile::run(a.left, a.x, m * Tile::kM, n * Tile::kN, a.s.m, a.s.n_padded, a.s.m, matrix, matrix, (LdsByte*)lds, acc);
    const int64_t i0 = m * Tile::kM + Tile::wave_m(), j0 = n * Tile::kN + Tile::wave_n();
#pragma unroll
    for (int bi = 0; bi < Tile::kBlocksM; ++bi)
#pragma unroll
        for (int bj = 0; bj < Tile::kBlocksN; ++bj) {
            const int64_t j = j0 + 32 * bj + lane_column();
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t i = i0 + 32 * bi + block_row(r);
                if (i >= a.s.m || j >= a.s.n_padded) continue;
                const int64_t at = (matrix * a.s.m + i) * a.s.n_padded + j;
                const float v = fmaf(a.keep, a.held[at], acc[bi][bj][r] * a.factor);
                if (a.planes) {
                    a.held[at] = v;
                    store_plane_values<kPl>(a.planes, a.plane, at, v * a.s.x_scale);
                } else if (j < a.s.n) {
                    const int64_t to = a.s.turned ? j * a.s.out_stride + i : i * a.s.out_stride + j;
                    result[matrix * a.s.out_batch + to] = static_cast<T>(v * a.s.out_scale);
                }
            }
        }
}

// ---- the call ----

template <typename T, int kSize>
using GramTile = TileProduct<Half, kUpdatePlanes<T>, kSize, kSize, 2, kSize / 64, false, false>;
template <typename T, int kSize>
using UpdateTile = TileProduct<Half, kUpdatePlanes<T>, kSize, kSize, 2, kSize / 64, false, true>;

Matrices matrices_of(const dllm_hip_orthogonalize_shape& sh) {
    Matrices s;
    s.batch = sh.batch;
    s.turned = sh.rows > sh.cols;
    s.m = std::min(sh.rows, sh.cols), s.n = std::max(sh.rows, sh.cols);
    s.m_padded = static_cast<int64_t>(round_up(s.m, 8)), s.n_padded = static_cast<int64_t>(round_up(s.n, 8));
    s.in_stride = sh.x_stride ? sh.x_stride : sh.cols;
    s.out_stride = sh.out_stride ? sh.out_stride : sh.cols;
    s.in_batch = sh.x_batch_stride ? sh.x_batch_stride : sh.rows * s.in_stride;
    s.out_batch = sh.out_batch_stride ? sh.out_batch_stride : sh.rows * s.out_stride;
    s.x_scale = static_cast<float>(std::ldexp(1.0, 4 + static_cast<int>(std::log2(static_cast<double>(s.n)) / 2)));
    s.eps = sh.eps;
    s.out_scale = static_cast<float>(sh.scale);
    return s;
}

struct UpdateLayout {
    size_t norm, held, planes, gram, bytes;
    UpdateLayout(const Matrices& s, int64_t dtype) {
        const size_t pl = dtype == kFloat32 ? 2 : 1;
        norm = static_cast<size_t>(s.batch) * kNormParts;
        held = static_cast<size_t>(s.batch) * s.m * s.n_padded;
        planes = pl * held;
        gram = pl * s.batch * s.m * s.m_padded;
        Layout l;
        l.add<double>(norm);
        l.add<float>(held);
        for (const size_t n : {planes, planes, gram, gram}) l.add<Half>(n);
        bytes = l.bytes;
    }
};

struct UpdateBuffers {
    double* norm;
    float* held;
    Half *planes[2], *gram, *left;
};

template <typename T, int kSize>
int launch_step(const Matrices& s, const UpdateBuffers& b, const double* c, int from, bool last, T* out, hipStream_t stream) {
    constexpr int kPl = kUpdatePlanes<T>;
    using Gram = GramTile<T, kSize>;
    using Update = UpdateTile<T, kSize>;
    const int64_t plane = s.batch * s.m * s.n_padded, gram_plane = s.batch * s.m * s.m_padded;
    const Operand x{reinterpret_cast<const char*>(b.planes[from]), s.n_padded * 2, plane * 2, s.m * s.n_padded * 2, s.m};
    const int64_t tiles = ceil_div(s.m, kSize), each = tiles * (tiles + 1) / 2;
    const dim3 grid(static_cast<unsigned>(each * s.batch));
    GramArgs g{};
    g.s = s, g.of = x, g.k = s.n_padded, g.out = b.gram, g.out_plane = gram_plane, g.factor = kGramScale / (s.x_scale * s.x_scale);
    gram_kernel<T, Gram><<<grid, Gram::kThreads, 0, stream>>>(g, tiles);
    const Operand gram{reinterpret_cast<const char*>(b.gram), s.m_padded * 2, gram_plane * 2, s.m * s.m_padded * 2, s.m};
    g.of = gram, g.k = s.m, g.out = b.left, g.factor = static_cast<float>(c[2]) / kGramScale, g.first = b.gram, g.first_factor = static_cast<float>(c[1]);
    gram_kernel<T, Gram><<<grid, Gram::kThreads, 0, stream>>>(g, tiles);
    UpdateArgs u{};
    u.s = s, u.left = gram, u.left.base = reinterpret_cast<const char*>(b.left), u.x = x;
    u.held = b.held, u.planes = last ? nullptr : b.planes[1 - from], u.plane = plane;
    u.keep = static_cast<float>(c[0]), u.factor = 1.0f / (kGramScale * s.x_scale);
    const int64_t n_tiles = ceil_div(s.n, kSize);
    update_kernel<T, Update><<<static_cast<unsigned>(tiles * n_tiles * s.batch), Update::kThreads, 0, stream>>>(out, u, tiles, n_tiles);
    (void)kPl;
    return check_launch("orthogonalize");
}

template <typename T>
int run(const dllm_hip_orthogonalize_shape& sh, const Matrices& s, const double* coefficients, const T* x, T* out, const UpdateBuffers& b,
        hipStream_t stream) {
    const int parts = static_cast<int>(std::min<int64_t>(kNormParts, sh.rows));
    squares_kernel<T><<<dim3(parts, static_cast<unsigned>(s.batch)), kNormThreads, 0, stream>>>(x, b.norm, sh.rows, sh.cols, s);
    const dim3 tiles(static_cast<unsigned>(ceil_div(s.n_padded, 64)), static_cast<unsigned>(ceil_div(s.m, 64)), static_cast<unsigned>(s.batch));
    start_kernel<T><<<tiles, 256, 0, stream>>>(x, b.norm, parts, b.held, b.planes[0], s.batch * s.m * s.n_padded, s);
    if (sh.steps == 0) {
        const size_t blocks = std::min<size_t>(ceil_div(s.m * s.n, 256), 4096);
        no_steps_kernel<T><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(s.batch)), 256, 0, stream>>>(b.held, out, s);
        return check_launch("orthogonalize");
    }
    static constexpr double kQuintic[3] = {3.4445, -4.7750, 2.0315};
    for (int64_t i = 0; i < sh.steps; ++i) {
        const double* const c = coefficients ? coefficients + 3 * i : kQuintic;
        DLLM_TRY((launch_step<T, 128>(s, b, c, static_cast<int>(i % 2), i == sh.steps - 1, out, stream)));
    }
    return kOk;
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
        DLLM_REQUIRE(row <= INT64_MAX / (1 << 17), "a row stride is too large");
        DLLM_REQUIRE(s[1] == 0 || s[1] >= (sh->rows - 1) * row + sh->cols, "a batch stride must be 0 or at least a matrix");
    }
    // a grid's x extent times its workgroup is below 2^32
    const int64_t tiles = ceil_div(sh->rows, 128) * ceil_div(sh->cols, 128) + ceil_div(std::min(sh->rows, sh->cols), 128);
    DLLM_REQUIRE(tiles * sh->batch < (1 << 23), "too many matrices for one call");
    return kOk;
}

}  // namespace

extern "C" {

size_t dllm_hip_orthogonalize_workspace(const dllm_hip_orthogonalize_shape* sh) {
    return check_shape(sh) == kOk ? UpdateLayout(matrices_of(*sh), sh->dtype).bytes : 0;
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
    const UpdateLayout layout(s, sh->dtype);
    DLLM_REQUIRE(workspace && workspace_bytes >= layout.bytes, "workspace too small for orthogonalize");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    Carve c(workspace, workspace_bytes);
    UpdateBuffers b;
    b.norm = c.take<double>(layout.norm);
    b.held = c.take<float>(layout.held);
    b.planes[0] = c.take<Half>(layout.planes);
    b.planes[1] = c.take<Half>(layout.planes);
    b.gram = c.take<Half>(layout.gram);
    b.left = c.take<Half>(layout.gram);
    auto st = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return run<float>(*sh, s, coefficients, static_cast<const float*>(x), static_cast<float*>(out), b, st);
        case kBFloat16: return run<__bf16>(*sh, s, coefficients, static_cast<const __bf16*>(x), static_cast<__bf16*>(out), b, st);
        default: return run<_Float16>(*sh, s, coefficients, static_cast<const _Float16*>(x), static_cast<_Float16*>(out), b, st);
    }
}

}  // extern "C"
