// Attention within packed documents, forward and backward (see doc_attention.h for the mask and the score).
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i)
//   dP = dout v^T,  dS = p (dP - dout . out) cap' scale,  dq = dS k,  dk = dS^T q,  dv = p^T dout
#include <float.h>

#include <algorithm>
#include <initializer_list>

#include "common.h"
#include "doc_attention.h"
#include "doc_tile.h"
#include "dllm_hip.h"
#include "workspace.h"

using namespace dllm_hip;

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;  // queries of a workgroup: 32 for each wave
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T, int kDim>
constexpr int kKeys = kDim * sizeof(T) <= 256 ? 64 : 32;  // keys of a tile: K and V twice in at most 64 KB of LDS, or 128 KB

// Forward. A wave's lane owns one query (two lanes: its halves); keys go through LDS in tiles, two buffers deep.
//
//   X = K Q^T (32 keys x 32 queries at a time)     s = X scale, capped, biased, in units of log 2
//   m = running maximum, P = 2^(s - m), l = sum P   O^T += V^T P
//
// The running maximum is moved only when some query of the wave has outgrown it by 2^8: until then P stays below 2^8, which
// float32 sums and 16-bit products hold as well as values below one.
template <typename T, int kDim, bool kDirect>
__global__ __launch_bounds__(kThreads, 2) void forward_kernel(DocAttention a, T* out) {
    using Shape = TileShape<T, kDim>;
    constexpr int kTile = kKeys<T, kDim>;
    constexpr int kTileBytes = kTile * Shape::kRowBytes;
    constexpr int kParts = kDim / 32;
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTileBytes];  // K, V of one buffer, K, V of the other

    // the heads that share keys are 8 workgroups (or a divisor of it) apart: on the same L2
    const int turn = static_cast<int>(blockIdx.x) % a.heads;
    const int head = (turn % a.kv_heads) * a.group + turn / a.kv_heads;
    const int kv = head / a.group;
    Document doc;
    int first;
    if (!locate_tile<kRows, true>(a, blockIdx.x / a.heads, doc, first)) return;

    const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5;
    const int wave_first = first + 32 * wave, wave_last = min(wave_first + 31, doc.end - 1);
    const bool working = wave_first < doc.end;
    const int i = min(wave_first + (lane & 31), doc.end - 1);
    const Span span = key_span(a, doc, i);

    Chunk<T> q[Shape::kSteps];
    load_column<T, kDim, kDirect>(static_cast<const T*>(a.q) + i * a.q_stride + static_cast<int64_t>(head) * a.head_dim,
                                  a.head_dim, q);

    // keys of the workgroup: [low, high) in whole tiles of the document, and the tiles of the prefix before them
    const int low = key_span(a, doc, first).low;
    const int high = max(key_span(a, doc, min(first + kRows, doc.end) - 1).high, doc.prefix_end);
    const int low_tile = (low - doc.start) / kTile, prefix_tiles = (doc.prefix_end - doc.start + kTile - 1) / kTile;
    const int tiles = (high - doc.start + kTile - 1) / kTile;
    // the wave's: keys that all its queries see, and that any sees
    const Span first_span = key_span(a, doc, wave_first), last_span = key_span(a, doc, wave_last);
    const int any_low = first_span.low, any_high = last_span.high, all_low = last_span.low, all_high = first_span.high;

    const TileCopy<T, kDim, kTile, kThreads, kDirect> copy_k(a.k, a.k_stride, kv, a.head_dim);
    const TileCopy<T, kDim, kTile, kThreads, kDirect> copy_v(a.v, a.v_stride, kv, a.head_dim);
    const TileView<T, kDim> view;
    LdsByte* const buffers = (LdsByte*)lds;

    const float unit = (a.softcap != 0.0f ? a.softcap : a.scale) * kLog2E;  // score of X (or of the tanh) in units of log 2
    const float cap_in = a.softcap != 0.0f ? a.scale / a.softcap : 0.0f;
    const float slope = a.slopes ? a.slopes[head] * kLog2E : 0.0f;

    Acc o[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[p][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    auto next_tile = [&](int t) { return t + 1 < prefix_tiles ? t + 1 : max(t + 1, low_tile); };
    auto fetch = [&](int t, int buffer) {
        const int from = doc.start + t * kTile;
        copy_k(from, doc.end - from, buffers + buffer * 2 * kTileBytes);
        copy_v(from, doc.end - from, buffers + buffer * 2 * kTileBytes + kTileBytes);
    };
    int t = next_tile(-1);
    fetch(t, 0);
    for (int buffer = 0; t < tiles; buffer ^= 1) {
        tile_barrier();
        const int next = next_tile(t);
        if (next < tiles) fetch(next, buffer ^ 1);
        const LdsByte* const k_tile = buffers + buffer * 2 * kTileBytes;
        const LdsByte* const v_tile = k_tile + kTileBytes;
        const int from = doc.start + t * kTile;
        t = next;
        const bool in_prefix = from < doc.prefix_end;
        if (!working || !((from < any_high && from + kTile > any_low) || in_prefix)) continue;
        const bool all_seen = (from >= all_low && from + kTile <= all_high) || from + kTile <= doc.prefix_end;

        float s[kTile / 32][16];
#pragma unroll
        for (int b = 0; b < kTile / 32; ++b) {
            Acc x;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = 0.0f;
#pragma unroll
            for (int step = 0; step < Shape::kSteps; ++step) multiply(view.rows(k_tile, b, step), q[step], x);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = x[r];
        }
        float times = unit;
        if (a.softcap != 0.0f) {
#pragma unroll
            for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = cap_tanh<T>(s[b][r] * cap_in);
        }
        if (a.slopes) {
            const float away = static_cast<float>(i - from - 4 * half);
#pragma unroll
            for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[b][r] = fmaf(-slope, fabsf(away - static_cast<float>(32 * b + 8 * (r / 4) + r % 4)), s[b][r] * unit);
            times = 1.0f;
        }
        if (!all_seen) {
            const int to_low = span.low - from - 4 * half;
            const unsigned width = static_cast<unsigned>(span.high - span.low);
            const int to_prefix = doc.prefix_end - from - 4 * half;
#pragma unroll
            for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = 32 * b + 8 * (r / 4) + r % 4;
                    const bool see = static_cast<unsigned>(j - to_low) < width || j < to_prefix;
                    s[b][r] = see ? s[b][r] : -INFINITY;
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
        top = fmaxf(top, other_half(top)) * times;
        if (__any(top > m + 8.0f)) {
            const float moved = fmaxf(m, top);
            const float keep = __builtin_amdgcn_exp2f(m - (moved == -INFINITY ? 0.0f : moved));
            m = moved;
            l *= keep;
#pragma unroll
            for (int p = 0; p < kParts; ++p)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[p][r] *= keep;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], times, -base));
                sum += s[b][r];
            }
        l += sum;
#pragma unroll
        for (int b = 0; b < kTile / 32; ++b) multiply_columns<T, kDim, kParts>(view, v_tile, b, s[b], o);
    }
    if (!working) return;
    l += other_half(l);

    // A hidden key counts as zero times its value: where that is infinite or NaN, the row is computed again from the keys
    // that it sees alone.
    bool spoilt = !(all_finite(o) && l * 0.0f == 0.0f && m * 0.0f == 0.0f);
    spoilt = (spoilt | __shfl_xor(static_cast<int>(spoilt), 32)) && wave_first + (lane & 31) < doc.end;
    if (!spoilt && wave_first + (lane & 31) < doc.end) {
        store_column<T, kParts, kDirect>(out + i * a.out_stride + static_cast<int64_t>(head) * a.head_dim, a.head_dim, o, 1.0f / l);
        if (a.lse && half == 0) a.lse[static_cast<int64_t>(head) * a.tokens + i] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
    for (uint32_t left = static_cast<uint32_t>(__ballot(spoilt)); left; left &= left - 1) {
        const int row = wave_first + __ffs(left) - 1;
        float value[kLaneDims], lse;
        attention_row<T>(a, doc, head, row, value, lse);
        store_row(out + row * a.out_stride + static_cast<int64_t>(head) * a.head_dim, value, a.head_dim);
        if (a.lse && lane == 0) a.lse[static_cast<int64_t>(head) * a.tokens + row] = lse;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void dq_rows_kernel(DocAttention a) {
    Document doc;
    int first;
    if (!locate_tile<4>(a, blockIdx.x, doc, first)) return;
    const int i = first + (static_cast<int>(threadIdx.x) >> 6), head = blockIdx.y, lane = threadIdx.x & 63;
    if (i >= doc.end) return;
    const int64_t at = i * a.out_stride + static_cast<int64_t>(head) * a.head_dim;
    const T *out = static_cast<const T*>(a.out) + at, *dout = static_cast<const T*>(a.dout) + at;
    float part = 0.0f;
    for (int d = lane; d < a.head_dim; d += 64) part = fmaf(static_cast<float>(out[d]), static_cast<float>(dout[d]), part);
    const float delta = wave_add(part);
    if (lane == 0) a.delta[static_cast<int64_t>(head) * a.tokens + i] = delta;
    float dq[kLaneDims];
    attention_row_dq<T>(a, doc, head, i, delta, dq);
    store_row(static_cast<T*>(a.dq) + i * a.q_stride + static_cast<int64_t>(head) * a.head_dim, dq, a.head_dim);
}

template <typename T>
__global__ __launch_bounds__(256) void dkv_rows_kernel(DocAttention a) {
    Document doc;
    int first;
    if (!locate_tile<4>(a, blockIdx.x, doc, first)) return;
    const int j = first + (static_cast<int>(threadIdx.x) >> 6), kv = blockIdx.y;
    if (j >= doc.end) return;
    float dk[kLaneDims] = {}, dv[kLaneDims] = {};
    for (int g = 0; g < a.group; ++g) {
        float dk1[kLaneDims], dv1[kLaneDims];
        attention_row_dkv<T>(a, doc, kv * a.group + g, j, dk1, dv1);
#pragma unroll
        for (int c = 0; c < kLaneDims; ++c) dk[c] += dk1[c], dv[c] += dv1[c];
    }
    store_row(static_cast<T*>(a.dk) + j * a.k_stride + static_cast<int64_t>(kv) * a.head_dim, dk, a.head_dim);
    store_row(static_cast<T*>(a.dv) + j * a.v_stride + static_cast<int64_t>(kv) * a.head_dim, dv, a.head_dim);
}

int check_shape(const dllm_hip_document_attention_shape* sh) {
    DLLM_REQUIRE(sh != nullptr, "null shape");
    DLLM_REQUIRE(sh->dtype >= 0 && sh->dtype <= 2, "dtype must be float32 (0), bfloat16 (1) or float16 (2)");
    DLLM_REQUIRE(sh->tokens >= 0 && sh->tokens < (int64_t{1} << 31) && sh->documents >= 0 &&
                     sh->documents < (int64_t{1} << 31),
                 "tokens and documents must be in [0, 2^31)");
    DLLM_REQUIRE(sh->kv_heads >= 1 && sh->heads >= 1 && sh->heads % sh->kv_heads == 0,
                 "heads must be a multiple of kv heads");
    DLLM_REQUIRE(sh->heads <= 65535, "at most 65535 heads");
    DLLM_REQUIRE(sh->head_dim >= 1 && sh->head_dim <= kMaxHeadDim, "head_dim must be in [1, 256]");
    DLLM_REQUIRE(sh->window >= 0, "window must not be negative");
    DLLM_REQUIRE(sh->softcap >= 0.0 && static_cast<float>(sh->softcap) <= FLT_MAX, "softcap must not be negative, nor infinite");
    DLLM_REQUIRE(static_cast<float>(sh->scale) > 0.0f && static_cast<float>(sh->scale) <= FLT_MAX, "scale must be positive and finite");
    const int64_t q = sh->heads * sh->head_dim, k = sh->kv_heads * sh->head_dim;
    for (const int64_t s : {sh->q_stride, sh->out_stride}) DLLM_REQUIRE(s == 0 || s >= q, "a token stride must be 0 or at least heads * head_dim");
    for (const int64_t s : {sh->k_stride, sh->v_stride}) DLLM_REQUIRE(s == 0 || s >= k, "a token stride must be 0 or at least heads * head_dim");
    // a grid's x extent times its workgroup is below 2^32
    DLLM_REQUIRE((static_cast<int64_t>(ceil_div(sh->tokens, kRows)) + std::min(sh->documents, sh->tokens)) * sh->heads < (1 << 24),
                 "too many tokens and documents for one call");
    return kOk;
}

DocAttention arguments(const dllm_hip_document_attention_shape& sh) {
    DocAttention a{};
    const int64_t q = sh.heads * sh.head_dim, k = sh.kv_heads * sh.head_dim;
    a.q_stride = sh.q_stride ? sh.q_stride : q;
    a.k_stride = sh.k_stride ? sh.k_stride : k;
    a.v_stride = sh.v_stride ? sh.v_stride : k;
    a.out_stride = sh.out_stride ? sh.out_stride : q;
    a.tokens = static_cast<int>(sh.tokens);
    a.documents = static_cast<int>(sh.documents);
    a.heads = static_cast<int>(sh.heads);
    a.kv_heads = static_cast<int>(sh.kv_heads);
    a.group = a.heads / a.kv_heads;
    a.head_dim = static_cast<int>(sh.head_dim);
    a.causal = sh.causal != 0;
    a.window = static_cast<int>(std::min<int64_t>(sh.window, INT32_MAX));
    a.scale = static_cast<float>(sh.scale);
    a.softcap = static_cast<float>(sh.softcap);
    return a;
}

// Parts of `rows` tokens of all documents, at most.
unsigned tiles(const DocAttention& a, int rows) {
    return static_cast<unsigned>(ceil_div(a.tokens, rows) + std::min(a.documents, a.tokens));
}

// Whole 16-byte chunks throughout: rows can be copied to LDS directly.
template <typename T>
bool whole_chunks(const DocAttention& a, std::initializer_list<const void*> arrays) {
    bool whole = a.head_dim % kChunk<T> == 0;
    for (const int64_t s : {a.q_stride, a.k_stride, a.v_stride, a.out_stride})
        whole = whole && s % kChunk<T> == 0 && s < (int64_t{1} << 25);  // a copy's lane offsets stay below 2^32 bytes
    for (const void* p : arrays) whole = whole && aligned_to(p, 16);
    return whole;
}

template <typename T, int kDim>
void launch_forward_dim(const DocAttention& a, T* out, bool direct, hipStream_t s) {
    const dim3 grid(tiles(a, kRows) * a.heads);
    if (direct)
        forward_kernel<T, kDim, true><<<grid, kThreads, 0, s>>>(a, out);
    else
        forward_kernel<T, kDim, false><<<grid, kThreads, 0, s>>>(a, out);
}

template <typename T>
int launch_forward(const DocAttention& a, void* out, hipStream_t s) {
    const bool direct = whole_chunks<T>(a, {a.q, a.k, a.v, out});
    T* const to = static_cast<T*>(out);
    if (a.head_dim <= 64)
        launch_forward_dim<T, 64>(a, to, direct, s);
    else if (a.head_dim <= 128)
        launch_forward_dim<T, 128>(a, to, direct, s);
    else
        launch_forward_dim<T, 256>(a, to, direct, s);
    return check_launch("document_attention");
}

template <typename T>
int launch_backward(const DocAttention& a, hipStream_t s) {
    dq_rows_kernel<T><<<dim3(tiles(a, 4), a.heads), 256, 0, s>>>(a);
    dkv_rows_kernel<T><<<dim3(tiles(a, 4), a.kv_heads), 256, 0, s>>>(a);
    return check_launch("document_attention_backward");
}

size_t backward_bytes(const DocAttention& a) {
    Layout l;
    l.add<float>(static_cast<size_t>(a.heads) * a.tokens);
    return l.bytes;
}

}  // namespace

extern "C" {

size_t dllm_hip_document_attention_workspace(const dllm_hip_document_attention_shape* sh) {
    (void)sh;
    return 0;
}

int dllm_hip_document_attention(const dllm_hip_document_attention_shape* sh, const void* q, const void* k,
                                const void* v, const int64_t* offsets, const int64_t* prefix, const float* slopes,
                                void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    (void)workspace, (void)workspace_bytes;
    DLLM_TRY(check_shape(sh));
    if (sh->tokens == 0 || sh->documents == 0) return kOk;
    DLLM_REQUIRE(q && k && v && offsets && out, "null q, k, v, offsets or out");
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(q, size) && aligned_to(k, size) && aligned_to(v, size) && aligned_to(out, size) &&
                     aligned_to(offsets, 8) && aligned_to(prefix, 8) && aligned_to(slopes, 4) && aligned_to(lse, 4),
                 "pointers must be aligned to the element");
    DocAttention a = arguments(*sh);
    a.q = q, a.k = k, a.v = v, a.offsets = offsets, a.prefix = prefix, a.slopes = slopes, a.lse = lse;
    auto s = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return launch_forward<float>(a, out, s);
        case kBFloat16: return launch_forward<__bf16>(a, out, s);
        default: return launch_forward<_Float16>(a, out, s);
    }
}

size_t dllm_hip_document_attention_backward_workspace(const dllm_hip_document_attention_shape* sh) {
    return check_shape(sh) == kOk ? backward_bytes(arguments(*sh)) : 0;
}

int dllm_hip_document_attention_backward(const dllm_hip_document_attention_shape* sh, const void* q, const void* k,
                                         const void* v, const int64_t* offsets, const int64_t* prefix,
                                         const float* slopes, const void* out, const float* lse, const void* dout,
                                         void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                         void* stream) {
    DLLM_TRY(check_shape(sh));
    if (sh->tokens == 0 || sh->documents == 0) return kOk;
    DLLM_REQUIRE(q && k && v && offsets && out && lse && dout && dq && dk && dv,
                 "null q, k, v, offsets, out, lse, dout, dq, dk or dv");
    const size_t size = element_bytes(sh->dtype);
    for (const void* p : {q, k, v, out, dout, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
        DLLM_REQUIRE(aligned_to(p, size), "pointers must be aligned to the element");
    DLLM_REQUIRE(aligned_to(offsets, 8) && aligned_to(prefix, 8) && aligned_to(slopes, 4) && aligned_to(lse, 4),
                 "pointers must be aligned to the element");
    DocAttention a = arguments(*sh);
    DLLM_REQUIRE(workspace && workspace_bytes >= backward_bytes(a), "workspace too small for document_attention_backward");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    a.q = q, a.k = k, a.v = v, a.offsets = offsets, a.prefix = prefix, a.slopes = slopes, a.out = out, a.dout = dout;
    a.lse = const_cast<float*>(lse);
    a.dq = dq, a.dk = dk, a.dv = dv;
    Carve c(workspace, workspace_bytes);
    a.delta = c.take<float>(static_cast<size_t>(a.heads) * a.tokens);
    auto s = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return launch_backward<float>(a, s);
        case kBFloat16: return launch_backward<__bf16>(a, s);
        default: return launch_backward<_Float16>(a, s);
    }
}

}  // extern "C"
