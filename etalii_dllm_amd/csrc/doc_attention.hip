// Attention within packed documents, forward and backward (see doc_attention.h for the mask and the score).
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i)
//   dP = dout v^T,  dS = p (dP - dout . out) cap' scale,  dq = dS k,  dk = dS^T q,  dv = p^T dout
#include <algorithm>

#include "common.h"
#include "doc_attention.h"
#include "dllm_hip.h"
#include "workspace.h"

using namespace dllm_hip;

namespace {

constexpr int kSmallestTile = 4;

template <typename T>
__global__ __launch_bounds__(256) void forward_rows_kernel(DocAttention a, T* out) {
    Document doc;
    int first;
    if (!locate_tile<4>(a, blockIdx.x, doc, first)) return;
    const int i = first + (static_cast<int>(threadIdx.x) >> 6), head = blockIdx.y;
    if (i >= doc.end) return;
    float o[kLaneDims], lse;
    attention_row<T>(a, doc, head, i, o, lse);
    store_row(out + i * a.out_stride + static_cast<int64_t>(head) * a.head_dim, o, a.head_dim);
    if (a.lse && (threadIdx.x & 63) == 0) a.lse[static_cast<int64_t>(head) * a.tokens + i] = lse;
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
    DLLM_REQUIRE(sh->softcap >= 0.0, "softcap must not be negative");
    const int64_t q = sh->heads * sh->head_dim, k = sh->kv_heads * sh->head_dim;
    for (const int64_t s : {sh->q_stride, sh->out_stride}) DLLM_REQUIRE(s == 0 || s >= q, "a token stride must be 0 or at least heads * head_dim");
    for (const int64_t s : {sh->k_stride, sh->v_stride}) DLLM_REQUIRE(s == 0 || s >= k, "a token stride must be 0 or at least heads * head_dim");
    // a grid's x extent times its workgroup is below 2^32
    DLLM_REQUIRE(static_cast<int64_t>(ceil_div(sh->tokens, kSmallestTile)) + std::min(sh->documents, sh->tokens) < (1 << 24),
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

template <typename T>
int launch_forward(const DocAttention& a, void* out, hipStream_t s) {
    forward_rows_kernel<T><<<dim3(tiles(a, 4), a.heads), 256, 0, s>>>(a, static_cast<T*>(out));
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
