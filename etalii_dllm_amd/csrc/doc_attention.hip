// Attention within packed documents: the entry points. The kernels are doc_attention_forward.h's and
// doc_attention_backward.h's, compiled for each type in doc_attention_{f32,bf16,f16}.hip.
#include <algorithm>
#include <initializer_list>

#include "common.h"
#include "dllm_hip.h"
#include "doc_attention.h"
#include "workspace.h"

using namespace dllm_hip;

namespace {

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
    // in float32 the scale, the cap, their quotient and any of them times 2 / log 2 are then ordinary numbers
    DLLM_REQUIRE(sh->softcap == 0.0 || (sh->softcap >= 0x1p-64 && sh->softcap <= 0x1p64), "softcap must be 0 or in [2^-64, 2^64]");
    DLLM_REQUIRE(sh->scale >= 0x1p-60 && sh->scale <= 0x1p60, "scale must be in [2^-60, 2^60]");
    const int64_t q = sh->heads * sh->head_dim, k = sh->kv_heads * sh->head_dim;
    for (const int64_t s : {sh->q_stride, sh->out_stride}) DLLM_REQUIRE(s == 0 || s >= q, "a token stride must be 0 or at least heads * head_dim");
    for (const int64_t s : {sh->k_stride, sh->v_stride}) DLLM_REQUIRE(s == 0 || s >= k, "a token stride must be 0 or at least heads * head_dim");
    // a grid's x extent times its workgroup is below 2^32
    DLLM_REQUIRE((static_cast<int64_t>(ceil_div(sh->tokens, kDocTileRows / 2)) + sh->documents) * sh->heads < (1 << 24),
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

size_t token_bytes(const DocAttention& a, int64_t dtype, bool backward) {
    return dtype == kFloat32 ? packed_token_bytes<float>(a, backward) : packed_token_bytes<__bf16>(a, backward);
}

// The sources' copies; backward, the rows' statistics and the parts of heads that share keys too.
struct AttentionLayout {
    size_t packed, stats, part, bytes;
    AttentionLayout(const DocAttention& a, int64_t dtype, bool backward) {
        packed = token_bytes(a, dtype, backward) * static_cast<size_t>(a.tokens);
        stats = backward ? static_cast<size_t>(a.heads) * a.tokens : 0;
        part = backward && a.group > 1 ? stats * a.head_dim : 0;
        Layout l;
        l.add<char>(packed);
        for (const size_t n : {stats, part, part}) l.add<float>(n);
        bytes = l.bytes;
    }
};

}  // namespace

extern "C" {

size_t dllm_hip_document_attention_workspace(const dllm_hip_document_attention_shape* sh) {
    return check_shape(sh) == kOk ? AttentionLayout(arguments(*sh), sh->dtype, false).bytes : 0;
}

int dllm_hip_document_attention(const dllm_hip_document_attention_shape* sh, const void* q, const void* k,
                                const void* v, const int64_t* offsets, const int64_t* prefix, const float* slopes,
                                void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    DLLM_TRY(check_shape(sh));
    if (sh->tokens == 0 || sh->documents == 0) return kOk;
    DLLM_REQUIRE(q && k && v && offsets && out, "null q, k, v, offsets or out");
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(q, size) && aligned_to(k, size) && aligned_to(v, size) && aligned_to(out, size) &&
                     aligned_to(offsets, 8) && aligned_to(prefix, 8) && aligned_to(slopes, 4) && aligned_to(lse, 4),
                 "pointers must be aligned to the element");
    DocAttention a = arguments(*sh);
    const AttentionLayout layout(a, sh->dtype, false);
    DLLM_REQUIRE(workspace && workspace_bytes >= layout.bytes, "workspace too small for document_attention");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    a.q = q, a.k = k, a.v = v, a.offsets = offsets, a.prefix = prefix, a.slopes = slopes, a.lse = lse;
    char* const packed = Carve(workspace, workspace_bytes).take<char>(layout.packed);
    auto s = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return launch_document_attention<float>(a, out, packed, s);
        case kBFloat16: return launch_document_attention<__bf16>(a, out, packed, s);
        default: return launch_document_attention<_Float16>(a, out, packed, s);
    }
}

size_t dllm_hip_document_attention_backward_workspace(const dllm_hip_document_attention_shape* sh) {
    return check_shape(sh) == kOk ? AttentionLayout(arguments(*sh), sh->dtype, true).bytes : 0;
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
    const AttentionLayout layout(a, sh->dtype, true);
    DLLM_REQUIRE(workspace && workspace_bytes >= layout.bytes, "workspace too small for document_attention_backward");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    a.q = q, a.k = k, a.v = v, a.offsets = offsets, a.prefix = prefix, a.slopes = slopes, a.out = out, a.dout = dout;
    a.lse = const_cast<float*>(lse);
    a.dq = dq, a.dk = dk, a.dv = dv;
    Carve c(workspace, workspace_bytes);
    char* const packed = c.take<char>(layout.packed);
    a.delta = c.take<float>(layout.stats);
    a.dk_part = c.take<float>(layout.part);
    a.dv_part = c.take<float>(layout.part);
    auto s = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return launch_document_attention_backward<float>(a, packed, s);
        case kBFloat16: return launch_document_attention_backward<__bf16>(a, packed, s);
        default: return launch_document_attention_backward<_Float16>(a, packed, s);
    }
}

}  // extern "C"
