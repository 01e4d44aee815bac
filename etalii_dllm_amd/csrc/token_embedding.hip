// Embedding lookup with scaling, and the table's gradient.
//
//   out[t] = scale * table[token t]          dtable[v] = (dtable[v] +) scale * sum over t with token v of dout[t]
//
// Bound: HBM. The lookup reads and writes each element once, a thread 16 bytes. The gradient writes the whole table, or with
// accumulate reads and writes the rows of tokens that occur; its sums are token_rows.hip's. Measured: 16384 tokens of 2304 in
// bfloat16 27 us, 5.5 TB/s (tokens that come again are read from the caches); the gradient of 8192 tokens onto 151936 x 1536
// 108 us, 78 of them the table's zeroes at 6.0 TB/s with the sort beside them. One token is a launch, 6.7 us.
#include "common.h"
#include "dllm_hip.h"
#include "element.h"
#include "token_rows.h"

using namespace dllm_hip;

namespace {

constexpr int kThreads = 256;

struct LookupArgs {
    const int64_t* tokens;
    int64_t count, vocabulary, dim, stride, chunks;
    float scale;
};

// Chunk i of a row of `chunks`; kWidth elements of it.
template <typename T, int kWidth, typename Index>
__global__ __launch_bounds__(kThreads) void lookup_kernel(const T* __restrict__ table, T* __restrict__ out, LookupArgs a) {
    const Index i = static_cast<Index>(block_id()) * kThreads + threadIdx.x;
    const Index t = i / static_cast<Index>(a.chunks), c = i - t * static_cast<Index>(a.chunks);
    if (t >= static_cast<Index>(a.count)) return;
    const int64_t token = a.tokens[t];
    float v[kWidth] = {};
    if (token >= 0 && token < a.vocabulary) {
        load_as_float<T, kWidth>(table + token * a.dim + static_cast<int64_t>(c) * kWidth, v);
#pragma unroll
        for (int j = 0; j < kWidth; ++j) v[j] *= a.scale;
    }
    store_from_float<T, kWidth>(out + static_cast<int64_t>(t) * a.stride + static_cast<int64_t>(c) * kWidth, v);
}

template <typename T, int kWidth>
int launch_lookup(const void* table, void* out, LookupArgs a, hipStream_t stream) {
    a.chunks = a.dim / kWidth;
    const size_t items = static_cast<size_t>(a.count) * a.chunks;
    const dim3 grid = grid_of(ceil_div(items, kThreads));
    const T* from = static_cast<const T*>(table);
    T* to = static_cast<T*>(out);
    // (threads past the last item, up to a row of workgroups, are counted too)
    if (items + (size_t{1} << 29) < (size_t{1} << 32))
        lookup_kernel<T, kWidth, uint32_t><<<grid, kThreads, 0, stream>>>(from, to, a);
    else
        lookup_kernel<T, kWidth, uint64_t><<<grid, kThreads, 0, stream>>>(from, to, a);
    return check_launch("token_embedding");
}

template <typename T>
int launch_lookup_of(const void* table, void* out, const LookupArgs& a, hipStream_t stream) {
    constexpr int kWide = kChunk<T>;
    const bool wide = a.dim % kWide == 0 && a.stride % kWide == 0 && aligned_to(table, 16) && aligned_to(out, 16);
    return wide ? launch_lookup<T, kWide>(table, out, a, stream) : launch_lookup<T, 1>(table, out, a, stream);
}

int check_shape(const dllm_hip_token_embedding_shape* sh) {
    DLLM_REQUIRE(sh != nullptr, "null shape");
    DLLM_REQUIRE(sh->dtype >= 0 && sh->dtype <= 2, "dtype must be float32 (0), bfloat16 (1) or float16 (2)");
    DLLM_REQUIRE(sh->tokens >= 0 && sh->tokens < kMaxSortTokens, "tokens must be in [0, 2^27)");
    DLLM_REQUIRE(sh->vocabulary >= 1 && sh->vocabulary < (int64_t{1} << 31), "vocabulary must be in [1, 2^31)");
    DLLM_REQUIRE(sh->dim >= 1 && sh->dim <= (1 << 20), "dim must be in [1, 2^20]");
    DLLM_REQUIRE(sh->tokens * sh->dim < (int64_t{1} << 40), "tokens * dim must be below 2^40");
    DLLM_REQUIRE(sh->stride == 0 || (sh->stride >= sh->dim && sh->stride < (int64_t{1} << 32)), "a token stride must be 0 or at least dim, below 2^32");
    DLLM_REQUIRE(sh->scale >= -0x1p60 && sh->scale <= 0x1p60, "scale must be in [-2^60, 2^60]");
    return kOk;
}

struct GradientLayout {
    size_t part, bytes;
    explicit GradientLayout(const dllm_hip_token_embedding_shape& sh) {
        part = token_sums_part_floats(sh.tokens, sh.dim);
        Layout l;
        add_token_order(l, sh.tokens);
        l.add<float>(part);
        bytes = l.bytes;
    }
};

}  // namespace

extern "C" {

int dllm_hip_token_embedding(const dllm_hip_token_embedding_shape* sh, const void* table, const int64_t* tokens, void* out,
                             void* stream) {
    DLLM_TRY(check_shape(sh));
    if (sh->tokens == 0) return kOk;
    DLLM_REQUIRE(table && tokens && out, "null table, tokens or out");
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(table, size) && aligned_to(out, size) && aligned_to(tokens, 8), "pointers must be aligned to the element");
    const LookupArgs a{tokens, sh->tokens, sh->vocabulary, sh->dim, sh->stride ? sh->stride : sh->dim, 0, static_cast<float>(sh->scale)};
    auto s = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return launch_lookup_of<float>(table, out, a, s);
        case kBFloat16: return launch_lookup_of<__bf16>(table, out, a, s);
        default: return launch_lookup_of<_Float16>(table, out, a, s);
    }
}

size_t dllm_hip_token_embedding_backward_workspace(const dllm_hip_token_embedding_shape* sh) {
    return check_shape(sh) == kOk ? GradientLayout(*sh).bytes : 0;
}

int dllm_hip_token_embedding_backward(const dllm_hip_token_embedding_shape* sh, const int64_t* tokens, const void* dout, void* dtable,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    DLLM_TRY(check_shape(sh));
    DLLM_REQUIRE(dtable || (sh->tokens == 0 && sh->accumulate), "null dtable");
    DLLM_REQUIRE(sh->tokens == 0 || (tokens && dout), "null tokens or dout");
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(dout, size) && aligned_to(dtable, size) && aligned_to(tokens, 8), "pointers must be aligned to the element");
    auto s = static_cast<hipStream_t>(stream);
    const size_t table_bytes = sh->accumulate ? 0 : static_cast<size_t>(sh->vocabulary) * sh->dim * size;
    if (sh->tokens == 0) return table_bytes ? fill_words(dtable, table_bytes, 0, s) : static_cast<int>(kOk);
    const GradientLayout layout(*sh);
    DLLM_REQUIRE(workspace && workspace_bytes >= layout.bytes, "workspace too small for token_embedding_backward");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    Carve c(workspace, workspace_bytes);
    TokenSums a{};
    a.order = take_token_order(c, sh->tokens);
    a.n = sh->tokens, a.vocabulary = sh->vocabulary, a.dim = sh->dim, a.stride = sh->stride ? sh->stride : sh->dim;
    a.rows = dout, a.scale = static_cast<float>(sh->scale), a.part = c.take<float>(layout.part);
    a.table = dtable, a.accumulate = sh->accumulate != 0;
    DLLM_TRY(sort_tokens(tokens, sh->tokens, sh->vocabulary, a.order, dtable, table_bytes, 0, s));
    return launch_token_sums(a, sh->dtype, s);
}

}  // extern "C"
