// Rotary positions of several axes for q and k in one launch, forward and inverse.
//
// Pair p of token t is turned by a = positions[axis(p)][t] inv_freq[p]: (u, v) -> (u cos a - v sin a, v cos a + u sin a),
// inverse with -a. The angle is formed in double and reduced to a fraction of a turn there (the turns are exact to 2^-53
// of their number), so the float32 sine and cosine see an argument of at most half a turn and are good to their last bits
// at any position. All heads of a token share its angles: a workgroup computes the sines and cosines of its tokens once
// into LDS, then turns every head of q and k.
//
// Bound: HBM, each element read and written once; per element a multiply, an FMA and 4 bytes of LDS. 16384 tokens, 12/2 heads of
// 128 in bfloat16: 28 us, 4.2 TB/s. One token: 7.5 us, the launch.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "dllm_hip.h"
#include "element.h"

using namespace dllm_hip;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;
constexpr int kTableEntries = 1024;  // (token, pair) angles of a workgroup: 8 KB of LDS

struct RopeArgs {
    const int64_t* positions;
    const double* inv_freq;
    const uint8_t* pair_axis;
    int64_t tokens;
    int64_t stride[2], out_stride[2];
    int heads[2];
    int head_dim, pairs, axes, inverse, block_tokens;
};

// kWidth elements of a head at once: kWidth consecutive pairs' first and second halves, or kWidth / 2 interleaved pairs
// (kWidth 1 interleaved: one whole pair of single elements).
template <typename T, int kWidth, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(const T* q, const T* k, T* q_out, T* k_out, RopeArgs a) {
    __shared__ float cos_of[kTableEntries], sin_of[kTableEntries];
    const int64_t t0 = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * a.block_tokens;
    if (t0 >= a.tokens) return;
    const int tokens = static_cast<int>(a.tokens - t0 < a.block_tokens ? a.tokens - t0 : a.block_tokens);
    for (int e = threadIdx.x; e < tokens * a.pairs; e += kThreads) {
        const int t = e / a.pairs, p = e - t * a.pairs;
        const int axis = a.pair_axis[p];
        float c = 1.0f, s = 0.0f;
        if (axis < a.axes) {
            const double position = static_cast<double>(a.positions[axis * a.tokens + t0 + t]);
            const double turns = position * a.inv_freq[p] * 0.15915494309189535;  // 1 / (2 pi)
            const float half_turns = static_cast<float>(2.0 * (turns - rint(turns)));
            sincospif(half_turns, &s, &c);
        }
        cos_of[e] = c;
        sin_of[e] = a.inverse ? -s : s;
    }
    __syncthreads();

    constexpr int kPairWidth = kInterleaved ? (kWidth > 1 ? kWidth / 2 : 1) : kWidth;  // pairs per item
    const int heads = a.heads[0] + a.heads[1];
    const int turned = a.pairs / kPairWidth;                   // items of a head that turn
    const int copied = (a.head_dim - 2 * a.pairs + kWidth - 1) / kWidth;  // items past the turned dimensions
    const int per_head = turned + copied;
    const int items = tokens * heads * per_head;
    for (int i = threadIdx.x; i < items; i += kThreads) {
        const int row = i / per_head, item = i - row * per_head;
        const int t = row / heads;
        int head = row - t * heads;
        const int which = head >= a.heads[0];
        head -= which ? a.heads[0] : 0;
        const T* src = (which ? k : q) + (t0 + t) * a.stride[which] + static_cast<int64_t>(head) * a.head_dim;
        T* dst = (which ? k_out : q_out) + (t0 + t) * a.out_stride[which] + static_cast<int64_t>(head) * a.head_dim;
        if (item >= turned) {
            const int d = 2 * a.pairs + (item - turned) * kWidth;
            if (src != dst) *reinterpret_cast<Pack<T, kWidth>*>(dst + d) = *reinterpret_cast<const Pack<T, kWidth>*>(src + d);
            continue;
        }
        const int p = item * kPairWidth;
        const float* c = cos_of + t * a.pairs + p;
        const float* s = sin_of + t * a.pairs + p;
        if constexpr (!kInterleaved) {
            float u[kWidth], v[kWidth], x[kWidth], y[kWidth];
            load_as_float<T, kWidth>(src + p, u);
            load_as_float<T, kWidth>(src + a.pairs + p, v);
#pragma unroll
            for (int j = 0; j < kWidth; ++j) {
                x[j] = fmaf(u[j], c[j], -(v[j] * s[j]));
                y[j] = fmaf(v[j], c[j], u[j] * s[j]);
            }
            store_from_float<T, kWidth>(dst + p, x);
            store_from_float<T, kWidth>(dst + a.pairs + p, y);
        } else if constexpr (kWidth == 1) {
            const float u = static_cast<float>(src[2 * p]), v = static_cast<float>(src[2 * p + 1]);
            dst[2 * p] = static_cast<T>(fmaf(u, c[0], -(v * s[0])));
            dst[2 * p + 1] = static_cast<T>(fmaf(v, c[0], u * s[0]));
        } else {
            float u[kWidth], x[kWidth];
            load_as_float<T, kWidth>(src + 2 * p, u);
#pragma unroll
            for (int j = 0; j < kWidth / 2; ++j) {
                x[2 * j] = fmaf(u[2 * j], c[j], -(u[2 * j + 1] * s[j]));
                x[2 * j + 1] = fmaf(u[2 * j + 1], c[j], u[2 * j] * s[j]);
            }
            store_from_float<T, kWidth>(dst + 2 * p, x);
        }
    }
}

template <typename T>
int launch_rope_axes(const void* q, const void* k, void* q_out, void* k_out, const RopeArgs& a, bool interleaved,
                     bool wide, hipStream_t stream) {
    const size_t blocks = ceil_div(static_cast<size_t>(a.tokens), static_cast<size_t>(a.block_tokens));
    const size_t x = std::min<size_t>(blocks, 1 << 20);  // a grid's x extent times its workgroup is below 2^32
    const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(ceil_div(blocks, x)));
    const T *qt = static_cast<const T*>(q), *kt = static_cast<const T*>(k);
    T *qo = static_cast<T*>(q_out), *ko = static_cast<T*>(k_out);
    if (wide && interleaved)
        rope_axes_kernel<T, kChunk<T>, true><<<grid, kThreads, 0, stream>>>(qt, kt, qo, ko, a);
    else if (wide)
        rope_axes_kernel<T, kChunk<T>, false><<<grid, kThreads, 0, stream>>>(qt, kt, qo, ko, a);
    else if (interleaved)
        rope_axes_kernel<T, 1, true><<<grid, kThreads, 0, stream>>>(qt, kt, qo, ko, a);
    else
        rope_axes_kernel<T, 1, false><<<grid, kThreads, 0, stream>>>(qt, kt, qo, ko, a);
    return check_launch("rope_axes");
}

}  // namespace

extern "C" int dllm_hip_rope_axes(const dllm_hip_rope_axes_shape* sh, const void* q, const void* k,
                                  const int64_t* positions, const double* inv_freq, const uint8_t* pair_axis,
                                  void* q_out, void* k_out, void* stream) {
    DLLM_REQUIRE(sh != nullptr, "null shape");
    DLLM_REQUIRE(sh->dtype >= 0 && sh->dtype <= 2, "dtype must be float32 (0), bfloat16 (1) or float16 (2)");
    DLLM_REQUIRE(sh->tokens >= 0 && sh->tokens < (int64_t{1} << 31), "tokens must be in [0, 2^31)");
    DLLM_REQUIRE(sh->q_heads >= 0 && sh->k_heads >= 0 && sh->q_heads <= 65535 && sh->k_heads <= 65535,
                 "head counts must be in [0, 65535]");
    DLLM_REQUIRE(sh->pairs >= 0 && sh->pairs <= kMaxPairs, "pairs must be in [0, 256]");
    DLLM_REQUIRE(sh->head_dim >= 1 && sh->head_dim <= 65536 && 2 * sh->pairs <= sh->head_dim,
                 "2 * pairs must not exceed head_dim");
    // (a thread counts them in steps of a workgroup, past the last)
    DLLM_REQUIRE((sh->q_heads + sh->k_heads) * sh->head_dim <= INT32_MAX - kThreads,
                 "a token's heads must have fewer than 2^31 - 256 elements");
    DLLM_REQUIRE(sh->axes >= 1 && sh->axes <= 255, "axes must be in [1, 255]");
    const int64_t heads[2] = {sh->q_heads, sh->k_heads};
    const int64_t in[2] = {sh->q_stride, sh->k_stride}, out[2] = {sh->q_out_stride, sh->k_out_stride};
    const void* const srcs[2] = {q, k};
    void* const dsts[2] = {q_out, k_out};
    const size_t size = element_bytes(sh->dtype);
    const int64_t chunk = static_cast<int64_t>(16 / size);
    RopeArgs a{};
    bool wide = sh->head_dim % chunk == 0 && (sh->interleaved ? 2 * sh->pairs : sh->pairs) % chunk == 0;
    for (int i = 0; i < 2; ++i) {
        const int64_t packed = heads[i] * sh->head_dim;
        DLLM_REQUIRE((in[i] == 0 || in[i] >= packed) && (out[i] == 0 || out[i] >= packed),
                     "a token stride must be 0 or at least heads * head_dim");
        a.heads[i] = static_cast<int>(heads[i]);
        a.stride[i] = in[i] ? in[i] : packed;
        a.out_stride[i] = out[i] ? out[i] : packed;
        if (sh->tokens == 0 || heads[i] == 0) continue;
        DLLM_REQUIRE(srcs[i] && dsts[i], "null q, k or output");
        DLLM_REQUIRE(aligned_to(srcs[i], size) && aligned_to(dsts[i], size), "pointers must be aligned to the element");
        DLLM_REQUIRE(srcs[i] != dsts[i] || a.stride[i] == a.out_stride[i], "in place needs equal strides");
        wide = wide && aligned_to(srcs[i], 16) && aligned_to(dsts[i], 16) && a.stride[i] % chunk == 0 &&
               a.out_stride[i] % chunk == 0;
    }
    if (sh->tokens == 0 || heads[0] + heads[1] == 0) return kOk;
    DLLM_REQUIRE(sh->pairs == 0 || (positions && inv_freq && pair_axis), "null positions, inv_freq or pair_axis");
    DLLM_REQUIRE(aligned_to(positions, 8) && aligned_to(inv_freq, 8), "positions and inv_freq must be aligned to the element");
    a.positions = positions;
    a.inv_freq = inv_freq;
    a.pair_axis = pair_axis;
    a.tokens = sh->tokens;
    a.head_dim = static_cast<int>(sh->head_dim);
    a.pairs = static_cast<int>(sh->pairs);
    a.axes = static_cast<int>(sh->axes);
    a.inverse = sh->inverse != 0;
    // Tokens of a workgroup: enough for about four items to a thread, as far as their angles fit the table and there are
    // workgroups for all CUs. (16384 tokens, 12/2 heads of 128 in bfloat16: 31 us with one token
    // each, 28 with these.)
    const int64_t width = wide ? chunk : 1, pair_width = sh->interleaved ? std::max<int64_t>(width / 2, 1) : width;
    const int64_t items = (sh->q_heads + sh->k_heads) * (sh->pairs / pair_width + (sh->head_dim - 2 * sh->pairs) / width);
    const int64_t by_items = 4 * kThreads / std::max<int64_t>(items, 1), by_table = kTableEntries / std::max<int64_t>(sh->pairs, 1);
    a.block_tokens = static_cast<int>(std::clamp<int64_t>(std::min({by_items, by_table, sh->tokens / 1024}), 1, kTableEntries));
    auto s = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return launch_rope_axes<float>(q, k, q_out, k_out, a, sh->interleaved != 0, wide, s);
        case kBFloat16: return launch_rope_axes<__bf16>(q, k, q_out, k_out, a, sh->interleaved != 0, wide, s);
        default: return launch_rope_axes<_Float16>(q, k, q_out, k_out, a, sh->interleaved != 0, wide, s);
    }
}
