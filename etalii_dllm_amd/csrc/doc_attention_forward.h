// Attention within packed documents: the forward kernel (doc_attention.h: the mask and the score).
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp s_ij
#pragma once

#include "common.h"
#include "doc_attention.h"
#include "doc_tile.h"

namespace dllm_hip {

// Keys of a tile, and whether two buffers of K and V tiles fit LDS: 64 or 128 KB for 16-bit types, 96 KB for float32's planes.
template <typename T, int kDim>
constexpr int kKeys = kPlanes<T> == 1 || kDim <= 64 ? 64 : 32;
template <typename T, int kDim>
constexpr int kBuffers = 4 * kKeys<T, kDim> * kDim * 2 * kPlanes<T> <= 128 * 1024 ? 2 : 1;

// Forward. A wave's lane owns one query (two lanes: its halves); keys go through LDS in tiles, two buffers deep.
//
//   X = K Q^T (32 keys x 32 queries at a time)     s = X scale, capped, biased, in units of log 2
//   m = running maximum, P = 2^(s - m), l = sum P   O^T += V^T P
//
// The running maximum is moved only when some query of the wave has outgrown it by 2^8: until then P stays below 2^8, which
// float32 sums and 16-bit products hold as well as values below one. P is rounded to the type for the second product, as the
// type's users expect of it; l is the sum of P before that.
//
// Bound: the way of few waves through products, softmax and waits in series; no unit is full. 8192 tokens in bfloat16 (matrix
// cores, vector units and LDS busy; waves waiting for memory or LDS, and for their turn to issue): 16/8 heads of 128, 41, 45 and
// 21%; 31 and 26% of 1.6 waves on a SIMD; heads of 64, 36, 63 and 19%; 31 and 28% of 2.5; 8/4 heads of 256, 32, 32 and 16%; 26 and
// 23% of 0.9. float32, 4096 tokens of 16/8 heads of 128: 45, 24 and 11%; 21 and 40% of 0.9. A loop of nothing but 16-bit products of
// random numbers reaches 1540 TFLOP/s; of the scores that count these are 320 to 364 us, 755 to 860 TFLOP/s, for heads of 128 (567 to
// 610 us and 900 to 970 without the causal mask), 170 to 197 us and 700 to 810 for 64, 355 to 390 us and 705 to 775 for 256, and
// 410 to 435 us for float32, of six products 945 to 1000. Short calls are bound by the way of one workgroup through a row's keys: about 1.1 us a tile
// of 64 (16-bit), 3.1 us one of 32 (float32).
template <typename T, int kDim, bool kLargeCap>
__global__ __launch_bounds__(kDocThreads, kPlanes<T> == 1 ? (kDim <= 64 ? 3 : kDim <= 128 ? 2 : 1) : 1) void forward_kernel(DocAttention a, T* out) {
    using Shape = TileShape<T, kDim>;
    constexpr int kTile = kKeys<T, kDim>;
    using Copy = TileCopy<T, kDim, kTile, kDocThreads>;
    constexpr int kTileBytes = Copy::kBytes;
    constexpr bool kPaired = kPair<T, kDim> == 2;
    constexpr int kParts = kWaveDim<T, kDim> / 32, kOwn = kBlockRows<T, kDim>;
    constexpr bool kAhead = kBuffers<T, kDim> == 2;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers<T, kDim> * 2 * kTileBytes];  // K, V of each buffer
    __shared__ __attribute__((aligned(16))) char pair_lds[kPaired ? kTile / 32 * 4 * 4096 : 16];

    // the heads that share keys are 8 workgroups (or a divisor of it) apart: on the same L2
    const int turn = static_cast<int>(blockIdx.x) % a.heads;
    const int head = (turn % a.kv_heads) * a.group + turn / a.kv_heads;
    const int kv = head / a.group;
    Document doc;
    int first;
    if (!locate_tile<kOwn, true>(a, blockIdx.x / a.heads, doc, first)) return;

    const int wave = uniform(static_cast<int>(threadIdx.x) >> 6), lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5;
    const int part = kPaired ? wave & 1 : 0, first_part = part * kParts;  // of the dimensions
    const int wave_first = first + 32 * (kPaired ? wave >> 1 : wave), wave_last = min(wave_first + 31, doc.end - 1);
    const bool working = wave_first < doc.end;
    const int i = min(wave_first + (lane & 31), doc.end - 1);
    const Span span = key_span(a, doc, i);
    const bool few = kPlanes<T> == 1 && all_see_few(doc, span);

    // keys of the workgroup: [low, high) in whole tiles of the document, and the tiles of the prefix before them
    const int low = key_span(a, doc, first).low;
    const int high = max(key_span(a, doc, min(first + kOwn, doc.end) - 1).high, doc.prefix_end);
    const int low_tile = (low - doc.start) / kTile, prefix_tiles = (doc.prefix_end - doc.start + kTile - 1) / kTile;
    const int tiles = (high - doc.start + kTile - 1) / kTile;
    // the wave's: keys that all its queries see, and that any sees
    const Span first_span = key_span(a, doc, wave_first), last_span = key_span(a, doc, wave_last);
    const int any_low = first_span.low, any_high = last_span.high, all_low = last_span.low, all_high = first_span.high;

    const Copy copy_k(a.sources[1], kv), copy_v(a.sources[2], kv);
    const TileView<T, kDim, kTile> view;
    LdsByte* const buffers = (LdsByte*)lds;

    // the first tile is on its way while the lane's row is read
    auto next_tile = [&](int t) { return t + 1 < prefix_tiles ? t + 1 : max(t + 1, low_tile); };
    auto fetch = [&](int t, int buffer) {
        const int from = doc.start + t * kTile;
        copy_k(from, doc.end - from, buffers + buffer * 2 * kTileBytes);
        copy_v(from, doc.end - from, buffers + buffer * 2 * kTileBytes + kTileBytes);
    };
    int t = next_tile(-1);
    if (kAhead) fetch(t, 0);
    const Column<T, kDim> q(a.sources[0], head, i, part);

    const CapTerms<T, kLargeCap> cap(a);
    const float slope = a.slopes ? a.slopes[head] * kLog2E : 0.0f;

    Acc o[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[p][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    loads_arrived();
    for (int buffer = 0; t < tiles; buffer ^= kAhead) {
        tile_barrier();
        const int next = next_tile(t);
        if (!kAhead) {
            fetch(t, 0);
            tile_barrier();
        } else if (next < tiles) {
            fetch(next, buffer ^ 1);
        }
        const LdsByte* const k_tile = buffers + buffer * 2 * kTileBytes;
        const LdsByte* const v_tile = k_tile + kTileBytes;
        const int from = doc.start + t * kTile;
        t = next;
        const bool in_prefix = from < doc.prefix_end;
        const bool idle = !working || !((from < any_high && from + kTile > any_low) || in_prefix);
        if (!kPaired && idle) continue;
        const bool all_seen = (from >= all_low && from + kTile <= all_high) || from + kTile <= doc.prefix_end;

        Acc x[kTile / 32];
#pragma unroll
        for (int b = 0; b < kTile / 32; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[b][r] = 0.0f;
            if (!kPaired || !idle) multiply_rows(view, k_tile, b, q, part, x[b]);
        }
        if constexpr (kPaired) {
            static_assert(kTile == 32);
            exchange({&x[0]}, (LdsByte*)pair_lds);
            if (idle) continue;
        }
        float s[kTile / 32][16];
#pragma unroll
        for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = x[b][r];
        float times = cap.times, plus = cap.plus;  // s times + plus: the score in units of log 2
        if (cap.capped) {
            float unused;
#pragma unroll
            for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = cap.bend(s[b][r], unused);
        }
        if (a.slopes) {
            const float away = static_cast<float>(i - from - 4 * half);
#pragma unroll
            for (int b = 0; b < kTile / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[b][r] = fmaf(-slope, fabsf(away - static_cast<float>(32 * b + 8 * (r / 4) + r % 4)), fmaf(s[b][r], times, plus));
            times = 1.0f, plus = 0.0f;
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
        top = fmaf(fmaxf(top, other_half(top)), times, plus);
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
        const float base = (m == -INFINITY ? 0.0f : m) - plus;
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
        for (int b = 0; b < kTile / 32; ++b) multiply_columns<T, kDim, kTile>(view, v_tile, b, Rows16<T>(s[b]), first_part, o);
        if (few) {
#pragma unroll
            for (int b = 0; b < kTile / 32; ++b) {
                keep_rest<T>(s[b]);
                multiply_columns<T, kDim, kTile>(view, v_tile, b, Rows16<T>(s[b]), first_part, o);
            }
        }
    }
    if (!kPaired && !working) return;
    l += other_half(l);

    // A hidden key counts as zero times its value: where that is infinite or NaN, the row is computed again from the keys
    // that it sees alone.
    const bool mine = wave_first + (lane & 31) < doc.end;
    const bool finite = all_finite(o) && l * 0.0f == 0.0f && m * 0.0f == 0.0f;
    const uint64_t marks = __ballot(!finite && mine);
    uint32_t spoilt = static_cast<uint32_t>(marks) | static_cast<uint32_t>(marks >> 32);
    if constexpr (kPaired) spoilt = pair_marks(spoilt, (LdsByte*)pair_lds);
    if (mine && !(spoilt >> (lane & 31) & 1)) {
        store_column(out + i * a.out_stride + static_cast<int64_t>(head) * a.head_dim, a.head_dim, a.whole, first_part, o, 1.0f / l);
        if (a.lse && half == 0 && part == 0) a.lse[static_cast<int64_t>(head) * a.tokens + i] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
    for (uint32_t left = part == 0 ? spoilt : 0; left; left &= left - 1) {
        const int row = wave_first + __ffs(left) - 1;
        float value[kLaneDims], lse;
        attention_row<T>(a, doc, head, row, value, lse);
        store_row(out + row * a.out_stride + static_cast<int64_t>(head) * a.head_dim, value, a.head_dim);
        if (a.lse && lane == 0) a.lse[static_cast<int64_t>(head) * a.tokens + row] = lse;
    }
}

template <typename T, int kDim>
void launch_forward(const DocAttention& a, T* out, hipStream_t s) {
    const unsigned blocks = doc_tiles(a, kBlockRows<T, kDim>) * a.heads;
    if constexpr (sizeof(T) == 2)
        if (large_cap(a)) {
            forward_kernel<T, kDim, true><<<blocks, kDocThreads, 0, s>>>(a, out);
            return;
        }
    forward_kernel<T, kDim, false><<<blocks, kDocThreads, 0, s>>>(a, out);
}

// doc_attention_wide.hip
extern template void launch_forward<__bf16, 256>(const DocAttention&, __bf16*, hipStream_t);
extern template void launch_forward<_Float16, 256>(const DocAttention&, _Float16*, hipStream_t);

template <typename T>
int launch_document_attention(DocAttention a, void* out, char* packed, hipStream_t s) {
    a.whole = whole_chunks(a, kChunk<T>, {a.q, a.k, a.v, out});
    set_sources<T>(a, false, packed, s);
    T* const to = static_cast<T*>(out);
    if (a.head_dim <= 64)
        launch_forward<T, 64>(a, to, s);
    else if (a.head_dim <= 128)
        launch_forward<T, 128>(a, to, s);
    else
        launch_forward<T, 256>(a, to, s);
    return check_launch("document_attention");
}

}  // namespace dllm_hip
