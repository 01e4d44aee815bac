// Attention within packed documents: the gradients (doc_attention.h: the mask and the score).
//
//   p_ij = exp(s_ij - lse_i),  dP = dout v^T,  dS = p (dP - dout . out) cap' scale,
//   dq = dS k,  dk = dS^T q,  dv = p^T dout
//
// dout . out of every row comes first (pack_kernel). Then there are two kinds of workgroups, each computing scores and dP for
// itself, so that every gradient is summed by one wave in one order: dq for 128 queries of a head over their keys, and dk and
// dv for 128 keys over the queries of one head that see them. That is seven products instead of five; sums of dq across
// workgroups by atomic additions would save two and give other bits every time. Heads that share keys leave their dk and dv in
// float32 and a last kernel adds them in head order.
//
// Both kinds run in one launch where that costs neither of them waves per CU (gradients_kernel): each fills the other's ends,
// and short calls have half the way (4 float32 documents of 256 tokens, 9/3 heads of 64: 71 to 48 us; 2447 tokens of
// 4/2 heads of 256: 655 to 383 us).
//
// Bound: as the forward, few waves' way through products, weights and waits in series, and two products more than the five that
// the gradients could not do without. 8192 tokens, 16/8 heads of 128 in bfloat16: dq 405 us, 1020 TFLOP/s of its three products
// (matrix cores, vector units and LDS busy 48, 38 and 24%; of its 1.7 waves on a SIMD 34% wait for memory or LDS and 29% for their
// turn); dk and dv 605 to 660 us, 830 to 910 of four (37, 24 and 23%; 38 and 17% of 0.9 waves); all together 1040 to 1150 us, 600 to
// 660 TFLOP/s of the five. 8/4 heads of 256, where dk and dv are two kinds of workgroups and eight products in all: 1200 us (38, 22
// and 21%; 32 and 28% of 0.9). float32, 4096 tokens of 16/8 heads of 128: 1210 us (55, 22 and 15%; 20 and 45% of 0.9).
// Another order of dk's and dv's products, with the next tile's scores formed before this one's sums, took 816 us for heads
// of 128.
#pragma once

#include <float.h>

#include <algorithm>

#include "common.h"
#include "doc_attention.h"
#include "doc_tile.h"

namespace dllm_hip {

// Rows of a tile that goes through LDS, and whether two buffers of two tiles fit it.
template <typename T, int kDim>
constexpr int kStream = kPlanes<T> == 1 || kDim <= 64 ? 64 : 32;
template <typename T, int kDim>
constexpr int kStreamBuffers = 4 * kStream<T, kDim> * kDim * 2 * kPlanes<T> <= 128 * 1024 ? 2 : 1;

constexpr int kTogether = 128;

// float16 loses values below 2^-14 bit by bit. The weights are at most one and are held times 2^15 where they are multiplied
// themselves (dv). dS has the sizes of upstream gradients, values and weights together, so each lane holds its column's (a
// query's for dq, a key's for dk) times a power of two of its own: one that brings the largest so far between 2^9 and 2^15, moved,
// with the sums, when a larger one comes. Hidden values count for nothing in it, so what a column does not see costs it no bits,
// and neither does what other columns see. Other types need none of it. (A power of two from the norms of all upstream gradients
// that a workgroup reads was 4% faster, 8192 tokens of 16/8 heads of 128: 1113 and 1152 us, and lost a key's bits to queries that
// do not see it.)
template <typename T>
constexpr bool kScaled = __is_same(T, _Float16);
template <typename T>
constexpr float kWeightShift = kScaled<T> ? 15.0f : 0.0f;

struct ColumnScale {
    float into = 0x1p60f;  // nothing seen yet (and values from 2^-45 down to 2^-74 need no other)

    // ds, times the power of two already, into range; sums: those of ds so far.
    template <int kParts>
    __device__ __forceinline__ void keep_in_range(float (&ds)[16], Acc (&sums)[kParts]) {
        float top = fabsf(ds[0]);
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
        if (!__any(top > 0x1p15f)) return;
        top = fmaxf(top, other_half(top));
        int e;
        frexpf(top, &e);  // (infinity: anything, the row is computed again)
        const float keep = top > 0x1p15f ? ldexpf(1.0f, 10 - min(e, 128)) : 1.0f;
        into *= keep;
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] *= keep;
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[p][r] *= keep;
    }
};

// ---- dq ----
template <typename T, int kDim, bool kLargeCap>
__device__ __forceinline__ void dq_tile(const DocAttention& a, unsigned block, LdsByte* buffers, LdsByte* pair_lds) {
    using Shape = TileShape<T, kDim>;
    constexpr int kTile = kStream<T, kDim>;
    using Copy = TileCopy<T, kDim, kTile, kDocThreads>;
    constexpr int kTileBytes = Copy::kBytes;
    constexpr bool kPaired = kPair<T, kDim> == 2;
    constexpr int kParts = kWaveDim<T, kDim> / 32, kOwn = kBlockRows<T, kDim>;
    constexpr bool kAhead = kStreamBuffers<T, kDim> == 2;

    const int turn = static_cast<int>(block) % a.heads;
    const int head = (turn % a.kv_heads) * a.group + turn / a.kv_heads;
    const int kv = head / a.group;
    Document doc;
    int first;
    if (!locate_tile<kOwn, true>(a, block / a.heads, doc, first)) return;

    const int wave = uniform(static_cast<int>(threadIdx.x) >> 6), lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5;
    const int part = kPaired ? wave & 1 : 0, first_part = part * kParts;  // of the dimensions
    const int wave_first = first + 32 * (kPaired ? wave >> 1 : wave), wave_last = min(wave_first + 31, doc.end - 1);
    const bool working = wave_first < doc.end;
    const bool mine = wave_first + (lane & 31) < doc.end;
    const int i = min(wave_first + (lane & 31), doc.end - 1);
    const Span span = key_span(a, doc, i);
    const bool few = kPlanes<T> == 1 && all_see_few(doc, span);
    const int64_t head_at = static_cast<int64_t>(head) * a.head_dim, stat_at = static_cast<int64_t>(head) * a.tokens + i;

    const int low = key_span(a, doc, first).low;
    const int high = max(key_span(a, doc, min(first + kOwn, doc.end) - 1).high, doc.prefix_end);
    const int low_tile = (low - doc.start) / kTile, prefix_tiles = (doc.prefix_end - doc.start + kTile - 1) / kTile;
    const int tiles = (high - doc.start + kTile - 1) / kTile;
    const Span first_span = key_span(a, doc, wave_first), last_span = key_span(a, doc, wave_last);
    const int any_low = first_span.low, any_high = last_span.high, all_low = last_span.low, all_high = first_span.high;

    const Copy copy_k(a.sources[1], kv), copy_v(a.sources[2], kv);
    const TileView<T, kDim, kTile> view;
    // the first tile is on its way while the lane's rows are read
    auto next_tile = [&](int t) { return t + 1 < prefix_tiles ? t + 1 : max(t + 1, low_tile); };
    auto fetch = [&](int t, int buffer) {
        const int from = doc.start + t * kTile;
        copy_k(from, doc.end - from, buffers + buffer * 2 * kTileBytes);
        copy_v(from, doc.end - from, buffers + buffer * 2 * kTileBytes + kTileBytes);
    };
    int t = next_tile(-1);
    if (kAhead) fetch(t, 0);

    const Column<T, kDim> q(a.sources[0], head, i, part), dout(a.sources[3], head, i, part);
    const float delta = a.delta[stat_at];
    ColumnScale scale;

    const CapTerms<T, kLargeCap> cap(a);
    const float slope = a.slopes ? a.slopes[head] * kLog2E : 0.0f;
    const float base = a.lse[stat_at] * kLog2E - cap.plus;

    Acc dq[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[p][r] = 0.0f;

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
        const bool idle = !working || !((from < any_high && from + kTile > any_low) || from < doc.prefix_end);
        if (!kPaired && idle) continue;
        const bool all_seen = (from >= all_low && from + kTile <= all_high) || from + kTile <= doc.prefix_end;
#pragma unroll
        for (int b = 0; b < kTile / 32; ++b) {
            Acc x, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = dp[r] = 0.0f;
            if (!kPaired || !idle) {
                multiply_rows(view, k_tile, b, q, part, x);
                multiply_rows(view, v_tile, b, dout, part, dp);
            }
            if constexpr (kPaired) {
                static_assert(kTile == 32);
                exchange({&x, &dp}, pair_lds);
                if (idle) continue;
            }
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = kScaled<T> ? fmaf(dp[r], scale.into, -delta * scale.into) : dp[r] - delta;
            if (cap.capped) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float derivative;
                    x[r] = cap.bend(x[r], derivative);
                    ds[r] *= derivative;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], cap.times, -base);
            if (a.slopes) {
                const float away = static_cast<float>(i - from - 32 * b - 4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = fmaf(-slope, fabsf(away - static_cast<float>(8 * (r / 4) + r % 4)), x[r]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] *= __builtin_amdgcn_exp2f(x[r]);
            if (!all_seen) {
                const int to_low = span.low - from - 32 * b - 4 * half;
                const unsigned width = static_cast<unsigned>(span.high - span.low);
                const int to_prefix = doc.prefix_end - from - 32 * b - 4 * half;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = 8 * (r / 4) + r % 4;
                    const bool see = static_cast<unsigned>(j - to_low) < width || j < to_prefix;
                    ds[r] = see ? ds[r] : 0.0f;
                }
            }
            if constexpr (kScaled<T>) scale.keep_in_range(ds, dq);
            multiply_columns<T, kDim, kTile>(view, k_tile, b, Rows16<T>(ds), first_part, dq);
            if (few) {
                keep_rest<T>(ds);
                multiply_columns<T, kDim, kTile>(view, k_tile, b, Rows16<T>(ds), first_part, dq);
            }
        }
    }
    if (!kPaired && !working) return;
    const uint64_t marks = __ballot(!all_finite(dq) && mine);
    uint32_t spoilt = static_cast<uint32_t>(marks) | static_cast<uint32_t>(marks >> 32);
    if constexpr (kPaired) spoilt = pair_marks(spoilt, pair_lds);
    T* const to = static_cast<T*>(a.dq) + head_at;
    if (mine && !(spoilt >> (lane & 31) & 1))
        store_column(to + i * a.q_stride, a.head_dim, a.whole, first_part, dq, kScaled<T> ? a.scale / scale.into : a.scale);
    for (uint32_t left = part == 0 ? spoilt : 0; left; left &= left - 1) {
        const int from_lane = __ffs(left) - 1, row = wave_first + from_lane;
        float value[kLaneDims];
        attention_row_dq<T>(a, doc, head, row, __shfl(delta, from_lane), value);
        store_row(to + row * a.q_stride, value, a.head_dim);
    }
}

// ---- dk and dv of one head ----
//
// kShared: into the float32 parts of heads that share keys. kDk, kDv: which of the two; rows of more than kTogether
// elements for a wave take a workgroup for each, since the sums of both and a lane's two rows are more than its registers (five products
// in all instead of four).
template <typename T, int kDim, bool kLargeCap, bool kShared, bool kDk, bool kDv>
__device__ __forceinline__ void dkv_tile(const DocAttention& a, unsigned block, LdsByte* buffers, LdsByte* pair_lds) {
    using Shape = TileShape<T, kDim>;
    constexpr int kTile = kStream<T, kDim>;
    using Copy = TileCopy<T, kDim, kTile, kDocThreads>;
    constexpr int kTileBytes = Copy::kBytes;
    constexpr bool kPaired = kPair<T, kDim> == 2;
    constexpr int kParts = kWaveDim<T, kDim> / 32, kOwn = kBlockRows<T, kDim>;
    constexpr bool kAhead = kStreamBuffers<T, kDim> == 2;
    __shared__ __attribute__((aligned(16))) float stats[2][2][kTile];  // lse in units of log 2, and dout . out, of a tile's queries

    const int turn = static_cast<int>(block) % a.heads;
    const int head = (turn % a.kv_heads) * a.group + turn / a.kv_heads;
    const int kv = head / a.group;
    Document doc;
    int first;
    if (!locate_tile<kOwn, false>(a, block / a.heads, doc, first)) return;

    const int wave = uniform(static_cast<int>(threadIdx.x) >> 6), lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5;
    const int part = kPaired ? wave & 1 : 0, first_part = part * kParts;  // of the dimensions
    const int wave_first = first + 32 * (kPaired ? wave >> 1 : wave), wave_last = min(wave_first + 31, doc.end - 1);
    const bool working = wave_first < doc.end;
    const bool mine = wave_first + (lane & 31) < doc.end;
    const int j = min(wave_first + (lane & 31), doc.end - 1);
    const Span span = query_span(a, doc, j);
    const bool few = kPlanes<T> == 1 && all_seen_by_few(span);
    const int64_t kv_at = static_cast<int64_t>(kv) * a.head_dim, stat_at = static_cast<int64_t>(head) * a.tokens;

    // the queries that see any key of the workgroup; keys in the prefix are seen from the document's start on
    const int last = min(first + kOwn, doc.end) - 1;
    const int low = query_span(a, doc, first).low;
    const int high = max(query_span(a, doc, first).high, query_span(a, doc, last).high);
    const int low_tile = (low - doc.start) / kTile, tiles = (high - doc.start + kTile - 1) / kTile;
    // the wave's: those that see any of its keys, and all
    const Span first_span = query_span(a, doc, min(wave_first, doc.end - 1)), last_span = query_span(a, doc, wave_last);
    const int any_low = first_span.low, any_high = max(first_span.high, last_span.high);
    // (a wave with keys on both sides of the prefix's end: the first key after it has the earliest end)
    const int edge = wave_first < doc.prefix_end && wave_last >= doc.prefix_end ? doc.prefix_end : wave_first;
    const int all_low = last_span.low, all_high = query_span(a, doc, min(edge, doc.end - 1)).high;

    const Copy copy_q(a.sources[0], head), copy_d(a.sources[3], head);
    const TileView<T, kDim, kTile> view;
    auto fetch = [&](int t, int buffer) {
        const int from = doc.start + t * kTile;
        copy_q(from, doc.end - from, buffers + buffer * 2 * kTileBytes);
        copy_d(from, doc.end - from, buffers + buffer * 2 * kTileBytes + kTileBytes);
    };
    // the first tile is on its way while the lane's rows are read
    int t = low_tile;
    if (kAhead) fetch(t, 0);
    const Column<T, kDim> k(a.sources[1], kv, j, part), v(a.sources[2], kv, j, part);

    ColumnScale scale;

    const CapTerms<T, kLargeCap> cap(a);
    const float slope = a.slopes ? a.slopes[head] * kLog2E : 0.0f;

    Acc dk[kDk ? kParts : 1], dv[kDv ? kParts : 1];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
        for (int p = 0; p < (kDk ? kParts : 1); ++p) dk[p][r] = 0.0f;
#pragma unroll
        for (int p = 0; p < (kDv ? kParts : 1); ++p) dv[p][r] = 0.0f;
    }

    // a tile's statistics, one value for each of the first 2 kTile threads
    auto read_stat = [&](int t) {
        const int which = static_cast<int>(threadIdx.x) / kTile, at = min(doc.start + t * kTile + static_cast<int>(threadIdx.x) % kTile, doc.end - 1);
        return which == 0 ? a.lse[stat_at + at] * kLog2E - kWeightShift<T> - cap.plus : which == 1 ? a.delta[stat_at + at] : 0.0f;
    };
    auto write_stat = [&](int buffer, float value) {
        if (static_cast<int>(threadIdx.x) < 2 * kTile) (&stats[buffer][0][0])[threadIdx.x] = value;
    };
    // (read a tile ahead of their writing to LDS, which is a tile ahead of their use)
    if (kAhead) write_stat(0, read_stat(t));
    float ahead = read_stat(t + (kAhead ? 1 : 0));
    loads_arrived();
    for (int buffer = 0; t < tiles; buffer ^= kAhead, ++t) {
        tile_barrier();
        if (!kAhead) {
            write_stat(0, ahead);
            fetch(t, 0);
            tile_barrier();
        } else if (t + 1 < tiles) {
            write_stat(buffer ^ 1, ahead);
        }
        ahead = read_stat(t + (kAhead ? 2 : 1));
        if (kAhead && t + 1 < tiles) fetch(t + 1, buffer ^ 1);
        const LdsByte* const q_tile = buffers + buffer * 2 * kTileBytes;
        const LdsByte* const d_tile = q_tile + kTileBytes;
        const int from = doc.start + t * kTile;
        const bool idle = !working || !(from < any_high && from + kTile > any_low);
        if (!kPaired && idle) continue;
        const bool all_seen = from >= all_low && from + kTile <= all_high;
        const float* const tile_base = &stats[buffer][0][4 * half];
        const float* const tile_delta = &stats[buffer][1][4 * half];
        using Four = float __attribute__((ext_vector_type(4)));

        // 32 queries' scores and dP ...
        auto products = [&](int b, Acc& x, Acc& dp) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = dp[r] = 0.0f;
            multiply_rows(view, q_tile, b, k, part, x);
            if constexpr (kDk) multiply_rows(view, d_tile, b, v, part, dp);
        };
        // ... their weights and dS ...
        auto weights = [&](int b, Acc& x, const Acc& dp, float (&p)[16], float (&ds)[16]) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const Four base = *reinterpret_cast<const Four*>(tile_base + 32 * b + 8 * g);
                const Four delta = *reinterpret_cast<const Four*>(tile_delta + 32 * b + 8 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[4 * g + r] = base[r];
                    ds[4 * g + r] = dp[4 * g + r] - delta[r];
                }
            }
            if (cap.capped) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float derivative;
                    x[r] = cap.bend(x[r], derivative);
                    ds[r] *= derivative;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = fmaf(x[r], cap.times, -p[r]);
            if (a.slopes) {
                const float away = static_cast<float>(from + 32 * b + 4 * half - j);
#pragma unroll
                for (int r = 0; r < 16; ++r) p[r] = fmaf(-slope, fabsf(away + static_cast<float>(8 * (r / 4) + r % 4)), p[r]);
            }
            if (!all_seen) {
                const int to_low = span.low - from - 32 * b - 4 * half;
                const unsigned width = static_cast<unsigned>(span.high - span.low);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool see = static_cast<unsigned>(8 * (r / 4) + r % 4 - to_low) < width;
                    p[r] = see ? p[r] : -INFINITY;
                    ds[r] = see ? ds[r] : 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(p[r]);
                ds[r] *= p[r];
            }
        };
        // ... and their part of the sums.
        auto add = [&](int b, const Rows16<T>& p, const Rows16<T>& ds) {
            if constexpr (kDv) multiply_columns<T, kDim, kTile>(view, d_tile, b, p, first_part, dv);
            if constexpr (kDk) multiply_columns<T, kDim, kTile>(view, q_tile, b, ds, first_part, dk);
        };
        constexpr int kBlocks = kTile / 32;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            Acc x{}, dp{};
            if (!kPaired || !idle) products(b, x, dp);
            if constexpr (kPaired) {
                static_assert(kBlocks == 1);
                if constexpr (kDk)
                    exchange({&x, &dp}, pair_lds);
                else
                    exchange({&x}, pair_lds);
                if (idle) continue;
            }
            float p[16], ds[16];
            weights(b, x, dp, p, ds);
            if constexpr (kScaled<T> && kDk) {
#pragma unroll
                for (int r = 0; r < 16; ++r) ds[r] *= scale.into;
                scale.keep_in_range(ds, dk);
            }
            add(b, Rows16<T>(p), Rows16<T>(ds));
            if (few) {
                keep_rest<T>(p);
                keep_rest<T>(ds);
                add(b, Rows16<T>(p), Rows16<T>(ds));
            }
        }
    }
    if (!kPaired && !working) return;
    const float unshift = __builtin_amdgcn_exp2f(-kWeightShift<T>), dk_factor = (kScaled<T> && kDk ? a.scale / scale.into : a.scale) * unshift;
    const uint64_t marks = __ballot(!(all_finite(dk) && all_finite(dv)) && mine);
    uint32_t spoilt = static_cast<uint32_t>(marks) | static_cast<uint32_t>(marks >> 32);
    if constexpr (kPaired) spoilt = pair_marks(spoilt, pair_lds);
    // row `at` of dk and dv, by `store` of its place and its factor
    auto rows_of = [&](int64_t at, auto&& store) {
        const int64_t part = (stat_at + at) * a.head_dim;
        if constexpr (kShared)
            store(a.dk_part + part, a.dv_part + part);
        else
            store(static_cast<T*>(a.dk) + at * a.k_stride + kv_at, static_cast<T*>(a.dv) + at * a.v_stride + kv_at);
    };
    if (mine && !(spoilt >> (lane & 31) & 1))
        rows_of(j, [&](auto* to_dk, auto* to_dv) {
            if constexpr (kDk) store_column(to_dk, a.head_dim, a.whole, first_part, dk, dk_factor);
            if constexpr (kDv) store_column(to_dv, a.head_dim, a.whole, first_part, dv, unshift);
        });
    for (uint32_t left = part == 0 ? spoilt : 0; left; left &= left - 1) {
        const int row = wave_first + __ffs(left) - 1;
        float dk1[kLaneDims], dv1[kLaneDims];
        attention_row_dkv<T>(a, doc, head, row, dk1, dv1);
        rows_of(row, [&](auto* to_dk, auto* to_dv) {
            if constexpr (kDk) store_row(to_dk, dk1, a.head_dim);
            if constexpr (kDv) store_row(to_dv, dv1, a.head_dim);
        });
    }
}

// LDS of a workgroup: the tiles, and what a pair of waves exchanges.
template <typename T, int kDim>
constexpr int kTilesBytes = kStreamBuffers<T, kDim> * 2 * TileCopy<T, kDim, kStream<T, kDim>, kDocThreads>::kBytes;
template <typename T, int kDim>
constexpr int kExchangeBytes = kPair<T, kDim> == 2 ? 2 * 4 * 4096 : 16;

// All gradients at once: dk and dv (blockIdx.y 0; dv 2 where it is on its own), whose workgroups take longer, before dq (1).
template <typename T, int kDim, bool kLargeCap, bool kShared>
__global__ __launch_bounds__(kDocThreads, kPlanes<T> == 1 && kDim <= 64 ? 2 : 1) void gradients_kernel(DocAttention a) {
    __shared__ __attribute__((aligned(1024))) char lds[kTilesBytes<T, kDim>];
    __shared__ __attribute__((aligned(16))) char exchanged[kExchangeBytes<T, kDim>];
    LdsByte* const buffers = (LdsByte*)lds;
    LdsByte* const pair_lds = (LdsByte*)exchanged;
    const unsigned block = blockIdx.x, turn = blockIdx.y;
    if constexpr (kWaveDim<T, kDim> <= kTogether) {
        if (turn == 0) return dkv_tile<T, kDim, kLargeCap, kShared, true, true>(a, block, buffers, pair_lds);
    } else {
        if (turn == 0) return dkv_tile<T, kDim, kLargeCap, kShared, true, false>(a, block, buffers, pair_lds);
        if (turn == 2) return dkv_tile<T, kDim, kLargeCap, kShared, false, true>(a, block, buffers, pair_lds);
    }
    dq_tile<T, kDim, kLargeCap>(a, block, buffers, pair_lds);
}

// 16-bit heads of 65 to 128 elements: dq alone fits twice on a CU, dk and dv do not. With more than kFewTiles workgroups of
// each kind a kernel for each is faster (16/8 heads of 128 in bfloat16, microseconds together and apart: 2048 tokens, 272
// workgroups, 111 and 163; 3071 tokens, 400, 215 and 234; 4096 tokens, 528, 339 and 329; 8192 tokens, 1040, 1184 and 1045).
// Both ways run the same code and give the same bits; large caps have the one launch alone.
template <typename T, int kDim>
constexpr bool kApart = kPlanes<T> == 1 && kDim == 128;
constexpr unsigned kFewTiles = 512;

// (two waves on a SIMD, 256 registers each; float16 keeps one more in scratch memory)
template <typename T, int kDim>
__global__ __launch_bounds__(kDocThreads, 2) void dq_kernel(DocAttention a) {
    static_assert(kApart<T, kDim>);
    __shared__ __attribute__((aligned(1024))) char lds[kTilesBytes<T, kDim>];
    dq_tile<T, kDim, false>(a, blockIdx.x, (LdsByte*)lds, nullptr);
}

template <typename T, int kDim, bool kShared>
__global__ __launch_bounds__(kDocThreads, 1) void dkv_kernel(DocAttention a) {
    static_assert(kApart<T, kDim>);
    __shared__ __attribute__((aligned(1024))) char lds[kTilesBytes<T, kDim>];
    dkv_tile<T, kDim, false, kShared, true, true>(a, blockIdx.x, (LdsByte*)lds, nullptr);
}

// dk and dv of the tokens of documents: the group's heads added in order. kWidth elements to a thread. Bound: HBM (8192 tokens,
// 16/8 heads of 128: 32 us, 5.2 TB/s).
template <typename T, int kWidth>
__global__ __launch_bounds__(kDocThreads) void add_heads_kernel(DocAttention a) {
    const int per_row = (a.head_dim + kWidth - 1) / kWidth, per_token = a.kv_heads * per_row;
    Document doc;
    int first;
    if (!locate_tile<kDocTileRows, false>(a, blockIdx.x, doc, first)) return;
    const int rows = min(kDocTileRows, doc.end - first);
    // (128 rows of at most 65535 heads of 64 groups of four: 32 bits)
    for (int e = static_cast<int>(blockIdx.y * kDocThreads + threadIdx.x); e < rows * per_token; e += static_cast<int>(gridDim.y) * kDocThreads) {
        const int row = e / per_token, in_token = e - row * per_token;
        const int kv = in_token / per_row, d = (in_token - kv * per_row) * kWidth;
        const int64_t j = first + row;
        const int64_t at = (static_cast<int64_t>(kv) * a.group * a.tokens + j) * a.head_dim + d, next = static_cast<int64_t>(a.tokens) * a.head_dim;
        float sum[2][kWidth] = {};  // (of zero and a first part of minus zero: plus zero, as a product's sum would be)
#pragma unroll 4
        for (int g = 0; g < a.group; ++g) {
            float more[2][kWidth];
            load_as_float<float, kWidth>(a.dk_part + at + g * next, more[0]);
            load_as_float<float, kWidth>(a.dv_part + at + g * next, more[1]);
#pragma unroll
            for (int c = 0; c < kWidth; ++c) sum[0][c] += more[0][c], sum[1][c] += more[1][c];
        }
        store_from_float<T, kWidth>(static_cast<T*>(a.dk) + j * a.k_stride + static_cast<int64_t>(kv) * a.head_dim + d, sum[0]);
        store_from_float<T, kWidth>(static_cast<T*>(a.dv) + j * a.v_stride + static_cast<int64_t>(kv) * a.head_dim + d, sum[1]);
    }
}

template <typename T, int kDim, bool kShared>
void launch_gradients(const DocAttention& a, hipStream_t s) {
    const unsigned tiles = doc_tiles(a, kBlockRows<T, kDim>) * a.heads;
    const dim3 together(tiles, kWaveDim<T, kDim> <= kTogether ? 2 : 3);
    if constexpr (sizeof(T) == 2)
        if (large_cap(a)) {
            gradients_kernel<T, kDim, true, kShared><<<together, kDocThreads, 0, s>>>(a);
            return;
        }
    if constexpr (kApart<T, kDim>) {
        if (tiles > kFewTiles) {
            dkv_kernel<T, kDim, kShared><<<tiles, kDocThreads, 0, s>>>(a);
            dq_kernel<T, kDim><<<tiles, kDocThreads, 0, s>>>(a);
            return;
        }
    }
    gradients_kernel<T, kDim, false, kShared><<<together, kDocThreads, 0, s>>>(a);
}

template <typename T, int kDim>
void launch_gradients(const DocAttention& a, hipStream_t s) {
    if (a.group == 1)
        launch_gradients<T, kDim, false>(a, s);
    else
        launch_gradients<T, kDim, true>(a, s);
}

template <typename T>
int launch_document_attention_backward(DocAttention a, char* packed, hipStream_t s) {
    a.whole = whole_chunks(a, kChunk<T>, {a.q, a.k, a.v, a.out, a.dout, a.dq, a.dk, a.dv});
    set_sources<T>(a, true, packed, s);
    if (a.head_dim <= 64)
        launch_gradients<T, 64>(a, s);
    else if (a.head_dim <= 128)
        launch_gradients<T, 128>(a, s);
    else
        launch_gradients<T, 256>(a, s);
    if (a.group > 1) {
        // about one turn for each thread, as far as 64 workgroups to a part of a document go
        const int64_t threads = static_cast<int64_t>(kDocTileRows) * a.kv_heads * a.head_dim / (a.whole ? 4 : 1);
        const dim3 grid(doc_tiles(a, kDocTileRows), static_cast<unsigned>(std::clamp<int64_t>(threads / kDocThreads, 1, 64)));
        if (a.whole)
            add_heads_kernel<T, 4><<<grid, kDocThreads, 0, s>>>(a);
        else
            add_heads_kernel<T, 1><<<grid, kDocThreads, 0, s>>>(a);
    }
    return check_launch("document_attention_backward");
}

}  // namespace dllm_hip
