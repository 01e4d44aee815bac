// Attention within packed documents: what the forward and backward kernels share. Which keys a query sees, how a
// workgroup finds its part of a document, and the score's bends (cap, distance bias).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

#include "common.h"
#include "doc_tile.h"
#include "element.h"
#include "softcap.h"

namespace dllm_hip {

constexpr int kDocThreads = 256;
constexpr int kDocTileRows = 128;  // tokens of a workgroup, 32 for each wave (64 of wide float32 heads)

struct DocAttention {
    const void *q, *k, *v, *out, *dout;  // out: written by the forward, read by the backward
    void *dq, *dk, *dv;
    float* lse;  // [heads][tokens]
    const int64_t *offsets, *prefix;
    const float* slopes;
    int64_t q_stride, k_stride, v_stride, out_stride;
    int tokens, documents, heads, kv_heads, group, head_dim;
    int causal, window;  // window 0: none
    float scale, softcap;  // softcap 0: none
    bool whole;  // every array's rows are whole 16-byte chunks, aligned to them
    Source sources[4];  // q, k, v, dout as the matrix cores read them
    // backward scratch
    float* delta;     // [heads][tokens]: dout . out
    float* dk_part;   // [heads][tokens][head_dim] float32, before the heads of a group are added
    float* dv_part;
};

// 16-bit weights (and dS) are rounded to their type for the second product: each is off by 2^-9 or 2^-12 of itself, which in a
// sum over many keys adds to about what the result's own rounding is. Rows that see so few keys (keys that so few queries see)
// that such errors do not average out have what the rounding left multiplied too, where that holds for all 32 of a wave: short
// documents, narrow windows, a long causal document's first queries and last keys. (128 documents of 64 tokens, 16/8 heads of 128
// in bfloat16: 37.7 to 39.3 us, gradients 193 to 202 us; the error of a document of 37: 1.8e-3 to 1.6e-3, which is the result's own
// rounding.)
constexpr int kFewTokens = 64;

// Token range of a document, and the end of the keys that all its tokens see.
struct Document {
    int start, end, prefix_end;
};

__device__ __forceinline__ int clamp_token(int64_t v, int low, int high) {
    return v < low ? low : v > high ? high : static_cast<int>(v);
}

__device__ __forceinline__ Document document_at(const DocAttention& a, int d) {
    Document r;
    r.start = clamp_token(a.offsets[d], 0, a.tokens);
    r.end = clamp_token(a.offsets[d + 1], r.start, a.tokens);
    r.prefix_end = a.prefix ? r.start + clamp_token(a.prefix[d], 0, r.end - r.start) : r.start;
    return r;
}

// The tile-th part of kRows tokens of all documents; each document starts a part of its own, so that what is computed for it
// does not depend on where it lies. Every lane of the wave returns the same. False where there is no such part: past the last one
// and, among many documents, in between.
//
// Parts come longest first, as far as that is cheap to know, so that the last workgroups to start are short ones: kFromEnd is
// for work that grows towards a document's end (a causal row's keys), else towards its start (a key's queries). Up to 64
// causal documents (one to a lane): the parts of the highest level first, of all documents that reach it, where a part's level
// counts from the end with less work. Else the documents in order, each from the end with more work. (Ten documents of 1 to 2048
// tokens, 8192 in all, 16/8 heads of 128 in bfloat16: 97 us in their order, 83 by level; gradients 363 and 345.)
//
// More documents than lanes are not counted through, which would take every workgroup a time that grows with their number. Part p
// of document d is tile start / kRows + d + p instead: that gives no tile twice (a document has at most one part more than
// start / kRows steps on to the next) and leaves some out, and grows with d, which is searched for, 64 documents at once. (5000
// documents of 10 tokens, 8/4 heads of 64 in bfloat16: counted 1523 us and 8.8 ms for the gradients, searched 256 us and 1.2 ms.)
constexpr int kFewDocuments = 64;

template <int kRows, bool kFromEnd>
__device__ __forceinline__ bool find_tile_of_many(const DocAttention& a, int tile, Document& doc, int& first) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int at = kFromEnd ? (a.tokens + kRows - 1) / kRows + a.documents - 1 - tile : tile;
    auto first_tile = [&](int d) { return clamp_token(a.offsets[d], 0, a.tokens) / kRows + d; };
    int low = 0, step;  // document low begins at or before the tile, low + count, if there is one, after it
    for (int count = a.documents; count > 0; count = step == 1 ? 0 : min(step, count)) {
        step = (count + 63) / 64;
        const int off = lane * step;
        const uint64_t begun = __ballot(off < count && first_tile(low + min(off, count - 1)) <= at);
        if (!begun) return false;
        const int last = (__popcll(begun) - 1) * step;
        low += last, count -= last;
    }
    doc = document_at(a, low);
    const int part = at - first_tile(low);
    if (part >= (doc.end - doc.start + kRows - 1) / kRows) return false;
    first = doc.start + part * kRows;
    return true;
}

template <int kRows, bool kFromEnd>
__device__ __forceinline__ bool find_tile(const DocAttention& a, int tile, Document& doc, int& first) {
    if (a.documents > kFewDocuments) return find_tile_of_many<kRows, kFromEnd>(a, tile, doc, first);
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int d = a.causal || !kFromEnd ? lane : a.documents - 1 - lane;
    Document mine{0, 0, 0};
    if (d >= 0 && d < a.documents) mine = document_at(a, d);
    const int parts = (mine.end - mine.start + kRows - 1) / kRows;
    auto found = [&](int owner, int level) {
        doc.start = __builtin_amdgcn_readlane(mine.start, owner);
        doc.end = __builtin_amdgcn_readlane(mine.end, owner);
        doc.prefix_end = __builtin_amdgcn_readlane(mine.prefix_end, owner);
        const int all = (doc.end - doc.start + kRows - 1) / kRows;
        first = doc.start + (kFromEnd ? level : all - 1 - level) * kRows;
        return true;
    };
    if (a.causal) {
        const int bits = 32 - __builtin_clz((a.tokens + kRows - 1) / kRows | 1);
        auto at_or_above = [&](int level) {  // parts of that level or higher, by the bits of each document's number of them
            const int n = parts > level ? parts - level : 0;
            int64_t sum = 0;
            for (int b = 0; b < bits; ++b) sum += static_cast<int64_t>(__popcll(__ballot(n >> b & 1))) << b;
            return sum;
        };
        if (tile >= at_or_above(0)) return false;
        int level = 0;
        for (int b = bits - 1; b >= 0; --b)
            if (at_or_above(level + (1 << b)) > tile) level += 1 << b;
        uint64_t reach = __ballot(parts > level);
        for (int64_t skip = tile - at_or_above(level + 1); skip > 0; --skip) reach &= reach - 1;
        return found(__builtin_ctzll(reach), level);
    }
    int64_t through = parts;  // parts of the lanes up to this one
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int64_t o = __shfl_up(through, s);
        if (lane >= s) through += o;
    }
    if (tile >= __shfl(through, 63)) return false;
    const int owner = __builtin_ctzll(__ballot(through > tile));
    const int part = static_cast<int>(tile - __shfl(through - parts, owner));
    return found(owner, __builtin_amdgcn_readfirstlane(__builtin_amdgcn_readlane(parts, owner) - 1 - part));
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// find_tile, with its results in scalar registers: what follows from them (loops, branches, addresses) is scalar too.
template <int kRows, bool kFromEnd>
__device__ __forceinline__ bool locate_tile(const DocAttention& a, unsigned tile, Document& doc, int& first) {
    Document d{0, 0, 0};
    int f = 0;
    const int found = find_tile<kRows, kFromEnd>(a, static_cast<int>(tile), d, f);
    doc.start = uniform(d.start), doc.end = uniform(d.end), doc.prefix_end = uniform(d.prefix_end);
    first = uniform(f);
    return uniform(found);
}

// Waits for the loads issued so far, where the compiler sees it: a load from before a loop that is first used in it is waited
// for in every turn otherwise, and with it the copies to LDS that the turn has just begun.
__device__ __forceinline__ void loads_arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// The keys that query i sees: [low, high) and [start, prefix_end).
struct Span {
    int low, high;
};

__device__ __forceinline__ Span key_span(const DocAttention& a, const Document& d, int i) {
    Span s;
    s.low = a.window && i - d.start >= a.window ? i - a.window + 1 : d.start;
    s.high = a.causal ? i + 1 : a.window && d.end - i > a.window ? i + a.window : d.end;
    return s;
}

// The queries that see key j: one range, since the prefix is seen by all.
__device__ __forceinline__ Span query_span(const DocAttention& a, const Document& d, int j) {
    if (j < d.prefix_end) return {d.start, d.end};
    Span s;
    s.low = a.causal ? j : a.window && j - d.start >= a.window ? j - a.window + 1 : d.start;
    s.high = a.window && d.end - j > a.window ? j + a.window : d.end;
    return s;
}

__device__ __forceinline__ bool visible(const Document& d, const Span& s, int j) {
    return (j >= s.low && j < s.high) || (j >= d.start && j < d.prefix_end);
}

// Of the 32 queries (keys) of a wave: whether each sees (is seen by) few.
__device__ __forceinline__ bool all_see_few(const Document& d, const Span& s) {
    const int before = max(min(d.prefix_end, s.low), d.start) - d.start, after = max(d.prefix_end - s.high, 0);
    return !__any(s.high - s.low + before + after > kFewTokens);
}

__device__ __forceinline__ bool all_seen_by_few(const Span& s) { return !__any(s.high - s.low > kFewTokens); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
    return v;
}

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

// The score of a dot product, and the cap's derivative there.
__device__ __forceinline__ float bend_score(const DocAttention& a, float slope, float dot, int distance, float& derivative) {
    float x = dot * a.scale;
    derivative = 1.0f;
    if (a.softcap != 0.0f) {
        const float t = tanhf(x / a.softcap);
        derivative = 1.0f - t * t;
        x = a.softcap * t;
    }
    return x - slope * static_cast<float>(distance < 0 ? -distance : distance);
}

// The score of a product x in units of log 2: bent(x) times + plus, which is x scale without a cap. bent grows with x, so the
// largest score is that of the largest bent. bent is tanh, as float32 has it from the library, exact to its last bits near zero
// too. With 16-bit types it is
// - of caps up to kSmallCap -1 / (1 + e^2z) = (tanh z - 1) / 2, whose rest falls into times and plus. It is off by at most about
//   6 x 2^-24 of the cap however small the score is: 2^-15 of a weight, which rounds to 2^-9 or 2^-12 of itself.
// - of larger ones, whose scores may be any part of the cap, tanh again (softcap.h).
// Large caps have kernels of their own: in the same ones, chosen by a branch, they cost other calls registers (8192 tokens of
// 16/8 heads of 64 in bfloat16, without a cap, 168 and 178 us). Caps of 50 and 100: 8000 + 192 tokens, 8/4 heads of 256, window 4096,
// 377 and 462 us; gradients of 8192 tokens, 16/8 heads of 128, 1323 and 1925.
constexpr float kSmallCap = 64.0f;

inline bool large_cap(const DocAttention& a) { return a.softcap > kSmallCap; }

template <typename T, bool kLargeCap>
struct CapTerms {
    static constexpr bool kHalved = sizeof(T) == 2 && !kLargeCap;  // bent is (tanh - 1) / 2
    bool capped;
    float in, times, plus;
    __device__ __forceinline__ explicit CapTerms(const DocAttention& a) {
        capped = a.softcap != 0.0f;
        const float unit = (capped ? a.softcap : a.scale) * kLog2E;
        in = capped ? a.scale / a.softcap : 0.0f;
        times = unit, plus = 0.0f;
        if (kHalved && capped) in *= 2.0f * kLog2E, times = 2.0f * unit, plus = unit;
    }
    // bent, and the cap's derivative: of a halved one 4 e b^2 with e = e^2z, which is right to its last bits where the cap is nearly
    // reached on either side (one minus the square of a tanh near one is not; float32 has it as any float32 evaluation would)
    __device__ __forceinline__ float bend(float x, float& derivative) const {
        if constexpr (kLargeCap) return tanh_of_any_size(x * in, derivative);
        if constexpr (sizeof(T) == 4) {
            const float t = tanhf(x * in);
            derivative = fmaf(-t, t, 1.0f);
            return t;
        }
        const float e = __builtin_amdgcn_exp2f(x * in), b = __builtin_amdgcn_rcpf(-1.0f - e);
        derivative = fminf(e, 0x1p126f) * b * (4.0f * b);
        return b;
    }
};

template <typename T>
__device__ __forceinline__ float dot_row(const T* a, const T* b, int n) {
    float s = 0.0f;
    for (int d = 0; d < n; ++d) s = fmaf(static_cast<float>(a[d]), static_cast<float>(b[d]), s);
    return s;
}

constexpr int kMaxHeadDim = 256;
constexpr int kLaneDims = kMaxHeadDim / 64;  // head dimensions that a lane of a row's wave holds

// ---- one row by one wave ----
//
// Exactly the formula over the visible keys (queries), 64 of them at a time, one per lane. Nothing of a hidden row
// is touched. A weight that is NaN ends it: whatever follows, the row is NaN (so a batch that is NaN throughout costs each row
// its first keys).

__device__ __forceinline__ void all_nan(float (&v)[kLaneDims]) {
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) v[c] = NAN;
}

template <typename T>
__device__ void attention_row(const DocAttention& a, const Document& doc, int head, int i, float (&o)[kLaneDims], float& lse) {
    const int lane = static_cast<int>(threadIdx.x) & 63, kv = head / a.group;
    const T* q = static_cast<const T*>(a.q) + i * a.q_stride + static_cast<int64_t>(head) * a.head_dim;
    const T* k = static_cast<const T*>(a.k) + static_cast<int64_t>(kv) * a.head_dim;
    const T* v = static_cast<const T*>(a.v) + static_cast<int64_t>(kv) * a.head_dim;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const Span s = key_span(a, doc, i);
    const int from = doc.prefix_end > doc.start ? doc.start : s.low;
    const int to = s.high > doc.prefix_end ? s.high : doc.prefix_end;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) o[c] = 0.0f;
    for (int base = from; base < to; base += 64) {
        const int j = base + lane;
        const bool see = j < to && visible(doc, s, j);
        if (!__any(see)) continue;
        float unused;
        const float x = see ? bend_score(a, slope, dot_row(q, k + j * a.k_stride, a.head_dim), i - j, unused) : -INFINITY;
        const float top = fmaxf(m, wave_max(x));
        const float p = x == -INFINITY ? 0.0f : expf(x - top);
        const float keep = m == top ? 1.0f : expf(m - top);
        m = top;
        l = l * keep + wave_add(p);
        if (l != l) {  // NaN, or infinity less itself
            all_nan(o);
            lse = NAN;
            return;
        }
#pragma unroll
        for (int c = 0; c < kLaneDims; ++c) o[c] *= keep;
        for (uint64_t left = __ballot(see); left; left &= left - 1) {
            const int from_lane = __ffsll(static_cast<unsigned long long>(left)) - 1;
            const float pj = __shfl(p, from_lane);
            const T* row = v + (base + from_lane) * a.v_stride;
#pragma unroll
            for (int c = 0; c < kLaneDims; ++c)
                if (lane + 64 * c < a.head_dim) o[c] = fmaf(pj, static_cast<float>(row[lane + 64 * c]), o[c]);
        }
    }
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) o[c] /= l;
    lse = m + logf(l);
}

template <typename T>
__device__ void attention_row_dq(const DocAttention& a, const Document& doc, int head, int i, float delta, float (&dq)[kLaneDims]) {
    const int lane = static_cast<int>(threadIdx.x) & 63, kv = head / a.group;
    const int64_t at = static_cast<int64_t>(head) * a.head_dim;
    const T* q = static_cast<const T*>(a.q) + i * a.q_stride + at;
    const T* dout = static_cast<const T*>(a.dout) + i * a.out_stride + at;
    const T* k = static_cast<const T*>(a.k) + static_cast<int64_t>(kv) * a.head_dim;
    const T* v = static_cast<const T*>(a.v) + static_cast<int64_t>(kv) * a.head_dim;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const float lse = a.lse[static_cast<int64_t>(head) * a.tokens + i];
    const Span s = key_span(a, doc, i);
    const int from = doc.prefix_end > doc.start ? doc.start : s.low;
    const int to = s.high > doc.prefix_end ? s.high : doc.prefix_end;
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) dq[c] = 0.0f;
    for (int base = from; base < to; base += 64) {
        const int j = base + lane;
        const bool see = j < to && visible(doc, s, j);
        float ds = 0.0f;
        if (see) {
            float derivative;
            const float x = bend_score(a, slope, dot_row(q, k + j * a.k_stride, a.head_dim), i - j, derivative);
            const float dp = dot_row(dout, v + j * a.v_stride, a.head_dim);
            ds = expf(x - lse) * (dp - delta) * derivative * a.scale;
        }
        if (__any(ds != ds)) return all_nan(dq);
        for (uint64_t left = __ballot(see); left; left &= left - 1) {
            const int from_lane = __ffsll(static_cast<unsigned long long>(left)) - 1;
            const float d = __shfl(ds, from_lane);
            const T* row = k + (base + from_lane) * a.k_stride;
#pragma unroll
            for (int c = 0; c < kLaneDims; ++c)
                if (lane + 64 * c < a.head_dim) dq[c] = fmaf(d, static_cast<float>(row[lane + 64 * c]), dq[c]);
        }
    }
}

// One head's part of dk and dv of key j.
template <typename T>
__device__ void attention_row_dkv(const DocAttention& a, const Document& doc, int head, int j, float (&dk)[kLaneDims],
                                  float (&dv)[kLaneDims]) {
    const int lane = static_cast<int>(threadIdx.x) & 63, kv = head / a.group;
    const int64_t at = static_cast<int64_t>(head) * a.head_dim;
    const T* q = static_cast<const T*>(a.q) + at;
    const T* dout = static_cast<const T*>(a.dout) + at;
    const T* k = static_cast<const T*>(a.k) + j * a.k_stride + static_cast<int64_t>(kv) * a.head_dim;
    const T* v = static_cast<const T*>(a.v) + j * a.v_stride + static_cast<int64_t>(kv) * a.head_dim;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const float* lse = a.lse + static_cast<int64_t>(head) * a.tokens;
    const float* delta = a.delta + static_cast<int64_t>(head) * a.tokens;
    const Span s = query_span(a, doc, j);
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) dk[c] = dv[c] = 0.0f;
    for (int base = s.low; base < s.high; base += 64) {
        const int i = base + lane;
        const bool see = i < s.high;
        float p = 0.0f, ds = 0.0f;
        if (see) {
            float derivative;
            const float x = bend_score(a, slope, dot_row(q + i * a.q_stride, k, a.head_dim), i - j, derivative);
            const float dp = dot_row(dout + i * a.out_stride, v, a.head_dim);
            p = expf(x - lse[i]);
            ds = p * (dp - delta[i]) * derivative * a.scale;
        }
        if (__any(p != p)) {
            all_nan(dk), all_nan(dv);
            return;
        }
        for (uint64_t left = __ballot(see); left; left &= left - 1) {
            const int from_lane = __ffsll(static_cast<unsigned long long>(left)) - 1;
            const float pj = __shfl(p, from_lane), dj = __shfl(ds, from_lane);
            const T* qi = q + (base + from_lane) * a.q_stride;
            const T* di = dout + (base + from_lane) * a.out_stride;
#pragma unroll
            for (int c = 0; c < kLaneDims; ++c)
                if (lane + 64 * c < a.head_dim) {
                    dk[c] = fmaf(dj, static_cast<float>(qi[lane + 64 * c]), dk[c]);
                    dv[c] = fmaf(pj, static_cast<float>(di[lane + 64 * c]), dv[c]);
                }
        }
    }
}

// A row of head_dim elements from a wave's registers.
template <typename To>
__device__ __forceinline__ void store_row(To* to, const float (&v)[kLaneDims], int head_dim) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c)
        if (lane + 64 * c < head_dim) to[lane + 64 * c] = static_cast<To>(v[c]);
}

// Tiles that find_tile gives parts of `rows` tokens, at most.
inline unsigned doc_tiles(const DocAttention& a, int rows) {
    const int parts_begun = a.documents > kFewDocuments ? a.documents : std::min(a.documents, a.tokens);
    return static_cast<unsigned>(ceil_div(a.tokens, rows) + parts_begun);
}

// Whole 16-byte chunks throughout, and strides that leave a copy's lane offsets below 2^32 bytes.
inline bool whole_chunks(const DocAttention& a, int64_t chunk, std::initializer_list<const void*> arrays) {
    bool whole = a.head_dim % chunk == 0;
    for (const int64_t s : {a.q_stride, a.k_stride, a.v_stride, a.out_stride})
        whole = whole && s % chunk == 0 && s < (int64_t{1} << 25);
    for (const void* p : arrays) whole = whole && aligned_to(p, 16);
    return whole;
}

// Bytes of one token of q, k, v (and dout) as packed sources.
template <typename T>
size_t packed_token_bytes(const DocAttention& a, bool backward) {
    const size_t heads = static_cast<size_t>(a.heads) * (backward ? 2 : 1) + 2 * static_cast<size_t>(a.kv_heads);
    return heads * round_up(a.head_dim, kPartChunk) * 2 * kPlanes<T>;
}

struct PackArgs {
    const void* from[4];
    int64_t stride[4];
    Source to[4];
    int heads[4];
    int tokens, head_dim;
    bool whole;
    const void* out;  // backward: with dout, for
    float* delta;
    int skip;  // arrays that need no copy: all four, or none
};

// dout . out of every token and head: 16 lanes to a row, 16 bytes of it to a lane at a time. Bound: HBM (8192 tokens, 16 heads of 128
// in bfloat16: 14 us, 4.8 TB/s) where a token has 16 heads or more; of a token with fewer the other lanes of a workgroup of 256
// have none (12 heads: 12 us).
template <typename T>
__device__ __forceinline__ void row_products(const PackArgs& a) {
    constexpr int kWide = kChunk<T>, kLanes = 16;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x)
        for (int head = static_cast<int>(threadIdx.x) / kLanes; head < a.heads[3]; head += 256 / kLanes) {
            const int64_t at = token * a.stride[3] + static_cast<int64_t>(head) * a.head_dim;
            const T* const out = static_cast<const T*>(a.out) + at;
            const T* const dout = static_cast<const T*>(a.from[3]) + at;
            float sum = 0.0f;
            for (int d = lane * kWide; d < a.head_dim; d += kLanes * kWide) {
                float o[kWide] = {}, g[kWide] = {};
                if (a.whole) {
                    load_as_float<T, kWide>(out + d, o);
                    load_as_float<T, kWide>(dout + d, g);
                } else {
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
                        if (d + j < a.head_dim) o[j] = static_cast<float>(out[d + j]), g[j] = static_cast<float>(dout[d + j]);
                }
#pragma unroll
                for (int j = 0; j < kWide; ++j) sum = fmaf(o[j], g[j], sum);
            }
#pragma unroll
            for (int s = kLanes / 2; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
            if (lane == 0) a.delta[static_cast<int64_t>(head) * a.tokens + token] = sum;
        }
}

// Copies arrays into sources: split into planes, heads filled up with zeroes to whole chunks. A workgroup has some tokens, a
// thread a chunk of 8 elements at a time. The gradients have row_products from here, too, in the same launch. Bound: HBM (4096
// tokens of 32 heads of 128 in float32: 26 us for 168 MB).
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
    const int which = static_cast<int>(blockIdx.y) + a.skip;
    if (which == 4) return row_products<T>(a);
    const Source to = a.to[which];
    const int per_token = a.heads[which] * to.chunks;
    const int at_once = per_token < 256 ? 256 / per_token : 1;  // tokens of a turn of the workgroup
    const int mine = static_cast<int>(threadIdx.x) / per_token, first = static_cast<int>(threadIdx.x) % per_token;
    if (per_token < 256 && mine >= at_once) return;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * at_once; base < a.tokens; base += static_cast<int64_t>(gridDim.x) * at_once) {
        const int64_t token = base + (per_token < 256 ? mine : 0);
        if (token >= a.tokens) return;
        for (int c = per_token < 256 ? first : static_cast<int>(threadIdx.x); c < per_token; c += per_token < 256 ? per_token : 256) {
            const int head = c / to.chunks, chunk = c - head * to.chunks;
            const T* from = static_cast<const T*>(a.from[which]) + token * a.stride[which] + static_cast<int64_t>(head) * a.head_dim + chunk * kPartChunk;
            const int there = a.head_dim - chunk * kPartChunk;  // elements of the head from here on
            T x[kPartChunk];
            if (a.whole && there >= kPartChunk) {
#pragma unroll
                for (int h = 0; h < kPartChunk; h += kChunk<T>)
                    *reinterpret_cast<Pack<T, kChunk<T>>*>(x + h) = *reinterpret_cast<const Pack<T, kChunk<T>>*>(from + h);
            } else {
#pragma unroll
                for (int j = 0; j < kPartChunk; ++j) x[j] = j < there ? from[j] : static_cast<T>(0.0f);
            }
            Pack<Part<T>, kPartChunk> planes[kPlanes<T>];
#pragma unroll
            for (int j = 0; j < kPartChunk; ++j) {
                Part<T> parts[kPlanes<T>];
                if constexpr (kPlanes<T> == 1)
                    parts[0] = x[j];
                else
                    split<T>(x[j], parts);
#pragma unroll
                for (int p = 0; p < kPlanes<T>; ++p) planes[p].v[j] = parts[p];
            }
#pragma unroll
            for (int p = 0; p < kPlanes<T>; ++p)
                *reinterpret_cast<Pack<Part<T>, kPartChunk>*>(const_cast<char*>(to.base) + p * to.plane + token * to.stride +
                                                              head * to.head + chunk * 16) = planes[p];
        }
    }
}

// a's sources: the arrays themselves where they are 16-bit and whole, else copies in the workspace.
template <typename T>
void set_sources(DocAttention& a, bool backward, char* packed, hipStream_t stream) {
    const void* const arrays[4] = {a.q, a.k, a.v, a.dout};
    const int64_t strides[4] = {a.q_stride, a.k_stride, a.v_stride, a.out_stride};
    const int heads[4] = {a.heads, a.kv_heads, a.kv_heads, a.heads};
    const int count = backward ? 4 : 3;
    const int chunks = static_cast<int>(ceil_div(a.head_dim, kPartChunk));
    const bool as_they_are = kPlanes<T> == 1 && a.whole;
    PackArgs p{};
    p.tokens = a.tokens;
    p.head_dim = a.head_dim;
    p.whole = a.whole;
    for (int i = 0; i < count; ++i) {
        const int64_t row = int64_t{heads[i]} * chunks * 16, plane = row * a.tokens;
        if (as_they_are) {
            a.sources[i] = {static_cast<const char*>(arrays[i]), strides[i] * 2, int64_t{a.head_dim} * 2, 0, chunks};
        } else {
            a.sources[i] = {packed, row, int64_t{chunks} * 16, plane, chunks};
            packed += plane * kPlanes<T>;
        }
        p.from[i] = arrays[i], p.stride[i] = strides[i], p.to[i] = a.sources[i], p.heads[i] = heads[i];
    }
    p.out = a.out, p.delta = a.delta;
    p.skip = as_they_are ? 4 : 0;
    const int parts = (as_they_are ? 0 : count) + (backward ? 1 : 0);
    if (!parts) return;
    const size_t blocks = ceil_div(static_cast<size_t>(a.tokens) * a.heads * chunks, 256);
    pack_kernel<T><<<dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), parts), 256, 0, stream>>>(p);
}

// doc_attention_{f32,bf16,f16}.hip
template <typename T>
int launch_document_attention(DocAttention a, void* out, char* packed, hipStream_t stream);
template <typename T>
int launch_document_attention_backward(DocAttention a, char* packed, hipStream_t stream);

}  // namespace dllm_hip
