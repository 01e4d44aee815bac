// The sort and the sums of token_rows.h.
//
// Sort by digits: least significant first, 9 bits at a time (a vocabulary of 2^18 takes two passes). A position's place is the
// number of smaller digits, the same digits in earlier waves (counts of each wave and digit, scanned), and those before it
// in its own wave, which 9 ballots per 64 positions give without any atomic operation, so the sort is stable and its result
// the same every time. Up to 16384 positions are first dealt to workgroups by a hash of the token, since one workgroup's ballots
// over all of them took 39 us; more go through memory, each pass three launches.
//
// Sums: a token's positions are added 8 at a time from its first one on, whatever tokens lie beside it, so a row of the sums is the
// same bits in any batch that has its positions. A wave takes the groups of 8 that begin among 8 sorted positions, and 16 bytes of
// columns to a lane; it reads all their rows (up to 15) at once and adds them in order. A token of at most 8 is done; the groups of
// others are float32 parts, added in their order by a second launch. Nothing depends on when a wave runs. 16381 rows of 576 in
// float32 onto a table that is added to: sort 22 us, sums 14 (2.7 TB/s of rows read), parts 9, a chain of additions as long as the
// most frequent token's; 16 positions to a wave were no faster.
#include "token_rows.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace dllm_hip {

namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortRounds = 16;  // positions of a thread
constexpr int kSortBlock = kSortThreads * kSortRounds;
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;

struct SortCounts {
    uint16_t wave[kSortWaves][kDigits];
    uint32_t digit[kDigits];
    uint32_t carry[kDigits / kWave];
};

// The items of a workgroup lie wave by wave, `rounds` times 64 to a wave.
__device__ __forceinline__ int sort_item(int rounds, int r) {
    return ((static_cast<int>(threadIdx.x) >> 6) * rounds + r) * kWave + (static_cast<int>(threadIdx.x) & 63);
}

// rank[i]: how many items with item i's digit come before it in its wave; then counts.wave: those in earlier waves;
// counts.digit: the items with smaller digits.
__device__ __forceinline__ void rank_digits(const uint32_t* keys, int rounds, int n, int shift, SortCounts& counts, uint16_t* ranks) {
    const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
    for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) (&counts.wave[0][0])[i] = 0;
    __syncthreads();
    volatile uint16_t* const mine = counts.wave[wave];
    for (int r = 0; r < rounds; ++r) {
        const int i = sort_item(rounds, r);
        const bool valid = i < n;
        const uint32_t d = valid ? (keys[i] >> shift) & (kDigits - 1) : 0;
        uint64_t same = __ballot(valid);
#pragma unroll
        for (int b = 0; b < kDigitBits; ++b) {
            const uint64_t set = __ballot((d >> b) & 1);
            same &= (d >> b) & 1 ? set : ~set;
        }
        const int before = __popcll(same & ((uint64_t{1} << lane) - 1));
        const int old = mine[d];
        __builtin_amdgcn_wave_barrier();
        if (valid) {
            ranks[i] = static_cast<uint16_t>(old + before);
            if (before == 0) mine[d] = static_cast<uint16_t>(old + __popcll(same));
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    uint32_t total = 0, sum = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const uint32_t c = counts.wave[w][threadIdx.x];
            counts.wave[w][threadIdx.x] = static_cast<uint16_t>(total);
            total += c;
        }
        sum = total;
#pragma unroll
        for (int s = 1; s < kWave; s *= 2) {
            const uint32_t o = __shfl_up(sum, s);
            if (lane >= s) sum += o;
        }
        if (lane == kWave - 1) counts.carry[wave] = sum;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
        uint32_t before = 0;
        for (int w = 0; w < wave; ++w) before += counts.carry[w];
        counts.digit[threadIdx.x] = before + sum - total;
    }
    __syncthreads();
}

__device__ __forceinline__ uint32_t token_key(int64_t token, int64_t vocabulary) {
    return static_cast<uint32_t>(token >= 0 && token < vocabulary ? token : vocabulary);
}

// word to every word of `bytes` bytes at `at` (aligned to 2), by workgroup `block` of `blocks`
__device__ __forceinline__ void fill_part(char* at, size_t bytes, uint32_t word, size_t block, size_t blocks) {
    const size_t head = min(bytes, (16 - reinterpret_cast<uintptr_t>(at) % 16) % 16), chunks = (bytes - head) / 16;
    uint4* const body = reinterpret_cast<uint4*>(at + head);
    for (size_t i = block * blockDim.x + threadIdx.x; i < chunks; i += blocks * blockDim.x) body[i] = make_uint4(word, word, word, word);
    const size_t tail = head + chunks * 16;
    if (block == 0) {
        for (size_t i = 2 * threadIdx.x; i + 2 <= head; i += 2 * blockDim.x) *reinterpret_cast<uint16_t*>(at + i) = static_cast<uint16_t>(word);
        for (size_t i = tail + 2 * threadIdx.x; i + 2 <= bytes; i += 2 * blockDim.x)
            *reinterpret_cast<uint16_t*>(at + i) = static_cast<uint16_t>(word);
    }
}

__global__ __launch_bounds__(256) void fill_kernel(char* at, size_t bytes, uint32_t word) {
    fill_part(at, bytes, word, blockIdx.x, gridDim.x);
}

// Up to kSortBlock positions. A workgroup to each of 2^bucket_bits parts of the tokens, by a hash, and one to those outside: it
// lists its positions in their order, counts those of the parts before it, and sorts its own by token; short lists by counting
// the smaller ones, longer ones by digits. The others fill. 16381 tokens of 49152 in 128 parts: 22 us (39 in one), most of
// it the longest list's, a frequent token's. Beside a fill, which takes longer, few workgroups sort.
constexpr int kBucketBits = 7, kBucketBitsWithFill = 4;
constexpr int kCountedList = 256;

__device__ __forceinline__ int bucket_of(uint32_t key, uint32_t outside, int bits) {
    return key == outside ? 1 << bits : static_cast<int>((key * 2654435769u) >> (32 - bits));
}

__global__ __launch_bounds__(kSortThreads) void sort_kernel(const int64_t* __restrict__ tokens, int n, int64_t vocabulary, int passes,
                                                            int bucket_bits, TokenOrder order, char* fill_at, size_t fill_bytes, uint32_t fill) {
    __shared__ SortCounts counts;
    __shared__ __attribute__((aligned(16))) uint32_t keys[kSortBlock];
    __shared__ uint16_t positions[kSortBlock], ranks[kSortBlock];
    __shared__ int mine_of[kSortWaves], before_of[kSortWaves];
    const int bucket = static_cast<int>(blockIdx.x), buckets = 1 << bucket_bits;
    if (bucket > buckets) {
        fill_part(fill_at, fill_bytes, fill, bucket - buckets - 1, gridDim.x - buckets - 1);
        return;
    }
    const uint32_t outside = static_cast<uint32_t>(vocabulary);
    const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
    const int rounds_all = (n + kSortThreads - 1) / kSortThreads;
    uint32_t key[kSortRounds];
    uint32_t in_bucket = 0;  // bit r: item r is this bucket's
    int mine = 0, before = 0;
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        if (r < rounds_all) {
            const int i = sort_item(rounds_all, r);
            key[r] = i < n ? token_key(tokens[i], vocabulary) : ~0u;
        }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        if (r < rounds_all) {
            const int of = key[r] == ~0u ? buckets + 1 : bucket_of(key[r], outside, bucket_bits);
            mine += __popcll(__ballot(of == bucket));
            before += __popcll(__ballot(of < bucket));
            in_bucket |= (of == bucket ? 1u : 0u) << r;
        }
    if (lane == 0) mine_of[wave] = mine, before_of[wave] = before;
    __syncthreads();
    int list = 0, base = 0, at = 0;
    for (int w = 0; w < kSortWaves; ++w) {
        if (w < wave) at += mine_of[w];
        list += mine_of[w];
        base += before_of[w];
    }
    if (bucket == buckets && threadIdx.x == 0) *order.kept = base;
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        if (r < rounds_all) {
            const uint64_t in = __ballot(in_bucket >> r & 1);
            if (in >> lane & 1) {
                const int to = at + __popcll(in & ((uint64_t{1} << lane) - 1));
                keys[to] = key[r];
                positions[to] = static_cast<uint16_t>(sort_item(rounds_all, r));
            }
            at += __popcll(in);
        }
    __syncthreads();
    bool alike = true;
    for (int i = threadIdx.x; i < list; i += kSortThreads) alike = alike && keys[i] == keys[0];
    if (__syncthreads_and(alike)) {  // the positions' order is theirs already
        for (int i = threadIdx.x; i < list; i += kSortThreads) order.token[base + i] = keys[i], order.position[base + i] = positions[i];
        return;
    }
    if (list <= kCountedList) {
        if (static_cast<int>(threadIdx.x) < list) {
            const uint32_t own = keys[threadIdx.x];
            const int self = static_cast<int>(threadIdx.x);
            int rank = 0;
#pragma unroll 4
            for (int i = 0; i < list; i += 4) {  // (what is read past the list does not count)
                const uint4 four = *reinterpret_cast<const uint4*>(keys + i);
                const uint32_t k[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) rank += i + e < list && (k[e] < own || (k[e] == own && i + e < self));
            }
            order.token[base + rank] = own;
            order.position[base + rank] = positions[threadIdx.x];
        }
        return;
    }
    const int rounds = (list + kSortThreads - 1) / kSortThreads;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * kDigitBits;
        rank_digits(keys, rounds, list, shift, counts, ranks);
        uint32_t moved[kSortRounds], to[kSortRounds];
        uint16_t position[kSortRounds];
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
            const int i = sort_item(rounds, r);
            if (r < rounds && i < list) {
                moved[r] = keys[i], position[r] = positions[i];
                const uint32_t d = (moved[r] >> shift) & (kDigits - 1);
                to[r] = counts.digit[d] + counts.wave[wave][d] + ranks[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r)
            if (r < rounds && sort_item(rounds, r) < list) keys[to[r]] = moved[r], positions[to[r]] = position[r];
        __syncthreads();
    }
    for (int i = threadIdx.x; i < list; i += kSortThreads) order.token[base + i] = keys[i], order.position[base + i] = positions[i];
}

// One pass over more positions: this workgroup's number of each digit, by digit and workgroup ...
__global__ __launch_bounds__(kSortThreads) void digit_counts_kernel(const int64_t* __restrict__ tokens, const uint32_t* __restrict__ key,
                                                                    int64_t n, int64_t vocabulary, int shift, int64_t each, uint32_t* __restrict__ counts) {
    __shared__ uint32_t of[kDigits];
    for (int i = threadIdx.x; i < kDigits; i += kSortThreads) of[i] = 0;
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * each, end = min(n, first + each);
    for (int64_t i = first + threadIdx.x; i < end; i += kSortThreads)
        atomicAdd(&of[((key ? key[i] : token_key(tokens[i], vocabulary)) >> shift) & (kDigits - 1)], 1u);
    __syncthreads();
    for (int i = threadIdx.x; i < kDigits; i += kSortThreads) counts[static_cast<size_t>(i) * gridDim.x + blockIdx.x] = of[i];
}

// ... their sums before each, by one workgroup, 8 to a thread (n is a multiple of 8) ...
__global__ __launch_bounds__(kSortThreads) void scan_kernel(uint32_t* __restrict__ counts, int64_t n) {
    __shared__ uint32_t carry[kSortWaves];
    const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
    uint32_t before = 0;
    for (int64_t base = 0; base < n; base += 8 * kSortThreads) {
        const int64_t i = base + 8 * threadIdx.x;
        Pack<uint32_t, 8> c = {};
        if (i < n) c = *reinterpret_cast<const Pack<uint32_t, 8>*>(counts + i);
        uint32_t own = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) own += c.v[e];
        uint32_t sum = own;
#pragma unroll
        for (int s = 1; s < kWave; s *= 2) {
            const uint32_t o = __shfl_up(sum, s);
            if (lane >= s) sum += o;
        }
        if (lane == kWave - 1) carry[wave] = sum;
        __syncthreads();
        uint32_t earlier = before + sum - own;
        for (int w = 0; w < kSortWaves; ++w) {
            if (w < wave) earlier += carry[w];
            before += carry[w];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t one = c.v[e];
            c.v[e] = earlier;
            earlier += one;
        }
        if (i < n) *reinterpret_cast<Pack<uint32_t, 8>*>(counts + i) = c;
        __syncthreads();
    }
}

// ... and the positions to their places.
__global__ __launch_bounds__(kSortThreads) void scatter_kernel(const int64_t* __restrict__ tokens, const uint32_t* __restrict__ key_in,
                                                               const uint32_t* __restrict__ position_in, int64_t n, int64_t vocabulary,
                                                               int shift, int rounds, const uint32_t* __restrict__ before, uint32_t* __restrict__ key_out,
                                                               uint32_t* __restrict__ position_out) {
    __shared__ SortCounts counts;
    __shared__ uint32_t keys[kSortBlock];
    __shared__ uint16_t ranks[kSortBlock];
    const int64_t each = static_cast<int64_t>(rounds) * kSortThreads, first = static_cast<int64_t>(blockIdx.x) * each;
    const int here = static_cast<int>(min(n - first, each));
    for (int i = threadIdx.x; i < here; i += kSortThreads) keys[i] = key_in ? key_in[first + i] : token_key(tokens[first + i], vocabulary);
    __syncthreads();
    rank_digits(keys, rounds, here, shift, counts, ranks);
    for (int i = threadIdx.x; i < here; i += kSortThreads) {
        const uint32_t key = keys[i], d = (key >> shift) & (kDigits - 1);
        const int wave = i / (kWave * rounds);  // the one that ranked it
        const uint32_t to = before[static_cast<size_t>(d) * gridDim.x + blockIdx.x] + counts.wave[wave][d] + ranks[i];
        key_out[to] = key;
        position_out[to] = position_in ? position_in[first + i] : static_cast<uint32_t>(first + i);
    }
}

__global__ __launch_bounds__(256) void kept_kernel(const uint32_t* __restrict__ token, int64_t n, uint32_t outside, uint32_t* __restrict__ kept) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n) return;
    if (token[i] != outside && (i == n - 1 || token[i + 1] == outside)) *kept = static_cast<uint32_t>(i + 1);
    if (i == 0 && token[0] == outside) *kept = 0;
}

// ---- sums ----

constexpr int kSumRows = 8;  // sorted positions of a wave

struct SumArgs {
    const uint32_t* token;
    const uint32_t* position;
    int64_t n, dim, stride, blocks;
    uint32_t outside;
    const float* coefficient;
    float scale;
    float* part;
    bool accumulate;
    float* sums;
    int32_t* first;
};

template <typename T, int kWidth>
__device__ __forceinline__ void finish_sum(const SumArgs& a, T* table, uint32_t token, int64_t index, int64_t column, float (&acc)[kWidth]) {
#pragma unroll
    for (int j = 0; j < kWidth; ++j) acc[j] *= a.scale;
    if (a.sums) {
        if (column == 0) a.first[token] = static_cast<int32_t>(index);
        store_from_float<float, kWidth>(a.sums + index * a.dim + column, acc);
        return;
    }
    T* const row = table + static_cast<int64_t>(token) * a.dim + column;
    if (a.accumulate) {
        float old[kWidth];
        load_as_float<T, kWidth>(row, old);
#pragma unroll
        for (int j = 0; j < kWidth; ++j) acc[j] += old[j];
    }
    store_from_float<T, kWidth>(row, acc);
}

// What a wave makes of the positions first .. first + 15, a lane each (16 lanes count): bit masks.
struct Runs {
    uint32_t inside;  // there is a position, of a token inside the vocabulary
    uint32_t starts;  // a token's first position
    uint32_t groups;  // the first of a token's 8
    int earlier;      // positions of the first one's token before it
};

// The start of the run of t that reaches up to `first` from below, where token[first - 1] is t: 64 probes at a time, since
// whether a position before `first` is the run's goes from no to yes once.
__device__ __forceinline__ int64_t run_start(const uint32_t* token, int64_t first, uint32_t t, int lane) {
    int64_t low = 0, high = first - 1;  // the start is in [low, high], and high is the run's
    {
        const int64_t at = first - 1 - lane;  // most runs are short
        const uint64_t in = __ballot(at >= 0 && token[at >= 0 ? at : 0] == t);
        if (~in) return first - (__ffsll(static_cast<unsigned long long>(~in)) - 1);
        high = first - kWave;
    }
    while (low < high) {
        const int64_t step = (high - low + kWave - 1) / kWave;
        const int64_t at = min(low + lane * step, high);
        const int in = __ffsll(static_cast<unsigned long long>(__ballot(token[at] == t))) - 1;
        if (in < 0) {  // (between the last probe and high)
            low = min(low + (kWave - 1) * step, high) + 1;
        } else {
            high = min(low + in * step, high);
            if (in > 0) low = min(low + (in - 1) * step, high - 1) + 1;
            else low = high;
        }
    }
    return low;
}

__device__ __forceinline__ Runs runs_of(const uint32_t* token, int64_t n, uint32_t outside, int64_t first, int lane, uint32_t own) {
    const uint32_t t0 = __builtin_amdgcn_readfirstlane(own), previous = first > 0 ? token[first - 1] : outside;
    const uint32_t before = __shfl_up(own, 1);
    Runs r;
    r.inside = static_cast<uint32_t>(__ballot(lane < 2 * kSumRows && first + lane < n && own != outside));
    r.starts = static_cast<uint32_t>(__ballot(lane < 2 * kSumRows && own != (lane == 0 ? previous : before))) & r.inside;
    r.earlier = 0;
    if (first > 0 && t0 != outside && t0 == previous) r.earlier = static_cast<int>((first - run_start(token, first, t0, lane)) & (kSumRows - 1));
    const uint32_t below = r.starts & ((2u << (lane & 31)) - 1);
    const int rank = below ? lane - (31 - __clz(below)) : lane + r.earlier;
    r.groups = static_cast<uint32_t>(__ballot(lane < 2 * kSumRows && (rank & (kSumRows - 1)) == 0)) & r.inside;
    return r;
}

// A wave forms the sums of the groups of 8 that begin among its 8 positions. part[block][0]: of a token that began earlier;
// part[block][1]: the first 8 of one that begins here and has more.
template <typename T, int kWidth>
__global__ __launch_bounds__(256) void token_sums_kernel(const T* __restrict__ rows, T* __restrict__ table, SumArgs a) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int64_t block = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)));
    if (block >= a.blocks) return;
    const int64_t first = block * kSumRows, column = (static_cast<int64_t>(blockIdx.y) * kWave + lane) * kWidth;
    uint32_t token = a.outside, position = 0;
    if (lane < 2 * kSumRows && first + lane < a.n) token = a.token[first + lane], position = a.position[first + lane];
    const Runs r = runs_of(a.token, a.n, a.outside, first, lane, token);
    // from the first group that begins here to the end of the last one
    const uint32_t here = r.groups & ((1u << kSumRows) - 1), past = (r.groups | ~r.inside) >> kSumRows;
    if (!here) return;
    const int begin = __ffs(here) - 1, end = kSumRows + __ffs(past | (1u << kSumRows)) - 1;
    const uint32_t mine = r.inside & ((1u << end) - 1) & ~((1u << begin) - 1);
    float weight = 1.0f;
    if (a.coefficient && mine >> (lane & 31) & 1 && lane < 2 * kSumRows) weight = a.coefficient[position];
    const bool inside = column < a.dim;
    constexpr int kMost = 2 * kSumRows - 1;
    using Words = uint32_t __attribute__((ext_vector_type(kWidth * sizeof(T) >= 8 ? kWidth * sizeof(T) / 4 : 2)));
    using Row = std::conditional_t<kWidth == 1, T, Words>;  // (16-bit elements one by one would take a register each)
    Row row[kMost] = {};
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const uint32_t p = __builtin_amdgcn_readlane(position, i);
        if (mine >> i & 1 && inside) row[i] = *reinterpret_cast<const Row*>(rows + static_cast<int64_t>(p) * a.stride + column);
    }
    // (all lanes stay: the tokens are read from lanes whose columns are past the row too)
    float acc[kWidth] = {};
    int group = begin;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        if (!(mine >> i & 1)) continue;
        const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), i));
        const Pack<T, kWidth> v = __builtin_bit_cast(Pack<T, kWidth>, row[i]);
#pragma unroll
        for (int j = 0; j < kWidth; ++j) acc[j] = fmaf(c, static_cast<float>(v.v[j]), acc[j]);
        if (!((r.groups | ~r.inside) >> (i + 1) & 1)) continue;
        if (inside) {
            const bool begins = r.starts >> group & 1, ends = (r.starts | ~r.inside) >> (i + 1) & 1;
            if (begins && ends)
                finish_sum<T, kWidth>(a, table, __builtin_amdgcn_readlane(token, i), first + group, column, acc);
            else
                store_from_float<float, kWidth>(a.part + (2 * block + (begins ? 1 : 0)) * a.dim + column, acc);
        }
#pragma unroll
        for (int j = 0; j < kWidth; ++j) acc[j] = 0.0f;
        group = i + 1;
    }
}

// Adds the groups' parts of a token that begins among this wave's positions and has more than 8.
template <typename T, int kWidth>
__global__ __launch_bounds__(256) void token_parts_kernel(T* __restrict__ table, SumArgs a) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int64_t block = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)));
    if (block >= a.blocks - 1) return;  // what begins in the last block has at most 8
    const int64_t first = block * kSumRows;
    const uint32_t own = lane < kSumRows ? a.token[first + lane] : a.outside;
    const uint32_t previous = lane > 0 ? a.token[first + min(lane, kSumRows) - 1] : first > 0 ? a.token[first - 1] : a.outside;
    const uint32_t starts = static_cast<uint32_t>(__ballot(lane < kSumRows && own != a.outside && own != previous));
    if (!starts) return;
    const int64_t index = first + 31 - __clz(starts);  // the last one alone can have more
    const uint32_t t = a.token[index];
    // further groups
    int64_t more = 0;
    for (;; more += kWave) {
        const int64_t at = index + (more + lane + 1) * kSumRows;
        const uint64_t stops = ~__ballot(at < a.n && a.token[min(at, a.n - 1)] == t);
        if (stops) {
            more += __ffsll(static_cast<unsigned long long>(stops)) - 1;
            break;
        }
    }
    if (more == 0) return;
    const int64_t column = (static_cast<int64_t>(blockIdx.y) * kWave + lane) * kWidth;
    if (column >= a.dim) return;
    float acc[kWidth];
    load_as_float<float, kWidth>(a.part + (2 * block + 1) * a.dim + column, acc);
    const float* part = a.part + 2 * (block + 1) * a.dim + column;
    int64_t i = 0;
    constexpr int kAhead = 16;
    for (; i + kAhead <= more; i += kAhead) {
        float v[kAhead][kWidth];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) load_as_float<float, kWidth>(part + 2 * (i + k) * a.dim, v[k]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int j = 0; j < kWidth; ++j) acc[j] += v[k][j];
    }
    for (; i < more; ++i) {
        float v[kWidth];
        load_as_float<float, kWidth>(part + 2 * i * a.dim, v);
#pragma unroll
        for (int j = 0; j < kWidth; ++j) acc[j] += v[j];
    }
    finish_sum<T, kWidth>(a, table, t, index, column, acc);
}

template <typename T, int kWidth>
int launch_sums(const TokenSums& s, const SumArgs& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.blocks, 4)), static_cast<unsigned>(ceil_div(a.dim, kWave * kWidth)));
    token_sums_kernel<T, kWidth><<<grid, 256, 0, stream>>>(static_cast<const T*>(s.rows), static_cast<T*>(s.table), a);
    if (a.blocks > 1) token_parts_kernel<T, kWidth><<<grid, 256, 0, stream>>>(static_cast<T*>(s.table), a);
    return check_launch("token_sums");
}

template <typename T>
int launch_sums_of(const TokenSums& s, hipStream_t stream) {
    SumArgs a{};
    a.token = s.order.token, a.position = s.order.position;
    a.n = s.n, a.dim = s.dim, a.stride = s.stride;
    a.blocks = static_cast<int64_t>(ceil_div(s.n, kSumRows));
    a.outside = static_cast<uint32_t>(s.vocabulary);
    a.coefficient = s.coefficient, a.scale = s.scale, a.part = s.part;
    a.accumulate = s.accumulate, a.sums = s.sums, a.first = s.first;
    constexpr int kWide = kChunk<T>;
    const bool wide = s.dim % kWide == 0 && s.stride % kWide == 0 && aligned_to(s.rows, 16) && aligned_to(s.table, 16);
    return wide ? launch_sums<T, kWide>(s, a, stream) : launch_sums<T, 1>(s, a, stream);
}

}  // namespace

namespace {
// Positions of a thread where the sort goes through memory: as many workgroups as one can scan the counts of (23234 tokens took
// 109 us for the gradient of a small table with workgroups of 16384).
int sort_rounds(int64_t n) { return static_cast<int>(std::clamp<int64_t>(static_cast<int64_t>(ceil_div(n, 64 * kSortThreads)), 1, kSortRounds)); }
}  // namespace

TokenOrderSizes::TokenOrderSizes(int64_t tokens) : n(static_cast<size_t>(tokens)) {
    const bool memory = tokens > kSortBlock;
    spare = memory ? n : 0;
    counts = memory ? ceil_div(n, sort_rounds(tokens) * kSortThreads) * kDigits : 0;
}

int fill_words(void* at, size_t bytes, uint32_t word, hipStream_t stream) {
    const size_t blocks = std::min<size_t>(ceil_div(bytes, 256 * 16), 2048);
    fill_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<char*>(at), bytes, word);
    return check_launch("fill_words");
}

int sort_tokens(const int64_t* tokens, int64_t n, int64_t vocabulary, const TokenOrder& o, void* fill_at, size_t fill_bytes, uint32_t fill,
                hipStream_t stream) {
    int bits = 1;
    while (bits < 32 && vocabulary >> bits) ++bits;
    const int passes = (bits + kDigitBits - 1) / kDigitBits;
    char* const to = static_cast<char*>(fill_at);
    if (n <= kSortBlock) {
        const bool long_fill = fill_bytes > (size_t{64} << 20);  // of more than a sort's time
        const int bits = long_fill ? kBucketBitsWithFill : kBucketBits, sorting = (1 << bits) + 1;
        const size_t fills = std::min<size_t>(ceil_div(fill_bytes, kSortThreads * 16), 256 - sorting);
        sort_kernel<<<static_cast<unsigned>(sorting + fills), kSortThreads, 0, stream>>>(tokens, static_cast<int>(n), vocabulary, passes, bits, o, to,
                                                                                    fill_bytes, fill);
        return check_launch("sort_tokens");
    }
    if (fill_bytes) DLLM_TRY(fill_words(fill_at, fill_bytes, fill, stream));
    const int rounds = sort_rounds(n);
    const int64_t each = static_cast<int64_t>(rounds) * kSortThreads;
    const unsigned blocks = static_cast<unsigned>(ceil_div(n, each));
    // the last pass ends in the order's own arrays
    uint32_t *key_in = nullptr, *position_in = nullptr;
    for (int pass = 0; pass < passes; ++pass) {
        const bool own = (passes - 1 - pass) % 2 == 0;
        uint32_t *const key_out = own ? o.token : o.spare_token, *const position_out = own ? o.position : o.spare_position;
        const int shift = pass * kDigitBits;
        digit_counts_kernel<<<blocks, kSortThreads, 0, stream>>>(tokens, key_in, n, vocabulary, shift, each, o.counts);
        scan_kernel<<<1, kSortThreads, 0, stream>>>(o.counts, static_cast<int64_t>(blocks) * kDigits);
        scatter_kernel<<<blocks, kSortThreads, 0, stream>>>(tokens, key_in, position_in, n, vocabulary, shift, rounds, o.counts, key_out, position_out);
        key_in = key_out, position_in = position_out;
    }
    kept_kernel<<<static_cast<unsigned>(ceil_div(n, 256)), 256, 0, stream>>>(o.token, n, static_cast<uint32_t>(vocabulary), o.kept);
    return check_launch("sort_tokens");
}

size_t token_sums_part_floats(int64_t n, int64_t dim) {
    const size_t blocks = ceil_div(static_cast<size_t>(n), kSumRows);
    return blocks > 1 ? 2 * blocks * static_cast<size_t>(dim) : 0;
}

int launch_token_sums(const TokenSums& a, int64_t dtype, hipStream_t stream) {
    switch (dtype) {
        case kFloat32: return launch_sums_of<float>(a, stream);
        case kBFloat16: return launch_sums_of<__bf16>(a, stream);
        default: return launch_sums_of<_Float16>(a, stream);
    }
}

}  // namespace dllm_hip
