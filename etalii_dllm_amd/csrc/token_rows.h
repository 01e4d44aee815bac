// Rows gathered by token: a stable grouping of positions by token, and the sums of the rows of each token in the order of their
// positions. The embedding table's gradient is such a sum, and so is the targets' part of the vocabulary loss's.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "element.h"
#include "workspace.h"

namespace dllm_hip {

constexpr int64_t kMaxSortTokens = int64_t{1} << 27;  // the counts of larger sorts would be scanned by one workgroup for long

// Positions 0 .. n - 1 grouped by token, and what the sort needs beside them.
struct TokenOrder {
    uint32_t* token;     // [n] each token's together; tokens outside the vocabulary count as `vocabulary` and come last
    uint32_t* position;  // [n] ascending within a token
    uint32_t* kept;      // [1] how many are inside
    uint32_t* spare_token;
    uint32_t* spare_position;
    uint32_t* counts;
};

struct TokenOrderSizes {
    size_t n, spare, counts;
    explicit TokenOrderSizes(int64_t tokens);
};

inline void add_token_order(Layout& l, int64_t n) {
    const TokenOrderSizes s(n);
    for (const size_t k : {s.n, s.n, size_t{1}, s.spare, s.spare, s.counts}) l.add<uint32_t>(k);
}

inline TokenOrder take_token_order(Carve& c, int64_t n) {
    const TokenOrderSizes s(n);
    TokenOrder o;
    o.token = c.take<uint32_t>(s.n);
    o.position = c.take<uint32_t>(s.n);
    o.kept = c.take<uint32_t>(1);
    o.spare_token = c.take<uint32_t>(s.spare);
    o.spare_position = c.take<uint32_t>(s.spare);
    o.counts = c.take<uint32_t>(s.counts);
    return o;
}

// Writes `word`, whose halves are alike, to every word of `bytes` bytes (an even number) at `at`, aligned to 2.
int fill_words(void* at, size_t bytes, uint32_t word, hipStream_t stream);

// Sorts n >= 1 tokens and fills fill_bytes bytes at fill_at as fill_words, in the sort's launch where that is one.
int sort_tokens(const int64_t* tokens, int64_t n, int64_t vocabulary, const TokenOrder& order, void* fill_at, size_t fill_bytes,
                uint32_t fill, hipStream_t stream);

// sums over a token's rows: scale * sum of coefficient[position] * rows[position]
struct TokenSums {
    TokenOrder order;
    int64_t n, vocabulary, dim, stride;
    const void* rows;
    const float* coefficient;  // by position; NULL: 1
    float scale;
    float* part;  // token_sums_part_floats
    // either the table's rows, of the rows' type, ...
    void* table;
    bool accumulate;
    // ... or float32 rows by the index in the order of a token's first position, and that index by token
    float* sums;
    int32_t* first;
};

size_t token_sums_part_floats(int64_t n, int64_t dim);

int launch_token_sums(const TokenSums& a, int64_t dtype, hipStream_t stream);

}  // namespace dllm_hip
