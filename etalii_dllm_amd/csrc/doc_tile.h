// Matrix-core tiles of the document attention kernels.
//
// Every product is laid out so that a lane owns one column: a query (forward, dq) or a key (dk, dv). A wave's 32 x 32
// product X = A B takes A's rows from LDS and B's columns from registers, and leaves column lane % 32 of X in the lane, rows
//     row(r) = 8 (r / 4) + 4 (lane / 32) + r % 4,   r = 0 .. 15,
// with lane / 32 = half. What is computed from X (a softmax weight) is then the next product's B as it stands: the contraction
// index may run in any order as long as A's rows are read in the same one, so no value moves between lanes.
//
// LDS holds a tile row by row in 16-byte chunks (8 elements of 16 bits, 4 of 32), chunk c of row r at place c ^ swizzle(r):
// 16 rows' reads of one chunk, and the transposing reads' 4 rows of 4 chunks, fall on different banks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element.h"
#include "lds_copy.h"

namespace dllm_hip {

using Acc = float __attribute__((ext_vector_type(16)));

template <typename T>
struct MatrixType;
template <>
struct MatrixType<__bf16> {
    using Chunk = __bf16 __attribute__((ext_vector_type(8)));
};
template <>
struct MatrixType<_Float16> {
    using Chunk = _Float16 __attribute__((ext_vector_type(8)));
};
template <>
struct MatrixType<float> {
    using Chunk = float __attribute__((ext_vector_type(4)));
};
template <typename T>
using Chunk = typename MatrixType<T>::Chunk;

// acc += A B over the elements of two chunks (a lane's half of 2 kChunk<T> contraction steps)
__device__ __forceinline__ void multiply(const Chunk<__bf16>& a, const Chunk<__bf16>& b, Acc& acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void multiply(const Chunk<_Float16>& a, const Chunk<_Float16>& b, Acc& acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void multiply(const Chunk<float>& a, const Chunk<float>& b, Acc& acc) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
}

typedef __attribute__((address_space(3))) char LdsByte;

// A tile's geometry: kDim padded elements per row.
template <typename T, int kDim>
struct TileShape {
    static constexpr int kChunks = kDim * sizeof(T) / 16;  // 16-byte chunks of a row
    static constexpr int kRowBytes = kDim * sizeof(T);
    static constexpr int kSteps = kChunks / 2;             // chunk pairs: multiply() calls of a whole row

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (kChunks >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
};

// Copies kRows rows to LDS, kThreads chunks to a turn. The direct copy leaves no trace in registers: each wave's instruction fills 1 KB of LDS in lane
// order, and the lanes fetch the chunks that belong there. Rows past `valid` repeat the last one and chunks past head_dim the
// last one: what they are multiplied by is zero, or what they yield is not stored.
template <typename T, int kDim, int kRows, int kThreads, bool kDirect>
struct TileCopy {
    using Shape = TileShape<T, kDim>;
    static constexpr int kSlots = kRows * Shape::kChunks;
    static constexpr int kTurns = kSlots / kThreads;
    static constexpr int kTurnRows = kThreads / Shape::kChunks;
    static constexpr int kPeriod = kTurnRows >= 16 ? 1 : 16 / kTurnRows;  // turns after which the swizzle repeats
    static_assert(kSlots % kThreads == 0 && kThreads % Shape::kChunks == 0 && kTurns % kPeriod == 0);

    const char* head;  // row 0 of the array, at the head's first element
    int64_t stride;    // bytes between rows
    int last_chunk;
    int head_dim;
    uint32_t offset[kPeriod];  // of the lane's chunks from the first row of kPeriod turns: below 32 strides

    __device__ __forceinline__ TileCopy(const void* array, int64_t stride_elements, int head_index, int dim) {
        head = static_cast<const char*>(array) + static_cast<int64_t>(head_index) * dim * sizeof(T);
        stride = stride_elements * static_cast<int64_t>(sizeof(T));
        head_dim = dim;
        last_chunk = (dim * static_cast<int>(sizeof(T)) + 15) / 16 - 1;
#pragma unroll
        for (int e = 0; e < kPeriod; ++e) {
            const int row = e * kTurnRows + static_cast<int>(threadIdx.x) / Shape::kChunks;
            const int chunk = (static_cast<int>(threadIdx.x) % Shape::kChunks) ^ Shape::swizzle(row);
            offset[e] = static_cast<uint32_t>(row * stride) + min(chunk, last_chunk) * 16;
        }
    }

    __device__ __forceinline__ void operator()(int first, int valid, LdsByte* lds) const {
        const int wave = static_cast<int>(threadIdx.x) >> 6;
        const char* base = head + first * stride;
        if constexpr (kDirect) {
            const char* to = (const char*)lds + wave * 1024;
            if (valid >= kRows) {
#pragma unroll
                for (int t = 0; t < kTurns; ++t)
                    copy16_to_lds_s(base + (t / kPeriod) * (kPeriod * kTurnRows * stride), offset[t % kPeriod],
                                    to + t * (kThreads * 16));
            } else {
#pragma unroll
                for (int t = 0; t < kTurns; ++t) {
                    const int row = t * kTurnRows + static_cast<int>(threadIdx.x) / Shape::kChunks;
                    const int chunk = (static_cast<int>(threadIdx.x) % Shape::kChunks) ^ Shape::swizzle(row);
                    copy16_to_lds(base + min(row, valid - 1) * stride + min(chunk, last_chunk) * 16, to + t * (kThreads * 16));
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < kTurns; ++t) {
                const int slot = t * kThreads + static_cast<int>(threadIdx.x);
                const int row = slot / Shape::kChunks;
                const int chunk = (slot % Shape::kChunks) ^ Shape::swizzle(row);
                const T* src = reinterpret_cast<const T*>(base + min(row, valid - 1) * stride);
                Chunk<T> c;
#pragma unroll
                for (int j = 0; j < kChunk<T>; ++j) {
                    const int d = chunk * kChunk<T> + j;
                    c[j] = d < head_dim ? src[d] : static_cast<T>(0.0f);
                }
                *(__attribute__((address_space(3))) Chunk<T>*)(lds + slot * 16) = c;
            }
        }
    }
};

// This wave's copies have arrived and its LDS reads are done; then all waves' are.
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A lane's view of a tile in LDS.
template <typename T, int kDim>
struct TileView {
    using Shape = TileShape<T, kDim>;
    int rows_at;        // row lane % 32, chunk half: the A operand of products along head_dim
    int columns_at[2];  // the transposing reads' place in rows 0..7 and 8..15 of a group of 16

    __device__ __forceinline__ TileView() {
        const int lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5, row = lane & 31;
        rows_at = row * Shape::kRowBytes + ((half ^ Shape::swizzle(row)) << 4);
        if constexpr (sizeof(T) == 2) {
            // 16 lanes read 4 rows of 16 columns and get a column each: rows 8 t + 4 half + 0 .. 3, columns 16 ((lane / 16) % 2)
            const int i = lane & 15;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int r = 8 * t + 4 * half + (i >> 2);
                const int chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                columns_at[t] = r * Shape::kRowBytes + ((chunk ^ Shape::swizzle(r)) << 4) + (i & 1) * 8;
            }
        } else {
            const int r = 4 * half, column = lane & 31;
            columns_at[0] = r * Shape::kRowBytes;
            columns_at[1] = column;
        }
    }

    // chunk pair `step` of rows 32 block ..
    __device__ __forceinline__ Chunk<T> rows(const LdsByte* tile, int block, int step) const {
        return *(const __attribute__((address_space(3))) Chunk<T>*)(tile + ((rows_at ^ (step << 5)) + block * 32 * Shape::kRowBytes));
    }
};

// acc += (tile's rows, 32 of them from 32 block, as columns 32 part ..)^T x: x is a product's 16 rows as they stand in a lane.
template <typename T, int kDim, int kParts>
__device__ __forceinline__ void multiply_columns(const TileView<T, kDim>& view, const LdsByte* tile, int block,
                                                 const float (&x)[16], Acc (&acc)[kParts]) {
    using Shape = TileShape<T, kDim>;
    if constexpr (sizeof(T) == 2) {
        using Half = short __attribute__((ext_vector_type(4)));
        union Both {
            Half h[2];
            Chunk<T> c;
        };
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // 16 rows at a time
            Chunk<T> b;
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = static_cast<T>(x[8 * c + j]);
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                Both a;
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    a.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) Half*)(tile + ((view.columns_at[t] ^ (p << 6)) +
                                                                          (32 * block + 16 * c) * Shape::kRowBytes)));
                multiply(a.c, b, acc[p]);
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = 32 * block + 8 * (r / 4) + r % 4;  // + 4 half
            const int sw = Shape::swizzle(8 * (r / 4) + r % 4);
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                const int half = (static_cast<int>(threadIdx.x) >> 5) & 1;
                const int column = 32 * p + view.columns_at[1];
                const int chunk = (column >> 2) ^ (sw ^ half);  // bit 2 of the row is the swizzle's lowest
                const float a = *(const __attribute__((address_space(3))) float*)(tile + (row * Shape::kRowBytes + view.columns_at[0] +
                                                                                          (chunk << 4) + (column & 3) * 4));
                acc[p] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[r], acc[p], 0, 0, 0);
            }
        }
    }
}

// A lane's own row, the B operand of products along head_dim: chunk pair `step`'s chunk of its half, zero past head_dim. Held
// in registers, or read again at each use where it would take more than 64 of them (a step's four float32 products take 256
// cycles, and the row stays in the caches).
template <typename T, int kDim, bool kDirect>
struct Column {
    static constexpr int kSteps = TileShape<T, kDim>::kSteps;
    static constexpr bool kHeld = sizeof(T) == 2 || kSteps <= 8;
    const T* row;
    int head_dim;
    Chunk<T> held[kHeld ? kSteps : 1];

    __device__ __forceinline__ Chunk<T> read(int step) const {
        const int d = (2 * step + ((static_cast<int>(threadIdx.x) >> 5) & 1)) * kChunk<T>;
        Chunk<T> c{};
        if constexpr (kDirect) {
            if (d < head_dim) c = *reinterpret_cast<const Chunk<T>*>(row + d);
        } else {
#pragma unroll
            for (int j = 0; j < kChunk<T>; ++j)
                if (d + j < head_dim) c[j] = row[d + j];
        }
        return c;
    }
    __device__ __forceinline__ Column(const T* from, int dim) : row(from), head_dim(dim) {
        if constexpr (kHeld)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) held[s] = read(s);
    }
    __device__ __forceinline__ Chunk<T> operator[](int step) const {
        if constexpr (kHeld) return held[step];
        return read(step);
    }
};

// The other half's value for the same column.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// Column values 32 p + 8 g + 4 half + 0 .. 3 of a lane, times factor, to its row.
template <bool kDirect, typename T, int kParts>
__device__ __forceinline__ void store_column(T* row, int head_dim, const Acc (&acc)[kParts], float factor) {
    const int half = (static_cast<int>(threadIdx.x) >> 5) & 1;
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * p + 8 * g + 4 * half;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = acc[p][4 * g + r] * factor;
            if constexpr (kDirect) {
                if (d < head_dim) store_from_float<T, 4>(row + d, v);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (d + r < head_dim) row[d + r] = static_cast<T>(v[r]);
            }
        }
}

// Whether every value is finite (a sum of products by zero is NaN otherwise).
template <int kParts>
__device__ __forceinline__ bool all_finite(const Acc (&acc)[kParts]) {
    float z = 0.0f;
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int r = 0; r < 16; ++r) z = fmaf(acc[p][r], 0.0f, z);
    return z == 0.0f;
}

}  // namespace dllm_hip
