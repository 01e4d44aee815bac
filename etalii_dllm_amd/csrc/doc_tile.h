// Matrix-core tiles of the document attention kernels.
//
// Every product is laid out so that a lane owns one column: a query (forward, dq) or a key (dk, dv). A wave's 32 x 32
// product X = A B takes A's rows from LDS and B's columns from registers, and leaves column lane % 32 of X in the lane, rows
//     row(r) = 8 (r / 4) + 4 (lane / 32) + r % 4,   r = 0 .. 15,
// with lane / 32 = half. What is computed from X (a softmax weight) is then the next product's B as it stands: the contraction
// index may run in any order as long as A's rows are read in the same one, so no value moves between lanes.
//
// float32 is multiplied as bfloat16: x = h + m + l with h, m and l the roundings of x, x - h and x - h - m, 8 bits each, which
// is x to its last bits. Of the nine products of two such sums the six of order h h, h m, m m and h l are formed (those left
// out are 2^-24 of the product), each exactly, and added in float32: float32's accuracy at 6/16 of the float32 matrix
// instructions' time. The arrays are split once, into three planes, before the kernels that read their rows many times.
//
// LDS holds a tile row by row in 16-byte chunks of 8 elements, chunk c of row r at place c ^ swizzle(r): 16 rows' reads of
// one chunk, and the transposing reads' 4 rows of 4 chunks, fall on different banks (measured: no conflicts).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "element.h"
#include "lds_copy.h"

namespace dllm_hip {

using Acc = float __attribute__((ext_vector_type(16)));

// What an activation type is multiplied as.
template <typename T>
struct Product {
    using Part = T;
    static constexpr int kPlanes = 1;
};
template <>
struct Product<float> {
    using Part = __bf16;
    static constexpr int kPlanes = 3;
};
template <typename T>
using Part = typename Product<T>::Part;
template <typename T>
constexpr int kPlanes = Product<T>::kPlanes;

using Chunk16 = short __attribute__((ext_vector_type(8)));  // 8 elements of either 16-bit type
constexpr int kPartChunk = 8;

template <typename P>
__device__ __forceinline__ void multiply(const Chunk16& a, const Chunk16& b, Acc& acc) {
    using V = P __attribute__((ext_vector_type(8)));
    if constexpr (__is_same(P, __bf16))
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), acc, 0, 0, 0);
    else
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), acc, 0, 0, 0);
}

// A value's chunk in each plane.
template <typename T>
struct Chunks {
    Chunk16 c[kPlanes<T>];
};

// acc += a b, the small products first.
template <typename T>
__device__ __forceinline__ void multiply(const Chunks<T>& a, const Chunks<T>& b, Acc& acc) {
    if constexpr (kPlanes<T> == 3) {
        multiply<Part<T>>(a.c[2], b.c[0], acc);
        multiply<Part<T>>(a.c[0], b.c[2], acc);
        multiply<Part<T>>(a.c[1], b.c[1], acc);
        multiply<Part<T>>(a.c[1], b.c[0], acc);
        multiply<Part<T>>(a.c[0], b.c[1], acc);
    }
    multiply<Part<T>>(a.c[0], b.c[0], acc);
}

// x's parts, kPlanes of them.
template <typename T>
__device__ __forceinline__ void split(float x, Part<T> (&out)[kPlanes<T>]) {
#pragma unroll
    for (int p = 0; p < kPlanes<T>; ++p) {
        out[p] = static_cast<Part<T>>(x);
        x -= static_cast<float>(out[p]);
    }
}

typedef __attribute__((address_space(3))) char LdsByte;

// An array [tokens, heads, head_dim] as the kernels read it: 16-bit elements, whole 16-byte chunks (`chunks` of them hold a
// head; zeroes fill the last), in kPlanes planes. Byte strides.
struct Source {
    const char* base;
    int64_t stride, head, plane;
    int chunks;
};

// A tile's geometry: kDim padded elements per row.
template <typename T, int kDim>
struct TileShape {
    static constexpr int kRowBytes = kDim * 2;
    static constexpr int kChunks = kRowBytes / 16;  // of a row
    static constexpr int kSteps = kChunks / 2;      // chunk pairs: multiply() calls of a whole row

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (kChunks >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
};

// Copies kRows rows (of each plane, one plane after another) to LDS, kThreads chunks to a turn, without a trace in registers:
// each wave's instruction fills 1 KB of LDS in lane order, and the lanes fetch the chunks that belong there. Rows past
// `valid` repeat the last one and chunks past the head the last one: what they are multiplied by is zero, or what they
// yield is not stored.
template <typename T, int kDim, int kRows, int kThreads>
struct TileCopy {
    using Shape = TileShape<T, kDim>;
    static constexpr int kPlaneBytes = kRows * Shape::kRowBytes;
    static constexpr int kBytes = kPlanes<T> * kPlaneBytes;
    static constexpr int kTurns = kRows * Shape::kChunks / kThreads;
    static constexpr int kTurnRows = kThreads / Shape::kChunks;
    static constexpr int kPeriod = kTurnRows >= 16 ? 1 : 16 / kTurnRows;  // turns after which the swizzle repeats
    static_assert(kRows * Shape::kChunks % kThreads == 0 && kThreads % Shape::kChunks == 0 && kTurns % kPeriod == 0);

    const char* head;  // row 0 of the array, at the head's first element
    int64_t stride, plane;
    int last_chunk;
    uint32_t offset[kPeriod];  // of the lane's chunks from the first row of kPeriod turns: below 32 strides

    __device__ __forceinline__ TileCopy(const Source& s, int head_index) {
        head = s.base + head_index * s.head;
        stride = s.stride;
        plane = s.plane;
        last_chunk = s.chunks - 1;
#pragma unroll
        for (int e = 0; e < kPeriod; ++e) {
            const int row = e * kTurnRows + static_cast<int>(threadIdx.x) / Shape::kChunks;
            const int chunk = (static_cast<int>(threadIdx.x) % Shape::kChunks) ^ Shape::swizzle(row);
            offset[e] = static_cast<uint32_t>(row * stride) + min(chunk, last_chunk) * 16;
        }
    }

    __device__ __forceinline__ void operator()(int first, int valid, LdsByte* lds) const {
        const char* to = (const char*)lds + (static_cast<int>(threadIdx.x) >> 6) * 1024;
#pragma unroll
        for (int p = 0; p < kPlanes<T>; ++p) {
            const char* base = head + first * stride + p * plane;
            if (valid >= kRows) {
#pragma unroll
                for (int t = 0; t < kTurns; ++t)
                    copy16_to_lds_s(base + (t / kPeriod) * (kPeriod * kTurnRows * stride), offset[t % kPeriod],
                                    to + p * kPlaneBytes + t * (kThreads * 16));
            } else {
#pragma unroll
                for (int t = 0; t < kTurns; ++t) {
                    const int row = t * kTurnRows + static_cast<int>(threadIdx.x) / Shape::kChunks;
                    const int chunk = (static_cast<int>(threadIdx.x) % Shape::kChunks) ^ Shape::swizzle(row);
                    copy16_to_lds(base + min(row, valid - 1) * stride + min(chunk, last_chunk) * 16,
                                  to + p * kPlaneBytes + t * (kThreads * 16));
                }
            }
        }
    }
};

// This wave's copies have arrived and its LDS reads are done; then all waves' are.
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A lane's view of a tile of kRows rows in LDS.
template <typename T, int kDim, int kRows>
struct TileView {
    using Shape = TileShape<T, kDim>;
    static constexpr int kPlaneBytes = kRows * Shape::kRowBytes;
    int rows_at;        // row lane % 32, chunk half: the A operand of products along head_dim
    int columns_at[2];  // the transposing reads' place in rows 0..7 and 8..15 of a group of 16

    __device__ __forceinline__ TileView() {
        const int lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5, row = lane & 31;
        rows_at = row * Shape::kRowBytes + ((half ^ Shape::swizzle(row)) << 4);
        // 16 lanes read 4 rows of 16 columns and get a column each: rows 8 t + 4 half + 0 .. 3, columns 16 ((lane / 16) % 2)
        const int i = lane & 15;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = 8 * t + 4 * half + (i >> 2);
            const int chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
            columns_at[t] = r * Shape::kRowBytes + ((chunk ^ Shape::swizzle(r)) << 4) + (i & 1) * 8;
        }
    }

    // chunk pair `step` of rows 32 block ..
    __device__ __forceinline__ Chunks<T> rows(const LdsByte* tile, int block, int step) const {
        Chunks<T> a;
#pragma unroll
        for (int p = 0; p < kPlanes<T>; ++p)
            a.c[p] = *(const __attribute__((address_space(3))) Chunk16*)(tile + ((rows_at ^ (step << 5)) + block * 32 * Shape::kRowBytes +
                                                                                 p * kPlaneBytes));
        return a;
    }

    // rows 32 block + 16 group .. as columns 32 part ..
    __device__ __forceinline__ Chunks<T> columns(const LdsByte* tile, int block, int group, int part) const {
        using Half = short __attribute__((ext_vector_type(4)));
        union Both {
            Half h[2];
            Chunk16 c;
        };
        Chunks<T> a;
#pragma unroll
        for (int p = 0; p < kPlanes<T>; ++p) {
            Both both;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                both.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) Half*)(tile + ((columns_at[t] ^ (part << 6)) +
                                                                      (32 * block + 16 * group) * Shape::kRowBytes + p * kPlaneBytes)));
            a.c[p] = both.c;
        }
        return a;
    }
};

// A product's 16 rows as they stand in a lane, as the B operand of the next.
template <typename T>
struct Rows16 {
    Chunks<T> group[2];
    __device__ __forceinline__ explicit Rows16(const float (&x)[16]) {
        using V = Part<T> __attribute__((ext_vector_type(8)));
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            V v[kPlanes<T>];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                Part<T> parts[kPlanes<T>];
                split<T>(x[8 * g + j], parts);
#pragma unroll
                for (int p = 0; p < kPlanes<T>; ++p) v[p][j] = parts[p];
            }
#pragma unroll
            for (int p = 0; p < kPlanes<T>; ++p) group[g].c[p] = __builtin_bit_cast(Chunk16, v[p]);
        }
    }
};

// What the type's rounding leaves of each value.
template <typename T>
__device__ __forceinline__ void keep_rest(float (&x)[16]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] -= static_cast<float>(static_cast<Part<T>>(x[r]));
}

// kSteps products, each of kReads LDS reads that are begun some steps before their use. Left alone the compiler reads an operand,
// waits for it and multiplies, which leaves the matrix cores idle for the LDS's latency every time.
//
// One wave on a SIMD (float32, heads of 256) has no other to fill such waits: the order is held by scheduling barriers that reads
// and products do not cross. More waves do better where the compiler is only asked for an order (microseconds, asked and held:
// 4096 float32 tokens of 16/8 heads of 128, gradients 1306 and 1228; 8192 bfloat16 tokens of 8/4 heads of 256, 1400 and
// 1222; of 16/8 heads of 128, 1154 and 1188; of 64, forward, 175 to 183 both).
template <typename T, int kDim>
constexpr bool kOrderHeld = kPlanes<T> == 3 || kDim > 128;
template <typename T, int kDim>
constexpr int kAheadSteps = kPlanes<T> == 3 ? 1 : 2;  // measured: one more, two more and four more are no faster, and take registers
template <typename T, int kDim, int kSteps, int kReads, typename Read, typename Multiply>
__device__ __forceinline__ void multiply_steps(Read&& read, Multiply&& multiply_step) {
    constexpr int kAhead = kAheadSteps<T, kDim>;
    if constexpr (kOrderHeld<T, kDim>) {
        constexpr int kMayCross = 0x2 | 0x4 | 0x400;  // vector, scalar and transcendental arithmetic
        decltype(read(0)) held[kAhead + 1];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) held[i] = read(i);
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            if (step + kAhead < kSteps) held[(step + kAhead) % (kAhead + 1)] = read(step + kAhead);
            __builtin_amdgcn_sched_barrier(kMayCross);
            multiply_step(step, held[step % (kAhead + 1)]);
            __builtin_amdgcn_sched_barrier(kMayCross);
        }
    } else {
#pragma unroll
        for (int step = 0; step < kSteps; ++step) multiply_step(step, read(step));
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead * kReads, 0);  // LDS reads, ...
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // ... a product, and the reads of a later one
            __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
        }
    }
}

// acc += (tile's rows, 32 of them from 32 block, as columns 32 (first + 0 .. kParts - 1) ..)^T x
template <typename T, int kDim, int kRows, int kParts>
__device__ __forceinline__ void multiply_columns(const TileView<T, kDim, kRows>& view, const LdsByte* tile, int block,
                                                 const Rows16<T>& x, int first, Acc (&acc)[kParts]) {
    multiply_steps<T, kDim, 2 * kParts, 2>(
        [&](int s) { return view.columns(tile, block, s / kParts, kParts * 32 == kDim ? s % kParts : first + s % kParts); },
        [&](int s, const Chunks<T>& a) { multiply<T>(a, x.group[s / kParts], acc[s % kParts]); });
}

// Wide float32 heads: a lane's rows and sums in three planes are more than the registers, so a pair of waves shares 32 rows
// and takes half of the head's dimensions each. Both then need the sums over all of them: see exchange(). (4096 tokens, 4/2
// heads of 256: forward 675 to 512 us, gradients 5.3 to 1.44 ms. Heads of 128 fit a wave, and sharing costs them more than it
// gives: 16/8 of them 430 to 655 us.)
template <typename T, int kDim>
constexpr int kPair = kPlanes<T> * kDim > 384 ? 2 : 1;
template <typename T, int kDim>
constexpr int kWaveDim = kDim / kPair<T, kDim>;
template <typename T, int kDim>
constexpr int kBlockRows = 128 / kPair<T, kDim>;  // of a workgroup's own, 32 for each wave or pair

// A lane's own row, the B operand of products along head_dim: each chunk pair's chunk of its half, zero past the head; of a
// wave's part of the dimensions.
template <typename T, int kDim>
struct Column {
    static constexpr int kSteps = kWaveDim<T, kDim> / 16;
    Chunks<T> held[kSteps];
    __device__ __forceinline__ Column(const Source& s, int head, int64_t token, int part) {
        const char* const row = s.base + token * s.stride + head * s.head;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int chunk = 2 * (i + part * kSteps) + ((static_cast<int>(threadIdx.x) >> 5) & 1);
#pragma unroll
            for (int p = 0; p < kPlanes<T>; ++p) {
                held[i].c[p] = Chunk16{};
                if (chunk < s.chunks) held[i].c[p] = *reinterpret_cast<const Chunk16*>(row + p * s.plane + chunk * 16);
            }
        }
    }
};

// acc += (rows 32 block .. of a tile) column, over the wave's part of the dimensions
template <typename T, int kDim, int kRows>
__device__ __forceinline__ void multiply_rows(const TileView<T, kDim, kRows>& view, const LdsByte* tile, int block,
                                              const Column<T, kDim>& column, int part, Acc& acc) {
    constexpr int kSteps = Column<T, kDim>::kSteps;
    multiply_steps<T, kDim, kSteps, 1>(
        [&](int s) { return view.rows(tile, block, kPair<T, kDim> == 1 ? s : s + part * kSteps); },
        [&](int s, const Chunks<T>& a) { multiply<T>(a, column.held[s], acc); });
}

// The pair's sums: each wave leaves its own in LDS (4 KB for each 32 x 32), and after the barrier adds the other's. All waves
// of the workgroup come here. area: kCount * 4 KB for each wave; the next exchange comes after another barrier.
template <int kCount>
__device__ __forceinline__ void exchange(Acc* const (&x)[kCount], LdsByte* area) {
    using Four = float __attribute__((ext_vector_type(4)));
    using LdsFour = __attribute__((address_space(3))) Four;
    const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
    LdsFour* const mine = (LdsFour*)(area + wave * kCount * 4096) + lane;
    LdsFour* const other = (LdsFour*)(area + (wave ^ 1) * kCount * 4096) + lane;
#pragma unroll
    for (int c = 0; c < kCount; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) mine[(4 * c + g) * 64] = Four{(*x[c])[4 * g], (*x[c])[4 * g + 1], (*x[c])[4 * g + 2], (*x[c])[4 * g + 3]};
    lds_barrier();
#pragma unroll
    for (int c = 0; c < kCount; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const Four v = other[(4 * c + g) * 64];
#pragma unroll
            for (int r = 0; r < 4; ++r) (*x[c])[4 * g + r] += v[r];
        }
}

// Which of a wave's rows either wave of the pair has marked. All waves of the workgroup come here.
__device__ __forceinline__ uint32_t pair_marks(uint32_t marks, LdsByte* area) {
    using LdsWord = __attribute__((address_space(3))) uint32_t;
    LdsWord* const words = (LdsWord*)area;
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) words[wave] = marks;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(words[wave & ~1] | words[wave | 1]);
}

// The other half's value for the same column.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// Column values 32 (first + p) + 8 g + 4 half + 0 .. 3 of a lane, times factor, to its row; whole: rows of whole groups of
// four, aligned to them.
template <typename T, int kParts>
__device__ __forceinline__ void store_column(T* row, int head_dim, bool whole, int first, const Acc (&acc)[kParts], float factor) {
    const int half = (static_cast<int>(threadIdx.x) >> 5) & 1;
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * (first + p) + 8 * g + 4 * half;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = acc[p][4 * g + r] * factor;
            if (whole) {
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
