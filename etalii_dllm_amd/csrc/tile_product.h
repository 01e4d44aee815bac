// Tiled products on the matrix cores: C[m][n] = sum over k of A[m][k] B[n][k], float32 sums, with an epilogue of the
// caller's on the tile in registers.
//
// Either operand lies in memory with k along its rows (kRows) or across them (kColumns: k is the row, m or n the column).
// Tiles of 64 k go through LDS in kStages buffers, copied without registers in 16-byte chunks; chunk c of LDS row r lies at place
// c ^ swizzle(r), so that neither the row reads nor the transposing reads of kColumns tiles (4 rows of 16 columns by 16
// lanes) meet on a bank. A wave holds a kWaveM x kWaveN part of the tile as blocks of 32 x 32.
//
// kPlanes 2: a value is a pair of 16-bit parts, multiplied as three products (second by first, first by second, first by first).
// A row holds 32 values' first parts, then their second parts, and so on, so a tile of 32 k has the bytes, lines and LDS places of
// one of 64 single values. (In planes of their own, multiplied pair after pair, the parts were read three times for two.)
//
// P float: values as they are, 32 k to a tile, only along the rows, on the float32 matrix instructions: a sixteenth of the 16-bit
// ones' rate, for products that wait for their operands.
//
// Measured, plain products of random bfloat16 values, 8192 x 8192: 1040 TFLOP/s over 1536 k and 1070 to 1230 over 8192 (256 x 256
// tiles), 1020 and 1120 (128 x 128, two workgroups to a CU); a library product reaches 1148. The matrix cores are busy 60% of
// the time at 1.86 GHz, to which power lowers the clock. Reading a step's operands ahead of the products before it, also over the
// stages' barrier, gave nothing; shorter stages (32 k), three and four of them, are slower where rows of 64 bytes are
// read, and wave priorities did not matter.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "doc_tile.h"

namespace dllm_hip {

// Bytes; base and strides are multiples of 16. kRows: m or n rows of k values. kColumns: k rows of m or n values, each readable up to
// the next whole chunk. `count`: how many m or n there are; indexes past it repeat others, what they yield is not
// stored.
struct Operand {
    const char* base;
    int64_t stride, batch;
    int64_t count;
};

static __device__ const uint4 kZeroChunk = {0, 0, 0, 0};

// Where value c of a row begins, in bytes; a pair's second part is kSecond bytes further. kBytes: of a part.
template <int kPlanes, int kBytes = 2>
__host__ __device__ __forceinline__ int64_t value_at(int64_t c) {
    return kPlanes == 1 ? c * kBytes : (c >> 5) * 128 + (c & 31) * 2;
}
constexpr int kSecond = 64;
// Values of a row that are there: whole chunks, or whole groups of pairs.
template <int kPlanes>
constexpr int kRowMultiple = kPlanes == 1 ? 8 : 32;

// 8 values, from one that is a multiple of 8 in its row on, as parts of type P. (A pair of an infinity is that and NaN, so products are NaN.)
template <typename P, int kPlanes>
__device__ __forceinline__ void store_eight(char* to, const float (&v)[8]) {
    using V = P __attribute__((ext_vector_type(8)));
    float left[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) left[e] = v[e];
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
        V part;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            part[e] = static_cast<P>(left[e]);
            left[e] -= static_cast<float>(part[e]);
        }
        *reinterpret_cast<V*>(to + p * kSecond) = part;
    }
}

template <int kChunks>
__device__ __forceinline__ int tile_swizzle(int row) {
    if constexpr (kChunks >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// One operand's tile of kSize m or n: its copy to LDS.
template <int kSize, int kPlanes, int kPartBytes, int kThreads, bool kColumns>
struct OperandTile {
    static constexpr int kTileK = 128 / (kPlanes * kPartBytes);
    static constexpr int kChunks = kColumns ? kSize * kPlanes / 8 : 8;  // of an LDS row
    static constexpr int kRows = kColumns ? kTileK : kSize;
    static constexpr int kBytes = kRows * kChunks * 16;
    static constexpr int kTurns = kRows * kChunks / kThreads;
    static constexpr int kTurnRows = kThreads / kChunks;
    static_assert(kRows * kChunks % kThreads == 0 && kThreads % kChunks == 0 && (kPartBytes == 2 || !kColumns));

    const char* base;  // of the tile's first m or n
    int64_t stride;
    uint32_t offset[kTurns];  // of the lane's chunk of each turn

    __device__ __forceinline__ static int lds_row(int turn) { return turn * kTurnRows + static_cast<int>(threadIdx.x) / kChunks; }
    __device__ __forceinline__ static int chunk(int turn) {
        return (static_cast<int>(threadIdx.x) % kChunks) ^ tile_swizzle<kChunks>(lds_row(turn));
    }
    // the first value of a chunk
    __device__ __forceinline__ static int value_of(int c) { return kPlanes == 1 ? c * (16 / kPartBytes) : c / 8 * 32 + (c & 3) * 8; }

    __device__ __forceinline__ void init(const Operand& op, int64_t first, int64_t count, int64_t batch) {
        stride = op.stride;
        const int64_t left = count - first;  // at least 1
        base = op.base + batch * op.batch + (kColumns ? value_at<kPlanes>(first) : first * stride);
#pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const int64_t row = lds_row(t);
            int c = chunk(t);
            if constexpr (kColumns) {
                if (value_of(c) >= left) c = kPlanes == 1 ? static_cast<int>((left - 1) / 8) : static_cast<int>((left - 1) / 32 * 8) + (c & 4);
                offset[t] = static_cast<uint32_t>(row * stride + c * 16);
            } else {
                offset[t] = static_cast<uint32_t>(min(row, left - 1) * stride + c * 16);
            }
        }
    }

    // The tile from k0 on to LDS; k at and past `k` are zero.
    __device__ __forceinline__ void copy(int64_t k0, int64_t k, LdsByte* lds) const {
        const char* to = (const char*)lds + (static_cast<int>(threadIdx.x) >> 6) * 1024;
        const char* from = base + (kColumns ? k0 * stride : value_at<kPlanes, kPartBytes>(k0));
        if (k0 + kTileK <= k) {
#pragma unroll
            for (int t = 0; t < kTurns; ++t) copy16_to_lds_s(from, offset[t], to + t * (kThreads * 16));
        } else {
#pragma unroll
            for (int t = 0; t < kTurns; ++t) {
                const bool inside = kColumns ? k0 + lds_row(t) < k : k0 + value_of(chunk(t)) < k;
                const char* src = inside ? from + offset[t] : reinterpret_cast<const char*>(&kZeroChunk);
                copy16_to_lds(src, to + t * (kThreads * 16));
            }
        }
    }
};

// A lane's reads of blocks of 32 m or n by 16 k (8 of float32) from a tile.
template <int kSize, int kPlanes, bool kColumns>
struct OperandView {
    static constexpr int kChunks = kColumns ? kSize * kPlanes / 8 : 8;
    static constexpr int kRowBytes = kChunks * 16;
    int at[2];

    __device__ __forceinline__ explicit OperandView(int first) {
        const int lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5;
        if constexpr (!kColumns) {
            const int row = lane & 31;
            at[0] = (first + row) * kRowBytes + ((half ^ tile_swizzle<kChunks>(row)) << 4);
            at[1] = 0;
        } else {
            // 16 lanes read 4 rows of 16 columns and get a column each: k 8 half + 4 t + 0 .. 3, columns 16 ((lane / 16) % 2) ..
            const int i = lane & 15;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int r = 8 * half + 4 * t + (i >> 2);
                const int chunk = first / 32 * (4 * kPlanes) + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                at[t] = r * kRowBytes + ((chunk ^ tile_swizzle<kChunks>(r)) << 4) + (i & 1) * 8;
            }
        }
    }

    // (the places that step, block and plane change are whole bits of the chunk's number)
    __device__ __forceinline__ Chunk16 read(const LdsByte* tile, int block, int step, int plane) const {
        if constexpr (!kColumns) {
            return *(const __attribute__((address_space(3))) Chunk16*)(tile + ((at[0] ^ (step << 5) ^ (plane << 6)) + block * 32 * kRowBytes));
        } else {
            using Half = short __attribute__((ext_vector_type(4)));
            union Both {
                Half h[2];
                Chunk16 c;
            } both;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                both.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) Half*)(tile + ((at[t] ^ (block << (5 + kPlanes)) ^ (plane << 6)) + step * 16 * kRowBytes)));
            return both.c;
        }
    }
};

// All but kCount of this wave's copies have arrived, and its LDS reads are done; then all waves' are.
template <int kCount>
__device__ __forceinline__ void stage_barrier() {
    static_assert(kCount < 64);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kCount) : "memory");
}

// acc += x y: 16 k of a 16-bit type, 8 of float32, of which each instruction takes one of either half's chunk.
template <typename P>
__device__ __forceinline__ void multiply_chunks(const Chunk16& x, const Chunk16& y, Acc& acc) {
    if constexpr (sizeof(P) == 4) {
        using Four = float __attribute__((ext_vector_type(4)));
        const Four a = __builtin_bit_cast(Four, x), b = __builtin_bit_cast(Four, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
    } else {
        multiply<P>(x, y, acc);
    }
}

// A tile of kM x kN by kWavesM x kWavesN waves, with kStages buffers.
template <typename P, int kPlanesOf, int kM_, int kN_, int kWavesM_, int kWavesN_, bool kAColumns, bool kBColumns, int kStages = 2>
struct TileProduct {
    static constexpr int kM = kM_, kN = kN_, kWavesM = kWavesM_, kWavesN = kWavesN_;
    static constexpr int kThreads = kWavesM * kWavesN * kWave;
    static constexpr int kWaveM = kM / kWavesM, kWaveN = kN / kWavesN;
    static constexpr int kBlocksM = kWaveM / 32, kBlocksN = kWaveN / 32;
    static constexpr int kTileK = 128 / (kPlanesOf * static_cast<int>(sizeof(P)));
    static_assert(kPlanesOf == 1 || (kPlanesOf == 2 && sizeof(P) == 2));
    using Part = P;
    using ATile = OperandTile<kM, kPlanesOf, sizeof(P), kThreads, kAColumns>;
    using BTile = OperandTile<kN, kPlanesOf, sizeof(P), kThreads, kBColumns>;
    static constexpr int kStage = ATile::kBytes + BTile::kBytes;
    static constexpr int kLds = kStages * kStage;
    static constexpr int kCopies = ATile::kTurns + BTile::kTurns;  // of a thread, for one stage
    using Sums = Acc[kBlocksM][kBlocksN];

    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6); }
    static __device__ __forceinline__ int wave_m() { return wave() / kWavesN * kWaveM; }
    static __device__ __forceinline__ int wave_n() { return wave() % kWavesN * kWaveN; }

    // acc = the tile at (m0, n0); all of m0 < a_count, n0 < b_count. LDS: kLds bytes. kSegments: k is summed in segments of `segment`
    // (a multiple of kTileK), each from zero, which are added in order.
    template <bool kSegments = false>
    static __device__ __forceinline__ void run(const Operand& a, const Operand& b, int64_t m0, int64_t n0, int64_t a_count, int64_t b_count,
                                               int64_t k, int64_t batch_a, int64_t batch_b, LdsByte* lds, Sums& acc, int64_t segment = 0) {
        ATile at;
        BTile bt;
        at.init(a, m0, a_count, batch_a);
        bt.init(b, n0, b_count, batch_b);
        const OperandView<kM, kPlanesOf, kAColumns> av(wave_m());
        const OperandView<kN, kPlanesOf, kBColumns> bv(wave_n());
        const auto clear = [&] {
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i)
#pragma unroll
                for (int j = 0; j < kBlocksN; ++j) acc[i][j] = Acc{};
        };
        clear();
        const int count = static_cast<int>((k + kTileK - 1) / kTileK);
        if (count == 0) return;
        int tile = 0, into = 0;  // of the next copy
        auto copy = [&] {
            LdsByte* const to = lds + into * kStage;
            at.copy(static_cast<int64_t>(tile) * kTileK, k, to);
            bt.copy(static_cast<int64_t>(tile) * kTileK, k, to + ATile::kBytes);
            ++tile;
            into = into + 1 == kStages ? 0 : into + 1;
        };
        for (int i = 0; i < kStages - 1 && i < count; ++i) copy();
        const int segment_tiles = kSegments ? static_cast<int>(segment / kTileK) : count;
        int from = 0, boundary = segment_tiles;
        Sums total;
        if constexpr (kSegments) {
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i)
#pragma unroll
                for (int j = 0; j < kBlocksN; ++j) total[i][j] = Acc{};
        }
        for (int i = 0; i < count; ++i) {
            // stage i has arrived, and the one that the next copy goes to is read
            if (kStages > 2 && i + kStages - 2 < count)
                stage_barrier<(kStages - 2) * kCopies>();
            else
                stage_barrier<0>();
            if (i + kStages - 1 < count) copy();
            if (kSegments && i == boundary) {
                boundary += segment_tiles;
#pragma unroll
                for (int m = 0; m < kBlocksM; ++m)
#pragma unroll
                    for (int n = 0; n < kBlocksN; ++n) total[m][n] += acc[m][n];
                clear();
            }
            const LdsByte* const stage = lds + from * kStage;
            from = from + 1 == kStages ? 0 : from + 1;
#pragma unroll
            for (int step = 0; step < 4 / kPlanesOf; ++step) {
                Chunk16 x[kPlanesOf][kBlocksM], y[kPlanesOf][kBlocksN];
#pragma unroll
                for (int p = 0; p < kPlanesOf; ++p) {
#pragma unroll
                    for (int m = 0; m < kBlocksM; ++m) x[p][m] = av.read(stage, m, step, p);
#pragma unroll
                    for (int n = 0; n < kBlocksN; ++n) y[p][n] = bv.read(stage + ATile::kBytes, n, step, p);
                }
#pragma unroll
                for (int product = kPlanesOf == 1 ? 2 : 0; product < 3; ++product)
#pragma unroll
                    for (int m = 0; m < kBlocksM; ++m)
#pragma unroll
                        for (int n = 0; n < kBlocksN; ++n) multiply_chunks<P>(x[product == 0][m], y[product == 1][n], acc[m][n]);
            }
        }
        if constexpr (kSegments) {
#pragma unroll
            for (int m = 0; m < kBlocksM; ++m)
#pragma unroll
                for (int n = 0; n < kBlocksN; ++n) acc[m][n] = total[m][n] + acc[m][n];
        }
    }
};

__device__ __forceinline__ int lane_half() { return (static_cast<int>(threadIdx.x) >> 5) & 1; }
__device__ __forceinline__ int lane_column() { return static_cast<int>(threadIdx.x) & 31; }

// Row of a 32 x 32 block that a lane holds in element r; its column is lane % 32.
__device__ __forceinline__ int block_row(int r) { return 8 * (r >> 2) + 4 * lane_half() + (r & 3); }

// A wave's sums by rows: f(row, column, v) with 8 consecutive columns' sums in each lane (row and column within the wave's part), for
// wide stores. The blocks go through LDS, 32 rows at a time; its 16-byte chunks lie at places that keep both ways free of
// conflicts on the 64 banks. What f reads from memory is read by load(row, column), for a block at once and ahead of its way
// through LDS, and handed to f. With columns, what f leaves in v goes by columns to g(row, column, v) with 8 consecutive rows of
// one column.
template <typename Tile, typename L, typename F, typename G>
__device__ __forceinline__ void by_rows_and_columns(const typename Tile::Sums& acc, LdsByte* lds, bool columns, L&& load, F&& f, G&& g) {
    constexpr int kColumns = Tile::kWaveN, kRowBytes = kColumns * 4, kLanes = kColumns / 8, kRowsAtOnce = kWave / kLanes;
    static_assert(Tile::kThreads / kWave * 32 * kRowBytes <= Tile::kLds && (kColumns == 64 || kColumns == 32));
    using Four = float __attribute__((ext_vector_type(4)));
    using LdsFour = __attribute__((address_space(3))) Four;
    using LdsFloat = __attribute__((address_space(3))) float;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    LdsByte* const area = lds + Tile::wave() * 32 * kRowBytes;
    const auto at = [](int row, int chunk) { return row * kRowBytes + ((chunk ^ (kColumns >= 64 ? ((row >> 2) & 1) << 3 | (row & 1) : row & 1)) << 4); };
    constexpr int kTurns = 32 / kRowsAtOnce;
    decltype(load(0, 0)) held[kTurns];
    const auto load_block = [&](int i) {
#pragma unroll
        for (int t = 0; t < kTurns; ++t) held[t] = load(32 * i + t * kRowsAtOnce + lane / kLanes, lane % kLanes * 8);
    };
    load_block(0);
    __syncthreads();  // the products' stages are read
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        if (i > 0) load_block(i);
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int column = 32 * j + lane_column();
                *(LdsFloat*)(area + at(block_row(r), column >> 2) + (column & 3) * 4) = acc[i][j][r];
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const int row = t * kRowsAtOnce + lane / kLanes, chunk = 2 * (lane % kLanes);
            LdsFour *const first = (LdsFour*)(area + at(row, chunk)), *const second = (LdsFour*)(area + at(row, chunk + 1));
            const Four one = *first, two = *second;
            float v[8] = {one[0], one[1], one[2], one[3], two[0], two[1], two[2], two[3]};
            f(32 * i + row, chunk * 4, v, held[t]);
            if (columns) *first = Four{v[0], v[1], v[2], v[3]}, *second = Four{v[4], v[5], v[6], v[7]};
        }
        __builtin_amdgcn_wave_barrier();
        if (columns) {
#pragma unroll
            for (int t = 0; t < kColumns / 16; ++t) {
                const int column = lane % kColumns, row = (kColumns == 64 ? t : 2 * t + lane / 32) * 8;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = *(LdsFloat*)(area + at(row + e, column >> 2) + (column & 3) * 4);
                g(32 * i + row, column, v);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

template <typename Tile, typename L, typename F>
__device__ __forceinline__ void by_rows(const typename Tile::Sums& acc, LdsByte* lds, L&& load, F&& f) {
    by_rows_and_columns<Tile>(acc, lds, false, load, f, [](int, int, float (&)[8]) {});
}

struct Nothing {};

// Workgroup id -> tile, such that each XCD (workgroups are dealt over the 8 in turn) takes a contiguous range of tiles, and those
// that run at once share panels: 8 tiles of n side by side, m after m.
__device__ __forceinline__ void tile_of(int64_t id, int64_t m_tiles, int64_t n_tiles, int64_t& m, int64_t& n) {
    constexpr int64_t kXcds = 8, kGroup = 8;
    const int64_t total = m_tiles * n_tiles, q = total / kXcds, r = total % kXcds, x = id % kXcds, i = id / kXcds;
    const int64_t t = x < r ? x * (q + 1) + i : r * (q + 1) + (x - r) * q + i;
    const int64_t group = t / (kGroup * m_tiles), inside = t - group * kGroup * m_tiles;
    const int64_t width = min(kGroup, n_tiles - group * kGroup);
    m = inside / width;
    n = group * kGroup + inside % width;
}

}  // namespace dllm_hip
