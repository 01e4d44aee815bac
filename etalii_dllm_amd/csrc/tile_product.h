// Tiled products on the 16-bit matrix cores: C[m][n] = sum over k of A[m][k] B[n][k], float32 sums, with an epilogue of the
// caller's on the tile in registers.
//
// Either operand lies in memory with k along its rows (kRows) or across them (kColumns: k is the row, m or n the column).
// Tiles of 64 k go through LDS two buffers deep, copied without registers in 16-byte chunks; chunk c of LDS row r lies at place
// c ^ swizzle(r), so that neither the row reads nor the transposing reads of kColumns tiles (4 rows of 16 columns by 16
// lanes) meet on a bank. A wave holds a kWaveM x kWaveN part of the tile as blocks of 32 x 32.
//
// Float32 operands come as planes of 16-bit parts: three of bfloat16, six products, or two of float16, three products; the
// smaller products first. The k loop runs once for each pair.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "doc_tile.h"

namespace dllm_hip {

// Bytes; base and strides are multiples of 16. kRows: m or n rows of k elements. kColumns: k rows of m or n elements, each
// readable up to the next multiple of 8 elements. `count`: how many m or n there are; indexes past it repeat others, what
// they yield is not stored.
struct Operand {
    const char* base;
    int64_t stride, plane, batch;
    int64_t count;
};

static __device__ const uint4 kZeroChunk = {0, 0, 0, 0};

template <int kPlanesOf>
struct PlanePairs {
    static constexpr int kCount = kPlanesOf == 1 ? 1 : kPlanesOf == 2 ? 3 : 6;
    // plane of A and of B in pair i
    static __device__ __forceinline__ int a(int i) {
        if constexpr (kPlanesOf == 1) return 0;
        if constexpr (kPlanesOf == 2) return i == 0 ? 1 : 0;
        return i == 0 ? 2 : i == 2 || i == 3 ? 1 : 0;
    }
    static __device__ __forceinline__ int b(int i) {
        if constexpr (kPlanesOf == 1) return 0;
        if constexpr (kPlanesOf == 2) return i == 1 ? 1 : 0;
        return i == 1 ? 2 : i == 2 || i == 4 ? 1 : 0;
    }
};

template <int kChunks>
__device__ __forceinline__ int tile_swizzle(int row) {
    if constexpr (kChunks >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
    if constexpr (kChunks == 4) return (row >> 2) & 3;
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// One operand's tile of kSize m or n by kTileK k: its copy to LDS.
template <int kSize, int kTileK, int kThreads, bool kColumns>
struct OperandTile {
    static constexpr int kChunks = kColumns ? kSize / 8 : kTileK / 8;  // of an LDS row
    static constexpr int kRows = kColumns ? kTileK : kSize;
    static constexpr int kRowBytes = kChunks * 16;
    static constexpr int kBytes = kRows * kRowBytes;
    static constexpr int kTurns = kRows * kChunks / kThreads;
    static constexpr int kTurnRows = kThreads / kChunks;
    static_assert(kRows * kChunks % kThreads == 0 && kThreads % kChunks == 0);

    const char* base;  // of the tile's first m or n
    int64_t stride, plane;
    uint32_t offset[kTurns];  // of the lane's chunk of each turn

    __device__ __forceinline__ static int lds_row(int turn) { return turn * kTurnRows + static_cast<int>(threadIdx.x) / kChunks; }
    __device__ __forceinline__ static int chunk(int turn) {
        return (static_cast<int>(threadIdx.x) % kChunks) ^ tile_swizzle<kChunks>(lds_row(turn));
    }

    __device__ __forceinline__ void init(const Operand& op, int64_t first, int64_t count, int64_t batch) {
        stride = op.stride;
        plane = op.plane;
        const int64_t left = count - first;  // at least 1
        base = op.base + batch * op.batch + (kColumns ? first * 2 : first * stride);
#pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const int64_t row = lds_row(t), c = chunk(t);
            if constexpr (kColumns)
                offset[t] = static_cast<uint32_t>(row * stride + min(c, (left - 1) / 8) * 16);
            else
                offset[t] = static_cast<uint32_t>(min(row, left - 1) * stride + c * 16);
        }
    }

    // The tile from k0 on of plane p to LDS; k at and past `k` are zero.
    __device__ __forceinline__ void copy(int64_t k0, int64_t k, int p, LdsByte* lds) const {
        const char* to = (const char*)lds + (static_cast<int>(threadIdx.x) >> 6) * 1024;
        const char* from = base + p * plane + (kColumns ? k0 * stride : k0 * 2);
        if (k0 + kTileK <= k) {
#pragma unroll
            for (int t = 0; t < kTurns; ++t) copy16_to_lds_s(from, offset[t], to + t * (kThreads * 16));
        } else {
#pragma unroll
            for (int t = 0; t < kTurns; ++t) {
                const bool inside = kColumns ? k0 + lds_row(t) < k : k0 + chunk(t) * 8 < k;
                const char* src = inside ? from + offset[t] : reinterpret_cast<const char*>(&kZeroChunk);
                copy16_to_lds(src, to + t * (kThreads * 16));
            }
        }
    }
};

// A lane's reads of blocks of 32 m or n by 16 k from a tile.
template <int kSize, int kTileK, bool kColumns>
struct OperandView {

    static constexpr int kRowBytes = (kColumns ? kSize / 8 : kTileK / 8) * 16;
    static constexpr int kChunks = kRowBytes / 16;
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
                const int chunk = first / 8 + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                at[t] = r * kRowBytes + ((chunk ^ tile_swizzle<kChunks>(r)) << 4) + (i & 1) * 8;
            }
        }
    }

    __device__ __forceinline__ Chunk16 read(const LdsByte* tile, int block, int step) const {
        if constexpr (!kColumns) {
            return *(const __attribute__((address_space(3))) Chunk16*)(tile + ((at[0] ^ (step << 5)) + block * 32 * kRowBytes));
        } else {
            using Half = short __attribute__((ext_vector_type(4)));
            union Both {
                Half h[2];
                Chunk16 c;
            } both;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                both.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) Half*)(tile + ((at[t] ^ (block << 6)) + step * 16 * kRowBytes)));
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

// A tile of kM x kN by kWavesM x kWavesN waves, kTileK k to each of kStages buffers.
template <typename P, int kPlanesOf, int kM_, int kN_, int kWavesM_, int kWavesN_, bool kAColumns, bool kBColumns, int kTileK = 64, int kStages = 2>
struct TileProduct {
    static constexpr int kM = kM_, kN = kN_, kWavesM = kWavesM_, kWavesN = kWavesN_;
    static constexpr int kThreads = kWavesM * kWavesN * kWave;
    static constexpr int kWaveM = kM / kWavesM, kWaveN = kN / kWavesN;
    static constexpr int kBlocksM = kWaveM / 32, kBlocksN = kWaveN / 32;
    using ATile = OperandTile<kM, kTileK, kThreads, kAColumns>;
    using BTile = OperandTile<kN, kTileK, kThreads, kBColumns>;
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
        constexpr int kPairs = PlanePairs<kPlanesOf>::kCount;
        ATile at;
        BTile bt;
        at.init(a, m0, a_count, batch_a);
        bt.init(b, n0, b_count, batch_b);
        const OperandView<kM, kTileK, kAColumns> av(wave_m());
        const OperandView<kN, kTileK, kBColumns> bv(wave_n());
        const auto clear = [&] {
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i)
#pragma unroll
                for (int j = 0; j < kBlocksN; ++j) acc[i][j] = Acc{};
        };
        clear();
        const int tiles = static_cast<int>((k + kTileK - 1) / kTileK), count = tiles * kPairs;
        if (count == 0) return;
        const int segment_tiles = kSegments ? static_cast<int>(segment / kTileK) : tiles;
        int pair = 0, tile = 0, into = 0, first = 0, end = min(segment_tiles, tiles);  // of the next copy; first, end: of its segment
        auto copy = [&] {
            LdsByte* const to = lds + into * kStage;
            at.copy(static_cast<int64_t>(tile) * kTileK, k, PlanePairs<kPlanesOf>::a(pair), to);
            bt.copy(static_cast<int64_t>(tile) * kTileK, k, PlanePairs<kPlanesOf>::b(pair), to + ATile::kBytes);
            if (++tile == end) {
                if (++pair == kPairs && kSegments) pair = 0, first = end, end = min(end + segment_tiles, tiles);
                tile = first;
            }
            into = into + 1 == kStages ? 0 : into + 1;
        };
        for (int i = 0; i < kStages - 1 && i < count; ++i) copy();
        int from = 0, boundary = segment_tiles * kPairs;
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
                boundary += segment_tiles * kPairs;
#pragma unroll
                for (int m = 0; m < kBlocksM; ++m)
#pragma unroll
                    for (int n = 0; n < kBlocksN; ++n) total[m][n] += acc[m][n];
                clear();
            }
            const LdsByte* const stage = lds + from * kStage;
            from = from + 1 == kStages ? 0 : from + 1;
#pragma unroll
            for (int step = 0; step < kTileK / 16; ++step) {
                Chunk16 x[kBlocksM], y[kBlocksN];
#pragma unroll
                for (int m = 0; m < kBlocksM; ++m) x[m] = av.read(stage, m, step);
#pragma unroll
                for (int n = 0; n < kBlocksN; ++n) y[n] = bv.read(stage + ATile::kBytes, n, step);
#pragma unroll
                for (int m = 0; m < kBlocksM; ++m)
#pragma unroll
                    for (int n = 0; n < kBlocksN; ++n) multiply<P>(x[m], y[n], acc[m][n]);
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
