// A projection shared by all rows beside low-rank adapters of which each row names one:
//
//     out[r] = x[r] weight^T + scale_a (x[r] down_a^T) up_a^T,   a = adapter_ids[r]
//
// The rows of a large batch are sorted by adapter, so that rows of one adapter are next to each other, and
// x and out are addressed through the order; few rows keep theirs. `low` = scale_a x[r] down_a^T is formed first, one group of
// up to 16 rows of one adapter at a time; the projection's kernel then adds low up_a^T to each tile's
// sums: out is written once for both.
//
// low between the two products. The products are the 16-bit matrix instructions', so low is handed over
// in parts of the operands' type, high + rest (+ rest of that), as many as keep a float32 output's digits:
// two of float16 hold 22 bits, three of bfloat16 all 24; a bfloat16 output takes two, of 16 bits. A float16 row is
// scaled by a power of two that brings its largest finite value to [2^14, 2^15), so that it neither overflows nor
// loses small parts; its inverse is applied to the sums in float32. bfloat16 has float32's range: only values from
// 2^126 on are scaled, down, since they could round to an infinity; up may hold values as large as float32's, with
// which scaled-up rows would overflow. float32 operands need no parts.
//
// Measured: 8192 rows 1024 -> 1024, 32 adapters of rank 32 in runs of 250, bfloat16: 57 us, of which the sort 9,
// low 12.5, the projection 23 (a library product 25) and the adapters' part 13; 300 mixed rows of 200 adapters
// 14.0 us, 8 rows of 64 9.7 us, in two launches.
//
// Rows are kept apart: a row's sums take the products with its own adapter only, chosen and not
// multiplied by zero, so infinities and NaN in one adapter stay in its rows.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"
#include "elements.hpp"
#include "matrix_plan.hpp"
#include "matrix_tile.hpp"
#include "pair_sort.hpp"

namespace zcgvs_hip {

namespace {

constexpr int kMaxRank = 128;
constexpr int kRankStep = 32;  // low's rows are padded to whole steps of the matrix instructions

template <typename T, typename Out>
constexpr int kParts = std::is_same_v<T, float> ? 1 : std::is_same_v<T, __bf16> && std::is_same_v<Out, float> ? 3 : 2;
constexpr int kMostParts = 3;

int paddedRank(int max_rank) { return (max_rank + kRankStep - 1) / kRankStep * kRankStep; }

struct AdaptedArgs {
    const void* x;
    std::int64_t x_stride;
    const void* weight;
    std::int64_t weight_stride;
    int rows;
    int dim;
    int out_dim;
    const void* down;
    const void* up;
    int adapter_count;
    int max_rank;
    int padded_rank;
    const int* ranks;
    const float* scales;
    const int* adapters;  // [rows] sorted, adapter_count: none; null: no row has one
    const int* order;     // [rows] the row at each sorted position
    int parts;
    void* low;            // [rows, parts, padded_rank] by sorted position
    float* low_scale;     // [rows]
    int tiles_m;
    int tiles_n;
    void* out;
    std::int64_t out_stride;
};

__device__ __forceinline__ int rankOf(const AdaptedArgs& args, int adapter) {
    return args.ranks == nullptr ? args.max_rank : min(max(args.ranks[adapter], 0), args.max_rank);
}

// 16 bytes of a row of which `valid` values from `from` on exist; the others are zeros.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::type loadChunk(const T* from, int valid) {
    typename Fragment<T>::type v = {};
    if (valid >= kChunk<T>) {
        __builtin_memcpy(&v, from, 16);
    } else {
#pragma unroll
        for (int e = 0; e < kChunk<T>; ++e) {
            if (e < valid) {
                v[e] = from[e];
            }
        }
    }
    return v;
}

// The same where the row has `stored` values from `from` on, of which the first `valid` are wanted.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::type loadMasked(const T* from, int stored, int valid) {
    typename Fragment<T>::type v = loadChunk(from, stored);
#pragma unroll
    for (int e = 0; e < kChunk<T>; ++e) {
        v[e] = e < valid ? v[e] : static_cast<T>(0.0f);
    }
    return v;
}

// Zeros in the place of infinities.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::type withoutInfinities(const typename Fragment<T>::type& v) {
    static_assert(sizeof(T) == 2, "16-bit values");
    typedef std::uint16_t Bits __attribute__((ext_vector_type(8)));
    constexpr std::uint16_t kInfinity = std::is_same_v<T, __bf16> ? 0x7F80 : 0x7C00;
    Bits bits = __builtin_bit_cast(Bits, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        bits[e] = (bits[e] & 0x7FFF) == kInfinity ? 0 : bits[e];
    }
    return __builtin_bit_cast(typename Fragment<T>::type, bits);
}

// ---- low = scale x down^T -----------------------------------------------------------------------

// A workgroup takes the groups that begin among `positions` sorted positions (1, or a block of 16; a group is
// the rows of one adapter within a block). Its eight wavefronts take an eighth of the steps over dim each and
// their sums are joined through LDS.
constexpr int kLowThreads = 512;
constexpr int kLowWaves = kLowThreads / kWave;

template <typename T, int kRankBlocks>
__global__ __launch_bounds__(kLowThreads) void lowKernel(AdaptedArgs args, int positions) {
    constexpr int kLowAhead = kRankBlocks <= 4 ? 4 : 2;  // steps whose loads are in flight
    constexpr int kRanks = kRankBlocks * 16;
    __shared__ float joined[kLowWaves][16][kRanks];
    __shared__ float row_peak[16][16];
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int r16 = lane & 15;
    const int h = lane >> 4;
    constexpr int kStepK = 4 * kChunk<T>;
    const int steps = (args.dim + kStepK - 1) / kStepK;
    const int share = (steps + kLowWaves - 1) / kLowWaves;
    const int first = static_cast<int>(blockIdx.x) * positions;
    const int block = first / 16 * 16;
    const int in_block = min(16, args.rows - block);
    // the block's adapters, a lane each
    const int at = block + min(r16, in_block - 1);
    const int my_adapter = args.adapters[at];
    const int my_row = args.order[at];
    const int adapter_before = __shfl_up(my_adapter, 1, kWave);
    const unsigned begins = static_cast<unsigned>(
        __ballot(lane < in_block && my_adapter < args.adapter_count && (lane == 0 || my_adapter != adapter_before)));
    unsigned left = positions == 1 ? begins & (1u << (first - block)) : begins;
    while (left != 0) {
        const int start = __builtin_ctz(left);
        left &= left - 1;
        const int adapter = __builtin_amdgcn_readlane(my_adapter, start);
        const int length = __popcll(__ballot(lane < in_block && my_adapter == adapter));
        const int p = block + start;
        const int rank = rankOf(args, adapter);
        const T* x = static_cast<const T*>(args.x) +
                     __shfl(my_row, start + min(r16, length - 1), kWave) * args.x_stride;
        const T* down = static_cast<const T*>(args.down) +
                        static_cast<std::int64_t>(adapter) * args.max_rank * args.dim;
        f32x4 sums[kRankBlocks];
        const T* rows_of[kRankBlocks];  // a row past the rank gives sums that are not used
#pragma unroll
        for (int j = 0; j < kRankBlocks; ++j) {
            sums[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            rows_of[j] = down + static_cast<std::int64_t>(min(j * 16 + r16, max(rank, 1) - 1)) * args.dim;
        }
        const int past_step = min((wave + 1) * share, steps);
        const int past_whole = min(past_step, args.dim / kStepK);
        int s = wave * share;
        for (; s + kLowAhead <= past_whole; s += kLowAhead) {
            typename Fragment<T>::type a[kLowAhead], b[kLowAhead][kRankBlocks];
#pragma unroll
            for (int u = 0; u < kLowAhead; ++u) {
                const int k = (s + u) * kStepK + h * kChunk<T>;
                __builtin_memcpy(&a[u], x + k, 16);
#pragma unroll
                for (int j = 0; j < kRankBlocks; ++j) {
                    __builtin_memcpy(&b[u][j], rows_of[j] + k, 16);
                }
            }
#pragma unroll
            for (int u = 0; u < kLowAhead; ++u) {
#pragma unroll
                for (int j = 0; j < kRankBlocks; ++j) {
                    sums[j] = multiplyAdd(b[u][j], a[u], sums[j]);
                }
            }
        }
        for (; s < past_step; ++s) {
            const int k = s * kStepK + h * kChunk<T>;
            const auto a = loadChunk(x + k, args.dim - k);
#pragma unroll
            for (int j = 0; j < kRankBlocks; ++j) {
                sums[j] = multiplyAdd(loadChunk(rows_of[j] + k, args.dim - k), a, sums[j]);
            }
        }
        __syncthreads();  // the last group's sums have been read
#pragma unroll
        for (int j = 0; j < kRankBlocks; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                joined[wave][r16][j * 16 + 4 * h + e] = sums[j][e];
            }
        }
        __syncthreads();
        // 16 threads a row; the others look on
        const int row = static_cast<int>(threadIdx.x) / 16 % 16;
        const int column = static_cast<int>(threadIdx.x) % 16;
        const float scale = args.scales == nullptr ? 1.0f : args.scales[adapter];
        float value[kRankBlocks];
        float peak = 0.0f;
#pragma unroll
        for (int j = 0; j < kRankBlocks; ++j) {
            const int r = j * 16 + column;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kLowWaves; ++w) {
                sum += joined[w][row][r];
            }
            value[j] = r < rank ? sum * scale : 0.0f;
            // of the finite ones: beside an infinity they still have to fit the parts
            peak = fmaxf(peak, fabsf(value[j]) <= 3.402823466e+38f ? fabsf(value[j]) : 0.0f);
        }
        if constexpr (sizeof(T) == 2) {
            row_peak[row][column] = peak;  // the same from both halves of the workgroup
            __syncthreads();
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                peak = fmaxf(peak, row_peak[row][c]);
            }
        }
        if (row < length && threadIdx.x < 256) {
            const std::int64_t at = p + row;
            if constexpr (sizeof(T) == 2) {
                int exponent = 0;
                if (peak > 0.0f) {
                    int e = 0;
                    frexpf(peak, &e);  // peak = m 2^e, m in [0.5, 1)
                    exponent = std::is_same_v<T, __bf16> ? min(0, 126 - e) : min(126, max(-126, 15 - e));
                }
                T* to = static_cast<T*>(args.low) + at * args.parts * args.padded_rank;
                const float up_by = ldexpf(1.0f, exponent);
#pragma unroll
                for (int j = 0; j < kRankBlocks; ++j) {
                    const int r = j * 16 + column;
                    float rest = value[j] * up_by;
                    if (r < args.padded_rank) {
                        for (int part = 0; part < args.parts; ++part) {
                            const T here = static_cast<T>(rest);
                            to[part * args.padded_rank + r] = here;
                            // an infinite value has no rest
                            rest = fabsf(rest) <= 3.402823466e+38f ? rest - static_cast<float>(here) : 0.0f;
                        }
                    }
                }
                for (int r = kRanks + column; r < args.padded_rank; r += 16) {
                    for (int part = 0; part < args.parts; ++part) {
                        to[part * args.padded_rank + r] = static_cast<T>(0.0f);
                    }
                }
                if (column == 0) {
                    args.low_scale[at] = ldexpf(1.0f, -exponent);
                }
            } else {
                float* to = static_cast<float*>(args.low) + at * args.padded_rank;
#pragma unroll
                for (int j = 0; j < kRankBlocks; ++j) {
                    if (j * 16 + column < args.padded_rank) {
                        to[j * 16 + column] = value[j];
                    }
                }
                for (int r = kRanks + column; r < args.padded_rank; r += 16) {
                    to[r] = 0.0f;
                }
                if (column == 0) {
                    args.low_scale[at] = 1.0f;
                }
            }
        }
        if constexpr (sizeof(T) == 2) {
            __syncthreads();  // row_peak is written again
        }
    }
}

// ---- the projection -----------------------------------------------------------------------------

// Adds low up^T to a tile's sums, in one of two ways.
// By adapter: one adapter of the tile's rows after the other. Its rows of low (zeros for the other rows) and
// its columns of up go through LDS like a stage of the products over dim, and the result is kept in the rows
// that are the adapter's. An adapter costs about 1.6 us for every 64 values of low's parts (float32: 32).
// By row: every lane forms its own results, 4 columns of a row, from its row's adapter: a fused
// multiply-add for each rank and result (64 x 32 results of rank 32 about 3 us), whatever the adapters; taken
// where the tile's rows have many.
// Every thread of the workgroup calls it, behind the products over dim.

// A tile's rows, 64 to a register: their adapters (adapter_count: none), ranks and low's scales. Read before
// the products over dim, behind which the latency is gone.
template <int kTileRows>
struct TileAdapters {
    static constexpr int kSets = kTileRows / kWave;
    int adapter[kSets];
    int rank[kSets];
    float scale[kSets];
    int changes;  // rows whose adapter is not that of the row before

    __device__ __forceinline__ void read(const AdaptedArgs& args, int m0) {
        const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
        int before[kSets];
#pragma unroll
        for (int i = 0; i < kSets; ++i) {
            const int p = min(m0 + i * kWave + lane, args.rows - 1);
            adapter[i] = args.adapters[p];
            before[i] = args.adapters[max(p - 1, 0)];
            scale[i] = args.low_scale[p];
        }
        changes = 0;
#pragma unroll
        for (int i = 0; i < kSets; ++i) {
            adapter[i] = m0 + i * kWave + lane < args.rows ? adapter[i] : args.adapter_count;
            const bool has = adapter[i] < args.adapter_count;
            rank[i] = has ? rankOf(args, adapter[i]) : 0;
            scale[i] = has ? scale[i] : 0.0f;
            changes += __popcll(__ballot(has && adapter[i] != before[i]));
        }
    }
    // Of the tile's row `row`, which may differ from lane to lane.
    template <typename V>
    static __device__ __forceinline__ V at(const V (&values)[kSets], int row) {
        V value = __shfl(values[0], row % kWave, kWave);
#pragma unroll
        for (int i = 1; i < kSets; ++i) {
            const V other = __shfl(values[i], row % kWave, kWave);
            value = row / kWave == i ? other : value;
        }
        return value;
    }
};

template <class Tile, typename Out>
__device__ __forceinline__ void addAdapters(const AdaptedArgs& args, const TileAdapters<Tile::kM>& rows,
                                            std::uint8_t* lds, int m0, int n0, typename Tile::Sums& sums) {
    using T = typename Tile::T;
    constexpr int kHere = kParts<T, Out>;
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int r16 = lane & 15;
    const int h = lane >> 4;
    int left = __builtin_amdgcn_readfirstlane(rows.adapter[0]);  // sorted: the first row's is the smallest
    if (left >= args.adapter_count) {
        return;
    }
    const int wave_row = Tile::waveM() * Tile::kBlocksM * 16 + r16;
    if (rows.changes > 2 + args.max_rank / 8) {
        const int wave_n0 = n0 + Tile::waveN() * Tile::kBlocksN * 16 + 4 * h;
#pragma unroll
        for (int i = 0; i < Tile::kBlocksM; ++i) {
            const int row = wave_row + i * 16;
            const int adapter = TileAdapters<Tile::kM>::at(rows.adapter, row);
            const int rank = TileAdapters<Tile::kM>::at(rows.rank, row);
            const float scale = TileAdapters<Tile::kM>::at(rows.scale, row);
            // a row without an adapter has rank 0
            const T* low = static_cast<const T*>(args.low) +
                           static_cast<std::int64_t>(m0 + row) * kHere * args.padded_rank;
            const T* up = static_cast<const T*>(args.up) + static_cast<std::int64_t>(adapter) * args.out_dim * args.max_rank;
#pragma unroll 1
            for (int r = 0; r < rank; r += kChunk<T>) {
                float values[kChunk<T>];
#pragma unroll
                for (int half = 0; half < kHere; ++half) {
                    const auto v = *reinterpret_cast<const typename Fragment<T>::type*>(low + half * args.padded_rank + r);
#pragma unroll
                    for (int e = 0; e < kChunk<T>; ++e) {
                        values[e] = (half == 0 ? 0.0f : values[e]) + static_cast<float>(v[e]) * scale;
                    }
                }
#pragma unroll
                for (int j = 0; j < Tile::kBlocksN; ++j) {
                    typename Fragment<T>::type b[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int n = min(wave_n0 + j * 16 + e, args.out_dim - 1);
                        b[e] = loadMasked(up + static_cast<std::int64_t>(n) * args.max_rank + r, args.max_rank - r, rank - r);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
#pragma unroll
                        for (int c = 0; c < kChunk<T>; ++c) {
                            sums[i][j][e] += values[c] * static_cast<float>(b[e][c]);
                        }
                    }
                }
            }
        }
        return;
    }
    using SideA = typename Tile::StageTile::SideA;
    using SideB = typename Tile::StageTile::SideB;
    const int low_values = kHere * args.padded_rank;
    while (left < args.adapter_count) {
        int rank = 0;
        int next = args.adapter_count;
#pragma unroll
        for (int i = 0; i < TileAdapters<Tile::kM>::kSets; ++i) {
            const unsigned long long mine = __ballot(rows.adapter[i] == left);
            const unsigned long long later = __ballot(rows.adapter[i] > left);
            rank = mine != 0 ? __builtin_amdgcn_readlane(rows.rank[i], __builtin_ctzll(mine)) : rank;
            if (later != 0) {  // the first of them is the next
                next = min(next, __builtin_amdgcn_readlane(rows.adapter[i], __builtin_ctzll(later)));
            }
        }
        const T* up = static_cast<const T*>(args.up) + static_cast<std::int64_t>(left) * args.out_dim * args.max_rank;
        typename Tile::Sums part;
        Tile::clear(part);
#pragma unroll 1
        for (int k0 = 0; k0 < low_values; k0 += kStageK<T>) {
            typename Fragment<T>::type a[SideA::kCopies], b[SideB::kCopies];
#pragma unroll
            for (int i = 0; i < SideA::kCopies; ++i) {
                int row, chunk;
                SideA::placeOf(i, row, chunk);
                const int k = k0 + chunk * kChunk<T>;
                const bool mine = TileAdapters<Tile::kM>::at(rows.adapter, row) == left && k < low_values;
                a[i] = typename Fragment<T>::type{};
                if (mine) {
                    a[i] = *reinterpret_cast<const typename Fragment<T>::type*>(
                        static_cast<const T*>(args.low) + static_cast<std::int64_t>(m0 + row) * low_values + k);
                }
            }
#pragma unroll
            for (int i = 0; i < SideB::kCopies; ++i) {
                int row, chunk;
                SideB::placeOf(i, row, chunk);
                const int n = min(n0 + row, args.out_dim - 1);
                const int k = k0 + chunk * kChunk<T>;
                const int r = k % args.padded_rank;  // every part meets the same columns of up
                b[i] = loadMasked(up + static_cast<std::int64_t>(n) * args.max_rank + r,
                                  k < low_values ? args.max_rank - r : 0, rank - r);
                if constexpr (kHere > 1) {
                    // an infinity times the first part is the result; a rest of 0 or of the other sign makes it NaN
                    if (k >= args.padded_rank) {
                        b[i] = withoutInfinities<T>(b[i]);
                    }
                }
            }
            __syncthreads();  // what stood in the LDS has been read
#pragma unroll
            for (int i = 0; i < SideA::kCopies; ++i) {
                *reinterpret_cast<typename Fragment<T>::type*>(lds + (i * Tile::kThreads + static_cast<int>(threadIdx.x)) * 16) = a[i];
            }
#pragma unroll
            for (int i = 0; i < SideB::kCopies; ++i) {
                *reinterpret_cast<typename Fragment<T>::type*>(
                    lds + SideA::kBytes + (i * Tile::kThreads + static_cast<int>(threadIdx.x)) * 16) = b[i];
            }
            __syncthreads();
            Tile::StageTile::multiplyStage(lds, part);
        }
#pragma unroll
        for (int i = 0; i < Tile::kBlocksM; ++i) {
            const int row = wave_row + i * 16;
            const bool mine = TileAdapters<Tile::kM>::at(rows.adapter, row) == left;
            const float scale = TileAdapters<Tile::kM>::at(rows.scale, row);
#pragma unroll
            for (int j = 0; j < Tile::kBlocksN; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sums[i][j][e] += mine ? part[i][j][e] * scale : 0.0f;
                }
            }
        }
        left = next;
    }
}

// 128 registers, so that a CU holds two workgroups of the 128 x 128 tile (float32's 64 x 64: three).
template <class Tile, typename Out>
__global__ __launch_bounds__(Tile::kThreads, Tile::kThreads >= 512 ? 4 : 3) void adaptedKernel(AdaptedArgs args) {
    using T = typename Tile::T;
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    int tile_m, tile_n;
    tileOf(static_cast<int>(blockIdx.x), args.tiles_m, args.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * Tile::kM;
    const int n0 = tile_n * Tile::kN;
    const T* x = static_cast<const T*>(args.x);
    const T* weight = static_cast<const T*>(args.weight);
    const auto row_at = [&](int p) { return args.order == nullptr ? p : args.order[p]; };
    typename Tile::Loads loads;
    loads.begin([&](int r) { return x + row_at(min(m0 + r, args.rows - 1)) * args.x_stride; }, args.x_stride, 0,
                [&](int r) { return weight + min(n0 + r, args.out_dim - 1) * args.weight_stride; },
                args.weight_stride, 0, args.dim);
    loads.start(lds);
    typename Tile::Sums sums;
    Tile::clear(sums);
    TileAdapters<Tile::kM> rows;
    if (args.adapters != nullptr) {
        rows.read(args, m0);
    }
    Tile::accumulate(lds, loads, args.dim, sums, [] {});
    if (args.adapters != nullptr) {
        addAdapters<Tile, Out>(args, rows, lds, m0, n0, sums);
    }
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        const int p = m0 + (Tile::waveM() * Tile::kBlocksM + i) * 16 + (lane & 15);
        if (p >= args.rows) {
            continue;
        }
        Out* out = static_cast<Out*>(args.out) + row_at(p) * args.out_stride;
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j) {
            const int n = n0 + (Tile::waveN() * Tile::kBlocksN + j) * 16 + 4 * (lane >> 4);
            if (n < args.out_dim) {
                storeFour(sums[i][j], out + n, args.out_dim - n);
            }
        }
    }
}

// ---- few rows -----------------------------------------------------------------------------------

// Few rows, in their own order: a workgroup forms 16 columns of 16 rows. Its 16 wavefronts form a sixteenth of
// the products over dim each; 256 threads add those up and their result's share of low up^T. low is formed
// either by every workgroup for itself (as many wavefronts to a row as there are for each, every one over its part
// of dim), which saves a launch while the rows of down that it reads are few, or by a launch before. All of
// low stays in float32. Measured, float16, rank 16, mixed adapters, against the sorted rows' three launches: 1 row
// of 768 -> 768 6.8 us (two launches 9.9), 8 rows 9.9 (one launch 12.2); 300 rows of 384 -> 384 9.6 against 18.1,
// 1000 rows 16.1 against 23.1; 300 rows of 1024 -> 1024 20.8 against 24.9, 500 rows 28.6 against 25.4.
constexpr int kFewRows = 16;
constexpr int kFewThreads = 1024;
constexpr int kFewWaves = kFewThreads / kWave;
constexpr std::int64_t kFewProducts = 400'000'000;  // rows * dim * out_dim up to which it is taken
constexpr std::int64_t kFewDownBytes = 50 * 1024;   // of down that a workgroup reads

// Products of 16 rows of `a_row` and 16 rows of `b_row` (a lane has its row l % 16 of each) over the steps
// [step, past).
template <typename T>
__device__ __forceinline__ f32x4 multiplyRows(const T* a_row, const T* b_row, int step, int past, int dim) {
    constexpr int kStepK = 4 * kChunk<T>;
    constexpr int kAhead = 4;
    const int h = (static_cast<int>(threadIdx.x) & (kWave - 1)) >> 4;
    const int past_whole = min(past, dim / kStepK);
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (; step + kAhead <= past_whole; step += kAhead) {
        typename Fragment<T>::type a[kAhead], b[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = (step + u) * kStepK + h * kChunk<T>;
            __builtin_memcpy(&a[u], a_row + k, 16);
            __builtin_memcpy(&b[u], b_row + k, 16);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            sum = multiplyAdd(b[u], a[u], sum);
        }
    }
    for (; step < past; ++step) {
        const int k = step * kStepK + h * kChunk<T>;
        sum = multiplyAdd(loadChunk(b_row + k, dim - k), loadChunk(a_row + k, dim - k), sum);
    }
    return sum;
}

// low of one row and 16 ranks: args.low is float32 [rows, max_rank] here.
constexpr int kLowFewThreads = 256;
constexpr int kLowFewWaves = kLowFewThreads / kWave;

template <typename T>
__global__ __launch_bounds__(kLowFewThreads) void lowFewKernel(AdaptedArgs args, const int* adapter_ids) {
    __shared__ float joined[kLowFewWaves][16];
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int row = static_cast<int>(blockIdx.x);
    const int r = static_cast<int>(blockIdx.y) * 16;
    const int adapter = adapter_ids[row];
    if (!counts(adapter, args.adapter_count, -1)) {
        return;
    }
    const int rank = rankOf(args, adapter);
    if (r >= rank) {
        return;
    }
    const int steps = (args.dim + 4 * kChunk<T> - 1) / (4 * kChunk<T>);
    const int share = (steps + kLowFewWaves - 1) / kLowFewWaves;
    const T* down = static_cast<const T*>(args.down) +
                    (static_cast<std::int64_t>(adapter) * args.max_rank + min(r + (lane & 15), rank - 1)) * args.dim;
    const f32x4 sum = multiplyRows(static_cast<const T*>(args.x) + row * args.x_stride, down, wave * share,
                                   min((wave + 1) * share, steps), args.dim);
    if ((lane & 15) == 0) {  // every column holds the row
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            joined[wave][4 * (lane >> 4) + e] = sum[e];
        }
    }
    __syncthreads();
    if (threadIdx.x < 16 && r + static_cast<int>(threadIdx.x) < rank) {
        float whole = 0.0f;
        for (int w = 0; w < kLowFewWaves; ++w) {
            whole += joined[w][threadIdx.x];
        }
        const float scale = args.scales == nullptr ? 1.0f : args.scales[adapter];
        static_cast<float*>(args.low)[static_cast<std::int64_t>(row) * args.max_rank + r + threadIdx.x] = whole * scale;
    }
}

// kFormLow: low is formed here; otherwise it stands in args.low.
template <typename T, typename Out, bool kFormLow>
__global__ __launch_bounds__(kFewThreads) void adaptedFewKernel(AdaptedArgs args, const int* adapter_ids) {
    __shared__ float low[kFormLow ? kFewWaves : 1][kMaxRank + 4];
    __shared__ float parts[kFewWaves][16][17];
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int r16 = lane & 15;
    const int h = lane >> 4;
    const int n0 = static_cast<int>(blockIdx.x) * 16;
    const int m0 = static_cast<int>(blockIdx.y) * kFewRows;
    const int rows = min(kFewRows, args.rows - m0);
    const int steps = (args.dim + 4 * kChunk<T> - 1) / (4 * kChunk<T>);
    const T* x_row = static_cast<const T*>(args.x) + (m0 + min(r16, rows - 1)) * args.x_stride;
    // wavefronts to a row of low: the largest power of two that serves all rows
    int helpers = kFewWaves;
    while (helpers * rows > kFewWaves) {
        helpers /= 2;
    }
    const int my_row = wave / helpers;
    const int my_adapter = kFormLow && adapter_ids != nullptr && my_row < rows ? adapter_ids[m0 + my_row] : -1;
    const int share = (steps + kFewWaves - 1) / kFewWaves;
    const T* weight_row = static_cast<const T*>(args.weight) + min(n0 + r16, args.out_dim - 1) * args.weight_stride;
    const f32x4 product = multiplyRows(x_row, weight_row, wave * share, min((wave + 1) * share, steps), args.dim);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        parts[wave][r16][4 * h + e] = product[e];
    }
    if (kFormLow && counts(my_adapter, args.adapter_count, -1)) {
        const int rank = rankOf(args, my_adapter);
        const float scale = args.scales == nullptr ? 1.0f : args.scales[my_adapter];
        const T* down = static_cast<const T*>(args.down) + static_cast<std::int64_t>(my_adapter) * args.max_rank * args.dim;
        const int low_share = (steps + helpers - 1) / helpers;
        const int first = wave % helpers * low_share;
        for (int r = 0; r < rank; r += 16) {
            const f32x4 sum = multiplyRows(x_row, down + static_cast<std::int64_t>(min(r + r16, rank - 1)) * args.dim, first,
                                           min(first + low_share, steps), args.dim);
            if (r16 == my_row) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    low[wave][r + 4 * h + e] = sum[e] * scale;
                }
            }
        }
    }
    __syncthreads();
    const int row = static_cast<int>(threadIdx.x) / 16;
    const int n = n0 + static_cast<int>(threadIdx.x) % 16;
    if (row >= rows || n >= args.out_dim) {
        return;
    }
    float sum = 0.0f;
    const int adapter = adapter_ids == nullptr ? -1 : adapter_ids[m0 + row];
    if (counts(adapter, args.adapter_count, -1)) {
        const int rank = rankOf(args, adapter);
        const T* up = static_cast<const T*>(args.up) +
                      (static_cast<std::int64_t>(adapter) * args.out_dim + n) * args.max_rank;
        for (int r = 0; r < rank; r += kChunk<T>) {
            const auto b = loadChunk(up + r, args.max_rank - r);
#pragma unroll
            for (int e = 0; e < kChunk<T>; ++e) {
                if (r + e < rank) {
                    float whole = 0.0f;
                    if constexpr (kFormLow) {
                        for (int w = 0; w < helpers; ++w) {
                            whole += low[row * helpers + w][r + e];
                        }
                    } else {
                        whole = static_cast<const float*>(args.low)[static_cast<std::int64_t>(m0 + row) * args.max_rank + r + e];
                    }
                    sum += whole * static_cast<float>(b[e]);
                }
            }
        }
    }
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
        sum += parts[w][row][static_cast<int>(threadIdx.x) % 16];
    }
    static_cast<Out*>(args.out)[(m0 + row) * args.out_stride + n] = static_cast<Out>(sum);
}

// ---- host ---------------------------------------------------------------------------------------

int invalid(const char* message) {
    return setError(ZCGVS_ERR_INVALID_ARGUMENT, std::string("zcgvs adapted projection: ") + message);
}

int checkAdapted(const zcgvs_adapted_desc* desc) {
    if (desc == nullptr) {
        return invalid("null descriptor");
    }
    const zcgvs_adapted_desc& d = *desc;
    if (!validElement(d.dtype)) {
        return invalid("the operands must hold float32, float16 or bfloat16");
    }
    if (d.dim <= 0 || d.out_dim <= 0) {
        return invalid("dim and out_dim must be positive");
    }
    if (d.dim > (1 << 24) || d.out_dim > (1 << 24)) {
        return invalid("dim and out_dim must be at most 2^24");
    }
    if (d.rows < 0 || d.rows > (1 << 29)) {
        return invalid("rows must lie in [0, 2^29]");
    }
    if (rowStride(d.x_stride, d.dim) < d.dim || rowStride(d.weight_stride, d.dim) < d.dim) {
        return invalid("a row stride is smaller than dim");
    }
    if (d.rows > 0 && (d.x == nullptr || d.weight == nullptr)) {
        return invalid("null device pointer");
    }
    if (d.adapter_ids != nullptr) {
        if (d.adapter_count < 0 || d.adapter_count == INT32_MAX) {
            return invalid("adapter_count must lie in [0, 2^31 - 2]");
        }
        if (d.adapter_count > 0 && (d.max_rank <= 0 || d.max_rank > kMaxRank)) {
            return invalid("max_rank must lie in [1, 128]");
        }
        if (d.rows > 0 && d.adapter_count > 0 && (d.down == nullptr || d.up == nullptr)) {
            return invalid("null adapter pointer");
        }
    }
    return ZCGVS_OK;
}

bool hasAdapters(const zcgvs_adapted_desc& d) { return d.adapter_ids != nullptr && d.adapter_count > 0; }

struct AdaptedSpace {
    std::size_t sort;
    std::size_t low;
    std::size_t low_scale;
    std::size_t bytes;
};

AdaptedSpace adaptedSpace(const zcgvs_adapted_desc& d) {
    AdaptedSpace s{};
    std::size_t at = 0;
    if (hasAdapters(d)) {
        const std::size_t rows = static_cast<std::size_t>(d.rows);
        const std::size_t parts = d.dtype == ZCGVS_DTYPE_F32 ? 1 : kMostParts;
        s.sort = at;
        at += pairSortBytes(rows);
        s.low = at;
        at += sortAligned(rows * parts * static_cast<std::size_t>(paddedRank(d.max_rank) * elementBytes(d.dtype)));
        s.low_scale = at;
        at += sortAligned(rows * 4);
    }
    s.bytes = std::max<std::size_t>(at, 256);
    return s;
}

template <typename T>
int launchLow(const AdaptedArgs& args, hipStream_t stream) {
    // many rows of few adapters begin few groups: a workgroup a block of 16 then; else one a group
    const int positions = args.rows <= 2048 ? 1 : 16;
    const int blocks_needed = divideUp(args.rows, positions);
    if (blocks_needed > (1 << 23) - 1) {
        return invalid("more rows than one launch can take");
    }
    const unsigned blocks = static_cast<unsigned>(blocks_needed);
    const int rank_blocks = (args.max_rank + 15) / 16;
    if (rank_blocks <= 1) {
        lowKernel<T, 1><<<blocks, kLowThreads, 0, stream>>>(args, positions);
    } else if (rank_blocks <= 2) {
        lowKernel<T, 2><<<blocks, kLowThreads, 0, stream>>>(args, positions);
    } else if (rank_blocks <= 4) {
        lowKernel<T, 4><<<blocks, kLowThreads, 0, stream>>>(args, positions);
    } else {
        lowKernel<T, 8><<<blocks, kLowThreads, 0, stream>>>(args, positions);
    }
    ZCGVS_LAUNCH_CHECK("adapted projection");
    return ZCGVS_OK;
}

template <class Tile, typename Out>
int launchTile(AdaptedArgs args, hipStream_t stream) {
    args.tiles_m = divideUp(args.rows, Tile::kM);
    args.tiles_n = divideUp(args.out_dim, Tile::kN);
    const long long blocks = static_cast<long long>(args.tiles_m) * args.tiles_n;
    if (blocks > kMaxBlocks) {
        return invalid("more output than one launch can write");
    }
    adaptedKernel<Tile, Out><<<static_cast<unsigned>(blocks), Tile::kThreads, 0, stream>>>(args);
    ZCGVS_LAUNCH_CHECK("adapted projection");
    return ZCGVS_OK;
}

template <typename T, typename Out>
int launchAdapted(const AdaptedArgs& args, int dtype, bool direct, hipStream_t stream) {
    if (args.adapters != nullptr) {
        const int status = launchLow<T>(args, stream);
        if (status != ZCGVS_OK) {
            return status;
        }
    }
    const ProductPlan plan = planProduct(args.rows, args.out_dim, args.dim, 1, dtype, 0, LargestTile::k128x128);
    return withTile<T, false, false, LargestTile::k128x128, false>(plan.shape, direct, [&](auto tile) {
        return launchTile<decltype(tile), Out>(args, stream);
    });
}

}  // namespace

}  // namespace zcgvs_hip

using namespace zcgvs_hip;

extern "C" {

int zcgvs_adapted_max_rank(void) { return kMaxRank; }

std::size_t zcgvs_adapted_projection_workspace_bytes(const zcgvs_adapted_desc* desc) {
    if (checkAdapted(desc) != ZCGVS_OK) {
        return 0;
    }
    clearError();
    return adaptedSpace(*desc).bytes;
}

int zcgvs_adapted_projection(const zcgvs_adapted_desc* desc, void* d_out, std::int64_t out_stride, int out_dtype,
                             void* d_workspace, std::size_t workspace_bytes, zcgvs_stream_t stream) {
    const int status = checkAdapted(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_adapted_desc& d = *desc;
    if (out_dtype != d.dtype && out_dtype != ZCGVS_DTYPE_F32) {
        return invalid("the output type is the operands' or float32");
    }
    const std::int64_t stride = rowStride(out_stride, d.out_dim);
    if (stride < d.out_dim) {
        return invalid("the output's row stride is smaller than out_dim");
    }
    if (d.rows == 0) {
        return clearError();
    }
    if (d_out == nullptr) {
        return invalid("null device pointer");
    }
    const AdaptedSpace space = adaptedSpace(d);
    if (hasAdapters(d) && (d_workspace == nullptr || workspace_bytes < space.bytes)) {
        return invalid("the workspace is too small");
    }
    if (hasAdapters(d) && !aligned16(d_workspace)) {
        return invalid("the workspace must be aligned to 16 bytes");
    }
    AdaptedArgs args{};
    args.x = d.x;
    args.x_stride = rowStride(d.x_stride, d.dim);
    args.weight = d.weight;
    args.weight_stride = rowStride(d.weight_stride, d.dim);
    args.rows = static_cast<int>(d.rows);
    args.dim = d.dim;
    args.out_dim = d.out_dim;
    args.out = d_out;
    args.out_stride = stride;
    const bool few = d.rows <= kFewRows ||
                     (hasAdapters(d) && d.rows <= 4096 && d.rows * d.dim * d.out_dim <= kFewProducts);
    const bool low_by_all =
        !hasAdapters(d) || (d.max_rank <= 16 && d.rows * d.max_rank * d.dim * elementBytes(d.dtype) <= kFewDownBytes);
    if (hasAdapters(d)) {
        char* workspace = static_cast<char*>(d_workspace);
        args.down = d.down;
        args.up = d.up;
        args.adapter_count = d.adapter_count;
        args.max_rank = d.max_rank;
        args.padded_rank = paddedRank(d.max_rank);
        args.ranks = d.ranks;
        args.scales = d.scales;
        args.low = workspace + space.low;
        args.low_scale = reinterpret_cast<float*>(workspace + space.low_scale);
    }
    if (hasAdapters(d) && !few) {
        SortInput input{};
        input.keys = d.adapter_ids;
        input.count = args.rows;
        input.key_end = d.adapter_count;
        input.skipped = -1;
        input.raw = true;
        const int sorted = sortPairs(input, static_cast<char*>(d_workspace) + space.sort, &args.adapters, &args.order,
                                     NoSideWork{}, toStream(stream));
        if (sorted != ZCGVS_OK) {
            return sorted;
        }
    }
    const bool direct = directRows(d.x, args.x_stride, d.dim, d.dtype) &&
                        directRows(d.weight, args.weight_stride, d.dim, d.dtype);
    const int launched = withElement(d.dtype, [&](auto in) {
        using T = decltype(in);
        return withElement(out_dtype, [&](auto element) {
            using Out = decltype(element);
            if constexpr (std::is_same_v<Out, T> || std::is_same_v<Out, float>) {
                if (few) {
                    const dim3 grid(static_cast<unsigned>(divideUp(d.out_dim, 16)),
                                    static_cast<unsigned>(divideUp(d.rows, kFewRows)));
                    const int* ids = hasAdapters(d) ? d.adapter_ids : nullptr;
                    if (low_by_all) {
                        adaptedFewKernel<T, Out, true><<<grid, kFewThreads, 0, toStream(stream)>>>(args, ids);
                    } else {
                        lowFewKernel<T><<<dim3(static_cast<unsigned>(d.rows), static_cast<unsigned>(divideUp(d.max_rank, 16))),
                                          kLowFewThreads, 0, toStream(stream)>>>(args, ids);
                        ZCGVS_LAUNCH_CHECK("adapted projection");
                        adaptedFewKernel<T, Out, false><<<grid, kFewThreads, 0, toStream(stream)>>>(args, ids);
                    }
                    ZCGVS_LAUNCH_CHECK("adapted projection");
                    return static_cast<int>(ZCGVS_OK);
                }
                args.parts = kParts<T, Out>;
                return launchAdapted<T, Out>(args, d.dtype, direct, toStream(stream));
            } else {
                return static_cast<int>(ZCGVS_ERR_INVALID_ARGUMENT);  // refused above
            }
        });
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

}  // extern "C"
