// Tiled matrix products on the matrix cores for the embedding-model operators.
//
// A workgroup forms a kM x kN tile of C[m, n] = sum_k A[m, k] B[n, k] in float32 accumulators. Each side
// comes in one of two layouts: rows whose k are neighbours ("plain": the activations and weights of
// a forward product), or k-rows whose m (or n) are neighbours ("turned": what the gradients contract).
// A stage is 128 bytes of k a row (64 16-bit values); two stages are in LDS, one being read by the matrix
// cores while the next arrives. float32 products are those of matrix_split.hpp, on planes of the same layouts;
// of float32 itself this file holds what multiplies one plain stage.
//
// LDS layout. A plain side's row r takes 128 bytes; its 16-byte chunk c stands in slot
// c ^ ((r >> 1) & 7), so that the 16 rows of one ds_read_b128 fall on 16 different 16-byte columns of
// the 256 bytes that the 64 banks hold. A turned side's k-row takes its m (or n) in order, in granules
// of 32 bytes whose place is exchanged by the k-row's number, read by ds_read_b64_tr_b16, which hands lane i
// of 16 the column i of four k-rows.
//
// Matrix instructions. 16-bit: v_mfma_f32_16x16x32, float32: v_mfma_f32_16x16x4. The first operand
// holds B's rows and the second A's, so that lane l of a 16 x 16 result has the four neighbouring columns
// n = 4 (l / 16) + e of row m = l % 16 and can store them together. Lane group h = l / 16 holds the
// 16 bytes of chunk 4 t + h in step t, on both sides: every k meets itself whatever the order.
//
// Bounds. Past a side's end its last row (plain) or chunk of columns (turned) is read again; those
// only reach results that are not stored. k past the end is read as zeros on both sides.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.hpp"
#include "elements.hpp"
#include "lds_copy.hpp"

namespace zcgvs_hip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kStageBytes = 128;  // of k in a plain side's row
constexpr int kStageSteps = 2;    // matrix instruction steps of 64 bytes of k

template <typename T>
constexpr int kStageK = kStageBytes / static_cast<int>(sizeof(T));
template <typename T>
constexpr int kChunk = 16 / static_cast<int>(sizeof(T));  // values in 16 bytes

template <typename T>
struct Fragment {
    typedef T type __attribute__((ext_vector_type(kChunk<T>)));
};

__device__ __forceinline__ f32x4 multiplyAdd(Fragment<_Float16>::type b, Fragment<_Float16>::type a, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(b, a, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiplyAdd(Fragment<__bf16>::type b, Fragment<__bf16>::type a, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiplyAdd(Fragment<float>::type b, Fragment<float>::type a, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(b[e], a[e], c, 0, 0, 0);
    }
    return c;
}

// What lanes read in the place of k past the end.
static __device__ const u32x4 zero_chunk = {0u, 0u, 0u, 0u};

// One side of a product: `rows` rows from `base` on, `stride` values apart (turned: `rows` columns of
// k-rows that are `stride` values apart).
template <typename T>
struct MatrixSide {
    const T* base;
    std::int64_t stride;
    int rows;
};

// Moves one side's stages into LDS: kRows rows of a tile, by a workgroup of kThreads threads.
// kDirect: 16-byte copies past the registers; rows start at multiples of 16 bytes and hold whole
// chunks. Otherwise through registers, from any alignment.
template <typename T, int kRows, bool kTurned, bool kDirect, int kThreads>
struct StageLoader {
    // 16-byte copies of a stage, by wavefronts of 64; where they do not split evenly the last ones have
    // one round less
    static constexpr int kWaves = kThreads / kWave;
    static constexpr int kWaveCopies = kRows * (kStageBytes / 16) / kWave;
    static constexpr int kCopies = (kWaveCopies + kWaves - 1) / kWaves;
    static constexpr bool kEven = kWaveCopies % kWaves == 0;
    static constexpr int kBytes = kRows * kStageBytes;
    static_assert(sizeof(T) == 2 || !kTurned, "a turned side is 16-bit");

    static __device__ __forceinline__ bool hasCopy(int i) {
        return kEven || i + 1 < kCopies ||
               i * kWaves + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave) < kWaveCopies;
    }

    static constexpr int kSlots = kRows * static_cast<int>(sizeof(T)) / 16;  // 16-byte chunks of a turned k-row

    const char* src[kCopies];
    std::int64_t step;  // bytes from stage to stage
    int k_left;         // from the next stage to load on
    int columns_left;   // that exist from the tile's first on (turned, not direct)
    u32x4 held[kDirect ? 1 : kCopies];

    // Row (plain) or k-row (turned) and chunk of the i-th copy of this thread.
    static __device__ __forceinline__ void placeOf(int i, int& row, int& chunk) {
        const int slot = i * kThreads + static_cast<int>(threadIdx.x);
        if constexpr (kTurned) {
            row = slot / kSlots;
            chunk = sourceChunk(row, slot % kSlots);
        } else {
            row = slot / 8;
            chunk = (slot % 8) ^ ((row >> 1) & 7);
        }
    }
    // k of the i-th copy's first value within a stage.
    static __device__ __forceinline__ int kOf(int i) {
        int row, chunk;
        placeOf(i, row, chunk);
        return kTurned ? row : chunk * kChunk<T>;
    }

    // row_of(r): the tile's row r of a plain side, at k = 0. A turned side starts at its tile's first
    // column, of which `columns` (at least one) exist; direct copies read the last chunk again past them.
    template <typename RowOf>
    __device__ __forceinline__ void begin(RowOf&& row_of, std::int64_t stride, int columns, int k_total) {
        k_left = k_total;
        columns_left = columns;
        step = kTurned ? stride * kStageK<T> * static_cast<std::int64_t>(sizeof(T)) : kStageBytes;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            int row, chunk;
            placeOf(i, row, chunk);
            if constexpr (kTurned) {
                const int from = kDirect ? min(chunk, (columns - 1) / kChunk<T>) : chunk;
                src[i] = reinterpret_cast<const char*>(row_of(0) + row * stride + from * kChunk<T>);
            } else {
                src[i] = reinterpret_cast<const char*>(row_of(row) + chunk * kChunk<T>);
            }
        }
    }

    // From the end of k (whose last stage, where it is not a whole one, does not advance) to k = 0 of an
    // operand `bytes` further on.
    __device__ __forceinline__ void moveOn(std::int64_t bytes, int k_total) {
        const std::int64_t by = bytes - (k_total / kStageK<T>)*step;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            src[i] += by;
        }
        k_left = k_total;
    }

    // Which chunk of k-row k stands in `slot` of its LDS row (an exchange, so also the reverse).
    static __device__ __forceinline__ int sourceChunk(int k, int slot) { return slot ^ (2 * turnOf(k)); }
    static __device__ __forceinline__ int turnOf(int k) { return ((k & 3) | ((k >> 1) & 4)) & (kRows / 16 - 1); }

    // Starts the next stage's copies into `stage` (direct).
    __device__ __forceinline__ void issue(const std::uint8_t* stage) {
        const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
        const std::uint32_t base = ldsAddress(stage) + static_cast<std::uint32_t>(wave * kWave * 16);
        if (k_left >= kStageK<T>) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                if (hasCopy(i)) {
                    copySharedToLds(src[i], __builtin_amdgcn_readfirstlane(base + i * kThreads * 16));
                }
                src[i] += step;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const char* from = kOf(i) < k_left ? src[i] : reinterpret_cast<const char*>(&zero_chunk);
                if (hasCopy(i)) {
                    copySharedToLds(from, __builtin_amdgcn_readfirstlane(base + i * kThreads * 16));
                }
            }
        }
        k_left -= kStageK<T>;
    }

    // Reads the next stage into registers, and later writes it to `stage` (not direct).
    __device__ __forceinline__ void fetch() {
        if (k_left >= kStageK<T> && (!kTurned || columns_left >= kRows)) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                if (hasCopy(i)) {
                    __builtin_memcpy(&held[i], src[i], 16);
                }
                src[i] += step;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                int row, chunk;
                placeOf(i, row, chunk);
                int valid = kTurned ? (row < k_left ? columns_left - chunk * kChunk<T> : 0) : k_left - chunk * kChunk<T>;
                valid = hasCopy(i) ? valid : 0;
                typename Fragment<T>::type v = {};
                const T* from = reinterpret_cast<const T*>(src[i]);
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
                held[i] = __builtin_bit_cast(u32x4, v);
                src[i] += k_left >= kStageK<T> ? step : 0;
            }
        }
        k_left -= kStageK<T>;
    }
    __device__ __forceinline__ void put(std::uint8_t* stage) const {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            if (hasCopy(i)) {
                *reinterpret_cast<u32x4*>(stage + (i * kThreads + static_cast<int>(threadIdx.x)) * 16) = held[i];
            }
        }
    }

    // The calling lane's fragment of rows 16 block .. 16 block + 15 in step t.
    static __device__ __forceinline__ typename Fragment<T>::type read(const std::uint8_t* stage, int block, int t) {
        const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
        const int r16 = lane & 15;
        const int h = lane >> 4;
        if constexpr (!kTurned) {
            const int slot = (4 * t + h) ^ ((r16 >> 1) & 7);
            return *reinterpret_cast<const typename Fragment<T>::type*>(stage + (16 * block + r16) * kStageBytes +
                                                                        16 * slot);
        } else {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) s16x4* LdsPointer;
            const int k = 32 * t + 8 * h + (r16 >> 2);
            const std::uint32_t offset =
                static_cast<std::uint32_t>(k * kRows * 2 + ((block ^ turnOf(k)) * 32) + (r16 & 3) * 8);
            const std::uint32_t address = ldsAddress(stage) + offset;
            const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsPointer>(address));
            const s16x4 high =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsPointer>(address + 4 * kRows * 2));
            const s16x8 both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(typename Fragment<T>::type, both);
        }
    }
};

// A tile's shape: kM x kN by kWavesM x kWavesN wavefronts, each (kM / kWavesM) x (kN / kWavesN).
template <typename Element, int kTileM, int kTileN, int kSplitM, int kSplitN, bool kTurnedA, bool kTurnedB,
          bool kDirectLoads>
struct MatrixTile {
    using T = Element;
    using StageTile = MatrixTile;  // whose multiplyStage() takes one stage of T
    static constexpr int kM = kTileM;
    static constexpr int kN = kTileN;
    static constexpr int kWavesM = kSplitM;
    static constexpr int kWavesN = kSplitN;
    static constexpr int kThreads = kWavesM * kWavesN * kWave;
    static constexpr int kBlocksM = kM / kWavesM / 16;
    static constexpr int kBlocksN = kN / kWavesN / 16;
    static constexpr bool kDirect = kDirectLoads;
    using SideA = StageLoader<T, kM, kTurnedA, kDirect, kThreads>;
    using SideB = StageLoader<T, kN, kTurnedB, kDirect, kThreads>;
    static constexpr int kStageLds = SideA::kBytes + SideB::kBytes;
    static constexpr int kLdsBytes = 2 * kStageLds;

    using Sums = f32x4[kBlocksM][kBlocksN];

    static __device__ __forceinline__ int waveId() {
        return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    }
    static __device__ __forceinline__ int waveM() { return waveId() / kWavesN; }
    static __device__ __forceinline__ int waveN() { return waveId() % kWavesN; }

    static __device__ __forceinline__ void clear(Sums& sums) {
#pragma unroll
        for (int i = 0; i < kBlocksM; ++i) {
#pragma unroll
            for (int j = 0; j < kBlocksN; ++j) {
                sums[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
    }

    static __device__ __forceinline__ void multiplyStage(const std::uint8_t* stage, Sums& sums) {
        const std::uint8_t* stage_b = stage + SideA::kBytes;
        const int block_m = waveM() * kBlocksM;
        const int block_n = waveN() * kBlocksN;
#pragma unroll
        for (int t = 0; t < kStageSteps; ++t) {
            typename Fragment<T>::type a[kBlocksM], b[kBlocksN];
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i) {
                a[i] = SideA::read(stage, block_m + i, t);
            }
#pragma unroll
            for (int j = 0; j < kBlocksN; ++j) {
                b[j] = SideB::read(stage_b, block_n + j, t);
            }
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i) {
#pragma unroll
                for (int j = 0; j < kBlocksN; ++j) {
                    sums[i][j] = multiplyAdd(b[j], a[i], sums[i][j]);
                }
            }
        }
    }

    // The loads of both sides. A workgroup that forms several tiles (or a tile of several products)
    // starts the next one's first stage while it multiplies the last stage of the one before, so that
    // it arrives behind that stage and the tile's results.
    struct Loads {
        SideA a;
        SideB b;
        int buffer = 0;       // of the next stage
        bool landed = false;  // the next stage is known to have arrived

        template <typename RowA, typename RowB>
        __device__ __forceinline__ void begin(RowA&& row_a, std::int64_t stride_a, int columns_a, RowB&& row_b,
                                              std::int64_t stride_b, int columns_b, int k_total) {
            a.begin(row_a, stride_a, columns_a, k_total);
            b.begin(row_b, stride_b, columns_b, k_total);
        }
        __device__ __forceinline__ void issue(std::uint8_t* lds, int to) {
            a.issue(lds + to * kStageLds);
            b.issue(lds + to * kStageLds + SideA::kBytes);
        }
        // Goes on with a second product over the same k, its operands so many bytes from the first's.
        __device__ __forceinline__ void moveOn(std::int64_t a_bytes, std::int64_t b_bytes, int k_total) {
            a.moveOn(a_bytes, k_total);
            b.moveOn(b_bytes, k_total);
        }
        // Starts the first stage after begin() or moveOn().
        __device__ __forceinline__ void start(std::uint8_t* lds) {
            if constexpr (kDirect) {
                issue(lds, buffer);
            }
        }
        // Waits for a started first stage; called before a tile's results are stored, so that the next
        // tile does not wait for the stores.
        __device__ __forceinline__ void land() {
            if constexpr (kDirect) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                landed = true;
            }
        }
    };

    // Adds the products over k_total values of k to `sums`, from the stage that `loads` has started on.
    // next(): called in the last stage; may begin and start what comes after (`loads.start(lds)`).
    // Every thread of the workgroup calls it; `lds` holds kLdsBytes.
    template <typename Next>
    static __device__ __forceinline__ void accumulate(std::uint8_t* lds, Loads& loads, int k_total, Sums& sums,
                                                      Next&& next) {
        const int stages = (k_total + kStageK<T> - 1) / kStageK<T>;
        if constexpr (kDirect) {
            for (int s = 0; s < stages; ++s) {
                // this stage's copies have arrived, and every wavefront has read the other buffer
                if (loads.landed) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    loads.landed = false;
                } else {
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                }
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                const std::uint8_t* here = lds + loads.buffer * kStageLds;
                loads.buffer ^= 1;
                if (s + 1 < stages) {
                    loads.issue(lds, loads.buffer);
                } else {
                    next();
                }
                multiplyStage(here, sums);
            }
        } else {
            __syncthreads();  // the LDS may still be read for the tile before
            loads.a.fetch();
            loads.b.fetch();
            loads.a.put(lds);
            loads.b.put(lds + SideA::kBytes);
            __syncthreads();
            for (int s = 0; s < stages; ++s) {
                std::uint8_t* here = lds + (s & 1) * kStageLds;
                std::uint8_t* other = lds + ((s & 1) ^ 1) * kStageLds;
                if (s + 1 < stages) {
                    loads.a.fetch();
                    loads.b.fetch();
                }
                multiplyStage(here, sums);
                if (s + 1 < stages) {
                    loads.a.put(other);
                    loads.b.put(other + SideA::kBytes);
                }
                __syncthreads();
            }
            next();
        }
    }
};

// The index-th tile (m, n) of a launch whose block b forms the tiles b, b + gridDim.x, ... (a multiple of
// kXcds apart where there are several). Blocks of one XCD (every eighth one) take neighbouring tiles, in
// bands of kBandRows tile rows walked column by column, so that an XCD's blocks share rows of both sides in
// its L2.
constexpr int kXcds = 8;
constexpr int kBandRows = 4;

__device__ __forceinline__ void tileOf(int index, int tiles_m, int tiles_n, int& m, int& n) {
    const int total = tiles_m * tiles_n;
    const int xcd = index % kXcds;
    const int whole = total / kXcds;
    const int more = total % kXcds;  // the first `more` XCDs have one tile more
    const int tile = xcd * whole + min(xcd, more) + index / kXcds;
    const int band_tiles = kBandRows * tiles_n;
    const int band = tile / band_tiles;
    const int in_band = tile - band * band_tiles;
    const int rows = min(kBandRows, tiles_m - band * kBandRows);
    m = band * kBandRows + in_band % rows;
    n = in_band / rows;
}

// Reads four neighbouring values of one row of which `left` exist; the others are zeros.
template <typename T>
__device__ __forceinline__ f32x4 loadFour(const T* from, int left) {
    f32x4 value = {0.0f, 0.0f, 0.0f, 0.0f};
    if (left >= 4) {
        float v[4];
        loadPack(from, v);
        value = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e < left) {
                value[e] = static_cast<float>(from[e]);
            }
        }
    }
    return value;
}

// Stores four neighbouring results of one row; `left` of them exist.
template <typename Out>
__device__ __forceinline__ void storeFour(const f32x4& value, Out* to, int left) {
    if (left >= 4) {
        const float v[4] = {value[0], value[1], value[2], value[3]};
        storePack(v, to);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e < left) {
                to[e] = static_cast<Out>(value[e]);
            }
        }
    }
}

}  // namespace zcgvs_hip
