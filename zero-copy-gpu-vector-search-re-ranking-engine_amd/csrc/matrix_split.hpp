// Tiled products of float32 operands on the bf16 matrix cores, in the interface of MatrixTile.
//
// A float32 value is the sum of three bf16 values, exactly: itself rounded to bf16, what is left rounded to
// bf16, and the rest. Rounded to nearest, each part is at most 2^-8 of the one before and has either sign. x y is
// formed as the six products of parts whose size is at least 2^-16 of it; the other three are together below
// 2^-24 (1 + 2^-8) of it, half of what a float32 sum may round away, and no sign is preferred. (Parts cut off
// instead have the value's sign, and the three products left out would reach 2^-21, all in one direction.)
// Six v_mfma_f32_16x16x32_bf16 take 3/8 of the time of the eight v_mfma_f32_16x16x4_f32 that they stand for
// (whose rate bounds a float32 product at 150 TFLOP/s).
// A stage's products are summed by themselves and then added to the tile's sums: the matrix cores' additions
// do not round to nearest, and cost a sum over 8192 a relative 1.5e-6 (2-norm) where all of them go to one sum;
// like this it is 2.4e-7, at up to 4% of the time (float32 matrix instructions: 1.7e-6).
// Operands are split once, between the registers that they are loaded into and LDS, where the three parts
// are planes of the 16-bit layouts of matrix_tile.hpp; a stage is 64 values of k. The next stage is on its way
// into registers while this one is multiplied. Loads take any alignment. Measured, gated products of 4096 rows,
// 8192 -> 2048: 128 x 128 tiles 195 TFLOP/s, 64 x 64 149, float32 matrix instructions 127.
// Infinite operands give NaN (which the last part of an infinity is), and values below about
// 2^-110 lose bits.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "matrix_tile.hpp"

namespace zcgvs_hip {

constexpr int kSplitParts = 3;
constexpr float kLargestPart = 3.38953139e38f;  // the largest finite bf16 value

template <int kRows, bool kTurned, int kThreads>
struct SplitLoader {
    using Plane = StageLoader<__bf16, kRows, kTurned, false, kThreads>;
    static constexpr int kValues = 8;  // of a copy: 16 bytes of every plane
    static constexpr int kCopies = Plane::kCopies;
    static constexpr int kBytes = kSplitParts * Plane::kBytes;
    static constexpr int kStage = kStageK<__bf16>;
    static_assert(Plane::kEven, "a stage splits over the threads");

    const float* src[kCopies];
    std::int64_t step;  // values from stage to stage
    int k_left;
    int columns_left;
    float held[kCopies][kValues];

    template <typename RowOf>
    __device__ __forceinline__ void begin(RowOf&& row_of, std::int64_t stride, int columns, int k_total) {
        k_left = k_total;
        columns_left = columns;
        step = kTurned ? stride * kStage : kStage;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            int row, chunk;
            Plane::placeOf(i, row, chunk);
            src[i] = kTurned ? row_of(0) + row * stride + chunk * kValues : row_of(row) + chunk * kValues;
        }
    }
    __device__ __forceinline__ void moveOn(std::int64_t bytes, int k_total) {
        const std::int64_t by = bytes / static_cast<std::int64_t>(sizeof(float)) - (k_total / kStage) * step;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            src[i] += by;
        }
        k_left = k_total;
    }
    __device__ __forceinline__ void fetch() {
        if (k_left >= kStage && (!kTurned || columns_left >= kRows)) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                __builtin_memcpy(&held[i][0], src[i], 16);
                __builtin_memcpy(&held[i][4], src[i] + 4, 16);
                src[i] += step;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                int row, chunk;
                Plane::placeOf(i, row, chunk);
                const int valid = kTurned ? (row < k_left ? columns_left - chunk * kValues : 0) : k_left - chunk * kValues;
#pragma unroll
                for (int e = 0; e < kValues; ++e) {
                    held[i][e] = 0.0f;
                    if (e < valid) {
                        held[i][e] = src[i][e];
                    }
                }
                src[i] += k_left >= kStage ? step : 0;
            }
        }
        k_left -= kStage;
    }
    __device__ __forceinline__ void put(std::uint8_t* stage) const {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            u32x4 part[kSplitParts];
#pragma unroll
            for (int e = 0; e < kValues; e += 2) {
                float rest[2] = {held[i][e], held[i][e + 1]};
#pragma unroll
                for (int p = 0; p < kSplitParts; ++p) {
                    f32x2 from = {rest[0], rest[1]};
                    if (p == 0) {  // a finite value's first part stays finite
                        from = f32x2{__builtin_amdgcn_fmed3f(rest[0], -kLargestPart, kLargestPart),
                                     __builtin_amdgcn_fmed3f(rest[1], -kLargestPart, kLargestPart)};
                    }
                    const std::uint32_t both = __builtin_bit_cast(std::uint32_t, __builtin_convertvector(from, bf16x2));
                    part[p][e / 2] = both;
                    rest[0] -= __uint_as_float(both << 16);
                    rest[1] -= __uint_as_float(both & 0xFFFF0000u);
                }
            }
#pragma unroll
            for (int p = 0; p < kSplitParts; ++p) {
                *reinterpret_cast<u32x4*>(stage + p * Plane::kBytes +
                                          (i * kThreads + static_cast<int>(threadIdx.x)) * 16) = part[p];
            }
        }
    }
};

template <int kTileM, int kTileN, int kSplitM, int kSplitN, bool kTurnedA, bool kTurnedB>
struct SplitTile {
    using T = float;
    // the tile of the same shape whose stages hold float32 as it is
    using StageTile = MatrixTile<float, kTileM, kTileN, kSplitM, kSplitN, false, false, false>;
    static constexpr int kM = kTileM;
    static constexpr int kN = kTileN;
    static constexpr int kWavesM = kSplitM;
    static constexpr int kWavesN = kSplitN;
    static constexpr int kThreads = kWavesM * kWavesN * kWave;
    static constexpr int kBlocksM = kM / kWavesM / 16;
    static constexpr int kBlocksN = kN / kWavesN / 16;
    using SideA = SplitLoader<kM, kTurnedA, kThreads>;
    using SideB = SplitLoader<kN, kTurnedB, kThreads>;
    static constexpr int kLdsBytes = SideA::kBytes + SideB::kBytes;
    using Sum = f32x4;
    using Sums = Sum[kBlocksM][kBlocksN];

    static __device__ __forceinline__ int waveM() { return StageTile::waveM(); }
    static __device__ __forceinline__ int waveN() { return StageTile::waveN(); }
    static __device__ __forceinline__ void clear(Sums& sums) { StageTile::clear(sums); }

    struct Loads {
        SideA a;
        SideB b;

        template <typename RowA, typename RowB>
        __device__ __forceinline__ void begin(RowA&& row_a, std::int64_t stride_a, int columns_a, RowB&& row_b,
                                              std::int64_t stride_b, int columns_b, int k_total) {
            a.begin(row_a, stride_a, columns_a, k_total);
            b.begin(row_b, stride_b, columns_b, k_total);
        }
        __device__ __forceinline__ void moveOn(std::int64_t a_bytes, std::int64_t b_bytes, int k_total) {
            a.moveOn(a_bytes, k_total);
            b.moveOn(b_bytes, k_total);
        }
        // Reads the first stage after begin() or moveOn() into registers.
        __device__ __forceinline__ void start(std::uint8_t*) {
            a.fetch();
            b.fetch();
        }
        __device__ __forceinline__ void land() {}
    };

    static __device__ __forceinline__ void multiplySplit(const std::uint8_t* stage, Sums& sums) {
        using Fragments = Fragment<__bf16>::type;
        const std::uint8_t* stage_b = stage + SideA::kBytes;
#pragma unroll
        for (int t = 0; t < kStageSteps; ++t) {
            Fragments a[kBlocksM][kSplitParts], b[kBlocksN][kSplitParts];
#pragma unroll
            for (int p = 0; p < kSplitParts; ++p) {
#pragma unroll
                for (int i = 0; i < kBlocksM; ++i) {
                    a[i][p] = SideA::Plane::read(stage + p * SideA::Plane::kBytes, waveM() * kBlocksM + i, t);
                }
#pragma unroll
                for (int j = 0; j < kBlocksN; ++j) {
                    b[j][p] = SideB::Plane::read(stage_b + p * SideB::Plane::kBytes, waveN() * kBlocksN + j, t);
                }
            }
            // the small products first; neighbouring instructions write different sums
#pragma unroll
            for (int size = kSplitParts - 1; size >= 0; --size) {
#pragma unroll
                for (int p = 0; p <= size; ++p) {
#pragma unroll
                    for (int i = 0; i < kBlocksM; ++i) {
#pragma unroll
                        for (int j = 0; j < kBlocksN; ++j) {
                            sums[i][j] = multiplyAdd(b[j][p], a[i][size - p], sums[i][j]);
                        }
                    }
                }
            }
        }
    }

    template <typename Next>
    static __device__ __forceinline__ void accumulate(std::uint8_t* lds, Loads& loads, int k_total, Sums& sums,
                                                      Next&& next) {
        const int stages = (k_total + SideA::kStage - 1) / SideA::kStage;
        for (int s = 0; s < stages; ++s) {
            __syncthreads();  // the stage before has been read
            loads.a.put(lds);
            loads.b.put(lds + SideA::kBytes);
            __syncthreads();
            if (s + 1 < stages) {
                loads.a.fetch();
                loads.b.fetch();
            } else {
                next();
            }
            Sums stage;
            clear(stage);
            multiplySplit(lds, stage);
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i) {
#pragma unroll
                for (int j = 0; j < kBlocksN; ++j) {
                    sums[i][j] += stage[i][j];
                }
            }
        }
    }
};

}  // namespace zcgvs_hip
