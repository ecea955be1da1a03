// Which tile a matrix product of the embedding-model operators takes, and over how many splits of k.
#pragma once

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.hpp"
#include "elements.hpp"
#include "matrix_split.hpp"
#include "matrix_tile.hpp"

namespace zcgvs_hip {

enum class TileShape { k256x256, k256x192, k128x128, k64x64 };

struct ProductPlan {
    TileShape shape;
    int splits;
    double us;  // the time it is planned for
};

namespace {

// a launch has less than 2^32 threads, of up to 1024 a block
constexpr long long kMaxBlocks = (1ll << 22) - 1;

inline std::int64_t rowStride(std::int64_t stride, int length) { return stride == 0 ? length : stride; }

inline int divideUp(std::int64_t a, std::int64_t b) { return static_cast<int>((a + b - 1) / b); }

// Rows that the 16-byte copies can read: whole aligned chunks.
inline bool directRows(const void* base, std::int64_t stride, int length, int dtype) {
    return alignedRows(base, stride, dtype, 16) && static_cast<std::int64_t>(length) * elementBytes(dtype) % 16 == 0;
}

// The largest tile a kernel is built with: those of 256 rows have 16 wavefronts of 128 registers.
enum class LargestTile { k256x256, k256x192, k128x128 };

// Rows that are no whole 16-byte chunks go through registers, for which the tiles of 256 rows have too few; they are
// planned for the tiles they take. (Gradient of 16,384 rows 767 -> 2047 bfloat16 825 us, 870 us with the splits of the
// larger tiles; rows of 768 and 2048 356 us. The stage times are those of whole chunks.)
inline LargestTile largestTile(LargestTile largest, bool direct) { return direct ? largest : LargestTile::k128x128; }

// Values of k of a stage, of every type.
constexpr int kPlanStageK = 64;

// The plan of `count` products of m x n over k: the least time of the CU with the most tiles. A stage of a
// tile takes alone_us, and more_us longer for every further tile that the CU holds beside it (as many as
// `together`); fixed_us are the tile's first loads and its results. Measured, 16-bit: 128 stages of one
// 64 x 64 tile a CU 58 us, of four 89 us; of one 128 x 128 tile 83 us, of two 111 us; 256 x 256 1.6 us a stage
// at any length (1326 TFLOP/s over 8192). float32: of one 64 x 64 tile 190 us, of three 330 us; of one
// 128 x 128 tile 343 us (198 TFLOP/s).
// Splits write and read float32 sums of the whole product once each, at the rate of a copy; they come in
// multiples of split_step, and only where a workspace can be had (split_step 0: one split).
inline ProductPlan planProduct(std::int64_t m, std::int64_t n, std::int64_t k, int count, int dtype, int split_step,
                               LargestTile largest) {
    struct Shape {
        TileShape shape;
        int m, n, together;
        double alone_us, more_us, fixed_us;
    };
    constexpr Shape kShapes16[] = {
        {TileShape::k256x256, 256, 256, 1, 1.60, 0.0, 6.0},
        {TileShape::k256x192, 256, 192, 1, 1.40, 0.0, 4.5},
        {TileShape::k128x128, 128, 128, 2, 0.65, 0.21, 3.0},
        {TileShape::k64x64, 64, 64, 4, 0.45, 0.083, 2.0},
    };
    constexpr Shape kShapes32[] = {
        {TileShape::k128x128, 128, 128, 1, 2.70, 0.0, 3.0},
        {TileShape::k64x64, 64, 64, 3, 1.50, 0.55, 3.0},
    };
    const bool wide = dtype == ZCGVS_DTYPE_F32;
    const Shape* shapes = wide ? kShapes32 : kShapes16;
    const int shape_count = wide ? 2 : 4;
    const std::int64_t stages = (k + kPlanStageK - 1) / kPlanStageK;
    const std::int64_t units = deviceComputeUnits();
    ProductPlan best{TileShape::k64x64, 1, 0.0};
    for (int i = 0; i < shape_count; ++i) {
        const Shape& s = shapes[i];
        if ((s.m > 128 && largest == LargestTile::k128x128) || (s.n > 192 && largest != LargestTile::k256x256)) {
            continue;
        }
        const std::int64_t tiles = count * ((m + s.m - 1) / s.m) * ((n + s.n - 1) / s.n);
        const int most = split_step == 0 ? 1 : 32;
        for (int splits = 1; splits <= most; splits += splits == 1 && split_step > 1 ? split_step - 1 : std::max(split_step, 1)) {
            if (splits > 1 && stages < 4 * splits) {
                break;
            }
            const std::int64_t on_unit = (tiles * splits + units - 1) / units;
            const std::int64_t rounds = on_unit / s.together;
            const std::int64_t rest = on_unit % s.together;
            const double length = static_cast<double>((stages + splits - 1) / splits);
            double us = static_cast<double>(rounds) * (length * (s.alone_us + (s.together - 1) * s.more_us) + s.fixed_us);
            us += rest > 0 ? length * (s.alone_us + static_cast<double>(rest - 1) * s.more_us) + s.fixed_us : 0.0;
            if (splits > 1) {
                us += 4.0 + 8.0 * static_cast<double>(count) * static_cast<double>(m) * static_cast<double>(n) * splits / 4.5e6;
            }
            if (best.us == 0.0 || us < best.us) {
                best = {s.shape, splits, us};
            }
        }
    }
    return best;
}

// Blocks of a launch whose blocks form several tiles each: two to a CU that holds one at a time, so that
// their results and first loads fall at different times.
inline int persistentBlocks(TileShape shape) {
    return shape == TileShape::k256x256 || shape == TileShape::k256x192 ? 2 * ((deviceComputeUnits() + 7) / 8 * 8)
                                                                          : static_cast<int>(kMaxBlocks) / 8 * 8;
}

// Calls body(Tile{}) with a shape's tile; loads past the registers where the rows allow (16-bit). kPaired: every
// wavefront has an even number of column blocks (256 x 192 by 8 x 2 wavefronts instead of 4 x 4).
template <typename T, bool kTurnedA, bool kTurnedB, LargestTile kLargest, bool kPaired, typename Body>
int withTile(TileShape shape, bool direct, Body&& body) {
    if constexpr (std::is_same_v<T, float>) {
        return shape == TileShape::k64x64 ? body(SplitTile<64, 64, 2, 2, kTurnedA, kTurnedB>{})
                                          : body(SplitTile<128, 128, 4, 4, kTurnedA, kTurnedB>{});
    } else {
        if (!direct) {
            return shape == TileShape::k64x64 ? body(MatrixTile<T, 64, 64, 2, 2, kTurnedA, kTurnedB, false>{})
                                              : body(MatrixTile<T, 128, 128, 2, 4, kTurnedA, kTurnedB, false>{});
        }
        if constexpr (kLargest == LargestTile::k256x256) {
            if (shape == TileShape::k256x256) {
                return body(MatrixTile<T, 256, 256, 4, 4, kTurnedA, kTurnedB, true>{});
            }
        }
        if constexpr (kLargest != LargestTile::k128x128) {
            if (shape == TileShape::k256x192) {
                return body(MatrixTile<T, 256, 192, kPaired ? 8 : 4, kPaired ? 2 : 4, kTurnedA, kTurnedB, true>{});
            }
        }
        return shape == TileShape::k64x64 ? body(MatrixTile<T, 64, 64, 2, 2, kTurnedA, kTurnedB, true>{})
                                          : body(MatrixTile<T, 128, 128, 2, 4, kTurnedA, kTurnedB, true>{});
    }
}

}  // namespace
}  // namespace zcgvs_hip
