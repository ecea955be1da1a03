// The gated half of a feed-forward block and its gradient.
//
//     g = x gate^T,  u = x up^T,  out = act(g) * u
//     dg = d_out * u * act'(g),  du = d_out * act(g)
//     x_gradient = dg gate + du up,  gate_gradient = dg^T x,  up_gradient = du^T x
//
// Forward: 4 rows dim hidden operations in one kernel. A tile's columns are half gate rows and half up
// rows, dealt so that each wavefront holds g and u of the same elements in the same lanes: the
// activation and the product stay in registers and g and u never exist in memory.
// Gradient: the same kernel forms g and u again and writes dg and du (4 rows dim hidden operations
// instead of reading and writing two stored tensors), then one product over hidden and two over rows,
// twelve rows dim hidden operations in all.
//
// dg and du are rounded to the operands' type where they are written, once each, as a model of that type stores them:
// the matrix instructions take 16-bit operands, and their sums are float32. A gradient's relative error (2-norm against
// 64 bits) is then 2.3e-3 in bfloat16 and 2.9e-4 in float16, of which 1.7e-3 and 2.1e-4 are the result's own rounding.
// A second part of dg and du would take that away, for twice the operations of the three products over them and
// twice the bytes between (16,384 rows of 768, hidden 2048: about 190 us beside the present 350). In float16 a value
// beyond 65504 becomes an infinity there. float32 keeps all digits.
//
// Bound by the matrix cores where there are many rows. Measured: 8192 rows 1024 -> 4096 bfloat16 119-125 us
// (1100-1155 TFLOP/s; a library product of that size without the activation 113-115 us); the gradient of 16,384
// rows of 768, hidden 2048: dg and du 138 us (103 GFLOP, and 200 MB in bursts between the tiles), dx 93, the
// weights' 101. One row 768 -> 2048 takes 6.6 us, a launch's time (float32: 19.7, operands split for 64 rows).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "activation.hpp"
#include "common.hpp"
#include "elements.hpp"
#include "matrix_join.hpp"
#include "matrix_plan.hpp"
#include "matrix_tile.hpp"

namespace zcgvs_hip {

namespace {

struct GatedArgs {
    const void* x;
    std::int64_t x_stride;
    const void* gate;
    const void* up;
    std::int64_t weight_stride;
    int rows;
    int dim;
    int hidden;
    int tiles_m;
    int tiles_n;
    void* out;
    std::int64_t out_stride;
    // gradient only: `out` is dg and du is out + du_offset, both [rows, out_stride] with the columns
    // past hidden written as zeros
    const void* out_gradient;
    std::int64_t out_gradient_stride;
    std::int64_t du_offset;
};

template <class Tile, int kActivation, bool kGradient>
__global__ __launch_bounds__(Tile::kThreads) void gatedKernel(GatedArgs args) {
    using T = typename Tile::T;
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    constexpr int kWaveN = Tile::kN / Tile::kWavesN;
    constexpr int kHalf = kWaveN / 2;
    constexpr int kPairs = Tile::kBlocksN / 2;
    static_assert(Tile::kBlocksN % 2 == 0, "a wavefront's columns are whole blocks of gate and of up rows");
    const T* x = static_cast<const T*>(args.x);
    const T* gate = static_cast<const T*>(args.gate);
    const T* up = static_cast<const T*>(args.up);
    const int total = args.tiles_m * args.tiles_n;
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    typename Tile::Loads loads;
    auto begin = [&](int index) {
        int tile_m, tile_n;
        tileOf(index, args.tiles_m, args.tiles_n, tile_m, tile_n);
        const int m0 = tile_m * Tile::kM;
        const int n0 = tile_n * (Tile::kN / 2);
        loads.begin([&](int r) { return x + min(m0 + r, args.rows - 1) * args.x_stride; }, args.x_stride, 0,
                    [&](int r) {
                        const int j = r % kWaveN;
                        const int n = min(n0 + r / kWaveN * kHalf + j % kHalf, args.hidden - 1);
                        return (j < kHalf ? gate : up) + n * args.weight_stride;
                    },
                    args.weight_stride, 0, args.dim);
        loads.start(lds);
    };
    begin(static_cast<int>(blockIdx.x));
    for (int index = static_cast<int>(blockIdx.x); index < total; index += static_cast<int>(gridDim.x)) {
        typename Tile::Sums sums;
        Tile::clear(sums);
        Tile::accumulate(lds, loads, args.dim, sums, [&] {
            if (index + static_cast<int>(gridDim.x) < total) {
                begin(index + static_cast<int>(gridDim.x));
            }
        });
        int tile_m, tile_n;
        tileOf(index, args.tiles_m, args.tiles_n, tile_m, tile_n);
        const int m0 = tile_m * Tile::kM + Tile::waveM() * Tile::kBlocksM * 16 + (lane & 15);
        const int n0 = tile_n * (Tile::kN / 2) + Tile::waveN() * kHalf + 4 * (lane >> 4);
        if constexpr (!kGradient) {
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sums[i][j][e] = activate<kActivation>(sums[i][j][e]) * sums[i][j + kPairs][e];
                    }
                }
            }
            loads.land();
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const int m = m0 + i * 16;
                    const int n = n0 + j * 16;
                    if (m < args.rows && n < args.hidden) {
                        storeFour(sums[i][j], static_cast<T*>(args.out) + m * args.out_stride + n, args.hidden - n);
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i) {
                const int m = m0 + i * 16;
                f32x4 from[kPairs];
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const int n = n0 + j * 16;
                    from[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (m < args.rows && n < args.hidden) {
                        from[j] = loadFour(static_cast<const T*>(args.out_gradient) + m * args.out_gradient_stride + n,
                                           args.hidden - n);
                    }
                }
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const int n = n0 + j * 16;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float value, slope;
                        activateBoth<kActivation>(sums[i][j][e], value, slope);
                        // columns past hidden are zeros whatever stands in for their weights
                        const bool inside = n + e < args.hidden;
                        sums[i][j][e] = inside ? from[j][e] * sums[i][j + kPairs][e] * slope : 0.0f;
                        sums[i][j + kPairs][e] = inside ? from[j][e] * value : 0.0f;
                    }
                }
            }
            loads.land();
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const int m = m0 + i * 16;
                    const int n = n0 + j * 16;
                    if (m < args.rows && n < args.out_stride) {
                        T* to = static_cast<T*>(args.out) + m * args.out_stride + n;
                        storeFour(sums[i][j], to, 4);
                        storeFour(sums[i][j + kPairs], to + args.du_offset, 4);
                    }
                }
            }
        }
    }
}

// A product with too few tiles for the GPU is split over k as well: every split writes float32 partial
// sums, which joinKernel adds in the order of the splits.

// x_gradient [rows, dim] = dg gate + du up.
struct InputGradientArgs {
    const void* dg;
    std::int64_t d_stride;
    std::int64_t du_offset;
    const void* gate;
    const void* up;
    std::int64_t weight_stride;
    int rows;
    int dim;
    int hidden;
    int tiles_m;
    int tiles_n;
    int splits;      // 1: both products in one; otherwise even, the first half of them for dg gate
    int split_k;     // values of k of a split
    float* partials;  // [splits, rows, dim]
    void* out;
    std::int64_t out_stride;
};

template <class Tile>
__device__ __forceinline__ void formInputGradient(const InputGradientArgs& args, std::uint8_t* lds, int tile, int split) {
    using T = typename Tile::T;
    int tile_m, tile_n;
    tileOf(tile, args.tiles_m, args.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * Tile::kM;
    const int n0 = tile_n * Tile::kN;
    const int half = args.splits / 2;
    int part = args.splits > 1 && split >= half ? 1 : 0;
    const int past_part = args.splits > 1 ? part + 1 : 2;
    const int k0 = args.splits > 1 ? (split - part * half) * args.split_k : 0;
    const int k_total = args.splits > 1 ? min(args.split_k, args.hidden - k0) : args.hidden;
    typename Tile::Sums sums;
    Tile::clear(sums);
    typename Tile::Loads loads;
    const T* d = static_cast<const T*>(args.dg) + (part == 0 ? 0 : args.du_offset) + k0;
    const T* weight = static_cast<const T*>(part == 0 ? args.gate : args.up) + k0 * args.weight_stride;
    loads.begin([&](int r) { return d + min(m0 + r, args.rows - 1) * args.d_stride; }, args.d_stride, 0,
                [&](int) { return weight + n0; }, args.weight_stride, args.dim - n0, k_total);
    loads.start(lds);
#pragma unroll 1
    for (; part < past_part; ++part) {
        Tile::accumulate(lds, loads, k_total, sums, [&] {
            if (part + 1 < past_part) {
                loads.moveOn(args.du_offset * static_cast<std::int64_t>(sizeof(T)),
                             static_cast<const char*>(args.up) - static_cast<const char*>(args.gate), k_total);
                loads.start(lds);
            }
        });
    }
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        const int m = m0 + (Tile::waveM() * Tile::kBlocksM + i) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j) {
            const int n = n0 + (Tile::waveN() * Tile::kBlocksN + j) * 16 + 4 * (lane >> 4);
            if (m < args.rows && n < args.dim) {
                if (args.splits > 1) {
                    float* to = args.partials + (static_cast<std::int64_t>(split) * args.rows + m) * args.dim + n;
                    storeFour(sums[i][j], to, args.dim - n);
                } else {
                    storeFour(sums[i][j], static_cast<T*>(args.out) + m * args.out_stride + n, args.dim - n);
                }
            }
        }
    }
}

// gate_gradient = dg^T x and up_gradient = du^T x, the second half of the grid's tiles for the latter.
struct WeightGradientArgs {
    const void* dg;
    std::int64_t d_stride;
    std::int64_t du_offset;
    const void* x;
    std::int64_t x_stride;
    int rows;
    int dim;
    int hidden;
    int tiles_m;  // of one of the two
    int tiles_n;
    int splits;
    int split_k;
    float* partials;  // [splits, 2, hidden, dim]
    void* gate_out;
    void* up_out;
    std::int64_t out_stride;
};

template <class Tile>
__device__ __forceinline__ void formWeightGradient(const WeightGradientArgs& args, std::uint8_t* lds, int tile,
                                                   int split) {
    using T = typename Tile::T;
    int tile_m, tile_n;
    tileOf(tile, 2 * args.tiles_m, args.tiles_n, tile_m, tile_n);
    const int k0 = split * args.split_k;
    const int k_total = min(args.split_k, args.rows - k0);
    const bool second = tile_m >= args.tiles_m;
    const int m0 = (second ? tile_m - args.tiles_m : tile_m) * Tile::kM;
    const int n0 = tile_n * Tile::kN;
    const T* d = static_cast<const T*>(args.dg) + (second ? args.du_offset : 0) + k0 * args.d_stride;
    const T* x = static_cast<const T*>(args.x) + k0 * args.x_stride;
    typename Tile::Sums sums;
    Tile::clear(sums);
    // the rows of dg and du are padded to whole chunks
    typename Tile::Loads loads;
    loads.begin([&](int) { return d + m0; }, args.d_stride, static_cast<int>(args.d_stride) - m0,
                [&](int) { return x + n0; }, args.x_stride, args.dim - n0, k_total);
    loads.start(lds);
    Tile::accumulate(lds, loads, k_total, sums, [] {});
    T* out = static_cast<T*>(second ? args.up_out : args.gate_out);
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        const int m = m0 + (Tile::waveM() * Tile::kBlocksM + i) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j) {
            const int n = n0 + (Tile::waveN() * Tile::kBlocksN + j) * 16 + 4 * (lane >> 4);
            if (m < args.hidden && n < args.dim) {
                if (args.splits > 1) {
                    const std::int64_t row = (2 * static_cast<std::int64_t>(split) + (second ? 1 : 0)) * args.hidden + m;
                    storeFour(sums[i][j], args.partials + row * args.dim + n, args.dim - n);
                } else {
                    storeFour(sums[i][j], out + m * args.out_stride + n, args.dim - n);
                }
            }
        }
    }
}

template <class Tile>
__global__ __launch_bounds__(Tile::kThreads) void inputGradientKernel(InputGradientArgs args) {
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    formInputGradient<Tile>(args, lds, static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.y));
}

template <class Tile>
__global__ __launch_bounds__(Tile::kThreads) void weightGradientKernel(WeightGradientArgs args) {
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    formWeightGradient<Tile>(args, lds, static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.y));
}

// Both in one launch, for products of few tiles: the first `input_blocks` blocks form the input's.
template <class InputTile, class WeightTile>
__global__ __launch_bounds__(InputTile::kThreads) void bothGradientsKernel(InputGradientArgs input,
                                                                           WeightGradientArgs weight, int input_blocks) {
    static_assert(InputTile::kThreads == WeightTile::kThreads, "one workgroup size");
    __shared__ __attribute__((aligned(256))) std::uint8_t
        lds[InputTile::kLdsBytes > WeightTile::kLdsBytes ? InputTile::kLdsBytes : WeightTile::kLdsBytes];
    const int block = static_cast<int>(blockIdx.x);
    if (block < input_blocks) {
        const int tiles = input.tiles_m * input.tiles_n;
        formInputGradient<InputTile>(input, lds, block % tiles, block / tiles);
    } else {
        const int tiles = 2 * weight.tiles_m * weight.tiles_n;
        formWeightGradient<WeightTile>(weight, lds, (block - input_blocks) % tiles, (block - input_blocks) / tiles);
    }
}

// ---- host ---------------------------------------------------------------------------------------

int invalid(const char* message) {
    return setError(ZCGVS_ERR_INVALID_ARGUMENT, std::string("zcgvs gated projection: ") + message);
}

int checkGated(const zcgvs_gated_desc* desc) {
    if (desc == nullptr) {
        return invalid("null descriptor");
    }
    const zcgvs_gated_desc& d = *desc;
    if (!validElement(d.dtype)) {
        return invalid("the operands must hold float32, float16 or bfloat16");
    }
    if (d.activation < ZCGVS_ACT_SILU || d.activation > ZCGVS_ACT_GELU_TANH) {
        return invalid("unknown activation");
    }
    if (d.dim <= 0 || d.hidden <= 0) {
        return invalid("dim and hidden must be positive");
    }
    if (d.dim > (1 << 24) || d.hidden > (1 << 24)) {
        return invalid("dim and hidden must be at most 2^24");
    }
    if (d.rows < 0 || d.rows > (1 << 30)) {
        return invalid("rows must lie in [0, 2^30]");
    }
    if (rowStride(d.x_stride, d.dim) < d.dim || rowStride(d.weight_stride, d.dim) < d.dim) {
        return invalid("a row stride is smaller than dim");
    }
    if (d.rows > 0 && (d.x == nullptr || d.gate == nullptr || d.up == nullptr)) {
        return invalid("null device pointer");
    }
    return ZCGVS_OK;
}

template <typename T, bool kGradient>
int launchGated(const zcgvs_gated_desc& d, GatedArgs args, hipStream_t stream) {
    args.x = d.x;
    args.x_stride = rowStride(d.x_stride, d.dim);
    args.gate = d.gate;
    args.up = d.up;
    args.weight_stride = rowStride(d.weight_stride, d.dim);
    args.rows = static_cast<int>(d.rows);
    args.dim = d.dim;
    args.hidden = d.hidden;
    const bool direct = directRows(args.x, args.x_stride, d.dim, d.dtype) &&
                        directRows(args.gate, args.weight_stride, d.dim, d.dtype) &&
                        directRows(args.up, args.weight_stride, d.dim, d.dtype);
    return withActivation(d.activation, [&](auto activation) {
        // the error function's terms do not fit the registers beside the sums of 256 x 256
        constexpr LargestTile kLargest = decltype(activation)::value == ZCGVS_ACT_GELU ? LargestTile::k256x192
                                                                                        : LargestTile::k256x256;
        const ProductPlan plan = planProduct(d.rows, 2 * static_cast<std::int64_t>(d.hidden), d.dim, 1, d.dtype, 0,
                                             largestTile(kLargest, direct));
        return withTile<T, false, false, kLargest, true>(plan.shape, direct, [&](auto tile) {
            using Tile = decltype(tile);
            args.tiles_m = divideUp(d.rows, Tile::kM);
            args.tiles_n = divideUp(d.hidden, Tile::kN / 2);
            const long long tiles = static_cast<long long>(args.tiles_m) * args.tiles_n;
            if (tiles > INT32_MAX) {
                return invalid("more output than one launch can write");
            }
            const long long blocks = std::min(tiles, static_cast<long long>(persistentBlocks(plan.shape)));
            gatedKernel<Tile, decltype(activation)::value, kGradient>
                <<<static_cast<unsigned>(blocks), Tile::kThreads, 0, stream>>>(args);
            ZCGVS_LAUNCH_CHECK("gated projection");
            return static_cast<int>(ZCGVS_OK);
        });
    });
}

// Elements from row to row of dg and du in the workspace; the partial sums follow them.
std::int64_t gradientStride(const zcgvs_gated_desc& d) { return (static_cast<std::int64_t>(d.hidden) + 7) / 8 * 8; }

std::size_t partialsOffset(const zcgvs_gated_desc& d) {
    const std::size_t both = 2 * static_cast<std::size_t>(d.rows) * static_cast<std::size_t>(gradientStride(d));
    return (both * static_cast<std::size_t>(elementBytes(d.dtype)) + 255) / 256 * 256;
}

ProductPlan inputPlan(const zcgvs_gated_desc& d, bool direct) {
    // an even number of splits, each within one of the two products; 256 x 256 tiles of two products one
    // after the other do not fit the registers (measured 140 us for what 256 x 192 take 93)
    return planProduct(d.rows, d.dim, 2 * static_cast<std::int64_t>(d.hidden), 1, d.dtype, 2,
                       largestTile(LargestTile::k256x192, direct));
}

ProductPlan weightPlan(const zcgvs_gated_desc& d, bool direct) {
    return planProduct(d.hidden, d.dim, d.rows, 2, d.dtype, 1, largestTile(LargestTile::k256x256, direct));
}

// float32 partial sums of the two products: the input's, then the weights'. A call's workspace holds those of either
// kind of rows, so that its size goes by the sizes and the type alone.
std::size_t inputPartials(const zcgvs_gated_desc& d) {
    const int splits = std::max(inputPlan(d, false).splits, inputPlan(d, true).splits);
    const std::size_t values = static_cast<std::size_t>(d.rows) * static_cast<std::size_t>(d.dim);
    return splits > 1 ? static_cast<std::size_t>(splits) * values / 4 * 4 + 4 : 0;
}

std::size_t weightPartials(const zcgvs_gated_desc& d) {
    const int splits = std::max(weightPlan(d, false).splits, weightPlan(d, true).splits);
    const std::size_t values = 2 * static_cast<std::size_t>(d.hidden) * static_cast<std::size_t>(d.dim);
    return splits > 1 ? static_cast<std::size_t>(splits) * values : 0;
}

// The splits of a plan: whole stages each, which may leave fewer than planned.
void splitInput(const zcgvs_gated_desc& d, const ProductPlan& plan, InputGradientArgs& args) {
    args.splits = 1;
    args.split_k = d.hidden;
    if (plan.splits > 1) {
        args.split_k = divideUp(divideUp(d.hidden, plan.splits / 2), kPlanStageK) * kPlanStageK;
        args.splits = 2 * divideUp(d.hidden, args.split_k);
    }
}

void splitWeight(const zcgvs_gated_desc& d, const ProductPlan& plan, WeightGradientArgs& args) {
    args.split_k = divideUp(divideUp(d.rows, plan.splits), kPlanStageK) * kPlanStageK;
    args.splits = divideUp(d.rows, args.split_k);
}

template <typename T>
int launchInputGradient(const zcgvs_gated_desc& d, const ProductPlan& plan, bool direct, InputGradientArgs args,
                        hipStream_t stream) {
    return withTile<T, false, true, LargestTile::k256x192, false>(plan.shape, direct, [&](auto tile) {
        using Tile = decltype(tile);
        args.tiles_m = divideUp(d.rows, Tile::kM);
        args.tiles_n = divideUp(d.dim, Tile::kN);
        const long long blocks = static_cast<long long>(args.tiles_m) * args.tiles_n;
        if (blocks > kMaxBlocks) {
            return invalid("more output than one launch can write");
        }
        inputGradientKernel<Tile><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(args.splits)),
                                    Tile::kThreads, 0, stream>>>(args);
        ZCGVS_LAUNCH_CHECK("gated gradient");
        return static_cast<int>(ZCGVS_OK);
    });
}

template <typename T>
int launchWeightGradient(const zcgvs_gated_desc& d, const ProductPlan& plan, bool direct, WeightGradientArgs args,
                         hipStream_t stream) {
    return withTile<T, true, true, LargestTile::k256x256, false>(plan.shape, direct, [&](auto tile) {
        using Tile = decltype(tile);
        args.tiles_m = divideUp(d.hidden, Tile::kM);
        args.tiles_n = divideUp(d.dim, Tile::kN);
        const long long blocks = 2ll * args.tiles_m * args.tiles_n;
        if (blocks > kMaxBlocks) {
            return invalid("more output than one launch can write");
        }
        weightGradientKernel<Tile><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(args.splits)),
                                     Tile::kThreads, 0, stream>>>(args);
        ZCGVS_LAUNCH_CHECK("gated gradient");
        return static_cast<int>(ZCGVS_OK);
    });
}

// Both products where both take 64 x 64 tiles, which leave the GPU idle between launches (500 rows of 384,
// hidden 1024: 19.4 us instead of 22.8).
template <class InputTile, class WeightTile>
int launchBothGradients(const zcgvs_gated_desc& d, InputGradientArgs input, WeightGradientArgs weight,
                        hipStream_t stream) {
    input.tiles_m = divideUp(d.rows, InputTile::kM);
    input.tiles_n = divideUp(d.dim, InputTile::kN);
    weight.tiles_m = divideUp(d.hidden, WeightTile::kM);
    weight.tiles_n = divideUp(d.dim, WeightTile::kN);
    const long long input_blocks = static_cast<long long>(input.tiles_m) * input.tiles_n * input.splits;
    const long long weight_blocks = 2ll * weight.tiles_m * weight.tiles_n * weight.splits;
    if (input_blocks + weight_blocks > kMaxBlocks) {
        return invalid("more output than one launch can write");
    }
    bothGradientsKernel<InputTile, WeightTile><<<static_cast<unsigned>(input_blocks + weight_blocks),
                                                 InputTile::kThreads, 0, stream>>>(input, weight,
                                                                                   static_cast<int>(input_blocks));
    ZCGVS_LAUNCH_CHECK("gated gradient");
    return ZCGVS_OK;
}

// The products with dg and du, and the sums over their splits. An output that is null is not wanted.
template <typename T>
int launchGradients(const zcgvs_gated_desc& d, InputGradientArgs input, WeightGradientArgs weight, hipStream_t stream) {
    const bool direct_input = directRows(input.gate, input.weight_stride, d.dim, d.dtype) &&
                              directRows(input.up, input.weight_stride, d.dim, d.dtype);
    const bool direct_weight = directRows(weight.x, weight.x_stride, d.dim, d.dtype);
    const ProductPlan input_plan = inputPlan(d, direct_input);
    const ProductPlan weight_plan = weightPlan(d, direct_weight);
    splitInput(d, input_plan, input);
    splitWeight(d, weight_plan, weight);
    const bool wants_input = input.out != nullptr;
    const bool wants_weight = weight.gate_out != nullptr;
    int status = ZCGVS_OK;
    if (wants_input && wants_weight && direct_input == direct_weight && input_plan.shape == TileShape::k64x64 &&
        weight_plan.shape == TileShape::k64x64) {
        if constexpr (std::is_same_v<T, float>) {
            status = launchBothGradients<SplitTile<64, 64, 2, 2, false, true>, SplitTile<64, 64, 2, 2, true, true>>(
                d, input, weight, stream);
        } else if (direct_input) {
            status = launchBothGradients<MatrixTile<T, 64, 64, 2, 2, false, true, true>,
                                         MatrixTile<T, 64, 64, 2, 2, true, true, true>>(d, input, weight, stream);
        } else {
            status = launchBothGradients<MatrixTile<T, 64, 64, 2, 2, false, true, false>,
                                         MatrixTile<T, 64, 64, 2, 2, true, true, false>>(d, input, weight, stream);
        }
    } else {
        if (wants_input) {
            status = launchInputGradient<T>(d, input_plan, direct_input, input, stream);
        }
        if (status == ZCGVS_OK && wants_weight) {
            status = launchWeightGradient<T>(d, weight_plan, direct_weight, weight, stream);
        }
    }
    if (status == ZCGVS_OK && wants_input && input.splits > 1) {
        status = launchJoin<T>(input.partials, input.splits, d.rows, d.dim, d.rows, input.out, nullptr,
                               input.out_stride, stream);
    }
    if (status == ZCGVS_OK && wants_weight && weight.splits > 1) {
        status = launchJoin<T>(weight.partials, weight.splits, 2 * static_cast<std::int64_t>(d.hidden), d.dim, d.hidden,
                               weight.gate_out, weight.up_out, weight.out_stride, stream);
    }
    return status;
}

// Zeros for the weight gradients of a batch without rows.
template <typename T>
__global__ __launch_bounds__(256) void clearMatrixKernel(T* out, std::int64_t stride, int rows, int columns) {
    for (int r = static_cast<int>(blockIdx.x); r < rows; r += static_cast<int>(gridDim.x)) {
        for (int c = static_cast<int>(threadIdx.x); c < columns; c += 256) {
            out[r * stride + c] = static_cast<T>(0.0f);
        }
    }
}

}  // namespace

}  // namespace zcgvs_hip

using namespace zcgvs_hip;

extern "C" {

int zcgvs_gated_projection(const zcgvs_gated_desc* desc, void* d_out, std::int64_t out_stride, zcgvs_stream_t stream) {
    const int status = checkGated(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_gated_desc& d = *desc;
    if (rowStride(out_stride, d.hidden) < d.hidden) {
        return invalid("the output's row stride is smaller than hidden");
    }
    if (d.rows == 0) {
        return clearError();
    }
    if (d_out == nullptr) {
        return invalid("null device pointer");
    }
    GatedArgs args{};
    args.out = d_out;
    args.out_stride = rowStride(out_stride, d.hidden);
    const int launched = withElement(d.dtype, [&](auto element) {
        return launchGated<decltype(element), false>(d, args, toStream(stream));
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

std::size_t zcgvs_gated_gradient_workspace_bytes(const zcgvs_gated_desc* desc) {
    if (checkGated(desc) != ZCGVS_OK) {
        return 0;
    }
    clearError();
    return desc->rows == 0 ? 256 : partialsOffset(*desc) + (inputPartials(*desc) + weightPartials(*desc)) * sizeof(float);
}

int zcgvs_gated_gradient(const zcgvs_gated_desc* desc, const void* d_out_gradient, std::int64_t out_gradient_stride,
                         void* d_x_gradient, std::int64_t x_gradient_stride, void* d_gate_gradient,
                         void* d_up_gradient, std::int64_t weight_gradient_stride, void* d_workspace,
                         std::size_t workspace_bytes, zcgvs_stream_t stream) {
    const int status = checkGated(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_gated_desc& d = *desc;
    const std::int64_t from_stride = rowStride(out_gradient_stride, d.hidden);
    const std::int64_t x_out_stride = rowStride(x_gradient_stride, d.dim);
    const std::int64_t weight_out_stride = rowStride(weight_gradient_stride, d.dim);
    if (from_stride < d.hidden || x_out_stride < d.dim || weight_out_stride < d.dim) {
        return invalid("a gradient's row stride is smaller than its row");
    }
    if ((d_gate_gradient == nullptr) != (d_up_gradient == nullptr)) {
        return invalid("gate_gradient and up_gradient are wanted both or neither");
    }
    if (d_x_gradient == nullptr && d_gate_gradient == nullptr) {
        return clearError();
    }
    if (d.rows == 0) {
        if (d_gate_gradient != nullptr) {
            const int cleared = withElement(d.dtype, [&](auto element) {
                using T = decltype(element);
                const unsigned blocks = static_cast<unsigned>(std::min(d.hidden, 4096));
                for (void* out : {d_gate_gradient, d_up_gradient}) {
                    clearMatrixKernel<T><<<blocks, 256, 0, toStream(stream)>>>(static_cast<T*>(out), weight_out_stride,
                                                                               d.hidden, d.dim);
                    ZCGVS_LAUNCH_CHECK("gated gradient");
                }
                return static_cast<int>(ZCGVS_OK);
            });
            if (cleared != ZCGVS_OK) {
                return cleared;
            }
        }
        return clearError();
    }
    if (d_out_gradient == nullptr) {
        return invalid("null device pointer");
    }
    if (d_workspace == nullptr || workspace_bytes < zcgvs_gated_gradient_workspace_bytes(desc)) {
        return invalid("the workspace is too small");
    }
    if (!aligned16(d_workspace)) {
        return invalid("the workspace must be aligned to 16 bytes");
    }
    const int launched = withElement(d.dtype, [&](auto element) {
        using T = decltype(element);
        GatedArgs form{};
        form.out = d_workspace;
        form.out_stride = gradientStride(d);
        form.out_gradient = d_out_gradient;
        form.out_gradient_stride = from_stride;
        form.du_offset = d.rows * form.out_stride;
        const int formed = launchGated<T, true>(d, form, toStream(stream));
        if (formed != ZCGVS_OK) {
            return formed;
        }
        float* partials = reinterpret_cast<float*>(static_cast<char*>(d_workspace) + partialsOffset(d));
        InputGradientArgs input{};
        input.dg = d_workspace;
        input.d_stride = form.out_stride;
        input.du_offset = form.du_offset;
        input.gate = d.gate;
        input.up = d.up;
        input.weight_stride = rowStride(d.weight_stride, d.dim);
        input.rows = static_cast<int>(d.rows);
        input.dim = d.dim;
        input.hidden = d.hidden;
        input.partials = partials;
        input.out = d_x_gradient;
        input.out_stride = x_out_stride;
        WeightGradientArgs weight{};
        weight.dg = d_workspace;
        weight.d_stride = form.out_stride;
        weight.du_offset = form.du_offset;
        weight.x = d.x;
        weight.x_stride = rowStride(d.x_stride, d.dim);
        weight.rows = input.rows;
        weight.dim = d.dim;
        weight.hidden = d.hidden;
        weight.partials = partials + inputPartials(d);
        weight.gate_out = d_gate_gradient;
        weight.up_out = d_up_gradient;
        weight.out_stride = weight_out_stride;
        return launchGradients<T>(d, input, weight, toStream(stream));
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

}  // extern "C"
