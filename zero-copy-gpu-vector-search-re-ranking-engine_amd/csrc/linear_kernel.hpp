// Kernels of the linear projection, forward and backward.
//
//     z = x W^T + b (int8: the codes' exact products in int32, times the scales),  out = act(z) + residual
//     dz = d_out act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// The tiles are those of matrix_tile.hpp and matrix_split.hpp; bias, activation and residual are applied to a
// tile's sums in registers, so each output is written once and nothing else is. The next tile's first stage is on
// its way while a tile's results are formed.
//
// Few rows (linearThinKernel) are bound by latency and by reading W once: a workgroup takes 16 columns and 16 or 32
// rows, its eight wavefronts every eighth 128 bytes of k, straight from memory into registers, and joins their sums
// through LDS. No LDS stages, no splits over workgroups, one launch.
//
// Measured: one row 768 -> 768 float16 6.6 us (the launch); 8192 rows 1024 -> 4096 int8, GELU by tanh 60-68 us (1.0-1.1 POP/s), bfloat16
// 84-95 (0.7-0.8 PFLOP/s); 8192 cubed bfloat16 1015-1034 us (1.07 PFLOP/s, a library product 1.45); the gradient of 16,384 rows
// 768 -> 2048 bfloat16 216-222 us (dz 91, dW 66, dx 55, joins 8). Bound by the product loop, dz also by its loads and stores between the
// tiles' products.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "activation.hpp"
#include "column_sums.hpp"
#include "common.hpp"
#include "elements.hpp"
#include "linear.hpp"
#include "matrix_plan.hpp"
#include "matrix_split.hpp"
#include "matrix_tile.hpp"

namespace zcgvs_hip {
namespace {

// Four neighbouring values of a bias or a residual.
template <typename T>
__device__ __forceinline__ f32x4 loadEpilogue(const LinearArgs& args, const void* base, std::int64_t index, int left) {
    if constexpr (std::is_same_v<T, std::int8_t>) {
        if (args.epilogue_dtype == ZCGVS_DTYPE_F16) {
            return loadFour(static_cast<const _Float16*>(base) + index, left);
        }
        if (args.epilogue_dtype == ZCGVS_DTYPE_BF16) {
            return loadFour(static_cast<const __bf16*>(base) + index, left);
        }
        return loadFour(static_cast<const float*>(base) + index, left);
    } else {
        return loadFour(static_cast<const T*>(base) + index, left);
    }
}

// The same as they are stored, until their values are wanted (int8 operands: the values).
template <typename T>
struct HeldFour {
    static constexpr bool kValues = std::is_same_v<T, std::int8_t>;
    using Stored = std::conditional_t<kValues, f32x4, typename Pack<T, 4>::type>;
    Stored stored = {};

    __device__ __forceinline__ void load(const LinearArgs& args, const void* base, std::int64_t index, int left) {
        if constexpr (kValues) {
            stored = loadEpilogue<T>(args, base, index, left);
        } else {
            const T* from = static_cast<const T*>(base) + index;
            if (left >= 4) {
                stored = *reinterpret_cast<const typename Pack<T, 4>::stored*>(from);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (e < left) {
                        stored[e] = from[e];
                    }
                }
            }
        }
    }
    __device__ __forceinline__ f32x4 values() const {
        if constexpr (kValues) {
            return stored;
        } else {
            return __builtin_convertvector(stored, f32x4);
        }
    }
};

template <typename T>
__device__ __forceinline__ void storeResult(const LinearArgs& args, const f32x4& value, std::int64_t index, int left) {
    if (args.out_dtype == ZCGVS_DTYPE_F32) {
        storeFour(value, static_cast<float*>(args.out) + index, left);
    } else if constexpr (std::is_same_v<T, std::int8_t>) {
        if (args.out_dtype == ZCGVS_DTYPE_F16) {
            storeFour(value, static_cast<_Float16*>(args.out) + index, left);
        } else {
            storeFour(value, static_cast<__bf16*>(args.out) + index, left);
        }
    } else {
        storeFour(value, static_cast<T*>(args.out) + index, left);
    }
}

// kMaxCodes products of -128 and -128 are 2^31, which wraps to -2^31; no other codes give that (-128 times 127 is more). The
// integer below 2^31 is the same float32.
__device__ __forceinline__ void exactSum(i32x4& sum) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        sum[e] = sum[e] == INT32_MIN ? INT32_MAX : sum[e];
    }
}

// z of four neighbouring columns n of row m from their sum of products.
template <typename T, typename Sum>
__device__ __forceinline__ f32x4 beforeActivation(const Sum& sum, float x_scale, const f32x4& weight_scales,
                                                  const f32x4& bias) {
    f32x4 z;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        z[e] = static_cast<float>(sum[e]);
        if constexpr (std::is_same_v<T, std::int8_t>) {
            z[e] *= x_scale * weight_scales[e];
        }
        z[e] += bias[e];
    }
    return z;
}

template <class Tile, int kActivation, bool kGradient>
__global__ __launch_bounds__(Tile::kThreads) void linearKernel(LinearArgs args) {
    using T = typename Tile::T;
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    const T* x = static_cast<const T*>(args.x);
    const T* weight = static_cast<const T*>(args.weight);
    const int total = args.tiles_m * args.tiles_n;
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    typename Tile::Loads loads;
    auto begin = [&](int index) {
        int tile_m, tile_n;
        tileOf(index, args.tiles_m, args.tiles_n, tile_m, tile_n);
        const int m0 = tile_m * Tile::kM;
        const int n0 = tile_n * Tile::kN;
        loads.begin([&](int r) { return x + min(m0 + r, args.rows - 1) * args.x_stride; }, args.x_stride, 0,
                    [&](int r) { return weight + min(n0 + r, args.out_dim - 1) * args.weight_stride; },
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
        if constexpr (std::is_same_v<T, std::int8_t>) {
            if (args.dim == kMaxCodes) {
#pragma unroll
                for (int i = 0; i < Tile::kBlocksM; ++i) {
#pragma unroll
                    for (int j = 0; j < Tile::kBlocksN; ++j) {
                        exactSum(sums[i][j]);
                    }
                }
            }
        }
        int tile_m, tile_n;
        tileOf(index, args.tiles_m, args.tiles_n, tile_m, tile_n);
        const int m0 = tile_m * Tile::kM + Tile::waveM() * Tile::kBlocksM * 16 + (lane & 15);
        const int n0 = tile_n * Tile::kN + Tile::waveN() * Tile::kBlocksN * 16 + 4 * (lane >> 4);
        // What a column block needs beside its sums is held as it is stored, that of the next one on its way where
        // the registers allow. Results take the place of their sums; the barriers keep the compiler from taking
        // several blocks at once, for which 256 x 256 tiles have no registers (up to 365 were spilled without them).
        constexpr int kHeld = Tile::kBlocksM * Tile::kBlocksN >= 16 || std::is_same_v<T, std::int8_t> ? 1 : 2;
        HeldFour<T> bias[kHeld], from[kHeld][Tile::kBlocksM];
        f32x4 scales = {0.0f, 0.0f, 0.0f, 0.0f};
        float x_scales[Tile::kBlocksM];
#pragma unroll
        for (int i = 0; i < Tile::kBlocksM; ++i) {
            x_scales[i] = std::is_same_v<T, std::int8_t> ? args.x_scales[min(m0 + i * 16, args.rows - 1)] : 1.0f;
        }
        const void* base = kGradient ? args.out_gradient : args.residual;
        const std::int64_t stride = kGradient ? args.out_gradient_stride : args.residual_stride;
        auto hold = [&](int j) {
            const int n = n0 + j * 16;
            const int left = args.out_dim - n;
            bias[j % kHeld] = HeldFour<T>{};
            if (args.bias != nullptr && left > 0) {
                bias[j % kHeld].load(args, args.bias, n, left);
            }
            if (std::is_same_v<T, std::int8_t> && left > 0) {
                scales = loadFour(args.weight_scales + n, left);
            }
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i) {
                const int m = m0 + i * 16;
                from[j % kHeld][i] = HeldFour<T>{};
                if (base != nullptr && m < args.rows && left > 0) {
                    from[j % kHeld][i].load(args, base, m * stride + n, left);
                }
            }
        };
        if constexpr (kHeld > 1) {
            hold(0);
        }
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j) {
            if constexpr (kHeld == 1) {
                hold(j);
            } else if (j + 1 < Tile::kBlocksN) {
                hold(j + 1);
            }
#pragma unroll
            for (int i = 0; i < Tile::kBlocksM; ++i) {
                const int m = m0 + i * 16;
                const f32x4 z = beforeActivation<T>(sums[i][j], x_scales[i], scales, bias[j % kHeld].values());
                const f32x4 more = from[j % kHeld][i].values();
                f32x4 result;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (kGradient) {
                        float value, slope;
                        activateBoth<kActivation>(z[e], value, slope);
                        // rows and columns past the ends are zeros whatever stands in for their operands
                        const bool inside = m < args.rows && n0 + j * 16 + e < args.out_dim;
                        result[e] = inside ? more[e] * slope : 0.0f;
                    } else {
                        result[e] = activate<kActivation>(z[e]) + more[e];
                    }
                }
                sums[i][j] = __builtin_bit_cast(typename Tile::Sum, result);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        loads.land();
#pragma unroll
        for (int i = 0; i < Tile::kBlocksM; ++i) {
            const int m = m0 + i * 16;
#pragma unroll
            for (int j = 0; j < Tile::kBlocksN; ++j) {
                const int n = n0 + j * 16;
                const f32x4 result = __builtin_bit_cast(f32x4, sums[i][j]);
                if constexpr (kGradient) {
                    if (m < args.rows && n < args.out_stride) {
                        storeFour(result, static_cast<T*>(args.out) + m * args.out_stride + n, 4);
                    }
                } else if (m < args.rows && n < args.out_dim) {
                    storeResult<T>(args, result, m * args.out_stride + n, args.out_dim - n);
                }
            }
        }
        if constexpr (kGradient) {
            if (args.bias_partials != nullptr) {
                float* to = args.bias_partials +
                            (static_cast<std::int64_t>(tile_m) * Tile::kWavesM + Tile::waveM()) * args.out_dim;
#pragma unroll
                for (int j = 0; j < Tile::kBlocksN; ++j) {
                    f32x4 sum = __builtin_bit_cast(f32x4, sums[0][j]);
#pragma unroll
                    for (int i = 1; i < Tile::kBlocksM; ++i) {
                        sum += __builtin_bit_cast(f32x4, sums[i][j]);
                    }
#pragma unroll
                    for (int offset = 1; offset < 16; offset *= 2) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            sum[e] += waveXor(sum[e], offset);
                        }
                    }
                    const int n = n0 + j * 16;
                    if ((lane & 15) == 0 && n < args.out_dim) {
                        storeFour(sum, to + n, args.out_dim - n);
                    }
                }
            }
        }
    }
}

// ---- few rows -----------------------------------------------------------------------------------

constexpr int kThinWaves = 8;
constexpr int kThinThreads = kThinWaves * kWave;
static_assert(kThinStageBytes == kThinWaves * kStageBytes, "a stage is 128 bytes of k for each wavefront");

// A row's chunk of 16 bytes at value k, of which `left` values exist; zeros past them.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::type loadChunk(const T* from, int left) {
    typename Fragment<T>::type v = {};
    if (left >= kChunk<T>) {
        __builtin_memcpy(&v, from, 16);
    } else {
#pragma unroll
        for (int e = 0; e < kChunk<T>; ++e) {
            if (e < left) {
                v[e] = from[e];
            }
        }
    }
    return v;
}

template <typename T, int kBlocksM, int kActivation>
__global__ __launch_bounds__(kThinThreads) void linearThinKernel(LinearArgs args) {
    using Sum = std::conditional_t<std::is_same_v<T, std::int8_t>, i32x4, f32x4>;
    __shared__ Sum shared[kThinWaves][kBlocksM][kWave];
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int r16 = lane & 15;
    const int h = lane >> 4;
    const int m0 = static_cast<int>(blockIdx.y) * kBlocksM * 16;
    const int n0 = static_cast<int>(blockIdx.x) * 16;
    const T* weight = static_cast<const T*>(args.weight) + min(n0 + r16, args.out_dim - 1) * args.weight_stride;
    const T* x[kBlocksM];
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) {
        x[i] = static_cast<const T*>(args.x) + min(m0 + i * 16 + r16, args.rows - 1) * args.x_stride;
    }
    Sum sums[kBlocksM];
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) {
        sums[i] = Sum{};
    }
    typename Fragment<T>::type a[kStageSteps][kBlocksM], b[kStageSteps];
    auto load = [&](int k0) {
#pragma unroll
        for (int t = 0; t < kStageSteps; ++t) {
            const int k = k0 + (4 * t + h) * kChunk<T>;
            b[t] = loadChunk(weight + k, args.dim - k);
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i) {
                a[t][i] = loadChunk(x[i] + k, args.dim - k);
            }
        }
    };
    const int step = kThinWaves * kStageK<T>;
    int k = wave * kStageK<T>;
    if (k < args.dim) {
        load(k);
    }
    for (; k < args.dim; k += step) {
        typename Fragment<T>::type now_a[kStageSteps][kBlocksM], now_b[kStageSteps];
#pragma unroll
        for (int t = 0; t < kStageSteps; ++t) {
            now_b[t] = b[t];
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i) {
                now_a[t][i] = a[t][i];
            }
        }
        if (k + step < args.dim) {
            load(k + step);
        }
#pragma unroll
        for (int t = 0; t < kStageSteps; ++t) {
#pragma unroll
            for (int i = 0; i < kBlocksM; ++i) {
                sums[i] = multiplyAdd(now_b[t], now_a[t][i], sums[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) {
        shared[wave][i][lane] = sums[i];
    }
    __syncthreads();
    if (wave >= kBlocksM) {
        return;
    }
    // wavefront i joins and finishes the rows of block i
    Sum sum = shared[0][wave][lane];
    if constexpr (std::is_same_v<T, std::int8_t>) {
        u32x4 wrapping = __builtin_bit_cast(u32x4, sum);
#pragma unroll
        for (int w = 1; w < kThinWaves; ++w) {
            wrapping += __builtin_bit_cast(u32x4, shared[w][wave][lane]);
        }
        sum = __builtin_bit_cast(Sum, wrapping);
        exactSum(sum);
    } else {
#pragma unroll
        for (int w = 1; w < kThinWaves; ++w) {
            sum += shared[w][wave][lane];
        }
    }
    const int m = m0 + wave * 16 + r16;
    const int n = n0 + 4 * h;
    if (m >= args.rows || n >= args.out_dim) {
        return;
    }
    const int left = args.out_dim - n;
    f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f}, scales = bias, from = bias;
    float x_scale = 1.0f;
    if (args.bias != nullptr) {
        bias = loadEpilogue<T>(args, args.bias, n, left);
    }
    if constexpr (std::is_same_v<T, std::int8_t>) {
        scales = loadFour(args.weight_scales + n, left);
        x_scale = args.x_scales[m];
    }
    if (args.residual != nullptr) {
        from = loadEpilogue<T>(args, args.residual, m * args.residual_stride + n, left);
    }
    f32x4 z = beforeActivation<T>(sum, x_scale, scales, bias);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        z[e] = activate<kActivation>(z[e]) + from[e];
    }
    storeResult<T>(args, z, m * args.out_stride + n, left);
}

// ---- the gradient's products --------------------------------------------------------------------

template <class Tile, bool kTurnedA>
__device__ __forceinline__ void formProduct(const ProductArgs& args, std::uint8_t* lds, int tile, int split) {
    using T = typename Tile::T;
    int tile_m, tile_n;
    tileOf(tile, args.tiles_m, args.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * Tile::kM;
    const int n0 = tile_n * Tile::kN;
    const int k0 = split * args.split_k;
    const int k_total = min(args.split_k, args.k - k0);
    const T* a = static_cast<const T*>(args.a) + (kTurnedA ? k0 * args.a_stride : static_cast<std::int64_t>(k0));
    const T* b = static_cast<const T*>(args.b) + k0 * args.b_stride;
    typename Tile::Sums sums;
    Tile::clear(sums);
    typename Tile::Loads loads;
    loads.begin([&](int r) { return kTurnedA ? a + m0 : a + min(m0 + r, args.m - 1) * args.a_stride; }, args.a_stride,
                args.a_columns - m0, [&](int) { return b + n0; }, args.b_stride, args.n - n0, k_total);
    loads.start(lds);
    Tile::accumulate(lds, loads, k_total, sums, [] {});
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        const int m = m0 + (Tile::waveM() * Tile::kBlocksM + i) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j) {
            const int n = n0 + (Tile::waveN() * Tile::kBlocksN + j) * 16 + 4 * (lane >> 4);
            if (m < args.m && n < args.n) {
                if (args.splits > 1) {
                    float* to = args.partials + (static_cast<std::int64_t>(split) * args.m + m) * args.n + n;
                    storeFour(sums[i][j], to, args.n - n);
                } else {
                    storeFour(sums[i][j], static_cast<T*>(args.out) + m * args.out_stride + n, args.n - n);
                }
            }
        }
    }
}

template <class Tile, bool kTurnedA>
__global__ __launch_bounds__(Tile::kThreads) void productKernel(ProductArgs args) {
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    formProduct<Tile, kTurnedA>(args, lds, static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.y));
}

// Both products in one launch where both take 64 x 64 tiles, which leave the GPU idle between launches: the first
// `input_blocks` blocks form dx.
template <class InputTile, class WeightTile>
__global__ __launch_bounds__(InputTile::kThreads) void bothProductsKernel(ProductArgs input, ProductArgs weight,
                                                                          int input_blocks, int weight_blocks, ColumnJoin bias) {
    static_assert(InputTile::kThreads == WeightTile::kThreads && InputTile::kThreads == kColumnThreads, "one workgroup size");
    __shared__ __attribute__((aligned(256))) std::uint8_t
        lds[InputTile::kLdsBytes > WeightTile::kLdsBytes ? InputTile::kLdsBytes : WeightTile::kLdsBytes];
    const int block = static_cast<int>(blockIdx.x);
    if (block < input_blocks) {
        const int tiles = input.tiles_m * input.tiles_n;
        formProduct<InputTile, false>(input, lds, block % tiles, block / tiles);
    } else if (block >= input_blocks + weight_blocks) {
        joinColumns(bias.partials, bias.rows, bias.columns, static_cast<typename InputTile::T*>(bias.out),
                    block - input_blocks - weight_blocks);
    } else {
        const int tiles = weight.tiles_m * weight.tiles_n;
        formProduct<WeightTile, true>(weight, lds, (block - input_blocks) % tiles, (block - input_blocks) / tiles);
    }
}

// ---- host ---------------------------------------------------------------------------------------

template <typename T, bool kGradient>
int launchTiles(const LinearPlan& plan, int activation, LinearArgs args, hipStream_t stream) {
    // (the sizes that linear.hip plans for)
    constexpr LargestTile kLargest = kGradient ? LargestTile::k256x256 : LargestTile::k256x192;
    return withTile<T, false, false, kLargest, false>(plan.product.shape, plan.direct, [&](auto tile) {
        using Tile = decltype(tile);
        args.tiles_m = divideUp(args.rows, Tile::kM);
        args.tiles_n = divideUp(args.out_dim, Tile::kN);
        const long long tiles = static_cast<long long>(args.tiles_m) * args.tiles_n;
        if (tiles > INT32_MAX) {
            return linearInvalid("more output than one launch can write");
        }
        const unsigned blocks =
            static_cast<unsigned>(std::min(tiles, static_cast<long long>(persistentBlocks(plan.product.shape))));
        const auto launch = [&](auto kind) {
            linearKernel<Tile, decltype(kind)::value, kGradient><<<blocks, Tile::kThreads, 0, stream>>>(args);
            ZCGVS_LAUNCH_CHECK("linear projection");
            return static_cast<int>(ZCGVS_OK);
        };
        if constexpr (!kGradient) {
            if (activation == ZCGVS_ACT_NONE) {
                return launch(std::integral_constant<int, ZCGVS_ACT_NONE>{});
            }
        }
        if constexpr (Tile::kM == 256 && Tile::kN == 256) {
            return activation == ZCGVS_ACT_SILU ? launch(std::integral_constant<int, ZCGVS_ACT_SILU>{})
                                                : launch(std::integral_constant<int, ZCGVS_ACT_GELU_TANH>{});
        } else {
            return withActivation(activation, launch);
        }
    });
}

template <typename T>
int launchThin(int row_blocks, int activation, const LinearArgs& args, hipStream_t stream) {
    const auto with = [&](auto blocks_m) {
        constexpr int kBlocksM = decltype(blocks_m)::value;
        const dim3 grid(static_cast<unsigned>(divideUp(args.out_dim, 16)),
                        static_cast<unsigned>(divideUp(args.rows, 16 * kBlocksM)));
        const auto launch = [&](auto kind) {
            linearThinKernel<T, kBlocksM, decltype(kind)::value><<<grid, kThinThreads, 0, stream>>>(args);
            ZCGVS_LAUNCH_CHECK("linear projection");
            return static_cast<int>(ZCGVS_OK);
        };
        return activation == ZCGVS_ACT_NONE ? launch(std::integral_constant<int, ZCGVS_ACT_NONE>{})
                                            : withActivation(activation, launch);
    };
    return row_blocks == 1 ? with(std::integral_constant<int, 1>{}) : with(std::integral_constant<int, 2>{});
}

template <typename T, bool kTurnedA>
int launchProduct(const ProductPlan& plan, bool direct, ProductArgs args, hipStream_t stream) {
    return withTile<T, kTurnedA, true, LargestTile::k256x256, false>(plan.shape, direct, [&](auto tile) {
        using Tile = decltype(tile);
        args.tiles_m = divideUp(args.m, Tile::kM);
        args.tiles_n = divideUp(args.n, Tile::kN);
        const long long blocks = static_cast<long long>(args.tiles_m) * args.tiles_n;
        if (blocks > kMaxBlocks) {
            return linearInvalid("more output than one launch can write");
        }
        productKernel<Tile, kTurnedA><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(args.splits)),
                                        Tile::kThreads, 0, stream>>>(args);
        ZCGVS_LAUNCH_CHECK("linear gradient");
        return static_cast<int>(ZCGVS_OK);
    });
}

template <class InputTile, class WeightTile>
int launchBothProducts(ProductArgs input, ProductArgs weight, ColumnJoin bias, hipStream_t stream) {
    input.tiles_m = divideUp(input.m, InputTile::kM);
    input.tiles_n = divideUp(input.n, InputTile::kN);
    weight.tiles_m = divideUp(weight.m, WeightTile::kM);
    weight.tiles_n = divideUp(weight.n, WeightTile::kN);
    const long long input_blocks = static_cast<long long>(input.tiles_m) * input.tiles_n * input.splits;
    const long long weight_blocks = static_cast<long long>(weight.tiles_m) * weight.tiles_n * weight.splits;
    const long long bias_blocks = bias.out == nullptr ? 0 : divideUp(bias.columns, kJoinColumns);
    if (input_blocks + weight_blocks + bias_blocks > kMaxBlocks) {
        return linearInvalid("more output than one launch can write");
    }
    bothProductsKernel<InputTile, WeightTile><<<static_cast<unsigned>(input_blocks + weight_blocks + bias_blocks),
                                                InputTile::kThreads, 0, stream>>>(
        input, weight, static_cast<int>(input_blocks), static_cast<int>(weight_blocks), bias);
    ZCGVS_LAUNCH_CHECK("linear gradient");
    return ZCGVS_OK;
}

// The sums of both products' splits and the bias's, whichever there are, in one launch: the first blocks take packs of
// four values of the products, the last ones 16 columns of the bias.
template <typename T>
__global__ __launch_bounds__(kColumnThreads) void joinProductsKernel(ProductArgs input, ProductArgs weight, int input_blocks,
                                                                     int weight_blocks, ColumnJoin bias) {
    const int block = static_cast<int>(blockIdx.x);
    if (block >= input_blocks + weight_blocks) {
        joinColumns(bias.partials, bias.rows, bias.columns, static_cast<T*>(bias.out), block - input_blocks - weight_blocks);
        return;
    }
    const bool first = block < input_blocks;
    const ProductArgs& args = first ? input : weight;
    const int blocks = first ? input_blocks : weight_blocks;
    const int packs_per_row = (args.n + 3) / 4;
    const long long packs = static_cast<long long>(args.m) * packs_per_row;
    const long long split_values = static_cast<long long>(args.m) * args.n;
    for (long long p = static_cast<long long>(first ? block : block - input_blocks) * kColumnThreads + threadIdx.x; p < packs;
         p += static_cast<long long>(blocks) * kColumnThreads) {
        const long long row = p / packs_per_row;
        const int column = 4 * static_cast<int>(p - row * packs_per_row);
        const int left = args.n - column;
        const float* from = args.partials + row * args.n + column;
        f32x4 sum = loadFour(from, left);
#pragma unroll 4
        for (int s = 1; s < args.splits; ++s) {
            sum += loadFour(from + s * split_values, left);
        }
        storeFour(sum, static_cast<T*>(args.out) + row * args.out_stride + column, left);
    }
}

inline int joinBlocks(const ProductArgs& args) {
    const long long packs = static_cast<long long>(args.m) * ((args.n + 3) / 4);
    return args.out == nullptr || args.splits == 1
               ? 0
               : static_cast<int>(std::min(4096ll, (packs + kColumnThreads - 1) / kColumnThreads));
}

template <typename T>
int launchJoins(const ProductArgs& input, const ProductArgs& weight, const ColumnJoin& bias, hipStream_t stream) {
    const int input_blocks = joinBlocks(input);
    const int weight_blocks = joinBlocks(weight);
    const int bias_blocks = bias.out == nullptr ? 0 : divideUp(bias.columns, kJoinColumns);
    if (input_blocks + weight_blocks + bias_blocks == 0) {
        return ZCGVS_OK;
    }
    joinProductsKernel<T><<<static_cast<unsigned>(input_blocks + weight_blocks + bias_blocks), kColumnThreads, 0, stream>>>(
        input, weight, input_blocks, weight_blocks, bias);
    ZCGVS_LAUNCH_CHECK("linear gradient");
    return ZCGVS_OK;
}

}  // namespace

template <typename T>
int launchLinear(const LinearPlan& plan, int activation, LinearArgs args, hipStream_t stream) {
    return plan.thin > 0 ? launchThin<T>(plan.thin, activation, args, stream) : launchTiles<T, false>(plan, activation, args, stream);
}

template <typename T>
int launchLinearSlope(const LinearPlan& plan, int activation, LinearArgs args, hipStream_t stream) {
    return launchTiles<T, true>(plan, activation, args, stream);
}

template <typename T>
int launchLinearProducts(ProductPlan input_plan, bool input_direct, ProductArgs input, ProductPlan weight_plan,
                         bool weight_direct, ProductArgs weight, ColumnJoin bias, hipStream_t stream) {
    const bool wants_input = input.out != nullptr;
    const bool wants_weight = weight.out != nullptr;
    int status = ZCGVS_OK;
    if (wants_input && wants_weight && input_direct == weight_direct && input_plan.shape == TileShape::k64x64 &&
        weight_plan.shape == TileShape::k64x64) {
        if constexpr (std::is_same_v<T, float>) {
            status = launchBothProducts<SplitTile<64, 64, 2, 2, false, true>, SplitTile<64, 64, 2, 2, true, true>>(
                input, weight, bias, stream);
        } else if (input_direct) {
            status = launchBothProducts<MatrixTile<T, 64, 64, 2, 2, false, true, true>,
                                        MatrixTile<T, 64, 64, 2, 2, true, true, true>>(input, weight, bias, stream);
        } else {
            status = launchBothProducts<MatrixTile<T, 64, 64, 2, 2, false, true, false>,
                                        MatrixTile<T, 64, 64, 2, 2, true, true, false>>(input, weight, bias, stream);
        }
        bias.out = nullptr;
    } else {
        if (wants_input) {
            status = launchProduct<T, false>(input_plan, input_direct, input, stream);
        }
        if (status == ZCGVS_OK && wants_weight) {
            status = launchProduct<T, true>(weight_plan, weight_direct, weight, stream);
        }
    }
    if (status == ZCGVS_OK) {
        status = launchJoins<T>(input, weight, bias, stream);
    }
    return status;
}

}  // namespace zcgvs_hip
