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
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"
#include "elements.hpp"
#include "matrix_tile.hpp"

namespace zcgvs_hip {

namespace {

// 1 / (1 + exp(-x)): exp2 and the reciprocal of the hardware, each within 1 ulp.
__device__ __forceinline__ float logistic(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}

// The activation's value and slope at g.
template <int kActivation>
__device__ __forceinline__ float activate(float g) {
    if constexpr (kActivation == ZCGVS_ACT_SILU) {
        return g * logistic(g);
    } else if constexpr (kActivation == ZCGVS_ACT_GELU) {
        return 0.5f * g * (1.0f + erff(g * 0.70710678f));
    } else {
        // 0.5 (1 + tanh(z)) is the logistic function of 2 z
        return g * logistic(1.59576912f * (g + 0.044715f * g * g * g));
    }
}

template <int kActivation>
__device__ __forceinline__ void activateBoth(float g, float& value, float& slope) {
    if constexpr (kActivation == ZCGVS_ACT_SILU) {
        const float y = logistic(g);
        value = g * y;
        slope = y + value * (1.0f - y);
    } else if constexpr (kActivation == ZCGVS_ACT_GELU) {
        const float y = 0.5f * (1.0f + erff(g * 0.70710678f));
        value = g * y;
        slope = y + g * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * g * g);
    } else {
        const float y = logistic(1.59576912f * (g + 0.044715f * g * g * g));
        value = g * y;
        slope = y + value * (1.0f - y) * (1.59576912f * (1.0f + 0.134145f * g * g));
    }
}

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
    bool out_packed;  // stores of four results are aligned
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
    int tile_m, tile_n;
    tileOf(args.tiles_m, args.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * Tile::kM;
    const int n0 = tile_n * (Tile::kN / 2);
    const T* x = static_cast<const T*>(args.x);
    const T* gate = static_cast<const T*>(args.gate);
    const T* up = static_cast<const T*>(args.up);

    typename Tile::Sums sums;
    Tile::clear(sums);
    Tile::accumulate(
        lds, [&](int r) { return x + min(m0 + r, args.rows - 1) * args.x_stride; }, args.x_stride, 0,
        [&](int r) {
            const int j = r % kWaveN;
            const int n = min(n0 + r / kWaveN * kHalf + j % kHalf, args.hidden - 1);
            return (j < kHalf ? gate : up) + n * args.weight_stride;
        },
        args.weight_stride, 0, args.dim, sums);

    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        const int m = m0 + (Tile::waveM() * Tile::kBlocksM + i) * 16 + (lane & 15);
        if (m >= args.rows) {
            continue;
        }
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            const int n = n0 + Tile::waveN() * kHalf + j * 16 + 4 * (lane >> 4);
            const f32x4 g = sums[i][j];
            const f32x4 u = sums[i][j + kPairs];
            T* to = static_cast<T*>(args.out) + m * args.out_stride + n;
            if constexpr (!kGradient) {
                if (n < args.hidden) {
                    f32x4 h;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[e] = activate<kActivation>(g[e]) * u[e];
                    }
                    storeFour(h, to, args.hidden - n, args.out_packed);
                }
            } else if (n < args.out_stride) {
                const T* d = static_cast<const T*>(args.out_gradient) + m * args.out_gradient_stride + n;
                f32x4 dg, du;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float from = n + e < args.hidden ? static_cast<float>(d[e]) : 0.0f;
                    float value, slope;
                    activateBoth<kActivation>(g[e], value, slope);
                    dg[e] = n + e < args.hidden ? from * u[e] * slope : 0.0f;
                    du[e] = n + e < args.hidden ? from * value : 0.0f;
                }
                storeFour(dg, to, 4, true);
                storeFour(du, to + args.du_offset, 4, true);
            }
        }
    }
}

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
    void* out;
    std::int64_t out_stride;
    bool out_packed;
};

template <class Tile>
__global__ __launch_bounds__(Tile::kThreads) void inputGradientKernel(InputGradientArgs args) {
    using T = typename Tile::T;
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    int tile_m, tile_n;
    tileOf(args.tiles_m, args.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * Tile::kM;
    const int n0 = tile_n * Tile::kN;
    typename Tile::Sums sums;
    Tile::clear(sums);
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const T* d = static_cast<const T*>(args.dg) + (part == 0 ? 0 : args.du_offset);
        const T* weight = static_cast<const T*>(part == 0 ? args.gate : args.up);
        Tile::accumulate(
            lds, [&](int r) { return d + min(m0 + r, args.rows - 1) * args.d_stride; }, args.d_stride, 0,
            [&](int) { return weight + n0; }, args.weight_stride, args.dim - n0, args.hidden, sums);
    }
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        const int m = m0 + (Tile::waveM() * Tile::kBlocksM + i) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j) {
            const int n = n0 + (Tile::waveN() * Tile::kBlocksN + j) * 16 + 4 * (lane >> 4);
            if (m < args.rows && n < args.dim) {
                storeFour(sums[i][j], static_cast<T*>(args.out) + m * args.out_stride + n, args.dim - n,
                          args.out_packed);
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
    void* gate_out;
    void* up_out;
    std::int64_t out_stride;
    bool out_packed;
};

template <class Tile>
__global__ __launch_bounds__(Tile::kThreads) void weightGradientKernel(WeightGradientArgs args) {
    using T = typename Tile::T;
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[Tile::kLdsBytes];
    int tile_m, tile_n;
    tileOf(2 * args.tiles_m, args.tiles_n, tile_m, tile_n);
    const bool second = tile_m >= args.tiles_m;
    const int m0 = (second ? tile_m - args.tiles_m : tile_m) * Tile::kM;
    const int n0 = tile_n * Tile::kN;
    const T* d = static_cast<const T*>(args.dg) + (second ? args.du_offset : 0);
    const T* x = static_cast<const T*>(args.x);
    typename Tile::Sums sums;
    Tile::clear(sums);
    // the rows of dg and du are padded to whole chunks
    Tile::accumulate(
        lds, [&](int) { return d + m0; }, args.d_stride, static_cast<int>(args.d_stride) - m0,
        [&](int) { return x + n0; }, args.x_stride, args.dim - n0, args.rows, sums);
    T* out = static_cast<T*>(second ? args.up_out : args.gate_out);
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int i = 0; i < Tile::kBlocksM; ++i) {
        const int m = m0 + (Tile::waveM() * Tile::kBlocksM + i) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < Tile::kBlocksN; ++j) {
            const int n = n0 + (Tile::waveN() * Tile::kBlocksN + j) * 16 + 4 * (lane >> 4);
            if (m < args.hidden && n < args.dim) {
                storeFour(sums[i][j], out + m * args.out_stride + n, args.dim - n, args.out_packed);
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------

constexpr long long kMaxBlocks = (1ll << 22) - 1;  // a launch has less than 2^32 threads

int invalid(const char* message) {
    return setError(ZCGVS_ERR_INVALID_ARGUMENT, std::string("zcgvs gated projection: ") + message);
}

std::int64_t rowStride(std::int64_t stride, int length) { return stride == 0 ? length : stride; }

int divideUp(std::int64_t a, int b) { return static_cast<int>((a + b - 1) / b); }

// Rows that the 16-byte copies can read: whole aligned chunks.
bool directRows(const void* base, std::int64_t stride, int length, int dtype) {
    return alignedRows(base, stride, dtype, 16) && length * elementBytes(dtype) % 16 == 0;
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

// Calls body(std::integral_constant<int, activation>).
template <typename Body>
int withActivation(int activation, Body&& body) {
    switch (activation) {
        case ZCGVS_ACT_GELU:
            return body(std::integral_constant<int, ZCGVS_ACT_GELU>{});
        case ZCGVS_ACT_GELU_TANH:
            return body(std::integral_constant<int, ZCGVS_ACT_GELU_TANH>{});
        default:
            return body(std::integral_constant<int, ZCGVS_ACT_SILU>{});
    }
}

// Calls body(Tile{}) with the tile for an m x n product: 128 x 128 where that fills the GPU, 64 x 64
// otherwise; loads past the registers where the rows allow.
template <typename T, bool kTurnedA, bool kTurnedB, typename Body>
int withTile(long long tiles_128, bool direct, Body&& body) {
    if (tiles_128 >= deviceComputeUnits()) {
        return direct ? body(MatrixTile<T, 128, 128, 2, 2, kTurnedA, kTurnedB, true>{})
                      : body(MatrixTile<T, 128, 128, 2, 2, kTurnedA, kTurnedB, false>{});
    }
    return direct ? body(MatrixTile<T, 64, 64, 2, 2, kTurnedA, kTurnedB, true>{})
                  : body(MatrixTile<T, 64, 64, 2, 2, kTurnedA, kTurnedB, false>{});
}

long long tilesOf(std::int64_t m, std::int64_t n, int side) {
    return static_cast<long long>(divideUp(m, side)) * divideUp(n, side);
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
    return withTile<T, false, false>(tilesOf(d.rows, 2 * static_cast<std::int64_t>(d.hidden), 128), direct, [&](auto tile) {
        using Tile = decltype(tile);
        return withActivation(d.activation, [&](auto activation) {
            args.tiles_m = divideUp(d.rows, Tile::kM);
            args.tiles_n = divideUp(d.hidden, Tile::kN / 2);
            const long long blocks = static_cast<long long>(args.tiles_m) * args.tiles_n;
            if (blocks > kMaxBlocks) {
                return invalid("more output than one launch can write");
            }
            gatedKernel<Tile, decltype(activation)::value, kGradient>
                <<<static_cast<unsigned>(blocks), Tile::kThreads, 0, stream>>>(args);
            ZCGVS_LAUNCH_CHECK("gated projection");
            return static_cast<int>(ZCGVS_OK);
        });
    });
}

// Elements from row to row of dg and du in the workspace.
std::int64_t gradientStride(const zcgvs_gated_desc& d) { return (static_cast<std::int64_t>(d.hidden) + 7) / 8 * 8; }

template <typename T>
int launchInputGradient(const zcgvs_gated_desc& d, InputGradientArgs args, hipStream_t stream) {
    const bool direct = directRows(args.gate, args.weight_stride, d.dim, d.dtype) &&
                        directRows(args.up, args.weight_stride, d.dim, d.dtype);
    return withTile<T, false, true>(tilesOf(d.rows, d.dim, 128), direct, [&](auto tile) {
        using Tile = decltype(tile);
        args.tiles_m = divideUp(d.rows, Tile::kM);
        args.tiles_n = divideUp(d.dim, Tile::kN);
        const long long blocks = static_cast<long long>(args.tiles_m) * args.tiles_n;
        if (blocks > kMaxBlocks) {
            return invalid("more output than one launch can write");
        }
        inputGradientKernel<Tile><<<static_cast<unsigned>(blocks), Tile::kThreads, 0, stream>>>(args);
        ZCGVS_LAUNCH_CHECK("gated gradient");
        return static_cast<int>(ZCGVS_OK);
    });
}

template <typename T>
int launchWeightGradient(const zcgvs_gated_desc& d, WeightGradientArgs args, hipStream_t stream) {
    const bool direct = directRows(args.x, args.x_stride, d.dim, d.dtype);
    return withTile<T, true, true>(2 * tilesOf(d.hidden, d.dim, 128), direct, [&](auto tile) {
        using Tile = decltype(tile);
        args.tiles_m = divideUp(d.hidden, Tile::kM);
        args.tiles_n = divideUp(d.dim, Tile::kN);
        const long long blocks = 2ll * args.tiles_m * args.tiles_n;
        if (blocks > kMaxBlocks) {
            return invalid("more output than one launch can write");
        }
        weightGradientKernel<Tile><<<static_cast<unsigned>(blocks), Tile::kThreads, 0, stream>>>(args);
        ZCGVS_LAUNCH_CHECK("gated gradient");
        return static_cast<int>(ZCGVS_OK);
    });
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
    args.out_packed = alignedRows(d_out, args.out_stride, d.dtype, 4 * elementBytes(d.dtype));
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
    const std::size_t one = static_cast<std::size_t>(desc->rows) * static_cast<std::size_t>(gradientStride(*desc));
    return std::max<std::size_t>(256, 2 * one * static_cast<std::size_t>(elementBytes(desc->dtype)));
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
        form.out_packed = true;
        form.out_gradient = d_out_gradient;
        form.out_gradient_stride = from_stride;
        form.du_offset = d.rows * form.out_stride;
        int done = launchGated<T, true>(d, form, toStream(stream));
        if (done == ZCGVS_OK && d_x_gradient != nullptr) {
            InputGradientArgs args{};
            args.dg = d_workspace;
            args.d_stride = form.out_stride;
            args.du_offset = form.du_offset;
            args.gate = d.gate;
            args.up = d.up;
            args.weight_stride = rowStride(d.weight_stride, d.dim);
            args.rows = static_cast<int>(d.rows);
            args.dim = d.dim;
            args.hidden = d.hidden;
            args.out = d_x_gradient;
            args.out_stride = x_out_stride;
            args.out_packed = alignedRows(d_x_gradient, x_out_stride, d.dtype, 4 * elementBytes(d.dtype));
            done = launchInputGradient<T>(d, args, toStream(stream));
        }
        if (done == ZCGVS_OK && d_gate_gradient != nullptr) {
            WeightGradientArgs args{};
            args.dg = d_workspace;
            args.d_stride = form.out_stride;
            args.du_offset = form.du_offset;
            args.x = d.x;
            args.x_stride = rowStride(d.x_stride, d.dim);
            args.rows = static_cast<int>(d.rows);
            args.dim = d.dim;
            args.hidden = d.hidden;
            args.gate_out = d_gate_gradient;
            args.up_out = d_up_gradient;
            args.out_stride = weight_out_stride;
            args.out_packed = alignedRows(d_gate_gradient, weight_out_stride, d.dtype, 4 * elementBytes(d.dtype)) &&
                              alignedRows(d_up_gradient, weight_out_stride, d.dtype, 4 * elementBytes(d.dtype));
            done = launchWeightGradient<T>(d, args, toStream(stream));
        }
        return done;
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

}  // extern "C"
