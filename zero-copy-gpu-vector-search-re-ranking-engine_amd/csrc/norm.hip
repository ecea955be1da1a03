// Root-mean-square norm of the sum of two rows, with int8 rows and scales as one of its outputs, and its gradient.
//
//     s = x + residual,  r = 1 / sqrt(mean(s^2) + eps),  y = s r (w + c)
//     ds = r (g - u mean(g u)) + ds',  u = s r,  g = dy (w + c);   dw = sum over rows of dy u
//
// Memory bound: every operand is read once and every result written once. A row stays in the registers of one
// wavefront (up to 2048 16-bit or 1024 float32 values) or of one workgroup between the sum of its squares and its
// results, so nothing is read twice. The squares' sum, the mean and the rows are float32 throughout; s is rounded
// where it is stored only.
// The gradient's workgroups take every gridDim.x-th row and keep their part of dw in registers; each writes
// one row of float32 sums, which a second launch adds in the order of the workgroups: the same bits on every call.
// Measured, 16,384 rows of 1024 bfloat16: 26.9 us with residual and sum (134 MB, 5.0 TB/s, a large copy's rate), the
// gradient 31.1 (24 and the second launch); 1001 rows of 384 float32, the gradient 10.7 (two launches of 5).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "column_sums.hpp"
#include "common.hpp"
#include "elements.hpp"
#include "matrix_plan.hpp"
#include "matrix_tile.hpp"

namespace zcgvs_hip {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / kWave;
constexpr int kNormMaxDim = 16384;
constexpr long long kNormMaxBlocks = (1ll << 24) - 1;  // a launch has less than 2^32 threads, of 256 a block

// Values of 16 bytes, which a thread takes at a time.
template <typename T>
constexpr int kNormPack = 16 / static_cast<int>(sizeof(T));

// kCount values to `to` on, of which `left` are wanted.
template <typename T, int kCount>
__device__ __forceinline__ void storeSome(const float (&from)[kCount], int left, T* to) {
    if (left >= kCount) {
        storePack(from, to);
    } else {
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            if (e < left) {
                to[e] = static_cast<T>(from[e]);
            }
        }
    }
}

// The int8 codes of kCount values.
template <int kCount>
__device__ __forceinline__ void storeCodes(const float (&from)[kCount], float inverse, int left, std::int8_t* to) {
    typename Pack<std::int8_t, kCount>::stored codes;
#pragma unroll
    for (int e = 0; e < kCount; ++e) {
        codes[e] = quantizeCode(from[e], inverse);
    }
    if (left >= kCount) {
        *reinterpret_cast<typename Pack<std::int8_t, kCount>::stored*>(to) = codes;
    } else {
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            if (e < left) {
                to[e] = codes[e];
            }
        }
    }
}

// op over a row's kThreads threads (a wavefront, or the whole workgroup through `shared`, which holds one value
// a wavefront and is free again after the next call's barrier); every thread gets the result.
template <int kThreads, typename Op>
__device__ __forceinline__ float overRow(float value, float* shared, Op op) {
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) {
        value = op(value, waveXor(value, offset));
    }
    if constexpr (kThreads > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0) {
            shared[threadIdx.x / kWave] = value;
        }
        __syncthreads();
        value = shared[0];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) {
            value = op(value, shared[w]);
        }
    }
    return value;
}

struct NormArgs {
    const void* x;
    std::int64_t x_stride;
    const void* residual;
    std::int64_t residual_stride;
    const void* weight;
    long long rows;
    long long first;  // row of the launch's first workgroup
    int dim;
    float weight_offset;
    float eps;
    void* out;
    std::int64_t out_stride;
    float* out_scales;
    void* sum;
    std::int64_t sum_stride;
};

// 1 / sqrt(mean + eps) of a row whose squares add up to `squares`.
__device__ __forceinline__ float rowFactor(float squares, int dim, float eps) {
    return 1.0f / sqrtf(squares / static_cast<float>(dim) + eps);
}

// The calling thread's kVectors packs of one row, as they are stored. Where rows are whole packs (`whole`) no load hangs
// on a branch, so that all are on their way together.
template <typename T, int kThreads, int kVectors>
struct RowPacks {
    typedef typename Pack<T, kNormPack<T>>::type Stored;
    Stored packs[kVectors];

    __device__ __forceinline__ void load(const T* row, int dim, bool whole) {
        constexpr int kPack = kNormPack<T>;
        const int lane = static_cast<int>(threadIdx.x) % kThreads;
        if (whole) {
#pragma unroll
            for (int i = 0; i < kVectors; ++i) {
                const int c = (i * kThreads + lane) * kPack;
                const void* from = c < dim ? static_cast<const void*>(row + c) : static_cast<const void*>(&zero_chunk);
                packs[i] = *static_cast<const typename Pack<T, kPack>::stored*>(from);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVectors; ++i) {
                const int c = (i * kThreads + lane) * kPack;
                packs[i] = Stored{};
                if (c + kPack <= dim) {
                    packs[i] = *reinterpret_cast<const typename Pack<T, kPack>::stored*>(row + c);
                } else {
#pragma unroll
                    for (int e = 0; e < kPack; ++e) {
                        if (c + e < dim) {
                            packs[i][e] = row[c + e];
                        }
                    }
                }
            }
        }
    }
    __device__ __forceinline__ float at(int i, int e) const { return static_cast<float>(packs[i][e]); }
};

// kThreads threads a row, kVectors packs each.
template <typename T, typename Out, int kThreads, int kVectors>
__global__ __launch_bounds__(kNormThreads) void residualNormKernel(NormArgs args) {
    constexpr int kPack = kNormPack<T>;
    __shared__ float shared[2][kNormWaves];
    const int lane = static_cast<int>(threadIdx.x) % kThreads;
    const long long row = args.first + static_cast<long long>(blockIdx.x) * (blockDim.x / kThreads) + threadIdx.x / kThreads;
    if (row >= args.rows) {
        return;  // (a whole row's threads, and the whole workgroup where they share memory)
    }
    float s[kVectors][kPack];
    const bool whole = args.dim % kPack == 0;
    RowPacks<T, kThreads, kVectors> x, residual, weight;
    x.load(static_cast<const T*>(args.x) + row * args.x_stride, args.dim, whole);
    if (args.residual != nullptr) {
        residual.load(static_cast<const T*>(args.residual) + row * args.residual_stride, args.dim, whole);
    }
    if (args.weight != nullptr) {
        weight.load(static_cast<const T*>(args.weight), args.dim, whole);
    }
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            s[i][e] = args.residual != nullptr ? x.at(i, e) + residual.at(i, e) : x.at(i, e);
        }
    }
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            squares = fmaf(s[i][e], s[i][e], squares);
        }
    }
    const auto add = [](float a, float b) { return a + b; };
    const float factor = rowFactor(overRow<kThreads>(squares, shared[0], add), args.dim, args.eps);
    if (args.sum != nullptr) {
        T* sum = static_cast<T*>(args.sum) + row * args.sum_stride;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const int c = (i * kThreads + lane) * kPack;
            storeSome(s[i], args.dim - c, sum + c);
        }
    }
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int c = (i * kThreads + lane) * kPack;
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            s[i][e] *= factor * ((args.weight != nullptr ? weight.at(i, e) : 1.0f) + args.weight_offset);
            peak = fmaxf(peak, c + e < args.dim ? fabsf(s[i][e]) : 0.0f);
        }
    }
    if constexpr (std::is_same_v<Out, std::int8_t>) {
        peak = overRow<kThreads>(peak, shared[1], [](float a, float b) { return fmaxf(a, b); });
        const float scale = peak > 0.0f ? peak / 127.0f : 1.0f;
        const float inverse = 1.0f / scale;
        std::int8_t* out = static_cast<std::int8_t*>(args.out) + row * args.out_stride;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const int c = (i * kThreads + lane) * kPack;
            storeCodes(s[i], inverse, args.dim - c, out + c);
        }
        if (lane == 0) {
            args.out_scales[row] = scale;
        }
    } else {
        Out* out = static_cast<Out*>(args.out) + row * args.out_stride;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const int c = (i * kThreads + lane) * kPack;
            storeSome(s[i], args.dim - c, out + c);
        }
    }
}

struct NormGradientArgs {
    const void* out_gradient;
    std::int64_t out_gradient_stride;
    const void* sum_gradient;
    std::int64_t sum_gradient_stride;
    void* x_gradient;
    std::int64_t x_gradient_stride;
    float* partials;  // [workgroups, dim] of the weight's gradient, or null: not wanted
};

template <typename T, int kThreads, int kVectors>
__global__ __launch_bounds__(kNormThreads) void residualNormGradientKernel(NormArgs args, NormGradientArgs more) {
    constexpr int kPack = kNormPack<T>;
    constexpr int kRows = kNormThreads / kThreads;
    // sums over the row of two values a wavefront, two sets by turns; a workgroup of several rows joins its sums
    // of the weight's gradient here
    __shared__ float shared[kThreads > kWave ? 4 * kNormWaves : kThreads * kPack];
    const int lane = static_cast<int>(threadIdx.x) % kThreads;
    const int slot = static_cast<int>(threadIdx.x) / kThreads;
    const bool whole = args.dim % kPack == 0;
    float w[kVectors][kPack], dw[kVectors][kPack];
    {
        RowPacks<T, kThreads, kVectors> weight;
        if (args.weight != nullptr) {
            weight.load(static_cast<const T*>(args.weight), args.dim, whole);
        }
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                w[i][e] = (args.weight != nullptr ? weight.at(i, e) : 1.0f) + args.weight_offset;
                dw[i][e] = 0.0f;
            }
        }
    }
    RowPacks<T, kThreads, kVectors> x_row, residual_row, d_row, through_row;
    auto load = [&](long long row) {
        x_row.load(static_cast<const T*>(args.x) + row * args.x_stride, args.dim, whole);
        d_row.load(static_cast<const T*>(more.out_gradient) + row * more.out_gradient_stride, args.dim, whole);
        if (args.residual != nullptr) {
            residual_row.load(static_cast<const T*>(args.residual) + row * args.residual_stride, args.dim, whole);
        }
        if (more.sum_gradient != nullptr) {
            through_row.load(static_cast<const T*>(more.sum_gradient) + row * more.sum_gradient_stride, args.dim, whole);
        }
    };
    int turn = 0;
    const long long first = static_cast<long long>(blockIdx.x) * kRows + slot;
    const long long step = static_cast<long long>(gridDim.x) * kRows;
    constexpr bool kAhead = kVectors * kPack <= 24;  // the registers do for the next row as well
    if (kAhead && first < args.rows) {
        load(first);
    }
    for (long long row = first; row < args.rows; row += step) {
        if (!kAhead) {
            load(row);
        }
        float s[kVectors][kPack], d[kVectors][kPack], result[kVectors][kPack];
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                s[i][e] = args.residual != nullptr ? x_row.at(i, e) + residual_row.at(i, e) : x_row.at(i, e);
                d[i][e] = d_row.at(i, e);
                result[i][e] = more.sum_gradient != nullptr ? through_row.at(i, e) : 0.0f;
            }
        }
        if (kAhead && row + step < args.rows) {
            load(row + step);  // on its way while this one is used
        }
        float squares = 0.0f, along = 0.0f;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                squares = fmaf(s[i][e], s[i][e], squares);
                along = fmaf(d[i][e] * w[i][e], s[i][e], along);
            }
        }
        const auto add = [](float a, float b) { return a + b; };
        if constexpr (kThreads > kWave) {
            // both sums with one barrier; the other set is the row's before, which every thread has read
            float* set = shared + turn * 2 * kNormWaves;
            turn ^= 1;
            squares = overRow<kWave>(squares, nullptr, add);
            along = overRow<kWave>(along, nullptr, add);
            if ((threadIdx.x & (kWave - 1)) == 0) {
                set[threadIdx.x / kWave] = squares;
                set[kNormWaves + threadIdx.x / kWave] = along;
            }
            __syncthreads();
            squares = set[0];
            along = set[kNormWaves];
#pragma unroll
            for (int v = 1; v < kNormWaves; ++v) {
                squares += set[v];
                along += set[kNormWaves + v];
            }
        } else {
            squares = overRow<kWave>(squares, nullptr, add);
            along = overRow<kWave>(along, nullptr, add);
        }
        const float factor = rowFactor(squares, args.dim, args.eps);
        const float mean = along * factor / static_cast<float>(args.dim);  // of g u
        T* to = static_cast<T*>(more.x_gradient) + row * more.x_gradient_stride;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const int c = (i * kThreads + lane) * kPack;
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                const float u = s[i][e] * factor;
                dw[i][e] = fmaf(d[i][e], u, dw[i][e]);
                result[i][e] += factor * (d[i][e] * w[i][e] - u * mean);
            }
            if (more.x_gradient != nullptr) {
                storeSome(result[i], args.dim - c, to + c);
            }
        }
    }
    if (more.partials == nullptr) {
        return;
    }
    float* to = more.partials + static_cast<long long>(blockIdx.x) * args.dim;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int c = (i * kThreads + lane) * kPack;
        if constexpr (kRows > 1) {
            // the rows' threads add theirs one after the other
            for (int turn_of = 0; turn_of < kRows; ++turn_of) {
                __syncthreads();
                if (slot == turn_of) {
#pragma unroll
                    for (int e = 0; e < kPack; ++e) {
                        float* at = shared + e * kThreads + lane;
                        dw[i][e] += turn_of > 0 ? *at : 0.0f;
                        *at = dw[i][e];
                    }
                }
            }
        }
        if (slot == kRows - 1) {
            storeSome(dw[i], args.dim - c, to + c);
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------

int invalid(const char* message) {
    return setError(ZCGVS_ERR_INVALID_ARGUMENT, std::string("zcgvs residual norm: ") + message);
}

int checkNorm(const zcgvs_norm_desc* desc) {
    if (desc == nullptr) {
        return invalid("null descriptor");
    }
    const zcgvs_norm_desc& d = *desc;
    if (!validElement(d.dtype)) {
        return invalid("the operands must hold float32, float16 or bfloat16");
    }
    if (d.dim <= 0 || d.dim > kNormMaxDim) {
        return invalid("dim must lie in [1, 16384]");
    }
    if (d.rows < 0 || d.rows > (1 << 30)) {
        return invalid("rows must lie in [0, 2^30]");
    }
    if (rowStride(d.x_stride, d.dim) < d.dim || (d.residual != nullptr && rowStride(d.residual_stride, d.dim) < d.dim)) {
        return invalid("a row stride is smaller than dim");
    }
    if (!(d.eps >= 0.0f) || !std::isfinite(d.eps) || !std::isfinite(d.weight_offset)) {
        return invalid("eps must be finite and at least 0, weight_offset finite");
    }
    if (d.rows > 0 && d.x == nullptr) {
        return invalid("null device pointer");
    }
    return ZCGVS_OK;
}

// Calls body(threads a row, packs a thread), both as integral constants: a wavefront a row where at most four packs
// a thread hold it.
template <typename T, typename Body>
int withRowShape(int dim, Body&& body) {
    const auto wave = std::integral_constant<int, kWave>{};
    const auto group = std::integral_constant<int, kNormThreads>{};
    const int packs = divideUp(dim, kNormPack<T>);
    switch (divideUp(packs, kWave)) {
        case 1: return body(wave, std::integral_constant<int, 1>{});
        case 2: return body(wave, std::integral_constant<int, 2>{});
        case 3: return body(wave, std::integral_constant<int, 3>{});
        case 4: return body(wave, std::integral_constant<int, 4>{});
        default: break;
    }
    const int each = divideUp(packs, kNormThreads);
    if (each <= 2) {
        return body(group, std::integral_constant<int, 2>{});
    }
    if (each <= 4) {
        return body(group, std::integral_constant<int, 4>{});
    }
    if constexpr (sizeof(T) == 4) {
        if (each > 8) {
            return body(group, std::integral_constant<int, 16>{});
        }
    }
    return body(group, std::integral_constant<int, 8>{});
}

NormArgs normArgs(const zcgvs_norm_desc& d) {
    NormArgs args{};
    args.x = d.x;
    args.x_stride = rowStride(d.x_stride, d.dim);
    args.residual = d.residual;
    args.residual_stride = rowStride(d.residual_stride, d.dim);
    args.weight = d.weight;
    args.rows = d.rows;
    args.dim = d.dim;
    args.weight_offset = d.weight_offset;
    args.eps = d.eps;
    return args;
}

// Workgroups of the gradient, rows of a wavefront four at a time: as many as are on a CU together by their registers, each
// with rows to load ahead. 16,384 x 1024 bfloat16 (two packs a thread): two to a CU 33.4 us, three 31.1, four 38.1; 30,000 x
// 200 (one): 34.3, 28.0, 24.9; 8192 x 2048 (four): 33.4, 38.8, 39.0.
int gradientBlocks(const zcgvs_norm_desc& d) {
    const int packs = divideUp(divideUp(d.dim, 16 / elementBytes(d.dtype)), kWave);
    const int rows_each = packs <= 4 ? kNormWaves : 1;
    const long long most = (packs == 1 ? 4ll : packs == 2 ? 3ll : 2ll) * deviceComputeUnits();
    return static_cast<int>(std::min<long long>(most, (d.rows + rows_each - 1) / rows_each));
}

}  // namespace

}  // namespace zcgvs_hip

using namespace zcgvs_hip;

extern "C" {

int zcgvs_residual_norm_max_dim(void) { return kNormMaxDim; }

int zcgvs_residual_norm(const zcgvs_norm_desc* desc, void* d_out, std::int64_t out_stride, int out_dtype,
                        float* d_out_scales, void* d_sum, std::int64_t sum_stride, zcgvs_stream_t stream) {
    const int status = checkNorm(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_norm_desc& d = *desc;
    const bool codes = out_dtype == ZCGVS_DTYPE_I8;
    if (!codes && out_dtype != d.dtype && out_dtype != ZCGVS_DTYPE_F32) {
        return invalid("the output must hold the operands' type, float32 or int8");
    }
    if (rowStride(out_stride, d.dim) < d.dim || (d_sum != nullptr && rowStride(sum_stride, d.dim) < d.dim)) {
        return invalid("an output's row stride is smaller than dim");
    }
    if (d.rows == 0) {
        return clearError();
    }
    if (d_out == nullptr || (codes && d_out_scales == nullptr)) {
        return invalid("null device pointer");
    }
    NormArgs args = normArgs(d);
    args.out = d_out;
    args.out_stride = rowStride(out_stride, d.dim);
    args.out_scales = d_out_scales;
    args.sum = d_sum;
    args.sum_stride = rowStride(sum_stride, d.dim);
    const int launched = withElement(d.dtype, [&](auto element) {
        using T = decltype(element);
        return withRowShape<T>(d.dim, [&](auto threads, auto vectors) {
            constexpr int kThreads = decltype(threads)::value;
            constexpr int kVectors = decltype(vectors)::value;
            // a wavefront's rows in workgroups of four, or of one where that leaves CUs without one
            const int rows_each =
                kThreads > kWave || d.rows <= kNormWaves * static_cast<std::int64_t>(deviceComputeUnits()) ? 1 : kNormWaves;
            const unsigned block_threads = static_cast<unsigned>(rows_each * kThreads);
            for (args.first = 0; args.first < d.rows; args.first += kNormMaxBlocks * rows_each) {
                const unsigned blocks =
                    static_cast<unsigned>(std::min<long long>(kNormMaxBlocks, (d.rows - args.first + rows_each - 1) / rows_each));
                if (codes) {
                    residualNormKernel<T, std::int8_t, kThreads, kVectors><<<blocks, block_threads, 0, toStream(stream)>>>(args);
                } else if (out_dtype == d.dtype) {
                    residualNormKernel<T, T, kThreads, kVectors><<<blocks, block_threads, 0, toStream(stream)>>>(args);
                } else {
                    residualNormKernel<T, float, kThreads, kVectors><<<blocks, block_threads, 0, toStream(stream)>>>(args);
                }
                ZCGVS_LAUNCH_CHECK("residual norm");
            }
            return static_cast<int>(ZCGVS_OK);
        });
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

std::size_t zcgvs_residual_norm_gradient_workspace_bytes(const zcgvs_norm_desc* desc) {
    if (checkNorm(desc) != ZCGVS_OK) {
        return 0;
    }
    clearError();
    return std::max<std::size_t>(256, static_cast<std::size_t>(gradientBlocks(*desc)) * desc->dim * sizeof(float));
}

int zcgvs_residual_norm_gradient(const zcgvs_norm_desc* desc, const void* d_out_gradient,
                                 std::int64_t out_gradient_stride, const void* d_sum_gradient,
                                 std::int64_t sum_gradient_stride, void* d_x_gradient, std::int64_t x_gradient_stride,
                                 void* d_weight_gradient, void* d_workspace, std::size_t workspace_bytes,
                                 zcgvs_stream_t stream) {
    const int status = checkNorm(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_norm_desc& d = *desc;
    if (rowStride(out_gradient_stride, d.dim) < d.dim || rowStride(sum_gradient_stride, d.dim) < d.dim ||
        rowStride(x_gradient_stride, d.dim) < d.dim) {
        return invalid("a gradient's row stride is smaller than dim");
    }
    if ((d_x_gradient == nullptr || d.rows == 0) && d_weight_gradient == nullptr) {
        return clearError();
    }
    if (d.rows > 0 && d_out_gradient == nullptr) {
        return invalid("null device pointer");
    }
    if (d_weight_gradient != nullptr && d.rows > 0) {
        if (d_workspace == nullptr || workspace_bytes < zcgvs_residual_norm_gradient_workspace_bytes(desc)) {
            return invalid("the workspace is too small");
        }
        if (!aligned16(d_workspace)) {
            return invalid("the workspace must be aligned to 16 bytes");
        }
    }
    NormGradientArgs more{};
    more.out_gradient = d_out_gradient;
    more.out_gradient_stride = rowStride(out_gradient_stride, d.dim);
    more.sum_gradient = d_sum_gradient;
    more.sum_gradient_stride = rowStride(sum_gradient_stride, d.dim);
    more.x_gradient = d_x_gradient;
    more.x_gradient_stride = rowStride(x_gradient_stride, d.dim);
    more.partials = d_weight_gradient == nullptr ? nullptr : static_cast<float*>(d_workspace);
    const int blocks = gradientBlocks(d);
    const int launched = withElement(d.dtype, [&](auto element) {
        using T = decltype(element);
        if (d.rows > 0) {
            const int formed = withRowShape<T>(d.dim, [&](auto threads, auto vectors) {
                residualNormGradientKernel<T, decltype(threads)::value, decltype(vectors)::value>
                    <<<static_cast<unsigned>(blocks), kNormThreads, 0, toStream(stream)>>>(normArgs(d), more);
                ZCGVS_LAUNCH_CHECK("residual norm gradient");
                return static_cast<int>(ZCGVS_OK);
            });
            if (formed != ZCGVS_OK) {
                return formed;
            }
        }
        if (d_weight_gradient != nullptr) {
            return launchJoinColumns<T>(more.partials, d.rows > 0 ? blocks : 0, d.dim, d_weight_gradient, toStream(stream));
        }
        return static_cast<int>(ZCGVS_OK);
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

}  // extern "C"
