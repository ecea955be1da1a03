// The linear projection with bias, activation and residual, and its gradient: checks, plans and the launches' order.
// The kernels are in linear_kernel.hpp, built for each operand type by a file of its own.
//
// dz is rounded to the operands' type where it is written, as a model of that type stores it: the products over it take
// 16-bit operands, their sums are float32. The bias's gradient is the sum of the unrounded dz, formed beside it.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "column_sums.hpp"
#include "common.hpp"
#include "elements.hpp"
#include "linear.hpp"
#include "matrix_plan.hpp"

namespace zcgvs_hip {

int linearInvalid(const char* message) {
    return setError(ZCGVS_ERR_INVALID_ARGUMENT, std::string("zcgvs linear projection: ") + message);
}

int linearWaveRows(const LinearPlan& plan, int dtype, std::int64_t rows) {
    switch (plan.product.shape) {
        case TileShape::k64x64:
            return 2 * divideUp(rows, 64);
        case TileShape::k128x128:
            return (dtype == ZCGVS_DTYPE_F32 ? 4 : 2) * divideUp(rows, 128);
        default:
            return 4 * divideUp(rows, 256);
    }
}

namespace {

// Column sums of a matrix [rows, columns]: workgroup (c, p) those of columns 32 c on and every kSumChunks-th stretch of
// rows, to partials [kSumChunks, columns].
constexpr int kSumColumns = 32;
constexpr int kSumChunks = 128;

template <typename T>
__global__ __launch_bounds__(kColumnThreads) void columnSumsKernel(const T* __restrict__ from, std::int64_t stride, int rows,
                                                                   int columns, float* __restrict__ partials) {
    constexpr int kLanes = kColumnThreads / kSumColumns;
    __shared__ float shared[kLanes][kSumColumns];
    const int column = static_cast<int>(threadIdx.x) % kSumColumns;
    const int part = static_cast<int>(threadIdx.x) / kSumColumns;
    const int c = static_cast<int>(blockIdx.x) * kSumColumns + column;
    float sum = 0.0f;
    if (c < columns) {
#pragma unroll 8
        for (int r = static_cast<int>(blockIdx.y) * kLanes + part; r < rows; r += kSumChunks * kLanes) {
            sum += static_cast<float>(from[r * stride + c]);
        }
    }
    shared[part][column] = sum;
    __syncthreads();
    if (part == 0 && c < columns) {
#pragma unroll
        for (int p = 1; p < kLanes; ++p) {
            sum += shared[p][column];
        }
        partials[static_cast<std::int64_t>(blockIdx.y) * columns + c] = sum;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void clearRowsKernel(T* out, std::int64_t stride, int rows, int columns) {
    for (int r = static_cast<int>(blockIdx.x); r < rows; r += static_cast<int>(gridDim.x)) {
        for (int c = static_cast<int>(threadIdx.x); c < columns; c += 256) {
            out[r * stride + c] = static_cast<T>(0.0f);
        }
    }
}

int checkLinear(const zcgvs_linear_desc* desc) {
    if (desc == nullptr) {
        return linearInvalid("null descriptor");
    }
    const zcgvs_linear_desc& d = *desc;
    const bool codes = d.dtype == ZCGVS_DTYPE_I8;
    if (!codes && !validElement(d.dtype)) {
        return linearInvalid("the operands must hold float32, float16, bfloat16 or int8");
    }
    if (codes ? !validElement(d.epilogue_dtype) : d.epilogue_dtype != d.dtype) {
        return linearInvalid("bias and residual must hold the operands' type, or with int8 operands a float type");
    }
    if (d.activation < ZCGVS_ACT_SILU || d.activation > ZCGVS_ACT_NONE) {
        return linearInvalid("unknown activation");
    }
    if (d.dim <= 0 || d.out_dim <= 0) {
        return linearInvalid("dim and out_dim must be positive");
    }
    if (d.dim > (1 << 24) || d.out_dim > (1 << 24)) {
        return linearInvalid("dim and out_dim must be at most 2^24");
    }
    if (codes && d.dim > kMaxCodes) {
        return linearInvalid("int8 rows hold at most 131072 codes");
    }
    if (d.rows < 0 || d.rows > (1 << 30)) {
        return linearInvalid("rows must lie in [0, 2^30]");
    }
    if (rowStride(d.x_stride, d.dim) < d.dim || rowStride(d.weight_stride, d.dim) < d.dim) {
        return linearInvalid("a row stride is smaller than dim");
    }
    if (d.residual != nullptr && rowStride(d.residual_stride, d.out_dim) < d.out_dim) {
        return linearInvalid("the residual's row stride is smaller than out_dim");
    }
    if (d.rows > 0 && (d.x == nullptr || d.weight == nullptr)) {
        return linearInvalid("null device pointer");
    }
    if (d.rows > 0 && codes && (d.x_scales == nullptr || d.weight_scales == nullptr)) {
        return linearInvalid("int8 operands need the scales of both");
    }
    return ZCGVS_OK;
}

bool directOperands(const zcgvs_linear_desc& d) {
    return directRows(d.x, rowStride(d.x_stride, d.dim), d.dim, d.dtype) &&
           directRows(d.weight, rowStride(d.weight_stride, d.dim), d.dim, d.dtype);
}

// The time of the kernel for few rows: each of its workgroups takes 16 columns and 16 or 32 rows, and stage after stage of
// 1024 bytes of k. A stage costs a CU c us for each of its workgroups, and the call 4 us. Measured, 16-bit 4096 -> 1024:
// 64 rows 9.9 us (32 at a time 13.3, 64 x 64 tiles 32.7), 128 rows 17.4 (13.5, 32.8), 512 rows 58 (44, 33.2); 1024 -> 4096:
// 64 rows 9.4 (7.9, 8.6), 256 rows 33 (26, 11.2); float32 4096 -> 1024, 64 rows 17.7 (24.1, 94), int8 8.8 (11.1, 15.3).
double thinTime(const zcgvs_linear_desc& d, int row_blocks) {
    const int values = kThinStageBytes / elementBytes(d.dtype);
    const double each = d.dtype == ZCGVS_DTYPE_I8 ? (row_blocks == 1 ? 1.5 : 2.4) : (row_blocks == 1 ? 0.9 : 1.35);
    const double groups = static_cast<double>(divideUp(d.out_dim, 16)) * divideUp(d.rows, 16 * row_blocks);
    return 4.0 + divideUp(d.dim, values) * std::max(1.0, groups / deviceComputeUnits()) * each;
}

LinearPlan planLinear(const zcgvs_linear_desc& d, bool direct, bool gradient) {
    // What the results need beside the sums of 256 x 256 does not fit the registers of the forward kernel (8192 rows
    // 1024 -> 4096 bfloat16 95 us, 87 with 256 x 192; int8 149 and 63), nor the error function's terms those of dz
    // (16,384 rows 768 -> 2048, GELU by tanh: 228 us, 236 with 256 x 192).
    const LargestTile largest = !gradient || d.activation == ZCGVS_ACT_GELU ? LargestTile::k256x192 : LargestTile::k256x256;
    // int8 stages hold twice the values and take the time of 16-bit ones
    const bool codes = d.dtype == ZCGVS_DTYPE_I8;
    const ProductPlan product = planProduct(d.rows, d.out_dim, codes ? (d.dim + 1) / 2 : d.dim, 1,
                                            codes ? static_cast<int>(ZCGVS_DTYPE_F16) : d.dtype, 0, largestTile(largest, direct));
    int thin = 0;
    if (!gradient && d.rows <= kThinMostRows) {
        const int row_blocks = thinTime(d, 1) <= thinTime(d, 2) ? 1 : 2;
        thin = thinTime(d, row_blocks) < product.us ? row_blocks : 0;
    }
    return {product, thin, direct};
}

LinearArgs linearArgs(const zcgvs_linear_desc& d) {
    LinearArgs args{};
    args.x = d.x;
    args.x_stride = rowStride(d.x_stride, d.dim);
    args.weight = d.weight;
    args.weight_stride = rowStride(d.weight_stride, d.dim);
    args.rows = static_cast<int>(d.rows);
    args.dim = d.dim;
    args.out_dim = d.out_dim;
    args.epilogue_dtype = d.epilogue_dtype;
    args.x_scales = d.x_scales;
    args.weight_scales = d.weight_scales;
    args.bias = d.bias;
    return args;
}

// ---- the gradient's workspace: dz, the bias's partial sums, the products' --------------------------

std::int64_t slopeStride(const zcgvs_linear_desc& d) { return (static_cast<std::int64_t>(d.out_dim) + 7) / 8 * 8; }

std::size_t roundUp256(std::size_t bytes) { return (bytes + 255) / 256 * 256; }

std::size_t slopeBytes(const zcgvs_linear_desc& d) {
    return d.activation == ZCGVS_ACT_NONE ? 0
                                          : roundUp256(static_cast<std::size_t>(d.rows) * static_cast<std::size_t>(slopeStride(d)) *
                                                       static_cast<std::size_t>(elementBytes(d.dtype)));
}

// A wavefront of the dz launch takes 32 rows of a tile or more.
std::size_t biasBytes(const zcgvs_linear_desc& d) {
    const std::size_t rows = d.activation == ZCGVS_ACT_NONE ? kSumChunks : static_cast<std::size_t>(divideUp(d.rows, 256)) * 8;
    return roundUp256(rows * static_cast<std::size_t>(d.out_dim) * sizeof(float));
}

ProductPlan inputPlan(const zcgvs_linear_desc& d, bool direct) {
    return planProduct(d.rows, d.dim, d.out_dim, 1, d.dtype, 1, largestTile(LargestTile::k256x256, direct));
}

ProductPlan weightPlan(const zcgvs_linear_desc& d, bool direct) {
    return planProduct(d.out_dim, d.dim, d.rows, 1, d.dtype, 1, largestTile(LargestTile::k256x256, direct));
}

// For either kind of rows, so that a call's workspace goes by the sizes and the type alone.
std::size_t partialBytes(int splits, std::int64_t m, std::int64_t n) {
    return splits > 1 ? roundUp256(static_cast<std::size_t>(splits) * static_cast<std::size_t>(m) * static_cast<std::size_t>(n) *
                                   sizeof(float))
                      : 0;
}

std::size_t inputPartialBytes(const zcgvs_linear_desc& d) {
    return partialBytes(std::max(inputPlan(d, false).splits, inputPlan(d, true).splits), d.rows, d.dim);
}

std::size_t weightPartialBytes(const zcgvs_linear_desc& d) {
    return partialBytes(std::max(weightPlan(d, false).splits, weightPlan(d, true).splits), d.out_dim, d.dim);
}

// Whole stages for each split, which may leave fewer than planned.
void splitProduct(const ProductPlan& plan, ProductArgs& args) {
    args.split_k = args.k;
    args.splits = 1;
    if (plan.splits > 1) {
        args.split_k = divideUp(divideUp(args.k, plan.splits), kPlanStageK) * kPlanStageK;
        args.splits = divideUp(args.k, args.split_k);
    }
}

template <typename T>
int clearRows(void* out, std::int64_t stride, int rows, int columns, hipStream_t stream) {
    clearRowsKernel<T><<<static_cast<unsigned>(std::min(rows, 4096)), 256, 0, stream>>>(static_cast<T*>(out), stride, rows, columns);
    ZCGVS_LAUNCH_CHECK("linear gradient");
    return ZCGVS_OK;
}

template <typename T>
int formGradients(const zcgvs_linear_desc& d, const void* out_gradient, std::int64_t out_gradient_stride, ProductArgs input,
                  ProductArgs weight, void* bias_gradient, char* workspace, hipStream_t stream) {
    float* bias_partials = reinterpret_cast<float*>(workspace + slopeBytes(d));
    const void* dz = out_gradient;
    std::int64_t dz_stride = out_gradient_stride;
    int dz_columns = d.out_dim;
    int bias_rows = kSumChunks;
    int status = ZCGVS_OK;
    if (d.activation != ZCGVS_ACT_NONE) {
        const LinearPlan plan = planLinear(d, directOperands(d), true);
        LinearArgs form = linearArgs(d);
        form.out = workspace;
        form.out_stride = slopeStride(d);
        form.out_gradient = out_gradient;
        form.out_gradient_stride = out_gradient_stride;
        form.bias_partials = bias_gradient == nullptr ? nullptr : bias_partials;
        status = launchLinearSlope<T>(plan, d.activation, form, stream);
        bias_rows = linearWaveRows(plan, d.dtype, d.rows);
        dz = workspace;
        dz_stride = form.out_stride;
        dz_columns = static_cast<int>(dz_stride);
    } else if (bias_gradient != nullptr) {
        columnSumsKernel<T><<<dim3(static_cast<unsigned>(divideUp(d.out_dim, kSumColumns)), kSumChunks), kColumnThreads, 0,
                              stream>>>(static_cast<const T*>(dz), dz_stride, static_cast<int>(d.rows), d.out_dim, bias_partials);
        ZCGVS_LAUNCH_CHECK("linear gradient");
    }
    if (status != ZCGVS_OK) {
        return status;
    }
    const bool direct_dz = directRows(dz, dz_stride, dz_columns, d.dtype);
    const bool direct_input = direct_dz && directRows(input.b, input.b_stride, d.dim, d.dtype);
    const bool direct_weight = direct_dz && directRows(weight.b, weight.b_stride, d.dim, d.dtype);
    const ProductPlan input_plan = inputPlan(d, direct_input);
    const ProductPlan weight_plan = weightPlan(d, direct_weight);
    input.a = weight.a = dz;
    input.a_stride = weight.a_stride = dz_stride;
    input.a_columns = weight.a_columns = dz_columns;
    splitProduct(input_plan, input);
    splitProduct(weight_plan, weight);
    const ColumnJoin bias{bias_partials, bias_rows, d.out_dim, bias_gradient};
    return launchLinearProducts<T>(input_plan, direct_input, input, weight_plan, direct_weight, weight, bias, stream);
}

}  // namespace

}  // namespace zcgvs_hip

using namespace zcgvs_hip;

extern "C" {

int zcgvs_linear(const zcgvs_linear_desc* desc, void* d_out, std::int64_t out_stride, int out_dtype, zcgvs_stream_t stream) {
    const int status = checkLinear(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_linear_desc& d = *desc;
    if (out_dtype != d.epilogue_dtype && out_dtype != ZCGVS_DTYPE_F32) {
        return linearInvalid("the output must hold the bias's type or float32");
    }
    if (rowStride(out_stride, d.out_dim) < d.out_dim) {
        return linearInvalid("the output's row stride is smaller than out_dim");
    }
    if (d.rows == 0) {
        return clearError();
    }
    if (d_out == nullptr) {
        return linearInvalid("null device pointer");
    }
    LinearArgs args = linearArgs(d);
    args.out_dtype = out_dtype;
    args.residual = d.residual;
    args.residual_stride = rowStride(d.residual_stride, d.out_dim);
    args.out = d_out;
    args.out_stride = rowStride(out_stride, d.out_dim);
    const LinearPlan plan = planLinear(d, directOperands(d), false);
    const int launched =
        d.dtype == ZCGVS_DTYPE_I8 ? launchLinear<std::int8_t>(plan, d.activation, args, toStream(stream))
                                  : withElement(d.dtype, [&](auto element) {
                                        return launchLinear<decltype(element)>(plan, d.activation, args, toStream(stream));
                                    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

std::size_t zcgvs_linear_gradient_workspace_bytes(const zcgvs_linear_desc* desc) {
    if (checkLinear(desc) != ZCGVS_OK) {
        return 0;
    }
    if (desc->dtype == ZCGVS_DTYPE_I8) {
        linearInvalid("the gradient takes float operands");
        return 0;
    }
    clearError();
    const zcgvs_linear_desc& d = *desc;
    return d.rows == 0 ? 256 : slopeBytes(d) + biasBytes(d) + inputPartialBytes(d) + weightPartialBytes(d);
}

int zcgvs_linear_gradient(const zcgvs_linear_desc* desc, const void* d_out_gradient, std::int64_t out_gradient_stride,
                          void* d_x_gradient, std::int64_t x_gradient_stride, void* d_weight_gradient,
                          std::int64_t weight_gradient_stride, void* d_bias_gradient, void* d_workspace,
                          std::size_t workspace_bytes, zcgvs_stream_t stream) {
    const int status = checkLinear(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_linear_desc& d = *desc;
    if (d.dtype == ZCGVS_DTYPE_I8) {
        return linearInvalid("the gradient takes float operands");
    }
    const std::int64_t from_stride = rowStride(out_gradient_stride, d.out_dim);
    const std::int64_t x_out_stride = rowStride(x_gradient_stride, d.dim);
    const std::int64_t weight_out_stride = rowStride(weight_gradient_stride, d.dim);
    if (from_stride < d.out_dim || x_out_stride < d.dim || weight_out_stride < d.dim) {
        return linearInvalid("a gradient's row stride is smaller than its row");
    }
    if (d_x_gradient == nullptr && d_weight_gradient == nullptr && d_bias_gradient == nullptr) {
        return clearError();
    }
    if (d.rows == 0) {
        const int cleared = withElement(d.dtype, [&](auto element) {
            using T = decltype(element);
            int done = ZCGVS_OK;
            if (d_weight_gradient != nullptr) {
                done = clearRows<T>(d_weight_gradient, weight_out_stride, d.out_dim, d.dim, toStream(stream));
            }
            if (done == ZCGVS_OK && d_bias_gradient != nullptr) {
                done = clearRows<T>(d_bias_gradient, d.out_dim, 1, d.out_dim, toStream(stream));
            }
            return done;
        });
        return cleared == ZCGVS_OK ? clearError() : cleared;
    }
    if (d_out_gradient == nullptr) {
        return linearInvalid("null device pointer");
    }
    if (d_workspace == nullptr || workspace_bytes < zcgvs_linear_gradient_workspace_bytes(desc)) {
        return linearInvalid("the workspace is too small");
    }
    if (!aligned16(d_workspace)) {
        return linearInvalid("the workspace must be aligned to 16 bytes");
    }
    char* workspace = static_cast<char*>(d_workspace);
    float* partials = reinterpret_cast<float*>(workspace + slopeBytes(d) + biasBytes(d));
    ProductArgs input{};
    input.b = d.weight;
    input.b_stride = rowStride(d.weight_stride, d.dim);
    input.m = static_cast<int>(d.rows);
    input.n = d.dim;
    input.k = d.out_dim;
    input.partials = partials;
    input.out = d_x_gradient;
    input.out_stride = x_out_stride;
    ProductArgs weight{};
    weight.b = d.x;
    weight.b_stride = rowStride(d.x_stride, d.dim);
    weight.m = d.out_dim;
    weight.n = d.dim;
    weight.k = static_cast<int>(d.rows);
    weight.partials = reinterpret_cast<float*>(reinterpret_cast<char*>(partials) + inputPartialBytes(d));
    weight.out = d_weight_gradient;
    weight.out_stride = weight_out_stride;
    const int launched = withElement(d.dtype, [&](auto element) {
        return formGradients<decltype(element)>(d, d_out_gradient, from_stride, input, weight, d_bias_gradient, workspace,
                                                toStream(stream));
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

}  // extern "C"
