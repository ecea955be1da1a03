// What the linear projection's translation units share: the launches that linear.hip chooses between, built for
// each operand type by linear_f32.hip, linear_f16.hip, linear_bf16.hip and linear_i8.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "matrix_plan.hpp"

namespace zcgvs_hip {

struct LinearArgs {
    const void* x;
    std::int64_t x_stride;
    const void* weight;
    std::int64_t weight_stride;
    int rows;
    int dim;
    int out_dim;
    int tiles_m;
    int tiles_n;
    int epilogue_dtype;  // of bias and residual (int8 operands; otherwise the operands')
    int out_dtype;       // epilogue_dtype or float32
    const float* x_scales;
    const float* weight_scales;
    const void* bias;
    const void* residual;
    std::int64_t residual_stride;
    void* out;
    std::int64_t out_stride;
    // gradient only: `out` is dz of the operands' type, its columns past out_dim written as zeros, and
    // `bias_partials` (or null) takes float32 sums of dz over each wavefront's rows
    const void* out_gradient;
    std::int64_t out_gradient_stride;
    float* bias_partials;  // [rows of wavefronts, out_dim]
};

// out [m, n] = sum over k of a and b, each side plain or turned (matrix_tile.hpp); splits over k write their sums to
// `partials` [splits, m, n].
struct ProductArgs {
    const void* a;
    std::int64_t a_stride;
    const void* b;
    std::int64_t b_stride;
    int m;
    int n;
    int k;
    int a_columns;  // of a turned side a that can be read
    int tiles_m;
    int tiles_n;
    int splits;
    int split_k;
    float* partials;
    void* out;
    std::int64_t out_stride;
};

constexpr int kMaxCodes = 131072;  // of an int8 row: products of -128 add up to 2^31 (exactSum)
constexpr int kThinStageBytes = 1024;  // of k that a workgroup of the kernel for few rows takes at a time
constexpr int kThinMostRows = 4096;

// The bias's gradient: out [columns] = the sums over `rows` rows of partials, by a launch's last blocks (out null: none).
struct ColumnJoin {
    const float* partials;
    int rows;
    int columns;
    void* out;
};

// How linear.hip runs a call.
struct LinearPlan {
    ProductPlan product;
    int thin;     // few rows: blocks of 16 of them that a workgroup takes, its wavefronts splitting k; 0: tiles
    bool direct;  // rows of whole aligned chunks
};

// Rows of wavefronts of the dz launch under a plan, and so rows of bias_partials.
int linearWaveRows(const LinearPlan& plan, int dtype, std::int64_t rows);

template <typename T>
int launchLinear(const LinearPlan& plan, int activation, LinearArgs args, hipStream_t stream);
template <typename T>
int launchLinearSlope(const LinearPlan& plan, int activation, LinearArgs args, hipStream_t stream);
// dx = dz weight, dW = dz^T x and what is left of the bias's gradient; a null `out` is not wanted.
template <typename T>
int launchLinearProducts(ProductPlan input_plan, bool input_direct, ProductArgs input, ProductPlan weight_plan,
                         bool weight_direct, ProductArgs weight, ColumnJoin bias, hipStream_t stream);

int linearInvalid(const char* message);

}  // namespace zcgvs_hip
