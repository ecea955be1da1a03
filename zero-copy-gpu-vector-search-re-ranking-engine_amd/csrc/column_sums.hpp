// Sums over the rows of a matrix, a value a column, in a fixed order.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace zcgvs_hip {
namespace {

constexpr int kColumnThreads = 256;

// out[c] = the sum over `count` rows of partials [count, dim], kJoinLanes threads a column in a fixed order.
constexpr int kJoinColumns = 16;
constexpr int kJoinLanes = kColumnThreads / kJoinColumns;

template <typename T>
__device__ __forceinline__ void joinColumns(const float* __restrict__ partials, int count, int dim, T* __restrict__ out,
                                            int block) {
    __shared__ float shared[kJoinLanes][kJoinColumns];
    const int column = static_cast<int>(threadIdx.x) % kJoinColumns;
    const int part = static_cast<int>(threadIdx.x) / kJoinColumns;
    const int c = block * kJoinColumns + column;
    float sum = 0.0f;
    if (c < dim) {
#pragma unroll 8
        for (int r = part; r < count; r += kJoinLanes) {
            sum += partials[static_cast<long long>(r) * dim + c];
        }
    }
    shared[part][column] = sum;
    __syncthreads();
    if (part == 0 && c < dim) {
#pragma unroll
        for (int p = 1; p < kJoinLanes; ++p) {
            sum += shared[p][column];
        }
        out[c] = static_cast<T>(sum);
    }
}

template <typename T>
__global__ __launch_bounds__(kColumnThreads) void joinColumnsKernel(const float* __restrict__ partials, int count, int dim,
                                                                    T* __restrict__ out) {
    joinColumns(partials, count, dim, out, static_cast<int>(blockIdx.x));
}

template <typename T>
int launchJoinColumns(const float* partials, int count, int dim, void* out, hipStream_t stream) {
    joinColumnsKernel<T><<<static_cast<unsigned>((dim + kJoinColumns - 1) / kJoinColumns), kColumnThreads, 0, stream>>>(
        partials, count, dim, static_cast<T*>(out));
    ZCGVS_LAUNCH_CHECK("column sums");
    return ZCGVS_OK;
}

}  // namespace
}  // namespace zcgvs_hip
