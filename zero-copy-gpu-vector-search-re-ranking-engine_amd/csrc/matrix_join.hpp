// The sum of the float32 partial products that the splits of a product over k have written.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "common.hpp"
#include "elements.hpp"

namespace zcgvs_hip {
namespace {

// out = the sum of the splits' partials [splits, rows, columns]; rows from `rows_first` on go to `second`.
constexpr int kJoinThreads = 256;

template <typename T, int kPack>
__global__ __launch_bounds__(kJoinThreads) void joinKernel(const float* __restrict__ partials, int splits,
                                                           long long rows, int columns, long long rows_first,
                                                           T* __restrict__ first, T* __restrict__ second,
                                                           std::int64_t stride) {
    const int packs_per_row = (columns + kPack - 1) / kPack;
    const long long packs = rows * packs_per_row;
    const long long split_values = rows * columns;
    for (long long p = static_cast<long long>(blockIdx.x) * kJoinThreads + threadIdx.x; p < packs;
         p += static_cast<long long>(gridDim.x) * kJoinThreads) {
        const long long row = p / packs_per_row;
        const int column = packColumn<kPack>(static_cast<int>(p - row * packs_per_row), columns);
        const float* from = partials + row * columns + column;
        float sum[kPack];
        loadPack(from, sum);
#pragma unroll 4
        for (int s = 1; s < splits; ++s) {
            float more[kPack];
            loadPack(from + s * split_values, more);
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                sum[e] += more[e];
            }
        }
        T* to = row < rows_first ? first + row * stride : second + (row - rows_first) * stride;
        storePack(sum, to + column);
    }
}

template <typename T>
int launchJoin(const float* partials, int splits, std::int64_t rows, int columns, std::int64_t rows_first, void* first,
               void* second, std::int64_t stride, hipStream_t stream) {
    const bool four = columns >= 4;
    const long long packs = static_cast<long long>(rows) * (four ? (columns + 3) / 4 : columns);
    const unsigned blocks = static_cast<unsigned>(std::min(8192ll, (packs + kJoinThreads - 1) / kJoinThreads));
    if (four) {
        joinKernel<T, 4><<<blocks, kJoinThreads, 0, stream>>>(partials, splits, rows, columns, rows_first,
                                                              static_cast<T*>(first), static_cast<T*>(second), stride);
    } else {
        joinKernel<T, 1><<<blocks, kJoinThreads, 0, stream>>>(partials, splits, rows, columns, rows_first,
                                                              static_cast<T*>(first), static_cast<T*>(second), stride);
    }
    ZCGVS_LAUNCH_CHECK("join of splits");
    return ZCGVS_OK;
}

}  // namespace
}  // namespace zcgvs_hip
