// Element types of the embedding-model operators (float32, float16, bfloat16) and their checks.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "common.hpp"

namespace zcgvs_hip {

inline bool validElement(int dtype) {
    return dtype == ZCGVS_DTYPE_F32 || dtype == ZCGVS_DTYPE_F16 || dtype == ZCGVS_DTYPE_BF16;
}

__host__ __device__ constexpr int elementBytes(int dtype) { return dtype == ZCGVS_DTYPE_F32 ? 4 : 2; }

// Calls body(T{}) with the C++ type of a valid element dtype.
template <typename Body>
int withElement(int dtype, Body&& body) {
    switch (dtype) {
        case ZCGVS_DTYPE_F16:
            return body(_Float16{});
        case ZCGVS_DTYPE_BF16:
            return body(__bf16{});
        default:
            return body(float{});
    }
}

// Whether rows that start at `base`, `stride` elements apart, can be read `bytes` at a time.
inline bool alignedRows(const void* base, std::int64_t stride, int dtype, int bytes) {
    return reinterpret_cast<std::uintptr_t>(base) % static_cast<std::uintptr_t>(bytes) == 0 &&
           stride * elementBytes(dtype) % bytes == 0;
}

// kCount neighbouring elements as one load or store. `stored` may stand at any element: the hardware takes
// vector accesses at any alignment.
template <typename T, int kCount>
struct Pack {
    typedef T type __attribute__((ext_vector_type(kCount)));
    typedef T stored __attribute__((ext_vector_type(kCount), aligned(sizeof(T))));
};
template <typename T>
struct Pack<T, 1> {
    typedef T type;
    typedef T stored;
};

// The first column of a row's pack `pack`: the last pack of a row that is no whole number of them begins
// early and overlaps the one before.
template <int kCount>
__host__ __device__ __forceinline__ int packColumn(int pack, int columns) {
    const int column = pack * kCount;
    return column < columns - kCount ? column : columns - kCount;
}

template <typename T, int kCount>
__device__ __forceinline__ void loadPack(const T* from, float (&to)[kCount]) {
    if constexpr (kCount == 1) {
        to[0] = static_cast<float>(*from);
    } else {
        const auto v = *reinterpret_cast<const typename Pack<T, kCount>::stored*>(from);
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            to[e] = static_cast<float>(v[e]);
        }
    }
}

// sum += weight * the values of a pack as it was loaded.
template <int kCount, typename V>
__device__ __forceinline__ void addPack(const V& v, float weight, float (&sum)[kCount]) {
    if constexpr (kCount == 1) {
        sum[0] += weight * static_cast<float>(v);
    } else {
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            sum[e] += weight * static_cast<float>(v[e]);
        }
    }
}

// Rounds to nearest even where T is narrower than float32.
template <typename T, int kCount>
__device__ __forceinline__ void storePack(const float (&from)[kCount], T* to) {
    if constexpr (kCount == 1) {
        *to = static_cast<T>(from[0]);
    } else {
        typename Pack<T, kCount>::type v;
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            v[e] = static_cast<T>(from[e]);
        }
        *reinterpret_cast<typename Pack<T, kCount>::stored*>(to) = v;
    }
}

// The same with the hint that nobody reads it soon.
template <typename T, int kCount>
__device__ __forceinline__ void storePackOnce(const float (&from)[kCount], T* to) {
    typename Pack<T, kCount>::stored v;
    if constexpr (kCount == 1) {
        v = static_cast<T>(from[0]);
    } else {
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            v[e] = static_cast<T>(from[e]);
        }
    }
    __builtin_nontemporal_store(v, reinterpret_cast<typename Pack<T, kCount>::stored*>(to));
}

}  // namespace zcgvs_hip
