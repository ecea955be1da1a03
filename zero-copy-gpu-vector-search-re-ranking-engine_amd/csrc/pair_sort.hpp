// Stable sort of (key, row) pairs by small non-negative keys: token ids, adapter numbers.
//
// Least-significant-digit radix sort, at most kDigitBits bits a pass. The rank of an item among its
// wavefront's items of the same digit follows from ballots over the digit's bits, so equal keys keep
// their order and the result is the same on every run. Up to kSmallItems items one workgroup runs all
// passes in LDS (one launch); beyond, a pass is two launches: tiles count their digits, then place
// their items, each adding up the counts of the tiles before it by itself (there are at most kMaxTiles).
// What bounds it is latency, not the 16 bytes a pair and pass.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "common.hpp"

namespace zcgvs_hip {
namespace {

constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortItems = kSortThreads;  // an item a thread
constexpr int kMaxTiles = 128;
constexpr int kSmallThreads = 1024;
constexpr int kSmallWaves = kSmallThreads / kWave;
constexpr int kSmallItems = 8192;
constexpr int kSmallRounds = kSmallItems / kSmallThreads;

// Keys in [0, key_end) count; a raw key outside, or equal to `skipped`, becomes key_end (the largest).
struct SortInput {
    const int* keys;
    const int* rows;  // null: the position itself
    int count;
    int key_end;
    int skipped;
    bool raw;  // keys are not yet checked
};

__device__ __forceinline__ bool counts(int id, int end, int skipped) { return id >= 0 && id < end && id != skipped; }

__device__ __forceinline__ int checkedKey(const SortInput& in, int key) {
    return !in.raw || counts(key, in.key_end, in.skipped) ? key : in.key_end;
}

__device__ __forceinline__ int sortKey(const SortInput& in, int i) { return checkedKey(in, in.keys[i]); }

// Orders a wavefront's LDS accesses before and after it.
__device__ __forceinline__ void waveFence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Exclusive prefix sum over the block's threads; every thread of the block calls it.
__device__ __forceinline__ unsigned blockPrefix(unsigned value, unsigned* wave_sums) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    unsigned prefix = value;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const unsigned below = __shfl_up(prefix, d, kWave);
        prefix += lane >= d ? below : 0u;
    }
    if (lane == kWave - 1) {
        wave_sums[wave] = prefix;
    }
    __syncthreads();
    unsigned base = 0;
    for (int w = 0; w < wave; ++w) {
        base += wave_sums[w];
    }
    __syncthreads();
    return base + prefix - value;
}

// The rank of this lane's item behind its wavefront's earlier items of the same digit, which `seen`
// (the wavefront's own, in LDS) counts. Every lane of the wavefront calls it.
__device__ __forceinline__ unsigned digitRank(unsigned digit, int bits, bool ok, unsigned* seen) {
    const int lane = threadIdx.x & (kWave - 1);
    unsigned long long same = __ballot(ok);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((digit >> b) & 1u);
        same &= ((digit >> b) & 1u) ? set : ~set;
    }
    unsigned before = 0;
    if (ok) {
        before = seen[digit];
    }
    waveFence();
    const int below = __popcll(same & ((1ull << lane) - 1ull));
    if (ok && below == 0) {
        seen[digit] = before + static_cast<unsigned>(__popcll(same));
    }
    waveFence();
    return before + static_cast<unsigned>(below);
}

// What a sort's launches do beside it: sorting waits on latency and leaves the memory idle. Blocks past the
// sort's own call run(block, blocks) with what is theirs of launch `launch` out of `launches`.
struct NoSideWork {
    static constexpr int kBlocks = 0;
    __device__ void run(int, int, int, int) const {}
};

// ---- one workgroup ------------------------------------------------------------------------------

template <class Side>
__global__ __launch_bounds__(kSmallThreads) void sortSmallKernel(SortInput in, int bits, int passes,
                                                                 int* __restrict__ keys_out,
                                                                 int* __restrict__ rows_out, Side side) {
    if (blockIdx.x > 0) {
        side.run(static_cast<int>(blockIdx.x) - 1, static_cast<int>(gridDim.x) - 1, 0, 1);
        return;
    }
    __shared__ int keys[2][kSmallItems];
    __shared__ std::uint16_t places[2][kSmallItems];
    __shared__ unsigned seen[kSmallWaves][kDigits];
    __shared__ unsigned wave_sums[kSmallWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    // a wavefront owns `rounds` * 64 consecutive items
    const int rounds = (in.count + kSmallThreads - 1) / kSmallThreads;
    const int per_pass = (bits + passes - 1) / passes;
    for (int p = 0; p < passes; ++p) {
        const int shift = p * per_pass;
        const int here = min(per_pass, bits - shift);
        const int digits = 1 << here;
        const unsigned mask = static_cast<unsigned>(digits) - 1u;
        int key[kSmallRounds];
        unsigned rank[kSmallRounds];
        // all loads before the first use: one latency, not one a round
        if (p == 0) {
#pragma unroll
            for (int round = 0; round < kSmallRounds; ++round) {
                key[round] = in.keys[min((wave * rounds + round) * kWave + lane, in.count - 1)];
            }
#pragma unroll
            for (int round = 0; round < kSmallRounds; ++round) {
                key[round] = checkedKey(in, key[round]);
            }
        } else {
#pragma unroll
            for (int round = 0; round < kSmallRounds; ++round) {
                key[round] = keys[p & 1][min((wave * rounds + round) * kWave + lane, in.count - 1)];
            }
        }
        for (int d = lane; d < digits; d += kWave) {
            seen[wave][d] = 0;
        }
        waveFence();
#pragma unroll
        for (int round = 0; round < kSmallRounds; ++round) {
            if (round < rounds) {
                const bool ok = (wave * rounds + round) * kWave + lane < in.count;
                rank[round] = digitRank((static_cast<unsigned>(key[round]) >> shift) & mask, here, ok, seen[wave]);
            }
        }
        __syncthreads();
        unsigned total = 0;
        if (static_cast<int>(threadIdx.x) < digits) {
#pragma unroll
            for (int w = 0; w < kSmallWaves; ++w) {
                total += seen[w][threadIdx.x];
            }
        }
        unsigned at = blockPrefix(total, wave_sums);
        if (static_cast<int>(threadIdx.x) < digits) {
#pragma unroll
            for (int w = 0; w < kSmallWaves; ++w) {
                const unsigned count = seen[w][threadIdx.x];
                seen[w][threadIdx.x] = at;
                at += count;
            }
        }
        __syncthreads();
#pragma unroll
        for (int round = 0; round < kSmallRounds; ++round) {
            const int i = (wave * rounds + round) * kWave + lane;
            if (round < rounds && i < in.count) {
                const unsigned digit = (static_cast<unsigned>(key[round]) >> shift) & mask;
                const unsigned to = seen[wave][digit] + rank[round];
                const int place = p == 0 ? i : places[p & 1][i];
                if (p + 1 < passes) {
                    keys[(p & 1) ^ 1][to] = key[round];
                    places[(p & 1) ^ 1][to] = static_cast<std::uint16_t>(place);
                } else {
                    keys_out[to] = key[round];
                    rows_out[to] = in.rows == nullptr ? place : in.rows[place];
                }
            }
        }
        __syncthreads();
    }
}

// ---- many workgroups ----------------------------------------------------------------------------

// A tile is a run of items that one workgroup counts and then places, kSortItems at a time.
struct SortPass {
    SortInput in;
    int* keys_out;
    int* rows_out;
    unsigned* tile_counts;  // [tiles, kDigits]
    int tile_items;         // a multiple of kSortItems
    int tiles;
    int shift;
    int bits;
    int launch;    // of this pass's count; its placement is the next one
    int launches;
};

template <class Side>
__global__ __launch_bounds__(kSortThreads) void sortCountKernel(SortPass pass, Side side) {
    __shared__ unsigned histogram[kDigits];
    if (static_cast<int>(blockIdx.x) >= pass.tiles) {
        side.run(static_cast<int>(blockIdx.x) - pass.tiles, static_cast<int>(gridDim.x) - pass.tiles, pass.launch,
                 pass.launches);
        return;
    }
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) {
        histogram[d] = 0;
    }
    __syncthreads();
    const int begin = static_cast<int>(blockIdx.x) * pass.tile_items;
    const int end = min(begin + pass.tile_items, pass.in.count);
    const unsigned mask = (1u << pass.bits) - 1u;
    for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += kSortThreads) {
        atomicAdd(&histogram[(static_cast<unsigned>(sortKey(pass.in, i)) >> pass.shift) & mask], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) {
        pass.tile_counts[static_cast<std::size_t>(blockIdx.x) * kDigits + d] = histogram[d];
    }
}

template <class Side>
__global__ __launch_bounds__(kSortThreads) void sortPlaceKernel(SortPass pass, Side side) {
    __shared__ unsigned start[kDigits];
    __shared__ unsigned seen[kSortWaves][kDigits];
    __shared__ unsigned wave_sums[kSortWaves];
    if (static_cast<int>(blockIdx.x) >= pass.tiles) {
        side.run(static_cast<int>(blockIdx.x) - pass.tiles, static_cast<int>(gridDim.x) - pass.tiles, pass.launch + 1,
                 pass.launches);
        return;
    }
    const int wave = threadIdx.x / kWave;
    // digits of smaller value in all tiles, then the same digit in the tiles before this one: thread t adds
    // up digits 2 t' and 2 t' + 1 (t' = t % 256) over every fourth tile
    constexpr int kGroups = kSortThreads / (kDigits / 2);
    static_assert(kGroups * 2 * kDigits <= kSortWaves * kDigits, "the groups' sums fit where `seen` stands");
    const int pair = static_cast<int>(threadIdx.x) % (kDigits / 2);
    const int group = static_cast<int>(threadIdx.x) / (kDigits / 2);
    unsigned total[2] = {0, 0}, before[2] = {0, 0};
    const uint2* counts_of = reinterpret_cast<const uint2*>(pass.tile_counts) + pair;
#pragma unroll 8
    for (int t = group; t < pass.tiles; t += kGroups) {
        const uint2 c = counts_of[static_cast<std::size_t>(t) * (kDigits / 2)];
        total[0] += c.x;
        total[1] += c.y;
        if (t < static_cast<int>(blockIdx.x)) {
            before[0] += c.x;
            before[1] += c.y;
        }
    }
    unsigned* sums = &seen[0][0];  // [groups][2][digits]
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        sums[(group * 2 + 0) * kDigits + 2 * pair + e] = total[e];
        sums[(group * 2 + 1) * kDigits + 2 * pair + e] = before[e];
    }
    __syncthreads();
    unsigned all = 0, earlier = 0;
    if (threadIdx.x < kDigits) {
        for (int g = 0; g < kGroups; ++g) {
            all += sums[(g * 2 + 0) * kDigits + threadIdx.x];
            earlier += sums[(g * 2 + 1) * kDigits + threadIdx.x];
        }
    }
    const unsigned base = blockPrefix(all, wave_sums);
    if (threadIdx.x < kDigits) {
        start[threadIdx.x] = base + earlier;
    }
    const int begin = static_cast<int>(blockIdx.x) * pass.tile_items;
    const int end = min(begin + pass.tile_items, pass.in.count);
    const unsigned mask = (1u << pass.bits) - 1u;
    for (int first = begin; first < end; first += kSortItems) {
        __syncthreads();
        for (int d = threadIdx.x; d < kDigits * kSortWaves; d += kSortThreads) {
            (&seen[0][0])[d] = 0;
        }
        __syncthreads();
        const int i = first + static_cast<int>(threadIdx.x);
        const bool ok = i < end;
        const int key = ok ? sortKey(pass.in, i) : 0;
        const unsigned digit = (static_cast<unsigned>(key) >> pass.shift) & mask;
        const unsigned rank = digitRank(digit, pass.bits, ok, seen[wave]);
        __syncthreads();
        if (threadIdx.x < kDigits) {
            unsigned at = start[threadIdx.x];
            for (int w = 0; w < kSortWaves; ++w) {
                const unsigned here = seen[w][threadIdx.x];
                seen[w][threadIdx.x] = at;
                at += here;
            }
            start[threadIdx.x] = at;
        }
        __syncthreads();
        if (ok) {
            const unsigned at = seen[wave][digit] + rank;
            pass.keys_out[at] = key;
            pass.rows_out[at] = pass.in.rows == nullptr ? i : pass.in.rows[i];
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------

inline std::size_t sortAligned(std::size_t bytes) { return (bytes + 255) / 256 * 256; }

// Bytes of scratch for sorting `count` pairs; the sorted pairs stand in it too.
inline std::size_t pairSortBytes(std::size_t count) {
    return 4 * sortAligned(count * 4) + sortAligned(static_cast<std::size_t>(kMaxTiles) * kDigits * 4);
}

// Sorts count >= 1 pairs (at most 2^29); *keys and *rows are where they then stand, in `scratch`.
template <class Side>
int sortPairs(SortInput in, char* scratch, const int** keys, const int** rows, const Side& side, hipStream_t stream) {
    const std::size_t n = static_cast<std::size_t>(in.count);
    const std::size_t one = sortAligned(n * 4);
    int* key_buffer[2] = {reinterpret_cast<int*>(scratch), reinterpret_cast<int*>(scratch + one)};
    int* row_buffer[2] = {reinterpret_cast<int*>(scratch + 2 * one), reinterpret_cast<int*>(scratch + 3 * one)};
    int bits = 1;
    while ((static_cast<long long>(in.key_end) >> bits) != 0) {
        ++bits;
    }
    const int passes = (bits + kDigitBits - 1) / kDigitBits;
    if (in.count <= kSmallItems) {
        sortSmallKernel<Side><<<1 + Side::kBlocks, kSmallThreads, 0, stream>>>(in, bits, passes, key_buffer[0],
                                                                              row_buffer[0], side);
        ZCGVS_LAUNCH_CHECK("sort");
        *keys = key_buffer[0];
        *rows = row_buffer[0];
        return ZCGVS_OK;
    }
    SortPass pass{};
    pass.in = in;
    pass.tile_counts = reinterpret_cast<unsigned*>(scratch + 4 * one);
    const std::size_t tile = (n + kMaxTiles - 1) / kMaxTiles;
    pass.tile_items = static_cast<int>((tile + kSortItems - 1) / kSortItems) * kSortItems;
    pass.tiles = static_cast<int>((n + static_cast<std::size_t>(pass.tile_items) - 1) / static_cast<std::size_t>(pass.tile_items));
    const int per_pass = (bits + passes - 1) / passes;
    for (int p = 0; p < passes; ++p) {
        pass.shift = p * per_pass;
        pass.bits = std::min(per_pass, bits - pass.shift);
        pass.keys_out = key_buffer[p & 1];
        pass.rows_out = row_buffer[p & 1];
        pass.launch = 2 * p;
        pass.launches = 2 * passes;
        const unsigned blocks = static_cast<unsigned>(pass.tiles + Side::kBlocks);
        sortCountKernel<Side><<<blocks, kSortThreads, 0, stream>>>(pass, side);
        ZCGVS_LAUNCH_CHECK("sort");
        sortPlaceKernel<Side><<<blocks, kSortThreads, 0, stream>>>(pass, side);
        ZCGVS_LAUNCH_CHECK("sort");
        pass.in.keys = pass.keys_out;
        pass.in.rows = pass.rows_out;
        pass.in.raw = false;
    }
    *keys = pass.in.keys;
    *rows = pass.in.rows;
    return ZCGVS_OK;
}

}  // namespace
}  // namespace zcgvs_hip
