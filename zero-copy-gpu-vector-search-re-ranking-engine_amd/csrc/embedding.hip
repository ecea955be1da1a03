// Token-table lookup with scaling and pooling, and its gradient by sorted tokens.
//
// Lookup. out[r] = scale * w_r * sum of table[id] over the tokens of row r that count; w_r is 1, or
// 1 / (the number of those tokens) for the mean. Nothing is computed that a copy would not need, so
// the kernels are bound by memory: the rows of the tokens are read and the output is written. Measured: 1M
// Zipf-distributed tokens pooled into 16,384 rows of 384 floats 109-114 us, 1.5 GB of rows at 13-14 TB/s out of the
// caches (67% hits in the L2s; the 46 MB table does not fit one XCD's).
//
// Gradient. d_table[v] = scale * sum of w_r(j) * d_out[r(j)] over the tokens j with id v. A scatter
// with atomics would add in an order that changes from run to run and queue up on frequent tokens (the
// most frequent token of a text holds several percent of all positions); here the positions are sorted
// by id (a stable radix sort), runs of equal ids are summed in the order of the positions, in chunks
// of a fixed length, and the chunks' partial sums of a run that crosses chunks are joined in order (at
// most 512 tokens are searched instead of sorted).
// Rows of the table that no token names are zeros: all rows are cleared by blocks that the sort's launches
// leave idle. Measured for 262,144 tokens and 128,000 x 768 (bfloat16 in, float32 out): zeros and sort 83 us
// (393 MB at 4.7 TB/s), the sums 136 us (400 MB read and 136 MB written in single rows, 3.9 TB/s), the
// joins 15 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "elements.hpp"
#include "pair_sort.hpp"

namespace zcgvs_hip {

namespace {

constexpr int kThreads = 256;
constexpr int kWavesPerBlock = kThreads / kWave;
constexpr std::int64_t kMaxTokens = 1 << 28;          // a launch a chunk of 64 has less than 2^32 threads
constexpr long long kMaxBlocks = (1ll << 24) - 1;     // a launch has less than 2^32 threads
constexpr int kMaxDim = 1 << 23;                      // slices of 256 columns in a grid's second dimension

// ---- lookup, one output row per token ---------------------------------------------------------

// Output rows are cut into packs of kPack elements; a block writes kLookupPacks * 256 consecutive
// packs of the whole output, each thread kLookupPacks of them with their loads in flight together.
constexpr int kLookupPacks = 4;

template <typename In, typename Out, int kPack>
__global__ __launch_bounds__(kThreads) void lookupKernel(const In* __restrict__ table, std::int64_t table_stride,
                                                         int vocab, int dim, const int* __restrict__ ids,
                                                         long long packs, int padding_id, float scale,
                                                         Out* __restrict__ out, std::int64_t out_stride) {
    const int packs_per_row = (dim + kPack - 1) / kPack;
    const long long first = static_cast<long long>(blockIdx.x) * (kThreads * kLookupPacks);
    const long long first_row = first / packs_per_row;
    const unsigned first_pack = static_cast<unsigned>(first - first_row * packs_per_row);
    const int left = static_cast<int>(min(packs - first, static_cast<long long>(kThreads * kLookupPacks)));
    float value[kLookupPacks][kPack];
#pragma unroll
    for (int u = 0; u < kLookupPacks; ++u) {
        const int i = u * kThreads + static_cast<int>(threadIdx.x);
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            value[u][e] = 0.0f;
        }
        if (i < left) {
            const unsigned at = first_pack + static_cast<unsigned>(i);
            const unsigned row = at / static_cast<unsigned>(packs_per_row);
            const unsigned pack = at - row * static_cast<unsigned>(packs_per_row);
            const int id = ids[first_row + row];
            if (counts(id, vocab, padding_id)) {
                loadPack(table + id * table_stride + packColumn<kPack>(static_cast<int>(pack), dim), value[u]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kLookupPacks; ++u) {
        const int i = u * kThreads + static_cast<int>(threadIdx.x);
        if (i < left) {
            const unsigned at = first_pack + static_cast<unsigned>(i);
            const unsigned row = at / static_cast<unsigned>(packs_per_row);
            const unsigned pack = at - row * static_cast<unsigned>(packs_per_row);
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                value[u][e] *= scale;
            }
            storePack(value[u], out + (first_row + row) * out_stride + packColumn<kPack>(static_cast<int>(pack), dim));
        }
    }
}

// ---- lookup with bags -------------------------------------------------------------------------

// A wavefront pools a share of one bag's tokens over a slice of 64 packs. It reads 64 ids at a time, a lane
// each, and hands them on as scalars, so that the rows' loads wait for nothing but each other: kBagAhead of
// them are in flight. kShares wavefronts of a workgroup share a bag's tokens, every kShares-th one each, and
// their sums are joined through LDS in the order of the shares.
constexpr int kBagAhead = 16;

template <typename In, typename Out, int kPack, int kShares>
__global__ __launch_bounds__(kThreads) void bagKernel(const In* __restrict__ table, std::int64_t table_stride,
                                                      int vocab, int dim, const int* __restrict__ ids,
                                                      long long token_count,
                                                      const std::int64_t* __restrict__ bag_offsets, long long items,
                                                      int slices, bool mean, int padding_id, float scale,
                                                      Out* __restrict__ out, std::int64_t out_stride) {
    constexpr int kItems = kWavesPerBlock / kShares;  // of a workgroup
    __shared__ float sums[kShares > 1 ? kWavesPerBlock : 1][kWave * kPack];
    __shared__ int found[kWavesPerBlock];
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int share = wave % kShares;
    const long long item = static_cast<long long>(blockIdx.x) * kItems + wave / kShares;
    const bool has_item = item < items;
    const long long bag = has_item ? item / slices : 0;
    const int pack = static_cast<int>(item - bag * slices) * kWave + lane;
    const bool has_pack = has_item && pack < (dim + kPack - 1) / kPack;
    const int column = has_pack ? packColumn<kPack>(pack, dim) : 0;
    const long long begin = min(max(static_cast<long long>(bag_offsets[bag]), 0ll), token_count);
    const long long end = has_item ? min(static_cast<long long>(bag_offsets[bag + 1]), token_count) : begin;
    const In* from = table + column;

    float sum[kPack] = {};
    int count = 0;
    for (long long j = begin + share; j < end; j += kWave * kShares) {
        // 64 of this share's tokens, those that count first and in their order
        const long long mine = j + static_cast<long long>(lane) * kShares;
        const int id = mine < end ? ids[mine] : -1;
        unsigned long long left = __ballot(counts(id, vocab, padding_id));
        count += __popcll(left);
        while (left != 0) {
            typename Pack<In, kPack>::stored value[kBagAhead];
            int taken = 0;
#pragma unroll
            for (int u = 0; u < kBagAhead; ++u) {
                if (left != 0) {
                    const int next = __builtin_ctzll(left);
                    left &= left - 1;
                    const std::int64_t row = __builtin_amdgcn_readlane(id, next);
                    value[u] = *reinterpret_cast<const typename Pack<In, kPack>::stored*>(from + row * table_stride);
                    ++taken;
                }
            }
#pragma unroll
            for (int u = 0; u < kBagAhead; ++u) {
                if (u < taken) {
                    addPack(value[u], 1.0f, sum);
                }
            }
        }
    }
    if constexpr (kShares > 1) {
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            sums[wave][lane * kPack + e] = sum[e];
        }
        if (lane == 0) {
            found[wave] = count;
        }
        __syncthreads();
        if (share != 0) {
            return;
        }
        for (int w = 1; w < kShares; ++w) {
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                sum[e] += sums[wave + w][lane * kPack + e];
            }
            count += found[wave + w];
        }
    }
    if (has_pack) {
        const float weight = mean && count > 1 ? scale / static_cast<float>(count) : scale;
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            sum[e] *= weight;
        }
        storePack(sum, out + bag * out_stride + column);
    }
}

// ---- gradient: the tokens and their output rows ------------------------------------------------

// Output row of every token of a bag list, and how many of each bag's tokens count.
__global__ __launch_bounds__(kThreads) void bagRowsKernel(const int* __restrict__ ids, int count, int vocab,
                                                          int padding_id,
                                                          const std::int64_t* __restrict__ bag_offsets, int bags,
                                                          int* __restrict__ keys, int* __restrict__ rows,
                                                          unsigned* __restrict__ bag_counts) {
    const int j = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
    if (j >= count) {
        return;
    }
    // the last bag that starts at or before j
    int low = -1, high = bags;
    while (high - low > 1) {
        const int middle = low + (high - low) / 2;
        if (bag_offsets[middle] <= j) {
            low = middle;
        } else {
            high = middle;
        }
    }
    const bool ok = low >= 0 && j < bag_offsets[low + 1] && counts(ids[j], vocab, padding_id);
    keys[j] = ok ? ids[j] : vocab;
    rows[j] = ok ? low : 0;
    if (ok) {
        atomicAdd(bag_counts + low, 1u);  // an integer count: the same in any order
    }
}

__global__ __launch_bounds__(kThreads) void clearWordsKernel(unsigned* __restrict__ words, long long count) {
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < count;
         i += static_cast<long long>(gridDim.x) * kThreads) {
        words[i] = 0u;
    }
}

// ---- gradient ---------------------------------------------------------------------------------

struct GradientArgs {
    const int* keys;  // sorted
    const int* rows;
    int count;
    int chunk;  // sorted positions a block sums
    int vocab;
    int dim;
    const void* out_gradient;
    std::int64_t out_gradient_stride;
    const unsigned* bag_counts;  // null: no mean
    float scale;
    void* table_gradient;
    std::int64_t table_gradient_stride;
    bool accumulate;
    float* partials;  // [chunks, 2, dim]: sums of a chunk's first and last run where they cross chunks
};

// Writes pack `pack` of row `key`, or adds it to what is there: there only the columns that are not the pack
// before's too.
template <typename Out, int kPack>
__device__ __forceinline__ void finishRow(const GradientArgs& args, int key, int pack, float (&sum)[kPack]) {
    const int column = packColumn<kPack>(pack, args.dim);
    Out* to = static_cast<Out*>(args.table_gradient) + key * args.table_gradient_stride + column;
#pragma unroll
    for (int e = 0; e < kPack; ++e) {
        sum[e] *= args.scale;
    }
    if (!args.accumulate) {
        storePack(sum, to);
    } else if (column == pack * kPack) {
        float old[kPack];
        loadPack(static_cast<const Out*>(to), old);
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            sum[e] += old[e];
        }
        storePack(sum, to);
    } else {
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            if (column + e >= pack * kPack) {
                to[e] = static_cast<Out>(static_cast<float>(to[e]) + sum[e]);
            }
        }
    }
}

// A wavefront sums one chunk's rows over 64 packs of columns: it reads the chunk's ids and rows at once, a
// lane each (a chunk is at most 64 positions), and hands them on as scalars; kGradientAhead rows are in
// flight.
constexpr int kGradientAhead = 16;

template <typename In, typename Out, int kPack>
__global__ __launch_bounds__(kThreads) void gradientChunkKernel(GradientArgs args, long long items, int slices) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const long long item = static_cast<long long>(blockIdx.x) * kWavesPerBlock + wave;
    if (item >= items) {
        return;
    }
    const int chunk = static_cast<int>(item / slices);
    const int pack = static_cast<int>(item - static_cast<long long>(chunk) * slices) * kWave + lane;
    const bool has_column = pack < (args.dim + kPack - 1) / kPack;
    const int column = has_column ? packColumn<kPack>(pack, args.dim) : 0;
    const int begin = chunk * args.chunk;
    const int length = min(args.chunk, args.count - begin);
    const int at = begin + min(lane, length - 1);
    const int my_key = args.keys[at];
    const int my_row = args.rows[at];
    // tokens that do not count stand at the end
    const int valid = __popcll(__ballot(lane < length && my_key < args.vocab));
    if (valid == 0) {
        return;
    }
    float my_weight = 1.0f;
    if (args.bag_counts != nullptr && my_key < args.vocab) {
        my_weight = 1.0f / static_cast<float>(args.bag_counts[my_row]);
    }
    const int key_before = begin > 0 ? args.keys[begin - 1] : -1;
    const int key_after = begin + length < args.count ? args.keys[begin + length] : args.vocab;
    const In* from = static_cast<const In*>(args.out_gradient) + column;
    float* partials = args.partials + static_cast<std::size_t>(chunk) * 2 * args.dim + column;
    int current = __builtin_amdgcn_readlane(my_key, 0);
    bool continued = key_before == current;  // the run so far began before this chunk
    float sum[kPack] = {};
    for (int j = 0; j < valid; j += kGradientAhead) {
        typename Pack<In, kPack>::stored value[kGradientAhead];
#pragma unroll
        for (int u = 0; u < kGradientAhead; ++u) {
            if (j + u < valid) {
                const std::int64_t row = __builtin_amdgcn_readlane(my_row, j + u);
                value[u] = __builtin_nontemporal_load(
                    reinterpret_cast<const typename Pack<In, kPack>::stored*>(from + row * args.out_gradient_stride));
            }
        }
#pragma unroll
        for (int u = 0; u < kGradientAhead; ++u) {
            if (j + u < valid) {
                const int key = __builtin_amdgcn_readlane(my_key, j + u);
                if (key != current) {
                    if (has_column) {
                        if (continued) {
                            storePack(sum, partials);
                        } else {
                            finishRow<Out, kPack>(args, current, pack, sum);
                        }
                    }
                    continued = false;
                    current = key;
#pragma unroll
                    for (int e = 0; e < kPack; ++e) {
                        sum[e] = 0.0f;
                    }
                }
                const float weight = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_weight), j + u));
                addPack(value[u], weight, sum);
            }
        }
    }
    if (!has_column) {
        return;
    }
    if (continued) {
        storePack(sum, partials);
    } else if (valid == length && key_after == current) {
        storePack(sum, partials + args.dim);
    } else {
        finishRow<Out, kPack>(args, current, pack, sum);
    }
}

// Joins the runs that cross chunks: the sum of the chunk where a run begins and the first sums of the
// chunks it reaches, over a slice of 64 packs. A wavefront looks at one chunk's end each and joins a run that
// reaches few chunks by itself; the workgroup then takes the longer ones together, an equal share of the
// chunks a wavefront.
constexpr int kJoinThreads = 512;
constexpr int kJoinWaves = kJoinThreads / kWave;
constexpr int kJoinAlone = 16;  // chunks

template <typename Out, int kPack>
__global__ __launch_bounds__(kJoinThreads) void gradientJoinKernel(GradientArgs args) {
    __shared__ float sums[kJoinWaves][kWave * kPack];
    __shared__ int last_of[kJoinWaves];  // the last chunk of the run that begins in the wavefront's chunk
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int chunks = (args.count + args.chunk - 1) / args.chunk;
    const int pack = static_cast<int>(blockIdx.y) * kWave + lane;
    const bool has_column = pack < (args.dim + kPack - 1) / kPack;
    const std::size_t stride = 2 * static_cast<std::size_t>(args.dim);
    const float* partials = args.partials + (has_column ? packColumn<kPack>(pack, args.dim) : 0);
    const int first_chunk = static_cast<int>(blockIdx.x) * kJoinWaves;

    int chunk = first_chunk + wave;
    int last = chunk;  // no run to join
    if (chunk + 1 < chunks) {
        const int next = (chunk + 1) * args.chunk;
        const int begin = chunk * args.chunk;
        const int key = args.keys[next - 1];
        const bool crosses = key == args.keys[next] && key < args.vocab;
        const bool begins = begin == 0 || args.keys[begin] != key || args.keys[begin - 1] != key;
        if (crosses && begins) {
            // the last chunk whose first id is the run's
            last = chunk + 1;
            int past = chunks;
            while (past - last > 1) {
                const int middle = last + (past - last) / 2;
                if (args.keys[middle * args.chunk] == key) {
                    last = middle;
                } else {
                    past = middle;
                }
            }
        }
    }
    if (lane == 0) {
        last_of[wave] = last;
    }
    if (last > chunk && last - chunk <= kJoinAlone) {
        float sum[kPack];
        loadPack(partials + chunk * stride + args.dim, sum);
#pragma unroll 4
        for (int c = chunk + 1; c <= last; ++c) {
            float more[kPack];
            loadPack(partials + c * stride, more);
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                sum[e] += more[e];
            }
        }
        if (has_column) {
            finishRow<Out, kPack>(args, args.keys[last * args.chunk], pack, sum);
        }
    }
    __syncthreads();
    for (int w = 0; w < kJoinWaves; ++w) {
        chunk = first_chunk + w;
        last = last_of[w];
        const int reached = last - chunk;
        if (reached <= kJoinAlone) {
            continue;
        }
        const int share = (reached + kJoinWaves - 1) / kJoinWaves;
        const int from = chunk + 1 + wave * share;
        const int to = min(from + share, last + 1);
        float sum[kPack] = {};
        if (wave == 0) {
            loadPack(partials + chunk * stride + args.dim, sum);
        }
#pragma unroll 8
        for (int c = from; c < to; ++c) {
            float more[kPack];
            loadPack(partials + c * stride, more);
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                sum[e] += more[e];
            }
        }
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
            sums[wave][lane * kPack + e] = sum[e];
        }
        __syncthreads();
        if (wave == 0 && has_column) {
            for (int v = 1; v < kJoinWaves; ++v) {
#pragma unroll
                for (int e = 0; e < kPack; ++e) {
                    sum[e] += sums[v][lane * kPack + e];
                }
            }
            finishRow<Out, kPack>(args, args.keys[last * args.chunk], pack, sum);
        }
        __syncthreads();
    }
}

// Zeros for the rows of the gradient, written beside the sort: launch l of the sort's takes an equal part
// of the packs.
template <typename Out, int kPack>
struct ClearRows {
    static constexpr int kBlocks = 768;
    Out* out;  // null: nothing to clear
    std::int64_t stride;
    long long packs;
    int dim;

    __device__ void run(int block, int blocks, int launch, int launches) const {
        if (out == nullptr) {
            return;
        }
        const int packs_per_row = (dim + kPack - 1) / kPack;
        const long long begin = packs * launch / launches;
        const long long end = packs * (launch + 1) / launches;
        const float zeros[kPack] = {};
        const long long step = static_cast<long long>(blocks) * blockDim.x;
        long long at = begin + static_cast<long long>(block) * blockDim.x + threadIdx.x;
        long long row = at / packs_per_row;
        int pack = static_cast<int>(at - row * packs_per_row);
        const long long row_step = step / packs_per_row;
        const int pack_step = static_cast<int>(step - row_step * packs_per_row);
        for (; at < end; at += step) {
            storePackOnce(zeros, out + row * stride + packColumn<kPack>(pack, dim));
            row += row_step;
            pack += pack_step;
            if (pack >= packs_per_row) {
                pack -= packs_per_row;
                ++row;
            }
        }
    }
};

// Few tokens need no sort: a workgroup looks whether its token is the first of its id and sums the id's
// tokens then, over a slice of 64 packs. Every wavefront takes a quarter of the positions from the token's on, in
// their order; the quarters are joined in theirs. One launch instead of three: 500
// tokens of 384 columns take 9.9 us with the clearing of 30,000 rows, sorted 18.0 us, and 7.5 us against 15.9 us at
// 2,000 rows. The time grows with the tokens of one id, as its workgroup's loads do: 500 of the same take 11.7 us
// against 13.4 us, 1,000 about 24 us against 13.5 us, so more are sorted.
// Blocks past those of the sums clear the rows that no token names, a range of rows at a time, whose named ones
// they mark first: one launch for both, 2 to 3 us less than two (500 tokens and 30,000 rows of 384 columns
// 13.4 -> 9.9 us).
constexpr int kFewAhead = 16;
constexpr std::int64_t kFewTokens = 512;
constexpr int kFewClearBlocks = 2048;
constexpr int kFewClearRows = 1024;  // of a range

template <typename Out, int kPack>
__device__ __forceinline__ void clearUnnamed(const ClearRows<Out, kPack>& clear, const SortInput& in, int block) {
    __shared__ unsigned named[kFewClearRows / 32];
    const int packs_per_row = (clear.dim + kPack - 1) / kPack;
    const int range_rows = min(kFewClearRows, (in.key_end - 1) / kFewClearBlocks + 1);
    const int ranges = (in.key_end - 1) / range_rows + 1;
    const float zeros[kPack] = {};
    for (int range = block; range < ranges; range += kFewClearBlocks) {
        const int first = range * range_rows;
        const int rows = min(range_rows, in.key_end - first);
        if (threadIdx.x < kFewClearRows / 32) {
            named[threadIdx.x] = 0;
        }
        __syncthreads();
        for (int i = static_cast<int>(threadIdx.x); i < in.count; i += kThreads) {
            const int row = sortKey(in, i) - first;
            if (row >= 0 && row < rows) {
                atomicOr(&named[row / 32], 1u << (row % 32));
            }
        }
        __syncthreads();
        int row = static_cast<int>(threadIdx.x) / packs_per_row;
        int pack = static_cast<int>(threadIdx.x) - row * packs_per_row;
        const int row_step = kThreads / packs_per_row;
        const int pack_step = kThreads - row_step * packs_per_row;
        while (row < rows) {
            if (((named[row / 32] >> (row % 32)) & 1u) == 0) {
                storePackOnce(zeros, clear.out + static_cast<std::int64_t>(first + row) * clear.stride +
                                         packColumn<kPack>(pack, clear.dim));
            }
            row += row_step;
            pack += pack_step;
            if (pack >= packs_per_row) {
                pack -= packs_per_row;
                ++row;
            }
        }
        __syncthreads();
    }
}

template <typename In, typename Out, int kPack>
__global__ __launch_bounds__(kThreads) void gradientFewKernel(GradientArgs args, SortInput in, int slices,
                                                            ClearRows<Out, kPack> clear) {
    const int sum_blocks = in.count * slices;
    if (static_cast<int>(blockIdx.x) >= sum_blocks) {
        clearUnnamed<Out, kPack>(clear, in, static_cast<int>(blockIdx.x) - sum_blocks);
        return;
    }
    __shared__ float sums[kWavesPerBlock][kWave * kPack];
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int token = static_cast<int>(blockIdx.x) / slices;
    const int pack = (static_cast<int>(blockIdx.x) - token * slices) * kWave + lane;
    const int key = sortKey(in, token);
    if (key >= in.key_end) {
        return;
    }
    bool earlier = false;
    for (int i = static_cast<int>(threadIdx.x); i < token; i += kThreads) {
        earlier |= sortKey(in, i) == key;
    }
    if (__syncthreads_or(earlier ? 1 : 0) != 0) {
        return;
    }
    const bool has_column = pack < (args.dim + kPack - 1) / kPack;
    const In* from = static_cast<const In*>(args.out_gradient) + (has_column ? packColumn<kPack>(pack, args.dim) : 0);
    const int share = (in.count - token + kThreads - 1) / kThreads * kWave;
    const int end = min(token + (wave + 1) * share, in.count);
    float sum[kPack] = {};
    for (int base = token + wave * share; base < end; base += kWave) {
        const int position = min(base + lane, in.count - 1);
        const int my_row = in.rows == nullptr ? position : in.rows[position];
        const bool mine = base + lane < end && sortKey(in, position) == key;
        float my_weight = 1.0f;
        if (args.bag_counts != nullptr && mine) {
            my_weight = 1.0f / static_cast<float>(args.bag_counts[my_row]);
        }
        unsigned long long left = __ballot(mine);
        while (left != 0) {
            typename Pack<In, kPack>::stored value[kFewAhead];
            int at[kFewAhead];
            int taken = 0;
#pragma unroll
            for (int u = 0; u < kFewAhead; ++u) {
                if (left != 0) {
                    at[u] = __builtin_ctzll(left);
                    left &= left - 1;
                    const std::int64_t row = __builtin_amdgcn_readlane(my_row, at[u]);
                    value[u] = *reinterpret_cast<const typename Pack<In, kPack>::stored*>(
                        from + row * args.out_gradient_stride);
                    ++taken;
                }
            }
#pragma unroll
            for (int u = 0; u < kFewAhead; ++u) {
                if (u < taken) {
                    const float weight = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_weight), at[u]));
                    addPack(value[u], weight, sum);
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < kPack; ++e) {
        sums[wave][lane * kPack + e] = sum[e];
    }
    __syncthreads();
    if (wave == 0 && has_column) {
        for (int w = 1; w < kWavesPerBlock; ++w) {
#pragma unroll
            for (int e = 0; e < kPack; ++e) {
                sum[e] += sums[w][lane * kPack + e];
            }
        }
        finishRow<Out, kPack>(args, key, pack, sum);
    }
}

// ---- host ---------------------------------------------------------------------------------------

std::int64_t rowStride(std::int64_t stride, int length) { return stride == 0 ? length : stride; }

int invalid(const char* message) {
    return setError(ZCGVS_ERR_INVALID_ARGUMENT, std::string("zcgvs embedding: ") + message);
}

// Checks what lookup and gradient share.
int checkEmbedding(const zcgvs_embedding_desc* desc) {
    if (desc == nullptr) {
        return invalid("null descriptor");
    }
    if (desc->vocab <= 0 || desc->dim <= 0) {
        return invalid("vocab and dim must be positive");
    }
    if (desc->dim > kMaxDim) {
        return invalid("dim must be at most 2^23");
    }
    if (desc->vocab == INT32_MAX) {
        return invalid("vocab must be below 2^31 - 1");
    }
    if (desc->token_count < 0 || desc->token_count > kMaxTokens) {
        return invalid("token_count must lie in [0, 2^28]");
    }
    if (desc->bag_offsets != nullptr && (desc->bag_count < 0 || desc->bag_count > INT32_MAX)) {
        return invalid("bag_count must lie in [0, 2^31 - 1]");
    }
    if (desc->bag_offsets == nullptr && desc->bag_count > 0) {
        return invalid("bag_count needs bag_offsets");
    }
    if (desc->reduce != ZCGVS_EMBEDDING_SUM && desc->reduce != ZCGVS_EMBEDDING_MEAN) {
        return invalid("unknown reduction");
    }
    if (desc->token_count > 0 && desc->ids == nullptr) {
        return invalid("null token ids");
    }
    return ZCGVS_OK;
}

template <typename In, typename Out, int kPack>
int lookupTyped(const zcgvs_embedding_desc& d, Out* out, std::int64_t out_stride, hipStream_t stream) {
    const In* table = static_cast<const In*>(d.table);
    const std::int64_t table_stride = rowStride(d.table_stride, d.dim);
    const int packs_per_row = (d.dim + kPack - 1) / kPack;
    if (d.bag_offsets == nullptr) {
        const long long packs = static_cast<long long>(d.token_count) * packs_per_row;
        const long long blocks = (packs + kThreads * kLookupPacks - 1) / (kThreads * kLookupPacks);
        if (blocks > kMaxBlocks) {
            return invalid("more output than one launch can write");
        }
        lookupKernel<In, Out, kPack><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
            table, table_stride, d.vocab, d.dim, d.ids, packs, d.padding_id, d.scale, out, out_stride);
    } else {
        const int slices = (packs_per_row + kWave - 1) / kWave;
        // a wavefront a bag where that keeps the GPU's memory busy, else four
        const bool alone = d.bag_count * slices >= 16ll * deviceComputeUnits();
        const int items_per_block = alone ? kWavesPerBlock : 1;
        const std::int64_t most = std::max<std::int64_t>(1, kMaxBlocks * items_per_block / slices);
        for (std::int64_t bag = 0; bag < d.bag_count; bag += most) {
            const long long items = std::min<std::int64_t>(most, d.bag_count - bag) * slices;
            const unsigned blocks = static_cast<unsigned>((items + items_per_block - 1) / items_per_block);
            const auto kernel = alone ? bagKernel<In, Out, kPack, 1> : bagKernel<In, Out, kPack, kWavesPerBlock>;
            kernel<<<blocks, kThreads, 0, stream>>>(table, table_stride, d.vocab, d.dim, d.ids, d.token_count,
                                                    d.bag_offsets + bag, items, slices,
                                                    d.reduce == ZCGVS_EMBEDDING_MEAN, d.padding_id, d.scale,
                                                    out + bag * out_stride, out_stride);
        }
    }
    ZCGVS_LAUNCH_CHECK("embedding lookup");
    return ZCGVS_OK;
}

// Parts of the gradient's workspace, 256-byte aligned.
struct GradientSpace {
    std::size_t sort;
    std::size_t bag_keys;
    std::size_t bag_rows;
    std::size_t bag_counts;
    std::size_t partials;
    std::size_t bytes;
    int chunk;
};

GradientSpace gradientSpace(const zcgvs_embedding_desc& d) {
    GradientSpace s{};
    std::size_t at = 0;
    auto take = [&](std::size_t bytes) {
        const std::size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const std::size_t n = static_cast<std::size_t>(d.token_count);
    // enough chunks for the whole GPU where there are few tokens; long enough to read on beyond
    s.chunk = 64;
    while (s.chunk > 8 && n / static_cast<std::size_t>(s.chunk) < 1024) {
        s.chunk /= 2;
    }
    const bool bags = d.bag_offsets != nullptr;
    s.sort = take(pairSortBytes(n));
    s.bag_keys = take(bags ? n * 4 : 0);
    s.bag_rows = take(bags ? n * 4 : 0);
    s.bag_counts = take(bags ? static_cast<std::size_t>(d.bag_count) * 4 : 0);
    const std::size_t chunks = (n + static_cast<std::size_t>(s.chunk) - 1) / static_cast<std::size_t>(s.chunk);
    s.partials = take(chunks * 2 * static_cast<std::size_t>(d.dim) * 4);
    s.bytes = std::max<std::size_t>(at, 256);
    return s;
}

unsigned clearBlocks(long long words) {
    return static_cast<unsigned>(std::max(1ll, std::min(2048ll, (words + kThreads - 1) / kThreads)));
}

// The tokens' ids and output rows.
int tokenPairs(const zcgvs_embedding_desc& d, const GradientSpace& s, char* workspace, SortInput& input,
               hipStream_t stream) {
    const int n = static_cast<int>(d.token_count);
    input = SortInput{};
    input.keys = d.ids;
    input.count = n;
    input.key_end = d.vocab;
    input.skipped = d.padding_id;
    input.raw = true;
    if (d.bag_offsets != nullptr) {
        unsigned* bag_counts = reinterpret_cast<unsigned*>(workspace + s.bag_counts);
        int* bag_keys = reinterpret_cast<int*>(workspace + s.bag_keys);
        int* bag_rows = reinterpret_cast<int*>(workspace + s.bag_rows);
        clearWordsKernel<<<clearBlocks(d.bag_count), kThreads, 0, stream>>>(bag_counts, d.bag_count);
        ZCGVS_LAUNCH_CHECK("embedding gradient");
        bagRowsKernel<<<static_cast<unsigned>((n + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
            d.ids, n, d.vocab, d.padding_id, d.bag_offsets, static_cast<int>(d.bag_count), bag_keys, bag_rows,
            bag_counts);
        ZCGVS_LAUNCH_CHECK("embedding gradient");
        input.keys = bag_keys;
        input.rows = bag_rows;
        input.raw = false;
    }
    return ZCGVS_OK;
}

template <typename In, typename Out, int kPack>
int gradientTyped(const zcgvs_embedding_desc& d, const GradientSpace& s, GradientArgs args, char* workspace,
                  hipStream_t stream) {
    ClearRows<Out, kPack> clear{};
    if (!args.accumulate) {
        clear.out = static_cast<Out*>(args.table_gradient);
        clear.stride = args.table_gradient_stride;
        clear.dim = d.dim;
        clear.packs = static_cast<long long>(d.vocab) * ((d.dim + kPack - 1) / kPack);
    }
    SortInput input{};
    input.key_end = d.vocab;
    if (args.count > 0) {
        const int paired = tokenPairs(d, s, workspace, input, stream);
        if (paired != ZCGVS_OK) {
            return paired;
        }
    }
    const int slices = ((d.dim + kPack - 1) / kPack + kWave - 1) / kWave;
    const long long few_blocks =
        static_cast<long long>(args.count) * slices + (args.accumulate ? 0 : kFewClearBlocks);
    if (args.count == 0 || (args.count <= kFewTokens && few_blocks <= kMaxBlocks)) {
        gradientFewKernel<In, Out, kPack>
            <<<static_cast<unsigned>(few_blocks), kThreads, 0, stream>>>(args, input, slices, clear);
        ZCGVS_LAUNCH_CHECK("embedding gradient");
        return ZCGVS_OK;
    }
    const int sorted = args.accumulate
                           ? sortPairs(input, workspace + s.sort, &args.keys, &args.rows, NoSideWork{}, stream)
                           : sortPairs(input, workspace + s.sort, &args.keys, &args.rows, clear, stream);
    if (sorted != ZCGVS_OK) {
        return sorted;
    }
    const int chunks = static_cast<int>((static_cast<long long>(args.count) + s.chunk - 1) / s.chunk);
    const long long items = static_cast<long long>(chunks) * slices;
    const long long blocks = (items + kWavesPerBlock - 1) / kWavesPerBlock;
    if (blocks > kMaxBlocks) {
        return invalid("more tokens than one launch can take");
    }
    gradientChunkKernel<In, Out, kPack><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(args, items, slices);
    ZCGVS_LAUNCH_CHECK("embedding gradient");
    if (chunks > 1) {
        gradientJoinKernel<Out, kPack><<<dim3(static_cast<unsigned>((chunks - 1 + kJoinWaves - 1) / kJoinWaves),
                                              static_cast<unsigned>(slices)),
                                         kJoinThreads, 0, stream>>>(args);
        ZCGVS_LAUNCH_CHECK("embedding gradient");
    }
    return ZCGVS_OK;
}

}  // namespace

}  // namespace zcgvs_hip

using namespace zcgvs_hip;

extern "C" {

int zcgvs_embedding_lookup(const zcgvs_embedding_desc* desc, void* d_out, std::int64_t out_stride, int out_dtype,
                           zcgvs_stream_t stream) {
    const int status = checkEmbedding(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_embedding_desc& d = *desc;
    if (!validElement(d.dtype)) {
        return invalid("the table must hold float32, float16 or bfloat16");
    }
    if (out_dtype != d.dtype && out_dtype != ZCGVS_DTYPE_F32) {
        return invalid("the output type is the table's or float32");
    }
    const std::int64_t stride = rowStride(out_stride, d.dim);
    const std::int64_t table_stride = rowStride(d.table_stride, d.dim);
    if (stride < d.dim || table_stride < d.dim) {
        return invalid("a row stride is smaller than dim");
    }
    const std::int64_t rows = d.bag_offsets != nullptr ? d.bag_count : d.token_count;
    if (rows == 0) {
        return clearError();
    }
    if (d.table == nullptr || d_out == nullptr) {
        return invalid("null device pointer");
    }
    const int launched = withElement(d.dtype, [&](auto in) {
        using In = decltype(in);
        return withElement(out_dtype, [&](auto element) {
            using Out = decltype(element);
            if constexpr (std::is_same_v<Out, In> || std::is_same_v<Out, float>) {
                return d.dim >= 4 ? lookupTyped<In, Out, 4>(d, static_cast<Out*>(d_out), stride, toStream(stream))
                                 : lookupTyped<In, Out, 1>(d, static_cast<Out*>(d_out), stride, toStream(stream));
            } else {
                return static_cast<int>(ZCGVS_ERR_INVALID_ARGUMENT);  // refused above
            }
        });
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

std::size_t zcgvs_embedding_gradient_workspace_bytes(const zcgvs_embedding_desc* desc) {
    if (checkEmbedding(desc) != ZCGVS_OK) {
        return 0;
    }
    clearError();
    return gradientSpace(*desc).bytes;
}

int zcgvs_embedding_gradient(const zcgvs_embedding_desc* desc, const void* d_out_gradient,
                             std::int64_t out_gradient_stride, int gradient_dtype, void* d_table_gradient,
                             std::int64_t table_gradient_stride, int table_gradient_dtype, int accumulate,
                             void* d_workspace, std::size_t workspace_bytes, zcgvs_stream_t stream) {
    const int status = checkEmbedding(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_embedding_desc& d = *desc;
    if (!validElement(gradient_dtype)) {
        return invalid("the output gradient must hold float32, float16 or bfloat16");
    }
    if (table_gradient_dtype != gradient_dtype && table_gradient_dtype != ZCGVS_DTYPE_F32) {
        return invalid("the table gradient's type is the output gradient's or float32");
    }
    const std::int64_t from_stride = rowStride(out_gradient_stride, d.dim);
    const std::int64_t to_stride = rowStride(table_gradient_stride, d.dim);
    if (from_stride < d.dim || to_stride < d.dim) {
        return invalid("a row stride is smaller than dim");
    }
    const bool no_tokens = d.token_count == 0 || (d.bag_offsets != nullptr && d.bag_count == 0);
    if (no_tokens && accumulate != 0) {
        return clearError();
    }
    if (d_table_gradient == nullptr || (!no_tokens && d_out_gradient == nullptr)) {
        return invalid("null device pointer");
    }
    const GradientSpace space = gradientSpace(d);
    if (!no_tokens && (d_workspace == nullptr || workspace_bytes < space.bytes)) {
        return invalid("the workspace is too small");
    }
    if (!no_tokens && !aligned16(d_workspace)) {
        return invalid("the workspace must be aligned to 16 bytes");
    }
    char* workspace = static_cast<char*>(d_workspace);
    GradientArgs args{};
    if (!no_tokens) {
        args.partials = reinterpret_cast<float*>(workspace + space.partials);
    }
    args.count = no_tokens ? 0 : static_cast<int>(d.token_count);
    args.chunk = space.chunk;
    args.vocab = d.vocab;
    args.dim = d.dim;
    args.out_gradient = d_out_gradient;
    args.out_gradient_stride = from_stride;
    args.bag_counts = d.bag_offsets != nullptr && d.reduce == ZCGVS_EMBEDDING_MEAN
                          ? reinterpret_cast<const unsigned*>(workspace + space.bag_counts)
                          : nullptr;
    args.scale = d.scale;
    args.table_gradient = d_table_gradient;
    args.table_gradient_stride = to_stride;
    args.accumulate = accumulate != 0;
    const int launched = withElement(gradient_dtype, [&](auto in) {
        using In = decltype(in);
        return withElement(table_gradient_dtype, [&](auto element) {
            using Out = decltype(element);
            if constexpr (std::is_same_v<Out, In> || std::is_same_v<Out, float>) {
                return d.dim >= 4 ? gradientTyped<In, Out, 4>(d, space, args, workspace, toStream(stream))
                                 : gradientTyped<In, Out, 1>(d, space, args, workspace, toStream(stream));
            } else {
                return static_cast<int>(ZCGVS_ERR_INVALID_ARGUMENT);  // refused above
            }
        });
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

}  // extern "C"
