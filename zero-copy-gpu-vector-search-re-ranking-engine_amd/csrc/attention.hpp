// What the attention's translation units share: arguments, the texts' rows, the tiles of keys in LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "common.hpp"
#include "elements.hpp"
#include "lds_copy.hpp"
#include "matrix_tile.hpp"

namespace zcgvs_hip {

constexpr int kAttentionMaxDim = 128;
constexpr int kAttentionMaxDistance = 512;
constexpr long long kMaxAttentionBlocks = (1ll << 24) - 1;  // a launch has less than 2^32 threads, of 256 a block
constexpr float kLog2E = 1.44269504f;
constexpr float kLn2 = 0.69314718f;

// Rows of a batch's texts: those of text t are offsets[t] .. offsets[t + 1] - 1 (null: `each` rows a text), the first
// lengths[t] of them count (null: all).
struct TextRows {
    const std::int64_t* offsets;
    const int* lengths;
    std::int64_t total;
    int texts;
    int each;
};

struct AttentionArgs {
    const void* q;
    const void* k;
    const void* v;
    std::int64_t q_stride;
    std::int64_t k_stride;
    std::int64_t v_stride;
    TextRows q_texts;
    TextRows k_texts;
    int heads;
    int group;  // query heads to a key head
    int head_dim;
    int q_last;  // the query rows stand at the end of their text's keys
    int causal;
    const int* prefix;
    float scale;
    float cap;
    const float* slopes;
    const void* table;
    int max_distance;
};

struct AttentionOutput {
    void* out;
    std::int64_t out_stride;
    float* lse;
    int slots;   // tiles of query rows, empty ones among them
    int splits;  // parts of the keys, each with its own workgroups
    float* partial_rows;   // [splits, q_rows * heads, padded head_dim] of unfinished rows (splits > 1)
    float* partial_stats;  // [splits, q_rows * heads, 2]: the largest score and the sum of exponentials, base 2
};

// How attention.hip runs a call.
enum class AttentionShape { kNarrow, kShort, kLong };  // 16 rows of a workgroup, 64, 128
struct AttentionPlan {
    AttentionShape shape;
    bool direct;  // rows of whole aligned chunks
};

template <typename T>
int launchAttention(const AttentionPlan& plan, const AttentionArgs& args, const AttentionOutput& output, hipStream_t stream);

struct AttentionGradient {
    const void* out;
    std::int64_t out_stride;
    const float* lse;
    const void* out_gradient;
    std::int64_t out_gradient_stride;
    void* q_gradient;
    std::int64_t q_gradient_stride;
    void* k_gradient;
    std::int64_t k_gradient_stride;
    void* v_gradient;
    std::int64_t v_gradient_stride;
    void* table_gradient;
    float* stats;           // [heads, q_rows, 2]: lse in base 2, delta
    float* table_partials;  // [heads, key_slots, 2 * max_distance + 1], or null: not wanted
    int key_slots;          // tiles of keys, empty ones among them
    int key_parts;          // of a key head's query heads, each with its own workgroups
    float* key_partials;    // [2 (dk, dv), key_parts, k_rows, kv_heads * head_dim] (key_parts > 1)
    int query_slots;
};

// Blocks of 16 keys (query rows) of a wavefront; rows of whole aligned chunks: of q and the output's gradient, of k and v.
struct AttentionGradientPlan {
    int key_blocks;
    int query_blocks;
    bool direct_rows;
    bool direct_keys;
};

template <typename T>
int launchAttentionGradient(const AttentionGradientPlan& plan, const AttentionArgs& args, const AttentionGradient& more,
                            hipStream_t stream);

int attentionInvalid(const char* message);

// The head's width in LDS and registers: zeros fill it up.
inline int paddedDim(int head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128; }

// The narrow shape: keys of a wavefront's tile, those of 4 KB, but whole turned fragments of them and at most 64; floats of the
// tables of a key head's query heads that LDS holds, each with a margin on either side.
constexpr int narrowKeys(int padded_dim, int element_bytes) {
    return padded_dim * element_bytes <= 64 ? 64 : padded_dim * element_bytes <= 128 || element_bytes == 2 ? 32 : 16;
}
constexpr int kNarrowRows = 16;
constexpr int kNarrowTable = 4096;
constexpr int biasTableWidth(int max_distance, int margin) { return 2 * (max_distance + margin) + 1; }

namespace {

struct TextSpan {
    std::int64_t first;
    int rows;   // that there are
    int count;  // that count
};

// Offsets out of order or out of range give spans within the rows all the same.
__device__ __forceinline__ std::int64_t textStart(const TextRows& rows, int t) {
    if (rows.offsets == nullptr) {
        return static_cast<std::int64_t>(t) * rows.each;
    }
    const std::int64_t at = rows.offsets[t];
    return at < 0 ? 0 : at < rows.total ? at : rows.total;
}

__device__ __forceinline__ TextSpan textSpan(const TextRows& rows, int t) {
    TextSpan span;
    span.first = textStart(rows, t);
    const std::int64_t end = textStart(rows, t + 1);
    span.rows = end > span.first ? static_cast<int>(end - span.first) : 0;
    span.count = rows.lengths == nullptr ? span.rows : min(max(rows.lengths[t], 0), span.rows);
    return span;
}

// Tiles of kTile rows never hold rows of two texts. Text t's begin at slot floor(first row / kTile) + t, so that they are
// found without a list: the next text's begin at least as many slots on as this one has tiles.
// The text of a slot (-1: none), by a search of all lanes at a time, the same in every lane. `weight`: tile rows
// to a text's row.
template <int kTile>
__device__ __forceinline__ int textOfSlot(const TextRows& rows, int weight, int slot) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    int low = 0, high = rows.texts;
    while (true) {
        const int step = (high - low + kWave - 1) / kWave;
        const int t = low + lane * step;
        const bool at_or_before = t < high && textStart(rows, t) * weight / kTile + t <= slot;
        const int count = __popcll(__ballot(at_or_before));
        if (count == 0) {
            return -1;
        }
        low += (count - 1) * step;
        high = min(high, low + step);
        if (step == 1) {
            return __builtin_amdgcn_readfirstlane(low);
        }
    }
}

inline long long slotsOf(const TextRows& rows, int weight, int tile) { return rows.total * weight / tile + rows.texts; }

// Position b of a launch of `total` blocks: blocks of one XCD (every eighth one) get neighbouring positions, so that tiles
// of one head and text read its keys through one L2.
__device__ __forceinline__ int positionOf(int block, int total) {
    const int xcd = block % kXcds;
    const int whole = total / kXcds;
    return xcd * whole + min(xcd, total % kXcds) + block / kXcds;
}

// A row's 16-byte chunk from value `at` on, of which `left` exist; zeros past them.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::type loadRowChunk(const T* from, int left) {
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

// The calling lane's fragments of a row along its kSteps matrix instruction steps: `width` values exist (0: no row).
template <typename T, int kSteps>
__device__ __forceinline__ void loadRowFragments(const T* row, int width, bool whole_chunks, typename Fragment<T>::type (&to)[kSteps]) {
    const int h = (static_cast<int>(threadIdx.x) & (kWave - 1)) >> 4;
    if (whole_chunks) {
        // every chunk is there or not: all loads at once
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            const int d = (4 * t + h) * kChunk<T>;
            __builtin_memcpy(&to[t], d < width ? static_cast<const void*>(row + d) : static_cast<const void*>(&zero_chunk), 16);
        }
    } else {
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            const int d = (4 * t + h) * kChunk<T>;
            to[t] = loadRowChunk(row + d, width - d);
        }
    }
}

// kRows rows of kDim values in LDS, one behind the other. A row's chunk c stands in slot c ^ turn(row), so that what is
// read together falls on different columns of the 256 bytes that the banks hold. A 16-byte read takes 16 lanes at a time,
// of a lane group and the next one: rows 0-3 and 12-15 of chunk c with rows 4-11 of chunk c + 1, or the others. A
// transposing read (16-bit) takes half a wavefront: rows 0-7, or 8-15, two chunks of each.
template <typename T, int kRows, int kDim, int kTeam, bool kDirect>
struct RowTile {
    static constexpr int kRowBytes = kDim * static_cast<int>(sizeof(T));
    static constexpr int kBytes = kRows * kRowBytes;
    static constexpr int kRowChunks = kRowBytes / 16;
    static constexpr int kChunks = kRows * kRowChunks;
    static constexpr int kCopies = (kChunks + kTeam - 1) / kTeam;
    static constexpr int kSteps = kRowBytes / 64;  // matrix instruction steps over a row
    static_assert(kChunks % kTeam == 0 || (kChunks < kTeam && kChunks % kWave == 0), "a tile splits over its wavefronts");

    // Small tiles leave the last wavefronts without a copy.
    static __device__ __forceinline__ bool hasCopy() {
        return kChunks >= kTeam || __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) % kTeam / kWave) * kWave < kChunks;
    }

    static __device__ __forceinline__ int turn(int row) {
        constexpr int kPerLine = kRowBytes >= 256 ? 1 : 256 / kRowBytes;
        constexpr int kTurns = kRowChunks < 16 ? kRowChunks : 16;
        const int p = (row / kPerLine) & (kTurns - 1);
        if constexpr (sizeof(T) == 2) {
            return ((2 * p) & (kTurns - 1)) ^ (p / (kTurns / 2) * (kTurns / 2 + 1));
        } else {
            return p;
        }
    }

    const T* src[kCopies];
    std::int64_t step;  // values from tile to tile
    int rows_left;      // from the next tile's first row on
    int width;          // values of a row that exist
    u32x4 held[kDirect ? 1 : kCopies];

    static __device__ __forceinline__ void placeOf(int i, int& row, int& chunk) {
        const int slot = i * kTeam + static_cast<int>(threadIdx.x) % kTeam;
        row = slot / kRowChunks;
        chunk = (slot % kRowChunks) ^ turn(row);
    }

    // Rows `base`, base + stride, ..., `count` of them; tiles `tiles_apart` tiles apart.
    __device__ __forceinline__ void begin(const T* base, std::int64_t stride, int count, int row_width, int tiles_apart) {
        step = stride * kRows * tiles_apart;
        rows_left = count;
        width = row_width;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            int row, chunk;
            placeOf(i, row, chunk);
            src[i] = base + row * stride + chunk * kChunk<T>;
        }
    }
    __device__ __forceinline__ bool exists(int i) const {
        int row, chunk;
        placeOf(i, row, chunk);
        return row < rows_left && chunk * kChunk<T> < width;
    }
    // Starts the next tile's copies into `to` (direct).
    __device__ __forceinline__ void issue(const std::uint8_t* to, int tiles_apart) {
        const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) % kTeam / kWave);
        const std::uint32_t base = ldsAddress(to) + static_cast<std::uint32_t>(wave * kWave * 16);
        const bool whole = rows_left >= kRows && width == kDim;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const void* from = whole || exists(i) ? static_cast<const void*>(src[i]) : static_cast<const void*>(&zero_chunk);
            if (hasCopy()) {
                copySharedToLds(from, __builtin_amdgcn_readfirstlane(base + i * kTeam * 16));
            }
            src[i] += step;
        }
        rows_left -= kRows * tiles_apart;
    }
    // Reads the next tile into registers, and later writes it to `to` (not direct).
    __device__ __forceinline__ void fetch(int tiles_apart) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            int row, chunk;
            placeOf(i, row, chunk);
            const int left = hasCopy() && row < rows_left ? width - chunk * kChunk<T> : 0;
            held[i] = __builtin_bit_cast(u32x4, loadRowChunk(src[i], left));
            src[i] += step;
        }
        rows_left -= kRows * tiles_apart;
    }
    __device__ __forceinline__ void put(std::uint8_t* to) const {
        if (!hasCopy()) {
            return;
        }
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            *reinterpret_cast<u32x4*>(to + (i * kTeam + static_cast<int>(threadIdx.x) % kTeam) * 16) = held[i];
        }
    }

    // Where the calling lane's fragments begin within a tile: what follows from the lane alone, so that a tile's reads
    // differ by constants (turn() has the period of 16 rows).
    struct Lane {
        std::uint32_t plain[kSteps];
        std::uint32_t turned[kDim / 16][sizeof(T) == 2 ? 1 : 4];

        __device__ __forceinline__ Lane() {
            const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
            const int i = lane & 15;
            const int h = lane >> 4;
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                plain[t] = static_cast<std::uint32_t>(i * kRowBytes + 16 * ((4 * t + h) ^ turn(i)));
            }
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) {
                if constexpr (sizeof(T) == 2) {
                    const int row = 4 * h + (i >> 2);
                    const int chunk = 2 * d + ((i & 3) >> 1);
                    turned[d][0] = static_cast<std::uint32_t>(row * kRowBytes + 16 * (chunk ^ turn(row)) + 8 * (i & 1));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 4 * h + e;
                        turned[d][e] = static_cast<std::uint32_t>(row * kRowBytes + 16 * ((4 * d + (i >> 2)) ^ turn(row)) + 4 * (i & 3));
                    }
                }
            }
        }
    };

    // The calling lane's fragment of rows 16 block .. + 15, values of step t along the row. `tile`: an LDS address.
    static __device__ __forceinline__ typename Fragment<T>::type read(std::uint32_t tile, const Lane& lane, int block, int t) {
        typedef const __attribute__((address_space(3))) typename Fragment<T>::type* LdsPointer;
        return *reinterpret_cast<LdsPointer>(tile + lane.plain[t] + 16 * block * kRowBytes);
    }
    // The calling lane's fragment of columns 16 block .. + 15, contracted over rows: of lane group h the rows 4 h + e of
    // row block `pair` (float32), or of the row blocks 2 pair and 2 pair + 1 (16-bit): the rows whose products a lane
    // holds in its results, so that these are the other operand as they are.
    static __device__ __forceinline__ typename Fragment<T>::type readTurned(std::uint32_t tile, const Lane& lane, int block,
                                                                            int pair) {
        if constexpr (sizeof(T) == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* LdsPointer;
            const std::uint32_t low = tile + lane.turned[block][0] + 32 * pair * kRowBytes;
            const s16x4 first = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsPointer>(low));
            const s16x4 second = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsPointer>(low + 16 * kRowBytes));
            return __builtin_bit_cast(typename Fragment<T>::type,
                                      __builtin_shufflevector(first, second, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            typedef const __attribute__((address_space(3))) float* LdsPointer;
            typename Fragment<T>::type v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = *reinterpret_cast<LdsPointer>(tile + lane.turned[block][e] + 16 * pair * kRowBytes);
            }
            return v;
        }
    }
};

// Row blocks that one turned fragment contracts over.
template <typename T>
constexpr int kBlocksTurned = sizeof(T) == 2 ? 2 : 1;

// The largest of a lane's value over the four lanes of its row (NaN where one is).
__device__ __forceinline__ float overGroups(float value) {
    const auto pairs = __builtin_amdgcn_permlane16_swap(__float_as_uint(value), __float_as_uint(value), false, false);
    value = __builtin_elementwise_maximum(__uint_as_float(pairs[0]), __uint_as_float(pairs[1]));
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(value), __float_as_uint(value), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}

// Asks the scheduler for kReads LDS reads, each with kEach matrix instructions, in an order that keeps four reads ahead:
// left to itself it reads late and waits for every read.
template <int kReads, int kEach>
__device__ __forceinline__ void scheduleProducts() {
    constexpr int kAhead = kReads < 4 ? kReads : 4;
    constexpr int kMatrix = 0x8, kLdsRead = 0x100;
    __builtin_amdgcn_sched_group_barrier(kLdsRead, kAhead, 0);
#pragma unroll
    for (int i = 0; i < kReads - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMatrix, kEach, 0);
        __builtin_amdgcn_sched_group_barrier(kLdsRead, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMatrix, kAhead * kEach, 0);
}

// A lane's results for kBlocksTurned row blocks as the other operand of that contraction, rounded to T.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::type resultFragment(const f32x4* blocks) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_convertvector(__builtin_shufflevector(blocks[0], blocks[1], 0, 1, 2, 3, 4, 5, 6, 7),
                                       typename Fragment<T>::type);
    } else {
        return blocks[0];
    }
}

// Tiles that a team of threads (a workgroup, or a wavefront of its own) works through: the next one's copies are on their
// way while this one is used.
template <int kTeam>
__device__ __forceinline__ void teamSync() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if constexpr (kTeam > kWave) {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
}

// A head's values of the distance bias in LDS: `margin` copies of the end values on either side, times `factor`. Values of
// -1e30 and less are minus infinity, and stay so.
template <typename T>
__device__ __forceinline__ float biasValue(T value, float factor) {
    const float bias = static_cast<float>(value);
    return bias <= -1.0e30f ? -INFINITY : factor * bias;
}

// How scores follow from the raw products. Without a cap, biases are where the products' sums begin (divided by scale, so
// that one factor brings all to base 2); with a cap, or a scale too small to divide by, they are added to formed scores.
struct ScoreForm {
    bool capped;
    bool fine;           // the cap is too large for tangents that are off by 2^-21
    bool formed;         // scores in base 2 are formed before the biases
    float factor;        // log2(e) |scale| (the queries, or keys, carry scale's sign)
    float bias_factor;   // of the table's values and the slopes
    float cap;           // log2(e) cap
    float to_cap;        // |scale| / cap (16-bit operands: times 2 log2(e))

    __device__ __forceinline__ ScoreForm(const AttentionArgs& args, bool base_two) {
        capped = args.cap > 0.0f;
        // Up to 64 a score is off by 2^-15, and its exponential by that of itself: 1/16 of what float16 rounds off it.
        // 128 texts of 64 to 1024 bfloat16 under a cap of 30: 362 us, 452 with fine tangents; their gradient 466 and 521.
        fine = args.cap > 64.0f;
        // Larger caps only bend scores whose softmax is 0 or 1 in any case; up to this one, what follows stays finite.
        const float largest = fminf(args.cap, 0x1p96f);
        const float scale = fabsf(args.scale);
        formed = capped || scale < 0x1p-20f;
        factor = kLog2E * scale;
        bias_factor = formed ? kLog2E : 1.0f / scale;
        cap = kLog2E * largest;
        // (finite, so that a score of zero stays one under the smallest caps)
        to_cap = capped ? fminf((base_two ? 2.0f * kLog2E : 1.0f) * scale / largest, FLT_MAX) : 0.0f;
    }
};

// The hyperbolic tangent of a raw product times form.to_cap.
// 16-bit: of y, in base 2 and doubled, the quotient is off by up to 2^-21, and the score by that of the cap. kFine: within
// 2^-20 of its value instead, by an odd polynomial where tangents are small: fitted to tanh(y / (2 log2(e))) / y on |y| < 1,
// to 2^-24 of it.
template <typename T, bool kFine>
__device__ __forceinline__ float tanhOf(float y) {
    if constexpr (sizeof(T) == 2) {
        const float wide = fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y)), 1.0f);
        if constexpr (!kFine) {
            return wide;
        }
        const float w = y * y;
        const float narrow = y * fmaf(fmaf(fmaf(-2.94580081e-5f, w, 6.64870524e-4f), w, -1.38756690e-2f), w, 3.46573579e-1f);
        return fabsf(y) < 1.0f ? narrow : wide;
    } else {
        return tanhf(y);
    }
}

// Calls body(whether tangents are formed as kFine).
template <typename T, typename Body>
__device__ __forceinline__ void withTanh(const ScoreForm& form, Body&& body) {
    if (sizeof(T) == 2 && form.fine) {
        asm volatile("");  // stays a branch
        body(std::true_type{});
    } else {
        asm volatile("");  // stays a branch
        body(std::false_type{});
    }
}

}  // namespace
}  // namespace zcgvs_hip
