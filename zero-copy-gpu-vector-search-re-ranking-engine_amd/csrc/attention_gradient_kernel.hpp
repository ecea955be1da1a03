// The gradient of attention over packed texts.
//
//     delta = dout . out (a row),  p = exp(s - lse),  dp = dout v^T,  ds = p (dp - delta)
//     dbias = sums of ds along the diagonals,  dr = ds (1 - (c / cap)^2)
//     dq = scale dr k,  dk = scale dr^T q,  dv = p^T dout
//
// Two launches (one more each with the bias's gradient and with few keys), no atomics between workgroups: the same bits on
// every call.
// 1. dq: a wavefront keeps 16 or 32 query rows and goes through the keys, as the forward kernel does. Before, it forms delta
//    and the rows' lse in base 2, for itself and the second launch (in a launch of their own 16 us more than the 378 below).
// 2. dk and dv: a wavefront keeps 16 or 32 keys and their values in registers and goes through the queries of all heads of
//    its key head, in LDS tiles of 32 rows that the workgroup shares. Scores come out with a lane's four neighbouring query
//    rows of one key, which is how the products over the rows take p and dr: they stay in registers.
//    Where that leaves CUs idle, the query heads are split over workgroups and one more launch adds the parts.
// So p is formed twice: seven products instead of five, for sums in one order and no float32 copy of dq.
// The bias's gradient: a wavefront adds its tile up along the diagonals by moving rows along the lanes, and every lane
// group adds the result to a table of its own in LDS (its 16 lanes always meet 16 different distances, so the order of
// additions is the program's), with room for distances past the table's ends; tiles that lie past them altogether add
// to two registers. A workgroup joins its tables and writes
// one of partial sums a head, which the last launch adds in the order of the workgroups.
// 16-bit p and dr are rounded for the products over them, whose matrix instructions take 16-bit operands; the bias's gradient
// is the sum of the unrounded ds.
// Bound by waits: wavefronts, about two of them on a SIMD, stand half of their time at tiles whose copies were started one tile
// before. Counted for the 128 texts below, of all SIMD cycles: keys 36% vector and 14% matrix instructions, 1.6 wavefronts a SIMD;
// queries 46%, 19% and 2.3. Measured, bfloat16: 128 texts of 64 to 512, 12 heads of 64, a learned bias and its gradient 378-380 us
// (queries 149, keys 253 under the profiler), without a bias 321, float32 1963; 8 texts of 4096, 8 heads of 64 on 2 1046 us,
// of 128 2070. 3 texts of 20 to 77 float32, 6 heads of 32 on 2 23.5-24.5 us (the launches).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention.hpp"
#include "column_sums.hpp"
#include "matrix_plan.hpp"

namespace zcgvs_hip {
namespace {

constexpr int kGradientWaves = 4;
constexpr int kGradientThreads = kGradientWaves * kWave;
constexpr int kQueryTile = 32;

static __device__ const float no_row[2] = {INFINITY, 0.0f};  // p = 0

// ---- shared by both kernels ----------------------------------------------------------------------

// Raw products -> formed scores in base 2 before the biases; the tangent's square to `bent`.
template <typename T, int kCount>
__device__ __forceinline__ void formScores(const ScoreForm& form, f32x4 (&s)[kCount], f32x4 (&bent)[kCount]) {
    if (form.capped) {
        withTanh<T>(form, [&](auto fine) {
#pragma unroll
            for (int b = 0; b < kCount; ++b) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = tanhOf<T, decltype(fine)::value>(s[b][e] * form.to_cap);
                    bent[b][e] = t * t;
                    s[b][e] = form.cap * t;
                }
            }
        });
    } else {
        asm volatile("");  // stays a branch
#pragma unroll
        for (int b = 0; b < kCount; ++b) {
            s[b] *= form.factor;
        }
    }
}

// The table of a head with `margin` copies of its end values on either side.
template <typename T>
__device__ __forceinline__ void loadTable(const AttentionArgs& args, int head, int margin, float factor, float* table) {
    const int width = 2 * (args.max_distance + margin) + 1;
    const T* from = static_cast<const T*>(args.table) + static_cast<std::int64_t>(head) * (2 * args.max_distance + 1);
    for (int i = static_cast<int>(threadIdx.x); i < width; i += kGradientThreads) {
        table[i] = biasValue(from[min(max(i - margin, 0), 2 * args.max_distance)], factor);
    }
}

// ---- dk, dv and the bias's partial sums ----------------------------------------------------------

// The value of the lane kBy lanes after (before) within a group of 16, zero past its end.
template <int kBy>
__device__ __forceinline__ float fromLaneAfter(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x100 + kBy, 0xF, 0xF, true));
}
template <int kBy>
__device__ __forceinline__ float fromLaneBefore(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x110 + kBy, 0xF, 0xF, true));
}

// Wavefronts of a SIMD that the registers do for; the bound also keeps sums out of the accumulation registers.
// (The largest tables leave LDS for one workgroup.)
template <typename T, int kDim, int kBlocks, int kFar>
constexpr int kKeyResident = kBlocks * kDim * static_cast<int>(sizeof(T)) <= 256 && kFar <= 128 ? 2 : 1;
template <typename T, int kDim, int kBlocks>
constexpr int kQueryResident = kBlocks * kDim * static_cast<int>(sizeof(T)) <= 512 ? 2 : 1;

// kFar: the largest max_distance whose gradient is wanted (0: none).
template <typename T, int kDim, int kBlocks, bool kDirect, int kFar>
__global__ __launch_bounds__(kGradientThreads, (kKeyResident<T, kDim, kBlocks, kFar>)) void keyGradientKernel(AttentionArgs args, AttentionGradient more) {
    using Rows = RowTile<T, kQueryTile, kDim, kGradientThreads, kDirect>;
    constexpr int kWaveKeys = 16 * kBlocks;
    constexpr int kKeys = kWaveKeys * kGradientWaves;
    constexpr int kStageBytes = 2 * Rows::kBytes;  // queries, then the output's gradient
    constexpr int kDimBlocks = kDim / 16;
    constexpr int kRowBlocks = kQueryTile / 16;
    constexpr int kTurned = kBlocksTurned<T>;
    constexpr int kMargin = kQueryTile + kWaveKeys + 16;
    // the four groups of a wavefront add to 64 different banks
    constexpr int kBins = kFar > 0 ? (2 * (kFar + kMargin) + 1 + 43) / 64 * 64 + 20 : 1;
    static_assert(kFar == 0 || (kBins % 64 == 20 && kBins >= 2 * (kFar + kMargin) + 1), "a table holds its distances");
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[2 * kStageBytes];
    __shared__ __attribute__((aligned(256))) float stats[2][kQueryTile][2];
    __shared__ float table[2 * (kAttentionMaxDistance + kMargin) + 1];
    __shared__ float bins[kFar > 0 ? kGradientWaves * 4 : 1][kBins];
    __shared__ float past_ends[2];

    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int r16 = lane & 15;
    const int h = lane >> 4;
    const int position = positionOf(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
    const int slot = position % more.key_slots;
    const int key_heads = args.heads / args.group;
    const int key_head = position / more.key_slots % key_heads;
    const int part = position / more.key_slots / key_heads;
    const int first_head = part * args.group / more.key_parts;  // of the part, within the key head's
    const int end_head = (part + 1) * args.group / more.key_parts;
    const int table_columns = 2 * args.max_distance + 1;
    auto partialTable = [&](int head) {
        return more.table_partials + (static_cast<std::int64_t>(head) * more.key_slots + slot) * table_columns;
    };
    const int text = textOfSlot<kKeys>(args.k_texts, 1, slot);
    TextSpan keys{0, 0, 0};
    int tile_key = 0;
    if (text >= 0) {
        keys = textSpan(args.k_texts, text);
        tile_key = (slot - (static_cast<int>(keys.first / kKeys) + text)) * kKeys;
    }
    if (text < 0 || tile_key < 0 || tile_key >= keys.rows) {
        if constexpr (kFar > 0) {
            for (int g = first_head; g < end_head; ++g) {
                for (int i = static_cast<int>(threadIdx.x); i < table_columns; i += kGradientThreads) {
                    partialTable(key_head * args.group + g)[i] = 0.0f;
                }
            }
        }
        return;
    }
    const TextSpan queries = textSpan(args.q_texts, text);
    const int prefix = args.prefix == nullptr ? 0 : args.prefix[text];
    const int shift = args.q_last ? keys.count - queries.count : 0;
    const ScoreForm form(args, sizeof(T) == 2);

    const int wave_key = tile_key + wave * kWaveKeys;
    int key[kBlocks], seen_from[kBlocks];
    bool valid[kBlocks];
    const bool whole_chunks = args.head_dim % kChunk<T> == 0;
    typename Fragment<T>::type k[kBlocks][Rows::kSteps], v[kBlocks][Rows::kSteps];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
        key[n] = wave_key + 16 * n + r16;
        valid[n] = key[n] < keys.count;
        seen_from[n] = !args.causal || key[n] < prefix ? INT32_MIN / 2 : key[n];
        const std::int64_t row = keys.first + key[n];
        const int width = valid[n] ? args.head_dim : 0;
        loadRowFragments(static_cast<const T*>(args.k) + row * args.k_stride + key_head * args.head_dim, width, whole_chunks, k[n]);
        loadRowFragments(static_cast<const T*>(args.v) + row * args.v_stride + key_head * args.head_dim, width, whole_chunks, v[n]);
    }
    if (args.scale < 0.0f) {
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
            for (int t = 0; t < Rows::kSteps; ++t) {
                k[n][t] = -k[n][t];
            }
        }
    }
    // they have arrived before the loop: a wait within it would be one for the next tile too
    __builtin_amdgcn_s_waitcnt(vmcntOnly(0));
    f32x4 dk[kBlocks][kDimBlocks], dv[kBlocks][kDimBlocks];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) {
            dk[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            dv[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    const typename Rows::Lane own_lane;
    // query rows from the first that sees one of the workgroup's keys on
    const int query_begin = args.causal && tile_key >= prefix ? max(tile_key - shift, 0) : 0;
    const bool any_key = wave_key < keys.count;
    const int last_key = min(wave_key + kWaveKeys, keys.count) - 1;
    const bool hidden_keys = args.causal && last_key >= prefix;  // some key of the wavefront is not seen by all

    for (int g = first_head; g < end_head; ++g) {
        const int head = key_head * args.group + g;
        const float slope = args.slopes != nullptr ? form.bias_factor * args.slopes[head] : 0.0f;
        float past[2] = {};  // sums of ds at distances past the table's ends: before, behind
        __syncthreads();              // the tables and tiles of the head before have been used
        if (args.table != nullptr) {
            loadTable<T>(args, head, kMargin, form.bias_factor, table);
        }
        if constexpr (kFar > 0) {
            for (int i = static_cast<int>(threadIdx.x); i < kGradientWaves * 4 * kBins; i += kGradientThreads) {
                (&bins[0][0])[i] = 0.0f;
            }
        }
        const std::int64_t first = queries.first + query_begin;
        Rows q_tile, d_tile;
        q_tile.begin(static_cast<const T*>(args.q) + first * args.q_stride + head * args.head_dim, args.q_stride,
                     queries.count - query_begin, args.head_dim, 1);
        d_tile.begin(static_cast<const T*>(more.out_gradient) + first * more.out_gradient_stride + head * args.head_dim,
                     more.out_gradient_stride, queries.count - query_begin, args.head_dim, 1);
        const float* head_stats = more.stats + 2 * (head * args.q_texts.total + queries.first);
        auto issueStats = [&](int row0, int buffer) {
            // a dword for each lane of the first wavefront
            if (wave == 0) {
                const int row = row0 + (lane >> 1);
                const float* from = row < queries.count ? head_stats + 2 * row + (lane & 1) : no_row + (lane & 1);
                copyDwordToLds(from, __builtin_amdgcn_readfirstlane(ldsAddress(&stats[buffer][0][0])));
            }
        };
        if (query_begin < queries.count) {
            issueStats(query_begin, 0);
            if constexpr (kDirect) {
                q_tile.issue(lds, 1);
                d_tile.issue(lds + Rows::kBytes, 1);
            } else {
                q_tile.fetch(1);
                d_tile.fetch(1);
                q_tile.put(lds);
                d_tile.put(lds + Rows::kBytes);
            }
        }
        int buffer = 0;
        for (int row0 = query_begin; row0 < queries.count; row0 += kQueryTile) {
            teamSync<kGradientThreads>();
            const std::uint32_t q_stage = ldsAddress(lds) + buffer * kStageBytes;
            const std::uint32_t d_stage = q_stage + Rows::kBytes;
            const float* row_stats = &stats[buffer][0][0];
            buffer ^= 1;
            const bool next = row0 + kQueryTile < queries.count;
            std::uint8_t* other = lds + buffer * kStageBytes;
            if (next) {
                issueStats(row0 + kQueryTile, buffer);
                if constexpr (kDirect) {
                    q_tile.issue(other, 1);
                    d_tile.issue(other + Rows::kBytes, 1);
                } else {
                    q_tile.fetch(1);
                    d_tile.fetch(1);
                }
            }
            const int place0 = row0 + shift;  // of the tile's first row
            if (any_key && !(hidden_keys && wave_key >= prefix && place0 + kQueryTile - 1 < wave_key)) {
                float score_factor = form.factor, score_offset = 0.0f;
                const bool before = wave_key + kWaveKeys - 1 - place0 <= -args.max_distance;
                const bool behind = wave_key - (place0 + kQueryTile - 1) >= args.max_distance;
                const bool in_table = args.table != nullptr && !before && !behind;
                f32x4 s[kBlocks][kRowBlocks], dp[kBlocks][kRowBlocks], bent[kBlocks][kRowBlocks];
                auto loadBiases = [&](f32x4(&to)[kBlocks][kRowBlocks]) {
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) {
                        const float* from = table + key[n] - place0 - 4 * h + args.max_distance + kMargin;
#pragma unroll
                        for (int m = 0; m < kRowBlocks; ++m) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                to[n][m][e] = from[-(16 * m + e)];
                            }
                        }
                    }
                };
                auto addSlopes = [&](f32x4(&to)[kBlocks][kRowBlocks]) {
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) {
                        const float distance = static_cast<float>(key[n] - place0 - 4 * h);  // of the lane's first row
#pragma unroll
                        for (int m = 0; m < kRowBlocks; ++m) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                to[n][m][e] = fmaf(-slope, fabsf(distance - static_cast<float>(16 * m + e)), to[n][m][e]);
                            }
                        }
                    }
                };
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                    for (int m = 0; m < kRowBlocks; ++m) {
                        s[n][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        dp[n][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    }
                }
                if (in_table && !form.formed) {
                    loadBiases(s);
                }
                if (args.slopes != nullptr && !form.formed) {
                    addSlopes(s);
                }
#pragma unroll
                for (int m = 0; m < kRowBlocks; ++m) {
#pragma unroll
                    for (int t = 0; t < Rows::kSteps; ++t) {
                        const auto q = Rows::read(q_stage, own_lane, m, t);
                        const auto d = Rows::read(d_stage, own_lane, m, t);
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
                            s[n][m] = multiplyAdd(q, k[n][t], s[n][m]);
                            dp[n][m] = multiplyAdd(d, v[n][t], dp[n][m]);
                        }
                    }
                }
                if (form.formed) {
                    asm volatile("");  // stays a branch
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) {
                        formScores<T>(form, s[n], bent[n]);
                    }
                    score_factor = 1.0f;
                    if (in_table) {
                        f32x4 bias[kBlocks][kRowBlocks];
                        loadBiases(bias);
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                            for (int m = 0; m < kRowBlocks; ++m) {
                                s[n][m] += bias[n][m];
                            }
                        }
                    }
                    if (args.slopes != nullptr) {
                        addSlopes(s);
                    }
                }
                if (args.table != nullptr && !in_table) {
                    score_offset = score_factor * table[before ? 0 : 2 * (args.max_distance + kMargin)];
                }
#pragma unroll
                for (int m = 0; m < kRowBlocks; ++m) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float off = score_offset - row_stats[2 * (16 * m + 4 * h + e)];
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
                            s[n][m][e] = __builtin_amdgcn_exp2f(fmaf(s[n][m][e], score_factor, off));
                        }
                    }
                }
                if (hidden_keys && place0 < last_key) {
                    asm volatile("");  // stays a branch
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) {
                        const int seen = seen_from[n] - place0 - 4 * h;
#pragma unroll
                        for (int m = 0; m < kRowBlocks; ++m) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                s[n][m][e] = 16 * m + e >= seen ? s[n][m][e] : 0.0f;
                            }
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < kRowBlocks; ++m) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float delta = row_stats[2 * (16 * m + 4 * h + e) + 1];
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
                            dp[n][m][e] = s[n][m][e] * (dp[n][m][e] - delta);
                        }
                    }
                }
                if constexpr (kFar > 0) {
                    if (wave_key + kWaveKeys > keys.count) {
                        // keys past the text's end have zeros as their operands, and scores
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                            for (int m = 0; m < kRowBlocks; ++m) {
                                dp[n][m] = valid[n] ? dp[n][m] : f32x4{};
                            }
                        }
                    }
                    if (before || behind) {
                        float sum = 0.0f;
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                            for (int m = 0; m < kRowBlocks; ++m) {
                                sum += (dp[n][m][0] + dp[n][m][1]) + (dp[n][m][2] + dp[n][m][3]);
                            }
                        }
                        past[0] += before ? sum : 0.0f;
                        past[1] += before ? 0.0f : sum;
                    } else {
                        // Row e of a lane's four moved e lanes along: lane x then holds distance x - 4 h, and what moved
                        // past the group's end the distance 16 less. Blocks on one diagonal add up before they go to
                        // the table.
                        float along[kBlocks + kRowBlocks] = {};  // at distances 16 (i - kRowBlocks) more
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                            for (int m = 0; m < kRowBlocks; ++m) {
                                float& here = along[n - m + kRowBlocks];
                                float& less = along[n - m + kRowBlocks - 1];
                                here += dp[n][m][0];
                                here += fromLaneAfter<1>(dp[n][m][1]);
                                here += fromLaneAfter<2>(dp[n][m][2]);
                                here += fromLaneAfter<3>(dp[n][m][3]);
                                less += fromLaneBefore<15>(dp[n][m][1]);
                                less += fromLaneBefore<14>(dp[n][m][2]);
                                less += fromLaneBefore<13>(dp[n][m][3]);
                            }
                        }
                        float* own = &bins[wave * 4 + h][0] + wave_key + r16 - place0 - 4 * h + args.max_distance + kMargin;
                        // (no two lanes of a group, nor two diagonals, meet; LDS additions as one instruction took
                        // 128 cycles each)
                        float held[kBlocks + kRowBlocks];
#pragma unroll
                        for (int i = 0; i < kBlocks + kRowBlocks; ++i) {
                            held[i] = own[16 * (i - kRowBlocks)];
                        }
#pragma unroll
                        for (int i = 0; i < kBlocks + kRowBlocks; ++i) {
                            own[16 * (i - kRowBlocks)] = held[i] + along[i];
                        }
                    }
                }
                if (form.capped) {
                    asm volatile("");  // stays a branch
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                        for (int m = 0; m < kRowBlocks; ++m) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                dp[n][m][e] = fmaf(-dp[n][m][e], bent[n][m][e], dp[n][m][e]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int pair = 0; pair < kRowBlocks / kTurned; ++pair) {
                    typename Fragment<T>::type p[kBlocks], dr[kBlocks];
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) {
                        p[n] = resultFragment<T>(&s[n][pair * kTurned]);
                        dr[n] = resultFragment<T>(&dp[n][pair * kTurned]);
                    }
#pragma unroll
                    for (int d = 0; d < kDimBlocks; ++d) {
                        const auto dout = Rows::readTurned(d_stage, own_lane, d, pair);
                        const auto q = Rows::readTurned(q_stage, own_lane, d, pair);
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
                            dv[n][d] = multiplyAdd(dout, p[n], dv[n][d]);
                            dk[n][d] = multiplyAdd(q, dr[n], dk[n][d]);
                        }
                    }
                }
            }
            if constexpr (!kDirect) {
                if (next) {
                    q_tile.put(other);
                    d_tile.put(other + Rows::kBytes);
                }
            }
        }
        if constexpr (kFar > 0) {
            // the lanes' sums past the ends: over the wavefront, then to the ends of its first group's table
            float ends[2];
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                ends[side] = past[side];
#pragma unroll
                for (int offset = kWave / 2; offset > 0; offset >>= 1) {
                    ends[side] += waveXor(ends[side], offset);
                }
            }
            // (without a tile of rows the sums are zeros, and no barrier stands behind the tables' clearing yet)
            if (lane == 0 && query_begin < queries.count) {
                bins[wave * 4][kMargin] += ends[0];
                bins[wave * 4][2 * args.max_distance + kMargin] += ends[1];
            }
            __syncthreads();
            // the groups' tables one after the other, then what lies past either end by a wavefront
            const int width = table_columns + 2 * kMargin;
            for (int i = static_cast<int>(threadIdx.x); i < width; i += kGradientThreads) {
                float sum = bins[0][i];
#pragma unroll
                for (int w = 1; w < kGradientWaves * 4; ++w) {
                    sum += bins[w][i];
                }
                bins[0][i] = sum;
            }
            __syncthreads();
            if (wave < 2) {
                const int from = wave == 0 ? 0 : width - kMargin;
                float sum = 0.0f;
                for (int i = lane; i < kMargin; i += kWave) {
                    sum += bins[0][from + i];
                }
#pragma unroll
                for (int offset = kWave / 2; offset > 0; offset >>= 1) {
                    sum += waveXor(sum, offset);
                }
                if (lane == 0) {
                    // (one bin holds both ends where the table has one value)
                    past_ends[wave] = sum;
                }
            }
            __syncthreads();
            float* to = partialTable(head);
            for (int i = static_cast<int>(threadIdx.x); i < table_columns; i += kGradientThreads) {
                float sum = bins[0][kMargin + i];
                sum += i == 0 ? past_ends[0] : 0.0f;
                sum += i == table_columns - 1 ? past_ends[1] : 0.0f;
                to[i] = sum;
            }
        }
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
        if (key[n] >= keys.rows) {
            continue;
        }
        const std::int64_t row = keys.first + key[n];
        if (more.key_parts > 1) {
            const std::int64_t width = static_cast<std::int64_t>(key_heads) * args.head_dim;
            float* to = more.key_partials + (part * args.k_texts.total + row) * width + key_head * args.head_dim;
            const std::int64_t values_on = more.key_parts * args.k_texts.total * width;
#pragma unroll
            for (int d = 0; d < kDimBlocks; ++d) {
                const int column = 16 * d + 4 * h;
                if (column < args.head_dim) {
                    storeFour(valid[n] ? dk[n][d] * args.scale : f32x4{}, to + column, args.head_dim - column);
                    storeFour(valid[n] ? dv[n][d] : f32x4{}, to + values_on + column, args.head_dim - column);
                }
            }
            continue;
        }
        T* k_to = static_cast<T*>(more.k_gradient) + row * more.k_gradient_stride + key_head * args.head_dim;
        T* v_to = static_cast<T*>(more.v_gradient) + row * more.v_gradient_stride + key_head * args.head_dim;
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) {
            const int column = 16 * d + 4 * h;
            if (column < args.head_dim) {
                storeFour(valid[n] ? dk[n][d] * args.scale : f32x4{}, k_to + column, args.head_dim - column);
                storeFour(valid[n] ? dv[n][d] : f32x4{}, v_to + column, args.head_dim - column);
            }
        }
    }
}

// dk and dv from the parts of their query heads, in their order; rows of no text are left as they are.
template <typename T>
__global__ __launch_bounds__(kGradientThreads) void joinKeyPartsKernel(AttentionArgs args, AttentionGradient more) {
    const int width = args.heads / args.group * args.head_dim;
    const int packs = (width + 3) / 4;
    const std::int64_t first = textStart(args.k_texts, 0), end = textStart(args.k_texts, args.k_texts.texts);
    const std::int64_t part_values = args.k_texts.total * width;
    const bool values = blockIdx.y == 1;
    const float* partials = more.key_partials + (values ? more.key_parts * part_values : 0);
    T* out = static_cast<T*>(values ? more.v_gradient : more.k_gradient);
    const std::int64_t stride = values ? more.v_gradient_stride : more.k_gradient_stride;
    for (std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * kGradientThreads + threadIdx.x; i < (end - first) * packs;
         i += static_cast<std::int64_t>(gridDim.x) * kGradientThreads) {
        const std::int64_t row = first + i / packs;
        const int column = 4 * static_cast<int>(i % packs);
        const float* from = partials + row * width + column;
        f32x4 sum = loadFour(from, width - column);
#pragma unroll 4
        for (int p = 1; p < more.key_parts; ++p) {
            sum += loadFour(from + p * part_values, width - column);
        }
        storeFour(sum, out + row * stride + column, width - column);
    }
}

// ---- dq ------------------------------------------------------------------------------------------

template <typename T, int kDim, int kBlocks, bool kDirect>
__global__ __launch_bounds__(kGradientThreads, (kQueryResident<T, kDim, kBlocks>)) void queryGradientKernel(AttentionArgs args, AttentionGradient more) {
    constexpr int kTileKeys = sizeof(T) == 2 ? 64 : 32;
    using Keys = RowTile<T, kTileKeys, kDim, kGradientThreads, kDirect>;
    constexpr int kWaveRows = 16 * kBlocks;
    constexpr int kRows = kWaveRows * kGradientWaves;
    constexpr int kStageBytes = 2 * Keys::kBytes;  // keys, then values
    constexpr int kDimBlocks = kDim / 16;
    constexpr int kTurned = kBlocksTurned<T>;
    constexpr int kMargin = kTileKeys + kWaveRows;
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[2 * kStageBytes];
    __shared__ float table[2 * (kAttentionMaxDistance + kMargin) + 1];

    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int r16 = lane & 15;
    const int h = lane >> 4;
    const int position = positionOf(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
    const int slot = position % more.query_slots;
    const int head = position / more.query_slots;
    const int key_head = head / args.group;
    const int text = textOfSlot<kRows>(args.q_texts, 1, slot);
    if (text < 0) {
        return;
    }
    const TextSpan queries = textSpan(args.q_texts, text);
    const int tile_row = (slot - (static_cast<int>(queries.first / kRows) + text)) * kRows;
    if (tile_row < 0 || tile_row >= queries.rows) {
        return;
    }
    const TextSpan keys = textSpan(args.k_texts, text);
    const int prefix = args.prefix == nullptr ? 0 : args.prefix[text];
    const int shift = args.q_last ? keys.count - queries.count : 0;
    auto limitAt = [&](int at) { return args.causal ? min(keys.count, max(max(at + 1, prefix), 0)) : keys.count; };
    const ScoreForm form(args, sizeof(T) == 2);
    const float slope = args.slopes != nullptr ? form.bias_factor * args.slopes[head] : 0.0f;

    const int wave_row = tile_row + wave * kWaveRows;
    const bool whole_chunks = args.head_dim % kChunk<T> == 0;
    int place[kBlocks], limit[kBlocks];
    float lse[kBlocks], delta[kBlocks];
    typename Fragment<T>::type q[kBlocks][Keys::kSteps], dout[kBlocks][Keys::kSteps], out[kBlocks][Keys::kSteps];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        const int i = wave_row + 16 * m + r16;
        const bool valid = i < queries.count;
        const std::int64_t row = queries.first + i;
        place[m] = i + shift;
        limit[m] = valid ? limitAt(place[m]) : 0;
        const int width = valid ? args.head_dim : 0;
        lse[m] = valid ? more.lse[row * args.heads + head] : -INFINITY;
        loadRowFragments(static_cast<const T*>(more.out) + row * more.out_stride + head * args.head_dim, width, whole_chunks, out[m]);
        loadRowFragments(static_cast<const T*>(args.q) + row * args.q_stride + head * args.head_dim, width, whole_chunks, q[m]);
        loadRowFragments(static_cast<const T*>(more.out_gradient) + row * more.out_gradient_stride + head * args.head_dim, width,
                         whole_chunks, dout[m]);
    }
    if (args.scale < 0.0f) {
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
            for (int t = 0; t < Keys::kSteps; ++t) {
                q[m][t] = -q[m][t];
            }
        }
    }
    const int last_row = min(wave_row + kWaveRows, queries.count) - 1;
    const int first_place = wave_row + shift;
    const int last_place = last_row + shift;
    // a wavefront with rows that do not count has their limits of zero to mind
    const int least_limit = last_row - wave_row + 1 == kWaveRows ? limitAt(first_place) : 0;
    const int most_limit = last_row >= wave_row ? limitAt(last_place) : 0;
    const int tile_last = min(tile_row + kRows, queries.count) - 1;
    const int all_keys = tile_last >= tile_row ? limitAt(tile_last + shift) : 0;

    if (args.table != nullptr) {
        loadTable<T>(args, head, kMargin, form.bias_factor, table);
    }
    f32x4 dq[kBlocks][kDimBlocks];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) {
            dq[m][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    const typename Keys::Lane own_lane;
    Keys k_tile, v_tile;
    k_tile.begin(static_cast<const T*>(args.k) + keys.first * args.k_stride + key_head * args.head_dim, args.k_stride,
                 keys.count, args.head_dim, 1);
    v_tile.begin(static_cast<const T*>(args.v) + keys.first * args.v_stride + key_head * args.head_dim, args.v_stride,
                 keys.count, args.head_dim, 1);
    if (all_keys > 0) {
        if constexpr (kDirect) {
            k_tile.issue(lds, 1);
            v_tile.issue(lds + Keys::kBytes, 1);
        } else {
            k_tile.fetch(1);
            v_tile.fetch(1);
            k_tile.put(lds);
            v_tile.put(lds + Keys::kBytes);
        }
    }
    // delta, from the chunks of the row's four lanes, and lse in base 2, here and for the launch of the keys (a wait for the
    // rows within the loop would be one for the next tile too)
    __builtin_amdgcn_s_waitcnt(vmcntOnly(0));
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < Keys::kSteps; ++t) {
#pragma unroll
            for (int e = 0; e < kChunk<T>; ++e) {
                sum = fmaf(static_cast<float>(out[m][t][e]), static_cast<float>(dout[m][t][e]), sum);
            }
        }
        sum += waveXor(sum, 16);
        sum += waveXor(sum, 32);
        // a row that sees no key: p = 0
        const bool empty = lse[m] == -INFINITY;
        lse[m] = empty ? INFINITY : kLog2E * lse[m];
        delta[m] = empty ? 0.0f : sum;
        const int i = wave_row + 16 * m + r16;
        if (h == 0 && i < queries.count) {
            float* row_stats = more.stats + 2 * (head * args.q_texts.total + queries.first + i);
            row_stats[0] = lse[m];
            row_stats[1] = delta[m];
        }
    }
    int buffer = 0;
    for (int key0 = 0; key0 < all_keys; key0 += kTileKeys) {
        teamSync<kGradientThreads>();
        const std::uint32_t stage = ldsAddress(lds) + buffer * kStageBytes;
        const std::uint32_t values = stage + Keys::kBytes;
        buffer ^= 1;
        std::uint8_t* other = lds + buffer * kStageBytes;
        const bool next = key0 + kTileKeys < all_keys;
        if (next) {
            if constexpr (kDirect) {
                k_tile.issue(other, 1);
                v_tile.issue(other + Keys::kBytes, 1);
            } else {
                k_tile.fetch(1);
                v_tile.fetch(1);
            }
        }
#pragma unroll
        for (int pair = 0; pair < kTileKeys / 16 / kTurned; ++pair) {
            const int pair_key = key0 + pair * 16 * kTurned;
            if (pair_key >= most_limit) {
                continue;
            }
            float score_factor = form.factor, score_offset = 0.0f;
            const bool behind = pair_key - last_place >= args.max_distance;
            const bool before = pair_key + 16 * kTurned - 1 - first_place <= -args.max_distance;
            const bool in_table = args.table != nullptr && !before && !behind;
            f32x4 s[kBlocks][kTurned], dp[kBlocks][kTurned], bent[kBlocks][kTurned];
            auto loadBiases = [&](f32x4(&to)[kBlocks][kTurned]) {
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    // rows past the text's last one may reach beyond the margin
                    const float* from = table + max(pair_key + 4 * h - place[m] + args.max_distance + kMargin, 0);
#pragma unroll
                    for (int b = 0; b < kTurned; ++b) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            to[m][b][e] = from[16 * b + e];
                        }
                    }
                }
            };
            auto addSlopes = [&](f32x4(&to)[kBlocks][kTurned]) {
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    const float distance = static_cast<float>(pair_key + 4 * h - place[m]);
#pragma unroll
                    for (int b = 0; b < kTurned; ++b) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            to[m][b][e] = fmaf(-slope, fabsf(distance + static_cast<float>(16 * b + e)), to[m][b][e]);
                        }
                    }
                }
            };
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                for (int b = 0; b < kTurned; ++b) {
                    s[m][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    dp[m][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
            if (in_table && !form.formed) {
                loadBiases(s);
            }
            if (args.slopes != nullptr && !form.formed) {
                addSlopes(s);
            }
#pragma unroll
            for (int b = 0; b < kTurned; ++b) {
#pragma unroll
                for (int t = 0; t < Keys::kSteps; ++t) {
                    const auto k = Keys::read(stage, own_lane, pair * kTurned + b, t);
                    const auto v = Keys::read(values, own_lane, pair * kTurned + b, t);
#pragma unroll
                    for (int m = 0; m < kBlocks; ++m) {
                        s[m][b] = multiplyAdd(k, q[m][t], s[m][b]);
                        dp[m][b] = multiplyAdd(v, dout[m][t], dp[m][b]);
                    }
                }
            }
            if (form.formed) {
                asm volatile("");  // stays a branch
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    formScores<T>(form, s[m], bent[m]);
                }
                score_factor = 1.0f;
                if (in_table) {
                    f32x4 bias[kBlocks][kTurned];
                    loadBiases(bias);
#pragma unroll
                    for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                        for (int b = 0; b < kTurned; ++b) {
                            s[m][b] += bias[m][b];
                        }
                    }
                }
                if (args.slopes != nullptr) {
                    addSlopes(s);
                }
            }
            if (args.table != nullptr && !in_table) {
                score_offset = score_factor * table[before ? 0 : 2 * (args.max_distance + kMargin)];
            }
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const float off = score_offset - lse[m];
#pragma unroll
                for (int b = 0; b < kTurned; ++b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[m][b][e] = __builtin_amdgcn_exp2f(fmaf(s[m][b][e], score_factor, off));
                    }
                }
            }
            if (pair_key + 16 * kTurned > least_limit) {
                asm volatile("");  // stays a branch
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    const int left = limit[m] - pair_key - 4 * h;
#pragma unroll
                    for (int b = 0; b < kTurned; ++b) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[m][b][e] = 16 * b + e < left ? s[m][b][e] : 0.0f;
                        }
                    }
                }
            }
            typename Fragment<T>::type dr[kBlocks];
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                for (int b = 0; b < kTurned; ++b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        dp[m][b][e] = s[m][b][e] * (dp[m][b][e] - delta[m]);
                    }
                }
            }
            if (form.capped) {
                asm volatile("");  // stays a branch
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                    for (int b = 0; b < kTurned; ++b) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            dp[m][b][e] = fmaf(-dp[m][b][e], bent[m][b][e], dp[m][b][e]);
                        }
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                dr[m] = resultFragment<T>(dp[m]);
            }
#pragma unroll
            for (int d = 0; d < kDimBlocks; ++d) {
                const auto k = Keys::readTurned(stage, own_lane, d, pair);
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    dq[m][d] = multiplyAdd(k, dr[m], dq[m][d]);
                }
            }
        }
        if constexpr (!kDirect) {
            if (next) {
                k_tile.put(other);
                v_tile.put(other + Keys::kBytes);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        const int i = wave_row + 16 * m + r16;
        if (i >= queries.rows) {
            continue;
        }
        T* to = static_cast<T*>(more.q_gradient) + (queries.first + i) * more.q_gradient_stride + head * args.head_dim;
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) {
            const int column = 16 * d + 4 * h;
            if (column < args.head_dim) {
                storeFour(i < queries.count ? dq[m][d] * args.scale : f32x4{}, to + column, args.head_dim - column);
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------

template <typename T, int kDim, int kBlocks, bool kDirect>
int launchKeyGradient(const AttentionArgs& args, const AttentionGradient& more, hipStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(more.key_slots * (args.heads / args.group) * more.key_parts);
    if (more.table_partials == nullptr) {
        keyGradientKernel<T, kDim, kBlocks, kDirect, 0><<<blocks, kGradientThreads, 0, stream>>>(args, more);
    } else if (args.max_distance <= 128) {
        keyGradientKernel<T, kDim, kBlocks, kDirect, 128><<<blocks, kGradientThreads, 0, stream>>>(args, more);
    } else {
        keyGradientKernel<T, kDim, kBlocks, kDirect, kAttentionMaxDistance><<<blocks, kGradientThreads, 0, stream>>>(args, more);
    }
    ZCGVS_LAUNCH_CHECK("attention gradient");
    if (more.key_parts > 1) {
        const long long packs = args.k_texts.total * ((args.heads / args.group * args.head_dim + 3) / 4);
        const unsigned join_blocks = static_cast<unsigned>(std::min(4096ll, (packs + kGradientThreads - 1) / kGradientThreads));
        joinKeyPartsKernel<T><<<dim3(join_blocks, 2), kGradientThreads, 0, stream>>>(args, more);
        ZCGVS_LAUNCH_CHECK("attention gradient");
    }
    return ZCGVS_OK;
}

template <typename T, int kDim>
int launchGradientDim(const AttentionGradientPlan& plan, const AttentionArgs& args, const AttentionGradient& more,
                      hipStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(more.query_slots * args.heads);
    if (plan.query_blocks == 1) {
        if (plan.direct_keys) {
            queryGradientKernel<T, kDim, 1, true><<<blocks, kGradientThreads, 0, stream>>>(args, more);
        } else {
            queryGradientKernel<T, kDim, 1, false><<<blocks, kGradientThreads, 0, stream>>>(args, more);
        }
    } else if (plan.direct_keys) {
        queryGradientKernel<T, kDim, 2, true><<<blocks, kGradientThreads, 0, stream>>>(args, more);
    } else {
        queryGradientKernel<T, kDim, 2, false><<<blocks, kGradientThreads, 0, stream>>>(args, more);
    }
    ZCGVS_LAUNCH_CHECK("attention gradient");
    constexpr bool kTwo = sizeof(T) == 2 || kDim < 128;  // (as attention.hip plans)
    if constexpr (kTwo) {
        if (plan.key_blocks == 2) {
            return plan.direct_rows ? launchKeyGradient<T, kDim, 2, true>(args, more, stream)
                                    : launchKeyGradient<T, kDim, 2, false>(args, more, stream);
        }
    }
    return plan.direct_rows ? launchKeyGradient<T, kDim, 1, true>(args, more, stream)
                            : launchKeyGradient<T, kDim, 1, false>(args, more, stream);
}

// out [heads, columns] = the sums over the slots of partials [heads, slots, columns].
template <typename T>
__global__ __launch_bounds__(kColumnThreads) void joinTablesKernel(const float* __restrict__ partials, int slots, int columns,
                                                                   T* __restrict__ out) {
    joinColumns(partials + static_cast<std::int64_t>(blockIdx.y) * slots * columns, slots, columns,
                out + static_cast<std::int64_t>(blockIdx.y) * columns, static_cast<int>(blockIdx.x));
}

}  // namespace

template <typename T>
int launchAttentionGradient(const AttentionGradientPlan& plan, const AttentionArgs& args, const AttentionGradient& more,
                            hipStream_t stream) {
    int status;
    switch (paddedDim(args.head_dim)) {
        case 32:
            status = launchGradientDim<T, 32>(plan, args, more, stream);
            break;
        case 64:
            status = launchGradientDim<T, 64>(plan, args, more, stream);
            break;
        default:
            status = launchGradientDim<T, 128>(plan, args, more, stream);
            break;
    }
    if (status == ZCGVS_OK && more.table_partials != nullptr) {
        const int columns = 2 * args.max_distance + 1;
        joinTablesKernel<T><<<dim3(static_cast<unsigned>(divideUp(columns, kJoinColumns)), static_cast<unsigned>(args.heads)),
                              kColumnThreads, 0, stream>>>(more.table_partials, more.key_slots, columns,
                                                           static_cast<T*>(more.table_gradient));
        ZCGVS_LAUNCH_CHECK("attention gradient");
    }
    return status;
}

}  // namespace zcgvs_hip
