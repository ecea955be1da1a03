// Attention over packed texts, forward.
//
//     s = cap(scale q k^T) + bias(distance),  p = exp(s - max),  out = p v / sum p
//
// One pass over the keys: each wavefront keeps 16 or 32 query rows in registers (as the second operand of the
// matrix instructions) and, per row, the running maximum, the sum and the unfinished output. Scores come out of the
// matrix instruction with a lane's four neighbouring keys of one query row, which is also how the product with v takes
// them: the exponentials never leave their registers, and maximum, sum and rescaling are scalars of a lane. The
// maximum is only raised (and the output rescaled) when some row's scores exceed it by more than 8 in base 2, so that
// exponentials stay below 2^8 and most tiles rescale nothing.
// Tiles of 64 keys (float32: 32) and their values go to LDS by 16-byte copies, double buffered, one barrier a tile, read
// by the four wavefronts of a workgroup.
//
// Few query rows (the narrow shape): the rows are those of all heads of a key head, so that its keys are
// read once; the four wavefronts take every fourth tile each, from LDS of their own without a barrier, and the keys
// may be split over workgroups as well. The parts are joined by their maxima and sums.
//
// 16-bit exponentials are rounded for the product with v, since its matrix instructions take 16-bit operands (float32 ones have
// a sixteenth of their rate); their sum is that of the unrounded ones.
//
// Bound: by the vector units' issue up to heads of 64. Counted for heads of 64, SIMD cycles a score: over 8 texts of 4096 vector
// instructions 0.59 (76% of all cycles) and matrix instructions 0.25 of 0.77; over texts of 64 to 1024 with a learned bias 0.77
// (67%) and 0.27 of 1.15, wavefronts waiting a third of their time. The narrow shape by reading the keys once.
// Measured, bfloat16: 128 texts of 64 to 1024 tokens, 12 heads of 64, a learned bias 271-281 us (520-540 TFLOP/s of the pairs' four
// products' operations), without it 259, float32 1452; 8 texts of 4096, 8 heads of 64 346 us (790), of 80 and 96 (padded to 128)
// 541 and 550, of 128 580 (950), float32 of 64 2240. The last of 8193 rows, 16 heads of 128 on 4 float16 13.4 us (17 MB of keys,
// two launches).
#pragma once

#include <hip/hip_runtime.h>

#include "attention.hpp"
#include "matrix_plan.hpp"

namespace zcgvs_hip {
namespace {

constexpr int kAttentionWaves = 4;
constexpr int kAttentionThreads = kAttentionWaves * kWave;

template <typename T, int kDim, int kBlocks, bool kNarrow>
struct AttentionTile {
    static constexpr int kTileKeys = kNarrow ? narrowKeys(kDim, sizeof(T)) : sizeof(T) == 2 ? 64 : 32;
    static constexpr int kTeam = kNarrow ? kWave : kAttentionThreads;
    static constexpr int kWaveRows = 16 * kBlocks;
    static constexpr int kRows = kNarrow ? kWaveRows : kWaveRows * kAttentionWaves;
    static constexpr int kKeyBlocks = kTileKeys / 16;
    // distances past the table's ends that a tile which reaches into it can hold, on either side
    static constexpr int kMargin = kTileKeys + kWaveRows;
    static constexpr int kTableFloats = kNarrow ? kNarrowTable : biasTableWidth(kAttentionMaxDistance, kMargin);
    static_assert(!kNarrow || kWaveRows == kNarrowRows, "the margin that attention.hip plans with");
};

// Wavefronts of a SIMD: two, for which the registers of all but wide float32 rows do. The bound also keeps the sums in
// ordinary registers: with more of them to spend, tiles went through the accumulation registers and back
// (768 us for 128 texts of 64 to 1024 tokens, 12 heads of 64, that took 306 with the bound).
// The narrow shape's tiles of wide rows leave LDS for one workgroup.
template <typename T, int kDim, int kBlocks, bool kNarrow>
constexpr int kAttentionResident = kDim == 128 && (kNarrow || (sizeof(T) == 4 && kBlocks == 2)) ? 1 : 2;

template <typename T, int kDim, int kBlocks, bool kNarrow, bool kDirect>
__global__ __launch_bounds__(kAttentionThreads, (kAttentionResident<T, kDim, kBlocks, kNarrow>)) void attentionKernel(AttentionArgs args, AttentionOutput output) {
    using Tile = AttentionTile<T, kDim, kBlocks, kNarrow>;
    using Keys = RowTile<T, Tile::kTileKeys, kDim, Tile::kTeam, kDirect>;
    constexpr int kTeams = kNarrow ? kAttentionWaves : 1;
    constexpr int kStageBytes = 2 * Keys::kBytes;  // keys, then values
    constexpr int kJoinBytes = kNarrow ? kAttentionWaves * (kDim / 16 * kWave * 16 + 2 * 16 * 4) : 0;
    constexpr int kTileBytes = kTeams * 2 * kStageBytes;
    constexpr int kDimBlocks = kDim / 16;
    __shared__ __attribute__((aligned(256))) std::uint8_t lds[kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes];
    __shared__ float table[Tile::kTableFloats];

    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int r16 = lane & 15;
    const int h = lane >> 4;

    // this workgroup's part of the keys, head (or key head) and rows
    const int position = positionOf(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
    const int slot = position % output.slots;
    const int unit = position / output.slots % (kNarrow ? args.heads / args.group : args.heads);
    const int split = position / output.slots / (kNarrow ? args.heads / args.group : args.heads);
    const int group = kNarrow ? args.group : 1;
    const int text = textOfSlot<Tile::kRows>(args.q_texts, group, slot);
    if (text < 0) {
        return;
    }
    const TextSpan queries = textSpan(args.q_texts, text);
    const int first_slot = static_cast<int>(queries.first * group / Tile::kRows) + text;
    const int tile_row = (slot - first_slot) * Tile::kRows;
    if (tile_row < 0 || tile_row >= queries.rows * group) {
        return;
    }
    const TextSpan keys = textSpan(args.k_texts, text);
    const int key_head = kNarrow ? unit : unit / args.group;
    const int prefix = args.prefix == nullptr ? 0 : args.prefix[text];
    const int shift = args.q_last ? keys.count - queries.count : 0;  // position of query row 0
    // keys that the query row at a position sees: those before this one
    auto limitAt = [&](int at) { return args.causal ? min(keys.count, max(max(at + 1, prefix), 0)) : keys.count; };

    const int wave_row = tile_row + (kNarrow ? 0 : wave * Tile::kWaveRows);
    int place[kBlocks], head[kBlocks], limit[kBlocks];
    std::int64_t row[kBlocks];
    bool valid[kBlocks], exists[kBlocks];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        const int r = wave_row + 16 * m + r16;
        const int i = r / group;
        exists[m] = i < queries.rows;
        valid[m] = i < queries.count;
        row[m] = queries.first + i;
        head[m] = kNarrow ? unit * group + r % group : unit;
        place[m] = i + shift;
        limit[m] = valid[m] ? limitAt(place[m]) : INT32_MAX;  // the results of other rows are not used
    }
    // of the wavefront's rows that count, the first and the last
    const int last_row = min(wave_row + Tile::kWaveRows, queries.count * group) - 1;
    const bool any = last_row >= wave_row;
    const int first_place = wave_row / group + shift;
    const int last_place = last_row / group + shift;
    const int least_limit = any ? limitAt(first_place) : 0;
    const int most_limit = any ? limitAt(last_place) : 0;
    const int tile_last = min(tile_row + Tile::kRows, queries.count * group) - 1;
    const int all_keys = tile_last >= tile_row ? limitAt(tile_last / group + shift) : 0;

    // tiles of this part of the keys
    const int tiles_all = (all_keys + Tile::kTileKeys - 1) / Tile::kTileKeys;
    const int tiles_each = (tiles_all + output.splits - 1) / output.splits;
    const int tile_begin = split * tiles_each + (kNarrow ? wave : 0);
    const int tile_end = min(tiles_all, (split + 1) * tiles_each);

    std::uint8_t* own = lds + (kNarrow ? wave * 2 * kStageBytes : 0);
    Keys k_tile, v_tile;
    if (tile_begin < tile_end) {
        const int key0 = tile_begin * Tile::kTileKeys;
        const std::int64_t first = keys.first + key0;
        k_tile.begin(static_cast<const T*>(args.k) + first * args.k_stride + key_head * args.head_dim, args.k_stride,
                     keys.count - key0, args.head_dim, kTeams);
        v_tile.begin(static_cast<const T*>(args.v) + first * args.v_stride + key_head * args.head_dim, args.v_stride,
                     keys.count - key0, args.head_dim, kTeams);
        if constexpr (kDirect) {
            k_tile.issue(own, kTeams);
            v_tile.issue(own + Keys::kBytes, kTeams);
        } else {
            k_tile.fetch(kTeams);
            v_tile.fetch(kTeams);
            k_tile.put(own);
            v_tile.put(own + Keys::kBytes);
        }
    }

    const ScoreForm form(args, sizeof(T) == 2);
    float slope[kBlocks];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        slope[m] = args.slopes != nullptr && valid[m] ? form.bias_factor * args.slopes[head[m]] : 0.0f;
    }
    // the tables with kMargin copies of their end values on either side
    const int table_width = biasTableWidth(args.max_distance, Tile::kMargin);
    if (args.table != nullptr) {
        const T* from = static_cast<const T*>(args.table) +
                        static_cast<std::int64_t>(unit * group) * (2 * args.max_distance + 1);
        for (int i = static_cast<int>(threadIdx.x); i < group * table_width; i += kAttentionThreads) {
            const int distance = min(max(i % table_width - Tile::kMargin, 0), 2 * args.max_distance);
            table[i] = biasValue(from[i / table_width * (2 * args.max_distance + 1) + distance], form.bias_factor);
        }
        __syncthreads();
    }

    typename Fragment<T>::type q[kBlocks][Keys::kSteps];
    const bool whole_chunks = args.head_dim % kChunk<T> == 0;
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        const T* from = static_cast<const T*>(args.q) + row[m] * args.q_stride + head[m] * args.head_dim;
        loadRowFragments(from, valid[m] ? args.head_dim : 0, whole_chunks, q[m]);
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

    f32x4 sums[kBlocks][kDimBlocks];
    float largest[kBlocks], total[kBlocks];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        largest[m] = -INFINITY;
        total[m] = 0.0f;
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) {
            sums[m][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    const typename Keys::Lane own_lane;
    auto useTile = [&](std::uint32_t stage, int key0) {
        // scores are s * score_factor + score_offset in base 2
        float score_factor = form.factor;
        float score_offset[kBlocks] = {};
        const int nearest = key0 - last_place;                          // the least distance of the tile
        const int farthest = key0 + Tile::kTileKeys - 1 - first_place;  // the largest
        const bool behind = nearest >= args.max_distance, before = farthest <= -args.max_distance;
        // biases of the tile, or zeros
        f32x4 s[kBlocks][Tile::kKeyBlocks];
        auto loadBiases = [&](f32x4(&to)[kBlocks][Tile::kKeyBlocks]) {
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                // rows past the text's last one may reach beyond the margin
                const int at = min(max(key0 + 4 * h - place[m] + args.max_distance + Tile::kMargin, 0),
                                   table_width - Tile::kTileKeys + 12);
                const float* from = table + (kNarrow ? head[m] - unit * group : 0) * table_width + at;
#pragma unroll
                for (int b = 0; b < Tile::kKeyBlocks; ++b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        to[m][b][e] = from[16 * b + e];
                    }
                }
            }
        };
        auto addSlopes = [&](f32x4(&to)[kBlocks][Tile::kKeyBlocks]) {
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const float distance = static_cast<float>(key0 + 4 * h - place[m]);
#pragma unroll
                for (int b = 0; b < Tile::kKeyBlocks; ++b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        to[m][b][e] = fmaf(-slope[m], fabsf(distance + static_cast<float>(16 * b + e)), to[m][b][e]);
                    }
                }
            }
        };
        const bool in_table = args.table != nullptr && !behind && !before;
        const float offset_factor = form.formed ? 1.0f : form.factor;
        auto products = [&](auto from_zero) {
#pragma unroll
            for (int b = 0; b < Tile::kKeyBlocks; ++b) {
#pragma unroll
                for (int t = 0; t < Keys::kSteps; ++t) {
                    const auto k = Keys::read(stage, own_lane, b, t);
#pragma unroll
                    for (int m = 0; m < kBlocks; ++m) {
                        s[m][b] = multiplyAdd(k, q[m][t], decltype(from_zero)::value && t == 0 ? f32x4{} : s[m][b]);
                    }
                }
            }
            scheduleProducts<Tile::kKeyBlocks * Keys::kSteps, kBlocks * (sizeof(T) == 2 ? 1 : 4)>();
        };
        if (form.formed || (!in_table && args.slopes == nullptr)) {
            products(std::true_type{});
        } else {
            if (in_table) {
                loadBiases(s);
            } else {
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                    for (int b = 0; b < Tile::kKeyBlocks; ++b) {
                        s[m][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    }
                }
            }
            if (args.slopes != nullptr) {
                addSlopes(s);
            }
            products(std::false_type{});
        }
        if (form.capped) {
            withTanh<T>(form, [&](auto fine) {
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                    for (int b = 0; b < Tile::kKeyBlocks; ++b) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[m][b][e] = tanhOf<T, decltype(fine)::value>(s[m][b][e] * form.to_cap);
                        }
                    }
                }
            });
            score_factor = form.cap;
        }
        if (form.formed && (!form.capped || in_table || args.slopes != nullptr)) {
            asm volatile("");  // stays a branch
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                for (int b = 0; b < Tile::kKeyBlocks; ++b) {
                    s[m][b] *= score_factor;
                }
            }
            score_factor = 1.0f;
            if (in_table) {
                f32x4 bias[kBlocks][Tile::kKeyBlocks];
                loadBiases(bias);
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                    for (int b = 0; b < Tile::kKeyBlocks; ++b) {
                        s[m][b] += bias[m][b];
                    }
                }
            }
            if (args.slopes != nullptr) {
                addSlopes(s);
            }
        }
        if (args.table != nullptr && !in_table) {
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const int base = (kNarrow ? head[m] - unit * group : 0) * table_width;
                score_offset[m] = offset_factor * table[base + (behind ? table_width - 1 : 0)];
            }
        }
        if (key0 + Tile::kTileKeys > least_limit) {
            asm volatile("");  // stays a branch
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const int left = limit[m] - key0 - 4 * h;
#pragma unroll
                for (int b = 0; b < Tile::kKeyBlocks; ++b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[m][b][e] = 16 * b + e < left ? s[m][b][e] : -INFINITY;
                    }
                }
            }
        }
        bool raise = false;
        float peak[kBlocks];
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
            peak[m] = s[m][0][0];
#pragma unroll
            for (int b = 0; b < Tile::kKeyBlocks; ++b) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    peak[m] = __builtin_elementwise_maximum(peak[m], s[m][b][e]);
                }
            }
            peak[m] = fmaf(overGroups(peak[m]), score_factor, score_offset[m]);
            raise = raise || peak[m] > largest[m] + 8.0f;
        }
        if (__ballot(raise) != 0) {
            asm volatile("");  // stays a branch
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const float now = __builtin_elementwise_maximum(largest[m], peak[m]);
                const float keep = now == largest[m] ? 1.0f : __builtin_amdgcn_exp2f(largest[m] - now);
                largest[m] = now;
                total[m] *= keep;
#pragma unroll
                for (int d = 0; d < kDimBlocks; ++d) {
                    sums[m][d] *= keep;
                }
            }
        }
        typename Fragment<T>::type p[kBlocks][Tile::kKeyBlocks / kBlocksTurned<T>];
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
            // a row that has seen no key yet has only scores of minus infinity
            const float off = score_offset[m] - (largest[m] == -INFINITY ? 0.0f : largest[m]);
#pragma unroll
            for (int b = 0; b < Tile::kKeyBlocks; ++b) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[m][b][e] = __builtin_amdgcn_exp2f(fmaf(s[m][b][e], score_factor, off));
                    total[m] += s[m][b][e];
                }
            }
#pragma unroll
            for (int b = 0; b < Tile::kKeyBlocks / kBlocksTurned<T>; ++b) {
                p[m][b] = resultFragment<T>(&s[m][b * kBlocksTurned<T>]);
            }
        }
        const std::uint32_t values = stage + Keys::kBytes;
#pragma unroll
        for (int b = 0; b < Tile::kKeyBlocks / kBlocksTurned<T>; ++b) {
#pragma unroll
            for (int d = 0; d < kDimBlocks; ++d) {
                const auto v = Keys::readTurned(values, own_lane, d, b);
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    sums[m][d] = multiplyAdd(v, p[m][b], sums[m][d]);
                }
            }
        }
    };

    // the queries have arrived as well: a wait for them within the loop would be one for the next tile too
    __builtin_amdgcn_s_waitcnt(vmcntOnly(0));
    int buffer = 0;
    for (int tile = tile_begin; tile < tile_end; tile += kTeams) {
        // this tile has arrived, and every wavefront of the team has read the other buffer
        teamSync<Tile::kTeam>();
        const std::uint8_t* stage = own + buffer * kStageBytes;
        std::uint8_t* other = own + (buffer ^ 1) * kStageBytes;
        buffer ^= 1;
        const bool more = tile + kTeams < tile_end;
        if (more) {
            if constexpr (kDirect) {
                k_tile.issue(other, kTeams);
                v_tile.issue(other + Keys::kBytes, kTeams);
            } else {
                k_tile.fetch(kTeams);
                v_tile.fetch(kTeams);
            }
        }
        const int key0 = tile * Tile::kTileKeys;
        if (key0 < most_limit) {
            useTile(ldsAddress(stage), key0);
        }
        if constexpr (!kDirect) {
            if (more) {
                k_tile.put(other);
                v_tile.put(other + Keys::kBytes);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        total[m] += waveXor(total[m], 16);
        total[m] += waveXor(total[m], 32);
    }

    if constexpr (kNarrow) {
        // join the wavefronts' rows: each brings its own to the common maximum
        static_assert(kBlocks == 1, "one row block");
        __syncthreads();
        float* maxima = reinterpret_cast<float*>(lds + kAttentionWaves * kDimBlocks * kWave * 16);
        float* totals = maxima + kAttentionWaves * 16;
        f32x4* rows = reinterpret_cast<f32x4*>(lds);
        if (h == 0) {
            maxima[wave * 16 + r16] = largest[0];
        }
        __syncthreads();
        float now = maxima[r16];
#pragma unroll
        for (int w = 1; w < kAttentionWaves; ++w) {
            now = fmaxf(now, maxima[w * 16 + r16]);
        }
        const float keep = now == largest[0] ? 1.0f : __builtin_amdgcn_exp2f(largest[0] - now);
        if (h == 0) {
            totals[wave * 16 + r16] = total[0] * keep;
        }
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) {
            rows[(wave * kDimBlocks + d) * kWave + lane] = sums[0][d] * keep;
        }
        __syncthreads();
        largest[0] = now;
        total[0] = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttentionWaves; ++w) {
            total[0] += totals[w * 16 + r16];
        }
        // wavefront w finishes every fourth block of columns
        for (int d = wave; d < kDimBlocks; d += kAttentionWaves) {
            f32x4 sum = rows[d * kWave + lane];
#pragma unroll
            for (int w = 1; w < kAttentionWaves; ++w) {
                sum += rows[(w * kDimBlocks + d) * kWave + lane];
            }
            const int column = 16 * d + 4 * h;
            if (!exists[0]) {
                continue;
            }
            if (output.splits > 1) {
                const std::int64_t at = (split * args.q_texts.total + row[0]) * args.heads + head[0];
                *reinterpret_cast<f32x4*>(output.partial_rows + at * kDim + column) = valid[0] ? sum : f32x4{};
            } else if (column < args.head_dim) {
                const float scale = valid[0] && total[0] != 0.0f ? 1.0f / total[0] : 0.0f;
                const f32x4 result = valid[0] && total[0] != 0.0f ? sum * scale : f32x4{};
                storeFour(result, static_cast<T*>(output.out) + row[0] * output.out_stride + head[0] * args.head_dim + column,
                          args.head_dim - column);
            }
        }
        if (wave == 0 && h == 0 && exists[0]) {
            if (output.splits > 1) {
                const std::int64_t at = (split * args.q_texts.total + row[0]) * args.heads + head[0];
                output.partial_stats[2 * at] = valid[0] ? largest[0] : -INFINITY;
                output.partial_stats[2 * at + 1] = valid[0] ? total[0] : 0.0f;
            } else if (output.lse != nullptr) {
                output.lse[row[0] * args.heads + head[0]] =
                    valid[0] && total[0] != 0.0f ? kLn2 * (largest[0] + __builtin_amdgcn_logf(total[0])) : -INFINITY;
            }
        }
        return;
    }
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
        const bool empty = !valid[m] || total[m] == 0.0f;
        const float scale = empty ? 0.0f : 1.0f / total[m];
        if (!exists[m]) {
            continue;
        }
        T* to = static_cast<T*>(output.out) + row[m] * output.out_stride + head[m] * args.head_dim;
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) {
            const int column = 16 * d + 4 * h;
            if (column < args.head_dim) {
                storeFour(empty ? f32x4{} : sums[m][d] * scale, to + column, args.head_dim - column);
            }
        }
        if (output.lse != nullptr && h == 0) {
            output.lse[row[m] * args.heads + head[m]] =
                empty ? -INFINITY : kLn2 * (largest[m] + __builtin_amdgcn_logf(total[m]));
        }
    }
}

// Rows from the parts of their keys, a workgroup a row and head: its threads take four columns each of every
// kJoinParts-th part. Parts of rows of no text are not written and not read.
template <typename T, int kDim>
__global__ __launch_bounds__(kAttentionThreads) void joinAttentionKernel(AttentionArgs args, AttentionOutput output) {
    constexpr int kColumnThreads = kDim / 4;
    constexpr int kJoinParts = kAttentionThreads / kColumnThreads;
    __shared__ float maxima[kAttentionWaves], totals[kAttentionWaves];
    __shared__ f32x4 sums[kJoinParts][kColumnThreads];
    const std::int64_t rows = args.q_texts.total * args.heads;
    const std::int64_t at = blockIdx.x;
    const std::int64_t row = at / args.heads;
    const int head = static_cast<int>(at % args.heads);
    if (args.q_texts.offsets != nullptr) {
        const std::int64_t first = textStart(args.q_texts, 0), end = textStart(args.q_texts, args.q_texts.texts);
        if (row < first || row >= end) {
            return;
        }
    }
    // (at most as many parts as threads)
    const int thread = static_cast<int>(threadIdx.x);
    const int wave = thread / kWave;
    const float* stats = output.partial_stats + 2 * (thread * rows + at);
    const float own_largest = thread < output.splits ? stats[0] : -INFINITY;
    const float own_total = thread < output.splits ? stats[1] : 0.0f;
    const int column = 4 * (thread % kColumnThreads);
    const int part = thread / kColumnThreads;
    float largest = own_largest;
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) {
        largest = fmaxf(largest, waveXor(largest, offset));
    }
    if (thread % kWave == 0) {
        maxima[wave] = largest;
    }
    __syncthreads();
    largest = maxima[0];
#pragma unroll
    for (int w = 1; w < kAttentionWaves; ++w) {
        largest = fmaxf(largest, maxima[w]);
    }
    float total = own_total * (own_largest == largest ? 1.0f : __builtin_amdgcn_exp2f(own_largest - largest));
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) {
        total += waveXor(total, offset);
    }
    if (thread % kWave == 0) {
        totals[wave] = total;
    }
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = part; s < output.splits; s += kJoinParts) {
        const float at_part = output.partial_stats[2 * (s * rows + at)];
        const float keep = at_part == largest ? 1.0f : __builtin_amdgcn_exp2f(at_part - largest);
        sum += *reinterpret_cast<const f32x4*>(output.partial_rows + (s * rows + at) * kDim + column) * keep;
    }
    sums[part][thread % kColumnThreads] = sum;
    __syncthreads();
    if (part != 0) {
        return;
    }
    total = totals[0];
#pragma unroll
    for (int w = 1; w < kAttentionWaves; ++w) {
        total += totals[w];
    }
#pragma unroll
    for (int p = 1; p < kJoinParts; ++p) {
        sum += sums[p][thread];
    }
    const bool empty = total == 0.0f;
    if (column < args.head_dim) {
        storeFour(empty ? f32x4{} : sum * (1.0f / total),
                  static_cast<T*>(output.out) + row * output.out_stride + head * args.head_dim + column, args.head_dim - column);
    }
    if (output.lse != nullptr && thread == 0) {
        output.lse[at] = empty ? -INFINITY : kLn2 * (largest + __builtin_amdgcn_logf(total));
    }
}

// ---- host ---------------------------------------------------------------------------------------

template <typename T, int kDim, int kBlocks, bool kNarrow, bool kDirect>
int launchAttentionTiles(const AttentionArgs& args, AttentionOutput output, hipStream_t stream) {
    using Tile = AttentionTile<T, kDim, kBlocks, kNarrow>;
    const int units = kNarrow ? args.heads / args.group : args.heads;
    const long long slots = slotsOf(args.q_texts, kNarrow ? args.group : 1, Tile::kRows);
    if (slots * units * output.splits > kMaxAttentionBlocks) {
        return attentionInvalid("more texts and rows than one launch can take");
    }
    output.slots = static_cast<int>(slots);
    attentionKernel<T, kDim, kBlocks, kNarrow, kDirect>
        <<<static_cast<unsigned>(slots * units * output.splits), kAttentionThreads, 0, stream>>>(args, output);
    ZCGVS_LAUNCH_CHECK("attention");
    if (output.splits > 1) {
        const std::int64_t rows = args.q_texts.total * args.heads;
        joinAttentionKernel<T, kDim><<<static_cast<unsigned>(rows), kAttentionThreads, 0, stream>>>(args, output);
        ZCGVS_LAUNCH_CHECK("attention");
    }
    return ZCGVS_OK;
}

template <typename T, int kDim>
int launchAttentionDim(const AttentionPlan& plan, const AttentionArgs& args, const AttentionOutput& output, hipStream_t stream) {
    if (plan.shape == AttentionShape::kNarrow) {
        return plan.direct ? launchAttentionTiles<T, kDim, 1, true, true>(args, output, stream)
                           : launchAttentionTiles<T, kDim, 1, true, false>(args, output, stream);
    }
    if (!plan.direct) {
        return launchAttentionTiles<T, kDim, 1, false, false>(args, output, stream);
    }
    return plan.shape == AttentionShape::kShort ? launchAttentionTiles<T, kDim, 1, false, true>(args, output, stream)
                                                : launchAttentionTiles<T, kDim, 2, false, true>(args, output, stream);
}

}  // namespace

template <typename T>
int launchAttention(const AttentionPlan& plan, const AttentionArgs& args, const AttentionOutput& output, hipStream_t stream) {
    switch (paddedDim(args.head_dim)) {
        case 32:
            return launchAttentionDim<T, 32>(plan, args, output, stream);
        case 64:
            return launchAttentionDim<T, 64>(plan, args, output, stream);
        default:
            return launchAttentionDim<T, 128>(plan, args, output, stream);
    }
}

}  // namespace zcgvs_hip
