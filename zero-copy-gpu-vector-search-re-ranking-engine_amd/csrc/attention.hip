// Attention over packed texts: checks, plans and the launches' order. The kernels are in attention_kernel.hpp,
// built for each operand type by a file of its own.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attention.hpp"
#include "common.hpp"
#include "elements.hpp"
#include "matrix_plan.hpp"

namespace zcgvs_hip {

int attentionInvalid(const char* message) {
    return setError(ZCGVS_ERR_INVALID_ARGUMENT, std::string("zcgvs attention: ") + message);
}

namespace {

int checkAttention(const zcgvs_attention_desc* desc) {
    if (desc == nullptr) {
        return attentionInvalid("null descriptor");
    }
    const zcgvs_attention_desc& d = *desc;
    if (!validElement(d.dtype)) {
        return attentionInvalid("the operands must hold float32, float16 or bfloat16");
    }
    if (d.heads <= 0 || d.heads > 1024 || d.kv_heads <= 0 || d.heads % d.kv_heads != 0) {
        return attentionInvalid("heads must lie in [1, 1024] and be a multiple of kv_heads");
    }
    if (d.head_dim <= 0 || d.head_dim > kAttentionMaxDim) {
        return attentionInvalid("head_dim must lie in [1, 128]");
    }
    if (d.q_rows < 0 || d.q_rows > (1 << 28) || d.k_rows < 0 || d.k_rows > (1 << 28)) {
        return attentionInvalid("q_rows and k_rows must lie in [0, 2^28]");
    }
    if (d.texts < 0 || d.texts > (1 << 24)) {
        return attentionInvalid("texts must lie in [0, 2^24]");
    }
    if (d.texts > 0 && ((d.q_offsets == nullptr && d.q_rows % d.texts != 0) || (d.k_offsets == nullptr && d.k_rows % d.texts != 0))) {
        return attentionInvalid("rows without offsets must be a multiple of texts");
    }
    const int q_width = d.heads * d.head_dim;
    const int k_width = d.kv_heads * d.head_dim;
    if (rowStride(d.q_stride, q_width) < q_width || rowStride(d.k_stride, k_width) < k_width ||
        rowStride(d.v_stride, k_width) < k_width) {
        return attentionInvalid("a row stride is smaller than its heads");
    }
    if (d.q_align != ZCGVS_ATTENTION_FIRST && d.q_align != ZCGVS_ATTENTION_LAST) {
        return attentionInvalid("unknown alignment of the queries");
    }
    if (d.prefix_lengths != nullptr && d.causal == 0) {
        return attentionInvalid("prefix_lengths need the causal mask");
    }
    if (!std::isfinite(d.scale) || !std::isfinite(d.cap) || d.cap < 0.0f) {
        return attentionInvalid("scale and cap must be finite, cap at least 0");
    }
    if (d.distance_bias != nullptr && (d.max_distance < 0 || d.max_distance > kAttentionMaxDistance)) {
        return attentionInvalid("max_distance must lie in [0, 512]");
    }
    if (d.texts > 0 && d.q_rows > 0 && (d.q == nullptr || (d.k_rows > 0 && (d.k == nullptr || d.v == nullptr)))) {
        return attentionInvalid("null device pointer");
    }
    return ZCGVS_OK;
}

bool noWork(const zcgvs_attention_desc& d) { return d.texts == 0 || d.q_rows == 0; }

AttentionArgs attentionArgs(const zcgvs_attention_desc& d) {
    AttentionArgs args{};
    args.q = d.q;
    args.k = d.k;
    args.v = d.v;
    args.q_stride = rowStride(d.q_stride, d.heads * d.head_dim);
    args.k_stride = rowStride(d.k_stride, d.kv_heads * d.head_dim);
    args.v_stride = rowStride(d.v_stride, d.kv_heads * d.head_dim);
    const int texts = static_cast<int>(d.texts);
    args.q_texts = {d.q_offsets, d.q_lengths, d.q_rows, texts, static_cast<int>(d.q_rows / d.texts)};
    args.k_texts = {d.k_offsets, d.k_lengths, d.k_rows, texts, static_cast<int>(d.k_rows / d.texts)};
    args.heads = d.heads;
    args.group = d.heads / d.kv_heads;
    args.head_dim = d.head_dim;
    args.q_last = d.q_align == ZCGVS_ATTENTION_LAST ? 1 : 0;
    args.causal = d.causal != 0 ? 1 : 0;
    args.prefix = d.prefix_lengths;
    args.scale = d.scale;
    args.cap = d.cap;
    args.slopes = d.slopes;
    args.table = d.distance_bias;
    args.max_distance = d.distance_bias == nullptr ? 0 : d.max_distance;
    return args;
}

struct HostPlan {
    AttentionShape shape;
    int splits;
};

// By the mean rows and keys of a text: the narrow shape where a key head's query rows fit one workgroup's 16, or where the
// others leave most CUs idle over long keys.
HostPlan planAttention(const zcgvs_attention_desc& d) {
    const long long units = deviceComputeUnits();
    const int group = d.heads / d.kv_heads;
    const double rows = static_cast<double>(d.q_rows) / static_cast<double>(d.texts);
    const double keys = static_cast<double>(d.k_rows) / static_cast<double>(d.texts);
    const double short_blocks = d.heads * (static_cast<double>(d.q_rows) / 64.0 + static_cast<double>(d.texts));
    const int tile_keys = narrowKeys(paddedDim(d.head_dim), elementBytes(d.dtype));
    const long long table = d.distance_bias == nullptr ? 0 : biasTableWidth(d.max_distance, tile_keys + kNarrowRows);
    const bool fits = group * table <= kNarrowTable && d.q_rows * group < (1ll << 30);
    if (fits && (rows * group <= 16.0 || (short_blocks <= units / 2 && keys >= 512.0))) {
        const double blocks = d.kv_heads * (static_cast<double>(d.q_rows) * group / 16.0 + static_cast<double>(d.texts));
        // A workgroup a CU, and tiles for two of its wavefronts at least. The last of 32,000 rows, 16 heads of 128 on 4
        // float16: 20.3 us, 25.0 with two workgroups a CU (one of which wide heads leave LDS for); of 1500 float32 13.4, 17.1
        // with two tiles for every wavefront; of 8193 14.0, 14.0.
        const double most = keys / (2.0 * tile_keys);
        const double splits = std::min(static_cast<double>(units) / blocks, most);
        return {AttentionShape::kNarrow, std::max(1, std::min(128, static_cast<int>(splits)))};
    }
    return {rows <= 64.0 ? AttentionShape::kShort : AttentionShape::kLong, 1};
}

std::size_t partialFloats(const zcgvs_attention_desc& d, int splits, int each) {
    return splits == 1 ? 0 : static_cast<std::size_t>(splits) * static_cast<std::size_t>(d.q_rows) * d.heads * each;
}

// ---- the gradient's workspace: the rows' statistics, the bias's partial sums -----------------------

// Blocks of 16 rows of a wavefront by a text's mean rows: tiles of 128 where texts fill them. Two blocks of keys, their
// values and both gradients do not fit the registers for float32 heads of 128.
int gradientBlocks(std::int64_t rows, std::int64_t texts) { return rows <= 64 * texts ? 1 : 2; }

int keyBlocks(const zcgvs_attention_desc& d) {
    return paddedDim(d.head_dim) == 128 ? 1 : gradientBlocks(d.k_rows, d.texts);
}

long long slotsFor(std::int64_t rows, std::int64_t texts, int blocks) { return rows / (64 * blocks) + texts; }

std::size_t statsBytes(const zcgvs_attention_desc& d) {
    return (static_cast<std::size_t>(d.q_rows) * d.heads * 2 * sizeof(float) + 255) / 256 * 256;
}

std::size_t tableBytes(const zcgvs_attention_desc& d) {
    return d.distance_bias == nullptr ? 0
                                      : static_cast<std::size_t>(slotsFor(d.k_rows, d.texts, keyBlocks(d))) * d.heads *
                                            (2 * static_cast<std::size_t>(d.max_distance) + 1) * sizeof(float);
}

// Parts of a key head's query heads in the launch for dk and dv, joined by one more: as many as bring it to four
// workgroups a CU. 8 texts of 512, 16 heads of 64 on 1 bfloat16: 299 us without parts, 101 with a workgroup a CU, 79 with four,
// 80 with eight; 3 texts of 2048 on 2: 603, 360, 262, 262; 3 texts of up to 77 float32, 6 heads of 32 on 2: 40 and 28.
int keyParts(const zcgvs_attention_desc& d) {
    const int group = d.heads / d.kv_heads;
    const long long blocks = slotsFor(d.k_rows, d.texts, keyBlocks(d)) * d.kv_heads;
    return static_cast<int>(std::max(1ll, std::min<long long>(group, 4 * deviceComputeUnits() / blocks)));
}

std::size_t keyPartBytes(const zcgvs_attention_desc& d) {
    const int parts = keyParts(d);
    return parts == 1 ? 0
                      : 2 * static_cast<std::size_t>(parts) * static_cast<std::size_t>(d.k_rows) * d.kv_heads * d.head_dim * sizeof(float);
}

template <typename T>
__global__ __launch_bounds__(256) void clearTextRowsKernel(TextRows rows, int width, std::int64_t stride, T* out) {
    const std::int64_t first = textStart(rows, 0), end = textStart(rows, rows.texts);
    for (std::int64_t r = first + blockIdx.x; r < end; r += gridDim.x) {
        for (int c = static_cast<int>(threadIdx.x); c < width; c += 256) {
            out[r * stride + c] = static_cast<T>(0.0f);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void clearTableKernel(int count, T* out) {
    for (int i = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x); i < count;
         i += static_cast<int>(gridDim.x) * 256) {
        out[i] = static_cast<T>(0.0f);
    }
}

}  // namespace

}  // namespace zcgvs_hip

using namespace zcgvs_hip;

extern "C" {

int zcgvs_attention_max_head_dim(void) { return kAttentionMaxDim; }

int zcgvs_attention_max_distance(void) { return kAttentionMaxDistance; }

std::size_t zcgvs_attention_workspace_bytes(const zcgvs_attention_desc* desc) {
    if (checkAttention(desc) != ZCGVS_OK) {
        return 0;
    }
    clearError();
    if (noWork(*desc)) {
        return 256;
    }
    const int splits = planAttention(*desc).splits;
    return std::max<std::size_t>(256, partialFloats(*desc, splits, paddedDim(desc->head_dim) + 2) * sizeof(float));
}

int zcgvs_attention(const zcgvs_attention_desc* desc, void* d_out, std::int64_t out_stride, float* d_lse,
                    void* d_workspace, std::size_t workspace_bytes, zcgvs_stream_t stream) {
    const int status = checkAttention(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_attention_desc& d = *desc;
    const int width = d.heads * d.head_dim;
    if (rowStride(out_stride, width) < width) {
        return attentionInvalid("the output's row stride is smaller than its heads");
    }
    if (noWork(d)) {
        return clearError();
    }
    if (d_out == nullptr) {
        return attentionInvalid("null device pointer");
    }
    const HostPlan plan = planAttention(d);
    const AttentionArgs args = attentionArgs(d);
    AttentionOutput output{};
    output.out = d_out;
    output.out_stride = rowStride(out_stride, width);
    output.lse = d_lse;
    output.splits = plan.splits;
    if (plan.splits > 1) {
        if (d_workspace == nullptr || workspace_bytes < zcgvs_attention_workspace_bytes(desc)) {
            return attentionInvalid("the workspace is too small");
        }
        if (!aligned16(d_workspace)) {
            return attentionInvalid("the workspace must be aligned to 16 bytes");
        }
        output.partial_rows = static_cast<float*>(d_workspace);
        output.partial_stats = output.partial_rows + partialFloats(d, plan.splits, paddedDim(d.head_dim));
    }
    const bool direct = directRows(d.k, args.k_stride, d.head_dim, d.dtype) && directRows(d.v, args.v_stride, d.head_dim, d.dtype);
    const int launched = withElement(d.dtype, [&](auto element) {
        return launchAttention<decltype(element)>({plan.shape, direct}, args, output, toStream(stream));
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

std::size_t zcgvs_attention_gradient_workspace_bytes(const zcgvs_attention_desc* desc) {
    if (checkAttention(desc) != ZCGVS_OK) {
        return 0;
    }
    clearError();
    return desc->texts == 0 ? 256 : std::max<std::size_t>(256, statsBytes(*desc) + tableBytes(*desc) + keyPartBytes(*desc));
}

int zcgvs_attention_gradient(const zcgvs_attention_desc* desc, const void* d_out, std::int64_t out_stride, const float* d_lse,
                             const void* d_out_gradient, std::int64_t out_gradient_stride, void* d_q_gradient,
                             std::int64_t q_gradient_stride, void* d_k_gradient, std::int64_t k_gradient_stride,
                             void* d_v_gradient, std::int64_t v_gradient_stride, void* d_distance_bias_gradient,
                             void* d_workspace, std::size_t workspace_bytes, zcgvs_stream_t stream) {
    const int status = checkAttention(desc);
    if (status != ZCGVS_OK) {
        return status;
    }
    const zcgvs_attention_desc& d = *desc;
    const int q_width = d.heads * d.head_dim;
    const int k_width = d.kv_heads * d.head_dim;
    AttentionGradient more{};
    more.out_stride = rowStride(out_stride, q_width);
    more.out_gradient_stride = rowStride(out_gradient_stride, q_width);
    more.q_gradient_stride = rowStride(q_gradient_stride, q_width);
    more.k_gradient_stride = rowStride(k_gradient_stride, k_width);
    more.v_gradient_stride = rowStride(v_gradient_stride, k_width);
    if (more.out_stride < q_width || more.out_gradient_stride < q_width || more.q_gradient_stride < q_width ||
        more.k_gradient_stride < k_width || more.v_gradient_stride < k_width) {
        return attentionInvalid("a row stride is smaller than its heads");
    }
    if (d_distance_bias_gradient != nullptr && d.distance_bias == nullptr) {
        return attentionInvalid("a gradient of the distance bias needs the distance bias");
    }
    const int table_count = d.distance_bias == nullptr ? 0 : d.heads * (2 * d.max_distance + 1);
    if (d.texts == 0 || (d.q_rows == 0 && d.k_rows == 0)) {
        if (d_distance_bias_gradient != nullptr) {
            return withElement(d.dtype, [&](auto element) {
                using T = decltype(element);
                clearTableKernel<T><<<64, 256, 0, toStream(stream)>>>(table_count, static_cast<T*>(d_distance_bias_gradient));
                ZCGVS_LAUNCH_CHECK("attention gradient");
                return clearError();
            });
        }
        return clearError();
    }
    if ((d.q_rows > 0 && (d_out == nullptr || d_lse == nullptr || d_out_gradient == nullptr || d_q_gradient == nullptr)) ||
        (d.k_rows > 0 && (d_k_gradient == nullptr || d_v_gradient == nullptr))) {
        return attentionInvalid("null device pointer");
    }
    if (d_workspace == nullptr || workspace_bytes < zcgvs_attention_gradient_workspace_bytes(desc)) {
        return attentionInvalid("the workspace is too small");
    }
    if (!aligned16(d_workspace)) {
        return attentionInvalid("the workspace must be aligned to 16 bytes");
    }
    const AttentionArgs args = attentionArgs(d);
    more.out = d_out;
    more.lse = d_lse;
    more.out_gradient = d_out_gradient;
    more.q_gradient = d_q_gradient;
    more.k_gradient = d_k_gradient;
    more.v_gradient = d_v_gradient;
    more.table_gradient = d_distance_bias_gradient;
    const int launched = withElement(d.dtype, [&](auto element) {
        using T = decltype(element);
        if (d.q_rows == 0 || d.k_rows == 0) {
            // nothing sees anything: zeros for the rows of the texts
            const TextRows& rows = d.q_rows == 0 ? args.k_texts : args.q_texts;
            const int width = d.q_rows == 0 ? k_width : q_width;
            if (d.q_rows == 0) {
                clearTextRowsKernel<T><<<1024, 256, 0, toStream(stream)>>>(rows, width, more.k_gradient_stride,
                                                                           static_cast<T*>(d_k_gradient));
                clearTextRowsKernel<T><<<1024, 256, 0, toStream(stream)>>>(rows, width, more.v_gradient_stride,
                                                                           static_cast<T*>(d_v_gradient));
            } else {
                clearTextRowsKernel<T><<<1024, 256, 0, toStream(stream)>>>(rows, width, more.q_gradient_stride,
                                                                           static_cast<T*>(d_q_gradient));
            }
            if (d_distance_bias_gradient != nullptr) {
                clearTableKernel<T><<<64, 256, 0, toStream(stream)>>>(table_count, static_cast<T*>(d_distance_bias_gradient));
            }
            ZCGVS_LAUNCH_CHECK("attention gradient");
            return static_cast<int>(ZCGVS_OK);
        }
        AttentionGradientPlan plan{};
        plan.key_blocks = keyBlocks(d);
        plan.query_blocks = gradientBlocks(d.q_rows, d.texts);
        const long long key_slots = slotsFor(d.k_rows, d.texts, plan.key_blocks);
        const long long query_slots = slotsFor(d.q_rows, d.texts, plan.query_blocks);
        if (key_slots * d.kv_heads > kMaxAttentionBlocks || query_slots * d.heads > kMaxAttentionBlocks) {
            return attentionInvalid("more texts and rows than one launch can take");
        }
        more.key_slots = static_cast<int>(key_slots);
        more.query_slots = static_cast<int>(query_slots);
        more.key_parts = keyParts(d);
        more.stats = static_cast<float*>(d_workspace);
        more.key_partials = reinterpret_cast<float*>(static_cast<char*>(d_workspace) + statsBytes(d) + tableBytes(d));
        if (d_distance_bias_gradient != nullptr) {
            more.table_partials = reinterpret_cast<float*>(static_cast<char*>(d_workspace) + statsBytes(d));
        }
        plan.direct_rows = directRows(d.q, args.q_stride, d.head_dim, d.dtype) &&
                           directRows(d_out_gradient, more.out_gradient_stride, d.head_dim, d.dtype);
        plan.direct_keys = directRows(d.k, args.k_stride, d.head_dim, d.dtype) &&
                           directRows(d.v, args.v_stride, d.head_dim, d.dtype);
        return launchAttentionGradient<T>(plan, args, more, toStream(stream));
    });
    return launched == ZCGVS_OK ? clearError() : launched;
}

}  // extern "C"
