/*
 * zcgvs_hip.h - C ABI of the MI355X (gfx950) zero-copy search hot path.
 *
 * Every entry point takes plain device pointers, sizes and a stream handle and returns a
 * zcgvs_status code. Nothing here throws, and no C++ or torch type crosses the boundary.
 * The message describing the most recent failure on the calling thread is returned by
 * zcgvs_last_error().
 *
 * Error contract (mirrors the reference's exception split, include/zcgvs/core/cuda_check.hpp
 * and src/search/searcher.cpp:91-135):
 *   ZCGVS_ERR_INVALID_ARGUMENT  - the reference throws std::invalid_argument;
 *   ZCGVS_ERR_RUNTIME           - the reference throws std::runtime_error (e.g. N > INT32_MAX);
 *   ZCGVS_ERR_HIP               - a HIP runtime call failed (the reference's CudaError).
 * Launchers that receive empty work (count <= 0) return ZCGVS_OK without launching, exactly
 * like the reference launchers (src/cuda/similarity.cu:356-358, topk.cu:143-145).
 *
 * Launchers are asynchronous on the given stream, never allocate device memory, never
 * synchronize, and are safe to record into a HIP graph (zcgvs_graph_begin_capture). The one
 * exception is zcgvs_memset, which must not be recorded into a graph; use zcgvs_fill_u32.
 *
 * Enumerations keep the reference's numeric codes, which are part of its on-disk format:
 *   metric (include/zcgvs/core/metric.hpp:8-12), dtype (include/zcgvs/core/scalar_type.hpp:12-17).
 *
 * Top-k ordering (all selection entry points): score descending, ties broken by the lower
 * corpus index, i.e. the order std::stable_sort gives in tests/cpp/cpu_reference.hpp:26-34.
 * -0.0f ranks equal to +0.0f; a NaN score ranks below every other score.
 */
#ifndef ZCGVS_HIP_H
#define ZCGVS_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------------------------
 * Status, enums, opaque handles
 * ---------------------------------------------------------------------------------------- */
enum zcgvs_status {
    ZCGVS_OK = 0,
    ZCGVS_ERR_INVALID_ARGUMENT = 1,
    ZCGVS_ERR_RUNTIME = 2,
    ZCGVS_ERR_HIP = 3,
    ZCGVS_ERR_UNSUPPORTED = 4
};

/* include/zcgvs/core/metric.hpp:8-12 */
enum zcgvs_metric { ZCGVS_METRIC_COSINE = 0, ZCGVS_METRIC_DOT = 1, ZCGVS_METRIC_L2 = 2 };

/* include/zcgvs/core/scalar_type.hpp:12-17 */
enum zcgvs_dtype {
    ZCGVS_DTYPE_F32 = 0,
    ZCGVS_DTYPE_F16 = 1,
    ZCGVS_DTYPE_I8 = 2,
    ZCGVS_DTYPE_BINARY = 3,
    /* bfloat16: the embedding-model operators only; no store or search takes it */
    ZCGVS_DTYPE_BF16 = 4
};

/* How an int8 corpus is scored.
 *  REFERENCE: (int8 * one matrix-wide scale) against a float32 query, accumulated in float32,
 *             as src/cuda/similarity.cu:59-67 and include/zcgvs/cuda/decode.cuh:24-26 do.
 *  PER_VECTOR: each row r carries its own scale s_r = max|x_r| / 127; queries are quantized the
 *             same way on the device; score = (float)(int32 dot) * (s_q * s_r), evaluated in
 *             exactly that order. No counterpart in the reference (its format has one scale). */
enum zcgvs_int8_mode { ZCGVS_INT8_REFERENCE = 0, ZCGVS_INT8_PER_VECTOR = 1 };

typedef void* zcgvs_stream_t; /* hipStream_t; NULL is the null stream   */
typedef void* zcgvs_event_t;  /* hipEvent_t                               */
typedef void* zcgvs_graph_t;  /* hipGraphExec_t (instantiated graph)      */

/* Message for the most recent non-OK status returned on this thread ("" if none). */
const char* zcgvs_last_error(void);
/* Library version string, e.g. "zcgvs-hip 0.1.0 gfx950". */
const char* zcgvs_version(void);

/* ------------------------------------------------------------------------------------------
 * Device, memory, streams, events, graphs - the thin runtime layer the C++17 host uses in
 * place of include/zcgvs/core/{cuda_context,device_buffer,pinned_buffer,cuda_stream}.hpp.
 * ---------------------------------------------------------------------------------------- */
typedef struct zcgvs_device_info {
    char name[256];
    char arch[64];             /* gcnArchName, e.g. "gfx950:sramecc+:xnack-" */
    size_t total_memory;       /* bytes */
    int compute_units;
    int clock_khz;
    int memory_clock_khz;
    int memory_bus_width;      /* bits */
    int l2_cache_bytes;
    int major;
    int minor;
    /* 2 * memory clock * bus width / 8, the formula of include/zcgvs/core/cuda_context.hpp:20-23 */
    double peak_bandwidth_gbs;
} zcgvs_device_info;

int zcgvs_device_count(int* count);
int zcgvs_set_device(int device);                       /* src/core/cuda_context.cpp:9 */
int zcgvs_get_device(int* device);
int zcgvs_device_query(int device, zcgvs_device_info* out); /* src/core/cuda_context.cpp:23-45 */
int zcgvs_device_synchronize(void);

/* Measured HBM rates of the current device, the achievable counterpart of peak_bandwidth_gbs
 * (the reference derives only that nominal peak, include/zcgvs/core/cuda_context.hpp:20-23, and
 * prints each scan's GB/s against it, apps/bench_kernels.cu:133-143). A streaming read and a
 * streaming copy over two `bytes`-byte buffers (at least 64 MiB; use several times the 256 MiB
 * last-level cache) are each timed `iterations` times at a few grid sizes; the best launch gives
 * *read_gbs (bytes read per second) and *copy_gbs (bytes read + written per second), in 1e9
 * bytes/s. Allocates, frees and synchronizes: never call it inside a graph capture. */
int zcgvs_measure_hbm_bandwidth(size_t bytes, int iterations, double* read_gbs, double* copy_gbs);

int zcgvs_malloc(void** ptr, size_t bytes);           /* device_buffer.hpp:40-56 */
int zcgvs_free(void* ptr);
int zcgvs_host_alloc(void** ptr, size_t bytes);       /* pinned_buffer.hpp:14-67 */
int zcgvs_host_free(void* ptr);
int zcgvs_memcpy_h2d(void* dst, const void* src, size_t bytes, zcgvs_stream_t stream);
int zcgvs_memcpy_d2h(void* dst, const void* src, size_t bytes, zcgvs_stream_t stream);
int zcgvs_memcpy_d2d(void* dst, const void* src, size_t bytes, zcgvs_stream_t stream);
/* Not graph-capture safe (records a memset node); use zcgvs_fill_u32 inside captures. */
int zcgvs_memset(void* dst, int value, size_t bytes, zcgvs_stream_t stream);
/* Fills `count` 32-bit words with `value` using a kernel (capture safe). */
int zcgvs_fill_u32(void* dst, uint32_t value, size_t count, zcgvs_stream_t stream);

int zcgvs_stream_create(zcgvs_stream_t* stream);      /* cuda_stream.hpp:9-43 */
int zcgvs_stream_destroy(zcgvs_stream_t stream);
int zcgvs_stream_synchronize(zcgvs_stream_t stream);

int zcgvs_event_create(zcgvs_event_t* event);
int zcgvs_event_destroy(zcgvs_event_t event);
int zcgvs_event_record(zcgvs_event_t event, zcgvs_stream_t stream);
int zcgvs_event_synchronize(zcgvs_event_t event);
int zcgvs_event_elapsed_ms(float* ms, zcgvs_event_t start, zcgvs_event_t end);

/* Stream capture into an instantiated graph (src/search/searcher.cpp:305-342). Capture uses
 * the thread-local mode. end_capture instantiates and returns the executable graph. */
int zcgvs_graph_begin_capture(zcgvs_stream_t stream);
int zcgvs_graph_end_capture(zcgvs_stream_t stream, zcgvs_graph_t* graph);
int zcgvs_graph_launch(zcgvs_graph_t graph, zcgvs_stream_t stream);
int zcgvs_graph_destroy(zcgvs_graph_t graph);

/* ------------------------------------------------------------------------------------------
 * Kernel launchers. Each one replaces the reference launcher named in its comment, with the
 * same argument order and meaning, a HIP stream in place of the CUDA stream, and a status code
 * in place of exceptions.
 * ---------------------------------------------------------------------------------------- */

/* src/cuda/similarity.cu:345-398 launchSimilarity.
 * d_scores[q * doc_count + doc] = score of query q against document doc.
 * d_queries: [batch, dim] float32, or [batch, ceil(dim/32)] packed uint32 words for a BINARY
 * corpus (bit b of word w = dimension 32w+b, set iff value >= 0). Masked documents (mask byte 0)
 * score -FLT_MAX. Cosine is a raw dot product (inputs are assumed L2-normalized). L2 scores are
 * the negated squared distance. Binary scores are (dim - 2*hamming) / dim. Unmasked cosine/dot
 * batches of at least 4 float32/float16 queries with dim 128, 256, 384 or 512 are computed on the
 * matrix cores (float32 products and sums in another order: equal to the scalar loop within
 * float32 rounding). */
int zcgvs_launch_similarity(const void* d_corpus, int dtype, float scale, int doc_count, int dim,
                            const void* d_queries, int batch, const uint8_t* d_mask, int metric,
                            float* d_scores, zcgvs_stream_t stream);

/* Same contract as zcgvs_launch_similarity for an int8 corpus in ZCGVS_INT8_PER_VECTOR mode:
 * d_corpus [doc_count, dim] int8 with d_row_scales [doc_count]; d_queries [batch, dim] int8 with
 * d_query_scales [batch]. Metric must be COSINE or DOT. No reference counterpart. Scores are
 * (float)(int32 dot) * (s_q * s_r) on every path (unmasked batches of at least 8 queries over a
 * whole number of 64-row tiles with dim 256-1024 run on the matrix cores). */
int zcgvs_launch_similarity_i8i8(const int8_t* d_corpus, const float* d_row_scales,
                                 int doc_count, int dim, const int8_t* d_queries,
                                 const float* d_query_scales, int batch, const uint8_t* d_mask,
                                 int metric, float* d_scores, zcgvs_stream_t stream);

int zcgvs_similarity_query_tile(void);                                /* similarity.cu:309 */
size_t zcgvs_similarity_shared_bytes(int dtype, int dim, int batch);  /* similarity.cu:337-343 */

/* src/cuda/topk.cu:112-130 sizing helpers. zcgvs_topk_scratch_elements is the per-query element
 * count of EACH of the four scratch buffers zcgvs_launch_topk takes. */
int zcgvs_topk_tile_size(void);
int zcgvs_topk_merge_tile(void);
int zcgvs_topk_max_k(void);
int zcgvs_topk_block_count(int doc_count);
int zcgvs_topk_scratch_elements(int doc_count, int k);

/* src/cuda/topk.cu:132-189 launchTopK. Selects the k best of each [batch, doc_count] score row,
 * descending, lowest index first on equal scores. Scratch buffers are each
 * batch * zcgvs_topk_scratch_elements(doc_count, k) elements. k <= zcgvs_topk_max_k() and
 * k <= doc_count or ZCGVS_ERR_INVALID_ARGUMENT. */
int zcgvs_launch_topk(const float* d_scores, int doc_count, int k, int batch, int* d_out_indices,
                      float* d_out_values, float* d_scratch_values_a, int* d_scratch_indices_a,
                      float* d_scratch_values_b, int* d_scratch_indices_b,
                      zcgvs_stream_t stream);

/* src/cuda/rescore.cu:83-130 launchGatherRescore / rescoreSharedBytes.
 * d_values[q * C + slot] = exact score of corpus row d_candidate_indices[q * C + slot] against
 * float32 query q; an index < 0 or >= doc_count gives -FLT_MAX. BINARY storage is rejected. */
size_t zcgvs_rescore_shared_bytes(int dim);
int zcgvs_launch_gather_rescore(const void* d_corpus, int dtype, float scale, int doc_count,
                                int dim, const float* d_queries, int batch,
                                const int* d_candidate_indices, int candidate_count, int metric,
                                float* d_values, zcgvs_stream_t stream);

/* src/cuda/rescore.cu:132-146 launchRemapIndices. */
int zcgvs_launch_remap_indices(const int* d_candidate_indices, const int* d_local_indices,
                               int candidate_count, int k, int batch, int* d_out_indices,
                               zcgvs_stream_t stream);

/* src/cuda/lexical.cu:78-92 launchBm25. Scatter-adds the posting weights of the query's terms
 * into d_scores (zeroed by the caller). Terms < 0 are skipped, as are documents outside
 * [0, doc_count); term ids must be below the index's vocabulary size, as in the reference.
 * Terms are accumulated in slot order, so every document's sum is formed in the same order on
 * every run. */
int zcgvs_launch_bm25(const int64_t* d_offsets, const int* d_docs, const float* d_weights,
                      const int* d_query_terms, int term_count, int doc_count, float* d_scores,
                      zcgvs_stream_t stream);

/* Batched form of zcgvs_launch_bm25: d_query_terms [batch, term_stride], d_scores
 * [batch, doc_count] (zeroed by the caller). One launch per term slot instead of one per
 * (query, slot) as src/search/searcher.cpp:241-249 does. */
int zcgvs_launch_bm25_batched(const int64_t* d_offsets, const int* d_docs,
                              const float* d_weights, const int* d_query_terms, int term_stride,
                              int batch, int doc_count, float* d_scores, zcgvs_stream_t stream);

/* Slice table of a lexical index whose postings ascend strictly by document (the
 * ZCGVS_SEARCH_SORTED_POSTINGS layout): d_table[t * S + c] = the number of term t's postings whose
 * document is below c * 4096 for c < S - 1, and below doc_count for c = S - 1, with
 * S = ceil(doc_count / 4096) + 1 (doc_count <= 2^31 - 1). Built once per index (one binary search
 * per entry), it lets every hybrid search take its terms' 4096-document slice bounds from the
 * table (zcgvs_search_desc.lex_slice_table). No reference counterpart: the reference's BM25
 * (src/cuda/lexical.cu:17-42) scatters every posting with atomics and keeps no such table.
 * zcgvs_lexical_slice_table_bytes returns 0 for an empty index or too many documents. */
size_t zcgvs_lexical_slice_table_bytes(int vocab_size, int64_t doc_count);
int zcgvs_build_lexical_slice_table(const int64_t* d_offsets, const int* d_docs, int vocab_size,
                                    int64_t doc_count, uint32_t* d_table, zcgvs_stream_t stream);

/* src/cuda/lexical.cu:94-105 launchMaxPositive: *d_max = max(*d_max, max_i values[i]) for
 * values >= 0 (caller zeroes *d_max). */
int zcgvs_launch_max_positive(const float* d_values, int count, float* d_max,
                              zcgvs_stream_t stream);

/* src/cuda/lexical.cu:107-123 launchFuseScores, in place:
 * dense[i] = weight * dense[i] + (1 - weight) * lexical[i] * (max > 0 ? 1/max : 0). */
int zcgvs_launch_fuse_scores(float* d_dense, const float* d_lexical, const float* d_lexical_max,
                             float weight, int count, zcgvs_stream_t stream);

/* src/cuda/convert.cu:55-93 launchConvertF32ToF16 / launchConvertF32ToI8 / launchPackBinary. */
int zcgvs_launch_convert_f32_to_f16(const float* d_src, void* d_dst_half, size_t count,
                                    zcgvs_stream_t stream);
int zcgvs_launch_convert_f32_to_i8(const float* d_src, void* d_dst_int8, size_t count,
                                   float scale, zcgvs_stream_t stream);
int zcgvs_launch_pack_binary(const float* d_src, void* d_dst_words, int rows, int dim,
                             zcgvs_stream_t stream);

/* Per-row symmetric int8 quantization (ZCGVS_INT8_PER_VECTOR): for every row,
 * s = max|x| / 127 (1.0 for an all-zero row), q = clamp(rint(x * (1/s)), -127, 127).
 * No reference counterpart; the reciprocal rule is that of src/cuda/convert.cu:25-32. */
int zcgvs_launch_quantize_rows_i8(const float* d_src, int rows, int dim, int8_t* d_dst,
                                  float* d_scales, zcgvs_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * Fused search: the whole device pipeline of src/search/searcher.cpp:209-285 (scan, optional
 * BM25 fusion, top-k, optional gather rescore + second top-k + remap) without a [batch, N]
 * score matrix. Only [batch, k] ids and scores are written.
 * ---------------------------------------------------------------------------------------- */
typedef struct zcgvs_store_desc {
    const void* data;          /* [doc_count, row_stride] device rows                         */
    int64_t doc_count;
    int dim;
    int dtype;                 /* enum zcgvs_dtype                                             */
    float scale;               /* matrix-wide int8 scale (ZCGVS_INT8_REFERENCE)               */
    const float* row_scales;   /* [doc_count] per-row int8 scales (ZCGVS_INT8_PER_VECTOR)     */
} zcgvs_store_desc;

typedef struct zcgvs_search_desc {
    zcgvs_store_desc corpus;   /* primary (scanned) store                                      */
    zcgvs_store_desc rescore;  /* rescore store; data == NULL disables the rescore stage        */
    const float* queries;      /* [batch, dim] float32 device queries                           */
    int batch;
    int k;                     /* final top-k, 1..zcgvs_topk_max_k()                            */
    int metric;                /* enum zcgvs_metric                                             */
    int int8_mode;             /* enum zcgvs_int8_mode (int8 corpus only)                       */
    const uint8_t* mask;       /* optional [doc_count] allow-mask                               */
    int rescore_candidates;    /* C; > 0 with rescore.data enables the rescore stage           */
    /* Hybrid lexical stage (src/search/searcher.cpp:235-259); enabled when query_terms != NULL
     * and lexical_stride > 0. */
    const int64_t* lex_offsets;
    const int* lex_docs;
    const float* lex_weights;
    int64_t lex_doc_count;
    int lex_vocab_size;        /* term ids >= this are skipped                                  */
    const int* query_terms;    /* [batch, lexical_stride] device term ids, -1 padded           */
    int lexical_stride;
    float dense_weight;
    int flags;                 /* zcgvs_search_flags bits; 0 for the default pipeline           */
    /* Optional slice table of the lexical index (zcgvs_build_lexical_slice_table over
     * lex_doc_count documents); with ZCGVS_SEARCH_SORTED_POSTINGS the BM25 stage reads its terms'
     * slice bounds from it instead of searching the postings. NULL: searched per call. */
    const uint32_t* lex_slice_table;
} zcgvs_search_desc;

/* zcgvs_search_desc.flags. ZCGVS_SEARCH_MATERIALIZE runs the reference-order pipeline (a
 * [batch, doc_count] score matrix in the workspace, then zcgvs_launch_topk) instead of the fused
 * scan; its workspace is correspondingly larger.
 * By default the BM25 stage scatters each query's postings term slot by term slot, which takes
 * postings in any order, like the reference's launchBm25 (src/cuda/lexical.cu:78-92).
 * ZCGVS_SEARCH_SORTED_POSTINGS states that every term's postings ascend strictly by document, one
 * per document (the layout the reference's index builder writes,
 * python/zcgvs_tools/build_lexical.py:147-163); the stage then reads them in document-range
 * slices instead, with no atomics and no clearing pass. Scores are bit-identical between the
 * two forms; with the flag set on postings that break the contract they are undefined.
 * ZCGVS_SEARCH_UNSORTED_POSTINGS names the default explicitly; setting it together with
 * ZCGVS_SEARCH_SORTED_POSTINGS is an invalid argument.
 * ZCGVS_SEARCH_FORCE_EXACT_PASS runs the exact device fallback (see zcgvs_search_topk) for every
 * query instead of only the ones whose candidate buffers overflowed; for tests and verification.
 * ZCGVS_SEARCH_TEST_TINY_SEGMENTS gives every candidate segment of the first attempt two slots, so
 * that almost every query overflows and takes the fallback through its overflow flag; for tests
 * only.
 * ZCGVS_SEARCH_TEST_HIGH_THRESHOLD sets the speculative threshold of a sketch-planned search (see
 * zcgvs_search_topk) to the best sampled score, so that most queries find fewer than k candidates
 * and take the fallback; for tests only (no effect on other plans).
 * ZCGVS_SEARCH_TEST_TINY_RERUN gives the rerun of flagged queries (sketch-planned and int8
 * matrix-core searches) segments of two slots per listed query when every query is listed, so
 * that, with ZCGVS_SEARCH_TEST_TINY_SEGMENTS listing almost every query, the reruns overflow too
 * and the last resort runs; for tests only. */
enum zcgvs_search_flags {
    ZCGVS_SEARCH_MATERIALIZE = 1,
    ZCGVS_SEARCH_UNSORTED_POSTINGS = 2,
    ZCGVS_SEARCH_SORTED_POSTINGS = 4,
    ZCGVS_SEARCH_FORCE_EXACT_PASS = 8,
    ZCGVS_SEARCH_TEST_TINY_SEGMENTS = 16,
    ZCGVS_SEARCH_TEST_HIGH_THRESHOLD = 32,
    ZCGVS_SEARCH_TEST_TINY_RERUN = 64
};

/* Bytes of device workspace zcgvs_search_topk needs for this descriptor (0 on error). */
size_t zcgvs_search_workspace_bytes(const zcgvs_search_desc* desc);

/* Runs the fused pipeline. d_out_indices/d_out_values are [batch, k]. The workspace must be
 * zcgvs_search_workspace_bytes(desc) bytes; its contents need no initialization. Capture safe.
 * The result is the exact top-k for every input: the scan keeps only candidates above a sampled
 * threshold in bounded per-workgroup buffers. A per-vector int8 search on the matrix cores, or a
 * binary search of 4 or more queries at 512 or 1024 bits, over a large corpus is sketch-planned: a first launch over
 * every 32nd block (64th for binary) records per slot (a row half of an int8 workgroup, a pair of a binary
 * workgroup's wavefronts) the best score of each query, and one scan of the whole corpus keeps
 * the keys at or above the j-th best of those scores (a threshold that is likely, not certain, to
 * lie below the k-th best key); other searches run threshold phases whose thresholds are certain
 * lower bounds. The search's last merge flags a query whose buffers overflowed (a corpus whose
 * best rows crowd into a few blocks) or which found fewer than k keys above a speculative
 * threshold; flagged queries are completed on the device, in the same call and stream, by the
 * exact fallback: for a sketch-planned search the scan runs once more over the whole corpus for
 * just those queries with a threshold that is a certain lower bound and the batch's candidate
 * buffers shared among them, and the selection is taken from that; for other scans, or when that
 * rerun overflows too, one workgroup per query selects over recomputed scores (a few corpus
 * reads).
 * zcgvs_search_overflow_flags tells which queries took the fallback. A search of at most four
 * queries selecting at most 1024 keys each (k, or rescore_candidates with a rescore store) that
 * no matrix-core scan takes reads the corpus in a single pass whose per-workgroup lists are exact
 * (selections above 32 keys merge groups of workgroups first); it never overflows.
 * Non-finite inputs: float32 rows of 256 or 384 dims searched with 32 to 128 queries per launch
 * are scanned on the bf16 matrix cores as exact three-part splits, where a row or query with an
 * infinite or NaN component scores NaN (it ranks last); every other scan follows the IEEE sum,
 * where such a score can be +inf and rank first. So with non-finite data the result can depend
 * on the batch size (the reference defines no order for non-finite scores either). */
int zcgvs_search_topk(const zcgvs_search_desc* desc, void* d_workspace, size_t workspace_bytes,
                      int* d_out_indices, float* d_out_values, zcgvs_stream_t stream);

/* No counterpart in the reference. For callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc): zcgvs_search_topk with
 * its workspace in a library-owned static device array of zcgvs_static_scratch_bytes() bytes
 * (64 MiB) per device instead of a caller's buffer. A search whose workspace
 * (zcgvs_search_workspace_bytes) exceeds that size is rejected with ZCGVS_ERR_INVALID_ARGUMENT;
 * nothing is allocated or freed, on the host's HIP side or the device. Every call on one device
 * shares that device's array: calls that overlap on one GPU (concurrent streams, threads) race
 * and must be serialized by the caller. The results equal zcgvs_search_topk's. The array's device
 * address is looked up on the first call on a device, or earlier by zcgvs_graph_begin_capture,
 * so a call recorded into a graph performs no lookup. */
size_t zcgvs_static_scratch_bytes(void);
int zcgvs_search_topk_noalloc(const zcgvs_search_desc* desc, int* d_out_indices, float* d_out_values,
                              zcgvs_stream_t stream);

/* Measurement hook: zcgvs_search_topk that also records events[2p] and events[2p + 1] on `stream`
 * immediately before and after the scan launches of phase p, for p < max_phases, and returns the
 * number of phases in *phases. A fused hybrid search also brackets its lexical (BM25) stage with
 * the next pair, events[2 * phases] and events[2 * phases + 1], when max_phases > *phases. The events must have been created with zcgvs_event_create. Not
 * meant for graph capture. No reference counterpart (the reference times the whole pipeline with
 * one event pair, src/search/searcher.cpp:358-365). */
int zcgvs_search_topk_profiled(const zcgvs_search_desc* desc, void* d_workspace,
                               size_t workspace_bytes, int* d_out_indices, float* d_out_values,
                               zcgvs_stream_t stream, zcgvs_event_t* events, int max_phases,
                               int* phases);

/* Corpus rows each scan phase of the fused pipeline visits for `desc` (rows[p] for p <
 * max_phases; the phase count in *phases; 0 phases when the pipeline materializes the score
 * matrix instead; one phase of doc_count rows for the single pass; the sample of rows from which a
 * filter scan in two phases takes its first threshold belongs to the launches of phase 0 and is not
 * counted). Host only; used to price the
 * scan launches. No reference counterpart. */
int zcgvs_search_phase_rows(const zcgvs_search_desc* desc, long long* rows, int max_phases,
                            int* phases);

/* Device address of the [batch] uint32 overflow flags inside a workspace laid out for `desc`,
 * valid after the stream has completed the search: non-zero when that query's candidate buffers
 * overflowed and its result came from the exact device fallback (the result is exact either way;
 * the flags are for monitoring). */
int zcgvs_search_overflow_flags(const zcgvs_search_desc* desc, void* d_workspace,
                                uint32_t** d_flags);

/* Device addresses, inside a workspace laid out for `desc`, of a sketch-planned search's sketch
 * state, valid after the stream has completed the search: the slot scores (*slots x batch
 * float32, slot-major: the best score of each query over the slot's rows, -inf for a slot that
 * saw none) and two [batch] threshold keys (a key is kept when it is at least the threshold):
 * the speculative one, ordered32(the *rank-th best slot score) << 32 (for a flagged query the
 * merge replaces it by its rerun's threshold), and the certain one, of the *width-th best slot
 * score. In a filter scan the slot scores are lower bounds of the rows' scores, and both thresholds are
 * the certain one (of all ones for a query of zeros, which that scan leaves to the last merge); where it
 * runs in two phases the speculative one is the first phase's. A search that is not sketch-planned sets
 * *slots and *rank to 0 and the addresses to
 * null. For monitoring and tests; no reference counterpart. */
int zcgvs_search_sketch_state(const zcgvs_search_desc* desc, void* d_workspace, float** d_slot_scores,
                              int* slots, int* rank, int* width, uint64_t** d_tau, uint64_t** d_tau_safe);

/* ------------------------------------------------------------------------------------------
 * Synthetic data on the device (benchmarks and large parity runs). Row r of a matrix generated
 * with `seed` depends only on (seed, r): a counter-based splitmix64 stream, Box-Muller in
 * double precision, rounded to float32, then L2-normalized in float32 in dimension order.
 * ---------------------------------------------------------------------------------------- */
int zcgvs_generate_normalized(float* d_out, int64_t rows, int dim, uint64_t seed,
                              int64_t row_offset, zcgvs_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * Embedding-model operators: from token ids to query vectors on the device, and their gradients.
 * No counterpart in the reference, whose QueryEmbedder runs a model outside its device code
 * (include/zcgvs/embed/query_embedder.hpp:8-15). A model's call in front of a search:
 * zcgvs_embedding_lookup (token rows, or the mean of each text's rows), zcgvs_gated_projection,
 * zcgvs_adapted_projection with float32 output, which is the `queries` of zcgvs_search_topk.
 *
 * Types: float32, float16 or bfloat16 operands (ZCGVS_DTYPE_F32 / F16 / BF16). Products and sums are
 * held in float32 whatever the type; results are rounded once, where they are written. Matrix products of
 * float32 operands are formed from exact parts of them, to within 2^-23 of each product; an infinite
 * operand may give NaN there where the formula gives an infinity. Matrices are
 * row-major with a row stride in elements (at least the row's length). Rows may start at any address
 * that is aligned to their element; rows whose address and stride are multiples of 16 bytes take the
 * faster kernels. The same inputs give the same bits on every call: no result depends on the order of
 * atomic operations. Outputs must not overlap inputs, except where a function says so.
 * Like the launchers, these functions are asynchronous on `stream`, allocate nothing, never
 * synchronize and may be recorded into a HIP graph. Workspaces need no initialization and must not be
 * shared by calls that can overlap; one of more bytes than asked for is fine.
 * ---------------------------------------------------------------------------------------- */
enum zcgvs_embedding_reduce { ZCGVS_EMBEDDING_SUM = 0, ZCGVS_EMBEDDING_MEAN = 1 };

/* A table of token rows and the tokens to look up.
 * A token counts when its id lies in [0, vocab) and differs from padding_id (-1: no padding id);
 * any other token stands for a row of zeros and has no gradient.
 * Without bags, output row j is scale * table[ids[j]]. With bag_offsets, output row r is scale times
 * the sum (or the mean over the tokens that count) of the rows of tokens bag_offsets[r] ..
 * bag_offsets[r + 1] - 1; a bag with no token that counts gives zeros. Offsets ascend and lie in
 * [0, token_count]. */
typedef struct zcgvs_embedding_desc {
    const void* table;           /* [vocab, dim] rows of `dtype` (not read by the gradient)      */
    int64_t table_stride;        /* elements from row to row; 0: dim                             */
    int vocab;
    int dim;                     /* at most 2^23                                                 */
    int dtype;                   /* of the table                                                 */
    const int* ids;              /* [token_count]                                                */
    int64_t token_count;         /* at most 2^28                                                 */
    const int64_t* bag_offsets;  /* [bag_count + 1], or NULL: one output row per token           */
    int64_t bag_count;           /* at most 2^31 - 1                                             */
    int reduce;                  /* enum zcgvs_embedding_reduce (with bags)                      */
    int padding_id;
    float scale;
} zcgvs_embedding_desc;

/* d_out [token_count or bag_count, dim]; out_dtype is the table's type or ZCGVS_DTYPE_F32;
 * out_stride 0: dim. */
int zcgvs_embedding_lookup(const zcgvs_embedding_desc* desc, void* d_out, int64_t out_stride,
                           int out_dtype, zcgvs_stream_t stream);

/* The gradient of zcgvs_embedding_lookup with respect to the table, from the gradient of its output
 * rows (d_out_gradient, of `gradient_dtype`): d_table_gradient[v] = scale * the sum of the output
 * gradients of v's tokens (with ZCGVS_EMBEDDING_MEAN each over its bag's counting tokens). Each
 * row's terms are added in a fixed grouping of the tokens' order.
 * accumulate == 0: every row of d_table_gradient [vocab, dim] is written, those of tokens that do not
 * occur with zeros. accumulate != 0: the sums are added to d_table_gradient and only rows of tokens
 * that occur are touched. table_gradient_dtype is gradient_dtype or ZCGVS_DTYPE_F32. */
size_t zcgvs_embedding_gradient_workspace_bytes(const zcgvs_embedding_desc* desc);
int zcgvs_embedding_gradient(const zcgvs_embedding_desc* desc, const void* d_out_gradient,
                             int64_t out_gradient_stride, int gradient_dtype, void* d_table_gradient,
                             int64_t table_gradient_stride, int table_gradient_dtype, int accumulate,
                             void* d_workspace, size_t workspace_bytes, zcgvs_stream_t stream);

/* Activations of the gated block: x * sigmoid(x); x * Phi(x) with the normal distribution function
 * Phi; and the latter's usual tanh approximation 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))). */
enum zcgvs_activation { ZCGVS_ACT_SILU = 0, ZCGVS_ACT_GELU = 1, ZCGVS_ACT_GELU_TANH = 2 };

/* The gated half of a feed-forward block: out = act(x gate^T) * (x up^T), both products, the
 * activation and the product in one kernel. All matrices hold `dtype`. */
typedef struct zcgvs_gated_desc {
    const void* x;         /* [rows, dim]                                                  */
    int64_t x_stride;      /* 0: dim                                                       */
    const void* gate;      /* [hidden, dim]                                                */
    const void* up;        /* [hidden, dim]; one [2 hidden, dim] matrix may hold both       */
    int64_t weight_stride; /* of gate and up; 0: dim                                       */
    int64_t rows;          /* at most 2^30                                                 */
    int dim;
    int hidden;
    int dtype;
    int activation;        /* enum zcgvs_activation                                        */
} zcgvs_gated_desc;

/* d_out [rows, hidden] of desc->dtype; out_stride 0: hidden. */
int zcgvs_gated_projection(const zcgvs_gated_desc* desc, void* d_out, int64_t out_stride,
                           zcgvs_stream_t stream);

/* The gradient of zcgvs_gated_projection. With g = x gate^T and u = x up^T (computed again, nothing of
 * the forward pass is kept): dg = d_out * u * act'(g), du = d_out * act(g), and
 *     x_gradient [rows, dim] = dg gate + du up,
 *     gate_gradient [hidden, dim] = dg^T x,   up_gradient [hidden, dim] = du^T x,
 * all of desc->dtype. dg and du are rounded to desc->dtype between the products, as tensors of a model
 * of that type are (float16: to an infinity beyond 65504, so scale the loss as for stored tensors).
 * x_gradient may be NULL (not wanted), and so may gate_gradient and up_gradient, both together. A stride
 * of 0 is the row's length; gate_gradient and up_gradient share theirs. */
size_t zcgvs_gated_gradient_workspace_bytes(const zcgvs_gated_desc* desc);
int zcgvs_gated_gradient(const zcgvs_gated_desc* desc, const void* d_out_gradient,
                         int64_t out_gradient_stride, void* d_x_gradient, int64_t x_gradient_stride,
                         void* d_gate_gradient, void* d_up_gradient, int64_t weight_gradient_stride,
                         void* d_workspace, size_t workspace_bytes, zcgvs_stream_t stream);

/* A projection that every row shares, beside low-rank adapters of which each row names one:
 *     out[r] = x[r] weight^T + scales[a] * (x[r] down[a]^T) up[a]^T,   a = adapter_ids[r].
 * A row whose id lies outside [0, adapter_count) has no adapter, as have all rows where adapter_ids is
 * NULL. Of adapter a the first ranks[a] of max_rank rows of down[a] and columns of up[a] count; what
 * lies beyond is not used. Rows may come in any order; rows of one adapter next to each other (the
 * tokens of a request) cost least. Of the other rows and their adapters a row's result takes nothing, also
 * where those hold infinities or NaN; but how many they are and how they mix chooses the kernel and the
 * order of a row's sums, so in another batch it may be rounded otherwise. */
typedef struct zcgvs_adapted_desc {
    const void* x;          /* [rows, dim]                                                  */
    int64_t x_stride;       /* 0: dim                                                       */
    const void* weight;     /* [out_dim, dim]                                               */
    int64_t weight_stride;  /* 0: dim                                                       */
    int64_t rows;           /* at most 2^29                                                 */
    int dim;
    int out_dim;
    int dtype;              /* of x, weight, down and up                                    */
    const void* down;       /* [adapter_count, max_rank, dim]                               */
    const void* up;         /* [adapter_count, out_dim, max_rank]                           */
    int adapter_count;
    int max_rank;           /* at most zcgvs_adapted_max_rank()                             */
    const int* ranks;       /* [adapter_count], clamped to [0, max_rank]; NULL: max_rank    */
    const float* scales;    /* [adapter_count]; NULL: 1                                     */
    const int* adapter_ids; /* [rows]; NULL: no adapters (down and up are not read)         */
} zcgvs_adapted_desc;

int zcgvs_adapted_max_rank(void); /* 128 */
/* d_out [rows, out_dim]; out_dtype is desc->dtype or ZCGVS_DTYPE_F32 (the `queries` of a search);
 * out_stride 0: out_dim. */
size_t zcgvs_adapted_projection_workspace_bytes(const zcgvs_adapted_desc* desc);
int zcgvs_adapted_projection(const zcgvs_adapted_desc* desc, void* d_out, int64_t out_stride,
                             int out_dtype, void* d_workspace, size_t workspace_bytes,
                             zcgvs_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * Operators of an encoder block: what stands between the token rows of zcgvs_embedding_lookup and
 * the row that is pooled, beside zcgvs_gated_projection. No counterpart in the reference, whose
 * QueryEmbedder runs a model outside its device code (include/zcgvs/embed/query_embedder.hpp:8-15).
 * What the embedding-model operators above promise of types, sums, strides, alignment, streams,
 * workspaces and equal bits on every call holds for these as well.
 * ---------------------------------------------------------------------------------------- */

/* Root-mean-square norm of the sum of two rows (of one, where residual is NULL):
 *     s = x + residual,   y = s / sqrt(mean(s^2) + eps) * (weight + weight_offset).
 * s and y are formed in float32 of the operands as stored; the norm is that of the float32 sum, also where
 * a rounded copy of the sum is written. eps > 0 keeps rows of zeros finite; a row whose squares pass
 * float32's range gives zeros. */
typedef struct zcgvs_norm_desc {
    const void* x;          /* [rows, dim]                                                  */
    int64_t x_stride;       /* 0: dim                                                       */
    const void* residual;   /* [rows, dim], or NULL: none                                   */
    int64_t residual_stride; /* 0: dim                                                      */
    const void* weight;     /* [dim], or NULL: ones                                         */
    int64_t rows;           /* at most 2^30                                                 */
    int dim;                /* at most zcgvs_residual_norm_max_dim()                        */
    int dtype;              /* of x, residual and weight                                    */
    float weight_offset;    /* 1 for weights stored as their distance from one              */
    float eps;              /* at least 0                                                   */
} zcgvs_norm_desc;

int zcgvs_residual_norm_max_dim(void); /* 16384 */
/* d_out [rows, dim]: out_dtype is desc->dtype, ZCGVS_DTYPE_F32 or ZCGVS_DTYPE_I8. int8 rows are those of
 * zcgvs_launch_quantize_rows_i8 over y: q = max|y| / 127 (1 for a row of zeros) goes to d_out_scales [rows],
 * code = clamp(rint(y * (1/q)), -127, 127) to d_out: operands of zcgvs_linear, or rows of a
 * ZCGVS_INT8_PER_VECTOR store. d_out_scales is not read or written otherwise. d_sum, NULL or [rows, dim] of
 * desc->dtype, takes s, rounded once; it may be x or residual itself (with the same stride), and d_out may
 * be x or residual where it has their type and stride and d_sum is another buffer. */
int zcgvs_residual_norm(const zcgvs_norm_desc* desc, void* d_out, int64_t out_stride, int out_dtype,
                        float* d_out_scales, void* d_sum, int64_t sum_stride, zcgvs_stream_t stream);

/* The gradient of zcgvs_residual_norm (float output) from that of y and, where d_sum_gradient is not NULL,
 * that of s. With u = s / sqrt(mean(s^2) + eps) and g = d_out_gradient * (weight + weight_offset):
 *     x_gradient [rows, dim] = (g - u mean(g u)) / sqrt(mean(s^2) + eps) + d_sum_gradient,
 *     weight_gradient [dim] = the sum over rows of d_out_gradient * u,
 * all of desc->dtype. x_gradient is that of x and of residual alike. desc may give x and residual, or as x the
 * sum that the forward call wrote. Either output may be NULL (not wanted); x_gradient may be d_out_gradient or
 * d_sum_gradient itself (with the same stride). No rows: weight_gradient is zeros. */
size_t zcgvs_residual_norm_gradient_workspace_bytes(const zcgvs_norm_desc* desc);
int zcgvs_residual_norm_gradient(const zcgvs_norm_desc* desc, const void* d_out_gradient,
                                 int64_t out_gradient_stride, const void* d_sum_gradient,
                                 int64_t sum_gradient_stride, void* d_x_gradient, int64_t x_gradient_stride,
                                 void* d_weight_gradient, void* d_workspace, size_t workspace_bytes,
                                 zcgvs_stream_t stream);

/* A projection with its epilogue: out = act(x weight^T + bias) + residual, act one of enum
 * zcgvs_activation or ZCGVS_ACT_NONE.
 * int8 operands (dtype ZCGVS_DTYPE_I8, at most 131072 codes a row): x weight^T is the exact sum of the codes'
 * products times x_scales[row] * weight_scales[column] (in this order). */
enum { ZCGVS_ACT_NONE = 3 };

typedef struct zcgvs_linear_desc {
    const void* x;           /* [rows, dim]                                                  */
    int64_t x_stride;        /* 0: dim                                                       */
    const void* weight;      /* [out_dim, dim]                                               */
    int64_t weight_stride;   /* 0: dim                                                       */
    int64_t rows;            /* at most 2^30                                                 */
    int dim;
    int out_dim;
    int dtype;               /* of x and weight: float32, float16, bfloat16 or int8          */
    int activation;
    int epilogue_dtype;      /* of bias and residual: dtype, or with int8 operands a float type */
    const float* x_scales;      /* [rows] (int8)                                             */
    const float* weight_scales; /* [out_dim] (int8)                                          */
    const void* bias;        /* [out_dim], or NULL: none                                     */
    const void* residual;    /* [rows, out_dim], or NULL: none                               */
    int64_t residual_stride; /* 0: out_dim                                                   */
} zcgvs_linear_desc;

/* d_out [rows, out_dim]; out_dtype is epilogue_dtype or ZCGVS_DTYPE_F32; out_stride 0: out_dim. d_out may be
 * the residual itself where it has its type and stride. */
int zcgvs_linear(const zcgvs_linear_desc* desc, void* d_out, int64_t out_stride, int out_dtype,
                 zcgvs_stream_t stream);

/* The gradient of zcgvs_linear (float operands) from that of its output. With z = x weight^T + bias (computed
 * again; not needed without an activation) and dz = d_out_gradient * act'(z):
 *     x_gradient [rows, dim] = dz weight,   weight_gradient [out_dim, dim] = dz^T x,
 *     bias_gradient [out_dim] = the sum of dz over rows,
 * all of desc->dtype; that of the residual is d_out_gradient itself. dz is rounded to desc->dtype between the
 * products where there is an activation. Any output may be NULL (not wanted). */
size_t zcgvs_linear_gradient_workspace_bytes(const zcgvs_linear_desc* desc);
int zcgvs_linear_gradient(const zcgvs_linear_desc* desc, const void* d_out_gradient, int64_t out_gradient_stride,
                          void* d_x_gradient, int64_t x_gradient_stride, void* d_weight_gradient,
                          int64_t weight_gradient_stride, void* d_bias_gradient, void* d_workspace,
                          size_t workspace_bytes, zcgvs_stream_t stream);

/* Where the query rows of a text stand among its keys: from the first one on, or so that the last one
 * stands at the last key. */
enum zcgvs_attention_align { ZCGVS_ATTENTION_FIRST = 0, ZCGVS_ATTENTION_LAST = 1 };

/* Attention within each text of a batch. Query row i of text t stands at position p = i (or
 * p = key_count - query_count + i), key j of the text at position j; with head h of the query and key head
 * h / (heads / kv_heads):
 *     c = scale * q_i . k_j,  with cap > 0: c = cap * tanh(c / cap)
 *     s_j = c - slopes[h] * |j - p| + distance_bias[h][clamp(j - p, -max_distance, max_distance) + max_distance]
 *     out_i = sum_j softmax(s)_j v_j   over the keys that i sees.
 * A query row sees the keys of its own text; with `causal` those at j <= p and, where prefix_lengths is
 * given, those at j < prefix_lengths[t] as well. A distance_bias of -1e30 or less leaves the keys at its distances
 * out, as minus infinity does. A row that sees no key gives zeros.
 * The rows of text t are q_offsets[t] .. q_offsets[t + 1] - 1 (offsets ascend and lie in [0, q_rows]), or
 * with q_offsets NULL t * (q_rows / texts) on (q_rows a multiple of texts): one query row a text, or a padded
 * batch. Of these the first q_lengths[t] count (clamped to [0, the text's rows]; NULL: all); the rest are padding:
 * their output rows are zeros, and so are the gradients of padding rows. Rows of no text (before the first
 * offset, behind the last) are neither read nor written. Likewise for the keys.
 * Padding rows, rows of no text and other texts may hold anything, infinities and NaN included. A key of the
 * row's own text that only the causal mask or a bias hides must be finite, as must the queries that do not see
 * a key for that key's gradient.
 * A call may take (q_rows / 64 + 2 * texts) * heads workgroups, its gradient also (k_rows / 64 + texts) * kv_heads:
 * calls that need 2^24 of either are refused. */
typedef struct zcgvs_attention_desc {
    const void* q;             /* [q_rows, heads, head_dim]                                     */
    int64_t q_stride;          /* elements from row to row; 0: heads * head_dim                 */
    const void* k;             /* [k_rows, kv_heads, head_dim]                                  */
    int64_t k_stride;          /* 0: kv_heads * head_dim                                        */
    const void* v;             /* [k_rows, kv_heads, head_dim]                                  */
    int64_t v_stride;          /* 0: kv_heads * head_dim                                        */
    int64_t q_rows;            /* at most 2^28                                                  */
    int64_t k_rows;            /* at most 2^28                                                  */
    int64_t texts;             /* at most 2^24                                                  */
    const int64_t* q_offsets;  /* [texts + 1], or NULL                                          */
    const int64_t* k_offsets;  /* [texts + 1], or NULL                                          */
    const int* q_lengths;      /* [texts], or NULL                                              */
    const int* k_lengths;      /* [texts], or NULL                                              */
    int heads;                 /* a multiple of kv_heads, at most 1024                          */
    int kv_heads;
    int head_dim;              /* at most zcgvs_attention_max_head_dim()                        */
    int dtype;                 /* of q, k, v and distance_bias                                  */
    int q_align;               /* enum zcgvs_attention_align                                    */
    int causal;
    const int* prefix_lengths; /* [texts] (causal), or NULL                                     */
    float scale;               /* finite                                                        */
    float cap;                 /* 0: none. 16-bit: c within 2^-21 cap up to caps of 64, 2^-19 c above */
    const float* slopes;       /* [heads], or NULL: none                                        */
    const void* distance_bias; /* [heads, 2 * max_distance + 1], or NULL: none                  */
    int max_distance;          /* at most zcgvs_attention_max_distance()                        */
} zcgvs_attention_desc;

int zcgvs_attention_max_head_dim(void); /* 128 */
int zcgvs_attention_max_distance(void); /* 512 */
/* d_out [q_rows, heads, head_dim] of desc->dtype (out_stride 0: heads * head_dim). d_lse, NULL or
 * [q_rows, heads] float32, takes each row's logarithm of the sum of exponentials of s (minus infinity where
 * it sees no key), which the gradient needs. With 16-bit operands the softmax's exponentials are rounded to
 * that type for the product with v; their sum is that of the unrounded ones. */
size_t zcgvs_attention_workspace_bytes(const zcgvs_attention_desc* desc);
int zcgvs_attention(const zcgvs_attention_desc* desc, void* d_out, int64_t out_stride, float* d_lse,
                    void* d_workspace, size_t workspace_bytes, zcgvs_stream_t stream);

/* The gradient of zcgvs_attention from that of its output, with what the forward call wrote (d_out with
 * out_stride, d_lse). q_gradient, k_gradient and v_gradient have the shapes of q, k and v and desc->dtype;
 * distance_bias_gradient (NULL: not wanted) that of distance_bias and desc->dtype. The softmax and its
 * gradient are rounded to desc->dtype between the products (float16: to an infinity beyond 65504 and to
 * multiples of 2^-24 below 2^-14, so scale the loss as for stored tensors; probabilities over more than 2^14
 * keys lose bits). A stride of 0 is the row's length. */
size_t zcgvs_attention_gradient_workspace_bytes(const zcgvs_attention_desc* desc);
int zcgvs_attention_gradient(const zcgvs_attention_desc* desc, const void* d_out, int64_t out_stride,
                             const float* d_lse, const void* d_out_gradient, int64_t out_gradient_stride,
                             void* d_q_gradient, int64_t q_gradient_stride, void* d_k_gradient,
                             int64_t k_gradient_stride, void* d_v_gradient, int64_t v_gradient_stride,
                             void* d_distance_bias_gradient, void* d_workspace, size_t workspace_bytes,
                             zcgvs_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* ZCGVS_HIP_H */
