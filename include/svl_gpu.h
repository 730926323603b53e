/*
 * svl_gpu.h -- C ABI of the B200 (sm_100a) text-embedding and exact-search
 * library (libsvl_gpu.so).
 *
 * The library replaces the bodies of these reference (Seldon Vault Lite,
 * Rust) entry points; each declaration below names the one it stands behind:
 *
 *   TextModel::new / from_files        src/model/text.rs:104-126, weights.rs:125-241
 *   TextModel::forward                 src/model/text.rs:150
 *   TextModel::forward_with_features   src/model/text.rs:167
 *   TextModel::embed_ids               src/model/text.rs:546
 *   ForwardOutput::embedding           src/model/text.rs:72 (truncate_and_normalize)
 *   vector::rank                       src/index/vector.rs:17-97
 *   Index::search (vector mode)        src/index/mod.rs:325-388
 *   Chunk::new normalisation           src/storage/model.rs:325, 546-581
 *
 * Conventions (mirroring the reference):
 *   - every call returns an svl_status; the enumerators map one to one onto
 *     the reference's Error variants (src/error.rs:24-36).  A human-readable
 *     message is written to `err` (NUL-terminated, truncated to err_len) when
 *     err is non-NULL.  No call aborts the process.
 *   - inputs are borrowed; outputs are caller-owned buffers of the stated
 *     size; the library never retains caller pointers after returning.
 *   - plain pointers and sizes only: no C++ or PyTorch types cross the ABI.
 *   - an svl_model / svl_index is bound to one CUDA device.  Calls on one
 *     handle are serialised by an internal mutex, so a handle may be shared
 *     between threads (TextModel is Send + Sync in the reference).
 *   - *_device entry points take device pointers and an optional cudaStream_t
 *     (passed as void*; NULL = the handle's own stream) and return once the
 *     work is queued; the host-pointer entry points copy in, run and copy out
 *     synchronously.
 */
#ifndef SVL_GPU_H
#define SVL_GPU_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SVL_ABI_VERSION 1u

/* src/error.rs:24-36 */
typedef enum svl_status {
  SVL_OK = 0,
  SVL_USAGE = 1,           /* Error::Usage         */
  SVL_IO = 2,              /* Error::Io            */
  SVL_CORRUPT = 3,         /* Error::Corrupt       */
  SVL_LIMIT_EXCEEDED = 4,  /* Error::LimitExceeded */
  SVL_UNSUPPORTED = 5,     /* Error::Unsupported   */
  SVL_INTERNAL = 6         /* Error::Internal      */
} svl_status;

/* src/model/config.rs:55-70 */
typedef enum svl_layer_type { SVL_LAYER_SLIDING = 0, SVL_LAYER_FULL = 1 } svl_layer_type;

typedef struct svl_layer_config {
  uint32_t layer_type;           /* svl_layer_type */
  uint32_t head_dim;
  uint32_t num_key_value_heads;
} svl_layer_config;

/* Validated text configuration (TextConfig, src/model/config.rs:76-97).  The
 * host side parses config.json (config.rs:112-269) and fills this struct;
 * embedding_scale = sqrt(hidden_size) and ple_scale = 1 / embedding_scale are
 * the f32 values config.rs:241-242 computes. */
typedef struct svl_text_config {
  uint32_t vocab_size;
  uint32_t hidden_size;
  uint32_t intermediate_size;
  uint32_t num_hidden_layers;
  uint32_t num_attention_heads;
  uint32_t hidden_size_per_layer_input;
  uint32_t embedding_dim;
  uint32_t max_position_embeddings;
  uint32_t sliding_window;       /* inclusive two-sided radius */
  int64_t pad_token_id;          /* -1 when the config declares none */
  float rms_norm_eps;
  float embedding_scale;
  float ple_scale;
  float full_rope_theta;
  float sliding_rope_theta;
  const svl_layer_config* layers; /* num_hidden_layers entries */
} svl_text_config;

/* SVL_DTYPE_F16 is an operand type of the operators below; weight tensors are F32 or BF16. */
typedef enum svl_dtype { SVL_DTYPE_F32 = 0, SVL_DTYPE_BF16 = 1, SVL_DTYPE_F16 = 2 } svl_dtype;

/* One named weight tensor in host memory (a Safetensors entry,
 * src/binary/safetensors.rs:69-123).  BF16 data is widened to FP32 exactly
 * (src/binary/bf16.rs:40) while it is uploaded. */
typedef struct svl_tensor_view {
  const char* name;              /* e.g. "language_model.layers.0.mlp.up_proj.weight" */
  const void* data;
  uint32_t dtype;                /* svl_dtype */
  uint32_t ndim;
  uint64_t shape[4];
} svl_tensor_view;

/* Soft-token override of a row range of one sequence
 * (TextModel::forward_with_features, src/model/text.rs:167, 226-275). */
typedef struct svl_feature_span {
  uint32_t sequence;             /* index into the batch */
  uint32_t start;                /* first row within the sequence */
  uint32_t count;                /* rows replaced (>= 1) */
  uint32_t reserved;
  uint64_t feature_offset;       /* first float of this span in `features` */
} svl_feature_span;

typedef struct svl_model svl_model;
typedef struct svl_index svl_index;

/* ---------------------------------------------------------------- model -- */

/* Library ABI version (SVL_ABI_VERSION). */
uint32_t svl_abi_version(void);

/* Number of visible CUDA devices, or a negative value on error. */
int svl_device_count(void);

/* TextModel::new (text.rs:117) over TextWeights::decode (weights.rs:125-189):
 * checks the tensor inventory against the configuration (missing, extra
 * "language_model." tensor, shape mismatch -> SVL_CORRUPT; non-finite weight
 * -> SVL_CORRUPT), uploads the weights to `device` in FP32 and builds the
 * fused device layouts.  Weights are copied; `tensors` may be freed after. */
int svl_model_create(const svl_text_config* config, const svl_tensor_view* tensors,
                     size_t n_tensors, int device, svl_model** out, char* err, size_t err_len);
void svl_model_destroy(svl_model* model);

/* Arithmetic of the encoder's tensor-core products (no counterpart in the
 * reference, whose scalar path is FP32 throughout):
 *   SVL_PRECISION_FAST  (default) every projection and attention product on
 *       11-bit-significand operands (FP16 with power-of-two scales, or TF32)
 *       accumulated in FP32: the fastest path.
 *   SVL_PRECISION_SPLIT each operand x is split into hi = TF32(x) and
 *       lo = TF32(x - hi) and every projection accumulates hi*hi + hi*lo +
 *       lo*hi in one TF32 product over three times the reduction width
 *       (~22-bit products); attention runs in FP32 on the CUDA cores.  For
 *       trained weights whose activations amplify rounding, at several times
 *       the cost of the default.
 * svl_model_create takes SVL_PRECISION_SPLIT when the environment variable
 * SVL_PRECISION is "split" at creation, else SVL_PRECISION_FAST. */
typedef enum svl_precision { SVL_PRECISION_FAST = 0, SVL_PRECISION_SPLIT = 1 } svl_precision;

typedef struct svl_model_options {
  uint32_t precision;            /* svl_precision */
  uint32_t reserved[7];          /* zero */
} svl_model_options;

/* svl_model_create with explicit options (NULL = defaults, environment
 * ignored).  An unknown precision or non-zero reserved word -> SVL_USAGE. */
int svl_model_create_ex(const svl_text_config* config, const svl_tensor_view* tensors,
                        size_t n_tensors, int device, const svl_model_options* options,
                        svl_model** out, char* err, size_t err_len);

/* The model's svl_precision. */
int svl_model_precision(const svl_model* model, uint32_t* out);

/* TextModel::parameters (text.rs:139). */
int svl_model_parameters(const svl_model* model, uint64_t* out);

/* TextModel::forward / forward_with_features over a packed batch of
 * sequences (text.rs:150, 167, 182-538).  Host pointers.
 *   ids        : cu_seqlens[batch] token ids, sequence b = ids[cu_seqlens[b] .. cu_seqlens[b+1])
 *   cu_seqlens : batch + 1 offsets, cu_seqlens[0] = 0
 *   features / spans : optional soft-token rows (n_spans may be 0)
 *   normalized : batch x embedding_dim   (ForwardOutput::normalized)
 *   pooled     : batch x embedding_dim or NULL (ForwardOutput::pooled)
 *   projected  : T x embedding_dim or NULL     (ForwardOutput::projected)
 *   hidden_states : (num_hidden_layers + 1) x T x hidden_size or NULL
 *               (ForwardOutput::hidden_states, capture_hidden = true)
 * Errors follow text.rs:188-218: empty sequence / id >= vocab -> SVL_CORRUPT,
 * sequence > 8192 or > max_position_embeddings -> SVL_LIMIT_EXCEEDED,
 * non-finite activation -> SVL_INTERNAL. */
int svl_forward_batch(svl_model* model, const uint32_t* ids, const uint64_t* cu_seqlens,
                      uint32_t batch, const float* features, const svl_feature_span* spans,
                      uint32_t n_spans, float* normalized, float* pooled, float* projected,
                      float* hidden_states, char* err, size_t err_len);

/* TextModel::embed_ids (text.rs:546-554) for a batch: forward, then
 * truncate_and_normalize to `dimension` (kernels.rs:916-927).  Host pointers;
 * out is batch x dimension.  dimension outside 1..=embedding_dim ->
 * SVL_INTERNAL before any work, as in the reference. */
int svl_embed_batch(svl_model* model, const uint32_t* ids, const uint64_t* cu_seqlens,
                    uint32_t batch, uint32_t dimension, float* out, char* err, size_t err_len);

/* Same as svl_embed_batch with ids and out in device memory of the model's
 * device (cu_seqlens stays on the host: it drives the tile schedule).  ids
 * are validated on the device; an out-of-vocabulary id is reported by the
 * next call to svl_model_check (SVL_CORRUPT) because this call does not
 * synchronise. */
int svl_embed_batch_device(svl_model* model, const uint32_t* d_ids, const uint64_t* cu_seqlens,
                           uint32_t batch, uint32_t dimension, float* d_out, void* stream,
                           char* err, size_t err_len);

/* Synchronises the model's stream and reports a deferred device-side error
 * (out-of-vocabulary id, non-finite activation) raised by *_device calls. */
int svl_model_check(svl_model* model, char* err, size_t err_len);

/* ---------------------------------------------------------------- index -- */

/* A device-resident, append-only store of unit-norm embedding rows with their
 * chunk ids (the in-memory Index view, src/index/mod.rs:271-308).
 * `capacity` rows of `dim` floats are reserved in HBM up front. */
int svl_index_create(int device, uint32_t dim, uint64_t capacity, svl_index** out, char* err,
                     size_t err_len);
void svl_index_destroy(svl_index* index);
uint64_t svl_index_len(const svl_index* index);
uint32_t svl_index_dim(const svl_index* index);

/* Appends n host rows; each row is L2-normalised in f64 exactly as
 * Chunk::new does (src/storage/model.rs:546-581: zero or non-finite norm ->
 * SVL_USAGE).  chunk_ids are the rows' ChunkId values (tie-break key). */
int svl_index_append(svl_index* index, const float* rows, const uint64_t* chunk_ids, uint64_t n,
                     char* err, size_t err_len);
/* Device-pointer variant (rows and chunk_ids in device memory). */
int svl_index_append_device(svl_index* index, const float* d_rows, const uint64_t* d_chunk_ids,
                            uint64_t n, void* stream, char* err, size_t err_len);

/* Document ingest into the device index (Store::put_document's chunk
 * embedding, src/storage/store.rs:524, then Chunk::new's normalisation and
 * the index append): embeds `batch` packed sequences (host ids and cu_seqlens
 * as for svl_embed_batch) at the index's dimension (Matryoshka truncation and
 * L2 normalisation, text.rs:546-554) and appends the embeddings with
 * `chunk_ids` (host, one per sequence) without copying them to the host.  The
 * model and the index must live on the same GPU and the index dimension must
 * be 1..=embedding_dim (else SVL_USAGE); a batch that does not fit the
 * index's remaining capacity is rejected before any work
 * (SVL_LIMIT_EXCEEDED).  Model errors (bad ids, non-finite activations) are
 * reported before anything is appended.  Synchronous, like svl_embed_batch. */
int svl_ingest_batch(svl_model* model, svl_index* index, const uint32_t* ids, const uint64_t* cu_seqlens,
                     uint32_t batch, const uint64_t* chunk_ids, char* err, size_t err_len);

/* Exact cosine top-k for a batch of queries: for each query the first k
 * entries of vector::rank (src/index/vector.rs:17-97), i.e. rows sorted by
 * f64 score = dot / (|q| |v|) descending, ties by ascending chunk id, and the
 * slice Index::search takes (offset + limit = k, src/index/mod.rs:349-359).
 *   queries   : n_queries x dim (host)
 *   row_mask  : NULL, or svl_index_len bytes; rows whose byte is 0 are
 *               filtered out (Filters::matches, src/index/mod.rs:63-72)
 *   out_rows / out_chunk_ids / out_scores : n_queries x k (entries past
 *               out_counts[q] are unspecified); out_chunk_ids may be NULL
 *   out_counts: n_queries, min(k, rows surviving the filter)
 * Query validation follows vector.rs:23-55 (empty, non-finite, zero norm,
 * dimension mismatch -> SVL_USAGE; dim > 8192 -> SVL_LIMIT_EXCEEDED). */
int svl_index_search(svl_index* index, const float* queries, uint32_t n_queries, uint32_t dim,
                     const uint8_t* row_mask, uint32_t k, uint64_t* out_rows,
                     uint64_t* out_chunk_ids, double* out_scores, uint32_t* out_counts,
                     char* err, size_t err_len);

/* Device-pointer variant: queries, outputs and row_mask in device memory;
 * returns once queued on `stream`.  Queries are not validated on the host;
 * an invalid query is reported by svl_index_check. */
int svl_index_search_device(svl_index* index, const float* d_queries, uint32_t n_queries,
                            const uint8_t* d_row_mask, uint32_t k, uint64_t* d_out_rows,
                            uint64_t* d_out_chunk_ids, double* d_out_scores,
                            uint32_t* d_out_counts, void* stream, char* err, size_t err_len);

/* Synchronises the index's stream and reports deferred device-side errors. */
int svl_index_check(svl_index* index, char* err, size_t err_len);

/* Merges per-shard top-k lists (gathered from every GPU of a row-sharded
 * index) into the global top-k, in device memory on `device`:
 *   d_scores / d_chunk_ids / d_rows : n_shards x n_queries x k (shard-major,
 *       as an all-gather lays them out); d_counts n_shards x n_queries
 *   outputs n_queries x k plus d_out_shard (which shard each hit came from)
 * Order: score descending, chunk id ascending (vector.rs:90-95). */
int svl_merge_topk_device(int device, const double* d_scores, const uint64_t* d_chunk_ids,
                          const uint64_t* d_rows, const uint32_t* d_counts, uint32_t n_shards,
                          uint32_t n_queries, uint32_t k, double* d_out_scores,
                          uint64_t* d_out_chunk_ids, uint64_t* d_out_rows,
                          uint32_t* d_out_shard, uint32_t* d_out_counts, void* stream,
                          char* err, size_t err_len);

/* ------------------------------------------------------------ multi-GPU --
 * One process per GPU over an NCCL communicator (NVLink / NVSwitch).  The
 * reference is single-process, so these have no counterpart there: they are
 * how the row-sharded index of this build reaches vector::rank
 * (src/index/vector.rs:17-97) over several GPUs.  NCCL is opened at run time
 * (libnccl.so.2; the copy already loaded in the process when there is one):
 * without it these calls return SVL_UNSUPPORTED.  Every rank must make the
 * same calls in the same order with the same sizes. */

/* 128 bytes (an ncclUniqueId) for svl_nccl_comm_create, made on one rank and
 * handed to the others by the host. */
int svl_nccl_unique_id(void* id_out, char* err, size_t err_len);

/* Joins rank `rank` of `n_ranks` (1..64) on `device`; *comm_out is the
 * communicator (an ncclComm_t) the calls below take.  Blocks until every
 * rank has joined. */
int svl_nccl_comm_create(int device, int n_ranks, int rank, const void* id, void** comm_out, char* err,
                         size_t err_len);

/* Destroys (abort = 0) or aborts (abort = 1: after an error that left other
 * ranks waiting) a communicator from svl_nccl_comm_create. */
int svl_nccl_comm_destroy(void* comm, int abort);

/* Query stage of ingest-then-query: every rank passes n_local x dim floats
 * (the same n_local on every rank); d_all (n_ranks * n_local x dim, rank
 * major) receives every rank's rows on every rank.  Queued on `stream`. */
int svl_allgather_rows(void* comm, const float* d_local, uint64_t n_local, uint32_t dim, float* d_all,
                       void* stream, char* err, size_t err_len);

#define SVL_SHARDED_MAX_K 4096u

/* Exact top-k over a corpus row-sharded across the communicator's ranks:
 * every rank passes its shard (an svl_index whose rows start at global row
 * `row_offset`) and the SAME n_queries x dim queries (device memory).  Each
 * rank searches its shard (svl_index_search's exact path, near-ties
 * included), the per-shard lists are exchanged in one all-gather, and every
 * rank receives the global answer in reference order (score descending, chunk
 * id ascending; vector.rs:90-95):
 *   d_out_rows      n_queries x k global rows (row_offset + local row)
 *   d_out_chunk_ids n_queries x k (may be NULL); d_out_scores n_queries x k
 *   d_out_counts    n_queries: min(k, total rows)
 * k is 1..SVL_SHARDED_MAX_K.  The call synchronises `stream` once (between
 * the shard search and the exchange) and returns with the exchange and the
 * merge queued.  A rank whose own search fails still takes part in the
 * exchange and returns the error; the other ranks skip its list and report
 * SVL_INTERNAL ("another rank's shard search failed") at svl_index_check.
 * If the exchange buffers cannot be allocated the call returns
 * SVL_LIMIT_EXCEEDED without taking part: abort the communicator on every
 * rank. */
int svl_sharded_search(void* comm, svl_index* shard, uint64_t row_offset, const float* d_queries,
                       uint32_t n_queries, uint32_t k, uint64_t* d_out_rows, uint64_t* d_out_chunk_ids,
                       double* d_out_scores, uint32_t* d_out_counts, void* stream, char* err,
                       size_t err_len);

/* Exact cosine top-k like svl_index_search_device, for callers that cannot
 * allocate device memory: no counterpart in the reference.  Some hosts cannot
 * let a library call cudaMalloc -- device memory is carved up up front by a
 * pool this library must not bypass, a serving loop runs under a fixed memory
 * budget, or the calling thread may not take the driver's allocation lock.
 * This entry point allocates nothing: its scratch is one static device array
 * of about 2.6 MiB that every GPU loading the library holds until the process
 * exits.
 *   d_rows     : n_rows x dim unit-norm rows (as svl_index_append stores them),
 *                16-byte aligned, on the current device; d_chunk_ids n_rows
 *   d_queries  : n_queries x dim, 16-byte aligned; d_row_mask NULL or n_rows
 *                bytes (0 = filtered); a misaligned pointer is SVL_USAGE
 *   outputs    : as svl_index_search_device (n_queries x k, counts n_queries);
 *                d_out_chunk_ids may be NULL
 * Limits: 1..128 queries, dim a multiple of 4 up to 1024, k 1..32; larger
 * requests are rejected with SVL_LIMIT_EXCEEDED.  Synchronous: returns after
 * `stream` has finished the search; a query with too many near-ties for the
 * candidate screen returns SVL_UNSUPPORTED (svl_index_search answers it).
 * The first call on each device looks up the scratch address and sets kernel
 * attributes, so make it before any stream capture.  Every call on a device
 * shares the one scratch array: calls that overlap on the GPU (other threads
 * or streams) race and must be serialised by the caller. */
int svl_search_noalloc(const float* d_rows, const uint64_t* d_chunk_ids, uint64_t n_rows, uint32_t dim,
                       const float* d_queries, uint32_t n_queries, const uint8_t* d_row_mask, uint32_t k,
                       uint64_t* d_out_rows, uint64_t* d_out_chunk_ids, double* d_out_scores,
                       uint32_t* d_out_counts, void* stream, char* err, size_t err_len);

/* ------------------------------------------------------------- operators --
 * Blocks of the towers and encoders that stand beside the text model: what
 * makes the soft tokens of svl_feature_span, or another encoder's rows, from
 * projections (svl_q4_linear_device), positions (svl_rope_apply_device) and
 * attention (svl_attention_device).  The reference runs these towers on the
 * CPU; the entry points have no one counterpart there.
 *
 * Operands are rows of device memory: row t starts at pointer + t * ld
 * elements and holds its heads one after another, as the fused q, k, v rows
 * of a projection do.  Every pointer belongs to the device of the handle (or
 * of the `device` argument), whatever the calling thread's current device is,
 * which stays as it was.  The *_device calls follow `stream` (NULL = the
 * legacy default stream): they return once queued, allocate nothing and never
 * wait, so they may be captured into a CUDA graph; a captured call keeps
 * referring to the handle, which has to outlive the graph, and a queued one
 * has to be over before its handle is destroyed.  Destroying a handle frees its
 * memory at once and may wait for the device; it may happen while a capture
 * is open, on any thread.  Creating or reading one allocates, copies and waits,
 * and checking a plan waits: not for an open capture.  A handle is never
 * changed by a call, so threads, streams and graphs may share it; outputs and
 * workspaces are the caller's and must not be shared by calls that may overlap.  Outputs must not overlap
 * inputs except where stated.  NULL pointers are accepted where nothing is
 * read or written through them. */

/* How the axes of a multi-axis rotary embedding share a head.  An axis with n
 * pairs turns n pairs of dimensions by angles position * frequency:
 *   SVL_ROPE_SPLIT        axis a owns the next 2 n_a dimensions and pairs d
 *                         with d + n_a inside them; pair i has the frequency
 *                         theta[a]^(-i / n_a).  (Images: half a head turns
 *                         with the row, half with the column.)
 *   SVL_ROPE_SECTIONS     with n = sum n_a, pair p is (p, p + n) and has the
 *                         frequency theta[0]^(-p / n); each axis owns a run of
 *                         pairs, in order.
 *   SVL_ROPE_INTERLEAVED  the same pairs and frequencies, dealt to the axes
 *                         in turn, an axis dropping out once it has its n_a.
 * Dimensions behind 2 * sum n_a are copied. */
typedef enum svl_rope_arrangement {
  SVL_ROPE_SPLIT = 0,
  SVL_ROPE_SECTIONS = 1,
  SVL_ROPE_INTERLEAVED = 2
} svl_rope_arrangement;

#define SVL_ROPE_MAX_AXES 4u
#define SVL_ROPE_MAX_HEAD_DIM 512u

typedef struct svl_rope_config {
  uint32_t head_dim;             /* 2..SVL_ROPE_MAX_HEAD_DIM */
  uint32_t n_axes;               /* 1..SVL_ROPE_MAX_AXES */
  uint32_t pairs[4];             /* per axis; >= 1 for the first n_axes, 2 * sum <= head_dim */
  uint32_t arrangement;          /* svl_rope_arrangement */
  uint32_t reserved;             /* zero */
  double theta[4];               /* finite, >= 1/128; theta[0] alone unless SVL_ROPE_SPLIT */
} svl_rope_config;

typedef struct svl_rope svl_rope;

/* A rotary embedding's tables, in host memory: no device is touched, and any
 * device may use it.  A bad configuration -> SVL_USAGE. */
int svl_rope_create(const svl_rope_config* config, svl_rope** out, char* err, size_t err_len);
void svl_rope_destroy(svl_rope* rope);

/* Rotates n_tokens rows of q_heads query heads and k_heads key heads (either
 * may be 0) of `dtype` (svl_dtype).  d_positions: n_axes x n_tokens, one axis
 * after another, any int32 values; however far the position, the angle that sine
 * and cosine are taken of is within 2^-25 of a turn (2^-26 by its rounding to
 * FP32), and products are rounded once to the type.  An output may
 * be its own input (same pointer and ld: in place).  Element alignment
 * suffices (4 bytes for the positions; else SVL_USAGE); 16-byte aligned rows with an even head are faster.  heads *
 * head_dim <= ld < 2^36, n_tokens < 2^31 (else SVL_USAGE). */
int svl_rope_apply_device(const svl_rope* rope, int device, uint32_t dtype, const int32_t* d_positions,
                          uint64_t n_tokens, const void* d_q, uint64_t ld_q, uint32_t q_heads, void* d_q_out,
                          uint64_t ld_q_out, const void* d_k, uint64_t ld_k, uint32_t k_heads, void* d_k_out,
                          uint64_t ld_k_out, void* stream, char* err, size_t err_len);

/* Attention over packed sequences: for query i of a sequence (of n_q queries
 * and n_k keys) at position p = i + n_k - n_q, and key j,
 *   visible(i, j) = doc_q[i] == doc_k[j], or j < prefix        (documents)
 *                   and doc_q[i] >= 0 and doc_k[j] >= 0
 *                   and (j < prefix, or j <= p if causal)      (order)
 *                   and (j < prefix, or |p - j| <= window if window >= 0)
 *   t(i, j) = scale * q_i . k_j;  cap > 0: t = cap * tanh(t / cap)
 *             then t -= slope[head] * |p - j|
 *   out_i   = sum over the visible j of softmax(t)_j v_j
 *   lse_i   = log of the sum over the visible j of exp(t(i, j))
 * A row that sees no key gets out = 0 and lse = -inf.  A masked key's values
 * never reach a row, be they NaN or infinite; rows of other sequences and
 * rows behind the last one are neither read into a result nor written.
 * Scores, softmax statistics and sums are FP32 (a capped score is off by up to
 * 2^-20 of the cap where it comes near it; FP16 / BF16: the weights of the
 * visible keys are rounded to the type before they multiply v). */
typedef struct svl_attention_config {
  uint32_t dtype;                /* svl_dtype of q, k, v and out */
  uint32_t q_heads;              /* a multiple of kv_heads; q_heads / kv_heads <= 65535 */
  uint32_t kv_heads;             /* 1..65535; query head h reads kv head h / (q_heads / kv_heads) */
  uint32_t head_dim;             /* 1..512 */
  float scale;                   /* 1e-30..1e30 */
  float cap;                     /* 0 = none; 1e-30..1e30, scale / cap at most 1e30 */
  uint32_t causal;               /* 0 or 1 */
  int32_t window;                /* < 0 = none */
  uint32_t reserved[4];          /* zero */
} svl_attention_config;

typedef struct svl_attention_plan svl_attention_plan;

/* Checks a batch's layout and masks and puts its tile schedule on `device`.
 * Host pointers, copied; synchronous.  One plan serves every layer that
 * attends over the batch.
 *   cu_q, cu_k : batch + 1 offsets each, as cu_seqlens; cu_k NULL = cu_q
 *   prefix     : batch entries, or NULL (0 for all)
 *   doc_q, doc_k : the document of every packed query / key, or both NULL;
 *                any values, negative = padding; doc_k NULL alone = doc_q, if
 *                cu_k is NULL too
 *   slopes     : q_heads values in -1e20..1e20, or NULL
 * Errors: SVL_USAGE (bad configuration, offsets that start off 0 or fall,
 * slopes out of range), SVL_LIMIT_EXCEEDED (2^31 or more keys, or query rows
 * times group, in one sequence; out of memory). */
int svl_attention_plan_create(int device, const svl_attention_config* config, const uint64_t* cu_q,
                              const uint64_t* cu_k, uint32_t batch, const uint64_t* prefix, const int32_t* doc_q,
                              const int32_t* doc_k, const float* slopes, svl_attention_plan** out, char* err,
                              size_t err_len);
void svl_attention_plan_destroy(svl_attention_plan* plan);

/* Bytes of workspace that svl_attention_device needs (0 unless the plan cuts
 * a long key axis over several blocks). */
int svl_attention_plan_workspace(const svl_attention_plan* plan, uint64_t* bytes);

/* One attention over the plan's batch.  d_lse: q rows x q_heads, or NULL.
 * d_workspace: 16-byte aligned, svl_attention_plan_workspace bytes, contents
 * irrelevant before and after.  heads * head_dim <= ld < 2^36.  With FP16 / BF16 and
 * a head_dim that is a multiple of 8, q, k, v and out have to be 16-byte
 * aligned with ld a multiple of 8 (else SVL_USAGE); otherwise element
 * alignment suffices. */
int svl_attention_device(const svl_attention_plan* plan, const void* d_q, uint64_t ld_q, const void* d_k,
                         uint64_t ld_k, const void* d_v, uint64_t ld_v, void* d_out, uint64_t ld_out, float* d_lse,
                         void* d_workspace, uint64_t workspace_bytes, void* stream, char* err, size_t err_len);

/* Synchronises the plan's device and reports a deferred device-side error (a
 * bounded wait that ran out -> SVL_INTERNAL). */
int svl_attention_check(const svl_attention_plan* plan, char* err, size_t err_len);

/* A weight matrix W [n, k] in 4 bits: W[i, j] = (code - zero) * scale with
 * codes and zeros 0..15 and one scale (and zero) per row and group of `group`
 * columns (32, 64 or 128; k a multiple of it, n and k below 2^31). */
typedef struct svl_q4 svl_q4;

/* From existing codes, in host or in device memory (work that writes them has
 * to be complete); copied into the handle's own layout; synchronous.
 *   codes  : n x k/2 bytes, column 2c in the low half of byte c
 *   scales : n x k/group of scale_dtype (SVL_DTYPE_F16 or SVL_DTYPE_BF16); 2-byte
 *            aligned where they are in device memory (else SVL_USAGE)
 *   zeros  : n x k/group bytes (the low four bits), or NULL (8 for all) */
int svl_q4_create(int device, const uint8_t* codes, const void* scales, uint32_t scale_dtype, const uint8_t* zeros,
                  uint32_t n, uint32_t k, uint32_t group, svl_q4** out, char* err, size_t err_len);

/* Quantises a host weight tensor (2-D, F32 or BF16) on the device: per group,
 * with asymmetric = 0 scale = max|w| / 7 and zero 8 (codes 1..15), else scale
 * = (max - min) / 15 over the values and 0, and zero = -min / scale rounded;
 * scales are rounded to BF16 before the codes are chosen, codes are the
 * nearest (ties to even).  A non-finite weight -> SVL_CORRUPT. */
int svl_q4_quantize(int device, const svl_tensor_view* weight, uint32_t group, uint32_t asymmetric, svl_q4** out,
                    char* err, size_t err_len);
void svl_q4_destroy(svl_q4* weight);

/* The matrix as svl_q4_create takes it, into host memory (any pointer may be
 * NULL): sizes and scale type, codes, scales, zeros (all 8 when it has none). */
int svl_q4_read(const svl_q4* weight, uint32_t* n, uint32_t* k, uint32_t* group, uint32_t* scale_dtype,
                uint8_t* codes, void* scales, uint8_t* zeros, char* err, size_t err_len);

/* y = x W^T: `rows` rows of x (k values each, row stride ld_x) into y (n
 * values, row stride ld_y), both of `dtype`.  Made for few rows (a query's
 * tokens, down to a single one); any count below 2^31 works.  Products and
 * sums are FP32 (an F32 x keeps its 24 bits, but none below 2^-133), y is rounded once.  A row with a
 * NaN or infinite value gets non-finite results; the others do not.  Element
 * alignment suffices.  Strides are below 2^36.  Columns of y behind n are left
 * as they were. */
int svl_q4_linear_device(const svl_q4* weight, uint32_t dtype, const void* d_x, uint64_t ld_x, uint64_t rows,
                         void* d_y, uint64_t ld_y, void* stream, char* err, size_t err_len);

#ifdef __cplusplus
}
#endif
#endif /* SVL_GPU_H */
