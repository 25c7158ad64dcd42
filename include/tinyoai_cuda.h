/*
 * tinyoai_cuda.h - C ABI of the B200 (sm_100a) inference backend for tinyoai.
 *
 * The Go package binds these entry points through cgo (build tag `cuda`) in
 * place of its native MLX forwarders. Each entry point names the reference
 * interface it replaces (path:line inside the wbrown/tinyoai project).
 *
 * Conventions
 *  - Every function returns an int status: TCU_OK (0) or a negative TCU_E*
 *    code. The message of the last failure on the calling thread is returned
 *    by tcu_last_error() (pattern of internal/mlx/bridge.c:13-33).
 *  - Buffers are plain host pointers owned by the caller. Nothing is retained
 *    after a call returns except where stated (weights are copied to the GPU
 *    during load, so the caller may free its tensor bytes afterwards).
 *  - Handles are opaque. A session (and its branches) must be used from one
 *    thread at a time, as the Go wrapper guarantees with its request gate
 *    (mlx.go:32, 291-296). Distinct sessions may run concurrently.
 *  - No call allocates host memory for the caller, and no call falls back to
 *    the CPU: without a usable sm_100a GPU, loading fails with TCU_ENODEV.
 */
#ifndef TINYOAI_CUDA_H
#define TINYOAI_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TCU_ABI_VERSION 1

/* Status codes. */
#define TCU_OK 0
#define TCU_EINVAL (-1)    /* bad argument: token, prefix, length, shape, dtype */
#define TCU_ENODEV (-2)    /* no usable sm_100 device */
#define TCU_ENOMEM (-3)    /* device memory or KV pool exhausted */
#define TCU_ECUDA (-4)     /* CUDA runtime error (message has the detail) */
#define TCU_ECLOSED (-5)   /* handle already closed */
#define TCU_EUNSUP (-6)    /* valid request this backend does not implement */
#define TCU_ETIMEOUT (-7)  /* a bounded device wait expired */

/* Tensor dtypes: GGUF type codes (gguf.go:177-205). */
#define TCU_F32 0
#define TCU_F16 1
#define TCU_Q5_1 7
#define TCU_Q8_0 8
#define TCU_Q5_K 13
#define TCU_Q6_K 14
#define TCU_BF16 30

/* One checkpoint tensor as the Go loaders hold it: weightTensor{data, dtype,
 * shape} (safetensors.go:193-197), row-major with the file's block encoding.
 * Names use the Hugging Face convention (stablelm.go:180-191). */
typedef struct {
  const char* name;
  int32_t dtype;
  int32_t ndim;       /* 1 or 2 */
  int64_t shape[2];   /* shape[0] = rows (or length), shape[1] = cols */
  const void* data;
  uint64_t nbytes;
} tcu_tensor;

/* StableLMConfig after validate() (stablelm.go:18-111). */
typedef struct {
  int32_t vocab_size, hidden_size, intermediate_size, num_hidden_layers;
  int32_t num_attention_heads, num_key_value_heads, max_position_embeddings;
  int32_t bos_token_id, eos_token_id;
  double layer_norm_eps, rope_theta, partial_rotary_factor;
} tcu_stablelm_config;

/* Load-time options. Zero-initialise for defaults. */
typedef struct {
  int32_t device;         /* CUDA ordinal */
  int32_t kv_page_tokens; /* positions per KV page; 0 -> 32 */
  int64_t kv_pool_bytes;  /* KV pool budget per KV dtype; 0 -> 1/4 of free HBM after weights */
} tcu_load_options;

typedef struct tcu_model tcu_model;
typedef struct tcu_session tcu_session;
typedef struct tcu_branches tcu_branches;

/* Library and device queries. */
int tcu_abi_version(void);
const char* tcu_last_error(void);
int tcu_device_count(int32_t* count);

/* Replaces LoadStableLM/loadStableWeights (stablelm.go:136-199) and
 * LoadMLXNative (mlx_native.go:56-160): validates the config, checks every
 * tensor's shape, uploads and repacks weights into the device layout. */
int tcu_stablelm_load(const tcu_stablelm_config* config, const tcu_tensor* tensors, int32_t n_tensors,
                      const tcu_load_options* options, tcu_model** out);

/* Head-parallel tensor parallelism for one long sequence (an 8K-token
 * prefill, say): `world` processes, one GPU each, load the same checkpoint
 * and each keeps a contiguous block of query heads (and their KV heads),
 * the matching rows of q/k/v, a block of MLP rows (gate/up rows, down
 * columns) and the matching columns of o_proj; embedding, norms and lm_head
 * are replicated. Every layer sums the ranks' out + down partials with one
 * NCCL all-reduce (the parallel residual, stablelm.go:365-377, lets both
 * products share it) and adds the sum to the residual. Rank 0 makes the
 * communicator id with tcu_tp_unique_id and shares its 128 bytes with the
 * others (any host channel); every rank then calls tcu_stablelm_load_tp with
 * the same id. world must divide the heads, KV heads and MLP width, and the
 * o/down column slices must be whole quantisation blocks. A tensor-parallel
 * model serves one session at a time (every rank runs the same calls, in the
 * same order, with the same tokens). NCCL is loaded at run time
 * (libnccl.so.2); without it these return TCU_EUNSUP. */
typedef struct {
  int32_t world;
  int32_t rank;
  uint8_t nccl_id[128];
} tcu_tp_options;
int tcu_tp_unique_id(uint8_t* id);
int tcu_stablelm_load_tp(const tcu_stablelm_config* config, const tcu_tensor* tensors, int32_t n_tensors,
                         const tcu_load_options* options, const tcu_tp_options* tp, tcu_model** out);
/* The share of rank `rank`: out[0..6) = first query head, query heads, first
 * KV head, KV heads, first MLP row, MLP rows. Needs no GPU. */
int tcu_tp_plan(const tcu_stablelm_config* config, int32_t world, int32_t rank, int32_t* out);

/* The per-layer exchange over NVLink peer memory instead of NCCL (no
 * counterpart in the reference): every rank calls tcu_tp_exchange_handle
 * (allocates its exchange buffer, returns its CUDA IPC handle), the ranks
 * share the handles (any host channel), and every rank calls
 * tcu_tp_exchange_open with all of them in rank order. From then on the
 * exchange of up to 64 rows (decode steps) is one kernel per layer that stores
 * this rank's partial into every rank's buffer, waits (bounded) for the
 * others' and adds the rank-ordered sum to the residual, and tensor-parallel
 * decode steps replay a captured CUDA graph; prefill chunks keep NCCL. Ranks
 * on one node, at most 8. A wait that runs out returns TCU_ETIMEOUT. */
#define TCU_TP_HANDLE_BYTES 64
int tcu_tp_exchange_handle(tcu_model* model, uint8_t* handle);
int tcu_tp_exchange_open(tcu_model* model, const uint8_t* handles);

/* GGUF StableLM checkpoints (readGGUF and loadStableGGUF, gguf.go:139-357):
 * tcu_gguf_open memory-maps a GGUF v3 file, validates its header as the
 * reference does (magic and version, counts, metadata types, tensor ranks,
 * dimensions and types, alignment, bounds, overlap, the StableLM metadata and
 * tensor set) and derives the configuration. The vocabulary size is the
 * length of tokenizer.ggml.tokens; comparing that vocabulary with the
 * tokenizer.json beside the file stays with the caller's tokenizer.
 * tcu_gguf_tensor returns tensor i under its Hugging Face name (the inverse of
 * ggufNames, gguf.go:250-255) with data pointing into the mapping, valid until
 * tcu_gguf_close. tcu_gguf_load_stablelm uploads the model straight from the
 * mapping (no host copy of the weights); tp may be NULL (the whole model) or a
 * rank's share as for tcu_stablelm_load_tp. Needs no GPU except the load. */
typedef struct tcu_gguf tcu_gguf;
int tcu_gguf_open(const char* path, tcu_gguf** out);
int tcu_gguf_config(const tcu_gguf* gguf, tcu_stablelm_config* config);
int tcu_gguf_tensor_count(const tcu_gguf* gguf, int32_t* n);
int tcu_gguf_tensor(const tcu_gguf* gguf, int32_t index, tcu_tensor* out);
int tcu_gguf_load_stablelm(const tcu_gguf* gguf, const tcu_load_options* options, const tcu_tp_options* tp, tcu_model** out);
int tcu_gguf_close(tcu_gguf* gguf);

/* Replaces LoadModel/readWeights (model.go:90-166) for the legacy llama2.c
 * checkpoint (7 x int32 header then float32 tensors), and DefaultMLX /
 * LoadLlamaMLX (mlx_llama.go:37-53). */
int tcu_llama_load(const void* checkpoint, uint64_t nbytes, const tcu_load_options* options, tcu_model** out);

/* Model dimensions: vocab, hidden, layers, heads, kv heads, max positions. */
int tcu_model_info(const tcu_model* model, int32_t* vocab, int32_t* hidden, int32_t* layers, int32_t* heads,
                   int32_t* kv_heads, int32_t* max_positions);
/* Device bytes held by weights, and by the KV pool (allocated / in use). */
int tcu_model_memory(const tcu_model* model, uint64_t* weight_bytes, uint64_t* kv_pool_bytes, uint64_t* kv_used_bytes);
/* Releases weights and the KV pool. Every session must be closed first. */
int tcu_model_free(tcu_model* model);

/* weightTensor.readValues (matmul.go:12-50, decodeKBlock quant_k.go:31-86) on
 * the device: decodes n values, starting at row-major element `offset`, of a
 * rows x cols tensor given in its file encoding (host bytes, checked against
 * the format's size), into out (n host floats). `decoder` names which of the
 * device decoders produces them:
 *   TCU_DECODE_ELEMENT  the per-element decoder of the matrix-vector kernels
 *                       (every format);
 *   TCU_DECODE_GROUP8   the 8-value decoder of the batched products (Q6_K,
 *                       Q5_K);
 *   TCU_DECODE_TC       the tensor-core operand: the binary16 pieces the
 *                       tcgen05 GEMM multiplies, summed back and unscaled
 *                       (Q8_0, Q6_K, Q5_K).
 * Each returns the reference's float32 values bit for bit, which is what this
 * entry point lets a host check (quant_k_test.go:14-48 checks the Go decoder
 * the same way). It allocates and frees its own device buffers. */
#define TCU_DECODE_ELEMENT 0
#define TCU_DECODE_GROUP8 1
#define TCU_DECODE_TC 2
int tcu_read_values(int32_t device, int32_t dtype, const void* data, uint64_t nbytes, int32_t rows, int32_t cols,
                    int64_t offset, int64_t n, int32_t decoder, float* out);

/* A generation session: the resident token prefix of one request stream and
 * its paged KV (the state nativeMLX keeps per model, mlx_native.go:24-45).
 * kv_dtype is TCU_F32 or TCU_F16 (StableLMOptions.KVCache, kv_cache.go:8-24). */
int tcu_session_new(tcu_model* model, int32_t kv_dtype, tcu_session** out);
int tcu_session_free(tcu_session* session);
/* Number of resident positions (nativeMLX.offset). */
int tcu_session_length(const tcu_session* session, int32_t* length);

/* mlxForwarder.Forward (mlx.go:45-51, mlx_native.go:294-297): evaluates tokens
 * at positions prefix.. after keeping the first `prefix` resident positions.
 * When want_logits != 0 the final vocabulary row is written to logits_out
 * (vocab floats). Requires 0 <= prefix <= length and prefix + n <= max
 * positions. On failure the resident prefix is discarded (mlx_native.go:487-489). */
int tcu_session_forward(tcu_session* session, int32_t prefix, const int32_t* tokens, int32_t n, int32_t want_logits,
                        float* logits_out);

/* llamaMLXForwarder.Forward with allLogits (mlx_llama.go:27-35): one logits
 * row per input token (n x vocab floats). */
int tcu_session_forward_all(tcu_session* session, int32_t prefix, const int32_t* tokens, int32_t n, float* logits_out);

/* Greedy decoding on the device (sampleWithOptions with Temperature == 0,
 * sampling.go:150-163 / model.go:622-630, inside the loops of
 * stablelm.go:519-540 and mlx.go:414-468): evaluates tokens after `prefix`,
 * then emits `steps` argmax tokens, feeding each back without a host round
 * trip. The resident prefix afterwards holds prompt + steps-1 tokens, as in
 * the reference loop (the final sampled token is not evaluated). */
int tcu_session_generate_greedy(tcu_session* session, int32_t prefix, const int32_t* tokens, int32_t n, int32_t steps,
                                int32_t* out_tokens);

/* Device-side sampling shortlist over the logits of the last forward:
 * samplingCandidates (sampling.go:112-143) over float32 logits, returning up to
 * k (id, logit) pairs in descending order with ties broken by lower id, plus
 * the full-vocabulary log-sum-exp (logprobs.go:64-95). */
int tcu_session_shortlist(tcu_session* session, int32_t k, int32_t* ids, float* logits, double* logsumexp,
                          int32_t* n_out);

/* mlxProbabilityForwarder.ForwardWithLogprobs (mlx.go:53-57,
 * mlx_native.go:303-313 and 436-478) with summarizeLogits semantics
 * (logprobs.go:64-95): evaluates tokens[0..n) after `prefix` as
 * tcu_session_forward does, and for every input position i writes
 *   chosen[i]                          log P(targets[i]) after position i,
 *   top_ids[i * count .. + count)      the count most likely next ids,
 *   top_logprobs[i * count .. + count) their log probabilities,
 * descending, ties by lower id, all normalised over the full vocabulary in
 * float64. logits_out (vocab floats, may be NULL) receives the final row.
 * targets pair one-for-one with tokens; 1 <= count <= min(256, vocab).
 * On failure the resident prefix is discarded, as for tcu_session_forward. */
int tcu_session_forward_logprobs(tcu_session* session, int32_t prefix, const int32_t* tokens, const int32_t* targets, int32_t n,
                                 int32_t count, double* chosen, int32_t* top_ids, double* top_logprobs, float* logits_out);

/* SamplingOptions' penalties (sampling.go:12-58), validated as Validate does:
 * finite, repetition_penalty >= 1, repetition_range >= 0 (0: the whole
 * history), repetition_slope >= 0. Neutral: {1, 0, 0, 0, 0}. */
typedef struct {
  double repetition_penalty;
  double presence_penalty;
  double frequency_penalty;
  double repetition_slope;
  int32_t repetition_range;
} tcu_penalties;

/* samplingCandidates(penalizedLogits(logits, history, opts), k)
 * (sampling.go:76-143) over the logits of the session's last forward, on
 * the device: float64 scores with recency-weighted frequency, presence and
 * logarithmic repetition penalties from `history` (the story's token ids,
 * oldest first), then the k best (id, score) pairs, descending, ties by
 * lower id (1 <= k <= 256). ids[0] is the greedy choice of sampleWithOptions
 * (sampling.go:155-163). The caller draws from the pairs with its own RNG
 * (temperature, top-p and tail-free filtering run on these k scores). At most
 * 16384 distinct ids may carry a penalty. */
int tcu_session_sample_candidates(tcu_session* session, const int32_t* history, int32_t n_history, const tcu_penalties* penalties,
                                  int32_t k, int32_t* ids, double* scores, int32_t* n_out);

/* SaveCache / LoadCache (cache_file.go:55-176) for a session, in the
 * reference's TNYKV001 format: "TNYKV001", the header length, the JSON header
 * {"model_sha256", "float16", "tokens"} as encoding/json writes it, the
 * resident positions' KV in layer -> KV head -> keys, values order (float32
 * little-endian or binary16 bits, cachePayload cache_file.go:203-258), then
 * the SHA-256 of all of that. model_sha256 is the caller's model identity
 * (modelIdentity, cache_file.go:26-48: the config and tensor bytes), tokens
 * the session's resident token ids (n_tokens == its length).
 * Save writes a 0600 temporary file beside `path`, syncs it and renames it
 * over `path`. Load checks, in LoadCache's order, the format, header size,
 * context length, token ids, model identity, KV precision, file size and
 * checksum; only then do the restored positions replace the session's
 * context (on any error the session is unchanged) and the tokens go to
 * tokens[0 .. *n_tokens) (capacity entries available). */
int tcu_session_save_cache(tcu_session* session, const char* path, const uint8_t* model_sha256, const int32_t* tokens,
                           int32_t n_tokens);
int tcu_session_load_cache(tcu_session* session, const char* path, const uint8_t* model_sha256, int32_t* tokens, int32_t capacity,
                           int32_t* n_tokens);

/* mlxForker.Fork (sessions.go:26-30, mlx_sessions.go:10-71): the child shares
 * every full KV page copy-free (reference counted) and copies only the
 * partially filled tail page. Parent and child then diverge independently. */
int tcu_session_fork(tcu_session* session, tcu_session** child);

/* LimitCache / SetKVBits (mlx_native.go:231-244, mlx_kv.go:78-91). cleared
 * reports whether resident KV was discarded. */
int tcu_session_limit(tcu_session* session, int32_t window, int32_t* cleared);
int tcu_session_set_kv_dtype(tcu_session* session, int32_t kv_dtype, int32_t* cleared);
/* llamaMLXForwarder.Reset: drop all resident positions. */
int tcu_session_reset(tcu_session* session);

/* Runs the session's work on a caller-owned CUDA stream (a cudaStream_t;
 * NULL restores the session's own stream). Lets a host that already owns a
 * stream order its copies and events with the session's kernels. */
int tcu_session_set_stream(tcu_session* session, void* stream);

/* Opt-in stage timing, the device counterpart of stableProfile
 * (stablelm.go:229-250): when enabled, CUDA events bracket every kernel and
 * the per-stage launch counts and milliseconds accumulate. Stages, in order:
 * embedding, norm+q/k/v/gate/up projection, decode attention, out/down
 * projection + residual, final norm+head, prefill projection, prefill
 * attention, other, whole persistent decode step, tensor-parallel
 * all-reduce. tcu_session_profile_read returns the number of stages (10) and
 * fills up to n_stages entries;
 * reset != 0 clears the totals.
 * Profiling synchronises after every decode step, so it is for diagnosis,
 * not for throughput runs. */
int tcu_session_profile(tcu_session* session, int32_t enable);
int tcu_session_profile_read(tcu_session* session, int32_t n_stages, int64_t* launches, double* ms, int32_t reset);

/* mlxBrancher.NewBranches (branches.go:55-59, mlx_branches.go:25-32): count
 * suffixes that share the first `prefix` resident positions read-only.
 * Unlike the MLX backend, grouped-query attention is supported. */
int tcu_branches_open(tcu_session* session, int32_t prefix, int32_t count, tcu_branches** out);
/* mlxBranches.Forward (mlx_branches.go:120-184): one token per branch at the
 * same absolute position; writes count x vocab logits (rows_out may be NULL
 * to skip the copy). */
int tcu_branches_forward(tcu_branches* branches, const int32_t* tokens, float* rows_out);
/* Greedy argmax of each branch's last row (count ints). */
int tcu_branches_argmax(tcu_branches* branches, int32_t* ids);
/* mlxBranches.Close: releases suffix pages (the shared prefix stays resident)
 * and frees the handle, which must not be used afterwards. A failed
 * tcu_branches_forward already released the pages; close it all the same. */
int tcu_branches_close(tcu_branches* branches);

/* Continuous batching (a serving load of many sessions). The reference's
 * Go server runs one request at a time per model (the request gate,
 * mlx.go:291-296); a batching scheduler instead advances all active
 * sessions together. tcu_batch_open reserves a workspace and stream for up
 * to max_rows rows (1..1024) so that steps allocate no device memory. */
typedef struct tcu_batch tcu_batch;
int tcu_batch_open(tcu_model* model, int32_t max_rows, tcu_batch** out);
/* One decode step for n sessions of the batch's model that share one KV
 * precision: tokens[i] is appended to sessions[i] at its current length
 * (which must be >= 1) and its logits row computed, exactly as
 * tcu_session_forward(sessions[i], length, &tokens[i], 1, 1, row) would.
 * Writes n x vocab logits (rows_out may be NULL) and each row's greedy
 * argmax (ids_out may be NULL); each session's length then grows by one.
 * Sessions with open branches, repeated or closed sessions are rejected.
 * Work already queued on a session's own stream completes first. */
int tcu_batch_forward(tcu_batch* batch, tcu_session* const* sessions, const int32_t* tokens, int32_t n, float* rows_out,
                      int32_t* ids_out);
/* tcu_session_sample_candidates for every row of the batch's last step
 * (n = that step's row count): row i's history is history[off_i ..
 * off_i + history_len[i]) with off_i the sum of the earlier lengths, its
 * penalties penalties[i]; writes n x k ids and scores. */
int tcu_batch_sample_candidates(tcu_batch* batch, int32_t n, const int32_t* history, const int32_t* history_len,
                                const tcu_penalties* penalties, int32_t k, int32_t* ids, double* scores);
/* Lets steps of this batch whose sessions all begin with the same KV pages
 * (forks of one session, tcu_session_fork) read those pages once for all of
 * them: a step of two rows or more that share at least min_positions positions
 * in whole pages attends through tcu_paged_append and tcu_paged_attend (below)
 * instead of row by row. 0 (the default) turns it off. A layer's attention then
 * differs from the unshared step's by the order of float32 sums (and, over
 * binary16 KV, by weights of 22 bits), not in what it computes; keys and values
 * are rotated and rounded alike. What a later layer appends follows from
 * attention so rounded: a binary16 key or value there may be its neighbour.
 * Allocates the step's buffers; a step whose workspace has to grow allocates
 * again. Not for tensor-parallel models, nor for shapes outside the limits of
 * the operators below (TCU_EUNSUP). */
int tcu_batch_share_prefix(tcu_batch* batch, int32_t min_positions);
int tcu_batch_close(tcu_batch* batch);

/* Sampling shortlist over a logits row the caller already holds in device
 * memory, allocating no device memory. This entry point has no counterpart in
 * the reference (its Go path keeps logits on the host); it serves callers that
 * must not allocate on the device when they call, for example a host whose
 * own caching allocator already holds the free HBM.
 *
 * Same kernel and results as tcu_session_shortlist: up to k (id, logit)
 * pairs, descending, ties by lower id (sampling.go:112-143), plus the float64
 * log-sum-exp of the whole row (logprobs.go:64-95). logits: `vocab` floats on
 * `device`; stream: a CUDA stream of that device, or NULL for the legacy
 * default stream. The call makes `device` current, returns after the stream
 * has synchronised, and writes *n_out = min(k, vocab) entries to the host
 * arrays ids and values.
 *
 * The kernel's results pass through one fixed device array of
 * TCU_SHORTLIST_STATIC_SCRATCH_BYTES per device, so k is limited to
 * TCU_SHORTLIST_STATIC_MAX_K. vocab is limited to
 * TCU_SHORTLIST_STATIC_MAX_VOCAB (the kernel marks taken ids in shared memory).
 * Larger values fail with TCU_EINVAL. The first call on a device does the set-up
 * (it looks up that array's device address). The call synchronises the stream
 * and copies into host memory, so it cannot be captured into a CUDA graph: a
 * stream under capture fails with TCU_EINVAL before any work is queued.
 * Calls on one device share the array: two calls in flight at the same time on
 * one device, from different host threads, overwrite each other's results. */
#define TCU_SHORTLIST_STATIC_MAX_K 256
#define TCU_SHORTLIST_STATIC_MAX_VOCAB 1048576
#define TCU_SHORTLIST_STATIC_SCRATCH_BYTES 4096
int tcu_shortlist_static(int32_t device, const float* logits, int32_t vocab, int32_t k, void* stream, int32_t* ids,
                         float* values, double* logsumexp, int32_t* n_out);

/* ---------------------------------------------------------------------------
 * Operators over a paged KV cache the caller holds in device memory.
 *
 * One serving step of a host that keeps its own cache: tcu_plan_step builds
 * the step's block tables, positions and slots; tcu_paged_append normalises
 * and rotates the step's queries and keys and appends keys and values;
 * tcu_paged_means keeps the mean key of every completed page;
 * tcu_paged_attend and tcu_paged_attend_sparse attend. No counterpart in the
 * reference, whose native sessions own their KV (mlx_native.go:24-45): these
 * serve hosts that already hold their activations and cache on the GPU.
 *
 * Conventions of the section
 *  - Pointers named in a structure or argument list are device memory of
 *    `device` unless stated; counts, strides and the structures themselves
 *    are host values read during the call.
 *  - Work is queued on `stream` (a cudaStream_t of that device; NULL: the
 *    legacy default stream) and the call returns. Nothing is allocated,
 *    synchronised or kept, so the calls can be captured into CUDA graphs and
 *    may run concurrently as long as their outputs and workspaces differ. The
 *    caller's current device is left as it was.
 *  - Types: TCU_F32, TCU_F16 or TCU_BF16. Query rows and outputs have the
 *    cache's type, or are float32 over a TCU_F16 cache. Sums, norms and
 *    softmax statistics are float32 or wider; a result is rounded once, when
 *    it is stored. Softmax weights are operands of 16-bit matrix products over
 *    16-bit caches: with 16-bit rows each is rounded to the cache's type (by
 *    half a step of it; binary16 weights below 2^-25 of a part's largest by 2^-36
 *    of that at most), with float32 rows to a pair of binary16 values (22
 *    bits; below 2^-17 of the largest by 2^-39 of that), and so are those rows'
 *    queries (below 2^-16 of a row's largest by 2^-38 of that).
 *  - Strides count values, and the last dimension (a head's values) is
 *    contiguous. Rows, strides and bases of q, out, k and v are multiples of
 *    16 bytes. Head sizes: multiples of 8 up to TCU_PAGED_MAX_HEAD_DIM.
 *    Rows that are written (out, and k and v in an append) must not overlap;
 *    rows that are read may (stride 0: one head, or one row, for several).
 *  - Page ids outside [0, num_pages) stand for no page: their positions are
 *    not attended and nothing is written there. Values in a page behind a
 *    request's length are never read into a result.
 * ------------------------------------------------------------------------ */
#define TCU_PAGED_MAX_HEAD_DIM 256
#define TCU_PAGED_MAX_GROUP 64           /* query heads per KV head */
#define TCU_PAGED_MAX_PAGE_TOKENS 65536
#define TCU_PAGED_MAX_SELECTED 65536     /* first + last + top of a sparse call */
/* Tables, prefixes and selections map at most 2^30 positions. */

/* Value d of position r of page p, KV head g of k (and of v) is at
 * p * page_stride + g * head_stride + r * token_stride + d. */
typedef struct {
  void* k;
  void* v;
  int32_t dtype;
  int32_t num_pages, page_tokens, kv_heads, head_dim;
  int64_t page_stride, head_stride, token_stride;
} tcu_paged_kv;

/* Block tables, positions and slots of a step, from request lengths. Request
 * i holds held[i] positions and adds fresh[i] >= 0 tokens. Its table (row i,
 * table_width entries, rows table_stride apart) maps its pages; entries for
 * the positions it holds are read, ceil((held + fresh) / P) - ceil(held / P)
 * entries after them are written with pages from the front of free_pages, in
 * request order; other entries are left as they were. Outputs:
 *   starts[0 .. n]      first token of each request; starts[n] = tokens planned
 *   lengths[0 .. n)     held + fresh
 *   positions[t], slots[t] (t < capacity)  position of token t and its place
 *                       page * P + offset in the pool; -1 and -1 behind the
 *                       last token, and slot -1 where the table has no page
 *   counts[0 .. 3)      requests planned, tokens planned, pages taken
 * Requests are planned in order up to the first that does not fit (capacity
 * tokens, n_free pages, table_width) or has a negative count; that one and
 * the later ones keep lengths[i] = held[i] and get no tokens. lengths may be
 * the array held (or fresh) itself, starts the array fresh; no other arrays may
 * overlap. A page that a
 * request appends to (its last, partly filled one) must be its own.
 * page_tokens P: 1 .. TCU_PAGED_MAX_PAGE_TOKENS. */
int tcu_plan_step(int32_t device, void* stream, int32_t n, const int32_t* held, const int32_t* fresh, int32_t page_tokens, int32_t* tables,
                  int32_t table_width, int64_t table_stride, const int32_t* free_pages, int32_t n_free, int32_t capacity, int32_t* starts,
                  int32_t* lengths, int32_t* positions, int64_t* slots, int32_t* counts);

/* Rotary table: max_positions x pairs float32 pairs (cos, sin), 8-byte
 * aligned. Pair i is features (i, i + pairs) of a head, or (2i, 2i + 1) when
 * adjacent != 0; features from 2 * pairs on pass unchanged. Products and sums
 * are each rounded to float32. */
typedef struct {
  const float* table;
  int32_t max_positions, pairs, adjacent;
} tcu_rotary;

/* Norm of each query and key head over its head_dim features, before the
 * rotation: x / sqrt(mean x^2 + eps) * w (TCU_NORM_RMS) or (x - mean) /
 * sqrt(variance + eps) * w (TCU_NORM_LAYER). Weights are float32, one row of
 * head_dim for all heads (head_stride 0) or a row per head (head_stride
 * head_dim): q_weight for the query heads, k_weight for the KV heads. */
#define TCU_NORM_NONE 0
#define TCU_NORM_RMS 1
#define TCU_NORM_LAYER 2
typedef struct {
  int32_t kind;
  double eps;
  const float* q_weight;
  const float* k_weight;
  int64_t head_stride;
} tcu_head_norm;

/* Normalises (norm, may be NULL) and rotates (rotary, may be NULL) the query
 * and key heads of `rows` rows [heads | kv_heads | kv_heads] x head_dim of
 * type dtype, rows qkv_stride apart; writes queries to q_out (rows q_stride
 * apart, same type) and keys and values to the cache at slots[row] =
 * page * page_tokens + offset. Rows whose slot is outside the pool (-1: a
 * padding row) or whose position is outside the rotary table are skipped:
 * nothing of theirs is written. Two rows must not name one slot. q_out may be
 * the queries' own place in qkv (the same address and stride) and must not
 * overlap it otherwise. */
int tcu_paged_append(int32_t device, void* stream, const tcu_paged_kv* kv, int32_t dtype, int32_t rows, int32_t heads, const void* qkv,
                     int64_t qkv_stride, const int32_t* positions, const int64_t* slots, const tcu_rotary* rotary, const tcu_head_norm* norm,
                     void* q_out, int64_t q_stride);

/* For every slot that is the last of its page: means[page][g] = mean over the
 * page's positions of its keys, for each KV head g. means: [num_pages]
 * [kv_heads][head_dim], contiguous, the cache's type. The pages' other
 * positions must hold their keys already (an append of the same slots before
 * it on the stream); slots of other positions and outside the pool do
 * nothing. kv->v is not read. */
int tcu_paged_means(int32_t device, void* stream, const tcu_paged_kv* kv, int32_t rows, const int64_t* slots, void* means);

/* The queries of a ragged step. Rows starts[i] .. starts[i + 1] of q (rows
 * rows in all, heads x head_dim values each) are request i's last tokens:
 * row starts[i] + j is at position lengths[i] - (starts[i + 1] - starts[i])
 * + j and attends to the request's positions up to its own. Row i of tables
 * maps its pages. max_fresh is at least the largest starts[i + 1] - starts[i]
 * (later rows of a longer request are left as they were), and rows behind
 * starts[requests] are left as they were. A row at a negative position
 * attends to nothing and is zero. What lies at positions that a row does not
 * attend to never reaches it, infinities and NaN among them. heads is a
 * multiple of kv_heads; query head h reads KV head h / (heads / kv_heads). out
 * may be q itself (address and strides) and must not overlap it otherwise. The
 * weight of position t is softmax(scale * q . k_t). */
typedef struct {
  int32_t dtype;
  int32_t requests, rows, heads, max_fresh;
  int32_t table_width;
  const void* q;
  int64_t q_token_stride, q_head_stride;
  void* out;
  int64_t out_token_stride, out_head_stride;
  const int32_t* starts;
  const int32_t* lengths;
  const int32_t* tables;
  int64_t table_stride;
  float scale;
} tcu_paged_queries;

/* Attention of the step. The first prefix_pages pages of every request are
 * prefix[0 .. prefix_pages) (a long prompt they share): they are read from
 * there, once for all requests, and the tables' entries for them are not
 * read. prefix_pages 0: nothing is shared. max_length bounds the requests'
 * lengths (0: what the tables and the prefix map); positions from it on are
 * not attended. workspace: at least the bytes that the _workspace call
 * reports for the same arguments (it reads no device memory; 0: the call
 * needs none and workspace may be NULL), 256-byte aligned, its content
 * irrelevant before and after; calls that may run at the same time (two
 * streams, two captured graphs) need one each. A wait inside the kernel that
 * runs out after about a second (it should not: nothing but the kernel's own
 * copies and products is waited for) leaves NaN in the rows concerned; the call
 * has returned by then and gives no status. */
int tcu_paged_attend_workspace(const tcu_paged_kv* kv, const tcu_paged_queries* queries, int32_t prefix_pages, int32_t max_length,
                               uint64_t* bytes);
int tcu_paged_attend(int32_t device, void* stream, const tcu_paged_kv* kv, const tcu_paged_queries* queries, const int32_t* prefix,
                     int32_t prefix_pages, int32_t max_length, void* workspace, uint64_t workspace_bytes);

/* Attention of each query over the pages that a cheap score selects. A query
 * at position p has npages = p / page_tokens + 1 pages. For each KV head it
 * attends to the first `first` pages, the last `last` pages (at least 1, so
 * that the page being filled is among them) and, of those between, the `top`
 * with the largest max over the KV head's query heads h of q_h . means[page]
 * (float64; ties to the lower page, NaN and missing pages last). means is
 * tcu_paged_means' array, read for complete pages only. pages
 * [rows][kv_heads][first + last + top] receives the logical pages attended
 * to, ascending, -1 behind them. The workspace is as for tcu_paged_attend. */
int tcu_paged_attend_sparse_workspace(const tcu_paged_kv* kv, const tcu_paged_queries* queries, int32_t first, int32_t last, int32_t top,
                                      uint64_t* bytes);
int tcu_paged_attend_sparse(int32_t device, void* stream, const tcu_paged_kv* kv, const tcu_paged_queries* queries, const void* means,
                            int32_t first, int32_t last, int32_t top, int32_t* pages, void* workspace, uint64_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif
