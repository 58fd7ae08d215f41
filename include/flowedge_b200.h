/*
 * flowedge_b200 - B200 (sm_100a) implementation of FlowEdge's policy-sampling
 * hot path behind FlowEdge's own C ABI.
 *
 * Part 1 declares the reference ABI unchanged: same names, argument meaning,
 * status codes, struct layouts and error behaviour.  Each declaration cites
 * the reference declaration it replaces (paths inside the FlowEdge repository:
 * src/core/api/engine.h and src/core/protocol/contracts.h).  A program built
 * against the reference header links against libflowedge_b200.so unchanged.
 *
 * Part 2 adds what the reference has no equivalent for: batched entry points
 * (the reference is batch-1 only), device-pointer entry points, load options,
 * capacity reservation and allocation / launch counters.
 *
 * Part 3 declares operators on device buffers: the Mamba mixer's convolution
 * and selective scan over ragged sequences with slot states, products with
 * 4-bit weights, and the residual norm.
 *
 * All work runs on a B200; there is no CPU fallback.  Loading fails with a
 * message when no sm_100 device is present.
 */
#ifndef FLOWEDGE_B200_H
#define FLOWEDGE_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* ------------------------------------------------------------------------- */
/* contracts (src/core/protocol/contracts.h:11-121)                           */

enum { FE_PROTOCOL_VERSION = 1, FE_MODEL_DIGEST_BYTES = 16 };

enum {
  FE_ARCH_UNKNOWN = 0,
  FE_ARCH_MAMBA = 1,
  FE_ARCH_FLOW_HEAD = 2,
  FE_ARCH_MAMBA_FLOW = 3,
  FE_ARCH_DIFFUSION_HEAD = 4,
  FE_ARCH_TRANSFORMER = 5,
  FE_ARCH_TRANSFORMER_FLOW = 6,
  FE_ARCH_SMOLVLA_ACTION_EXPERT = 7,
};

enum { FE_PRECISION_UNKNOWN = 0, FE_PRECISION_F32 = 1, FE_PRECISION_BF16 = 2, FE_PRECISION_MIXED = 3 };

enum { FE_ACTION_RUNNING = 0, FE_ACTION_COMPLETE = 1, FE_ACTION_CANCELLED = 2, FE_ACTION_FAILED = 3 };

enum { FE_ACTION_UNITS_NORMALIZED = 0, FE_ACTION_UNITS_PHYSICAL = 1 };

enum { FE_NORMALIZATION_NONE = 0, FE_NORMALIZATION_MINMAX = 1 };

enum { FE_PROFILE_SOLVER_EULER = 0, FE_PROFILE_SOLVER_HEUN = 1, FE_PROFILE_SOLVER_RK4 = 2 };

typedef struct fe_model_digest {
  uint8_t bytes[FE_MODEL_DIGEST_BYTES];
} fe_model_digest;

typedef struct fe_model_metadata {
  uint32_t struct_size;
  uint32_t protocol_version;
  uint32_t architecture;
  uint32_t precision;
  fe_model_digest model_digest;
  uint64_t d_model;
  uint64_t n_layers;
  uint64_t d_inner;
  uint64_t d_state;
  uint64_t d_conv;
  uint64_t action_dim;
  uint64_t condition_dim;
  uint64_t decode_snapshot_bytes;
} fe_model_metadata;

typedef struct fe_deployment_profile {
  uint32_t struct_size;
  uint32_t profile_version;
  uint32_t model_compatibility_version;
  uint32_t action_units;
  uint32_t normalization_type;
  uint32_t solver_default;
  uint32_t reserved;
  const char* observation_schema_hash;
  const float* normalization_min;
  const float* normalization_max;
  uint64_t action_dim;
  uint64_t action_horizon;
  uint64_t normalization_count;
  uint64_t solver_min_steps;
  uint64_t solver_max_steps;
} fe_deployment_profile;

typedef struct fe_condition_metadata {
  uint32_t struct_size;
  uint32_t protocol_version;
  uint32_t solver;
  uint32_t reserved;
  fe_model_digest model_digest;
  uint64_t timestamp_ns;
  uint64_t deadline_ns;
  uint64_t generation;
  uint64_t condition_dim;
  uint64_t action_dim;
  uint64_t solver_steps;
  uint64_t remaining_nfe;
} fe_condition_metadata;

typedef struct fe_action_metadata {
  uint32_t struct_size;
  uint32_t protocol_version;
  uint32_t solver;
  uint32_t status;
  fe_model_digest model_digest;
  uint64_t timestamp_ns;
  uint64_t deadline_ns;
  uint64_t generation;
  uint64_t condition_dim;
  uint64_t action_dim;
  uint64_t remaining_nfe;
} fe_action_metadata;

/* ------------------------------------------------------------------------- */
/* Part 1: the reference C ABI (src/core/api/engine.h)                        */

typedef struct FeEngine fe_engine;
typedef struct FeWeights fe_weights;

enum { FE_SOLVER_EULER = 0, FE_SOLVER_HEUN = 1, FE_SOLVER_RK4 = 2 }; /* engine.h:16-21 */

enum { FE_DIFFUSION_DDIM = 0, FE_DIFFUSION_DDPM = 1 }; /* engine.h:23-27 */

typedef struct fe_diffusion_metadata { /* engine.h:29-44 */
  uint32_t struct_size;
  uint32_t protocol_version;
  uint32_t clip_sample;
  uint32_t reserved;
  uint64_t action_dim;
  uint64_t condition_dim;
  uint64_t horizon;
  uint64_t action_steps;
  uint64_t observation_steps;
  uint64_t train_timesteps;
  float clip_sample_range;
  float reserved_float;
} fe_diffusion_metadata;

enum { /* engine.h:46-59 */
  FE_STATUS_OK = 0,
  FE_STATUS_INVALID_ARGUMENT = 1,
  FE_STATUS_RESOURCE_EXHAUSTED = 2,
  FE_STATUS_TOKEN_OUT_OF_RANGE = 3,
  FE_STATUS_UNSUPPORTED_MODEL = 4,
  FE_STATUS_INVALID_SOLVER = 5,
  FE_STATUS_NO_ACTIVE_OPERATION = 6,
  FE_STATUS_STATE_UNAVAILABLE = 7,
  FE_STATUS_CANCELLED = 8,
  FE_STATUS_INCOMPATIBLE_STATE = 9,
  FE_STATUS_CORRUPT_STATE = 10,
};

/* engine.h:60-63: last error of this thread, valid until the next call, never NULL */
const char* fe_engine_last_error(void);

/* engine.h:65-71: load with FLOWEDGE_THREADS (0..8). FLOWEDGE_CUDA_FORCE_HOST=1
 * is a load error here (no host kernels exist); FLOWEDGE_CUDA_REQUIRED=1 is
 * always satisfied by a successful load. */
fe_engine* fe_engine_load(const char* path);
/* engine.h:73-82: worker_threads above 8 are rejected */
fe_engine* fe_engine_load_with_threads(const char* path, unsigned worker_threads);
/* engine.h:84-85 */
fe_weights* fe_weights_load(const char* path);
/* engine.h:87-88 */
size_t fe_weights_size_bytes(const fe_weights* weights);
/* engine.h:90-91 */
void fe_weights_free(fe_weights* weights);
/* engine.h:93-94 */
fe_engine* fe_engine_create_from_weights(const fe_weights* weights, unsigned worker_threads);
/* engine.h:96-97 */
fe_engine* fe_engine_create_from_weights_auto(const fe_weights* weights);
/* engine.h:99-105 */
void fe_engine_dims(const fe_engine* engine, size_t* d_model, size_t* n_layers);
/* engine.h:107-114: Mamba prefill, out [seq_len][d_model] */
int fe_engine_run(fe_engine* engine, const int32_t* tokens, size_t seq_len, float* out);
/* engine.h:116-124: Transformer backbone (not built: FE_STATUS_UNSUPPORTED_MODEL) */
int fe_engine_run_embeddings(fe_engine* engine, const float* embeddings, size_t seq_len, float* out);
/* engine.h:126-134 (not built: FE_STATUS_UNSUPPORTED_MODEL) */
int fe_engine_run_embeddings_masked(fe_engine* engine, const float* embeddings, const uint8_t* attention_mask,
                                    size_t seq_len, float* out);
/* engine.h:136-146: SmolVLA suffix embedding, out [chunk_size][expert_width] */
int fe_engine_smolvla_embed_suffix(fe_engine* engine, const float* noisy_actions, size_t chunk_size,
                                   float timestep, float* out);
/* engine.h:148-161: the expert's layers over a caller-supplied prefix cache
 * [expert_layers][prefix_length][cache_width] (cache_width = the K / V width in
 * the reference's layout; this build also accepts a wider cache that the
 * cross-attention layers project, e.g. a 960-wide prefix for 12 heads of 60) */
int fe_engine_smolvla_run_expert(fe_engine* engine, const float* suffix, size_t chunk_size,
                                 const float* prefix_keys, const float* prefix_values, const uint8_t* prefix_mask,
                                 size_t prefix_length, float* out);
/* engine.h:163-171 */
int fe_engine_smolvla_project_actions(fe_engine* engine, const float* hidden, size_t chunk_size, float* out);
/* engine.h:173-183 */
int fe_engine_smolvla_denoise(fe_engine* engine, const float* noisy_actions, size_t chunk_size, float timestep,
                              const float* prefix_keys, const float* prefix_values, const uint8_t* prefix_mask,
                              size_t prefix_length, float* out);
/* engine.h:185-196: Euler sample, t = 1 - step / steps */
int fe_engine_smolvla_sample(fe_engine* engine, const float* initial_noise, size_t chunk_size, size_t steps,
                             const float* prefix_keys, const float* prefix_values, const uint8_t* prefix_mask,
                             size_t prefix_length, float* out);
/* engine.h:198-205: streaming Mamba decode of one token, out [d_model] */
int fe_engine_step(fe_engine* engine, int32_t token, float* out);
/* engine.h:207-211 */
void fe_engine_reset(fe_engine* engine);
/* engine.h:213-218 */
unsigned fe_engine_thread_count(const fe_engine* engine);
/* engine.h:220-228: always 1 for a loaded engine (weights are device-resident) */
int fe_engine_cuda_resident(const fe_engine* engine);
/* engine.h:230-231 */
int fe_engine_model_metadata(const fe_engine* engine, fe_model_metadata* metadata);
/* engine.h:233-239: returns 2 when the checkpoint has no deployment profile */
int fe_engine_deployment_profile(const fe_engine* engine, fe_deployment_profile* profile);
/* engine.h:241-246 */
size_t fe_engine_action_dim(const fe_engine* engine);
/* engine.h:248-251 */
size_t fe_engine_action_horizon(const fe_engine* engine);
/* engine.h:253-254 */
int fe_engine_diffusion_metadata(const fe_engine* engine, fe_diffusion_metadata* metadata);
/* engine.h:256-261 */
size_t fe_engine_condition_dim(const fe_engine* engine);
/* engine.h:263-279: DDIM (eta 0) / DDPM sample, action in original units */
int fe_engine_sample_diffusion(fe_engine* engine, const float* condition, const float* noise, size_t steps,
                               int scheduler, uint64_t seed, float* action);
/* engine.h:281-284: one epsilon prediction in normalized action space */
int fe_engine_diffusion_denoise(fe_engine* engine, const float* condition, const float* normalized_sample,
                                float timestep, float* predicted_noise);
/* engine.h:286-303: Mamba condition from tokens, then the flow ODE */
int fe_engine_sample(fe_engine* engine, const int32_t* tokens, size_t seq_len, const float* noise, size_t steps,
                     int method, float* action);
/* engine.h:305-322 */
int fe_engine_sample_condition(fe_engine* engine, const float* condition, const float* noise, size_t steps,
                               int method, float* action);
/* engine.h:324-333 */
int fe_engine_flow_begin(fe_engine* engine, const float* condition, const float* noise, size_t steps, int method);
/* engine.h:335-341 */
int fe_engine_make_condition_metadata(const fe_engine* engine, uint64_t timestamp_ns, uint64_t deadline_ns,
                                      uint64_t generation, size_t steps, int method,
                                      fe_condition_metadata* metadata);
/* engine.h:343-345 */
int fe_engine_flow_begin_request(fe_engine* engine, const float* condition, const float* noise,
                                 const fe_condition_metadata* metadata);
/* engine.h:347-351: the one call that is safe concurrently with fe_engine_flow_advance */
void fe_engine_cancel_before(fe_engine* engine, uint64_t generation);
/* engine.h:353-365 */
int fe_engine_flow_advance(fe_engine* engine, size_t step_budget, float* action, size_t* steps_remaining);
/* engine.h:367-368 */
int fe_engine_flow_action_metadata(const fe_engine* engine, fe_action_metadata* metadata);
/* engine.h:370-375: 96-byte header + decode state */
size_t fe_engine_decode_state_bytes(const fe_engine* engine);
/* engine.h:377-383 */
int fe_engine_export_decode_state(const fe_engine* engine, void* destination, size_t bytes);
/* engine.h:385-391 */
int fe_engine_import_decode_state(fe_engine* engine, const void* source, size_t bytes);
/* engine.h:393-397 */
void fe_engine_free(fe_engine* engine);

/* ------------------------------------------------------------------------- */
/* Part 2: extensions (no counterpart in the reference, which is batch 1)     */

enum { FE_PRECISION_MODE_AUTO = 0, FE_PRECISION_MODE_F32 = 1, FE_PRECISION_MODE_BF16 = 2 };

typedef struct fe_engine_options {
  uint32_t struct_size;    /* sizeof(fe_engine_options) */
  uint32_t worker_threads; /* 0..8, kept for fe_engine_thread_count */
  int32_t device;          /* CUDA device index; -1 = FLOWEDGE_DEVICE or 0 */
  uint32_t precision;      /* FE_PRECISION_MODE_*; AUTO = bf16 if the file stores bf16 weights */
  uint64_t max_batch;      /* batch capacity reserved at load (0 = FLOWEDGE_MAX_BATCH or 1) */
  uint64_t max_sequence;   /* Mamba prefill capacity in tokens (0 = 512) */
  /* 32, 64 or 128: the Mamba in / x / out projections' weights are rounded to
   * 4 bits with one scale per that many inputs (the rule of
   * fe_w4_quantize_device), and every Mamba entry point computes with them.
   * Calls over slots read the packed form for fewer than 128 rows, and for any
   * number in projections whose inputs (d_model; d_inner) are no multiple of
   * 64, which the tensor path does not take.  All others read the full-width
   * copy, which a bf16 engine holds in fp16 (rounded once more) and which stays
   * beside the packed one: the option saves time, not memory.  0: off.  A
   * structure that ends before this field (struct_size 32) reads as 0. */
  uint32_t weights4_group;
  uint32_t reserved; /* 0 (of a structure that holds it, struct_size 40) */
} fe_engine_options;

/* Load with explicit options (device, precision, batch capacity). */
fe_engine* fe_engine_load_with_options(const char* path, const fe_engine_options* options);
/* Shared-weight variant of fe_engine_load_with_options. */
fe_engine* fe_engine_create_from_weights_with_options(const fe_weights* weights, const fe_engine_options* options);

/* Grow the device workspace to hold `max_batch` independent samples.  This is
 * the only call besides loading that allocates device memory; calls with
 * batch <= the reserved capacity never allocate. */
int fe_engine_reserve_batch(fe_engine* engine, size_t max_batch);

/* Batched fe_engine_sample_diffusion: condition [batch][C], noise and action
 * [batch][H][A].  Sample b uses DDPM seed `seed + b`. */
int fe_engine_sample_diffusion_batch(fe_engine* engine, const float* condition, const float* noise, size_t batch,
                                     size_t steps, int scheduler, uint64_t seed, float* action);
/* Batched fe_engine_diffusion_denoise. */
int fe_engine_diffusion_denoise_batch(fe_engine* engine, const float* condition, const float* normalized_sample,
                                      size_t batch, float timestep, float* predicted_noise);
/* As fe_engine_sample_diffusion_batch with DEVICE pointers, enqueued on
 * `stream` (a cudaStream_t, NULL = the engine's stream); returns before the
 * work completes. */
int fe_engine_sample_diffusion_device(fe_engine* engine, const float* condition, const float* noise, size_t batch,
                                      size_t steps, int scheduler, uint64_t seed, float* action, void* stream);
/* Batched fe_engine_sample_condition: condition [batch][C], noise/action [batch][A]. */
int fe_engine_sample_condition_batch(fe_engine* engine, const float* condition, const float* noise, size_t batch,
                                     size_t steps, int method, float* action);
/* Device-pointer variant of fe_engine_sample_condition_batch. */
int fe_engine_sample_condition_device(fe_engine* engine, const float* condition, const float* noise, size_t batch,
                                      size_t steps, int method, float* action, void* stream);
/* Allocation-free variant of fe_engine_sample_condition_device (no
 * counterpart in the reference ABI).  For callers that cannot call cudaMalloc
 * while they sample - a fixed-period control loop, where cudaMalloc may block
 * and synchronise the device, or a host process whose device memory another
 * runtime's pool allocator claimed at start-up - it runs the flow ODE solve on caller device buffers (condition [batch][C],
 * noise / action [batch][A], enqueued on `stream`) with its scratch in a
 * fixed 4 MiB static device array that every GPU loading the library holds
 * until exit, never touching the engine's reserved workspace.  Requests whose
 * scratch exceeds 4 MiB are rejected with FE_STATUS_RESOURCE_EXHAUSTED.  The
 * first call on a device looks up the array's address; make it before any
 * stream capture.  Calls share the array: calls that overlap on the GPU race. */
int fe_engine_sample_condition_static(fe_engine* engine, const float* condition, const float* noise, size_t batch,
                                      size_t steps, int method, float* action, void* stream);
/* Batched Mamba prefill: tokens [batch][seq_len], out [batch][seq_len][d_model]. */
int fe_engine_run_batch(fe_engine* engine, const int32_t* tokens, size_t batch, size_t seq_len, float* out);
/* Mamba prefill on DEVICE buffers, enqueued on `stream` (NULL = the engine's
 * stream): tokens [batch][seq_len] (ids are not range-checked on the host),
 * last_hidden [batch][d_model] = the final-normed hidden state of each
 * sequence's last position (the flow condition).  Returns before the work
 * completes; batch * seq_len must fit the reserved capacity. */
int fe_engine_run_device(fe_engine* engine, const int32_t* tokens, size_t batch, size_t seq_len, float* last_hidden,
                         void* stream);
/* Many sequences over slots: a pool of decode states on the device, so that
 * ragged prompts leave the state that single tokens then continue from.
 * fe_engine_reserve_slots makes room for slots 0 .. n_slots - 1 (zero states;
 * a larger pool keeps the states of a smaller one) and, together with
 * fe_engine_reserve_batch and max_batch x max_sequence, is what allocates.
 * Slots are apart from the one state of fe_engine_step.  A call takes at most
 * 2^16 sequences.  Growth moves buffers:
 * a graph in which the caller captured one of the calls below is no longer
 * valid behind it (a prompt_batch or step_batch of more rows than there is
 * room for grows too, and a growth that fails for want of memory may have moved
 * them all the same; it changes no state and no capacity otherwise). */
int fe_engine_reserve_slots(fe_engine* engine, size_t n_slots);
/* Zero states for n slots. */
int fe_engine_reset_slots(fe_engine* engine, const int32_t* slots, size_t n);
/* Prompts of lengths[s] >= 1 tokens, one after the other in `tokens`, each
 * for a slot of its own: from a zero state, or with resume != 0 from the
 * slot's.  last_hidden [n_seq][d_model] takes the final-normed hidden state
 * of each prompt's last token (the flow condition); the slots take the states
 * behind it.  Host buffers, synchronous. */
int fe_engine_prompt_batch(fe_engine* engine, const int32_t* tokens, const size_t* lengths, const int32_t* slots,
                           size_t n_seq, int resume, float* last_hidden);
/* The same with DEVICE pointers, enqueued on `stream` (NULL = the engine's
 * stream): offsets [n_seq + 1] into the rows, slots [n_seq] (negative: the
 * sequence is skipped), fresh [n_seq] (nonzero: from a zero state; NULL: all
 * continue), sequences checked as in part 3 with their bits in *status (may
 * be NULL).  Rows of last_hidden without a sequence that ran are left as they
 * were.  A token outside the vocabulary reads as a zero embedding, and where its
 * sequence ran fe_engine_synchronize reports it (what rows that do not run hold
 * is no fault).  Any other fault of a call on device buffers is reported by the
 * next call on host buffers before that changes a state.  rows must fit max_batch x max_sequence
 * and n_seq the reserved slots.  Calls of one engine share its workspace:
 * they must not overlap. */
int fe_engine_prompt_device(fe_engine* engine, const int32_t* tokens, size_t rows, const int32_t* offsets,
                            const int32_t* slots, const uint8_t* fresh, size_t n_seq, float* last_hidden,
                            int32_t* status, void* stream);
/* One token for each of n slots: out [n][d_model].  Host buffers, synchronous. */
int fe_engine_step_batch(fe_engine* engine, const int32_t* tokens, const int32_t* slots, size_t n, float* out);
/* The same with DEVICE pointers, as fe_engine_prompt_device; rows of out with
 * a negative slot are left as they were (a padded batch). */
int fe_engine_step_device(fe_engine* engine, const int32_t* tokens, const int32_t* slots, size_t n, float* out,
                          int32_t* status, void* stream);
/* Batched fe_engine_sample: tokens [batch][seq_len], noise/action [batch][A]. */
int fe_engine_sample_batch(fe_engine* engine, const int32_t* tokens, size_t batch, size_t seq_len,
                           const float* noise, size_t steps, int method, float* action);
/* Batched fe_engine_smolvla_sample: initial_noise / out [batch][chunk_size][max_action_dim];
 * prefix_keys / prefix_values [batch][expert_layers][prefix_length][cache_width] and
 * prefix_mask [batch][prefix_length], or one prefix for every sample when
 * shared_prefix != 0. */
int fe_engine_smolvla_sample_batch(fe_engine* engine, const float* initial_noise, size_t batch, size_t chunk_size,
                                   size_t steps, const float* prefix_keys, const float* prefix_values,
                                   const uint8_t* prefix_mask, size_t prefix_length, int shared_prefix, float* out);
/* As fe_engine_smolvla_sample_batch with DEVICE pointers, enqueued on `stream`
 * (NULL = the engine's stream); returns before the work completes.  The mask is
 * not validated on the host. */
int fe_engine_smolvla_sample_device(fe_engine* engine, const float* initial_noise, size_t batch, size_t chunk_size,
                                    size_t steps, const float* prefix_keys, const float* prefix_values,
                                    const uint8_t* prefix_mask, size_t prefix_length, int shared_prefix, float* out,
                                    void* stream);
/* Reserve the SmolVLA workspace for `batch` chunks of `chunk_size` tokens and
 * prefixes of `prefix_length` slots (the only SmolVLA call besides the first
 * sample of a larger shape that allocates device memory). */
int fe_engine_smolvla_reserve(fe_engine* engine, size_t batch, size_t chunk_size, size_t prefix_length,
                              int shared_prefix);
/* Wait for all work enqueued by this engine. */
int fe_engine_synchronize(fe_engine* engine);

/* Profile one U-Net forward of `batch` samples on the tensor-core path with
 * CUDA events around every convolution GEMM: metrics[0] = summed GEMM kernel
 * milliseconds, [1] = GEMM launches, [2] = algorithmic GEMM FLOPs,
 * [3] = whole forward milliseconds.  The batch must be within the reserved
 * capacity and use the tensor-core path (bf16 mode). */
int fe_engine_profile_diffusion(fe_engine* engine, size_t batch, double* metrics);

/* Process-wide counts of device / pinned-host allocations made by this library. */
uint64_t fe_device_malloc_count(void);
uint64_t fe_host_malloc_count(void);
/* Kernel launches issued by this engine so far (graph replays counted per node). */
uint64_t fe_engine_kernel_launches(const fe_engine* engine);

/* ------------------------------------------------------------------------- */
/* Part 3: operators on device buffers (no counterpart in the reference)      */
/*
 * The operators of a Mamba layer over many independent sequences, the mixer's
 * state kept in slots.  Every pointer is a device pointer; the work is enqueued on
 * `stream` (a cudaStream_t; NULL is the default stream) of the device
 * args->device (-1: the calling thread's current device) and the call returns
 * before it completes.  No call allocates, synchronises or keeps anything, so
 * calls may be captured into CUDA graphs and may run at the same time on
 * different streams as long as their outputs, states and workspaces differ.
 * Returns FE_STATUS_OK, FE_STATUS_INVALID_ARGUMENT (nothing was launched;
 * fe_engine_last_error names the argument) or FE_STATUS_RESOURCE_EXHAUSTED
 * (the launch failed).
 *
 * Rows and sequences.  Activations are matrices of `rows` rows; a row is
 * contiguous and `*_ld` elements from the next.  With `offsets` ([n_seq + 1],
 * not decreasing, within 0 .. rows) sequence s is the rows offsets[s] ..
 * offsets[s + 1] - 1, possibly none; rows outside every sequence are left as
 * they were.  Without offsets every row is a sequence of one token and n_seq
 * must equal rows.  Sequence s has slot slots[s] (without slots, slot s); a
 * negative slot skips the sequence: neither its rows nor any slot change.  A
 * sequence with fresh[s] != 0 starts from a zero state whatever its slot
 * holds.  A state pointer of NULL means: every sequence starts from zero and
 * no state is kept.
 *
 * A call with states and slots has at most 2^16 sequences (each looks for its
 * slot among those before it, so the cost grows with their square: up to some
 * 8192 it is a small part of the call).
 *
 * Offsets and slots are read on the device.  A sequence whose offsets lie
 * outside the rows, whose slot is n_slots or more, or whose slot an earlier
 * sequence of the call has, is skipped, and the FE_SEQ_* bit is set in
 * *status (an int32 in device memory that the call only adds bits to; may be
 * NULL).  Offsets that decrease set the bit too; which of the call's other
 * sequences run is then undefined, as is what rows and slots of sequences that
 * overlap hold, but nothing outside the call's buffers is touched.
 */
enum { FE_DTYPE_F32 = 0, FE_DTYPE_BF16 = 1, FE_DTYPE_F16 = 2 };

enum { FE_SEQ_BAD_OFFSETS = 1, FE_SEQ_BAD_SLOT = 2, FE_SEQ_DUPLICATE_SLOT = 4 };

/* u[t][c] = SiLU(b[c] + sum_k w[c][k] x[t - (d_conv - 1) + k][c]), the inputs
 * before a sequence's first row taken from its slot's window; then the window
 * takes the sequence's last d_conv inputs (the layout of the decode state:
 * [d_inner][d_conv], newest last, fp32; slot i is slot_stride floats after
 * slot i - 1).  x and u are `dtype`, w and b fp32, sums fp32.  d_conv 1 .. 8.
 * u may share no element with x. */
typedef struct fe_conv_args {
  uint32_t struct_size; /* sizeof(fe_conv_args) */
  int32_t device;
  uint32_t dtype; /* FE_DTYPE_* of x and u */
  uint32_t d_conv;
  uint64_t rows, d_inner, n_seq, n_slots;
  int64_t x_ld, u_ld, slot_stride;
  const void* x;
  const float* w; /* [d_inner][d_conv] */
  const float* b; /* [d_inner] */
  void* u;
  float* window; /* [n_slots][slot_stride], or NULL */
  const int32_t* offsets;
  const int32_t* slots;
  const uint8_t* fresh;
  int32_t* status;
} fe_conv_args;
int fe_causal_conv_device(const fe_conv_args* args, void* stream);

/* The selective scan.  A row of proj is [dt_in (dt_rank) | B (d_state) | C
 * (d_state)]; per row t and channel c
 *   dt = softplus(dt_b[c] + sum_r dt_in[r] dt_w[r][c])
 *   h_n = exp(dt a[n][c]) h_n + dt B_n u[t][c]
 *   y[t][c] = (d[c] u[t][c] + sum_n h_n C_n) SiLU(z[t][c])    (no z: no gate)
 * u, proj, z and y are `dtype`; weights, states ([d_state][d_inner] per slot)
 * and all sums are fp32.  d_state 1 .. 32, dt_rank 1 .. 512.  y may share no
 * element with u, z or proj.  `workspace` holds the rows' steps dt (of
 * prompts, and of many single tokens) and the partial states of prompts that
 * are scanned in parallel pieces: at least fe_selective_scan_workspace(args)
 * bytes (0 for few single tokens), 16-byte aligned, in use until the call's
 * work completes. */
typedef struct fe_scan_args {
  uint32_t struct_size; /* sizeof(fe_scan_args) */
  int32_t device;
  uint32_t dtype; /* FE_DTYPE_* of u, proj, z and y */
  uint32_t d_state;
  uint64_t rows, d_inner, dt_rank, n_seq, n_slots;
  int64_t u_ld, proj_ld, z_ld, y_ld, slot_stride;
  const void* u;
  const void* proj;
  const void* z; /* or NULL */
  const float* a;    /* [d_state][d_inner], negative */
  const float* d;    /* [d_inner] */
  const float* dt_w; /* [dt_rank][d_inner] */
  const float* dt_b; /* [d_inner] */
  void* y;
  float* state; /* [n_slots][slot_stride], or NULL */
  const int32_t* offsets;
  const int32_t* slots;
  const uint8_t* fresh;
  int32_t* status;
  void* workspace;
  uint64_t workspace_bytes;
} fe_scan_args;
int fe_selective_scan_device(const fe_scan_args* args, void* stream);
/* Reads the sizes, device and offsets (only whether given) of args. */
size_t fe_selective_scan_workspace(const fe_scan_args* args);

/* Weights of 4 bits with group scales: w[m][k] = (q[m][k] - 8) scales[m][k / group],
 * q from 0 to 15, scales fp16 [m][ceil(k / group)], group 32, 64 or 128.
 * `packed` is 16-byte aligned.  A 32-bit word holds eight neighbouring elements;
 * its nibbles 0 .. 7, lowest first, are the elements 0, 2, 4, 6, 1, 3, 5, 7 of
 * the eight (so that one mask takes out two neighbours).  Elements behind the
 * last are 8, that is zero.  The words' order:
 * FE_W4_ROWS: [m][ceil(k / 32)][16 bytes], the words in the order of their
 * elements.
 * FE_W4_BLOCKS: [m][ceil(k / 128)][64 bytes]; the word at place 4 t + j (t, j
 * from 0 to 3) of a block of 128 elements holds those from 32 j + 8 t on, so
 * that a thread's words of four groups come in one load.
 * A structure that ends before `layout` (struct_size 88) reads as FE_W4_BLOCKS.
 *
 * fe_w4_matvec_device: y[r][m] = sum_k x[r][k] w[m][k] for a few rows; x and y
 * are `dtype`, sums fp32 (an fp32 x enters the products unrounded).  Up to 32
 * rows read the weights once; more rows run in passes of 32.  y may share no
 * element with x.
 * fe_w4_quantize_device: packed and scales from the weight matrix x
 * ([m][x_ld], `dtype`, finite): scale = the group's largest magnitude / 7
 * rounded to fp16 (at most 65504), q = round(w / scale) + 8 within 0 .. 15,
 * ties to even (rows is not read).
 * fe_w4_dequantize_device: the weights as `dtype` into y ([m][y_ld]). */
enum { FE_W4_BLOCKS = 0, FE_W4_ROWS = 1 };

typedef struct fe_w4_args {
  uint32_t struct_size; /* sizeof(fe_w4_args) */
  int32_t device;
  uint32_t dtype;
  uint32_t group;
  uint64_t rows, m, k;
  int64_t x_ld, y_ld;
  const void* x;
  void* packed;
  void* scales;
  void* y;
  uint32_t layout;   /* FE_W4_* of packed */
  uint32_t reserved; /* 0 */
} fe_w4_args;
int fe_w4_matvec_device(const fe_w4_args* args, void* stream);
int fe_w4_quantize_device(const fe_w4_args* args, void* stream);
int fe_w4_dequantize_device(const fe_w4_args* args, void* stream);

/* The residual between two blocks and the norms around it, per row:
 *   t = x post_weight / sqrt(mean(x^2) + eps)      (t = x without post_weight)
 *   residual = residual + scale gate t             (gate 1 without gate)
 *   out = residual weight / sqrt(mean(residual^2) + eps)
 * x, gate and out are `dtype`, the residual (updated in place) fp32 or
 * `dtype`, weights fp32; sums and the norm's input are fp32, before the
 * residual's rounding.  gate_ld 0 gives every row the same gate.  dim 1 ..
 * 16384, scale and eps finite.  out, residual, x and gate share no element. */
typedef struct fe_norm_args {
  uint32_t struct_size; /* sizeof(fe_norm_args) */
  int32_t device;
  uint32_t dtype;
  uint32_t residual_dtype;
  uint64_t rows, dim;
  int64_t x_ld, residual_ld, gate_ld, out_ld;
  const void* x;
  const float* post_weight; /* [dim], or NULL */
  const void* gate;         /* or NULL */
  void* residual;
  const float* weight; /* [dim] */
  void* out;
  float scale;
  float eps;
} fe_norm_args;
int fe_residual_norm_device(const fe_norm_args* args, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif

#endif /* FLOWEDGE_B200_H */
