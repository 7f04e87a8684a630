/*
 * kleos_b200 — C ABI of the B200-native distributed MoE layer forward pass.
 *
 * Every entry point below replaces one inline C++ host function of the reference project
 * (namespace kleos); the reference file:line each one stands in for is cited beside it.
 * All functions return 0 on success or a negative KLEOS_E_* code; none of them exits the
 * process (the reference prints and calls exit()/quick_exit(), debug.cuh:19-43).
 *
 * Threading model is the reference's: one host thread per process, one process per GPU,
 * global state, not re-entrant (types.cuh:440,1011-1013).
 */
#ifndef KLEOS_B200_H
#define KLEOS_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    KLEOS_OK = 0,
    KLEOS_E_CONFIG = -1,      /* unreadable or invalid kleos_config.json            */
    KLEOS_E_STATE = -2,       /* call order: not initialised / already initialised  */
    KLEOS_E_CUDA = -3,        /* a CUDA runtime or driver call failed               */
    KLEOS_E_BOOTSTRAP = -4,   /* NCCL bootstrap or peer mapping failed              */
    KLEOS_E_MISMATCH = -5,    /* ranks disagree on the configuration                */
    KLEOS_E_DEVICE = -6,      /* the device reported a timeout or a bounds error    */
    KLEOS_E_UNSUPPORTED = -7, /* dtype / shape outside what the kernels implement   */
    KLEOS_E_ARG = -8          /* null pointer or out-of-range argument              */
};

/* Where a device-side problem was detected (kleos_status.where). */
enum {
    KLEOS_AT_NONE = 0,
    KLEOS_AT_PLAN_WAIT = 1,     /* waiting for dispatch flags from the source ranks */
    KLEOS_AT_COMBINE_WAIT = 2,  /* waiting for result flags from the expert ranks   */
    KLEOS_AT_GEMM_PRODUCER = 3, /* TMA producer waiting for a free pipeline stage   */
    KLEOS_AT_GEMM_MMA = 4,      /* MMA issuer waiting for operands or accumulator   */
    KLEOS_AT_GEMM_EPILOGUE = 5, /* epilogue waiting for an accumulator              */
    KLEOS_AT_BOUNDS = 6,        /* an index outside its table                       */
    KLEOS_AT_GRID_BARRIER = 7   /* blocks of the persistent kernel waiting for one another */
};

typedef struct kleos_status {
    int32_t code;   /* 0, or KLEOS_E_DEVICE */
    int32_t where;  /* KLEOS_AT_*           */
    int32_t detail; /* rank / cell / tile the detector was looking at */
    int32_t epoch;  /* forward-call counter when it happened */
} kleos_status;

typedef struct kleos_layer_info {
    int32_t rank, world, local_experts;
    int32_t S, H, I, E, K, EC, pEC, PX;
    int32_t torch_dtype, hidden_act, elem_bytes;
    int64_t input_elems;  /* elements in the packed input buffer  iP */
    int64_t output_elems; /* elements in the packed output buffer oP */
} kleos_layer_info;

/* Bootstrap helper: rank 0 creates the 128-byte NCCL unique id that every rank passes to
 * kleos_initialize.  The reference bootstraps through nvshmem_init() under an MPI/PMI
 * launcher instead (bootstrap.cuh:295). */
int kleos_get_unique_id(void* out_id128);

/* Select the CUDA device before kleos_initialize (reference: setDevice(),
 * bootstrap.cuh:549-553).  Default is rank % device count. */
int kleos_set_device(int device);

/* Read kleos_config.json (same keys as kleos_config.schema.json:5-89, parsed at run time
 * instead of being baked in by CMake), allocate the symmetric cells, flags and bookkeeping,
 * and map every peer's cells.  Replaces kleos::initialize() (bootstrap.cuh:532-547).
 * nccl_id may be NULL when world == 1. */
int kleos_initialize(const char* config_json_path, int rank, int world, const void* nccl_id);

/* Parse a kleos_config.json and report the derived sizes for a given world size without
 * touching the GPU (rank is reported as 0).  Same derivations as the reference's compile-time
 * ACC struct (types.cuh:442-513). */
int kleos_config_probe(const char* config_json_path, int world, kleos_layer_info* out);

/* Optional per-expert logit bias (E floats, host memory).  The reference gate has no bias
 * (moe/gate.cuh:87-88); the load-imbalanced benchmark layer needs one.  NULL clears it. */
int kleos_set_gate_bias(const float* host_bias, int n);

/* One layer forward, asynchronous on `stream` (a cudaStream_t, or NULL for the per-thread
 * default stream the reference uses, types.cuh:1013).  iP and oP are DEVICE pointers to the
 * packed buffers of moe.cuh:92-98:
 *   iP = [A S*H][Wg PX*H][W1 nLx*I*H][W2 nLx*H*I][b1 nLx*I][b2 nLx*H]
 *   oP = [gate probabilities S*PX][layer output S*H]
 * With num_experts == 1 the layer is the plain FFN over the rank's own tokens, as in the
 * reference (moe/moe.cuh:197-204 launches moe/fffn.cuh:31-167): no gate and no exchange, every
 * rank holds the one expert (nLx = 1, any world size, no NCCL id needed), and the packed
 * buffers lose their gate sections:
 *   iP = [A S*H][W1 I*H][W2 H*I][b1 I][b2 H]      oP = [layer output S*H]
 * Replaces kleos::moe::forwardHost(iP, oP) (moe/moe.cuh:186-205). */
int kleos_forward(const void* iP, void* oP, void* stream);

/* skip warm-up forwards, then trials forwards between two CUDA events; *ms = mean per
 * forward.  Synchronises.  Replaces forwardHostBench<skip,trials> (moe/moe.cuh:146-184). */
int kleos_forward_bench(const void* iP, void* oP, int skip, int trials, float* ms);

/* End-to-end call with HOST buffers: copies S*H activations host->device into the A section
 * of iP, runs one forward, copies the S*H layer output device->host, and synchronises.
 * Weights stay resident in iP.  The reference driver does the same copies by hand
 * (main.cu:64-66). */
int kleos_forward_host(const void* host_activations, void* iP, void* oP, void* host_output);

/* Pipelined form of kleos_forward_host for a stream of batches: returns as soon as the step is
 * queued.  Activations and layer output are double-buffered inside the library, so the
 * host->device copy of step i+1 and the device->host copy of step i-1 overlap the forward of
 * step i (three streams).  host_output of a step is valid after kleos_host_sync(), which also
 * reports device-side errors.  The gate probabilities still land in oP.  The reference has no
 * counterpart (its driver copies once and loops on the device, main.cu:64-68). */
int kleos_forward_host_async(const void* host_activations, void* iP, void* oP, void* host_output);
int kleos_host_sync(void);

/* Reference: getRank() (bootstrap.cuh:555-559) and hostBookkeeping.nLx (main.cu:22). */
int kleos_get_rank(void);
int kleos_local_experts(void);
int kleos_get_info(kleos_layer_info* out);

/* Device-side status of the last forward calls; synchronises the library's stream.
 * The reference has no equivalent: its device waits spin forever (atomics.cuh:96-138). */
int kleos_last_status(kleos_status* out);
/* Forget a recorded device-side error (the first one sticks until cleared). */
int kleos_clear_status(void);

/* Routing results of the last forward, copied to host memory (any pointer may be NULL):
 * topk [S*K] expert ids, slots [S*K] slot inside the expert cell or -1 when dropped,
 * counts [E] unclamped tokens per expert, mcw [S] sum of the k winning probabilities.
 * The reference keeps these in its bookkeeping arena (types.cuh:697-1008) without an
 * accessor; parity tests need them. */
int kleos_debug_routing(int32_t* topk, int32_t* slots, uint32_t* counts, float* mcw);

/* Per-phase device time of the most recent kleos_forward_bench, in milliseconds averaged over
 * its trials: [0] route, [1] slots, [2] dispatch, [3] plan(wait), [4] GEMM1, [5] GEMM2,
 * [6] combine, [7] whole forward.  n = number of floats the caller provides (>= 8). */
int kleos_phase_times(float* ms, int n);

/* With KLEOS_FLOW=1 16-bit routed layers run the router, dispatch, plan, both expert GEMMs and the
 * combine as ONE persistent kernel (the reference's arrangement, moe/moe.cuh:77-144); the phases above are
 * then read from the blocks' global-timer stamps: [0] gate GEMM + top-k up to the first grid
 * barrier, [1] slots up to the second; [2] last row dispatched and [3] tile plan known, both
 * counted from the second barrier; [4] span of the GEMM1 tiles; [5] from the last GEMM1 tile to
 * the last tile; [6] from the last tile to the kernel's end.  This call returns the raw
 * milestones of the most recent kleos_forward_bench, milliseconds after the earliest block's
 * start, latest block each: [0] 0, [1] plan known, [2] first tile begins (earliest block),
 * [3] last GEMM1 tile done, [4] last tile done, [5] last row dispatched, [6] last token combined,
 * [7] last block ends, [8] routing done (first grid barrier), [9] slots done (second),
 * [10] gate logits of the last token tile complete, [11] ... and turned into choices; with
 * n >= 19 also the router's inner steps: [12] top-k and softmax sum known, [13] near-ties
 * re-evaluated and probabilities stored, [14] base slots of the block's tile known, [15] slots
 * written, [16] set-up over and gate GEMM begins, [17] first K slice of the gate GEMM in shared
 * memory, [18] first pass over the logits done.  n >= 12.
 * KLEOS_E_STATE when the layer runs as separate launches (float and TF32 layers, the dense
 * layer, and every layer unless KLEOS_FLOW=1 is set). */
int kleos_flow_timeline(float* ms, int n);

/* The same stamps block by block, as written by the last timed forward of kleos_forward_bench:
 * ns[b * per_block + k] = global-timer nanoseconds of milestone k in block b (0: that block never
 * passed it).  *blocks and *per_block are always set; ns may be null to ask for the sizes only,
 * otherwise capacity >= *blocks * *per_block.  A tuning aid with no counterpart in the reference. */
int kleos_debug_flow_stamps(long long* ns, int capacity, int* blocks, int* per_block);

/* Wait times of the persistent kernel's tile-stream roles in the LAST timed forward of
 * kleos_forward_bench, milliseconds averaged over the blocks that recorded a value:
 * [0] producer waiting for a free stage, [1] for cell data / GEMM1 counters, [2] producer total,
 * [3] MMA issuer waiting for an accumulator, [4] for operands, [5] for the next claimed tile,
 * [6] issuer total, [7] read-back warp waiting for an accumulator, [8] publishing, [9] reading back
 * and storing, [10] read-back total, [11] producer's proxy fences.  n >= 12.  A tuning aid with no counterpart in
 * the reference. */
int kleos_debug_flow_stalls(float* ms, int n);

/* The segment order of the persistent kernel's tile queue for `local_experts` experts and a lag
 * of `lag` segments: phase[s] is 0 for the first expert GEMM and 1 for the second, expert[s] the
 * local expert of segment s; returns the number of segments (2 * local_experts).  Host only,
 * needs no GPU and no kleos_initialize; lets a test check that every second-GEMM segment follows
 * the first-GEMM segment it consumes (the reference chains the two per row panel at run time,
 * os/processor/processor.cuh:717-729). */
int kleos_debug_tile_order(int local_experts, int lag, int32_t* phase, int32_t* expert);

/* Kernels this library has launched for forward calls since kleos_initialize (every launch site
 * counts itself; memory copies and memsets are not kernels).  A benchmark reads it before and
 * after its timed region.  Negative (KLEOS_E_STATE) when not initialised.  No counterpart in the
 * reference, whose forward is always one launch (moe/moe.cuh:198). */
long long kleos_launch_count(void);

/* Stall counters of the last GEMM1 and GEMM2 launches, only when the environment variable
 * KLEOS_GEMM_STATS=1 was set at initialise time: [2][blocks][12] clock cycles per block
 * {producer wait-empty, producer total, MMA wait-accumulator, MMA wait-operands, MMA total,
 *  epilogue wait-accumulator, epilogue total, unused, prologue, unused, unused, unused}.  Returns the number of values written.
 * A tuning aid with no counterpart in the reference. */
int kleos_debug_gemm_stats(long long* out, int max_values);

/* Router only, for callers that cannot allocate device memory when they call (inside another
 * runtime's allocator callback, in a serving loop with a frozen memory budget, ...).  It has no
 * counterpart in the reference, which always routes inside its fused kernel.  It needs no
 * kleos_initialize: the scratch it uses (near-tie list, fp64 logits, counters; 2,130,432 bytes)
 * is a fixed array inside the library that every GPU loading it keeps until the process ends,
 * and the call performs no cudaMalloc / cudaFree.
 *   A [S,H], Wg [64,H] (row e = expert e, rows >= E zero), gate_bias [E] floats or NULL,
 *   probs [S,64] (element type), topk [S,K], mcw [S]: all DEVICE pointers owned by the caller;
 *   A and Wg must be 16-byte aligned (KLEOS_E_ARG otherwise).
 *   Limits: S <= 4096, E <= 64, K <= min(E, 8), H a multiple of 64, torch_dtype 0 or 2; anything
 *   larger is refused with KLEOS_E_ARG and a message on stderr.
 * The first call on each device looks up the array's device address; make that call before any
 * stream capture.  Float calls share the array, and each clears the part that must start at zero, so two
 * float calls that overlap on the GPU (different streams, different threads) race: serialise them.
 * bf16 calls only read the zero bias there and may overlap.  Asynchronous on `stream` (NULL = per-thread
 * default stream).  The bf16 kernel's waits are bounded (KLEOS_WAIT_MS at the first call on the device, about ten
 * seconds without it): a token whose logits did not come in time has topk = -1 and mcw = NaN. */
int kleos_route_static(const void* A, const void* Wg, const float* gate_bias, int S, int H, int E,
                       int K, int torch_dtype, void* probs, int32_t* topk, float* mcw,
                       void* stream);

/* Training-mode gate statistics of the last forward on this rank (is_training = 1 in the
 * configuration, num_experts > 1), the three quantities the reference keeps in its device
 * bookkeeping (types.cuh:944-960) and never copies out:
 *   mean_prob[e]  = (1/S) sum_t p(t,e), fp32 softmax probabilities      (moe/gate.cuh:607-635)
 *   mean_count[e] = (tokens of this rank that chose e, before capacity) / S   (:698-705)
 *   loss          = sum_e mean_prob[e] * mean_count[e] / E              (:763-773)
 * Host pointers, E floats / E floats / 1 float; any may be NULL.  The reference accumulates
 * with atomicAdd and never clears between launches; here every forward overwrites the values
 * and the sums run in a fixed order.  KLEOS_E_STATE when the layer was not set up for training. */
int kleos_gate_stats(float* mean_prob, float* mean_count, float* loss);

/* Init-time placement planner (host only, needs no GPU and no kleos_initialize): restates the
 * reference's Decider and expert assignment (os/decider/decider.cuh:37-329, used at start-up in
 * bootstrap.cuh:170-265).  From a latency / inverse-bandwidth matrix (alpha in ms, beta in ms per
 * MB, entry [i*world + j] = link i -> j), per-device throughput and the number of experts each
 * device can hold, it merges devices into expert-parallel groups and assigns the experts of the
 * asking rank's group to its members in proportion to throughput.
 *   device_to_group  [world]  representative device of every device's group
 *   group_ranks      [world]  first group_size entries: devices of rank's group, ascending
 *   expert_to_member [E]      index into group_ranks of the device that holds each expert
 * Output pointers may be NULL.  matches_data_path is 1 when the plan is the even contiguous
 * sharding over all ranks that kleos_initialize implements (the case of one NVSwitch node with
 * identical GPUs); other plans are reported but not executed by this library. */
typedef struct kleos_placement_request {
    int32_t world, rank, num_experts, expert_cost, is_training;
    uint32_t moe_stages, p2p_buffer_mb, grad_buffer_mb; /* see kleos_placement_model */
    const float* alpha;  /* [world*world] */
    const float* beta;   /* [world*world] */
    const float* rate;   /* [world] expert cost units per ms */
    const uint32_t* mem; /* [world] experts that fit */
} kleos_placement_request;

typedef struct kleos_placement_result {
    int32_t feasible, group_size, group_rank, local_experts, expert_slots, widest_group;
    int32_t matches_data_path;
} kleos_placement_result;

int kleos_plan_placement(const kleos_placement_request* request, kleos_placement_result* result,
                         uint32_t* device_to_group, uint32_t* group_ranks, uint32_t* expert_to_member);

/* The three cost-model constants the reference derives from the compiled layer
 * (types.cuh:487-494): global MoE stages, and the dispatch and gradient buffers in MB. */
int kleos_placement_model(const char* config_json_path, uint32_t* moe_stages, uint32_t* p2p_buffer_mb,
                          uint32_t* grad_buffer_mb);

/* ------------------------------------------------------------------------------------------------
 * Operators around the experts, for programs that train an MoE block, or serve one whose experts
 * kleos_forward does not compute: layer norm, the sort of tokens by expert with the rows there and
 * back, and the experts' products over the sorted rows, each with its gradients.  No counterpart
 * in the reference, whose layer is one fused forward.
 *
 * None of them needs kleos_initialize, allocates, synchronises with the host or keeps anything
 * from one call to the next, so they may be captured and calls may overlap on different streams.
 * They run on the current device, asynchronously on `stream` (NULL = per-thread default stream);
 * every pointer is a DEVICE pointer owned by the caller, and no output may overlap an input.
 * torch_dtype is 0 (float), 2 (bf16) or 3 (fp16); anything else is KLEOS_E_UNSUPPORTED.  A row
 * stride (ld...) counts elements and is at least the row's length.  Sums are kept in 32 bits and
 * rounded once, in a fixed order: the same call gives the same bits.  Where addresses, strides and
 * lengths are multiples of 16 bytes the kernels move 16 bytes at a time; others are taken too, more slowly. */

/* y = (x - mean) * rstd * weight + bias of every row, rstd = 1 / sqrt(var + eps), var the mean square of
 * x - mean.  x [rows, H] and y of torch_dtype, rows up to 2^31 - 2^16; weight [H] and bias [H] of param_dtype, 0 (float) or
 * torch_dtype, NULL for ones and zeros.  mean [rows] and rstd [rows] are floats for the backward pass and
 * may be NULL. */
int kleos_layer_norm(const void* x, long long ldx, const void* weight, const void* bias, int rows, int H, float eps,
                     int torch_dtype, int param_dtype, void* y, long long ldy, float* mean, float* rstd, void* stream);

/* Gradients of kleos_layer_norm: dx [rows, H] of torch_dtype, dweight [H] and dbias [H] of param_dtype (each may be
 * NULL), from dy and the mean and rstd that the forward pass gave.  dweight and dbias are overwritten (zeros when
 * rows is 0) and need a 16-byte aligned workspace of kleos_layer_norm_workspace(H) bytes, whose contents do not
 * matter: 296 partial sums of two rows of floats. */
long long kleos_layer_norm_workspace(int H);
int kleos_layer_norm_backward(const void* dy, long long lddy, const void* x, long long ldx, const void* weight,
                              const float* mean, const float* rstd, int rows, int H, int torch_dtype, int param_dtype,
                              void* dx, long long lddx, void* dweight, void* dbias, void* workspace,
                              long long workspace_bytes, void* stream);

/* Where the rows of each expert lie.  topk [T, K] holds the experts of every token (as kleos_route_static gives them);
 * an id outside 0 .. E - 1 is a place without an expert.
 *   offsets [E + 1]   rows of expert e: offsets[e] .. offsets[e + 1] - 1; offsets[E] = places with an expert
 *   row_of [T, K]     row of every place, in the order of the tokens within an expert; -1 without an expert
 *   source [T * K]    t * K + k of every row, -1 from offsets[E] on; may be NULL
 * K from 1 to 8, E from 1 to 1024. */
int kleos_sort_tokens(const int32_t* topk, int T, int K, int E, int32_t* offsets, int32_t* row_of, int32_t* source,
                      void* stream);

/* rows[row_of[t, k]] = x[t]: rows [T * K, H] sorted by expert, zeros from offsets[E] on. */
int kleos_gather_tokens(const void* x, long long ldx, const int32_t* row_of, const int32_t* offsets, int T, int K, int E,
                        int H, int torch_dtype, void* rows, void* stream);

/* out[t] = sum over k of weights[t, k] * rows[row_of[t, k]], places without an expert left out (zeros for a token that
 * has none).  weights [T, K] are floats; NULL for ones, which makes it the gradient of kleos_gather_tokens. */
int kleos_combine_tokens(const void* rows, const int32_t* row_of, const float* weights, int T, int K, int H, int torch_dtype,
                         void* out, long long ldo, void* stream);

/* Gradients of kleos_combine_tokens: drows[row_of[t, k]] = weights[t, k] * dout[t], zeros from offsets[E] on, and
 * dweights[t, k] = <dout[t], rows[row_of[t, k]]>, 0 without an expert; dweights may be NULL. */
int kleos_combine_tokens_backward(const void* dout, long long ldd, const void* rows, const int32_t* row_of,
                                  const float* weights, const int32_t* offsets, int T, int K, int E, int H,
                                  int torch_dtype, void* drows, float* dweights, void* stream);

/* y[r] = x[r] W[e]^T + bias[e] for the rows r of expert e, offsets[e] <= r < offsets[e + 1]; zeros for rows from
 * offsets[E] on.  x [rows, K], W [E, N, K], bias [E, N] or NULL, y [rows, N].  offsets is ascending from 0; what it says
 * beyond `rows` is not read.  E from 1 to 1024, rows up to 2^31 - 2^16. */
int kleos_expert_products(const void* x, long long ldx, const int32_t* offsets, const void* w, const void* bias, int rows,
                          int E, int N, int K, int torch_dtype, void* y, long long ldy, void* stream);

/* Gradients of kleos_expert_products: dx[r] = dy[r] W[e], zeros for rows from offsets[E] on; dW[e] = sum over the rows
 * of expert e of dy[r]^T x[r] and dbias[e] = sum of dy[r], zeros for an expert without rows.  dW [E, N, K] and
 * dbias [E, N] (or NULL) of grad_dtype, 0 (float) or torch_dtype.
 *
 * The sums of 16-bit products that become 16-bit results stay on the matrix unit, which cuts them off instead of rounding
 * them: up to about 2^-27 of the sum of the terms' magnitudes for every term, half a unit of fp16 after 2^16 terms of one
 * sign, of bf16 after 2^19.  dW in floats is read back every 256 rows instead and is within 1.4e-6 of the
 * 2-norm (measured up to 262144 rows). */
int kleos_expert_products_dx(const void* dy, long long lddy, const int32_t* offsets, const void* w, int rows, int E, int N,
                             int K, int torch_dtype, void* dx, long long lddx, void* stream);
int kleos_expert_products_dw(const void* dy, long long lddy, const void* x, long long ldx, const int32_t* offsets, int rows,
                             int E, int N, int K, int torch_dtype, int grad_dtype, void* dw, void* dbias, void* stream);

/* The activation between an expert's two products: h = f(z), or gated h = f(z[:, :I]) * z[:, I:], with f of hidden_act
 * 0 (ReLU), 1 (GELU, erf form) or 2 (SiLU, z / (1 + e^-z)).  z [rows, I], gated [rows, 2 I] (an expert's W1 has the rows of the
 * activated half first), h [rows, I].  Elements are computed in 32 bits. */
int kleos_activation(const void* z, long long ldz, long long rows, int I, int hidden_act, int gated, int torch_dtype, void* h,
                     long long ldh, void* stream);

/* Gradient of kleos_activation: dz from dh and z.  ReLU's slope at 0 is 0. */
int kleos_activation_backward(const void* dh, long long lddh, const void* z, long long ldz, long long rows, int I, int hidden_act,
                              int gated, int torch_dtype, void* dz, long long lddz, void* stream);

/* A whole MoE layer for the few tokens of a decode step.
 *   l = x gate^T + gate_bias;  the K largest l of a token (ties: the lower expert), their softmax as weights;
 *   out = sum over k of weights[t, k] (W2[e] h + b2[e]),  h as kleos_activation makes it of W1[e] x + b1[e],  e = topk[t, k]
 * x [T, H] and out [T, H] with row strides, gate [E, H], gate_bias [E] floats or NULL, W1 [E, I, H] (gated [E, 2 I, H]) and W2 [E, H, I]
 * as the products above take them, b1 and b2 or NULL; T from 0 to 128, K from 1 to 8.
 * topk [T, K] and weights [T, K] are written; with gate NULL they are what the caller's own router chose and are read: an id outside
 * 0 .. E - 1 is a place without an expert, and an expert may be named twice.  Logits are exact to about 2^-46 (those with
 * infinities in them, or past the floats' range on the way, are sums of 64 bits), h is rounded to
 * torch_dtype between the products (fp16: a value past 65504 is kept with 18 bits), everything else is 32 bits and one
 * rounding (sums of 16-bit products stay on the matrix unit, see above, for 8192 terms at most).  An expert
 * whose logit is minus infinity (a gate_bias that takes it out of service, a gate row, a token) is never chosen: its place has topk -1 and weight 0, and a
 * token without any expert has zeros.  NaN counts as the largest logit and makes its token's weights and results NaN.
 * The workspace (16-byte aligned, kleos_moe_tokens_workspace(T, I, K) bytes, contents of no matter) belongs to the call while it runs:
 * calls that may overlap have one each. */
long long kleos_moe_tokens_workspace(int T, int I, int K);
int kleos_moe_tokens(const void* x, long long ldx, const void* gate, const float* gate_bias, const void* w1, const void* b1,
                     const void* w2, const void* b2, int T, int H, int I, int E, int K, int hidden_act, int gated, int torch_dtype,
                     void* out, long long ldo, int32_t* topk, float* weights, void* workspace, long long workspace_bytes, void* stream);

/* Low-rank adapters of many requests beside a projection that they share: for the rows of request i, offsets[i] <= row <
 * offsets[i + 1], with l = adapter[i]
 *   u = x A[l]^T,   y = base + scale[l] u B[l]^T
 * x [rows, K], base and y [rows, N], A [L, r, K], B [L, N, r], scale [L] floats or NULL for ones, u [rows, r] floats for the backward
 * pass, or NULL.  base (what the shared projection gave) may be y itself, or NULL for zeros.  offsets [R + 1] is ascending; rows before the
 * first request or behind the last, and those of requests whose adapter is outside 0 .. L - 1, have y = base and u = 0.  On the tensor
 * cores (16-bit rows on 16-byte boundaries, r a multiple of 8, or of 4 up to 16) u, and v below, enter the second products rounded to
 * torch_dtype, fp16 after a division by a power of two: a row's values there, a rank's in the gradients.  Of those divided together the ones down
 * to 2^-28 of the largest keep fp16's bits.
 * R from 1 to 65536, L from 1 to 65535, r from 1 to 128. */
int kleos_adapter_products(const void* x, long long ldx, const int32_t* offsets, const int32_t* adapter, const void* a, const void* b,
                           const float* scale, const void* base, long long ldb, int rows, int R, int L, int r, int N, int K,
                           int torch_dtype, void* y, long long ldy, float* u, void* stream);

/* Gradients of kleos_adapter_products, from dy, x and the u of the forward pass:
 *   v = scale[l] dy B[l],   dx = dbase + v A[l],   dA[l] = sum of v^T x,   dB[l] = scale[l] sum of dy^T u
 * dbase (the shared projection's dx) may be dx itself, or NULL for zeros.  dA [L, r, K] and dB [L, N, r] of grad_dtype, 0 (float) or
 * torch_dtype, zeros for an adapter without rows, may be NULL.  On the tensor cores (as above, r even) results in 16 bits
 * of more than 512 rows are of u and v rounded to torch_dtype, and their long sums stay on the matrix unit, as those of kleos_expert_products_dw; those of fewer rows and results in floats are of u
 * and v in two parts (2^-16 of them in bf16, 2^-22 in fp16) and, floats, within 3e-6 of the 2-norm beside that.  dA needs a 16-byte aligned workspace of
 * kleos_adapter_products_workspace(rows, r) bytes, whose contents do not matter. */
long long kleos_adapter_products_workspace(int rows, int r);
int kleos_adapter_products_backward(const void* dy, long long lddy, const void* x, long long ldx, const float* u, const int32_t* offsets,
                                    const int32_t* adapter, const void* a, const void* b, const float* scale, const void* dbase,
                                    long long ldb, int rows, int R, int L, int r, int N, int K, int torch_dtype, int grad_dtype,
                                    void* dx, long long lddx, void* da, void* db, void* workspace, long long workspace_bytes,
                                    void* stream);

/* Test hook for the failure path: while on, the expert FFN does not raise its "results
 * returned" flags, so the combine's bounded wait runs out, the forward records
 * {KLEOS_E_DEVICE, KLEOS_AT_COMBINE_WAIT} and returns with the context intact.  Nothing is
 * faulted or hung; the wait budget is KLEOS_WAIT_MS.  No counterpart in the reference, whose
 * waits spin forever (atomics.cuh:96-138). */
int kleos_debug_suppress_return_flag(int on);

/* Free everything.  Replaces kleos::finalize() (bootstrap.cuh:561-588). */
int kleos_finalize(void);

const char* kleos_error_string(int code);

#ifdef __cplusplus
}
#endif
#endif /* KLEOS_B200_H */
