/*
 * tcu_scope.h -- C ABI of the B200 (sm_100a) segmented / full reduce and
 * inclusive-scan library for fp16 arrays.
 *
 * The reference project (c3sr/tcu_scope) has no FFI; its operator surface is
 * a set of header-only kernel templates
 *     compute_wmma_<op>_<variant><SEGMENT_SIZE, WARPS_PER_BLOCK, ...>
 *         (const half* d_in, OUT* d_out, [half* partial_sums,] size_t num_segments)
 * launched by one Google-Benchmark driver per variant.  Each entry point below
 * names the kernels / drivers it stands in for.  Conventions shared by all of
 * them, taken from those call sites:
 *   - the caller owns every device buffer (the drivers cudaMalloc them,
 *     src/reduction/seg_wmma_16n.cu:35-36); nothing here allocates or frees;
 *   - segment j occupies in[j*segment_size, (j+1)*segment_size)
 *     (src/reduction/seg_wmma_16n.cu:14-25);
 *   - work is queued on the given stream and the call returns at once;
 *   - the return value is a tcu_status; nothing throws, nothing resets the
 *     device (the reference does both, src/utils/error.hpp:28-46).
 * Pointers are plain device pointers (void*), streams are cudaStream_t passed
 * as void*; there are no C++ or torch types in any signature.
 */
#ifndef TCU_SCOPE_H_
#define TCU_SCOPE_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  TCU_OK              = 0,
  TCU_ERR_INVALID_ARG = 1, /* null / misaligned pointer, size overflow                  */
  TCU_ERR_UNSUPPORTED = 2, /* segment size 0, unknown algo/type, algo without that size   */
  TCU_ERR_CUDA        = 3, /* a CUDA runtime call failed (see cudaGetLastError)         */
  TCU_ERR_TIMEOUT     = 4, /* a bounded device-side wait ran out (tcu_device_error)     */
  TCU_ERR_WORKSPACE   = 5, /* workspace missing or smaller than tcu_workspace_bytes()   */
  TCU_ERR_TOO_LARGE   = 6, /* more elements than TCU_STATIC_SCAN_MAX_ELEMENTS           */
  TCU_ERR_INDEX       = 7  /* an index in device memory was wrong (tcu_device_error)    */
} tcu_status;

typedef enum {
  TCU_ALGO_AUTO    = 0, /* the fastest tensor-core kernel for the size: mma.sync, or
                           tcgen05 for large scans with 16-bit outputs                  */
  TCU_ALGO_MMA     = 1, /* TMA ring + mma.sync m16n8k16 against ones / triangular ones  */
  TCU_ALGO_SHUFFLE = 2, /* same pipeline, CUDA-core adds + warp shuffles: the ablation  */
  TCU_ALGO_TCGEN05 = 3  /* tcgen05.mma, accumulators in tensor memory; powers of two,
                           num_elements % 64 == 0: segmented reduction of 16 ... 2048
                           elements (plain fp32 accumulation), inclusive segmented scan
                           of 16 ... 16384 elements (exact parts, like TCU_ALGO_MMA),
                           with 16-bit outputs of up to 2^20 elements (2 segments or more) */
} tcu_algo;

typedef enum { TCU_OUT_F16 = 0, TCU_OUT_F32 = 1 } tcu_out_type;

typedef enum {
  TCU_OP_SEGMENTED_REDUCE = 0,
  TCU_OP_SEGMENTED_SCAN   = 1,
  TCU_OP_FULL_REDUCE      = 2,
  TCU_OP_FULL_SCAN        = 3
} tcu_op;

/* Input distributions of tcu_fill_f16 (bit-identical to the CPU oracle's). */
typedef enum {
  TCU_DIST_UNIFORM_PM1 = 0, /* uniform in [-1, 1)                                       */
  TCU_DIST_UNIFORM_01  = 1, /* uniform in [0, 1)                                        */
  TCU_DIST_SMALL_INT   = 2, /* integers -2..2 (every sum exact in any precision)        */
  TCU_DIST_CONST_0P001 = 3  /* half(0.001f): the reference's fill,
                               src/reduction/seg_wmma_16n.cu:38                          */
} tcu_dist;

/*
 * Segmented sum reduction: out[j] = sum of segment j.
 * Replaces compute_wmma_segmented_reduction_16n (src/reduction/kernel.cuh:80-125),
 * ..._256n (:301-356) and ..._256n_block (:418-485) and their drivers
 * CUDA_WMMA_SEGMENTED_REDUCTION_16N / _256N / _256N_BLOCK
 * (src/reduction/seg_wmma_16n.cu:137-221, seg_wmma_256n.cu:149-229).
 * segment_size: any size >= 1.  Powers of two >= 16 (the sizes of the
 * reference's dispatch table, seg_wmma_16n.cu:146-172, and of all its
 * benchmarks) run the tiled kernels at HBM speed; the other multiples of 16
 * the reference accepts run kernels that give a warp 16 segments (reduction,
 * also for multiples of 8 and for any size up to 255) or 16 rows of 16
 * elements (scan) at a time, up to 2048 elements; every other size (tails
 * masked) runs a one-warp-per-segment kernel (TCU_ALGO_AUTO or TCU_ALGO_MMA
 * only).
 * d_out: num_segments floats or halves.
 * A workspace is needed only when segment_size > 16384.
 */
int tcu_segmented_reduce_f16(const void* d_in, void* d_out, int out_type, size_t num_segments,
                             size_t segment_size, int algo, void* d_workspace,
                             size_t workspace_bytes, void* stream);

/*
 * Segmented inclusive prefix sum: out[j*S + i] = in[j*S] + ... + in[j*S + i].
 * Replaces compute_wmma_segmented_prefixsum_16n (src/prefixsum/kernel.cuh:86-150),
 * ..._256n (:441-506), ..._256n_block (:586-678) and their drivers
 * CUDA_WMMA_SEGMENTED_PREFIXSUM_16N / _256N (src/prefixsum/seg_wmma_16n.cu:139-223,
 * seg_wmma_256n.cu:143-222).  d_out: num_segments*segment_size halves or floats.
 * A workspace is needed only when segment_size > 16384.
 */
int tcu_segmented_scan_f16(const void* d_in, void* d_out, int out_type, size_t num_segments,
                           size_t segment_size, int algo, void* d_workspace,
                           size_t workspace_bytes, void* stream);

/*
 * Sum of all num_elements inputs (a multiple of 16) into *d_out (float) and,
 * if d_out_f64 is not null, into *d_out_f64 (double; what a multi-GPU caller
 * gathers).  Replaces CUDA_WMMA_FULL_REDUCTION_2KERS[_BLOCK]_BASE_{16,256}
 * (src/reduction/wmma_2kers.cu:17-193): segmented kernel + cub::DeviceReduce.
 * Always needs a workspace.
 */
int tcu_full_reduce_f16(const void* d_in, float* d_out, double* d_out_f64, size_t num_elements,
                        int algo, void* d_workspace, size_t workspace_bytes, void* stream);

/*
 * Inclusive prefix sum over all num_elements inputs (a multiple of 16).
 * Replaces CUDA_WMMA_FULL_PREFIXSUM_3KERS[_BLOCK] (src/prefixsum/wmma_3kers.cu:14-177):
 * ..._256n_ps + cub::DeviceScan::ExclusiveSum + add_partial_sums, here one pass.
 * For a scan sharded over several GPUs, d_shard_totals points at the gathered
 * per-shard totals (device memory, doubles) and shard_index is this GPU's
 * position: the sum of the earlier shards' totals seeds the scan.  Pass NULL
 * and 0 on one GPU.  Always needs a workspace.
 */
int tcu_full_scan_f16(const void* d_in, void* d_out, int out_type, size_t num_elements,
                      const double* d_shard_totals, int shard_index, int algo,
                      void* d_workspace, size_t workspace_bytes, void* stream);

/*
 * Exclusive variants: out[i] = sum of the elements of the segment BEFORE i (0 for
 * the first).  The reference has inclusive scans only (U has ones on its
 * diagonal, src/prefixsum/kernel.cuh:60); callers that turn counts into offsets
 * need this form, and on the tensor core it is the same product with the
 * diagonal of U removed.  Arguments as for the inclusive entry points; always
 * the tensor-core algorithm.
 */
int tcu_segmented_exclusive_scan_f16(const void* d_in, void* d_out, int out_type,
                                     size_t num_segments, size_t segment_size, void* d_workspace,
                                     size_t workspace_bytes, void* stream);
int tcu_full_exclusive_scan_f16(const void* d_in, void* d_out, int out_type, size_t num_elements,
                                void* d_workspace, size_t workspace_bytes, void* stream);

/*
 * bfloat16 inputs.  Same operations, arguments, status codes, workspace sizes
 * and segment sizes as the *_f16 entry points of the same name; d_in holds
 * bfloat16 values and out_type TCU_OUT_F16 means "16-bit outputs in the type
 * of the input", i.e. bfloat16.  No counterpart in the reference, which is
 * fp16 only (half everywhere in src/reduction/kernel.cuh and
 * src/prefixsum/kernel.cuh); the step next to it that mixed-precision callers
 * need first.  Same kernels, compiled a second time with the bf16 form of the
 * MMA, of the constant matrices and of the exact hi/lo split.  algo:
 * TCU_ALGO_AUTO / _MMA / _SHUFFLE / _TCGEN05 as for fp16.
 */
int tcu_segmented_reduce_bf16(const void* d_in, void* d_out, int out_type, size_t num_segments,
                              size_t segment_size, int algo, void* d_workspace,
                              size_t workspace_bytes, void* stream);
int tcu_segmented_scan_bf16(const void* d_in, void* d_out, int out_type, size_t num_segments,
                            size_t segment_size, int algo, void* d_workspace,
                            size_t workspace_bytes, void* stream);
int tcu_segmented_exclusive_scan_bf16(const void* d_in, void* d_out, int out_type,
                                      size_t num_segments, size_t segment_size, void* d_workspace,
                                      size_t workspace_bytes, void* stream);
int tcu_full_exclusive_scan_bf16(const void* d_in, void* d_out, int out_type, size_t num_elements,
                                 void* d_workspace, size_t workspace_bytes, void* stream);
int tcu_full_reduce_bf16(const void* d_in, float* d_out, double* d_out_f64, size_t num_elements,
                         int algo, void* d_workspace, size_t workspace_bytes, void* stream);
int tcu_full_scan_bf16(const void* d_in, void* d_out, int out_type, size_t num_elements,
                       const double* d_shard_totals, int shard_index, int algo,
                       void* d_workspace, size_t workspace_bytes, void* stream);
/* tcu_fill_f16 rounding the same values to bfloat16 instead. */
int tcu_fill_bf16(void* d_out, size_t n, uint64_t seed, uint64_t first_index, int dist,
                  void* stream);

/*
 * tcu_full_scan_f16 for callers that must not allocate device memory.  It has
 * no counterpart in the reference, whose drivers cudaMalloc whatever they need.
 *
 * Who needs it: code that runs where cudaMalloc / cudaFree are off limits or
 * too expensive -- a plugin that was handed its input and output buffers and
 * nothing else by a host framework that owns all device memory, a service
 * loop with a latency budget (cudaMalloc and cudaFree synchronise the whole
 * device), or a step that sits between other asynchronous work and must not
 * stall it.  Such a caller cannot produce the workspace tcu_full_scan_f16 asks
 * for, so this variant brings its own: a fixed array in the library's device
 * image, TCU_STATIC_SCAN_SCRATCH_BYTES (about 0.8 MiB) on every GPU the
 * library is loaded on, held until the process exits.
 *
 * Same arguments and results as tcu_full_scan_f16 minus the workspace.  Limits
 * and rules that come with the shared array:
 *   - num_elements <= TCU_STATIC_SCAN_MAX_ELEMENTS (2^30), else TCU_ERR_TOO_LARGE
 *     and nothing is launched;
 *   - the first call on each device looks up the array's device address (with
 *     that device current); make that first call outside any stream capture;
 *   - every call uses the same array and clears the part it needs on `stream`
 *     before its kernel, so calls in one stream are fine back to back, but two
 *     calls that can run at the same time on one GPU (different streams,
 *     different host threads) race on it: serialise them, or give the second
 *     one a workspace and use tcu_full_scan_f16;
 *   - no cudaMalloc, cudaFree or allocating library routine is called.
 */
#define TCU_STATIC_SCAN_MAX_ELEMENTS ((size_t)1 << 30)
#define TCU_STATIC_SCAN_MAX_TILES (TCU_STATIC_SCAN_MAX_ELEMENTS / 16384)
#define TCU_STATIC_SCAN_SCRATCH_BYTES \
  (256 + TCU_STATIC_SCAN_MAX_TILES * 8 + (TCU_STATIC_SCAN_MAX_TILES / 32 + TCU_STATIC_SCAN_MAX_TILES / 2 + 2) * 8)
int tcu_full_scan_f16_static(const void* d_in, void* d_out, int out_type, size_t num_elements,
                             const double* d_shard_totals, int shard_index, int algo,
                             void* stream);

/* Bytes of device workspace the operation needs (0 = none).  The workspace
 * needs no initialisation; one workspace must not be shared by calls that can
 * run at the same time. */
size_t tcu_workspace_bytes(int op, size_t num_elements, size_t segment_size);

/*
 * Seeded input fill, element i = f(seed, first_index + i): the build's
 * replacement for cuda_memory_set / setFP16 (src/utils/cuda_helpers.cuh:123-181).
 * Shards of one logical array are filled independently by passing their
 * first global index.  n must be a multiple of 8.
 */
int tcu_fill_f16(void* d_out, size_t n, uint64_t seed, uint64_t first_index, int dist,
                 void* stream);

/*
 * Same operations with HOST buffers: input is copied to the device in chunks
 * of whole segments that overlap with the kernels, results are copied back.
 * h_in / h_out should be pinned for full copy bandwidth.  The context owns
 * its staging buffers and streams (created once; this is the only place the
 * library allocates).  op selects the operation; for the full operations
 * segment_size is ignored.  The call returns when h_out is complete.
 */
typedef struct tcu_host_ctx tcu_host_ctx;
int tcu_host_ctx_create(tcu_host_ctx** ctx, size_t chunk_elements);
void tcu_host_ctx_destroy(tcu_host_ctx* ctx);
int tcu_host_run_f16(tcu_host_ctx* ctx, int op, const void* h_in, void* h_out, int out_type,
                     size_t num_elements, size_t segment_size, int algo);

/*
 * The reference's segment-size sweep (one array, many segment sizes:
 * SEG_16_ARGS ... SEG_16384_ARGS over the same element counts,
 * src/reduction/args.hpp:64-75) for an array in HOST memory: every chunk is
 * copied to the device once and reduced at all num_sizes segment sizes while
 * the next chunk is on its way; h_outs[i] receives num_elements /
 * segment_sizes[i] sums.  Saves num_sizes - 1 of num_sizes host-to-device
 * passes compared with num_sizes calls of tcu_host_run_f16.
 */
int tcu_host_segmented_reduce_sweep_f16(tcu_host_ctx* ctx, const void* h_in, size_t num_elements,
                                        int num_sizes, const size_t* segment_sizes,
                                        void* const* h_outs, int out_type, int algo);

/*
 * Full reduction and full scan of ONE array sharded contiguously over the GPUs
 * of a node: rank r holds elements [begin_r, end_r) in its own device memory
 * and keeps its part of the output.  The reference is single-device
 * (src/init/cuda.cpp:45 selects one GPU and nothing in src/ talks to another),
 * so these entry points have no counterpart there; they are what its full
 * operations (src/reduction/wmma_2kers.cu:65-81, src/prefixsum/wmma_3kers.cu:63-70)
 * become when the array does not live on one GPU.
 *
 * One context per GPU.  The GPUs exchange one double each per call -- the
 * shard totals -- which the reduction kernel's last thread block stores
 * straight into a small slot array in every rank's memory; the scan kernel of
 * rank r waits (bounded) for the totals of ranks < r in its own memory.  No
 * library collective runs per call.  Set-up:
 *   - one process per GPU: every rank calls tcu_mgpu_ctx_create, which fills
 *     handle_out (TCU_MGPU_HANDLE_BYTES bytes, a CUDA IPC handle of its slot
 *     array); the ranks exchange the handles by any means they have (one
 *     all-gather at start-up) and pass all of them, in rank order, to
 *     tcu_mgpu_ctx_connect;
 *   - one process driving several devices: create one context per device (with
 *     that device current; handle_out may be NULL) and call
 *     tcu_mgpu_ctx_connect_local on each with the array of all contexts.
 * Rules: every rank makes the same sequence of tcu_mgpu_full_* calls, each on
 * one stream of its own GPU, and the calls of one context do not overlap;
 * a rank whose peers never make the matching call gives up after about two
 * seconds and reports TCU_ERR_TIMEOUT through tcu_device_error (bit 2).
 * Destroy a context only after EVERY rank has finished its last call
 * (synchronise, then meet at a host barrier): peers store into its memory.
 *
 * tcu_mgpu_full_reduce_f16: *d_out (and *d_out_f64 if not NULL) receive the
 * sum over all ranks' shards, on every rank.
 * tcu_mgpu_full_scan_f16: d_out[i] = (sum of all earlier ranks' shards) +
 * in[0] + ... + in[i]; two passes over the shard (reduce, then scan).
 * num_elements: this rank's shard, a multiple of 16, may be 0.
 * tcu_mgpu_ctx_set_l2_keep_bytes: how much of the shard the first pass asks
 * L2 to keep for the second (default 64 MiB; 0 = nothing).
 */
#define TCU_MGPU_HANDLE_BYTES 64
#define TCU_MGPU_MAX_RANKS 16
typedef struct tcu_mgpu_ctx tcu_mgpu_ctx;
int tcu_mgpu_ctx_create(tcu_mgpu_ctx** ctx, int rank, int world, void* handle_out);
int tcu_mgpu_ctx_connect(tcu_mgpu_ctx* ctx, const void* handles);
int tcu_mgpu_ctx_connect_local(tcu_mgpu_ctx* ctx, tcu_mgpu_ctx* const* group);
int tcu_mgpu_ctx_set_l2_keep_bytes(tcu_mgpu_ctx* ctx, size_t bytes);
void tcu_mgpu_ctx_destroy(tcu_mgpu_ctx* ctx);
int tcu_mgpu_full_reduce_f16(tcu_mgpu_ctx* ctx, const void* d_in, float* d_out, double* d_out_f64,
                             size_t num_elements, void* stream);
int tcu_mgpu_full_scan_f16(tcu_mgpu_ctx* ctx, const void* d_in, void* d_out, int out_type,
                           size_t num_elements, void* stream);

/*
 * Language-model operators: the scan and the segmented reductions above, with
 * weights.  A gated linear recurrence is a segmented scan whose running sum
 * decays; a norm is a segmented sum of squares and its use; the log
 * probability of a token is a segmented sum of exponentials and its use.
 * They have no counterpart in the reference.
 *
 * Conventions they share, next to those at the top of this file:
 *   - arguments come in a struct of 8-byte fields; a field left 0 means "not
 *     given" where it says so;
 *   - element types are tcu_type codes; everything is computed in 32 bits and
 *     rounded to the type of the output once;
 *   - inputs have a stride in elements between rows (any, 0 and negative
 *     included), the elements of a row lie side by side; outputs are
 *     contiguous;
 *   - pointers are aligned to their element's size; 16-byte aligned rows are
 *     faster;
 *   - results do not depend on timing: the same call gives the same bits;
 *   - an index in device memory that is out of range raises bit 3 of
 *     tcu_device_error, and what it names is left out.
 */
typedef enum { TCU_TYPE_F16 = 0, TCU_TYPE_F32 = 1, TCU_TYPE_BF16 = 2 } tcu_type;

/*
 * Gated linear recurrence along time, for every channel by itself:
 *     h_t = f_t * h_{t-1} + u_t,    h_{-1} = h0 (0 if not given)
 *   TCU_GATE_DECAY:    f = a,            u = x
 *   TCU_GATE_LOG:      f = exp(a),       u = x
 *   TCU_GATE_SIGMOID:  f = 1/(1+exp(-a)) u = (1 - f) * x
 * Gates are meant to have |f| <= 1: the product of up to 1024 of them in a
 * row must stay within float32.
 *
 * x, a: `batch` sequences of `tokens` rows of `dim` (up to 2^21) elements; h: contiguous.
 * With `offsets` (batch + 1 values, not decreasing, 32- or 64-bit) the
 * sequences lie one behind the other instead, sequence b being the rows
 * offsets[b] ... offsets[b+1]-1 of `tokens` rows in all (batch strides
 * are not used); rows before the first and behind the last sequence are left as
 * they were, or become 0 where clear_rest is not 0, and a sequence whose offsets are out of range or decrease counts as
 * empty.  Of sequences that then share rows or lie in another order than their
 * numbers at most one is not empty, always the same.  a_type: the type of x, or TCU_TYPE_F32.
 * h0, last: batch x dim floats; last (may be h0) receives the state behind
 * each sequence's last row, h0's if the sequence is empty.
 * states: NULL, or tcu_linear_scan_states_rows() x dim floats that
 * tcu_linear_scan_backward() wants (the state before every 16th row).
 */
typedef enum { TCU_GATE_DECAY = 0, TCU_GATE_LOG = 1, TCU_GATE_SIGMOID = 2 } tcu_gate;

typedef struct {
  const void* a;
  const void* x;
  void* h;
  const float* h0;     /* may be NULL */
  float* last;         /* may be NULL */
  float* states;       /* may be NULL */
  const void* offsets; /* may be NULL */
  int64_t batch, tokens, dim;
  int64_t a_batch_stride, a_row_stride, x_batch_stride, x_row_stride;
  int64_t gate, a_type, type, offsets_are_64bit, clear_rest;
} tcu_linear_scan_args;
int tcu_linear_scan(const tcu_linear_scan_args* args, void* stream);

size_t tcu_linear_scan_states_rows(size_t batch, size_t tokens, int packed);

/*
 * Its gradient: from dh (of h; may be NULL: zeros), dlast (of last, batch x dim floats; may be
 * NULL) and the states of the forward call, da and dx (contiguous, in the
 * types of a and x) and dh0 (batch x dim floats; may be NULL).  a, x, gate and
 * offsets as in the forward call.
 */
typedef struct {
  const void* dh;
  const void* a;
  const void* x;
  const float* states;
  const float* dlast; /* may be NULL */
  void* da;
  void* dx;
  float* dh0;          /* may be NULL */
  const void* offsets; /* may be NULL */
  int64_t batch, tokens, dim;
  int64_t dh_batch_stride, dh_row_stride, a_batch_stride, a_row_stride, x_batch_stride, x_row_stride;
  int64_t gate, a_type, type, offsets_are_64bit, clear_rest;
} tcu_linear_scan_backward_args;
int tcu_linear_scan_backward(const tcu_linear_scan_backward_args* args, void* stream);

/*
 * One token for each of `batch` sequences: row b of a and x advances the state
 * state[slots[b]] (state: `pool` x dim floats, contiguous, updated in place;
 * slots NULL: state b) and writes it to row b of h.  A negative slot marks a
 * padded row: its row of h is left as it was (becomes 0 where clear_rest is not
 * 0), and so it is, with bit 3 of tcu_device_error, for a slot >= pool and for
 * one that an earlier row names.
 */
typedef struct {
  const void* a;
  const void* x;
  void* h;
  float* state;
  const void* slots; /* may be NULL */
  int64_t batch, pool, dim;
  int64_t a_row_stride, x_row_stride;
  int64_t gate, a_type, type, slots_are_64bit, clear_rest;
} tcu_linear_scan_step_args;
int tcu_linear_scan_step(const tcu_linear_scan_step_args* args, void* stream);

/*
 * The norms around a block of a model, fused with its gate and its residual
 * connection, for `rows` rows of `dim` elements (up to 16384):
 *     n = z / rms(z) * post_weight                  (z itself without post_weight)
 *     out = residual + scale * act(gate) * n        (residual 0, act(gate) 1 if not given)
 *     normed = out / rms(out) * pre_weight          (only with pre_weight)
 * with rms(y) = sqrt(mean(y^2) + eps), and out not rounded before it is normed.
 * (Sums of squares of a row must stay within float32.)
 * gate: gate_rows rows, each for rows / gate_rows consecutive rows (1: one
 * learned vector; rows: a gate for every element); gate_rows divides rows.
 * type: of z, residual, gate, out and normed; weight_type: that type or
 * TCU_TYPE_F32.  out may be z's or residual's buffer, normed z's, if that is
 * contiguous.
 */
typedef enum { TCU_ACT_NONE = 0, TCU_ACT_SIGMOID = 1, TCU_ACT_SILU = 2 } tcu_act;

typedef struct {
  const void* z;
  const void* residual;    /* may be NULL */
  const void* post_weight; /* may be NULL */
  const void* gate;        /* may be NULL */
  const void* pre_weight;  /* may be NULL */
  void* out;
  void* normed;            /* only with pre_weight */
  int64_t rows, dim, gate_rows;
  int64_t z_row_stride, residual_row_stride, gate_row_stride;
  int64_t act, type, weight_type;
  double scale, eps;
} tcu_norm_residual_args;
int tcu_norm_residual(const tcu_norm_residual_args* args, void* stream);

/*
 * Its gradient: from dout and dnormed (NULL: zeros) dz, and whichever of the
 * others are not NULL, each in the type of what it is the gradient of.  The
 * sums over rows are made in a fixed order.  dresidual may be dout's buffer,
 * dz may be z's, dout's (if that is not dresidual too) or dnormed's, if that is
 * contiguous.  The workspace is 16-byte aligned, of
 * tcu_norm_residual_workspace_bytes(), needs no initialisation, and must not be
 * shared by calls that can run at the same time.
 */
typedef struct {
  const void* dout;        /* may be NULL */
  const void* dnormed;     /* may be NULL */
  const void* z;
  const void* residual;    /* may be NULL */
  const void* post_weight; /* may be NULL */
  const void* gate;        /* may be NULL */
  const void* pre_weight;  /* may be NULL */
  void* dz;
  void* dresidual;         /* may be NULL */
  void* dpost_weight;      /* may be NULL */
  void* dgate;             /* may be NULL; gate_rows x dim */
  void* dpre_weight;       /* may be NULL */
  void* workspace;
  int64_t workspace_bytes;
  int64_t rows, dim, gate_rows;
  int64_t dout_row_stride, dnormed_row_stride, z_row_stride, residual_row_stride, gate_row_stride;
  int64_t act, type, weight_type;
  double scale, eps;
} tcu_norm_residual_backward_args;
int tcu_norm_residual_backward(const tcu_norm_residual_backward_args* args, void* stream);

size_t tcu_norm_residual_workspace_bytes(size_t rows, size_t dim, size_t gate_rows);

/*
 * Log probabilities of given tokens, for `rows` rows of `vocab` (up to 2^30) logits:
 *     lse = log sum_j exp(x_j),  logprob = x_target - lse,
 *     entropy = - sum_j p_j log p_j,  p_j = exp(x_j - lse),
 * and the `top` (0 ... TCU_MAX_TOP, at most vocab) most probable tokens: their log
 * probabilities, falling, and indices (ties: the lowest index first; NaN counts as the largest).  Logits of -inf
 * are tokens left out; a row of nothing else has lse and log probabilities
 * -inf and entropy 0.  A row with NaN or +inf gives NaN.
 * targets: 32- or 64-bit; a row whose target is ignore_index has logprob 0,
 * and so, with bit 3 of tcu_device_error, has one whose target is out of range.
 */
#define TCU_MAX_TOP 32
typedef struct {
  const void* logits;
  const void* targets; /* may be NULL if logprob is */
  float* logprob;      /* rows; may be NULL */
  float* entropy;      /* rows; may be NULL */
  float* lse;          /* rows; may be NULL */
  float* top_logprob;  /* rows x top */
  int64_t* top_index;  /* rows x top */
  int64_t rows, vocab, row_stride, top, ignore_index;
  int64_t type, targets_are_64bit;
} tcu_token_logprobs_args;
int tcu_token_logprobs(const tcu_token_logprobs_args* args, void* stream);

/*
 * Its gradient: from dlogprob and dentropy (rows floats each; NULL: zeros) and
 * the lse and entropy of the forward call, dlogits (contiguous, the type of the
 * logits; may be their buffer if that is contiguous).  Rows whose target counts
 * for nothing have no part of dlogprob; a row of -inf has gradient 0.
 * Probabilities go by lse, whose rounding to 32 bits is their relative error;
 * above |lse| of 32 (TCU_TYPE_F32) or 256 the row is summed once more instead.
 */
typedef struct {
  const void* logits;
  const void* targets;   /* may be NULL if dlogprob is */
  const float* lse;
  const float* entropy;  /* may be NULL if dentropy is */
  const float* dlogprob; /* may be NULL */
  const float* dentropy; /* may be NULL */
  void* dlogits;
  int64_t rows, vocab, row_stride, ignore_index;
  int64_t type, targets_are_64bit;
} tcu_token_logprobs_backward_args;
int tcu_token_logprobs_backward(const tcu_token_logprobs_backward_args* args, void* stream);

/* Reads (and optionally clears) the device-side error word of the current
 * device: bit 0 = an mbarrier wait ran out, bit 1 = a tile-status poll ran
 * out, bit 2 = a wait for another GPU's total ran out, bit 3 = an index in
 * device memory was wrong.  Synchronises the device.  Returns
 * TCU_ERR_TIMEOUT if any of the bits 0 to 2 is set, TCU_ERR_INDEX if bit 3
 * alone is. */
int tcu_device_error(unsigned int* bits, int clear);

/*
 * Test hooks for the bounded waits (the reference has none: its one
 * device-side spin barrier is disabled as a dead lock,
 * src/prefixsum/wmma_atomic.cu:189).  Every device-side wait of the library
 * gives up after a limit and raises a bit of the error word instead of
 * hanging; these two calls let a test see that happen within a millisecond.
 * tcu_test_set_wait_limits: attempts before an mbarrier wait, a tile-status
 * poll, a shared-memory flag poll and a peer-total poll give up, on the
 * current device; 0 restores that limit's default.
 * tcu_test_inject: arms ONE stall for the next matching call on this host
 * thread's library state -- TCU_TEST_SKIP_TILE_LOAD: the next segmented or
 * full reduction never loads tile `arg` of CTA 0's tiles (its consumers'
 * barrier is never armed); TCU_TEST_LOOKBACK_TICKET: the next look-back scan
 * hands out tiles starting at `arg` instead of 0 (tile `arg` polls status
 * words nobody publishes).  Nothing faults or traps: the waits run out, the
 * kernels return, the outputs of that call are wrong and flagged.
 */
typedef enum { TCU_TEST_NONE = 0, TCU_TEST_SKIP_TILE_LOAD = 1, TCU_TEST_LOOKBACK_TICKET = 2 } tcu_test_stall;
int tcu_test_set_wait_limits(unsigned barrier_attempts, unsigned status_polls, unsigned flag_polls,
                             unsigned peer_polls);
int tcu_test_inject(int what, unsigned long long arg);

/* Geometry the kernels were built with, for callers that size experiments. */
int tcu_tile_elements(void);
int tcu_num_sms(void);

const char* tcu_status_string(int status);

#ifdef __cplusplus
}
#endif
#endif /* TCU_SCOPE_H_ */
