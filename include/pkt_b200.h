/*
 * pkt_b200 — C-ABI of the B200-native (sm_100a) persistent training megakernel.
 *
 * This is the drop-in boundary for Marco-Christiani/pkt's hot path. Plain C
 * types only (pointers, sizes, ints); device pointers are passed as void* /
 * float*, CUDA streams as void*. Every function returns an int status
 * (0 = ok, < 0 = error; pkt_last_error() gives the message) where pkt's own
 * host API returned nothing and checked no CUDA call (include/runtime.hpp:27-449).
 *
 * The C++ header include/pk/runtime.hpp wraps the runtime half of this ABI in
 * pkt's own class (pk::Runtime) so pkt programs compile unchanged against it.
 */
#ifndef PKT_B200_H
#define PKT_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define PKT_OK 0
#define PKT_ERR_ARGS -1        /* bad argument / out of capacity */
#define PKT_ERR_CUDA -2        /* a CUDA runtime / driver call failed */
#define PKT_ERR_TIMEOUT -3     /* a device wait ran out of time (see pkt_runtime_status) */
#define PKT_ERR_OPCODE -4      /* device met an opcode it does not implement */
#define PKT_ERR_NCCL -5        /* an NCCL call failed */
#define PKT_ERR_UNSUPPORTED -6 /* shape / dtype / layout the kernel cannot run */

/* Device-side status word codes (pkt_runtime_status / pkt_mlp_status). */
#define PKT_DEV_OK 0
#define PKT_DEV_TIMEOUT_DEPS 1    /* controller waited too long for a dependency token */
#define PKT_DEV_TIMEOUT_PIPE 2    /* an intra-CTA pipeline wait (mbarrier) ran out */
#define PKT_DEV_BAD_OPCODE 3      /* unknown opcode in the task list */
#define PKT_DEV_BAD_ARGS 4        /* task arguments failed a device-side bounds check */

/* ---- task descriptor (byte-identical to pkt's pk::Task, include/task.cuh:22-40) */
typedef struct pkt_task_header {
  uint16_t opcode;          /* offset 0 */
  uint16_t arg_bytes;       /* offset 2 */
  uint32_t user_tag;        /* offset 4: overwritten with the task index on device */
  uint16_t buffer_read_id;  /* offset 8: dependency token waited on (0 = none) */
  uint16_t buffer_write_id; /* offset 10: token marked when the task completes (0 = none) */
  uint32_t wait_count;      /* offset 12: token count needed */
  uint32_t read_epoch;      /* offset 16: token epoch needed */
  uint32_t write_epoch;     /* offset 20: epoch published (atomic max) */
  /* offset 24: reserved[0] in pkt. Extension (0 keeps pkt semantics):
   *   bits 0-15  second token waited on, bits 16-31 second token marked. */
  uint32_t ext_ids;
  uint32_t ext_wait_count; /* offset 28: reserved[1] in pkt; count needed on the second token */
} pkt_task_header;

typedef struct pkt_task {
  pkt_task_header header;
  uint8_t args[64];
} __attribute__((aligned(16))) pkt_task;

/* Opcodes. 0-3 and 10-13 are pkt's (include/task.cuh:11-20); the rest are new. */
enum pkt_opcode {
  PKT_OP_INVALID = 0,
  PKT_OP_ZERO_MEMORY = 1,     /* pkt ZeroMemoryArgs */
  PKT_OP_AXPY = 2,            /* pkt AxpyArgs */
  PKT_OP_GEMM = 3,            /* pkt's reserved Gemm: one tcgen05 tile, pkt_gemm_tile_args */
  PKT_OP_LINEAR_FORWARD = 10, /* pkt LinearForwardArgs (fp32 SIMT tile, any shape) */
  PKT_OP_MSE_LOSS = 11,       /* pkt MSELossArgs */
  PKT_OP_LINEAR_BACKWARD = 12,/* pkt LinearBackwardArgs */
  PKT_OP_SGD_UPDATE = 13,     /* pkt SGDUpdateArgs */
  PKT_OP_BIAS_SGD = 20,       /* pkt_bias_sgd_args: reduce column partials, update bias */
  PKT_OP_LOSS_REDUCE = 21,    /* pkt_loss_reduce_args: deterministic sum of tile partials */
  PKT_OP_SGD_MIXED = 22,      /* pkt_sgd_mixed_args: fp32 master -= lr*g, bf16 shadow write */
  /* Fused data parallel (MLP grad_mode 2; peer memory between the ranks' GPUs): */
  PKT_OP_DP_WAIT = 30,        /* pkt_dp_wait_args: the next step's weights of a layer have arrived */
  PKT_OP_DP_BIAS_SEND = 31,   /* pkt_dp_bias_args: this rank's bias gradient to every rank */
  PKT_OP_DP_BIAS_APPLY = 32,  /* pkt_dp_bias_args: sum the ranks' bias gradients, SGD */
  PKT_OP_DP_REDUCE = 33       /* pkt_gemm_tile_args: an owned weight tile: sum the ranks' partials,
                                 SGD on the fp32 master, new bf16 tile to every rank */
};

/* Args of PKT_OP_GEMM: tile (tile_m, tile_n) of registered GEMM `gemm`. */
typedef struct pkt_gemm_tile_args {
  uint32_t gemm;
  uint32_t tile_m;
  uint32_t tile_n;
  uint32_t pad;
} pkt_gemm_tile_args;

typedef struct pkt_bias_sgd_args {
  const float* partials; /* [num_partials, ld] column partial sums */
  float* bias;           /* [n] updated in place (may be null: grads only) */
  float* grad_out;       /* [n] optional: the reduced gradient */
  int num_partials;
  int ld;
  int col_begin;
  int col_end;
  float lr;
  int pad;
} pkt_bias_sgd_args;

typedef struct pkt_loss_reduce_args {
  const float* partials;
  float* loss;     /* loss[0] = sum(partials) * scale, or loss[(*step)++] when step != null */
  int count;
  float scale;
  int* step;       /* optional device step counter */
} pkt_loss_reduce_args;

typedef struct pkt_sgd_mixed_args {
  const float* w;       /* fp32 master read */
  const float* g;       /* gradient */
  float* w_out;         /* fp32 master written (may equal w) */
  uint16_t* w_bf16;     /* optional bf16 copy written from the new master (may be null) */
  long long n;
  float lr;
  int pad;
} pkt_sgd_mixed_args;

/* Args of the fused data-parallel tasks. Offsets are bytes into a rank's
 * exchange region (identical layout on every rank); the region bases of all
 * ranks reach the kernel through the launch, not through the task. */
typedef struct pkt_dp_wait_args {
  int layer;
  int tiles;           /* weight tiles of the layer (each published once per CTA of a pair) */
} pkt_dp_wait_args;

typedef struct pkt_dp_bias_args {
  const float* partials; /* SEND: [num_partials, ld] column partial sums */
  float* bias;           /* APPLY: [n] updated in place */
  int num_partials;
  int ld;
  int n;
  int layer;
  int bias_off;          /* float offset of the layer in a rank's bias gradient vector */
  float lr;              /* APPLY: learning rate x gradient scale */
} pkt_dp_bias_args;

/* ---- dtypes and GEMM registration -------------------------------------- */
#define PKT_DTYPE_BF16 1
#define PKT_DTYPE_TF32 2 /* fp32 storage, TF32 tensor-core inputs */
#define PKT_DTYPE_F32 3  /* fp32 output storage */
#define PKT_DTYPE_E4M3 4 /* 8-bit float: 4 exponent bits, largest value 448, no infinity */
#define PKT_DTYPE_E5M2 5 /* 8-bit float: 5 exponent bits, largest finite value 57344 */

#define PKT_MAJOR_K 0  /* operand stored [rows][K] (K contiguous) */
#define PKT_MAJOR_MN 1 /* operand stored [K][rows] (rows contiguous) */

enum pkt_epilogue {
  PKT_EPI_STORE = 0,      /* out = acc */
  PKT_EPI_BIAS_ACT = 1,   /* out = act(acc + bias) */
  PKT_EPI_MSE = 2,        /* y = acc + bias; out = dY = scale*(y - target); loss partials */
  PKT_EPI_DGRAD_RELU = 3, /* out = acc * (aux > 0) */
  PKT_EPI_WGRAD_SGD = 4,  /* w_out = w_in - lr*acc (fp32), w_bf16 = bf16(w_out) */
  PKT_EPI_WGRAD_STORE = 5, /* out = acc (fp32 gradient) */
  PKT_EPI_WGRAD_PEER = 6   /* fused data parallel (MLP grad_mode 2 only): a rank that
                              does not own the tile sends its fp32 partial to the
                              owner's exchange region; the owner sums the ranks'
                              partials, applies SGD (w_in/w_out, lr) and writes the
                              bf16 copy (w_shadow) on every rank */
};

/* One D[M,N] = sum_k A[m,k] B[n,k] problem, tiled 128 x bn. */
typedef struct pkt_gemm_desc {
  int M, N, K;
  int bn;            /* tile N: 16..256, multiple of 16 */
  int in_dtype;      /* PKT_DTYPE_BF16 or PKT_DTYPE_TF32 */
  const void* a;     /* device pointer */
  int lda;           /* elements between consecutive stored rows */
  int a_major;       /* PKT_MAJOR_K: a[m*lda+k]; PKT_MAJOR_MN: a[k*lda+m] */
  const void* b;
  int ldb;
  int b_major;
  int epilogue;      /* pkt_epilogue */
  void* out;         /* D / dY / dH / dW output */
  int ldo;           /* columns N.. of a row are not written (ldw too) */
  int out_dtype;     /* PKT_DTYPE_BF16 or PKT_DTYPE_F32 */
  int relu;          /* PKT_EPI_BIAS_ACT: apply ReLU */
  const float* bias; /* [N] or null */
  const void* aux;   /* MSE: target [M,ldaux] (in_dtype storage); DGRAD: relu source H [M,ldaux] */
  int ldaux;
  float scale;       /* MSE: 2/(B*N) */
  float* loss_partials; /* MSE: [tiles_m*tiles_n] sum of squared error per tile */
  float* colsum;     /* MSE / DGRAD: [tiles_m, ldcol] per-row-block column sums of stored out */
  int ldcol;
  const float* w_in; /* WGRAD_SGD: fp32 master read (may equal w_out) [M, ldw] */
  float* w_out;      /* WGRAD_SGD: fp32 master written */
  void* w_shadow;    /* WGRAD_SGD: bf16 copy written (may be null) */
  int ldw;
  float lr;
  void* y_out;       /* MSE: optional fp32 copy of y = acc + bias */
  int ldy;
  int cta_pair;      /* 0/1: one CTA per 128 x bn tile; 2: a CTA pair per 256 x bn tile
                        (tcgen05 cta_group::2, each CTA loads its A rows and half of B);
                        must match the launch mode (pkt_runtime_set_cta_pair) */
} pkt_gemm_desc;

/* ---- runtime (pk::Runtime's C half) ------------------------------------ */
typedef struct pkt_runtime pkt_runtime;

int pkt_runtime_create(int device, pkt_runtime** out);
int pkt_runtime_destroy(pkt_runtime* rt);
/* Allocates room for max_tasks tasks (runtime.hpp:27-90). */
int pkt_runtime_initialize(pkt_runtime* rt, int max_tasks);
/* Copies the task list to the device and resets cursor, tokens and status (runtime.hpp:92-157). */
int pkt_runtime_submit(pkt_runtime* rt, const pkt_task* tasks, int n);
/* Stream-ordered variant: tasks from pinned host memory, no host sync. */
int pkt_runtime_submit_async(pkt_runtime* rt, const pkt_task* tasks, int n, void* stream);
/* Segments are accepted and kept as scheduling hints (runtime.hpp:159-173). */
int pkt_runtime_set_segments(pkt_runtime* rt, const int* begin_end_pairs, int n);
int pkt_runtime_set_segment_window_size(pkt_runtime* rt, int window);
/* One persistent launch over the submitted list (runtime.hpp:175-228). num_blocks <= 0: one CTA per SM. */
int pkt_runtime_launch(pkt_runtime* rt, int num_blocks, void* stream);
int pkt_runtime_synchronize(pkt_runtime* rt);
/* Device status word of the last launch: code (PKT_DEV_*), task index, token. */
int pkt_runtime_status(pkt_runtime* rt, int* code, int* task_index, int* detail);
/* Registers GEMM descriptors (builds their TMA tensor maps); returns the first id in *first_id. */
int pkt_runtime_register_gemms(pkt_runtime* rt, const pkt_gemm_desc* descs, int n, int* first_id);
int pkt_runtime_clear_gemms(pkt_runtime* rt);
/* Number of tiles of a registered GEMM (tiles_m * tiles_n). */
int pkt_gemm_tiles(const pkt_gemm_desc* d, int* tiles_m, int* tiles_n);
/* Wait budget of every device-side spin, in nanoseconds (default 2e9). */
int pkt_runtime_set_timeout_ns(pkt_runtime* rt, unsigned long long ns);
/* Launch mode: 1 = one CTA per SM works alone (default); 2 = CTA pairs (clusters of
 * two SMs) share 256-row GEMM tiles. pkt_runtime_launch clamps the grid to the CTAs
 * that can be resident at once and, in pair mode, rounds it to whole clusters. */
int pkt_runtime_set_cta_pair(pkt_runtime* rt, int pair);
int pkt_runtime_set_task_accounting(pkt_runtime* rt, int enabled);
int pkt_runtime_fetch_task_counter(pkt_runtime* rt, unsigned long long* out);
int pkt_runtime_set_perf(pkt_runtime* rt, int enabled);
/* Per-CTA role cycle counters of the last launch: blocks x PKT_PERF_WORDS u64. */
#define PKT_PERF_WORDS 16
int pkt_runtime_fetch_perf(pkt_runtime* rt, unsigned long long* out, int max_blocks, int* blocks);
int pkt_runtime_last_launch_blocks(pkt_runtime* rt);
/* For launching the megakernel instantiated with a program's own pk::OpTraits ops
 * (pk/kernel.cuh, pk::launch_with_ops; no counterpart in pkt, whose ops are
 * compiled into its one kernel): prepares the submitted list exactly as
 * pkt_runtime_launch does (grid clamped to the resident CTAs, counters cleared on
 * `stream`) and returns the kernel's parameter block (kparams_bytes must equal the
 * caller's sizeof(pkb::KParams)), the grid and the CTA-pair mode. */
int pkt_runtime_prepare_launch(pkt_runtime* rt, int num_blocks, void* stream, void* kparams, int kparams_bytes,
                               int* blocks, int* pair);
/* Effective SM clock of the launches since the last reset (no counterpart in pkt):
 * out3 = {SM cycles, nanoseconds, launches} summed over CTA 0's lifetime in every
 * launch; cycles * 1000 / ns is the mean SM clock in MHz. reset != 0 clears the
 * sums after reading them (out3 may be NULL to clear only). */
int pkt_runtime_clock_stats(pkt_runtime* rt, unsigned long long* out3, int reset);
/* Per-task trace of launches (no counterpart in pkt; its closest is the per-role
 * PerfBlock cycle counters): when enabled, every launch records for each task
 * PKT_TRACE_WORDS u64 = {CTA | opcode << 16 (GEMM tiles also: GEMM id << 32,
 * tile_m & 255 << 48, tile_n & 255 << 56), then %globaltimer ns at: dequeue, dependencies
 * satisfied, first TMA load issued, first MMA issued, last MMA committed, compute
 * warps started (GEMM: accumulator complete), compute warps finished}; stages a
 * task does not have stay 0. fetch copies the last launch's records (synchronous). */
#define PKT_TRACE_WORDS 8
int pkt_runtime_set_trace(pkt_runtime* rt, int enabled);
int pkt_runtime_fetch_trace(pkt_runtime* rt, unsigned long long* out, int max_tasks, int* n);
int pkt_num_sms(int device);
const char* pkt_last_error(void);

/* ---- axpy entry point (pkt examples/axpy_example.cu) --------------------- */
/* y = a*x + y over n floats on device memory, as one streaming task list. */
int pkt_axpy(const float* x, float* y, float a, long long n, void* stream);
/* Same result as pkt_axpy for callers that must not allocate device memory
 * (no counterpart in pkt: its runtime always cudaMallocs its task list). The
 * task list and status words live in a fixed ~192 KB array inside the library;
 * n is limited to 67,108,864 floats (larger n: PKT_ERR_ARGS, nothing launched).
 * Calls on one device share that array, so calls that overlap on the GPU race;
 * order them on one stream. The first call on a device looks up the array's
 * address and should come before any stream capture. */
int pkt_axpy_noalloc(const float* x, float* y, float a, long long n, void* stream);
/* Device status words of the last pkt_axpy_noalloc launch on the current device
 * (code PKT_DEV_*, task index, detail; all 0 when it ran cleanly), read from the
 * same fixed array without allocating. Synchronises the device first, so call it
 * after the work to check, not inside a stream capture. Every wait in that launch
 * has a fixed budget of 2 s; a launch that ran out of it reports
 * PKT_DEV_TIMEOUT_PIPE or PKT_DEV_TIMEOUT_DEPS here. The next pkt_axpy_noalloc
 * call clears the words. */
int pkt_axpy_noalloc_status(int* code, int* task_index, int* detail);

/* ---- stand-alone operators ---------------------------------------------- */
/* These run on the current device and in the order of `stream`; every pointer is
 * memory of that device (checked: a host pointer or another device's memory is
 * PKT_ERR_ARGS, and so is what the captured graph will allocate itself, by an
 * allocation node of the same capture: it is not memory yet). They allocate nothing and may be captured into a CUDA graph
 * (pkt_adamw_create and pkt_ops_status, which allocate or synchronise, may not).
 * A descriptor is read during the call only. Outputs must not overlap inputs
 * unless an operator says so. Only a result's own rows and columns are written. Of
 * an input, bytes beside a row may be read, within the 16-byte granules that hold
 * the row's first and last value; they never change a result. No counterpart in pkt. */

/* Every wait inside their kernels is bounded (about 2 s). code: PKT_DEV_TIMEOUT_PIPE
 * when one has run out on the current device since the last call (results since then
 * are not valid), else PKT_DEV_OK. Synchronises the device and clears the word. */
int pkt_ops_status(int* code);

/* Layer norm over the last dimension of [rows, cols]. Statistics and sums are
 * fp32; each result is rounded to its type once.
 *   forward   mean = sum x / C, rstd = 1/sqrt(sum (x-mean)^2 / C + eps),
 *             y = (x - mean) rstd gamma + beta
 *   backward  dx, and the sums over all rows dgamma = sum dy (x-mean) rstd,
 *             dbeta = sum dy, from x, dy and the forward pass's mean and rstd
 * Any cols >= 1 and row strides >= cols. Fastest where every row and gamma and beta
 * start on 16 bytes and a row is a multiple of 16 bytes; else the call goes value by
 * value. y may be x, dx may be dy or x, with the same row stride. The columns of a
 * padded row past cols do not count and are not written. rows = 0 is allowed (dgamma
 * and dbeta are then zero). */
typedef struct pkt_layernorm_desc {
  long long rows;
  int cols;
  int dtype;         /* of x, y, dy, dx: PKT_DTYPE_BF16 or PKT_DTYPE_F32 */
  int param_dtype;   /* of gamma, beta: PKT_DTYPE_BF16 or PKT_DTYPE_F32 */
  float eps;         /* forward */
  const void* x;     /* row stride ldx, in elements (so the other ld*) */
  long long ldx;
  const void* gamma; /* [cols], null: ones */
  const void* beta;  /* forward: [cols], null: zeros */
  void* y;           /* forward */
  long long ldy;
  float* mean;       /* [rows]: forward writes it (may be null), backward reads it */
  float* rstd;
  const void* dy;    /* backward */
  long long lddy;
  void* dx;          /* backward, may be null */
  long long lddx;
  float* dgamma;     /* backward: [cols], overwritten; may be null */
  float* dbeta;
  void* workspace;   /* backward: pkt_layernorm_backward_workspace bytes, used during the
                        call alone; calls that overlap on the GPU (two graphs, two
                        streams) need one each */
  size_t workspace_bytes;
} pkt_layernorm_desc;
int pkt_layernorm_forward(const pkt_layernorm_desc* d, void* stream);
/* Workspace of a backward call with these rows and cols on the current device. */
int pkt_layernorm_backward_workspace(const pkt_layernorm_desc* d, size_t* bytes);
int pkt_layernorm_backward(const pkt_layernorm_desc* d, void* stream);

/* Block-scaled 8-bit floats: a block of values with the largest magnitude `amax`
 * is held as q = round(x * (most / amax)) and scale = amax / most, where `most` is
 * the type's largest value (448 or 57344); x is about q * scale. Rounding is to
 * nearest, ties to even. A block with amax < 2^-100 is zeros with scale 0; a block
 * that holds an infinity or NaN has a non-finite scale. */

/* Quantises x [rows, cols]:
 *   q  [rows, cols]: blocks of 128 columns x block_rows rows,
 *      scale [ceil(cols/128), ceil(rows/block_rows)]: one row of scales per 128 columns
 *   qt [cols, rows]: the transposed matrix quantised the same way (blocks of 128 rows
 *      of x x block_rows columns), scale_t [ceil(rows/128), ceil(cols/block_rows)]
 * Either may be left out (null); both together read x once. These are operands of
 * pkt_fp8_gemm whose summed dimension is the contiguous one. Bytes of padded rows
 * past the matrix are not written. */
typedef struct pkt_fp8_quantize_desc {
  int rows, cols;
  int dtype;        /* of x: PKT_DTYPE_BF16 or PKT_DTYPE_F32 */
  int q_dtype;      /* PKT_DTYPE_E4M3 or PKT_DTYPE_E5M2 */
  int block_rows;   /* 1 (activations, gradients) or 128 (weights) */
  const void* x;
  long long ldx;
  void* q;          /* 16-byte aligned, ldq a multiple of 16 */
  long long ldq;
  float* scale;
  long long ld_scale;
  void* qt;         /* 16-byte aligned, ldqt a multiple of 16 */
  long long ldqt;
  float* scale_t;
  long long ld_scale_t;
} pkt_fp8_quantize_desc;
int pkt_fp8_quantize(const pkt_fp8_quantize_desc* d, void* stream);

/* out[m, n] = sum over blocks kb of 128 along K of
 *             scale_a[kb, m / a_block_rows] * scale_b[kb, n / b_block_rows]
 *             * sum over k in kb of a[m, k] * b[n, k]
 * on the tensor cores (tcgen05, fp32 accumulators); the scales are applied to each
 * block's fp32 sum and the blocks are added in fp32; the two scales may be multiplied
 * with one another first, so their product should not leave fp32's normal range
 * (below 2^-126 it loses bits). Any M, N, K >= 0 (K = 0:
 * zeros); a and b are 16-byte aligned with row strides that are multiples of 16.
 * The result of a call does not depend on timing. */
typedef struct pkt_fp8_gemm_desc {
  int M, N, K;
  int a_dtype, b_dtype; /* PKT_DTYPE_E4M3 or PKT_DTYPE_E5M2, each on its own */
  const void* a;        /* [M, K], row stride lda */
  long long lda;
  const float* scale_a; /* [ceil(K/128), ceil(M/a_block_rows)], row stride ld_scale_a */
  long long ld_scale_a;
  int a_block_rows;     /* 1 or 128 */
  const void* b;        /* [N, K], row stride ldb */
  long long ldb;
  const float* scale_b; /* [ceil(K/128), ceil(N/b_block_rows)], row stride ld_scale_b */
  long long ld_scale_b;
  int b_block_rows;     /* 1 or 128 */
  void* out;            /* [M, N], row stride ldo */
  long long ldo;
  int out_dtype;        /* PKT_DTYPE_BF16 or PKT_DTYPE_F32 */
} pkt_fp8_gemm_desc;
int pkt_fp8_gemm(const pkt_fp8_gemm_desc* d, void* stream);
/* AdamW over many tensors in one launch. For step t of a tensor, with g = grad *
 * gradient scale:
 *   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
 *   param = param (1 - lr weight_decay)
 *           - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * in fp32. state_dtype PKT_DTYPE_F32 keeps m and v as fp32. PKT_DTYPE_E4M3 keeps m
 * and sqrt(v) as block-scaled 8-bit floats (blocks of 128 consecutive values from
 * the tensor's start, scales m_scale / v_scale): 2 1/16 bytes per parameter instead
 * of 8; beside larger ones of its block a positive sqrt(v) is held as at least the
 * smallest 8-bit value, so that it does not turn into a division by eps alone (in a
 * block that is held as zeros it does). States start as zeros (scales too). Fastest
 * where all arrays of a tensor start on boundaries of 4 of their values; a tensor with
 * one that does not goes value by value.
 * The plan keeps the pointers and, on the device, the step count: replaying a
 * captured step advances it. Calls on a plan are ordered by the caller (one
 * stream, or events), also against replays of a captured step, and a plan outlives the
 * graphs that captured it. Arrays that a step writes must not overlap one another or a
 * gradient (PKT_ERR_ARGS); gradients may be shared. */
typedef struct pkt_adamw pkt_adamw;
typedef struct pkt_adamw_tensor {
  void* param;           /* [n], param_dtype, updated in place */
  const void* grad;      /* [n], grad_dtype; null: the tensor is left alone */
  void* m;               /* [n], state_dtype */
  void* v;               /* [n], state_dtype */
  float* m_scale;        /* 8-bit states: [ceil(n/128)] */
  float* v_scale;
  void* copy_bf16;       /* optional [n]: the new parameters rounded to bf16 */
  long long n;           /* 0: no pointer of the tensor is looked at */
  float weight_decay;
  int pad;
} pkt_adamw_tensor;
typedef struct pkt_adamw_config {
  int num_tensors;
  const pkt_adamw_tensor* tensors; /* read by pkt_adamw_create only */
  int param_dtype;                 /* PKT_DTYPE_F32 or PKT_DTYPE_BF16 */
  int grad_dtype;                  /* PKT_DTYPE_F32 or PKT_DTYPE_BF16 */
  int state_dtype;                 /* PKT_DTYPE_F32 or PKT_DTYPE_E4M3 */
  double beta1, beta2, eps;
  long long step;                  /* steps taken before the first call */
} pkt_adamw_config;
int pkt_adamw_create(int device, const pkt_adamw_config* cfg, pkt_adamw** out);
int pkt_adamw_destroy(pkt_adamw* h);
/* One step. `scales` (device memory, may be null): lr is multiplied by scales[0] and
 * the gradients by scales[1], read when the step runs (a schedule or a clipping
 * factor computed on the device, also under graph replay). grad_scale multiplies
 * the gradients too. */
int pkt_adamw_step(pkt_adamw* h, float lr, float grad_scale, const float* scales, void* stream);
/* New gradient pointers (num_tensors of them), for steps enqueued from now on. Not
 * inside a stream capture: steps captured before then read the new pointers too. */
int pkt_adamw_set_grads(pkt_adamw* h, const void* const* grads, void* stream);
/* Steps taken: set (stream-ordered), and read (synchronises the stream; not inside a
 * stream capture). */
int pkt_adamw_set_step(pkt_adamw* h, long long step, void* stream);
int pkt_adamw_get_step(pkt_adamw* h, long long* step, void* stream);

/* ---- MLP training engine (the hot path) -------------------------------- */
typedef struct pkt_mlp pkt_mlp;

typedef struct pkt_mlp_config {
  int num_layers;   /* L */
  const int* dims;  /* L+1 layer widths, dims[0] = input, dims[L] = output */
  int batch;        /* rows per GPU per step */
  int dtype;        /* PKT_DTYPE_BF16 (bf16 weights/acts, fp32 master) or PKT_DTYPE_TF32 */
  int has_bias;
  int relu_last;    /* ReLU after the output layer too (0 for plain regression) */
  float lr;
  int grad_mode;    /* 0: SGD fused into the weight-gradient epilogue; 1: store fp32
                       gradients, separate SGD pass (data parallel over NCCL /
                       inspection); 2: fused data parallel over peer memory
                       (pkt_mlp_dp_handle / pkt_mlp_dp_connect) */
  int max_bn;       /* largest tile N to use (0: 256) */
  int cta_pair;     /* 2: CTA pairs share 256-row tiles (tcgen05 cta_group::2);
                       1: every CTA computes its own 128-row tiles; 0: automatic
                       (pairs when the widest layer gives every pair a 256 x 256
                       tile, single CTAs for narrow, latency-bound networks) */
} pkt_mlp_config;

int pkt_mlp_create(int device, const pkt_mlp_config* cfg, pkt_mlp** out);
int pkt_mlp_destroy(pkt_mlp* m);
/* Parameters as fp32 host arrays: W concatenated [d_{l+1}, d_l] row-major, b concatenated. */
int pkt_mlp_set_params(pkt_mlp* m, const float* W, const float* b);
int pkt_mlp_get_params(pkt_mlp* m, float* W, float* b);
/* Gradients of the last step (grad_mode 1 only). */
int pkt_mlp_get_grads(pkt_mlp* m, float* dW, float* db);
/* Batch upload: x [batch, d0], target [batch, dL], host or device memory, in the
 * engine's storage type (uint16 bf16 bits for PKT_DTYPE_BF16, fp32 for TF32).
 * Stream-ordered (host memory should be pinned for async copies). The engine
 * has two input slots: each call fills the slot the previous call did not use
 * and makes it the one later training steps read, so a copy on another stream
 * can overlap the step still reading the other slot (the caller orders the
 * copy after the step that last read its slot, two loads back). */
int pkt_mlp_load_batch(pkt_mlp* m, const void* x, const void* target, int on_device, void* stream);
/* Enqueue `steps` training steps on the loaded batch. */
int pkt_mlp_train(pkt_mlp* m, int steps, void* stream);
/* Loss of each enqueued step since the last reset (device -> host, syncs). */
int pkt_mlp_losses(pkt_mlp* m, float* out, int max_n, int* n);
int pkt_mlp_reset_losses(pkt_mlp* m);
/* Device pointer of the loss of step i (for async reads). */
int pkt_mlp_loss_ptr(pkt_mlp* m, int i, float** out);
/* Output activations of the last step: y = last layer (fp32), [batch, dL]. */
int pkt_mlp_get_output(pkt_mlp* m, float* y);
int pkt_mlp_status(pkt_mlp* m, int* code, int* task_index, int* detail);
/* Tasks and GEMM tiles one step enqueues (for accounting). */
int pkt_mlp_step_info(pkt_mlp* m, int* tasks, int* gemm_tiles, double* flops);
/* Capture y = output layer (fp32) during training steps, for pkt_mlp_get_output. */
int pkt_mlp_set_output_capture(pkt_mlp* m, int enabled);
/* Data parallel (grad_mode 1). One step = pkt_mlp_forward_backward, then an
 * all-reduce (sum) of the fp32 gradient buffer by the caller (NCCL on the same
 * stream), then pkt_mlp_apply_update. grad_scale multiplies lr in the update
 * (1/world_size turns the summed per-rank mean gradients into the global mean). */
int pkt_mlp_grad_buffer(pkt_mlp* m, float** ptr, long long* count);
int pkt_mlp_set_grad_scale(pkt_mlp* m, float scale);
/* AdamW (pkt_adamw) in the place of SGD, in grad_mode 1: pkt_mlp_train and
 * pkt_mlp_apply_update then update the fp32 masters (and their bf16 copies) with it,
 * with the engine's lr and gradient scale; weight decay is for the weights, not the
 * biases. Starts with empty states and step 0; cfg = NULL goes back to SGD. A call that
 * fails leaves what was set before. pkt_mlp_set_params keeps the states, which (with
 * their step count) are the engine's own and cannot be read or set. Synchronises
 * the device. */
typedef struct pkt_mlp_adamw {
  double beta1, beta2, eps;
  float weight_decay;
  int state_dtype; /* PKT_DTYPE_F32 or PKT_DTYPE_E4M3 (8-bit states) */
} pkt_mlp_adamw;
int pkt_mlp_set_adamw(pkt_mlp* m, const pkt_mlp_adamw* cfg);
int pkt_mlp_forward_backward(pkt_mlp* m, void* stream);
int pkt_mlp_apply_update(pkt_mlp* m, void* stream);
/* The same step as pkt_mlp_forward_backward in L launches (grad_mode 1), so the
 * caller can all-reduce each layer's gradient on another stream as soon as it is
 * complete, overlapped with the rest of the backward: after segment s (0..L-1)
 * the bucket of layer L-1-s (pkt_mlp_grad_bucket: offset and count in floats
 * within pkt_mlp_grad_buffer, dW then db) is final. Segment 0 also runs the
 * forward and the loss. pkt_mlp_set_reserved_sms leaves that many SMs out of
 * the persistent grid, so a collective kernel on another stream has SMs to run
 * on while a segment runs (0 by default). */
int pkt_mlp_backward_segments(pkt_mlp* m, int* count);
int pkt_mlp_forward_backward_segment(pkt_mlp* m, int segment, void* stream);
int pkt_mlp_grad_bucket(pkt_mlp* m, int layer, long long* offset, long long* count);
int pkt_mlp_set_reserved_sms(pkt_mlp* m, int sms);
/* Fused data parallel (grad_mode 2): one launch per step on every rank; the
 * weight-gradient tiles go to their owner rank (tile index mod world) over
 * peer memory as they finish, the owner sums the ranks' partials in rank
 * order, applies SGD (lr x grad_scale) to its shard of the fp32 masters and
 * writes the new bf16 weights into every rank; the next step's forward tiles of
 * a layer start once that layer's weights have all arrived. Set-up: every rank
 * creates its engine, exports its exchange region (pkt_mlp_dp_handle, 64 bytes
 * of CUDA IPC handle), the caller exchanges the handles (e.g. an all-gather over
 * torch.distributed) and passes them, in rank order, to pkt_mlp_dp_connect.
 * world = 1 needs no handles. All ranks must run the same number of steps;
 * a rank that stops early makes the others' waits time out (PKT_ERR_TIMEOUT). */
#define PKT_DP_MAX_RANKS 8
int pkt_mlp_dp_handle(pkt_mlp* m, void* handle64);
int pkt_mlp_dp_connect(pkt_mlp* m, int rank, int world, const void* handles);
/* Per-CTA role cycle counters of the last launch (same layout as pkt_runtime_fetch_perf). */
int pkt_mlp_set_perf(pkt_mlp* m, int enabled);
int pkt_mlp_fetch_perf(pkt_mlp* m, unsigned long long* out, int max_blocks, int* blocks);
/* Effective SM clock of the engine's launches, as pkt_runtime_clock_stats. */
int pkt_mlp_clock_stats(pkt_mlp* m, unsigned long long* out3, int reset);
/* Per-task trace of the engine's launches, as pkt_runtime_set_trace / _fetch_trace
 * (task indices are those of one step's task list). */
int pkt_mlp_set_trace(pkt_mlp* m, int enabled);
int pkt_mlp_fetch_trace(pkt_mlp* m, unsigned long long* out, int max_tasks, int* n);

#ifdef __cplusplus
}
#endif

#endif /* PKT_B200_H */
