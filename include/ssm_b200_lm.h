/*
 * ssm_b200 — C ABI of the operators that stand beside the state-space operators of ssm_b200.h in a language model: the gated
 * delta rule (whole sequences and single tokens), log probabilities of given tokens, distillation from a teacher's top logits, the norms around
 * a block, cross entropy from hidden states, the norm over many tensors with clipping.
 * Same conventions: plain argument structs of raw device pointers, sizes, element strides and SSM_* dtype codes; kernels are
 * enqueued on the given stream; nothing is allocated or synchronised; 0, a negative SSM_ERR_* or a positive cudaError_t is returned
 * and ssm_b200_last_error() describes the last failure.
 */
#ifndef SSM_B200_LM_H_
#define SSM_B200_LM_H_

#include "ssm_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Raised with every change of a struct's layout, of an entry point's signature or of the set of entry points below. */
#define SSM_B200_LM_ABI_VERSION 2
int ssm_b200_lm_abi_version(void);

/* ---------------------------------------------------------------------------------------
 * Gated delta rule.  Per head, with a_t = exp(g_t) and a state S of (vdim, kdim):
 *
 *   S' = a_t S_{t-1};   r_t = v_t - S' k_t;   S_t = S' + beta_t r_t k_t^T;   o_t = scale S_t q_t
 *
 * q, k: (batch, len, key_heads, kdim), v: (batch, len, heads, vdim), io_dtype, innermost axis contiguous, the others at the given
 * element strides; head h reads key head h / (heads / key_heads).  g (natural logarithm of the decay; NULL: no decay), beta:
 * (batch, len, heads) of their own types and strides.  o: (batch, len, heads, vdim) dense, io_dtype.
 * kdim <= 256, vdim <= 65536.
 *
 * Packed sequences (num_seqs > 0): batch is 1, cu_seqlens (num_seqs + 1 entries on the device, 64-bit integers with cu_is_64, else
 * 32-bit) rises from 0 to at most len.  Boundaries are used where they lie; entries out of order or range are clamped so that no access
 * leaves the tensors.  Rows behind the last sequence are written as zeros.
 * States: initial (fp32) and final (final_dtype): (batch or num_seqs, heads, vdim, kdim) dense.
 *
 * table: scratch of ssm_gated_delta_table_ints(batch, len, num_seqs) 32-bit integers, needed when num_seqs > 0; the forward call
 * writes it, the backward call reads it.  For a backward pass to follow: rest (batch, len, heads, vdim) fp32 receives r, states fp32
 * of ssm_gated_delta_chunks(batch, len, num_seqs) x heads x vdim x kdim receives the state before every chunk of 32 tokens.
 * ------------------------------------------------------------------------------------- */
typedef struct {
  int32_t batch, len, heads, key_heads;
  int32_t kdim, vdim, io_dtype, g_dtype;
  int32_t beta_dtype, final_dtype, num_seqs, cu_is_64;
  float scale;
  int32_t reserved0;
  const void* q;
  const void* k;
  const void* v;
  const void* g; /* nullable */
  const void* beta;
  int64_t q_sb, q_st, q_sh;
  int64_t k_sb, k_st, k_sh;
  int64_t v_sb, v_st, v_sh;
  int64_t g_sb, g_st, g_sh;
  int64_t beta_sb, beta_st, beta_sh;
  const void* cu_seqlens;     /* nullable */
  const float* initial_state; /* nullable: zeros */
  void* o;
  void* final_state; /* nullable */
  int32_t* table;    /* nullable without packed sequences */
  float* rest;       /* nullable */
  float* states;     /* nullable */
} ssm_gated_delta_args;

int64_t ssm_gated_delta_chunks(int32_t batch, int32_t len, int32_t num_seqs);
int64_t ssm_gated_delta_table_ints(int32_t batch, int32_t len, int32_t num_seqs);
int ssm_gated_delta_fwd(const ssm_gated_delta_args* args, ssm_stream_t stream);

/* Backward.  fwd: the forward call's arguments with what it left in table, rest and states (o, final_state unused).
 * dout (batch, len, heads, vdim) dense, io_dtype; dfinal fp32 or NULL.  Written: dq, dk (batch, len, key_heads, kdim), dv, all dense
 * io_dtype; dg, dbeta (batch, len, heads) dense fp32; dinitial fp32 or NULL.  Scratch: dv32 (batch, len, heads, vdim) fp32 (may be dv
 * itself where io_dtype is fp32), dstates of the size of fwd.states, and with heads > key_heads dqk:
 * 2 x batch x len x heads x kdim fp32. */
typedef struct {
  ssm_gated_delta_args fwd;
  const void* dout;
  const float* dfinal; /* nullable */
  void* dq;
  void* dk;
  void* dv;
  float* dg;
  float* dbeta;
  float* dinitial; /* nullable */
  float* dv32;
  float* dstates;
  float* dqk; /* nullable where heads == key_heads */
} ssm_gated_delta_bwd_args;

int ssm_gated_delta_bwd(const ssm_gated_delta_bwd_args* args, ssm_stream_t stream);

/* The same on the tensor cores, in chunks of 64 tokens: 16-bit operands, kdim and vdim multiples of 8, kdim <= 128, q, k, v with rows on
 * 16-byte boundaries (strides multiples of 8 elements, none of zero), o and initial_state 16-byte aligned: ..._supported() tells, without
 * looking at anything on the device.  rest and states of the arguments are not used.  scratch is free again when the call's work is done,
 * kept holds what a backward pass reads (`train` nonzero) and is needed without one too; both 256-byte aligned.  They grow with the chunks, of
 * which packed sequences have up to len / 64 + num_seqs + 1: for kdim above 64, 40 KiB of scratch and 9 KiB kept a chunk and head; with a backward
 * pass to follow 25 KiB and 384 vdim bytes kept, and 256 vdim bytes of scratch in the backward call.  State, adjoint state and operands of products are
 * rounded to io_dtype once a chunk (results in bf16: 0.3 % off in norm for independent keys, more where keys hardly differ).  status: a 32-bit
 * word in memory that the device can write, set if a bounded wait ran out. */
int ssm_gated_delta_chunked_supported(const ssm_gated_delta_args* args);
int64_t ssm_gated_delta_chunked_scratch_bytes(int32_t batch, int32_t len, int32_t num_seqs, int32_t heads, int32_t kdim);
int64_t ssm_gated_delta_chunked_kept_bytes(int32_t batch, int32_t len, int32_t num_seqs, int32_t heads, int32_t kdim, int32_t vdim, int32_t train);
int ssm_gated_delta_chunked_fwd(const ssm_gated_delta_args* args, void* scratch, void* kept, int32_t train, int32_t* status, ssm_stream_t stream);
/* Its backward: dv32 and dstates of the arguments are not used (scratch takes their place); dout, dq, dk, dv, dfinal, dqk 16-byte aligned. */
int64_t ssm_gated_delta_chunked_bwd_scratch_bytes(int32_t batch, int32_t len, int32_t num_seqs, int32_t heads, int32_t kdim, int32_t vdim);
int ssm_gated_delta_chunked_bwd(const ssm_gated_delta_bwd_args* args, void* kept, void* scratch, int32_t* status, ssm_stream_t stream);

/* One token: state (batch, heads, vdim, kdim) fp32, 16-byte aligned, updated in place; q, k (batch, key_heads, kdim), v (batch, heads,
 * vdim), g, beta (batch, heads) at strides; o (batch, heads, vdim) dense. */
typedef struct {
  int32_t batch, heads, key_heads, kdim;
  int32_t vdim, io_dtype, g_dtype, beta_dtype;
  float scale;
  int32_t reserved0;
  float* state;
  const void* q;
  const void* k;
  const void* v;
  const void* g; /* nullable */
  const void* beta;
  int64_t q_sb, q_sh;
  int64_t k_sb, k_sh;
  int64_t v_sb, v_sh;
  int64_t g_sb, g_sh;
  int64_t beta_sb, beta_sh;
  void* o;
} ssm_gated_delta_step_args;

int ssm_gated_delta_step(const ssm_gated_delta_step_args* args, ssm_stream_t stream);

/* ---------------------------------------------------------------------------------------
 * Log probabilities of given tokens.  logits (rows, vocab) of io_dtype, contiguous rows at row_stride; x = logits / temperature,
 * p = softmax(x).  logp[r] = log p[targets[r]]; 0 where targets[r] == ignore_index; NaN for any other target outside of the vocabulary.
 * entropy[r] = -sum p log p.  top_ids / top_logp (rows, top_k): the top_k largest logits in falling order, equal ones by rising id.
 * stats (rows, 4) fp32: what the backward pass needs.  A row of -inf alone has no distribution: log probabilities -inf, entropy 0,
 * gradients 0; a NaN or +inf in a row makes its results NaN.  vocab <= 2^30, top_k <= min(vocab, 128).
 *
 * Backward: dlogits (rows, vocab) dense, from dlogp, dentropy, dtop_logp (each nullable).
 * ------------------------------------------------------------------------------------- */
typedef struct {
  int64_t rows, row_stride;
  int32_t vocab, io_dtype, top_k, reserved0;
  int64_t ignore_index;
  float temperature;
  int32_t reserved1;
  const void* logits;
  const int64_t* targets;
  float* logp;
  float* entropy;   /* nullable */
  float* top_logp;  /* nullable without top_k */
  int64_t* top_ids; /* nullable without top_k */
  float* stats;     /* nullable */
} ssm_token_logp_args;

typedef struct {
  ssm_token_logp_args fwd; /* logits, targets, top_ids and stats are read */
  const float* dlogp;      /* nullable */
  const float* dentropy;   /* nullable */
  const float* dtop_logp;  /* nullable */
  void* dlogits;
} ssm_token_logp_bwd_args;

int ssm_token_logp(const ssm_token_logp_args* args, ssm_stream_t stream);
int ssm_token_logp_bwd(const ssm_token_logp_bwd_args* args, ssm_stream_t stream);

/* ---------------------------------------------------------------------------------------
 * Distillation from a teacher's top logits: t = softmax(teacher / temperature) over a row's top_k entries (those with a negative id
 * left out), loss[r] = sum_j t_j (log t_j - log softmax(logits / temperature)[ids_j]).  An id of vocab or above whose t_j is not 0 makes a row's loss
 * and gradient NaN; with a teacher logit of -inf, or one so low that t_j is 0, it counts for nothing.
 * A row without entries, or with entries of -inf alone, has loss 0 and no gradient; a student row of -inf alone has loss inf and no gradient.
 * teacher, ids: (rows, top_k) dense.  top_k <= 1024.  Backward: dlogits (rows, vocab) dense from dloss; an id given twice counts twice.
 * ------------------------------------------------------------------------------------- */
typedef struct {
  int64_t rows, row_stride;
  int32_t vocab, io_dtype, top_k, teacher_dtype;
  float temperature;
  int32_t reserved0;
  const void* logits;
  const void* teacher;
  const int64_t* ids;
  float* loss;
  float* stats; /* nullable: (rows, 4) fp32 for the backward pass */
} ssm_topk_distill_args;

typedef struct {
  ssm_topk_distill_args fwd;
  const float* dloss;
  void* dlogits;
} ssm_topk_distill_bwd_args;

int ssm_topk_distill(const ssm_topk_distill_args* args, ssm_stream_t stream);
int ssm_topk_distill_bwd(const ssm_topk_distill_bwd_args* args, ssm_stream_t stream);

/* ---------------------------------------------------------------------------------------
 * The norms after and before a block with its gate, residual scale and residual add:
 *   n = norm(x) post_weight + post_bias;   residual_out = residual + scale gate n;   y = norm(residual_out) weight + bias
 * norm(x) = (x - m) / sqrt(mean (x - m)^2 + eps), m the row's mean, or 0 with is_rms; post_eps and eps for the two.  All tensors dense: x, y (rows, dim) of io_dtype,
 * residual (nullable: 0) of res_dtype, residual_out of resout_dtype (rounded there; y is formed from what it was before), parameters (dim) of param_dtype,
 * both biases or neither.  gate of gate_dtype: gate_kind 0 none (1), 1 (dim), 2 (rows / len, dim), one row for `len` rows, 3 (rows, dim).
 * stats (rows, 4) fp32, 16-byte aligned, for the backward pass; nullable.  dim <= 8192.
 *
 * Backward: from dy and dresidual_out (nullable) writes dx, dresidual (nullable; res_dtype), the parameters' gradients (param_dtype; biases' nullable) and dgate
 * (gate's shape and type).  partial: ssm_block_norm_bwd_scratch_floats floats, 16-byte aligned.
 * ------------------------------------------------------------------------------------- */
typedef struct {
  int64_t rows, len;
  int32_t dim, io_dtype, res_dtype, resout_dtype;
  int32_t param_dtype, gate_dtype, gate_kind, is_rms;
  float eps, post_eps, scale;
  int32_t reserved0;
  const void* x;
  const void* residual; /* nullable */
  const void* post_weight;
  const void* weight;
  const void* post_bias; /* nullable */
  const void* bias;      /* nullable */
  const void* gate;      /* nullable */
  void* y;
  void* residual_out;
  float* stats; /* nullable */
} ssm_block_norm_args;

typedef struct {
  ssm_block_norm_args fwd; /* y and residual_out are not read */
  const void* dy;
  const void* dresidual_out; /* nullable */
  void* dx;
  void* dresidual; /* nullable */
  void* dpost_weight;
  void* dweight;
  void* dpost_bias; /* nullable */
  void* dbias;      /* nullable */
  void* dgate;      /* nullable without a gate */
  float* partial;
} ssm_block_norm_bwd_args;

int ssm_block_norm_fwd(const ssm_block_norm_args* args, ssm_stream_t stream);
int64_t ssm_block_norm_bwd_scratch_floats(int64_t rows, int32_t dim);
int ssm_block_norm_bwd(const ssm_block_norm_bwd_args* args, ssm_stream_t stream);

/* ---------------------------------------------------------------------------------------
 * Cross entropy from hidden states: z = hidden weight^T, log_z[r] = ln sum_v exp z[r, v], loss[r] = log_z[r] - z[r, targets[r]], without a (rows, vocab) matrix.
 * hidden (rows, dim), weight (vocab, dim) of io_dtype, rows at their strides.  A row whose target is ignore_index costs nothing, is not read and gives 0; any other target outside
 * of the vocabulary gives a loss of NaN.  row_loss and log_z (rows) fp32; loss, with reduction 1 (sum) or 2 (mean over the rows that count, 0 without any), one float.
 * stats (rows, 4) fp32, 16-byte aligned, keeps what the backward pass needs (nullable).  status: a word in host memory that the device writes, set where a bounded wait ran out.
 *
 * Backward: from dloss (rows, or one float with a reduction) and dlog_z (rows, nullable) writes dhidden (rows, dim; io_dtype) and dweight (vocab, dim; dweight_dtype),
 * dense, each nullable, via pieces of the logits' gradient in 16 bits (three times 16 for fp32): at most SSM_LINEAR_CE_PIECE_BYTES and 16384 rows, or 256 rows where those are larger.
 * packs, 256-byte aligned, ssm_linear_ce_packs_bytes(args) bytes (which go by weight and weight_stride too: a weight that cannot be copied from its place is packed, so both are set before it
 * is asked): the rows that count (and, in fp32, the weight) as the products read them, written by the forward pass and read by
 * the backward pass.  scratch: ssm_linear_ce_scratch_bytes(args, pass) bytes, 256-byte aligned; pass 0 forward, 1 backward, 2 both at once.
 *
 * ssm_linear_ce_train, for bf16 with a reduction: the forward pass and, for a dloss that is known later, dhidden (rows, dim) and dweight (vocab, dim rounded up to a multiple of
 * 4) in fp32, 16-byte aligned, each nullable; kept: three words.  ssm_linear_ce_scale then multiplies either, (rows, dim) at the row stride ld, by dloss and what `kept` holds.
 * ------------------------------------------------------------------------------------- */
#define SSM_LINEAR_CE_PIECE_BYTES (512 << 20)
typedef struct {
  int64_t rows, hidden_stride, weight_stride, ignore_index;
  int32_t dim, vocab, io_dtype, reduction;
  const void* hidden;
  const void* weight;
  const int64_t* targets;
  float* row_loss;
  float* log_z;
  float* loss;  /* nullable without a reduction */
  float* stats; /* nullable */
  void* packs;
  void* scratch;
  int32_t* status;
} ssm_linear_ce_args;

typedef struct {
  ssm_linear_ce_args fwd; /* hidden, weight, targets, stats and packs are read */
  const float* dloss;
  const float* dlog_z; /* nullable */
  void* dhidden;       /* nullable */
  void* dweight;       /* nullable */
  int32_t dweight_dtype, reserved0;
} ssm_linear_ce_bwd_args;

int64_t ssm_linear_ce_packs_bytes(const ssm_linear_ce_args* args);
int64_t ssm_linear_ce_scratch_bytes(const ssm_linear_ce_args* args, int32_t pass);
int ssm_linear_ce_fwd(const ssm_linear_ce_args* args, ssm_stream_t stream);
int ssm_linear_ce_bwd(const ssm_linear_ce_bwd_args* args, ssm_stream_t stream);
int ssm_linear_ce_train(const ssm_linear_ce_args* args, float* dhidden, float* dweight, float* kept, ssm_stream_t stream);
int ssm_linear_ce_scale(const float* src, int64_t ld, int64_t rows, int32_t dim, const float* kept, const float* dloss, void* out, int32_t dtype, ssm_stream_t stream);

/* ---------------------------------------------------------------------------------------
 * The norm over all elements of many tensors: sqrt(sum x^2), or max |x| with is_max, into *norm (device, fp32); NaN once there is one.  Clipping multiplies
 * every element in place by min(1, max_norm / (norm + 1e-6)) and leaves all as it is where that is 1 or max_norm infinite.  The list is read by the
 * host during the call; every tensor is dense memory of its type.  scratch: ssm_global_norm_scratch_bytes(count) bytes, 8-byte aligned.
 * ------------------------------------------------------------------------------------- */
typedef struct {
  const void* data;
  int64_t numel;
  int32_t dtype, reserved0;
} ssm_tensor_ref;

int64_t ssm_global_norm_scratch_bytes(int64_t count);
int ssm_global_norm(const ssm_tensor_ref* tensors, int64_t count, int32_t is_max, void* scratch, float* norm, ssm_stream_t stream);
int ssm_clip_global_norm(const ssm_tensor_ref* tensors, int64_t count, int32_t is_max, float max_norm, void* scratch, float* norm, ssm_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SSM_B200_LM_H_ */
