// What the kernels of the gated delta rule share: where sequences and their chunks lie, operands at strides.
//
//   S' = a_t S_{t-1};  r_t = v_t - S' k_t;  S_t = S' + beta_t r_t k_t^T;  o_t = scale S_t q_t        (S: vdim x kdim, a = e^g)
#pragma once

#include "../../include/ssm_b200_lm.h"
#include "common.cuh"

namespace ssmb {
namespace gd {

constexpr int kChunk = 32;  // tokens between two states that the forward pass leaves for the backward

// Packed sequences.  Chunks are counted from a sequence's first token; behind the last sequence's chunks come those of the
// rows that belong to none (their gradients are zeros).  Layout of the table: 2 ints a sequence (first token, end), one int a sequence
// (its first chunk), then 3 ints a chunk (first token, end, sequence or -1); unused chunks have no tokens.
__host__ __device__ inline int64_t chunk_bound(int64_t batch, int64_t len, int64_t seqs, int chunk) {
  return seqs > 0 ? len / chunk + seqs + 1 : batch * ((len + chunk - 1) / chunk);
}

struct Seqs {
  const int32_t* table;  // NULL: dense (batch, len)
  int len, seqs, per;    // per: chunks of a dense sequence
};
struct Span {
  int b, t0, t1, seq, chunk;
};
__device__ __forceinline__ Span sequence(const Seqs& s, int i) {
  if (!s.table) return {i, 0, s.len, i, i * s.per};
  return {0, s.table[2 * i], s.table[2 * i + 1], i, s.table[2 * s.seqs + i]};
}
__device__ __forceinline__ Span chunk_of(const Seqs& s, int c, int chunk) {
  if (!s.table) {
    const int b = c / s.per, t0 = (c % s.per) * chunk;
    return {b, t0, min(s.len, t0 + chunk), b, c};
  }
  const int32_t* e = s.table + 3 * s.seqs + 3 * c;
  return {0, e[0], e[1], e[2], c};
}

struct Rows {  // an operand at strides (batch, token, head)
  const void* p;
  int64_t sb, st, sh;
};
struct Args {
  Rows q, k, v, g, beta;
  int io, g_dtype, beta_dtype, kd, vd, heads, group, len, seqs, final_dtype;  // group: value heads of a key head
  float scale;
  Seqs where;
};

// decay and write strength of a token
__device__ __forceinline__ float decay_of(const Args& a, int b, int t, int h) {
  return a.g.p ? expf(load_dyn(a.g.p, b * a.g.sb + t * a.g.st + h * a.g.sh, a.g_dtype)) : 1.f;
}
__device__ __forceinline__ float beta_of(const Args& a, int b, int t, int h) {
  return load_dyn(a.beta.p, b * a.beta.sb + t * a.beta.st + h * a.beta.sh, a.beta_dtype);
}

int check(const ssm_gated_delta_args& a, Args& d);
int check_gradients(const ssm_gated_delta_bwd_args& g);  // of the backward call's own pointers, their alignment
// sums the fp32 gradients of a key head's value heads (dq, then dk of all tokens) into dq and dk
int fold_heads(const float* dqk, void* dq, void* dk, int64_t tokens, int kd, int key_heads, int group, int dtype, cudaStream_t st);
// forms the table on the device; a no-op without packed sequences
int make_table(const ssm_gated_delta_args& a, int chunk, cudaStream_t st);

}  // namespace gd
}  // namespace ssmb
