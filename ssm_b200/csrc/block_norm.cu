// The norms after and before a block, fused with the block's gate, its residual scale and the residual add; forward and backward.
//
//   n = h1 w1 + b1,  h1 = (x - m1) s1;   r = residual + scale gate n;   y = h2 w2 + b2,  h2 = (r - m2) s2
//
// with m the mean of a row (0 for RMSNorm) and s = 1 / sqrt(mean (x - m)^2 + eps).  Backward, with means over a row, from dy and dr (the gradient of r):
//
//   g2 = w2 dy;   dr' = dr + s2 (g2 - [mean g2] - h2 mean(g2 h2));   dn = scale gate dr';   dgate = scale dr' n
//   g1 = w1 dn;   dx = s1 (g1 - [mean g1] - h1 mean(g1 h1));   dresidual = dr';   dw1 = sum dn h1, db1 = sum dn, dw2 = sum dy h2, db2 = sum dy
//
// Bound: HBM, 12 bytes an element forward and 20 back with 16-bit activations and a 32-bit stream.  A row is owned by 32 to 512 threads and lies in their
// registers, read once; everything is computed in 32 bits.  The forward pass leaves m1, s1, m2, s2 of each row for the backward pass, which forms r
// again from x and the residual (it would have to read one of the two anyway).  Backward blocks take runs of neighbouring rows and keep the parameters' gradients of their
// columns in registers; partial rows are added up by a second kernel in a fixed order, so that the bits repeat.  A gate given per sequence has its
// gradient finished where a block holds the whole sequence, and through partial rows where it does not.
#include <algorithm>

#include "../../include/ssm_b200_lm.h"
#include "common.cuh"

namespace ssmb {
namespace {

constexpr int kMaxRuns = 148 * 8;  // backward blocks

template <int V>
__device__ __forceinline__ void load_vec(const void* base, int64_t i, int dtype, float (&f)[V]) {
  if constexpr (V == 1) f[0] = load_dyn(base, i, dtype);
  else load_param_vec<V>(base, i, dtype, f);
}
template <int V>
__device__ __forceinline__ void store_vec(void* base, int64_t i, int dtype, const float (&f)[V]) {
  if constexpr (V == 1) {
    store_dyn(base, i, dtype, f[0]);
  } else if (dtype == SSM_F32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i);
#pragma unroll
    for (int k = 0; k < V / 4; ++k) __stcs(p + k, make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]));
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      if (dtype == SSM_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    uint16_t* p = reinterpret_cast<uint16_t*>(base) + i;
    if constexpr (V == 8) __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    else __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
  }
}

// a row's pieces of one tensor: all loads first, conversions afterwards
template <int V>
struct Raw {
  uint4 a, b;
};
template <int V>
__device__ __forceinline__ void issue(const void* base, int64_t i, int dtype, Raw<V>& r) {
  if constexpr (V == 1) {
    if (dtype == SSM_F32) r.a.x = __ldcs(reinterpret_cast<const uint32_t*>(base) + i);
    else r.a.x = __ldcs(reinterpret_cast<const uint16_t*>(base) + i);
  } else if (dtype == SSM_F32) {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + i);
    r.a = __ldcs(p);
    if constexpr (V == 8) r.b = __ldcs(p + 1);
  } else if constexpr (V == 8) {
    r.a = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + i));
  } else {
    const uint2 t = __ldcs(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(base) + i));
    r.a.x = t.x, r.a.y = t.y;
  }
}
__device__ __forceinline__ void halves(uint32_t w, int dtype, float& lo, float& hi) {
  if (dtype == SSM_BF16) {
    lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = h.x, hi = h.y;
  }
}
template <int V>
__device__ __forceinline__ void convert(const Raw<V>& r, int dtype, float (&f)[V]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if (dtype == SSM_F32) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = __uint_as_float(w[k]);
  } else if constexpr (V == 1) {
    float hi;
    halves(w[0], dtype, f[0], hi);
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) halves(w[k], dtype, f[2 * k], f[2 * k + 1]);
  }
}

// sums of two values over the G threads of a block
template <int G>
__device__ __forceinline__ void allsum2(float& a, float& b, float2 (*scratch)[16], int& turn) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off), b += __shfl_xor_sync(0xffffffffu, b, off);
  if constexpr (G > 32) {  // two rows of scratch in turn: a barrier a sum
    if (threadIdx.x % 32 == 0) scratch[turn][threadIdx.x / 32] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) a += scratch[turn][w].x, b += scratch[turn][w].y;
    turn ^= 1;
  }
}

enum Gate { kNone = 0, kChannel = 1, kSequence = 2, kToken = 3 };

// No load of these kernels depends on a condition for its address: what a call does not have (a residual, an incoming gradient) points at what it has, with a flag to leave it
// out, and in the forward pass a thread beyond the row's end reads the row's last piece.

// Mean and 1 / std of a row; V elements to a piece, MC pieces to a thread: piece c of thread t is c G + t, and there are n of them
template <int V, int G, int MC>
__device__ __forceinline__ void row_stats(const float (&f)[MC][V], int n, float inv, bool rms, float eps, float2 (*scratch)[16], int& turn, float& mean, float& rstd) {
  float t = 0.f, q = 0.f;
  mean = 0.f;
  if (!rms) {
#pragma unroll
    for (int c = 0; c < MC; ++c) {
#pragma unroll
      for (int k = 0; k < V; ++k) t += c * G + (int)threadIdx.x < n ? f[c][k] : 0.f;
    }
    allsum2<G>(t, q, scratch, turn);
    mean = t * inv, q = 0.f;
  }
#pragma unroll
  for (int c = 0; c < MC; ++c) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = c * G + (int)threadIdx.x < n ? f[c][k] - mean : 0.f;
      q = fmaf(d, d, q);
    }
  }
  t = 0.f;
  allsum2<G>(q, t, scratch, turn);
  rstd = rsqrtf(q * inv + eps);
}

// h, n and the factor of n in r, for a row's piece; w is left as post_weight
template <int V, bool BIAS, bool GATE>
__device__ __forceinline__ void branch(const ssm_block_norm_args& a, int col, int64_t gate_at, float m1, float s1, const float (&x)[V], float (&h)[V], float (&n)[V], float (&ga)[V],
                                       float (&w)[V]) {
  load_vec<V>(a.post_weight, col, a.param_dtype, w);
  if (BIAS) load_vec<V>(a.post_bias, col, a.param_dtype, n);
  if (GATE) load_vec<V>(a.gate, gate_at + col, a.gate_dtype, ga);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    h[k] = (x[k] - m1) * s1;
    n[k] = BIAS ? fmaf(h[k], w[k], n[k]) : h[k] * w[k];
    ga[k] = GATE ? a.scale * ga[k] : a.scale;
  }
}

struct FwdArgs {
  ssm_block_norm_args a;
  int len, has_r;  // rows of a sequence; the residual is one
};

template <int V, int G, int MC, bool BIAS, bool GATE>
__global__ void __launch_bounds__(G) block_norm_kernel(const __grid_constant__ FwdArgs args) {
  const ssm_block_norm_args& a = args.a;
  __shared__ float2 scratch[2][16];
  int turn = 0;
  const int tid = threadIdx.x, dim = a.dim, n = dim / V, row = blockIdx.x;
  const float inv = 1.f / (float)dim;
  const int64_t at = (int64_t)row * dim, gate_at = a.gate_kind == kToken ? at : a.gate_kind == kSequence ? (int64_t)(row / args.len) * dim : 0;
  float v[MC][V];
  Raw<V> rx[MC], rr[MC];
#pragma unroll
  for (int c = 0; c < MC; ++c) issue<V>(a.x, at + min(c * G + tid, n - 1) * V, a.io_dtype, rx[c]);
#pragma unroll
  for (int c = 0; c < MC; ++c) issue<V>(a.residual, at + min(c * G + tid, n - 1) * V, a.res_dtype, rr[c]);
#pragma unroll
  for (int c = 0; c < MC; ++c) convert<V>(rx[c], a.io_dtype, v[c]);
  float m1, s1, m2, s2;
  row_stats<V, G, MC>(v, n, inv, a.is_rms, a.post_eps, scratch, turn, m1, s1);
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int col = min(c * G + tid, n - 1) * V;
    float h[V], b[V], ga[V], w[V], r[V];
    branch<V, BIAS, GATE>(a, col, gate_at, m1, s1, v[c], h, b, ga, w);
    convert<V>(rr[c], a.res_dtype, r);
#pragma unroll
    for (int k = 0; k < V; ++k) v[c][k] = args.has_r ? fmaf(ga[k], b[k], r[k]) : ga[k] * b[k];
    if (c * G + tid < n) store_vec<V>(a.residual_out, at + col, a.resout_dtype, v[c]);
  }
  row_stats<V, G, MC>(v, n, inv, a.is_rms, a.eps, scratch, turn, m2, s2);
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int col = min(c * G + tid, n - 1) * V;
    float w[V], b[V], y[V];
    load_vec<V>(a.weight, col, a.param_dtype, w);
    if (BIAS) load_vec<V>(a.bias, col, a.param_dtype, b);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float h = (v[c][k] - m2) * s2;
      y[k] = BIAS ? fmaf(h, w[k], b[k]) : h * w[k];
    }
    if (c * G + tid < n) store_vec<V>(a.y, at + col, a.io_dtype, y);
  }
  if (a.stats && tid == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(m1, s1, m2, s2);
}

// where a run of rows leaves its sums: [run][which][dim]; which: dpost_weight, dweight, dpost_bias, dbias, dgate (of its first sequence, of its last)
constexpr int kSlots = 6;

// The backward pass of a run of rows.  V elements to a piece, piece c of thread t is c G + t.  A row's chain is long (loads, two rounds of sums, stores), so the next row is on its way
// into shared memory while this one is worked on: each thread copies its own pieces (asynchronous copies, no barrier) and reads them there again where it needs them,
// which leaves the registers to the sums of its columns.
template <int V, int G, int MC>
struct RowRing {
  static constexpr int kBytes = MC * G * V * 4;  // of one tensor, 32-bit elements
};
template <int V>
__device__ __forceinline__ void copy_piece(uint32_t dst, const void* base, int64_t i, int dtype) {
  if constexpr (V == 4) {
    if (dtype == SSM_F32) {
      const float* src = reinterpret_cast<const float*>(base) + i;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
    } else {
      const uint16_t* src = reinterpret_cast<const uint16_t*>(base) + i;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(dst), "l"(src) : "memory");
    }
  } else {  // element by element, through the registers
    if (dtype == SSM_F32) asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(dst), "r"(reinterpret_cast<const uint32_t*>(base)[i]) : "memory");
    else asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(dst), "r"((uint32_t) reinterpret_cast<const uint16_t*>(base)[i]) : "memory");
  }
}
template <int V>
__device__ __forceinline__ void read_piece(const unsigned char* at, int dtype, float (&f)[V]) {
  if constexpr (V == 4) {
    if (dtype == SSM_F32) {
      const float4 v = *reinterpret_cast<const float4*>(at);
      f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(at);
      halves(v.x, dtype, f[0], f[1]), halves(v.y, dtype, f[2], f[3]);
    }
  } else {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(at);
    float hi;
    if (dtype == SSM_F32) f[0] = __uint_as_float(v);
    else halves(v, dtype, f[0], hi);
  }
}

struct BwdArgs {
  ssm_block_norm_bwd_args g;
  int rows, per, len, unit;  // rows in all, of a run, of a sequence, that share a gate
  int stages, has_r, has_d, d_dtype;  // rows in shared memory; the residual is one, and the gradient that came through it
};

template <int V, int G, int MC, bool BIAS, bool GATE>
__global__ void __launch_bounds__(G) block_norm_bwd_kernel(const __grid_constant__ BwdArgs args) {
  const ssm_block_norm_bwd_args& g = args.g;
  const ssm_block_norm_args& a = g.fwd;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 scratch[2][16];
  constexpr int kT = RowRing<V, G, MC>::kBytes, kB = BIAS ? MC : 1, kG = GATE ? MC : 1;
  int turn = 0;
  const int tid = threadIdx.x, dim = a.dim, n = dim / V;
  const float inv = 1.f / (float)dim;
  const int first = blockIdx.x * args.per, last = min(args.rows, first + args.per);
  const bool has_r = args.has_r, has_d = args.has_d, two = args.stages == 2;
  float dpw[MC][V], dw[MC][V], dpb[kB][V], db[kB][V], dg[kG][V];
#pragma unroll
  for (int c = 0; c < MC; ++c) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      dpw[c][k] = dw[c][k] = 0.f;
      if (BIAS) dpb[BIAS ? c : 0][k] = db[BIAS ? c : 0][k] = 0.f;
      if (GATE) dg[GATE ? c : 0][k] = 0.f;
    }
  }
  float* const part = g.partial + (int64_t)blockIdx.x * kSlots * dim;
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring);

  int stage = 0;
  for (int next = first; next <= last; ++next) {  // the row `next` sets out, the one before it is worked on
    const int into = two ? (next - first) & 1 : 0;
    if (next < last && (two || next == first)) {
      const int64_t at = (int64_t)next * dim;
#pragma unroll
      for (int c = 0; c < MC; ++c) {
        const int p = c * G + tid;
        if (p < n) {
          const uint32_t to = ring0 + into * 4 * kT + p * V * 4;
          copy_piece<V>(to, a.x, at + p * V, a.io_dtype);
          copy_piece<V>(to + kT, g.dy, at + p * V, a.io_dtype);
          copy_piece<V>(to + 2 * kT, a.residual, at + p * V, a.res_dtype);
          copy_piece<V>(to + 3 * kT, g.dresidual_out, at + p * V, args.d_dtype);
        }
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    if (next == first) continue;
    if (two) asm volatile("cp.async.wait_group 1;\n" ::: "memory");
    else asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    const int row = next - 1;
    const int64_t at = (int64_t)row * dim, gate_at = a.gate_kind == kToken ? at : a.gate_kind == kSequence ? (int64_t)(row / args.len) * dim : 0;
    const unsigned char* const mine = ring + stage * 4 * kT;
    const float4 stats = reinterpret_cast<const float4*>(a.stats)[row];
    const float m1 = stats.x, s1 = stats.y, m2 = stats.z, s2 = stats.w;
    float h2[MC][V], d[MC][V];
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * G + tid;
      if (p < n) {
        float x[V], h[V], b[V], ga[V], w[V], r[V], dy[V];
        read_piece<V>(mine + p * V * 4, a.io_dtype, x);
        branch<V, BIAS, GATE>(a, p * V, gate_at, m1, s1, x, h, b, ga, w);
        read_piece<V>(mine + kT + p * V * 4, a.io_dtype, dy);
        read_piece<V>(mine + 2 * kT + p * V * 4, a.res_dtype, r);
        load_vec<V>(a.weight, p * V, a.param_dtype, w);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = has_r ? fmaf(ga[k], b[k], r[k]) : ga[k] * b[k];
          h2[c][k] = (v - m2) * s2;
          dw[c][k] = fmaf(dy[k], h2[c][k], dw[c][k]);
          if (BIAS) db[BIAS ? c : 0][k] += dy[k];
          d[c][k] = w[k] * dy[k];
          sum0 += d[c][k], sum1 = fmaf(d[c][k], h2[c][k], sum1);
        }
      }
    }
    allsum2<G>(sum0, sum1, scratch, turn);
    const float c2 = a.is_rms ? 0.f : sum0 * inv, e2 = sum1 * inv;
    sum0 = sum1 = 0.f;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * G + tid;
      if (p < n) {
        float x[V], h[V], b[V], ga[V], w[V], o[V], gg[V];
        read_piece<V>(mine + p * V * 4, a.io_dtype, x);
        branch<V, BIAS, GATE>(a, p * V, gate_at, m1, s1, x, h, b, ga, w);
        read_piece<V>(mine + 3 * kT + p * V * 4, args.d_dtype, o);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float t = s2 * (d[c][k] - c2 - h2[c][k] * e2);
          if (has_d) t += o[k];
          o[k] = t;
          gg[k] = a.scale * t * b[k];
          if (GATE) dg[GATE ? c : 0][k] += gg[k];
          const float dn = ga[k] * t;
          dpw[c][k] = fmaf(dn, h[k], dpw[c][k]);
          if (BIAS) dpb[BIAS ? c : 0][k] += dn;
          d[c][k] = w[k] * dn;
          sum0 += d[c][k], sum1 = fmaf(d[c][k], h[k], sum1);
        }
        if (g.dresidual) store_vec<V>(g.dresidual, at + p * V, a.res_dtype, o);
        if (a.gate_kind == kToken) store_vec<V>(g.dgate, at + p * V, a.gate_dtype, gg);
      }
    }
    allsum2<G>(sum0, sum1, scratch, turn);
    const float c1 = a.is_rms ? 0.f : sum0 * inv, e1 = sum1 * inv;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * G + tid;
      if (p < n) {
        float x[V];
        read_piece<V>(mine + p * V * 4, a.io_dtype, x);
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = s1 * (d[c][k] - c1 - (x[k] - m1) * s1 * e1);
        store_vec<V>(g.dx, at + p * V, a.io_dtype, x);
      }
    }
    if (GATE && a.gate_kind != kToken && (row + 1 == last || (row + 1) % args.unit == 0)) {  // the gate's rows end here, or the run does
      const int seq = row / args.unit, begin = seq * args.unit, end = begin + args.unit;
#pragma unroll
      for (int c = 0; c < MC; ++c) {
        const int p = c * G + tid;
        if (p < n) {
          if (begin >= first && end <= last) store_vec<V>(g.dgate, (int64_t)seq * dim + p * V, a.gate_dtype, dg[GATE ? c : 0]);
          else if (begin < first) store_vec<V>(part, 4 * dim + p * V, SSM_F32, dg[GATE ? c : 0]);
          else store_vec<V>(part, 5 * dim + p * V, SSM_F32, dg[GATE ? c : 0]);
#pragma unroll
          for (int k = 0; k < V; ++k) dg[GATE ? c : 0][k] = 0.f;
        }
      }
    }
    stage = two ? stage ^ 1 : 0;
    if (!two && next < last) {  // one row's room: the next one sets out now
      const int64_t to_row = (int64_t)next * dim;
#pragma unroll
      for (int c = 0; c < MC; ++c) {
        const int p = c * G + tid;
        if (p < n) {
          const uint32_t to = ring0 + p * V * 4;
          copy_piece<V>(to, a.x, to_row + p * V, a.io_dtype);
          copy_piece<V>(to + kT, g.dy, to_row + p * V, a.io_dtype);
          copy_piece<V>(to + 2 * kT, a.residual, to_row + p * V, a.res_dtype);
          copy_piece<V>(to + 3 * kT, g.dresidual_out, to_row + p * V, args.d_dtype);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int p = c * G + tid;
    if (p < n) {
      store_vec<V>(part, p * V, SSM_F32, dpw[c]);
      store_vec<V>(part, dim + p * V, SSM_F32, dw[c]);
      if (BIAS) store_vec<V>(part, 2 * dim + p * V, SSM_F32, dpb[BIAS ? c : 0]), store_vec<V>(part, 3 * dim + p * V, SSM_F32, db[BIAS ? c : 0]);
    }
  }
}

// Columns' sums over all runs (y = 0 .. 3), and over the runs that share a gate's rows (y = 4 + sequence)
struct FoldArgs {
  const float* partial;
  void *dpost_weight, *dweight, *dpost_bias, *dbias, *dgate;  // the biases' and the gate's nullable
  int per, runs, unit, units;  // rows of a run; runs; rows that share a gate, how often
  int dim, param_dtype, gate_dtype;
};
__global__ void __launch_bounds__(256) block_norm_fold_kernel(const __grid_constant__ FoldArgs f) {
  __shared__ float sums[8][32];
  const int lane = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int col = blockIdx.x * 32 + lane;
  for (int what = blockIdx.y; what < 4 + f.units; what += gridDim.y) {
    int from = 0, to = f.runs, begin = 0;
    bool here = what < 2 || (what == 2 && f.dpost_bias) || (what == 3 && f.dbias);
    if (what >= 4) {
      begin = (what - 4) * f.unit;
      from = begin / f.per, to = (begin + f.unit - 1) / f.per + 1;
      here = to - from > 1;  // else written by its run
    }
    float t = 0.f;
    if (here && col < f.dim) {
      for (int r = from + slice; r < to; r += 8) {
        const int slot = what < 4 ? what : begin < r * f.per ? 4 : 5;
        t += f.partial[((int64_t)r * kSlots + slot) * f.dim + col];
      }
    }
    __syncthreads();
    sums[slice][lane] = t;
    __syncthreads();
    if (here && slice == 0 && col < f.dim) {
#pragma unroll
      for (int w = 1; w < 8; ++w) t += sums[w][lane];
      if (what == 0) store_dyn(f.dpost_weight, col, f.param_dtype, t);
      else if (what == 1) store_dyn(f.dweight, col, f.param_dtype, t);
      else if (what == 2) store_dyn(f.dpost_bias, col, f.param_dtype, t);
      else if (what == 3) store_dyn(f.dbias, col, f.param_dtype, t);
      else store_dyn(f.dgate, (int64_t)(what - 4) * f.dim + col, f.gate_dtype, t);
    }
  }
}

// runs of neighbouring rows: as many as blocks run at once, at least one row each
int64_t rows_per_run(int64_t rows, int threads) {
  const int64_t runs = std::min<int64_t>(kMaxRuns, (int64_t)sm_count() * std::max(1, 1024 / threads / 2));
  return std::max<int64_t>(1, (rows + runs - 1) / runs);
}

template <int V, int G, int MC>
int launch_fwd(const ssm_block_norm_args& a, cudaStream_t st) {
  FwdArgs f{a, (int)std::min<int64_t>(a.len, a.rows), a.residual != nullptr};
  if (!f.has_r) f.a.residual = a.x, f.a.res_dtype = a.io_dtype;
  const unsigned grid = (unsigned)a.rows;
  if (a.bias) {
    if (a.gate_kind) block_norm_kernel<V, G, MC, true, true><<<grid, G, 0, st>>>(f);
    else block_norm_kernel<V, G, MC, true, false><<<grid, G, 0, st>>>(f);
  } else {
    if (a.gate_kind) block_norm_kernel<V, G, MC, false, true><<<grid, G, 0, st>>>(f);
    else block_norm_kernel<V, G, MC, false, false><<<grid, G, 0, st>>>(f);
  }
  return launch_status("block_norm_kernel");
}
template <int V, int G, int MC, bool BIAS, bool GATE>
int launch_bwd2(const ssm_block_norm_bwd_args& g, cudaStream_t st) {
  const ssm_block_norm_args& a = g.fwd;
  const int per = (int)rows_per_run(a.rows, G), runs = (int)((a.rows + per - 1) / per);
  BwdArgs b{};
  b.g = g, b.rows = (int)a.rows, b.per = per, b.len = (int)std::min<int64_t>(a.len, a.rows);
  b.unit = a.gate_kind == kSequence ? b.len : b.rows;
  b.has_r = a.residual != nullptr, b.has_d = g.dresidual_out != nullptr, b.d_dtype = b.has_d ? a.resout_dtype : a.io_dtype;
  if (!b.has_r) b.g.fwd.residual = a.x, b.g.fwd.res_dtype = a.io_dtype;
  if (!b.has_d) b.g.dresidual_out = g.dy;
  constexpr int kRow = 4 * RowRing<V, G, MC>::kBytes;
  static_assert(kRow <= 200 * 1024, "a row's pieces lie in shared memory");
  b.stages = 2 * kRow <= 200 * 1024 ? 2 : 1;
  const int smem = b.stages * kRow;
  auto kern = block_norm_bwd_kernel<V, G, MC, BIAS, GATE>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  kern<<<runs, G, smem, st>>>(b);
  if (const int rc = launch_status("block_norm_bwd_kernel")) return rc;
  FoldArgs f{};
  f.partial = g.partial, f.dpost_weight = g.dpost_weight, f.dweight = g.dweight, f.dpost_bias = g.dpost_bias, f.dbias = g.dbias, f.dgate = g.dgate;
  f.per = per, f.runs = runs, f.dim = a.dim, f.param_dtype = a.param_dtype, f.gate_dtype = a.gate_dtype, f.unit = b.unit, f.units = a.gate_kind == kChannel || a.gate_kind == kSequence ? b.rows / b.unit : 0;
  block_norm_fold_kernel<<<dim3((a.dim + 31) / 32, std::min(4 + f.units, 1024)), 256, 0, st>>>(f);
  return launch_status("block_norm_fold_kernel");
}
template <int V, int G, int MC>
int launch_bwd(const ssm_block_norm_bwd_args& g, cudaStream_t st) {
  const bool bias = g.fwd.bias, gate = g.fwd.gate_kind;
  if (bias) return gate ? launch_bwd2<V, G, MC, true, true>(g, st) : launch_bwd2<V, G, MC, true, false>(g, st);
  return gate ? launch_bwd2<V, G, MC, false, true>(g, st) : launch_bwd2<V, G, MC, false, false>(g, st);
}

constexpr int kMaxDim = 8192;

// threads and pieces of a row: n pieces of V elements
#define SSM_ROW_CASES(WHAT, V, n, ...)                    \
  if ((n) <= 32) return WHAT<V, 32, 1>(__VA_ARGS__);      \
  if ((n) <= 64) return WHAT<V, 32, 2>(__VA_ARGS__);      \
  if ((n) <= 128) return WHAT<V, 64, 2>(__VA_ARGS__);     \
  if ((n) <= 256) return WHAT<V, 128, 2>(__VA_ARGS__);    \
  if ((n) <= 384) return WHAT<V, 128, 3>(__VA_ARGS__);    \
  if ((n) <= 512) return WHAT<V, 256, 2>(__VA_ARGS__);    \
  if ((n) <= 768) return WHAT<V, 256, 3>(__VA_ARGS__);    \
  if ((n) <= 1024) return WHAT<V, 512, 2>(__VA_ARGS__);   \
  if ((n) <= 2048) return WHAT<V, 512, 4>(__VA_ARGS__);

int dispatch_fwd(const ssm_block_norm_args& a, bool wide, cudaStream_t st) {
  if (wide && a.io_dtype != SSM_F32 && a.dim % 8 == 0) {
    SSM_ROW_CASES(launch_fwd, 8, a.dim / 8, a, st)
  }
  if (wide && a.dim % 4 == 0) {
    SSM_ROW_CASES(launch_fwd, 4, a.dim / 4, a, st)
  }
  SSM_ROW_CASES(launch_fwd, 1, a.dim, a, st)
  return launch_fwd<1, 512, kMaxDim / 512>(a, st);
}
// four elements to a piece also in 16 bits: the sums of a thread's columns stay in registers
int dispatch_bwd(const ssm_block_norm_bwd_args& g, bool wide, cudaStream_t st) {
  if (wide && g.fwd.dim % 4 == 0) {
    SSM_ROW_CASES(launch_bwd, 4, g.fwd.dim / 4, g, st)
  }
  SSM_ROW_CASES(launch_bwd, 1, g.fwd.dim, g, st)
  return launch_bwd<1, 512, kMaxDim / 512>(g, st);
}

int check(const ssm_block_norm_args& a) {
  SSM_REQUIRE(a.rows >= 0 && a.dim >= 1 && a.len >= 1, SSM_ERR_SHAPE, "fused_block_norm: bad shape");
  SSM_REQUIRE(a.dim <= kMaxDim, SSM_ERR_TOO_LARGE, "fused_block_norm: more than 8192 columns");
  SSM_REQUIRE(a.rows < ((int64_t)1 << 31), SSM_ERR_TOO_LARGE, "fused_block_norm: 2^31 rows or more");
  SSM_REQUIRE(valid_dtype(a.io_dtype) && valid_dtype(a.res_dtype) && valid_dtype(a.resout_dtype) && valid_dtype(a.param_dtype) && valid_dtype(a.gate_dtype), SSM_ERR_DTYPE,
              "fused_block_norm: unknown dtype");
  SSM_REQUIRE(a.gate_kind >= kNone && a.gate_kind <= kToken && (a.gate_kind != kSequence || a.rows % a.len == 0), SSM_ERR_SHAPE, "fused_block_norm: bad gate");
  SSM_REQUIRE(a.rows == 0 || (a.x && a.post_weight && a.weight && (a.gate || !a.gate_kind)), SSM_ERR_NULL, "fused_block_norm: NULL pointer");
  SSM_REQUIRE(!a.bias == !a.post_bias, SSM_ERR_NULL, "fused_block_norm: both biases or neither");
  SSM_REQUIRE(aligned_to(a.x, dtype_size(a.io_dtype)) && aligned_to(a.residual, dtype_size(a.res_dtype)) && aligned_to({a.post_weight, a.weight, a.post_bias, a.bias}, dtype_size(a.param_dtype)) &&
                  aligned_to(a.gate, dtype_size(a.gate_dtype)) && aligned_to(a.y, dtype_size(a.io_dtype)) && aligned_to(a.residual_out, dtype_size(a.resout_dtype)) && aligned_to(a.stats, 16),
              SSM_ERR_ALIGN, "fused_block_norm: misaligned pointer");
  return SSM_OK;
}
bool wide_reads(const ssm_block_norm_args& a) { return aligned_to({a.x, a.residual, a.post_weight, a.weight, a.post_bias, a.bias, a.gate, a.y, a.residual_out}, 16); }

}  // namespace
}  // namespace ssmb

using namespace ssmb;

extern "C" int ssm_block_norm_fwd(const ssm_block_norm_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "fused_block_norm: NULL arguments");
  if (const int rc = check(*args)) return rc;
  if (args->rows == 0) return SSM_OK;
  SSM_REQUIRE(args->y && args->residual_out, SSM_ERR_NULL, "fused_block_norm: NULL output");
  return dispatch_fwd(*args, wide_reads(*args), reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int64_t ssm_block_norm_bwd_scratch_floats(int64_t rows, int32_t dim) { return std::min<int64_t>(std::max<int64_t>(rows, 1), kMaxRuns) * kSlots * (int64_t)dim; }

extern "C" int ssm_block_norm_bwd(const ssm_block_norm_bwd_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "fused_block_norm: NULL arguments");
  if (const int rc = check(args->fwd)) return rc;
  if (args->fwd.rows == 0) return SSM_OK;
  const ssm_block_norm_args& a = args->fwd;
  SSM_REQUIRE(a.stats && args->dy && args->dx && args->dpost_weight && args->dweight && args->partial && (args->dgate || !a.gate_kind) && (!args->dresidual || a.residual), SSM_ERR_NULL, "fused_block_norm backward: NULL pointer");
  SSM_REQUIRE(aligned_to({args->dy, args->dx}, dtype_size(a.io_dtype)) && aligned_to(args->dresidual_out, dtype_size(a.resout_dtype)) && aligned_to(args->dresidual, dtype_size(a.res_dtype)) &&
                  aligned_to({args->dpost_weight, args->dweight, args->dpost_bias, args->dbias}, dtype_size(a.param_dtype)) && aligned_to(args->dgate, dtype_size(a.gate_dtype)) &&
                  aligned_to(args->partial, 16),
              SSM_ERR_ALIGN, "fused_block_norm backward: misaligned pointer");
  const bool wide = wide_reads(a) && aligned_to({args->dy, args->dx, args->dresidual_out, args->dresidual, args->dgate}, 16);
  return dispatch_bwd(*args, wide, reinterpret_cast<cudaStream_t>(stream));
}
