// The norms after and before a block, fused with the block's gate, its residual scale and the residual add; forward and backward.
//
//   n = h1 w1 + b1,  h1 = (x - m1) s1;   r = residual + scale gate n;   y = h2 w2 + b2,  h2 = (r - m2) s2
//
// with m the mean of a row (0 for RMSNorm) and s = 1 / sqrt(mean (x - m)^2 + eps).  Backward, with means over a row, from dy and dr (the gradient of r):
//
//   g2 = w2 dy;   dr' = dr + s2 (g2 - [mean g2] - h2 mean(g2 h2));   dn = scale gate dr';   dgate = scale dr' n
//   g1 = w1 dn;   dx = s1 (g1 - [mean g1] - h1 mean(g1 h1));   dresidual = dr';   dw1 = sum dn h1, db1 = sum dn, dw2 = sum dy h2, db2 = sum dy
//
// Bound: HBM, 12 bytes an element forward and 18 back with 16-bit activations and a 32-bit stream.  A row is owned by 32 to 512 threads and lies in their
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
constexpr int kMaxDim = 8192;

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

// sums of two values over a block, or of the second alone.  A warp's sums meet in shared memory, where each warp adds them up by shuffles (every thread reading all of them: 25 of the
// backward pass's 81 instructions an element); two rows of scratch in turn, so that a sum takes one barrier.
template <bool BOTH>
__device__ __forceinline__ void allsum(float& a, float& b, float2 (*scratch)[16], int& turn) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    if (BOTH) a += __shfl_xor_sync(0xffffffffu, a, off);
    b += __shfl_xor_sync(0xffffffffu, b, off);
  }
  const int warps = blockDim.x / 32, lane = threadIdx.x % 32;
  if (warps > 1) {
    if (lane == 0) scratch[turn][threadIdx.x / 32] = make_float2(a, b);
    __syncthreads();
    const float2 v = scratch[turn][lane % 16];
    a = lane % 16 < warps ? v.x : 0.f, b = lane % 16 < warps ? v.y : 0.f;
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) {
      if (BOTH) a += __shfl_xor_sync(0xffffffffu, a, off);
      b += __shfl_xor_sync(0xffffffffu, b, off);
    }
    turn ^= 1;
  }
}
__device__ __forceinline__ void allsum2(float& a, float& b, float2 (*scratch)[16], int& turn) { allsum<true>(a, b, scratch, turn); }

enum Gate { kNone = 0, kChannel = 1, kSequence = 2, kToken = 3 };

// No load of these kernels depends on a condition for its address: what a call does not have (a residual, an incoming gradient) points at what it has, with a flag to leave it
// out, and in the forward pass a thread beyond the row's end reads the row's last piece.

// Types known at compile time: 0 none; 1 bf16, 2 fp16, 3 fp32 activations, gate and parameters, with a residual stream of fp32, in and out
template <int TYPES>
__device__ __forceinline__ int io_type(int dtype) {
  return TYPES == 1 ? SSM_BF16 : TYPES == 2 ? SSM_F16 : TYPES == 3 ? SSM_F32 : dtype;
}
template <int TYPES>
__device__ __forceinline__ int stream_type(int dtype) {
  return TYPES ? SSM_F32 : dtype;
}

// Mean and 1 / std of a row; V elements to a piece, MC pieces to a thread: piece c of thread t is c blockDim + t, and there are n of them
template <int V, int MC>
__device__ __forceinline__ void row_stats(const float (&f)[MC][V], int n, float inv, bool rms, float eps, float2 (*scratch)[16], int& turn, float& mean, float& rstd) {
  float t = 0.f, q = 0.f;
  mean = 0.f;
  if (!rms) {
#pragma unroll
    for (int c = 0; c < MC; ++c) {
#pragma unroll
      for (int k = 0; k < V; ++k) t += (int)(c * blockDim.x + threadIdx.x) < n ? f[c][k] : 0.f;
    }
    allsum<false>(q, t, scratch, turn);
    mean = t * inv, q = 0.f;
  }
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const bool live = (int)(c * blockDim.x + threadIdx.x) < n;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = live ? f[c][k] - mean : 0.f;
      q = fmaf(d, d, q);
    }
  }
  t = 0.f;
  allsum<false>(t, q, scratch, turn);
  rstd = rsqrtf(q * inv + eps);
}

struct FwdArgs {
  ssm_block_norm_args a;
  int len, has_r;  // rows of a sequence; the residual is one
};

template <int V, int MC, bool BIAS, bool GATE, int TYPES>
__global__ void __launch_bounds__(512) block_norm_kernel(const __grid_constant__ FwdArgs args) {
  const ssm_block_norm_args& a = args.a;
  __shared__ float2 scratch[2][16];
  int turn = 0;
  const int io = io_type<TYPES>(a.io_dtype), rt = stream_type<TYPES>(a.res_dtype), ot = stream_type<TYPES>(a.resout_dtype), pt = io_type<TYPES>(a.param_dtype), gt = io_type<TYPES>(a.gate_dtype);
  const bool has_r = TYPES || args.has_r;
  const int tid = threadIdx.x, threads = blockDim.x, dim = a.dim, n = dim / V, row = blockIdx.x;
  const float inv = 1.f / (float)dim;
  const int64_t at = (int64_t)row * dim, gate_at = a.gate_kind == kToken ? at : a.gate_kind == kSequence ? (int64_t)(row / args.len) * dim : 0;
  float v[MC][V];
  Raw<V> rx[MC], rr[MC];
  int col[MC];
#pragma unroll
  for (int c = 0; c < MC; ++c) col[c] = min(c * threads + tid, n - 1) * V;
#pragma unroll
  for (int c = 0; c < MC; ++c) issue<V>(a.x, at + col[c], io, rx[c]);
#pragma unroll
  for (int c = 0; c < MC; ++c) issue<V>(a.residual, at + col[c], rt, rr[c]);
#pragma unroll
  for (int c = 0; c < MC; ++c) convert<V>(rx[c], io, v[c]);
  float m1, s1, m2, s2;
  row_stats<V, MC>(v, n, inv, a.is_rms, a.post_eps, scratch, turn, m1, s1);
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    float b[V], ga[V], w[V], r[V];
    load_vec<V>(a.post_weight, col[c], pt, w);
    if (BIAS) load_vec<V>(a.post_bias, col[c], pt, b);
    if (GATE) load_vec<V>(a.gate, gate_at + col[c], gt, ga);
    convert<V>(rr[c], rt, r);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float h = (v[c][k] - m1) * s1, y = BIAS ? fmaf(h, w[k], b[k]) : h * w[k], f = GATE ? a.scale * ga[k] : a.scale;
      v[c][k] = has_r ? fmaf(f, y, r[k]) : f * y;
    }
    if (c * threads + tid < n) store_vec<V>(a.residual_out, at + col[c], ot, v[c]);
  }
  row_stats<V, MC>(v, n, inv, a.is_rms, a.eps, scratch, turn, m2, s2);
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    float w[V], b[V], y[V];
    load_vec<V>(a.weight, col[c], pt, w);
    if (BIAS) load_vec<V>(a.bias, col[c], pt, b);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float h = (v[c][k] - m2) * s2;
      y[k] = BIAS ? fmaf(h, w[k], b[k]) : h * w[k];
    }
    if (c * threads + tid < n) store_vec<V>(a.y, at + col[c], io, y);
  }
  if (a.stats && tid == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(m1, s1, m2, s2);
}

// where a run of rows leaves its sums: [run][which][dim]; which: dpost_weight, dweight, dpost_bias, dbias, dgate (of its first sequence, of its last)
constexpr int kSlots = 6;

// The backward pass of a run of rows.  V elements to a piece, piece c of thread t is c blockDim + t.  A row's chain is long (loads, two rounds of sums, stores), so the next row is on its way
// into shared memory while this one is worked on: each thread copies its own pieces (asynchronous copies, no barrier) and reads them there again where it needs them,
// which leaves the registers to the sums of its columns.  The parameters, and a gate per channel or sequence, lie beside them in fp32, loaded once (a sequence).
// pieces of four
__device__ __forceinline__ void copy_piece(uint32_t dst, const void* base, int64_t i, int dtype) {
  if (dtype == SSM_F32) {
    const float* src = reinterpret_cast<const float*>(base) + i;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
  } else {
    const uint16_t* src = reinterpret_cast<const uint16_t*>(base) + i;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(dst), "l"(src) : "memory");
  }
}
// single elements of a row, a thread's MC of them: 32 bits by an asynchronous copy, 16 bits through registers, all loads ahead of the first store (one after another, 1519 rows
// of 2502 bf16 columns with a gate per token: backward 112 us, so 48)
template <int MC>
struct Loose {
  uint16_t v[MC];
  __device__ __forceinline__ void load(uint32_t dst, const void* base, int64_t at, int dtype, int n) {
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * (int)blockDim.x + (int)threadIdx.x;
      v[c] = 0;
      if (p < n) {
        if (dtype == SSM_F32) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst + p * 4), "l"(reinterpret_cast<const float*>(base) + at + p) : "memory");
        else v[c] = reinterpret_cast<const uint16_t*>(base)[at + p];
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t dst, int dtype, int n) const {
    if (dtype == SSM_F32) return;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * (int)blockDim.x + (int)threadIdx.x;
      if (p < n) asm volatile("st.shared.b16 [%0], %1;\n" ::"r"(dst + p * 2), "h"(v[c]) : "memory");
    }
  }
};
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
    float hi;
    if (dtype == SSM_F32) f[0] = *reinterpret_cast<const float*>(at);
    else halves(*reinterpret_cast<const uint16_t*>(at), dtype, f[0], hi);
  }
}

struct BwdArgs {
  ssm_block_norm_bwd_args g;
  int rows, per, len, unit;  // rows in all, of a run, of a sequence, that share a gate
  int stages, has_r, has_d, d_dtype;  // rows in shared memory; the residual is one, and the gradient that came through it
  int o_dy, o_r, o_d, o_g, stage;     // places in a row's part of shared memory, its size; parameters behind the rows
};

template <int V, int MC, bool BIAS, int GATE, int TYPES>  // GATE: 0 none, 1 per channel or sequence, 2 per token
__global__ void __launch_bounds__(512) block_norm_bwd_kernel(const __grid_constant__ BwdArgs args) {
  const ssm_block_norm_bwd_args& g = args.g;
  const ssm_block_norm_args& a = g.fwd;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 scratch[2][16];
  constexpr int kB = BIAS ? MC : 1, kG = GATE == 1 ? MC : 1;
  constexpr bool kCached = MC * V <= 8;  // the parameters of rows of up to 4096 columns have room in shared memory
  const int io = io_type<TYPES>(a.io_dtype), rt = stream_type<TYPES>(a.res_dtype), dt = stream_type<TYPES>(args.d_dtype), pt = io_type<TYPES>(a.param_dtype), gt = io_type<TYPES>(a.gate_dtype);
  const int ie = io == SSM_F32 ? 4 : 2, re = rt == SSM_F32 ? 4 : 2, de = dt == SSM_F32 ? 4 : 2, ge = gt == SSM_F32 ? 4 : 2;
  const bool has_r = TYPES || args.has_r, has_d = TYPES || args.has_d, two = args.stages == 2;
  int turn = 0;
  const int tid = threadIdx.x, threads = blockDim.x, dim = a.dim, n = dim / V;
  const float inv = 1.f / (float)dim;
  const int first = blockIdx.x * args.per, last = min(args.rows, first + args.per);
  float dpw[MC][V], dw[MC][V], dpb[kB][V], db[kB][V], dg[kG][V];
#pragma unroll
  for (int c = 0; c < MC; ++c) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      dpw[c][k] = dw[c][k] = 0.f;
      if (BIAS) dpb[BIAS ? c : 0][k] = db[BIAS ? c : 0][k] = 0.f;
      if (GATE == 1) dg[GATE == 1 ? c : 0][k] = 0.f;
    }
  }
  static_assert(V == 1, "pieces of four have a kernel of their own");
  float* const part = g.partial + (int64_t)blockIdx.x * kSlots * dim;
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring);
  // post_weight, weight, post_bias, gate times scale: [which][dim], a thread's own pieces
  float* const par = reinterpret_cast<float*>(ring + args.stages * args.stage);
  const int dim4 = (dim + 3) / 4 * 4;
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int p = c * threads + tid;
    if (kCached && p < n) {
      float w[V];
      load_vec<V>(a.post_weight, p * V, pt, w);
#pragma unroll
      for (int k = 0; k < V; ++k) par[p * V + k] = w[k];
      load_vec<V>(a.weight, p * V, pt, w);
#pragma unroll
      for (int k = 0; k < V; ++k) par[dim4 + p * V + k] = w[k];
      if (BIAS) {
        load_vec<V>(a.post_bias, p * V, pt, w);
#pragma unroll
        for (int k = 0; k < V; ++k) par[2 * dim4 + p * V + k] = w[k];
      }
    }
  }
  auto set_out = [&](int row, int into) {
    const int64_t at = (int64_t)row * dim;
    const uint32_t to = ring0 + into * args.stage;
    Loose<MC> x, dy, r, d, gate;
    x.load(to, a.x, at, io, n), dy.load(to + args.o_dy, g.dy, at, io, n), r.load(to + args.o_r, a.residual, at, rt, n), d.load(to + args.o_d, g.dresidual_out, at, dt, n);
    if (GATE == 2) gate.load(to + args.o_g, a.gate, at, gt, n);
    x.store(to, io, n), dy.store(to + args.o_dy, io, n), r.store(to + args.o_r, rt, n), d.store(to + args.o_d, dt, n);
    if (GATE == 2) gate.store(to + args.o_g, gt, n);
  };

  int stage = 0, gate_of = -1;
  if (two && first < last) set_out(first, 0);
  asm volatile("cp.async.commit_group;\n" ::: "memory");
  for (int row = first; row < last; ++row) {
    if (two) {
      if (row + 1 < last) set_out(row + 1, stage ^ 1);
      asm volatile("cp.async.commit_group;\n" ::: "memory");
      asm volatile("cp.async.wait_group 1;\n" ::: "memory");
    } else {
      set_out(row, 0);
      asm volatile("cp.async.commit_group;\n" ::: "memory");
      asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    }
    const int64_t at = (int64_t)row * dim;
    const unsigned char* const mine = ring + stage * args.stage;
    const float4 stats = reinterpret_cast<const float4*>(a.stats)[row];
    const float m1 = stats.x, s1 = stats.y, m2 = stats.z, s2 = stats.w;
    const int64_t gate_at = GATE == 1 ? (int64_t)(row / args.unit) * dim : 0;
    if (GATE == 1 && kCached) {
      const int seq = row / args.unit;
      if (seq != gate_of) {  // a thread's own pieces: no barrier
#pragma unroll
        for (int c = 0; c < MC; ++c) {
          const int p = c * threads + tid;
          if (p < n) {
            float w[V];
            load_vec<V>(a.gate, (int64_t)seq * dim + p * V, gt, w);
#pragma unroll
            for (int k = 0; k < V; ++k) par[3 * dim4 + p * V + k] = a.scale * w[k];
          }
        }
        gate_of = seq;
      }
    }
    auto param = [&](int which, const void* from, int p, float (&w)[V]) {
      if (kCached) read_piece<V>(reinterpret_cast<const unsigned char*>(par + which * dim4 + p * V), SSM_F32, w);
      else load_vec<V>(from, p * V, pt, w);
    };
    // h, n and the factor of n in r, for a piece
    auto branch = [&](int p, float (&h)[V], float (&nn)[V], float (&ga)[V], float (&w)[V]) {
      float x[V], b[V];
      read_piece<V>(mine + p * V * ie, io, x);
      param(0, a.post_weight, p, w);
      if (BIAS) param(2, a.post_bias, p, b);
      if (GATE == 1) {
        if (kCached) read_piece<V>(reinterpret_cast<const unsigned char*>(par + 3 * dim4 + p * V), SSM_F32, ga);
        else load_vec<V>(a.gate, gate_at + p * V, gt, ga);
      }
      if (GATE == 2) read_piece<V>(mine + args.o_g + p * V * ge, gt, ga);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        h[k] = (x[k] - m1) * s1;
        nn[k] = BIAS ? fmaf(h[k], w[k], b[k]) : h[k] * w[k];
        ga[k] = GATE == 2 || (GATE == 1 && !kCached) ? a.scale * ga[k] : GATE == 1 ? ga[k] : a.scale;
      }
    };
    float h2[MC][V], d[MC][V];
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * threads + tid;
      if (p < n) {
        float h[V], b[V], ga[V], w[V], r[V], dy[V];
        branch(p, h, b, ga, w);
        read_piece<V>(mine + args.o_dy + p * V * ie, io, dy);
        read_piece<V>(mine + args.o_r + p * V * re, rt, r);
        param(1, a.weight, p, w);
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
    allsum2(sum0, sum1, scratch, turn);
    const float c2 = a.is_rms ? 0.f : sum0 * inv, e2 = sum1 * inv;
    sum0 = sum1 = 0.f;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * threads + tid;
      if (p < n) {
        float h[V], b[V], ga[V], w[V], o[V], gg[V];
        branch(p, h, b, ga, w);
        read_piece<V>(mine + args.o_d + p * V * de, dt, o);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float t = s2 * (d[c][k] - c2 - h2[c][k] * e2);
          if (has_d) t += o[k];
          o[k] = t;
          gg[k] = a.scale * t * b[k];
          if (GATE == 1) dg[GATE == 1 ? c : 0][k] += gg[k];
          const float dn = ga[k] * t;
          dpw[c][k] = fmaf(dn, h[k], dpw[c][k]);
          if (BIAS) dpb[BIAS ? c : 0][k] += dn;
          d[c][k] = w[k] * dn;
          sum0 += d[c][k], sum1 = fmaf(d[c][k], h[k], sum1);
        }
        if (TYPES || g.dresidual) store_vec<V>(g.dresidual, at + p * V, rt, o);
        if (GATE == 2) store_vec<V>(g.dgate, at + p * V, gt, gg);
      }
    }
    allsum2(sum0, sum1, scratch, turn);
    const float c1 = a.is_rms ? 0.f : sum0 * inv, e1 = sum1 * inv;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * threads + tid;
      if (p < n) {
        float x[V];
        read_piece<V>(mine + p * V * ie, io, x);
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = s1 * (d[c][k] - c1 - (x[k] - m1) * s1 * e1);
        store_vec<V>(g.dx, at + p * V, io, x);
      }
    }
    if (GATE == 1 && (row + 1 == last || (row + 1) % args.unit == 0)) {  // the gate's rows end here, or the run does
      const int seq = row / args.unit, begin = seq * args.unit, end = begin + args.unit;
#pragma unroll
      for (int c = 0; c < MC; ++c) {
        const int p = c * threads + tid;
        if (p < n) {
          if (begin >= first && end <= last) store_vec<V>(g.dgate, (int64_t)seq * dim + p * V, gt, dg[GATE == 1 ? c : 0]);
          else if (begin < first) store_vec<V>(part, 4 * dim + p * V, SSM_F32, dg[GATE == 1 ? c : 0]);
          else store_vec<V>(part, 5 * dim + p * V, SSM_F32, dg[GATE == 1 ? c : 0]);
#pragma unroll
          for (int k = 0; k < V; ++k) dg[GATE == 1 ? c : 0][k] = 0.f;
        }
      }
    }
    stage = two ? stage ^ 1 : 0;
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int p = c * threads + tid;
    if (p < n) {
      store_vec<V>(part, p * V, SSM_F32, dpw[c]);
      store_vec<V>(part, dim + p * V, SSM_F32, dw[c]);
      if (BIAS) store_vec<V>(part, 2 * dim + p * V, SSM_F32, dpb[BIAS ? c : 0]), store_vec<V>(part, 3 * dim + p * V, SSM_F32, db[BIAS ? c : 0]);
    }
  }
}

// The same for pieces of four, in pairs of fp32 (one instruction for two).  THREADS: at most; rows of up to 2560 columns, all that 320 threads hold, leave room for two blocks to an SM.  42M elements
// with a gate per channel, us: 2560 columns 138, with up to 512 threads and one block 185; 2048: 146 and 144; 1024: 136 and 140; beyond, with one block: 2564 columns 197, 2816 174, 4096 149.
// 16384 rows of 2560 bf16 columns: scalar arithmetic, 91 instructions an element, one block to an SM: 254 us.
struct Quad {
  float2 a, b;
};
__device__ __forceinline__ Quad quad(float x) { return {make_float2(x, x), make_float2(x, x)}; }
__device__ __forceinline__ Quad fma4(const Quad& x, const Quad& y, const Quad& z) { return {__ffma2_rn(x.a, y.a, z.a), __ffma2_rn(x.b, y.b, z.b)}; }
__device__ __forceinline__ Quad mul4(const Quad& x, const Quad& y) { return {__fmul2_rn(x.a, y.a), __fmul2_rn(x.b, y.b)}; }
__device__ __forceinline__ Quad add4(const Quad& x, const Quad& y) { return {__fadd2_rn(x.a, y.a), __fadd2_rn(x.b, y.b)}; }
__device__ __forceinline__ float sum4(const Quad& x) { return (x.a.x + x.a.y) + (x.b.x + x.b.y); }
__device__ __forceinline__ Quad read_quad(const unsigned char* at, int dtype) {
  Quad q;
  if (dtype == SSM_F32) {
    const float4 v = *reinterpret_cast<const float4*>(at);
    q.a = make_float2(v.x, v.y), q.b = make_float2(v.z, v.w);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    halves(v.x, dtype, q.a.x, q.a.y), halves(v.y, dtype, q.b.x, q.b.y);
  }
  return q;
}
__device__ __forceinline__ Quad load_quad(const void* base, int64_t i, int dtype) {
  float f[4];
  load_param_vec<4>(base, i, dtype, f);
  return {make_float2(f[0], f[1]), make_float2(f[2], f[3])};
}
__device__ __forceinline__ void store_quad(void* base, int64_t i, int dtype, const Quad& q) {
  const float f[4] = {q.a.x, q.a.y, q.b.x, q.b.y};
  store_vec<4>(base, i, dtype, f);
}

template <int THREADS, int MC, bool BIAS, int GATE, int TYPES>  // GATE: 0 none, 1 per channel or sequence, 2 per token
__global__ void __launch_bounds__(THREADS, THREADS <= 320 ? 2 : 1) block_norm_bwd4_kernel(const __grid_constant__ BwdArgs args) {
  const ssm_block_norm_bwd_args& g = args.g;
  const ssm_block_norm_args& a = g.fwd;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 scratch[2][16];
  constexpr int kB = BIAS ? MC : 1, kG = GATE == 1 ? MC : 1;
  constexpr bool kCached = MC <= 2;  // the parameters of rows of up to 4096 columns have room in shared memory
  const int io = io_type<TYPES>(a.io_dtype), rt = stream_type<TYPES>(a.res_dtype), dt = stream_type<TYPES>(args.d_dtype), pt = io_type<TYPES>(a.param_dtype), gt = io_type<TYPES>(a.gate_dtype);
  const int ie = io == SSM_F32 ? 16 : 8, re = rt == SSM_F32 ? 16 : 8, de = dt == SSM_F32 ? 16 : 8, ge = gt == SSM_F32 ? 16 : 8;
  const bool has_r = TYPES || args.has_r, has_d = TYPES || args.has_d, two = args.stages == 2, rms = a.is_rms;
  int turn = 0;
  const int tid = threadIdx.x, threads = blockDim.x, dim = a.dim, n = dim / 4;
  const float inv = 1.f / (float)dim;
  const int first = blockIdx.x * args.per, last = min(args.rows, first + args.per);
  Quad dpw[MC], dw[MC], dpb[kB], db[kB], dg[kG];
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    dpw[c] = dw[c] = quad(0.f);
    if (BIAS) dpb[BIAS ? c : 0] = db[BIAS ? c : 0] = quad(0.f);
    if (GATE == 1) dg[GATE == 1 ? c : 0] = quad(0.f);
  }
  float* const part = g.partial + (int64_t)blockIdx.x * kSlots * dim;
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring);
  unsigned char* const par = ring + args.stages * args.stage;  // post_weight, weight, post_bias, gate times scale: [which][dim] fp32, a thread's own pieces
  const Quad scale4 = quad(a.scale);
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int p = c * threads + tid;
    if (kCached && p < n) {
      Quad w = load_quad(a.post_weight, p * 4, pt);
      *reinterpret_cast<float4*>(par + p * 16) = make_float4(w.a.x, w.a.y, w.b.x, w.b.y);
      w = load_quad(a.weight, p * 4, pt);
      *reinterpret_cast<float4*>(par + (n + p) * 16) = make_float4(w.a.x, w.a.y, w.b.x, w.b.y);
      if (BIAS) {
        w = load_quad(a.post_bias, p * 4, pt);
        *reinterpret_cast<float4*>(par + (2 * n + p) * 16) = make_float4(w.a.x, w.a.y, w.b.x, w.b.y);
      }
    }
  }
  auto set_out = [&](int row, int into) {
    const int64_t at = (int64_t)row * dim;
    const uint32_t to = ring0 + into * args.stage;
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * threads + tid;
      if (p < n) {
        copy_piece(to + p * ie, a.x, at + p * 4, io);
        copy_piece(to + args.o_dy + p * ie, g.dy, at + p * 4, io);
        copy_piece(to + args.o_r + p * re, a.residual, at + p * 4, rt);
        copy_piece(to + args.o_d + p * de, g.dresidual_out, at + p * 4, dt);
        if (GATE == 2) copy_piece(to + args.o_g + p * ge, a.gate, at + p * 4, gt);
      }
    }
  };

  int stage = 0, gate_of = -1;
  if (two && first < last) set_out(first, 0);
  asm volatile("cp.async.commit_group;\n" ::: "memory");
  float4 stats = first < last ? __ldg(reinterpret_cast<const float4*>(a.stats) + first) : make_float4(0.f, 0.f, 0.f, 0.f);
  for (int row = first; row < last; ++row) {
    const float4 now = stats;
    if (row + 1 < last) stats = __ldg(reinterpret_cast<const float4*>(a.stats) + row + 1);
    if (two) {
      if (row + 1 < last) set_out(row + 1, stage ^ 1);
      asm volatile("cp.async.commit_group;\n" ::: "memory");
      asm volatile("cp.async.wait_group 1;\n" ::: "memory");
    } else {
      set_out(row, 0);
      asm volatile("cp.async.commit_group;\n" ::: "memory");
      asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    }
    const int64_t at = (int64_t)row * dim;
    const unsigned char* const mine = ring + stage * args.stage;
    const Quad s1 = quad(now.y), o1 = quad(-now.x * now.y), s2 = quad(now.w), o2 = quad(-now.z * now.w);  // h = x s1 + o1
    const int64_t gate_at = GATE == 1 ? (int64_t)(row / args.unit) * dim : 0;
    if (GATE == 1 && kCached) {
      const int seq = row / args.unit;
      if (seq != gate_of) {  // a thread's own pieces: no barrier
#pragma unroll
        for (int c = 0; c < MC; ++c) {
          const int p = c * threads + tid;
          if (p < n) {
            const Quad w = mul4(load_quad(a.gate, gate_at + p * 4, gt), scale4);
            *reinterpret_cast<float4*>(par + (3 * n + p) * 16) = make_float4(w.a.x, w.a.y, w.b.x, w.b.y);
          }
        }
        gate_of = seq;
      }
    }
    auto param = [&](int which, const void* from, int p) { return kCached ? read_quad(par + (which * n + p) * 16, SSM_F32) : load_quad(from, p * 4, pt); };
    auto factor = [&](int p) {  // of n in r
      if (GATE == 1) return kCached ? read_quad(par + (3 * n + p) * 16, SSM_F32) : mul4(load_quad(a.gate, gate_at + p * 4, gt), scale4);
      if (GATE == 2) return mul4(read_quad(mine + args.o_g + p * ge, gt), scale4);
      return scale4;
    };
    Quad h2[MC], d[MC];
    Quad sum = quad(0.f), dot = quad(0.f);
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * threads + tid;
      if (p < n) {
        const Quad h = fma4(read_quad(mine + p * ie, io), s1, o1), w1 = param(0, a.post_weight, p), y = BIAS ? fma4(h, w1, param(2, a.post_bias, p)) : mul4(h, w1);
        const Quad v = has_r ? fma4(factor(p), y, read_quad(mine + args.o_r + p * re, rt)) : mul4(factor(p), y), dy = read_quad(mine + args.o_dy + p * ie, io);
        h2[c] = fma4(v, s2, o2);
        dw[c] = fma4(dy, h2[c], dw[c]);
        if (BIAS) db[BIAS ? c : 0] = add4(db[BIAS ? c : 0], dy);
        d[c] = mul4(param(1, a.weight, p), dy);
        if (!rms) sum = add4(sum, d[c]);
        dot = fma4(d[c], h2[c], dot);
      }
    }
    float sum0 = sum4(sum), sum1 = sum4(dot);
    if (rms) allsum<false>(sum0, sum1, scratch, turn);
    else allsum<true>(sum0, sum1, scratch, turn);
    const Quad k2 = quad(-now.w * sum0 * inv), e2 = quad(-sum1 * inv);  // -s2 mean g, -mean(g h)
    sum = dot = quad(0.f);
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * threads + tid;
      if (p < n) {
        const Quad h = fma4(read_quad(mine + p * ie, io), s1, o1), w1 = param(0, a.post_weight, p), y = BIAS ? fma4(h, w1, param(2, a.post_bias, p)) : mul4(h, w1);
        Quad t = fma4(h2[c], e2, d[c]);
        t = has_d ? fma4(t, s2, read_quad(mine + args.o_d + p * de, dt)) : mul4(t, s2);
        if (!rms) t = add4(t, k2);
        if (TYPES || g.dresidual) store_quad(g.dresidual, at + p * 4, rt, t);
        if (GATE == 1) dg[GATE == 1 ? c : 0] = fma4(t, y, dg[GATE == 1 ? c : 0]);
        if (GATE == 2) store_quad(g.dgate, at + p * 4, gt, mul4(mul4(t, scale4), y));
        const Quad dn = mul4(factor(p), t);
        dpw[c] = fma4(dn, h, dpw[c]);
        if (BIAS) dpb[BIAS ? c : 0] = add4(dpb[BIAS ? c : 0], dn);
        d[c] = mul4(w1, dn);
        h2[c] = h;
        if (!rms) sum = add4(sum, d[c]);
        dot = fma4(d[c], h, dot);
      }
    }
    sum0 = sum4(sum), sum1 = sum4(dot);
    if (rms) allsum<false>(sum0, sum1, scratch, turn);
    else allsum<true>(sum0, sum1, scratch, turn);
    const Quad k1 = quad(-now.y * sum0 * inv), e1 = quad(-sum1 * inv);
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const int p = c * threads + tid;
      if (p < n) store_quad(g.dx, at + p * 4, io, rms ? mul4(fma4(h2[c], e1, d[c]), s1) : fma4(fma4(h2[c], e1, d[c]), s1, k1));
    }
    if (GATE == 1 && (row + 1 == last || (row + 1) % args.unit == 0)) {  // the gate's rows end here, or the run does
      const int seq = row / args.unit, begin = seq * args.unit, end = begin + args.unit;
#pragma unroll
      for (int c = 0; c < MC; ++c) {
        const int p = c * threads + tid;
        if (p < n) {
          const Quad v = mul4(dg[GATE == 1 ? c : 0], scale4);
          if (begin >= first && end <= last) store_quad(g.dgate, (int64_t)seq * dim + p * 4, gt, v);
          else if (begin < first) store_quad(part, 4 * dim + p * 4, SSM_F32, v);
          else store_quad(part, 5 * dim + p * 4, SSM_F32, v);
          dg[GATE == 1 ? c : 0] = quad(0.f);
        }
      }
    }
    stage = two ? stage ^ 1 : 0;
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int p = c * threads + tid;
    if (p < n) {
      store_quad(part, p * 4, SSM_F32, dpw[c]);
      store_quad(part, dim + p * 4, SSM_F32, dw[c]);
      if (BIAS) store_quad(part, 2 * dim + p * 4, SSM_F32, dpb[BIAS ? c : 0]), store_quad(part, 3 * dim + p * 4, SSM_F32, db[BIAS ? c : 0]);
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
// 32 pieces of V columns to a block, 32 slices of the runs (293 runs of 2560 columns, in the L2: 6.6 us; element by element 15, with eight slices 13)
template <int V>
__global__ void __launch_bounds__(1024) block_norm_fold_kernel(const __grid_constant__ FoldArgs f) {
  __shared__ float sums[V][32][33];
  const int lane = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int col = (blockIdx.x * 32 + lane) * V;
  for (int what = blockIdx.y; what < 4 + f.units; what += gridDim.y) {
    int from = 0, to = f.runs, begin = 0;
    bool here = what < 2 || (what == 2 && f.dpost_bias) || (what == 3 && f.dbias);
    if (what >= 4) {
      begin = (what - 4) * f.unit;
      from = begin / f.per, to = (begin + f.unit - 1) / f.per + 1;
      here = to - from > 1;  // else written by its run
    }
    if (!here) continue;  // the whole block
    float t[V];
#pragma unroll
    for (int k = 0; k < V; ++k) t[k] = 0.f;
    if (col < f.dim) {
#pragma unroll 4
      for (int r = from + slice; r < to; r += 32) {
        const int slot = what < 4 ? what : begin < r * f.per ? 4 : 5;
        float v[V];
        load_vec<V>(f.partial, ((int64_t)r * kSlots + slot) * f.dim + col, SSM_F32, v);
#pragma unroll
        for (int k = 0; k < V; ++k) t[k] += v[k];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) sums[k][slice][lane] = t[k];
    __syncthreads();
    const int c = (blockIdx.x * 32 + slice) * V;  // a warp has the slices of a piece
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float s = warp_sum(sums[k][lane][slice]);
      if (lane == 0 && c < f.dim) {
        if (what == 0) store_dyn(f.dpost_weight, c + k, f.param_dtype, s);
        else if (what == 1) store_dyn(f.dweight, c + k, f.param_dtype, s);
        else if (what == 2) store_dyn(f.dpost_bias, c + k, f.param_dtype, s);
        else if (what == 3) store_dyn(f.dbias, c + k, f.param_dtype, s);
        else store_dyn(f.dgate, (int64_t)(what - 4) * f.dim + c + k, f.gate_dtype, s);
      }
    }
  }
}

int types_of(const ssm_block_norm_args& a) {  // see io_type
  const bool same = a.param_dtype == a.io_dtype && (!a.gate_kind || a.gate_dtype == a.io_dtype), stream = a.residual && a.res_dtype == SSM_F32 && a.resout_dtype == SSM_F32;
  return !same || !stream ? 0 : a.io_dtype == SSM_BF16 ? 1 : a.io_dtype == SSM_F16 ? 2 : 3;
}
// whole warps for `n` pieces, MC each
int threads_for(int n, int mc) { return std::max(32, ((n + mc - 1) / mc + 31) / 32 * 32); }

template <int V, int MC, int TYPES>
int launch_fwd(const ssm_block_norm_args& a, cudaStream_t st) {
  FwdArgs f{a, (int)std::min<int64_t>(a.len, a.rows), a.residual != nullptr};
  if (!f.has_r) f.a.residual = a.x, f.a.res_dtype = a.io_dtype;
  const unsigned grid = (unsigned)a.rows;
  const int threads = threads_for(a.dim / V, MC);
  if (a.bias) {
    if (a.gate_kind) block_norm_kernel<V, MC, true, true, TYPES><<<grid, threads, 0, st>>>(f);
    else block_norm_kernel<V, MC, true, false, TYPES><<<grid, threads, 0, st>>>(f);
  } else {
    if (a.gate_kind) block_norm_kernel<V, MC, false, true, TYPES><<<grid, threads, 0, st>>>(f);
    else block_norm_kernel<V, MC, false, false, TYPES><<<grid, threads, 0, st>>>(f);
  }
  return launch_status("block_norm_kernel");
}
// One piece to a thread where a row is short, two up to 1024, so that all threads have work whatever the width, more only where 512 threads cannot hold the row
template <int TYPES>
int fwd_of(const ssm_block_norm_args& a, bool wide, cudaStream_t st) {
  constexpr int kWide = TYPES == 3 ? 4 : 8;
  if (TYPES && wide && a.dim % kWide == 0) {
    const int n = a.dim / kWide;
    if (n <= 64) return launch_fwd<kWide, 1, TYPES>(a, st);
    if (n <= 1024) return launch_fwd<kWide, 2, TYPES>(a, st);
    return launch_fwd<kWide, 4, TYPES>(a, st);
  }
  if (wide && a.dim % 4 == 0) return a.dim <= 4096 ? launch_fwd<4, 2, 0>(a, st) : launch_fwd<4, 4, 0>(a, st);
  return a.dim <= 1024 ? launch_fwd<1, 2, TYPES>(a, st) : a.dim <= 4096 ? launch_fwd<1, 8, TYPES>(a, st) : launch_fwd<1, 16, 0>(a, st);
}
int dispatch_fwd(const ssm_block_norm_args& a, bool wide, cudaStream_t st) {
  switch (types_of(a)) {
    case 1: return fwd_of<1>(a, wide, st);
    case 2: return fwd_of<2>(a, wide, st);
    case 3: return fwd_of<3>(a, wide, st);
    default: return fwd_of<0>(a, wide, st);
  }
}

constexpr int kRing = 200 * 1024;
template <int V, int THREADS, int MC, bool BIAS, int GATE, int TYPES>
int launch_bwd2(const ssm_block_norm_bwd_args& g, cudaStream_t st) {
  const ssm_block_norm_args& a = g.fwd;
  const int threads = threads_for(a.dim / V, MC);
  BwdArgs b{};
  b.g = g, b.rows = (int)a.rows, b.len = (int)std::min<int64_t>(a.len, a.rows);
  b.unit = a.gate_kind == kSequence ? b.len : b.rows;
  b.has_r = a.residual != nullptr, b.has_d = g.dresidual_out != nullptr, b.d_dtype = b.has_d ? a.resout_dtype : a.io_dtype;
  if (!b.has_r) b.g.fwd.residual = a.x, b.g.fwd.res_dtype = a.io_dtype;
  if (!b.has_d) b.g.dresidual_out = g.dy;
  auto room = [&](int dtype) { return (a.dim * dtype_size(dtype) + 15) / 16 * 16; };
  b.o_dy = room(a.io_dtype), b.o_r = 2 * b.o_dy, b.o_d = b.o_r + room(b.g.fwd.res_dtype), b.o_g = b.o_d + room(b.d_dtype), b.stage = b.o_g + (GATE == 2 ? room(a.gate_dtype) : 0);
  const int params = MC * V <= 8 ? (GATE == 1 ? 4 : BIAS ? 3 : 2) * ((a.dim + 3) / 4 * 16) : 0;
  b.stages = 2 * b.stage + params <= kRing ? 2 : 1;
  const int smem = b.stages * b.stage + params;
  SSM_REQUIRE(smem <= 227 * 1024 - 512, SSM_ERR_TOO_LARGE, "fused_block_norm: a row does not fit");
  void (*kern)(BwdArgs);
  if constexpr (V == 4) kern = block_norm_bwd4_kernel<THREADS, MC, BIAS, GATE, TYPES>;
  else kern = block_norm_bwd_kernel<V, MC, BIAS, GATE, TYPES>;
  // what the device says of this kernel, asked once for a size (it takes longer than a launch)
  struct Known {
    int device = -1, threads = 0, smem = 0, fit = 0;
  };
  static thread_local Known known;
  int device = 0;
  cudaGetDevice(&device);
  if (known.device != device || known.threads != threads || known.smem != smem) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 512);  // the same for all calls, whichever thread makes them
    int fit = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, threads, smem) != cudaSuccess || fit < 1) cudaGetLastError(), fit = 1;
    known = Known{device, threads, smem, fit * sm_count()};
  }
  // runs of neighbouring rows, as many as run at once
  const int64_t most = std::min(kMaxRuns, known.fit);
  b.per = (int)std::max<int64_t>(1, (a.rows + most - 1) / most);
  const int runs = (int)((a.rows + b.per - 1) / b.per);
  kern<<<runs, threads, smem, st>>>(b);
  if (const int rc = launch_status("block_norm_bwd_kernel")) return rc;
  FoldArgs f{};
  f.partial = g.partial, f.dpost_weight = g.dpost_weight, f.dweight = g.dweight, f.dpost_bias = g.dpost_bias, f.dbias = g.dbias, f.dgate = g.dgate;
  f.per = b.per, f.runs = runs, f.dim = a.dim, f.param_dtype = a.param_dtype, f.gate_dtype = a.gate_dtype, f.unit = b.unit, f.units = GATE == 1 ? b.rows / b.unit : 0;
  constexpr int kFold = V == 1 ? 1 : 4;
  block_norm_fold_kernel<kFold><<<dim3((a.dim + 32 * kFold - 1) / (32 * kFold), std::min(4 + f.units, 1024)), 1024, 0, st>>>(f);
  return launch_status("block_norm_fold_kernel");
}
template <int V, int THREADS, int MC, int TYPES>
int launch_bwd(const ssm_block_norm_bwd_args& g, cudaStream_t st) {
  const int gate = g.fwd.gate_kind == kNone ? 0 : g.fwd.gate_kind == kToken ? 2 : 1;
  if (g.fwd.bias) return gate == 0 ? launch_bwd2<V, THREADS, MC, true, 0, TYPES>(g, st) : gate == 1 ? launch_bwd2<V, THREADS, MC, true, 1, TYPES>(g, st) : launch_bwd2<V, THREADS, MC, true, 2, TYPES>(g, st);
  return gate == 0 ? launch_bwd2<V, THREADS, MC, false, 0, TYPES>(g, st) : gate == 1 ? launch_bwd2<V, THREADS, MC, false, 1, TYPES>(g, st) : launch_bwd2<V, THREADS, MC, false, 2, TYPES>(g, st);
}
// four elements to a piece also in 16 bits: the sums of a thread's columns stay in registers
template <int TYPES>
int bwd_of(const ssm_block_norm_bwd_args& g, bool wide, cudaStream_t st) {
  const int dim = g.fwd.dim;
  if (wide && dim % 4 == 0)
    return dim <= 256 ? launch_bwd<4, 320, 1, TYPES>(g, st) : dim <= 2560 ? launch_bwd<4, 320, 2, TYPES>(g, st) : dim <= 4096 ? launch_bwd<4, 512, 2, TYPES>(g, st) : launch_bwd<4, 512, 4, TYPES>(g, st);
  return dim <= 1024 ? launch_bwd<1, 512, 2, TYPES>(g, st) : dim <= 4096 ? launch_bwd<1, 512, 8, TYPES>(g, st) : launch_bwd<1, 512, 16, 0>(g, st);
}
int dispatch_bwd(const ssm_block_norm_bwd_args& g, bool wide, cudaStream_t st) {
  switch (g.dresidual && g.dresidual_out ? types_of(g.fwd) : 0) {
    case 1: return bwd_of<1>(g, wide, st);
    case 2: return bwd_of<2>(g, wide, st);
    case 3: return bwd_of<3>(g, wide, st);
    default: return bwd_of<0>(g, wide, st);
  }
}

int check(const ssm_block_norm_args& a) {
  SSM_REQUIRE(a.rows >= 0 && a.dim >= 1 && a.len >= 1, SSM_ERR_SHAPE, "fused_block_norm: bad shape");
  SSM_REQUIRE(a.dim <= kMaxDim, SSM_ERR_TOO_LARGE, "fused_block_norm: more than 8192 columns");
  SSM_REQUIRE(a.rows < ((int64_t)1 << 30), SSM_ERR_TOO_LARGE, "fused_block_norm: 2^30 rows or more");
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
