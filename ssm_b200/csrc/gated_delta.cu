// Gated delta rule, any sizes (kdim <= 256) and types, in fp32 throughout: the recurrence token by token, forward and back, and the
// gradients of a chunk's tokens from the states around it; the single-token step; the C entry points.
//
// The columns of v are independent rows of the state, so a CTA walks a sequence with 32 of them: four lanes share a row (eight above kdim 128),
// each with its part of kdim in registers, in pairs for packed fp32 instructions.  A token is one sum over the lanes, S k, behind which the
// correction follows; o = S q after it does not hold up the next token.  Bound: one token after another, each some 110 instructions of a warp that has its
// scheduler to itself (four warps an SM, 22 % of the issue slots): 0.26 us a token forward and 0.22 back on as few SMs as there are rows (777
// tokens, kdim 64, 18 CTAs: 200 and 170 us; with eight lanes, a barrier more and loads converted as they were asked for 285 and 244).
//
// Backward: the adjoint state walks the same way from the end (dS' = dS + scale do q^T; w = beta dS' k = dv; dS <- a (dS' - w k^T)),
// and needs nothing of the states.  What the other gradients need of them is the state before and the adjoint state behind each
// chunk; within a chunk they are sums over pairs of tokens (see grad_kernel), all chunks at once.
#include <algorithm>

#include "gated_delta.cuh"

namespace ssmb {
namespace gd {

// ---------------------------------------------------------------------------------------------
// packed sequences
// ---------------------------------------------------------------------------------------------
constexpr int kTableThreads = 1024;
__global__ void __launch_bounds__(kTableThreads) table_kernel(const void* cu, int is64, int seqs, int len, int chunk, int nchunks, int32_t* table) {
  __shared__ int ends[kTableThreads], firsts[kTableThreads];
  const int tid = threadIdx.x;
  int at = 0, used = 0;  // end and chunks of the sequences so far
  for (int i0 = 0; i0 < seqs; i0 += kTableThreads) {
    const int i = i0 + tid;
    int end = 0;  // entries are clamped to [0, len] and to rise
    if (i < seqs) {
      const int64_t raw = is64 ? reinterpret_cast<const int64_t*>(cu)[i + 1] : reinterpret_cast<const int32_t*>(cu)[i + 1];
      end = (int)max((int64_t)0, min((int64_t)len, raw));
    }
    ends[tid] = max(end, at);
    __syncthreads();
    for (int off = 1; off < kTableThreads; off *= 2) {
      const int o = tid >= off ? ends[tid - off] : 0;
      __syncthreads();
      ends[tid] = max(ends[tid], o);
      __syncthreads();
    }
    const int start = tid ? ends[tid - 1] : at, stop = ends[tid], mine = i < seqs ? (stop - start + chunk - 1) / chunk : 0;
    firsts[tid] = mine;
    __syncthreads();
    for (int off = 1; off < kTableThreads; off *= 2) {
      const int o = tid >= off ? firsts[tid - off] : 0;
      __syncthreads();
      firsts[tid] += o;
      __syncthreads();
    }
    if (i < seqs) table[2 * i] = start, table[2 * i + 1] = stop, table[2 * seqs + i] = used + firsts[tid] - mine;
    used += firsts[kTableThreads - 1], at = ends[kTableThreads - 1];
    __syncthreads();
  }
  int32_t* e = table + 3 * seqs;
  const int32_t* first = table + 2 * seqs;
  for (int c = tid; c < nchunks; c += kTableThreads) {
    int t0 = 0, t1 = 0, seq = -1;
    if (c < used) {  // the last sequence whose first chunk is not behind c
      int lo = 0, hi = seqs - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first[mid] <= c) lo = mid;
        else hi = mid - 1;
      }
      seq = lo, t0 = table[2 * lo] + (c - first[lo]) * chunk, t1 = min(table[2 * lo + 1], t0 + chunk);
    } else if (at + (int64_t)(c - used) * chunk < len) {  // rows behind the last sequence
      t0 = at + (c - used) * chunk, t1 = min(len, t0 + chunk);
    }
    e[3 * c] = t0, e[3 * c + 1] = t1, e[3 * c + 2] = seq;
  }
}
int make_table(const ssm_gated_delta_args& a, int chunk, cudaStream_t st) {
  if (a.num_seqs <= 0) return SSM_OK;
  table_kernel<<<1, kTableThreads, 0, st>>>(a.cu_seqlens, a.cu_is_64, a.num_seqs, a.len, chunk, (int)chunk_bound(1, a.len, a.num_seqs, chunk), a.table);
  return launch_status("table_kernel");
}

// ---------------------------------------------------------------------------------------------
// the walks
// ---------------------------------------------------------------------------------------------
constexpr int kLanes = 8, kRows = 32, kThreads = kLanes * kRows;

struct WalkArgs {
  Args a;
  const float* initial;  // forward: the state; backward: the gradient of the final state
  void* o;               // forward: o; backward: dv (nullable)
  const void* dout;      // backward
  void* last;            // forward: final state; backward: gradient of the initial state (fp32)
  int last_dtype;
  float* rest;    // forward: r; backward: w
  float* states;  // forward: the state before every chunk; backward: the adjoint state behind it
};

template <typename T, int kLanes, int E, bool BACK>
__global__ void __launch_bounds__(kLanes* kRows) walk_kernel(const WalkArgs w) {
  constexpr int KP = kLanes * E, kThreads = kLanes * kRows, kTile = KP > 128 ? 8 : 16, kOuts = BACK ? 1 : 2;  // two buffers within 48 KB
  __shared__ __align__(16) float ks[2][kTile][KP], qs[2][kTile][KP];
  __shared__ float vs[2][kTile][kRows], decay[2][kTile], beta[2][kTile], out_s[2][kOuts][kTile][kRows];
  const Args& a = w.a;
  const int tid = threadIdx.x, lane = tid % kLanes, row = tid / kLanes, h = blockIdx.y, v0 = blockIdx.x * kRows, kh = h / a.group;
  T* o = reinterpret_cast<T*>(w.o);
  const int64_t vd = a.vd;
  if ((int)blockIdx.z == a.seqs) {  // packed: rows behind the last sequence are zeros
    const int from = a.where.table[2 * a.seqs - 1];
    if (o)
      for (int64_t i = tid; i < (int64_t)(a.len - from) * kRows; i += kThreads) {
        const int t = from + (int)(i / kRows), c = v0 + (int)(i % kRows);
        if (c < a.vd) o[((int64_t)t * a.heads + h) * vd + c] = from_f<T>(0.f);
      }
    return;
  }
  const Span s = sequence(a.where, blockIdx.z);
  const int n = s.t1 - s.t0, v = v0 + row;
  const bool live = v < a.vd;
  const T* qp = reinterpret_cast<const T*>(a.q.p) + s.b * a.q.sb + kh * a.q.sh;
  const T* kp = reinterpret_cast<const T*>(a.k.p) + s.b * a.k.sb + kh * a.k.sh;
  // backward: the incoming gradient, dense, in the place of v
  const T* vp = BACK ? reinterpret_cast<const T*>(w.dout) + ((int64_t)s.b * a.len * a.heads + h) * vd
                     : reinterpret_cast<const T*>(a.v.p) + s.b * a.v.sb + h * a.v.sh;
  const int64_t v_st = BACK ? (int64_t)a.heads * vd : a.v.st;
  const int64_t state_at = (((int64_t)s.seq * a.heads + h) * vd + v) * a.kd;

  float2 S[E / 2];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (e / 4) * (4 * kLanes) + lane * 4 + e % 4;
    (e % 2 ? S[e / 2].y : S[e / 2].x) = w.initial && live && c < a.kd ? w.initial[state_at + c] : 0.f;
  }
  auto keep = [&](int chunk) {
    float* to = w.states + (((int64_t)chunk * a.heads + h) * vd + v) * a.kd;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (e / 4) * (4 * kLanes) + lane * 4 + e % 4;
      if (live && c < a.kd) to[c] = e % 2 ? S[e / 2].y : S[e / 2].x;
    }
  };

  // tile i holds tokens t(i * kTile + j), counted from the end in the backward walk.  Its chunk boundaries lie on tile boundaries: forward
  // tiles start at multiples of kTile, backward the first tile is the ragged one
  const int ragged = BACK && n % kTile ? n % kTile : kTile;
  const int tiles = n == 0 ? 0 : BACK ? 1 + (n - ragged + kTile - 1) / kTile : (n + kTile - 1) / kTile;
  auto tile_at = [&](int i, int& from, int& count) {  // tokens [from, from + count)
    if (BACK) {
      count = i == 0 ? ragged : kTile;
      from = s.t0 + (i == 0 ? n - count : n - ragged - i * kTile);
    } else {
      from = s.t0 + i * kTile, count = min(kTile, s.t1 - from);
    }
  };
  constexpr int NK = kTile * KP / kThreads, NV = kTile * kRows / kThreads;
  // As they lie in memory: a conversion here would wait for them.
  T kr[NK], qr[NK], vr[NV];
  uint32_t raw = 0;
  auto raw_at = [&](const Rows& x, int dtype, int t) -> uint32_t {
    const int64_t at = s.b * x.sb + t * x.st + h * x.sh;
    return dtype == SSM_F32 ? __ldg(reinterpret_cast<const uint32_t*>(x.p) + at) : __ldg(reinterpret_cast<const uint16_t*>(x.p) + at);
  };
  auto value = [&](int dtype) { return dtype == SSM_F32 ? __uint_as_float(raw) : dtype == SSM_BF16 ? __uint_as_float(raw << 16) : __half2float(__ushort_as_half((uint16_t)raw)); };
  auto request = [&](int i) {
    int from, count;
    tile_at(i, from, count);
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int at = tid + j * kThreads, t = at / KP, c = at % KP;
      const bool in = t < count && c < a.kd;
      kr[j] = in ? kp[(int64_t)(from + t) * a.k.st + c] : from_f<T>(0.f);
      qr[j] = in ? qp[(int64_t)(from + t) * a.q.st + c] : from_f<T>(0.f);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = tid + j * kThreads, t = at / kRows, c = v0 + at % kRows;
      vr[j] = t < count && c < a.vd ? vp[(int64_t)(from + t) * v_st + c] : from_f<T>(0.f);
    }
    if (tid < kTile) raw = tid < count && a.g.p ? raw_at(a.g, a.g_dtype, from + tid) : 0;
    else if (tid < 2 * kTile) raw = tid - kTile < count ? raw_at(a.beta, a.beta_dtype, from + tid - kTile) : 0;
  };
  auto place = [&](int buf) {
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int at = tid + j * kThreads;
      ks[buf][at / KP][at % KP] = to_f<T>(kr[j]), qs[buf][at / KP][at % KP] = to_f<T>(qr[j]) * a.scale;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = tid + j * kThreads;
      vs[buf][at / kRows][at % kRows] = to_f<T>(vr[j]);
    }
    if (tid < kTile) decay[buf][tid] = expf(value(a.g_dtype));  // without decays e^0
    else if (tid < 2 * kTile) beta[buf][tid - kTile] = value(a.beta_dtype);
  };
  auto flush = [&](int i, int buf) {  // forward o and r, back w
    int from, count;
    tile_at(i, from, count);
    for (int at = tid; at < count * kRows; at += kThreads) {
      const int t = at / kRows, c = v0 + at % kRows;
      if (c >= a.vd) continue;
      const int64_t to = (((int64_t)s.b * a.len + from + t) * a.heads + h) * vd + c;
      if (o) o[to] = from_f<T>(out_s[buf][0][t][at % kRows]);
      if (w.rest) w.rest[to] = out_s[buf][kOuts - 1][t][at % kRows];
    }
  };
  if (tiles > 0) {
    request(0);
    place(0);
  }
  __syncthreads();
  for (int i = 0; i < tiles; ++i) {
    const int buf = i & 1;
    int from, count;
    tile_at(i, from, count);
    if (i + 1 < tiles) request(i + 1);
    if (w.states) {  // forward: before a chunk's first token; backward: behind its last
      const int local = from - s.t0;
      if (!BACK && local % kChunk == 0) keep(s.chunk + local / kChunk);
      if (BACK && ((local + count) % kChunk == 0 || i == 0)) keep(s.chunk + (local + count - 1) / kChunk);
    }
    auto row_of = [&](const float(&from)[kTile][KP], int t, float2(&x)[E / 2]) {
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const float4 z = *reinterpret_cast<const float4*>(&from[t][e * kLanes + lane * 4]);
        x[e / 2] = make_float2(z.x, z.y), x[e / 2 + 1] = make_float2(z.z, z.w);
      }
    };
    auto dot = [&](const float2(&x)[E / 2]) {
      float2 d[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int e = 0; e < E / 2; ++e) d[e % 2] = __ffma2_rn(S[e], x[e], d[e % 2]);
      return group_sum<kLanes, 1>((d[0].x + d[1].x) + (d[0].y + d[1].y));
    };
    auto token = [&](int t) {
      const float al = decay[buf][t], be = beta[buf][t], x = vs[buf][t][row];
      float2 kk[E / 2], qq[E / 2];
      row_of(ks[buf], t, kk), row_of(qs[buf], t, qq);
      if constexpr (!BACK) {
        const float r = fmaf(-al, dot(kk), x), u = be * r;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) S[e] = __ffma2_rn(make_float2(u, u), kk[e], __fmul2_rn(make_float2(al, al), S[e]));
        const float y = dot(qq);
        out_s[buf][lane & 1][t][row] = lane & 1 ? r : y;  // lanes agree; no branch
      } else {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) S[e] = __ffma2_rn(make_float2(x, x), qq[e], S[e]);
        const float ww = be * dot(kk), aw = -al * ww;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) S[e] = __ffma2_rn(make_float2(aw, aw), kk[e], __fmul2_rn(make_float2(al, al), S[e]));
        out_s[buf][0][t][row] = ww;
      }
    };
    if (count == kTile) {  // tokens side by side in the instruction stream: only the state runs from one to the next
#pragma unroll 4
      for (int j = 0; j < kTile; ++j) token(BACK ? kTile - 1 - j : j);
    } else {
      for (int j = 0; j < count; ++j) token(BACK ? count - 1 - j : j);
    }
    if (i + 1 < tiles) place(buf ^ 1);
    __syncthreads();
    flush(i, buf);  // its place is written again after the next barrier
  }
  if (w.last && live) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (e / 4) * (4 * kLanes) + lane * 4 + e % 4;
      if (c < a.kd) store_dyn(w.last, state_at + c, w.last_dtype, e % 2 ? S[e / 2].y : S[e / 2].x);
    }
  }
}

template <typename T, bool BACK>
int launch_walk(const WalkArgs& w, cudaStream_t st) {
  const dim3 grid((w.a.vd + kRows - 1) / kRows, w.a.heads, w.a.seqs + (w.a.where.table ? 1 : 0));
  if (w.a.kd <= 32) walk_kernel<T, 4, 8, BACK><<<grid, 4 * kRows, 0, st>>>(w);
  else if (w.a.kd <= 64) walk_kernel<T, 4, 16, BACK><<<grid, 4 * kRows, 0, st>>>(w);
  else if (w.a.kd <= 128) walk_kernel<T, 4, 32, BACK><<<grid, 4 * kRows, 0, st>>>(w);
  else walk_kernel<T, 8, 32, BACK><<<grid, 8 * kRows, 0, st>>>(w);
  return launch_status(BACK ? "walk_kernel (backward)" : "walk_kernel");
}
template <bool BACK>
int walk_of(const WalkArgs& w, cudaStream_t st) {
  switch (w.a.io) {
    case SSM_F32: return launch_walk<float, BACK>(w, st);
    case SSM_BF16: return launch_walk<__nv_bfloat16, BACK>(w, st);
    default: return launch_walk<__half, BACK>(w, st);
  }
}

// ---------------------------------------------------------------------------------------------
// gradients of a chunk's tokens
// ---------------------------------------------------------------------------------------------
// With G_ij = a_{j+1} .. a_i, gam_i = a_1 .. a_i, suf_i = a_{i+1} .. a_C (products, so that a decay of zero is exact), S0 the state
// before and dS the adjoint state behind the chunk, N1_ij = do_i.r_j, N2_ij = w_i.r_j:
//   dq_i = scale (gam_i S0^T do_i + sum_{j<=i} G_ij N1_ij beta_j k_j)
//   y_i = scale sum_{j>=i} G_ji N1_ji q_j - sum_{j>i} G_ji N2_ji k_j + suf_i dS^T r_i;   dbeta_i = k_i.y_i
//   dk_i = beta_i y_i - gam_i S0^T w_i - sum_{j<i} G_ij N2_ij beta_j k_j
//   dg_t = <S'_t, dS'_t>: every path from before t to t or behind it, i.e. the pairs j < t <= i of
//   M_ij = G_ij beta_j (scale N1_ij q_i.k_j - N2_ij k_i.k_j), from S0 into i >= t, from j < t into dS, and gam_C <S0, dS>.
// Summed path by path: no large sums that cancel.
struct GradArgs {
  Args a;
  const void* dout;
  const float* rest;
  const float* w;
  const float* states;
  const float* dstates;
  void* dq;
  void* dk;
  float* dqk;  // fp32, per value head: dq then dk; NULL where heads do not share keys
  float* dg;
  float* dbeta;
  int64_t tokens;
};

__host__ __device__ inline int padded(int n) { return (n + 3) / 4 * 4 + 4; }
inline size_t grad_smem(int kd, int vd_tile) { return sizeof(float) * (2 * kChunk * padded(kd) + 3 * kChunk * padded(vd_tile) + 5 * kChunk * (kChunk + 1) + 16 * kChunk); }
constexpr int kVTile = 128;  // columns of v at a time

__device__ __forceinline__ float4 at4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float dot4(float4 a, float4 b, float sum) { return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, sum)))); }

// A thread owns one element of kdim (rounds of kThreads of them where there are more) and all tokens of the chunk.
template <typename T>
__global__ void __launch_bounds__(kThreads) grad_kernel(const GradArgs g) {
  constexpr int C = kChunk, MP = C + 1;
  extern __shared__ __align__(16) float sm[];
  const Args& a = g.a;
  const int tid = threadIdx.x, h = blockIdx.y, kh = h / a.group, KS = padded(a.kd), VS = padded(kVTile);
  const Span s = chunk_of(a.where, blockIdx.x, C);
  const int n = s.t1 - s.t0;
  if (n <= 0) return;
  const int64_t vd = a.vd, tok = (int64_t)s.b * a.len + s.t0;
  T* dq = reinterpret_cast<T*>(g.dq);
  T* dk = reinterpret_cast<T*>(g.dk);
  auto put = [&](int i, int c, float xq, float xk) {
    if (g.dqk) {
      const int64_t to = ((tok + i) * a.heads + h) * a.kd + c;
      g.dqk[to] = xq, g.dqk[g.tokens * a.heads * a.kd + to] = xk;
    } else {
      const int64_t to = ((tok + i) * a.heads + h) * a.kd + c;
      dq[to] = from_f<T>(xq), dk[to] = from_f<T>(xk);
    }
  };
  if (s.seq < 0) {  // rows of no sequence
    for (int at = tid; at < n * a.kd; at += kThreads) put(at / a.kd, at % a.kd, 0.f, 0.f);
    for (int i = tid; i < n; i += kThreads) g.dg[(tok + i) * a.heads + h] = 0.f, g.dbeta[(tok + i) * a.heads + h] = 0.f;
    return;
  }
  float *q = sm, *k = q + C * KS, *r = k + C * KS, *w = r + C * VS, *d = w + C * VS;
  float *G = d + C * VS, *N1 = G + C * MP, *N2 = N1 + C * MP, *QK = N2 + C * MP, *KK = QK + C * MP;
  float *al = KK + C * MP, *be = al + C, *gam = be + C, *suf = gam + C, *into = suf + C, *outof = into + C, *db = outof + C, *inner = db + C;
  const T* qp = reinterpret_cast<const T*>(a.q.p) + s.b * a.q.sb + kh * a.q.sh;
  const T* kp = reinterpret_cast<const T*>(a.k.p) + s.b * a.k.sb + kh * a.k.sh;
  for (int at = tid; at < C * (KS - 4); at += kThreads) {
    const int i = at / (KS - 4), c = at % (KS - 4);
    const bool in = i < n && c < a.kd;
    q[i * KS + c] = in ? to_f<T>(qp[(int64_t)(s.t0 + i) * a.q.st + c]) * a.scale : 0.f;  // scale rides on q
    k[i * KS + c] = in ? to_f<T>(kp[(int64_t)(s.t0 + i) * a.k.st + c]) : 0.f;
  }
  if (tid < C) {
    al[tid] = tid < n ? decay_of(a, s.b, s.t0 + tid, h) : 1.f;
    be[tid] = tid < n ? beta_of(a, s.b, s.t0 + tid, h) : 0.f;
    into[tid] = outof[tid] = db[tid] = 0.f;
    inner[tid] = 0.f;
  }
  for (int at = tid; at < C * C; at += kThreads) N1[at / C * MP + at % C] = N2[at / C * MP + at % C] = 0.f;
  __syncthreads();
  if (tid < C) {
    float x = 1.f;
    for (int i = 0; i < C; ++i) {
      if (i > tid) x *= al[i];
      G[i * MP + tid] = i >= tid ? x : 0.f;
    }
    suf[tid] = x;  // tokens behind the chunk's last decay nothing
    x = 1.f;
    for (int i = 0; i <= tid; ++i) x *= al[i];
    gam[tid] = x;
  }
  for (int at = tid; at < C * C; at += kThreads) {
    const int i = at / C, j = at % C;
    float x = 0.f, y = 0.f;
    if (j <= i)
      for (int c = 0; c < a.kd; c += 4) {  // rows are padded with zeros to whole vectors
        const float4 kj = at4(&k[j * KS + c]);
        x = dot4(at4(&q[i * KS + c]), kj, x), y = dot4(at4(&k[i * KS + c]), kj, y);
      }
    QK[i * MP + j] = x, KK[i * MP + j] = y;
  }
  const float* S0 = g.states + ((int64_t)s.chunk * a.heads + h) * vd * a.kd;
  const float* dS = g.dstates + ((int64_t)s.chunk * a.heads + h) * vd * a.kd;
  const int per = kThreads / 32;
  float whole = 0.f;  // <S0, dS>
  // the products with the states, of which a thread forms those of one element c of kdim with C / `parts` tokens at a time
  const int cols = min(a.kd, kThreads);
  for (int c0 = 0; c0 < a.kd; c0 += cols) {
    const int c = c0 + tid % cols, parts = kThreads / cols, part = tid / cols;
    const bool on = c < a.kd && part < parts;
    for (int i0 = 0; i0 < C; i0 += 8) {  // eight tokens at a time in registers
      if (i0 >= n) break;
      float D1[8], D2[8], Z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) D1[i] = D2[i] = Z[i] = 0.f;
      for (int v0 = 0; v0 < a.vd; v0 += kVTile) {
        const int nv = min(kVTile, a.vd - v0);
        const bool loaded = a.vd <= kVTile && (c0 > 0 || i0 > 0);
        if (!loaded) {
          __syncthreads();
          const int whole_v = (nv + 3) / 4 * 4;
          for (int at = tid; at < C * whole_v; at += kThreads) {
            const int i = at / whole_v, x = at % whole_v;
            const int64_t from = ((tok + i) * a.heads + h) * vd + v0 + x;
            const bool in = i < n && x < nv;
            r[i * VS + x] = in ? g.rest[from] : 0.f;
            w[i * VS + x] = in ? g.w[from] : 0.f;
            d[i * VS + x] = in ? to_f<T>(reinterpret_cast<const T*>(g.dout)[from]) : 0.f;
          }
          __syncthreads();
          if (c0 == 0 && i0 == 0)  // N1, N2 once over all of v
            for (int at = tid; at < C * C; at += kThreads) {
              const int i = at / C, j = at % C;
              if (j > i) continue;
              float x = N1[i * MP + j], y = N2[i * MP + j];
              for (int v = 0; v < nv; v += 4) {
                const float4 rj = at4(&r[j * VS + v]);
                x = dot4(at4(&d[i * VS + v]), rj, x), y = dot4(at4(&w[i * VS + v]), rj, y);
              }
              N1[i * MP + j] = x, N2[i * MP + j] = y;
            }
        }
        if (on)
          for (int v = 4 * part; v < nv; v += 4 * parts) {
            float s0[4], ds[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) s0[e] = v + e < nv ? S0[(int64_t)(v0 + v + e) * a.kd + c] : 0.f, ds[e] = v + e < nv ? dS[(int64_t)(v0 + v + e) * a.kd + c] : 0.f;
            const float4 s4 = make_float4(s0[0], s0[1], s0[2], s0[3]), d4 = make_float4(ds[0], ds[1], ds[2], ds[3]);
            if (i0 == 0) whole = dot4(s4, d4, whole);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              D1[i] = dot4(s4, at4(&d[(i0 + i) * VS + v]), D1[i]);
              D2[i] = dot4(s4, at4(&w[(i0 + i) * VS + v]), D2[i]);
              Z[i] = dot4(d4, at4(&r[(i0 + i) * VS + v]), Z[i]);
            }
          }
      }
      __syncthreads();
      if (c0 == 0 && i0 == 0)  // the decays between the tokens of a pair
        for (int at = tid; at < C * C; at += kThreads) N1[at / C * MP + at % C] *= G[at / C * MP + at % C], N2[at / C * MP + at % C] *= G[at / C * MP + at % C];
      // the parts of v meet in shared memory (a buffer of its own behind the arrays); the tokens are dealt out to the parts
      float* meet = sm + 2 * C * KS + 3 * C * VS + 5 * C * MP + 16 * C;
      if (on)
#pragma unroll
        for (int i = 0; i < 8; ++i) meet[(i * 3 + 0) * kThreads + tid] = D1[i], meet[(i * 3 + 1) * kThreads + tid] = D2[i], meet[(i * 3 + 2) * kThreads + tid] = Z[i];
      __syncthreads();
      float xb[8], xi[8], xo[8];
#pragma unroll
      for (int ii = 0; ii < 8; ++ii) {
        const int i = i0 + ii;
        xb[ii] = xi[ii] = xo[ii] = 0.f;
        if (!on || ii % parts != part || i >= n) continue;
        float d1 = 0.f, d2 = 0.f, z = 0.f, sq = 0.f, sk = 0.f, y = 0.f;
        for (int p = tid % cols; p < parts * cols; p += cols) d1 += meet[(ii * 3 + 0) * kThreads + p], d2 += meet[(ii * 3 + 1) * kThreads + p], z += meet[(ii * 3 + 2) * kThreads + p];
        for (int j = 0; j < i; ++j) {
          const float m = be[j] * k[j * KS + c];
          sq = fmaf(m, N1[i * MP + j], sq), sk = fmaf(m, N2[i * MP + j], sk);
        }
        const float kc = k[i * KS + c], qc = q[i * KS + c];
        sq = fmaf(be[i] * kc, N1[i * MP + i], sq);
        y = N1[i * MP + i] * qc;
        for (int j = i + 1; j < n; ++j) y = fmaf(N1[j * MP + i], q[j * KS + c], y), y = fmaf(-N2[j * MP + i], k[j * KS + c], y);
        y = fmaf(suf[i], z, y);
        put(i, c, a.scale * fmaf(gam[i], d1, sq), be[i] * y - fmaf(gam[i], d2, sk));
        xb[ii] = kc * y;
        xi[ii] = gam[i] * (qc * d1 - kc * d2);  // S0 into token i
        xo[ii] = be[i] * suf[i] * kc * z;       // token i into dS
      }
      __syncthreads();
      // sums over kdim: warps in order, no atomics
#pragma unroll
      for (int ii = 0; ii < 8; ++ii) {
        const float b0 = warp_sum(xb[ii]), b1 = warp_sum(xi[ii]), b2 = warp_sum(xo[ii]);
        if (tid % 32 == 0) meet[(ii * 3 + 0) * per + tid / 32] = b0, meet[(ii * 3 + 1) * per + tid / 32] = b1, meet[(ii * 3 + 2) * per + tid / 32] = b2;
      }
      __syncthreads();
      if (tid < 24) {
        float x = 0.f;
        for (int p = 0; p < per; ++p) x += meet[tid * per + p];
        const int i = i0 + tid / 3;
        (tid % 3 == 0 ? db : tid % 3 == 1 ? into : outof)[i] += x;
      }
    }
  }
  __syncthreads();
  float* meet = sm + 2 * C * KS + 3 * C * VS + 5 * C * MP + 16 * C;
  whole = warp_sum(whole);
  if (tid % 32 == 0) meet[tid / 32] = whole;
  // M over N1's place
  for (int at = tid; at < C * C; at += kThreads) {
    const int i = at / C, j = at % C;
    if (j < i) N1[i * MP + j] = be[j] * (N1[i * MP + j] * QK[i * MP + j] - N2[i * MP + j] * KK[i * MP + j]);
  }
  __syncthreads();
  for (int t = tid / 32; t < n; t += per) {
    float x = 0.f;
    for (int i = t + tid % 32; i < n; i += 32)
      for (int j = 0; j < t; ++j) x += N1[i * MP + j];
    x = warp_sum(x);
    if (tid % 32 == 0) {
      float all = 0.f;
      for (int p = 0; p < per; ++p) all += meet[p];
      x = fmaf(gam[n - 1], all, x);
      for (int i = t; i < n; ++i) x += into[i];
      for (int j = 0; j < t; ++j) x += outof[j];
      g.dg[(tok + t) * a.heads + h] = x;
      g.dbeta[(tok + t) * a.heads + h] = db[t];
    }
  }
}

// gradients of shared keys and queries: the sum over the value heads of each, in their order
template <typename T>
__global__ void __launch_bounds__(256) fold_heads_kernel(const float* dqk, T* dq, T* dk, int64_t n, int kd, int key_heads, int group, int64_t half) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t c = i % kd, kh = i / kd % key_heads, t = i / kd / key_heads;
    const float* from = dqk + ((t * key_heads + kh) * group) * kd + c;
    float x = 0.f, y = 0.f;
    for (int j = 0; j < group; ++j) x += from[(int64_t)j * kd], y += from[half + (int64_t)j * kd];
    dq[i] = from_f<T>(x), dk[i] = from_f<T>(y);
  }
}
int fold_heads(const float* dqk, void* dq, void* dk, int64_t tokens, int kd, int key_heads, int group, int dtype, cudaStream_t st) {
  const int64_t n = tokens * key_heads * kd, half = n * group;
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 8 * sm_count());
  auto go = [&](auto type) {
    using T = decltype(type);
    fold_heads_kernel<T><<<grid, 256, 0, st>>>(dqk, reinterpret_cast<T*>(dq), reinterpret_cast<T*>(dk), n, kd, key_heads, group, half);
  };
  if (dtype == SSM_F32) go(float());
  else if (dtype == SSM_BF16) go(__nv_bfloat16());
  else go(__half());
  return launch_status("fold_heads_kernel");
}
template <typename T>
int launch_grad(const GradArgs& g, int64_t chunks, cudaStream_t st) {
  const size_t smem = grad_smem(g.a.kd, kVTile) + sizeof(float) * 24 * kThreads;
  static_assert(sizeof(float) * (2 * kChunk * 260 + 3 * kChunk * 132 + 5 * kChunk * 33 + 16 * kChunk + 24 * kThreads) <= 227 * 1024, "kdim of 256 fits");
  const cudaError_t e = cudaFuncSetAttribute(grad_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    set_error("grad_kernel: %s", cudaGetErrorString(e));
    return (int)e;
  }
  grad_kernel<T><<<dim3((unsigned)chunks, g.a.heads), kThreads, smem, st>>>(g);
  if (const int rc = launch_status("grad_kernel")) return rc;
  return g.dqk ? fold_heads(g.dqk, g.dq, g.dk, g.tokens, g.a.kd, g.a.heads / g.a.group, g.a.group, g.a.io, st) : (int)SSM_OK;
}

// ---------------------------------------------------------------------------------------------
// one token
// ---------------------------------------------------------------------------------------------
// Bound: HBM, the fp32 state read and written (8 bytes an element).  Eight lanes share a row of the state, in pieces of 16 bytes: a warp's
// request covers whole lines of four rows, and all of a thread's pieces are in flight before the first product.
struct StepArgs {
  Rows q, k, v, g, beta;  // st unused
  int g_dtype, beta_dtype, kd, vd, heads, group;
  float scale;
  float* state;
  void* o;
};

template <typename T, int E, bool WHOLE>  // WHOLE: kdim is a multiple of 4 and q, k can be read four at a time
__global__ void __launch_bounds__(kThreads) step_kernel(const StepArgs a) {
  const int tid = threadIdx.x, lane = tid % kLanes, v = blockIdx.x * kRows + tid / kLanes, h = blockIdx.y, b = blockIdx.z, kh = h / a.group;
  const bool live = v < a.vd;
  float* st = a.state + (((int64_t)b * a.heads + h) * a.vd + (live ? v : 0)) * a.kd;
  const T* kp = reinterpret_cast<const T*>(a.k.p) + b * a.k.sb + kh * a.k.sh;
  const T* qp = reinterpret_cast<const T*>(a.q.p) + b * a.q.sb + kh * a.q.sh;
  float S[E], kk[E], qq[E];
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int c = e * kLanes + lane * 4;
    if constexpr (WHOLE) {
      const float4 x = live && c < a.kd ? __ldcs(reinterpret_cast<const float4*>(st + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[e] = x.x, S[e + 1] = x.y, S[e + 2] = x.z, S[e + 3] = x.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) S[e + i] = live && c + i < a.kd ? st[c + i] : 0.f;
    }
  }
  const float x = live ? to_f<T>(reinterpret_cast<const T*>(a.v.p)[b * a.v.sb + h * a.v.sh + v]) : 0.f;
  const float al = a.g.p ? expf(load_dyn(a.g.p, b * a.g.sb + h * a.g.sh, a.g_dtype)) : 1.f;
  const float be = load_dyn(a.beta.p, b * a.beta.sb + h * a.beta.sh, a.beta_dtype);
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int c = e * kLanes + lane * 4;
    if constexpr (WHOLE && sizeof(T) == 2) {
      const uint2 rk = c < a.kd ? __ldg(reinterpret_cast<const uint2*>(kp + c)) : make_uint2(0, 0), rq = c < a.kd ? __ldg(reinterpret_cast<const uint2*>(qp + c)) : make_uint2(0, 0);
      const T *k4 = reinterpret_cast<const T*>(&rk), *q4 = reinterpret_cast<const T*>(&rq);
#pragma unroll
      for (int i = 0; i < 4; ++i) kk[e + i] = to_f<T>(k4[i]), qq[e + i] = to_f<T>(q4[i]) * a.scale;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kk[e + i] = c + i < a.kd ? to_f<T>(kp[c + i]) : 0.f;
        qq[e + i] = c + i < a.kd ? to_f<T>(qp[c + i]) * a.scale : 0.f;
      }
    }
  }
  float sk = 0.f, sq = 0.f, kq = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    S[e] *= al;
    sk = fmaf(S[e], kk[e], sk), sq = fmaf(S[e], qq[e], sq), kq = fmaf(kk[e], qq[e], kq);
  }
  sk = group_sum<kLanes, 1>(sk), sq = group_sum<kLanes, 1>(sq), kq = group_sum<kLanes, 1>(kq);
  const float u = be * (x - sk);
  if (!live) return;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int c = e * kLanes + lane * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) S[e + i] = fmaf(u, kk[e + i], S[e + i]);
    if constexpr (WHOLE) {
      if (c < a.kd) __stcs(reinterpret_cast<float4*>(st + c), make_float4(S[e], S[e + 1], S[e + 2], S[e + 3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < a.kd) st[c + i] = S[e + i];
    }
  }
  if (lane == 0) reinterpret_cast<T*>(a.o)[((int64_t)b * a.heads + h) * a.vd + v] = from_f<T>(fmaf(kq, u, sq));
}
template <typename T, int E>
void launch_step(const StepArgs& a, int batch, bool whole, cudaStream_t st) {
  const dim3 grid((a.vd + kRows - 1) / kRows, a.heads, batch);
  if (whole) step_kernel<T, E, true><<<grid, kThreads, 0, st>>>(a);
  else step_kernel<T, E, false><<<grid, kThreads, 0, st>>>(a);
}
template <typename T>
void step_of(const StepArgs& a, int batch, bool whole, cudaStream_t st) {
  if (a.kd <= 32) launch_step<T, 4>(a, batch, whole, st);
  else if (a.kd <= 64) launch_step<T, 8>(a, batch, whole, st);
  else if (a.kd <= 128) launch_step<T, 16>(a, batch, whole, st);
  else launch_step<T, 32>(a, batch, whole, st);
}

// ---------------------------------------------------------------------------------------------
// arguments
// ---------------------------------------------------------------------------------------------
static int check_heads(int heads, int key_heads, int kd, int vd, int io, int g_dtype, int beta_dtype) {
  SSM_REQUIRE(heads >= 1 && key_heads >= 1 && heads % key_heads == 0, SSM_ERR_SHAPE, "gated_delta: the key heads must divide the heads");
  SSM_REQUIRE(kd >= 1 && vd >= 1, SSM_ERR_SHAPE, "gated_delta: the head sizes must be positive");
  SSM_REQUIRE(kd <= 256, SSM_ERR_TOO_LARGE, "gated_delta: the key size is at most 256");
  SSM_REQUIRE(vd <= 65536 && heads <= 65535, SSM_ERR_TOO_LARGE, "gated_delta: the value size is at most 65536, the heads at most 65535");
  SSM_REQUIRE(valid_dtype(io) && valid_dtype(g_dtype) && valid_dtype(beta_dtype), SSM_ERR_DTYPE, "gated_delta: unknown dtype");
  return SSM_OK;
}
int check(const ssm_gated_delta_args& a, Args& d) {
  SSM_REQUIRE(a.batch >= 0 && a.len >= 0, SSM_ERR_SHAPE, "gated_delta: negative size");
  if (const int rc = check_heads(a.heads, a.key_heads, a.kdim, a.vdim, a.io_dtype, a.g_dtype, a.beta_dtype)) return rc;
  SSM_REQUIRE(a.num_seqs >= 0 && (a.num_seqs == 0 || a.batch == 1), SSM_ERR_SHAPE, "gated_delta: packed sequences need a batch of one");
  SSM_REQUIRE(a.len <= (1 << 30), SSM_ERR_TOO_LARGE, "gated_delta: more than 2^30 tokens");
  SSM_REQUIRE(a.batch <= 65534 && a.num_seqs <= 65534, SSM_ERR_TOO_LARGE, "gated_delta: more than 65534 sequences");
  SSM_REQUIRE(a.num_seqs == 0 || (a.cu_seqlens && a.table), SSM_ERR_NULL, "gated_delta: packed sequences need cu_seqlens and table");
  SSM_REQUIRE((int64_t)a.batch * a.len == 0 || (a.q && a.k && a.v && a.beta), SSM_ERR_NULL, "gated_delta: NULL pointer");
  SSM_REQUIRE(a.final_state == nullptr || valid_dtype(a.final_dtype), SSM_ERR_DTYPE, "gated_delta: unknown state dtype");
  SSM_REQUIRE(aligned_to({a.q, a.k, a.v, a.o}, dtype_size(a.io_dtype)) && aligned_to(a.g, dtype_size(a.g_dtype)) && aligned_to(a.beta, dtype_size(a.beta_dtype)) &&
                  (a.num_seqs == 0 || aligned_to(a.cu_seqlens, a.cu_is_64 ? 8 : 4)) && aligned_to({a.initial_state, a.table, a.rest, a.states}, 4) &&
                  (a.final_state == nullptr || aligned_to(a.final_state, dtype_size(a.final_dtype))),
              SSM_ERR_ALIGN, "gated_delta: misaligned pointer");
  d.q = {a.q, a.q_sb, a.q_st, a.q_sh}, d.k = {a.k, a.k_sb, a.k_st, a.k_sh}, d.v = {a.v, a.v_sb, a.v_st, a.v_sh};
  d.g = {a.g, a.g_sb, a.g_st, a.g_sh}, d.beta = {a.beta, a.beta_sb, a.beta_st, a.beta_sh};
  d.io = a.io_dtype, d.g_dtype = a.g_dtype, d.beta_dtype = a.beta_dtype, d.kd = a.kdim, d.vd = a.vdim, d.heads = a.heads, d.group = a.heads / a.key_heads;
  d.len = a.len, d.seqs = a.num_seqs > 0 ? a.num_seqs : a.batch, d.final_dtype = a.final_dtype, d.scale = a.scale;
  d.where = {a.num_seqs > 0 ? a.table : nullptr, a.len, d.seqs, (a.len + kChunk - 1) / kChunk};
  return SSM_OK;
}

int check_gradients(const ssm_gated_delta_bwd_args& g) {
  SSM_REQUIRE(aligned_to({g.dout, g.dq, g.dk, g.dv}, dtype_size(g.fwd.io_dtype)) && aligned_to({g.dfinal, g.dg, g.dbeta, g.dinitial, g.dv32, g.dstates, g.dqk}, 4), SSM_ERR_ALIGN,
              "gated_delta backward: misaligned pointer");
  return SSM_OK;
}

}  // namespace gd
}  // namespace ssmb

using namespace ssmb;

extern "C" int64_t ssm_gated_delta_chunks(int32_t batch, int32_t len, int32_t num_seqs) { return gd::chunk_bound(batch, len, num_seqs, gd::kChunk); }
extern "C" int64_t ssm_gated_delta_table_ints(int32_t batch, int32_t len, int32_t num_seqs) {
  return num_seqs > 0 ? 3 * (int64_t)num_seqs + 3 * gd::chunk_bound(batch, len, num_seqs, gd::kChunk) : 0;
}

extern "C" int ssm_gated_delta_fwd(const ssm_gated_delta_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "gated_delta: NULL arguments");
  gd::WalkArgs w{};
  if (const int rc = gd::check(*args, w.a)) return rc;
  if (w.a.seqs == 0) return SSM_OK;
  SSM_REQUIRE(args->o || args->len == 0, SSM_ERR_NULL, "gated_delta: NULL output");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (const int rc = gd::make_table(*args, gd::kChunk, st)) return rc;
  w.initial = args->initial_state, w.o = args->o, w.last = args->final_state, w.last_dtype = args->final_dtype, w.rest = args->rest, w.states = args->states;
  return gd::walk_of<false>(w, st);
}

extern "C" int ssm_gated_delta_bwd(const ssm_gated_delta_bwd_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "gated_delta: NULL arguments");
  gd::WalkArgs w{};
  if (const int rc = gd::check(args->fwd, w.a)) return rc;
  if (w.a.seqs == 0) return SSM_OK;
  const bool any = args->fwd.len > 0;
  SSM_REQUIRE(!any || (args->dout && args->dq && args->dk && args->dv && args->dg && args->dbeta && args->dv32 && args->dstates && args->fwd.rest && args->fwd.states),
              SSM_ERR_NULL, "gated_delta backward: NULL pointer");
  SSM_REQUIRE(!any || w.a.group == 1 || args->dqk, SSM_ERR_NULL, "gated_delta backward: shared keys need the dqk scratch");
  if (const int rc = gd::check_gradients(*args)) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  w.initial = args->dfinal, w.dout = args->dout, w.last = args->dinitial, w.last_dtype = SSM_F32;
  w.o = args->dv == (void*)args->dv32 ? nullptr : args->dv, w.rest = args->dv32, w.states = args->dstates;
  if (w.a.where.table && !w.o) w.o = args->dv;  // rows of no sequence are written through it
  if (const int rc = gd::walk_of<true>(w, st)) return rc;
  if (!any) return SSM_OK;
  gd::GradArgs g{};
  g.a = w.a, g.dout = args->dout, g.rest = args->fwd.rest, g.w = args->dv32, g.states = args->fwd.states, g.dstates = args->dstates;
  g.dq = args->dq, g.dk = args->dk, g.dqk = w.a.group > 1 ? args->dqk : nullptr, g.dg = args->dg, g.dbeta = args->dbeta;
  g.tokens = (int64_t)args->fwd.batch * args->fwd.len;
  const int64_t chunks = ssm_gated_delta_chunks(args->fwd.batch, args->fwd.len, args->fwd.num_seqs);
  switch (w.a.io) {
    case SSM_F32: return gd::launch_grad<float>(g, chunks, st);
    case SSM_BF16: return gd::launch_grad<__nv_bfloat16>(g, chunks, st);
    default: return gd::launch_grad<__half>(g, chunks, st);
  }
}

extern "C" int ssm_gated_delta_step(const ssm_gated_delta_step_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "gated_delta_step: NULL arguments");
  const ssm_gated_delta_step_args& a = *args;
  SSM_REQUIRE(a.batch >= 0, SSM_ERR_SHAPE, "gated_delta_step: negative size");
  if (const int rc = gd::check_heads(a.heads, a.key_heads, a.kdim, a.vdim, a.io_dtype, a.g_dtype, a.beta_dtype)) return rc;
  SSM_REQUIRE(a.batch <= 65535, SSM_ERR_TOO_LARGE, "gated_delta_step: more than 65535 sequences");
  if (a.batch == 0) return SSM_OK;
  SSM_REQUIRE(a.state && a.q && a.k && a.v && a.beta && a.o, SSM_ERR_NULL, "gated_delta_step: NULL pointer");
  SSM_REQUIRE(aligned_to(a.state, 4) && aligned_to({a.q, a.k, a.v, a.o}, dtype_size(a.io_dtype)) && aligned_to(a.g, dtype_size(a.g_dtype)) && aligned_to(a.beta, dtype_size(a.beta_dtype)),
              SSM_ERR_ALIGN, "gated_delta_step: misaligned pointer");
  gd::StepArgs s{};
  s.q = {a.q, a.q_sb, 0, a.q_sh}, s.k = {a.k, a.k_sb, 0, a.k_sh}, s.v = {a.v, a.v_sb, 0, a.v_sh};
  s.g = {a.g, a.g_sb, 0, a.g_sh}, s.beta = {a.beta, a.beta_sb, 0, a.beta_sh};
  s.g_dtype = a.g_dtype, s.beta_dtype = a.beta_dtype, s.kd = a.kdim, s.vd = a.vdim, s.heads = a.heads, s.group = a.heads / a.key_heads;
  s.scale = a.scale, s.state = a.state, s.o = a.o;
  bool whole = a.kdim % 4 == 0 && aligned_to(a.state, 16);
  if (a.io_dtype != SSM_F32)  // q and k are read in pieces of 8 bytes
    whole = whole && aligned_to(a.q, 8) && aligned_to(a.k, 8) && a.q_sb % 4 == 0 && a.q_sh % 4 == 0 && a.k_sb % 4 == 0 && a.k_sh % 4 == 0;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a.io_dtype) {
    case SSM_F32: gd::step_of<float>(s, a.batch, whole, st); break;
    case SSM_BF16: gd::step_of<__nv_bfloat16>(s, a.batch, whole, st); break;
    default: gd::step_of<__half>(s, a.batch, whole, st);
  }
  return launch_status("step_kernel");
}
