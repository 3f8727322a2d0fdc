// Log probabilities of given tokens (with entropy and top alternatives) and distillation from a teacher's top logits.
//
// Both are one pass over a row of logits with a running maximum m, s = sum e^{(x - m)/T} and, for the entropy,
// w = sum (x - m)/T e^{(x - m)/T}: log p_i = (x_i - m)/T - ln s and H = ln s - w / s.  The backward pass is one more read of the row and
// one write of its gradient.  Bound: HBM (two or four bytes an element each way).  A row goes to one CTA, or to a cluster of up to
// eight that join their sums through distributed shared memory where the rows alone would not fill the GPU.
//
// Top alternatives: the k-th largest of the threads' own maxima bounds the k-th largest logit from below, so a second
// pass over the row (which then lies in the L2) keeps the few elements at or above it, and ranks them by (value, lowest id).
#include <cooperative_groups.h>

#include "../../include/ssm_b200_lm.h"
#include "common.cuh"

namespace ssmb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kUnroll = 4;       // 16-byte pieces a thread has in flight
constexpr int kCandidates = 1024;  // kept elements of a slice; more (many equal logits) go through rounds of one maximum each
constexpr int kMaxTop = 128;
constexpr int kMaxTeacher = 1024;

enum Flags { kEntropy = 1, kTop = 2 };

// order of floats as integers: NaN above everything, -0 equal to 0
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// larger key: larger value, among equal ones the lower id
__device__ __forceinline__ uint64_t key_of(float x, int id) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~id; }

// f(x, id) for the elements [lo, hi) of a row: 16-byte pieces between a ragged head and tail.  `lanes` threads share the work; this one is `me`.
// P pieces are requested before the first is used.
template <typename T, int P, typename F, typename G>
__device__ __forceinline__ void walk(const T* row, int lo, int hi, int me, int lanes, F&& one, G&& piece) {
  constexpr int V = Vec16<T>::N;
  const int skew = (int)((reinterpret_cast<uintptr_t>(row + lo) % 16) / sizeof(T));
  const int head = min(hi - lo, skew ? V - skew : 0);
  if (me < head) one(to_f<T>(row[lo + me]), lo + me);
  const int body = (hi - lo - head) / V, at = lo + head;
  const uint4* src = reinterpret_cast<const uint4*>(row + at);
  int i = me;
  for (; i + (P - 1) * lanes < body; i += P * lanes) {
    Vec16<T> r[P];
#pragma unroll
    for (int p = 0; p < P; ++p) r[p].raw = src[i + p * lanes];
    float f[P][V];
#pragma unroll
    for (int p = 0; p < P; ++p) r[p].unpack(f[p]);
    int ids[P];
#pragma unroll
    for (int p = 0; p < P; ++p) ids[p] = at + (i + p * lanes) * V;
    piece(f, ids, std::integral_constant<int, P>{});
  }
  for (; i < body; i += lanes) {
    Vec16<T> r;
    r.raw = src[i];
    float f[1][V];
    r.unpack(f[0]);
    const int ids[1] = {at + i * V};
    piece(f, ids, std::integral_constant<int, 1>{});
  }
  const int tail = at + body * V;
  if (me < hi - tail) one(to_f<T>(row[tail + me]), tail + me);
}

struct Sums {
  float m, s, w;
};
// c: log2(e) / T.  w in units of base-2 exponents
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, 0.f};  // NaN sums stay NaN
  const float da = fmaxf((a.m - m) * c, -1e30f), db = fmaxf((b.m - m) * c, -1e30f);
  const float ea = ex2_approx(da), eb = ex2_approx(db);
  return {m, a.s * ea + b.s * eb, ea * fmaf(a.s, da, a.w) + eb * fmaf(b.s, db, b.w)};
}

struct StatsArgs {
  int64_t rows, row_stride, ignore;
  int vocab, top_k, teacher_dtype;
  float c, inv_t;
  const void* logits;
  const int64_t* targets;
  const void* teacher;
  const int64_t* ids;
  float* logp;  // or the loss
  float* entropy;
  float* top_logp;
  int64_t* top_ids;
  float4* stats;  // m, log2 s, entropy, unused
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// softmax of a row's teacher entries by one warp: t_j into `t` (0 for those left out), the largest and ln of the sum returned
__device__ __forceinline__ void teacher_softmax(const StatsArgs& a, int64_t r, int lane, float* t, float& top, float& lns, bool& any) {
  const int64_t base = r * a.top_k;
  top = -INFINITY;
  float seen = 0.f;  // 1: an entry above -inf, or NaN
  for (int j = lane; j < a.top_k; j += 32) {
    const float x = load_dyn(a.teacher, base + j, a.teacher_dtype);
    if (a.ids[base + j] >= 0 && !(x == -INFINITY)) top = fmaxf(top, x), seen = 1.f;
  }
  top = warp_max(top);
  any = warp_max(seen) != 0.f;
  float s = 0.f;
  for (int j = lane; j < a.top_k; j += 32) {
    const bool in = any && a.ids[base + j] >= 0;
    const float x = in ? load_dyn(a.teacher, base + j, a.teacher_dtype) : 0.f;
    const float e = in ? expf((x - top) * a.inv_t) : 0.f;
    t[j] = e, s += e;
  }
  s = warp_sum(s);
  lns = logf(s);
  const float inv = any ? 1.f / s : 0.f;
  for (int j = lane; j < a.top_k; j += 32) t[j] *= inv;
}

template <typename T, int FLAGS, bool DISTILL>
__global__ void __launch_bounds__(kThreads) row_stats_kernel(const StatsArgs a, const int cluster) {
  __shared__ Sums part[kThreads / 32];
  __shared__ Sums mine;
  __shared__ __align__(16) float maxima[kThreads];
  __shared__ uint64_t cand[kCandidates];
  __shared__ uint64_t best[kMaxTop];
  __shared__ uint64_t round_best[kThreads / 32];
  __shared__ int count;
  __shared__ float bound_s;
  __shared__ float teach[DISTILL ? kMaxTeacher : 1];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int64_t r = blockIdx.x / cluster;
  const int part_of = (int)(blockIdx.x % cluster);
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  // slices of whole 16-byte pieces; the last takes the rest
  const int per = ((a.vocab + cluster - 1) / cluster + 63) / 64 * 64;
  const int lo = min(a.vocab, part_of * per), hi = part_of == cluster - 1 ? a.vocab : min(a.vocab, lo + per);

  Sums me{-INFINITY, 0.f, 0.f};
  const float c = a.c;
  auto raise = [&](float top) {
    if (top > me.m) {
      const float d = fmaxf((me.m - top) * c, -1e30f), e = ex2_approx(d);
      if constexpr ((FLAGS & kEntropy) != 0) me.w = e * fmaf(me.s, d, me.w);
      me.s *= e, me.m = top;
    }
  };
  auto add = [&](float x, float base) {
    const float d = (x - base) * c, e = ex2_approx(d);
    me.s += e;
    if constexpr ((FLAGS & kEntropy) != 0) me.w = fmaf(e, fmaxf(d, -1e30f), me.w);
  };
  walk<T, kUnroll>(
      row, lo, hi, tid, kThreads,
      [&](float x, int) {
        raise(x);
        add(x, me.m == -INFINITY ? 0.f : me.m);
      },
      [&](const auto& f, const int*, auto pieces) {
        constexpr int V = Vec16<T>::N;
        float top = f[0][0];
#pragma unroll
        for (int p = 0; p < decltype(pieces)::value; ++p)
#pragma unroll
          for (int j = 0; j < V; ++j) top = fmaxf(top, f[p][j]);
        raise(top);
        const float base = me.m == -INFINITY ? 0.f : me.m;
#pragma unroll
        for (int p = 0; p < decltype(pieces)::value; ++p)
#pragma unroll
          for (int j = 0; j < V; ++j) add(f[p][j], base);
      });

  if constexpr ((FLAGS & kTop) != 0) maxima[tid] = me.m;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const Sums o{__shfl_xor_sync(0xffffffffu, me.m, off), __shfl_xor_sync(0xffffffffu, me.s, off), __shfl_xor_sync(0xffffffffu, me.w, off)};
    me = lane & off ? join(o, me, c) : join(me, o, c);  // the same order on both sides
  }
  if (lane == 0) part[warp] = me;
  if (tid == 0) count = 0, bound_s = -INFINITY;
  __syncthreads();
  if (warp == 0) {
    me = lane < kThreads / 32 ? part[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      const Sums o{__shfl_xor_sync(0xffffffffu, me.m, off), __shfl_xor_sync(0xffffffffu, me.s, off), __shfl_xor_sync(0xffffffffu, me.w, off)};
      me = lane & off ? join(o, me, c) : join(me, o, c);
    }
    if (lane == 0) mine = me;
  }

  if constexpr ((FLAGS & kTop) != 0) {
    const int k = a.top_k;
    {  // the k-th largest of the threads' maxima
      const float own = maxima[tid];
      int above = 0;
      for (int i = 0; i < kThreads; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&maxima[i]);
        above += (v.x > own || (v.x == own && i < tid)) + (v.y > own || (v.y == own && i + 1 < tid)) + (v.z > own || (v.z == own && i + 2 < tid)) +
                 (v.w > own || (v.w == own && i + 3 < tid));
      }
      if (above == k - 1) bound_s = own;
    }
    __syncthreads();
    const uint32_t bound = order_of(bound_s);
    auto keep = [&](float x, int id) {
      if (order_of(x) >= bound) {
        const int at = atomicAdd(&count, 1);
        if (at < kCandidates) cand[at] = key_of(x, id);
      }
    };
    walk<T, 2>(row, lo, hi, tid, kThreads, keep, [&](const auto& f, const int* ids, auto pieces) {
      constexpr int V = Vec16<T>::N;
#pragma unroll
      for (int p = 0; p < decltype(pieces)::value; ++p)
#pragma unroll
        for (int j = 0; j < V; ++j) keep(f[p][j], ids[p] + j);
    });
    if (tid < kMaxTop) best[tid] = 0;  // below every key
    __syncthreads();
    const int n = count;
    if (n <= kCandidates) {
      for (int i = tid; i < n; i += kThreads) {  // keys differ (ids do), so ranks do
        const uint64_t own = cand[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += cand[j] > own;
        if (above < k) best[above] = own;
      }
    } else {  // more equal logits than fit: one maximum at a time
      uint64_t last = ~0ull;
      for (int j = 0; j < k; ++j) {
        uint64_t top = 0;
        auto look = [&](float x, int id) {
          const uint64_t key = key_of(x, id);
          if (key < last && key > top) top = key;
        };
        walk<T, 2>(row, lo, hi, tid, kThreads, look, [&](const auto& f, const int* ids, auto pieces) {
          constexpr int V = Vec16<T>::N;
#pragma unroll
          for (int p = 0; p < decltype(pieces)::value; ++p)
#pragma unroll
            for (int e = 0; e < V; ++e) look(f[p][e], ids[p] + e);
        });
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
          const uint64_t o = __shfl_xor_sync(0xffffffffu, top, off);
          top = o > top ? o : top;
        }
        if (lane == 0) round_best[warp] = top;
        __syncthreads();
        top = round_best[0];
        for (int i = 1; i < kThreads / 32; ++i) top = round_best[i] > top ? round_best[i] : top;
        __syncthreads();
        last = top;
        if (tid == 0) best[j] = top;
      }
    }
  }

  Sums all;
  if (cluster > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    if (part_of == 0) {
      all = *cl.map_shared_rank(&mine, 0);
      for (int i = 1; i < cluster; ++i) all = join(all, *cl.map_shared_rank(&mine, i), c);
      if constexpr ((FLAGS & kTop) != 0) {  // the slices' best, joined
        const int k = a.top_k, n = cluster * k;
        for (int i = tid; i < n; i += kThreads) cand[i] = cl.map_shared_rank(&best[0], i / k)[i % k];
      }
    }
    cl.sync();  // the other CTAs' shared memory stays until it has been read
    if (part_of != 0) return;
    if constexpr ((FLAGS & kTop) != 0) {
      const int k = a.top_k, n = cluster * k;
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t own = cand[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += cand[j] > own;
        if (own != 0 && above < k) best[above] = own;
      }
      __syncthreads();
    }
  } else {
    __syncthreads();
    all = mine;
  }

  const bool none = all.m == -INFINITY && all.s == 0.f;  // a row of -inf
  const float log2s = none ? 0.f : log2f(all.s), lns = log2s * kLn2;
  const float entropy = none ? 0.f : lns - kLn2 * all.w / all.s;
  auto logp_of = [&](float x) { return none ? -INFINITY : fmaf(x - all.m, a.inv_t, -lns); };
  if (tid == 0) {
    if (a.stats) a.stats[r] = make_float4(all.s != all.s ? all.s : all.m, log2s, entropy, 0.f);
    if constexpr (!DISTILL) {
      const int64_t t = a.targets[r];
      a.logp[r] = t == a.ignore ? 0.f : t < 0 || t >= a.vocab ? __uint_as_float(0x7fc00000u) : logp_of(to_f<T>(row[t]));
      if constexpr ((FLAGS & kEntropy) != 0) a.entropy[r] = entropy;
    }
  }
  if constexpr ((FLAGS & kTop) != 0) {
    for (int j = tid; j < a.top_k; j += kThreads) {
      const int id = (int)~(uint32_t)best[j];
      a.top_ids[r * a.top_k + j] = id;
      a.top_logp[r * a.top_k + j] = logp_of(to_f<T>(row[id]));
    }
  }
  if constexpr (DISTILL) {
    if (warp == 0) {
      float top, ln_t;
      bool any;
      teacher_softmax(a, r, lane, teach, top, ln_t, any);
      float loss = 0.f;
      const int64_t base = r * a.top_k;
      if (any)
        for (int j = lane; j < a.top_k; j += 32) {
          const int64_t id = a.ids[base + j];
          const float t = teach[j];
          if (id < 0 || t == 0.f) continue;
          const float log_t = (load_dyn(a.teacher, base + j, a.teacher_dtype) - top) * a.inv_t - ln_t;
          loss += id >= a.vocab ? __uint_as_float(0x7fc00000u) : t * (log_t - logp_of(to_f<T>(row[id])));
        }
      loss = warp_sum(loss);
      if (lane == 0) a.logp[r] = loss;
    }
  }
}

struct GradArgs {
  StatsArgs f;
  const float* dlogp;  // or dloss
  const float* dentropy;
  const float* dtop;
  void* out;
  int splits;
};

// d logits = (sum_e coef_e 1[id_e] - p (sum_e coef_e + dH (log p + H))) / T for the log probabilities (an entry e per given token and per
// alternative); dloss (q - sum_j t_j 1[id_j]) / T for the distillation.
template <typename T, bool DISTILL>
__global__ void __launch_bounds__(kThreads) row_grad_kernel(const GradArgs g) {
  constexpr int V = Vec16<T>::N;
  constexpr int kEntries = DISTILL ? kMaxTeacher : kMaxTop + 1;
  __shared__ int col[kEntries];
  __shared__ float coef[kEntries];
  const StatsArgs& a = g.f;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / g.splits;
  const int part_of = (int)(blockIdx.x % g.splits);
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* out = reinterpret_cast<T*>(g.out) + r * (int64_t)a.vocab;
  const int per = ((a.vocab + g.splits - 1) / g.splits + 63) / 64 * 64;
  const int lo = min(a.vocab, part_of * per), hi = part_of == g.splits - 1 ? a.vocab : min(a.vocab, lo + per);
  const float4 st = a.stats[r];
  const bool none = st.x == -INFINITY;
  const float dl = g.dlogp ? g.dlogp[r] : 0.f, dh = !DISTILL && g.dentropy ? g.dentropy[r] : 0.f;
  int n;
  float on_p;  // gradient = p (on_p + on_plogp log2 p) + entries
  if constexpr (DISTILL) {
    n = a.top_k;
    bool any = true;
    if (tid < 32) {
      float top, lns;
      teacher_softmax(a, r, tid, coef, top, lns, any);
    }
    any = __syncthreads_or(tid < 32 && any);
    on_p = any ? dl * a.inv_t : 0.f;
    for (int j = tid; j < n; j += kThreads) {
      const int64_t id = a.ids[r * n + j];
      coef[j] = -coef[j] * dl * a.inv_t;
      col[j] = id < 0 || id >= a.vocab ? -1 : (int)id;
    }
    // an id outside of the vocabulary made the loss NaN
    bool bad = false;
    for (int j = tid; j < n; j += kThreads) bad = bad || a.ids[r * n + j] >= a.vocab;
    if (__syncthreads_or(bad)) on_p = __uint_as_float(0x7fc00000u);
  } else {
    const int k = g.dtop ? a.top_k : 0;
    n = k + 1;
    float sum = 0.f;
    const int64_t t = a.targets[r];
    const bool in = t >= 0 && t < a.vocab;
    const float dt = t == a.ignore ? 0.f : in ? dl : __uint_as_float(0x7fc00000u);
    for (int j = 0; j < k; ++j) sum += g.dtop[r * k + j];
    on_p = -(sum + dt + dh * st.z) * a.inv_t;
    for (int j = tid; j < n; j += kThreads) {
      coef[j] = (j < k ? g.dtop[r * k + j] : dt) * a.inv_t;
      col[j] = j < k ? (int)a.top_ids[r * k + j] : in && t != a.ignore ? (int)t : -1;
    }
  }
  const float on_plogp = -dh * kLn2 * a.inv_t, c = a.c;
  const float base = none ? 0.f : st.x;
  auto grad = [&](float x) {
    const float e = fmaf(x - base, c, -st.y);
    const float p = ex2_approx(e);
    return none ? 0.f : p * fmaf(on_plogp, fmaxf(e, -1e30f), on_p);
  };
  // the rows of the gradient are dense, those of the logits need not be: whole pieces where both lie alike
  const bool alike = (reinterpret_cast<uintptr_t>(row + lo) % 16) == (reinterpret_cast<uintptr_t>(out + lo) % 16);
  auto one = [&](float x, int id) { out[id] = from_f<T>(grad(x)); };
  auto piece = [&](const auto& f, const int* ids, auto pieces) {
#pragma unroll
    for (int p = 0; p < decltype(pieces)::value; ++p) {
      float d[V];
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = grad(f[p][j]);
      if (alike) {
        Vec16<T> o;
        o.pack(d);
        o.store_stream(out + ids[p]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) out[ids[p] + j] = from_f<T>(d[j]);
      }
    }
  };
  walk<T, kUnroll>(row, lo, hi, tid, kThreads, one, piece);
  __syncthreads();  // the entries' columns are written again, with all that falls on them; a column given several times by its first entry
  if (none) return;
  for (int j = tid; j < n; j += kThreads) {
    const int id = col[j];
    if (id < lo || id >= hi) continue;
    float add = 0.f;
    bool first = true;
    for (int i = 0; i < n; ++i) {
      if (col[i] != id) continue;
      if (i < j) first = false;
      add += coef[i];
    }
    if (first) out[id] = from_f<T>(grad(to_f<T>(row[id])) + add);
  }
}

// CTAs a row: as many as keep about two waves of CTAs busy, each with at least 4096 elements
int splits_of(int64_t rows, int vocab, int most) {
  int n = 1;
  while (n < most && rows * n * 2 <= 2 * sm_count() && vocab / (n * 2) >= 4096) n *= 2;
  return n;
}

template <typename T, int FLAGS, bool DISTILL>
int launch_stats(const StatsArgs& a, cudaStream_t st) {
  const int cluster = splits_of(a.rows, a.vocab, 8);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * cluster)), cfg.blockDim = dim3(kThreads), cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, row_stats_kernel<T, FLAGS, DISTILL>, a, cluster);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("row_stats_kernel: %s", cudaGetErrorString(e));
    return (int)e;
  }
  return launch_status("row_stats_kernel");
}
template <int FLAGS, bool DISTILL>
int stats_of(const StatsArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case SSM_F32: return launch_stats<float, FLAGS, DISTILL>(a, st);
    case SSM_BF16: return launch_stats<__nv_bfloat16, FLAGS, DISTILL>(a, st);
    default: return launch_stats<__half, FLAGS, DISTILL>(a, st);
  }
}
template <bool DISTILL>
int grad_of(GradArgs& g, int dtype, cudaStream_t st) {
  g.splits = splits_of(g.f.rows, g.f.vocab, 64);
  const dim3 grid((unsigned)(g.f.rows * g.splits));
  switch (dtype) {
    case SSM_F32: row_grad_kernel<float, DISTILL><<<grid, kThreads, 0, st>>>(g); break;
    case SSM_BF16: row_grad_kernel<__nv_bfloat16, DISTILL><<<grid, kThreads, 0, st>>>(g); break;
    default: row_grad_kernel<__half, DISTILL><<<grid, kThreads, 0, st>>>(g);
  }
  return launch_status("row_grad_kernel");
}

int check_rows(int64_t rows, int64_t stride, int vocab, int dtype, float temperature) {
  SSM_REQUIRE(rows >= 0 && vocab >= 1, SSM_ERR_SHAPE, "logits must have at least one column");
  SSM_REQUIRE(rows <= (1 << 28) && vocab <= 0x7fffff00, SSM_ERR_TOO_LARGE, "logits: more than 2^28 rows or 2^31 columns");
  SSM_REQUIRE(stride >= 0, SSM_ERR_SHAPE, "logits: negative row stride");
  SSM_REQUIRE(valid_dtype(dtype), SSM_ERR_DTYPE, "logits: unknown dtype");
  SSM_REQUIRE(temperature > 0.f && temperature <= 3e38f, SSM_ERR_SHAPE, "temperature must be positive and finite");
  return SSM_OK;
}
int fill(const ssm_token_logp_args& a, StatsArgs& s) {
  if (const int rc = check_rows(a.rows, a.row_stride, a.vocab, a.io_dtype, a.temperature)) return rc;
  SSM_REQUIRE(a.top_k >= 0 && a.top_k <= a.vocab, SSM_ERR_SHAPE, "token_log_probs: top_k must lie between 0 and the vocabulary's size");
  SSM_REQUIRE(a.top_k <= kMaxTop, SSM_ERR_TOO_LARGE, "token_log_probs: top_k is at most 128");
  SSM_REQUIRE(a.rows == 0 || (a.logits && a.targets), SSM_ERR_NULL, "token_log_probs: NULL pointer");
  SSM_REQUIRE(aligned_to(a.logits, dtype_size(a.io_dtype)) && aligned_to(a.stats, 16), SSM_ERR_ALIGN, "token_log_probs: misaligned pointer");
  s.rows = a.rows, s.row_stride = a.row_stride, s.ignore = a.ignore_index, s.vocab = a.vocab, s.top_k = a.top_k;
  s.inv_t = 1.f / a.temperature, s.c = kLog2e / a.temperature;
  s.logits = a.logits, s.targets = a.targets, s.logp = a.logp, s.entropy = a.entropy, s.top_logp = a.top_logp, s.top_ids = a.top_ids;
  s.stats = reinterpret_cast<float4*>(a.stats);
  return SSM_OK;
}
int fill(const ssm_topk_distill_args& a, StatsArgs& s) {
  if (const int rc = check_rows(a.rows, a.row_stride, a.vocab, a.io_dtype, a.temperature)) return rc;
  SSM_REQUIRE(a.top_k >= 1, SSM_ERR_SHAPE, "topk_distill_loss: the teacher must have at least one entry a row");
  SSM_REQUIRE(a.top_k <= kMaxTeacher, SSM_ERR_TOO_LARGE, "topk_distill_loss: at most 1024 teacher entries a row");
  SSM_REQUIRE(valid_dtype(a.teacher_dtype), SSM_ERR_DTYPE, "topk_distill_loss: unknown teacher dtype");
  SSM_REQUIRE(a.rows == 0 || (a.logits && a.teacher && a.ids), SSM_ERR_NULL, "topk_distill_loss: NULL pointer");
  SSM_REQUIRE(aligned_to(a.logits, dtype_size(a.io_dtype)) && aligned_to(a.stats, 16), SSM_ERR_ALIGN, "topk_distill_loss: misaligned pointer");
  s.rows = a.rows, s.row_stride = a.row_stride, s.vocab = a.vocab, s.top_k = a.top_k, s.teacher_dtype = a.teacher_dtype;
  s.inv_t = 1.f / a.temperature, s.c = kLog2e / a.temperature;
  s.logits = a.logits, s.teacher = a.teacher, s.ids = a.ids, s.logp = a.loss, s.stats = reinterpret_cast<float4*>(a.stats);
  return SSM_OK;
}

}  // namespace
}  // namespace ssmb

using namespace ssmb;

extern "C" int ssm_b200_lm_abi_version(void) { return SSM_B200_LM_ABI_VERSION; }

extern "C" int ssm_token_logp(const ssm_token_logp_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "token_log_probs: NULL arguments");
  StatsArgs s{};
  if (const int rc = fill(*args, s)) return rc;
  if (s.rows == 0) return SSM_OK;
  SSM_REQUIRE(s.logp && (s.top_k == 0 || (s.top_logp && s.top_ids)), SSM_ERR_NULL, "token_log_probs: NULL output");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (s.top_k) return s.entropy ? stats_of<kTop | kEntropy, false>(s, args->io_dtype, st) : stats_of<kTop, false>(s, args->io_dtype, st);
  return s.entropy ? stats_of<kEntropy, false>(s, args->io_dtype, st) : stats_of<0, false>(s, args->io_dtype, st);
}

extern "C" int ssm_token_logp_bwd(const ssm_token_logp_bwd_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "token_log_probs: NULL arguments");
  GradArgs g{};
  if (const int rc = fill(args->fwd, g.f)) return rc;
  if (g.f.rows == 0) return SSM_OK;
  SSM_REQUIRE(args->dlogits && g.f.stats && (!args->dtop_logp || g.f.top_ids), SSM_ERR_NULL, "token_log_probs backward: NULL pointer");
  g.dlogp = args->dlogp, g.dentropy = args->dentropy, g.dtop = g.f.top_k ? args->dtop_logp : nullptr, g.out = args->dlogits;
  return grad_of<false>(g, args->fwd.io_dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ssm_topk_distill(const ssm_topk_distill_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "topk_distill_loss: NULL arguments");
  StatsArgs s{};
  if (const int rc = fill(*args, s)) return rc;
  if (s.rows == 0) return SSM_OK;
  SSM_REQUIRE(s.logp, SSM_ERR_NULL, "topk_distill_loss: NULL output");
  return stats_of<0, true>(s, args->io_dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ssm_topk_distill_bwd(const ssm_topk_distill_bwd_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "topk_distill_loss: NULL arguments");
  GradArgs g{};
  if (const int rc = fill(args->fwd, g.f)) return rc;
  if (g.f.rows == 0) return SSM_OK;
  SSM_REQUIRE(args->dlogits && g.f.stats && args->dloss, SSM_ERR_NULL, "topk_distill_loss backward: NULL pointer");
  g.dlogp = args->dloss, g.out = args->dlogits;
  return grad_of<true>(g, args->fwd.io_dtype, reinterpret_cast<cudaStream_t>(stream));
}
