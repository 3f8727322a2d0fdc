// Log probabilities of given tokens (with entropy and top alternatives) and distillation from a teacher's top logits.
//
// Both are one pass over a row of logits.  With c = log2(e) / T and a running reference M (c times the largest logit so far), d = c x - M:
// s = sum 2^d and, for the entropy, w = sum d 2^d; then log2 p_i = d_i - log2 s and H = (log2 s - w / s) ln 2.  M is rounded, by at most half a step of
// its own size, but the same in every term, so that it drops out as long as 2 to that power is a number to reckon with: rows whose M is
// beyond kFar are summed once more with differences before products.  The backward pass is one more read of the row and one write of its gradient.
// Bound: HBM (two or four bytes an element each way), beside 16 exponentials a cycle and SM: 91 us of them where 8192 x 50280 bf16 logits take 126 us
// to read.  A row goes to one CTA, or to a cluster of up to eight that join their sums through distributed shared memory where the rows alone would not
// fill the GPU.
//
// Top alternatives: the k-th largest of the maxima of groups of threads bounds the k-th largest logit from below, so a second
// pass over the row (which then lies in the L2) keeps the few elements at or above it, and ranks them by (value, lowest id).
#include <cooperative_groups.h>

#include <algorithm>

#include "../../include/ssm_b200_lm.h"
#include "common.cuh"

namespace ssmb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;  // forward and backward of 8192 rows of 50280 bf16 logits: 436 us, 442 with 128, 454 with 512
constexpr int kUnroll = 4;  // 16-byte pieces a thread has in flight; with entropy and alternatives, 4096 rows and 5 of them: 107 us, 125 with two
constexpr int kCandidates = 1024;  // kept elements of a slice above the bound, and at it
constexpr int kMaxTop = 128;
constexpr int kGroups = kThreads;  // groups of threads whose maxima are looked at, at most
constexpr int kMaxTeacher = 1024;

// threads of a group: twice as many groups as alternatives
__device__ __forceinline__ int group_size(int k) { return k <= kThreads / 16 ? 8 : k <= kThreads / 8 ? 4 : k <= kThreads / 4 ? 2 : 1; }
static_assert(2 * kMaxTop <= kThreads, "a group has a thread");

enum Flags { kEntropy = 1, kTop = 2 };

// order of floats as integers: NaN above everything, -0 equal to 0
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// larger key: larger value, among equal ones the lower id
__device__ __forceinline__ uint64_t key_of(float x, int id) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~id; }

// one(x, id) for the elements [lo, hi) of a row in a ragged head and tail, piece(raw, ids) for the 16-byte pieces between, P of them requested before
// the first is used.  `lanes` threads share the work; this one is `me`.
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
    int ids[P];
#pragma unroll
    for (int p = 0; p < P; ++p) r[p].raw = src[i + p * lanes], ids[p] = at + (i + p * lanes) * V;
    piece(r, ids);
  }
  for (; i < body; i += lanes) {
    Vec16<T> r[1];
    r[0].raw = src[i];
    const int ids[1] = {at + i * V};
    piece(r, ids);
  }
  const int tail = at + body * V;
  if (me < hi - tail) one(to_f<T>(row[tail + me]), tail + me);
}

// two fp32 values in a register pair: one instruction for both
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pair_of(float x, float y) {
  pair_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void parts_of(pair_t p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
  pair_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
  pair_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// one element of a piece, chosen at run time
template <typename T>
__device__ __forceinline__ float element(const Vec16<T>& v, int j) {
  const int word = j * (int)sizeof(T) / 4;
  const uint32_t w = word < 2 ? (word == 0 ? v.raw.x : v.raw.y) : word == 2 ? v.raw.z : v.raw.w;
  if constexpr (std::is_same<T, float>::value) return __uint_as_float(w);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  else return __half2float(__ushort_as_half((uint16_t)(j & 1 ? w >> 16 : w)));
}

// the largest (BIG) or smallest value of 16-byte pieces; a NaN makes the result NaN (NAN_COUNTS), or is passed over
template <bool BIG, bool NAN_COUNTS, typename T, int P>
__device__ __forceinline__ float extreme(const Vec16<T> (&r)[P]) {
  if constexpr (std::is_same<T, float>::value) {
    float top = BIG ? -INFINITY : INFINITY;
    bool bad = false;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float f[4];
      r[p].unpack(f);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = BIG ? fmaxf(top, f[e]) : fminf(top, f[e]), bad = bad || f[e] != f[e];
    }
    return NAN_COUNTS && bad ? __uint_as_float(0x7fc00000u) : top;
  } else {
    using V2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
    auto of2 = [](V2 a, V2 b) { return !BIG ? __hmin2(a, b) : NAN_COUNTS ? __hmax2_nan(a, b) : __hmax2(a, b); };
    V2 top;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t w[4] = {r[p].raw.x, r[p].raw.y, r[p].raw.z, r[p].raw.w};
      const V2 a = of2(*reinterpret_cast<const V2*>(&w[0]), *reinterpret_cast<const V2*>(&w[1])), b = of2(*reinterpret_cast<const V2*>(&w[2]), *reinterpret_cast<const V2*>(&w[3]));
      top = p ? of2(top, of2(a, b)) : of2(a, b);
    }
    const float lo = to_f<T>(top.x), hi = to_f<T>(top.y);
    if constexpr (NAN_COUNTS) return lo != lo ? lo : hi != hi ? hi : fmaxf(lo, hi);
    else return BIG ? fmaxf(lo, hi) : fminf(lo, hi);
  }
}

// m: the largest logit seen, M: the reference of s and w, c m but no less than -kFar.  Against that one, logits far below count for nothing: beside any above it
// they do not, and rows without one are looked at again, as those with c m beyond kFar are.  A NaN in s stays
constexpr float kFar = 268435456.f;  // 2^28, rounded by 16 at most: s between 2^-16 and V 2^16, log2 s and d off by 2^-20 each
struct Sums {
  float m, M, s, w;
};
__device__ __forceinline__ Sums nothing() { return {-INFINITY, -kFar, 0.f, 0.f}; }
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const bool first = a.m >= b.m;
  const Sums &hi = first ? a : b, &lo = first ? b : a;
  const float d = lo.M - hi.M, e = ex2_approx(d);
  return {hi.m, hi.M, hi.s + lo.s * e, hi.w + e * fmaf(lo.s, fmaxf(d, -1e30f), lo.w)};
}
__device__ __forceinline__ Sums exchanged(const Sums& a, int off) {
  return {__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.M, off), __shfl_xor_sync(0xffffffffu, a.s, off), __shfl_xor_sync(0xffffffffu, a.w, off)};
}

struct StatsArgs {
  int64_t rows, row_stride, ignore;
  int vocab, top_k, teacher_dtype;
  float c, inv_t, low;  // of logits from `low` on c x is a number
  const void* logits;
  const int64_t* targets;
  const void* teacher;
  const int64_t* ids;
  float* logp;  // or the loss
  float* entropy;
  float* top_logp;
  int64_t* top_ids;
  float4* stats;  // M, log2 s, entropy, 0; m in M's place and 2 where the row was summed by differences; 1 for a row of -inf
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
  __shared__ __align__(16) float maxima[kGroups];
  __shared__ uint64_t cand[(FLAGS & kTop) ? 2 * kCandidates : 1];  // above the bound; at it
  __shared__ uint64_t best[kMaxTop];
  __shared__ uint64_t round_best[kThreads / 32];
  __shared__ int count, equals;
  __shared__ float bound_s;
  __shared__ float teach[DISTILL ? kMaxTeacher : 1];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int64_t r = blockIdx.x / cluster;
  const int part_of = (int)(blockIdx.x % cluster);
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  // slices of whole 16-byte pieces; the last takes the rest
  const int per = ((a.vocab + cluster - 1) / cluster + 63) / 64 * 64;
  const int lo = min(a.vocab, part_of * per), hi = part_of == cluster - 1 ? a.vocab : min(a.vocab, lo + per);

  const float c = a.c;
  const pair_t c2 = pair_of(c, c);
  Sums me = nothing();
  {
    pair_t s2 = pair_of(0.f, 0.f), w2 = s2, M2 = pair_of(kFar, kFar);
    auto raise = [&](float top) {
      if (top > me.m) {
        const float M = fmaxf(top * c, -kFar), d = me.M - M, e = ex2_approx(d);
        const pair_t e2 = pair_of(e, e), none = pair_of(0.f, 0.f);
        if constexpr ((FLAGS & kEntropy) != 0) w2 = fma2(e2, fma2(s2, pair_of(d, d), w2), none);
        s2 = fma2(e2, s2, none);
        me.m = top, me.M = M, M2 = pair_of(-M, -M);
      }
    };
    walk<T, kUnroll>(
        row, lo, hi, tid, kThreads,
        [&](float x, int) {
          raise(x);
          const float d = fmaf(x, c, -me.M), e = ex2_approx(d);
          s2 = add2(s2, pair_of(e, 0.f));
          if constexpr ((FLAGS & kEntropy) != 0) w2 = add2(w2, pair_of(e * fmaxf(d, -1e30f), 0.f));
        },
        [&](const auto& r, const int*) {
          constexpr int V = Vec16<T>::N, P = sizeof(r) / sizeof(r[0]);
          raise(extreme<true, false>(r));
          auto add = [&](auto masked) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
              float f[V];
              r[p].unpack(f);
#pragma unroll
              for (int j = 0; j < V; j += 2) {
                const pair_t d2 = fma2(pair_of(f[j], f[j + 1]), c2, M2);
                float d0, d1;
                parts_of(d2, d0, d1);
                const pair_t e2 = pair_of(ex2_approx(d0), ex2_approx(d1));
                s2 = add2(s2, e2);
                if constexpr ((FLAGS & kEntropy) != 0) w2 = fma2(e2, decltype(masked)::value ? pair_of(fmaxf(d0, -1e30f), fmaxf(d1, -1e30f)) : d2, w2);
              }
            }
          };
          if ((FLAGS & kEntropy) != 0 && extreme<false, false>(r) < a.low) add(std::true_type());  // 0 times -inf
          else add(std::false_type());
        });
    float x, y;
    parts_of(s2, x, y), me.s = x + y;
    parts_of(w2, x, y), me.w = x + y;
  }

  if constexpr ((FLAGS & kTop) != 0) {  // maxima of groups of threads, at least twice as many as alternatives
    const int size = group_size(a.top_k);
    float top = me.m;
    for (int off = 1; off < size; off *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (tid % size == 0) maxima[tid / size] = top;
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const Sums o = exchanged(me, off);
    me = lane & off ? join(o, me) : join(me, o);  // the same order on both sides
  }
  if (lane == 0) part[warp] = me;
  if (tid == 0) count = equals = 0, bound_s = -INFINITY;
  __syncthreads();
  if (warp == 0) {
    me = lane < kThreads / 32 ? part[lane] : nothing();
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      const Sums o = exchanged(me, off);
      me = lane & off ? join(o, me) : join(me, o);
    }
    if (lane == 0) mine = me;
  }

  if constexpr ((FLAGS & kTop) != 0) {
    const int k = a.top_k;
    const int groups = kThreads / group_size(k);
    if (tid < groups) {  // the k-th largest of the groups' maxima
      const float own = maxima[tid];
      int above = 0;
      for (int i = 0; i < groups; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&maxima[i]);
        above += (v.x > own || (v.x == own && i < tid)) + (v.y > own || (v.y == own && i + 1 < tid)) + (v.z > own || (v.z == own && i + 2 < tid)) +
                 (v.w > own || (v.w == own && i + 3 < tid));
      }
      if (above == k - 1) bound_s = own;
    }
    __syncthreads();
    const float bound = bound_s;
    auto keep = [&](float x, int id) {
      if (x == bound) {
        const int at = atomicAdd(&equals, 1);
        if (at < kCandidates) cand[kCandidates + at] = key_of(x, id);
      } else if (!(x < bound)) {  // NaN counts as the largest
        const int at = atomicAdd(&count, 1);
        if (at < kCandidates) cand[at] = key_of(x, id);
      }
    };
    walk<T, kUnroll>(row, lo, hi, tid, kThreads, keep, [&](const auto& r, const int* ids) {
      constexpr int V = Vec16<T>::N, P = sizeof(r) / sizeof(r[0]);
      if (extreme<true, true>(r) < bound) return;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float f[V];
        r[p].unpack(f);
        uint32_t reach = 0;  // a branch for each of the few, not for each element: 4096 rows, 20 alternatives: 137 us, 158
#pragma unroll
        for (int j = 0; j < V; ++j) reach |= f[j] < bound ? 0u : 1u << j;
        for (; reach; reach &= reach - 1) {
          const int j = __ffs(reach) - 1;
          keep(element(r[p], j), ids[p] + j);
        }
      }
    });
    if (tid < kMaxTop) best[tid] = 0;  // below every key
    __syncthreads();
    const int n = count;
    int m = equals;
    if (m > kCandidates) {  // many at the bound: the first of them in the row's order
      if (warp == 0) {
        int found = 0;
        for (int id = lo; id < hi && found < k; id += 32) {
          const bool is = id + lane < hi && to_f<T>(row[id + lane]) == bound;
          const uint32_t votes = __ballot_sync(0xffffffffu, is);
          const int at = found + __popc(votes & ((1u << lane) - 1));
          if (is && at < k) cand[kCandidates + at] = key_of(bound, id + lane);
          found += __popc(votes);
        }
      }
      m = k;
      __syncthreads();
    }
    if (n <= kCandidates) {
      for (int i = tid; i < n + m; i += kThreads) {  // keys differ (ids do), so ranks do
        const uint64_t own = cand[i < n ? i : kCandidates + i - n];
        int above = 0;
        for (int j = 0; j < n; ++j) above += cand[j] > own;
        if (i >= n && above < k)
          for (int j = 0; j < m; ++j) above += cand[kCandidates + j] > own;
        if (above < k) best[above] = own;
      }
    } else {  // a few threads hold most of the largest: one maximum at a time
      uint64_t last = 0;
      for (int j = 0; j < k; ++j) {
        uint64_t top = 0;
        auto look = [&](float x, int id) {
          const uint64_t key = key_of(x, id);
          if ((j == 0 || key < last) && key > top) top = key;  // NaN in the first column has the largest of keys
        };
        walk<T, 1>(row, lo, hi, tid, kThreads, look, [&](const auto& r, const int* ids) {
          constexpr int V = Vec16<T>::N;
          float f[V];
          r[0].unpack(f);
#pragma unroll
          for (int e = 0; e < V; ++e) look(f[e], ids[0] + e);
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
      for (int i = 1; i < cluster; ++i) all = join(all, *cl.map_shared_rank(&mine, i));
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

  float kind = 0.f;
  if (!(fabsf(all.M) < kFar)) {  // the whole row once more, by this CTA, with differences before products
    __syncthreads();
    auto over = [&](float v, auto f) {  // over the threads
      for (int off = 16; off >= 1; off >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
      if (lane == 0) part[warp].m = v;
      __syncthreads();
      v = part[0].m;
      for (int i = 1; i < kThreads / 32; ++i) v = f(v, part[i].m);
      __syncthreads();
      return v;
    };
    auto each = [&](auto f) {
      walk<T, 2>(row, 0, a.vocab, tid, kThreads, [&](float x, int) { f(x); }, [&](const auto& r, const int*) {
        constexpr int V = Vec16<T>::N, P = sizeof(r) / sizeof(r[0]);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          float x[V];
          r[p].unpack(x);
#pragma unroll
          for (int j = 0; j < V; ++j) f(x[j]);
        }
      });
    };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto sum = [](float x, float y) { return x + y; };
    float m = -INFINITY, bad = 0.f, s = 0.f, w = 0.f;
    each([&](float x) { m = fmaxf(m, x), bad = x != x ? 1.f : bad; });
    m = over(m, larger), bad = over(bad, larger);
    if (m != -INFINITY)
      each([&](float x) {
        const float d = (x - m) * c, e = ex2_approx(d);
        s += e, w = fmaf(e, fmaxf(d, -1e30f), w);
      });
    s = over(s, sum), w = over(w, sum);
    if (bad != 0.f) s = w = __uint_as_float(0x7fc00000u);  // beside -inf alone too
    all = {m, m, s, w};
    kind = m == -INFINITY && bad == 0.f ? 1.f : 2.f;
  }
  const bool none = kind == 1.f;
  const float log2s = none ? 0.f : log2f(all.s), entropy = none ? 0.f : kLn2 * (log2s - all.w / all.s);
  auto logp_of = [&](float x) {
    if (none) return -INFINITY;
    const float l = kLn2 * (fmaf(x, c, -all.M) - log2s);
    return kind == 2.f || l == -INFINITY ? fmaf(x - all.m, a.inv_t, -kLn2 * log2s) : l;  // c x can be beyond the numbers where x / T is not
  };
  if (tid == 0) {
    if (a.stats) a.stats[r] = make_float4(all.M, log2s, entropy, kind);
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
template <typename T, bool DISTILL, bool PLAIN>
__device__ __forceinline__ void row_grad(const GradArgs& g, const float4 st, int* col, float* coef) {
  constexpr int V = Vec16<T>::N;
  const StatsArgs& a = g.f;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / g.splits;
  const int part_of = (int)(blockIdx.x % g.splits);
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* out = reinterpret_cast<T*>(g.out) + r * (int64_t)a.vocab;
  const int per = ((a.vocab + g.splits - 1) / g.splits + 63) / 64 * 64;
  const int lo = min(a.vocab, part_of * per), hi = part_of == g.splits - 1 ? a.vocab : min(a.vocab, lo + per);
  bool none = st.w == 1.f;
  const float dl = g.dlogp ? g.dlogp[r] : 0.f, dh = !DISTILL && g.dentropy ? g.dentropy[r] : 0.f;
  int n;
  float on_p;  // gradient = p (on_p + on_plogp log2 p) + entries
  if constexpr (DISTILL) {
    n = a.top_k;
    bool any = true, bad = false;  // the loss is NaN where a teacher's sum is, and by an id outside of the vocabulary that has a weight
    if (tid < 32) {
      float top, lns;
      teacher_softmax(a, r, tid, coef, top, lns, any);
      bad = any && lns != lns;
    }
    none = !__syncthreads_or(tid < 32 && any) || none;  // nothing asked of the row, whatever its logits are
    on_p = dl * a.inv_t;
    for (int j = tid; j < n; j += kThreads) {
      const int64_t id = a.ids[r * n + j];
      bad = bad || (id >= a.vocab && coef[j] != 0.f);
      coef[j] = -coef[j] * dl * a.inv_t;
      col[j] = id < 0 || id >= a.vocab ? -1 : (int)id;
    }
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
  auto grad = [&](float x) {
    const float e = (PLAIN ? fmaf(x, c, -st.x) : (x - st.x) * c) - st.y;
    const float p = ex2_approx(e);
    if constexpr (DISTILL) return none ? 0.f : p * on_p;
    else return none ? 0.f : p * fmaf(on_plogp, fmaxf(e, -160.f), on_p);  // p is 0 from there on, and e may be -inf or, times 1 / T, beyond the numbers
  };
  // The rows of the gradient are dense, those of the logits need not be: whole pieces where both lie alike (4096 rows of 50277 bf16 logits: 148 us), single
  // elements where they do not (540 us)
  const bool alike = (reinterpret_cast<uintptr_t>(row + lo) % 16) == (reinterpret_cast<uintptr_t>(out + lo) % 16);
  auto one = [&](float x, int id) { out[id] = from_f<T>(grad(x)); };
  auto piece = [&](const auto& r, const int* ids) {
    constexpr int P = sizeof(r) / sizeof(r[0]);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float f[V];
      r[p].unpack(f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = grad(f[j]);
      if (alike) {
        Vec16<T> o;
        o.pack(f);
        o.store_stream(out + ids[p]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) out[ids[p] + j] = from_f<T>(f[j]);
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

template <typename T, bool DISTILL>
__global__ void __launch_bounds__(kThreads) row_grad_kernel(const GradArgs g) {
  constexpr int kEntries = DISTILL ? kMaxTeacher : kMaxTop + 1;
  __shared__ int col[kEntries];
  __shared__ float coef[kEntries];
  const float4 st = g.f.stats[blockIdx.x / g.splits];
  if (st.w == 2.f) row_grad<T, DISTILL, false>(g, st, col, coef);  // summed by differences
  else row_grad<T, DISTILL, true>(g, st, col, coef);
}

// CTAs a row: twice as many until there are two an SM, or fewer than 4096 elements each, or `most`.  Sums | sums with 20 alternatives | gradient, us, bf16.
// Two an SM against one: 148 rows of 151936 23 | 31 | 31 against 29 | 38 | 45; 74 of them 16 | 25 | 21 against 21 | 29 | 27.  Against four: 148 rows of 50280 14 | 19 | 16
// against 14 | 23 | 14, 296 rows of 151936 35 | 55 | 51 against 30 | 49 | 41.  A cluster of eight against four: one row of 151936 12 | 17 against 14 | 19, of
// 50280 10 | 16 against 10 | 14.  4096 elements against 2048: nothing (74 rows of 8192 10 | 12 against 10 | 14); against 8192: one row of 50280 10 | 16 | 10 against 10 | 14 | 12.
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
  SSM_REQUIRE(rows <= (1 << 28) && vocab <= (1 << 30), SSM_ERR_TOO_LARGE, "logits: more than 2^28 rows or 2^30 columns");
  SSM_REQUIRE(stride >= 0, SSM_ERR_SHAPE, "logits: negative row stride");
  SSM_REQUIRE(valid_dtype(dtype), SSM_ERR_DTYPE, "logits: unknown dtype");
  SSM_REQUIRE(temperature >= 1e-37f && temperature <= 3e38f, SSM_ERR_SHAPE, "temperature must be positive and finite, and so its inverse");
  return SSM_OK;
}
void set_temperature(StatsArgs& s, float t) {
  s.inv_t = 1.f / t, s.c = kLog2e / t;
  s.low = std::max(-1e30f, -3.3e38f / s.c);
}
int fill(const ssm_token_logp_args& a, StatsArgs& s) {
  if (const int rc = check_rows(a.rows, a.row_stride, a.vocab, a.io_dtype, a.temperature)) return rc;
  SSM_REQUIRE(a.top_k >= 0 && a.top_k <= a.vocab, SSM_ERR_SHAPE, "token_log_probs: top_k must lie between 0 and the vocabulary's size");
  SSM_REQUIRE(a.top_k <= kMaxTop, SSM_ERR_TOO_LARGE, "token_log_probs: top_k is at most 128");
  SSM_REQUIRE(a.rows == 0 || (a.logits && a.targets), SSM_ERR_NULL, "token_log_probs: NULL pointer");
  SSM_REQUIRE(aligned_to(a.logits, dtype_size(a.io_dtype)) && aligned_to(a.stats, 16) && aligned_to({a.targets, a.top_ids}, 8) && aligned_to({a.logp, a.entropy, a.top_logp}, 4), SSM_ERR_ALIGN,
              "token_log_probs: misaligned pointer");
  s.rows = a.rows, s.row_stride = a.row_stride, s.ignore = a.ignore_index, s.vocab = a.vocab, s.top_k = a.top_k;
  set_temperature(s, a.temperature);
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
  SSM_REQUIRE(aligned_to(a.logits, dtype_size(a.io_dtype)) && aligned_to(a.teacher, dtype_size(a.teacher_dtype)) && aligned_to(a.stats, 16) && aligned_to(a.ids, 8) && aligned_to(a.loss, 4),
              SSM_ERR_ALIGN, "topk_distill_loss: misaligned pointer");
  s.rows = a.rows, s.row_stride = a.row_stride, s.vocab = a.vocab, s.top_k = a.top_k, s.teacher_dtype = a.teacher_dtype;
  set_temperature(s, a.temperature);
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
  SSM_REQUIRE(aligned_to({args->dlogp, args->dentropy, args->dtop_logp}, 4) && aligned_to(args->dlogits, dtype_size(args->fwd.io_dtype)), SSM_ERR_ALIGN,
              "token_log_probs backward: misaligned pointer");
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
  SSM_REQUIRE(aligned_to(args->dloss, 4) && aligned_to(args->dlogits, dtype_size(args->fwd.io_dtype)), SSM_ERR_ALIGN, "topk_distill_loss backward: misaligned pointer");
  g.dlogp = args->dloss, g.out = args->dlogits;
  return grad_of<true>(g, args->fwd.io_dtype, reinterpret_cast<cudaStream_t>(stream));
}
