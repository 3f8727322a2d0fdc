// The norm over many tensors at once, and clipping by it.
//
// norm = sqrt(sum x^2) (or max |x|) over all elements of all tensors; clipping multiplies every element by min(1, max_norm / (norm + 1e-6)).
// Bound: HBM; one read for the norm, one more read and a write where it clips.  The tensors' places come as kernel arguments (no table to copy, so a
// capture holds everything), cut into pieces of 16 KB; a block takes a run of neighbouring pieces, sums in a fixed order and writes one partial sum, and
// whoever needs the norm adds the partial sums up itself, again in a fixed order: two launches for up to a thousand tensors, the same bits every time.
// The scaling pass walks each run from its end, so that what the first pass read last is still in the L2.
//
// Sums: sixteen bytes' squares in fp32, where they neither overflow nor vanish (a sum within 2^-100 .. 2^100); otherwise in fp64, as the sums of these are.
#include <algorithm>

#include "../../include/ssm_b200_lm.h"
#include "common.cuh"

namespace ssmb {
namespace {

constexpr int kThreads = 256, kPieceBytes = 16384, kVecs = kPieceBytes / 16 / kThreads;  // 16-byte vectors of a piece per thread
constexpr int kTensors = 1024;  // of a launch
constexpr int kMaxBlocks = 148 * 8;

struct Table {
  const void* data[kTensors];
  int64_t bytes_and_type[kTensors];  // (bytes << 2) | dtype
  uint32_t first[kTensors + 1];      // a tensor's first piece
};
struct NormArgs {
  int tensors, blocks, is_max;
};

// a tensor as its aligned 16-byte vectors and the elements before and behind them
struct Spot {
  const unsigned char* base;  // first aligned vector
  int64_t vecs;
  int dtype, head, tail;  // elements
};
__device__ __forceinline__ Spot spot_of(const Table& t, int i) {
  Spot s;
  const unsigned char* p = reinterpret_cast<const unsigned char*>(t.data[i]);
  const int64_t bytes = t.bytes_and_type[i] >> 2;
  s.dtype = (int)(t.bytes_and_type[i] & 3);
  const int shift = s.dtype == SSM_F32 ? 2 : 1;
  const int64_t before = min((int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15), bytes);
  s.base = p + before, s.vecs = (bytes - before) >> 4;
  s.head = (int)(before >> shift), s.tail = (int)((bytes - before - (s.vecs << 4)) >> shift);
  return s;
}
__device__ __forceinline__ float element_of(const void* p, int64_t i, int dtype) {
  if (dtype == SSM_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == SSM_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ int unpack(const uint4& v, int dtype, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if (dtype == SSM_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]), f[4 + i] = 0.f;
    return 4;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == SSM_BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = h.x, f[2 * i + 1] = h.y;
    }
  }
  return 8;
}

// the tensor of piece `p`, by bisection
__device__ __forceinline__ int tensor_of(const Table& t, int n, uint32_t p) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= p) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// pieces [from, to) of a block
__device__ __forceinline__ void run_of(const Table& t, const NormArgs& a, uint32_t& from, uint32_t& to) {
  const uint64_t all = t.first[a.tensors];
  from = (uint32_t)(all * blockIdx.x / a.blocks), to = (uint32_t)(all * (blockIdx.x + 1) / a.blocks);
}

struct Running {
  double sum;
  float top;  // max |x|, NaN once there is one
};
__device__ __forceinline__ void see(Running& r, float x) {
  const float a = fabsf(x);
  if (!(a <= r.top)) r.top = r.top != r.top ? r.top : a;
}
__device__ __forceinline__ double wide_squares(const float (&f)[8]) {
  double q = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) q = fma((double)f[i], (double)f[i], q);
  return q;
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_partial_kernel(const __grid_constant__ Table t, const NormArgs a, double* __restrict__ partial) {
  __shared__ double sums[kThreads / 32];
  const int tid = threadIdx.x;
  Running r{0.0, 0.f};
  uint32_t from, to;
  run_of(t, a, from, to);
  int i = from < to ? tensor_of(t, a.tensors, from) : 0;
  Spot s{};
  if (from < to) s = spot_of(t, i);
  for (uint32_t p = from; p < to; ++p) {
    while (p >= t.first[i + 1]) s = spot_of(t, ++i);
    const int64_t v0 = (int64_t)(p - t.first[i]) * (kPieceBytes / 16) + tid;
    const uint4* src = reinterpret_cast<const uint4*>(s.base);
    uint4 v[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) v[k] = v0 + k * kThreads < s.vecs ? __ldg(src + v0 + k * kThreads) : make_uint4(0, 0, 0, 0);
    float all = 0.f;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      float f[8];
      unpack(v[k], s.dtype, f);
      if constexpr (MAX) {
#pragma unroll
        for (int e = 0; e < 8; ++e) see(r, f[e]);
      } else {
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) q = fmaf(f[e], f[e], q);
        if (q >= 0x1p-100f && q <= 0x1p100f) all += q;
        else if ((v[k].x | v[k].y | v[k].z | v[k].w) != 0u) r.sum += wide_squares(f);  // rows of zeros are common
      }
    }
    if constexpr (!MAX) r.sum += (double)all;
    if (p == t.first[i]) {  // the ends, at most 14 elements
      const int shift = s.dtype == SSM_F32 ? 2 : 1;
      if (tid < s.head + s.tail) {
        const float x = tid < s.head ? element_of(s.base - (s.head << shift), tid, s.dtype) : element_of(s.base + (s.vecs << 4), tid - s.head, s.dtype);
        if constexpr (MAX) see(r, x);
        else r.sum += (double)x * (double)x;
      }
    }
  }
  double mine = r.sum;
  if constexpr (MAX) mine = r.top;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const double o = __shfl_xor_sync(0xffffffffu, mine, off);
    if constexpr (MAX) mine = mine != mine || o <= mine ? mine : o;
    else mine += o;
  }
  if (tid % 32 == 0) sums[tid / 32] = mine;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w) {
      if constexpr (MAX) mine = mine != mine || sums[w] <= mine ? mine : sums[w];
      else mine += sums[w];
    }
    partial[blockIdx.x] = mine;
  }
}

// the norm from all partial sums, by a block; every thread gets it
__device__ __forceinline__ float joined(const double* partial, int n, int is_max, double* sums) {
  const int tid = threadIdx.x;
  double mine = 0;
  for (int i = tid; i < n; i += kThreads) {
    const double o = partial[i];
    if (is_max) mine = mine != mine || o <= mine ? mine : o;
    else mine += o;
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const double o = __shfl_xor_sync(0xffffffffu, mine, off);
    if (is_max) mine = mine != mine || o <= mine ? mine : o;
    else mine += o;
  }
  if (tid % 32 == 0) sums[tid / 32] = mine;
  __syncthreads();
  mine = sums[0];
  for (int w = 1; w < kThreads / 32; ++w) {
    if (is_max) mine = mine != mine || sums[w] <= mine ? mine : sums[w];
    else mine += sums[w];
  }
  return (float)(is_max ? mine : sqrt(mine));
}

__global__ void __launch_bounds__(kThreads) norm_join_kernel(const double* partial, int n, int is_max, float* norm) {
  __shared__ double sums[kThreads / 32];
  const float v = joined(partial, n, is_max, sums);
  if (threadIdx.x == 0) *norm = v;
}

__device__ __forceinline__ uint4 scaled(const uint4& v, int dtype, float c) {
  float f[8];
  unpack(v, dtype, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] *= c;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == SSM_F32) {
      w[i] = __float_as_uint(f[i]);
    } else if (dtype == SSM_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// `n` partial sums of all launches; block 0 of the first launch writes the norm
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ Table t, const NormArgs a, const double* partial, int n, float max_norm, float* norm, const bool first) {
  __shared__ double sums[kThreads / 32];
  const int tid = threadIdx.x;
  const float v = joined(partial, n, a.is_max, sums);
  if (first && blockIdx.x == 0 && tid == 0) *norm = v;
  const float c = max_norm / (v + 1e-6f);
  if (c >= 1.f || max_norm == INFINITY) return;  // a NaN goes on: it shows in every tensor
  uint32_t from, to;
  run_of(t, a, from, to);
  if (from >= to) return;
  int i = tensor_of(t, a.tensors, to - 1);
  Spot s = spot_of(t, i);
  for (uint32_t p = to; p-- > from;) {
    while (p < t.first[i]) s = spot_of(t, --i);
    const int64_t v0 = (int64_t)(p - t.first[i]) * (kPieceBytes / 16) + tid;
    uint4* at = reinterpret_cast<uint4*>(const_cast<unsigned char*>(s.base));
    uint4 x[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      if (v0 + k * kThreads < s.vecs) x[k] = at[v0 + k * kThreads];
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      if (v0 + k * kThreads < s.vecs) at[v0 + k * kThreads] = scaled(x[k], s.dtype, c);
    if (p == t.first[i] && tid < s.head + s.tail) {
      const int shift = s.dtype == SSM_F32 ? 2 : 1;
      void* q = const_cast<unsigned char*>(tid < s.head ? s.base - (s.head << shift) : s.base + (s.vecs << 4));
      const int at_e = tid < s.head ? tid : tid - s.head;
      store_dyn(q, at_e, s.dtype, element_of(q, at_e, s.dtype) * c);
    }
  }
}

int check_list(const ssm_tensor_ref* tensors, int64_t count, const void* scratch, const float* norm) {
  SSM_REQUIRE(count >= 0 && count <= (1 << 24), SSM_ERR_SHAPE, "global_norm: bad number of tensors");
  SSM_REQUIRE((count == 0 || tensors) && scratch && norm, SSM_ERR_NULL, "global_norm: NULL pointer");
  SSM_REQUIRE(aligned_to(scratch, 8) && aligned_to(norm, 4), SSM_ERR_ALIGN, "global_norm: misaligned pointer");
  for (int64_t i = 0; i < count; ++i) {
    const ssm_tensor_ref& r = tensors[i];
    SSM_REQUIRE(valid_dtype(r.dtype), SSM_ERR_DTYPE, "global_norm: unknown dtype");
    SSM_REQUIRE(r.numel >= 0, SSM_ERR_SHAPE, "global_norm: negative size");
    SSM_REQUIRE(r.numel <= (int64_t)1 << 40, SSM_ERR_TOO_LARGE, "global_norm: more than 2^40 elements");
    SSM_REQUIRE(r.numel == 0 || r.data, SSM_ERR_NULL, "global_norm: NULL tensor");
    SSM_REQUIRE(aligned_to(r.data, dtype_size(r.dtype)), SSM_ERR_ALIGN, "global_norm: misaligned tensor");
  }
  return SSM_OK;
}
int64_t launches_of(int64_t count) { return std::max<int64_t>(1, (count + kTensors - 1) / kTensors); }

// one launch's tensors and its blocks
int fill_table(const ssm_tensor_ref* tensors, int64_t count, Table& t, NormArgs& a) {
  uint64_t pieces = 0;
  a.tensors = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].numel == 0) continue;
    const int64_t bytes = tensors[i].numel * dtype_size(tensors[i].dtype);
    t.data[a.tensors] = tensors[i].data, t.bytes_and_type[a.tensors] = bytes << 2 | tensors[i].dtype;
    t.first[a.tensors++] = (uint32_t)pieces;
    pieces += (uint64_t)(bytes + kPieceBytes - 1) / kPieceBytes;
    SSM_REQUIRE(pieces < 0xffffffffu, SSM_ERR_TOO_LARGE, "global_norm: more than 64 TB in a thousand tensors");
  }
  t.first[a.tensors] = (uint32_t)pieces;
  a.blocks = (int)std::min<uint64_t>(std::max<uint64_t>(pieces, 1), std::min(kMaxBlocks, sm_count() * 8));
  return SSM_OK;
}

int partial_sums(const ssm_tensor_ref* tensors, int64_t count, int kind, double* scratch, cudaStream_t st, int& n) {
  n = 0;
  Table t;
  for (int64_t l = 0; l < launches_of(count); ++l) {
    NormArgs a{0, 0, kind};
    if (const int rc = fill_table(tensors + l * kTensors, std::min<int64_t>(kTensors, count - l * kTensors), t, a)) return rc;
    if (kind) norm_partial_kernel<true><<<a.blocks, kThreads, 0, st>>>(t, a, scratch + n);
    else norm_partial_kernel<false><<<a.blocks, kThreads, 0, st>>>(t, a, scratch + n);
    if (const int rc = launch_status("norm_partial_kernel")) return rc;
    n += a.blocks;
  }
  return SSM_OK;
}

}  // namespace
}  // namespace ssmb

using namespace ssmb;

extern "C" int64_t ssm_global_norm_scratch_bytes(int64_t count) { return launches_of(std::max<int64_t>(count, 0)) * kMaxBlocks * (int64_t)sizeof(double); }

extern "C" int ssm_global_norm(const ssm_tensor_ref* tensors, int64_t count, int32_t is_max, void* scratch, float* norm, ssm_stream_t stream) {
  if (const int rc = check_list(tensors, count, scratch, norm)) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int n = 0;
  if (const int rc = partial_sums(tensors, count, is_max != 0, static_cast<double*>(scratch), st, n)) return rc;
  norm_join_kernel<<<1, kThreads, 0, st>>>(static_cast<double*>(scratch), n, is_max != 0, norm);
  return launch_status("norm_join_kernel");
}

extern "C" int ssm_clip_global_norm(const ssm_tensor_ref* tensors, int64_t count, int32_t is_max, float max_norm, void* scratch, float* norm, ssm_stream_t stream) {
  if (const int rc = check_list(tensors, count, scratch, norm)) return rc;
  SSM_REQUIRE(max_norm >= 0.f, SSM_ERR_SHAPE, "clip_global_norm: max_norm must not be negative");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int n = 0;
  if (const int rc = partial_sums(tensors, count, is_max != 0, static_cast<double*>(scratch), st, n)) return rc;
  Table t;
  for (int64_t l = 0; l < launches_of(count); ++l) {
    NormArgs a{0, 0, is_max != 0};
    if (const int rc = fill_table(tensors + l * kTensors, std::min<int64_t>(kTensors, count - l * kTensors), t, a)) return rc;
    clip_kernel<<<a.blocks, kThreads, 0, st>>>(t, a, static_cast<double*>(scratch), n, max_norm, norm, l == 0);
    if (const int rc = launch_status("clip_kernel")) return rc;
  }
  return SSM_OK;
}
