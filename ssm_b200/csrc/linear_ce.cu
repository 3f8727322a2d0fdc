// Cross entropy from hidden states and the head's weight, without the logits: z = h W^T, log Z = ln sum exp z, loss = log Z - z_t.
//
// Forward: one product whose tiles end in a row's maximum and sum of exponentials (of powers of two, 2^(c z - M), c = log2 e, M the maximum rounded up to a whole number); a second
// kernel joins the tiles.  Backward, from w = dloss and wz = dlog_z of a row: G = p (w + wz) - [v = t] w, dh = G W, dW = G^T h.  G is formed again by the same product, a piece of the rows at a
// time, rounded to the operands' type (its sums are held in 32 bits), and read by the two others: 2 + 6 N D V operations where 6 are the least.
// Bound: the tensor cores; for few rows, reading W.
//
// Rows that are left out are not computed: the others are packed first, behind one another (which also gives the copies their alignment), and how many
// there are is known on the device alone, so that every kernel reads it there.
//
// Products: pairs of CTAs (cta_group::2) on tiles of 256 x 256 (x 128 for narrow outputs), a CTA holding 128 rows of the accumulator; operands by TMA in the 128-byte swizzle, blocks of 64 x 64, two to
// an operand, with K innermost (h, W, G as stored) or M / N innermost (G^T, W and h as the second factor).  One thread copies, one multiplies, eight
// warps read an accumulator while the next one is formed.  fp32 operands are taken as sums of three bf16 numbers (24 bits of mantissa in all) and
// multiplied in six products, the smallest first; what is left out is below 2^-24.
#include <algorithm>

#include "../../include/ssm_b200_lm.h"
#include "ssd_common.cuh"

namespace ssmb {
namespace {

constexpr int kTile = 256, kK = 64, kStages = 6, kThreads = 384, kEpilogueWarps = 8;
constexpr int kBoxBytes = 64 * kK * 2, kStageBytes = 4 * kBoxBytes;
constexpr size_t kSmem = (size_t)kStages * kStageBytes + 1024;
constexpr int kStatus = 128;           // status of a wait that ran out
constexpr float kFar = 268435456.f;    // M of a tile is no less than minus this
constexpr int kPairs = 6;
__constant__ const signed char kPlaneA[kPairs] = {2, 0, 1, 1, 0, 0}, kPlaneB[kPairs] = {0, 2, 1, 0, 1, 0};

enum Epilogue { kStats = 0, kGrad = 1, kOut = 2 };

struct GemmArgs {
  int m_tiles, n_tiles, splits, k_blocks, bn, m_inner;
  int a_mn, b_mn;              // innermost axis of an operand: its M / N instead of K
  int a_m0, a_k0, b_k0;        // where the operands' rows begin
  int planes, fmt;             // 3 for fp32; 0 fp16, 1 bf16
  int row0, rows, k_is_rows;   // the packed rows of this call: its M, or its K
  const int* count;            // packed rows in all
  int32_t* status;
  // kStats, kGrad
  int vocab;
  const int* targets;          // of packed rows; -1: outside of the vocabulary
  float2* part;                // [128 columns][rows of this call]: M, sum 2^(c z - M)
  int part_ld;
  float* z_target;
  const float4* row;           // of packed rows: M, 1 / s, w, w + wz
  uint16_t* g;                 // [plane][row][ldg]
  int64_t ldg, g_plane;
  // kOut
  float* out;                  // [split][row][ld]
  int64_t ld, out_split;
  int out_rows, add;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t leader_address(uint32_t smem) {  // the same place in the pair's first CTA
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem), "r"(0));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_address) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_address) : "memory");
}
// a box into this CTA's shared memory, counted on a barrier of the pair's first CTA
__device__ __forceinline__ void load_box(uint32_t dst, const void* map, uint32_t leader_bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(dst), "l"(map),
               "r"(leader_bar), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  const uint32_t acc = accumulate ? 1u : 0u;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// the barrier at this place in both CTAs follows all products issued so far
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// x as a sum of three bf16 numbers; what is not finite stays in the first
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
  p[0] = __float2bfloat16_rn(x);
  const float r = x - __bfloat162float(p[0]);
  const bool finite = fabsf(r) < INFINITY;
  p[1] = __float2bfloat16_rn(finite ? r : 0.f);
  p[2] = __float2bfloat16_rn(finite ? r - __bfloat162float(p[1]) : 0.f);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct TileAt {
  int m, n, split, kb0, kb1;
};

template <int EPI, typename T, int PLANES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const __grid_constant__ GemmArgs g) {
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t ring = (tc::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t full = tc::smem_u32(bars), empty = full + 8 * kStages, tfull = empty + 8 * kStages, tempty = tfull + 16;
  const int live = min(g.rows, max(0, *g.count - g.row0));
  const int m_tiles = g.k_is_rows ? g.m_tiles : (live + kTile - 1) / kTile, k_blocks = g.k_is_rows ? (live + kK - 1) / kK : g.k_blocks;
  const int tiles = live > 0 ? m_tiles * g.n_tiles * g.splits : 0;
  constexpr int kProducts = PLANES == 1 ? 1 : kPairs;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) tc::mbar_init(full + 8 * s, 1), tc::mbar_init(empty + 8 * s, 1);
    for (int b = 0; b < 2; ++b) tc::mbar_init(tfull + 8 * b, 1), tc::mbar_init(tempty + 8 * b, 2 * kEpilogueWarps);
    gave_up = 0;
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc::smem_u32(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  tc::fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;

  auto ran_out = [&]() {
    gave_up = 1;
    *reinterpret_cast<volatile int32_t*>(g.status) = kStatus;
  };
  auto place = [&](int t) {
    TileAt p;
    const int per = m_tiles * g.n_tiles;
    p.split = t / per, t -= p.split * per;
    if (g.m_inner) p.m = t % m_tiles, p.n = t / m_tiles;
    else p.n = t % g.n_tiles, p.m = t / g.n_tiles;
    p.kb0 = (int)((int64_t)k_blocks * p.split / g.splits), p.kb1 = (int)((int64_t)k_blocks * (p.split + 1) / g.splits);
    return p;
  };

  if (warp == 0) {
    if (tc::elect_one()) {  // copies
      const int half = g.bn / 2, bytes = 2 * (2 * kBoxBytes + half * kK * 2);
      const uint32_t full0 = leader_address(full);
      int it = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        const TileAt p = place(t);
        const int am = g.a_m0 + p.m * kTile + rank * 128, bn = p.n * g.bn + rank * half;
        for (int q = 0; q < kProducts && ok; ++q) {
          const int pa = PLANES == 1 ? 0 : kPlaneA[q], pb = PLANES == 1 ? 0 : kPlaneB[q];
          for (int kb = p.kb0; kb < p.kb1; ++kb, ++it) {
            const int s = it % kStages, round = it / kStages;
            if (round > 0 && !tc::mbar_wait(empty + 8 * s, (round - 1) & 1)) {
              ran_out();
              ok = false;
              break;
            }
            if (rank == 0) tc::mbar_expect_tx(full + 8 * s, bytes);
            const uint32_t at = ring + s * kStageBytes, bar = full0 + 8 * s;
            const int ka = g.a_k0 + kb * kK, kb_at = g.b_k0 + kb * kK;
#pragma unroll
            for (int j = 0; j < 2; ++j) load_box(at + j * kBoxBytes, &ma, bar, g.a_mn ? am + 64 * j : ka, g.a_mn ? ka : am + 64 * j, pa);
            for (int j = 0; j < half / 64; ++j) load_box(at + (2 + j) * kBoxBytes, &mb, bar, g.b_mn ? bn + 64 * j : kb_at, g.b_mn ? kb_at : bn + 64 * j, pb);
          }
        }
      }
      for (int i = max(0, it - kStages); ok && i < it; ++i)  // nothing is under way when the pair parts
        if (!tc::mbar_wait(empty + 8 * (i % kStages), (i / kStages) & 1)) {
          ran_out();
          break;
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && tc::elect_one()) {  // products
      const uint32_t idesc = tc::instr_desc(kTile, g.bn, g.fmt, g.a_mn, g.b_mn);
      const uint32_t a_lbo = g.a_mn ? kBoxBytes : 16, b_lbo = g.b_mn ? kBoxBytes : 16;
      const int a_step = g.a_mn ? 128 : 2, b_step = g.b_mn ? 128 : 2;
      int it = 0, n = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, ++n) {
        const TileAt p = place(t);
        const int b = n & 1;
        if (n >= 2 && !tc::mbar_wait(tempty + 8 * b, ((n >> 1) - 1) & 1)) {
          ran_out();
          break;
        }
        tc::fence_after_sync();
        const uint32_t d = tmem + b * 256;
        const int steps = (p.kb1 - p.kb0) * kProducts;
        for (int i = 0; i < steps; ++i, ++it) {
          const int s = it % kStages;
          if (!tc::mbar_wait(full + 8 * s, (it / kStages) & 1)) {
            ran_out();
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t at = ring + s * kStageBytes;
          const uint64_t da = tc::smem_desc_sw128(at, a_lbo, 1024), db = tc::smem_desc_sw128(at + 2 * kBoxBytes, b_lbo, 1024);
#pragma unroll
          for (int kk = 0; kk < kK / 16; ++kk) mma_pair(d, da + kk * a_step, db + kk * b_step, idesc, i > 0 || kk > 0);
          commit_pair(empty + 8 * s);
        }
        if (ok) commit_pair(tfull + 8 * b);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {  // accumulators
    const uint32_t tempty0 = leader_address(tempty);
    const int half = (warp - 4) >> 2, row_in = rank * 128 + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    int n = 0;
    for (int t = pair; t < tiles; t += pairs, ++n) {
      const TileAt p = place(t);
      const int b = n & 1;
      if (!__all_sync(0xffffffffu, tc::mbar_wait(tfull + 8 * b, (n >> 1) & 1))) {
        if (lane == 0) ran_out();
        break;
      }
      tc::fence_after_sync();
      const uint32_t from = tmem + lanes + b * 256 + half * (g.bn / 2);
      const int row = p.m * kTile + row_in;
      if constexpr (EPI == kOut) {
        float* out = g.out + p.split * g.out_split + row * g.ld + p.n * g.bn + half * (g.bn / 2);
        const int cols = (int)min((int64_t)(g.bn / 2), g.ld - p.n * g.bn - half * (g.bn / 2));
        for (int c = 0; c < g.bn / 2; c += 32) {
          uint32_t v[32];
          tmem_ld32_issue(from + c, v);
          tmem_wait_ld();
          if (row < g.out_rows) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              if (c + j < cols) {
                if (g.add) asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"l"(out + c + j), "f"(__uint_as_float(v[j])), "f"(__uint_as_float(v[j + 1])),
                                        "f"(__uint_as_float(v[j + 2])), "f"(__uint_as_float(v[j + 3]))
                                        : "memory");
                else *reinterpret_cast<uint4*>(out + c + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
              }
            }
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_at(tempty0 + 8 * b);
      } else {
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32_issue(from + 32 * c, v[c]);
        tmem_wait_ld();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_at(tempty0 + 8 * b);
        const int col0 = p.n * kTile + half * 128, left = g.vocab - col0;
        const bool in = row < live;
        const int at = in ? g.targets[g.row0 + row] - col0 : -1;  // the target's column here
        if constexpr (EPI == kStats) {
          float m = -INFINITY, s = 0.f;
          if (left < 128) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (32 * c + j >= left) v[c][j] = 0xff800000u;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j) m = fmaxf(m, __uint_as_float(v[c][j]));
          const float M = fmaxf(ceilf(m * kLog2e), -kFar);
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j) s += ex2_approx(fmaf(__uint_as_float(v[c][j]), kLog2e, -M));
          if (in) {
            g.part[(int64_t)(p.n * 2 + half) * g.part_ld + row] = make_float2(M, s);
            if (at >= 0 && at < 128) {
              float z = 0.f;
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = 0; j < 32; ++j) z = 32 * c + j == at ? __uint_as_float(v[c][j]) : z;
              g.z_target[g.row0 + row] = z;
            }
          }
        } else {
          float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
          if (in) r = g.row[g.row0 + row];
          uint16_t* to = g.g + row * g.ldg + col0;
          const int room = (int)min((int64_t)128, g.ldg - col0);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float e = ex2_approx(fmaf(__uint_as_float(v[c][j]), kLog2e, -r.x)) * r.y;
              float x = e * r.w;
              if (32 * c + j == at) x -= r.z;
              v[c][j] = in && 32 * c + j < left ? __float_as_uint(x) : 0u;
            }
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              if (32 * c + j < room) {
                if constexpr (PLANES == 1) {
                  uint32_t w[4];
#pragma unroll
                  for (int k = 0; k < 4; ++k) w[k] = pack2<T>(__uint_as_float(v[c][j + 2 * k]), __uint_as_float(v[c][j + 2 * k + 1]));
                  *reinterpret_cast<uint4*>(to + 32 * c + j) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                  __nv_bfloat16 e[8][3];
#pragma unroll
                  for (int k = 0; k < 8; ++k) split3(__uint_as_float(v[c][j + k]), e[k]);
#pragma unroll
                  for (int q = 0; q < 3; ++q) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)__bfloat16_as_ushort(e[2 * k][q]) | (uint32_t)__bfloat16_as_ushort(e[2 * k + 1][q]) << 16;
                    *reinterpret_cast<uint4*>(to + q * g.g_plane + 32 * c + j) = make_uint4(w[0], w[1], w[2], w[3]);
                  }
                }
              }
            }
          }
        }
      }
    }
  }
  __syncthreads();
  if (gave_up) {  // copies that are still under way land before the pair parts
    for (int i = 0; i < 100; ++i) __nanosleep(10000);
  }
  tc::fence_before_sync();
  cluster_sync();
  tc::fence_after_sync();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

// ---- around the products ------------------------------------------------------------------------------------------------------

// Rows whose target counts, in their order, from the front of idx; the others from its end.  One block.
__global__ void __launch_bounds__(1024) rows_kernel(const int64_t* __restrict__ targets, int rows, int64_t ignore, int vocab, int* __restrict__ idx, int* __restrict__ packed, int* __restrict__ count,
                                                    float* __restrict__ row_loss, float* __restrict__ log_z, const int write) {
  __shared__ int sums[32];
  __shared__ int base_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  for (int first = 0; first < rows; first += 8192) {
    int64_t t[8];
    int mine = 0;
    const int at = first + tid * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      t[k] = at + k < rows ? targets[at + k] : ignore;
      mine += t[k] != ignore;
    }
    int scan = mine;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, scan, off);
      if (lane >= off) scan += o;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    if (warp == 0) {
      int w = sums[lane];
#pragma unroll
      for (int off = 1; off < 32; off *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, w, off);
        if (lane >= off) w += o;
      }
      sums[lane] = w;
      if (lane == 31) base_s = base + w;
    }
    __syncthreads();
    int pos = base + scan - mine + (warp ? sums[warp - 1] : 0);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (at + k < rows) {
        if (t[k] != ignore) {
          idx[pos] = at + k, packed[pos] = t[k] >= 0 && t[k] < vocab ? (int)t[k] : -1;
          ++pos;
        } else {
          idx[rows - 1 - (at + k - pos)] = at + k;
          if (write) row_loss[at + k] = 0.f, log_z[at + k] = 0.f;
        }
      }
    }
    base = base_s;
    __syncthreads();
  }
  if (tid == 0) *count = base;
}

// (rows, dim) at a stride -> planes of 16-bit elements with rows of `ld`; with idx the packed rows, and zeros behind them to the end of their tile.  A warp per row.
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) pack_kernel(const void* src, int64_t stride, int64_t rows, int dim, const int* idx, const int* count, uint16_t* dst, int64_t ld, int64_t plane) {
  const int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (r >= rows) return;
  int64_t from = r;
  bool zero = false;
  if (idx != nullptr) {
    const int n = *count;
    if (r >= (n + kTile - 1) / kTile * kTile) return;
    zero = r >= n, from = idx[r];
  }
  const T* row = reinterpret_cast<const T*>(src) + from * stride;
  uint16_t* to = dst + r * ld;
  if constexpr (PLANES == 1) {
    const uint16_t* bits = reinterpret_cast<const uint16_t*>(row);
    if (dim % 8 == 0 && reinterpret_cast<uintptr_t>(bits) % 16 == 0) {
      for (int c = lane * 8; c < dim; c += 256) {
        uint4 v = *reinterpret_cast<const uint4*>(bits + c);
        if (zero) v = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(to + c) = v;
      }
    } else {
      for (int c = lane; c < dim; c += 32) to[c] = zero ? (uint16_t)0 : bits[c];
    }
  } else {
    for (int c = lane; c < dim; c += 32) {
      __nv_bfloat16 p[3];
      split3(zero ? 0.f : to_f<T>(row[c]), p);
#pragma unroll
      for (int q = 0; q < 3; ++q) to[q * plane + c] = __bfloat16_as_ushort(p[q]);
    }
  }
}

// The tiles of a row joined: 32 rows of a call to a block, eight slices of the columns.
__global__ void __launch_bounds__(256) join_kernel(const float2* __restrict__ part, int ld, int parts, const int* __restrict__ count, int row0, int rows, const int* __restrict__ idx,
                                                   const int* __restrict__ targets, const float* __restrict__ z_target, float2* __restrict__ stats, float* __restrict__ row_loss,
                                                   float* __restrict__ log_z) {
  __shared__ float2 slices[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  const int live = min(rows, *count - row0);
  if ((int)blockIdx.x * 32 >= live) return;
  float M = -INFINITY, s = 0.f;
  if (row < live) {
#pragma unroll 4
    for (int p = slice; p < parts; p += 8) {
      const float2 v = part[(int64_t)p * ld + row];
      const float top = fmaxf(M, v.x);
      s = s * ex2_approx(M - top) + v.y * ex2_approx(v.x - top);
      M = top;
    }
  }
  slices[slice][lane] = make_float2(M, s);
  __syncthreads();
  if (slice == 0 && row < live) {
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      const float2 v = slices[w][lane];
      if (v.x == -INFINITY) continue;
      const float top = fmaxf(M, v.x);
      s = s * ex2_approx(M - top) + v.y * ex2_approx(v.x - top);
      M = top;
    }
    const int r = row0 + row, t = targets[r], out = idx[r];
    stats[r] = make_float2(M, s);
    const float ln_s = logf(s);
    // log Z - z_t as differences from M, which take no bits from a small loss
    const float z = z_target[r];
    row_loss[out] = t < 0 ? NAN : ln_s - kLn2 * fmaf(z, kLog2e, -M);
    log_z[out] = fmaf(M, kLn2, ln_s);
  }
}

// sum or mean of the rows' losses, in a fixed order and 64 bits
__global__ void __launch_bounds__(1024) reduce_kernel(const float* __restrict__ row_loss, int rows, const int* __restrict__ count, int mean, float* __restrict__ loss) {
  __shared__ double sums[32];
  double s = 0;
  for (int i = threadIdx.x; i < rows; i += 1024) s += row_loss[i];
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) s += sums[w];
    if (mean) s /= max(1, *count);
    *loss = (float)s;
  }
}

// What the backward pass needs of a packed row, and the power of two that brings the largest weight to 2^13 .. 2^14 where the pieces are fp16 (products of small weights would vanish there).
__global__ void __launch_bounds__(1024) weights_kernel(const float2* __restrict__ stats, const int* __restrict__ idx, const int* __restrict__ targets, const int* __restrict__ count, const float* __restrict__ dloss, int reduction,
                                                       const float* __restrict__ dlog_z, int has_z, int half, float4* __restrict__ row, float* __restrict__ scales) {
  __shared__ float tops[32];
  const int n = *count, tid = threadIdx.x;
  const float all = reduction == 0 ? 0.f : reduction == 1 ? dloss[0] : dloss[0] / (float)max(1, n);
  float top = 0.f;
  for (int i = tid; i < n; i += 1024) {
    const float w = reduction ? all : dloss[idx[i]], z = has_z ? dlog_z[idx[i]] : 0.f;
    top = fmaxf(top, fmaxf(fabsf(w), fabsf(w + z)));
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (tid % 32 == 0) tops[tid / 32] = top;
  __syncthreads();
  for (int w = 0; w < 32; ++w) top = fmaxf(top, tops[w]);
  float scale = 1.f;
  if (half && top > 1e-30f && top < 1e30f) scale = exp2f((float)(13 - ilogbf(top)));
  if (tid == 0) scales[0] = scale, scales[1] = 1.f / scale;
  for (int i = tid; i < n; i += 1024) {
    const float w = reduction ? all : dloss[idx[i]], z = has_z ? dlog_z[idx[i]] : 0.f;
    const float2 s = stats[i];
    const float bad = targets[i] < 0 ? NAN : 0.f;  // a target outside of the vocabulary
    row[i] = make_float4(s.x, 1.f / s.y, w * scale + bad, (w + z) * scale + bad);
  }
}

// dhidden: a packed row's partial sums joined, into its place; zeros for rows that are left out.  Rows [row0, row0 + rows) of idx.
__global__ void __launch_bounds__(256) dhidden_kernel(const float* __restrict__ part, int splits, int64_t split, int64_t ld, int dim, const int* __restrict__ idx, const int* __restrict__ count, int row0,
                                                      int rows, const float* __restrict__ scales, void* out, int dtype) {
  const int n = *count;
  const float inv = scales[1];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * dim; i += (int64_t)gridDim.x * 256) {
    const int r = (int)(i / dim), c = (int)(i - (int64_t)r * dim);
    float v = 0.f;
    if (row0 + r < n) {
      for (int s = 0; s < splits; ++s) v += part[s * split + r * ld + c];
      v *= inv;
    }
    store_dyn(out, (int64_t)idx[row0 + r] * dim + c, dtype, v);
  }
}
__global__ void __launch_bounds__(256) dweight_kernel(const float* __restrict__ sums, int64_t ld, int vocab, int dim, const int* __restrict__ count, const float* __restrict__ scales, void* out, int dtype) {
  const bool none = *count == 0;
  const float inv = scales[1];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)vocab * dim; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / dim, c = i - r * dim;
    store_dyn(out, i, dtype, none ? 0.f : sums[r * ld + c] * inv);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// (outer, inner) matrices of 16-bit elements, `planes` of them; boxes of 64 x 64
int encode(CUtensorMap* m, const void* base, int64_t inner, int64_t outer, int planes, int64_t ld, int64_t plane, int fmt) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(SSM_ERR_DEVICE, "linear_cross_entropy: cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)planes}, strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
  const cuuint32_t box[3] = {64, 64, 1}, estr[3] = {1, 1, 1};
  const CUresult rc = fn(m, fmt ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? SSM_OK : fail(SSM_ERR_DEVICE, "linear_cross_entropy: cuTensorMapEncodeTiled rejected the matrix");
}

// sizes and places of a call
struct Plan {
  int planes, fmt, pairs_at_once;
  int64_t rows, dim, vocab, ldh, ldg, ldo;  // leading dimensions: packed h, pieces of G, fp32 outputs
  bool copy_w;
  int64_t piece;      // rows of a piece, forward and backward
  int splits, bn;     // of dh = G W
  int parts;
  // offsets into scratch
  int64_t idx, packed, count, scales, h, w, part, z, row, g, dh, dw, bytes;
};
constexpr int64_t kForwardRows = 16384;

Plan plan_of(const ssm_linear_ce_args& a, bool backward) {
  Plan p{};
  p.splits = 1;
  p.planes = a.io_dtype == SSM_F32 ? 3 : 1, p.fmt = a.io_dtype != SSM_F16;
  p.rows = std::max<int64_t>(a.rows, 1), p.dim = a.dim, p.vocab = a.vocab;
  p.ldh = up(p.dim, 8), p.ldg = up(p.vocab, 64), p.ldo = up(p.dim, 4);
  p.copy_w = p.planes == 3 || a.weight_stride % 8 != 0 || a.weight_stride < a.dim || !aligned_to(a.weight, 16);
  p.parts = (int)((p.vocab + kTile - 1) / kTile) * 2;
  p.pairs_at_once = sm_count() / 2;
  p.bn = p.dim <= 128 ? 128 : 256;
  p.piece = std::min<int64_t>(up(p.rows, kTile), kForwardRows);
  if (backward) {
    const int64_t fit = std::max<int64_t>(1, SSM_LINEAR_CE_PIECE_BYTES / (p.ldg * 2 * p.planes) / kTile) * kTile;
    p.piece = up((p.rows + (p.rows + fit - 1) / fit - 1) / ((p.rows + fit - 1) / fit), kTile);  // pieces of one size
    const int64_t tiles = p.piece / kTile * ((p.dim + p.bn - 1) / p.bn), kb = (p.vocab + kK - 1) / kK;
    // as many splits of the vocabulary as leave the pairs least idle, each of at least 16 steps
    double least = 1e300;
    for (int s = 1; s <= 32 && (s == 1 || kb / s >= 16); ++s) {
      const double rounds = (double)((tiles * s + p.pairs_at_once - 1) / p.pairs_at_once);
      const double cost = rounds * ((double)kb / s + 8.0) + 0.2 * (double)s * (double)tiles;
      if (cost < least) least = cost, p.splits = s;
    }
  }
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  p.idx = take(p.rows * 4), p.packed = take(p.rows * 4), p.count = take(4), p.scales = take(8);
  p.h = take(p.planes * up(p.rows, kTile) * p.ldh * 2);
  p.w = take(p.copy_w ? p.planes * p.vocab * p.ldh * 2 : 0);
  if (!backward) {
    p.part = take((int64_t)p.parts * p.piece * 8), p.z = take(p.rows * 4);
    p.row = take(p.rows * 8);  // stats of a call that keeps none
  } else {
    p.row = take(p.rows * 16), p.g = take(p.planes * p.piece * p.ldg * 2);
    p.dh = take((int64_t)p.splits * p.piece * p.ldo * 4), p.dw = take(p.vocab * p.ldo * 4);
  }
  p.bytes = at;
  return p;
}

int check(const ssm_linear_ce_args& a) {
  SSM_REQUIRE(a.rows >= 0 && a.dim >= 1 && a.vocab >= 1 && a.hidden_stride >= 0 && a.weight_stride >= 0, SSM_ERR_SHAPE, "linear_cross_entropy: bad shape");
  SSM_REQUIRE(a.rows <= (1 << 28) && a.vocab <= (1 << 28) && a.dim <= (1 << 20), SSM_ERR_TOO_LARGE, "linear_cross_entropy: more than 2^28 rows or columns, or 2^20 channels");
  SSM_REQUIRE(valid_dtype(a.io_dtype), SSM_ERR_DTYPE, "linear_cross_entropy: unknown dtype");
  SSM_REQUIRE(a.reduction >= 0 && a.reduction <= 2, SSM_ERR_SHAPE, "linear_cross_entropy: unknown reduction");
  SSM_REQUIRE(a.weight && (a.rows == 0 || (a.hidden && a.targets)) && a.scratch && a.status, SSM_ERR_NULL, "linear_cross_entropy: NULL pointer");
  SSM_REQUIRE(aligned_to({a.hidden, a.weight}, dtype_size(a.io_dtype)) && aligned_to({a.targets, a.stats}, 8) && aligned_to({a.row_loss, a.log_z, a.loss, a.status}, 4) && aligned_to(a.scratch, 256),
              SSM_ERR_ALIGN, "linear_cross_entropy: misaligned pointer");
  return SSM_OK;
}

template <int EPI, typename T, int PLANES>
int launch_gemm(const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& g, int pairs_at_once, cudaStream_t st) {
  auto kern = gemm_kernel<EPI, T, PLANES>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  const int64_t tiles = (int64_t)g.m_tiles * g.n_tiles * g.splits;
  kern<<<(unsigned)(2 * std::min<int64_t>(tiles, pairs_at_once)), kThreads, kSmem, st>>>(ma, mb, g);
  return launch_status("linear_ce gemm_kernel");
}
template <int EPI>
int gemm_of(const Plan& p, const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& g, cudaStream_t st) {
  if (p.planes == 3) return launch_gemm<EPI, __nv_bfloat16, 3>(ma, mb, g, p.pairs_at_once, st);
  if (EPI == kGrad && p.fmt == 0) return launch_gemm<EPI, __half, 1>(ma, mb, g, p.pairs_at_once, st);
  return launch_gemm<EPI, __nv_bfloat16, 1>(ma, mb, g, p.pairs_at_once, st);
}

struct Run {
  const ssm_linear_ce_args& a;
  Plan p;
  char* base;
  CUtensorMap mh, mw;
  template <typename U>
  U* at(int64_t off) const { return reinterpret_cast<U*>(base + off); }
};
// packs the rows (and the weight, where it cannot be copied from its place) and describes them to the copies
int prepare(Run& r, bool write, cudaStream_t st) {
  const ssm_linear_ce_args& a = r.a;
  const Plan& p = r.p;
  int *idx = r.at<int>(p.idx), *count = r.at<int>(p.count);
  rows_kernel<<<1, 1024, 0, st>>>(a.targets, (int)p.rows, a.ignore_index, (int)p.vocab, idx, r.at<int>(p.packed), count, a.row_loss, a.log_z, write);
  if (const int rc = launch_status("linear_ce rows_kernel")) return rc;
  const int64_t plane_h = up(p.rows, kTile) * p.ldh, plane_w = p.vocab * p.ldh;
  auto pack = [&](const void* src, int64_t stride, int64_t rows, const int* map, uint16_t* dst, int64_t plane) {
    const unsigned grid = (unsigned)((rows + 7) / 8);
    if (p.planes == 3) pack_kernel<float, 3><<<grid, 256, 0, st>>>(src, stride, rows, (int)p.dim, map, count, dst, p.ldh, plane);
    else pack_kernel<uint16_t, 1><<<grid, 256, 0, st>>>(src, stride, rows, (int)p.dim, map, count, dst, p.ldh, plane);
    return launch_status("linear_ce pack_kernel");
  };
  if (const int rc = pack(a.hidden, a.hidden_stride, p.rows, idx, r.at<uint16_t>(p.h), plane_h)) return rc;
  if (p.copy_w)
    if (const int rc = pack(a.weight, a.weight_stride, p.vocab, nullptr, r.at<uint16_t>(p.w), plane_w)) return rc;
  if (const int rc = encode(&r.mh, r.at<void>(p.h), p.dim, p.rows, p.planes, p.ldh, plane_h, p.fmt)) return rc;
  return encode(&r.mw, p.copy_w ? r.at<void>(p.w) : a.weight, p.dim, p.vocab, p.planes, p.copy_w ? p.ldh : a.weight_stride, p.copy_w ? plane_w : p.vocab * a.weight_stride, p.fmt);
}
// z = h W^T for the packed rows [row0, row0 + rows)
GemmArgs logits_args(const Run& r, int64_t row0, int64_t rows) {
  const Plan& p = r.p;
  GemmArgs g{};
  g.m_tiles = (int)((rows + kTile - 1) / kTile), g.n_tiles = (int)((p.vocab + kTile - 1) / kTile), g.splits = 1, g.k_blocks = (int)((p.dim + kK - 1) / kK), g.bn = kTile, g.m_inner = 1;
  g.a_m0 = (int)row0, g.planes = p.planes, g.fmt = p.fmt, g.row0 = (int)row0, g.rows = (int)rows, g.count = r.at<int>(p.count), g.status = r.a.status;
  g.vocab = (int)p.vocab, g.targets = r.at<int>(p.packed);
  return g;
}

}  // namespace
}  // namespace ssmb

using namespace ssmb;

extern "C" int64_t ssm_linear_ce_scratch_bytes(const ssm_linear_ce_args* args, int32_t backward) {
  if (!args || args->rows < 0 || args->dim < 1 || args->vocab < 1) return 0;
  return plan_of(*args, backward != 0).bytes;
}

extern "C" int ssm_linear_ce_fwd(const ssm_linear_ce_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "linear_cross_entropy: NULL arguments");
  if (const int rc = check(*args)) return rc;
  const ssm_linear_ce_args& a = *args;
  SSM_REQUIRE((a.rows == 0 || (a.row_loss && a.log_z)) && (a.reduction == 0 || a.loss), SSM_ERR_NULL, "linear_cross_entropy: NULL output");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  Run r{a, plan_of(a, false), static_cast<char*>(a.scratch)};
  const Plan& p = r.p;
  if (a.rows) {
    if (const int rc = prepare(r, true, st)) return rc;
    float2* stats = a.stats ? reinterpret_cast<float2*>(a.stats) : r.at<float2>(p.row);
    for (int64_t row0 = 0; row0 < p.rows; row0 += p.piece) {
      const int64_t rows = std::min(p.piece, p.rows - row0);
      GemmArgs g = logits_args(r, row0, rows);
      g.part = r.at<float2>(p.part), g.part_ld = (int)p.piece, g.z_target = r.at<float>(p.z);
      if (const int rc = gemm_of<kStats>(p, r.mh, r.mw, g, st)) return rc;
      join_kernel<<<(unsigned)((rows + 31) / 32), 256, 0, st>>>(g.part, g.part_ld, p.parts, g.count, (int)row0, (int)rows, r.at<int>(p.idx), r.at<int>(p.packed), g.z_target, stats, a.row_loss, a.log_z);
      if (const int rc = launch_status("linear_ce join_kernel")) return rc;
    }
  }
  if (a.reduction == 0) return SSM_OK;
  if (a.rows == 0) {
    const cudaError_t e = cudaMemsetAsync(a.loss, 0, 4, st);
    return e == cudaSuccess ? SSM_OK : (set_error("linear_cross_entropy: %s", cudaGetErrorString(e)), (int)e);
  }
  reduce_kernel<<<1, 1024, 0, st>>>(a.row_loss, (int)a.rows, r.at<int>(p.count), a.reduction == 2, a.loss);
  return launch_status("linear_ce reduce_kernel");
}

extern "C" int ssm_linear_ce_bwd(const ssm_linear_ce_bwd_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "linear_cross_entropy: NULL arguments");
  if (const int rc = check(args->fwd)) return rc;
  const ssm_linear_ce_args& a = args->fwd;
  SSM_REQUIRE(valid_dtype(args->dweight_dtype), SSM_ERR_DTYPE, "linear_cross_entropy: unknown dtype");
  SSM_REQUIRE(a.rows == 0 || (a.stats && args->dloss), SSM_ERR_NULL, "linear_cross_entropy backward: NULL pointer");
  SSM_REQUIRE(aligned_to({args->dloss, args->dlog_z}, 4) && aligned_to(args->dhidden, dtype_size(a.io_dtype)) && aligned_to(args->dweight, dtype_size(args->dweight_dtype)), SSM_ERR_ALIGN,
              "linear_cross_entropy backward: misaligned pointer");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.rows == 0) {
    if (!args->dweight) return SSM_OK;
    const cudaError_t e = cudaMemsetAsync(args->dweight, 0, (size_t)a.vocab * a.dim * dtype_size(args->dweight_dtype), st);
    return e == cudaSuccess ? SSM_OK : (set_error("linear_cross_entropy: %s", cudaGetErrorString(e)), (int)e);
  }
  Run r{a, plan_of(a, true), static_cast<char*>(a.scratch)};
  const Plan& p = r.p;
  if (const int rc = prepare(r, false, st)) return rc;
  int *idx = r.at<int>(p.idx), *count = r.at<int>(p.count);
  float* scales = r.at<float>(p.scales);
  weights_kernel<<<1, 1024, 0, st>>>(reinterpret_cast<const float2*>(a.stats), idx, r.at<int>(p.packed), count, args->dloss, a.reduction, args->dlog_z ? args->dlog_z : args->dloss, args->dlog_z != nullptr,
                                     a.io_dtype == SSM_F16, r.at<float4>(p.row), scales);
  if (const int rc = launch_status("linear_ce weights_kernel")) return rc;
  CUtensorMap mg;
  if (const int rc = encode(&mg, r.at<void>(p.g), p.vocab, p.piece, p.planes, p.ldg, p.piece * p.ldg, p.fmt)) return rc;
  const int d_tiles = (int)((p.dim + p.bn - 1) / p.bn);
  for (int64_t row0 = 0; row0 < p.rows; row0 += p.piece) {
    const int64_t rows = std::min(p.piece, p.rows - row0);
    GemmArgs z = logits_args(r, row0, rows);
    z.row = r.at<float4>(p.row), z.g = r.at<uint16_t>(p.g), z.ldg = p.ldg, z.g_plane = p.piece * p.ldg;
    if (const int rc = gemm_of<kGrad>(p, r.mh, r.mw, z, st)) return rc;
    GemmArgs g{};
    g.bn = p.bn, g.n_tiles = d_tiles, g.b_mn = 1, g.planes = p.planes, g.fmt = p.fmt, g.row0 = (int)row0, g.rows = (int)rows, g.count = count, g.status = a.status, g.ld = p.ldo;
    if (args->dhidden) {  // dh = G W
      GemmArgs d = g;
      d.m_tiles = z.m_tiles, d.splits = p.splits, d.k_blocks = (int)((p.vocab + kK - 1) / kK);
      d.out = r.at<float>(p.dh), d.out_split = p.piece * p.ldo, d.out_rows = (int)rows;
      if (const int rc = gemm_of<kOut>(p, mg, r.mw, d, st)) return rc;
      dhidden_kernel<<<(unsigned)std::min<int64_t>((rows * p.dim + 255) / 256, 148 * 8), 256, 0, st>>>(d.out, d.splits, d.out_split, p.ldo, (int)p.dim, idx, count, (int)row0, (int)rows, scales,
                                                                                                       args->dhidden, a.io_dtype);
      if (const int rc = launch_status("linear_ce dhidden_kernel")) return rc;
    }
    if (args->dweight) {  // dW += G^T h
      GemmArgs d = g;
      d.m_tiles = (int)((p.vocab + kTile - 1) / kTile), d.splits = 1, d.a_mn = 1, d.k_is_rows = 1, d.b_k0 = (int)row0;
      d.out = r.at<float>(p.dw), d.out_rows = (int)p.vocab, d.add = row0 > 0;
      if (const int rc = gemm_of<kOut>(p, mg, r.mh, d, st)) return rc;
    }
  }
  if (!args->dweight) return SSM_OK;
  dweight_kernel<<<(unsigned)std::min<int64_t>((p.vocab * p.dim + 255) / 256, 148 * 16), 256, 0, st>>>(r.at<float>(p.dw), p.ldo, (int)p.vocab, (int)p.dim, count, scales, args->dweight, args->dweight_dtype);
  return launch_status("linear_ce dweight_kernel");
}
