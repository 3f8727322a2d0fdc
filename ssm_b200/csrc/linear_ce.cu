// Cross entropy from hidden states and the head's weight, without the logits: z = h W^T, log Z = ln sum exp z, loss = log Z - z_t.
//
// Forward: one product whose tiles end in a row's maximum and sum of exponentials (of powers of two, 2^(c z - M), c = log2 e, M the maximum rounded up to a whole number); a second
// kernel joins the tiles.  Backward, from w = dloss and wz = dlog_z of a row: G = p (w + wz), q = p_t (w + wz) - w; dh = G' W + q W_t, dW = G'^T h + sum q h at the targets' rows, with
// G' = G but 0 at the target.  G' is formed again by the same product, a piece of the rows at a time, rounded to the operands' type, and read by the two others:
// 2 + 6 N D V operations where 6 are the least.  q, as a rule the largest number of its row by far, keeps 32 bits and goes to the results apart (rounded into G it gave
// most of the gradients' error: 0.31e-3 in fp16 where the result's own rounding is 0.21e-3).  In fp16 a row of G' is taken times a power of two of the row's own weight, which its row of dh is
// divided by and, where the weights differ, its row of h for dW: with one power for all, rows of 2^-20 of the largest weight lost their softmax part in G'.
//
// Loss and gradient in one pass, for sums and means in bf16: what the loss is multiplied by is one number, known later, and 6 N D V do.  The first product leaves
// 2^(c z - M) in bf16 with M from the target's logit: bf16 reaches as far as fp32, so that any M within 2^60 of the maximum will do, and it needs not be known before.  A row's factor
// 1 / sum goes to h for dW (rounded to bf16 there once more: rows of dW without a target are off by 2.8e-3, 2.3e-3 in two passes, the rounding of the result being 1.65e-3), and to the result
// for dh.  Rows whose maximum is further away are noticed when their tiles are joined, and their tiles formed again.
//
// Bound: the tensor cores; for few rows, reading W.
//
// Rows that are left out are not computed: the others are packed first, behind one another (which also gives the copies their alignment), and how many
// there are is known on the device alone, so that every kernel reads it there.
//
// Launches overlap: each kernel waits for the one before ahead of its first access (7 rows: 37 -> 29 us then, 500 fp32 rows with gradients 257 -> 241), and what kernels of a call write for one
// another is not marked as constant, so that no read of it moves ahead of the wait.  Operands and packed rows are read as constants where the address, or a branch around the read, depends on a
// load behind the wait (a row's place or target, how many rows count).
//
// Products: pairs of CTAs (cta_group::2) on tiles of 256 x 256 (x 128 for narrow outputs), a CTA holding 128 rows of the accumulator; operands by TMA in the 128-byte swizzle, blocks of 64 x 64, two to
// an operand, with K innermost (h, W, G as stored) or M / N innermost (G^T, W and h as the second factor).  One thread copies, one multiplies, eight
// warps read an accumulator while the next one is formed.  Logits, and products of fp32 operands, leave the accumulator every 512 terms and are added up by the warps that read it: the tensor core
// cuts its sums off (4096 rows of 2560: the losses were off by 1.0e-6, 2.4e-7 so).  Gradients of 16-bit operands, also those that leave in fp32, are the tensor core's own sums: their terms were
// rounded to 2^-9 or 2^-12 before, and so are the logits that two passes form again for them.  fp32 operands are taken as sums of three bf16 numbers (24 bits of mantissa in all) and
// multiplied in six products, the smallest first; what is left out is below 2^-24.
#include <algorithm>
#include <cmath>

#include "../../include/ssm_b200_lm.h"
#include "ssd_common.cuh"

namespace ssmb {
namespace {

constexpr int kTile = 256, kK = 64, kStages = 6, kThreads = 384, kEpilogueWarps = 8;
constexpr int kBoxBytes = 64 * kK * 2, kStageBytes = 4 * kBoxBytes;
constexpr int kSmem = kStages * kStageBytes + 1024;
constexpr int kStagePitch = 33, kStaging = kEpilogueWarps * 32 * kStagePitch * 4;  // kOut: a warp's rows on their way to places that are not aligned
constexpr int kStatus = 128;           // status of a wait that ran out
constexpr float kFar = 536870912.f;    // 2^29: rows whose M reaches this, either way, give NaN (their logits' steps are larger than any difference that matters); M of a tile is no less than minus this
constexpr int kPairs = 6;
__constant__ const signed char kPlaneA[kPairs] = {2, 0, 1, 1, 0, 0}, kPlaneB[kPairs] = {0, 2, 1, 0, 1, 0};

enum Epilogue { kStats = 0, kGrad = 1, kOut = 2, kKeep = 3, kFew = 4 };  // kFew: kStats with the weight's rows as M
// Up to which rows it is taken; a tile has no room for more.  Both sides, 7 / 32 / 64 rows: 50277 x 768 bf16 19 / 20 / 22 us against 33 / 33 / 34, 50280 x 2560 57 / 58 / 66 against 78 / 65 / 67,
// 16003 x 512 fp32 35 / 36 / 44 against 40 / 40 / 40 (launches replayed in a graph).
constexpr int kFewRows = 64;
constexpr int kLeastTop = -90;         // tops_kernel: no less, so that 2^(26 - top) is a number
constexpr float kReach = 60.f;         // how far a row's maximum may be from the M of the one-pass form

// one product: M x N in tiles, K in blocks of 64, cut into `splits`
struct Job {
  int m_tiles, n_tiles, splits, k_blocks, m_inner;
  int a_mn, b_mn;              // innermost axis of an operand: its M / N instead of K
  int a_m0, a_k0, b_k0;        // where the operands' rows begin
  int k_is_rows;               // the packed rows of the call are its K, not its M
  float* out;                  // kOut: [split][row][ld]
  int64_t ld, out_split;
  int out_rows, add;
  int last;                    // the last piece of dW: rounded into its place
};
struct GemmArgs {
  Job job[2];                  // kOut takes two; no tiles: none
  int bn, fmt;                 // columns of a tile; 0 fp16, 1 bf16
  int row0, rows;              // the packed rows of this call
  const int* count;            // packed rows in all
  int32_t* status;
  // kStats, kGrad, kKeep
  int vocab;
  const int* targets;          // of packed rows; -1: outside of the vocabulary
  float2* part;                // [128 columns][rows of this call]: M, sum 2^(c z - M); kKeep: the maximum, the sum; kFew: [row][32 columns]
  int part_ld;
  float* z_target;
  const float4* row;           // of packed rows: M, dh's factor, G's, q; kKeep: M
  uint16_t* g;                 // [plane][row][ldg]
  int64_t ldg, g_plane;
  const int* again;            // kKeep, nullable: the tiles of rows to be formed again
  // kOut, dW: the targets' rows, and for the last piece dw = sums scales[1]
  void* dw;
  int64_t dw_ld;
  int dw_dtype, dw_wide, dim;  // dw_wide: rows on boundaries of 16 bytes (1), of 32 (2)
  const float* scales;
  const int* heads;            // [sort][vocab]: the target's row in target_sums, or -1
  int sorts;
  const float* target_sums;    // [row][ld of the job]
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

// 32 columns, a value of each in every lane, joined over the lanes: lane l gets column l in v[0].  31 exchanges, half of the columns going on each time (a column after another
// 5 each, one waiting for the last: 43 rows, 106299 x 128: 69 us)
template <typename Join>
__device__ __forceinline__ void to_lanes(float (&v)[32], int lane, Join join) {
#pragma unroll
  for (int h = 16; h >= 1; h /= 2) {
    const bool upper = lane & h;
#pragma unroll
    for (int i = 0; i < h; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + h], h);
      v[i] = join(upper ? v[i + h] : v[i], other);
    }
  }
}

// 32 bytes; `whole`: on a boundary of 32, else of 16.  The rows of a warp's threads lie apart, so that halves of a sector would be two writes
__device__ __forceinline__ void put_sector(void* to, const uint32_t (&w)[8], bool whole) {
  if (whole) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
  } else {
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    *(reinterpret_cast<uint4*>(to) + 1) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

struct TileAt {
  int job, m, n, split, kb0, kb1;  // job -1: no more
};

// 32 columns of a row of dW from `col` on, of which `cols` are there: the targets' part
__device__ __forceinline__ void add_columns(const float* from, int cols, uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    if (i < cols) {  // the rows of these buffers have room for whole pieces
      const float4 o = *reinterpret_cast<const float4*>(from + i);
      v[i] = __float_as_uint(__uint_as_float(v[i]) + o.x), v[i + 1] = __float_as_uint(__uint_as_float(v[i + 1]) + o.y);
      v[i + 2] = __float_as_uint(__uint_as_float(v[i + 2]) + o.z), v[i + 3] = __float_as_uint(__uint_as_float(v[i + 3]) + o.w);
    }
  }
}
// where the targets' part of a row of dW is, in each sort of a piece (two at most); -1: nowhere
struct Heads {
  int at[2];
};
__device__ __forceinline__ Heads heads_of(const GemmArgs& g, const Job& j, int row) {
  Heads h{{-1, -1}};
  if (row < j.out_rows) {
    h.at[0] = g.heads[row];
    if (g.sorts > 1) h.at[1] = g.heads[(int64_t)j.out_rows + row];
  }
  return h;
}
__device__ __forceinline__ void add_target(const GemmArgs& g, const Job& j, const Heads& h, int64_t col, uint32_t (&v)[32]) {
  const int cols = (int)min((int64_t)32, g.dim - col);
#pragma unroll
  for (int b = 0; b < 2; ++b)
    if (h.at[b] >= 0) add_columns(g.target_sums + h.at[b] * j.ld + col, cols, v);
}
template <typename O>
__device__ __forceinline__ void put_column(O* to, int64_t ld, const float* from, int rows) {
#pragma unroll 8
  for (int r = 0; r < rows; ++r, to += ld) *to = from_f<O>(from[r * kStagePitch]);
}
// ... and their way into dW, a warp's 32 rows from `row0` on.  Rows that are not aligned go through shared memory, so that a warp writes neighbouring columns (20 rows, 30855 x 1219 bf16:
// the product with a thread to a row 645 us, so 113)
__device__ __forceinline__ void last_columns(const GemmArgs& g, const Job& j, bool add, int row0, int64_t col, uint32_t (&v)[32], float* staging) {
  const int cols = (int)min((int64_t)32, g.dim - col), lane = threadIdx.x & 31, row = row0 + lane;
  if (cols <= 0) return;
  if (add && row < j.out_rows) add_columns(j.out + row * j.ld + col, cols, v);
  const float f = g.scales[1];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
  if (g.dw_wide && cols == 32) {
    if (row >= j.out_rows) return;
    const int64_t to = row * g.dw_ld + col;
    if (g.dw_dtype == SSM_F32) {
      float* out = reinterpret_cast<float*>(g.dw) + to;
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const uint32_t w[8] = {v[i], v[i + 1], v[i + 2], v[i + 3], v[i + 4], v[i + 5], v[i + 6], v[i + 7]};
        put_sector(out + i, w, g.dw_wide > 1);
      }
    } else {
      uint16_t* out = reinterpret_cast<uint16_t*>(g.dw) + to;
#pragma unroll
      for (int i = 0; i < 32; i += 16) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float a = __uint_as_float(v[i + 2 * k]), b = __uint_as_float(v[i + 2 * k + 1]);
          w[k] = g.dw_dtype == SSM_BF16 ? pack2<__nv_bfloat16>(a, b) : pack2<__half>(a, b);
        }
        put_sector(out + i, w, g.dw_wide > 1);
      }
    }
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i) staging[lane * kStagePitch + i] = __uint_as_float(v[i]);
    __syncwarp();
    const int rows = min(32, j.out_rows - row0);
    if (lane < cols) {
      const float* from = staging + lane;
      const int64_t to = row0 * g.dw_ld + col + lane;
      if (g.dw_dtype == SSM_F32) put_column(reinterpret_cast<float*>(g.dw) + to, g.dw_ld, from, rows);
      else if (g.dw_dtype == SSM_BF16) put_column(reinterpret_cast<__nv_bfloat16*>(g.dw) + to, g.dw_ld, from, rows);
      else put_column(reinterpret_cast<__half*>(g.dw) + to, g.dw_ld, from, rows);
    }
  }
}

template <int EPI, typename T, int PLANES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const __grid_constant__ CUtensorMap mb1, const __grid_constant__ GemmArgs g) {
  // Blocks of K between two readings of an accumulator; the logits' gradient in 16 bits asks for no more than the tensor core's own sums (1999 rows of 1024: 180 us with segments)
  constexpr int kSegment = EPI == kGrad && PLANES == 1 ? 1 << 20 : 8;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t ring = (tc::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t full = tc::smem_u32(bars), empty = full + 8 * kStages, tfull = empty + 8 * kStages, tempty = tfull + 16;
  constexpr int kProducts = PLANES == 1 ? 1 : kPairs;
  constexpr bool kSegments = EPI != kOut || PLANES > 1;

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

  pdl_wait();  // all above overlaps with the kernel before
  pdl_trigger();
  int live = min(g.rows, max(0, *g.count - g.row0));
  if (EPI == kKeep && g.again != nullptr) {
    bool any = false;
    for (int i = 0; i < (live + kTile - 1) / kTile; ++i) any = any || g.again[i] != 0;
    if (!any) live = 0;
  }
  // This pair's k-th tile.  The first job's tiles (long ones) go round the pairs; pairs that have one less of them take as many rounds of the second job's alone as fit into
  // its time, then all take turns: the tiles that run at one time stay neighbours, and share operands in the L2.
  const int m0 = (live + kTile - 1) / kTile, kb_rows = (live + kK - 1) / kK;
  const int tiles0 = live > 0 ? (g.job[0].k_is_rows || EPI == kFew ? g.job[0].m_tiles : min(g.job[0].m_tiles, m0)) * g.job[0].n_tiles * g.job[0].splits : 0;
  const int tiles1 = EPI == kOut && (live > 0 || g.job[1].last) ? (g.job[1].k_is_rows ? g.job[1].m_tiles : min(g.job[1].m_tiles, m0)) * g.job[1].n_tiles * g.job[1].splits : 0;
  const int extra = tiles0 % pairs, mine0 = tiles0 / pairs + (pair < extra ? 1 : 0);
  const int alone = EPI == kOut && extra ? g.job[0].k_blocks / g.job[0].splits / max(1, g.job[1].k_is_rows ? kb_rows : g.job[1].k_blocks) : 0;
  auto place = [&](int k) {
    TileAt p;
    int t;
    p.job = 0;
    if (k < mine0) {
      t = pair + k * pairs;
    } else {
      if (EPI != kOut) {
        p.job = -1;
        return p;
      }
      k -= mine0;
      if (pair < extra) t = alone * (pairs - extra) + k * pairs + pair;
      else if (k < alone) t = k * (pairs - extra) + pair - extra;
      else t = alone * (pairs - extra) + (k - alone) * pairs + pair;
      p.job = t < tiles1 ? 1 : -1;
      if (p.job < 0) return p;
    }
    const Job& j = g.job[p.job];
    const int m_tiles = j.k_is_rows || EPI == kFew ? j.m_tiles : min(j.m_tiles, m0), k_blocks = j.k_is_rows ? kb_rows : j.k_blocks, per = m_tiles * j.n_tiles;
    p.split = t / per, t -= p.split * per;
    if (j.m_inner) p.m = t % m_tiles, p.n = t / m_tiles;
    else p.n = t % j.n_tiles, p.m = t / j.n_tiles;
    p.kb0 = (int)((int64_t)k_blocks * p.split / j.splits), p.kb1 = (int)((int64_t)k_blocks * (p.split + 1) / j.splits);
    if (EPI == kKeep && g.again != nullptr && !g.again[p.m]) p.kb1 = p.kb0;  // nothing to do
    return p;
  };

  auto ran_out = [&]() {
    gave_up = 1;
    *reinterpret_cast<volatile int32_t*>(g.status) = kStatus;
  };

  if (warp == 0) {
    if (tc::elect_one()) {  // copies
      const int half = g.bn / 2, bytes = 2 * (2 * kBoxBytes + half * kK * 2);
      const uint32_t full0 = leader_address(full);
      int it = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const TileAt p = place(k);
        if (p.job < 0) break;
        const Job& j = g.job[p.job];
        const CUtensorMap* const map_b = EPI == kOut && p.job ? &mb1 : &mb;
        const int am = j.a_m0 + p.m * kTile + rank * 128, bn = p.n * g.bn + rank * half;
        for (int seg = p.kb0; seg < p.kb1 && ok; seg += kSegment) {
          const int end = min(seg + kSegment, p.kb1);
          for (int q = 0; q < kProducts && ok; ++q) {
            const int pa = PLANES == 1 ? 0 : kPlaneA[q], pb = PLANES == 1 ? 0 : kPlaneB[q];
            for (int kb = seg; kb < end; ++kb, ++it) {
              const int s = it % kStages, round = it / kStages;
              if (round > 0 && !tc::mbar_wait(empty + 8 * s, (round - 1) & 1)) {
                ran_out();
                ok = false;
                break;
              }
              if (rank == 0) tc::mbar_expect_tx(full + 8 * s, bytes);
              const uint32_t at = ring + s * kStageBytes, bar = full0 + 8 * s;
              const int ka = j.a_k0 + kb * kK, kb_at = j.b_k0 + kb * kK;
#pragma unroll
              for (int i = 0; i < 2; ++i) load_box(at + i * kBoxBytes, &ma, bar, j.a_mn ? am + 64 * i : ka, j.a_mn ? ka : am + 64 * i, pa);
              if (EPI == kFew) load_box(at + 2 * kBoxBytes, map_b, bar, kb_at, bn, pb);  // a box of half the rows
              else
                for (int i = 0; i < half / 64; ++i) load_box(at + (2 + i) * kBoxBytes, map_b, bar, j.b_mn ? bn + 64 * i : kb_at, j.b_mn ? kb_at : bn + 64 * i, pb);
            }
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
      int it = 0, n = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const TileAt p = place(k);
        if (p.job < 0) break;
        const Job& j = g.job[p.job];
        const uint32_t idesc = tc::instr_desc(kTile, g.bn, g.fmt, j.a_mn, j.b_mn);
        const uint32_t a_lbo = j.a_mn ? kBoxBytes : 16, b_lbo = j.b_mn ? kBoxBytes : 16;
        const int a_step = j.a_mn ? 128 : 2, b_step = j.b_mn ? 128 : 2;
        const int length = kSegments ? kSegment : p.kb1 - p.kb0;
        for (int seg = p.kb0; seg < p.kb1 && ok; seg += length, ++n) {
          const int b = n & 1, steps = (min(seg + length, p.kb1) - seg) * kProducts;
          if (n >= 2 && !tc::mbar_wait(tempty + 8 * b, ((n >> 1) - 1) & 1)) {
            ran_out();
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t d = tmem + b * 256;
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
    }
    __syncwarp();
  } else if (warp >= 4) {  // accumulators
    const uint32_t tempty0 = leader_address(tempty);
    const int half = (warp - 4) >> 2, row_in = rank * 128 + (warp & 3) * 32 + lane;
    float* const staging = reinterpret_cast<float*>(raw + (ring - tc::smem_u32(raw)) + kStages * kStageBytes) + (warp - 4) * 32 * kStagePitch;  // kOut alone has it
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    int n = 0;
    bool ok = true;
    auto arrived = [&](int b) {
      ok = __all_sync(0xffffffffu, tc::mbar_wait(tfull + 8 * b, (n >> 1) & 1));
      if (!ok && lane == 0) ran_out();
      tc::fence_after_sync();
      return ok;
    };
    auto release = [&](int b) {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_at(tempty0 + 8 * b);
    };
    for (int k = 0; ok; ++k) {
      const TileAt p = place(k);
      if (p.job < 0) break;
      if (p.kb0 == p.kb1 && EPI == kKeep) continue;
      const Job& j = g.job[p.job];
      const int row = p.m * kTile + row_in, width = g.bn / 2;
      const int64_t out_col = p.n * g.bn + half * width;
      const bool none = p.kb0 == p.kb1;  // no rows in the last piece
      const bool add = EPI == kOut && j.add && *g.count > 0;
      Heads heads{{-1, -1}};
      if (EPI == kOut && p.job) heads = heads_of(g, j, row);  // before the accumulator is there
      // a warp whose rows nobody reads: of a piece of G those up to the next block of K are (zeros), of all else those that are live
      const bool idle = EPI != kFew && !(EPI == kOut && p.job) && row - lane >= (EPI == kGrad || EPI == kKeep ? (live + kK - 1) / kK * kK : live);
      if constexpr (!kSegments) {
        const int b = n & 1;
        if (!none && !arrived(b)) break;
        const uint32_t from = tmem + lanes + b * 256 + half * width;
        float* out = j.out + p.split * j.out_split + row * j.ld + out_col;
        const int cols = (int)min((int64_t)width, j.ld - out_col);
        for (int c = 0; c < width && !idle; c += 32) {
          uint32_t v[32];
          if (none) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
          } else {
            tmem_ld32_issue(from + c, v);
            tmem_wait_ld();
          }
          if (p.job) add_target(g, j, heads, out_col + c, v);
          if (j.last) {
            last_columns(g, j, add, row - lane, out_col + c, v, staging);
          } else if (row < j.out_rows) {
            const bool whole = j.ld % 8 == 0 && reinterpret_cast<uintptr_t>(j.out) % 32 == 0;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              if (!add && c + i + 8 <= cols) {
                const uint32_t w[8] = {v[i], v[i + 1], v[i + 2], v[i + 3], v[i + 4], v[i + 5], v[i + 6], v[i + 7]};
                put_sector(out + c + i, w, whole);
              } else {
#pragma unroll
                for (int k = i; k < i + 8; k += 4) {
                  if (c + k < cols) {
                    if (add) asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"l"(out + c + k), "f"(__uint_as_float(v[k])), "f"(__uint_as_float(v[k + 1])),
                                          "f"(__uint_as_float(v[k + 2])), "f"(__uint_as_float(v[k + 3]))
                                          : "memory");
                    else *reinterpret_cast<uint4*>(out + c + k) = make_uint4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                  }
                }
              }
            }
          }
          __syncwarp();  // the next columns are read by the whole warp
        }
        if (!none) {
          release(b);
          ++n;
        }
      } else {
        constexpr int kChunks = EPI == kFew ? 1 : 4;
        uint32_t v[kChunks][32];
        for (int seg = p.kb0; seg < p.kb1 && ok; seg += kSegment, ++n) {
          const int b = n & 1;
          if (!arrived(b)) break;
          const uint32_t from = tmem + lanes + b * 256 + half * width;
          if (idle) {
          } else if (seg == p.kb0) {
            if (EPI == kFew && width == 16) {
              float w[16];
              tc::tmem_ld16(from, w);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[0][i] = __float_as_uint(w[i]), v[0][16 + i] = 0u;
            } else {
#pragma unroll
              for (int c = 0; c < kChunks; ++c)
                if (32 * c < width) tmem_ld32_issue(from + 32 * c, v[c]);
              tmem_wait_ld();
            }
          } else {
#pragma unroll
            for (int c = 0; c < 2 * kChunks; ++c) {
              if (16 * c < width) {
                float w[16];
                tc::tmem_ld16(from + 16 * c, w);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[c / 2][c % 2 * 16 + i] = __float_as_uint(__uint_as_float(v[c / 2][c % 2 * 16 + i]) + w[i]);
              }
            }
          }
          release(b);
        }
        if (!ok) break;
        if (idle) continue;
        if (EPI == kOut && none) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[c][i] = 0u;
        }
        if constexpr (EPI == kFew) {  // a thread has a row of the weight, its registers packed rows
          const int id = p.m * kTile + row_in, first = half * width, cols = min(width, live - first);
          if (cols > 0) {
            const int target = lane < cols ? g.targets[g.row0 + first + lane] - (id - lane) : -1;  // lane l for column l: a row of this warp, or none
            for (uint32_t hits = __ballot_sync(0xffffffffu, target >= 0 && target < 32); hits; hits &= hits - 1) {
              const int i = __ffs(hits) - 1;
              if (lane == __shfl_sync(0xffffffffu, target, i) && id < g.vocab) {
                float z = 0.f;
#pragma unroll
                for (int k = 0; k < 32; ++k) z = k == i ? __uint_as_float(v[0][k]) : z;
                g.z_target[g.row0 + first + i] = z;
              }
            }
            float z[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] = id < g.vocab ? __uint_as_float(v[0][i]) : -INFINITY;
            float e[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) e[i] = z[i];
            to_lanes(e, lane, [](float x, float y) { return fmaxf(x, y); });
            const float M = fmaxf(ceilf(e[0] * kLog2e), -kFar);  // of column `lane`
#pragma unroll
            for (int i = 0; i < 32; ++i) e[i] = ex2_approx(fmaf(z[i], kLog2e, -__shfl_sync(0xffffffffu, M, i)));
            to_lanes(e, lane, [](float x, float y) { return x + y; });
            if (lane < cols) g.part[(int64_t)(first + lane) * g.part_ld + (p.m * 2 + rank) * 4 + (warp & 3)] = make_float2(M, e[0]);
          }
        } else if constexpr (EPI == kOut) {
          float* out = j.out + p.split * j.out_split + row * j.ld + out_col;
          const int cols = (int)min((int64_t)width, j.ld - out_col);
          if (p.job) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (32 * c < width) add_target(g, j, heads, out_col + 32 * c, v[c]);
          }
          if (j.last) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (32 * c < width) last_columns(g, j, add, row - lane, out_col + 32 * c, v[c], staging);
          } else if (row < j.out_rows) {
#pragma unroll
            for (int i = 0; i < 128; i += 4) {
              if (i < cols) {
                float4 w = make_float4(__uint_as_float(v[i / 32][i % 32]), __uint_as_float(v[i / 32][i % 32 + 1]), __uint_as_float(v[i / 32][i % 32 + 2]), __uint_as_float(v[i / 32][i % 32 + 3]));
                float4* to = reinterpret_cast<float4*>(out + i);
                if (add) {
                  const float4 o = *to;
                  w.x += o.x, w.y += o.y, w.z += o.z, w.w += o.w;
                }
                *to = w;
              }
            }
          }
        } else {
          const int col0 = p.n * kTile + half * 128, left = g.vocab - col0;
          const bool in = row < live;
          const int at = in ? g.targets[g.row0 + row] - col0 : -1;  // the target's column here
          if constexpr (EPI == kStats) {
            float m = -INFINITY, s = 0.f;
            if (left < 128) {
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (32 * c + i >= left) v[c][i] = 0xff800000u;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i) m = fmaxf(m, __uint_as_float(v[c][i]));
            const float M = fmaxf(ceilf(m * kLog2e), -kFar);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i) s += ex2_approx(fmaf(__uint_as_float(v[c][i]), kLog2e, -M));
            if (in) {
              g.part[(int64_t)(p.n * 2 + half) * g.part_ld + row] = make_float2(M, s);
              if (at >= 0 && at < 128) {
                float z = 0.f;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                  for (int i = 0; i < 32; ++i) z = 32 * c + i == at ? __uint_as_float(v[c][i]) : z;
                g.z_target[g.row0 + row] = z;
              }
            }
          } else {
            float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
            if (in) r = g.row[g.row0 + row];
            uint16_t* to = g.g + row * g.ldg + col0;
            const int room = (int)min((int64_t)128, g.ldg - col0);
            const float f = r.z;
            float m = -INFINITY, s = 0.f;
            if (EPI == kKeep && at >= 0 && at < 128) {  // with the sum's own errors, which a loss near zero takes the difference of
              float z = 0.f;
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i) z = 32 * c + i == at ? __uint_as_float(v[c][i]) : z;
              g.z_target[g.row0 + row] = z;
            }
            if (left < 128 || !in) {  // columns behind the vocabulary, rows behind the last one: zeros
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!in || 32 * c + i >= left) v[c][i] = 0xff800000u;
              if (!in) r.x = 0.f;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float z = __uint_as_float(v[c][i]);
                float e = ex2_approx(fmaf(z, kLog2e, -r.x));
                if constexpr (EPI == kKeep) m = fmaxf(m, z), s += e;
                else e *= f;
                v[c][i] = __float_as_uint(e);
              }
              // whole sectors of 32 bytes: the rows of a warp's threads lie apart
              if constexpr (PLANES == 1) {
#pragma unroll
                for (int i = 0; i < 32; i += 16) {
                  if (32 * c + i < room) {
                    uint32_t w[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) w[q] = pack2<T>(__uint_as_float(v[c][i + 2 * q]), __uint_as_float(v[c][i + 2 * q + 1]));
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to + 32 * c + i), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]),
                                 "r"(w[7])
                                 : "memory");
                  }
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; i += 16) {
                  if (32 * c + i < room) {
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
                      uint32_t w[8];
#pragma unroll
                      for (int h = 0; h < 8; ++h) {
                        float x[2] = {__uint_as_float(v[c][i + 2 * h]), __uint_as_float(v[c][i + 2 * h + 1])};
                        w[h] = pack2<__nv_bfloat16>(x[0], x[1]);
                        x[0] -= __uint_as_float(w[h] << 16), x[1] -= __uint_as_float(w[h] & 0xffff0000u);  // what is not finite stays in the first
                        v[c][i + 2 * h] = fabsf(x[0]) < INFINITY ? __float_as_uint(x[0]) : 0u, v[c][i + 2 * h + 1] = fabsf(x[1]) < INFINITY ? __float_as_uint(x[1]) : 0u;
                      }
                      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to + q * g.g_plane + 32 * c + i), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                                   "r"(w[5]), "r"(w[6]), "r"(w[7])
                                   : "memory");
                    }
                  }
                }
              }
            }
            if (at >= 0 && at < 128) {  // the target's own part goes to the gradients apart
#pragma unroll
              for (int q = 0; q < PLANES; ++q) to[q * g.g_plane + at] = 0;
            }
            if (EPI == kKeep && in) g.part[(int64_t)(p.n * 2 + half) * g.part_ld + row] = make_float2(m, s);
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
__global__ void __launch_bounds__(1024) rows_kernel(const int64_t* targets, int rows, int64_t ignore, int vocab, int* __restrict__ idx, int* __restrict__ packed, int* __restrict__ count,
                                                    float* __restrict__ row_loss, float* __restrict__ log_z) {
  pdl_wait();
  pdl_trigger();
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
          row_loss[at + k] = 0.f, log_z[at + k] = 0.f;
        }
      }
    }
    base = base_s;
    __syncthreads();
  }
  if (tid == 0) *count = base;
}

// a row that is not aligned, by a warp, eight loads ahead of their stores (left to the compiler, 30855 rows of 1219: 66 us)
__device__ __forceinline__ void copy_bits(const uint16_t* from, int dim, int lane, bool zero, uint16_t* to) {
  for (int c = lane; c < dim; c += 256) {
    uint16_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + 32 * k < dim ? from[c + 32 * k] : (uint16_t)0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + 32 * k < dim) to[c + 32 * k] = zero ? (uint16_t)0 : v[k];
  }
}
// (rows, dim) at a stride -> planes of 16-bit elements with rows of `ld`; with idx the packed rows, and zeros behind them to the end of their tile.  A warp per row.
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) pack_kernel(const void* src, int64_t stride, int64_t rows, int dim, const int* idx, const int* count, uint16_t* dst, int64_t ld, int64_t plane) {
  pdl_wait();
  pdl_trigger();
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
      copy_bits(bits, dim, lane, zero, to);
    }
  } else if (dim % 4 == 0 && reinterpret_cast<uintptr_t>(row) % 16 == 0) {
#pragma unroll 4
    for (int c = lane * 4; c < dim; c += 128) {
      const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + c);
      const float f[4] = {v.x, v.y, v.z, v.w};
      __nv_bfloat16 p[4][3];
#pragma unroll
      for (int k = 0; k < 4; ++k) split3(zero ? 0.f : f[k], p[k]);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        *reinterpret_cast<uint2*>(to + q * plane + c) = make_uint2((uint32_t)__bfloat16_as_ushort(p[0][q]) | (uint32_t)__bfloat16_as_ushort(p[1][q]) << 16,
                                                                   (uint32_t)__bfloat16_as_ushort(p[2][q]) | (uint32_t)__bfloat16_as_ushort(p[3][q]) << 16);
    }
  } else {
    for (int c = lane; c < dim; c += 256) {  // loads ahead of the stores
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = c + 32 * k < dim && !zero ? to_f<T>(row[c + 32 * k]) : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (c + 32 * k < dim) {
          __nv_bfloat16 p[3];
          split3(f[k], p);
#pragma unroll
          for (int q = 0; q < 3; ++q) to[q * plane + c + 32 * k] = __bfloat16_as_ushort(p[q]);
        }
      }
    }
  }
}

// Both for up to 64 rows, in one launch
template <typename T, int PLANES>
__global__ void __launch_bounds__(1024) few_rows_kernel(const int64_t* targets, int rows, int64_t ignore, int vocab, const void* src, int64_t stride, int dim, int* __restrict__ idx,
                                                        int* __restrict__ packed, int* __restrict__ count, float* __restrict__ row_loss, float* __restrict__ log_z, uint16_t* dst, int64_t ld,
                                                        int64_t plane) {
  pdl_wait();
  pdl_trigger();
  __shared__ int rows_of[kFewRows];
  __shared__ int kept_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 0) {
    int base = 0;
    for (int first = 0; first < rows; first += 32) {
      const int i = first + lane;
      const int64_t t = i < rows ? targets[i] : ignore;
      const bool counts = t != ignore;
      const uint32_t votes = __ballot_sync(0xffffffffu, counts);
      const int before = base + __popc(votes & ((1u << lane) - 1));
      if (i < rows) {
        if (counts) {
          idx[before] = i, packed[before] = t >= 0 && t < vocab ? (int)t : -1, rows_of[before] = i;
        } else {
          idx[rows - 1 - (i - before)] = i;
          row_loss[i] = 0.f, log_z[i] = 0.f;
        }
      }
      base += __popc(votes);
    }
    if (lane == 0) *count = kept_s = base;
  }
  __syncthreads();
  const int n = kept_s;
  for (int r = warp; r < rows; r += 32) {  // zeros behind the last one that counts
    const T* row = reinterpret_cast<const T*>(src) + (r < n ? rows_of[r] : 0) * stride;
    if (PLANES == 1 && dim % 8 == 0 && reinterpret_cast<uintptr_t>(row) % 16 == 0) {
#pragma unroll 4
      for (int c = lane * 8; c < dim; c += 256) {
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(row) + c);
        *reinterpret_cast<uint4*>(dst + r * ld + c) = r < n ? v : make_uint4(0, 0, 0, 0);
      }
      continue;
    }
    if (PLANES == 1) {
      copy_bits(reinterpret_cast<const uint16_t*>(row), dim, lane, r >= n, dst + r * ld);
      continue;
    }
#pragma unroll 4
    for (int c = lane; c < dim; c += 32) {
      if constexpr (PLANES > 1) {
        __nv_bfloat16 p[3];
        split3(r < n ? to_f<T>(row[c]) : 0.f, p);
#pragma unroll
        for (int q = 0; q < 3; ++q) dst[q * plane + r * ld + c] = __bfloat16_as_ushort(p[q]);
      }
    }
  }
}

__device__ __forceinline__ float within_reach(float M) { return fabsf(M) < kFar ? 0.f : NAN; }

// The tiles of a row joined: 32 rows of a call to a block, 32 slices of the columns (7 rows, 394 tiles: 21 us with eight slices).
__global__ void __launch_bounds__(1024) join_kernel(const float2* part, int ld, int parts, const int* count, int row0, int rows, const int* idx,
                                                   const int* targets, const float* z_target, float4* __restrict__ stats, float* __restrict__ row_loss,
                                                   float* __restrict__ log_z) {
  pdl_wait();
  pdl_trigger();
  __shared__ float2 slices[32][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  const int live = min(rows, *count - row0);
  if ((int)blockIdx.x * 32 >= live) return;
  float M = -INFINITY, s = 0.f;
  if (row < live) {
#pragma unroll 4
    for (int p = slice; p < parts; p += 32) {
      const float2 v = part[(int64_t)p * ld + row];
      const float top = fmaxf(M, v.x);
      s = s * ex2_approx(M - top) + v.y * ex2_approx(v.x - top);
      M = top;
    }
  }
  slices[slice][lane] = make_float2(M, s);
  __syncthreads();
  if (slice == 0 && row < live) {
#pragma unroll 8
    for (int w = 1; w < 32; ++w) {
      const float2 v = slices[w][lane];
      if (v.x == -INFINITY) continue;
      const float top = fmaxf(M, v.x);
      s = s * ex2_approx(M - top) + v.y * ex2_approx(v.x - top);
      M = top;
    }
    const int r = row0 + row, t = targets[r], out = idx[r];
    const float ln_s = logf(s) + within_reach(M), z = (t < 0 ? NAN : z_target[r]) + within_reach(M);
    stats[r] = make_float4(M, s, z, 0.f);
    row_loss[out] = ln_s - kLn2 * fmaf(z, kLog2e, -M);  // log Z - z_t as differences from M, which take no bits from a small loss
    log_z[out] = fmaf(M, kLn2, ln_s);
  }
}

// The tiles of up to 64 rows joined, a block to a row
__global__ void __launch_bounds__(256) few_join_kernel(const float2* part, int parts, const int* count, const int* idx, const int* targets,
                                                       const float* z_target, float4* __restrict__ stats, float* __restrict__ row_loss, float* __restrict__ log_z) {
  pdl_wait();
  pdl_trigger();
  __shared__ float2 warps[8];
  const int r = blockIdx.x, tid = threadIdx.x;
  if (r >= *count) return;
  float M = -INFINITY, s = 0.f;
  auto add = [&](float2 v) {
    const float top = fmaxf(M, v.x);
    s = (M == top ? s : s * ex2_approx(M - top)) + (v.x == top ? v.y : v.y * ex2_approx(v.x - top));
    M = top;
  };
#pragma unroll 4
  for (int p = tid; p < parts; p += 256) add(part[(int64_t)r * parts + p]);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const float2 o = make_float2(__shfl_xor_sync(0xffffffffu, M, off), __shfl_xor_sync(0xffffffffu, s, off));
    if (tid & off) {  // the same order on both sides
      const float2 mine = make_float2(M, s);
      M = o.x, s = o.y;
      add(mine);
    } else {
      add(o);
    }
  }
  if (tid % 32 == 0) warps[tid / 32] = make_float2(M, s);
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 8; ++w) add(warps[w]);
    const int t = targets[r], out = idx[r];
    const float ln_s = logf(s) + within_reach(M), z = (t < 0 ? NAN : z_target[r]) + within_reach(M);
    stats[r] = make_float4(M, s, z, 0.f);
    row_loss[out] = ln_s - kLn2 * fmaf(z, kLog2e, -M);
    log_z[out] = fmaf(M, kLn2, ln_s);
  }
}

// ---- loss and gradient in one pass: the target's logit of packed rows, which M comes from (the product then leaves its own in z_target: 3 rows, 900 x 2048, losses of 1: off by 7.1e-6
// with this one, 1.1e-6 with that)
__global__ void __launch_bounds__(256) reference_kernel(const __nv_bfloat16* h, const __nv_bfloat16* w, int64_t ldh, int64_t ldw, int dim, const int* targets,
                                                        const int* count, int row0, int rows, float* __restrict__ z_target, float4* __restrict__ row, int* __restrict__ again) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x & 31, r = row0 + i;
  if (i >= rows) return;
  if (lane == 0 && i % kTile == 0) again[i / kTile] = 0;
  if (r >= *count) return;
  const int t = targets[r];
  const __nv_bfloat16 *a = h + r * ldh, *b = w + (int64_t)max(t, 0) * ldw;
  float z = 0.f;
  for (int c = lane * 8; c < dim; c += 256) {
    if (c + 8 <= dim) {
      Vec16<__nv_bfloat16> x, y;
      float f[8], e[8];
      x.load(a + c), y.load(b + c);
      x.unpack(f), y.unpack(e);
#pragma unroll
      for (int k = 0; k < 8; ++k) z = fmaf(f[k], e[k], z);
    } else {
      for (int k = c; k < dim; ++k) z = fmaf(__bfloat162float(a[k]), __bfloat162float(b[k]), z);
    }
  }
  z = warp_sum(z);
  if (lane == 0) {
    const float M = t < 0 || !(fabsf(z) < 1e30f) ? 0.f : ceilf(z * kLog2e);
    z_target[r] = t < 0 ? NAN : z;
    row[r] = make_float4(M, 0.f, 0.f, 0.f);
  }
}
// Its tiles joined.  A row whose maximum is too far from M gets one from its maximum, and its tile of rows is formed again; the second call (`second`) then joins those.
__global__ void __launch_bounds__(1024) join_keep_kernel(const float2* part, int ld, int parts, const int* count, int row0, int rows, const int* idx,
                                                        const float* z_target, float4* __restrict__ row, int* __restrict__ again, int second, float* __restrict__ row_loss,
                                                        float* __restrict__ log_z) {
  pdl_wait();
  pdl_trigger();
  __shared__ float2 slices[32][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  const int live = min(rows, *count - row0);
  if ((int)blockIdx.x * 32 >= live || (second && !again[blockIdx.x * 32 / kTile])) return;
  float m = -INFINITY, s = 0.f;
  if (i < live) {
#pragma unroll 4
    for (int p = slice; p < parts; p += 32) {
      const float2 v = part[(int64_t)p * ld + i];
      m = fmaxf(m, v.x), s += v.y;
    }
  }
  slices[slice][lane] = make_float2(m, s);
  __syncthreads();
  if (slice == 0 && i < live) {
#pragma unroll 8
    for (int w = 1; w < 32; ++w) m = fmaxf(m, slices[w][lane].x), s += slices[w][lane].y;
    const int r = row0 + i, out = idx[r];
    const float z = z_target[r], top = ceilf(m * kLog2e);
    float4 v = row[r];
    if (!second && fabsf(top) < 1e30f && fabsf(top - v.x) > kReach) {
      again[i / kTile] = 1;
      row[r] = make_float4(top, 0.f, 0.f, 0.f);
      return;
    }
    const float d = fmaf(z, kLog2e, -v.x), inv = s < INFINITY ? 1.f / s : NAN, ln_s = (s < INFINITY ? logf(s) : NAN) + within_reach(v.x);
    const float bad = (z != z ? NAN : 0.f) + within_reach(v.x);  // a target outside of the vocabulary, or a NaN
    v.y = inv + bad, v.z = 1.f, v.w = ex2_approx(d) * inv - 1.f;
    row[r] = v;
    row_loss[out] = ln_s - kLn2 * d;
    log_z[out] = fmaf(v.x, kLn2, ln_s);
  }
}
// Packed rows times their factors, zeros behind them to the end of their tile: 1 / sum in the one-pass form.  With `top` the other part of the rows' weights in dW's scale 2^(26 - top):
// at most 2^14 then, and exact but for elements that lie 2^28 and more below the largest product of an element and its row's weight.
template <typename T>
__global__ void __launch_bounds__(256) scaled_rows_kernel(const T* h, int64_t ld, int dim, const float4* row, const int* count, int64_t row0, int64_t rows, T* __restrict__ out,
                                                          const int* top, float* __restrict__ scales) {
  pdl_wait();
  pdl_trigger();
  const int64_t r = row0 + (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x & 31, n = *count;
  const float all = top != nullptr ? scalbnf(1.f, 26 - *top) : 1.f;
  if (top != nullptr && blockIdx.x == 0 && threadIdx.x == 0) scales[0] = all, scales[1] = 1.f / all;
  if (r >= row0 + rows || r >= (n + kTile - 1) / kTile * kTile) return;
  const bool zero = r >= n;
  const float f = zero ? 0.f : row[r].y * all;
  for (int c = lane * 8; c < dim; c += 256) {  // rows have room for whole pieces
    Vec16<T> v;
    float e[8];
    v.load(h + r * ld + c);
    v.unpack(e);
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = zero ? 0.f : e[k] * f;
    v.pack(e);
    v.store(out + r * ld + c);
  }
}

// sum or mean of the rows' losses, in a fixed order and 64 bits
__global__ void __launch_bounds__(1024) reduce_kernel(const float* row_loss, int rows, const int* count, int mean, float* __restrict__ loss) {
  pdl_wait();
  pdl_trigger();
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

// What the backward pass needs of a packed row.  Where the pieces are fp16, a power of two brings a row's weight to 2^13 .. 2^14 (products of small weights would vanish there): with
// `each` the row's own, else that of the largest weight, which all share.
__global__ void __launch_bounds__(1024) weights_kernel(const float4* stats, const int* idx, const int* count, const float* dloss, int reduction,
                                                       const float* dlog_z, int has_z, int half, int each, float4* __restrict__ row, float* __restrict__ scales) {
  pdl_wait();
  pdl_trigger();
  __shared__ float tops[32];
  const int n = *count, tid = threadIdx.x;
  const float all = reduction == 0 ? 0.f : reduction == 1 ? dloss[0] : dloss[0] / (float)max(1, n);
  float top = 0.f;
  for (int i = tid; i < n; i += 1024) {
    const float w = reduction ? all : dloss[idx[i]], z = has_z ? dlog_z[idx[i]] : 0.f;
    top = fmaxf(top, fabsf(w + z));
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (tid % 32 == 0) tops[tid / 32] = top;
  __syncthreads();
  for (int w = 0; w < 32; ++w) top = fmaxf(top, tops[w]);
  float scale = 1.f;
  if (half && !each && top > 1e-30f && top < 1e30f) scale = exp2f((float)(13 - ilogbf(top)));
  if (tid == 0) scales[0] = scale, scales[1] = 1.f / scale, reinterpret_cast<int*>(scales)[2] = kLeastTop;
  for (int i = tid; i < n; i += 1024) {
    const float w = reduction ? all : dloss[idx[i]], z = has_z ? dlog_z[idx[i]] : 0.f;
    const float4 s = stats[i];
    const float inv = 1.f / s.y, d = fmaf(s.z, kLog2e, -s.x), bad = s.z != s.z ? NAN : 0.f;  // a target outside of the vocabulary, or a NaN
    float mine = scale, back = 1.f / scale;
    if (each) {
      const int e = max(-100, min(99, ilogbf(w + z)));  // of zero, and of what is not finite, one of the two ends
      mine = scalbnf(1.f, 13 - e), back = scalbnf(1.f, e - 13);
    }
    row[i] = make_float4(s.x, back, inv * ((w + z) * mine + bad), ex2_approx(d) * inv * (w + z) - w);
  }
}
// With `each`, the largest product of a row's weight (or q, which is more where dloss and dlog_z cancel) and its largest element, as an exponent of two (0 and what is not finite left
// out): dW's scale.  A warp per packed row, bound by its start (1999 rows of 1024: 5 us, as scaled_rows_kernel behind it).
__global__ void __launch_bounds__(256) tops_kernel(const __half* h, int64_t ld, int dim, const float4* row, const int* count, int* __restrict__ top) {
  pdl_wait();
  pdl_trigger();
  const int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (r >= *count) return;
  float m = 0.f;
  for (int c = lane * 8; c < dim; c += 256) {  // rows have room for whole pieces
    Vec16<__half> v;
    float e[8];
    v.load(h + r * ld + c);
    v.unpack(e);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, c + k < dim && fabsf(e[k]) < INFINITY ? fabsf(e[k]) : 0.f);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0 && m > 0.f) {
    const float4 w = row[r];
    atomicMax(top, max(13 + ilogbf(w.y), max(-100, min(99, ilogbf(w.w)))) + ilogbf(m));
  }
}

// dhidden: a packed row's partial sums joined, times its factor, and q W_t, into its place; zeros for rows that are left out (-0 with `later`: a factor
// still to come, infinite or NaN, leaves those as they are).  Rows [row0, row0 + rows) of idx, a
// warp each.  V columns at a time.
template <int V>
__global__ void __launch_bounds__(256) dhidden_kernel(const float* part, int splits, int64_t split, int64_t ld, int dim, const int* idx, const int* targets,
                                                      const int* count, int row0, int rows, const float4* row, int later, const void* weight,
                                                      int64_t weight_stride, int weight_dtype, void* out, int dtype) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x & 31, r = row0 + i;
  if (i >= rows) return;
  const bool in = r < *count;
  const int64_t to = (int64_t)idx[r] * dim;
  const int t = in ? max(targets[r], 0) : 0;
  const float4 w = in ? row[r] : make_float4(0.f, 0.f, 0.f, 0.f);
  const float f = w.y;
  if (in && V == 4) {  // four pieces in flight
    for (int c0 = blockIdx.y * 512 + lane * 4; c0 < dim; c0 += 512 * gridDim.y) {
      float4 x[4];
      float e[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = __ldcs(reinterpret_cast<const float4*>(part + i * ld + min(c0 + 128 * k, dim - 4)));
#pragma unroll 4
      for (int s = 1; s < splits; ++s) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 o = __ldcs(reinterpret_cast<const float4*>(part + s * split + i * ld + min(c0 + 128 * k, dim - 4)));
          x[k].x += o.x, x[k].y += o.y, x[k].z += o.z, x[k].w += o.w;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) load_param_vec<4>(weight, t * weight_stride + min(c0 + 128 * k, dim - 4), weight_dtype, e[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = c0 + 128 * k;
        if (c >= dim) break;
        const float v[4] = {fmaf(w.w, e[k][0], x[k].x * f), fmaf(w.w, e[k][1], x[k].y * f), fmaf(w.w, e[k][2], x[k].z * f), fmaf(w.w, e[k][3], x[k].w * f)};
        if (dtype == SSM_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + to + c) = make_float4(v[0], v[1], v[2], v[3]);
        else
          *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + to + c) =
              dtype == SSM_BF16 ? make_uint2(pack2<__nv_bfloat16>(v[0], v[1]), pack2<__nv_bfloat16>(v[2], v[3])) : make_uint2(pack2<__half>(v[0], v[1]), pack2<__half>(v[2], v[3]));
      }
    }
    return;
  }
  for (int c = (blockIdx.y * 32 + lane) * V; c < dim; c += 32 * V * gridDim.y) {
    float v[V] = {}, e[V];
    if (!in && later) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = -0.f;
    }
    if (in) {
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const float* from = part + s * split + i * ld + c;
        if constexpr (V == 4) {
          const float4 x = *reinterpret_cast<const float4*>(from);
          v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        } else {
          v[0] += *from;
        }
      }
      if constexpr (V == 4) load_param_vec<4>(weight, t * weight_stride + c, weight_dtype, e);
      else e[0] = load_dyn(weight, t * weight_stride + c, weight_dtype);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = fmaf(w.w, e[k], v[k] * f);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) store_dyn(out, to + c + k, dtype, v[k]);
  }
}

// A call's packed rows [8192 b, ..) in the order of their targets: keys (target, packed row), all ones behind them.  A block each; eight keys to a thread, compared in registers, by shuffles
// within a warp and through shared memory beyond (8192 keys all through shared memory: 97 us).  Key: uint32_t where target and place fit.
constexpr int kSort = 8192;
template <typename Key>
__device__ __forceinline__ Key shuffled(Key v, int lanes) { return __shfl_xor_sync(0xffffffffu, v, lanes); }
template <typename Key>
__global__ void __launch_bounds__(1024) sort_kernel(const int* targets, const int* count, int row0, int rows, int size, uint64_t* __restrict__ keys) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(8) unsigned char sort_raw[];
  Key* const other = reinterpret_cast<Key*>(sort_raw);
  const int first = blockIdx.x * kSort, n = min(rows, *count - row0), tid = threadIdx.x, threads = blockDim.x;
  Key key[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = tid * 8 + e, r = first + i, t = i < size && r < n ? targets[row0 + r] : -1;
    key[e] = t >= 0 ? (Key)t << 13 | (Key)i : ~(Key)0;
  }
  auto ordered = [](Key& a, Key& b, bool up) {  // a <= b where up
    const Key lo = a < b ? a : b, hi = a < b ? b : a;
    a = up ? lo : hi, b = up ? hi : lo;
  };
  for (int k = 2; k <= size; k *= 2) {
    int j = k / 2;
    for (; j >= 256; j /= 2) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) other[e * threads + tid] = key[e];
      __syncthreads();
      const bool up = ((tid * 8) & k) == 0, low = (tid & (j / 8)) == 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Key o = other[e * threads + (tid ^ (j / 8))];
        key[e] = (key[e] < o) == (up == low) ? key[e] : o;
      }
    }
    for (; j >= 8; j /= 2) {
      const bool up = ((tid * 8) & k) == 0, low = (tid & (j / 8)) == 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Key o = shuffled(key[e], j / 8);
        key[e] = (key[e] < o) == (up == low) ? key[e] : o;
      }
    }
    if (k >= 8) {
      const bool up = ((tid * 8) & k) == 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) ordered(key[e], key[e + 4], up);
#pragma unroll
      for (int e = 0; e < 8; e += 4) ordered(key[e], key[e + 2], up), ordered(key[e + 1], key[e + 3], up);
#pragma unroll
      for (int e = 0; e < 8; e += 2) ordered(key[e], key[e + 1], up);
    } else if (k == 4) {
#pragma unroll
      for (int e = 0; e < 8; e += 4) ordered(key[e], key[e + 2], (e & 4) == 0), ordered(key[e + 1], key[e + 3], (e & 4) == 0);
#pragma unroll
      for (int e = 0; e < 8; e += 2) ordered(key[e], key[e + 1], (e & 4) == 0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) ordered(key[e], key[e + 1], (e & 2) == 0);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (tid * 8 + e < size) keys[first + tid * 8 + e] = key[e] == ~(Key)0 ? ~0ull : (uint64_t)(key[e] >> 13) << 32 | (uint32_t)(row0 + first + (int)(key[e] & (kSort - 1)));
}
// The sum of q h over the rows that have a target, in their order, at the place of the first of them, and that place by target: one block (of 128 V columns) for each run of equal
// targets, eight rows on their way at a time (a common token has hundreds).
template <int V>
__global__ void __launch_bounds__(128) target_rows_kernel(const uint64_t* keys, int size, const float4* row, const int* idx, const void* hidden, int64_t stride, int dtype,
                                                          int dim, const float* scales, float* __restrict__ sums, int64_t ld, int* __restrict__ heads, int place) {
  pdl_wait();
  pdl_trigger();
  const int p = blockIdx.x;
  const uint64_t key = keys[p];
  if (key == ~0ull || (p > 0 && keys[p - 1] >> 32 == key >> 32)) return;
  if (blockIdx.y == 0 && threadIdx.x == 0) heads[key >> 32] = place + p;
  const int c = (blockIdx.y * 128 + threadIdx.x) * V;
  if (c >= dim) return;
  float v[V] = {};
  int q = p;
  if (p + 1 >= size || keys[p + 1] >> 32 != key >> 32) {  // the only row
    const int r = (int)(uint32_t)key;
    const float w = row[r].w;
    if constexpr (V == 4) load_param_vec<4>(hidden, idx[r] * stride + c, dtype, v);
    else v[0] = load_dyn(hidden, idx[r] * stride + c, dtype);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] *= w;
    q = size;
  }
  for (; q < size; q += 8) {
    float w[8], e[8][V];
    int r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t k = keys[min(q + i, size - 1)];
      r[i] = q + i < size && k >> 32 == key >> 32 ? (int)(uint32_t)k : -1;
    }
    const int none = (int)(uint32_t)key;  // a row to read where there are no more
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int from = r[i] >= 0 ? r[i] : none;
      w[i] = row[from].w;
      const int64_t at = idx[from] * stride + c;
      if constexpr (V == 4) load_param_vec<4>(hidden, at, dtype, e[i]);
      else e[i][0] = load_dyn(hidden, at, dtype);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = r[i] >= 0 ? fmaf(w[i], e[i][k], v[k]) : v[k];
    }
    if (r[7] < 0) break;
  }
  const float scale = scales[0];
  float* to = sums + (int64_t)(place + p) * ld + c;
  if constexpr (V == 4) *reinterpret_cast<float4*>(to) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
  else *to = v[0] * scale;
}

// out = factor * src, the factor scales[1] (dloss NULL) or scales[1] dloss; zeros where no row counts, and for -0.  V elements at a time.
template <int V>
__global__ void __launch_bounds__(256) scaled_copy_kernel(const float* src, int64_t ld, int64_t rows, int dim, const int* count, const float* scales,
                                                          const float* dloss, int has_dloss, void* out, int dtype) {
  pdl_wait();
  pdl_trigger();
  const bool none = *count == 0;
  const float f = has_dloss ? scales[1] * dloss[0] : scales[1];
  const int per = dim / V;
  const int64_t all = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * V;
    float v[V];
    if constexpr (V == 4) {
      const float4 x = __ldcs(reinterpret_cast<const float4*>(src + r * ld + c));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      v[0] = src[r * ld + c];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = none || __float_as_uint(v[k]) == 0x80000000u ? 0.f : v[k] * f;
    if constexpr (V == 4) {
      if (dtype == SSM_F32) {
        __stcs(reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + r * dim + c), make_float4(v[0], v[1], v[2], v[3]));
      } else {
        const uint2 w = dtype == SSM_BF16 ? make_uint2(pack2<__nv_bfloat16>(v[0], v[1]), pack2<__nv_bfloat16>(v[2], v[3])) : make_uint2(pack2<__half>(v[0], v[1]), pack2<__half>(v[2], v[3]));
        __stcs(reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + r * dim + c), w);
      }
    } else {
      store_dyn(out, r * dim + c, dtype, v[0]);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// (outer, inner) matrices of 16-bit elements, `planes` of them; boxes of 64 x `high`
int encode(CUtensorMap* m, const void* base, int64_t inner, int64_t outer, int planes, int64_t ld, int64_t plane, int fmt, int high = 64) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(SSM_ERR_DEVICE, "linear_cross_entropy: cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)planes}, strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)high, 1}, estr[3] = {1, 1, 1};
  const CUresult rc = fn(m, fmt ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? SSM_OK : fail(SSM_ERR_DEVICE, "linear_cross_entropy: cuTensorMapEncodeTiled rejected the matrix");
}

enum Pass { kForward = 0, kBackward = 1, kBoth = 2 };
// sizes and places of a call
struct Plan {
  int planes, fmt, pairs;
  int64_t rows, dim, vocab, ldh, ldg, ldo;  // leading dimensions: packed h, pieces of G, fp32 outputs
  bool copy_w;
  int64_t piece;      // rows of a piece
  int splits, bn;     // of dh = G W
  int parts, sort, sorts;
  // offsets: what both passes use (kept between them), then scratch
  int64_t idx, packed, count, h, w, kept, scales, part, z, row, g, dh, dw, keys, heads, sums, again, hs, bytes;
};
constexpr int64_t kPieceRows = 16384;  // at most, so that what a piece needs beside the logits' gradient has a bound

Plan plan_of(const ssm_linear_ce_args& a, int pass) {
  Plan p{};
  p.planes = a.io_dtype == SSM_F32 ? 3 : 1, p.fmt = a.io_dtype != SSM_F16;
  p.rows = std::max<int64_t>(a.rows, 1), p.dim = a.dim, p.vocab = a.vocab;
  p.ldh = up(p.dim, 8), p.ldg = up(p.vocab, 64), p.ldo = up(p.dim, 4);
  p.copy_w = p.planes == 3 || a.weight_stride % 8 != 0 || a.weight_stride < a.dim || !aligned_to(a.weight, 16);
  p.parts = (int)((p.vocab + kTile - 1) / kTile) * 2;
  p.pairs = std::max(1, sm_count() / 2);
  p.bn = p.dim <= 128 ? 128 : 256;
  p.splits = 1, p.sort = 1;
  p.piece = std::min<int64_t>(up(p.rows, kTile), kPieceRows);
  if (pass != kForward) {
    const int64_t fit = std::min(kPieceRows, std::max<int64_t>(1, SSM_LINEAR_CE_PIECE_BYTES / (p.ldg * 2 * p.planes) / kTile) * kTile), n = (p.rows + fit - 1) / fit;
    p.piece = up((p.rows + n - 1) / n, kTile);  // pieces of one size
    while (p.sort < kSort && p.sort < std::min(p.piece, p.rows)) p.sort *= 2;
    p.sorts = (int)((p.piece + kSort - 1) / kSort);
    // Splits of the vocabulary for dh: the pairs share its tiles and those of dW, which fill up where dh's do not come out even, as long as none of dh's takes longer than all of
    // a pair's share.  A split costs its partial sums' way through memory, 0.3 blocks of K a tile.
    const double t0 = (double)(p.piece / kTile) * (double)((p.dim + p.bn - 1) / p.bn), kb0 = (double)((p.vocab + kK - 1) / kK);
    const double t1 = (double)((p.vocab + kTile - 1) / kTile) * (double)((p.dim + p.bn - 1) / p.bn), share = (t0 * kb0 + t1 * (double)(p.piece / kK)) / p.pairs;
    double least = 1e300;
    for (int s = 1; s <= 32 && (s == 1 || kb0 / s >= 16); ++s) {
      const double cost = std::max(share, std::ceil(t0 * s / p.pairs) * (kb0 / s)) + 0.3 * s * t0;
      if (cost < least) least = cost, p.splits = s;
    }
  }
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  p.idx = take(p.rows * 4), p.packed = take(p.rows * 4), p.count = take(4);
  p.h = take(p.planes * up(p.rows, kTile) * p.ldh * 2);
  p.w = take(p.copy_w ? p.planes * p.vocab * p.ldh * 2 : 0);
  p.kept = at;
  p.scales = take(12), p.row = take(p.rows * 16);  // row: stats of a forward pass that keeps none
  if (pass != kBackward) p.part = take((int64_t)p.parts * p.piece * 8), p.z = take(p.rows * 4);
  if (pass != kForward) {
    p.g = take(p.planes * p.piece * p.ldg * 2), p.dh = take((int64_t)p.splits * p.piece * p.ldo * 4), p.keys = take((int64_t)p.sorts * kSort * 8);
    p.heads = take((int64_t)p.sorts * p.vocab * 4), p.sums = take((int64_t)p.sorts * p.sort * p.ldo * 4);
    if (pass == kBackward) p.dw = take(p.piece < p.rows ? p.vocab * p.ldo * 4 : 0);
    else p.again = take(p.piece / kTile * 4);
    if (pass == kBoth || p.fmt == 0) p.hs = take(up(p.rows, kTile) * p.ldh * 2);
  }
  p.bytes = at - p.kept;
  return p;
}

int check(const ssm_linear_ce_args& a) {
  SSM_REQUIRE(a.rows >= 0 && a.dim >= 1 && a.vocab >= 1 && a.hidden_stride >= 0 && a.weight_stride >= 0, SSM_ERR_SHAPE, "linear_cross_entropy: bad shape");
  SSM_REQUIRE(a.rows <= (1 << 28) && a.vocab <= (1 << 28) && a.dim <= (1 << 20), SSM_ERR_TOO_LARGE, "linear_cross_entropy: more than 2^28 rows or columns, or 2^20 channels");
  SSM_REQUIRE(valid_dtype(a.io_dtype), SSM_ERR_DTYPE, "linear_cross_entropy: unknown dtype");
  SSM_REQUIRE(a.reduction >= 0 && a.reduction <= 2, SSM_ERR_SHAPE, "linear_cross_entropy: unknown reduction");
  SSM_REQUIRE(a.weight && (a.rows == 0 || (a.hidden && a.targets)) && a.scratch && a.packs && a.status, SSM_ERR_NULL, "linear_cross_entropy: NULL pointer");
  SSM_REQUIRE(aligned_to({a.hidden, a.weight}, dtype_size(a.io_dtype)) && aligned_to(a.targets, 8) && aligned_to(a.stats, 16) && aligned_to({a.row_loss, a.log_z, a.loss, a.status}, 4) && aligned_to({a.scratch, a.packs}, 256),
              SSM_ERR_ALIGN, "linear_cross_entropy: misaligned pointer");
  return SSM_OK;
}

template <int EPI, typename T, int PLANES>
int launch_gemm(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mb1, const GemmArgs& g, int pairs, cudaStream_t st) {
  auto kern = gemm_kernel<EPI, T, PLANES>;
  constexpr int smem = kSmem + (EPI == kOut ? kStaging : 0);
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  int64_t tiles = 0;
  for (const Job& j : g.job) tiles += (int64_t)j.m_tiles * j.n_tiles * j.splits;
  return launch_overlapped("linear_ce gemm_kernel", kern, (unsigned)(2 * std::max<int64_t>(1, std::min<int64_t>(tiles, pairs))), kThreads, smem, st, ma, mb, mb1, g);
}
template <int EPI>
int gemm_of(const Plan& p, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mb1, const GemmArgs& g, cudaStream_t st) {
  if constexpr (EPI == kKeep) {
    return launch_gemm<EPI, __nv_bfloat16, 1>(ma, mb, mb1, g, p.pairs, st);
  } else {
    if (p.planes == 3) return launch_gemm<EPI, __nv_bfloat16, 3>(ma, mb, mb1, g, p.pairs, st);
    if (EPI == kGrad && p.fmt == 0) return launch_gemm<EPI, __half, 1>(ma, mb, mb1, g, p.pairs, st);
    return launch_gemm<EPI, __nv_bfloat16, 1>(ma, mb, mb1, g, p.pairs, st);
  }
}

struct Run {
  const ssm_linear_ce_args& a;
  Plan p;
  char* base;
  cudaStream_t st;
  CUtensorMap mh, mw, mg;
  template <typename U>
  U* at(int64_t off) const { return reinterpret_cast<U*>(off < p.kept ? static_cast<char*>(a.packs) + off : base + (off - p.kept)); }
  int* idx() const { return at<int>(p.idx); }
  int* packed() const { return at<int>(p.packed); }
  int* count() const { return at<int>(p.count); }
  float4* row() const { return at<float4>(p.row); }
  const void* w() const { return p.copy_w ? at<void>(p.w) : a.weight; }
  int64_t ldw() const { return p.copy_w ? p.ldh : a.weight_stride; }
};
// packs the rows (and the weight, where it cannot be copied from its place), unless they are from the pass before, and describes them to the copies
int prepare(Run& r, bool packs) {
  const ssm_linear_ce_args& a = r.a;
  const Plan& p = r.p;
  int device = 0;  // a thread's first call into the runtime makes the context current, which the description of a matrix needs (a backward pass runs on a thread of its own)
  if (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return fail(SSM_ERR_DEVICE, "linear_cross_entropy: no device");
  const int64_t plane_h = up(p.rows, kTile) * p.ldh, plane_w = p.copy_w ? p.vocab * p.ldh : p.vocab * a.weight_stride;
  auto pack = [&](const void* src, int64_t stride, int64_t rows, const int* map, uint16_t* dst, int64_t plane) {
    const unsigned grid = (unsigned)((rows + 7) / 8);
    auto kern = p.planes == 3 ? pack_kernel<float, 3> : pack_kernel<uint16_t, 1>;
    return launch_overlapped("linear_ce pack_kernel", kern, grid, 256, 0, r.st, src, stride, rows, (int)p.dim, map, r.count(), dst, p.ldh, plane);
  };
  if (packs && p.rows <= kFewRows) {
    auto kern = p.planes == 3 ? few_rows_kernel<float, 3> : few_rows_kernel<uint16_t, 1>;
    if (const int rc = launch_overlapped("linear_ce few_rows_kernel", kern, 1, 1024, 0, r.st,
                                         a.targets, (int)p.rows, a.ignore_index, (int)p.vocab, a.hidden, a.hidden_stride, (int)p.dim, r.idx(), r.packed(), r.count(), a.row_loss, a.log_z,
                                         r.at<uint16_t>(p.h), p.ldh, plane_h)) return rc;
  } else if (packs) {
    if (const int rc = launch_overlapped("linear_ce rows_kernel", rows_kernel, 1, 1024, 0, r.st,
                                         a.targets, (int)p.rows, a.ignore_index, (int)p.vocab, r.idx(), r.packed(), r.count(), a.row_loss, a.log_z)) return rc;
    if (const int rc = pack(a.hidden, a.hidden_stride, p.rows, r.idx(), r.at<uint16_t>(p.h), plane_h)) return rc;
  }
  if (packs && p.copy_w)
    if (const int rc = pack(a.weight, a.weight_stride, p.vocab, nullptr, r.at<uint16_t>(p.w), plane_w)) return rc;
  if (const int rc = encode(&r.mh, r.at<void>(p.h), p.dim, p.rows, p.planes, p.ldh, plane_h, p.fmt)) return rc;
  if (const int rc = encode(&r.mw, r.w(), p.dim, p.vocab, p.planes, r.ldw(), plane_w, p.fmt)) return rc;
  return p.g > 0 ? encode(&r.mg, r.at<void>(p.g), p.vocab, p.piece, p.planes, p.ldg, p.piece * p.ldg, p.fmt) : SSM_OK;
}
// z = h W^T for the packed rows [row0, row0 + rows)
GemmArgs logits_args(const Run& r, int64_t row0, int64_t rows) {
  const Plan& p = r.p;
  GemmArgs g{};
  Job& j = g.job[0];
  j.m_tiles = (int)((rows + kTile - 1) / kTile), j.n_tiles = (int)((p.vocab + kTile - 1) / kTile), j.splits = 1, j.k_blocks = (int)((p.dim + kK - 1) / kK), j.m_inner = 1, j.a_m0 = (int)row0;
  g.job[1].splits = 1;
  g.bn = kTile, g.fmt = p.fmt, g.row0 = (int)row0, g.rows = (int)rows, g.count = r.count(), g.status = r.a.status;
  g.vocab = (int)p.vocab, g.targets = r.packed(), g.row = r.row();
  g.part = r.at<float2>(p.part), g.part_ld = (int)p.piece, g.z_target = r.at<float>(p.z);
  g.g = r.at<uint16_t>(p.g), g.ldg = p.ldg, g.g_plane = p.piece * p.ldg;
  return g;
}
int zero(void* p, size_t bytes, cudaStream_t st, int byte = 0) {
  const cudaError_t e = cudaMemsetAsync(p, byte, bytes, st);
  if (e == cudaSuccess) return SSM_OK;
  set_error("linear_cross_entropy: %s", cudaGetErrorString(e));
  return (int)e;
}
// the part of a piece's targets in dW, by target
int target_rows(const Run& r, int64_t row0, int64_t rows) {
  const Plan& p = r.p;
  uint64_t* keys = r.at<uint64_t>(p.keys);
  const unsigned threads = (unsigned)std::max(32, p.sort / 8);
  const bool narrow = p.vocab < 1 << 19;  // a key's target and place in 32 bits
  auto sort = narrow ? sort_kernel<uint32_t> : sort_kernel<uint64_t>;
  if (!narrow) cudaFuncSetAttribute(sort_kernel<uint64_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSort * 8);
  if (const int rc = launch_overlapped("linear_ce sort_kernel", sort, p.sorts, threads, threads * (narrow ? 32 : 64), r.st,
                                       r.packed(), r.count(), (int)row0, (int)rows, p.sort, keys)) return rc;
  if (const int rc = zero(r.at<void>(p.heads), (size_t)p.sorts * p.vocab * 4, r.st, 0xff)) return rc;
  const bool wide = p.dim % 4 == 0 && r.a.hidden_stride % 4 == 0 && aligned_to(r.a.hidden, 16);
  auto kern = wide ? target_rows_kernel<4> : target_rows_kernel<1>;
  const int per = wide ? 512 : 128;
  for (int i = 0; i < p.sorts; ++i) {
    if (const int rc = launch_overlapped("linear_ce target_rows_kernel", kern, dim3((unsigned)p.sort, (unsigned)((p.dim + per - 1) / per)), 128, 0, r.st,
                                         keys + (int64_t)i * kSort, p.sort, r.row(), r.idx(), r.a.hidden, r.a.hidden_stride, r.a.io_dtype, (int)p.dim, r.at<float>(p.scales), r.at<float>(p.sums),
                                         p.ldo, r.at<int>(p.heads) + (int64_t)i * p.vocab, i * p.sort)) return rc;
  }
  return SSM_OK;
}
// dW's place: fp32 sums of the pieces before the last, and where the last one leaves it
struct WeightGrad {
  float* sums;
  void* out;
  int64_t ld;
  int dtype;
};
// dh = G W and dW += G^T h of a piece, `h2` for h, and dh's way to its rows; each nullable
int gradients(const Run& r, int64_t row0, int64_t rows, const CUtensorMap& h2, bool later, void* dh, int dh_dtype, const WeightGrad* dw) {
  const Plan& p = r.p;
  GemmArgs g{};
  g.bn = p.bn, g.fmt = p.fmt, g.row0 = (int)row0, g.rows = (int)rows, g.count = r.count(), g.status = r.a.status;
  const int d_tiles = (int)((p.dim + p.bn - 1) / p.bn);
  Job &a = g.job[0], &b = g.job[1];
  a.splits = b.splits = 1;
  if (dh) {
    a.m_tiles = (int)((rows + kTile - 1) / kTile), a.n_tiles = d_tiles, a.splits = p.splits, a.k_blocks = (int)((p.vocab + kK - 1) / kK), a.b_mn = 1;
    a.out = r.at<float>(p.dh), a.ld = p.ldo, a.out_split = p.piece * p.ldo, a.out_rows = (int)rows;
  }
  if (dw) {
    b.m_tiles = (int)((p.vocab + kTile - 1) / kTile), b.n_tiles = d_tiles, b.a_mn = b.b_mn = 1, b.k_is_rows = 1, b.b_k0 = (int)row0;
    b.out = dw->sums, b.ld = p.ldo, b.out_rows = (int)p.vocab, b.add = row0 > 0, b.last = row0 + rows >= p.rows && dw->out != dw->sums;
    if (const int rc = target_rows(r, row0, rows)) return rc;
    const int64_t bytes = dw->ld * dtype_size(dw->dtype);
    g.dw_wide = bytes % 32 == 0 && aligned_to(dw->out, 32) ? 2 : bytes % 16 == 0 && aligned_to(dw->out, 16) ? 1 : 0;
    g.dw = dw->out, g.dw_ld = dw->ld, g.dw_dtype = dw->dtype, g.dim = (int)p.dim;
    g.scales = r.at<float>(p.scales), g.heads = r.at<int>(p.heads), g.sorts = p.sorts, g.target_sums = r.at<float>(p.sums);
  }
  if (const int rc = gemm_of<kOut>(p, r.mg, r.mw, h2, g, r.st)) return rc;
  if (!dh) return SSM_OK;
  const bool wide = p.dim % 4 == 0 && r.a.weight_stride % 4 == 0 && aligned_to({r.a.weight, dh}, 16);
  auto kern = wide ? dhidden_kernel<4> : dhidden_kernel<1>;
  // few rows: their columns shared out too (20 rows of 1219 columns, a warp to a row: 53 us)
  const int64_t blocks = (rows + 7) / 8, shares = (p.dim + (wide ? 511 : 31)) / (wide ? 512 : 32);
  const dim3 grid((unsigned)blocks, (unsigned)std::max<int64_t>(1, std::min(shares, 4 * 148 / blocks)));
  return launch_overlapped("linear_ce dhidden_kernel", kern, grid, 256, 0, r.st,
                           a.out, a.splits, a.out_split, p.ldo, (int)p.dim, r.idx(), r.packed(), r.count(), (int)row0, (int)rows, r.row(), later, r.a.weight,
                           r.a.weight_stride, r.a.io_dtype, dh, dh_dtype);
}
int scaled_copy(const float* src, int64_t ld, int64_t rows, int64_t dim, const int* count, const float* scales, const float* dloss, void* out, int dtype, cudaStream_t st) {
  const bool wide = dim % 4 == 0 && ld % 4 == 0 && aligned_to({src, out}, 16);
  const int64_t all = rows * (wide ? dim / 4 : dim);
  const unsigned grid = (unsigned)std::min<int64_t>((all + 255) / 256, 148 * 32);
  auto kern = wide ? scaled_copy_kernel<4> : scaled_copy_kernel<1>;
  return launch_overlapped("linear_ce scaled_copy_kernel", kern, grid, 256, 0, st, src, ld, rows, (int)dim, count, scales, dloss ? dloss : scales, dloss != nullptr, out, dtype);
}
int reduce(const Run& r) {
  if (r.a.reduction == 0) return SSM_OK;
  if (r.a.rows == 0) return zero(r.a.loss, 4, r.st);
  return launch_overlapped("linear_ce reduce_kernel", reduce_kernel, 1, 1024, 0, r.st, r.a.row_loss, (int)r.a.rows, r.count(), r.a.reduction == 2, r.a.loss);
}
// what the one-pass form's gradients are multiplied by: kept[0] 1 / rows that count for a mean, kept[1] how many count (as an integer); scales of this call
__global__ void share_kernel(const int* count, int mean, float* kept, float* scales) {
  pdl_wait();
  pdl_trigger();
  kept[0] = scales[0] = 1.f;
  scales[1] = 1.f;
  kept[1] = mean ? 1.f / (float)max(1, *count) : 1.f;
  reinterpret_cast<int*>(kept)[2] = *count;
}

}  // namespace
}  // namespace ssmb

using namespace ssmb;

extern "C" int64_t ssm_linear_ce_packs_bytes(const ssm_linear_ce_args* args) {
  if (!args || args->rows < 0 || args->dim < 1 || args->vocab < 1) return 0;
  return plan_of(*args, kForward).kept;
}

extern "C" int64_t ssm_linear_ce_scratch_bytes(const ssm_linear_ce_args* args, int32_t pass) {
  if (!args || args->rows < 0 || args->dim < 1 || args->vocab < 1) return 0;
  return plan_of(*args, pass).bytes;
}

extern "C" int ssm_linear_ce_fwd(const ssm_linear_ce_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "linear_cross_entropy: NULL arguments");
  if (const int rc = check(*args)) return rc;
  const ssm_linear_ce_args& a = *args;
  SSM_REQUIRE((a.rows == 0 || (a.row_loss && a.log_z)) && (a.reduction == 0 || a.loss), SSM_ERR_NULL, "linear_cross_entropy: NULL output");
  Run r{a, plan_of(a, kForward), static_cast<char*>(a.scratch), reinterpret_cast<cudaStream_t>(stream)};
  const Plan& p = r.p;
  if (a.rows) {
    if (const int rc = prepare(r, true)) return rc;
    float4* stats = a.stats ? reinterpret_cast<float4*>(a.stats) : r.row();
    for (int64_t row0 = 0; row0 < p.rows; row0 += p.piece) {
      const int64_t rows = std::min(p.piece, p.rows - row0);
      GemmArgs g = logits_args(r, row0, rows);
      // Up to 64 rows the weight's rows are M and the packed rows N (32 or 64 columns of a tile instead of 256 rows): the products then take no longer than the weight's way from
      // memory (7 rows, 50277 x 768: 31 us the other way round)
      if (p.rows <= kFewRows) {
        g.bn = p.rows <= 32 ? 32 : 64;
        Job& j = g.job[0];
        j.m_tiles = j.n_tiles, j.n_tiles = 1, j.a_m0 = 0;
        g.part_ld = 8 * j.m_tiles;
        CUtensorMap mf;
        if (const int rc = encode(&mf, r.at<void>(p.h), p.dim, p.rows, p.planes, p.ldh, up(p.rows, kTile) * p.ldh, p.fmt, g.bn / 2)) return rc;
        if (const int rc = gemm_of<kFew>(p, r.mw, mf, mf, g, r.st)) return rc;
        if (const int rc = launch_overlapped("linear_ce few_join_kernel", few_join_kernel, (unsigned)p.rows, 256, 0, r.st,
                                             g.part, g.part_ld, g.count, r.idx(), r.packed(), g.z_target, stats, a.row_loss, a.log_z)) return rc;
        continue;
      }
      if (const int rc = gemm_of<kStats>(p, r.mh, r.mw, r.mw, g, r.st)) return rc;
      if (const int rc = launch_overlapped("linear_ce join_kernel", join_kernel, (unsigned)((rows + 31) / 32), 1024, 0, r.st,
                                           g.part, g.part_ld, p.parts, g.count, (int)row0, (int)rows, r.idx(), r.packed(), g.z_target, stats, a.row_loss, a.log_z)) return rc;
    }
  }
  return reduce(r);
}

extern "C" int ssm_linear_ce_bwd(const ssm_linear_ce_bwd_args* args, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "linear_cross_entropy: NULL arguments");
  if (const int rc = check(args->fwd)) return rc;
  const ssm_linear_ce_args& a = args->fwd;
  SSM_REQUIRE(valid_dtype(args->dweight_dtype), SSM_ERR_DTYPE, "linear_cross_entropy: unknown dtype");
  SSM_REQUIRE(a.rows == 0 || (a.stats && args->dloss), SSM_ERR_NULL, "linear_cross_entropy backward: NULL pointer");
  SSM_REQUIRE(aligned_to({args->dloss, args->dlog_z}, 4) && aligned_to(args->dhidden, dtype_size(a.io_dtype)) && aligned_to(args->dweight, dtype_size(args->dweight_dtype)), SSM_ERR_ALIGN,
              "linear_cross_entropy backward: misaligned pointer");
  Run r{a, plan_of(a, kBackward), static_cast<char*>(a.scratch), reinterpret_cast<cudaStream_t>(stream)};
  const Plan& p = r.p;
  if (a.rows == 0) return args->dweight ? zero(args->dweight, (size_t)a.vocab * a.dim * dtype_size(args->dweight_dtype), r.st) : SSM_OK;
  if (const int rc = prepare(r, false)) return rc;
  float* scales = r.at<float>(p.scales);
  const bool each = a.io_dtype == SSM_F16 && (a.reduction == 0 || args->dlog_z);  // weights that may differ
  const WeightGrad dw{r.at<float>(p.dw), args->dweight, p.dim, args->dweight_dtype};
  if (const int rc = launch_overlapped("linear_ce weights_kernel", weights_kernel, 1, 1024, 0, r.st,
                                       reinterpret_cast<const float4*>(a.stats), r.idx(), r.count(), args->dloss, a.reduction, args->dlog_z ? args->dlog_z : args->dloss, args->dlog_z != nullptr,
                                       a.io_dtype == SSM_F16, each, r.row(), scales)) return rc;
  const __half* h = r.at<__half>(p.h);
  CUtensorMap mhs = r.mh;
  int* top = reinterpret_cast<int*>(scales) + 2;
  if (each && args->dweight) {
    if (const int rc = launch_overlapped("linear_ce tops_kernel", tops_kernel, (unsigned)((p.rows + 7) / 8), 256, 0, r.st, h, p.ldh, (int)p.dim, r.row(), r.count(), top)) return rc;
    if (const int rc = encode(&mhs, r.at<void>(p.hs), p.dim, p.rows, 1, p.ldh, up(p.rows, kTile) * p.ldh, p.fmt)) return rc;
  }
  for (int64_t row0 = 0; row0 < p.rows; row0 += p.piece) {
    const int64_t rows = std::min(p.piece, p.rows - row0);
    if (const int rc = gemm_of<kGrad>(p, r.mh, r.mw, r.mw, logits_args(r, row0, rows), r.st)) return rc;
    if (each && args->dweight) {
      if (const int rc = launch_overlapped("linear_ce scaled_rows_kernel", scaled_rows_kernel<__half>, (unsigned)((rows + 7) / 8), 256, 0, r.st, h, p.ldh, (int)p.dim, r.row(), r.count(), row0,
                                           rows, r.at<__half>(p.hs), top, scales)) return rc;
    }
    if (const int rc = gradients(r, row0, rows, mhs, false, args->dhidden, a.io_dtype, args->dweight ? &dw : nullptr)) return rc;
  }
  return SSM_OK;
}

extern "C" int ssm_linear_ce_train(const ssm_linear_ce_args* args, float* dhidden, float* dweight, float* kept, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "linear_cross_entropy: NULL arguments");
  if (const int rc = check(*args)) return rc;
  const ssm_linear_ce_args& a = *args;
  SSM_REQUIRE(a.io_dtype == SSM_BF16 && a.reduction != 0 && a.rows > 0, SSM_ERR_UNSUPPORTED, "linear_cross_entropy: loss and gradient in one pass are built for sums and means of bf16");
  SSM_REQUIRE(a.row_loss && a.log_z && a.loss && kept, SSM_ERR_NULL, "linear_cross_entropy: NULL output");
  SSM_REQUIRE(aligned_to({dhidden, dweight}, 16) && aligned_to(kept, 4), SSM_ERR_ALIGN, "linear_cross_entropy: misaligned pointer");
  Run r{a, plan_of(a, kBoth), static_cast<char*>(a.scratch), reinterpret_cast<cudaStream_t>(stream)};
  const Plan& p = r.p;
  if (const int rc = prepare(r, true)) return rc;
  if (const int rc = launch_overlapped("linear_ce share_kernel", share_kernel, 1, 1, 0, r.st, r.count(), a.reduction == 2, kept, r.at<float>(p.scales))) return rc;
  const __nv_bfloat16* h = r.at<__nv_bfloat16>(p.h);
  __nv_bfloat16* hs = r.at<__nv_bfloat16>(p.hs);
  CUtensorMap mhs;
  if (const int rc = encode(&mhs, hs, p.dim, p.rows, 1, p.ldh, up(p.rows, kTile) * p.ldh, p.fmt)) return rc;
  int* again = r.at<int>(p.again);
  const WeightGrad dw{dweight, dweight, p.ldo, SSM_F32};
  for (int64_t row0 = 0; row0 < p.rows; row0 += p.piece) {
    const int64_t rows = std::min(p.piece, p.rows - row0);
    const unsigned warps = (unsigned)((rows + 7) / 8);
    GemmArgs g = logits_args(r, row0, rows);
    if (const int rc = launch_overlapped("linear_ce reference_kernel", reference_kernel, warps, 256, 0, r.st,
                                         h, static_cast<const __nv_bfloat16*>(r.w()), p.ldh, r.ldw(), (int)p.dim, r.packed(), r.count(), (int)row0, (int)rows, g.z_target, r.row(),
                                         again)) return rc;
    for (int second = 0; second < 2; ++second) {
      g.again = second ? again : nullptr;
      if (const int rc = gemm_of<kKeep>(p, r.mh, r.mw, r.mw, g, r.st)) return rc;
      if (const int rc = launch_overlapped("linear_ce join_keep_kernel", join_keep_kernel, (unsigned)((rows + 31) / 32), 1024, 0, r.st,
                                           g.part, g.part_ld, p.parts, g.count, (int)row0, (int)rows, r.idx(), g.z_target, r.row(), again, second, a.row_loss, a.log_z)) return rc;
    }
    if (dweight) {
      if (const int rc = launch_overlapped("linear_ce scaled_rows_kernel", scaled_rows_kernel<__nv_bfloat16>, warps, 256, 0, r.st, h, p.ldh, (int)p.dim, r.row(), r.count(), row0, rows, hs,
                                           static_cast<const int*>(nullptr), r.at<float>(p.scales))) return rc;
    }
    if (const int rc = gradients(r, row0, rows, mhs, true, dhidden, SSM_F32, dweight ? &dw : nullptr)) return rc;
  }
  return reduce(r);
}

extern "C" int ssm_linear_ce_scale(const float* src, int64_t ld, int64_t rows, int32_t dim, const float* kept, const float* dloss, void* out, int32_t dtype, ssm_stream_t stream) {
  SSM_REQUIRE(rows >= 0 && dim >= 1 && ld >= dim, SSM_ERR_SHAPE, "linear_cross_entropy: bad shape");
  SSM_REQUIRE(valid_dtype(dtype), SSM_ERR_DTYPE, "linear_cross_entropy: unknown dtype");
  SSM_REQUIRE(rows == 0 || (src && kept && dloss && out), SSM_ERR_NULL, "linear_cross_entropy: NULL pointer");
  SSM_REQUIRE(aligned_to({src, kept, dloss}, 4) && aligned_to(out, dtype_size(dtype)), SSM_ERR_ALIGN, "linear_cross_entropy: misaligned pointer");
  if (rows == 0) return SSM_OK;
  return scaled_copy(src, ld, rows, dim, reinterpret_cast<const int*>(kept) + 2, kept, dloss, out, dtype, reinterpret_cast<cudaStream_t>(stream));
}
