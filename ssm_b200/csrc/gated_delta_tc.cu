// Gated delta rule on the tensor cores: 16-bit operands, kdim and vdim multiples of 8, kdim <= 128.
//
// A sequence is cut into chunks of 64 tokens.  With a = e^g, gam_i = a_1 .. a_i, suf_i = a_{i+1} .. a_64, G_ij = a_{j+1} .. a_i, S0 (vdim x kdim)
// the state before the chunk, the rows r_i = v_i - S'_i k_i solve a unit lower triangular system:
//   (I + A) r = V - diag(gam) K S0^T,  A_ij = beta_j G_ij k_i.k_j (j < i);   X = (I + A)^-1,  W = X diag(gam) K;   r = X V - W S0^T
//   S = gam_64 S0 + r^T diag(beta suf) K
//   o = scale diag(gam) Q S0^T + P r = Y V + Z S0^T,  P_ij = scale beta_j G_ij q_i.k_j (j <= i),  Y = P X,  Z = scale diag(gam) Q - P W
// and the adjoint state, from the end, with D the gradient of the state behind the chunk and Wb = X^T diag(beta suf) K:
//   w = dv = Y^T do + Wb D^T;   D0 = gam_64 D + do^T diag(scale gam) Q - w^T diag(gam) K
//
//   pairs_kernel   one CTA per (chunk, value head): X, Y, W, Z (and Wb), which depend on no state: all chunks at once.  Products by
//                  mma.sync on 16 rows a warp; the inverse is kept in fp32: blocks of 16 by substitution, then two rounds of products of
//                  blocks whose factors are split into two 16-bit pieces.  Bound: shared memory, 70 % of its cycles: 24 ns a chunk and head
//                  on the whole GPU (196 us for 8192 at K = 128), 42 with Wb, whose registers spill.
//   chunks_kernel  one CTA per (sequence, value head, 128 rows of the state): the walk over the chunks, forward or back (BACK).
//   grads_kernel   a CTA per SM over all (chunk, value head): the other gradients from what both walks left (the formulas stand there).
//
// The walk is bound by its chain, the state of a chunk depending on the one before through two products and the conversions between
// them.  So the state lies transposed, with vdim on the 128 lanes of tensor memory, and both products take their A operand from tensor memory,
// written there by the threads that hold the rows: S (16 bits) x W^T, added to V^T X^T -> r -> times beta suf x K -> added to the state,
// which stays in registers.  o needs neither r nor a product of its own: Y and Z are 64 more rows of the operands X and W.
// Measured, K = V = 128: 1.2 us a chunk with 32 walks side by side (tensor pipe 48 % busy on the SMs that have one), 1.9 where a training call's
// states and rest are stored, forward and back; 128 walks move 796 MB in 144 us, 5.5 TB/s.
// Roundings to 16 bits, each half a step of the type, because the tensor cores take such operands; two pieces of each would double the walk's products and
// bytes.  Forward: S as an operand, X, W (from X gam), P, Y (from rounded P and X), Z (from rounded P and W), the weighted r.  Backward: the kept S, D and r,
// w as it is read again, gam w, the scaled q, Wb (from X^T beta suf) and the four matrices of pairs in grads_kernel.  The inverse's products split their factors
// into two pieces each (16 bits of bf16, 22 of fp16).  Sums, the state and its adjoint from chunk to chunk are fp32.
// Off 64 bits in norm, bf16 (fp16 an eighth of it), with the result's own rounding of 0.17 %: 0.31 % for keys in all directions, gradients 0.33 %.  Keys that
// hardly differ make X and W large against r = X V - W S0: 0.8 % where they are 0.3 of their length apart and strengths come from a sigmoid, gradients
// up to 1.3 %; 1.2 and 2.1 % at strength 1; 3.2 and 8 % at 1.9.  (The answers as Q S0 and P r of a rounded r: 1.3 % in place of 0.8.)
#include <algorithm>

#include "gated_delta.cuh"
#include "ssd_common.cuh"

namespace ssmb {
namespace gd {
namespace {

constexpr int C = 64;  // tokens of a chunk
constexpr int kTileBytes = C * 128;  // 64 rows of 128 bytes
constexpr float kReset = -150.f;     // base-2 logarithm of a decay that is zero in fp32

// What pairs_kernel leaves per (chunk, value head), matrices as tiles of 64 rows of 128 bytes in the 128-byte swizzle
struct Chunks {
  unsigned char* x;   // X
  unsigned char* wz;  // per 64 columns of kdim: -W, Z
  unsigned char* y;   // Y
  unsigned char* wb;  // Wb; NULL without a backward pass to follow
  float* vec;         // gam, beta, beta suf, scale gam: 64 each
  int32_t* status;
};

// not 0 where one of a 16-byte unit's elements is not finite: an exponent of ones carries into the sign
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint4 x) {
  constexpr uint32_t ones = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u, carry = std::is_same<T, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;
  return ((((x.x & ones) + carry) | ((x.y & ones) + carry) | ((x.z & ones) + carry) | ((x.w & ones) + carry)) & 0x80008000u);
}
__device__ __forceinline__ uint32_t swz(int row, int unit) { return (uint32_t)(row * 128 + ((unit ^ (row & 7)) << 4)); }  // 16-byte unit of a row

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// ---------------------------------------------------------------------------------------------
// warp-level products (pairs, gradients): 16 x 8 x 16
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Tiles of 64 rows: element (row, col) lies in block col / 64 of 8 KB, at swz(row, col % 64 / 8).
// A fragment of rows r0 .. r0 + 15, columns c0 .. c0 + 15
__device__ __forceinline__ void load_a(uint32_t (&f)[4], uint32_t tile, int r0, int c0, int lane) {
  const int row = r0 + (lane & 15), unit = c0 / 8 + (lane >> 4);
  ldsm4(f, tile + (unit >> 3) * kTileBytes + swz(row, unit & 7));
}
// B fragments of two neighbouring blocks of eight columns n0 .. n0 + 15, depth k0 .. k0 + 15; B[k][n] = tile[n][k]
__device__ __forceinline__ void load_b(uint32_t (&f)[4], uint32_t tile, int n0, int k0, int lane) {
  const int row = n0 + (lane & 7) + ((lane >> 4) << 3), unit = k0 / 8 + ((lane >> 3) & 1);
  ldsm4(f, tile + (unit >> 3) * kTileBytes + swz(row, unit & 7));
}
// B[k][n] = tile[k][n]
__device__ __forceinline__ void load_bt(uint32_t (&f)[4], uint32_t tile, int n0, int k0, int lane) {
  const int row = k0 + (lane & 15), unit = n0 / 8 + (lane >> 4);
  ldsm4t(f, tile + (unit >> 3) * kTileBytes + swz(row, unit & 7));
}

// ---------------------------------------------------------------------------------------------
// pairs of tokens
// ---------------------------------------------------------------------------------------------
constexpr int kPairThreads = 128, kAS = 68, kTS = 36;  // row strides of the fp32 blocks, in floats

template <int KD>
struct PairSmem {
  static constexpr int KT = (KD / 64) * kTileBytes;
  static constexpr int QT = KT > 2 * kTileBytes ? KT : 2 * kTileBytes;
  static constexpr int AT = C * kAS * 4 > KT ? C * kAS * 4 : KT;
  // k's rows, later Z; q's rows, later X and P (then Y); A, then X in fp32, later W (then Wb)
  static constexpr int K = 0, X = KT, P = X + kTileBytes, A = KT + QT, TMP = A + (AT + 1023) / 1024 * 1024, VEC = TMP + 32 * kTS * 4, TOTAL = VEC + 5 * C * 4;
  static constexpr int ALLOC = TOTAL + 1024;
};

// log decays and strengths of tokens 2 lane, 2 lane + 1 of a chunk, by one warp; tokens from n on decay nothing
struct TokenPair {
  float g[2], beta[2];
};
__device__ __forceinline__ TokenPair token_pair(const Args& a, const Span& s, int n, int h, int lane) {
  TokenPair x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = 2 * lane + i;
    x.g[i] = t < n && a.g.p ? load_dyn(a.g.p, s.b * a.g.sb + (s.t0 + t) * a.g.st + h * a.g.sh, a.g_dtype) : 0.f;
    x.beta[i] = t < n ? beta_of(a, s.b, s.t0 + t, h) : 0.f;
  }
  return x;
}
// their cumulative base-2 logarithms
__device__ __forceinline__ void decay_logs(const TokenPair& p, float* c, float* beta, int lane) {
  float x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[i] = p.g[i] * kLog2e, beta[2 * lane + i] = p.beta[i];
    if (x[i] < kReset) x[i] = kReset;  // NaN stays
  }
  float sum = x[0] + x[1];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const float o = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += o;
  }
  c[2 * lane + 1] = sum, c[2 * lane] = sum - x[1];
}

// k.k and q.k of this warp's 16 rows with all up to them, and the rows of q, which stay in the registers
template <typename T, int KD>
__device__ __forceinline__ void rows_products(float (&kk)[8][4], float (&qk)[8][4], uint32_t (&q)[KD / 16][4], uint32_t tk, uint32_t tq, int r0, int lane) {
#pragma unroll
  for (int nb = 0; nb < 8; ++nb)
#pragma unroll
    for (int e = 0; e < 4; ++e) kk[nb][e] = qk[nb][e] = 0.f;
#pragma unroll
  for (int k0 = 0; k0 < KD; k0 += 16) {
    uint32_t fk[4];
    load_a(fk, tk, r0, k0, lane);
    load_a(q[k0 / 16], tq, r0, k0, lane);
#pragma unroll
    for (int n0 = 0; n0 < C; n0 += 16) {
      if (n0 > r0) continue;
      uint32_t fb[4];
      load_b(fb, tk, n0, k0, lane);
      mma16816<T>(kk[n0 / 8], fk, fb[0], fb[1]);
      mma16816<T>(kk[n0 / 8 + 1], fk, fb[2], fb[3]);
      mma16816<T>(qk[n0 / 8], q[k0 / 16], fb[0], fb[1]);
      mma16816<T>(qk[n0 / 8 + 1], q[k0 / 16], fb[2], fb[3]);
    }
  }
}

// contiguous shared -> global; both addresses 16-byte aligned, size a multiple of 16
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

// 16 x 8 NB of a product of fp32 blocks in shared memory with an inner extent of K, by one warp: `left` points to its rows, `right` to its columns.
// Each factor in two 16-bit pieces, three products
template <typename T, int K, int NB>
__device__ __forceinline__ void block_product(float (&d)[NB][4], const float* left, int ls, const float* right, int rs, int lane) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) d[nb][0] = d[nb][1] = d[nb][2] = d[nb][3] = 0.f;
  auto split = [](float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = pack2<T>(x, y);
    const float2 z = unpack2<T>(hi);
    lo = pack2<T>(x - z.x, y - z.y);
  };
#pragma unroll
  for (int k0 = 0; k0 < K; k0 += 16) {
    uint32_t ah[4], al[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = *reinterpret_cast<const float2*>(&left[((lane >> 2) + (e & 1) * 8) * ls + k0 + (lane & 3) * 2 + (e >> 1) * 8]);
      split(x.x, x.y, ah[e], al[e]);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      uint32_t bh[2], bl[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float* at = &right[(k0 + (lane & 3) * 2 + e * 8) * rs + nb * 8 + (lane >> 2)];
        split(at[0], at[rs], bh[e], bl[e]);
      }
      mma16816<T>(d[nb], ah, bh[0], bh[1]);
      mma16816<T>(d[nb], al, bh[0], bh[1]);
      mma16816<T>(d[nb], ah, bl[0], bl[1]);
    }
  }
}

struct PairMaps {
  CUtensorMap q, k;
};

// Decays and strengths of a chunk's tokens, by one warp, here (c, beta, gam, beta suf, scale gam: 64 each) and for the kernels behind, there NaN from token
// `gone` on
__device__ __forceinline__ void leave_decays(const Args& a, const Chunks& out, int64_t at, const TokenPair& p, float* c, int gone, int lane) {
  float *beta = c + C, *gam = beta + C, *bsuf = gam + C, *sgam = bsuf + C, *v = out.vec + at * (4 * C);
  decay_logs(p, c, beta, lane);
  __syncwarp();
  for (int i = lane; i < C; i += 32) {
    const float x = ex2_approx(c[i]), y = beta[i] * ex2_approx(c[C - 1] - c[i]), none = i >= gone ? __uint_as_float(0x7fc00000u) : 0.f;
    gam[i] = x, bsuf[i] = y, sgam[i] = x * a.scale;
    v[i] = x + none, v[C + i] = beta[i] + none, v[2 * C + i] = y + none, v[3 * C + i] = x * a.scale + none;
  }
}
// A chunk without the tokens from `lost` on; not inline, and its products once more beside the first ones rather than in a loop: both would cost registers
template <int KD>
__device__ __noinline__ void cut_chunk(const Args& a, const Chunks& out, unsigned char* tK, float* c, int lost) {
  const Span s = chunk_of(a.where, blockIdx.x, C);
  constexpr int U = KD / 8;
  for (int i = threadIdx.x; i < (C - lost) * U; i += kPairThreads) *reinterpret_cast<uint4*>(tK + (i % U >> 3) * kTileBytes + swz(lost + i / U, i % U & 7)) = make_uint4(0, 0, 0, 0);
  if (threadIdx.x < 32) leave_decays(a, out, (int64_t)s.chunk * a.heads + blockIdx.y, token_pair(a, s, min(s.t1 - s.t0, lost), blockIdx.y, threadIdx.x), c, lost, threadIdx.x);
}

template <typename T, int KD, bool TRAIN>
__global__ void __launch_bounds__(kPairThreads, 4) pairs_kernel(const __grid_constant__ Args a, const __grid_constant__ Chunks out, const __grid_constant__ PairMaps maps) {
  using M = PairSmem<KD>;
  extern __shared__ unsigned char smdyn[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smdyn) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t mbar;
  __shared__ int lost;  // the first token whose key, decay or strength is not finite
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const Span s = chunk_of(a.where, blockIdx.x, C);
  const int n = s.t1 - s.t0, h = blockIdx.y, kh = h / a.group;
  if (n <= 0 || s.seq < 0) return;
  const int64_t at = (int64_t)s.chunk * a.heads + h;
  unsigned char *tK = sm + M::K, *tQ = sm + M::X, *tX = sm + M::X, *tP = sm + M::P, *tW = sm + M::A;
  float* A = reinterpret_cast<float*>(sm + M::A);
  float *tmp = reinterpret_cast<float*>(sm + M::TMP), *c = reinterpret_cast<float*>(sm + M::VEC), *beta = c + C, *gam = beta + C, *bsuf = gam + C, *sgam = bsuf + C;
  const uint32_t landed = tc::smem_u32(&mbar);
  if (tid == 0) {
    tc::mbar_init(landed, 1);
    tc::mbar_expect_tx(landed, 2 * M::KT);
    for (int b = 0; b < KD / 64; ++b) {
      tc::tma_load_4d(tc::smem_u32(tK + b * kTileBytes), &maps.k, landed, b * 64, kh, s.t0, s.b);
      tc::tma_load_4d(tc::smem_u32(tQ + b * kTileBytes), &maps.q, landed, b * 64, kh, s.t0, s.b);
    }
  }
  if (warp == 0) {  // beside the copies
    const TokenPair p = token_pair(a, s, n, h, lane);
    leave_decays(a, out, at, p, c, C, lane);
    const uint32_t even = __ballot_sync(0xffffffffu, !(p.g[0] * kLog2e < INFINITY && fabsf(p.beta[0]) < INFINITY)),
                   odd = __ballot_sync(0xffffffffu, !(p.g[1] * kLog2e < INFINITY && fabsf(p.beta[1]) < INFINITY));
    if (lane == 0) lost = min(even ? 2 * __ffs(even) - 2 : C, odd ? 2 * __ffs(odd) - 1 : C);
  }
  __syncthreads();
  if (!__syncthreads_and(tc::mbar_wait(landed, 0))) {
    if (tid == 0 && out.status) *(volatile int32_t*)out.status = 6;
    tc::mbar_wait(landed, 0);  // nothing is under way when the block ends, as far as a second limit goes
    return;
  }
  if (a.where.table && n < C) {  // rows of the next sequence: nothing of them may enter a product, not even times zero
    constexpr int U = KD / 8;
    for (int i = tid; i < (C - n) * U; i += kPairThreads)
      *reinterpret_cast<uint4*>(tK + (i % U >> 3) * kTileBytes + swz(n + i / U, i % U & 7)) = *reinterpret_cast<uint4*>(tQ + (i % U >> 3) * kTileBytes + swz(n + i / U, i % U & 7)) =
          make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const int r0 = warp * 16, gi = lane >> 2, gj = (lane & 3) * 2;
  const uint32_t bK = tc::smem_u32(tK);
  float kk[8][4], qk[8][4];
  uint32_t fq[KD / 16][4];
  rows_products<T, KD>(kk, qk, fq, bK, tc::smem_u32(tQ), r0, lane);
  // What is not finite would meet the zeros of the triangles below, and so reach tokens before it.  From the first such token on the chunk is formed
  // without keys, strengths and decays; those rows of X and Y and the decay of the whole chunk are NaN when they leave.  A key shows in its product with itself
  int own = C;
#pragma unroll
  for (int nb = 7; nb >= 0; --nb)
    if (nb >> 1 == warp && (gi & ~1) == gj && !(fabsf(gi & 1 ? kk[nb][2 * (nb & 1) + 1] : kk[nb][2 * (nb & 1)]) < INFINITY)) own = r0 + gi + (nb & 1) * 8;
  if (__syncthreads_or(own < C || lost < C)) {  // and the rows of q have been read
    if (own < C) atomicMin(&lost, own);
    __syncthreads();
    cut_chunk<KD>(a, out, tK, c, lost);
    __syncthreads();
    rows_products<T, KD>(kk, qk, fq, bK, tc::smem_u32(tQ), r0, lane);
    __syncthreads();
  }
  {
    const float ci[2] = {c[r0 + gi], c[r0 + gi + 8]};
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      float x[4] = {}, p[4] = {};
      if (nb * 8 <= r0 + 8) {
        const float2 cj = *reinterpret_cast<const float2*>(&c[nb * 8 + gj]), bj = *reinterpret_cast<const float2*>(&beta[nb * 8 + gj]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = r0 + gi + (e >> 1) * 8 - (nb * 8 + gj + (e & 1));
          const float G = ex2_approx(ci[e >> 1] - (e & 1 ? cj.y : cj.x)) * (e & 1 ? bj.y : bj.x);
          x[e] = d > 0 ? G * kk[nb][e] : 0.f;
          p[e] = d >= 0 ? G * a.scale * qk[nb][e] : 0.f;
        }
      }
      const int i = r0 + gi;
      *reinterpret_cast<float2*>(&A[i * kAS + nb * 8 + gj]) = make_float2(x[0], x[1]);
      *reinterpret_cast<float2*>(&A[(i + 8) * kAS + nb * 8 + gj]) = make_float2(x[2], x[3]);
      *reinterpret_cast<uint32_t*>(tP + swz(i, nb) + gj * 2) = pack2<T>(p[0], p[1]);
      *reinterpret_cast<uint32_t*>(tP + swz(i + 8, nb) + gj * 2) = pack2<T>(p[2], p[3]);
    }
  }
  __syncwarp();  // the diagonal block is this warp's own
  {              // its inverse, a column a lane (both halves of the warp the same ones)
    const float* D = A + r0 * kAS + r0;
    float x[16];
    const int col = lane & 15;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == col ? 1.f : 0.f, v1 = 0.f;
#pragma unroll
      for (int j = 0; j < i; j += 4) {
        const float4 m = *reinterpret_cast<const float4*>(&D[i * kAS + j]);  // zeros from the diagonal on
        v = fmaf(-m.x, x[j], v);
        if (j + 1 < i) v1 = fmaf(-m.y, x[j + 1], v1);
        if (j + 2 < i) v = fmaf(-m.z, x[j + 2], v);
        if (j + 3 < i) v1 = fmaf(-m.w, x[j + 3], v1);
      }
      x[i] = v + v1;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((i & 1) == lane >> 4) A[(r0 + i) * kAS + r0 + col] = x[i];
  }
  __syncthreads();
  auto put_rows = [&](float* to, int stride, const float (&d)[4], float sign) {  // 16 x 8 of a block
    *reinterpret_cast<float2*>(&to[gi * stride + gj]) = make_float2(sign * d[0], sign * d[1]);
    *reinterpret_cast<float2*>(&to[(gi + 8) * stride + gj]) = make_float2(sign * d[2], sign * d[3]);
  };
  {  // pairs of blocks: X10 = -X11 (A10 X00), two warps each
    const int n0 = (warp & 1) * 8;
    float* block = A + (warp >> 1) * 32 * (kAS + 1);
    float *half = tmp + (warp >> 1) * 16 * kTS + n0, d[1][4];
    block_product<T, 16>(d, block + 16 * kAS, kAS, block + n0, kAS, lane);
    put_rows(half, kTS, d[0], 1.f);
    __syncthreads();
    block_product<T, 16>(d, block + 16 * kAS + 16, kAS, half, kTS, lane);
    put_rows(block + 16 * kAS + n0, kAS, d[0], -1.f);
  }
  __syncthreads();
  {  // the same for the halves, 16 x 16 of it a warp
    const int br = (warp >> 1) * 16, bc = (warp & 1) * 16;
    float d[2][4];
    block_product<T, 32>(d, A + (32 + br) * kAS, kAS, A + bc, kAS, lane);
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) put_rows(tmp + br * kTS + bc + nb * 8, kTS, d[nb], 1.f);
    __syncthreads();
    block_product<T, 32>(d, A + (32 + br) * kAS + 32, kAS, tmp + bc, kTS, lane);
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) put_rows(A + (32 + br) * kAS + bc + nb * 8, kAS, d[nb], -1.f);
  }
  __syncthreads();
  // X in 16 bits, and the operands of W (X with columns times -gam) and Wb (X^T with columns times beta suf)
  uint32_t fw[4][4], fb[TRAIN ? 4 : 1][4];
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = r0 + gi + (e & 1) * 8, j = kb * 16 + gj + (e >> 1) * 8;
      float2 x = make_float2(0.f, 0.f);
      if (kb <= warp) {
        x = *reinterpret_cast<const float2*>(&A[i * kAS + j]);
        const float2 m = *reinterpret_cast<const float2*>(&gam[j]);
        fw[kb][e] = pack2<T>(-x.x * m.x, -x.y * m.y);
      }
      *reinterpret_cast<uint32_t*>(tX + swz(i, j >> 3) + gj * 2) = pack2<T>(x.x, x.y);
      if constexpr (TRAIN) {
        if (kb >= warp) {
          const float2 m = *reinterpret_cast<const float2*>(&bsuf[j]);
          fb[kb][e] = pack2<T>(A[j * kAS + i] * m.x, A[(j + 1) * kAS + i] * m.y);
        }
      }
    }
  }
  __syncthreads();  // A has been read, X is written
  // 64 columns of rows x a tile, from the accumulator given
  auto times = [&](float (&d)[8][4], const uint32_t (&fa)[4][4], uint32_t tile, int from, int to) {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      if (kb < from || kb > to) continue;
#pragma unroll
      for (int n0 = 0; n0 < 64; n0 += 16) {
        uint32_t b[4];
        load_bt(b, tile, n0, kb * 16, lane);
        mma16816<T>(d[n0 / 8], fa[kb], b[0], b[1]);
        mma16816<T>(d[n0 / 8 + 1], fa[kb], b[2], b[3]);
      }
    }
  };
  auto put = [&](unsigned char* tile, const float (&d)[8][4]) {  // this warp's rows
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      *reinterpret_cast<uint32_t*>(tile + swz(r0 + gi, nb) + gj * 2) = pack2<T>(d[nb][0], d[nb][1]);
      *reinterpret_cast<uint32_t*>(tile + swz(r0 + gi + 8, nb) + gj * 2) = pack2<T>(d[nb][2], d[nb][3]);
    }
  };
  // Wb waits in the registers for W's place; k's rows are not needed after it
  uint32_t wb[TRAIN ? KD / 64 : 1][8][2];
#pragma unroll
  for (int half = 0; half < KD / 64; ++half) {
    float d[8][4] = {};
    times(d, fw, bK + half * kTileBytes, 0, warp);
    put(tW + half * kTileBytes, d);
    if constexpr (TRAIN) {
      float e[8][4] = {};
      times(e, fb, bK + half * kTileBytes, warp, 3);
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) wb[half][nb][0] = pack2<T>(e[nb][0], e[nb][1]), wb[half][nb][1] = pack2<T>(e[nb][2], e[nb][3]);
    }
  }
  uint32_t fp[4][4];
#pragma unroll
  for (int kb = 0; kb < 4; ++kb)
    if (kb <= warp) load_a(fp[kb], tc::smem_u32(tP), r0, kb * 16, lane);
  {
    float d[8][4] = {};
    times(d, fp, tc::smem_u32(tX), 0, warp);
    __syncwarp();
    put(tP, d);
  }
  __syncthreads();  // W is written, the rows of k have been read
  const float s0 = sgam[r0 + gi], s1 = sgam[r0 + gi + 8];
#pragma unroll
  for (int half = 0; half < KD / 64; ++half) {
    float d[8][4];
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      const uint32_t* q = &fq[half * 4 + nb / 2][(nb & 1) * 2];
      const float2 x = unpack2<T>(q[0]), y = unpack2<T>(q[1]);
      d[nb][0] = s0 * x.x, d[nb][1] = s0 * x.y, d[nb][2] = s1 * y.x, d[nb][3] = s1 * y.y;
    }
    times(d, fp, tc::smem_u32(tW) + half * kTileBytes, 0, warp);
    put(tK + half * kTileBytes, d);
  }
  for (int i = lost * 8 + tid; i < C * 8; i += kPairThreads)  // NaN in either type
    *reinterpret_cast<uint4*>(tX + swz(i / 8, i % 8)) = *reinterpret_cast<uint4*>(tP + swz(i / 8, i % 8)) = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  tc::fence_async_smem();
  __syncthreads();
  if (tid == 0) {
    bulk_store(out.x + at * kTileBytes, tc::smem_u32(tX), kTileBytes);
    bulk_store(out.y + at * kTileBytes, tc::smem_u32(tP), kTileBytes);
    unsigned char* to = out.wz + at * (2 * M::KT);
#pragma unroll
    for (int half = 0; half < KD / 64; ++half) {
      bulk_store(to + 2 * half * kTileBytes, tc::smem_u32(tW) + half * kTileBytes, kTileBytes);
      bulk_store(to + (2 * half + 1) * kTileBytes, bK + half * kTileBytes, kTileBytes);
    }
    tc::bulk_commit();
    if constexpr (TRAIN) tc::bulk_wait_read();
  }
  if constexpr (TRAIN) {
    __syncthreads();  // W has left
#pragma unroll
    for (int half = 0; half < KD / 64; ++half)
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) {
        *reinterpret_cast<uint32_t*>(tW + half * kTileBytes + swz(r0 + gi, nb) + gj * 2) = wb[half][nb][0];
        *reinterpret_cast<uint32_t*>(tW + half * kTileBytes + swz(r0 + gi + 8, nb) + gj * 2) = wb[half][nb][1];
      }
    tc::fence_async_smem();
    __syncthreads();
    if (tid == 0) {
      bulk_store(out.wb + at * M::KT, tc::smem_u32(tW), M::KT);
      tc::bulk_commit();
    }
  }
  if (tid == 0) tc::bulk_wait_all();  // shared memory outlives the copies that read it
}

// ---------------------------------------------------------------------------------------------
// the walk over the chunks
// ---------------------------------------------------------------------------------------------
constexpr int kSlice = 64;  // columns of v that the gradients take at a time
struct WalkMaps {
  CUtensorMap q, k, v, o;  // boxes of 64 columns of one head x 64 tokens; BACK: v is do, o is dv
};
struct ChunkWalk {
  Args a;
  Chunks in;
  const float* initial;  // BACK: gradient of the final state
  void* o;               // BACK: dv
  void* last;            // final state; BACK: gradient of the initial one, fp32
  int last_dtype;
  void* rest;    // 16-bit r for the backward pass, [slice of vdim][token / 8][column][8] per (chunk, head); nullable
  void* states;  // 16-bit state before every chunk (BACK: adjoint state behind it), [kdim / 8][vdim][8]; nullable
};

// Warps 0-7 hold the rows of the state (a lane a row, two warps share the columns of 32 rows; with four of them 2240 cycles a chunk instead of 1940), 8-11
// prepare operands and store what leaves, 12 copies, 13 issues the products, 14 and 15 look at v (forward).  Launched with 128 registers a thread
// (512 x 128 = 65536), of which the groups of four warps keep 168, 168, 104 and 40.
constexpr int kParts = 2, kCompute = 128 * kParts, kHelp = 128, kWalkThreads = kCompute + kHelp + 128;
constexpr int kComputeRegs = 168, kHelpRegs = 104, kIssueRegs = 40;
static_assert(kCompute * kComputeRegs + kHelp * kHelpRegs + 128 * kIssueRegs <= kWalkThreads * 128, "the split draws on what the block was launched with");
// Operands in two rings: what the first product reads is free again a third into its chunk, the rest at its end.  (One ring of two stages of 81 KB:
// 4200 cycles a chunk, of which 1800 waiting for copies.)
template <int KD, bool BACK>
struct WalkSmem {
  static constexpr int KB = (KD / 64) * kTileBytes, VB = 2 * kTileBytes, VEC_BYTES = 4 * C * 4;
  static constexpr int WB = BACK ? KB : 2 * KB, XB = BACK ? kTileBytes : 2 * kTileBytes;
  static constexpr int V = 0, X = VB, W = X + XB, EARLY = W + WB;                       // v, X and Y, W and Z; BACK: do, Y, Wb
  static constexpr int K = 0, Q = KB, VEC = Q + (BACK ? KB : 0), LATE = VEC + VEC_BYTES;  // k, vectors; BACK: q too
  static constexpr int NE = 2, NL = 3;
  static constexpr int OUT = NE * EARLY + NL * LATE, ALLOC = OUT + 2 * VB + 1024;
};
static_assert(WalkSmem<128, false>::ALLOC <= 227 * 1024 && WalkSmem<128, true>::ALLOC <= 227 * 1024, "shared memory of an SM");

// tensor memory, in columns: operands (the state; the weighted r) and accumulators: r and o side by side, twice; the state's increment
struct Cols {
  static constexpr int S = 0, U = 64, RO = 128, DS = 384;
};

// A wait by parity must not fall two completions behind: each barrier's next completion but one needs what its waiter does after this one (two of
// kPrep and kSeen for that)
enum Bar { kFullE = 0, kFreeE = 2, kFullL = 4, kFreeL = 7, kPrep = 10, kSeen = 12, kFullV = 14, kState = 16, kR, kU, kDS, kO, kOut, kEnd, kBars };

// a load from tensor memory that is under way until `landed`
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// ... and its registers hang on the wait, so that no use of them moves in front of it
__device__ __forceinline__ void landed(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
// One probe that returns at once, then the suspending ones, which take 300 cycles even where the phase is complete.  (Polling instead costs the warps
// that work more than the ones that wait gain: 2170 to 2300 cycles a chunk against 1940.)
__device__ __forceinline__ bool phase_done(uint32_t mbar, uint32_t parity) { return tc::mbar_test(mbar, parity) || tc::mbar_wait(mbar, parity); }
__device__ __forceinline__ void put16(uint32_t saddr, uint16_t x) { asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(saddr), "h"(x) : "memory"); }
__device__ __forceinline__ float f(uint32_t x) { return __uint_as_float(x); }

template <typename T, int KD, bool BACK>
__global__ void __launch_bounds__(kWalkThreads, 1) chunks_kernel(const ChunkWalk w, const __grid_constant__ WalkMaps maps) {
  using M = WalkSmem<KD, BACK>;
  using TC = Cols;
  extern __shared__ unsigned char smdyn[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smdyn) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t mbar[kBars];
  __shared__ uint32_t tmem_slot;
  // Forward: what is not finite in v would meet the zeros of X and Y, and so reach tokens before it.  Two warps look at a chunk's v while the first products
  // run.  Where they find something they put zeros in its place, the products are issued once more before they count, and answers, rest and state of
  // such a column are NaN from its first such token on: `lost`, of halves of 64 columns that have any.  A chunk's place is used again four chunks later: its v
  // is there only when the rows and the answers of the one three before it have been read.  v has a barrier of its own, as it lands before the rest.
  // 1 x 16384 x 32 heads: 498 us, 493 without a look; 658 when v landed with the rest, 569 when the products waited for it, 568 with a look in pairs_kernel.
  __shared__ int lost[BACK ? 1 : 4][BACK ? 1 : 128], any_lost[BACK ? 1 : 4][2];
  const Args& a = w.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int h = blockIdx.y, kh = h / a.group, v0 = blockIdx.x * 128;
  if ((int)blockIdx.z == a.seqs) {  // packed: rows behind the last sequence are zeros
    const int from = a.where.table[2 * a.seqs - 1], cols = min(128, a.vd - v0) / 8;
    T* o = reinterpret_cast<T*>(w.o);
    for (int64_t i = tid; i < (int64_t)(a.len - from) * cols; i += kWalkThreads)
      *reinterpret_cast<uint4*>(o + ((from + i / cols) * a.heads + h) * (int64_t)a.vd + v0 + i % cols * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const Span s = sequence(a.where, blockIdx.z);
  const int nchunks = (s.t1 - s.t0 + C - 1) / C;
  const bool packed = a.where.table != nullptr;
  auto bar = [&](int i) { return tc::smem_u32(&mbar[i]); };
  auto wait = [&](int i, int n) { return (bool)__all_sync(0xffffffffu, phase_done(bar(i), n & 1)); };  // for the n-th completion
  if (warp == 0) tc::tmem_alloc(tc::smem_u32(&tmem_slot), 512);
  if (tid == 0) {
    for (int i = 0; i < kBars; ++i) {
      const bool rows = i == kState || i == kU, help = i == kPrep || i == kPrep + 1 || i == kOut, seen = i == kSeen || i == kSeen + 1;
      tc::mbar_init(bar(i), i >= kFreeL && i < kFreeL + M::NL ? 1 + (kCompute + kHelp) / 32 : rows ? kCompute / 32 : help ? kHelp / 32 : seen ? 2 : 1);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  auto chunk_at = [&](int p) { return BACK ? nchunks - 1 - p : p; };  // position in the walk -> chunk of the sequence
  auto done = [&](int i) {                                            // this warp's part of a phase
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(bar(i));
  };
  auto together = [](bool mine) {  // the helping warps meet, with one verdict
    uint32_t all;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.aligned.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}\n"
        : "=r"(all)
        : "r"((uint32_t)mine), "n"(kHelp)
        : "memory");
    return all != 0;
  };
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const int row = (warp & 3) * 32 + lane, v = v0 + row;  // rows of the state: a warp reaches the lanes of its quarter
  const bool live = v < a.vd;
  bool ok = true;

  if (warp >= (kCompute + kHelp) / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kIssueRegs));
    if (warp == (kCompute + kHelp) / 32) {  // ---- copies
      auto pair_at = [&](int p) { return (int64_t)(s.chunk + chunk_at(p)) * a.heads + h; };
      const unsigned char* wide = BACK ? w.in.wb : w.in.wz;
      auto early = [&](int p) {
        if (lane == 0) {
          const uint32_t full = bar(kFullE + p % M::NE), full_v = BACK ? full : bar(kFullV + p % M::NE), d = tc::smem_u32(sm + p % M::NE * M::EARLY);
          if constexpr (!BACK) tc::mbar_expect_tx(full_v, M::VB);
          tc::mbar_expect_tx(full, BACK ? M::EARLY : M::EARLY - M::VB);
          for (int b = 0; b < 2; ++b) tc::tma_load_4d(d + M::V + b * kTileBytes, &maps.v, full_v, v0 + b * 64, h, s.t0 + chunk_at(p) * C, s.b);
          if constexpr (!BACK) tc::bulk_load(d + M::X, w.in.x + pair_at(p) * kTileBytes, kTileBytes, full);
          tc::bulk_load(d + M::X + M::XB - kTileBytes, w.in.y + pair_at(p) * kTileBytes, kTileBytes, full);
          tc::bulk_load(d + M::W, wide + pair_at(p) * M::WB, M::WB, full);
        }
        __syncwarp();
      };
      auto late = [&](int p) {
        if (lane == 0) {
          const int t = s.t0 + chunk_at(p) * C;
          const uint32_t full = bar(kFullL + p % M::NL), d = tc::smem_u32(sm + M::NE * M::EARLY + p % M::NL * M::LATE);
          tc::mbar_expect_tx(full, M::LATE);
          for (int b = 0; b < KD / 64; ++b) {
            tc::tma_load_4d(d + M::K + b * kTileBytes, &maps.k, full, b * 64, kh, t, s.b);
            if constexpr (BACK) tc::tma_load_4d(d + M::Q + b * kTileBytes, &maps.q, full, b * 64, kh, t, s.b);
          }
          tc::bulk_load(d + M::VEC, w.in.vec + pair_at(p) * (4 * C), M::VEC_BYTES, full);
        }
        __syncwarp();
      };
      int ne = 0, nl = 0;
      while (ne < min(M::NE, nchunks)) early(ne++);
      while (nl < min(M::NL, nchunks)) late(nl++);
      for (int p = 0; p < nchunks && ok; ++p) {
        if (ne < nchunks && (ok = wait(kFreeE + p % M::NE, p / M::NE))) {
          if (ne + 1 < nchunks && lane == 0) {  // the next one's on their way into the L2
            for (int b = 0; b < 2 && v0 + b * 64 < a.vd; ++b) tc::tma_prefetch_4d(&maps.v, v0 + b * 64, h, s.t0 + chunk_at(ne + 1) * C, s.b);
            tc::bulk_prefetch(wide + pair_at(ne + 1) * M::WB, M::WB);
            tc::bulk_prefetch(w.in.y + pair_at(ne + 1) * kTileBytes, kTileBytes);
            if constexpr (!BACK) tc::bulk_prefetch(w.in.x + pair_at(ne + 1) * kTileBytes, kTileBytes);
          }
          early(ne++);
        }
        if (ok && nl < nchunks && (ok = wait(kFreeL + p % M::NL, p / M::NL))) late(nl++);
      }
      // nothing is under way when the block ends
      for (int p = max(0, ne - M::NE); p < ne; ++p) ok = wait(kFullE + p % M::NE, p / M::NE) && (BACK || wait(kFullV + p % M::NE, p / M::NE)) && ok;
      for (int p = max(0, nl - M::NL); p < nl; ++p) ok = wait(kFullL + p % M::NL, p / M::NL) && ok;
    } else if (warp == (kCompute + kHelp) / 32 + 1) {  // ---- products
      constexpr int fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      constexpr int N1 = BACK ? C : 2 * C;  // r, and forward o beside it
      constexpr uint32_t id_s = tc::instr_desc(128, C, fmt, 0, 0);               // state x W^T, Z^T; Wb^T
      constexpr uint32_t id_v = tc::instr_desc(128, N1, fmt, 1, BACK ? 1 : 0);   // V^T x X^T, Y^T; do^T x Y
      constexpr uint32_t id_k = tc::instr_desc(128, KD, fmt, 0, 1);              // weighted rows x K
      constexpr uint32_t id_doq = tc::instr_desc(128, KD, fmt, 1, 1);            // do^T Q
      for (int p = 0; p < nchunks; ++p) {
        const int se = p % M::NE, sl = p % M::NL;
        if (!(ok = wait(kFullE + se, p / M::NE) && (BACK || wait(kFullV + se, p / M::NE)) && wait(kFullL + sl, p / M::NL) && wait(kPrep + (p & 1), p >> 1)))
          break;  // rows of another sequence cut; BACK: q scaled
        tc::fence_after_sync();
        const uint32_t e = tc::smem_u32(sm + se * M::EARLY), l = tc::smem_u32(sm + M::NE * M::EARLY + sl * M::LATE), R = tmem + TC::RO + (p & 1) * 128;
        const uint64_t w_rows = tc::smem_desc_sw128(e + M::W, 16, 1024), v_cols = tc::smem_desc_sw128(e + M::V, kTileBytes, 1024);
        const uint64_t x_rows = tc::smem_desc_sw128(e + M::X, 16, 1024), y_cols = tc::smem_desc_sw128(e + M::X, kTileBytes, 1024);
        const uint64_t k_cols = tc::smem_desc_sw128(l + M::K, kTileBytes, 1024), q_cols = tc::smem_desc_sw128(l + M::Q, kTileBytes, 1024);
        auto along = [](int kk) { return (uint64_t)(((kk >> 2) * (N1 * 128) + (kk & 3) * 32) >> 4); };  // 16 columns further in a tile of N1 rows
        auto down = [](int kk) { return (uint64_t)(kk * (2048 >> 4)); };                                // 16 rows further
        auto first = [&] {
#pragma unroll
          for (int kk = 0; kk < C / 16; ++kk) tc::mma_ss(R, v_cols + down(kk), BACK ? y_cols + down(kk) : x_rows + along(kk), id_v, kk > 0);
        };
        auto second = [&] {
#pragma unroll
          for (int kk = 0; kk < KD / 16; ++kk) tc::mma_ts(R, tmem + TC::S + kk * 8, w_rows + along(kk), id_s, true);
        };
        if (tc::elect_one()) first();
        __syncwarp();
        if (BACK && p > 0 && !(ok = wait(kOut, p - 1))) break;  // the results before these have been read: kR is not two ahead of the helping warps
        if (!(ok = wait(kState, p))) break;
        tc::fence_after_sync();
        if (tc::elect_one()) {
          second();
          if constexpr (BACK) tc::commit(bar(kR));
        }
        __syncwarp();
        if constexpr (!BACK) {
          if (!(ok = wait(kSeen + (p & 1), p >> 1))) break;
          const bool again = any_lost[p & 3][0] + any_lost[p & 3][1] != 0;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            if (again) first(), second();
            tc::commit(bar(kR));
          }
          __syncwarp();
        }
        // beside the rows' step
        if (!BACK && p > 0 && !(ok = wait(kOut, p - 1))) break;
        tc::fence_after_sync();
        if (tc::elect_one()) {
          if constexpr (BACK) {
#pragma unroll
            for (int kk = 0; kk < C / 16; ++kk) tc::mma_ss(tmem + TC::DS, v_cols + down(kk), q_cols + down(kk), id_doq, kk > 0);
          } else {
#pragma unroll
            for (int kk = 0; kk < KD / 16; ++kk) tc::mma_ts(R + C, tmem + TC::S + kk * 8, w_rows + (uint64_t)(kTileBytes >> 4) + along(kk), id_s, true);
            tc::commit(bar(kO));
          }
          tc::commit(bar(kFreeE + se));
        }
        __syncwarp();
        if (!(ok = wait(kU, p))) break;
        tc::fence_after_sync();
        if (tc::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < C / 16; ++kk) tc::mma_ts(tmem + TC::DS, tmem + TC::U + kk * 8, k_cols + down(kk), id_k, BACK || kk > 0);
          tc::commit(bar(kDS));
          tc::commit(bar(kFreeL + sl));
        }
        __syncwarp();
      }
      if (tc::elect_one()) tc::commit(bar(kEnd));  // nothing is under way when the block ends, nor where a wait ran out
      __syncwarp();
      ok = wait(kEnd, 0) && ok;
    } else if (!BACK) {  // ---- a look at 64 columns of v
      const int half = warp & 1;
      for (int p = 0; p < nchunks && (ok = wait(kFullV + p % M::NE, p / M::NE)); ++p) {
        int* mine = &lost[BACK ? 0 : p & 3][BACK ? 0 : half * 64];
        mine[lane] = mine[lane + 32] = C;
        __syncwarp();
        const int n = min(C, s.t1 - (s.t0 + p * C));  // what lies behind belongs to the next sequence
        unsigned char* tile = sm + p % M::NE * M::EARLY + M::V + half * kTileBytes;
        uint32_t hits = 0;
#pragma unroll 4
        for (int i = 0; i < C / 4; ++i) {
          const int r = lane / 8 + i * 4;
          const uint32_t hit = not_finite<T>(*reinterpret_cast<const uint4*>(tile + swz(r, lane & 7)));
          hits |= r < n ? hit : 0u;
        }
        const bool found = __any_sync(0xffffffffu, hits != 0);
        if (found) {
          for (int i = lane; i < n * 64; i += 32) {
            constexpr uint16_t ones = std::is_same<T, __nv_bfloat16>::value ? 0x7f80 : 0x7c00;
            uint16_t* x = reinterpret_cast<uint16_t*>(tile + swz(i / 64, i % 64 / 8)) + i % 8;
            if ((*x & ones) == ones) *x = 0, atomicMin(&mine[i % 64], i / 64);
          }
          tc::fence_async_smem();
        }
        if (lane == 0) any_lost[BACK ? 0 : p & 3][half] = found;
        done(kSeen + (p & 1));
      }
    }
  } else if (warp >= kCompute / 32) {  // ---- operands prepared, results stored
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kHelpRegs));
    const int me = tid - kCompute;
    auto tokens_of = [&](int p) { return min(C, s.t1 - (s.t0 + chunk_at(p) * C)); };
    // rows of another sequence cut from the products over tokens; BACK: q times scale gam
    auto late_at = [&](int p) { return sm + M::NE * M::EARLY + p % M::NL * M::LATE; };
    auto prepare = [&](int p) {
      const int n = tokens_of(p);
      const bool cut = packed && n < C;
      if (!wait(kFullL + p % M::NL, p / M::NL) || (cut && !wait((BACK ? kFullE : kFullV) + p % M::NE, p / M::NE))) return false;
      unsigned char *d = late_at(p), *e = sm + p % M::NE * M::EARLY;
      constexpr int U = KD / 8;
      if constexpr (BACK) {
        const float* sg = reinterpret_cast<const float*>(d + M::VEC) + 3 * C;
#pragma unroll 4
        for (int i = me; i < C * U; i += kHelp) {
          const int r = i / U, u = i % U;
          uint4* at = reinterpret_cast<uint4*>(d + M::Q + (u >> 3) * kTileBytes + swz(r, u & 7));
          const float m = sg[r];
          const uint4 x = *at;
          const uint32_t in[4] = {x.x, x.y, x.z, x.w};
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 z = unpack2<T>(in[e]);
            y[e] = r < n ? pack2<T>(z.x * m, z.y * m) : 0u;
          }
          *at = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
      if (cut) {
        for (int i = me; i < (C - n) * U; i += kHelp) *reinterpret_cast<uint4*>(d + M::K + (i % U >> 3) * kTileBytes + swz(n + i / U, i % U & 7)) = make_uint4(0, 0, 0, 0);
        for (int i = me; i < (C - n) * 16; i += kHelp) *reinterpret_cast<uint4*>(e + M::V + (i % 16 >> 3) * kTileBytes + swz(n + i / 16, i % 16 & 7)) = make_uint4(0, 0, 0, 0);
      }
      if (BACK || cut) tc::fence_async_smem();
      done(kPrep + (p & 1));
      return true;
    };
    unsigned char* out = sm + M::OUT;  // rows of tokens on their way out, two blocks of 64 columns
    uint32_t unit[8];                  // where this thread's column lies in them, by the row's place in the swizzle
#pragma unroll
    for (int e = 0; e < 8; ++e) unit[e] = tc::smem_u32(out) + (row >> 6) * kTileBytes + swz(e, (row & 63) >> 3) + (row & 7) * 2;
    if (nchunks > 0) ok = prepare(0);
    for (int p = 0; p < nchunks; ++p) {
      ok = ok && (p + 1 >= nchunks || prepare(p + 1)) && wait(BACK ? kR : kO, p);
      if (!(ok = together(ok))) break;  // all four warps or none
      tc::fence_after_sync();
      const int n = tokens_of(p), t = s.t0 + chunk_at(p) * C, buf = (p & 1) * M::VB;
      uint32_t x[2][32];  // 64 tokens of this thread's row
#pragma unroll
      for (int q = 0; q < 2; ++q) ld32(tmem + lanes + TC::RO + (p & 1) * 128 + (BACK ? 0 : C) + q * 32, x[q]);
      landed(x[0]), landed(x[1]);
      done(kOut);
      if (!BACK && any_lost[BACK ? 0 : p & 3][row >> 6]) {
        const int from = lost[BACK ? 0 : p & 3][BACK ? 0 : row];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (q * 32 + e >= from) x[q][e] = 0x7fc00000u;
      }
      if (me == 0) asm volatile("cp.async.bulk.wait_group.read 1;\n" ::: "memory");  // the tile of the chunk before the last has left
      together(true);
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint32_t z = pack2<T>(f(x[q][e]), f(x[q][e + 1]));
          put16(unit[e & 7] + buf + (q * 32 + (e & ~7)) * 128, (uint16_t)z);
          put16(unit[(e + 1) & 7] + buf + (q * 32 + (e & ~7)) * 128, (uint16_t)(z >> 16));
        }
      tc::fence_async_smem();
      together(true);
      if (!packed || n == C) {  // TMA cuts at the tensor's end
        if (me == 0) {
          tc::tma_store_4d(&maps.o, tc::smem_u32(out + buf), v0, h, t, s.b);
          if (v0 + 64 < a.vd) tc::tma_store_4d(&maps.o, tc::smem_u32(out + buf + kTileBytes), v0 + 64, h, t, s.b);
          tc::bulk_commit();
        }
      } else {  // what follows belongs to the next sequence
        T* o = reinterpret_cast<T*>(w.o);
        const int units = min(128, a.vd - v0) / 8;
        for (int i = me; i < n * units; i += kHelp)
          *reinterpret_cast<uint4*>(o + ((int64_t)(t + i / units) * a.heads + h) * a.vd + v0 + i % units * 8) =
              *reinterpret_cast<const uint4*>(out + buf + (i % units >> 3) * kTileBytes + swz(i / units, i % units & 7));
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar(kFreeL + p % M::NL));
    }
    if (me == 0) tc::bulk_wait_all();
  } else {  // ---- rows of the state: lane = row, the warps of a lane quarter share the columns
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kComputeRegs));
    const int part = warp >> 2;
    constexpr int NS = KD / kParts, NT = C / kParts;  // columns of the state and tokens of a thread
    float S[NS];
    const int64_t state_at = (((int64_t)s.seq * a.heads + h) * a.vd + v) * a.kd + part * NS;
#pragma unroll
    for (int e = 0; e < NS; e += 4) {
      const bool in = w.initial && live && part * NS + e < a.kd;  // kdim is a multiple of 8
      const float4 x = in ? __ldg(reinterpret_cast<const float4*>(w.initial + state_at + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[e] = x.x, S[e + 1] = x.y, S[e + 2] = x.z, S[e + 3] = x.w;
    }
    // kept for a backward pass: slices of 64 columns v (`width` in the last one), of each its units of eight elements, of each its columns
    const int width = min(kSlice, a.vd - v / kSlice * kSlice);
    auto unit_at = [&](int units, int u) { return v / kSlice * kSlice * units + u * width + v % kSlice; };
    // the state as an operand, and for a backward pass to follow
    uint32_t x16[NS / 2];
    auto keep_units = [&](int p, int from, int to) {
      uint4* keep = reinterpret_cast<uint4*>(w.states) + ((int64_t)(s.chunk + chunk_at(p)) * a.heads + h) * (KD / 8) * a.vd + unit_at(KD / 8, part * (NS / 8));
#pragma unroll
      for (int u = 0; u < NS / 8; ++u)
        if (u >= from && u < to) keep[u * width] = make_uint4(x16[4 * u], x16[4 * u + 1], x16[4 * u + 2], x16[4 * u + 3]);
    };
    auto publish = [&](int p) {
      auto& x = x16;
#pragma unroll
      for (int e = 0; e < NS / 2; ++e) x[e] = pack2<T>(S[2 * e], S[2 * e + 1]);
#pragma unroll
      for (int q = 0; q < NS / 32; ++q) tc::tmem_st16(tmem + lanes + TC::S + part * (NS / 2) + q * 16, reinterpret_cast<const uint32_t(&)[16]>(x[q * 16]));
      tc::tmem_wait_st();
      done(kState);
      if (w.states && live) keep_units(p, 0, BACK ? NS / 16 : NS / 8);
    };
    if (nchunks > 0) publish(0);
    for (int p = 0; p < nchunks; ++p) {
      const int sl = p % M::NL;
      if (!(ok = wait(kFullL + sl, p / M::NL))) break;
      const float* vec = reinterpret_cast<const float*>(sm + M::NE * M::EARLY + sl * M::LATE + M::VEC);
      const float* weight = vec + (BACK ? 0 : 2 * C) + part * NT;  // beta suf; BACK: gam
      const float whole = vec[C - 1];
      float4 m[NT / 4];
#pragma unroll
      for (int e = 0; e < NT / 4; ++e) m[e] = *reinterpret_cast<const float4*>(weight + 4 * e);
      uint32_t x[NT];
      if (!(ok = wait(kR, p))) break;
      tc::fence_after_sync();
      const bool spoilt = !BACK && any_lost[BACK ? 0 : p & 3][row >> 6];
      ld32(tmem + lanes + TC::RO + (p & 1) * 128 + part * NT, x);
      landed(x);
      {
        uint32_t y[NT / 2];
        constexpr float sign = BACK ? -1.f : 1.f;
#pragma unroll
        for (int e = 0; e < NT / 4; ++e)
          y[2 * e] = pack2<T>(sign * f(x[4 * e]) * m[e].x, sign * f(x[4 * e + 1]) * m[e].y), y[2 * e + 1] = pack2<T>(sign * f(x[4 * e + 2]) * m[e].z, sign * f(x[4 * e + 3]) * m[e].w);
        tc::tmem_st16(tmem + lanes + TC::U + part * (NT / 2), y);
        tc::tmem_wait_st();
        done(kU);
        if constexpr (BACK)  // the rest of the state here, where the rows wait again: 124 us, 141 in one piece
          if (w.states && live) keep_units(p, NS / 16, NS / 8);
        if constexpr (!BACK)
          if (w.rest && live) {
            if (spoilt) {
              const int from = lost[p & 3][row] - part * NT;
#pragma unroll
              for (int e = 0; e < NT; ++e)
                if (e >= from) x[e] = 0x7fc00000u;
            }
#pragma unroll
            for (int e = 0; e < NT / 2; ++e) y[e] = pack2<T>(f(x[2 * e]), f(x[2 * e + 1]));
            uint4* to = reinterpret_cast<uint4*>(w.rest) + ((int64_t)(s.chunk + chunk_at(p)) * a.heads + h) * (C / 8) * a.vd + unit_at(C / 8, part * (NT / 8));
#pragma unroll
            for (int q = 0; q < NT / 8; ++q) to[q * width] = make_uint4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
          }
      }
      if (!(ok = wait(kDS, p))) break;
      tc::fence_after_sync();
      uint32_t z[NS / 32][32];
#pragma unroll
      for (int q = 0; q < NS / 32; ++q) ld32(tmem + lanes + TC::DS + part * NS + q * 32, z[q]);
#pragma unroll
      for (int q = 0; q < NS / 32; ++q) {
        landed(z[q]);
#pragma unroll
        for (int e = 0; e < 32; ++e) S[q * 32 + e] = fmaf(whole, S[q * 32 + e], f(z[q][e]));
      }
      if (spoilt && lost[BACK ? 0 : p & 3][BACK ? 0 : row] < C) {
#pragma unroll
        for (int e = 0; e < NS; ++e) S[e] = f(0x7fc00000u);
      }
      if (p + 1 < nchunks) publish(p + 1);
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar(kFreeL + sl));
    }
    if (ok && live && w.last) {
#pragma unroll
      for (int e = 0; e < NS; ++e)
        if (part * NS + e < a.kd) store_dyn(w.last, state_at + e, w.last_dtype, S[e]);
    }
  }
  if (!ok && lane == 0 && w.in.status) *(volatile int32_t*)w.in.status = BACK ? 5 : 4;
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem_slot, 512);
}

// ---------------------------------------------------------------------------------------------
// gradients of a chunk's tokens
// ---------------------------------------------------------------------------------------------
// With N1_ij = do_i.r_j, N2_ij = w_i.r_j, S0 the state before and D the adjoint state behind the chunk:
//   dq_i = scale gam_i S0^T do_i + sum_{j<=i} scale G_ij N1_ij beta_j k_j
//   y_i = suf_i D^T r_i + scale sum_{j>=i} G_ji N1_ji q_j - sum_{j>i} G_ji N2_ji k_j;   dbeta_i = k_i.y_i
//   dk_i = beta_i y_i - gam_i S0^T w_i - sum_{j<i} G_ij N2_ij beta_j k_j
//   dg_t = gam_64 <S0, D> + sum_{i<t} beta_i suf_i k_i.(D^T r_i) + sum_{i>=t} gam_i (scale q_i.(S0^T do_i) - k_i.(S0^T w_i)) + sum_{j<t<=i} M_ij,
//   M_ij = G_ij beta_j (scale N1_ij q_i.k_j - N2_ij k_i.k_j): every path from before t to t or behind it
// Sixteen warps, each 16 tokens x a quarter of the columns, products by mma.sync (15 Mflop a chunk); one block an SM that walks over its
// chunks, 64 columns of v at a time, with the next two slices' copies under way (145 KB read and 32 KB written a chunk).  A slice of the states
// lies in one piece, since copies of a kilobyte each cost their warp more than its products (187 -> 164 us).  Bound: instructions, some 2100 a
// warp and chunk at 1.7 a cycle, of which 200 are products.  2 x 4096 tokens x 16 heads: 160 us, 2.2 TB/s; with eight warps and a block a chunk 204.
struct GradMaps {
  CUtensorMap q, k, d, w;
};
struct ChunkGrads {
  Args a;
  const void* rest;     // [slice of vdim][token / 8][column][8]
  const void* states;   // [slice of vdim][kdim / 8][column][8]
  const void* dstates;
  void* dq;
  void* dk;
  float* dqk;  // fp32, per value head: dq then dk; NULL where heads do not share keys
  float* dg;
  float* dbeta;
  int64_t tokens;
  int chunks;
  int32_t* status;
};
constexpr int kGradThreads = 512;
template <int KD>
struct GradSmem {
  static constexpr int KT = (KD / 64) * kTileBytes, RT = (C / 8) * kSlice * 16, ST = (KD / 8) * kSlice * 16;
  // a slice of the columns of v (two of them), q and k (two of them), the matrices of pairs, later dq and dk
  static constexpr int D = 0, W = kTileBytes, R = 2 * kTileBytes, S = R + RT, DS = S + ST, SLICE = DS + ST, Q = 0, K = KT, QK = 2 * SLICE, Y1 = QK + 4 * KT, Y2 = Y1 + kTileBytes,
                       A1 = Y2 + kTileBytes, A2 = A1 + kTileBytes, VEC = A2 + kTileBytes, TOTAL = VEC + (24 * C + kGradThreads / 32) * 4;
  static constexpr int ALLOC = TOTAL + 1024;
};
static_assert(GradSmem<128>::ALLOC <= 227 * 1024, "shared memory of an SM");

// Units of 16 bytes (8 elements along the first axis of a matrix, one place v): unit (c, v) at (c kSlice + v) 16.
// B[k = v][n]: two neighbouring blocks of eight columns n0 .., depth v0 ..
__device__ __forceinline__ void units_b(uint32_t (&f)[4], uint32_t base, int n0, int v0, int lane) { ldsm4t(f, base + (((n0 >> 3) + (lane >> 4)) * kSlice + v0 + (lane & 15)) * 16); }
// A[m][k = v]: rows m0 .. + 15
__device__ __forceinline__ void units_a(uint32_t (&f)[4], uint32_t base, int m0, int v0, int lane) {
  ldsm4t(f, base + (((m0 >> 3) + ((lane >> 3) & 1)) * kSlice + v0 + (lane & 7) + ((lane >> 4) << 3)) * 16);
}
// A[m][k] = tile[k][m]
__device__ __forceinline__ void load_at(uint32_t (&f)[4], uint32_t tile, int m0, int k0, int lane) {
  const int row = k0 + (lane & 7) + ((lane >> 4) << 3), unit = m0 / 8 + ((lane >> 3) & 1);
  ldsm4t(f, tile + (unit >> 3) * kTileBytes + swz(row, unit & 7));
}

template <typename T, int KD>
__global__ void __launch_bounds__(kGradThreads, 1) grads_kernel(const ChunkGrads g, const __grid_constant__ GradMaps maps) {
  using M = GradSmem<KD>;
  constexpr int NB = KD / 32;  // blocks of eight columns of a warp: a quarter of kdim
  extern __shared__ unsigned char smdyn[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smdyn) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t mbar[2];
  const Args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  T* dq = reinterpret_cast<T*>(g.dq);
  T* dk = reinterpret_cast<T*>(g.dk);
  const int items = g.chunks * a.heads, slices = (a.vd + kSlice - 1) / kSlice;
  if (a.where.table)  // rows of no sequence
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
      const Span s = chunk_of(a.where, it % g.chunks, C);
      const int n = s.t1 - s.t0, h = it / g.chunks;
      if (n <= 0 || s.seq >= 0) continue;
      const int64_t tok = (int64_t)s.b * a.len + s.t0;
      for (int at = tid; at < n * a.kd; at += kGradThreads) {
        const int64_t to = ((tok + at / a.kd) * a.heads + h) * a.kd + at % a.kd;
        if (g.dqk) g.dqk[to] = 0.f, g.dqk[g.tokens * a.heads * a.kd + to] = 0.f;
        else dq[to] = from_f<T>(0.f), dk[to] = from_f<T>(0.f);
      }
      for (int i = tid; i < n; i += kGradThreads) g.dg[(tok + i) * a.heads + h] = 0.f, g.dbeta[(tok + i) * a.heads + h] = 0.f;
    }
  // the others, in this block's order
  struct Item {
    int it, h;
    Span s;
  };
  auto from_on = [&](int it) {
    Item x{it, 0, {}};
    for (; x.it < items; x.it += gridDim.x) {
      x.h = x.it / g.chunks, x.s = chunk_of(a.where, x.it - x.h * g.chunks, C);
      if (x.s.t1 > x.s.t0 && x.s.seq >= 0) break;
    }
    return x;
  };
  const uint32_t base = tc::smem_u32(sm), bars = tc::smem_u32(mbar);
  float* c = reinterpret_cast<float*>(sm + M::VEC);
  float *beta = c + C, *gam = beta + C, *suf = gam + C, *rows = suf + C, *cols = rows + 4 * C;  // [4][C] each: sums of M
  float *into = cols + 4 * C, *outof = into + 4 * C, *db = outof + 4 * C, *part = db + 4 * C;   // [4][C] each; a partial sum of every warp
  // a slice's copies, by warp 0: what follows is on its way while a chunk is worked on
  auto request = [&](const Item& x, int slice, int to_slice, int to_qk) {
    const Span& s = x.s;
    const int h = x.h, kh = h / a.group, v0 = slice * kSlice, nv = min(kSlice, a.vd - v0);
    const int64_t pair = (int64_t)s.chunk * a.heads + h;
    const uint32_t bar = bars + to_slice * 8, to = base + to_slice * M::SLICE, qk = base + M::QK + to_qk * 2 * M::KT;
    if (lane == 0) {
      tc::mbar_expect_tx(bar, 2 * kTileBytes + (C / 8 + 2 * (KD / 8)) * nv * 16 + (v0 ? 0 : 2 * M::KT));
      for (int b = 0; b < KD / 64 && v0 == 0; ++b) {
        tc::tma_load_4d(qk + M::Q + b * kTileBytes, &maps.q, bar, b * 64, kh, s.t0, s.b);
        tc::tma_load_4d(qk + M::K + b * kTileBytes, &maps.k, bar, b * 64, kh, s.t0, s.b);
      }
      tc::tma_load_4d(to + M::D, &maps.d, bar, v0, h, s.t0, s.b);
      tc::tma_load_4d(to + M::W, &maps.w, bar, v0, h, s.t0, s.b);
    }
    __syncwarp();
    if (nv == kSlice) {  // in one piece
      if (lane == 0) {
        const int64_t from = (pair * a.vd + v0) * 16;
        auto piece = [&](int at, const void* p, int units) { tc::bulk_load(to + at, reinterpret_cast<const unsigned char*>(p) + from * units, units * (kSlice * 16), bar); };
        piece(M::R, g.rest, C / 8), piece(M::S, g.states, KD / 8), piece(M::DS, g.dstates, KD / 8);
      }
      __syncwarp();
      return;
    }
    for (int u = lane; u < C / 8 + 2 * (KD / 8); u += 32) {
      const int i = u < C / 8 ? u : (u - C / 8) % (KD / 8), units = u < C / 8 ? C / 8 : KD / 8;
      const void* from = u < C / 8 ? g.rest : u < C / 8 + KD / 8 ? g.states : g.dstates;
      const int at = u < C / 8 ? M::R : u < C / 8 + KD / 8 ? M::S : M::DS;
      tc::bulk_load(to + at + i * (kSlice * 16), reinterpret_cast<const unsigned char*>(from) + ((pair * a.vd + v0) * units + i * nv) * 16, nv * 16, bar);
    }
  };
  if (tid == 0) tc::mbar_init(bars, 1), tc::mbar_init(bars + 8, 1);
  __syncthreads();
  Item now = from_on(blockIdx.x);
  int used = 0, asked = 0, ahead = 0, ahead_slice = 0;  // slices worked on and asked for; the next to ask for, `ahead` chunks from the current one
  const int r0 = (warp >> 2) * 16, quarter = (warp + (warp >> 2)) & 3, c0 = quarter * 16, k_cols = quarter * (KD / 4), gi = lane >> 2, gj = (lane & 3) * 2;
  TokenPair token{};
  auto tokens_of = [&](const Item& x) {
    if (x.it < items) token = token_pair(a, x.s, x.s.t1 - x.s.t0, x.h, lane);
  };
  constexpr int kDecays = 5, kSums = 10;  // warps that do more than their share, each with another scheduler; warp 0 asks for the copies
  if (warp == kDecays) tokens_of(now);
  for (int order = 0; now.it < items; ++order) {
    const Item next = from_on(now.it + gridDim.x);
    const Span s = now.s;
    const int n = s.t1 - s.t0, h = now.h;
    const int64_t tok = (int64_t)s.b * a.len + s.t0;
    unsigned char* qk = sm + M::QK + (order & 1) * 2 * M::KT;
    const uint32_t qk_base = tc::smem_u32(qk);
    auto feed = [&] {  // as far as there are buffers: two of slices, and for q and k this chunk's and the next one's
      for (; asked - used < 2 && ahead < 2 && (ahead ? next.it : now.it) < items; ++asked) {
        if (warp == 0) request(ahead ? next : now, ahead_slice, asked & 1, (order + ahead) & 1);
        if (++ahead_slice == slices) ahead_slice = 0, ++ahead;
      }
    };
    feed();
    if (warp == kDecays) {
      decay_logs(token, c, beta, lane);
      __syncwarp();
      for (int i = lane; i < C; i += 32) gam[i] = ex2_approx(c[i]), suf[i] = ex2_approx(c[C - 1] - c[i]);
    }
    float N1[2][4] = {}, N2[2][4] = {}, dQ[NB][4] = {}, dK[NB][4] = {}, y[NB][4] = {}, whole = 0.f;
    for (int v0 = 0; v0 < a.vd; v0 += kSlice) {
      const int nv = min(kSlice, a.vd - v0);
      unsigned char* sl = sm + (used & 1) * M::SLICE;
      const uint32_t slice = tc::smem_u32(sl);
      if (!__syncthreads_and(phase_done(bars + (used & 1) * 8, used >> 1 & 1))) {
        if (tid == 0 && g.status) *(volatile int32_t*)g.status = 7;
        for (; used < asked; ++used) phase_done(bars + (used & 1) * 8, used >> 1 & 1);  // nothing is under way when the block ends
        return;
      }
      if (a.where.table && n < C) {  // rows of the next sequence: nothing of them may enter a product, not even times zero
        constexpr int U = KD / 8;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < (C - n) * U; i += kGradThreads) {
          const int at = (i % U >> 3) * kTileBytes + swz(n + i / U, i % U & 7);
          *reinterpret_cast<uint4*>(qk + M::Q + at) = zero, *reinterpret_cast<uint4*>(qk + M::K + at) = zero;
        }
        for (int i = tid; i < (C - n) * 8; i += kGradThreads) {
          const int at = swz(n + i / 8, i % 8);
          *reinterpret_cast<uint4*>(sl + M::D + at) = zero, *reinterpret_cast<uint4*>(sl + M::W + at) = zero;
        }
      }
      if (nv % 16) {  // products take 16 columns of v at a time
        for (int i = tid; i < (C / 8 + 2 * (KD / 8)) * 8; i += kGradThreads) {
          const int u = i / 8, at = u < C / 8 ? M::R + u * (kSlice * 16) : M::S + (u - C / 8) * (kSlice * 16);  // the adjoint state follows the state
          *reinterpret_cast<uint4*>(sl + at + (nv + i % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      if (nv % 16 || (a.where.table && n < C)) __syncthreads();
      for (int k0 = 0; k0 < nv; k0 += 16) {
        uint32_t fd[4], fw[4], fr[4], b[4];
        load_a(fd, slice + M::D, r0, k0, lane);
        load_a(fw, slice + M::W, r0, k0, lane);
        units_a(fr, slice + M::R, r0, k0, lane);
        if (c0 <= r0) {
          units_b(b, slice + M::R, c0, k0, lane);
          mma16816<T>(N1[0], fd, b[0], b[1]), mma16816<T>(N1[1], fd, b[2], b[3]);
          mma16816<T>(N2[0], fw, b[0], b[1]), mma16816<T>(N2[1], fw, b[2], b[3]);
        }
#pragma unroll
        for (int n0 = 0; n0 < NB * 8; n0 += 16) {
          units_b(b, slice + M::S, k_cols + n0, k0, lane);
          mma16816<T>(dQ[n0 / 8], fd, b[0], b[1]), mma16816<T>(dQ[n0 / 8 + 1], fd, b[2], b[3]);
          mma16816<T>(dK[n0 / 8], fw, b[0], b[1]), mma16816<T>(dK[n0 / 8 + 1], fw, b[2], b[3]);
          units_b(b, slice + M::DS, k_cols + n0, k0, lane);
          mma16816<T>(y[n0 / 8], fr, b[0], b[1]), mma16816<T>(y[n0 / 8 + 1], fr, b[2], b[3]);
        }
      }
#pragma unroll
      for (int i = tid; i < (KD / 8) * kSlice; i += kGradThreads) {
        const int at = i * 16;
        if (i % kSlice >= nv) continue;
        const uint4 x = *reinterpret_cast<const uint4*>(sl + M::S + at), z = *reinterpret_cast<const uint4*>(sl + M::DS + at);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 p = unpack2<T>(xs[e]), q = unpack2<T>(zs[e]);
          whole = fmaf(p.x, q.x, fmaf(p.y, q.y, whole));
        }
      }
      tc::fence_async_smem();  // what was read and written here, before the next copies
      __syncthreads();
      ++used;
      feed();
    }
    if (warp == kDecays) tokens_of(next);
    whole = warp_sum(whole);
    if (lane == 0) part[warp] = gam[C - 1] * whole;  // here: the next chunk's decays may be written during the last sums
    {  // pairs of tokens: this warp's 16 x 16
      float QK[2][4] = {}, KK[2][4] = {};
      if (c0 <= r0) {
#pragma unroll
        for (int k0 = 0; k0 < KD; k0 += 16) {
          uint32_t fq[4], fk[4], b[4];
          load_a(fq, qk_base + M::Q, r0, k0, lane);
          load_a(fk, qk_base + M::K, r0, k0, lane);
          load_b(b, qk_base + M::K, c0, k0, lane);
          mma16816<T>(QK[0], fq, b[0], b[1]), mma16816<T>(QK[1], fq, b[2], b[3]);
          mma16816<T>(KK[0], fk, b[0], b[1]), mma16816<T>(KK[1], fk, b[2], b[3]);
        }
      }
      float row[2] = {0.f, 0.f};
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        const int j0 = c0 + nb * 8 + gj;
        float y1[4], y2[4], a1[4], a2[4], col[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = r0 + gi + (e >> 1) * 8, j = j0 + (e & 1);
          const float G = ex2_approx(c[i] - c[j]), b = beta[j];
          y1[e] = j <= i ? G * a.scale * N1[nb][e] : 0.f;
          y2[e] = j < i ? -G * N2[nb][e] : 0.f;
          a1[e] = b * y1[e], a2[e] = b * y2[e];
          const float m = j < i ? a1[e] * QK[nb][e] + a2[e] * KK[nb][e] : 0.f;
          row[e >> 1] += m, col[e & 1] += m;
        }
#pragma unroll
        for (int off = 4; off <= 16; off *= 2) col[0] += __shfl_xor_sync(0xffffffffu, col[0], off), col[1] += __shfl_xor_sync(0xffffffffu, col[1], off);
        if (gi == 0) cols[(warp >> 2) * C + j0] = col[0], cols[(warp >> 2) * C + j0 + 1] = col[1];
        const int lo = swz(r0 + gi, j0 >> 3) + gj * 2, hi = swz(r0 + gi + 8, j0 >> 3) + gj * 2;
        *reinterpret_cast<uint32_t*>(sm + M::Y1 + lo) = pack2<T>(y1[0], y1[1]), *reinterpret_cast<uint32_t*>(sm + M::Y1 + hi) = pack2<T>(y1[2], y1[3]);
        *reinterpret_cast<uint32_t*>(sm + M::Y2 + lo) = pack2<T>(y2[0], y2[1]), *reinterpret_cast<uint32_t*>(sm + M::Y2 + hi) = pack2<T>(y2[2], y2[3]);
        *reinterpret_cast<uint32_t*>(sm + M::A1 + lo) = pack2<T>(a1[0], a1[1]), *reinterpret_cast<uint32_t*>(sm + M::A1 + hi) = pack2<T>(a1[2], a1[3]);
        *reinterpret_cast<uint32_t*>(sm + M::A2 + lo) = pack2<T>(a2[0], a2[1]), *reinterpret_cast<uint32_t*>(sm + M::A2 + hi) = pack2<T>(a2[2], a2[3]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row[e] += __shfl_xor_sync(0xffffffffu, row[e], 1), row[e] += __shfl_xor_sync(0xffffffffu, row[e], 2);
        if ((lane & 3) == 0) rows[quarter * C + r0 + gi + e * 8] = row[e];
      }
    }
    // the states' parts, scaled, and what dg takes of them
    const float gm[2] = {gam[r0 + gi], gam[r0 + gi + 8]}, sf[2] = {suf[r0 + gi], suf[r0 + gi + 8]}, bt[2] = {beta[r0 + gi], beta[r0 + gi + 8]};
    auto row_sums = [&](float (&x)[2], float* to) {  // over the four lanes of a row, to this quarter's place
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[e] += __shfl_xor_sync(0xffffffffu, x[e], 1), x[e] += __shfl_xor_sync(0xffffffffu, x[e], 2);
        if ((lane & 3) == 0) to[quarter * C + r0 + gi + e * 8] = x[e];
      }
    };
    auto pair_at = [&](int tile, int e, int nb) {  // two neighbouring elements of q or k
      const int col = k_cols + nb * 8;
      return unpack2<T>(*reinterpret_cast<const uint32_t*>(qk + tile + (col >> 6) * kTileBytes + swz(r0 + gi + e * 8, (col & 63) >> 3) + gj * 2));
    };
    {
      float in[2] = {0.f, 0.f}, outp[2] = {0.f, 0.f};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 q = pair_at(M::Q, e, nb), k = pair_at(M::K, e, nb);
          dQ[nb][2 * e] *= gm[e] * a.scale, dQ[nb][2 * e + 1] *= gm[e] * a.scale;
          dK[nb][2 * e] *= -gm[e], dK[nb][2 * e + 1] *= -gm[e];
          y[nb][2 * e] *= sf[e], y[nb][2 * e + 1] *= sf[e];
          in[e] += dQ[nb][2 * e] * q.x + dQ[nb][2 * e + 1] * q.y + dK[nb][2 * e] * k.x + dK[nb][2 * e + 1] * k.y;
          outp[e] += bt[e] * (y[nb][2 * e] * k.x + y[nb][2 * e + 1] * k.y);
        }
      row_sums(in, into), row_sums(outp, outof);
    }
    __syncthreads();  // the pair matrices are written, the states have been read
#pragma unroll
    for (int k0 = 0; k0 < C; k0 += 16) {
      uint32_t fa[4], fb[4], b[4];
      if (k0 <= r0) {  // pairs with tokens before
        load_a(fa, base + M::A1, r0, k0, lane);
        load_a(fb, base + M::A2, r0, k0, lane);
#pragma unroll
        for (int n0 = 0; n0 < NB * 8; n0 += 16) {
          const int col = k_cols + n0;
          load_bt(b, qk_base + M::K + (col >> 6) * kTileBytes, col & 63, k0, lane);
          mma16816<T>(dQ[n0 / 8], fa, b[0], b[1]), mma16816<T>(dQ[n0 / 8 + 1], fa, b[2], b[3]);
          mma16816<T>(dK[n0 / 8], fb, b[0], b[1]), mma16816<T>(dK[n0 / 8 + 1], fb, b[2], b[3]);
        }
      }
      if (k0 >= r0) {  // and with those behind
        load_at(fa, base + M::Y1, r0, k0, lane);
        load_at(fb, base + M::Y2, r0, k0, lane);
#pragma unroll
        for (int n0 = 0; n0 < NB * 8; n0 += 16) {
          const int col = k_cols + n0;
          load_bt(b, qk_base + M::Q + (col >> 6) * kTileBytes, col & 63, k0, lane);
          mma16816<T>(y[n0 / 8], fa, b[0], b[1]), mma16816<T>(y[n0 / 8 + 1], fa, b[2], b[3]);
          load_bt(b, qk_base + M::K + (col >> 6) * kTileBytes, col & 63, k0, lane);
          mma16816<T>(y[n0 / 8], fb, b[0], b[1]), mma16816<T>(y[n0 / 8 + 1], fb, b[2], b[3]);
        }
      }
    }
    __syncthreads();  // and the pair matrices
    {
      float sum[2] = {0.f, 0.f};
      float* wide = g.dqk ? g.dqk + ((tok + r0 + gi) * a.heads + h) * a.kd : nullptr;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int col = k_cols + nb * 8 + gj;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 k = pair_at(M::K, e, nb);
          sum[e] += y[nb][2 * e] * k.x + y[nb][2 * e + 1] * k.y;
          const float k0 = fmaf(bt[e], y[nb][2 * e], dK[nb][2 * e]), k1 = fmaf(bt[e], y[nb][2 * e + 1], dK[nb][2 * e + 1]);
          if (wide) {
            if (r0 + gi + e * 8 < n && col < a.kd) {
              float* to = wide + (int64_t)e * 8 * a.heads * a.kd + col;
              *reinterpret_cast<float2*>(to) = make_float2(dQ[nb][2 * e], dQ[nb][2 * e + 1]);
              *reinterpret_cast<float2*>(to + g.tokens * a.heads * a.kd) = make_float2(k0, k1);
            }
          } else {  // over the pair matrices, to leave in whole pieces
            const int at = (col >> 6) * kTileBytes + swz(r0 + gi + e * 8, (col & 63) >> 3) + gj * 2;
            *reinterpret_cast<uint32_t*>(sm + M::Y1 + at) = pack2<T>(dQ[nb][2 * e], dQ[nb][2 * e + 1]);
            *reinterpret_cast<uint32_t*>(sm + M::A1 + at) = pack2<T>(k0, k1);
          }
        }
      }
      row_sums(sum, db);
    }
    __syncthreads();
    if (!g.dqk)
#pragma unroll
      for (int i = tid; i < C * (KD / 8); i += kGradThreads) {
        const int r = i / (KD / 8), u = i % (KD / 8), at = (u >> 3) * kTileBytes + swz(r, u & 7);
        if (r >= n || u * 8 >= a.kd) continue;
        const int64_t to = ((tok + r) * a.heads + h) * a.kd + u * 8;
        *reinterpret_cast<uint4*>(dq + to) = *reinterpret_cast<const uint4*>(sm + M::Y1 + at);
        *reinterpret_cast<uint4*>(dk + to) = *reinterpret_cast<const uint4*>(sm + M::A1 + at);
      }
    if (warp == kSums) {
      float all = 0.f;
      for (int i = 0; i < kGradThreads / 32; ++i) all += part[i];
      float x[2], z[2];  // of tokens 2 lane, 2 lane + 1: into them, out of them
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        x[e] = z[e] = 0.f;
        for (int b = 0; b < 4; ++b) x[e] += into[b * C + i] + rows[b * C + i] - (b * 16 + 15 > i ? cols[b * C + i] : 0.f), z[e] += outof[b * C + i];
      }
      float behind = x[0] + x[1], before = z[0] + z[1];  // inclusive sums from the end, and from the start
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const float u = __shfl_down_sync(0xffffffffu, behind, off), v = __shfl_up_sync(0xffffffffu, before, off);
        if (lane + off < 32) behind += u;
        if (lane >= off) before += v;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        if (i < n) {
          g.dg[(tok + i) * a.heads + h] = all + (e ? behind - x[0] : behind) + (e ? before - z[1] : before - z[0] - z[1]);
          g.dbeta[(tok + i) * a.heads + h] = db[i] + db[C + i] + db[2 * C + i] + db[3 * C + i];
        }
      }
    }
    now = next, --ahead;  // all of this chunk's slices have been asked for
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
// The driver's call below wants a context, which a thread that has launched nothing yet (autograd's, on its first call) does not have.
void bind_context() {
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaSetDevice(dev);
}
// (batch, len, heads, inner) at strides, as rank 4 (inner, head, token, batch); boxes of 64 columns of one head x 64 tokens
int encode_map(CUtensorMap* m, const void* base, int inner, int heads, int len, int batch, int64_t sh, int64_t st, int64_t sb, int dtype) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(SSM_ERR_DEVICE, "gated_delta: cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)heads, (cuuint64_t)len, (cuuint64_t)batch};
  // an extent of one may have any stride
  const cuuint64_t strides[3] = {(cuuint64_t)(heads > 1 ? sh : inner) * 2, (cuuint64_t)(len > 1 ? st : inner) * 2, (cuuint64_t)(batch > 1 ? sb : inner) * 2};
  const cuuint32_t box[4] = {64, 1, C, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult rc = fn(m, dtype == SSM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(SSM_ERR_DEVICE, "gated_delta: cuTensorMapEncodeTiled rejected the tensor");
  return SSM_OK;
}
bool lies(const void* p, int heads, int len, int batch, int64_t sh, int64_t st, int64_t sb) {
  auto ok = [](int n, int64_t stride) { return n <= 1 || (stride > 0 && stride % 8 == 0 && stride < ((int64_t)1 << 38)); };
  return aligned_to(p, 16) && ok(heads, sh) && ok(len, st) && ok(batch, sb);
}

template <typename T, int KD, bool TRAIN>
int launch_pairs(const Args& a, const Chunks& c, const PairMaps& maps, int64_t chunks, cudaStream_t st) {
  const int smem = PairSmem<KD>::ALLOC;
  if (const cudaError_t e = cudaFuncSetAttribute(pairs_kernel<T, KD, TRAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return set_error("pairs_kernel: %s", cudaGetErrorString(e)), (int)e;
  pairs_kernel<T, KD, TRAIN><<<dim3((unsigned)chunks, a.heads), kPairThreads, smem, st>>>(a, c, maps);
  return launch_status("pairs_kernel");
}
template <typename T, int KD, bool BACK>
int launch_chunks(const ChunkWalk& w, const WalkMaps& maps, cudaStream_t st) {
  const int smem = WalkSmem<KD, BACK>::ALLOC;
  if (const cudaError_t e = cudaFuncSetAttribute(chunks_kernel<T, KD, BACK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return set_error("chunks_kernel: %s", cudaGetErrorString(e)), (int)e;
  chunks_kernel<T, KD, BACK><<<dim3((w.a.vd + 127) / 128, w.a.heads, w.a.seqs + (w.a.where.table ? 1 : 0)), kWalkThreads, smem, st>>>(w, maps);
  return launch_status("chunks_kernel");
}

int64_t chunks_of(const ssm_gated_delta_args& a) { return chunk_bound(a.batch, a.len, a.num_seqs, C); }
int width(int kd) { return kd <= 64 ? 64 : 128; }

// what a call leaves for its backward pass, in this order; without one the vectors and Y alone
struct Layout {
  int64_t vec, y, wb, rest, states, total;
};
int64_t up(int64_t n) { return (n + 255) / 256 * 256; }
Layout layout_of(int64_t chunks, int heads, int kd, int vd, bool train) {
  Layout l{};
  const int64_t n = chunks * heads;
  l.y = up(n * 4 * C * 4);
  l.wb = l.y + up(n * kTileBytes);
  l.rest = l.wb + (train ? up(n * (width(kd) / 64) * kTileBytes) : 0);
  l.states = l.rest + (train ? up(n * C * vd * 2) : 0);
  l.total = l.states + (train ? up(n * (int64_t)width(kd) * vd * 2) : 0);
  return l;
}
int64_t fwd_bytes(int64_t chunks, int heads, int kd) { return up(chunks * heads * (1 + 2 * (width(kd) / 64)) * kTileBytes); }

}  // namespace

}  // namespace gd
}  // namespace ssmb

using namespace ssmb;

extern "C" int ssm_gated_delta_chunked_supported(const ssm_gated_delta_args* a) {
  return a && (a->io_dtype == SSM_BF16 || a->io_dtype == SSM_F16) && a->kdim >= 8 && a->kdim <= 128 && a->kdim % 8 == 0 && a->vdim >= 8 && a->vdim % 8 == 0 && a->len >= 1 &&
         a->key_heads >= 1 && a->heads >= 1 && gd::lies(a->q, a->key_heads, a->len, a->batch, a->q_sh, a->q_st, a->q_sb) &&
         gd::lies(a->k, a->key_heads, a->len, a->batch, a->k_sh, a->k_st, a->k_sb) && gd::lies(a->v, a->heads, a->len, a->batch, a->v_sh, a->v_st, a->v_sb) &&
         aligned_to(a->o, 16) && aligned_to(a->initial_state, 16);
}
extern "C" int64_t ssm_gated_delta_chunked_scratch_bytes(int32_t batch, int32_t len, int32_t num_seqs, int32_t heads, int32_t kdim) {
  return gd::fwd_bytes(gd::chunk_bound(batch, len, num_seqs, gd::C), heads, kdim);
}
extern "C" int64_t ssm_gated_delta_chunked_kept_bytes(int32_t batch, int32_t len, int32_t num_seqs, int32_t heads, int32_t kdim, int32_t vdim, int32_t train) {
  return gd::layout_of(gd::chunk_bound(batch, len, num_seqs, gd::C), heads, kdim, vdim, train != 0).total;
}

extern "C" int ssm_gated_delta_chunked_fwd(const ssm_gated_delta_args* args, void* scratch, void* kept, int32_t train, int32_t* status, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "gated_delta: NULL arguments");
  const ssm_gated_delta_args& f = *args;
  gd::ChunkWalk w{};
  if (const int rc = gd::check(f, w.a)) return rc;
  SSM_REQUIRE(ssm_gated_delta_chunked_supported(args), SSM_ERR_UNSUPPORTED, "gated_delta: these operands do not go to the tensor cores");
  if (w.a.seqs == 0) return SSM_OK;
  SSM_REQUIRE(f.o && scratch && kept, SSM_ERR_NULL, "gated_delta: NULL output or scratch");
  SSM_REQUIRE(aligned_to({scratch, kept}, 256) && aligned_to(status, 4), SSM_ERR_ALIGN, "gated_delta: misaligned scratch");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  w.a.where.per = (f.len + gd::C - 1) / gd::C;
  const int64_t chunks = gd::chunks_of(f);
  SSM_REQUIRE(chunks * f.heads < 0x7f000000, SSM_ERR_TOO_LARGE, "gated_delta: too many chunks");
  const gd::Layout l = gd::layout_of(chunks, f.heads, f.kdim, f.vdim, train != 0);
  unsigned char* base = reinterpret_cast<unsigned char*>(kept);
  unsigned char* wz = reinterpret_cast<unsigned char*>(scratch);
  w.in = {wz + chunks * f.heads * (2 * (gd::width(f.kdim) / 64)) * gd::kTileBytes, wz, base + l.y, train ? base + l.wb : nullptr, reinterpret_cast<float*>(base + l.vec), status};
  w.initial = f.initial_state, w.o = f.o, w.last = f.final_state, w.last_dtype = f.final_dtype;
  if (train) w.rest = base + l.rest, w.states = base + l.states;
  gd::bind_context();
  gd::WalkMaps maps;
  if (const int rc = gd::encode_map(&maps.q, f.q, f.kdim, f.key_heads, f.len, f.batch, f.q_sh, f.q_st, f.q_sb, f.io_dtype)) return rc;
  if (const int rc = gd::encode_map(&maps.k, f.k, f.kdim, f.key_heads, f.len, f.batch, f.k_sh, f.k_st, f.k_sb, f.io_dtype)) return rc;
  if (const int rc = gd::encode_map(&maps.v, f.v, f.vdim, f.heads, f.len, f.batch, f.v_sh, f.v_st, f.v_sb, f.io_dtype)) return rc;
  const int64_t row = (int64_t)f.heads * f.vdim;
  if (const int rc = gd::encode_map(&maps.o, f.o, f.vdim, f.heads, f.len, f.batch, f.vdim, row, row * f.len, f.io_dtype)) return rc;
  const gd::PairMaps pm{maps.q, maps.k};
  if (const int rc = gd::make_table(f, gd::C, st)) return rc;
  auto go = [&](auto type, auto kd) {
    using T = decltype(type);
    constexpr int KD = decltype(kd)::value;
    const int rc = train ? gd::launch_pairs<T, KD, true>(w.a, w.in, pm, chunks, st) : gd::launch_pairs<T, KD, false>(w.a, w.in, pm, chunks, st);
    return rc ? rc : gd::launch_chunks<T, KD, false>(w, maps, st);
  };
  const bool wide = f.kdim > 64;
  if (f.io_dtype == SSM_BF16) return wide ? go(__nv_bfloat16(), std::integral_constant<int, 128>()) : go(__nv_bfloat16(), std::integral_constant<int, 64>());
  return wide ? go(__half(), std::integral_constant<int, 128>()) : go(__half(), std::integral_constant<int, 64>());
}

extern "C" int64_t ssm_gated_delta_chunked_bwd_scratch_bytes(int32_t batch, int32_t len, int32_t num_seqs, int32_t heads, int32_t kdim, int32_t vdim) {
  return gd::up(gd::chunk_bound(batch, len, num_seqs, gd::C) * heads * (int64_t)gd::width(kdim) * vdim * 2);
}

extern "C" int ssm_gated_delta_chunked_bwd(const ssm_gated_delta_bwd_args* args, void* kept, void* scratch, int32_t* status, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "gated_delta: NULL arguments");
  const ssm_gated_delta_args& f = args->fwd;
  gd::ChunkWalk w{};
  if (const int rc = gd::check(f, w.a)) return rc;
  SSM_REQUIRE(ssm_gated_delta_chunked_supported(&f), SSM_ERR_UNSUPPORTED, "gated_delta: these operands do not go to the tensor cores");
  if (w.a.seqs == 0) return SSM_OK;
  SSM_REQUIRE(args->dout && args->dq && args->dk && args->dv && args->dg && args->dbeta && kept && scratch, SSM_ERR_NULL, "gated_delta backward: NULL pointer");
  SSM_REQUIRE(w.a.group == 1 || args->dqk, SSM_ERR_NULL, "gated_delta backward: shared keys need the dqk scratch");
  SSM_REQUIRE(aligned_to(args->dout, 16) && aligned_to(args->dv, 16) && aligned_to(args->dq, 16) && aligned_to(args->dk, 16) && aligned_to(args->dfinal, 16) && aligned_to(args->dqk, 16) &&
                  aligned_to(kept, 256) && aligned_to(scratch, 256),
              SSM_ERR_ALIGN, "gated_delta backward: misaligned pointer");
  if (const int rc = gd::check_gradients(*args)) return rc;
  SSM_REQUIRE(aligned_to(status, 4), SSM_ERR_ALIGN, "gated_delta backward: misaligned pointer");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  w.a.where.per = (f.len + gd::C - 1) / gd::C;
  const int64_t chunks = gd::chunks_of(f);
  SSM_REQUIRE(chunks * f.heads < 0x7f000000, SSM_ERR_TOO_LARGE, "gated_delta: too many chunks");
  const gd::Layout l = gd::layout_of(chunks, f.heads, f.kdim, f.vdim, true);
  unsigned char* base = reinterpret_cast<unsigned char*>(kept);
  w.in = {nullptr, nullptr, base + l.y, base + l.wb, reinterpret_cast<float*>(base + l.vec), status};
  w.initial = args->dfinal, w.o = args->dv, w.last = args->dinitial, w.last_dtype = SSM_F32, w.states = scratch;
  const int64_t row = (int64_t)f.heads * f.vdim;
  gd::bind_context();
  gd::WalkMaps maps;
  if (const int rc = gd::encode_map(&maps.q, f.q, f.kdim, f.key_heads, f.len, f.batch, f.q_sh, f.q_st, f.q_sb, f.io_dtype)) return rc;
  if (const int rc = gd::encode_map(&maps.k, f.k, f.kdim, f.key_heads, f.len, f.batch, f.k_sh, f.k_st, f.k_sb, f.io_dtype)) return rc;
  if (const int rc = gd::encode_map(&maps.v, args->dout, f.vdim, f.heads, f.len, f.batch, f.vdim, row, row * f.len, f.io_dtype)) return rc;
  if (const int rc = gd::encode_map(&maps.o, args->dv, f.vdim, f.heads, f.len, f.batch, f.vdim, row, row * f.len, f.io_dtype)) return rc;
  const gd::GradMaps gm{maps.q, maps.k, maps.v, maps.o};
  gd::ChunkGrads g{};
  g.a = w.a, g.rest = base + l.rest, g.states = base + l.states, g.dstates = scratch, g.dq = args->dq, g.dk = args->dk, g.dqk = w.a.group > 1 ? args->dqk : nullptr;
  g.dg = args->dg, g.dbeta = args->dbeta, g.tokens = (int64_t)f.batch * f.len, g.chunks = (int)chunks, g.status = status;
  auto go = [&](auto type, auto kd) {
    using T = decltype(type);
    constexpr int KD = decltype(kd)::value;
    if (const int rc = gd::launch_chunks<T, KD, true>(w, maps, st)) return rc;
    const int smem = gd::GradSmem<KD>::ALLOC;
    if (const cudaError_t e = cudaFuncSetAttribute(gd::grads_kernel<T, KD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return set_error("grads_kernel: %s", cudaGetErrorString(e)), (int)e;
    gd::grads_kernel<T, KD><<<(unsigned)std::min<int64_t>(chunks * f.heads, sm_count()), gd::kGradThreads, smem, st>>>(g, gm);
    if (const int rc = launch_status("grads_kernel")) return rc;
    return g.dqk ? gd::fold_heads(g.dqk, g.dq, g.dk, g.tokens, f.kdim, f.key_heads, w.a.group, f.io_dtype, st) : (int)SSM_OK;
  };
  const bool wide = f.kdim > 64;
  if (f.io_dtype == SSM_BF16) return wide ? go(__nv_bfloat16(), std::integral_constant<int, 128>()) : go(__nv_bfloat16(), std::integral_constant<int, 64>());
  return wide ? go(__half(), std::integral_constant<int, 128>()) : go(__half(), std::integral_constant<int, 64>());
}
