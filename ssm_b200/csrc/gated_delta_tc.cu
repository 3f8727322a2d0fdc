// Gated delta rule on the tensor cores: 16-bit operands, kdim and vdim multiples of 8, kdim <= 128.
//
// A sequence is cut into chunks of 64 tokens.  With a = e^g, gam_i = a_1 .. a_i, suf_i = a_{i+1} .. a_64, G_ij = a_{j+1} .. a_i, S0 the state
// before the chunk, the rows r_i = v_i - S'_i k_i solve a unit lower triangular system:
//   (I + A) r = V - diag(gam) K S0^T,  A_ij = beta_j G_ij k_i.k_j (j < i);   X = (I + A)^-1;   P_ij = scale beta_j G_ij q_i.k_j (j <= i)
//   r = X V - X diag(gam) K S0^T;   o = scale diag(gam) Q S0^T + P r;   S = gam_64 S0 + r^T diag(beta suf) K
// and the adjoint state, from the end, with D the gradient of the state behind the chunk and Y = P X:
//   w = dv = Y^T do + X^T diag(beta suf) K D^T;   D0 = gam_64 D + do^T diag(scale gam) Q - w^T diag(gam) K
//
//   pairs_kernel   one CTA per (chunk, key head): X, P (and Y) of its value heads.  The two 64 x 64 x kdim products are mma.sync; the inverse is
//                  fp32, blocks of 16 by substitution, then two rounds of block products.
//   chunks_kernel  one CTA per (sequence, value head, 128 rows of the state): the walk over the chunks, forward or back (BACK).
//
// The walk is bound by its chain: the state of a chunk depends on the one before through three products and the conversions between
// them.  So the state lies transposed, (vdim, kdim) with vdim on the 128 lanes of tensor memory, and every product of the chain takes its A
// operand from tensor memory, written there by the threads that hold the rows: no shared memory round trip, no transposes.
//   S (bf16, A) x K^T -> times -gam -> (A) x X^T, added to V^T X^T -> r -> times beta suf (A) x K -> added to the state in registers
// What does not depend on the state (V X^T; do Y; do Q) or is not on the chain (o) is issued beside it.
// Roundings to 16 bits: the operands above (S, gam K S, r and its weighted copy, X, P, Y, gam q), each half a step of the type; sums and the
// state between chunks are fp32.  For bf16 the outputs and gradients of random inputs are 0.3 % off in norm (0.17 of it their own rounding).
#include <algorithm>

#include "gated_delta.cuh"
#include "ssd_common.cuh"

namespace ssmb {
namespace gd {
namespace {

constexpr int C = 64;  // tokens of a chunk
constexpr int kTileBytes = C * 128;  // 64 rows of 128 bytes
constexpr float kReset = -150.f;     // base-2 logarithm of a decay that is zero in fp32

struct Chunks {  // what pairs_kernel leaves per (chunk, value head)
  unsigned char* pairs;  // X, P and (train) Y: tiles of 64 rows of 128 bytes in the 128-byte swizzle
  float* vec;            // gam, beta, beta suf, scale gam: 64 each
  int tiles;             // 2, or 3 with Y
};

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

// rows of an operand into a tile of KD columns; rows from n on and columns from kd on are zeros.  kd is a multiple of 8, rows lie on 16 bytes
template <typename T, int KD>
__device__ __forceinline__ void fill_tile(unsigned char* tile, const T* from, int64_t st, int n, int kd, int tid, int threads) {
  constexpr int U = KD / 8;
  for (int i = tid; i < C * U; i += threads) {
    const int row = i / U, unit = i % U;
    const uint4 v = row < n && unit * 8 < kd ? __ldg(reinterpret_cast<const uint4*>(from + (int64_t)row * st + unit * 8)) : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(tile + (unit >> 3) * kTileBytes + swz(row, unit & 7)) = v;
  }
}

// ---------------------------------------------------------------------------------------------
// pairs of tokens
// ---------------------------------------------------------------------------------------------
constexpr int kPairThreads = 128, kAS = 68, kTS = 36;  // row strides of the fp32 blocks, in floats

template <int KD>
struct PairSmem {
  static constexpr int QK = (KD / 64) * kTileBytes;
  static constexpr int TILES = 2 * QK > 3 * kTileBytes ? 2 * QK : 3 * kTileBytes;  // k and q rows; later X, P, Y on their way out
  static constexpr int TOTAL = TILES + (C * kAS + 32 * kTS + 5 * C) * 4;
  static constexpr int ALLOC = TOTAL + 128;
};

// cumulative base-2 logarithms of the decays of a chunk's tokens, by one warp; tokens from n on decay nothing
__device__ __forceinline__ void decay_logs(const Args& a, const Span& s, int n, int h, float* c, float* beta, int lane) {
  float x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = 2 * lane + i;
    x[i] = t < n && a.g.p ? fmaxf(load_dyn(a.g.p, s.b * a.g.sb + (s.t0 + t) * a.g.st + h * a.g.sh, a.g_dtype) * kLog2e, kReset) : 0.f;
    beta[t] = t < n ? beta_of(a, s.b, s.t0 + t, h) : 0.f;
  }
  float sum = x[0] + x[1];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const float o = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += o;
  }
  c[2 * lane + 1] = sum, c[2 * lane] = sum - x[1];
}

// acc[i][j] of `rows` x 64 with A rows r0.. of `ta` and B rows of `tb`, over KD columns: 8 blocks of 8 columns
template <typename T, int KD>
__device__ __forceinline__ void rows_product(float (&acc)[8][4], uint32_t ta, uint32_t tb, int r0, int lane) {
#pragma unroll
  for (int nb = 0; nb < 8; ++nb)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[nb][e] = 0.f;
#pragma unroll
  for (int k0 = 0; k0 < KD; k0 += 16) {
    uint32_t fa[4];
    load_a(fa, ta, r0, k0, lane);
#pragma unroll
    for (int n0 = 0; n0 < C; n0 += 16) {
      if (n0 > r0) continue;  // only pairs j <= i are looked at
      uint32_t fb[4];
      load_b(fb, tb, n0, k0, lane);
      mma16816<T>(acc[n0 / 8], fa, fb[0], fb[1]);
      mma16816<T>(acc[n0 / 8 + 1], fa, fb[2], fb[3]);
    }
  }
}

template <typename T, int KD, bool TRAIN>
__global__ void __launch_bounds__(kPairThreads) pairs_kernel(const Args a, const Chunks out) {
  using M = PairSmem<KD>;
  extern __shared__ unsigned char smdyn[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smdyn) + 127) & ~(uintptr_t)127);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const Span s = chunk_of(a.where, blockIdx.x, C);
  const int n = s.t1 - s.t0;
  if (n <= 0 || s.seq < 0) return;
  float* A = reinterpret_cast<float*>(sm + M::TILES);  // A, then X, in place
  float *tmp = A + C * kAS, *c = tmp + 32 * kTS, *beta = c + C;
  const int kh = blockIdx.y;
  fill_tile<T, KD>(sm, reinterpret_cast<const T*>(a.k.p) + s.b * a.k.sb + s.t0 * a.k.st + kh * a.k.sh, a.k.st, n, a.kd, tid, kPairThreads);
  fill_tile<T, KD>(sm + M::QK, reinterpret_cast<const T*>(a.q.p) + s.b * a.q.sb + s.t0 * a.q.st + kh * a.q.sh, a.q.st, n, a.kd, tid, kPairThreads);
  __syncthreads();
  const int r0 = warp * 16;
  float kk[8][4], qk[8][4];
  rows_product<T, KD>(kk, tc::smem_u32(sm), tc::smem_u32(sm), r0, lane);
  rows_product<T, KD>(qk, tc::smem_u32(sm + M::QK), tc::smem_u32(sm), r0, lane);
  unsigned char *tX = sm, *tP = sm + kTileBytes, *tY = sm + 2 * kTileBytes;
  for (int hh = 0; hh < a.group; ++hh) {
    const int h = kh * a.group + hh;
    __syncthreads();  // the rows of k and q, or the tiles of the head before, have been read
    if (warp == 0) decay_logs(a, s, n, h, c, beta, lane);
    __syncthreads();
    uint32_t pa[TRAIN ? 8 : 1][2], pl[TRAIN ? 8 : 1][2];  // P as an A operand, and what its rounding leaves
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      const int j = nb * 8 + (lane & 3) * 2;
      float x[4], p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = r0 + (lane >> 2) + (e >> 1) * 8, jj = j + (e & 1);
        const float G = jj <= i ? ex2_approx(c[i] - c[jj]) * beta[jj] : 0.f;
        x[e] = jj < i ? G * kk[nb][e] : 0.f;
        p[e] = jj <= i ? G * qk[nb][e] * a.scale : 0.f;
      }
      const int i = r0 + (lane >> 2);
      *reinterpret_cast<float2*>(&A[i * kAS + j]) = make_float2(x[0], x[1]);
      *reinterpret_cast<float2*>(&A[(i + 8) * kAS + j]) = make_float2(x[2], x[3]);
      const uint32_t w0 = pack2<T>(p[0], p[1]), w1 = pack2<T>(p[2], p[3]);
      *reinterpret_cast<uint32_t*>(tP + swz(i, nb) + (lane & 3) * 4) = w0;
      *reinterpret_cast<uint32_t*>(tP + swz(i + 8, nb) + (lane & 3) * 4) = w1;
      if constexpr (TRAIN) {
        const float2 u0 = unpack2<T>(w0), u1 = unpack2<T>(w1);
        pa[nb][0] = w0, pa[nb][1] = w1, pl[nb][0] = pack2<T>(p[0] - u0.x, p[1] - u0.y), pl[nb][1] = pack2<T>(p[2] - u1.x, p[3] - u1.y);
      }
    }
    __syncthreads();
    {  // the diagonal blocks, one a warp, a column a lane (both halves of the warp the same ones)
      const float* D = A + r0 * kAS + r0;
      float x[16];
      const int col = lane & 15;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = i == col ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) v = fmaf(-D[i * kAS + j], x[j], v);
        x[i] = v;
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((i & 1) == lane >> 4) A[(r0 + i) * kAS + r0 + col] = x[i];
    }
    __syncthreads();
    {  // pairs of blocks: X10 = -X11 (A10 X00); a thread has a row and four columns of one of the two
      const int b = tid >> 6, row = (tid & 63) >> 2, c4 = (tid & 3) * 4;
      const float* A10 = A + (b * 32 + 16) * kAS + b * 32;
      const float* X00 = A + (b * 32) * kAS + b * 32;
      const float* X11 = A + (b * 32 + 16) * kAS + b * 32 + 16;
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float m = A10[row * kAS + k];
        const float4 y = *reinterpret_cast<const float4*>(&X00[k * kAS + c4]);
        t.x = fmaf(m, y.x, t.x), t.y = fmaf(m, y.y, t.y), t.z = fmaf(m, y.z, t.z), t.w = fmaf(m, y.w, t.w);
      }
      *reinterpret_cast<float4*>(&tmp[(b * 16 + row) * kTS + c4]) = t;
      __syncthreads();
      t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float m = -X11[row * kAS + k];
        const float4 y = *reinterpret_cast<const float4*>(&tmp[(b * 16 + k) * kTS + c4]);
        t.x = fmaf(m, y.x, t.x), t.y = fmaf(m, y.y, t.y), t.z = fmaf(m, y.z, t.z), t.w = fmaf(m, y.w, t.w);
      }
      *reinterpret_cast<float4*>(&A[(b * 32 + 16 + row) * kAS + b * 32 + c4]) = t;
    }
    __syncthreads();
    {  // the same for the halves: two rows and four columns a thread
      const int row = (tid >> 3) * 2, c4 = (tid & 7) * 4;
      const float* A10 = A + 32 * kAS;
      float4 t[2];
      auto product = [&](const float* left, int ls, const float* right, int rs, float sign) {
        t[0] = t[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int k = 0; k < 32; ++k) {
          const float m0 = sign * left[row * ls + k], m1 = sign * left[(row + 1) * ls + k];
          const float4 y = *reinterpret_cast<const float4*>(&right[k * rs + c4]);
          t[0].x = fmaf(m0, y.x, t[0].x), t[0].y = fmaf(m0, y.y, t[0].y), t[0].z = fmaf(m0, y.z, t[0].z), t[0].w = fmaf(m0, y.w, t[0].w);
          t[1].x = fmaf(m1, y.x, t[1].x), t[1].y = fmaf(m1, y.y, t[1].y), t[1].z = fmaf(m1, y.z, t[1].z), t[1].w = fmaf(m1, y.w, t[1].w);
        }
      };
      product(A10, kAS, A, kAS, 1.f);
      *reinterpret_cast<float4*>(&tmp[row * kTS + c4]) = t[0];
      *reinterpret_cast<float4*>(&tmp[(row + 1) * kTS + c4]) = t[1];
      __syncthreads();
      product(A + 32 * kAS + 32, kAS, tmp, kTS, -1.f);
      __syncthreads();
      *reinterpret_cast<float4*>(&A[(32 + row) * kAS + c4]) = t[0];
      *reinterpret_cast<float4*>(&A[(33 + row) * kAS + c4]) = t[1];
    }
    __syncthreads();
    for (int i = tid; i < C * 8; i += kPairThreads) {  // X in 16 bits
      const int row = i >> 3, unit = i & 7;
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = unit * 8 + e * 2;
        const float2 v = *reinterpret_cast<const float2*>(&A[row * kAS + j]);
        w[e] = pack2<T>(j <= row ? v.x : 0.f, j + 1 <= row ? v.y : 0.f);
      }
      *reinterpret_cast<uint4*>(tX + swz(row, unit)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncthreads();
    if constexpr (TRAIN) {  // Y = P X, columns up to the rows' own; P in two pieces
      const uint32_t bX = tc::smem_u32(tX);
#pragma unroll
      for (int n0 = 0; n0 < C; n0 += 16) {
        float y[2][4] = {};
#pragma unroll
        for (int k0 = 0; k0 < C; k0 += 16) {
          if (k0 < n0 || k0 > r0) continue;
          uint32_t fb[4];
          load_bt(fb, bX, n0, k0, lane);
          const uint32_t hi[4] = {pa[k0 / 8][0], pa[k0 / 8][1], pa[k0 / 8 + 1][0], pa[k0 / 8 + 1][1]};
          const uint32_t lo[4] = {pl[k0 / 8][0], pl[k0 / 8][1], pl[k0 / 8 + 1][0], pl[k0 / 8 + 1][1]};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma16816<T>(y[e], hi, fb[2 * e], fb[2 * e + 1]);
            mma16816<T>(y[e], lo, fb[2 * e], fb[2 * e + 1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = r0 + (lane >> 2);
          *reinterpret_cast<uint32_t*>(tY + swz(i, n0 / 8 + e) + (lane & 3) * 4) = pack2<T>(y[e][0], y[e][1]);
          *reinterpret_cast<uint32_t*>(tY + swz(i + 8, n0 / 8 + e) + (lane & 3) * 4) = pack2<T>(y[e][2], y[e][3]);
        }
      }
      __syncthreads();
    }
    const int64_t at = (int64_t)s.chunk * a.heads + h;
    uint4* to = reinterpret_cast<uint4*>(out.pairs + at * (out.tiles * kTileBytes));
    for (int i = tid; i < (TRAIN ? 3 : 2) * (kTileBytes / 16); i += kPairThreads) to[i] = reinterpret_cast<const uint4*>(sm)[i];
    if (tid < C) {
      float* v = out.vec + at * (4 * C);
      const float gam = ex2_approx(c[tid]);
      v[tid] = gam, v[C + tid] = beta[tid], v[2 * C + tid] = beta[tid] * ex2_approx(c[C - 1] - c[tid]), v[3 * C + tid] = gam * a.scale;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// the walk over the chunks
// ---------------------------------------------------------------------------------------------
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
  void* rest;    // 16-bit r for the backward pass, [token / 8][vdim][8] per (chunk, head); nullable
  void* states;  // 16-bit state before every chunk (BACK: adjoint state behind it), [kdim / 8][vdim][8]; nullable
  int32_t* status;
};

constexpr int kCompute = 256, kWalkThreads = kCompute + 128;  // eight warps of rows; one each for copies, products, stores (and an idle one)
template <int KD>
struct WalkSmem {
  static constexpr int K_BYTES = (KD / 64) * kTileBytes;
  static constexpr int V_BYTES = 2 * kTileBytes;
  static constexpr int VEC_BYTES = 4 * C * 4;
  static constexpr int K = 0, Q = K_BYTES, V = Q + K_BYTES, X = V + V_BYTES, P = X + kTileBytes, VEC = P + kTileBytes;  // BACK: Y in P's place
  static constexpr int STAGE = VEC + VEC_BYTES;
  static constexpr int STAGES = 3;
  static constexpr int OUT = 2 * kTileBytes;
  static constexpr int ALLOC = STAGES * STAGE + OUT + 1024;
  static constexpr uint32_t BYTES = 2 * K_BYTES + V_BYTES + 2 * kTileBytes + VEC_BYTES;
};

// tensor memory, in columns: the state as an operand, the scaled product (then r), the weighted r; accumulators
template <int KD>
struct Cols {
  static constexpr int S = 0, A2 = 64, U = 96, KS = 128, R = 192, O = 256, DS = 384;  // O: two of 64
};

enum Bar { kFull = 0, kFree = 3, kPrep = 6, kState = 7, kKS = 8, kA2 = 9, kR = 10, kU = 11, kDS = 12, kO = 13, kOut = 14, kOutFree = 15, kEnd = 16, kBars = 17 };

template <typename T, int KD, bool BACK>
__global__ void __launch_bounds__(kWalkThreads, 1) chunks_kernel(const ChunkWalk w, const __grid_constant__ WalkMaps maps) {
  using M = WalkSmem<KD>;
  using TC = Cols<KD>;
  extern __shared__ unsigned char smdyn[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smdyn) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t mbar[kBars];
  __shared__ uint32_t tmem_slot;
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
  auto wait = [&](int i, int n) { return (bool)__all_sync(0xffffffffu, tc::mbar_test(bar(i), n & 1) || tc::mbar_wait(bar(i), n & 1)); };  // the n-th completion
  if (warp == 0) tc::tmem_alloc(tc::smem_u32(&tmem_slot), 512);
  if (tid == 0) {
    for (int i = 0; i < kBars; ++i) {
      const bool all = i == kPrep || i == kState || i == kA2 || i == kU || i == kOut;
      tc::mbar_init(bar(i), i >= kFree && i < kFree + M::STAGES ? 1 + kCompute / 32 : all ? kCompute / 32 : 1);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  // position p in the walk -> chunk of the sequence
  auto chunk_at = [&](int p) { return BACK ? nchunks - 1 - p : p; };
  unsigned char* out = sm + M::STAGES * M::STAGE;
  bool ok = true;

  if (warp == kCompute / 32) {  // ---- copies
    int sent = 0;
    for (int p = 0; p < nchunks && ok; ++p) {
      const int st = p % M::STAGES;
      if (p >= M::STAGES) ok = wait(kFree + st, p / M::STAGES - 1);
      if (!ok) break;
      if (lane == 0) {
        const int c = chunk_at(p), t = s.t0 + c * C;
        unsigned char* d = sm + st * M::STAGE;
        const uint32_t full = bar(kFull + st);
        tc::mbar_expect_tx(full, M::BYTES);
        for (int b = 0; b < KD / 64; ++b) {
          tc::tma_load_4d(tc::smem_u32(d + M::K + b * kTileBytes), &maps.k, full, b * 64, kh, t, s.b);
          tc::tma_load_4d(tc::smem_u32(d + M::Q + b * kTileBytes), &maps.q, full, b * 64, kh, t, s.b);
        }
        for (int b = 0; b < 2; ++b) tc::tma_load_4d(tc::smem_u32(d + M::V + b * kTileBytes), &maps.v, full, v0 + b * 64, h, t, s.b);
        const int64_t at = (int64_t)(s.chunk + c) * a.heads + h;
        const unsigned char* pairs = w.in.pairs + at * (w.in.tiles * kTileBytes);
        tc::bulk_load(tc::smem_u32(d + M::X), pairs, kTileBytes, full);
        tc::bulk_load(tc::smem_u32(d + M::P), pairs + (BACK ? 2 : 1) * kTileBytes, kTileBytes, full);
        tc::bulk_load(tc::smem_u32(d + M::VEC), w.in.vec + at * (4 * C), M::VEC_BYTES, full);
      }
      __syncwarp();
      sent = p + 1;
    }
    for (int p = max(0, sent - M::STAGES); p < sent; ++p) ok = wait(kFull + p % M::STAGES, p / M::STAGES) && ok;  // nothing is under way when the block ends
  } else if (warp == kCompute / 32 + 1) {  // ---- products
    constexpr int fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr uint32_t id_row = tc::instr_desc(128, C, fmt, 0, BACK ? 1 : 0);       // rows (tensor memory) x X or, transposed, X^T
    constexpr uint32_t id_kt = tc::instr_desc(128, C, fmt, 0, 0);                   // state x K^T, Q^T; r x P^T
    constexpr uint32_t id_vx = tc::instr_desc(128, C, fmt, 1, BACK ? 1 : 0);        // V^T X^T; do^T Y
    constexpr uint32_t id_k = tc::instr_desc(128, KD, fmt, 0, 1);                   // weighted rows x K
    constexpr uint32_t id_doq = tc::instr_desc(128, KD, fmt, 1, 1);                 // do^T Q
    for (int p = 0; p < nchunks && ok; ++p) {
      const int st = p % M::STAGES;
      ok = wait(kFull + st, p / M::STAGES) && wait(kPrep, p);  // rows of another sequence cut, q scaled
      if (!ok) break;
      tc::fence_after_sync();
      const uint32_t base = tc::smem_u32(sm + st * M::STAGE);
      const uint64_t k_rows = tc::smem_desc_sw128(base + M::K, 16, 1024), q_rows = tc::smem_desc_sw128(base + M::Q, 16, 1024);
      const uint64_t k_cols = tc::smem_desc_sw128(base + M::K, kTileBytes, 1024), q_cols = tc::smem_desc_sw128(base + M::Q, kTileBytes, 1024);
      const uint64_t v_cols = tc::smem_desc_sw128(base + M::V, kTileBytes, 1024);
      const uint64_t x_rows = tc::smem_desc_sw128(base + M::X, 16, 1024), p_rows = tc::smem_desc_sw128(base + M::P, 16, 1024);
      const uint64_t x_cols = tc::smem_desc_sw128(base + M::X, kTileBytes, 1024), y_cols = tc::smem_desc_sw128(base + M::P, kTileBytes, 1024);
      auto along = [](int kk) { return (uint64_t)(((kk >> 2) * kTileBytes + (kk & 3) * 32) >> 4); };  // 16 columns further
      auto down = [](int kk) { return (uint64_t)(kk * (2048 >> 4)); };                                // 16 rows further
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < C / 16; ++kk)
          tc::mma_ss(tmem + TC::R, v_cols + down(kk), BACK ? y_cols + down(kk) : x_rows + along(kk), id_vx, kk > 0);
      }
      __syncwarp();
      ok = wait(kState, p);
      if (!ok) break;
      tc::fence_after_sync();
      const uint32_t dO = tmem + TC::O + (p & 1) * 64;
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < KD / 16; ++kk) tc::mma_ts(tmem + TC::KS, tmem + TC::S + kk * 8, k_rows + along(kk), id_kt, kk > 0);
        tc::commit(bar(kKS));
        if constexpr (BACK) {
#pragma unroll
          for (int kk = 0; kk < C / 16; ++kk) tc::mma_ss(tmem + TC::DS, v_cols + down(kk), q_cols + down(kk), id_doq, kk > 0);
        } else {
#pragma unroll
          for (int kk = 0; kk < KD / 16; ++kk) tc::mma_ts(dO, tmem + TC::S + kk * 8, q_rows + along(kk), id_kt, kk > 0);
        }
      }
      __syncwarp();
      ok = wait(kA2, p);
      if (!ok) break;
      tc::fence_after_sync();
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < C / 16; ++kk) tc::mma_ts(tmem + TC::R, tmem + TC::A2 + kk * 8, BACK ? x_cols + down(kk) : x_rows + along(kk), id_row, true);
        tc::commit(bar(kR));
      }
      __syncwarp();
      ok = wait(kU, p);
      if (!ok) break;
      tc::fence_after_sync();
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < C / 16; ++kk) tc::mma_ts(tmem + TC::DS, tmem + TC::U + kk * 8, k_cols + down(kk), id_k, BACK || kk > 0);
        tc::commit(bar(kDS));
        if constexpr (!BACK) {
#pragma unroll
          for (int kk = 0; kk < C / 16; ++kk) tc::mma_ts(dO, tmem + TC::A2 + kk * 8, p_rows + along(kk), id_kt, true);
          tc::commit(bar(kO));
        }
        tc::commit(bar(kFree + st));
      }
      __syncwarp();
    }
    if (tc::elect_one()) tc::commit(bar(kEnd));  // nothing is under way when the block ends, nor where a wait ran out
    __syncwarp();
    ok = wait(kEnd, 0) && ok;
  } else if (warp == kCompute / 32 + 2) {  // ---- stores of o (BACK: dv)
    for (int p = 0; p < nchunks && ok; ++p) {
      ok = wait(kOut, p);
      if (!ok) break;
      const int t = s.t0 + chunk_at(p) * C, n = min(C, s.t1 - t);
      if (!packed || n == C) {  // TMA cuts at the tensor's end
        if (lane == 0) {
          tc::tma_store_4d(&maps.o, tc::smem_u32(out), v0, h, t, s.b);
          if (v0 + 64 < a.vd) tc::tma_store_4d(&maps.o, tc::smem_u32(out + kTileBytes), v0 + 64, h, t, s.b);
          tc::bulk_commit();
          tc::bulk_wait_read();
        }
        __syncwarp();
      } else {  // what follows belongs to the next sequence
        T* o = reinterpret_cast<T*>(w.o);
        const int units = min(128, a.vd - v0) / 8;
        for (int i = lane; i < n * units; i += 32) {
          const int row = i / units, u = i % units;
          *reinterpret_cast<uint4*>(o + ((int64_t)(t + row) * a.heads + h) * a.vd + v0 + u * 8) =
              *reinterpret_cast<const uint4*>(out + (u >> 3) * kTileBytes + swz(row, u & 7));
        }
        __syncwarp();
      }
      if (lane == 0) tc::mbar_arrive(bar(kOutFree));
      __syncwarp();
    }
    if (lane == 0) tc::bulk_wait_all();
  } else if (warp < kCompute / 32) {  // ---- rows of the state: lane = row, the warps of a lane quarter have half of the columns each
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int half = warp >> 2, row = (warp & 3) * 32 + lane, v = v0 + row;
    const bool live = v < a.vd;
    constexpr int NS = KD / 2;  // columns of the state a thread holds
    float S[NS];
    const int64_t state_at = (((int64_t)s.seq * a.heads + h) * a.vd + v) * a.kd + half * NS;
#pragma unroll
    for (int e = 0; e < NS; e += 4) {
      const bool in = w.initial && live && half * NS + e < a.kd;  // kdim is a multiple of 8
      const float4 x = in ? __ldg(reinterpret_cast<const float4*>(w.initial + state_at + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[e] = x.x, S[e + 1] = x.y, S[e + 2] = x.z, S[e + 3] = x.w;
    }
    auto done = [&](int i) {  // this warp's part of a phase
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar(i));
    };
    // the state as an operand, and for a backward pass to follow
    auto publish = [&](int p) {
      uint4* keep = w.states && p < nchunks && live
                        ? reinterpret_cast<uint4*>(w.states) + (((int64_t)(s.chunk + chunk_at(p)) * a.heads + h) * (KD / 8) + half * (NS / 8)) * a.vd + v
                        : nullptr;
#pragma unroll
      for (int q = 0; q < NS / 32; ++q) {
        uint32_t x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = pack2<T>(S[q * 32 + 2 * e], S[q * 32 + 2 * e + 1]);
        tc::tmem_st16(tmem + lanes + TC::S + half * (NS / 2) + q * 16, x);
        if (keep)
#pragma unroll
          for (int u = 0; u < 4; ++u) keep[(int64_t)(q * 4 + u) * a.vd] = make_uint4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
      }
      tc::tmem_wait_st();
      done(kState);
    };
    // rows of another sequence cut from the products over tokens; q times scale gam
    auto prepare = [&](int p) {
      const int st = p % M::STAGES;
      if (!wait(kFull + st, p / M::STAGES)) return false;
      unsigned char* d = sm + st * M::STAGE;
      const float* sg = reinterpret_cast<const float*>(d + M::VEC) + 3 * C;
      const int n = min(C, s.t1 - (s.t0 + chunk_at(p) * C));
      constexpr int U = KD / 8;
      for (int i = tid; i < C * U; i += kCompute) {
        const int r = i / U, u = i % U;
        uint4* at = reinterpret_cast<uint4*>(d + M::Q + (u >> 3) * kTileBytes + swz(r, u & 7));
        const float m = sg[r];
        const uint4 x = *at;
        const uint32_t in[4] = {x.x, x.y, x.z, x.w};
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<T>(in[e]);
          y[e] = r < n ? pack2<T>(f.x * m, f.y * m) : 0u;
        }
        *at = make_uint4(y[0], y[1], y[2], y[3]);
      }
      if (packed && n < C) {
        for (int i = tid; i < (C - n) * U; i += kCompute) *reinterpret_cast<uint4*>(d + M::K + (i % U >> 3) * kTileBytes + swz(n + i / U, i % U & 7)) = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < (C - n) * 16; i += kCompute) *reinterpret_cast<uint4*>(d + M::V + (i % 16 >> 3) * kTileBytes + swz(n + i / 16, i % 16 & 7)) = make_uint4(0, 0, 0, 0);
      }
      tc::fence_async_smem();
      done(kPrep);
      return true;
    };
    // 32 values of this thread's row (tokens 32 half ..) into the tile of rows of tokens that leaves by TMA
    auto stage_out = [&](const float (&x)[32]) {
      unsigned char* at = out + (row >> 6) * kTileBytes + (row & 7) * 2;
#pragma unroll
      for (int e = 0; e < 32; ++e) *reinterpret_cast<T*>(at + swz(half * 32 + e, (row & 63) >> 3)) = from_f<T>(x[e]);
      tc::fence_async_smem();
      done(kOut);
    };
    if (nchunks > 0) ok = prepare(0);
    publish(0);
    for (int p = 0; p < nchunks && ok; ++p) {
      const int st = p % M::STAGES;
      const float* vec = reinterpret_cast<const float*>(sm + st * M::STAGE + M::VEC);
      const float* first = vec + (BACK ? 2 * C : 0) + half * 32;   // gam; BACK: beta suf
      const float* second = vec + (BACK ? 0 : 2 * C) + half * 32;  // beta suf; BACK: gam
      float x[32];
      if (!(ok = wait(kKS, p))) break;
      tc::fence_after_sync();
      tc::tmem_ld32(tmem + lanes + TC::KS + half * 32, x);
      {
        uint32_t y[16];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 m = *reinterpret_cast<const float4*>(first + 2 * e);
          if constexpr (BACK) y[e] = pack2<T>(x[2 * e] * m.x, x[2 * e + 1] * m.y), y[e + 1] = pack2<T>(x[2 * e + 2] * m.z, x[2 * e + 3] * m.w);
          else y[e] = pack2<T>(-x[2 * e] * m.x, -x[2 * e + 1] * m.y), y[e + 1] = pack2<T>(-x[2 * e + 2] * m.z, -x[2 * e + 3] * m.w);
        }
        tc::tmem_st16(tmem + lanes + TC::A2 + half * 16, y);
        tc::tmem_wait_st();
      }
      done(kA2);
      if (!(ok = wait(kR, p))) break;
      tc::fence_after_sync();
      tc::tmem_ld32(tmem + lanes + TC::R + half * 32, x);
      {
        uint32_t y[16], u[16];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 m = *reinterpret_cast<const float4*>(second + 2 * e);
          if constexpr (BACK) u[e] = pack2<T>(-x[2 * e] * m.x, -x[2 * e + 1] * m.y), u[e + 1] = pack2<T>(-x[2 * e + 2] * m.z, -x[2 * e + 3] * m.w);
          else u[e] = pack2<T>(x[2 * e] * m.x, x[2 * e + 1] * m.y), u[e + 1] = pack2<T>(x[2 * e + 2] * m.z, x[2 * e + 3] * m.w);
          if constexpr (!BACK) y[e] = pack2<T>(x[2 * e], x[2 * e + 1]), y[e + 1] = pack2<T>(x[2 * e + 2], x[2 * e + 3]);
        }
        tc::tmem_st16(tmem + lanes + TC::U + half * 16, u);
        if constexpr (!BACK) tc::tmem_st16(tmem + lanes + TC::A2 + half * 16, y);
        tc::tmem_wait_st();
        done(kU);
        if constexpr (!BACK)
          if (w.rest && live) {
            uint4* to = reinterpret_cast<uint4*>(w.rest) + (((int64_t)(s.chunk + chunk_at(p)) * a.heads + h) * (C / 8) + half * 4) * a.vd + v;
#pragma unroll
            for (int q = 0; q < 4; ++q) to[(int64_t)q * a.vd] = make_uint4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
          }
      }
      if constexpr (BACK) {
        if (p > 0 && !(ok = wait(kOutFree, p - 1))) break;
        stage_out(x);
      }
      const float whole = vec[C - 1];
      if (p + 1 < nchunks && !(ok = prepare(p + 1))) break;
      if (!(ok = wait(kDS, p))) break;
      tc::fence_after_sync();
#pragma unroll
      for (int q = 0; q < NS / 32; ++q) {
        tc::tmem_ld32(tmem + lanes + TC::DS + half * NS + q * 32, x);
#pragma unroll
        for (int e = 0; e < 32; ++e) S[q * 32 + e] = fmaf(whole, S[q * 32 + e], x[e]);
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar(kFree + st));
      publish(p + 1);
      if constexpr (!BACK) {
        if (!(ok = wait(kO, p))) break;
        tc::fence_after_sync();
        tc::tmem_ld32(tmem + lanes + TC::O + (p & 1) * 64 + half * 32, x);
        if (p > 0 && !(ok = wait(kOutFree, p - 1))) break;
        stage_out(x);
      }
    }
    if (ok && live && w.last) {
#pragma unroll
      for (int e = 0; e < NS; ++e)
        if (half * NS + e < a.kd) store_dyn(w.last, state_at + e, w.last_dtype, S[e]);
    }
  }
  if (!ok && lane == 0 && w.status) *(volatile int32_t*)w.status = BACK ? 5 : 4;
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem_slot, 512);
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
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
int launch_pairs(const Args& a, const Chunks& c, int64_t chunks, cudaStream_t st) {
  const int smem = PairSmem<KD>::ALLOC;
  if (const cudaError_t e = cudaFuncSetAttribute(pairs_kernel<T, KD, TRAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return set_error("pairs_kernel: %s", cudaGetErrorString(e)), (int)e;
  pairs_kernel<T, KD, TRAIN><<<dim3((unsigned)chunks, a.heads / a.group), kPairThreads, smem, st>>>(a, c);
  return launch_status("pairs_kernel");
}
template <typename T, int KD, bool BACK>
int launch_chunks(const ChunkWalk& w, const WalkMaps& maps, cudaStream_t st) {
  const int smem = WalkSmem<KD>::ALLOC;
  if (const cudaError_t e = cudaFuncSetAttribute(chunks_kernel<T, KD, BACK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return set_error("chunks_kernel: %s", cudaGetErrorString(e)), (int)e;
  chunks_kernel<T, KD, BACK><<<dim3((w.a.vd + 127) / 128, w.a.heads, w.a.seqs + (w.a.where.table ? 1 : 0)), kWalkThreads, smem, st>>>(w, maps);
  return launch_status("chunks_kernel");
}

int64_t chunks_of(const ssm_gated_delta_args& a) { return chunk_bound(a.batch, a.len, a.num_seqs, C); }
int width(int kd) { return kd <= 64 ? 64 : 128; }

// scratch of a call, in this order: tiles of pairs, vectors, and for a backward pass the rests and the states
struct Layout {
  int64_t pairs, vec, rest, states, total;
  int tiles;
};
Layout layout_of(int64_t chunks, int heads, int kd, int vd, bool train) {
  Layout l{};
  l.tiles = train ? 3 : 2;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  l.pairs = 0;
  l.vec = up(chunks * heads * l.tiles * kTileBytes);
  l.rest = l.vec + up(chunks * heads * 4 * C * 4);
  l.states = l.rest + (train ? up(chunks * heads * C * vd * 2) : 0);
  l.total = l.states + (train ? up(chunks * heads * (int64_t)width(kd) * vd * 2) : 0);
  return l;
}

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
extern "C" int64_t ssm_gated_delta_chunked_scratch_bytes(int32_t batch, int32_t len, int32_t num_seqs, int32_t heads, int32_t kdim, int32_t vdim, int32_t train) {
  return gd::layout_of(gd::chunk_bound(batch, len, num_seqs, gd::C), heads, kdim, vdim, train != 0).total;
}

extern "C" int ssm_gated_delta_chunked_fwd(const ssm_gated_delta_args* args, void* scratch, int32_t train, int32_t* status, ssm_stream_t stream) {
  SSM_REQUIRE(args, SSM_ERR_NULL, "gated_delta: NULL arguments");
  const ssm_gated_delta_args& f = *args;
  gd::ChunkWalk w{};
  if (const int rc = gd::check(f, w.a)) return rc;
  SSM_REQUIRE(ssm_gated_delta_chunked_supported(args), SSM_ERR_UNSUPPORTED, "gated_delta: these operands do not go to the tensor cores");
  if (w.a.seqs == 0) return SSM_OK;
  SSM_REQUIRE(f.o && scratch && aligned_to(scratch, 256), SSM_ERR_NULL, "gated_delta: NULL output or scratch");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  w.a.where.per = (f.len + gd::C - 1) / gd::C;
  const int64_t chunks = gd::chunks_of(f);
  SSM_REQUIRE(chunks < 0x7fffffff && f.key_heads <= 65535, SSM_ERR_TOO_LARGE, "gated_delta: too many chunks");
  const gd::Layout l = gd::layout_of(chunks, f.heads, f.kdim, f.vdim, train != 0);
  unsigned char* base = reinterpret_cast<unsigned char*>(scratch);
  w.in = {base + l.pairs, reinterpret_cast<float*>(base + l.vec), l.tiles};
  w.initial = f.initial_state, w.o = f.o, w.last = f.final_state, w.last_dtype = f.final_dtype, w.status = status;
  if (train) w.rest = base + l.rest, w.states = base + l.states;
  gd::WalkMaps maps;
  if (const int rc = gd::encode_map(&maps.q, f.q, f.kdim, f.key_heads, f.len, f.batch, f.q_sh, f.q_st, f.q_sb, f.io_dtype)) return rc;
  if (const int rc = gd::encode_map(&maps.k, f.k, f.kdim, f.key_heads, f.len, f.batch, f.k_sh, f.k_st, f.k_sb, f.io_dtype)) return rc;
  if (const int rc = gd::encode_map(&maps.v, f.v, f.vdim, f.heads, f.len, f.batch, f.v_sh, f.v_st, f.v_sb, f.io_dtype)) return rc;
  const int64_t row = (int64_t)f.heads * f.vdim;
  if (const int rc = gd::encode_map(&maps.o, f.o, f.vdim, f.heads, f.len, f.batch, f.vdim, row, row * f.len, f.io_dtype)) return rc;
  if (const int rc = gd::make_table(f, gd::C, st)) return rc;
  auto go = [&](auto type, auto kd) {
    using T = decltype(type);
    constexpr int KD = decltype(kd)::value;
    const int rc = train ? gd::launch_pairs<T, KD, true>(w.a, w.in, chunks, st) : gd::launch_pairs<T, KD, false>(w.a, w.in, chunks, st);
    return rc ? rc : gd::launch_chunks<T, KD, false>(w, maps, st);
  };
  const bool wide = f.kdim > 64;
  if (f.io_dtype == SSM_BF16) return wide ? go(__nv_bfloat16(), std::integral_constant<int, 128>()) : go(__nv_bfloat16(), std::integral_constant<int, 64>());
  return wide ? go(__half(), std::integral_constant<int, 128>()) : go(__half(), std::integral_constant<int, 64>());
}
