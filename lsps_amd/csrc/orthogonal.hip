// Orthogonalised updates: Newton-Schulz iteration on stacks of matrices and the whole Muon step over the matrices of a net.
//
//   X0 = G / (|G|_F + eps)      X <- a X + (b A + c A^2) X,  A = X X^T   (`steps` times, on the side where X is wide)
//   Muon: m <- mu m + g,  G = g + mu m (nesterov) or m,  p <- p (1 - lr wd) - lr rms sqrt(max(rows, cols)) X
//
// Work on the short side.  With A = X X^T (M x M, M <= N) n steps are X <- (a^n I + R) X, where S = b A + c A^2 of the current
// Gram matrix and, from step to step, R <- a R + a^n S + R S and A <- A P^2 with P = a I + S: products of M x M matrices only,
// every one of them symmetric (they are polynomials of one symmetric matrix), so only the tiles on and above the diagonal are
// computed.  Two products with the long side (A, and the last one) per restart instead of two per step: 3 M^2 N + O(M^3)
// operations instead of 15 M^2 N for five steps.  A is formed anew from X after at most ORTHO_CHAINS steps: an error d of A is
// one of |b| / a (a^2)^k d, relatively, in the directions of small singular values after k more steps, so that chains of three
// cost about what the plain iteration in f32 costs and longer ones more (ortho_chain has the measurements).
//
// Operands.  Every matrix lives in the workspace as three bf16 limbs, which hold an f32 value exactly: 24 bits with an exponent of
// their own, so that rows and columns far below the others (1e-9 and less) keep the relative accuracy they have in f32 arithmetic;
// they grow by `a` a step and are as large as the others in the end.  (Two f16 limbs under one scale per matrix need half the
// MFMAs, but are good for 22 bits down to 1e-5 of the norm only: rows of 1e-8 were off by 4 %.)  A product is six
// v_mfma_f32_32x32x16_bf16 with f32 accumulation (limbs 0 0, 0 1, 1 0, 1 1, 0 2, 2 0; the dropped ones are at most
// 2^-24 of it, half a step of f32): 1.3 x the rate of the f32 MFMAs.
// Layout of a matrix with R rows: [column / 32][R][limb][(column % 32) / 8][8], rows and columns padded with zeros to multiples of 64:
// a 32-deep chunk of a row is one line of 192 bytes and the rows of a chunk follow each other, so that a tile's chunk is one
// contiguous run.  LDS-DMA copies it in 16-byte units whose source addresses carry the bank swizzle.  X is kept one way round only:
// Q X reads it transposed from LDS (28 x 256 x 2304 with an earlier loop on two limbs: 407 us, 451 with X^T beside X).
//
// Times (MI355X): 28 x 256 x 2304 440 us (prologue 45, two Gram matrices 51 each, twelve 256 x 256 products 14.5 to 22, Q X 65 to 70 each),
// the generator's 38 matrices 553, 2048 x 9216 2375 and 2795 with the discriminator's other eight: 0.9 PFLOP/s of bf16 MFMAs, a large
// library product at 1.21.  The 256 x 256 products are latency: launch, first and last bytes.
// All matrices of a call go through one launch per product (a block finds its group of equal matrices in the kernel's arguments).
#include <limits.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include "c8util.h"
#include "common.h"

namespace lsps {

typedef __bf16 og_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 og_b4 __attribute__((ext_vector_type(4)));
typedef float og_f16v __attribute__((ext_vector_type(16)));
typedef float og_f2 __attribute__((ext_vector_type(2)));
typedef __bf16 og_b2 __attribute__((ext_vector_type(2)));
typedef float og_f4 __attribute__((ext_vector_type(4)));
typedef float og_f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short og_u4u __attribute__((ext_vector_type(4), aligned(2)));

#define OG_BYTES 6             // of an element: three limbs
#define OG_LINE (32 * OG_BYTES) // 32 columns of a row
#define OG_BAND 512            // columns of a band of tiles of a symmetric product
#define ORTHO_GROUPS 16        // shapes per pass (they travel in the kernels' arguments)
#define ORTHO_MATRICES 1024    // matrices with pointers of their own per pass
#define ORTHO_CHAINS 3         // longest chain: steps between two Gram matrices of the long side
#define ORTHO_NORM_BLOCK 8192  // elements per block of the norm pass
#define ORTHO_PTR_PART 96      // matrices per table launch (passed by value: nothing on the host has to outlive the call)
#define ORTHO_STEPS 64
enum { OB_A, OB_S, OB_T, OB_R0, OB_R1, OB_SMALL, OB_X0 = OB_SMALL, OB_X1, OB_NONE };
enum { OM_F32, OM_BF16, OM_MUON };
enum { OL_SYM, OL_RECT, OL_LAST };

struct OrthoPtr {
  const void *g;
  void *out;           // OM_MUON: the weights
  float *m;            // OM_MUON: the momentum
};

// `count` matrices of one shape, and what one launch does with them.  48 bytes: a lane fetches a group's
struct OrthoGroup {
  int first;                      // blocks in front of the group's
  int aux;                        // norm and split passes: partial sums of squares in front of the group's; a product: ranges of its reduction
  int type, jobs;                 // a product: OL_*, and how many of them; panels: jobs = 32-column chunks of one
  int rows, cols, count;
  int ptr;                        // first of the matrices' pointers in the table; < 0: they lie one behind the other
  unsigned x_off, s_off, p_off;   // workspace offsets in 256-byte units: long-side matrices, M x M matrices, partial products
  float step;                     // OM_MUON: lr rms sqrt(max(rows, cols))
};
struct OrthoGroups {
  OrthoGroup g[ORTHO_GROUPS];     // (first = INT_MAX behind the last one)
  OrthoPtr base;                  // the only group's matrices if they lie one behind the other
  const OrthoPtr *table;
};

struct OrthoPtrPart {
  OrthoPtr p[ORTHO_PTR_PART];
};

__host__ __device__ static inline int og_pad(int n) { return (n + 63) & ~63; }
__host__ __device__ static inline int og_short(const OrthoGroup &g) { return g.rows < g.cols ? g.rows : g.cols; }
__host__ __device__ static inline int og_long(const OrthoGroup &g) { return g.rows < g.cols ? g.cols : g.rows; }
__host__ __device__ static inline int og_norm_blocks(const OrthoGroup &g) {
  return (int)(((long)g.rows * g.cols + ORTHO_NORM_BLOCK - 1) / ORTHO_NORM_BLOCK);
}
__host__ __device__ static inline int og_split_blocks(const OrthoGroup &g) { return og_pad(g.rows) / 64 * (og_pad(g.cols) / 64); }
// tiles of T x T per matrix of a product
__host__ __device__ static inline int og_tiles(const OrthoGroup &g, int type, int T) {
  const int m = (og_pad(og_short(g)) + T - 1) / T, n = (og_pad(og_long(g)) + T - 1) / T;
  return type == OL_SYM ? m * (m + 1) / 2 : m * n;
}

__global__ void ortho_ptr_kernel(OrthoPtrPart part, OrthoPtr *t, int base, int n) {
  if ((int)threadIdx.x < n) t[base + threadIdx.x] = part.p[threadIdx.x];
}

template <typename T>
__device__ __forceinline__ T og_readlane(const T &v, int lane) {
  constexpr int W = sizeof(T) / 4;
  int w[W];
  __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = __builtin_amdgcn_readlane(w[i], lane);
  T r;
  __builtin_memcpy(&r, w, sizeof(T));
  return r;
}

// The group of block b (the last one whose first block is not behind it): lane i looks at group i, so that one trip to the
// arguments' memory brings them all (through a table and its index it was three, 1.2 us of every launch).
__device__ __forceinline__ OrthoGroup ortho_group_of(const OrthoGroups &gs, int b, int &index) {
  const int lane = threadIdx.x & 63;
  const OrthoGroup mine = gs.g[lane < ORTHO_GROUPS ? lane : 0];
  index = __builtin_amdgcn_readfirstlane(63 - __clzll(__ballot(lane < ORTHO_GROUPS && mine.first <= b)));
  return og_readlane(mine, index);
}

__device__ __forceinline__ OrthoPtr ortho_ptr(const OrthoGroups &gs, const OrthoGroup &g, int mat, int bytes) {
  if (g.ptr >= 0) return gs.table[g.ptr + mat];
  const long o = (long)g.rows * g.cols * mat * bytes;
  return OrthoPtr{(const char *)gs.base.g + o, (char *)gs.base.out + o, nullptr};
}

__device__ __forceinline__ char *ortho_buffer(char *ws, const OrthoGroup &g, int id, int mat) {
  const long M = og_pad(og_short(g)), N = og_pad(og_long(g));
  if (id < OB_SMALL) return ws + (size_t)g.s_off * 256 + ((long)id * g.count + mat) * M * M * OG_BYTES;
  return ws + (size_t)g.x_off * 256 + ((long)(id - OB_X0) * g.count + mat) * M * N * OG_BYTES;
}
// byte of element (row, col) of a matrix of R rows: its first limb (the others lie 64 and 128 bytes on)
__device__ __forceinline__ long og_at(long R, int row, int col) {
  return ((col >> 5) * R + row) * OG_LINE + ((col >> 3) & 3) * 16 + (col & 7) * 2;
}

template <typename T>
__device__ __forceinline__ void og_load4(const T *p, long left, float (&v)[4]) {
  if (left >= 4) {
    if constexpr (sizeof(T) == 4) {
      const og_f4u q = *reinterpret_cast<const og_f4u *>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = q[e];
    } else {
      const og_u4u q = *reinterpret_cast<const og_u4u *>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float((unsigned)q[e] << 16);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? (float)p[e] : 0.f;
  }
}

struct OrthoMomentum {
  float mu, gscale;
  int nesterov;
};

// sums of squares of G in 64 bits (squares of f32 values neither overflow nor vanish there), one partial sum per block; Muon:
// the momentum is updated on the way.  Memory bound: 4 (Muon: 12) bytes per element.
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoGroups gs, double *__restrict__ sums, OrthoMomentum mo) {
  __shared__ double red[4];
  int grp;
  const OrthoGroup g = ortho_group_of(gs, blockIdx.x, grp);
  const int rel = blockIdx.x - g.first, nb = og_norm_blocks(g), mat = rel / nb, tile = rel - mat * nb;
  const long size = (long)g.rows * g.cols, lo = (long)tile * ORTHO_NORM_BLOCK;
  const OrthoPtr ptr = ortho_ptr(gs, g, mat, sizeof(T));
  const T *src = (const T *)ptr.g;
  float *m = ptr.m;
  double s = 0.;
#pragma unroll 4
  for (int i = 0; i < ORTHO_NORM_BLOCK / 1024; ++i) {
    const long at4 = lo + i * 1024 + threadIdx.x * 4;
    if (at4 >= size) break;
    float v[4];
    og_load4<T>(src + at4, size - at4, v);
    if constexpr (MUON) {
      float o[4];
      og_load4<float>(m + at4, size - at4, o);
      og_f4u q;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] *= mo.gscale;
        o[e] = fmaf(mo.mu, o[e], v[e]);
        q[e] = o[e];
        v[e] = mo.nesterov ? fmaf(mo.mu, o[e], v[e]) : o[e];
      }
      if (size - at4 >= 4) *reinterpret_cast<og_f4u *>(m + at4) = q;
      else
        for (int e = 0; e < 4; ++e)
          if (e < size - at4) m[at4 + e] = o[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s += (double)v[e] * (double)v[e];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) sums[g.aux + rel] = red[0] + red[1] + red[2] + red[3];
}

// 4 values as three limbs each: what is left of one rounding to bf16 is exact, and so is the third limb of an f32 value
__device__ __forceinline__ void og_split(const float (&v)[4], og_b4 (&l)[3]) {
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    og_f2 r = {v[e], v[e + 1]};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const og_b2 b = __builtin_convertvector(r, og_b2);
      l[k][e] = b[0];
      l[k][e + 1] = b[1];
      r = og_f2{r[0] - (float)b[0], r[1] - (float)b[1]};
    }
  }
}
// the 4 values: sums of limbs, smallest first, are exact
__device__ __forceinline__ void og_value(const og_b4 (&l)[3], float (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = (float)l[0][k] + ((float)l[1][k] + (float)l[2][k]);
}

// In front of the first use of accumulators behind a join of paths: an MFMA's last registers arrive 12 wait states behind it, and the
// compiler counts them along one of the paths only (seen: 15 instructions on a path round a conditional load, 7 on the one without;
// the last product of every 16th value was lost).
__device__ __forceinline__ void og_settle(og_f16v &a, og_f16v &b) { asm volatile("s_nop 15" : "+v"(a), "+v"(b)); }

__device__ __forceinline__ og_b8 og_join(const og_b4 &a, const og_b4 &b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// v / norm as f32: norm = mantissa * 2^ex, v 2^-ex rounded by one factor, so that nothing overflows on the way for any norm
struct OgUnit {
  float f;
  int ex;
  __device__ __forceinline__ explicit OgUnit(double norm) { f = (float)(1. / frexp(norm, &ex)); }
  __device__ __forceinline__ float operator()(float v) const { return ldexpf(v, -ex) * f; }
};

// X0 as limbs, the short side in rows.  One 64 x 64 tile of G per block, through LDS (turned round there for a tall G).
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoGroups gs, char *__restrict__ ws, const double *__restrict__ sums,
                                                          OrthoMomentum mo, float eps) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  int grp;
  const OrthoGroup g = ortho_group_of(gs, blockIdx.x, grp);
  const int rel = blockIdx.x - g.first, per = og_split_blocks(g), mat = rel / per, tix = rel - mat * per;
  const int nb = og_norm_blocks(g);
  const double *part = sums + g.aux + (long)mat * nb;
  double s = 0.;
  for (int i = threadIdx.x; i < nb; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  const int tc = og_pad(g.cols) / 64;
  const int r0 = tix / tc * 64, c0 = (tix - tix / tc * tc) * 64;
  const OrthoPtr ptr = ortho_ptr(gs, g, mat, sizeof(T));
  const T *src = (const T *)ptr.g;
  const float *m = ptr.m;
  float v[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + (threadIdx.x >> 4) + k * 16, c = c0 + (threadIdx.x & 15) * 4;
    const long left = r < g.rows ? g.cols - c : 0, o = (long)r * g.cols + c;
    og_load4<T>(src + o, left, v[k]);
    if constexpr (MUON) {
      float mv[4];
      og_load4<float>(m + o, left, mv);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = mo.nesterov ? fmaf(mo.mu, mv[e], v[k][e] * mo.gscale) : mv[e];
    }
  }
  __syncthreads();
  const OgUnit unit(sqrt(red[0] + red[1] + red[2] + red[3]) + (double)eps);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[(threadIdx.x >> 4) + k * 16][(threadIdx.x & 15) * 4 + e] = unit(v[k][e]);
  __syncthreads();
  const bool tall = g.rows > g.cols;
  char *dst = ortho_buffer(ws, g, OB_X0, mat);
  const int M = og_pad(og_short(g)), i0 = tall ? c0 : r0, j0 = tall ? r0 : c0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int u = threadIdx.x + k * 256, i = u >> 3, j = (u & 7) * 8;
    og_b4 l[2][3];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      float x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = tall ? tile[j + e + c][i] : tile[i][j + e + c];
      og_split(x, l[e / 4]);
    }
    char *o = dst + og_at(M, i0 + i, j0 + j);
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<og_b8 *>(o + q * 64) = og_join(l[0][q], l[1][q]);
  }
}

__device__ __forceinline__ void og_result(void *out, long o, float v, int mode, float step, float decay) {
  if (mode == OM_F32) ((float *)out)[o] = v;
  else if (mode == OM_BF16) ((__bf16 *)out)[o] = (__bf16)v;               // the one rounding of the result
  else ((float *)out)[o] = fmaf(-step, v, ((float *)out)[o] * decay);
}

// a / b for 0 <= a < 2^23, b > 0: a tenth of the instructions of an integer division, all of them in a block's first microsecond
__device__ __forceinline__ int og_div(int a, int b) {
  int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
  q -= q * b > a;
  q += (q + 1) * b <= a;
  return __builtin_amdgcn_readfirstlane(q);
}

// the largest j with j (j + 1) / 2 <= t
__device__ __forceinline__ int og_triangle(int t) {
  int j = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while ((j + 1) * (j + 2) / 2 <= t) ++j;
  while (j * (j + 1) / 2 > t) --j;
  return j;
}

struct OgTrue {
  static constexpr bool value = true;
};
struct OgFalse {
  static constexpr bool value = false;
};
struct OrthoJob {                   // out = k0 (product) + k1 E1 + k2 E2 + diag I
  int l, r, e1, e2, out;
  float k0, k1, k2, diag;
};
struct OrthoLevel {
  OrthoGroups gs;
  OrthoJob job[ORTHO_GROUPS * 2];   // of group i: 2 i, 2 i + 1
  int joining;                      // second launch of a split product: the ranges it was split into
  int mode;                         // of the last level: OM_*
  float decay;                      // 1 - lr wd
};

// One product per block: a T x T tile.  WI x WJ waves, each (T / WI) x (T / WJ) in 32x32 MFMA tiles; the MFMA's row index is the tile's
// COLUMN, so a lane holds one row of the result and runs of 4 columns (8-byte stores per limb).  The product of the first limbs has an
// accumulator of its own: the small cross products, added to it, would cost it a rounding each (measured: that halves the error of
// the whole iteration).  LDS: S stages of a KC-deep chunk of both operands, S - 1 of them requested ahead by LDS-DMA (from inline asm:
// in front of a transposing read the compiler would wait for all requests); one barrier per chunk.
//   OL_SYM : L R^T, symmetric: tiles on and above the diagonal, the mirrored tile is stored from an LDS transpose
//   OL_RECT: L X, X of the next chain: the reduction runs down the rows of X, whose chunks are read transposed from LDS
//   OL_LAST: the same, the result in the caller's layout and type, or the weight update
// A product with few tiles and a long reduction is split into kz ranges of it: f32 partial tiles in the workspace, added in a
// fixed order by a second launch of this kernel.
// Registers: as many waves per SIMD as fit beside each other in LDS (the second argument of the launch bounds); the accumulators have to
// stay in VGPRs, and nothing may spill: one reload in the loop waits for every request under way.
template <int T, int KC, int S, int WI, int WJ>
__global__ __launch_bounds__(WI * WJ * 64, T == 64 && S == 2 ? 3 : 2) void ortho_product_kernel(char *__restrict__ ws, OrthoLevel lv) {
  constexpr int WAVES = WI * WJ, STAGE = T * KC * OG_BYTES, PIECES = STAGE / 1024 / WAVES, FI = T / WI / 32, FJ = T / WJ / 32, TP = OG_LINE + 16;
  static_assert(PIECES * WAVES * 1024 == STAGE, "whole requests of a wave");
  static_assert(S * 2 * STAGE >= WAVES * 32 * TP, "the exchange buffers of the epilogue lie in the stages");
  static_assert((S - 1) * 2 * PIECES < 64, "the range of s_waitcnt vmcnt");
  extern __shared__ __align__(1024) char smem[];
  const int lane = threadIdx.x & 63;
  const OrthoJob mine = lv.job[lane < 2 * ORTHO_GROUPS ? lane : 0];
  int grp;
  const OrthoGroup g = ortho_group_of(lv.gs, blockIdx.x, grp);
  const int type = g.type, kz = lv.joining ? 1 : g.aux;
  const int M = og_pad(og_short(g)), N = og_pad(og_long(g));
  const int per = og_tiles(g, type, T) * kz, total = per * g.count * g.jobs;
  // consecutive blocks go to the eight XCDs in turn: block x + 8 y takes unit x q + y, so that an XCD's blocks share operands in its L2
  const int rel = blockIdx.x - g.first, q8 = (total + 7) / 8, unit0 = (rel & 7) * q8 + (rel >> 3);
  if ((rel >> 3) >= q8 || unit0 >= total) return;
  const int second = unit0 >= per * g.count;
  const OrthoJob job = og_readlane(mine, __builtin_amdgcn_readfirstlane(grp * 2 + second));
  const int u1 = unit0 - second * per * g.count, mat = og_div(u1, per), u2 = u1 - mat * per, tile = og_div(u2, kz), z = u2 - tile * kz;
  int bi, bj;
  if (type == OL_SYM) {
    // bands of W column tiles, in each row by row down to its triangle on the diagonal: an XCD's tiles make a block of about W x W
    constexpr int W = OG_BAND / T;
    const int m = (M + T - 1) / T;
    int b = og_triangle(tile) & -W, t = tile - b * (b + 1) / 2;  // the band's first column (the tiles in front of it make a triangle too)
    const int w = m - b < W ? m - b : W;
    if (t < b * w) {
      bi = og_div(t, w);
      bj = b + t - bi * w;
    } else {
      t -= b * w;
      bj = og_triangle(t);
      bi = b + t - bj * (bj + 1) / 2;
      bj += b;
    }
  } else {
    const int tm = (M + T - 1) / T;                              // the row tiles of one column panel one after the other
    bj = og_div(tile, tm);
    bi = tile - bj * tm;
  }
  const int cols = type == OL_SYM ? M : N;                       // of the result; rows: M
  const int K = job.l >= OB_SMALL ? N : M;
  const int chunks = K / KC, c0 = og_div(chunks * z, kz), c1 = og_div(chunks * (z + 1), kz);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ, l31 = lane & 31, lh = lane >> 5;
  og_f16v acc[FI][FJ], acx[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = acx[i][j][e] = 0.f;
  float *part = reinterpret_cast<float *>(ws + (size_t)g.p_off * 256);   // [mat][tile][z][fi][fj][q][thread][4]
  const char *e1 = job.e1 == OB_NONE ? nullptr : ortho_buffer(ws, g, job.e1, mat);
  const char *e2 = job.e2 == OB_NONE ? nullptr : ortho_buffer(ws, g, job.e2, mat);
  // one fragment per wave: E1 and E2 are fetched behind the product's first requests
  constexpr bool EARLY = FI * FJ == 1;
  og_b4 el[EARLY ? 8 : 1][3];
  auto early = [&]() {
    if constexpr (EARLY) {
      const long at = og_at(M, (bi * WI + wi) * 32 + l31, (bj * WJ + wj) * 32 + lh * 4);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const char *e = q < 4 ? e1 : e2;
        if (e) {
#pragma unroll
          for (int k = 0; k < 3; ++k) el[q][k] = *reinterpret_cast<const og_b4 *>(e + at + (q & 3) * 16 + k * 64);
        }
      }
    }
  };
  if (!lv.joining) {
    // a piece = 64 units of 16 bytes = one DMA request of a wave; a line = 12 units, [limb][8 columns] of a row of the tile; for X in
    // OL_RECT / OL_LAST: [32 columns][row of the chunk].  The unit of columns q of line r lies at q ^ (r / 4): 16 lanes reading 16
    // consecutive lines, or four lines of the 64-bit transposing reads, touch all 64 banks once
    const bool turned = type != OL_SYM;
    const c8_i32x4 lrs = c8_rsrc_words(ortho_buffer(ws, g, job.l, mat), (unsigned)((long)M * K * OG_BYTES));
    const c8_i32x4 rrs = c8_rsrc_words(ortho_buffer(ws, g, job.r, mat), (unsigned)((long)M * (turned ? N : K) * OG_BYTES));
    unsigned lo[PIECES], ro[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int u = (wave + WAVES * p) * 64 + lane, line = u / 12, unit = ((u - line * 12) ^ ((line >> 2) & 3)) * 16;
      const int li = bi * T + line < M ? bi * T + line : M - 1;
      lo[p] = (unsigned)(li * OG_LINE + unit);
      if (!turned) {
        const int rj = bj * T + line < M ? bj * T + line : M - 1;
        ro[p] = (unsigned)(rj * OG_LINE + unit);
      } else {                                                            // T / 32 column chunks of KC rows each
        const int cc = line / KC, r = line % KC;
        const int c = bj * (T / 32) + cc < N / 32 ? bj * (T / 32) + cc : N / 32 - 1;
        ro[p] = (unsigned)((c * (long)M + r) * OG_LINE + unit);
      }
    }
    const unsigned lstep = (unsigned)M * OG_LINE, rstep = turned ? KC * OG_LINE : lstep, lds0 = c8_lds_addr(smem);
    auto stage = [&](int buf, int c) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        c8_dma16_asm(lrs, lds0 + buf * 2 * STAGE + (wave + WAVES * p) * 1024, lo[p], c * lstep);
        c8_dma16_asm(rrs, lds0 + buf * 2 * STAGE + STAGE + (wave + WAVES * p) * 1024, ro[p], c * rstep);
      }
    };
    // Fragments are read from LDS one half chunk ahead of their MFMAs, across the barrier too: the barrier of chunk c comes when its
    // last fragments are in registers, so its stage is free for chunk c + S, and chunk c + 1 has landed.  The chunks go round the
    // stages in a loop unrolled S times, so that a lane's LDS addresses are eight registers and constants, and the last chunk has code
    // of its own: where paths meet, the compiler would wait for every LDS read in flight.
    static_assert(KC == 32, "two halves per chunk, lines of one chunk");
    og_b8 lf[2][FI][3], rf[2][FJ][3];
    auto product = [&](auto turn) {
      // lines of 32 columns: halves differ in bits of the unit, limbs by 64 bytes; chunks of X: lane i of 16 points at 4 columns of row
      // i / 4 and receives 4 rows of column i
      const char *la[2], *ra[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int unit = h * 2 + lh, li = wi * FI * 32 + l31, rj = wj * FJ * 32 + l31;
        la[h] = smem + li * OG_LINE + ((unit ^ ((li >> 2) & 3)) * 16);
        if constexpr (!turn.value) {
          ra[h] = smem + STAGE + rj * OG_LINE + ((unit ^ ((rj >> 2) & 3)) * 16);
        } else {                                                 // [4 rows further]
          const int r = lh * 8 + ((lane & 15) >> 2) + h * 4, u = ((lane >> 4) & 1) * 2 + ((lane & 2) >> 1);
          ra[h] = smem + STAGE + (wj * FJ * KC + r) * OG_LINE + (lane & 1) * 8 + ((u ^ ((r >> 2) & 3)) * 16);
        }
      }
      auto load = [&](int h, int at) {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
#pragma unroll
          for (int f = 0; f < FJ; ++f)
            if constexpr (!turn.value)
              rf[h][f][q] = *reinterpret_cast<const og_b8 *>(ra[h] + at * 2 * STAGE + f * 32 * OG_LINE + q * 64);
            else
              rf[h][f][q] = c8_tr_frag((const unsigned char *)ra[0] + at * 2 * STAGE + (f * KC + h * 16) * OG_LINE + q * 64,
                                       (const unsigned char *)ra[1] + at * 2 * STAGE + (f * KC + h * 16) * OG_LINE + q * 64);
#pragma unroll
          for (int f = 0; f < FI; ++f) lf[h][f][q] = *reinterpret_cast<const og_b8 *>(la[h] + at * 2 * STAGE + f * 32 * OG_LINE + q * 64);
        }
      };
      // limbs (r, l) of the products, the smallest first; 1 2, 2 1 and 2 2 are at most 2^-24 of the product
      auto multiply = [&](int h) {
        auto add = [&](int r, int l, og_f16v (&to)[FI][FJ]) {
#pragma unroll
          for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) to[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rf[h][j][r], lf[h][i][l], to[i][j], 0, 0, 0);
        };
        add(0, 2, acx);
        add(2, 0, acx);
        add(1, 1, acx);
        add(0, 0, acc);
        add(0, 1, acx);
        add(1, 0, acx);
      };
      const int n = c1 - c0;
#pragma unroll
      for (int c = 0; c < S; ++c)
        if (c < n) stage(c, c0 + c);
      if (kz == 1) early();
      // requests are served in order: those of the S - 1 chunks behind the first may still be on their way
      if (n >= S) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * 2 * PIECES) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      load(0, 0);
      int c = 0, left = n - 1;                                   // chunks with one behind them
      auto step = [&](int at) {                                  // chunk c, in stage `at`
        load(1, at);
        __builtin_amdgcn_sched_barrier(0);
        multiply(0);
        __builtin_amdgcn_sched_barrier(0);
        // chunks c + 1 ... c + S - 1 are requested
        if (S == 2 || left < S - 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * 2 * PIECES) : "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);                      // lgkmcnt(0), in the compiler's sight
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (left >= S) stage(at, c0 + c + S);
        load(0, at + 1 == S ? 0 : at + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(1);
        ++c;
        --left;
      };
      while (left >= S)
#pragma unroll
        for (int at = 0; at < S; ++at) step(at);
      int at = 0;
      while (left > 0) step(at++);
      load(1, at);
      multiply(0);
      multiply(1);
#pragma unroll
      for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) og_settle(acc[i][j], acx[i][j]);
    };
    if (c0 < c1) {
      if (turned) product(OgTrue());
      else product(OgFalse());
    }
    if (kz > 1) {
      og_f4 *dst = reinterpret_cast<og_f4 *>(part) + ((long)(mat * (per / kz) + tile) * kz + z) * (T * T / 4) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            og_f4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][j][q * 4 + e] + acx[i][j][q * 4 + e];
            dst[((i * FJ + j) * 4 + q) * WAVES * 64] = v;
          }
      return;
    }
  } else {
    early();
    const int nz = g.aux;
    const og_f4 *src = reinterpret_cast<const og_f4 *>(part) + (long)(mat * per + tile) * nz * (T * T / 4) + threadIdx.x;
    for (int k = 0; k < nz; ++k, src += T * T / 4)
#pragma unroll
      for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const og_f4 v = src[((i * FJ + j) * 4 + q) * WAVES * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][q * 4 + e] += v[e];
          }
  }
  auto stored = [&](int which, int q, int i, int j, float (&v)[4]) {     // 4 stored values of row i from column j on
    if constexpr (EARLY) {
      og_value(el[which * 4 + q], v);
    } else {
      const char *p = (which ? e2 : e1) + og_at(M, i, j);
      og_b4 l[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) l[k] = *reinterpret_cast<const og_b4 *>(p + k * 64);
      og_value(l, v);
    }
  };
  const bool last = type == OL_LAST, mirrored = type == OL_SYM && bi != bj;
  const OrthoPtr ptr = ortho_ptr(lv.gs, g, mat, lv.mode == OM_BF16 ? 2 : 4);
  const int m = og_short(g), nn = og_long(g);
  const bool tall = g.rows > g.cols;
  char *out = last ? nullptr : ortho_buffer(ws, g, job.out, mat);
  if (!last) __syncthreads();                                            // the stages become the waves' exchange buffers
  char *tp = smem + wave * 32 * TP;
#pragma unroll
  for (int fi = 0; fi < FI; ++fi)
#pragma unroll
    for (int fj = 0; fj < FJ; ++fj) {
      const int i0 = bi * T + (wi * FI + fi) * 32, j0 = bj * T + (wj * FJ + fj) * 32, i = i0 + l31;
      if (i0 >= M || j0 >= cols) continue;                               // (T = 128 on an odd number of 64-row halves)
      og_b4 lq[4][3];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = j0 + q * 8 + lh * 4;
        float v[4], x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = job.k0 * (acc[fi][fj][q * 4 + k] + acx[fi][fj][q * 4 + k]);
        if (e1) {
          stored(0, q, i, j, x);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = fmaf(job.k1, x[k], v[k]);
        }
        if (e2) {
          stored(1, q, i, j, x);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = fmaf(job.k2, x[k], v[k]);
        }
        if (!last) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (i == j + k) v[k] += job.diag;
          og_split(v, lq[q]);
#pragma unroll
          for (int k = 0; k < 3; ++k) *reinterpret_cast<og_b4 *>(tp + l31 * TP + k * 64 + q * 16 + lh * 8) = lq[q][k];
        } else if (i < m) {
          if (!tall && j + 4 <= nn && lv.mode != OM_BF16) {
            og_f4u *o = reinterpret_cast<og_f4u *>((float *)ptr.out + (long)i * nn + j);
            og_f4u y;
            if (lv.mode == OM_MUON) {
              const og_f4u w = *o;
#pragma unroll
              for (int k = 0; k < 4; ++k) y[k] = fmaf(-g.step, v[k], w[k] * lv.decay);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) y[k] = v[k];
            }
            *o = y;
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (j + k < nn) og_result(ptr.out, tall ? (long)(j + k) * m + i : (long)i * nn + j + k, v[k], lv.mode, g.step, lv.decay);
          }
        }
      }
      if (!last) {
        // 32 lines of the result lie one behind the other: 16 bytes per lane, six full stores
        auto leave = [&](char *o) {
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
          for (int s = 0; s < 6; ++s) {
            const int u = lane + s * 64;
            *reinterpret_cast<og_b8 *>(o + u * 16) = *reinterpret_cast<const og_b8 *>(tp + u / 12 * TP + u % 12 * 16);
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        };
        leave(out + og_at(M, i0, j0));
        if (mirrored) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              char *d = tp + (q * 8 + lh * 4 + k) * TP + (l31 >> 3) * 16 + (l31 & 7) * 2;
#pragma unroll
              for (int n = 0; n < 3; ++n) *reinterpret_cast<__bf16 *>(d + n * 64) = lq[q][n][k];
            }
          leave(out + og_at(M, j0, i0));
        }
      }
    }
}

// ---- short sides of up to 64 ---------------------------------------------------------------------------------------------
// A and Q (one after the other) and up to 320 columns of X of 33 to 64 rows (24 + 120 KB), 704 of up to 32 (6 + 132 KB), fit into LDS as
// limbs, so one workgroup can take a step's products one after the other with barriers between them; as launches they cost 5 us each
// at these sizes.  Such matrices run their whole iteration in one workgroup (ortho_small_kernel).  Longer ones are cut into panels of
// columns, one workgroup each: a launch per step adds the panels' shares of the Gram matrix up (every workgroup for itself, in a fixed
// order), forms Q, multiplies its panel by it and leaves the panel's share of the next Gram matrix (ortho_panel_kernel).
// Five steps, panels / the products as launches, us (one workgroup: 50 x 108 30, 64 x 256 43, 64 x 320 55, 20 x 700 59, 1000 of 20 x 330 82):
//   64 x 449  57 / 115     8 of 33 x 1000  67 / 132     100 of 64 x 576  121 / 166     64 x 4096   83 / 141     16 of 64 x 8192 273 / 259
//   20 x 8192 83 / 154    40 of 64 x 576  75 / 133      256 of 64 x 576 240 / 251     64 x 10240 122 / 164     30 of 64 x 4096 261 / 253
// The right-hand column takes more than one workgroup per CU (two rounds of them, 98 KB of LDS and more each): those go as products.
// Narrowest panels of 2 / 4 / 6 chunks: 8 of 33 x 1000 70 / 67 / 78, 20 of 64 x 576 69 / 65 / 73, 64 x 449 53 / 56 / 70.
#define ORTHO_SMALL_M 64
#define ORTHO_SMALL_LDS 147456 // 320 columns of 64 rows, 704 of 32
#define ORTHO_WIDE 4           // narrowest panel, in chunks of 32 columns
#define ORTHO_WIDEST 10        // widest: 320 columns
#define ORTHO_PANELS 32        // longest row of panels: every workgroup reads 16 KB of each
#define ORTHO_FEW 16           // pointers that travel in the kernels' arguments, without a launch that fills the table
struct OrthoSmall {
  OrthoGroups gs;
  OrthoPtr few[ORTHO_FEW];          // read one per lane, as the groups are
  OrthoMomentum mo;
  int steps;
  float a, b, c;
  float decay, eps;
};

// MT: the short side in tiles of 32 rows
__host__ __device__ static inline int og_mt(const OrthoGroup &g) { return og_short(g) <= 32 ? 1 : 2; }
// bytes of 32 MT rows x 32 columns in LDS
__host__ __device__ static constexpr int og_chunk(int MT) { return 32 * MT * OG_LINE; }
// byte of columns 8 q ... 8 q + 7 of row r, one limb, in a chunk in LDS
__device__ __forceinline__ int og_unit(int r, int q, int limb) { return r * OG_LINE + limb * 64 + ((q ^ ((r >> 2) & 3)) << 4); }
// 8 columns of a row, half chunk `half`, one limb: a lane's MFMA operand
__device__ __forceinline__ og_b8 og_frag(const char *chunk, int row, int half, int limb) {
  return *reinterpret_cast<const og_b8 *>(chunk + og_unit(row, half * 2 + ((threadIdx.x >> 5) & 1), limb));
}
// 4 values of a row from column 8 q + 4 (lane / 32) on
__device__ __forceinline__ void og_put(char *chunk, int row, int q, const float (&v)[4]) {
  og_b4 l[3];
  og_split(v, l);
#pragma unroll
  for (int k = 0; k < 3; ++k) *reinterpret_cast<og_b4 *>(chunk + og_unit(row, q, k) + ((threadIdx.x >> 5) & 1) * 8) = l[k];
}
// acc, acx += (limbs of y)(limbs of x)^T; the smallest first, 0 0 apart from the others as in ortho_product_kernel
__device__ __forceinline__ void og_multiply(const og_b8 (&y)[3], const og_b8 (&x)[3], og_f16v &acc, og_f16v &acx) {
  acx = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], x[2], acx, 0, 0, 0);
  acx = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[2], x[0], acx, 0, 0, 0);
  acx = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[1], x[1], acx, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], x[0], acc, 0, 0, 0);
  acx = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], x[1], acx, 0, 0, 0);
  acx = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[1], x[0], acx, 0, 0, 0);
}

// A panel's elements, 256 threads, 64 columns at a time (8 MT elements per thread); lanes run along the rows of G (TALL: along the
// short side).  Loads and stores go through buffer descriptors, whose bounds check does the padding's zeros: no branch stands between them.
template <bool TALL, int MT>
struct OgWalk {
  static constexpr int E = 8 * MT, COLS = TALL ? 8 / MT : 1, CH = og_chunk(MT);      // COLS: columns from one of a thread's elements to the next
  int so, valid, row;             // elements between two of a thread's; how many it has there; bytes of its row and column in LDS
  int o, step, left;              // first element; to the next 64 columns; columns left
  int lane, wave, m, r, c;        // r, c: TALL: its row and first column
  __device__ __forceinline__ OgWalk(const OrthoGroup &g, int j0, int chunks) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    m = og_short(g);
    const int n = og_long(g);
    left = n - j0 < chunks * 32 ? n - j0 : chunks * 32;
    r = lane & (32 * MT - 1);
    c = MT == 1 ? wave * 2 + (lane >> 5) : wave;
    so = TALL ? COLS * m : 4 * n;
    step = TALL ? 64 * m : 64;
    o = TALL ? (j0 + c) * m + r : wave * n + j0 + lane;
    row = TALL ? r * OG_LINE + ((c >> 2) & 1) * 64 + (c & 3) * 4 : (lane >> 5) * CH + wave * OG_LINE + ((lane >> 2) & 1) * 64 + (lane & 3) * 4;
    count();
  }
  __device__ __forceinline__ void count() { valid = TALL ? (r < m ? (left - c + COLS - 1) / COLS : 0) : lane < left ? (m - wave + 3) >> 2 : 0; }
  __device__ __forceinline__ void next() {
    left -= 64;
    o += step;
    row += 2 * CH;
    count();
  }
  __device__ __forceinline__ int at(int e) const { return e < valid ? o + e * so : -1; }      // -1: behind every buffer
  __device__ __forceinline__ int lds(int e) const {
    if constexpr (TALL) {
      const int first = e * COLS;                                                              // c + first: the column of 64
      return row + (first >> 5) * CH + ((first >> 2) & 1) * 64 + ((((first >> 3) & 3) ^ ((r >> 2) & 3)) << 4);
    } else {
      return row + e * 4 * OG_LINE + ((((lane & 31) >> 3) ^ (e & 3)) << 4);
    }
  }
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t og_buffer(void *p, int bytes) { return __builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, 0x00027000); }
template <typename T>
__device__ __forceinline__ float og_get(__amdgpu_buffer_rsrc_t b, int o) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, o < 0 ? -1 : o * 4, 0, 0));
  else return __uint_as_float((unsigned)__builtin_amdgcn_raw_buffer_load_b16(b, o < 0 ? -1 : o * 2, 0, 0) << 16);
}
__device__ __forceinline__ void og_set(__amdgpu_buffer_rsrc_t b, int o, float v) {
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), b, o < 0 ? -1 : o * 4, 0, 0);
}

// G (Muon: the momentum, updated on the way) as f32 into the place of its first two limbs (columns 8 q ... 8 q + 3 | 8 q + 4 ... 8 q + 7);
// returns the thread's sum of squares
template <typename T, bool MUON, bool TALL, int MT>
__device__ __forceinline__ double og_fetch(const OrthoGroup &g, int j0, int chunks, const OrthoPtr &ptr, const OrthoMomentum &mo, char *X) {
  const int size = g.rows * g.cols;
  const __amdgpu_buffer_rsrc_t src = og_buffer(const_cast<void *>((const void *)ptr.g), size * (int)sizeof(T));
  const __amdgpu_buffer_rsrc_t mom = og_buffer(ptr.m, MUON ? size * 4 : 0);
  OgWalk<TALL, MT> w(g, j0, chunks);
  constexpr int E = 8 * MT;
  double sum = 0.;
  for (int c = 0; c < chunks; c += 2, w.next()) {
    float v[E], mm[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = og_get<T>(src, w.at(e));
    if constexpr (MUON)
#pragma unroll
      for (int e = 0; e < E; ++e) mm[e] = og_get<float>(mom, w.at(e));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (MUON) {
        v[e] *= mo.gscale;
        mm[e] = fmaf(mo.mu, mm[e], v[e]);
        og_set(mom, w.at(e), mm[e]);
        v[e] = mo.nesterov ? fmaf(mo.mu, mm[e], v[e]) : mm[e];
      }
      sum += (double)v[e] * (double)v[e];
      *reinterpret_cast<float *>(X + w.lds(e)) = v[e];
    }
  }
  return sum;
}

// f32 into limbs in place: X0 = G / norm
template <int MT>
__device__ __forceinline__ void og_limbs(char *X, int chunks, double norm) {
  const OgUnit unit(norm);
  for (int t = threadIdx.x; t < chunks * 128 * MT; t += 256) {
    const int row = t & (32 * MT - 1), q = t / (32 * MT);
    char *p = X + (q >> 2) * og_chunk(MT) + og_unit(row, q & 3, 0);
    const og_f4 x[2] = {*reinterpret_cast<og_f4 *>(p), *reinterpret_cast<og_f4 *>(p + 64)};
    og_b4 l[2][3];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float v[4] = {unit(x[e][0]), unit(x[e][1]), unit(x[e][2]), unit(x[e][3])};
      og_split(v, l[e]);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<og_b8 *>(p + k * 64) = og_join(l[0][k], l[1][k]);
  }
}

// the results, f32 in X, to where they belong
template <typename T, bool MUON, bool TALL, int MT>
__device__ __forceinline__ void og_deliver(const OrthoGroup &g, int j0, int chunks, const OrthoPtr &ptr, const char *X, float decay) {
  const __amdgpu_buffer_rsrc_t out = og_buffer(ptr.out, g.rows * g.cols * (int)sizeof(T));
  OgWalk<TALL, MT> w(g, j0, chunks);
  constexpr int E = 8 * MT;
  for (int c = 0; c < chunks; c += 2, w.next()) {
    float old[E];
    if constexpr (MUON)
#pragma unroll
      for (int e = 0; e < E; ++e) old[e] = og_get<float>(out, w.at(e));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = *reinterpret_cast<const float *>(X + w.lds(e));
      const int o = w.at(e);
      if constexpr (MUON) og_set(out, o, fmaf(-g.step, v, old[e] * decay));
      else if constexpr (sizeof(T) == 4) og_set(out, o, v);
      else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)v), out, o < 0 ? -1 : o * 2, 0, 0);  // the one rounding
    }
  }
}

// this wave's 32 x 32 tile of Y Y^T, Y = `chunks` chunks at `in`, each chunk's operands requested a chunk ahead
template <bool DIAG, int MT>
__device__ __forceinline__ void og_square_tile(const char *in, int chunks, int ti, int tj, float (&v)[16]) {
  const int l31 = threadIdx.x & 31;
  og_f16v acc, acx;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = acx[e] = 0.f;
  og_b8 f[2][2][3], g[2][2][3];
  auto load = [&](int c, int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        f[b][h][k] = og_frag(in + c * og_chunk(MT), ti + l31, h, k);
        if constexpr (!DIAG) g[b][h][k] = og_frag(in + c * og_chunk(MT), tj + l31, h, k);
      }
  };
  auto multiply = [&](int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) og_multiply(DIAG ? f[b][h] : g[b][h], f[b][h], acc, acx);
  };
  load(0, 0);
  for (int c = 0;;) {
    load(c + 1 < chunks ? c + 1 : c, 1);
    multiply(0);
    if (++c == chunks) break;
    load(c + 1 < chunks ? c + 1 : c, 0);
    multiply(1);
    if (++c == chunks) break;
  }
  og_settle(acc, acx);
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = acc[e] + acx[e];
}
template <int MT>
__device__ __forceinline__ void og_square(const char *in, int chunks, int ti, int tj, float (&v)[16]) {
  if (MT == 1 || ti == tj) og_square_tile<true, MT>(in, chunks, ti, tj, v);
  else og_square_tile<false, MT>(in, chunks, ti, tj, v);
}

// Q = a I + b A + c A A from the wave's tile v of A; A passes through Q's place.  Two barriers in between, none behind
template <int MT>
__device__ __forceinline__ void og_make_q(char *Q, int ti, int tj, const float (&v)[16], const OrthoSmall &co) {
  const int l31 = threadIdx.x & 31, lh = (threadIdx.x >> 5) & 1;
  const bool mine = MT > 1 || threadIdx.x < 64;
  auto put = [&](const float (&t)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float w[4] = {t[q * 4], t[q * 4 + 1], t[q * 4 + 2], t[q * 4 + 3]};
      og_put(Q + (tj >> 5) * og_chunk(MT), ti + l31, q, w);
    }
  };
  if (mine) put(v);
  __syncthreads();
  float p[16];
  if (mine) og_square<MT>(Q, MT, ti, tj, p);
  __syncthreads();
  if (mine) {
#pragma unroll
    for (int e = 0; e < 16; ++e) p[e] = fmaf(co.c, p[e], fmaf(co.b, v[e], ti + l31 == tj + (e >> 2) * 8 + lh * 4 + (e & 3) ? co.a : 0.f));
    put(p);
  }
}

// X <- factor Q X, a wave's chunks one after the other (so a result may go where the chunk was read).  Begins with a barrier, in front
// of which the first chunk is requested (transposing reads).  `last`: f32 instead of limbs.
template <int MT>
__device__ __forceinline__ void og_apply(const char *Q, char *X, int chunks, float factor, bool last) {
  const int lane = threadIdx.x & 63, l31 = lane & 31, lh = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  og_b8 x[2 * MT][3], qf[2 * MT][MT][3];
  auto load = [&](const char *chunk) {
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) {
      const int r = h * 16 + lh * 8 + ((lane & 15) >> 2), u = ((lane >> 4) & 1) * 2 + ((lane & 2) >> 1);
#pragma unroll
      for (int k = 0; k < 3; ++k)
        x[h][k] = c8_tr_frag((const unsigned char *)chunk + og_unit(r, u, k) + (lane & 1) * 8,
                             (const unsigned char *)chunk + og_unit(r + 4, u, k) + (lane & 1) * 8);
    }
  };
  if (wave < chunks) load(X + wave * og_chunk(MT));
  __syncthreads();
  if (wave >= chunks) return;
#pragma unroll
  for (int h = 0; h < 2 * MT; ++h)
#pragma unroll
    for (int f = 0; f < MT; ++f)
#pragma unroll
      for (int k = 0; k < 3; ++k) qf[h][f][k] = og_frag(Q + (h >> 1) * og_chunk(MT), f * 32 + l31, h & 1, k);
  for (int ch = wave; ch < chunks; ch += 4) {
    char *chunk = X + ch * og_chunk(MT);
    og_f16v acc[MT], acx[MT];
#pragma unroll
    for (int f = 0; f < MT; ++f)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[f][e] = acx[f][e] = 0.f;
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h)
#pragma unroll
      for (int f = 0; f < MT; ++f) og_multiply(x[h], qf[h][f], acc[f], acx[f]);
    if (ch + 4 < chunks) load(chunk + 4 * og_chunk(MT));
#pragma unroll
    for (int f = 0; f < MT; ++f) og_settle(acc[f], acx[f]);
#pragma unroll
    for (int f = 0; f < MT; ++f)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[f][e] = factor * (acc[f][e] + acx[f][e]);
    auto each = [&](auto store) {
#pragma unroll
      for (int f = 0; f < MT; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v[4] = {acc[f][q * 4], acc[f][q * 4 + 1], acc[f][q * 4 + 2], acc[f][q * 4 + 3]};
          store(f * 32 + l31, q, v);
        }
    };
    if (last)
      each([&](int i, int q, const float(&v)[4]) { *reinterpret_cast<og_f4 *>(chunk + og_unit(i, q, lh)) = og_f4{v[0], v[1], v[2], v[3]}; });
    else
      each([&](int i, int q, const float(&v)[4]) { og_put(chunk, i, q, v); });
  }
}

// sum over 256 threads, the same in all of them; a barrier inside
template <int CTRL>
__device__ __forceinline__ double og_dpp(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, 0xf, 0xf, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, true);
  return v + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double og_block_sum(double s, double *red) {
  s = og_dpp<0xB1>(s);           // lane ^ 1, lane ^ 2, mirrored in 8, in 16
  s = og_dpp<0x4E>(s);
  s = og_dpp<0x141>(s);
  s = og_dpp<0x140>(s);
  if ((threadIdx.x & 15) == 0) red[threadIdx.x >> 4] = s;
  __syncthreads();
  double t = 0.;
#pragma unroll
  for (int i = 0; i < 16; ++i) t += red[i];
  return t;
}

__device__ __forceinline__ OrthoPtr og_small_ptr(const OrthoSmall &c, const OrthoGroup &g, int mat, int bytes) {
  if (g.ptr < 0 || c.gs.table) return ortho_ptr(c.gs, g, mat, bytes);
  const OrthoPtr mine = c.few[threadIdx.x & (ORTHO_FEW - 1)];
  return og_readlane(mine, __builtin_amdgcn_readfirstlane(g.ptr + mat));
}

template <typename T, bool MUON, int MT>
__device__ __forceinline__ void ortho_alone(const OrthoSmall &c, const OrthoGroup &g, const OrthoPtr &ptr, char *smem, double *red) {
  const int chunks = (og_long(g) + 31) / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char *Q = smem, *X = smem + MT * og_chunk(MT);
  const bool tall = g.rows > g.cols;
  const double sum = tall ? og_fetch<T, MUON, true, MT>(g, 0, chunks, ptr, c.mo, X) : og_fetch<T, MUON, false, MT>(g, 0, chunks, ptr, c.mo, X);
  og_limbs<MT>(X, chunks, sqrt(og_block_sum(sum, red)) + (double)c.eps);
  const int ti = MT > 1 ? (wave >> 1) * 32 : 0, tj = MT > 1 ? (wave & 1) * 32 : 0;          // this wave's tile of A and Q
  for (int k = 0; k < c.steps; ++k) {
    float v[16];
    __syncthreads();
    if (MT > 1 || wave == 0) og_square<MT>(X, chunks, ti, tj, v);
    og_make_q<MT>(Q, ti, tj, v, c);
    og_apply<MT>(Q, X, chunks, 1.f, k + 1 == c.steps);
  }
  __syncthreads();
  if (tall) og_deliver<T, MUON, true, MT>(g, 0, chunks, ptr, X, c.decay);
  else og_deliver<T, MUON, false, MT>(g, 0, chunks, ptr, X, c.decay);
}

template <typename T, bool MUON>
__global__ __launch_bounds__(256, 2) void ortho_small_kernel(OrthoSmall c) {
  extern __shared__ __align__(1024) char smem[];
  __shared__ double red[16];
  int grp;
  const OrthoGroup g = ortho_group_of(c.gs, blockIdx.x, grp);
  const OrthoPtr ptr = og_small_ptr(c, g, blockIdx.x - g.first, sizeof(T));
  if (og_mt(g) == 1) ortho_alone<T, MUON, 1>(c, g, ptr, smem, red);
  else ortho_alone<T, MUON, 2>(c, g, ptr, smem, red);
}

// LDS of a workgroup that keeps `chunks` chunks of X: A or Q, and an even number of chunks (OgWalk goes over 64 columns at a time)
static inline int og_small_lds(const OrthoGroup &g, int chunks) { return (og_mt(g) + (chunks + 1) / 2 * 2) * og_chunk(og_mt(g)); }
__host__ __device__ static inline int og_panels(const OrthoGroup &g) { return ((og_long(g) + 31) / 32 + g.jobs - 1) / g.jobs; }

// Launch k of a chain of panels: k = 0 forms X0's panel and its share of the first Gram matrix, launch k > 0 takes step k - 1.  X's
// panels lie in the workspace as they lie in LDS; the shares (f32, as the MFMAs leave them) go to one of two sets in turn, since
// other workgroups may still read the last launch's.  Launch 0 knows only its own panel's norm and divides by that; launch 1 knows
// all of them and puts it right: a panel's share counts (its norm / the matrix' norm)^2 times, its result their quotient times.
template <typename T, bool MUON, int MT>
__device__ __forceinline__ void ortho_panel(const OrthoSmall &c, const OrthoGroup &g, char *ws, double *sums, int k, char *smem, double *red) {
  const int panels = og_panels(g), wide = g.jobs, mat = og_div(blockIdx.x - g.first, panels), pan = blockIdx.x - g.first - mat * panels;
  const int all = (og_long(g) + 31) / 32, chunks = all - pan * wide < wide ? all - pan * wide : wide;
  char *Q = smem, *X = smem + MT * og_chunk(MT);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ti = MT > 1 ? (wave >> 1) * 32 : 0, tj = MT > 1 ? (wave & 1) * 32 : 0;
  const bool square = MT > 1 || wave == 0;
  const OrthoPtr ptr = og_small_ptr(c, g, mat, sizeof(T));
  const bool tall = g.rows > g.cols;
  const int j0 = pan * wide * 32;
  char *mine = ws + (size_t)g.x_off * 256 + ((size_t)mat * all + pan * wide) * og_chunk(MT);
  og_f4 *share = reinterpret_cast<og_f4 *>(ws + (size_t)g.p_off * 256);                       // [set][mat][panel][q][thread]
  const size_t set = (size_t)g.count * panels * 1024;
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = 0.f;
  if (k == 0) {
    const double part = tall ? og_fetch<T, MUON, true, MT>(g, j0, chunks, ptr, c.mo, X) : og_fetch<T, MUON, false, MT>(g, j0, chunks, ptr, c.mo, X);
    const double sum = og_block_sum(part, red);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
    og_limbs<MT>(X, chunks, sum == 0. ? 1. : sqrt(sum));
  } else {
    for (int t = threadIdx.x; t < chunks * (og_chunk(MT) / 16); t += 256)
      reinterpret_cast<og_b8 *>(X)[t] = reinterpret_cast<const og_b8 *>(mine)[t];
    const og_f4 *p = share + ((k - 1) & 1) * set + (size_t)mat * panels * 1024 + threadIdx.x;
    float own = 1.f;
    float *weight = reinterpret_cast<float *>(red + 16);
    if (k == 1) {
      const int lane = threadIdx.x & 63;
      const double part = lane < panels ? sums[blockIdx.x - pan + lane] : 0.;
      double norm = part;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) norm += __shfl_xor(norm, o, 64);
      norm = sqrt(norm) + (double)c.eps;
      const float quotient = (float)(sqrt(part) / norm);
      own = __shfl(quotient, pan, 64);
      if (lane < panels) weight[lane] = quotient * quotient;     // (every wave the same)
    }
    auto gather = [&](auto part) {
#pragma unroll 4
      for (int z = 0; z < panels; ++z, p += 1024) {
        const float share = part(z);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const og_f4 s = p[q * 256];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[q * 4 + e] = fmaf(s[e], share, v[q * 4 + e]);
        }
      }
    };
    if (square && k == 1) gather([&](int z) { return weight[z]; });
    else if (square) gather([](int) { return 1.f; });
    og_make_q<MT>(Q, ti, tj, v, c);
    og_apply<MT>(Q, X, chunks, own, k == c.steps);
  }
  __syncthreads();
  if (k == c.steps) {
    if (tall) og_deliver<T, MUON, true, MT>(g, j0, chunks, ptr, X, c.decay);
    else og_deliver<T, MUON, false, MT>(g, j0, chunks, ptr, X, c.decay);
    return;
  }
  if (square) {
    og_square<MT>(X, chunks, ti, tj, v);
    og_f4 *o = share + (k & 1) * set + ((size_t)mat * panels + pan) * 1024 + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q * 256] = og_f4{v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]};
  }
  for (int t = threadIdx.x; t < chunks * (og_chunk(MT) / 16); t += 256) reinterpret_cast<og_b8 *>(mine)[t] = reinterpret_cast<const og_b8 *>(X)[t];
}

template <typename T, bool MUON>
__global__ __launch_bounds__(256, 2) void ortho_panel_kernel(OrthoSmall c, char *__restrict__ ws, double *__restrict__ sums, int k) {
  extern __shared__ __align__(1024) char smem[];
  __shared__ double red[16 + ORTHO_PANELS / 2];
  int grp;
  const OrthoGroup g = ortho_group_of(c.gs, blockIdx.x, grp);
  if (og_mt(g) == 1) ortho_panel<T, MUON, 1>(c, g, ws, sums, k, smem, red);
  else ortho_panel<T, MUON, 2>(c, g, ws, sums, k, smem, red);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
struct OrthoCall {
  int steps;
  float a, b, c, eps;
  int mode;
  bool bf16;
  float decay;
  OrthoMomentum mo;
};

// Steps between two Gram matrices.  Longer chains save products with the long side and add M x M products, so they pay from N = 2 M
// on, and only where the long side's products fill the chip (`tiles`: 128 x 128 tiles of Q X of the whole pass; below, the number of
// launches counts, and chains of one have the fewest).  They carry rounding further, the more the smaller M: the lengths taken stay
// below the error of the plain iteration in f32.  Five steps with chains of 1 / 2 / 3, time and relative error against 64 bits (plain f32):
//   28 x 256 x 2304  663 / 526 / 460 us    1.3 / 1.5 / 2.6e-6  (3.4e-6)      4 x 256 x 1152   185 / 190 / 182 us    0.9 / 1.5 / 2.5e-6  (2.7e-6)
//   2048 x 9216     3796 / 2903 / 2422     1.8 / 1.8 / 2.5e-6  (5.4e-6)      3 x 333 x 1021   199 / 207 / 206       0.9 / 1.4 / 2.4e-6  (2.7e-6)
//   20 x 200 x 1000  251 / 234 / 226       1.0 / 1.8 / 3.1e-6  (2.5e-6)      1500 x 2000      657 / 670 / 668       1.2 / 1.3 / 4.0e-6  (3.5e-6)
//   1024 x 4608      647 / 533 / 469       1.2 / 1.2 / 3.0e-6  (3.7e-6)      4 x 128 x 576    134 / 148 / 145       0.6 / 2.3 / 2.8e-6  (1.7e-6)
static int ortho_chain(const OrthoGroup &g, long tiles) {
  const int M = og_short(g), N = og_long(g);
  if (tiles < 256 || M < 192 || N < 2 * M) return 1;
  return M < 256 || N < 4 * M ? 2 : 3;
}

// Coefficients that let a singular value of [0, 1] grow out of hand are refused: what a chain computes of it would pass the range of
// f32, and its rounding would drown the others.  One chain of n steps from the singular values sv, which are advanced to those
// behind the chain; every matrix of the chain (X, A, S, T = A P, R, Q = a^n I + R) has polynomials of them as singular values.
#define ORTHO_SAMPLES 257
#define ORTHO_GROWTH 1e4
static bool ortho_bounded(double *sv, int n, const OrthoCall &c) {
  bool ok = true;
  for (int i = 0; i < ORTHO_SAMPLES; ++i) {
    auto see = [&ok](double v) { ok = ok && fabs(v) <= ORTHO_GROWTH; };    // (false for a NaN)
    double lam = sv[i] * sv[i], r = 0., an = 1.;
    see(sv[i]);
    for (int k = 0; k < n; ++k) {
      const double A = lam, S = c.b * A + c.c * A * A, P = c.a + S;
      r = k ? c.a * r + an * S + r * S : S;
      lam = A * P * P;
      see(A);
      see(S);
      see(A * P);
      see(r);
      an *= c.a;
    }
    see(an + r);
    sv[i] *= an + r;
    see(sv[i]);
  }
  return ok;
}

// the products of one chain length, in order
struct OrthoPlan {
  struct {
    OrthoJob job[2];
    int jobs, type;
  } level[3 * ORTHO_STEPS + ORTHO_STEPS];
  int levels;                       // 0: not asked for yet
};

static bool ortho_plan(OrthoPlan *p, int most, const OrthoCall &c) {
  p->levels = 0;
  double sv[ORTHO_SAMPLES];
  for (int i = 0; i < ORTHO_SAMPLES; ++i) {                              // denser towards 0
    const double u = (double)i / (ORTHO_SAMPLES - 1);
    sv[i] = 1.00001 * u * u * u;
  }
  auto add = [p](int type, const OrthoJob &job) {
    p->level[p->levels].type = type;
    p->level[p->levels].jobs = 1;
    p->level[p->levels++].job[0] = job;
  };
  for (int left = c.steps, set = 0; left > 0; set ^= 1) {
    const int chain = left < most ? left : most;
    if (!ortho_bounded(sv, chain, c)) return false;
    const int x = set ? OB_X1 : OB_X0;
    add(OL_SYM, OrthoJob{x, x, OB_NONE, OB_NONE, OB_A, 1.f, 0.f, 0.f, 0.f});
    int r = OB_R0;                                                         // R of the first step is its S
    float an = c.a;                                                        // a^k
    for (int k = 0; k < chain; ++k) {
      const bool more = k + 1 < chain;
      const int s = k ? OB_S : OB_R0;
      // S = b A + c A A (the whole chain's Q = a I + S if it is one step)
      add(OL_SYM, OrthoJob{OB_A, OB_A, OB_A, OB_NONE, s, c.c, c.b, 0.f, k || more ? 0.f : an});
      OrthoJob todo[2];
      int jobs = 0;
      if (more) todo[jobs++] = OrthoJob{OB_A, s, OB_A, OB_NONE, OB_T, 1.f, c.a, 0.f, 0.f};                         // T = a A + A S
      if (k) {                                                                            // R = a R + a^k S + R S (+ a^(k+1) I: Q)
        const int to = r == OB_R0 ? OB_R1 : OB_R0;
        todo[jobs++] = OrthoJob{r, s, r, s, to, 1.f, c.a, an, more ? 0.f : an * c.a};
        r = to;
        an *= c.a;
      }
      if (jobs) {
        add(OL_SYM, todo[0]);
        p->level[p->levels - 1].job[1] = todo[1];
        p->level[p->levels - 1].jobs = jobs;
      }
      if (more) add(OL_SYM, OrthoJob{OB_T, s, OB_T, OB_NONE, OB_A, 1.f, c.a, 0.f, 0.f});                           // A = a T + T S
    }
    left -= chain;
    add(left > 0 ? OL_RECT : OL_LAST, OrthoJob{r, x, OB_NONE, OB_NONE, set ? OB_X0 : OB_X1, 1.f, 0.f, 0.f, 0.f});  // X = Q X
  }
  return true;
}

// Ranges of a Gram matrix' reduction.  A product whose tiles leave CUs idle splits a long reduction into ranges of 512 columns, at the
// price of the launch that adds them up: no block longer than its share of the pass' whole reduction (`work`: columns times tiles)
// on 256 CUs; of 4096 columns and more on 768 blocks, three to a CU, since one alone waits for its loads (0.75 us a chunk, 0.17 of
// MFMAs).  Five steps, no ranges / 1024 / 512 / 256 columns: 512 x 2304 292 / 248 / 226 / 226 us, 200 x 4000 322 / 213 / 184 / 186,
// 128 x 8192 508 / 194 / 186 / 185, 3 x 333 x 1021 209 / 211 / 204 / 198, 4 x 128 x 576 137 / 136 / 137 / 147.  Shares of 256 / 768: a step of
// the generator and the pose mapping (1024 x 16384 and 1024 x 8192 among 42) 2377 / 2066, 1024 x 16384 949 / 905, 1024 x 4608 486 / 469, 1300 x
// 9000 943 / 968; below 4096 columns: 1024 x 1024 263 / 284, 2 x 600 x 2000 300 / 314, 28 x 256 x 2304 441 / 457.
#define ORTHO_KZ 16
static int ortho_kz(int K, long own, long work) {
  long z = (K >= 4096 ? 768L : 256L) * K / work;
  if (own <= 16 && z < K / 1024) z = K / 1024;             // few tiles in the company of many: not the launch's last ones
  const long most = K / 512;
  if (z > most) z = most;
  if (z > ORTHO_KZ) z = ORTHO_KZ;
  return z < 2 ? 1 : (int)z;
}

struct OrthoLayout {
  size_t sums, bytes;
  bool small, panels;               // every matrix fits ortho_small_kernel, ortho_panel_kernel
  int chain[ORTHO_GROUPS];
  int kz[ORTHO_GROUPS];             // of the Gram matrices
  int norm_first[ORTHO_GROUPS], split_first[ORTHO_GROUPS];
  int norm_blocks, split_blocks;
};

// Widths of the panels (g[i].jobs): the smallest from ORTHO_WIDE chunks on that leaves the pass no more workgroups than CUs and no
// matrix more than ORTHO_PANELS panels.  False if there is none.
static bool ortho_panel_chunks(OrthoGroup *g, int n) {
  for (int w = ORTHO_WIDE; w <= ORTHO_WIDEST; ++w) {
    long blocks = 0, most = 0;
    for (int i = 0; i < n; ++i) {
      g[i].jobs = w;
      blocks += (long)g[i].count * og_panels(g[i]);
      if (og_panels(g[i]) > most) most = og_panels(g[i]);
    }
    if (blocks <= 256 && most <= ORTHO_PANELS) return true;
  }
  return false;
}

// workspace: pointers | partial sums of squares | per group X (two when there is more than one chain), the M x M matrices, the
// partial Gram matrices
static OrthoLayout ortho_layout(OrthoGroup *g, int n, int steps) {
  OrthoLayout lo;
  memset(&lo, 0, sizeof lo);
  lo.sums = align_up(sizeof(OrthoPtr) * ORTHO_MATRICES, 256);
  lo.small = lo.panels = true;
  for (int i = 0; i < n; ++i) {
    lo.chain[i] = 1;
    lo.norm_first[i] = lo.norm_blocks;
    lo.norm_blocks += g[i].count * og_norm_blocks(g[i]);
    lo.panels = lo.panels && og_short(g[i]) <= ORTHO_SMALL_M;
    lo.small = lo.small && lo.panels && og_small_lds(g[i], (og_long(g[i]) + 31) / 32) <= ORTHO_SMALL_LDS;
  }
  size_t at = lo.sums + align_up(lo.norm_blocks * sizeof(double), 256);
  lo.panels = lo.panels && !lo.small && ortho_panel_chunks(g, n);
  if (lo.small) {
    lo.bytes = lo.sums;
    return lo;
  }
  if (lo.panels) {                                                       // the panels' sums of squares | X | two sets of their shares
    long blocks = 0;
    for (int i = 0; i < n; ++i) blocks += (long)g[i].count * og_panels(g[i]);
    at = lo.sums + align_up(blocks * sizeof(double), 256);
    for (int i = 0; i < n; ++i) {
      g[i].x_off = (unsigned)(at / 256);
      at += (size_t)g[i].count * ((og_long(g[i]) + 31) / 32) * og_chunk(og_mt(g[i]));
      g[i].p_off = (unsigned)(at / 256);
      at += (size_t)g[i].count * og_panels(g[i]) * 2 * 16384;
    }
    lo.bytes = at;
    return lo;
  }
  long work = 0, rect = 0;
  for (int i = 0; i < n; ++i) rect += (long)g[i].count * og_tiles(g[i], OL_RECT, 128);
  for (int i = 0; i < n; ++i) {
    lo.chain[i] = ortho_chain(g[i], rect);
    lo.split_first[i] = lo.split_blocks;
    lo.split_blocks += g[i].count * og_split_blocks(g[i]);
    work += (long)g[i].count * og_tiles(g[i], OL_SYM, 64) * og_pad(og_long(g[i]));
  }
  for (int i = 0; i < n; ++i) {
    const size_t M = og_pad(og_short(g[i])), N = og_pad(og_long(g[i]));
    g[i].x_off = (unsigned)(at / 256);
    at += M * N * OG_BYTES * g[i].count * (steps > lo.chain[i] ? 2 : 1);  // multiples of 64 x 64 x 6 bytes
    g[i].s_off = (unsigned)(at / 256);
    at += M * M * OG_BYTES * g[i].count * OB_SMALL;
    g[i].p_off = (unsigned)(at / 256);
    lo.kz[i] = ortho_kz((int)N, (long)g[i].count * og_tiles(g[i], OL_SYM, 64), work);
    if (lo.kz[i] > 1) at += (size_t)lo.kz[i] * g[i].count * og_tiles(g[i], OL_SYM, 64) * 64 * 64 * 4;
  }
  lo.bytes = at;
  return lo;
}

template <int T, int KC, int S, int WI, int WJ>
static int ortho_launch(char *ws, const OrthoLevel &lv, int blocks, hipStream_t st) {
  const int lds = S * 2 * T * KC * OG_BYTES;
  if (const int rc = lds_optin(reinterpret_cast<const void *>(&ortho_product_kernel<T, KC, S, WI, WJ>), lds, "ortho_product_kernel")) return rc;
  hipLaunchKernelGGL((ortho_product_kernel<T, KC, S, WI, WJ>), dim3(blocks), dim3(WI * WJ * 64), lds, st, ws, lv);
  return 0;
}

// one pass over at most ORTHO_GROUPS groups and ORTHO_MATRICES pointers
static int ortho_run(OrthoGroup *g, int n, const OrthoPtr &base, const OrthoPtr *ptrs, int nptr, const OrthoCall &c, const OrthoPlan *plan,
                     char *ws, hipStream_t st) {
  const OrthoLayout lo = ortho_layout(g, n, c.steps);
  double *sums = (double *)(ws + lo.sums);
  int levels = 0;
  for (int i = 0; i < n; ++i)
    if (plan[lo.chain[i] - 1].levels > levels) levels = plan[lo.chain[i] - 1].levels;
  const bool few = (lo.small || lo.panels) && nptr <= ORTHO_FEW;
  for (int i = 0; i < nptr && !few; i += ORTHO_PTR_PART) {
    OrthoPtrPart part;
    const int k = nptr - i < ORTHO_PTR_PART ? nptr - i : ORTHO_PTR_PART;
    memcpy(part.p, ptrs + i, k * sizeof(OrthoPtr));
    hipLaunchKernelGGL(ortho_ptr_kernel, dim3(1), dim3(128), 0, st, part, (OrthoPtr *)ws, i, k);
  }
  OrthoLevel lv;
  memset(&lv, 0, sizeof lv);
  lv.mode = c.mode;
  lv.decay = c.decay;
  lv.gs.base = base;
  lv.gs.table = few ? nullptr : (const OrthoPtr *)ws;
  for (int i = 0; i < ORTHO_GROUPS; ++i) {
    if (i < n) lv.gs.g[i] = g[i];
    lv.gs.g[i].first = i < n ? lo.norm_first[i] : INT_MAX;
    lv.gs.g[i].aux = lo.norm_first[i];
  }
  if (lo.small || lo.panels) {
    OrthoSmall sm;
    memset(&sm, 0, sizeof sm);
    sm.gs = lv.gs;
    if (few && nptr) memcpy(sm.few, ptrs, nptr * sizeof(OrthoPtr));
    sm.mo = c.mo;
    sm.steps = c.steps;
    sm.a = c.a;
    sm.b = c.b;
    sm.c = c.c;
    sm.decay = c.decay;
    sm.eps = c.eps;
    int blocks = 0, lds = 0;
    for (int i = 0; i < n; ++i) {
      const int chunks = (og_long(g[i]) + 31) / 32, kept = lo.panels && g[i].jobs < chunks ? g[i].jobs : chunks;
      sm.gs.g[i].first = blocks;
      blocks += lo.panels ? g[i].count * og_panels(g[i]) : g[i].count;
      if (og_small_lds(g[i], kept) > lds) lds = og_small_lds(g[i], kept);
    }
#define ORTHO_SMALL(T, MUON)                                                                                                            \
  do {                                                                                                                                  \
    const void *fn = lo.small ? reinterpret_cast<const void *>(&ortho_small_kernel<T, MUON>) : reinterpret_cast<const void *>(&ortho_panel_kernel<T, MUON>); \
    if (const int rc = lds_optin(fn, ORTHO_SMALL_LDS, "ortho_small_kernel")) return rc;                               \
    if (lo.small) {                                                                                                                     \
      hipLaunchKernelGGL((ortho_small_kernel<T, MUON>), dim3(blocks), dim3(256), lds, st, sm);                                          \
    } else {                                                                                                                            \
      for (int k = 0; k <= c.steps; ++k)                                                                                                \
        hipLaunchKernelGGL((ortho_panel_kernel<T, MUON>), dim3(blocks), dim3(256), lds, st, sm, ws, sums, k);                           \
    }                                                                                                                                   \
  } while (0)
    if (c.mode == OM_MUON) ORTHO_SMALL(float, true);
    else if (!c.bf16) ORTHO_SMALL(float, false);
    else ORTHO_SMALL(__bf16, false);
#undef ORTHO_SMALL
    LSPS_CHECK_LAUNCH("newton_schulz");
    return 0;
  }
  OrthoGroups split = lv.gs;
  for (int i = 0; i < n; ++i) split.g[i].first = lo.split_first[i];
#define ORTHO_PRE(T, MUON)                                                                                                            \
  do {                                                                                                                                \
    hipLaunchKernelGGL((ortho_norm_kernel<T, MUON>), dim3(lo.norm_blocks), dim3(256), 0, st, lv.gs, sums, c.mo);                      \
    hipLaunchKernelGGL((ortho_split_kernel<T, MUON>), dim3(lo.split_blocks), dim3(256), 0, st, split, ws, sums, c.mo, c.eps);         \
  } while (0)
  if (c.mode == OM_MUON) ORTHO_PRE(float, true);
  else if (!c.bf16) ORTHO_PRE(float, false);
  else ORTHO_PRE(__bf16, false);
#undef ORTHO_PRE
  for (int l = 0; l < levels; ++l) {
    long wide = 0;                                                       // 128 x 128 tiles of short sides from 1024 on
    bool square = true, narrow = false;
    for (int i = 0; i < n; ++i) {
      const OrthoPlan &p = plan[lo.chain[i] - 1];
      lv.gs.g[i].type = l < p.levels ? p.level[l].type : OL_SYM;
      lv.gs.g[i].jobs = l < p.levels ? p.level[l].jobs : 0;
      if (l < p.levels) memcpy(lv.job + 2 * i, p.level[l].job, sizeof p.level[l].job);
      square = square && lv.gs.g[i].type == OL_SYM;
      if (og_short(g[i]) >= 1024) wide += (long)g[i].count * lv.gs.g[i].jobs * og_tiles(g[i], lv.gs.g[i].type, 128);
      else narrow |= lv.gs.g[i].jobs > 0;
    }
    // 128 x 128 tiles read each operand half as often, but there are fewer of them and one at a time on a CU (98 KB of LDS): for short
    // sides from 1024 on where they go round the 256 CUs once, most of them busy, or (Q X) more than twice; symmetric ones not in the
    // company of shorter sides, which need their reductions split (the discriminator's step 3170 us so, 2830 on 64).  Five steps, us, 64 / 128 wide:
    //   symmetric: 1800 x 3000 (120 tiles) 1205 / 1409, 2048 x 9216 (136) 2416 / 2364, 2300 x 2300 (171) 1608 / 1579, 2500 x 9000 (210) 4225 /
    //   3914, 6 x 1024 x 1024 (216) 915 / 847; two rounds: 8 x 1024 x 1024 (288) 1073 / 1260, 3000 x 3000 (300) 3255 / 3687, 3700 x 3700
    //   (435) 5659 / 5485, 4096 x 4096 (528) 7465 / 7850; sides below 1024: 64 x 512 x 512 (640) 1387 / 1432, 200 x 256 x 500 (600) 1291 / 1381
    //   Q X: 1500 x 2000 (192) 678 / 654, 2048 x 2048 (256) 1268 / 1134, 1024 x 4608 (288) 488 / 518, 1200 x 9000 (710) 814 / 787, 2048 x 9216
    //   (1152) 2576 / 2416; sides below 1024: 40 x 512 x 512 (640) 846 / 856, 4 x 700 x 700 (144) 314 / 350
    const int T = square ? (!narrow && wide > 160 && wide <= 256 ? 128 : 64) : (wide > 160 && wide <= 256) || wide > 512 ? 128 : 64;
    bool split_any = false;
    for (int pass = 0; pass < 2; ++pass) {
      int blocks = 0;
      lv.joining = pass;
      for (int i = 0; i < n; ++i) {
        OrthoGroup &q = lv.gs.g[i];
        const bool gram = q.jobs && q.type == OL_SYM && lv.job[2 * i].l >= OB_SMALL && T == 64;
        q.aux = gram ? lo.kz[i] : 1;
        split_any |= q.aux > 1;
        q.first = blocks;
        const long units = (long)q.count * q.jobs * og_tiles(q, q.type, T) * (pass ? q.aux > 1 : q.aux);
        blocks += (int)((units + 7) / 8 * 8);
      }
      if (!blocks) break;
      // Stages hide latency as long as the blocks that a CU gets fit beside each other: 64-wide tiles with 3 (73 KB) for two blocks per CU
      // (28 x 256 x 2304 452 us, 463 with 2; 1024 x 1024 263 / 327; no more with 4 or 6 for one), else 2, three blocks (28 x 256 x 2304
      // with 3: 471; 200 x 128 x 576 456 / 507).  128-wide ones: 8 waves of 64 x 32 (2048 x 9216 2464, 4 waves of 64 x 64 2687; 3 stages 2443)
      const int rc = T == 128       ? ortho_launch<128, 32, 2, 2, 4>(ws, lv, blocks, st)
                     : blocks > 512 ? ortho_launch<64, 32, 2, 2, 2>(ws, lv, blocks, st)
                                    : ortho_launch<64, 32, 3, 2, 2>(ws, lv, blocks, st);
      if (rc) return rc;
      if (!split_any) break;
    }
  }
  LSPS_CHECK_LAUNCH("newton_schulz");
  return 0;
}

}  // namespace lsps

using namespace lsps;

extern "C" {

static bool ortho_sane(const OrthoGroup &g) {
  return g.rows > 0 && g.cols > 0 && g.count > 0 && g.rows <= 1 << 20 && g.cols <= 1 << 20 &&
         (double)og_pad(g.rows) * og_pad(g.cols) <= (double)(1 << 29) &&      // a matrix of limbs: 32-bit offsets
         (double)og_pad(g.rows) * og_pad(g.cols) * g.count <= (double)(1L << 36);
}

// this thread's plans, none made yet
static OrthoPlan *ortho_plans() {
  static thread_local OrthoPlan plan[ORTHO_CHAINS];
  for (int k = 0; k < ORTHO_CHAINS; ++k) plan[k].levels = 0;
  return plan;
}

// checks one pass; plan[k]: made for the chain lengths that it needs, kept for the call's other passes
static int ortho_check(const char *what, OrthoGroup *g, int n, const OrthoCall &c, OrthoPlan *plan, const void *ws, size_t ws_bytes) {
  LSPS_CHECK_ARG(c.steps >= 1 && c.steps <= ORTHO_STEPS, "%s: %d steps (1 to %d)", what, c.steps, ORTHO_STEPS);
  LSPS_CHECK_ARG(c.eps >= 0.f, "%s: eps %g", what, (double)c.eps);
  double blocks = 0;
  for (int i = 0; i < n; ++i) {
    LSPS_CHECK_ARG(ortho_sane(g[i]), "%s: %d matrices of %d x %d", what, g[i].count, g[i].rows, g[i].cols);
    // the finest launch: 64 x 64 tiles, two jobs or split reductions
    blocks += (double)g[i].count * ((double)og_pad(g[i].rows) / 64 * og_pad(g[i].cols) / 64 + 8) * 2;
  }
  LSPS_CHECK_ARG(blocks < (double)(1L << 23), "%s: too many matrices for one call", what);
  const OrthoLayout lo = ortho_layout(g, n, c.steps);
  for (int i = 0; i < n; ++i) {
    OrthoPlan *p = plan + lo.chain[i] - 1;
    LSPS_CHECK_ARG(p->levels || ortho_plan(p, lo.chain[i], c), "%s: the iteration with (%g, %g, %g) grows out of bounds on [0, 1]",
                   what, (double)c.a, (double)c.b, (double)c.c);
  }
  LSPS_CHECK_ARG(!((uintptr_t)ws & 15), "%s: the workspace is not 16-byte aligned", what);
  if (!ws || ws_bytes < lo.bytes) {
    set_error("%s: workspace of %zu bytes, %zu needed", what, ws_bytes, lo.bytes);
    return LSPS_E_WS;
  }
  return 0;
}

static OrthoGroup ortho_group(int count, int rows, int cols) {
  OrthoGroup g;
  memset(&g, 0, sizeof g);
  g.count = count;
  g.rows = rows;
  g.cols = cols;
  g.ptr = -1;
  return g;
}

size_t lsps_newton_schulz_workspace_bytes(int count, int rows, int cols, int steps) {
  OrthoGroup g = ortho_group(count, rows, cols);
  if (!ortho_sane(g) || steps < 1) return 0;
  return ortho_layout(&g, 1, steps).bytes;
}

int lsps_newton_schulz(const void *g, void *out, int count, int rows, int cols, int dtype, int steps, float a, float b, float c, float eps,
                       void *ws, size_t ws_bytes, void *stream) {
  (void)hipGetLastError();   // clear stale sticky errors left by other users of the runtime
  LSPS_CHECK_ARG(g && out, "newton_schulz: null pointer");
  LSPS_CHECK_ARG(dtype == LSPS_F32 || dtype == LSPS_BF16, "newton_schulz: dtype %d (LSPS_F32 or LSPS_BF16)", dtype);
  OrthoGroup grp = ortho_group(count, rows, cols);
  const OrthoCall call = {steps, a, b, c, eps, dtype == LSPS_F32 ? OM_F32 : OM_BF16, dtype == LSPS_BF16, 1.f, {0.f, 1.f, 0}};
  OrthoPlan *plan = ortho_plans();
  if (const int rc = ortho_check("newton_schulz", &grp, 1, call, plan, ws, ws_bytes)) return rc;
  return ortho_run(&grp, 1, OrthoPtr{g, out, nullptr}, nullptr, 0, call, plan, (char *)ws, (hipStream_t)stream);
}

// The next pass of a Muon step from matrix `at` on: as many as fit ORTHO_GROUPS shapes and ORTHO_MATRICES pointers, sorted into
// shapes, the longest shapes first (the long blocks of a product start first).  Returns the number of matrices taken.
struct MuonPass {
  OrthoGroup g[ORTHO_GROUPS];
  OrthoPtr ptr[ORTHO_MATRICES];
  int n, taken;
};
static void muon_pass(const LspsMuonMatrix *mats, int n, int at, float lr, float rms, MuonPass *p) {
  int shape[ORTHO_MATRICES];
  p->n = p->taken = 0;
  for (; at + p->taken < n && p->taken < ORTHO_MATRICES; ++p->taken) {
    const LspsMuonMatrix &m = mats[at + p->taken];
    int k = 0;
    while (k < p->n && (p->g[k].rows != m.rows || p->g[k].cols != m.cols)) ++k;
    if (k == p->n) {
      if (p->n == ORTHO_GROUPS) break;
      p->g[p->n] = ortho_group(0, m.rows, m.cols);
      p->g[p->n++].step = lr * rms * sqrtf((float)(m.rows > m.cols ? m.rows : m.cols));
    }
    ++p->g[k].count;
    shape[p->taken] = k;
  }
  int order[ORTHO_GROUPS], next = 0;
  for (int i = 0; i < p->n; ++i) {
    int j = i;
    for (; j > 0 && og_long(p->g[order[j - 1]]) < og_long(p->g[i]); --j) order[j] = order[j - 1];
    order[j] = i;
  }
  OrthoGroup sorted[ORTHO_GROUPS];
  for (int i = 0; i < p->n; ++i) {
    sorted[i] = p->g[order[i]];
    sorted[i].ptr = next;
    for (int k = 0; k < p->taken; ++k)
      if (shape[k] == order[i]) p->ptr[next++] = OrthoPtr{mats[at + k].g, mats[at + k].p, mats[at + k].m};
  }
  memcpy(p->g, sorted, p->n * sizeof(OrthoGroup));
}

size_t lsps_muon_workspace_bytes(const LspsMuonMatrix *mats, int n, int steps) {
  static thread_local MuonPass p;
  size_t most = 0;
  if (!mats || n < 1 || steps < 1) return 0;
  for (int i = 0; i < n; ++i)
    if (!ortho_sane(ortho_group(1, mats[i].rows, mats[i].cols))) return 0;
  for (int at = 0; at < n; at += p.taken) {
    muon_pass(mats, n, at, 0.f, 0.f, &p);
    const size_t need = ortho_layout(p.g, p.n, steps).bytes;
    if (need > most) most = need;
  }
  return most;
}

// Does memory that the step writes overlap other memory of it?  (-1: no memory to look.)
struct MuonSpan {
  uintptr_t lo, hi;
  int written;
};
static int muon_before(const void *a, const void *b) {
  const MuonSpan *x = (const MuonSpan *)a, *y = (const MuonSpan *)b;
  return x->lo < y->lo ? -1 : x->lo > y->lo;
}
static int muon_overlap(const LspsMuonMatrix *mats, int n) {
  MuonSpan few[96], *v = n <= 32 ? few : (MuonSpan *)malloc(sizeof(MuonSpan) * 3 * n);
  if (!v) return -1;
  for (int i = 0; i < n; ++i) {
    const uintptr_t size = (uintptr_t)mats[i].rows * mats[i].cols * sizeof(float);
    const uintptr_t at[3] = {(uintptr_t)mats[i].p, (uintptr_t)mats[i].m, (uintptr_t)mats[i].g};
    for (int k = 0; k < 3; ++k) v[3 * i + k] = MuonSpan{at[k], at[k] + size, k < 2};
  }
  qsort(v, 3 * (size_t)n, sizeof *v, muon_before);
  uintptr_t end = 0, end_written = 0;
  int found = 0;
  for (int i = 0; i < 3 * n && !found; ++i) {
    found = v[i].lo < end_written || (v[i].written && v[i].lo < end);
    if (v[i].hi > end) end = v[i].hi;
    if (v[i].written && v[i].hi > end_written) end_written = v[i].hi;
  }
  if (v != few) free(v);
  return found;
}

int lsps_muon_step(const LspsMuonMatrix *mats, int n, float lr, float momentum, int nesterov, float weight_decay, float rms, float grad_scale,
                   int steps, float a, float b, float c, float eps, void *ws, size_t ws_bytes, void *stream) {
  static thread_local MuonPass p;
  (void)hipGetLastError();   // clear stale sticky errors left by other users of the runtime
  LSPS_CHECK_ARG(mats && n > 0, "muon_step: no matrices");
  LSPS_CHECK_ARG(isfinite(lr) && isfinite(weight_decay) && isfinite(rms) && isfinite(grad_scale) && momentum >= 0.f && momentum < 1.f,
                 "muon_step: lr %g, momentum %g, weight decay %g, rms %g, gradient scale %g", (double)lr, (double)momentum,
                 (double)weight_decay, (double)rms, (double)grad_scale);
  for (int i = 0; i < n; ++i) {
    LSPS_CHECK_ARG(mats[i].p && mats[i].g && mats[i].m, "muon_step: null pointer in matrix %d", i);
    LSPS_CHECK_ARG(ortho_sane(ortho_group(1, mats[i].rows, mats[i].cols)), "muon_step: matrix %d of %d x %d", i, mats[i].rows, mats[i].cols);
  }
  const int overlap = muon_overlap(mats, n);
  LSPS_CHECK_ARG(overlap == 0, "muon_step: %s", overlap < 0 ? "out of host memory" : "weights, momenta or gradients overlap");
  const OrthoCall call = {steps, a, b, c, eps, OM_MUON, false, 1.f - lr * weight_decay, {momentum, grad_scale, nesterov != 0}};
  OrthoPlan *plan = ortho_plans();
  for (int at = 0; at < n; at += p.taken) {
    muon_pass(mats, n, at, lr, rms, &p);
    if (const int rc = ortho_check("muon_step", p.g, p.n, call, plan, ws, ws_bytes)) return rc;
  }
  for (int at = 0; at < n; at += p.taken) {
    muon_pass(mats, n, at, lr, rms, &p);
    if (const int rc = ortho_run(p.g, p.n, OrthoPtr{nullptr, nullptr, nullptr}, p.ptr, p.taken, call, plan, (char *)ws, (hipStream_t)stream)) return rc;
  }
  return 0;
}

}  // extern "C"
