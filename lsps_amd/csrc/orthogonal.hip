// Orthogonalised updates: Newton-Schulz iteration on stacks of matrices and the whole Muon step over the matrices of a net.
//
//   X0 = G / (|G|_F + eps)      X <- a X + (b A + c A^2) X,  A = X X^T   (`steps` times, on the side where X is wide)
//   Muon: m <- mu m + g,  G = g + mu m (nesterov) or m,  p <- p (1 - lr wd) - lr rms sqrt(max(rows, cols)) X
//
// Work on the short side.  With A = X X^T (M x M, M <= N) n steps are X <- (a^n I + R) X, where S = b A + c A^2 of the current
// Gram matrix and, from step to step, R <- a R + a^n S + R S and A <- A P^2 with P = a I + S: products of M x M matrices only,
// every one of them symmetric (they are polynomials of one symmetric matrix), so only the tiles on and above the diagonal are
// computed.  Two products with the long side (A, and the last one) per restart instead of two per step: 3 M^2 N + O(M^3)
// operations instead of 15 M^2 N for five steps.  A is formed anew from X after at most ORTHO_CHAIN steps: an error d of A is
// one of |b| / a (a^2)^k d, relatively, in the directions of small singular values after k more steps, so three steps cost
// what the plain iteration in f32 costs (measured: no larger error than it) and five do not.
//
// Operands.  Every matrix lives in the workspace as two f16 limbs, v s = hi + lo with a power of two s chosen from a bound of
// the matrix' entries (22 significand bits; the entries are bounded by the spectral norm, which is a polynomial of values in
// [0, 1], see ortho_bounds), and a product is three v_mfma_f32_32x32x16_f16 (hi hi + hi lo + lo hi, f32 accumulation; the
// dropped lo lo is below 2^-22 of the product): f32-class results at a third of the f16 rate, 5 x the f32 MFMA rate.
// Layout: [row][k / 8][hi 8 | lo 8], rows and columns padded with zeros to multiples of 64: a k-chunk of 32 is one 128-byte line
// of a row, copied to LDS by 16-byte LDS-DMA whose source addresses carry the bank swizzle (unit ^ (row & 7)).
// All matrices of a call go through one launch per product (the blocks find their matrix in a table in the workspace).
#include <math.h>
#include <string.h>

#include "common.h"

namespace lsps {

typedef _Float16 og_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 og_h4 __attribute__((ext_vector_type(4)));
typedef float og_f16v __attribute__((ext_vector_type(16)));
typedef float og_f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short og_u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef __attribute__((address_space(3))) void *og_lds;
typedef const __attribute__((address_space(1))) void *og_glb;

#define ORTHO_GROUPS 64        // groups of equal matrices per pass (the blocks search them with one ballot)
#define ORTHO_CHAIN 3          // steps between two Gram matrices of the long side
#define ORTHO_NORM_BLOCK 16384 // elements per block of the norm pass
#define ORTHO_TABLE_PART 32    // groups per table launch (passed by value: nothing on the host has to outlive the call)
enum { OK_NORM, OK_SPLIT, OK_SYM64, OK_SYM128, OK_RECT64, OK_RECT128, ORTHO_KINDS };
enum { OB_A, OB_S, OB_T, OB_R0, OB_R1, OB_SMALL, OB_X0 = OB_SMALL, OB_X1, OB_XT0, OB_XT1, OB_NONE };
enum { OM_F32, OM_BF16, OM_MUON };

struct OrthoGroup {
  const void *g;       // count matrices of rows x cols, contiguous
  void *out;           // OM_MUON: the weights
  float *m;            // OM_MUON: the momentum
  unsigned x_off, s_off;          // workspace offsets in 256-byte units: long-side matrices, M x M matrices
  int norm_off;                   // first of the matrices' partial sums of squares
  int rows, cols, count;
  float step;                     // OM_MUON: lr rms sqrt(max(rows, cols))
  int first[ORTHO_KINDS];         // blocks in front of this group, for each way of cutting it into blocks
};

struct OrthoTable {
  OrthoGroup g[ORTHO_GROUPS];
  int first[ORTHO_KINDS][ORTHO_GROUPS];
};

struct OrthoPart {
  OrthoGroup g[ORTHO_TABLE_PART];
};

__host__ __device__ static inline int og_pad(int n) { return (n + 63) & ~63; }
__host__ __device__ static inline int og_short(const OrthoGroup &g) { return g.rows < g.cols ? g.rows : g.cols; }
__host__ __device__ static inline int og_long(const OrthoGroup &g) { return g.rows < g.cols ? g.cols : g.rows; }
__host__ __device__ static inline int og_norm_blocks(const OrthoGroup &g) {
  return (int)(((long)g.rows * g.cols + ORTHO_NORM_BLOCK - 1) / ORTHO_NORM_BLOCK);
}
// blocks per matrix
__host__ __device__ static inline int og_blocks(const OrthoGroup &g, int kind) {
  const int M = og_pad(og_short(g)), N = og_pad(og_long(g));
  switch (kind) {
    case OK_NORM: return og_norm_blocks(g);
    case OK_SPLIT: return (M / 64) * (N / 64);
    case OK_SYM64: return (M / 64) * (M / 64 + 1) / 2;
    case OK_SYM128: return ((M + 127) / 128) * ((M + 127) / 128 + 1) / 2;
    case OK_RECT64: return (M / 64) * (N / 64);
    default: return ((M + 127) / 128) * ((N + 127) / 128);
  }
}

__global__ void ortho_table_kernel(OrthoPart part, OrthoTable *t, int base, int n) {
  const int i = threadIdx.x;
  if (i >= n) return;
  t->g[base + i] = part.g[i];
  for (int k = 0; k < ORTHO_KINDS; ++k) t->first[k][base + i] = part.g[i].first[k];
}

struct OrthoAt {
  int grp, mat, tile;
};
// group, matrix and tile of block b: the group is the last one whose first block is not behind b
__device__ __forceinline__ OrthoAt ortho_at(const OrthoTable *t, int n, int kind, int b) {
  const int lane = threadIdx.x & 63;
  const bool le = lane < n && t->first[kind][lane] <= b;
  OrthoAt at;
  at.grp = __builtin_amdgcn_readfirstlane(63 - __clzll(__ballot(le)));
  const int per = og_blocks(t->g[at.grp], kind), rel = b - t->g[at.grp].first[kind];
  at.mat = rel / per;
  at.tile = rel - at.mat * per;
  return at;
}

__device__ __forceinline__ char *ortho_buffer(char *ws, const OrthoGroup &g, int id, int mat) {
  const long M = og_pad(og_short(g)), N = og_pad(og_long(g));
  if (id < OB_SMALL) return ws + (size_t)g.s_off * 256 + ((long)id * g.count + mat) * M * M * 4;
  const int which = id == OB_X0 ? 0 : id == OB_XT0 ? 1 : id == OB_X1 ? 2 : 3;
  return ws + (size_t)g.x_off * 256 + ((long)which * g.count + mat) * M * N * 4;
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
__global__ __launch_bounds__(256) void ortho_norm_kernel(const OrthoTable *__restrict__ t, int n, double *__restrict__ sums,
                                                         OrthoMomentum mo) {
  __shared__ double red[4];
  const OrthoAt at = ortho_at(t, n, OK_NORM, blockIdx.x);
  const OrthoGroup &g = t->g[at.grp];
  const long size = (long)g.rows * g.cols, lo = (long)at.tile * ORTHO_NORM_BLOCK;
  const T *src = (const T *)g.g + at.mat * size;
  float *m = MUON ? g.m + at.mat * size : nullptr;
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
  if (threadIdx.x == 0) sums[g.norm_off + at.mat * og_norm_blocks(g) + at.tile] = red[0] + red[1] + red[2] + red[3];
}

__device__ __forceinline__ void og_split(float v, _Float16 &hi, _Float16 &lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// X0 as limbs, both ways round: X (short side in rows) and its transpose.  One 64 x 64 tile of G per block, through LDS.
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_split_kernel(const OrthoTable *__restrict__ t, int n, char *__restrict__ ws,
                                                          const double *__restrict__ sums, OrthoMomentum mo, float eps, float scale) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const OrthoAt at = ortho_at(t, n, OK_SPLIT, blockIdx.x);
  const OrthoGroup &g = t->g[at.grp];
  const int nb = og_norm_blocks(g);
  const double *part = sums + g.norm_off + (long)at.mat * nb;
  double s = 0.;
  for (int i = threadIdx.x; i < nb; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  const int tc = og_pad(g.cols) / 64;
  const int r0 = at.tile / tc * 64, c0 = (at.tile - at.tile / tc * tc) * 64;
  const long size = (long)g.rows * g.cols;
  const T *src = (const T *)g.g + at.mat * size;
  const float *m = MUON ? g.m + at.mat * size : nullptr;
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
  // one division of the 64-bit norm; the f32 quotient below is the rounding X / (|G| + eps) has in f32 arithmetic
  const float norm = (float)(sqrt(red[0] + red[1] + red[2] + red[3]) + (double)eps);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[(threadIdx.x >> 4) + k * 16][(threadIdx.x & 15) * 4 + e] = v[k][e] / norm * scale;
  __syncthreads();
  const bool tall = g.rows > g.cols;
  char *d0 = ortho_buffer(ws, g, tall ? OB_XT0 : OB_X0, at.mat), *d1 = ortho_buffer(ws, g, tall ? OB_X0 : OB_XT0, at.mat);
  const long p0 = (long)og_pad(g.cols) * 4, p1 = (long)og_pad(g.rows) * 4;     // row pitches in bytes
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int u = threadIdx.x + k * 256, a = u >> 3, q = u & 7;
    og_h8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 x, y;
      og_split(tile[a][q * 8 + e], x, y);
      h[e] = x;
      l[e] = y;
    }
    og_h8 *dst = reinterpret_cast<og_h8 *>(d0 + (r0 + a) * p0 + (c0 / 8 + q) * 32);
    dst[0] = h;
    dst[1] = l;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int u = threadIdx.x + k * 256, a = u >> 3, q = u & 7;
    og_h8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 x, y;
      og_split(tile[q * 8 + e][a], x, y);
      h[e] = x;
      l[e] = y;
    }
    og_h8 *dst = reinterpret_cast<og_h8 *>(d1 + (c0 + a) * p1 + (r0 / 8 + q) * 32);
    dst[0] = h;
    dst[1] = l;
  }
}

// out = k0 (L R^T) + k1 E1 + k2 E2 on stored (scaled) values: the scales are folded into the factors
struct OrthoJob {
  int l, r, e1, e2, out, mirror;
  float k0, k1, k2;
};
struct OrthoLevel {
  OrthoJob job[2];
  int blocks;              // per job
  int mode;                // of the last level: OM_*
  float decay;             // 1 - lr wd
};

enum { OL_SYM, OL_RECT, OL_LAST };

// One product per block: a T x T tile of L R^T, both with the reduction along their rows.  4 waves, 2 x 2, each (T/2) x (T/2)
// in 32x32 MFMA tiles; the MFMA's row index is the tile's COLUMN, so a lane holds one row of the result and runs of 4 columns
// (8-byte stores per limb).  LDS: two stages of a KC-deep chunk of both operands, filled by LDS-DMA while the other one is
// multiplied; one barrier per chunk.
//   OL_SYM : L R^T symmetric; tiles on and above the diagonal, the mirrored tile is stored from an LDS transpose
//   OL_RECT: X of the next chain, stored both ways round
//   OL_LAST: the result in the caller's layout and type, or the weight update
template <int T, int KC, int LEVEL>
__global__ __launch_bounds__(256) void ortho_product_kernel(const OrthoTable *__restrict__ t, int n, char *__restrict__ ws, OrthoLevel lv) {
  constexpr int UPR = KC / 4, STAGE = T * KC * 4, PIECES = T * UPR / 256, RPP = 64 / UPR, WT = T / 2, FR = WT / 32, TP = 144;
  constexpr int KIND = LEVEL == OL_SYM ? (T == 64 ? OK_SYM64 : OK_SYM128) : (T == 64 ? OK_RECT64 : OK_RECT128);
  static_assert(4 * STAGE >= 4 * 32 * TP, "the transpose of the epilogue reuses the stages");
  extern __shared__ __align__(1024) char smem[];
  const int second = (int)blockIdx.x >= lv.blocks;
  const OrthoJob job = lv.job[second];
  const OrthoAt at = ortho_at(t, n, KIND, blockIdx.x - second * lv.blocks);
  const OrthoGroup g = t->g[at.grp];
  const int M = og_pad(og_short(g)), N = og_pad(og_long(g));
  int bi, bj;
  if (LEVEL == OL_SYM) {
    bj = (int)((sqrtf(8.f * at.tile + 1.f) - 1.f) * 0.5f);
    while ((bj + 1) * (bj + 2) / 2 <= at.tile) ++bj;
    while (bj * (bj + 1) / 2 > at.tile) --bj;
    bi = at.tile - bj * (bj + 1) / 2;
  } else {
    const int tn = (N + T - 1) / T;
    bi = at.tile / tn;
    bj = at.tile - bi * tn;
  }
  const int cols = LEVEL == OL_SYM ? M : N;                      // of the result; rows: M
  const int K = job.l >= OB_SMALL ? N : M;
  const long pitch = (long)K * 4;
  const char *L = ortho_buffer(ws, g, job.l, at.mat), *R = ortho_buffer(ws, g, job.r, at.mat);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const char *lp[PIECES], *rp[PIECES];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int row = (wave + 4 * p) * RPP + lane / UPR, unit = (lane % UPR) ^ (row & 7);
    const int li = bi * T + row < M ? bi * T + row : M - 1, rj = bj * T + row < cols ? bj * T + row : cols - 1;
    lp[p] = L + li * pitch + unit * 16;
    rp[p] = R + rj * pitch + unit * 16;
  }
  auto stage = [&](int buf) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      __builtin_amdgcn_global_load_lds((og_glb)lp[p], (og_lds)(smem + buf * 2 * STAGE + (wave + 4 * p) * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((og_glb)rp[p], (og_lds)(smem + buf * 2 * STAGE + STAGE + (wave + 4 * p) * 1024), 16, 0, 0);
      lp[p] += KC * 4;
      rp[p] += KC * 4;
    }
  };
  const int wi = wave >> 1, wj = wave & 1, l31 = lane & 31, lh = lane >> 5;
  og_f16v acc[FR][FR];
#pragma unroll
  for (int i = 0; i < FR; ++i)
#pragma unroll
    for (int j = 0; j < FR; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  stage(0);
  const int chunks = K / KC;
  for (int c = 0; c < chunks; ++c) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (c + 1 < chunks) stage((c + 1) & 1);
    const char *sl = smem + (c & 1) * 2 * STAGE, *sr = sl + STAGE;
#pragma unroll
    for (int ks = 0; ks < KC / 16; ++ks) {
      const int kg = ks * 2 + lh;
      og_h8 lf[FR][2], rf[FR][2];
#pragma unroll
      for (int f = 0; f < FR; ++f)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int li = wi * WT + f * 32 + l31, rj = wj * WT + f * 32 + l31;
          lf[f][q] = *reinterpret_cast<const og_h8 *>(sl + li * (UPR * 16) + (((kg * 2 + q) ^ (li & 7)) * 16));
          rf[f][q] = *reinterpret_cast<const og_h8 *>(sr + rj * (UPR * 16) + (((kg * 2 + q) ^ (rj & 7)) * 16));
        }
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FR; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rf[j][0], lf[i][1], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rf[j][1], lf[i][0], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rf[j][0], lf[i][0], acc[i][j], 0, 0, 0);
        }
    }
  }
  const char *e1 = job.e1 == OB_NONE ? nullptr : ortho_buffer(ws, g, job.e1, at.mat);
  const char *e2 = job.e2 == OB_NONE ? nullptr : ortho_buffer(ws, g, job.e2, at.mat);
  const long opitch = (long)cols * 4;
  auto stored = [&](const char *e, int i, int j, float (&v)[4]) {        // 4 stored values of row i from column j on
    const og_h4 *p = reinterpret_cast<const og_h4 *>(e + i * opitch + (j >> 3) * 32 + (j & 7) * 2);
    const og_h4 h = p[0], l = p[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (float)h[k] + (float)l[k];
  };
  if (LEVEL != OL_LAST) __syncthreads();                                 // the stages become the waves' transpose buffers
  char *tp = smem + wave * 32 * TP;
#pragma unroll
  for (int fi = 0; fi < FR; ++fi)
#pragma unroll
    for (int fj = 0; fj < FR; ++fj) {
      const int i0 = bi * T + wi * WT + fi * 32, j0 = bj * T + wj * WT + fj * 32, i = i0 + l31;
      if (i0 >= M || j0 >= cols) continue;                               // (T = 128 on an odd number of 64-row halves)
      const bool mirrored = LEVEL == OL_RECT || (LEVEL == OL_SYM && bi != bj);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = j0 + q * 8 + lh * 4;
        float v[4], x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = job.k0 * acc[fi][fj][q * 4 + k];
        if (e1) {
          stored(e1, i, j, x);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = fmaf(job.k1, x[k], v[k]);
        }
        if (e2) {
          stored(e2, i, j, x);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = fmaf(job.k2, x[k], v[k]);
        }
        if constexpr (LEVEL != OL_LAST) {
          og_h4 h, l;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            _Float16 a, b;
            og_split(v[k], a, b);
            h[k] = a;
            l[k] = b;
          }
          og_h4 *p = reinterpret_cast<og_h4 *>(ortho_buffer(ws, g, job.out, at.mat) + i * opitch + (j >> 3) * 32 + (j & 7) * 2);
          p[0] = h;
          p[2] = l;
          if (mirrored) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              char *d = tp + (q * 8 + lh * 4 + k) * TP + l31 * 2;
              *reinterpret_cast<_Float16 *>(d) = h[k];
              *reinterpret_cast<_Float16 *>(d + 64) = l[k];
            }
          }
        } else {
          const int m = og_short(g), nn = og_long(g);
          const bool tall = g.rows > g.cols;
          const long size = (long)g.rows * g.cols;
          if (i < m) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (j + k < nn) {
                const long o = at.mat * size + (tall ? (long)(j + k) * m + i : (long)i * nn + j + k);
                if (lv.mode == OM_F32) ((float *)g.out)[o] = v[k];
                else if (lv.mode == OM_BF16) ((__bf16 *)g.out)[o] = (__bf16)v[k];       // the one rounding of the result
                else ((float *)g.out)[o] = fmaf(-g.step, v[k], ((float *)g.out)[o] * lv.decay);
              }
          }
        }
      }
      if constexpr (LEVEL != OL_LAST) {
        if (mirrored) {
          char *dst = ortho_buffer(ws, g, job.mirror, at.mat);
          const long mp = (long)M * 4;                                   // the mirrored matrix has the result's rows as columns
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int u = lane + s * 64, jr = u >> 3, ig = (u & 7) >> 1, limb = u & 1;
            const og_h8 x = *reinterpret_cast<const og_h8 *>(tp + jr * TP + limb * 64 + ig * 16);
            *reinterpret_cast<og_h8 *>(dst + (j0 + jr) * mp + (i0 / 8 + ig) * 32 + limb * 16) = x;
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
      }
    }
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

// Bounds of the matrices' spectral norms (hence of their entries) along the iteration: every one of them is a polynomial of
// X0's singular values, which lie in [0, 1].  bx: X; ba, bs, bt, br: A, S, T = A P, R of one chain.  False if the coefficients
// let the iteration grow out of hand (or are not finite).
struct OrthoScale {
  float x[ORTHO_CHAIN + 1], a[ORTHO_CHAIN], s[ORTHO_CHAIN], t[ORTHO_CHAIN], r[ORTHO_CHAIN];
};
#define ORTHO_SAMPLES 1025
#define ORTHO_GROWTH 1e4
static bool ortho_scale_of(double bound, float *scale) {
  if (!(bound <= ORTHO_GROWTH)) return false;
  if (bound < 1e-6) bound = 1e-6;
  *scale = (float)exp2(floor(log2(16384. / bound)));     // a factor of 4 below the largest f16 for rounding and between the samples
  return true;
}
// one chain of n steps from the singular values sv (advanced to those behind the chain)
static bool ortho_bounds(double *sv, int n, const OrthoCall &c, OrthoScale *o) {
  double r[ORTHO_SAMPLES], lam[ORTHO_SAMPLES], most = 0.;
  for (int i = 0; i < ORTHO_SAMPLES; ++i) {
    lam[i] = sv[i] * sv[i];
    most = fmax(most, fabs(sv[i]));
    if (!isfinite(sv[i])) return false;
  }
  if (!ortho_scale_of(most, &o->x[0])) return false;
  double an = 1.;
  for (int k = 0; k < n; ++k) {
    double ma = 0., ms = 0., mt = 0., mr = 0.;
    for (int i = 0; i < ORTHO_SAMPLES; ++i) {
      const double A = lam[i], S = c.b * A + c.c * A * A, P = c.a + S;
      r[i] = k ? c.a * r[i] + an * S + r[i] * S : S;
      lam[i] = A * P * P;
      if (!isfinite(lam[i]) || !isfinite(r[i])) return false;
      ma = fmax(ma, fabs(A));
      ms = fmax(ms, fabs(S));
      mt = fmax(mt, fabs(A * P));
      mr = fmax(mr, fabs(r[i]));
    }
    if (!ortho_scale_of(ma, &o->a[k]) || !ortho_scale_of(ms, &o->s[k]) || !ortho_scale_of(mt, &o->t[k]) || !ortho_scale_of(mr, &o->r[k]))
      return false;
    an *= c.a;
  }
  most = 0.;
  for (int i = 0; i < ORTHO_SAMPLES; ++i) {
    sv[i] *= an + r[i];
    if (!isfinite(sv[i])) return false;
    most = fmax(most, fabs(sv[i]));
  }
  return ortho_scale_of(most, &o->x[1]);
}

static void ortho_samples(double *sv) {
  for (int i = 0; i < ORTHO_SAMPLES; ++i) sv[i] = 1.00001 * pow((double)i / (ORTHO_SAMPLES - 1), 3.);    // denser towards 0
}

static bool ortho_converges(const OrthoCall &c) {
  double sv[ORTHO_SAMPLES];
  OrthoScale sc;
  ortho_samples(sv);
  for (int left = c.steps; left > 0;) {
    const int n = left < ORTHO_CHAIN ? left : ORTHO_CHAIN;
    if (!ortho_bounds(sv, n, c, &sc)) return false;
    left -= n;
  }
  return true;
}

struct OrthoLayout {
  size_t sums, data, bytes;
  int total[ORTHO_KINDS];
};

// workspace: table | partial sums of squares | per group X, X^T (twice when the chain restarts) | per group the M x M matrices
static OrthoLayout ortho_layout(OrthoGroup *g, int n, int steps) {
  OrthoLayout lo;
  memset(&lo, 0, sizeof lo);
  lo.sums = align_up(sizeof(OrthoTable), 256);
  long parts = 0;
  for (int i = 0; i < n; ++i) {
    for (int k = 0; k < ORTHO_KINDS; ++k) {
      g[i].first[k] = lo.total[k];
      lo.total[k] += g[i].count * og_blocks(g[i], k);
    }
    g[i].norm_off = (int)parts;
    parts += (long)g[i].count * og_norm_blocks(g[i]);
  }
  size_t at = lo.sums + align_up(parts * sizeof(double), 256);
  for (int i = 0; i < n; ++i) {
    const size_t M = og_pad(og_short(g[i])), N = og_pad(og_long(g[i]));
    g[i].x_off = (unsigned)(at / 256);
    at += M * N * 4 * g[i].count * (steps > ORTHO_CHAIN ? 4 : 2);        // multiples of 64 x 64 x 4 bytes
    g[i].s_off = (unsigned)(at / 256);
    at += M * M * 4 * g[i].count * OB_SMALL;
  }
  lo.bytes = at;
  return lo;
}

template <int T, int KC, int LEVEL>
static int ortho_launch(const OrthoTable *t, int n, char *ws, const OrthoLevel &lv, int jobs, hipStream_t st) {
  const int lds = 4 * T * KC * 4;
  if (const int rc = lds_optin(reinterpret_cast<const void *>(&ortho_product_kernel<T, KC, LEVEL>), lds, "ortho_product_kernel")) return rc;
  hipLaunchKernelGGL((ortho_product_kernel<T, KC, LEVEL>), dim3(lv.blocks * jobs), dim3(256), lds, st, t, n, ws, lv);
  return 0;
}

// 128 x 128 tiles read each operand half as often but need enough of them to fill the 256 CUs
template <int LEVEL>
static int ortho_product(const OrthoTable *t, int n, char *ws, const OrthoLayout &lo, OrthoLevel lv, int jobs, hipStream_t st) {
  const int k128 = LEVEL == OL_SYM ? OK_SYM128 : OK_RECT128, k64 = LEVEL == OL_SYM ? OK_SYM64 : OK_RECT64;
  if (lo.total[k128] * jobs >= 256) {
    lv.blocks = lo.total[k128];
    return ortho_launch<128, 32, LEVEL>(t, n, ws, lv, jobs, st);
  }
  lv.blocks = lo.total[k64];
  return ortho_launch<64, 64, LEVEL>(t, n, ws, lv, jobs, st);
}

// one pass over at most ORTHO_GROUPS groups
static int ortho_run(OrthoGroup *g, int n, const OrthoCall &c, char *ws, hipStream_t st) {
  const OrthoLayout lo = ortho_layout(g, n, c.steps);
  OrthoTable *table = (OrthoTable *)ws;
  double *sums = (double *)(ws + lo.sums);
  for (int i = 0; i < n; i += ORTHO_TABLE_PART) {
    OrthoPart part;
    const int k = n - i < ORTHO_TABLE_PART ? n - i : ORTHO_TABLE_PART;
    memcpy(part.g, g + i, k * sizeof(OrthoGroup));
    hipLaunchKernelGGL(ortho_table_kernel, dim3(1), dim3(64), 0, st, part, table, i, k);
  }
  double sv[ORTHO_SAMPLES];
  OrthoScale sc;
  ortho_samples(sv);
  int left = c.steps, set = 0;
  int chain = left < ORTHO_CHAIN ? left : ORTHO_CHAIN;
  LSPS_CHECK_ARG(ortho_bounds(sv, chain, c, &sc), "newton_schulz: coefficients");
  if (c.mode == OM_MUON) {
    hipLaunchKernelGGL((ortho_norm_kernel<float, true>), dim3(lo.total[OK_NORM]), dim3(256), 0, st, table, n, sums, c.mo);
    hipLaunchKernelGGL((ortho_split_kernel<float, true>), dim3(lo.total[OK_SPLIT]), dim3(256), 0, st, table, n, ws, sums, c.mo, c.eps, sc.x[0]);
  } else if (!c.bf16) {
    hipLaunchKernelGGL((ortho_norm_kernel<float, false>), dim3(lo.total[OK_NORM]), dim3(256), 0, st, table, n, sums, c.mo);
    hipLaunchKernelGGL((ortho_split_kernel<float, false>), dim3(lo.total[OK_SPLIT]), dim3(256), 0, st, table, n, ws, sums, c.mo, c.eps, sc.x[0]);
  } else {
    hipLaunchKernelGGL((ortho_norm_kernel<__bf16, false>), dim3(lo.total[OK_NORM]), dim3(256), 0, st, table, n, sums, c.mo);
    hipLaunchKernelGGL((ortho_split_kernel<__bf16, false>), dim3(lo.total[OK_SPLIT]), dim3(256), 0, st, table, n, ws, sums, c.mo, c.eps, sc.x[0]);
  }
  while (left > 0) {
    const OrthoJob none = {OB_A, OB_A, OB_NONE, OB_NONE, OB_A, OB_A, 0.f, 0.f, 0.f};
    OrthoLevel lv = {{none, none}, 0, c.mode, c.decay};
    const int x = set ? OB_X1 : OB_X0, xt = set ? OB_XT1 : OB_XT0;
    lv.job[0] = OrthoJob{x, x, OB_NONE, OB_NONE, OB_A, OB_A, sc.a[0] / (sc.x[0] * sc.x[0]), 0.f, 0.f};
    if (const int rc = ortho_product<OL_SYM>(table, n, ws, lo, lv, 1, st)) return rc;
    int r = OB_R0;                                                         // R of the first step is its S
    float rs = sc.s[0];                                                    // its scale
    float an = c.a;                                                        // a^k
    for (int k = 0; k < chain; ++k) {
      const bool more = k + 1 < chain;
      const float sa = sc.a[k], ss = sc.s[k];
      const int s = k ? OB_S : OB_R0;
      // S = b A + c A A
      lv.job[0] = OrthoJob{OB_A, OB_A, OB_A, OB_NONE, s, s, c.c * ss / (sa * sa), c.b * ss / sa, 0.f};
      if (const int rc = ortho_product<OL_SYM>(table, n, ws, lo, lv, 1, st)) return rc;
      int jobs = 0;
      if (more)                                                            // T = a A + A S
        lv.job[jobs++] = OrthoJob{OB_A, s, OB_A, OB_NONE, OB_T, OB_T, sc.t[k] / (sa * ss), c.a * sc.t[k] / sa, 0.f};
      if (k) {                                                             // R = a R + a^k S + R S
        const int to = r == OB_R0 ? OB_R1 : OB_R0;
        lv.job[jobs++] = OrthoJob{r, s, r, s, to, to, sc.r[k] / (rs * ss), c.a * sc.r[k] / rs, an * sc.r[k] / ss};
        r = to;
        rs = sc.r[k];
        an *= c.a;
      }
      if (jobs)
        if (const int rc = ortho_product<OL_SYM>(table, n, ws, lo, lv, jobs, st)) return rc;
      if (!more) break;
      // A = a T + T S
      lv.job[0] = OrthoJob{OB_T, s, OB_T, OB_NONE, OB_A, OB_A, sc.a[k + 1] / (sc.t[k] * ss), c.a * sc.a[k + 1] / sc.t[k], 0.f};
      if (const int rc = ortho_product<OL_SYM>(table, n, ws, lo, lv, 1, st)) return rc;
    }
    left -= chain;
    const float sx = sc.x[0], sx1 = sc.x[1];
    if (left > 0) {                                                        // X = a^n X + R X, both ways round
      lv.job[0] = OrthoJob{r, xt, x, OB_NONE, set ? OB_X0 : OB_X1, set ? OB_XT0 : OB_XT1, sx1 / (rs * sx), an * sx1 / sx, 0.f};
      if (const int rc = ortho_product<OL_RECT>(table, n, ws, lo, lv, 1, st)) return rc;
      set ^= 1;
      chain = left < ORTHO_CHAIN ? left : ORTHO_CHAIN;
      LSPS_CHECK_ARG(ortho_bounds(sv, chain, c, &sc), "newton_schulz: coefficients");
    } else {
      lv.job[0] = OrthoJob{r, xt, x, OB_NONE, OB_NONE, OB_NONE, 1.f / (rs * sx), an / sx, 0.f};
      if (const int rc = ortho_product<OL_LAST>(table, n, ws, lo, lv, 1, st)) return rc;
    }
  }
  LSPS_CHECK_LAUNCH("newton_schulz");
  return 0;
}

}  // namespace lsps

using namespace lsps;

extern "C" {

static int ortho_check(const char *what, OrthoGroup *g, int n, const OrthoCall &c, const void *ws, size_t ws_bytes) {
  LSPS_CHECK_ARG(c.steps >= 1 && c.steps <= 64, "%s: %d steps (1 to 64)", what, c.steps);
  LSPS_CHECK_ARG(c.eps >= 0.f, "%s: eps %g", what, (double)c.eps);
  LSPS_CHECK_ARG(ortho_converges(c), "%s: the iteration with (%g, %g, %g) leaves the range of its 16-bit limbs on [0, 1]", what, (double)c.a,
                 (double)c.b, (double)c.c);
  long blocks[ORTHO_KINDS] = {0};
  for (int i = 0; i < n; ++i) {
    LSPS_CHECK_ARG(g[i].rows > 0 && g[i].cols > 0 && g[i].count > 0 && g[i].rows <= 1 << 20 && g[i].cols <= 1 << 20,
                   "%s: %d matrices of %d x %d", what, g[i].count, g[i].rows, g[i].cols);
    LSPS_CHECK_ARG((long)og_pad(g[i].rows) * og_pad(g[i].cols) <= 1L << 34, "%s: a matrix of %d x %d", what, g[i].rows, g[i].cols);
    for (int k = 0; k < ORTHO_KINDS; ++k) {
      blocks[k] += (long)g[i].count * og_blocks(g[i], k);
      LSPS_CHECK_ARG(blocks[k] < 1L << 22, "%s: too many matrices for one call", what);
    }
  }
  const size_t need = ortho_layout(g, n, c.steps).bytes;
  LSPS_CHECK_ARG(!((uintptr_t)ws & 15), "%s: the workspace is not 16-byte aligned", what);
  if (!ws || ws_bytes < need) {
    set_error("%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
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
  return g;
}

static bool ortho_sane(const OrthoGroup &g) {
  return g.rows > 0 && g.cols > 0 && g.count > 0 && g.rows <= 1 << 20 && g.cols <= 1 << 20 &&
         (double)og_pad(g.rows) * og_pad(g.cols) * g.count <= 1e12;
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
  grp.g = g;
  grp.out = out;
  const OrthoCall call = {steps, a, b, c, eps, dtype == LSPS_F32 ? OM_F32 : OM_BF16, dtype == LSPS_BF16, 1.f, {0.f, 1.f, 0}};
  if (const int rc = ortho_check("newton_schulz", &grp, 1, call, ws, ws_bytes)) return rc;
  return ortho_run(&grp, 1, call, (char *)ws, (hipStream_t)stream);
}

// the matrices of one pass: the largest of the call first, so that the long blocks of a product start first
static int muon_pass(const LspsMuonMatrix *mats, int n, int at, float lr, float rms, OrthoGroup *g) {
  const int k = n - at < ORTHO_GROUPS ? n - at : ORTHO_GROUPS;
  for (int i = 0; i < k; ++i) {
    const LspsMuonMatrix &m = mats[at + i];
    OrthoGroup q = ortho_group(1, m.rows, m.cols);
    q.g = m.g;
    q.out = m.p;
    q.m = m.m;
    q.step = lr * rms * sqrtf((float)(m.rows > m.cols ? m.rows : m.cols));
    int j = i;
    for (; j > 0 && og_long(g[j - 1]) < og_long(q); --j) g[j] = g[j - 1];
    g[j] = q;
  }
  return k;
}

size_t lsps_muon_workspace_bytes(const LspsMuonMatrix *mats, int n, int steps) {
  size_t most = 0;
  if (!mats || n < 1 || steps < 1) return 0;
  for (int i = 0; i < n; ++i)
    if (!ortho_sane(ortho_group(1, mats[i].rows, mats[i].cols))) return 0;
  for (int at = 0; at < n; at += ORTHO_GROUPS) {
    OrthoGroup g[ORTHO_GROUPS];
    const size_t need = ortho_layout(g, muon_pass(mats, n, at, 0.f, 0.f, g), steps).bytes;
    if (need > most) most = need;
  }
  return most;
}

int lsps_muon_step(const LspsMuonMatrix *mats, int n, float lr, float momentum, int nesterov, float weight_decay, float rms, float grad_scale,
                   int steps, float a, float b, float c, float eps, void *ws, size_t ws_bytes, void *stream) {
  (void)hipGetLastError();   // clear stale sticky errors left by other users of the runtime
  LSPS_CHECK_ARG(mats && n > 0, "muon_step: no matrices");
  LSPS_CHECK_ARG(isfinite(lr) && isfinite(weight_decay) && isfinite(rms) && isfinite(grad_scale) && momentum >= 0.f && momentum < 1.f,
                 "muon_step: lr %g, momentum %g, weight decay %g, rms %g, gradient scale %g", (double)lr, (double)momentum,
                 (double)weight_decay, (double)rms, (double)grad_scale);
  for (int i = 0; i < n; ++i) LSPS_CHECK_ARG(mats[i].p && mats[i].g && mats[i].m, "muon_step: null pointer in matrix %d", i);
  const OrthoCall call = {steps, a, b, c, eps, OM_MUON, false, 1.f - lr * weight_decay, {momentum, grad_scale, nesterov != 0}};
  OrthoGroup g[ORTHO_GROUPS];
  for (int at = 0; at < n; at += ORTHO_GROUPS)
    if (const int rc = ortho_check("muon_step", g, muon_pass(mats, n, at, lr, rms, g), call, ws, ws_bytes)) return rc;
  for (int at = 0; at < n; at += ORTHO_GROUPS)
    if (const int rc = ortho_run(g, muon_pass(mats, n, at, lr, rms, g), call, (char *)ws, (hipStream_t)stream)) return rc;
  return 0;
}

}  // extern "C"
