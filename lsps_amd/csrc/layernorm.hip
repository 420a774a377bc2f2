// Layer normalisation over the last dimension of a row-major [rows][cols] tensor (f32 or bf16 activations, f32 statistics and
// parameters), forward and backward with the reduction of the gain's and the bias' gradients.
//
//   mu = mean(x)   v = mean((x - mu)^2)   r = 1 / sqrt(v + eps)   h = (x - mu) r   y = h w + b
//   g = dy w       dx = r (g - mean(g) - h mean(g h))             dw = sum_rows dy h   db = sum_rows dy
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx.  A row is held in registers by the
// threads that own it, so x is read once although the variance is taken around the exact mean (two passes over registers; sums
// in f32).  TPR threads share a row and walk rows with a grid stride (w, b and the dw / db partial sums stay in registers):
//   TPR = 16 or 64 lanes of a wave (up to 256 / 1024 columns): reductions by DPP / shuffles only, no barrier;
//   TPR = 256 ... 1024 threads, the whole workgroup (up to 16 columns per thread): one LDS exchange per reduction;
//   longer rows: chunks of LN_CHUNK columns per workgroup, statistics of the chunks in one launch, application in a second one
//   (a row that long would otherwise be one workgroup's serial work; the second read comes from L2 / MALL at these sizes).
// Rows are read in 16-byte units that start at the row's own address (global memory takes them at element alignment), so odd
// widths and row pitches have no path of their own; a row's last, partial unit is moved back to end with the row, its columns that
// the unit in front holds too stay out of the sums (read element by element instead: 21 -> 17 us forward at 30000 x 700 bf16, 85 -> 52 us
// backward at 500000 x 50 f32).
// dw / db: each workgroup leaves its sums in the workspace, ln_params_kernel adds them in a fixed order (no atomics: the same
// inputs give the same bits).
//
// Times (MI355X; a large copy moves 4.9 TB/s, 8.5 out of the cache): 131072 x 256 f32 forward 42 us (6.3 TB/s), backward 72 + 4 us
// (5.6); bf16 22 us (6.1), 37 + 4 (5.4); 4096 x 4096 f32 22 + 35 + 4 us; 8191 x 2049 bf16 19 + 31 + 5 us (3.4 TB/s: 257 units on 256
// threads, every second request is one thread's); 32 x 262144 f32 7 + 12 us, 13 + 21 + 4 us.
#include "common.h"

namespace lsps {

typedef __bf16 ln_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 ln_bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef float ln_f32x4 __attribute__((ext_vector_type(4)));
typedef float ln_f32x4u __attribute__((ext_vector_type(4), aligned(4)));

template <typename T>
struct LnVec;
template <>
struct LnVec<float> {
  static constexpr int V = 4;
  typedef float type;
  typedef ln_f32x4 reg;
  typedef ln_f32x4u mem;
};
template <>
struct LnVec<__bf16> {
  static constexpr int V = 8;
  typedef __bf16 type;
  typedef ln_bf16x8 reg;
  typedef ln_bf16x8u mem;
};
// rows shorter than a unit
template <typename T>
struct LnOne {
  static constexpr int V = 1;
  typedef T type;
  typedef T reg __attribute__((ext_vector_type(1)));
  typedef reg mem;
};

#define LN_CHUNK 4096        // columns per workgroup of the split variant (256 threads x 16)
#define LN_FWD_COLS 16384    // longest row that one workgroup holds: forward 1024 threads x 16 columns;
#define LN_BWD_COLS 8192     // backward 512 x 16 (its ~185 registers a thread leave no room for 1024 threads)
#define LN_ROWS_LDS 64       // rows per workgroup of the split backward (their two means sit in LDS)

// `left` columns remain from p on; a unit past the row's end reads nothing and holds zeros
template <typename T>
__device__ __forceinline__ typename LnVec<T>::reg ln_load(const T *p, long left) {
  constexpr int V = LnVec<T>::V;
  typename LnVec<T>::reg r;
  if (left >= V) return *reinterpret_cast<const typename LnVec<T>::mem *>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) r[e] = e < left ? p[e] : (T)0.f;
  return r;
}

template <typename T>
__device__ __forceinline__ void ln_store(T *p, long left, const float (&v)[LnVec<T>::V]) {
  constexpr int V = LnVec<T>::V;
  typename LnVec<T>::reg r;
#pragma unroll
  for (int e = 0; e < V; ++e) r[e] = (T)v[e];        // bf16: the one rounding of the result (nearest even)
  if (left >= V) {
    *reinterpret_cast<typename LnVec<T>::mem *>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) p[e] = r[e];
  }
}

// the unit at p, or zeros; the one rounding of a bf16 result is the store's (nearest even)
template <typename U>
__device__ __forceinline__ typename U::reg ln_unit(const typename U::type *p, bool on) {
  if (on) return *reinterpret_cast<const typename U::mem *>(p);
  typename U::reg r;
#pragma unroll
  for (int e = 0; e < U::V; ++e) r[e] = (typename U::type)0.f;
  return r;
}
template <typename U>
__device__ __forceinline__ void ln_put(typename U::type *p, const float (&v)[U::V]) {
  typename U::reg r;
#pragma unroll
  for (int e = 0; e < U::V; ++e) r[e] = (typename U::type)v[e];
  *reinterpret_cast<typename U::mem *>(p) = r;
}

// V consecutive parameters from column c on (`fill` where there is no parameter tensor or no column)
template <int V>
__device__ __forceinline__ void ln_load_param(const float *p, long c, long cols, float fill, float (&v)[V]) {
  if (V % 4 == 0 && p && c + V <= cols) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const ln_f32x4 t = *reinterpret_cast<const ln_f32x4u *>(p + c + q * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[q * 4 + e] = t[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = p && c + e < cols ? p[c + e] : fill;
  }
}

template <int CTRL>
__device__ __forceinline__ float ln_dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// sum over the TPR threads of a row, every one of them receives it.  16 lanes: quad permutes and the two mirrors (xor 1, 2,
// then each half / row reversed); 64: two shuffles more; a whole workgroup: the waves' sums through `red` (2 x 16 floats,
// alternating halves so that one barrier per call is enough)
template <int TPR>
__device__ __forceinline__ float ln_row_sum(float v, float *red, int &phase) {
  v = ln_dpp_add<0xB1>(v);
  v = ln_dpp_add<0x4E>(v);
  v = ln_dpp_add<0x141>(v);
  v = ln_dpp_add<0x140>(v);
  if constexpr (TPR >= 64) {
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
  }
  if constexpr (TPR > 64) {
    float *slot = red + phase * 16;
    phase ^= 1;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v += slot[w];
  }
  return v;
}

// where the units of thread t of a row start, and how many of their leading columns the unit in front holds (V: no unit)
template <int V, int TPR, int NU>
__device__ __forceinline__ void ln_units(int t, int cols, int (&at)[NU], int (&skip)[NU]) {
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int c = (t + u * TPR) * V;
    at[u] = c < cols - V ? c : cols - V;
    skip[u] = c < cols ? c - at[u] : V;
  }
}

template <typename U, int TPR, int WG, int NU>
__global__ __launch_bounds__(WG) void ln_fwd_kernel(const typename U::type *__restrict__ x, long ldx, const float *__restrict__ w,
                                                    const float *__restrict__ b, typename U::type *__restrict__ y,
                                                    float *__restrict__ mean, float *__restrict__ rstd, long rows, int cols, float eps) {
  constexpr int V = U::V, RPW = WG / TPR;
  __shared__ float red[32];
  int phase = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  int at[NU], skip[NU];
  ln_units<V, TPR, NU>(t, cols, at, skip);
  float wv[NU][V], bv[NU][V];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    ln_load_param<V>(w, at[u], cols, 1.f, wv[u]);
    ln_load_param<V>(b, at[u], cols, 0.f, bv[u]);
  }
  const float n = (float)cols;                           // divided by: times 1 / n rounds twice, and a constant row has a variance then
  const long step = (long)gridDim.x * RPW, first = (long)blockIdx.x * RPW;
  typename U::reg q[NU];
  auto fetch = [&](long r0) {
    const bool on = r0 + sub < rows;
    const typename U::type *xr = x + (on ? r0 + sub : 0) * ldx;
#pragma unroll
    for (int u = 0; u < NU; ++u) q[u] = ln_unit<U>(xr + at[u], on && skip[u] < V);
  };
  if (first < rows) fetch(first);
  for (long r0 = first; r0 < rows; r0 += step) {                                       // the same trip count in all threads
    const long r = r0 + sub;
    float v[NU][V];
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[u][e] = (float)q[u][e];
        s += e >= skip[u] ? v[u][e] : 0.f;
      }
    if (r0 + step < rows) fetch(r0 + step);                                            // the next row, before this one's reductions
    const float mu = ln_row_sum<TPR>(s, red, phase) / n;
    float s2 = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[u][e] -= mu;
        s2 += e >= skip[u] ? v[u][e] * v[u][e] : 0.f;
      }
    const float rs = 1.f / sqrtf(ln_row_sum<TPR>(s2, red, phase) / n + eps);
    if (r >= rows) continue;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(v[u][e] * rs, wv[u][e], bv[u][e]);
      if (skip[u] < V) ln_put<U>(y + r * cols + at[u], o);                             // (columns of two units get the same bits twice)
    }
    if (t == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

// One pass over x and dy: dx, and this workgroup's share of dw / db in part[block][2][cols] (dw / db themselves for a grid of
// one workgroup).  The next row's x and dy are loaded before the current row's reductions.
template <typename U, int TPR, int WG, int NU>
__global__ __launch_bounds__(WG) void ln_bwd_kernel(const typename U::type *__restrict__ dy, long lddy,
                                                    const typename U::type *__restrict__ x, long ldx, const float *__restrict__ mean,
                                                    const float *__restrict__ rstd, const float *__restrict__ w,
                                                    typename U::type *__restrict__ dx, float *__restrict__ part, float *__restrict__ dw,
                                                    float *__restrict__ db, long rows, int cols) {
  constexpr int V = U::V, RPW = WG / TPR, ROW = TPR * NU * V;
  __shared__ float red[32];
  __shared__ float sums[RPW > 1 ? 2 * ROW : 1];
  int phase = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  int at[NU], skip[NU];
  ln_units<V, TPR, NU>(t, cols, at, skip);
  float wv[NU][V], aw[NU][V], ab[NU][V];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    ln_load_param<V>(w, at[u], cols, 1.f, wv[u]);
#pragma unroll
    for (int e = 0; e < V; ++e) aw[u][e] = ab[u][e] = 0.f;
  }
  const float n = (float)cols;
  const long step = (long)gridDim.x * RPW;
  typename U::reg xq[NU], gq[NU];
  float mu = 0.f, rs = 0.f;
  auto fetch = [&](long r0) {
    const long r = r0 + sub;
    const bool on = r < rows;
    const typename U::type *xr = x + (on ? r : 0) * ldx, *gr = dy + (on ? r : 0) * lddy;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      xq[u] = ln_unit<U>(xr + at[u], on && skip[u] < V);
      gq[u] = ln_unit<U>(gr + at[u], on && skip[u] < V);
    }
    mu = on ? mean[r] : 0.f;
    rs = on ? rstd[r] : 0.f;
  };
  const long first = (long)blockIdx.x * RPW;
  if (first < rows) fetch(first);
  for (long r0 = first; r0 < rows; r0 += step) {
    const long r = r0 + sub;
    float h[NU][V], g[NU][V];
    float s1 = 0.f, s2 = 0.f;
    const float rsc = rs;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (float)gq[u][e], once = e >= skip[u] ? d : 0.f;
        h[u][e] = ((float)xq[u][e] - mu) * rsc;
        aw[u][e] = fmaf(once, h[u][e], aw[u][e]);
        ab[u][e] += once;
        g[u][e] = d * wv[u][e];
        s1 = fmaf(once, wv[u][e], s1);
        s2 = fmaf(once * wv[u][e], h[u][e], s2);
      }
    if (r0 + step < rows) fetch(r0 + step);
    const float m1 = ln_row_sum<TPR>(s1, red, phase) / n, m2 = ln_row_sum<TPR>(s2, red, phase) / n;
    if (r >= rows || !dx) continue;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = rsc * (g[u][e] - m1 - h[u][e] * m2);
      if (skip[u] < V) ln_put<U>(dx + r * cols + at[u], o);
    }
  }
  if (!dw && !db) return;
  float *pw = gridDim.x == 1 ? dw : part + (long)blockIdx.x * 2 * cols, *pb = gridDim.x == 1 ? db : pw + cols;
  if constexpr (RPW > 1) {                               // the row groups of the workgroup, one after the other
    for (int k = 0; k < RPW; ++k) {
      __syncthreads();
      if (sub == k) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int c = (t + u * TPR) * V + e;
            sums[c] = k ? sums[c] + aw[u][e] : aw[u][e];
            sums[ROW + c] = k ? sums[ROW + c] + ab[u][e] : ab[u][e];
          }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += WG) {       // column c: unit c / V, moved back by its skip in the row's last unit
      const int u = c / V * V, k = u < cols - V ? c : c + u - (cols - V);
      if (pw) pw[c] = sums[k];
      if (pb) pb[c] = sums[ROW + k];
    }
  } else {
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e >= skip[u]) {
          if (pw) pw[at[u] + e] = aw[u][e];
          if (pb) pb[at[u] + e] = ab[u][e];
        }
  }
}

// dw / db = sum over the `parts` rows of part[parts][2][cols], in a fixed order (the partial sums come from L2).  Many parts: a
// workgroup takes 16 of the 2 * cols columns with 64 threads each (runs of 64 bytes).  Few: a thread walks one column.
__global__ __launch_bounds__(1024) void ln_params_kernel(const float *__restrict__ part, int parts, long cols, float *__restrict__ dw,
                                                         float *__restrict__ db) {
  __shared__ float red[16][16];
  const int k = threadIdx.x & 15, s = threadIdx.x >> 4;
  for (long c0 = (long)blockIdx.x * 16; c0 < 2 * cols; c0 += (long)gridDim.x * 16) {
    const long c = c0 + k;
    float a = 0.f;
    if (c < 2 * cols) {
#pragma unroll 4
      for (int i = s; i < parts; i += 64) a += part[(long)i * 2 * cols + c];
    }
    a += __shfl_xor(a, 16, 64);
    a += __shfl_xor(a, 32, 64);
    __syncthreads();
    if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][k] = a;
    __syncthreads();
    if (threadIdx.x < 16 && c < 2 * cols) {
      a = 0.f;
#pragma unroll
      for (int w = 0; w < 16; ++w) a += red[w][k];
      float *dst = c < cols ? dw : db;
      if (dst) dst[c < cols ? c : c - cols] = a;
    }
  }
}
__global__ __launch_bounds__(256) void ln_params_few_kernel(const float *__restrict__ part, int parts, long cols, float *__restrict__ dw,
                                                            float *__restrict__ db) {
  for (long c = (long)blockIdx.x * 256 + threadIdx.x; c < 2 * cols; c += (long)gridDim.x * 256) {
    float a = 0.f;
#pragma unroll 8
    for (int i = 0; i < parts; ++i) a += part[(long)i * 2 * cols + c];
    float *dst = c < cols ? dw : db;
    if (dst) dst[c < cols ? c : c - cols] = a;
  }
}

// ---- rows longer than a workgroup holds ---------------------------------------------------------------------------------------
// (mean, sum of squares around it) of every chunk of a row: st[row][chunk][2]
template <typename T>
__global__ __launch_bounds__(256) void ln_split_stats_kernel(const T *__restrict__ x, long ldx, float *__restrict__ st, long rows,
                                                             long cols, int chunks) {
  constexpr int V = LnVec<T>::V, NU = LN_CHUNK / (256 * V);
  __shared__ float red[32];
  int phase = 0;
  for (long i = blockIdx.x; i < rows * chunks; i += gridDim.x) {
    const long r = i / chunks, c0 = (i - r * chunks) * LN_CHUNK;
    const long n = cols - c0 < LN_CHUNK ? cols - c0 : LN_CHUNK;
    const T *xr = x + r * ldx + c0;
    float v[NU][V], s = 0.f, s2 = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int c = (threadIdx.x + u * 256) * V;
      const typename LnVec<T>::reg q = ln_load<T>(xr + c, n - c);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[u][e] = (float)q[e];
        s += v[u][e];
      }
    }
    const float mu = ln_row_sum<256>(s, red, phase) / (float)n;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = v[u][e] - mu;
        s2 += (threadIdx.x + u * 256) * V + e < n ? d * d : 0.f;
      }
    s2 = ln_row_sum<256>(s2, red, phase);
    if (threadIdx.x == 0) {
      st[2 * i] = mu;
      st[2 * i + 1] = s2;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_split_fwd_kernel(const T *__restrict__ x, long ldx, const float *__restrict__ w,
                                                           const float *__restrict__ b, const float *__restrict__ st,
                                                           T *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd,
                                                           long rows, long cols, int chunks, float eps) {
  constexpr int V = LnVec<T>::V, NU = LN_CHUNK / (256 * V);
  __shared__ float red[32];
  int phase = 0;
  for (long i = blockIdx.x; i < rows * chunks; i += gridDim.x) {
    const long r = i / chunks, c0 = (i - r * chunks) * LN_CHUNK;
    const long n = cols - c0 < LN_CHUNK ? cols - c0 : LN_CHUNK;
    const T *xr = x + r * ldx + c0;
    typename LnVec<T>::reg q[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int c = (threadIdx.x + u * 256) * V;
      q[u] = ln_load<T>(xr + c, n - c);
    }
    const float *sr = st + r * chunks * 2;
    float s = 0.f;
    for (int k = threadIdx.x; k < chunks; k += 256) s += sr[2 * k] * (float)(k + 1 < chunks ? LN_CHUNK : cols - (long)k * LN_CHUNK);
    const float mu = ln_row_sum<256>(s, red, phase) / (float)cols;
    s = 0.f;
    for (int k = threadIdx.x; k < chunks; k += 256) {
      const float d = sr[2 * k] - mu;
      s += sr[2 * k + 1] + d * d * (float)(k + 1 < chunks ? LN_CHUNK : cols - (long)k * LN_CHUNK);
    }
    const float rs = 1.f / sqrtf(ln_row_sum<256>(s, red, phase) / (float)cols + eps);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int c = (threadIdx.x + u * 256) * V;
      if (c < n) {
        float wv[V], bv[V], o[V];
        ln_load_param<V>(w, c0 + c, cols, 1.f, wv);
        ln_load_param<V>(b, c0 + c, cols, 0.f, bv);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(((float)q[u][e] - mu) * rs, wv[e], bv[e]);
        ln_store<T>(y + r * cols + c0 + c, n - c, o);
      }
    }
    if (threadIdx.x == 0 && c0 == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

// sum of g and of g h over every chunk of a row: st[row][chunk][2]
template <typename T>
__global__ __launch_bounds__(256) void ln_split_dots_kernel(const T *__restrict__ dy, long lddy, const T *__restrict__ x, long ldx,
                                                            const float *__restrict__ mean, const float *__restrict__ rstd,
                                                            const float *__restrict__ w, float *__restrict__ st, long rows, long cols,
                                                            int chunks) {
  constexpr int V = LnVec<T>::V, NU = LN_CHUNK / (256 * V);
  __shared__ float red[32];
  int phase = 0;
  for (long i = blockIdx.x; i < rows * chunks; i += gridDim.x) {
    const long r = i / chunks, c0 = (i - r * chunks) * LN_CHUNK;
    const long n = cols - c0 < LN_CHUNK ? cols - c0 : LN_CHUNK;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int c = (threadIdx.x + u * 256) * V;
      const typename LnVec<T>::reg xq = ln_load<T>(x + r * ldx + c0 + c, n - c), gq = ln_load<T>(dy + r * lddy + c0 + c, n - c);
      float wv[V];
      ln_load_param<V>(w, c0 + c, cols, 1.f, wv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float g = (float)gq[e] * wv[e];
        s1 += g;
        s2 += c + e < n ? g * (((float)xq[e] - mu) * rs) : 0.f;
      }
    }
    s1 = ln_row_sum<256>(s1, red, phase);
    s2 = ln_row_sum<256>(s2, red, phase);
    if (threadIdx.x == 0) {
      st[2 * i] = s1;
      st[2 * i + 1] = s2;
    }
  }
}

// dx, and dw / db summed over the `rpg` rows of a group: a workgroup owns 256 V columns of one group
template <typename T>
__global__ __launch_bounds__(256) void ln_split_bwd_kernel(const T *__restrict__ dy, long lddy, const T *__restrict__ x, long ldx,
                                                           const float *__restrict__ mean, const float *__restrict__ rstd,
                                                           const float *__restrict__ w, const float *__restrict__ st,
                                                           T *__restrict__ dx, float *__restrict__ part, float *__restrict__ dw,
                                                           float *__restrict__ db, long rows, long cols, int chunks, int rpg, int groups) {
  constexpr int V = LnVec<T>::V;
  __shared__ float m1s[LN_ROWS_LDS], m2s[LN_ROWS_LDS], mus[LN_ROWS_LDS], rss[LN_ROWS_LDS];
  const long blocks = (cols + 256 * V - 1) / (256 * V);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (long i = blockIdx.x; i < blocks * groups; i += gridDim.x) {
    const long grp = i / blocks, c = ((i - grp * blocks) * 256 + threadIdx.x) * V;
    const long r0 = grp * rpg;
    const int n = (int)(rows - r0 < rpg ? rows - r0 : rpg);
    __syncthreads();
    for (int k = wave; k < n; k += 4) {
      const float *sr = st + (r0 + k) * chunks * 2;
      float s1 = 0.f, s2 = 0.f;
      for (int q = lane; q < chunks; q += 64) {
        s1 += sr[2 * q];
        s2 += sr[2 * q + 1];
      }
      s1 = wave_sum(s1);
      s2 = wave_sum(s2);
      if (lane == 0) {
        m1s[k] = s1 / (float)cols;
        m2s[k] = s2 / (float)cols;
        mus[k] = mean[r0 + k];
        rss[k] = rstd[r0 + k];
      }
    }
    __syncthreads();
    if (c < cols) {
      float wv[V], aw[V], ab[V];
      ln_load_param<V>(w, c, cols, 1.f, wv);
#pragma unroll
      for (int e = 0; e < V; ++e) aw[e] = ab[e] = 0.f;
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const typename LnVec<T>::reg xq = ln_load<T>(x + (r0 + k) * ldx + c, cols - c), gq = ln_load<T>(dy + (r0 + k) * lddy + c, cols - c);
        const float mu = mus[k], rs = rss[k], m1 = m1s[k], m2 = m2s[k];
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = (float)gq[e], h = ((float)xq[e] - mu) * rs;
          aw[e] = fmaf(d, h, aw[e]);
          ab[e] += d;
          o[e] = rs * (d * wv[e] - m1 - h * m2);
        }
        if (dx) ln_store<T>(dx + (r0 + k) * cols + c, cols - c, o);
      }
      float *pw = groups == 1 ? dw : part + grp * 2 * cols, *pb = groups == 1 ? db : pw + cols;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e < cols) {
          if (pw && (dw || groups > 1)) pw[c + e] = aw[e];
          if (pb && (db || groups > 1)) pb[c + e] = ab[e];
        }
    }
  }
}

// ---- launch shapes ------------------------------------------------------------------------------------------------------
static int ln_chunks(long cols) { return (int)((cols + LN_CHUNK - 1) / LN_CHUNK); }

// rows per workgroup pass of the register variants
static int ln_rows_per_pass(long cols) { return cols <= 256 ? 16 : cols <= 1024 ? 4 : 1; }

// workgroups of the register backward: one per CU as soon as there are passes for them (300 x 1500 f32 18 us with one for 16 rows, 9 so;
// 100 x 8000 30 / 16; 1000 x 700 13 / 9), then enough to fill 256 CUs, few enough that the partial sums (8 bytes per column and
// workgroup) stay small next to the rows they stand for; a handful of rows is one workgroup and needs no second launch.
// Measured: 131072 x 256 f32 72 us with at most 768, 72 with 1024, 79 with 512, in bf16 37 / 41 / 36; one row per pass: 4096 x 4096
// f32 34.5 us with 16 rows a workgroup, 37 with 8.  One row per pass, 2^25 elements, with at most 256 / 512 / 768 / 1024 workgroups: f32
// of 1500 columns 98 / 78 / 82 / 88, 3000 79 / 85 / 96, 8000 (one workgroup per CU) 89 / 113; bf16 of 1100 118 / 69 / 58 / 51, 1500 90 / 55 /
// 47 / 47, 3000 54 / 45 / 48, 8000 50 / 73.
static int ln_bwd_groups(long rows, long cols, int V) {
  const int rpp = ln_rows_per_pass(cols);
  const long passes = (rows + rpp - 1) / rpp;
  if (passes <= 4) return 1;
  const long few = passes < 256 ? passes : 256, many = rpp > 1 ? (passes + 7) / 8 : (passes + 15) / 16, g = many > few ? many : few;
  const long most = rpp > 1 ? 768 : cols > 4096 ? 256 : V == 4 ? (cols > 2048 ? 256 : 512) : cols > 2048 ? 512 : 768;
  return (int)(g < most ? g : most);
}

// row groups of the split backward: a workgroup owns 256 V columns; more groups only while they are needed to fill the chip
static int ln_split_rows_per_group(long rows, long cols, int V) {
  const long blocks = (cols + 256L * V - 1) / (256L * V);
  long groups = (1024 + blocks - 1) / blocks;
  if (groups > rows) groups = rows;
  long rpg = (rows + groups - 1) / groups;
  if (rpg > LN_ROWS_LDS) rpg = LN_ROWS_LDS;
  return (int)rpg;
}

static size_t ln_ws_bytes(long rows, long cols, int V) {
  if (cols <= LN_BWD_COLS) {
    const int g = ln_bwd_groups(rows, cols, V);
    return g > 1 ? (size_t)g * 2 * cols * sizeof(float) : 0;
  }
  const int rpg = ln_split_rows_per_group(rows, cols, V);
  const long groups = (rows + rpg - 1) / rpg;
  return align_up((size_t)rows * ln_chunks(cols) * 2 * sizeof(float), 256) + (groups > 1 ? (size_t)groups * 2 * cols * sizeof(float) : 0);
}

static int ln_grid(long n, long most) { return (int)(n < most ? n : most); }

template <typename T>
static void ln_fwd_launch(const T *x, long ldx, const float *w, const float *b, T *y, float *mean, float *rstd, long rows, int cols,
                          float eps, hipStream_t st) {
  constexpr int V = LnVec<T>::V;
#define LN_F(TPR, WG, NU)                                                                                                    \
  hipLaunchKernelGGL((ln_fwd_kernel<U, TPR, WG, NU>), dim3(ln_grid((rows + WG / TPR - 1) / (WG / TPR), 256 * (2048 / WG))), \
                     dim3(WG), 0, st, x, ldx, w, b, y, mean, rstd, rows, cols, eps)
  if (cols < V) {
    typedef LnOne<T> U;
    LN_F(16, 256, 1);
    return;
  }
  typedef LnVec<T> U;
  if (cols <= 64) LN_F(16, 256, 64 / (16 * V) ? 64 / (16 * V) : 1);
  else if (cols <= 128) LN_F(16, 256, 128 / (16 * V));
  else if (cols <= 256) LN_F(16, 256, 256 / (16 * V));
  else if (cols <= 512) LN_F(64, 256, 512 / (64 * V));
  else if (cols <= 1024) LN_F(64, 256, 1024 / (64 * V));
  else if (cols <= 2048) LN_F(256, 256, 2048 / (256 * V));
  else if (cols <= 4096) LN_F(256, 256, 4096 / (256 * V));
  else if (cols <= 8192) LN_F(512, 512, 8192 / (512 * V));
  else LN_F(1024, 1024, 16384 / (1024 * V));
#undef LN_F
}

template <typename T>
static void ln_bwd_launch(const T *dy, long lddy, const T *x, long ldx, const float *mean, const float *rstd, const float *w, T *dx,
                          float *part, float *dw, float *db, long rows, int cols, int groups, hipStream_t st) {
  constexpr int V = LnVec<T>::V;
#define LN_B(TPR, WG, NU)                                                                                               \
  hipLaunchKernelGGL((ln_bwd_kernel<U, TPR, WG, NU>), dim3(groups), dim3(WG), 0, st, dy, lddy, x, ldx, mean, rstd, w, dx, \
                     part, dw, db, rows, cols)
  if (cols < V) {
    typedef LnOne<T> U;
    LN_B(16, 256, 1);
    return;
  }
  typedef LnVec<T> U;
  if (cols <= 64) LN_B(16, 256, 64 / (16 * V) ? 64 / (16 * V) : 1);
  else if (cols <= 128) LN_B(16, 256, 128 / (16 * V));
  else if (cols <= 256) LN_B(16, 256, 256 / (16 * V));
  else if (cols <= 512) LN_B(64, 256, 512 / (64 * V));
  else if (cols <= 1024) LN_B(64, 256, 1024 / (64 * V));
  else if (cols <= 2048) LN_B(256, 256, 2048 / (256 * V));
  else if (cols <= 4096) LN_B(256, 256, 4096 / (256 * V));
  else LN_B(512, 512, 8192 / (512 * V));
#undef LN_B
}

template <typename T>
static int ln_fwd(const void *x_, const float *w, const float *b, void *y_, float *mean, float *rstd, long rows, long cols, long ldx,
                  float eps, void *ws, hipStream_t st) {
  const T *x = (const T *)x_;
  T *y = (T *)y_;
  if (cols <= LN_FWD_COLS) {
    ln_fwd_launch<T>(x, ldx, w, b, y, mean, rstd, rows, (int)cols, eps, st);
  } else {
    const int chunks = ln_chunks(cols), grid = ln_grid(rows * chunks, 1 << 20);
    hipLaunchKernelGGL(ln_split_stats_kernel<T>, dim3(grid), dim3(256), 0, st, x, ldx, (float *)ws, rows, cols, chunks);
    hipLaunchKernelGGL(ln_split_fwd_kernel<T>, dim3(grid), dim3(256), 0, st, x, ldx, w, b, (const float *)ws, y, mean, rstd, rows, cols,
                       chunks, eps);
  }
  LSPS_CHECK_LAUNCH("layernorm_fwd");
  return 0;
}

template <typename T>
static int ln_bwd(const void *dy_, const void *x_, const float *mean, const float *rstd, const float *w, void *dx_, float *dw, float *db,
                  long rows, long cols, long ldx, long lddy, void *ws, hipStream_t st) {
  const T *x = (const T *)x_, *dy = (const T *)dy_;
  T *dx = (T *)dx_;
  float *part;
  int parts;
  if (cols <= LN_BWD_COLS) {
    part = (float *)ws;
    parts = ln_bwd_groups(rows, cols, LnVec<T>::V);
    ln_bwd_launch<T>(dy, lddy, x, ldx, mean, rstd, w, dx, part, dw, db, rows, (int)cols, parts, st);
  } else {
    const int chunks = ln_chunks(cols), rpg = ln_split_rows_per_group(rows, cols, LnVec<T>::V);
    const long blocks = (cols + 256L * LnVec<T>::V - 1) / (256L * LnVec<T>::V);
    parts = (int)((rows + rpg - 1) / rpg);
    part = (float *)((char *)ws + align_up((size_t)rows * chunks * 2 * sizeof(float), 256));
    hipLaunchKernelGGL(ln_split_dots_kernel<T>, dim3(ln_grid(rows * chunks, 1 << 20)), dim3(256), 0, st, dy, lddy, x, ldx, mean, rstd, w,
                       (float *)ws, rows, cols, chunks);
    hipLaunchKernelGGL(ln_split_bwd_kernel<T>, dim3(ln_grid(blocks * parts, 1 << 20)), dim3(256), 0, st, dy, lddy, x, ldx, mean, rstd, w,
                       (const float *)ws, dx, part, dw, db, rows, cols, chunks, rpg, parts);
  }
  if (parts > 1 && (dw || db)) {
    if (parts <= 64)
      hipLaunchKernelGGL(ln_params_few_kernel, dim3(ln_grid((2 * cols + 255) / 256, 1 << 16)), dim3(256), 0, st, part, parts, cols, dw, db);
    else
      hipLaunchKernelGGL(ln_params_kernel, dim3(ln_grid((2 * cols + 15) / 16, 1 << 16)), dim3(1024), 0, st, part, parts, cols, dw, db);
  }
  LSPS_CHECK_LAUNCH("layernorm_bwd");
  return 0;
}

}  // namespace lsps

using namespace lsps;

extern "C" {

size_t lsps_layernorm_workspace_bytes(long rows, long cols, int dtype) {
  if (rows <= 0 || cols <= 0 || (dtype != LSPS_F32 && dtype != LSPS_BF16)) return 0;
  return align_up(ln_ws_bytes(rows, cols, dtype == LSPS_F32 ? 4 : 8), 256);
}

static int ln_check(const char *what, const void *x, bool stats, long rows, long cols, long ldx, int dtype, void *ws, size_t ws_bytes,
                    bool needs_ws) {
  LSPS_CHECK_ARG(x && stats, "%s: null pointer", what);
  LSPS_CHECK_ARG(dtype == LSPS_F32 || dtype == LSPS_BF16, "%s: dtype %d (LSPS_F32 or LSPS_BF16)", what, dtype);
  LSPS_CHECK_ARG(rows > 0 && cols > 0 && rows <= (1L << 40) / cols, "%s: %ld rows of %ld columns", what, rows, cols);
  LSPS_CHECK_ARG(ldx >= cols || rows == 1, "%s: row pitch %ld below %ld columns", what, ldx, cols);
  if (needs_ws) {
    const size_t need = lsps_layernorm_workspace_bytes(rows, cols, dtype);
    if (need && (!ws || ws_bytes < need)) {
      set_error("%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
      return LSPS_E_WS;
    }
  }
  return 0;
}

int lsps_layernorm_fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, long rows, long cols,
                       long ldx, int dtype, float eps, void *ws, size_t ws_bytes, void *stream) {
  (void)hipGetLastError();   // clear stale sticky errors left by other users of the runtime
  if (const int rc = ln_check("layernorm_fwd", x, !mean == !rstd, rows, cols, ldx, dtype, ws, ws_bytes, cols > LN_FWD_COLS)) return rc;
  LSPS_CHECK_ARG(y, "layernorm_fwd: null output");
  LSPS_CHECK_ARG(eps >= 0.f, "layernorm_fwd: eps %g", (double)eps);
  return dtype == LSPS_F32 ? ln_fwd<float>(x, gamma, beta, y, mean, rstd, rows, cols, ldx, eps, ws, (hipStream_t)stream)
                           : ln_fwd<__bf16>(x, gamma, beta, y, mean, rstd, rows, cols, ldx, eps, ws, (hipStream_t)stream);
}

int lsps_layernorm_bwd(const void *dy, const void *x, const float *mean, const float *rstd, const float *gamma, void *dx, float *dgamma,
                       float *dbeta, long rows, long cols, long ldx, long lddy, int dtype, void *ws, size_t ws_bytes, void *stream) {
  (void)hipGetLastError();   // clear stale sticky errors left by other users of the runtime
  if (const int rc = ln_check("layernorm_bwd", x, mean && rstd, rows, cols, ldx, dtype, ws, ws_bytes, true)) return rc;
  LSPS_CHECK_ARG(dy && (dx || dgamma || dbeta), "layernorm_bwd: null gradient");
  LSPS_CHECK_ARG(lddy >= cols || rows == 1, "layernorm_bwd: row pitch %ld below %ld columns", lddy, cols);
  return dtype == LSPS_F32 ? ln_bwd<float>(dy, x, mean, rstd, gamma, dx, dgamma, dbeta, rows, cols, ldx, lddy, ws, (hipStream_t)stream)
                           : ln_bwd<__bf16>(dy, x, mean, rstd, gamma, dx, dgamma, dbeta, rows, cols, ldx, lddy, ws, (hipStream_t)stream);
}

}  // extern "C"
