// Layer norm over the last axis, forward and backward.
//   mean = <x>, rstd = 1 / sqrt(<(x - mean)^2> + eps), h = (x - mean) rstd, y = h w + b
//   g = dy w:  dx = rstd (g - <g> - h <g h>),  dw = sum_rows dy h,  db = sum_rows dy
//
// Bound by memory.  A row is read once and stays in registers (fp32, fp64 rows in fp64).  A first mean is taken, then the deviations from it: their own mean is what the
// first one is off by, which for a row far from zero is many times the last place of its deviations, and is taken off again (fp32 columns of unit spread around
// 1e5: y off by 4.5e-7, without it by 9e-3; the backward pass takes the mean as it is stored, rounded to its type).  That costs 0.4 of 7.1 us for 65 536 x 21 of fp64.
// 16-bit elements go without: the fp32 sum of 2^13 fp16 or 2^16 bf16 numbers of one binade is exact, the mean off by 2^-24 of it, where the elements' own steps are
// 2^-11 and 2^-8 of it (with it 16384 x 8192 of bf16, at the clocks of a long run, took 134 us instead of 118).  16, 64, 256 or 1024 lanes share a row, so that a lane holds at most four 16-byte
// vectors; longer rows go through the kernels that read them again.  Loads and stores are 16 bytes a lane at any
// alignment (global memory takes them unaligned).  A row's last, partial vector is moved back to end with the row: it repeats columns of the lane before,
// which it leaves out of the row's sums and otherwise computes and writes a second time, with the same result.  So a row is loaded without a branch, and
// the next row's loads fly while one is reduced.
// The weights' gradients: every workgroup takes every gridDim-th group of rows and adds its columns in registers; the workgroups' sums are
// added in index order by a second launch -- no atomics, the same bits every time.
// 16384 x 8192 of bf16: 94 us, 150 us backward (5.3 TB/s); 10 000 x 1001 of fp32 16 and 22 us; 65 536 x 21 of fp64 9.0 and 8.5 us.
#include <algorithm>

#include "layers.hpp"

using namespace vmcpde;

namespace {

template <typename A> __device__ __forceinline__ A reciprocal_root(A v);
template <> __device__ __forceinline__ float reciprocal_root(float v) { return 1.0f / sqrtf(v); }
template <> __device__ __forceinline__ double reciprocal_root(double v) { return 1.0 / sqrt(v); }

// whether the deviations' mean is taken off (above)
template <typename T> constexpr bool refined() { return sizeof(T) > 2; }

// the variance from the mean of the squared deviations from a mean that is off by `off` (rounding may leave less than nothing of it; NaN stays)
template <typename A>
__device__ __forceinline__ A variance(A squares, A off) {
  const A v = squares - off * off;
  return v < 0 ? 0 : v;
}

// Sums of K values over the LANES lanes that share a row; every lane returns them.  `sh`: K x waves values, one slot a call in a row's turn.
template <int LANES, int K, typename A>
__device__ __forceinline__ void row_sum(A (&v)[K], A* sh) {
  if constexpr (LANES <= 64) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = group_sum<LANES>(v[k]);
  } else {
    constexpr int WAVES = LANES / 64;
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = group_sum<64>(v[k]);
      if ((threadIdx.x & 63) == 0) sh[k * WAVES + wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = sh[k * WAVES];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) v[k] += sh[k * WAVES + w];
    }
  }
}

// Where a lane's vectors lie in a row of cols >= V: from column base[i], of which the first skip[i] belong to the lane before (V or more: all of them).
template <int LANES, int ITER, int V>
struct Span {
  int base[ITER], skip[ITER];
  __device__ __forceinline__ explicit Span(int64_t cols) {
    const int lane = threadIdx.x % LANES;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int col = (i * LANES + lane) * V;
      base[i] = min(col, (int)cols - V);
      skip[i] = col - base[i];
    }
  }
};
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[V]; };
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> raw_at(const T* p) { return *reinterpret_cast<const Raw<T, V>*>(p); }
template <typename T, int V, typename A>
__device__ __forceinline__ void put(T* p, const A (&v)[V]) {
  Raw<T, V> r;
#pragma unroll
  for (int k = 0; k < V; ++k) r.v[k] = (T)v[k];
  *reinterpret_cast<Raw<T, V>*>(p) = r;
}
// a weight's or bias' vector; `none` where there is none
template <typename W, int V, typename A>
__device__ __forceinline__ void weights_at(const W* p, int64_t base, A none, A (&out)[V]) {
  if (p) {
    const Raw<W, V> r = raw_at<W, V>(p + base);
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = (A)r.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = none;
  }
}

// Every workgroup takes every gridDim-th group of rows.  The weights stay in registers where a lane holds at most 16 elements: read anew for every row
// they are up to four times the row's own traffic, from the caches.  EXACT: the row is LANES * ITER vectors.
template <typename T, typename W, int LANES, int ITER, int THREADS, bool EXACT>
__global__ __launch_bounds__(THREADS) void norm_forward_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ weight, const W* __restrict__ bias,
                                                               typename Wide<T>::type eps, int64_t rows, int64_t cols, T* __restrict__ y, int64_t ldy,
                                                               typename Wide<T>::type* __restrict__ mean_out, typename Wide<T>::type* __restrict__ rstd_out) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>(), GROUPS = THREADS / LANES, WAVES = THREADS / 64;
  constexpr bool KEEP = ITER * V <= 16, REFINED = refined<T>();
  __shared__ A sh[2][3][WAVES];                // (two sets of slots in turn: a wave may be a row ahead of the slowest)
  const int lane = threadIdx.x % LANES;
  const A inv = (A)1 / (A)cols;
  const Span<LANES, ITER, V> at(cols);
  A w[KEEP ? ITER : 1][V], b[KEEP ? ITER : 1][V];
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      weights_at<W, V>(weight, at.base[i], (A)1, w[i]);
      weights_at<W, V>(bias, at.base[i], (A)0, b[i]);
    }
  }
  Raw<T, V> next[ITER];
  auto fetch = [&](int64_t row) {
    const T* xr = x + (GROUPS == 1 || row < rows ? row : 0) * ldx;
#pragma unroll
    for (int i = 0; i < ITER; ++i) next[i] = raw_at<T, V>(xr + at.base[i]);
  };
  int64_t first = (int64_t)blockIdx.x * GROUPS;
  fetch(first + threadIdx.x / LANES);
  for (int turn = 0; first < rows; turn ^= 1) {
    const int64_t row = first + threadIdx.x / LANES;
    first += (int64_t)gridDim.x * GROUPS;
    A v[ITER][V], s[1] = {0}, q[REFINED ? 2 : 1] = {};
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[i][k] = (A)next[i].v[k];
        s[0] += EXACT || k >= at.skip[i] ? v[i][k] : (A)0;
      }
    if (first < rows) fetch(first + threadIdx.x / LANES);
    row_sum<LANES>(s, sh[turn][0]);
    const A mean = s[0] / (A)cols;
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[i][k] -= mean;
        const A d = EXACT || k >= at.skip[i] ? v[i][k] : (A)0;
        q[0] += d * d;
        if constexpr (REFINED) q[1] += d;
      }
    row_sum<LANES>(q, sh[turn][1]);
    A off = 0;
    if constexpr (REFINED) off = q[1] * inv;
    const A rstd = reciprocal_root<A>(variance(q[0] * inv, off) + eps), less = -off * rstd;
    if (GROUPS > 1 && row >= rows) continue;   // (a whole group of lanes; the sums above need every lane of a wave)
    if (lane == 0 && mean_out) {
      mean_out[row] = mean + off;
      rstd_out[row] = rstd;
    }
    T* yr = y + row * ldy;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      A wi[V], bi[V];
      if constexpr (KEEP) {
#pragma unroll
        for (int k = 0; k < V; ++k) wi[k] = w[i][k], bi[k] = b[i][k];
      } else {
        weights_at<W, V>(weight, at.base[i], (A)1, wi);
        weights_at<W, V>(bias, at.base[i], (A)0, bi);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] = (REFINED ? fma(v[i][k], rstd, less) : v[i][k] * rstd) * wi[k] + bi[k];
      if (EXACT || at.skip[i] < V) put<T, V>(yr + at.base[i], v[i]);
    }
  }
}

// Rows that no 1024 lanes hold: read three times, the second and third time from the caches.  A lane takes four vectors at a time, whose loads fly together
// (the last one moved back, as above): 4096 x 8200 of fp64 143 us (one after the other it lost 24); the backward pass of 4096 x 20000 of bf16 220, 372.
template <int V, typename F>
__device__ __forceinline__ void wide_row(int64_t cols, F f) {
  for (int64_t first = (int64_t)threadIdx.x * V; first < cols; first += 4 * 1024 * V) {
    int64_t base[4];
    int skip[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t col = first + (int64_t)u * 1024 * V;
      base[u] = col < cols - V ? col : cols - V;
      skip[u] = col - base[u] < V ? (int)(col - base[u]) : V;
    }
    f(base, skip);
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_forward_wide_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ weight, const W* __restrict__ bias,
                                                                 typename Wide<T>::type eps, int64_t cols, T* __restrict__ y, int64_t ldy,
                                                                 typename Wide<T>::type* __restrict__ mean_out, typename Wide<T>::type* __restrict__ rstd_out) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>();
  __shared__ A sh[3][16];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  constexpr bool REFINED = refined<T>();
  A s[1] = {0}, q[REFINED ? 2 : 1] = {};
  auto load = [&](const int64_t (&base)[4], Raw<T, V> (&r)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = raw_at<T, V>(xr + base[u]);
  };
  wide_row<V>(cols, [&](const int64_t (&base)[4], const int (&skip)[4]) {
    Raw<T, V> r[4];
    load(base, r);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) s[0] += k >= skip[u] ? (A)r[u].v[k] : (A)0;
  });
  row_sum<1024>(s, sh[0]);
  const A mean = s[0] / (A)cols;
  wide_row<V>(cols, [&](const int64_t (&base)[4], const int (&skip)[4]) {
    Raw<T, V> r[4];
    load(base, r);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const A d = k >= skip[u] ? (A)r[u].v[k] - mean : (A)0;
        q[0] += d * d;
        if constexpr (REFINED) q[1] += d;
      }
  });
  row_sum<1024>(q, sh[1]);
  A off = 0;
  if constexpr (REFINED) off = q[1] / (A)cols;
  const A rstd = reciprocal_root<A>(variance(q[0] / (A)cols, off) + eps), less = -off * rstd;
  if (threadIdx.x == 0 && mean_out) {
    mean_out[row] = mean + off;
    rstd_out[row] = rstd;
  }
  wide_row<V>(cols, [&](const int64_t (&base)[4], const int (&skip)[4]) {
    Raw<T, V> r[4];
    load(base, r);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      A w[V], b[V], v[V];
      weights_at<W, V>(weight, base[u], (A)1, w);
      weights_at<W, V>(bias, base[u], (A)0, b);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = (REFINED ? fma((A)r[u].v[k] - mean, rstd, less) : ((A)r[u].v[k] - mean) * rstd) * w[k] + b[k];
      if (skip[u] < V) put<T, V>(y + row * ldy + base[u], v);
    }
  });
}

// dx (may be null) and, with `partial`, this workgroup's column sums: partial[group][2][cols] = { sum dy h, sum dy }; a single workgroup writes them to
// dweight and dbias (either may be null) itself.
template <typename T, typename W, int LANES, int ITER, int THREADS, bool EXACT>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(const T* __restrict__ dy, int64_t ldd, const T* __restrict__ x, int64_t ldx,
                                                                const typename Wide<T>::type* __restrict__ mean_in,
                                                                const typename Wide<T>::type* __restrict__ rstd_in, const W* __restrict__ weight,
                                                                int64_t rows, int64_t cols, T* __restrict__ dx, typename Wide<T>::type* __restrict__ partial,
                                                                W* __restrict__ dweight, W* __restrict__ dbias) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>(), GROUPS = THREADS / LANES, WAVES = THREADS / 64;
  constexpr int SHARED = LANES <= 64 ? WAVES * LANES * ITER * V : 4 * WAVES;   // column sums of every wave, or the slots of the row sums
  constexpr bool KEEP = LANES < 1024 || ITER * V <= 8, AHEAD = LANES < 1024 || ITER * (int)sizeof(T) <= 8;      // (1024 lanes have 128 registers each)
  __shared__ A sh[SHARED];
  const int lane = threadIdx.x % LANES;
  const A inv = (A)1 / (A)cols;
  const Span<LANES, ITER, V> at(cols);
  A dw[ITER][V], db[ITER][V], w[KEEP ? ITER : 1][V];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    if constexpr (KEEP) weights_at<W, V>(weight, at.base[i], (A)1, w[i]);
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0;
  }
  Raw<T, V> next_x[ITER], next_d[ITER];
  A next_mean, next_rstd;
  auto fetch = [&](int64_t row) {
    const int64_t r = GROUPS == 1 || row < rows ? row : 0;
    next_mean = mean_in[r], next_rstd = rstd_in[r];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      next_d[i] = raw_at<T, V>(dy + r * ldd + at.base[i]);
      next_x[i] = raw_at<T, V>(x + r * ldx + at.base[i]);
    }
  };
  int64_t first = (int64_t)blockIdx.x * GROUPS;
  if (AHEAD && first < rows) fetch(first + threadIdx.x / LANES);
  for (int turn = 0; first < rows; turn ^= 1) {
    const int64_t row = first + threadIdx.x / LANES;
    if (!AHEAD) fetch(row);
    const bool live = GROUPS == 1 || row < rows;                 // lanes of no row add zeros
    first += (int64_t)gridDim.x * GROUPS;
    const A mean = next_mean, rstd = next_rstd;
    A h[ITER][V], g[ITER][V], s[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        h[i][k] = live ? ((A)next_x[i].v[k] - mean) * rstd : (A)0;
        g[i][k] = live ? (A)next_d[i].v[k] : (A)0;
      }
    if (AHEAD && first < rows) fetch(first + threadIdx.x / LANES);
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      A wi[V];
      if constexpr (KEEP) {
#pragma unroll
        for (int k = 0; k < V; ++k) wi[k] = w[i][k];
      } else {
        weights_at<W, V>(weight, at.base[i], (A)1, wi);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dw[i][k] += g[i][k] * h[i][k];
        db[i][k] += g[i][k];
        g[i][k] *= wi[k];
        const bool mine = EXACT || k >= at.skip[i];
        s[0] += mine ? g[i][k] : (A)0;
        s[1] += mine ? g[i][k] * h[i][k] : (A)0;
      }
    }
    if (dx) {
      row_sum<LANES>(s, sh + (LANES > 64 ? turn * 2 * WAVES : 0));   // (two slots in turn: a wave may be a row ahead of the slowest)
      const A c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) g[i][k] = rstd * (g[i][k] - c1 - h[i][k] * c2);
        if (live && (EXACT || at.skip[i] < V)) put<T, V>(dx + row * cols + at.base[i], g[i]);
      }
    }
  }
  if (!partial) return;
  const bool alone = gridDim.x == 1;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    A* out = partial + ((int64_t)blockIdx.x * 2 + which) * cols;
    W* last = which ? dbias : dweight;
    if (alone && !last) continue;
    if constexpr (LANES > 64) {
#pragma unroll
      for (int i = 0; i < ITER; ++i)
        if (EXACT || at.skip[i] < V) {
          if (alone) put<W, V>(last + at.base[i], which ? db[i] : dw[i]);
          else put<A, V>(out + at.base[i], which ? db[i] : dw[i]);
        }
    } else {
      const int wave = threadIdx.x >> 6;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          A v = which ? db[i][k] : dw[i][k];
          if constexpr (LANES == 16) {
            v += __shfl_xor(v, 16);
            v += __shfl_xor(v, 32);
          }
          if ((threadIdx.x & 63) < LANES) sh[((wave * ITER + i) * LANES + lane) * V + k] = v;
        }
      __syncthreads();
      for (int c = threadIdx.x; c < ITER * LANES * V; c += THREADS) {
        A v = 0;
        for (int w = 0; w < WAVES; ++w) v += sh[w * ITER * LANES * V + c];
        const int nominal = c / V * V, col = min(nominal, (int)cols - V) + c % V;
        if (nominal < cols) {
          if (alone) last[col] = (W)v;
          else out[col] = v;
        }
      }
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_backward_wide_kernel(const T* __restrict__ dy, int64_t ldd, const T* __restrict__ x, int64_t ldx,
                                                                  const typename Wide<T>::type* __restrict__ mean_in,
                                                                  const typename Wide<T>::type* __restrict__ rstd_in, const W* __restrict__ weight,
                                                                  int64_t cols, T* __restrict__ dx) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>();
  __shared__ A sh[2 * 16];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  const T* dr = dy + row * ldd;
  const A mean = mean_in[row], rstd = rstd_in[row], inv = (A)1 / (A)cols;
  A s[2] = {0, 0};
  // g = dy w and h of a lane's four vectors
  auto load = [&](const int64_t (&base)[4], A (&g)[4][V], A (&h)[4][V]) {
    Raw<T, V> a[4], b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      a[u] = raw_at<T, V>(dr + base[u]);
      b[u] = raw_at<T, V>(xr + base[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      A w[V];
      weights_at<W, V>(weight, base[u], (A)1, w);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        g[u][k] = (A)a[u].v[k] * w[k];
        h[u][k] = ((A)b[u].v[k] - mean) * rstd;
      }
    }
  };
  wide_row<V>(cols, [&](const int64_t (&base)[4], const int (&skip)[4]) {
    A g[4][V], h[4][V];
    load(base, g, h);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        s[0] += k >= skip[u] ? g[u][k] : (A)0;
        s[1] += k >= skip[u] ? g[u][k] * h[u][k] : (A)0;
      }
  });
  row_sum<1024>(s, sh);
  const A c1 = s[0] * inv, c2 = s[1] * inv;
  wide_row<V>(cols, [&](const int64_t (&base)[4], const int (&skip)[4]) {
    A g[4][V], h[4][V];
    load(base, g, h);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int k = 0; k < V; ++k) g[u][k] = rstd * (g[u][k] - c1 - h[u][k] * c2);
      if (skip[u] < V) put<T, V>(dx + row * cols + base[u], g[u]);
    }
  });
}

// Rows shorter than a vector: a lane each, in registers.  4 000 000 x 3 of bf16 take 19 us, 37 us backward; with a workgroup a row, as the long rows have, they
// took 26 000 us.
template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_forward_narrow_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ weight, const W* __restrict__ bias,
                                                                  typename Wide<T>::type eps, int64_t rows, int cols, T* __restrict__ y, int64_t ldy,
                                                                  typename Wide<T>::type* __restrict__ mean_out, typename Wide<T>::type* __restrict__ rstd_out) {
  typedef typename Wide<T>::type A;
  constexpr int MOST = vec_of<T>() - 1;
  const A inv = (A)1 / (A)cols;
  A w[MOST], b[MOST];
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    w[k] = weight && k < cols ? (A)weight[k] : (A)1;
    b[k] = bias && k < cols ? (A)bias[k] : (A)0;
  }
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < rows; row += (int64_t)gridDim.x * 256) {
    A v[MOST], s = 0, q = 0, off = 0;
#pragma unroll
    for (int k = 0; k < MOST; ++k) v[k] = k < cols ? (A)x[row * ldx + k] : (A)0;
#pragma unroll
    for (int k = 0; k < MOST; ++k) s += v[k];
    const A mean = s / (A)cols;
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
      v[k] -= mean;
      const A d = k < cols ? v[k] : (A)0;
      q += d * d;
      if constexpr (refined<T>()) off += d;
    }
    off *= inv;
    const A rstd = reciprocal_root<A>(variance(q * inv, off) + eps);
    if (mean_out) {
      mean_out[row] = mean + off;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < MOST; ++k)
      if (k < cols) y[row * ldy + k] = (T)((v[k] - off) * rstd * w[k] + b[k]);
  }
}

// as norm_backward_kernel
template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_backward_narrow_kernel(const T* __restrict__ dy, int64_t ldd, const T* __restrict__ x, int64_t ldx,
                                                                   const typename Wide<T>::type* __restrict__ mean_in,
                                                                   const typename Wide<T>::type* __restrict__ rstd_in, const W* __restrict__ weight,
                                                                   int64_t rows, int cols, T* __restrict__ dx, typename Wide<T>::type* __restrict__ partial,
                                                                   W* __restrict__ dweight, W* __restrict__ dbias) {
  typedef typename Wide<T>::type A;
  constexpr int MOST = vec_of<T>() - 1;
  __shared__ A sh[4][2][MOST];
  const A inv = (A)1 / (A)cols;
  A w[MOST], sum[2][MOST];
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    w[k] = weight && k < cols ? (A)weight[k] : (A)1;
    sum[0][k] = sum[1][k] = 0;
  }
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < rows; row += (int64_t)gridDim.x * 256) {
    const A mean = mean_in[row], rstd = rstd_in[row];
    A h[MOST], g[MOST], c1 = 0, c2 = 0;
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
      g[k] = k < cols ? (A)dy[row * ldd + k] : (A)0;
      h[k] = k < cols ? ((A)x[row * ldx + k] - mean) * rstd : (A)0;
    }
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
      sum[0][k] += g[k] * h[k];
      sum[1][k] += g[k];
      g[k] *= w[k];
      c1 += g[k];
      c2 += g[k] * h[k];
    }
    c1 *= inv;
    c2 *= inv;
#pragma unroll
    for (int k = 0; k < MOST; ++k)
      if (dx && k < cols) dx[row * cols + k] = (T)(rstd * (g[k] - c1 - h[k] * c2));
  }
  if (!partial) return;
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
      const A v = group_sum<64>(sum[which][k]);
      if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6][which][k] = v;
    }
  __syncthreads();
  const int which = threadIdx.x / MOST, k = threadIdx.x % MOST;
  if (which > 1 || k >= cols) return;
  A v = sh[0][which][k];
  for (int wave = 1; wave < 4; ++wave) v += sh[wave][which][k];
  W* last = which ? dbias : dweight;
  if (gridDim.x > 1) partial[((int64_t)blockIdx.x * 2 + which) * cols + k] = v;
  else if (last) last[k] = (W)v;
}

// column sums of rows blockIdx.y, blockIdx.y + gridDim.y, ...: four waves of rows x 64 vectors, the waves added in their order
template <typename T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const T* __restrict__ dy, int64_t ldd, const T* __restrict__ x, int64_t ldx,
                                                           const typename Wide<T>::type* __restrict__ mean_in,
                                                           const typename Wide<T>::type* __restrict__ rstd_in, int64_t rows, int64_t cols,
                                                           typename Wide<T>::type* __restrict__ partial) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>();
  __shared__ A sh[2][4][64 * V];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const int64_t nominal = ((int64_t)blockIdx.x * 64 + lane) * V, base = nominal < cols - V ? nominal : cols - V;
  A dw[V], db[V];
#pragma unroll
  for (int k = 0; k < V; ++k) dw[k] = db[k] = 0;
#pragma unroll 2
  for (int64_t r = (int64_t)blockIdx.y * 4 + part; r < rows; r += (int64_t)gridDim.y * 4) {
    const Raw<T, V> d = raw_at<T, V>(dy + r * ldd + base), v = raw_at<T, V>(x + r * ldx + base);
    const A mean = mean_in[r], rstd = rstd_in[r];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      dw[k] += (A)d.v[k] * (((A)v.v[k] - mean) * rstd);
      db[k] += (A)d.v[k];
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    sh[0][part][lane * V + k] = dw[k];
    sh[1][part][lane * V + k] = db[k];
  }
  __syncthreads();
  if (part < 2 && nominal < cols) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      A v = 0;
      for (int w = 0; w < 4; ++w) v += sh[part][w][lane * V + k];
      partial[((int64_t)blockIdx.y * 2 + part) * cols + base + k] = v;
    }
  }
}

// lanes that share a row, vectors a lane holds of it, workgroup size; lanes = 1: rows shorter than a vector, lanes = 0: the kernels for wide rows
struct Shape { int lanes, iter, threads; };

// Vectors that a lane may hold, below 1024 lanes and with them (128 registers each).  Forward (the row and two weights): two of 16-bit elements, else four; with
// 1024 lanes four (4096 x 20000 of bf16 86 us, 126 by the kernel for wide rows).  Backward (five arrays of the row): two, four of fp32 at 1024 lanes.
Shape shape_of(int64_t cols, int vec, int most, int most_1024) {
  if (cols < vec) return {1, 1, 256};
  for (int lanes : {16, 64, 256, 1024}) {
    const int limit = lanes == 1024 ? most_1024 : most;
    const int64_t vectors = ceil_div(cols, (int64_t)lanes * vec);
    if (vectors <= limit) return {lanes, vectors <= 1 ? 1 : vectors <= 2 ? 2 : 4, lanes <= 256 ? 256 : 1024};
  }
  return {0, 0, 1024};
}

// workgroups of the backward pass: enough to fill the card, few enough that their column sums stay small beside the rows; one for up to four rows each of
// its groups of lanes, which then needs no second launch
int64_t backward_groups(const Shape& s, int64_t rows) {
  const int64_t per = s.lanes ? s.threads / s.lanes : 4;
  const int64_t most = s.threads == 1024 ? 256 : 1024;
  const int64_t n = ceil_div(rows, per);
  return n <= 4 ? 1 : n < most ? n : most;
}

template <typename T, typename W>
struct Norm {
  typedef typename Wide<T>::type A;
  static constexpr int V = vec_of<T>();

  template <int LANES, int ITER, int THREADS>
  static void forward_as(const vmcpde_norm_args& a, hipStream_t s) {
    if (a.cols == (int64_t)LANES * ITER * V) forward_exactly<LANES, ITER, THREADS, true>(a, s);
    else forward_exactly<LANES, ITER, THREADS, false>(a, s);
  }
  template <int LANES, int ITER, int THREADS, bool EXACT>
  static void forward_exactly(const vmcpde_norm_args& a, hipStream_t s) {
    norm_forward_kernel<T, W, LANES, ITER, THREADS, EXACT><<<(unsigned)std::min<int64_t>(ceil_div(a.rows, THREADS / LANES), THREADS == 1024 ? 512 : 2048), THREADS, 0, s>>>(
        static_cast<const T*>(a.x), a.ldx, static_cast<const W*>(a.weight), static_cast<const W*>(a.bias), (A)a.eps, a.rows, a.cols, static_cast<T*>(a.y), a.ldy,
        static_cast<A*>(a.mean), static_cast<A*>(a.rstd));
  }
  template <int LANES, int THREADS>
  static void forward_iter(int iter, const vmcpde_norm_args& a, hipStream_t s) {
    if (iter == 1) forward_as<LANES, 1, THREADS>(a, s);
    else if (iter == 2) forward_as<LANES, 2, THREADS>(a, s);
    else if constexpr (sizeof(T) > 2 || LANES == 1024) forward_as<LANES, 4, THREADS>(a, s);
  }
  static void forward(const vmcpde_norm_args& a, hipStream_t s) {
    const Shape p = shape_of(a.cols, V, sizeof(T) == 2 ? 2 : 4, 4);
    if (p.lanes == 1)
      norm_forward_narrow_kernel<T, W><<<(unsigned)std::min<int64_t>(ceil_div(a.rows, 256), 4096), 256, 0, s>>>(
          static_cast<const T*>(a.x), a.ldx, static_cast<const W*>(a.weight), static_cast<const W*>(a.bias), (A)a.eps, a.rows, (int)a.cols, static_cast<T*>(a.y), a.ldy,
          static_cast<A*>(a.mean), static_cast<A*>(a.rstd));
    else if (p.lanes == 16) forward_iter<16, 256>(p.iter, a, s);
    else if (p.lanes == 64) forward_iter<64, 256>(p.iter, a, s);
    else if (p.lanes == 256) forward_iter<256, 256>(p.iter, a, s);
    else if (p.lanes == 1024) forward_iter<1024, 1024>(p.iter, a, s);
    else
      norm_forward_wide_kernel<T, W><<<(unsigned)a.rows, 1024, 0, s>>>(static_cast<const T*>(a.x), a.ldx, static_cast<const W*>(a.weight), static_cast<const W*>(a.bias),
                                                                       (A)a.eps, a.cols, static_cast<T*>(a.y), a.ldy, static_cast<A*>(a.mean), static_cast<A*>(a.rstd));
  }

  template <int LANES, int ITER, int THREADS>
  static void backward_as(const vmcpde_norm_args& a, int64_t groups, A* partial, hipStream_t s) {
    if (a.cols == (int64_t)LANES * ITER * V) backward_exactly<LANES, ITER, THREADS, true>(a, groups, partial, s);
    else backward_exactly<LANES, ITER, THREADS, false>(a, groups, partial, s);
  }
  template <int LANES, int ITER, int THREADS, bool EXACT>
  static void backward_exactly(const vmcpde_norm_args& a, int64_t groups, A* partial, hipStream_t s) {
    norm_backward_kernel<T, W, LANES, ITER, THREADS, EXACT><<<(unsigned)groups, THREADS, 0, s>>>(
        static_cast<const T*>(a.dy), a.ldd, static_cast<const T*>(a.x), a.ldx, static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd),
        static_cast<const W*>(a.weight), a.rows, a.cols, static_cast<T*>(a.dx), partial, static_cast<W*>(a.dweight), static_cast<W*>(a.dbias));
  }
  template <int LANES, int THREADS>
  static void backward_iter(int iter, const vmcpde_norm_args& a, int64_t groups, A* partial, hipStream_t s) {
    if (iter == 1) backward_as<LANES, 1, THREADS>(a, groups, partial, s);
    else backward_as<LANES, 2, THREADS>(a, groups, partial, s);
  }
  static void backward(const vmcpde_norm_args& a, void* workspace, hipStream_t s) {
    const Shape p = shape_of(a.cols, V, 2, sizeof(T) == 4 ? 4 : 2);
    const int64_t groups = backward_groups(p, a.rows);
    A* partial = a.dweight || a.dbias ? static_cast<A*>(workspace) : nullptr;
    if (p.lanes == 1)
      norm_backward_narrow_kernel<T, W><<<(unsigned)groups, 256, 0, s>>>(
          static_cast<const T*>(a.dy), a.ldd, static_cast<const T*>(a.x), a.ldx, static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd),
          static_cast<const W*>(a.weight), a.rows, (int)a.cols, static_cast<T*>(a.dx), partial, static_cast<W*>(a.dweight), static_cast<W*>(a.dbias));
    else if (p.lanes == 16) backward_iter<16, 256>(p.iter, a, groups, partial, s);
    else if (p.lanes == 64) backward_iter<64, 256>(p.iter, a, groups, partial, s);
    else if (p.lanes == 256) backward_iter<256, 256>(p.iter, a, groups, partial, s);
    else if (p.lanes == 1024 && p.iter <= 2) backward_iter<1024, 1024>(p.iter, a, groups, partial, s);
    else if (p.lanes == 1024) {
      if constexpr (sizeof(T) == 4) backward_as<1024, 4, 1024>(a, groups, partial, s);
    } else {
      if (a.dx && a.rows)
        norm_backward_wide_kernel<T, W><<<(unsigned)a.rows, 1024, 0, s>>>(static_cast<const T*>(a.dy), a.ldd, static_cast<const T*>(a.x), a.ldx,
                                                                          static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd),
                                                                          static_cast<const W*>(a.weight), a.cols, static_cast<T*>(a.dx));
      if (partial)
        norm_columns_kernel<T><<<dim3((unsigned)ceil_div(a.cols, 64 * V), (unsigned)groups), 256, 0, s>>>(
            static_cast<const T*>(a.dy), a.ldd, static_cast<const T*>(a.x), a.ldx, static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd), a.rows, a.cols,
            partial);
    }
    if (partial && (groups > 1 || !p.lanes))
      add_columns<A, W>(partial, groups, 2 * a.cols, a.cols, a.cols, static_cast<W*>(a.dweight), static_cast<W*>(a.dbias), s);
  }
};

// calls F<T, W> of the element type and the weights' type
template <typename F>
int by_types(const vmcpde_norm_args& a, F f) {
  switch (a.dtype) {
    case VMCPDE_F64: f(Norm<double, double>()); break;
    case VMCPDE_F32: f(Norm<float, float>()); break;
    case VMCPDE_F16: a.weight_dtype == VMCPDE_F32 ? f(Norm<f16_t, float>()) : f(Norm<f16_t, f16_t>()); break;
    default: a.weight_dtype == VMCPDE_F32 ? f(Norm<bf16_t, float>()) : f(Norm<bf16_t, bf16_t>());
  }
  VMC_CHECK_HIP(hipGetLastError());
  return 0;
}

int check(const vmcpde_norm_args* a) {
  VMC_REQUIRE(a, "layer norm: null arguments");
  VMC_REQUIRE(dtype_ok(a->dtype), "layer norm: type %d", a->dtype);
  VMC_REQUIRE(a->weight_dtype == a->dtype || (a->weight_dtype == VMCPDE_F32 && dtype_size(a->dtype) == 2),
              "layer norm: weights of type %d for elements of type %d (the same, or fp32 for 16-bit elements)", a->weight_dtype, a->dtype);
  VMC_REQUIRE(a->rows >= 0 && a->rows < (int64_t)1 << 31, "layer norm: %lld rows", (long long)a->rows);
  VMC_REQUIRE(a->cols >= 1 && a->cols < (int64_t)1 << 27, "layer norm: %lld columns", (long long)a->cols);
  VMC_REQUIRE(a->rows < (int64_t)1 << 22 || shape_of(a->cols, 16 / dtype_size(a->dtype), 2, a->dtype == VMCPDE_F32 ? 4 : 2).lanes, "layer norm: %lld rows of %lld columns", (long long)a->rows, (long long)a->cols);   // (a workgroup each, and a launch has 2^32 lanes)
  VMC_REQUIRE(a->rows == 0 || (a->x && a->ldx >= a->cols), "layer norm: x is null or its row pitch %lld is below its %lld columns", (long long)a->ldx, (long long)a->cols);
  return 0;
}

}  // namespace

extern "C" {

int vmcpde_layer_norm(const vmcpde_norm_args* a, void* stream) {
  if (const int rc = check(a)) return rc;
  VMC_REQUIRE(a->eps >= 0, "vmcpde_layer_norm: eps = %g", a->eps);
  VMC_REQUIRE(!a->mean == !a->rstd, "vmcpde_layer_norm: mean and rstd go together");
  if (a->rows == 0) return 0;
  VMC_REQUIRE(a->y && a->ldy >= a->cols, "vmcpde_layer_norm: y is null or its row pitch is below its columns");
  return by_types(*a, [&](auto norm) { norm.forward(*a, static_cast<hipStream_t>(stream)); });
}

int64_t vmcpde_layer_norm_backward_workspace_bytes(const vmcpde_norm_args* a) {
  if (check(a)) return -1;
  const Shape p = shape_of(a->cols, 16 / dtype_size(a->dtype), 2, a->dtype == VMCPDE_F32 ? 4 : 2);
  return backward_groups(p, a->rows) * 2 * a->cols * (a->dtype == VMCPDE_F64 ? 8 : 4);
}

int vmcpde_layer_norm_backward(const vmcpde_norm_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check(a)) return rc;
  VMC_REQUIRE(a->rows == 0 || (a->dy && a->ldd >= a->cols && a->mean && a->rstd), "vmcpde_layer_norm_backward: null dy, mean or rstd, or a row pitch below the columns");
  if (a->dweight || a->dbias) {
    const int64_t need = vmcpde_layer_norm_backward_workspace_bytes(a);
    VMC_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "vmcpde_layer_norm_backward: the workspace is not aligned to 16 bytes");
    VMC_REQUIRE(workspace && workspace_bytes >= need, "vmcpde_layer_norm_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  } else if (a->rows == 0 || !a->dx) {
    return 0;
  }
  return by_types(*a, [&](auto norm) { norm.backward(*a, workspace, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
