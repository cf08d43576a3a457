// The dense layer  y = scale * act(x W + b) + r  and its gradients (dz = scale * slope * dy: dx = dz W^T, dW = x^T dz, db = sum_rows dz).
#include <algorithm>

#include "layers.hpp"

using namespace vmcpde;

namespace {

// ---- the epilogue ------------------------------------------------------------------------------------------------------------------

// act(z) and act'(z)
template <typename A>
__device__ __forceinline__ void activate(int act, A z, A& a, A& slope) {
  if (act == VMCPDE_ACT_NONE) {
    a = z;
    slope = 1;
  } else if (act == VMCPDE_ACT_TANH) {
    a = sizeof(A) == 8 ? (A)tanh((double)z) : (A)tanhf((float)z);
    slope = 1 - a * a;
  } else if (act == VMCPDE_ACT_GELU) {
    A cdf, density;
    if constexpr (sizeof(A) == 8) {
      cdf = 0.5 * erfc(-z * 0.70710678118654752440);
      density = 0.39894228040143267794 * exp(-0.5 * z * z);
    } else {
      cdf = 0.5f * erfcf(-z * 0.70710678f);
      density = 0.39894228f * expf(-0.5f * z * z);
    }
    a = z * cdf;
    slope = density != 0 ? cdf + z * density : cdf;      // (z = -inf: no inf * 0)
    if (z == -(A)INFINITY) a = 0;
  } else {
    const A e = sizeof(A) == 8 ? (A)exp(-(double)z) : (A)expf(-(float)z);
    const A gate = 1 / (1 + e);
    a = z == -(A)INFINITY ? 0 : z * gate;
    slope = gate != 0 && gate != 1 ? gate * (1 + z * (1 - gate)) : gate;
  }
}

template <typename T>
struct Epilogue {
  const T* bias;
  const T* residual;
  int64_t ldr;
  T* y;
  int64_t ldy;
  typename Slope<T>::type* slope;
  int64_t n;       // columns, the slope's pitch
  typename Wide<T>::type scale;
  int32_t act;
};

template <typename T, typename A>
__device__ __forceinline__ void finish(const Epilogue<T>& e, int64_t row, int64_t col, A z) {
  A a, slope;
  if (e.bias) z += (A)e.bias[col];
  activate<A>(e.act, z, a, slope);
  a *= e.scale;
  if (e.residual) a += (A)e.residual[row * e.ldr + col];
  e.y[row * e.ldy + col] = (T)a;
  if (e.slope) e.slope[row * e.n + col] = (typename Slope<T>::type)slope;
}

// ---- products ----------------------------------------------------------------------------------------------------------------------

// C [m][n] = sum_k P(row, k) Q(k, col).  An operand lies along k (element (r, k) at r * ld + k), or with `across` along its rows / columns
// (k * ld + r).
struct Product {
  const void* p;
  const void* q;
  int64_t ldp, ldq;
  int32_t m, n, k;
  int32_t p_across, q_across;
};

template <typename A> struct Acc;
template <> struct Acc<float> { typedef float type __attribute__((ext_vector_type(4))); };
template <> struct Acc<double> { typedef double type __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ Acc<float>::type mfma(float a, float b, Acc<float>::type c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ Acc<double>::type mfma(double a, double b, Acc<double>::type c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
// row of the 16 x 16 block that register `reg` of a lane with lane / 16 = g holds (the column is lane % 16)
template <typename A> __device__ __forceinline__ int block_row(int g, int reg) { return sizeof(A) == 8 ? g + 4 * reg : g * 4 + reg; }

constexpr int WIDE_K = 16;

// One step of an operand, 16 k x R rows: global -> registers, registers -> LDS [k][row].  Coalesced along whichever axis lies in memory.
template <typename T, typename A, int R>
struct WideStep {
  static constexpr int E = R * WIDE_K / 256;
  A v[E];
  __device__ __forceinline__ void load(const T* __restrict__ base, int64_t ld, int across, int row0, int rows, int k0, int k_end) {
    const int t = threadIdx.x;
    const bool inside = row0 + R <= rows && k0 + WIDE_K <= k_end;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int r = row0 + (across ? t % R : t / WIDE_K + j * (256 / WIDE_K)), k = k0 + (across ? t / R + j * (256 / R) : t % WIDE_K);
      v[j] = inside || (r < rows && k < k_end) ? (A)base[across ? k * ld + r : r * ld + k] : (A)0;
    }
  }
  __device__ __forceinline__ void store(A* __restrict__ lds, int across) const {
    const int t = threadIdx.x;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int r = across ? t % R : t / WIDE_K + j * (256 / WIDE_K), k = across ? t / R + j * (256 / R) : t % WIDE_K;
      lds[k * (R + 16) + r] = v[j];
    }
  }
};

// BM x BN of C per workgroup of four waves, WM x WN blocks of 16 x 16 a wave; slice blockIdx.y of the k range, `part` != null: its sums
template <typename T, int BM, int BN, int WAVES_M>
__global__ __launch_bounds__(256) void product_wide_kernel(Product g, int tiles_n, int k_slice, typename Wide<T>::type* __restrict__ part, Epilogue<T> e) {
  typedef typename Wide<T>::type A;
  constexpr int WAVES_N = 4 / WAVES_M, WM = BM / WAVES_M / 16, WN = BN / WAVES_N / 16, LP = BM + 16, LQ = BN + 16;
  __shared__ A lp[2][WIDE_K * LP], lq[2][WIDE_K * LQ];
  const int row0 = (blockIdx.x / tiles_n) * BM, col0 = (blockIdx.x % tiles_n) * BN;
  const int k_begin = blockIdx.y * k_slice, k_end = k_begin + k_slice < g.k ? k_begin + k_slice : g.k;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q4 = lane >> 4;
  const int wr = (wave / WAVES_N) * WM * 16, wc = (wave % WAVES_N) * WN * 16;
  typename Acc<A>::type acc[WM][WN];
#pragma unroll
  for (int a = 0; a < WM; ++a)
#pragma unroll
    for (int b = 0; b < WN; ++b) acc[a][b] = {0, 0, 0, 0};
  const T* p = static_cast<const T*>(g.p);
  const T* q = static_cast<const T*>(g.q);
  WideStep<T, A, BM> sp;
  WideStep<T, A, BN> sq;
  sp.load(p, g.ldp, g.p_across, row0, g.m, k_begin, k_end);
  sq.load(q, g.ldq, g.q_across, col0, g.n, k_begin, k_end);
  sp.store(lp[0], g.p_across);
  sq.store(lq[0], g.q_across);
  __syncthreads();
  int buf = 0;
  for (int k0 = k_begin; k0 < k_end; k0 += WIDE_K, buf ^= 1) {
    const bool more = k0 + WIDE_K < k_end;
    if (more) {
      sp.load(p, g.ldp, g.p_across, row0, g.m, k0 + WIDE_K, k_end);
      sq.load(q, g.ldq, g.q_across, col0, g.n, k0 + WIDE_K, k_end);
    }
#pragma unroll
    for (int s = 0; s < WIDE_K / 4; ++s) {
      A fp[WM], fq[WN];
#pragma unroll
      for (int a = 0; a < WM; ++a) fp[a] = lp[buf][(s * 4 + q4) * LP + wr + a * 16 + i];
#pragma unroll
      for (int b = 0; b < WN; ++b) fq[b] = lq[buf][(s * 4 + q4) * LQ + wc + b * 16 + i];
#pragma unroll
      for (int a = 0; a < WM; ++a)
#pragma unroll
        for (int b = 0; b < WN; ++b) acc[a][b] = mfma(fp[a], fq[b], acc[a][b]);
    }
    if (more) {
      sp.store(lp[buf ^ 1], g.p_across);      // (the other buffer: its last readers passed the barrier of the step before)
      sq.store(lq[buf ^ 1], g.q_across);
    }
    __syncthreads();
  }
#pragma unroll
  for (int a = 0; a < WM; ++a)
#pragma unroll
    for (int reg = 0; reg < 4; ++reg) {
      const int row = row0 + wr + a * 16 + block_row<A>(q4, reg);
      if (row >= g.m) continue;
#pragma unroll
      for (int b = 0; b < WN; ++b) {
        const int col = col0 + wc + b * 16 + i;
        if (col >= g.n) continue;
        if (part) part[((int64_t)blockIdx.y * g.m + row) * g.n + col] = acc[a][b][reg];
        else finish<T, A>(e, row, col, acc[a][b][reg]);
      }
    }
}

// the slices' sums added in their order, and the epilogue
template <typename T>
__global__ __launch_bounds__(256) void product_join_kernel(const typename Wide<T>::type* __restrict__ part, int slices, int64_t m, int64_t n, Epilogue<T> e) {
  typedef typename Wide<T>::type A;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= m * n) return;
  A z = 0;
  for (int s = 0; s < slices; ++s) z += part[(int64_t)s * m * n + at];
  finish<T, A>(e, at / n, at % n, z);
}

// ---- the gradient before the activation ----------------------------------------------------------------------------------------------

// dz = scale * slope * dy (dz may be null; its row pitch may exceed n: zeros there), and sums of its columns over the rows that this
// workgroup takes: partial[blockIdx.y][n] (may be null).  LANES lanes along the columns, 256 / LANES rows at a time.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void dense_dz_kernel(const T* __restrict__ dy, int64_t ldd, const typename Slope<T>::type* __restrict__ slope,
                                                       typename Wide<T>::type scale, int64_t rows, int64_t n, T* __restrict__ dz, int64_t ldz,
                                                       typename Wide<T>::type* __restrict__ partial) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>(), ROWS = 256 / LANES;
  __shared__ A sh[ROWS][LANES * V];
  const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
  const int64_t col = ((int64_t)blockIdx.x * LANES + lane) * V;
  A sum[V];
#pragma unroll
  for (int k = 0; k < V; ++k) sum[k] = 0;
  for (int64_t r = (int64_t)blockIdx.y * ROWS + part; r < rows; r += (int64_t)gridDim.y * ROWS) {
    A v[V], s[V];
    load_vec<T, V>(dy + r * ldd, col, n, v);
    if (slope) load_vec<typename Slope<T>::type, V>(slope + r * n, col, n, s);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      v[k] *= scale;
      if (slope) v[k] *= s[k];
      if (col + k >= n) v[k] = 0;
      sum[k] += v[k];
    }
    if (dz) store_vec<T, V>(dz + r * ldz, col, ldz, v);
  }
  if (!partial) return;
#pragma unroll
  for (int k = 0; k < V; ++k) sh[part][lane * V + k] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < LANES * V; c += 256) {
    A v = 0;
    for (int p = 0; p < ROWS; ++p) v += sh[p][c];
    const int64_t to = (int64_t)blockIdx.x * LANES * V + c;
    if (to < n) partial[blockIdx.y * n + to] = v;
  }
}

// ---- plans ---------------------------------------------------------------------------------------------------------------------------

struct Tiles { int bm, bn, slices, k_slice; };

template <typename T>
Tiles tiles_of(int64_t m, int64_t n, int64_t k) {
  Tiles t;
  t.bm = m <= 32 ? 32 : 128;
  t.bn = n <= 32 ? 32 : 128;
  const int64_t tiles = ceil_div(m, t.bm) * ceil_div(n, t.bn);
  int64_t slices = 1;
  if (tiles > 0 && tiles < 256) slices = std::min<int64_t>(std::min<int64_t>(ceil_div(512, tiles), ceil_div(k, 4 * WIDE_K)), 512);
  if (slices < 1) slices = 1;
  t.k_slice = (int)round_up(ceil_div(k, slices), WIDE_K);
  if (t.k_slice < WIDE_K) t.k_slice = WIDE_K;
  t.slices = (int)std::max<int64_t>(1, ceil_div(k, t.k_slice));
  return t;
}

template <typename T>
int64_t product_bytes(int64_t m, int64_t n, int64_t k) {
  const Tiles t = tiles_of<T>(m, n, k);
  return t.slices > 1 ? round_up((int64_t)t.slices * m * n * (int64_t)sizeof(typename Wide<T>::type), 256) : 0;
}

template <typename T>
void product(const Product& g, const Epilogue<T>& e, void* workspace, hipStream_t s) {
  typedef typename Wide<T>::type A;
  const Tiles t = tiles_of<T>(g.m, g.n, g.k);
  A* part = t.slices > 1 ? static_cast<A*>(workspace) : nullptr;
  const int tiles_n = (int)ceil_div(g.n, t.bn);
  const dim3 grid((unsigned)(ceil_div(g.m, t.bm) * tiles_n), (unsigned)t.slices);
  if (t.bm == 128 && t.bn == 128) product_wide_kernel<T, 128, 128, 2><<<grid, 256, 0, s>>>(g, tiles_n, t.k_slice, part, e);
  else if (t.bm == 128) product_wide_kernel<T, 128, 32, 4><<<grid, 256, 0, s>>>(g, tiles_n, t.k_slice, part, e);
  else if (t.bn == 128) product_wide_kernel<T, 32, 128, 1><<<grid, 256, 0, s>>>(g, tiles_n, t.k_slice, part, e);
  else product_wide_kernel<T, 32, 32, 2><<<grid, 256, 0, s>>>(g, tiles_n, t.k_slice, part, e);
  if (part) product_join_kernel<T><<<(unsigned)ceil_div((int64_t)g.m * g.n, 256), 256, 0, s>>>(part, t.slices, g.m, g.n, e);
}

// workgroups along the rows of the dz kernel
int64_t dz_groups(int64_t rows, int64_t cols_blocks, int rows_at_once) {
  const int64_t want = std::max<int64_t>(1, 2048 / cols_blocks), have = std::max<int64_t>(1, ceil_div(rows, rows_at_once));
  return std::min<int64_t>(std::min<int64_t>(want, have), 512);
}

template <typename T>
struct Backward {
  typedef typename Wide<T>::type A;
  bool need_dz, own_dz;          // dz is used by a product; dz is not dy itself
  int lanes;
  int64_t ldz, groups, dz_bytes, part_bytes, product_bytes_, total;
  explicit Backward(const vmcpde_dense_args& a) {
    need_dz = a.dx || a.dkernel;
    own_dz = need_dz && (a.slope || a.scale != 1.0);
    lanes = a.n_out <= 8 * vec_of<T>() ? 8 : 32;
    ldz = own_dz ? a.n_out : a.ldd;
    groups = dz_groups(a.rows, ceil_div(a.n_out, lanes * vec_of<T>()), 256 / lanes);
    dz_bytes = own_dz ? round_up(a.rows * ldz * (int64_t)sizeof(T), 256) : 0;
    part_bytes = a.dbias ? round_up(groups * a.n_out * (int64_t)sizeof(A), 256) : 0;
    product_bytes_ = std::max(a.dx ? product_bytes<T>(a.rows, a.n_in, a.n_out) : 0, a.dkernel ? product_bytes<T>(a.n_in, a.n_out, a.rows) : 0);
    total = dz_bytes + part_bytes + product_bytes_;
  }
};

template <typename T>
struct Dense {
  typedef typename Wide<T>::type A;
  typedef typename Slope<T>::type S;

  static int64_t bytes(const vmcpde_dense_args& a, bool backward) { return backward ? Backward<T>(a).total : product_bytes<T>(a.rows, a.n_out, a.n_in); }

  static void forward(const vmcpde_dense_args& a, void* workspace, hipStream_t s) {
    const Epilogue<T> e = {static_cast<const T*>(a.bias), static_cast<const T*>(a.residual), a.ldr, static_cast<T*>(a.y), a.ldy, static_cast<S*>(a.slope), a.n_out,
                           (A)a.scale, a.activation};
    product<T>({a.x, a.kernel, a.ldx, a.ldk, (int32_t)a.rows, (int32_t)a.n_out, (int32_t)a.n_in, 0, !a.kernel_t}, e, workspace, s);
  }

  static void backward(const vmcpde_dense_args& a, void* workspace, hipStream_t s) {
    const Backward<T> b(a);
    char* at = static_cast<char*>(workspace);
    T* own = b.own_dz ? reinterpret_cast<T*>(at) : nullptr;
    A* partial = a.dbias ? reinterpret_cast<A*>(at + b.dz_bytes) : nullptr;
    void* rest = at + b.dz_bytes + b.part_bytes;
    if (own || partial) {
      const T* dy = static_cast<const T*>(a.dy);
      const S* slope = static_cast<const S*>(a.slope);
      const dim3 grid((unsigned)ceil_div(a.n_out, b.lanes * vec_of<T>()), (unsigned)b.groups);
      if (b.lanes == 8) dense_dz_kernel<T, 8><<<grid, 256, 0, s>>>(dy, a.ldd, slope, (A)a.scale, a.rows, a.n_out, own, b.ldz, partial);
      else dense_dz_kernel<T, 32><<<grid, 256, 0, s>>>(dy, a.ldd, slope, (A)a.scale, a.rows, a.n_out, own, b.ldz, partial);
      if (partial)
        add_columns_kernel<A, T><<<dim3((unsigned)ceil_div(a.n_out, 64), 1), 1024, 0, s>>>(partial, (int)b.groups, a.n_out, a.n_out, static_cast<T*>(a.dbias), nullptr);
    }
    const void* dz = own ? own : a.dy;
    if (a.dx && a.rows) {
      const Epilogue<T> e = {nullptr, nullptr, 0, static_cast<T*>(a.dx), a.n_in, nullptr, a.n_in, 1, VMCPDE_ACT_NONE};
      product<T>({dz, a.kernel, b.ldz, a.ldk, (int32_t)a.rows, (int32_t)a.n_in, (int32_t)a.n_out, 0, a.kernel_t}, e, rest, s);
    }
    if (a.dkernel) {
      const Epilogue<T> e = {nullptr, nullptr, 0, static_cast<T*>(a.dkernel), a.n_out, nullptr, a.n_out, 1, VMCPDE_ACT_NONE};
      product<T>({a.x, dz, a.ldx, b.ldz, (int32_t)a.n_in, (int32_t)a.n_out, (int32_t)a.rows, 1, 1}, e, rest, s);
    }
  }
};

template <typename F>
void by_type(int dtype, F f) {
  switch (dtype) {
    case VMCPDE_F64: f(Dense<double>()); break;
    case VMCPDE_F32: f(Dense<float>()); break;
    case VMCPDE_F16: f(Dense<f16_t>()); break;
    default: f(Dense<bf16_t>());
  }
}

int check(const vmcpde_dense_args* a, bool backward) {
  constexpr int64_t LIMIT = (int64_t)1 << 30;
  VMC_REQUIRE(a, "dense: null arguments");
  VMC_REQUIRE(dtype_ok(a->dtype), "dense: type %d", a->dtype);
  VMC_REQUIRE(a->activation >= VMCPDE_ACT_NONE && a->activation <= VMCPDE_ACT_SILU, "dense: activation %d", a->activation);
  VMC_REQUIRE(a->rows >= 0 && a->rows < LIMIT && a->n_in >= 1 && a->n_in < LIMIT && a->n_out >= 1 && a->n_out < LIMIT,
              "dense: rows %lld, n_in %lld, n_out %lld (rows from 0, widths from 1, all below 2^30)", (long long)a->rows, (long long)a->n_in, (long long)a->n_out);
  VMC_REQUIRE(a->scale == a->scale, "dense: scale is NaN");
  VMC_REQUIRE(ceil_div(std::max(a->rows, a->n_in), 32) * ceil_div(std::max(a->n_in, a->n_out), 32) < (int64_t)1 << 31, "dense: more than 2^31 tiles");
  const int64_t kernel_row = a->kernel_t ? a->n_in : a->n_out;
  const bool need_x = (!backward && a->rows) || (backward && a->dkernel && a->rows), need_kernel = !backward || a->dx;
  VMC_REQUIRE(!need_x || (a->x && a->ldx >= a->n_in), "dense: x is null or its row pitch %lld is below n_in %lld", (long long)a->ldx, (long long)a->n_in);
  VMC_REQUIRE(!need_kernel || (a->kernel && a->ldk >= kernel_row), "dense: kernel is null or its row pitch %lld is below %lld", (long long)a->ldk, (long long)kernel_row);
  if (!backward) {
    VMC_REQUIRE(a->rows == 0 || (a->y && a->ldy >= a->n_out), "dense: y is null or its row pitch %lld is below n_out %lld", (long long)a->ldy, (long long)a->n_out);
    VMC_REQUIRE(!a->residual || a->ldr >= a->n_out, "dense: the residual's row pitch %lld is below n_out %lld", (long long)a->ldr, (long long)a->n_out);
  } else {
    VMC_REQUIRE(a->rows == 0 || (a->dy && a->ldd >= a->n_out), "dense: dy is null or its row pitch %lld is below n_out %lld", (long long)a->ldd, (long long)a->n_out);
  }
  return 0;
}

}  // namespace

extern "C" {

int64_t vmcpde_dense_workspace_bytes(const vmcpde_dense_args* a, int32_t backward) {
  if (check(a, backward != 0)) return -1;
  int64_t n = 0;
  by_type(a->dtype, [&](auto d) { n = d.bytes(*a, backward != 0); });
  return n;
}

static int run(const vmcpde_dense_args* a, bool backward, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check(a, backward)) return rc;
  if (!backward && a->rows == 0) return 0;
  const int64_t need = vmcpde_dense_workspace_bytes(a, backward);
  VMC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "dense: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  by_type(a->dtype, [&](auto d) {
    if (backward) d.backward(*a, workspace, static_cast<hipStream_t>(stream));
    else d.forward(*a, workspace, static_cast<hipStream_t>(stream));
  });
  VMC_CHECK_HIP(hipGetLastError());
  return 0;
}

int vmcpde_dense(const vmcpde_dense_args* a, void* workspace, int64_t workspace_bytes, void* stream) { return run(a, false, workspace, workspace_bytes, stream); }
int vmcpde_dense_backward(const vmcpde_dense_args* a, void* workspace, int64_t workspace_bytes, void* stream) { return run(a, true, workspace, workspace_bytes, stream); }

}  // extern "C"
