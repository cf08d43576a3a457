// The dense layer  y = scale * act(x W + b) + r  and its gradients (dz = scale * slope * dy: dx = dz W^T, dW = x^T dz, db = sum_rows dz).
#include <algorithm>
#include <cmath>

#include "layers.hpp"

using namespace vmcpde;

namespace {

// ---- the epilogue ------------------------------------------------------------------------------------------------------------------

// e^-x - 1 = 2^n p + 2^n - 1 for x >= 0: range reduction by ln 2, which is split in two so that n times its upper part is exact (Cody and Waite's way), and the Taylor series of e^r - 1 on |r| <= ln 2 / 2 (degree 13: remainder 4e-18 r, fp32
// degree 7: 1e-9 r), which leaves the small results their last places.  A quarter of the instructions of the library's functions, and no branches.
__device__ __forceinline__ double exp_minus_one(double x, double& two_n, double& p) {
  const double n = rint(x * -1.4426950408889634074);
  double r = fma(n, -0x1.62e42fefa3p-1, -x);
  r = fma(n, -0x1.3de6af278ece6p-42, r);
  p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p * r, r, r);
  two_n = ldexp(1.0, (int)n);
  return fma(two_n, p, two_n - 1.0);
}
__device__ __forceinline__ float exp_minus_one(float x, float& two_n, float& p) {
  const float n = rintf(x * -1.44269504f);
  float r = fmaf(n, -0x1.62ep-1f, -x);
  r = fmaf(n, -0x1.0bfbe8p-15f, r);
  p = 1.0f / 5040.0f;
  p = fmaf(p, r, 1.0f / 720.0f);
  p = fmaf(p, r, 1.0f / 120.0f);
  p = fmaf(p, r, 1.0f / 24.0f);
  p = fmaf(p, r, 1.0f / 6.0f);
  p = fmaf(p, r, 0.5f);
  p = fmaf(p * r, r, r);
  two_n = ldexpf(1.0f, (int)n);
  return fmaf(two_n, p, two_n - 1.0f);
}
// 1 / v for 1 <= v <= 2, within a unit in the last place
__device__ __forceinline__ double reciprocal(double v) {
  double q = __builtin_amdgcn_rcp(v);
  q = fma(fma(-v, q, 1.0), q, q);
  return fma(fma(-v, q, 1.0), q, q);
}
__device__ __forceinline__ float reciprocal(float v) {
  const float q = __builtin_amdgcn_rcpf(v);
  return fmaf(fmaf(-v, q, 1.0f), q, q);
}

// act(z) and act'(z), to a few units of the arithmetic type's last place
template <typename A>
__device__ __forceinline__ void activate_exact(int act, A z, A& a, A& slope) {
  const A x = fabs(z);
  if (act == VMCPDE_ACT_TANH) {             // with m = e^-2|z| - 1: tanh |z| = -m / (2 + m), the slope 4 (1 + m) / (2 + m)^2
    A two_n, p;
    const A m = exp_minus_one(x > 25 ? (A)50 : 2 * x, two_n, p), den = 2 + m, q = reciprocal(den);      // (NaN stays)
    A h = -m * q;
    h = fma(fma(-den, h, -m), q, h);
    a = copysign(h, z);
    slope = 4 * fma(two_n, p, two_n) * q * q;
  } else if (act == VMCPDE_ACT_GELU) {
    A cdf, density;
    if constexpr (sizeof(A) == 8) {
      cdf = 0.5 * erfc(-z * 0.70710678118654752440);
      density = 0.39894228040143267794 * exp(-0.5 * z * z);
    } else {
      cdf = 0.5f * erfcf(-z * 0.70710678f);
      density = 0.39894228f * expf(-0.5f * z * z);
    }
    a = z == -(A)INFINITY ? 0 : z * cdf;
    slope = density != 0 ? cdf + z * density : cdf;      // (z = +-inf: no inf * 0)
  } else {                                  // with e = e^-|z|: the gate is 1 / (1 + e), or e / (1 + e) for z < 0
    A two_n, p;
    const A far = sizeof(A) == 8 ? 800 : 120;
    const A q = reciprocal(2 + exp_minus_one(x > far ? far : x, two_n, p)), e = fma(two_n, p, two_n), gate = z < 0 ? e * q : q, rest = z < 0 ? q : e * q;
    a = z == -(A)INFINITY ? 0 : z * gate;
    slope = gate != 0 && rest != 0 ? gate * (1 + z * rest) : gate;
  }
}

// The same beside 16-bit elements, some 1e-7 absolute (2e-7 relative for small tanh), a tenth of the instructions: with the library's functions the
// epilogue of a large product took as long as a quarter of its multiplications.  erf: the rational approximation 7.1.26 of Abramowitz and Stegun.
__device__ __forceinline__ void activate_short(int act, const float z, float& a, float& slope) {
  const float x = fabsf(z);
  if (act == VMCPDE_ACT_TANH) {
    const float e = __expf(-2 * x), y = z * z;
    const float large = copysignf((1 - e) * __builtin_amdgcn_rcpf(1 + e), z);
    const float small = z * (1 + y * (-0.33333333f + y * (0.13333333f - y * 0.053968254f)));
    a = x < 0.2f ? small : large;
    slope = x < 0.2f ? 1 - a * a : 4 * e * __builtin_amdgcn_rcpf((1 + e) * (1 + e));
  } else if (act == VMCPDE_ACT_GELU) {
    const float e = __expf(-0.5f * z * z), t = __builtin_amdgcn_rcpf(1 + 0.3275911f * 0.70710678f * x);
    const float tail = 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    const float cdf = z < 0 ? tail : 1 - tail;
    a = z == -INFINITY ? 0 : z * cdf;
    slope = e != 0 ? cdf + z * (0.39894228f * e) : cdf;
  } else {
    const float gate = __builtin_amdgcn_rcpf(1 + __expf(-z));
    a = z == -INFINITY ? 0 : z * gate;
    slope = gate != 0 && gate != 1 ? gate * (1 + z * (1 - gate)) : gate;
  }
}

template <typename T, typename A>
__device__ __forceinline__ void activate(int act, A z, A& a, A& slope) {
  if (act == VMCPDE_ACT_NONE) {
    a = z;
    slope = 1;
  } else {
    activate_exact<A>(act, z, a, slope);
  }
}

// The choice is made once for all N (so that they overlap) and slopes are computed where they are wanted (one by one: 4096 x 4096 x 16384 with tanh 500 us, so 460;
// without activation 434).
template <int ACT, int N>
__device__ __forceinline__ void activate_shorts(bool want_slope, float (&z)[N], float (&slope)[N]) {
  if (want_slope) {
#pragma unroll
    for (int k = 0; k < N; ++k) activate_short(ACT, z[k], z[k], slope[k]);
  } else {
    float unused;
#pragma unroll
    for (int k = 0; k < N; ++k) activate_short(ACT, z[k], z[k], unused);
  }
}
template <int N>
__device__ __forceinline__ void activate_shorts(int act, bool want_slope, float (&z)[N], float (&slope)[N]) {
  if (act == VMCPDE_ACT_TANH) activate_shorts<VMCPDE_ACT_TANH, N>(want_slope, z, slope);
  else if (act == VMCPDE_ACT_GELU) activate_shorts<VMCPDE_ACT_GELU, N>(want_slope, z, slope);
  else if (act == VMCPDE_ACT_SILU) activate_shorts<VMCPDE_ACT_SILU, N>(want_slope, z, slope);
  else
#pragma unroll
    for (int k = 0; k < N; ++k) slope[k] = 1;
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

// N numbers as they lie in memory
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Held { T v[N]; };
// columns col .. col + N of a row, zero behind its end or without a row
template <typename T, int N>
__device__ __forceinline__ Held<T, N> held_at(const T* __restrict__ row, int64_t col, int64_t cols) {
  Held<T, N> h = {};
  if (!row) return h;
  if (col + N <= cols) return *reinterpret_cast<const Held<T, N>*>(row + col);
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (col + k < cols) h.v[k] = row[col + k];
  return h;
}

// columns col .. col + N of a row (those inside it), from their sums, the bias and the residual there
template <typename T, int N, typename A>
__device__ __forceinline__ void finish(const Epilogue<T>& e, int64_t row, int64_t col, A (&z)[N], const Held<T, N>& bias, const Held<T, N>& residual) {
  A slope[N];
  if (e.bias) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] += (A)bias.v[k];
  }
  activate_shorts<N>(e.act, e.slope != nullptr, z, slope);
#pragma unroll
  for (int k = 0; k < N; ++k) z[k] *= e.scale;
  if (e.residual) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] += (A)residual.v[k];
  }
  store_vec<T, N>(e.y + row * e.ldy, col, e.n, z);
  if (e.slope) store_vec<typename Slope<T>::type, N>(e.slope + row * e.n, col, e.n, slope);
}
template <typename T, int N>
__device__ __forceinline__ Held<T, N> residual_at(const Epilogue<T>& e, int64_t row, int64_t col) {
  return held_at<T, N>(e.residual ? e.residual + row * e.ldr : nullptr, col, e.n);
}
template <typename T, int N, typename A>
__device__ __forceinline__ void finish(const Epilogue<T>& e, int64_t row, int64_t col, A (&z)[N]) {
  if constexpr (sizeof(T) == 2) {
    finish<T, N, A>(e, row, col, z, held_at<T, N>(e.bias, col, e.n), residual_at<T, N>(e, row, col));
  } else {                                 // (one number after the other: fewer registers, of which the occupancy of fp64's products depends)
    A slope[N], more[N];
    if (e.bias) {
      load_vec<T, N>(e.bias, col, e.n, more);
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] += more[k];
    }
    if (e.residual) load_vec<T, N>(e.residual + row * e.ldr, col, e.n, more);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      activate<T, A>(e.act, z[k], z[k], slope[k]);
      z[k] *= e.scale;
      if (e.residual) z[k] += more[k];
    }
    store_vec<T, N>(e.y + row * e.ldy, col, e.n, z);
    if (e.slope) store_vec<typename Slope<T>::type, N>(e.slope + row * e.n, col, e.n, slope);
  }
}

// ---- products ----------------------------------------------------------------------------------------------------------------------

// C [m][n] = sum_k P(row, k) Q(k, col).  An operand lies along k (element (r, k) at r * ld + k), or with `across` along its rows / columns
// (k * ld + r).
struct Product {
  const void* p;
  const void* q;
  int64_t ldp, ldq;
  int32_t m, n, k;
};

typedef short short8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef double double2v __attribute__((ext_vector_type(2)));
typedef double double4v __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) short4v lds_short4;

constexpr int LINE = 128;                 // bytes of k a step: 64 16-bit numbers, 32 fp32, 16 fp64
constexpr int OUTSIDE = 0x7ffffff0;       // byte offset behind every record: such a lane reads zeros
template <typename T> constexpr int step_of() { return LINE / (int)sizeof(T); }
// buffers of a BM x BN tile: two; four where a step is shorter than a fetch (16-bit small tiles: 10000 x 1024 x 1024 of fp32 lost a tenth to the CU's fewer workgroups)
constexpr int stages_of(int size, int bm, int bn) { return bm * bn >= 128 * 128 || (size > 2 && bm * bn >= 64 * 64) ? 2 : 4; }
constexpr int tile_lds(int size, int bm, int bn) { return stages_of(size, bm, bn) * (bm + bn) * LINE; }

// What a lane holds of 16 rows: 16 bytes, E numbers behind each other in k; four groups of 16 lanes hold 4 E of them.  One instruction of 32 k for
// the 16-bit types; fp32 and fp64 instructions take four k, one of each group, so E of them take the numbers one by one.
template <typename T> struct Matrix;
template <> struct Matrix<bf16_t> {
  typedef short8 Frag;
  typedef float4v Acc;
  static constexpr int TURNS = 1;
  static __device__ __forceinline__ Acc mfma(Frag a, Frag b, Acc c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Matrix<f16_t> {
  typedef short8 Frag;
  typedef float4v Acc;
  static constexpr int TURNS = 1;
  static __device__ __forceinline__ Acc mfma(Frag a, Frag b, Acc c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <> struct Matrix<float> {
  typedef float4v Frag;
  typedef float4v Acc;
  static constexpr int TURNS = 4;
  static __device__ __forceinline__ Acc mfma(Frag a, Frag b, Acc c, int j) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0); }
};
template <> struct Matrix<double> {
  typedef double2v Frag;
  typedef double4v Acc;
  static constexpr int TURNS = 2;
  static __device__ __forceinline__ Acc mfma(Frag a, Frag b, Acc c, int j) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a[j], b[j], c, 0, 0, 0); }
};

// One operand's tile, R rows x one step of k, 16-byte chunks straight from memory into LDS.  Along k: [row][8 chunks], chunk c of row r at
// place c ^ (r & 7).  Across: [k][chunks of R rows], chunk c of line k at place c ^ swizzle(k); there a lane gathers its k line by line, by the
// transposing LDS read for the 16-bit types.  The places are permuted on the memory side (a lane fetches the chunk that belongs where it
// writes), so that the fragment reads of a wave fall on different banks.  Memory addresses are multiples of four bytes.
template <typename T, int R, bool ACROSS, int THREADS>
struct Tile {
  typedef typename Matrix<T>::Frag Frag;
  static constexpr int SIZE = sizeof(T), E = 16 / SIZE, STEP = step_of<T>();
  static constexpr int LOADS = R * 8 / THREADS, BYTES = R * LINE;
  static constexpr int PER_LINE = R / E;                       // chunks of a line of k
  static constexpr int READS = !ACROSS ? 1 : SIZE == 2 ? 2 : E;   // LDS instructions of a fragment
  static_assert(LOADS >= 1, "a chunk for every thread");
  const char* base;
  int64_t left, step;                                          // bytes from base to the operand's end; bytes a step of k moves on
  int offset[LOADS], chunk_k[LOADS];
  int frag;                                                    // this lane's place in a fragment read

  static __device__ __forceinline__ int swizzle(int k) {       // lines whose reads meet on the same banks without it
    if constexpr (SIZE == 8) return 8 * ((k >> 1) & 1);
    else if constexpr (SIZE == 4) return PER_LINE >= 16 ? 4 * ((k >> 2) & 3) : 4 * ((k >> 2) & 1);
    else if constexpr (PER_LINE >= 16) return 2 * ((k & 3) | ((k >> 1) & 4));
    else if constexpr (PER_LINE == 8) return 2 * (((k >> 1) & 1) | ((k >> 2) & 2));
    else return 2 * ((k >> 3) & 1);
  }

  // rows = the operand's rows (columns of C for Q), k_total its k; row0: this tile's first; row_w: the wave's first row in the tile
  __device__ __forceinline__ void init(const void* p, int64_t ld, int rows, int k_total, int row0, int k0, int row_w) {
    const int t = threadIdx.x, lane = t & 63, i = lane & 15, g = lane >> 4;
    const int64_t first = ACROSS ? (int64_t)k0 * ld + row0 : (int64_t)row0 * ld + k0;
    const int64_t end = ACROSS ? (int64_t)(k_total - 1) * ld + rows : (int64_t)(rows - 1) * ld + k_total;
    base = static_cast<const char*>(p) + first * SIZE;
    left = ((end - first) * SIZE + 3) & ~(int64_t)3;           // the record ends with a whole dword (of an odd 16-bit width's last one half is used)
    step = ACROSS ? STEP * ld * SIZE : LINE;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int u = j * THREADS + t;
      if constexpr (ACROSS) {
        const int k = u / PER_LINE, c = (u % PER_LINE) ^ swizzle(k);
        offset[j] = k * (int)ld * SIZE + c * 16;
        chunk_k[j] = 0;
      } else {
        const int r = u / 8, c = (u % 8) ^ (r & 7);
        offset[j] = r * (int)ld * SIZE + c * 16;
        chunk_k[j] = c * E;
      }
    }
    if constexpr (!ACROSS) {
      frag = (row_w + i) * LINE + ((g ^ (i & 7)) << 4);
    } else if constexpr (SIZE == 2) {
      const int k = g * 8 + (i >> 2), c = row_w / 8 + ((i & 3) >> 1);
      frag = k * (R * 2) + ((c ^ swizzle(k)) << 4) + (i & 1) * 8;
    } else {
      const int k = g * E, c = (row_w + i) / E;                // (the lane's E lines have one swizzle)
      frag = k * (R * SIZE) + ((c ^ swizzle(k)) << 4) + (i % E) * SIZE;
    }
  }

  // Fetch the tile at k (k_left of it inside the operand) and move on.  In assembly because the compiler, which cannot tell the buffers apart, makes every
  // fragment read wait for the fetches into the other one; nothing is returned in registers, and `arrived` waits for what lands in LDS.
  __device__ __forceinline__ void fetch(unsigned to, int k_left) {
    const int64_t l = left < 0 ? 0 : left;
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const int4v r = {(int)(uint32_t)b, (int)((b >> 32) & 0xffff), l < OUTSIDE ? (int)l : OUTSIDE, 0x00020000};
    const unsigned first = to + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int at = ACROSS || chunk_k[j] < k_left ? offset[j] : OUTSIDE;
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(first + j * THREADS * 16), "v"(at), "s"(r) : "memory", "m0");
    }
    base += step;
    left -= step;
  }

  // A chunk that a row along k ends in also brought what lies behind the row: zeros there.  `k` of the step's k are inside.
  static __device__ __forceinline__ void trim(char* tile, int k) {
    if constexpr (!ACROSS)
      for (int r = threadIdx.x; r < R; r += THREADS) {
        T* chunk = reinterpret_cast<T*>(tile + r * LINE + (((k / E) ^ (r & 7)) << 4));
        for (int e = k % E; e < E; ++e) chunk[e] = (T)0;
      }
  }

  // rows row_w + 16 t .. + 16, half s of the step's k
  __device__ __forceinline__ Frag fragment(const lds_char* tile, int t, int s) const {
    if constexpr (!ACROSS) {
      return *(const __attribute__((address_space(3))) Frag*)(tile + ((frag ^ (s << 6)) + t * 16 * LINE));
    } else if constexpr (SIZE == 2) {
      const lds_char* a = tile + ((frag ^ (t << 5)) + s * 32 * R * 2);
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)a), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(a + 4 * R * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const lds_char* a = tile + ((frag ^ (t * 16 * SIZE)) + s * (STEP / 2) * R * SIZE);
      Frag f;
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = *(const __attribute__((address_space(3))) T*)(a + j * R * SIZE);
      return f;
    }
  }
};

// BM x BN of C by WM x WN waves; k in [k_begin, k_end) (k_begin a multiple of the step).  The column operand goes in as the matrix instruction's first, so a lane's results lie along a row of C.
// out.put(row, col, v, ...): the sums of C[row][col .. col + N].
template <typename T, int BM, int BN, int WM, int WN, bool PX, bool QX, typename F>
__device__ __forceinline__ void tile_product(const Product& g, int row0, int col0, int k_begin, int k_end, const F& out) {
  typedef typename Wide<T>::type A;
  typedef typename Matrix<T>::Acc Acc;
  typedef typename Matrix<T>::Frag Frag;
  constexpr int THREADS = 64 * WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, STEP = step_of<T>();
  typedef Tile<T, BM, PX, THREADS> P;
  typedef Tile<T, BN, QX, THREADS> Q;
  constexpr int STAGES = stages_of(sizeof(T), BM, BN);
  __shared__ __attribute__((aligned(16))) char tiles[STAGES * (P::BYTES + Q::BYTES)];
  static_assert(sizeof(tiles) == tile_lds(sizeof(T), BM, BN), "what the plans reckon with");
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wr = (wave / WN) * TM * 16, wc = (wave % WN) * TN * 16;
  P p;
  Q q;
  p.init(g.p, g.ldp, g.m, k_end, row0, k_begin, wr);
  q.init(g.q, g.ldq, g.n, k_end, col0, k_begin, wc);
  Acc acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = {0, 0, 0, 0};
  // A step's k is multiplied in two halves.  While the first half is multiplied the second's fragments are read; then the next step's tiles have arrived
  // and everyone has read this step's: the buffer is free for a later step's, and while the second half is multiplied the next step's first
  // fragments are read.  One barrier a step, and the matrix pipe has work on both sides of it.
  Frag p0[TM], q0[TN], p1[TM], q1[TN];
  auto read = [&](const lds_char* from, int s, Frag (&fp)[TM], Frag (&fq)[TN]) {
#pragma unroll
    for (int b = 0; b < TN; ++b) fq[b] = q.fragment(from + P::BYTES, b, s);
#pragma unroll
    for (int a = 0; a < TM; ++a) fp[a] = p.fragment(from, a, s);
  };
  auto multiply = [&](const Frag (&fp)[TM], const Frag (&fq)[TN]) {
#pragma unroll
    for (int j = 0; j < Matrix<T>::TURNS; ++j)
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) acc[a][b] = Matrix<T>::mfma(fq[b], fp[a], acc[a][b], j);
  };
  // a half's reads spread between the multiplications that run meanwhile (left alone, the compiler puts them behind)
  constexpr int READS = TM * P::READS + TN * Q::READS, PRODUCTS = TM * TN * Matrix<T>::TURNS, EACH = PRODUCTS / READS > 2 ? 2 : 1;
  auto interleave = [&]() {
#pragma unroll
    for (int r = 0; r < READS; ++r) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      // an LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);   // matrix instructions
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int BUFFER = P::BYTES + Q::BYTES;
  const lds_char* const lds = (const lds_char*)tiles;
  const unsigned place = __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<uintptr_t>(lds));
  auto fetch = [&](int buffer, int k_left) {
    p.fetch(place + buffer, k_left);
    q.fetch(place + buffer + P::BYTES, k_left);
  };
  if (k_begin < k_end) {
    constexpr int FETCHES = P::LOADS + Q::LOADS;
    const int steps = (k_end - k_begin + STEP - 1) / STEP;
    int k_left = k_end - k_begin, now = 0;
    const int last = k_left - (steps - 1) * STEP;        // of the last step
    auto trim = [&](int buffer) {
      P::trim(tiles + buffer, last);
      Q::trim(tiles + buffer + P::BYTES, last);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    const bool ragged = (!PX || !QX) && last % P::E != 0;
    for (int s = 0; s < STAGES && s < steps; ++s) fetch(s * BUFFER, k_left - s * STEP);
    if (steps >= STAGES) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 1) * FETCHES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    if (ragged && steps == 1) trim(0);
    read(lds, 0, p0, q0);
    for (int left = steps - 1; left > 0; --left) {
      read(lds + now, 1, p1, q1);
      multiply(p0, q0);
      interleave();
      // the next step's tiles (behind them at most STAGES - 2 more have been asked for), and everyone's reads of this step's
      if (left >= STAGES - 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * FETCHES) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (left >= STAGES) fetch(now, k_left - STAGES * STEP);
      k_left -= STEP;
      now = now + BUFFER == STAGES * BUFFER ? 0 : now + BUFFER;
      if (ragged && left == 1) trim(now);
      read(lds + now, 0, p0, q0);
      multiply(p1, q1);
      interleave();
    }
    read(lds + now, 1, p1, q1);
    multiply(p0, q0);
    multiply(p1, q1);
  }
  // Sixteen rows at a time through a piece of LDS of the wave's own, so that a lane ends with N columns of a row and a row's lanes write whole lines.
  // The loop stays rolled (the epilogue is long); the registers are picked by number inside it.  A lane's columns are the same every time; what it needs of
  // the residual is asked for a turn ahead (4096 x 4096 x 16384 bf16 with a residual: 505 -> 482 us; fp32 and fp64, whose registers it would take from the
  // product's occupancy, lost 2 and 6 %).
  constexpr int N = TN == 1 ? 4 : 8, COLS = TN * 16, PITCH = COLS + 4, PARTS = 16 * COLS / N / 64;
  constexpr bool AHEAD = sizeof(T) == 2;
  static_assert(WM * WN * 16 * PITCH * (int)sizeof(A) <= STAGES * (P::BYTES + Q::BYTES), "the rows fit the tiles' LDS");
  static_assert(64 % (COLS / N) == 0, "a lane's columns are the same in every part");
  auto row_of = [&](int turn, int j) { return row0 + wr + turn * 16 + (j * 64 + lane) / (COLS / N); };
  Held<T, N> bias, residual[PARTS];
  int col;
  if constexpr (AHEAD) {
    col = col0 + wc + lane % (COLS / N) * N;
    bias = out.template bias<N>(col);
#pragma unroll
    for (int j = 0; j < PARTS; ++j) residual[j] = out.template residual<N>(row_of(0, j), col);
  }
  __syncthreads();
  A* rows = reinterpret_cast<A*>(tiles) + wave * 16 * PITCH;
  const int i = lane & 15, group = lane >> 4;
#pragma unroll 1
  for (int turn = 0; turn < TM; ++turn) {
#pragma unroll
    for (int a = 0; a < TM; ++a)
      if (a == turn) {
#pragma unroll
        for (int b = 0; b < TN; ++b) {
          if constexpr (sizeof(A) == 4) {
            *reinterpret_cast<float4v*>(rows + i * PITCH + b * 16 + group * 4) = acc[a][b];
          } else {                        // (the fp64 instruction's registers are four rows apart, not one)
#pragma unroll
            for (int r = 0; r < 4; ++r) rows[i * PITCH + b * 16 + group + 4 * r] = acc[a][b][r];
          }
        }
      }
    Held<T, N> now[PARTS];
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      if (AHEAD) now[j] = residual[j];
      if (AHEAD && turn + 1 < TM) residual[j] = out.template residual<N>(row_of(turn + 1, j), col);
    }
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      A v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = rows[(j * 64 + lane) / (COLS / N) * PITCH + lane % (COLS / N) * N + k];
      if constexpr (AHEAD) out.put(row_of(turn, j), col, v, bias, now[j]);
      else out.put(row_of(turn, j), col0 + wc + (j * 64 + lane) % (COLS / N) * N, v);
    }
  }
}

// Where a tile's sums go: through the epilogue, or as a k slice's to `part`.
template <typename T>
struct Target {
  typedef typename Wide<T>::type A;
  const Epilogue<T>& e;
  A* part;
  const Product& g;
  template <int N>
  __device__ __forceinline__ Held<T, N> bias(int col) const { return held_at<T, N>(part ? nullptr : e.bias, col, e.n); }
  template <int N>
  __device__ __forceinline__ Held<T, N> residual(int row, int col) const {
    if (part || !e.residual || row >= g.m) return {};
    return residual_at<T, N>(e, row, col);
  }
  template <int N>
  __device__ __forceinline__ void put(int row, int col, A (&v)[N], const Held<T, N>& bias, const Held<T, N>& residual) const {
    if (row >= g.m || col >= g.n) return;
    if (part) store_vec<A, N>(part + ((int64_t)blockIdx.y * g.m + row) * g.n, col, g.n, v);
    else finish<T, N, A>(e, row, col, v, bias, residual);
  }
  template <int N>
  __device__ __forceinline__ void put(int row, int col, A (&v)[N]) const {
    if (row >= g.m || col >= g.n) return;
    if (part) store_vec<A, N>(part + ((int64_t)blockIdx.y * g.m + row) * g.n, col, g.n, v);
    else finish<T, N, A>(e, row, col, v);
  }
};

// C in BM x BN tiles, slice blockIdx.y of the k range (`part` != null: its sums).  Workgroups go round the eight XCDs by their number: each
// XCD takes one contiguous eighth of the tiles, in bands of eight tile rows, so that the operands a band shares stay in its L2.  Bound by the matrix pipe, whose
// clock the card's power limits, and by the LDS reads beside it: bf16 8192 x 4096 x 16384 with gelu 941 us = 1.17 PFLOP/s; fp32 10 000 x 1024 x 1024 169 us = 124
// TFLOP/s, fp64 4000 x 2048 x 2048 549 us = 61 TFLOP/s.
template <typename T, int BM, int BN, int WM, int WN, bool PX, bool QX>
__global__ __launch_bounds__(64 * WM * WN, BM * BN >= 256 * 256 ? 1 : 2) void product_kernel(Product g, int tiles_m, int tiles_n, int k_slice, typename Wide<T>::type* __restrict__ part,
                                                               Epilogue<T> e) {
  typedef typename Wide<T>::type A;
  const int tiles = tiles_m * tiles_n, id = blockIdx.x, xcd = id & 7, each = tiles >> 3, more = tiles & 7;
  const int tile = xcd * each + (xcd < more ? xcd : more) + (id >> 3);
  const int64_t per_band = (int64_t)8 * tiles_n;
  const int band = (int)(tile / per_band), in_band = (int)(tile - band * per_band), height = min(8, tiles_m - band * 8);
  const int row0 = (band * 8 + in_band % height) * BM, col0 = (in_band / height) * BN;
  const int k_begin = blockIdx.y * k_slice, k_end = min(k_begin + k_slice, g.k);
  const Target<T> to = {e, part, g};
  tile_product<T, BM, BN, WM, WN, PX, QX>(g, row0, col0, k_begin, k_end, to);
}

// the slices' sums and the epilogue: four columns a lane.  PARTS lanes share them where there are many slices of a small product; a part's slices, then
// the parts, are added in their order.
template <typename T, int PARTS>
__global__ __launch_bounds__(256) void product_join_kernel(const typename Wide<T>::type* __restrict__ part, int slices, int64_t m, int64_t n, Epilogue<T> e) {
  typedef typename Wide<T>::type A;
  constexpr int LANES = 256 / PARTS;
  __shared__ A sh[PARTS > 1 ? PARTS : 1][LANES][4];
  const int lane = threadIdx.x % LANES, p = threadIdx.x / LANES;
  const int64_t at = (int64_t)blockIdx.x * LANES + lane, quads = (n + 3) / 4, row = at / quads, col = (at - row * quads) * 4;
  A z[4] = {0, 0, 0, 0};
  if (row < m) {
#pragma unroll 4
    for (int s = p; s < slices; s += PARTS) {
      A v[4];
      load_vec<A, 4>(part + ((int64_t)s * m + row) * n, col, n, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) z[k] += v[k];
    }
  }
  if constexpr (PARTS > 1) {
#pragma unroll
    for (int k = 0; k < 4; ++k) sh[p][lane][k] = z[k];
    __syncthreads();
    if (p) return;
    for (int q = 1; q < PARTS; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) z[k] += sh[q][lane][k];
  }
  if (row < m) finish<T, 4>(e, row, col, z);
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------

// Up to four rows of C (a token, a handful of samples): bound by reading Q once, each number of which is used m times, so the vector units do and the matrix
// pipe's tiles would be mostly empty.  Q goes from memory to registers, 16 bytes a lane at any alignment and pitch; k is shared by the waves of a workgroup,
// whose sums are joined in LDS (in their order).  One row, us against the tiles': bf16 4096 x 16384 stored transposed 23.8 / 27.4, 16384 x 4096 30 / 33, 768 x 2304
// 7.9 / 10.9; fp32 16384 x 4096 47 / 59 (5.7 TB/s), transposed 51 / 69.
constexpr int FEW_ALONG = 4, FEW_ACROSS = 2, FEW_COLS = 4;      // most rows by Q's layout (across k, four rows' registers leave too few waves: 32 against the tiles' 26 us for 4 x 4096 x 12288)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Packed { T v[vec_of<T>()]; };
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };

// Q across k: ALONG lanes along a line, 64 / ALONG of them along k, eight lines each at a time.  32 lanes (512 bytes of a line) reach 5.6 TB/s, eight (128
// bytes) 4.6, but make four times the workgroups, and where those suffice no second launch is needed.
template <typename T, int M, int ALONG>
__global__ __launch_bounds__(512) void few_across_kernel(Product g, int k_slice, typename Wide<T>::type* __restrict__ part, Epilogue<T> e) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>(), WAVES = 8, COLS = ALONG * V, CHUNK = 64 / ALONG * 8;
  constexpr bool X_AHEAD = M * (int)sizeof(T) <= 8;      // (registers)
  __shared__ A sh[WAVES][M][COLS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane % ALONG, s = lane / ALONG;
  const int col = blockIdx.x * COLS + i * V, from = min(col, g.n - V);             // (a vector that passes the end is moved back: the same sums twice)
  const int k_begin = blockIdx.y * k_slice, k_end = min(k_begin + k_slice, g.k);
  const T* q = static_cast<const T*>(g.q) + from;
  const T* p = static_cast<const T*>(g.p);
  A acc[M][V];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < V; ++c) acc[m][c] = 0;
  Packed<T> w[8], w_next[8];
  Eight<T> x[M], x_next[M];
  auto fetch = [&](int k0) {
    const T* at = q + (int64_t)(k0 + s * 8) * g.ldq;
#pragma unroll
    for (int u = 0; u < 8; ++u) w_next[u] = *reinterpret_cast<const Packed<T>*>(at + u * g.ldq);
  };
  auto fetch_x = [&](int k0) {
#pragma unroll
    for (int m = 0; m < M; ++m) x_next[m] = *reinterpret_cast<const Eight<T>*>(p + min(m, g.m - 1) * g.ldp + k0 + s * 8);
  };
  auto add = [&](int u, const Packed<T>& line, const A (&xk)[M]) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const A v = (A)line.v[c];
#pragma unroll
      for (int m = 0; m < M; ++m) acc[m][c] = fma(xk[m], v, acc[m][c]);
    }
  };
  int k0 = k_begin + wave * CHUNK;
  if (k0 + CHUNK <= k_end) {
    if (X_AHEAD) fetch_x(k0);
    fetch(k0);
  }
  for (; k0 + CHUNK <= k_end; k0 += WAVES * CHUNK) {
#pragma unroll
    for (int u = 0; u < 8; ++u) w[u] = w_next[u];
    if (!X_AHEAD) fetch_x(k0);
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] = x_next[m];
    if (k0 + (WAVES + 1) * CHUNK <= k_end) {
      if (X_AHEAD) fetch_x(k0 + WAVES * CHUNK);
      fetch(k0 + WAVES * CHUNK);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      A xk[M];
#pragma unroll
      for (int m = 0; m < M; ++m) xk[m] = (A)x[m].v[u];
      add(u, w[u], xk);
    }
  }
  if (k0 < k_end)                                                                // the last, partial chunk
    for (int k = k0 + s * 8; k < min(k0 + s * 8 + 8, k_end); ++k) {
      A xk[M];
#pragma unroll
      for (int m = 0; m < M; ++m) xk[m] = (A)p[min(m, g.m - 1) * g.ldp + k];
      add(0, *reinterpret_cast<const Packed<T>*>(q + k * g.ldq), xk);
    }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < V; ++c) {
      A v = acc[m][c];
#pragma unroll
      for (int d = ALONG; d < 64; d *= 2) v += __shfl_xor(v, d);
      if (s == 0) sh[wave][m][i * V + c] = v;
    }
  __syncthreads();
  for (int u = threadIdx.x; u < M * ALONG; u += 64 * WAVES) {
    const int m = u / ALONG, j = u % ALONG, nominal = blockIdx.x * COLS + j * V;
    if (m >= g.m || nominal >= g.n) continue;
    A z[V];
#pragma unroll
    for (int c = 0; c < V; ++c) z[c] = sh[0][m][j * V + c];
    for (int w = 1; w < WAVES; ++w)
#pragma unroll
      for (int c = 0; c < V; ++c) z[c] += sh[w][m][j * V + c];
    const int to = min(nominal, g.n - V);
    if (part) store_vec<A, V>(part + ((int64_t)blockIdx.y * g.m + m) * g.n, to, g.n, z);
    else finish<T, V>(e, m, to, z);
  }
}

// Q along k, the lanes too: a wave takes four columns, and SPLIT of a workgroup's four waves share them.
template <typename T, int M, int SPLIT>
__global__ __launch_bounds__(256) void few_along_kernel(Product g, int k_slice, typename Wide<T>::type* __restrict__ part, Epilogue<T> e) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>(), COLS = FEW_COLS, CHUNK = 64 * SPLIT * V;
  __shared__ A sh[4][M][COLS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col0 = (blockIdx.x * (4 / SPLIT) + wave / SPLIT) * COLS;
  const int k_begin = blockIdx.y * k_slice, k_end = min(k_begin + k_slice, g.k);
  const T* p = static_cast<const T*>(g.p);
  const T* q = static_cast<const T*>(g.q);
  A acc[M][COLS];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < COLS; ++c) acc[m][c] = 0;
  auto row = [&](int m) { return p + min(m, g.m - 1) * g.ldp; };                  // (rows and columns that are not there: the last one again)
  auto line = [&](int c) { return q + min(col0 + c, g.n - 1) * g.ldq; };
#pragma unroll 2
  for (int k = k_begin + (threadIdx.x % (64 * SPLIT)) * V; k < k_end; k += CHUNK) {
    if (k + V <= k_end) {
      Packed<T> w[COLS], x[M];
#pragma unroll
      for (int c = 0; c < COLS; ++c) w[c] = *reinterpret_cast<const Packed<T>*>(line(c) + k);
#pragma unroll
      for (int m = 0; m < M; ++m) x[m] = *reinterpret_cast<const Packed<T>*>(row(m) + k);
#pragma unroll
      for (int u = 0; u < V; ++u)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int c = 0; c < COLS; ++c) acc[m][c] = fma((A)x[m].v[u], (A)w[c].v[u], acc[m][c]);
    } else {
      for (int j = k; j < k_end; ++j)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int c = 0; c < COLS; ++c) acc[m][c] = fma((A)row(m)[j], (A)line(c)[j], acc[m][c]);
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const A v = group_sum<64>(acc[m][c]);
      if (lane == 0) sh[wave][m][c] = v;
    }
  __syncthreads();
  const int m = threadIdx.x % (64 * SPLIT);                                        // the first wave of those that share the columns
  if (m >= g.m || col0 >= g.n) return;
  A z[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) z[c] = sh[wave][m][c];
#pragma unroll
  for (int w = 1; w < SPLIT; ++w)
#pragma unroll
    for (int c = 0; c < COLS; ++c) z[c] += sh[wave + w][m][c];
  if (part) store_vec<A, COLS>(part + ((int64_t)blockIdx.y * g.m + m) * g.n, col0, g.n, z);
  else finish<T, COLS>(e, m, col0, z);
}

// ---- what is made ready before the products --------------------------------------------------------------------------------------------

// Up to three copies in one launch: lines of n elements to lines of ld_to (zeros behind n), times the slope: an operand into lines that the
// products can fetch, or dz / scale = slope * dy; `to` may be null.  With `sums` also the sums of dz's columns (unrounded numbers', scaled at the end), or where several
// groups of workgroups share the lines each one's part of them: partial[group][n].  The scale stays out of what is rounded and goes into the products' epilogue: fp16 has no
// room for it (10 * 7000 is beyond its largest number, 1e-4 * 1e-3 among its last subnormal ones, where the gradients themselves may well fit).  `lanes` (a power of two) lie along the columns, 256 / lanes lines are taken at a time.  Bound by memory:
// dz of 8192 x 4096 bf16 and its columns' sums 32 us = 6.2 TB/s.
template <typename T>
struct Job {
  const T* from;
  int64_t ld, lines, n;
  const typename Slope<T>::type* slope;
  typename Wide<T>::type scale;      // of the sums
  T* to;
  int64_t ld_to;
  typename Wide<T>::type* partial;
  T* sums;             // with one group: the sums themselves
  int32_t lanes_log2, col_blocks, groups, first;       // first: the job's first workgroup in the launch
};
template <typename T>
struct Jobs {
  Job<T> job[3];
  int32_t count, blocks;
};

template <typename T>
__global__ __launch_bounds__(256) void prepare_kernel(Jobs<T> jobs) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>();
  __shared__ A sh[256 * V];
  int which = 0;
  while (which + 1 < jobs.count && (int)blockIdx.x >= jobs.job[which + 1].first) ++which;
  const Job<T>& b = jobs.job[which];
  const int block = blockIdx.x - b.first, group = block / b.col_blocks, lanes = 1 << b.lanes_log2, at_once = 256 >> b.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1), part = threadIdx.x >> b.lanes_log2;
  const int64_t col0 = (int64_t)(block - group * b.col_blocks) * lanes * V, col = col0 + lane * V;
  A sum[V];
#pragma unroll
  for (int k = 0; k < V; ++k) sum[k] = 0;
  for (int64_t r = (int64_t)group * at_once + part; r < b.lines; r += (int64_t)b.groups * at_once) {
    A v[V], s[V];
    load_vec<T, V>(b.from + r * b.ld, col, b.n, v);
    if (b.slope) load_vec<typename Slope<T>::type, V>(b.slope + r * b.n, col, b.n, s);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (b.slope) v[k] *= s[k];
      if (col + k >= b.n) v[k] = 0;
      sum[k] += v[k];
    }
    if (b.to) store_vec<T, V>(b.to + r * b.ld_to, col, b.ld_to, v);
  }
  if (!b.sums) return;
#pragma unroll
  for (int k = 0; k < V; ++k) sh[(part * lanes + lane) * V + k] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < lanes * V; c += 256) {
    A v = 0;
    for (int p = 0; p < at_once; ++p) v += sh[p * lanes * V + c];
    v *= b.scale;
    if (col0 + c < b.n) {
      if (b.groups == 1) b.sums[col0 + c] = (T)v;
      else b.partial[(int64_t)group * b.n + col0 + c] = v;
    }
  }
}

// ---- thin layers ---------------------------------------------------------------------------------------------------------------------

// At most 48 inputs and outputs in fp32 or fp64 (the flow's own conditioners): bound by reading and writing the rows once.  The kernel's fragments
// stay in registers, a wave takes sixteen rows at a time, and no operand is copied.  Between memory and the matrix instruction's lane layout a tile
// passes through a piece of LDS of the wave's own: its elements are fetched and written in the order of the rows (whole lines at any pitch), and the
// epilogue runs over them in that order too, so that no lane evaluates an activation for a column that is not there.  65 536 rows, 21 -> 21 fp64 with tanh: 15 us and
// 16 backward; 48 wide 34 and 45, 49 wide, by the tiles, 33 and 68 (fp32 17 and 23; 17 and 42); wider ones' fragments leave the registers.
constexpr int THIN = 48, THIN_THREADS = 512, THIN_GROUPS = 256;
// pitch of a tile's rows in LDS: sixteen rows four or eight banks apart
constexpr int thin_pitch(int wide) { return wide <= 32 ? 36 : 52; }

__device__ __forceinline__ float4v mfma4(float a, float b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ double4v mfma4(double a, double b, double4v c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
// row of a 16 x 16 result that register r of a lane of group g holds
template <typename T> __device__ __forceinline__ int result_row(int g, int r) { return sizeof(T) == 8 ? g + 4 * r : g * 4 + r; }

// Element u < 16 n of sixteen rows of n <= 48 (the product is off by far less than the half that keeps it from a whole number)
template <int PITCH>
struct InOrder {
  int n;
  float inv;
  __device__ __forceinline__ explicit InOrder(int n_) : n(n_), inv(1.0f / (float)n_) {}
  __device__ __forceinline__ int row(int u) const { return (int)(((float)u + 0.5f) * inv); }
  __device__ __forceinline__ int place(int u, int r) const { return r * PITCH + u - r * n; }
};

// The kernel's element (k, n) is at w[k * sk + n * sn].  KS: steps of four inputs, NT: tiles of sixteen outputs.
template <typename T, int KS, int NT>
__global__ __launch_bounds__(256) void thin_forward_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t sk, int64_t sn, int64_t rows, int n_in,
                                                           Epilogue<T> e) {
  typedef typename Matrix<T>::Acc Acc;
  constexpr int PITCH = thin_pitch(KS * 4 > NT * 16 ? KS * 4 : NT * 16), TILE = 16 * PITCH;
  __shared__ T sh[4][2][TILE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4, n_out = (int)e.n;
  const int64_t tiles = (rows + 15) / 16, stride = (int64_t)gridDim.x * 4;
  int64_t tile = (int64_t)blockIdx.x * 4 + wave;
  if (tile >= tiles) return;
  T* tx = sh[wave][0];
  T* tz = sh[wave][1];
  const InOrder<PITCH> in(n_in), out(n_out);
  T wf[KS][NT], bias[NT], xv[KS];
#pragma unroll
  for (int b = 0; b < NT; ++b) {
    bias[b] = e.bias && b * 16 + i < n_out ? e.bias[b * 16 + i] : (T)0;
#pragma unroll
    for (int s = 0; s < KS; ++s) wf[s][b] = 4 * s + g < n_in && b * 16 + i < n_out ? w[(4 * s + g) * sk + (b * 16 + i) * sn] : (T)0;
  }
  for (int u = lane; u < TILE; u += 64) tx[u] = 0;          // (behind the inputs it stays zero)
  auto load = [&](int64_t at) {                                  // (no branches: a lane without an element reads the tile's first one, so that all loads fly at once)
    const T* p = x + at * 16 * ldx;
    const int live = (int)min((int64_t)16, rows - at * 16);
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const int u = lane + 64 * j, r = in.row(u);
      xv[j] = p[r < live ? r * (int)ldx + u - r * n_in : 0];
    }
  };
  load(tile);
  for (; tile < tiles; tile += stride) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const int u = lane + 64 * j, r = in.row(u);
      if (r < 16) tx[in.place(u, r)] = xv[j];                   // (a row that is not there takes any numbers: its results are not written)
    }
    if (tile + stride < tiles) load(tile + stride);
    __builtin_amdgcn_wave_barrier();
    Acc acc[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[b] = {bias[b], bias[b], bias[b], bias[b]};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const T xf = tx[i * PITCH + 4 * s + g];
#pragma unroll
      for (int b = 0; b < NT; ++b) acc[b] = mfma4(xf, wf[s][b], acc[b]);
    }
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) tz[result_row<T>(g, r) * PITCH + b * 16 + i] = acc[b][r];
    __builtin_amdgcn_wave_barrier();
    const int live = (int)min((int64_t)16, rows - tile * 16) * n_out;
#pragma unroll 1
    for (int u = lane; u < live; u += 64) {                      // (rolled: the activations' code is longer than the loop saves)
      const int r = out.row(u), n = u - r * n_out;
      const int64_t row = tile * 16 + r;
      T a, slope;
      activate<T, T>(e.act, tz[out.place(u, r)], a, slope);
      a *= e.scale;
      if (e.residual) a += e.residual[row * e.ldr + n];
      e.y[row * e.ldy + n] = a;
      if (e.slope) e.slope[row * n_out + n] = slope;
    }
  }
}

// dx (may be null) and this workgroup's sums partial[blockIdx.x][n_in * n_out + n_out] of x^T dz and dz (null: not wanted); a single workgroup writes them
// to dkernel and dbias (either may be null) itself.
template <typename T, int KT, int NT>
__global__ __launch_bounds__(THIN_THREADS) void thin_backward_kernel(const T* __restrict__ dy, int64_t ldd, const T* __restrict__ slope, T scale,
                                                                     const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t sk, int64_t sn, int64_t rows,
                                                                     int n_in, int n_out, T* __restrict__ dx, T* __restrict__ partial, T* __restrict__ dkernel,
                                                                     T* __restrict__ dbias) {
  typedef typename Matrix<T>::Acc Acc;
  constexpr int PITCH = thin_pitch(16 * (KT > NT ? KT : NT)), TILE = 16 * PITCH, NS = NT * 4, WAVES = THIN_THREADS / 64, SUMS = KT * 16 * NT * 16 + NT * 16;
  __shared__ T sh[WAVES * 2 * TILE], wt[KT * 16 * PITCH];
  static_assert(WAVES / 2 * SUMS <= WAVES * 2 * TILE, "the sums fit the tiles' LDS");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const int64_t tiles = (rows + 15) / 16, stride = (int64_t)gridDim.x * WAVES;
  T* tx = sh + wave * 2 * TILE;
  T* tz = tx + TILE;
  const InOrder<PITCH> in(n_in), out(n_out);
  for (int u = threadIdx.x; u < KT * 16 * NT * 16; u += THIN_THREADS) {
    const int k = u / (NT * 16), n = u % (NT * 16);
    wt[k * PITCH + n] = dx && k < n_in && n < n_out ? w[k * sk + n * sn] : (T)0;
  }
  for (int u = lane; u < 2 * TILE; u += 64) tx[u] = 0;      // (behind dz's columns it stays zero: they are summed over)
  __syncthreads();
  Acc sum[KT][NT];
  T bias[NT];
#pragma unroll
  for (int b = 0; b < NT; ++b) {
    bias[b] = 0;
#pragma unroll
    for (int a = 0; a < KT; ++a) sum[a][b] = {0, 0, 0, 0};
  }
  T dv[NS], sv[NS], xv[KT * 4];
  auto load = [&](int64_t at) {                                  // (no branches: see above)
    const T* pd = dy + at * 16 * ldd;
    const T* ps = slope + at * 16 * n_out;
    const T* px = x + at * 16 * ldx;
    const int live = (int)min((int64_t)16, rows - at * 16);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int u = lane + 64 * j, r = out.row(u);
      dv[j] = pd[r < live ? r * (int)ldd + u - r * n_out : 0];
      sv[j] = slope ? ps[r < live ? u : 0] : (T)1;
    }
    if (x)
#pragma unroll
      for (int j = 0; j < KT * 4; ++j) {
        const int u = lane + 64 * j, r = in.row(u);
        xv[j] = px[r < live ? r * (int)ldx + u - r * n_in : 0];
      }
  };
  int64_t tile = (int64_t)blockIdx.x * WAVES + wave;
  if (tile < tiles) load(tile);
  for (; tile < tiles; tile += stride) {
    const int live = (int)min((int64_t)16, rows - tile * 16);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int u = lane + 64 * j, r = out.row(u);
      if (r < 16) tz[out.place(u, r)] = r < live ? dv[j] * scale * sv[j] : (T)0;
    }
    if (x)
#pragma unroll
      for (int j = 0; j < KT * 4; ++j) {
        const int u = lane + 64 * j, r = in.row(u);
        if (r < 16) tx[in.place(u, r)] = r < live ? xv[j] : (T)0;
      }
    if (tile + stride < tiles) load(tile + stride);
    __builtin_amdgcn_wave_barrier();
    if (partial) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        T xc[KT];
#pragma unroll
        for (int a = 0; a < KT; ++a) xc[a] = tx[(4 * s + g) * PITCH + a * 16 + i];
#pragma unroll
        for (int b = 0; b < NT; ++b) {
          const T zc = tz[(4 * s + g) * PITCH + b * 16 + i];
          bias[b] += zc;
#pragma unroll
          for (int a = 0; a < KT; ++a) sum[a][b] = mfma4(xc[a], zc, sum[a][b]);
        }
      }
    }
    if (dx) {
      Acc acc[KT];
#pragma unroll
      for (int a = 0; a < KT; ++a) acc[a] = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const T zr = tz[i * PITCH + 4 * s + g];
#pragma unroll
        for (int a = 0; a < KT; ++a) acc[a] = mfma4(zr, wt[(a * 16 + i) * PITCH + 4 * s + g], acc[a]);
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int a = 0; a < KT; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) tx[result_row<T>(g, r) * PITCH + a * 16 + i] = acc[a][r];
      __builtin_amdgcn_wave_barrier();
      T* dxt = dx + tile * 16 * n_in;
#pragma unroll 4
      for (int u = lane; u < live * n_in; u += 64) dxt[u] = tx[in.place(u, in.row(u))];
    }
  }
  if (!partial) return;
#pragma unroll
  for (int b = 0; b < NT; ++b) {
    bias[b] += __shfl_xor(bias[b], 16);
    bias[b] += __shfl_xor(bias[b], 32);
  }
  __syncthreads();
  // the upper waves' sums onto the lower ones', then those in their order
  for (int half = 0; half < 2; ++half) {
    if (wave / (WAVES / 2) == half) {
      T* to = sh + wave % (WAVES / 2) * SUMS;
#pragma unroll
      for (int b = 0; b < NT; ++b) {
#pragma unroll
        for (int a = 0; a < KT; ++a)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            T& at = to[(a * 16 + result_row<T>(g, r)) * (NT * 16) + b * 16 + i];
            at = half ? at + sum[a][b][r] : sum[a][b][r];
          }
        T& at = to[KT * 16 * NT * 16 + b * 16 + i];
        if (g == 0) at = half ? at + bias[b] : bias[b];
      }
    }
    __syncthreads();
  }
  T* to = partial + (int64_t)blockIdx.x * (n_in + 1) * n_out;
  for (int u = threadIdx.x; u < SUMS; u += THIN_THREADS) {
    const int k = u / (NT * 16), n = u % (NT * 16);
    const bool is_bias = k == KT * 16;
    if (n < n_out && (is_bias || k < n_in)) {
      T v = sh[u];
      for (int s = 1; s < WAVES / 2; ++s) v += sh[s * SUMS + u];
      if (gridDim.x > 1) to[(is_bias ? n_in : k) * n_out + n] = v;
      else if (is_bias && dbias) dbias[n] = v;
      else if (!is_bias && dkernel) dkernel[k * n_out + n] = v;
    }
  }
}

// ---- plans ---------------------------------------------------------------------------------------------------------------------------

struct Tiles { int bm, bn, slices, slice_steps; };

// What a step of k costs a CU in microseconds, by type and square tile: alone (its fetches and barrier), and each of several workgroups that share the CU
// (the matrix pipe).  `held`: workgroups a CU holds, by its LDS (64-wide 16-bit tiles: 64 KB each) or, for fp32 and fp64, its registers.  Measured as the difference of
// products of 96 and 32 steps with one to eight tiles a CU: 64-wide bf16 tiles 0.34, 0.42, 0.70, 0.83 us for one to four, 128-wide 0.71, 0.85, 1.53, 1.74, 256-wide 1.46, 2.96,
// fp32 0.68, 1.07, 1.53, 1.97, 3.00 for one to five, fp64 0.64, 1.08, 1.58, 2.15.
struct Cost { int side, held; double alone, each; };
constexpr Cost HALF_COSTS[] = {{64, 2, 0.34, 0.21}, {128, 2, 0.71, 0.43}, {256, 1, 1.46, 1.48}};
constexpr Cost F32_COST = {64, 4, 0.65, 0.5}, F64_COST = {64, 4, 0.7, 0.55};
constexpr int CU_LDS = 160 * 1024;
constexpr bool fits(const Cost& c, int size) { return c.held * tile_lds(size, c.side, c.side) <= CU_LDS; }
static_assert(fits(HALF_COSTS[0], 2) && fits(HALF_COSTS[1], 2) && fits(HALF_COSTS[2], 2) && fits(F32_COST, 4) && fits(F64_COST, 8), "a CU's LDS holds what the costs say");

// Tile and k slices of a product of `steps` steps of k.  Sides of at most 32 rows or columns take 32, so that little is multiplied for nothing: those read
// one long operand once, and the k range is cut until two workgroups a CU do.  Everything else takes the tile and the number of slices of the least
// estimated time: the steps of the fullest CU, and with slices a second launch that reads and joins their sums (5 us, of which the host takes most, and their bytes at 4 TB/s).  Of 45
// shapes (three types, 0.05 to 140 GFLOP) it finds the best choice, or one within 10 % of it, for 43; 1537 x 776 x 1000 of fp32 is off by 18 %, 256 x 256 x 65536 of bf16, which is
// bound by reading, by 22 %.
template <typename T>
Tiles tiles_of(int64_t m, int64_t n, int64_t steps) {
  Tiles best = {m <= 32 ? 32 : 128, n <= 32 ? 32 : 128, 1, 0};
  int64_t slices = 1;
  if (best.bm == 32 || best.bn == 32) {
    const int64_t tiles = ceil_div(m, best.bm) * ceil_div(n, best.bn);
    if (tiles > 0 && tiles < 256) slices = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(ceil_div(512, tiles), ceil_div(steps, 4)), 256));
  } else {
    double least = INFINITY;
    auto consider = [&](const Cost& c) {
      const int64_t tiles = ceil_div(m, c.side) * ceil_div(n, c.side);
      for (const int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256}) {
        if (s > 1 && (steps < 2 * s || tiles * s > 2048)) break;
        const double on_one = (double)ceil_div(tiles * s, 256);
        const double time = (double)ceil_div(steps, s) * std::max(c.alone * std::ceil(on_one / c.held), on_one * c.each) +
                            (s > 1 ? 5 + (double)s * m * n * 2 * sizeof(typename Wide<T>::type) / 4e6 : 0);
        if (time < least) {
          least = time;
          best.bm = best.bn = c.side;
          slices = s;
        }
      }
    };
    if constexpr (sizeof(T) == 2)
      for (const Cost& c : HALF_COSTS) consider(c);
    else
      consider(sizeof(T) == 4 ? F32_COST : F64_COST);
  }
  best.slice_steps = (int)std::max<int64_t>(1, ceil_div(steps, slices));
  best.slices = (int)std::max<int64_t>(1, ceil_div(steps, best.slice_steps));
  return best;
}

// Whether, for at most 32 rows of 16-bit numbers and a kernel across k, tiles 64 wide in one launch beat slices and a second launch: with a workgroup a CU a step
// takes 0.32 us (8 x 4096 x 16384: 26 us against 30), slices reach 5.4 TB/s.  (fp32's and fp64's steps hold half the k and more.)
template <typename T>
bool one_launch(int64_t n, int64_t k) {
  return sizeof(T) == 2 && n > 32 && n <= 64 * 256 && 0.32 * ceil_div(k, step_of<T>()) < (double)n * k * sizeof(T) / 5.4e6 + 4.5;
}

// Products that the kernels for few rows take, in any layout of their operands.  `fetchable`: the tiles could take q as it lies.
template <typename T>
bool few(int64_t m, int64_t n, int64_t k, bool q_across, bool fetchable) {
  return m >= 1 && m <= (q_across ? FEW_ACROSS : FEW_ALONG) && n >= vec_of<T>() && !(q_across && fetchable && one_launch<T>(n, k));
}

// Their plan: bm = 0, bn = the lanes along a line (Q across k), slice_steps = a slice's k.  A CU gets 34 GB/s at most, all of them together 5.6 TB/s (28, 4.6 with eight lanes); slices of k
// spread a product of few columns over the CUs, evenly, and cost a second launch (4.5 us) and their bytes.
template <typename T>
Tiles few_plan(int64_t m, int64_t n, int64_t k, bool across) {
  const double bytes = (double)n * k * sizeof(T);
  int64_t slices = 1;
  Tiles best = {0, 32, 1, 0};
  double shortest = INFINITY;
  for (const int lanes : {32, 8}) {
    if (!across && lanes != 32) break;
    const int64_t groups = ceil_div(n, across ? lanes * vec_of<T>() : FEW_COLS), least = across ? 256 : 2048;
    const double rate = across && lanes == 8 ? 4.6e6 : 5.6e6;
    for (int64_t s = 1; s <= std::max<int64_t>(1, std::min<int64_t>(k / least, 64)); ++s) {
      const double all = (double)groups * s, on_one = std::ceil(all / 256);
      const double time = bytes / all * on_one / std::min(lanes == 8 ? 28e3 : 34e3, rate / std::min(all, 256.0)) +
                          (s > 1 ? 4.5 + (double)s * m * n * 2 * sizeof(typename Wide<T>::type) / 4e6 : 0);
      if (time < shortest) shortest = time, slices = s, best.bn = lanes;
    }
  }
  best.slice_steps = (int)round_up(ceil_div(k, slices), 64);
  best.slices = (int)ceil_div(k, best.slice_steps);
  return best;
}

template <typename T>
Tiles plan_of(int64_t m, int64_t n, int64_t k, bool p_across, bool q_across, bool few_rows) {
  if (few_rows) return few_plan<T>(m, n, k, q_across);
  const int64_t steps = ceil_div(k, step_of<T>());
  if (m <= 32 && !p_across && q_across && one_launch<T>(n, k)) return {32, 64, 1, (int)std::max<int64_t>(1, steps)};
  return tiles_of<T>(m, n, steps);
}

template <typename T>
int64_t product_bytes(const Tiles& t, int64_t m, int64_t n) {
  return t.slices > 1 ? round_up((int64_t)t.slices * m * n * (int64_t)sizeof(typename Wide<T>::type), 256) : 0;
}

template <typename T, int BM, int BN, int WM, int WN>
void product_as(const Product& g, bool p_across, bool q_across, const Tiles& t, typename Wide<T>::type* part, const Epilogue<T>& e, hipStream_t s) {
  const int tiles_m = (int)ceil_div(g.m, BM), tiles_n = (int)ceil_div(g.n, BN);
  const dim3 grid((unsigned)(tiles_m * tiles_n), (unsigned)t.slices);
  if (p_across) product_kernel<T, BM, BN, WM, WN, true, true><<<grid, 64 * WM * WN, 0, s>>>(g, tiles_m, tiles_n, t.slice_steps * step_of<T>(), part, e);      // (P across: x^T dz, Q too)
  else if (q_across) product_kernel<T, BM, BN, WM, WN, false, true><<<grid, 64 * WM * WN, 0, s>>>(g, tiles_m, tiles_n, t.slice_steps * step_of<T>(), part, e);
  else product_kernel<T, BM, BN, WM, WN, false, false><<<grid, 64 * WM * WN, 0, s>>>(g, tiles_m, tiles_n, t.slice_steps * step_of<T>(), part, e);
}

template <typename T, int M>
void product_few(const Product& g, bool q_across, const Tiles& t, typename Wide<T>::type* part, const Epilogue<T>& e, hipStream_t s) {
  const unsigned slices = (unsigned)t.slices;
  if (q_across) {
    if constexpr (M <= FEW_ACROSS) {
      if (t.bn == 32) few_across_kernel<T, M, 32><<<dim3((unsigned)ceil_div(g.n, 32 * vec_of<T>()), slices), 512, 0, s>>>(g, t.slice_steps, part, e);
      else few_across_kernel<T, M, 8><<<dim3((unsigned)ceil_div(g.n, 8 * vec_of<T>()), slices), 512, 0, s>>>(g, t.slice_steps, part, e);
    }
  } else if (g.k < 256 * vec_of<T>()) few_along_kernel<T, M, 1><<<dim3((unsigned)ceil_div(g.n, 4 * FEW_COLS), slices), 256, 0, s>>>(g, t.slice_steps, part, e);   // (four waves do not fill one turn)
  else few_along_kernel<T, M, 4><<<dim3((unsigned)ceil_div(g.n, FEW_COLS), slices), 256, 0, s>>>(g, t.slice_steps, part, e);
}

template <typename T>
void product(const Product& g, bool p_across, bool q_across, const Tiles& t, const Epilogue<T>& e, void* workspace, hipStream_t s) {
  typedef typename Wide<T>::type A;
  A* part = t.slices > 1 ? static_cast<A*>(workspace) : nullptr;
  if (t.bm == 0) {
    if (g.m == 1) product_few<T, 1>(g, q_across, t, part, e, s);
    else if (g.m == 2) product_few<T, 2>(g, q_across, t, part, e, s);
    else product_few<T, 4>(g, q_across, t, part, e, s);
  }
  if constexpr (sizeof(T) == 2) {
    if (t.bm == 256) product_as<T, 256, 256, 2, 4>(g, p_across, q_across, t, part, e, s);
    if (t.bm == 128 && t.bn == 128) product_as<T, 128, 128, 2, 2>(g, p_across, q_across, t, part, e, s);
    if (t.bm == 32 && t.bn == 64) {
      const int tiles = (int)ceil_div(g.n, 64);
      product_kernel<T, 32, 64, 1, 4, false, true><<<tiles, 256, 0, s>>>(g, 1, tiles, t.slice_steps * step_of<T>(), nullptr, e);
    }
  }
  if (t.bm == 64) product_as<T, 64, 64, 2, 2>(g, p_across, q_across, t, part, e, s);
  else if (t.bm == 128 && t.bn == 32) product_as<T, 128, 32, 4, 1>(g, p_across, q_across, t, part, e, s);
  else if (t.bm == 32 && t.bn == 128) product_as<T, 32, 128, 1, 4>(g, p_across, q_across, t, part, e, s);
  else if (t.bm == 32 && t.bn == 32) product_as<T, 32, 32, 2, 2>(g, p_across, q_across, t, part, e, s);
  if (!part) return;
  const int64_t lanes = (int64_t)g.m * ((g.n + 3) / 4);
  if (t.slices > 16) product_join_kernel<T, 32><<<(unsigned)ceil_div(lanes, 8), 256, 0, s>>>(part, t.slices, g.m, g.n, e);
  else product_join_kernel<T, 1><<<(unsigned)ceil_div(lanes, 256), 256, 0, s>>>(part, t.slices, g.m, g.n, e);
}

// A matrix operand in memory: `lines` of `n` elements behind each other, `ld` apart.
struct Lines {
  const void* p;
  int64_t lines, n, ld;
};

// Whether the products can fetch it: lines at multiples of four bytes (every fp32 and fp64 operand, 16-bit ones of an even pitch).  What they cannot is
// copied into lines of whole 16-byte chunks first.
template <typename T>
bool fetchable(const Lines& o) {
  return reinterpret_cast<uintptr_t>(o.p) % 4 == 0 && o.ld * (int64_t)sizeof(T) % 4 == 0;
}

template <typename T>
struct Dense {
  typedef typename Wide<T>::type A;
  typedef typename Slope<T>::type S;

  // A walk over a call's launches.  Without a workspace it only adds up what they need of one.
  char* workspace;
  hipStream_t stream;
  int64_t used = 0, most = 0;
  bool launch, too_many = false;      // too_many: a product's tiles are more than one launch takes
  Jobs<T> jobs;
  Dense(void* w, hipStream_t s, bool l) : workspace(static_cast<char*>(w)), stream(s), launch(l) { jobs.count = jobs.blocks = 0; }

  void* take(int64_t bytes) {
    void* p = workspace ? workspace + used : nullptr;
    used += round_up(bytes, 256);
    most = std::max(most, used);
    return p;
  }

  // A job of the launch before the products; its groups are also the rows of `partial`.
  Job<T> job_of(const Lines& o) {
    Job<T> b = {static_cast<const T*>(o.p), o.ld, o.lines, o.n, nullptr, 1, nullptr, o.n, nullptr, nullptr, 5, 1, 1, 0};
    while (b.lanes_log2 > 2 && (int64_t)vec_of<T>() << (b.lanes_log2 - 1) >= o.n) --b.lanes_log2;
    return b;
  }
  void add(Job<T> b) {
    Jobs<T>& all = jobs;
    b.first = all.blocks;
    all.job[all.count++] = b;
    all.blocks += b.col_blocks * b.groups;
  }
  // workgroups: some 2048 along both axes, at most 512 along the lines
  static void shape(Job<T>& b, int64_t width) {
    b.col_blocks = (int)ceil_div(width, (int64_t)vec_of<T>() << b.lanes_log2);
    const int64_t rounds = ceil_div(b.lines, 256 >> b.lanes_log2);
    b.groups = rounds <= 4 ? 1 : (int)std::min<int64_t>(std::min<int64_t>(512, std::max(1, 2048 / b.col_blocks)), rounds);
  }
  void launch_jobs() {
    if (launch && jobs.count) prepare_kernel<T><<<jobs.blocks, 256, 0, stream>>>(jobs);
    jobs.count = jobs.blocks = 0;
  }

  // an operand that the products can fetch
  Lines ready(Lines o) {
    if (fetchable<T>(o)) return o;
    const int64_t ld = round_up(o.n, vec_of<T>());
    Job<T> b = job_of(o);
    b.to = static_cast<T*>(take(o.lines * ld * (int64_t)sizeof(T)));
    b.ld_to = ld;
    shape(b, ld);
    if (o.lines) add(b);
    return {b.to, o.lines, o.n, ld};
  }

  void multiply(const Lines& p, bool p_across, const Lines& q, bool q_across, int64_t m, int64_t n, int64_t k, const Epilogue<T>& e) {
    const Tiles t = plan_of<T>(m, n, k, p_across, q_across, !p_across && few<T>(m, n, k, q_across, fetchable<T>(q)));
    if (t.bm && ceil_div(m, t.bm) * ceil_div(n, t.bn) * (t.bm == 256 ? 512 : 256) >= (int64_t)1 << 32) too_many = true;      // (a launch has 2^32 lanes along an axis)
    const int64_t bytes = product_bytes<T>(t, m, n);
    void* rest = bytes ? take(bytes) : nullptr;
    if (launch) product<T>({p.p, q.p, p.ld, q.ld, (int32_t)m, (int32_t)n, (int32_t)k}, p_across, q_across, t, e, rest, stream);
    used -= round_up(bytes, 256);
  }

  // The thin kernels' layers.  They read operands where they lie, so nothing else is asked of these.
  static bool thin(const vmcpde_dense_args& a) { return sizeof(T) > 2 && a.n_in <= THIN && a.n_out <= THIN; }

  template <int NT>
  void thin_forward(const vmcpde_dense_args& a, const Epilogue<T>& e) {
    const unsigned groups = (unsigned)std::min<int64_t>(ceil_div(a.rows, 64), 512);
    const T* x = static_cast<const T*>(a.x);
    const T* w = static_cast<const T*>(a.kernel);
    const int64_t sk = a.kernel_t ? 1 : a.ldk, sn = a.kernel_t ? a.ldk : 1;
    if (a.n_in <= 8) thin_forward_kernel<T, 2, NT><<<groups, 256, 0, stream>>>(x, a.ldx, w, sk, sn, a.rows, (int)a.n_in, e);
    else if (a.n_in <= 16) thin_forward_kernel<T, 4, NT><<<groups, 256, 0, stream>>>(x, a.ldx, w, sk, sn, a.rows, (int)a.n_in, e);
    else if (a.n_in <= 24) thin_forward_kernel<T, 6, NT><<<groups, 256, 0, stream>>>(x, a.ldx, w, sk, sn, a.rows, (int)a.n_in, e);
    else if (a.n_in <= 32) thin_forward_kernel<T, 8, NT><<<groups, 256, 0, stream>>>(x, a.ldx, w, sk, sn, a.rows, (int)a.n_in, e);
    else thin_forward_kernel<T, 12, NT><<<groups, 256, 0, stream>>>(x, a.ldx, w, sk, sn, a.rows, (int)a.n_in, e);
  }

  template <int KT, int NT>
  void thin_backward(const vmcpde_dense_args& a, unsigned groups, T* partial) {
    thin_backward_kernel<T, KT, NT><<<groups, THIN_THREADS, 0, stream>>>(
        static_cast<const T*>(a.dy), a.ldd, static_cast<const T*>(a.slope), (T)a.scale, a.dkernel ? static_cast<const T*>(a.x) : nullptr, a.ldx,
        static_cast<const T*>(a.kernel), a.kernel_t ? 1 : a.ldk, a.kernel_t ? a.ldk : 1, a.rows, (int)a.n_in, (int)a.n_out, static_cast<T*>(a.dx), partial,
        static_cast<T*>(a.dkernel), static_cast<T*>(a.dbias));
  }

  template <int KT>
  void thin_backward_outputs(const vmcpde_dense_args& a, unsigned groups, T* partial) {
    if (a.n_out <= 16) thin_backward<KT, 1>(a, groups, partial);
    else if (a.n_out <= 32) thin_backward<KT, 2>(a, groups, partial);
    else thin_backward<KT, 3>(a, groups, partial);
  }

  void thin_backward(const vmcpde_dense_args& a) {
    const int64_t rounds = ceil_div(a.rows, 16 * (THIN_THREADS / 64)), groups = rounds <= 4 ? 1 : std::min<int64_t>(rounds, THIN_GROUPS), sums = (a.n_in + 1) * a.n_out;
    T* partial = a.dkernel || a.dbias ? static_cast<T*>(take(groups * sums * (int64_t)sizeof(T))) : nullptr;
    if (!launch || (!partial && !(a.dx && a.rows))) return;
    if (a.n_in <= 16) thin_backward_outputs<1>(a, (unsigned)groups, partial);
    else if (a.n_in <= 32) thin_backward_outputs<2>(a, (unsigned)groups, partial);
    else thin_backward_outputs<3>(a, (unsigned)groups, partial);
    if (partial && groups > 1)
      add_columns<T, T>(partial, groups, sums, a.n_in * a.n_out, a.n_out, static_cast<T*>(a.dkernel), static_cast<T*>(a.dbias), stream);
  }

  void forward(const vmcpde_dense_args& a) {
    if (!a.rows) return;
    const Epilogue<T> e = {static_cast<const T*>(a.bias), static_cast<const T*>(a.residual), a.ldr, static_cast<T*>(a.y), a.ldy, static_cast<S*>(a.slope), a.n_out,
                           (A)a.scale, a.activation};
    if constexpr (sizeof(T) > 2) {
      if (thin(a)) {
        if (launch) a.n_out <= 16 ? thin_forward<1>(a, e) : a.n_out <= 32 ? thin_forward<2>(a, e) : thin_forward<3>(a, e);
        return;
      }
    }
    Lines x = {a.x, a.rows, a.n_in, a.ldx}, kernel = kernel_lines(a);
    if (!few<T>(a.rows, a.n_out, a.n_in, !a.kernel_t, fetchable<T>(kernel))) x = ready(x), kernel = ready(kernel);
    launch_jobs();
    multiply(x, false, kernel, !a.kernel_t, a.rows, a.n_out, a.n_in, e);
  }

  static Lines kernel_lines(const vmcpde_dense_args& a) {
    return a.kernel_t ? Lines{a.kernel, a.n_out, a.n_in, a.ldk} : Lines{a.kernel, a.n_in, a.n_out, a.ldk};
  }

  void backward(const vmcpde_dense_args& a) {
    if constexpr (sizeof(T) > 2) {
      if (thin(a)) return thin_backward(a);
    }
    const Lines dy = {a.dy, a.rows, a.n_out, a.ldd};
    Lines dz = dy;
    const bool own = (a.dx || a.dkernel) && (a.slope || !fetchable<T>(dy));
    Job<T> b = job_of(dy);
    if (own) {
      b.ld_to = round_up(a.n_out, vec_of<T>());
      b.to = static_cast<T*>(take(a.rows * b.ld_to * (int64_t)sizeof(T)));
      dz = {b.to, a.rows, a.n_out, b.ld_to};
    }
    shape(b, own ? b.ld_to : a.n_out);
    if (own || a.dbias) {
      b.slope = static_cast<const S*>(a.slope);
      b.scale = (A)a.scale;
      b.sums = static_cast<T*>(a.dbias);
      if (a.dbias && b.groups > 1) b.partial = static_cast<A*>(take(b.groups * a.n_out * (int64_t)sizeof(A)));
      add(b);
    }
    const bool want_x = a.dx && a.rows;
    Lines kernel = want_x ? kernel_lines(a) : Lines();
    if (want_x && !few<T>(a.rows, a.n_in, a.n_out, a.kernel_t, fetchable<T>(kernel))) kernel = ready(kernel);
    const Lines x = a.dkernel ? ready({a.x, a.rows, a.n_in, a.ldx}) : Lines();
    launch_jobs();
    if (launch && b.partial) add_columns<A, T>(b.partial, b.groups, a.n_out, a.n_out, 0, static_cast<T*>(a.dbias), nullptr, stream);
    if (want_x) {
      const Epilogue<T> e = {nullptr, nullptr, 0, static_cast<T*>(a.dx), a.n_in, nullptr, a.n_in, (A)a.scale, VMCPDE_ACT_NONE};
      multiply(dz, false, kernel, a.kernel_t, a.rows, a.n_in, a.n_out, e);
    }
    if (a.dkernel) {
      const Epilogue<T> e = {nullptr, nullptr, 0, static_cast<T*>(a.dkernel), a.n_out, nullptr, a.n_out, (A)a.scale, VMCPDE_ACT_NONE};
      multiply(x, true, dz, true, a.n_in, a.n_out, a.rows, e);
    }
  }
};

// the bytes of workspace that the call needs, -1: more tiles than a launch takes; `launch`: the call itself
template <typename T>
int64_t walk(const vmcpde_dense_args& a, bool backward, void* workspace, hipStream_t s, bool launch) {
  Dense<T> d(workspace, s, launch);
  if (backward) d.backward(a);
  else d.forward(a);
  return d.too_many ? -1 : d.most;
}

int64_t walk_type(const vmcpde_dense_args& a, bool backward, void* workspace, hipStream_t s, bool launch) {
  switch (a.dtype) {
    case VMCPDE_F64: return walk<double>(a, backward, workspace, s, launch);
    case VMCPDE_F32: return walk<float>(a, backward, workspace, s, launch);
    case VMCPDE_F16: return walk<f16_t>(a, backward, workspace, s, launch);
    default: return walk<bf16_t>(a, backward, workspace, s, launch);
  }
}

int check(const vmcpde_dense_args* a, bool backward) {
  constexpr int64_t LIMIT = (int64_t)1 << 30;
  VMC_REQUIRE(a, "dense: null arguments");
  VMC_REQUIRE(dtype_ok(a->dtype), "dense: type %d", a->dtype);
  VMC_REQUIRE(a->activation >= VMCPDE_ACT_NONE && a->activation <= VMCPDE_ACT_SILU, "dense: activation %d", a->activation);
  VMC_REQUIRE(a->rows >= 0 && a->rows < LIMIT && a->n_in >= 1 && a->n_in < LIMIT && a->n_out >= 1 && a->n_out < LIMIT,
              "dense: rows %lld, n_in %lld, n_out %lld (rows from 0, widths from 1, all below 2^30)", (long long)a->rows, (long long)a->n_in, (long long)a->n_out);
  const int64_t pitch = (int64_t)1 << (a->dtype == VMCPDE_F64 ? 21 : 22);
  VMC_REQUIRE(std::max(std::max(a->n_in, a->n_out), std::max(a->ldx, std::max(a->ldk, a->ldd))) < pitch, "dense: widths and row pitches are below %lld for this type",
              (long long)pitch);     // (a tile's rows lie within 2^31 bytes of each other)
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
  const int64_t bytes = walk_type(*a, backward != 0, nullptr, nullptr, false);
  VMC_REQUIRE(bytes >= 0, "dense: rows %lld, n_in %lld, n_out %lld: a product of 2^24 tiles and more (64 x 64 in fp32 and fp64)", (long long)a->rows, (long long)a->n_in,
              (long long)a->n_out);
  return bytes;
}

static int run(const vmcpde_dense_args* a, bool backward, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check(a, backward)) return rc;
  if (!backward && a->rows == 0) return 0;
  const int64_t need = vmcpde_dense_workspace_bytes(a, backward);
  if (need < 0) return -1;
  VMC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "dense: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  VMC_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "dense: the workspace is not aligned to 16 bytes");
  walk_type(*a, backward, workspace, static_cast<hipStream_t>(stream), true);
  VMC_CHECK_HIP(hipGetLastError());
  return 0;
}

int vmcpde_dense(const vmcpde_dense_args* a, void* workspace, int64_t workspace_bytes, void* stream) { return run(a, false, workspace, workspace_bytes, stream); }
int vmcpde_dense_backward(const vmcpde_dense_args* a, void* workspace, int64_t workspace_bytes, void* stream) { return run(a, true, workspace, workspace_bytes, stream); }

}  // extern "C"
