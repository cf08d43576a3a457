// Shared by the layer operators (dense.hip, layer_norm.hip, global_norm.hip): element types, reductions, small vectors.
#pragma once
#include "common.hpp"
#include "wave_ops.hpp"

namespace vmcpde {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Arithmetic type of an element type: sums, statistics and epilogues of 16-bit elements are held in fp32, of fp64 in fp64.
template <typename T> struct Wide { typedef float type; };
template <> struct Wide<double> { typedef double type; };
// act'(z) kept between the passes: fp16 for bf16, fp32 for fp16.  Every slope lies in [-0.13, 1.13]; rounded to the element type itself it would add an
// error as large as the output's own rounding to every gradient.  fp16 is finer than bf16 for slopes above 2^-16; below, its steps are 2^-24, and a slope under 2^-25
// is kept as zero: a bf16 tanh unit passes no gradient beyond |z| = 9.4 (where its output, rounded, has been +-1 since 3.5).  fp32 would keep those, for four bytes more
// an element written and read (8192 x 8192 x 4096: some 26 us of 1360).
template <typename T> struct Slope { typedef T type; };
template <> struct Slope<bf16_t> { typedef f16_t type; };
template <> struct Slope<f16_t> { typedef float type; };

inline int dtype_size(int dtype) { return dtype == VMCPDE_F64 ? 8 : dtype == VMCPDE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype >= VMCPDE_F64 && dtype <= VMCPDE_BF16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline int64_t ceil_div(int64_t v, int64_t m) { return (v + m - 1) / m; }

// Sum over groups of GROUP consecutive lanes (16 or 64), every lane of the group returns it, to the last bit: partners exchange in every step, so both add
// the same two numbers (rotations by four and eight do not: neighbouring quads' lanes added theirs in different orders).  DPP steps, no LDS.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int GROUP, typename A>
__device__ __forceinline__ A group_sum(A v) {
  static_assert(GROUP == 16 || GROUP == 64, "a DPP row or a wave");
  v += dpp_move<0xb1>(v);    // quad_perm [1,0,3,2]
  v += dpp_move<0x4e>(v);    // quad_perm [2,3,0,1]
  v += dpp_move<0x141>(v);   // row_half_mirror: the other quad of eight lanes, of which all lanes hold one sum
  v += dpp_move<0x140>(v);   // row_mirror: the other eight
  if constexpr (GROUP == 64) {
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
  }
  return v;
}

// elements of a 16-byte vector
template <typename T> constexpr int vec_of() { return 16 / (int)sizeof(T); }

// elements col .. col + V of a row, zero behind its end; 16 bytes a lane at any alignment (global memory takes unaligned vectors)
template <typename T, int V, typename A>
__device__ __forceinline__ void load_vec(const T* __restrict__ row, int64_t col, int64_t cols, A (&out)[V]) {
  struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[V]; };
  if (col + V <= cols) {
    const Raw r = *reinterpret_cast<const Raw*>(row + col);
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = (A)r.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = col + k < cols ? (A)row[col + k] : (A)0;
  }
}
template <typename T, int V, typename A>
__device__ __forceinline__ void store_vec(T* __restrict__ row, int64_t col, int64_t cols, const A (&in)[V]) {
  struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[V]; };
  if (col + V <= cols) {
    Raw r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = (T)in[k];
    *reinterpret_cast<Raw*>(row + col) = r;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (col + k < cols) row[col + k] = (T)in[k];
  }
}

// Last step of a sum over rows: columns col < cols0 of sum_g partial[g * pitch + col] go to out0, the cols1 behind them to out1 (a null one is skipped).
// 1024 / PARTS columns x PARTS parts of the groups a workgroup; a part's groups, then the parts, are added in their order.
template <typename A, typename W, int PARTS>
static __global__ __launch_bounds__(1024) void add_columns_kernel(const A* __restrict__ partial, int groups, int64_t pitch, int64_t cols0, int64_t cols1,
                                                                  W* __restrict__ out0, W* __restrict__ out1) {
  constexpr int COLS = 1024 / PARTS;
  __shared__ A sh[PARTS][COLS];
  const int part = threadIdx.x / COLS, c = threadIdx.x % COLS;
  const int64_t col = (int64_t)blockIdx.x * COLS + c;
  A v = 0;
  if (col < cols0 + cols1) {
#pragma unroll 8
    for (int g = part; g < groups; g += PARTS) v += partial[(int64_t)g * pitch + col];
  }
  sh[part][c] = v;
  __syncthreads();
  if (part == 0 && col < cols0 + cols1) {
#pragma unroll 8
    for (int p = 1; p < PARTS; ++p) v += sh[p][c];
    if (col < cols0) {
      if (out0) out0[col] = (W)v;
    } else if (out1) {
      out1[col - cols0] = (W)v;
    }
  }
}
// few columns: more lanes along the groups (42 columns of 1024 groups: one workgroup of 64 x 16 took 9 us)
template <typename A, typename W>
void add_columns(const A* partial, int64_t groups, int64_t pitch, int64_t cols0, int64_t cols1, W* out0, W* out1, hipStream_t s) {
  const int64_t cols = cols0 + cols1;
  if (cols <= 1024) add_columns_kernel<A, W, 64><<<(unsigned)ceil_div(cols, 16), 1024, 0, s>>>(partial, (int)groups, pitch, cols0, cols1, out0, out1);
  else add_columns_kernel<A, W, 16><<<(unsigned)ceil_div(cols, 64), 1024, 0, s>>>(partial, (int)groups, pitch, cols0, cols1, out0, out1);
}

}  // namespace vmcpde
