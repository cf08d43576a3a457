// Global norm of many tensors, and clipping by it:  n = sqrt(sum_t sum_i t_i^2),  out = t * (n > max ? max / n : 1).
//
// Bound by memory: the factor is known after the last element only, so clipping reads everything twice and writes it once.  Squares are
// summed in fp64 whatever the element type (fp32 and 16-bit squares neither overflow nor vanish there); fp64 elements are summed in three
// bins -- huge, ordinary, tiny, the outer two scaled by a power of two before they are squared -- so no finite norm overflows or vanishes.
// The tensors travel as a table in the kernel arguments (no copy to the device, and a captured launch keeps its own table).  Every
// workgroup reads one chunk of one tensor and leaves one partial; a single workgroup adds the partials in index order, so the norm does not
// depend on which workgroup ends first.  500 million bf16 and fp32 numbers (1 GB) in 290 tensors: 550 us, 5.5 TB/s over the three passes.
#include <algorithm>
#include <new>
#include <vector>

#include "layers.hpp"

using namespace vmcpde;

namespace {

constexpr int TABLE = 112;             // tensors a launch: 112 x 32 bytes of kernel arguments, below the 4 KB that a launch may carry
constexpr int THREADS = 256;
constexpr int SMALL_THREADS = 1024;
constexpr int64_t SMALL_TOTAL = 32768; // up to here one workgroup reads, reduces and scales: one launch instead of three
constexpr int64_t SMALL_SHARED = 512;  // a tensor of that launch that all its waves share
constexpr int64_t MIN_CHUNK = 8192;
constexpr int64_t GROUPS = 16384;      // workgroups a launch aims at: short ones balance better than eight a CU (1 GB clipped: 2048 651, 8192 584, 16384 573 us)

// Borders of the bins: the middle one's squares, from 2^-1000 to 2^960, leave room for 2^64 of them; so do the huge ones', from 2^-240 to 2^848, and the tiny ones', up to 2^200.
constexpr double BIG = 0x1p480, TINY = 0x1p-500, DOWN = 0x1p-600, UP = 0x1p600;

struct Entry {
  const void* in;
  void* out;
  int64_t n;
  int32_t dtype;
  int32_t first;   // first workgroup of this tensor in the launch
};
struct Table {
  Entry e[TABLE];
  int32_t count, groups, shared;
  int64_t chunk;
};

struct Bins { double big, mid, tiny; };

template <typename T>
__device__ __forceinline__ void add_square(Bins& b, T value) {
  if constexpr (sizeof(T) == 8) {
    const double a = fabs((double)value);
    if (a > BIG) { const double s = a * DOWN; b.big = fma(s, s, b.big); }
    else if (a < TINY) { const double s = a * UP; b.tiny = fma(s, s, b.tiny); }
    else b.mid = fma(a, a, b.mid);        // (NaN comes here)
  } else {
    const double a = (double)(float)value;
    b.mid = fma(a, a, b.mid);
  }
}

__device__ __forceinline__ double join(const Bins& b) {
  if (b.mid != b.mid) return b.mid;
  if (b.big > 0) return sqrt(b.big + b.mid * DOWN * DOWN) * UP;
  if (b.mid > 0) return sqrt(b.mid + b.tiny * DOWN * DOWN);
  return sqrt(b.tiny) * DOWN;
}

typedef unsigned int uint4v __attribute__((ext_vector_type(4), aligned(2)));   // what the nontemporal builtins take

// 16 bytes a lane at any alignment (global memory takes unaligned vectors): which lane adds which element goes by the index alone, so the norm
// of the same numbers has the same bits wherever they lie
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[16 / sizeof(T)]; };

template <typename T>
__device__ void square_span(const T* __restrict__ p, int64_t n, int t, int threads, Bins& b) {
  constexpr int V = vec_of<T>();
  const int64_t vecs = n / V, tail = vecs * V;
  const Raw<T>* q = reinterpret_cast<const Raw<T>*>(p);
  int64_t j = t;
  for (; j + 3 * threads < vecs; j += 4 * threads) {   // four loads in flight a thread
    Raw<T> r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = q[j + u * threads];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) add_square(b, r[u].v[k]);
  }
  for (; j < vecs; j += threads) {
    const Raw<T> r = q[j];
#pragma unroll
    for (int k = 0; k < V; ++k) add_square(b, r.v[k]);
  }
  if (tail + t < n) add_square(b, p[tail + t]);
}

// What clipping multiplies by: f 2^e.  Far below 1 (2^-100) f is kept in [1/4, 1), so that neither max / norm in fp64 nor f in fp32 is a subnormal number, which has lost
// digits that the clipped elements, ordinary numbers at most max_norm, still have.
struct Factor {
  double f;
  int32_t e;
};
__device__ __forceinline__ Factor clip_factor(double norm, double max_norm) {
  if (!(norm > max_norm)) return {1.0, 0};                   // (NaN comes here)
  const double q = max_norm / norm;
  if (q >= 0x1p-100 || max_norm == 0 || norm == INFINITY) return {q, 0};
  int en, em;
  const double mn = frexp(norm, &en), mm = frexp(max_norm, &em);
  return {0.5 * mm / mn, em - en + 1};
}
template <bool FAR = true, typename T, typename A>
__device__ __forceinline__ T scaled(T v, A f, int e) {
  const A r = (A)v * f;
  if constexpr (!FAR) return (T)r;
  else if constexpr (sizeof(A) == 8) return (T)ldexp(r, e);
  else return (T)ldexpf(r, e);
}

// FAR: e is not 0 (asked once: with its power of two for every element 1 GB clipped took 558 us, not 550)
template <bool FAR, typename T>
__device__ void scale_span(const T* p, T* o, int64_t n, int t, int threads, Factor factor) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>();
  const A f = (A)factor.f;
  const int e = factor.e;
  const int64_t vecs = n / V, tail = vecs * V;
  const Raw<T>* q = reinterpret_cast<const Raw<T>*>(p);
  Raw<T>* w = reinterpret_cast<Raw<T>*>(o);
  int64_t j = t;
  for (; j + 3 * threads < vecs; j += 4 * threads) {
    Raw<T> r[4];                                       // nobody reads these soon: past the caches (400 MB 233 -> 191 us, 1 GB 573 -> 550 us; up to 200 MB alike)
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = __builtin_bit_cast(Raw<T>, __builtin_nontemporal_load(reinterpret_cast<const uint4v*>(q + j + u * threads)));
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int k = 0; k < V; ++k) r[u].v[k] = scaled<FAR>(r[u].v[k], f, e);
      __builtin_nontemporal_store(__builtin_bit_cast(uint4v, r[u]), reinterpret_cast<uint4v*>(w + j + u * threads));
    }
  }
  for (; j < vecs; j += threads) {
    Raw<T> r = q[j];
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = scaled<FAR>(r.v[k], f, e);
    w[j] = r;
  }
  if (tail + t < n) o[tail + t] = scaled<FAR>(p[tail + t], f, e);
}

__device__ void square_any(const Entry& e, int64_t at, int64_t n, int t, int threads, Bins& b) {
  switch (e.dtype) {
    case VMCPDE_F64: square_span(static_cast<const double*>(e.in) + at, n, t, threads, b); break;
    case VMCPDE_F32: square_span(static_cast<const float*>(e.in) + at, n, t, threads, b); break;
    case VMCPDE_F16: square_span(static_cast<const f16_t*>(e.in) + at, n, t, threads, b); break;
    default: square_span(static_cast<const bf16_t*>(e.in) + at, n, t, threads, b);
  }
}

template <typename T>
__device__ __forceinline__ void scale_typed(const Entry& e, int64_t at, int64_t n, int t, int threads, Factor factor) {
  const T* p = static_cast<const T*>(e.in) + at;
  T* o = static_cast<T*>(e.out) + at;
  if (factor.e) scale_span<true>(p, o, n, t, threads, factor);
  else scale_span<false>(p, o, n, t, threads, factor);
}
__device__ void scale_any(const Entry& e, int64_t at, int64_t n, int t, int threads, Factor factor) {
  switch (e.dtype) {
    case VMCPDE_F64: scale_typed<double>(e, at, n, t, threads, factor); break;
    case VMCPDE_F32: scale_typed<float>(e, at, n, t, threads, factor); break;
    case VMCPDE_F16: scale_typed<f16_t>(e, at, n, t, threads, factor); break;
    default: scale_typed<bf16_t>(e, at, n, t, threads, factor);
  }
}

// sum over the workgroup, thread 0 has it; the waves are added in their order
template <int WAVES>
__device__ Bins group_bins(Bins b) {
  __shared__ Bins sh[WAVES];
  b.big = wave_sum(b.big);
  b.mid = wave_sum(b.mid);
  b.tiny = wave_sum(b.tiny);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = b;
  __syncthreads();
  Bins s = sh[0];
  for (int w = 1; w < WAVES; ++w) { s.big += sh[w].big; s.mid += sh[w].mid; s.tiny += sh[w].tiny; }
  return s;
}

// the tensor that workgroup g of the launch works on: the last whose first workgroup is not behind g
__device__ __forceinline__ int find(const Table& tab, int g) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.e[mid].first <= g) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(THREADS) void squares_kernel(Table tab, Bins* __restrict__ partial) {
  const int g = blockIdx.x;
  const Entry& e = tab.e[find(tab, g)];
  const int64_t at = (int64_t)(g - e.first) * tab.chunk, left = e.n - at;
  Bins b = {0, 0, 0};
  square_any(e, at, left < tab.chunk ? left : tab.chunk, threadIdx.x, THREADS, b);
  b = group_bins<THREADS / 64>(b);
  if (threadIdx.x == 0) partial[g] = b;
}

__global__ __launch_bounds__(SMALL_THREADS) void join_kernel(const Bins* __restrict__ partial, int n, double max_norm, double* __restrict__ norm,
                                                             Factor* __restrict__ factor) {
  Bins b = {0, 0, 0};
  for (int j = threadIdx.x; j < n; j += SMALL_THREADS) { b.big += partial[j].big; b.mid += partial[j].mid; b.tiny += partial[j].tiny; }
  b = group_bins<SMALL_THREADS / 64>(b);
  if (threadIdx.x == 0) {
    const double v = join(b);
    *norm = v;
    if (factor) *factor = clip_factor(v, max_norm);
  }
}

__global__ __launch_bounds__(THREADS) void scale_kernel(Table tab, const Factor* __restrict__ factor) {
  const int g = blockIdx.x;
  const Entry& e = tab.e[find(tab, g)];
  const Factor f = *factor;
  if (f.f == 1.0 && e.in == e.out) return;       // (a far factor's f is below 1)
  const int64_t at = (int64_t)(g - e.first) * tab.chunk, left = e.n - at;
  scale_any(e, at, left < tab.chunk ? left : tab.chunk, threadIdx.x, THREADS, f);
}

// The kernel's first argument, brought into LDS at once: the arguments lie in the host's memory, and entry after entry each is a trip of its own (2 us).
template <typename S>
__device__ __forceinline__ void stage_arguments(S& to) {
  static_assert(sizeof(S) % 4 == 0, "whole words");
  const auto* from = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
  for (int u = threadIdx.x; u < (int)(sizeof(S) / 4); u += blockDim.x) reinterpret_cast<uint32_t*>(&to)[u] = from[u];
  __syncthreads();
}

// everything in one workgroup: a few thousand numbers cost three launches more than their arithmetic
__global__ __launch_bounds__(SMALL_THREADS) void small_kernel(Table, int clip, double max_norm, double* __restrict__ norm) {
  __shared__ Factor shared_factor;
  __shared__ Table tab;
  stage_arguments(tab);
  Bins b = {0, 0, 0};
  // leaves are mostly shorter than a wave: a wave takes every sixteenth tensor, and all of them share one that is long
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int k = 0; k < tab.shared; ++k) square_any(tab.e[k], 0, tab.e[k].n, threadIdx.x, SMALL_THREADS, b);
  for (int k = tab.shared + wave; k < tab.count; k += SMALL_THREADS / 64) square_any(tab.e[k], 0, tab.e[k].n, lane, 64, b);
  b = group_bins<SMALL_THREADS / 64>(b);
  if (threadIdx.x == 0) {
    const double v = join(b);
    *norm = v;
    shared_factor = clip_factor(v, max_norm);
  }
  __syncthreads();
  if (!clip) return;
  const Factor f = shared_factor;
  for (int k = 0; k < tab.shared; ++k) scale_any(tab.e[k], 0, tab.e[k].n, threadIdx.x, SMALL_THREADS, f);
  for (int k = tab.shared + wave; k < tab.count; k += SMALL_THREADS / 64) scale_any(tab.e[k], 0, tab.e[k].n, lane, 64, f);
}

// The same for tensors of one type that fit the workgroup's registers, in pieces of 64 elements: every element is read once and all loads fly together.
// 4213 fp64 numbers in 51 tensors (the leaves of a flow): 5.2 us against 10.
template <int PIECES>      // of a wave: eight where they do, in fp64 (its three bins) the adding of absent ones takes 3 us
struct Flat {
  static constexpr int ALL = PIECES * SMALL_THREADS / 64;
  static_assert(TABLE <= 256, "a byte numbers the tensors");
  Entry e[TABLE];          // `first`: the tensor's first piece
  int32_t pieces;
  uint8_t tensor[ALL];
};

template <typename T, int PIECES>
__global__ __launch_bounds__(SMALL_THREADS) void flat_kernel(Flat<PIECES>, int clip, double max_norm, double* __restrict__ norm) {
  typedef typename Wide<T>::type A;
  __shared__ Factor shared_factor;
  __shared__ Flat<PIECES> tab;
  stage_arguments(tab);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, pieces = tab.pieces;
  T v[PIECES];
#pragma unroll
  for (int j = 0; j < PIECES; ++j) {                   // (no branches: a lane without an element reads the tensor's first, so that all loads fly at once)
    const int c = wave + j * (SMALL_THREADS / 64);
    const Entry& e = tab.e[tab.tensor[min(c, pieces - 1)]];
    const int at = (c - e.first) * 64 + lane;
    const bool mine = c < pieces && at < e.n;
    const T x = static_cast<const T*>(e.in)[mine ? at : 0];
    v[j] = mine ? x : (T)0;
  }
  Bins b = {0, 0, 0};
#pragma unroll
  for (int j = 0; j < PIECES; ++j) add_square(b, v[j]);
  b = group_bins<SMALL_THREADS / 64>(b);
  if (threadIdx.x == 0) {
    const double n = join(b);
    *norm = n;
    shared_factor = clip_factor(n, max_norm);
  }
  __syncthreads();
  if (!clip) return;
  const A f = (A)shared_factor.f;
  const int f_e = shared_factor.e;
#pragma unroll
  for (int j = 0; j < PIECES; ++j) {
    const int c = wave + j * (SMALL_THREADS / 64);
    if (c >= pieces) break;
    const Entry& e = tab.e[tab.tensor[c]];
    const int at = (c - e.first) * 64 + lane;
    if (at < e.n) static_cast<T*>(e.out)[at] = scaled(v[j], f, f_e);
  }
}

// Launches flat_kernel; false: it does not take these tensors (several types, or too many pieces).
template <int PIECES>
bool flat(const vmcpde_tensor* t, int32_t count, int clip, double max_norm, double* norm, hipStream_t s) {
  Flat<PIECES> tab;
  int32_t filled = 0, dtype = 0;
  tab.pieces = 0;
  for (int32_t k = 0; k < count; ++k) {
    if (t[k].n == 0) continue;
    const int64_t pieces = ceil_div(t[k].n, 64);
    if (filled == TABLE || (filled && t[k].dtype != dtype) || tab.pieces + pieces > tab.ALL) return false;
    dtype = t[k].dtype;
    tab.e[filled] = {t[k].in, t[k].out, t[k].n, t[k].dtype, tab.pieces};
    for (int64_t c = 0; c < pieces; ++c) tab.tensor[tab.pieces++] = (uint8_t)filled;
    ++filled;
  }
  if (!filled) return false;
  if (dtype == VMCPDE_F64) flat_kernel<double><<<1, SMALL_THREADS, 0, s>>>(tab, clip, max_norm, norm);
  else if (dtype == VMCPDE_F32) flat_kernel<float><<<1, SMALL_THREADS, 0, s>>>(tab, clip, max_norm, norm);
  else if (dtype == VMCPDE_F16) flat_kernel<f16_t><<<1, SMALL_THREADS, 0, s>>>(tab, clip, max_norm, norm);
  else flat_kernel<bf16_t><<<1, SMALL_THREADS, 0, s>>>(tab, clip, max_norm, norm);
  return true;
}

struct Plan {
  int64_t total = 0, chunk = MIN_CHUNK, groups = 0;   // groups: of all launches
  bool small = false;
};

// the whole call's chunk length, and how many workgroups (= partials) it makes
Plan plan_of(const vmcpde_tensor* t, int32_t count) {
  Plan p;
  for (int32_t k = 0; k < count; ++k) p.total += t[k].n;
  const int64_t launches = count > TABLE ? ceil_div(count, TABLE) : 1;
  p.chunk = round_up(ceil_div(p.total, GROUPS * launches), MIN_CHUNK);
  if (p.chunk < MIN_CHUNK) p.chunk = MIN_CHUNK;
  for (int32_t k = 0; k < count; ++k) p.groups += ceil_div(t[k].n, p.chunk);
  p.small = p.total <= SMALL_TOTAL && count <= TABLE;
  return p;
}

int check_tensors(const vmcpde_tensor* t, int32_t count, bool write) {
  VMC_REQUIRE(count >= 0, "global norm: count = %d", count);
  VMC_REQUIRE(t || count == 0, "global norm: null table");
  for (int32_t k = 0; k < count; ++k) {
    VMC_REQUIRE(dtype_ok(t[k].dtype), "global norm: tensor %d has type %d", k, t[k].dtype);
    VMC_REQUIRE(t[k].n >= 0, "global norm: tensor %d has %lld elements", k, (long long)t[k].n);
    VMC_REQUIRE(t[k].n == 0 || (t[k].in && (!write || t[k].out)), "global norm: tensor %d is null", k);
    const int size = dtype_size(t[k].dtype);
    VMC_REQUIRE(reinterpret_cast<uintptr_t>(t[k].in) % size == 0 && (!write || reinterpret_cast<uintptr_t>(t[k].out) % size == 0),
                "global norm: tensor %d is not aligned to its elements", k);
  }
  return 0;
}

// What is written must be nothing else that is read or written; a tensor may be clipped in place.
int check_overlap(const vmcpde_tensor* t, int32_t count) {
  struct Span { uintptr_t begin, end; bool write; };
  std::vector<Span> spans;
  spans.reserve(2 * (size_t)count);
  for (int32_t k = 0; k < count; ++k)
    if (t[k].n && t[k].in != t[k].out) {
      const uintptr_t b = reinterpret_cast<uintptr_t>(t[k].in);
      spans.push_back({b, b + (uintptr_t)t[k].n * dtype_size(t[k].dtype), false});
    }
  for (int32_t k = 0; k < count; ++k)
    if (t[k].n) {
      const uintptr_t b = reinterpret_cast<uintptr_t>(t[k].out);
      spans.push_back({b, b + (uintptr_t)t[k].n * dtype_size(t[k].dtype), true});
    }
  auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  if (!std::is_sorted(spans.begin(), spans.end(), before)) std::sort(spans.begin(), spans.end(), before);
  uintptr_t any = 0, written = 0;
  for (const Span& s : spans) {
    VMC_REQUIRE(s.begin >= (s.write ? any : written), "vmcpde_global_norm: what one tensor is clipped into overlaps another tensor (the same tensor twice?)");
    any = std::max(any, s.end);
    if (s.write) written = std::max(written, s.end);
  }
  return 0;
}

// Fills tables of at most TABLE non-empty tensors and hands each to `launch(table, groups before it)`.
template <typename F>
int for_tables(const vmcpde_tensor* t, int32_t count, const Plan& p, F launch) {
  Table tab;
  tab.chunk = p.chunk;
  int64_t before = 0;
  for (int32_t j = 0; j < count;) {
    tab.count = 0;
    int64_t groups = 0;
    for (; j < count && tab.count < TABLE; ++j) {
      const vmcpde_tensor& e = t[j];
      if (e.n == 0) continue;
      tab.e[tab.count++] = {e.in, e.out, e.n, e.dtype, (int32_t)groups};
      groups += ceil_div(e.n, p.chunk);
    }
    tab.groups = (int32_t)groups;
    if (tab.count) {
      launch(tab, before);
      VMC_CHECK_HIP(hipGetLastError());
    }
    before += groups;
  }
  return 0;
}

}  // namespace

extern "C" {

int64_t vmcpde_global_norm_workspace_bytes(const vmcpde_tensor* tensors, int32_t count) {
  if (check_tensors(tensors, count, false)) return -1;
  const Plan p = plan_of(tensors, count);
  return p.small ? 0 : round_up(p.groups * (int64_t)sizeof(Bins) + (int64_t)sizeof(Factor), 256);
}

int vmcpde_global_norm(const vmcpde_tensor* tensors, int32_t count, int32_t clip, double max_norm, double* norm, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  if (const int rc = check_tensors(tensors, count, clip != 0)) return rc;
  VMC_REQUIRE(norm, "vmcpde_global_norm: null norm");
  VMC_REQUIRE(!clip || max_norm >= 0, "vmcpde_global_norm: max_norm = %g", max_norm);   // (refuses NaN too)
  if (clip) {
    try {
      if (const int rc = check_overlap(tensors, count)) return rc;
    } catch (const std::bad_alloc&) {
      VMC_REQUIRE(false, "vmcpde_global_norm: out of host memory");
    }
  }
  const Plan p = plan_of(tensors, count);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.small && (flat<8>(tensors, count, clip, max_norm, norm, s) || flat<16>(tensors, count, clip, max_norm, norm, s))) {
    VMC_CHECK_HIP(hipGetLastError());
    return 0;
  }
  if (p.small) {
    Table tab;
    tab.count = 0;
    for (bool shared : {true, false}) {      // the tensors that all waves share come first
      for (int32_t k = 0; k < count; ++k)
        if (tensors[k].n && (tensors[k].n > SMALL_SHARED) == shared) tab.e[tab.count++] = {tensors[k].in, tensors[k].out, tensors[k].n, tensors[k].dtype, 0};
      if (shared) tab.shared = tab.count;
    }
    small_kernel<<<1, SMALL_THREADS, 0, s>>>(tab, clip, max_norm, norm);
    VMC_CHECK_HIP(hipGetLastError());
    return 0;
  }
  const int64_t need = p.groups * (int64_t)sizeof(Bins) + (int64_t)sizeof(Factor);
  VMC_REQUIRE(workspace && workspace_bytes >= need, "vmcpde_global_norm: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  VMC_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "vmcpde_global_norm: the workspace is not aligned to 16 bytes");
  Bins* partial = static_cast<Bins*>(workspace);
  Factor* factor = reinterpret_cast<Factor*>(partial + p.groups);
  int rc = for_tables(tensors, count, p, [&](const Table& tab, int64_t before) { squares_kernel<<<tab.groups, THREADS, 0, s>>>(tab, partial + before); });
  if (rc) return rc;
  join_kernel<<<1, SMALL_THREADS, 0, s>>>(partial, (int)p.groups, max_norm, norm, clip ? factor : nullptr);
  VMC_CHECK_HIP(hipGetLastError());
  if (!clip) return 0;
  return for_tables(tensors, count, p, [&](const Table& tab, int64_t) { scale_kernel<<<tab.groups, THREADS, 0, s>>>(tab, factor); });
}

}  // extern "C"
