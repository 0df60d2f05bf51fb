// Norm of many tensors taken as one vector, and clipping by it.
//
//   norm = (sum |g|^p)^(1/p) over every entry of every tensor, p = 1, 2 or infinity
//   coef = min(1, max_norm / (norm + 1e-6));   out = round(g * coef)
//
// HBM-bound: the norm reads every entry once; clipping reads it again (the tensors of a model do
// not fit on the chip) and writes it once. The tensor list travels in the kernel's parameters, so a
// call copies nothing to the device and can be captured into a graph as it is. Tensors are cut into
// chunks of GR_CHUNK entries that the blocks take round robin: a list of large matrices and
// 1600-entry biases is spread evenly whatever its order.
// Every block leaves one partial sum; whoever needs the norm adds the partials in one fixed order,
// so the result does not depend on the order in which blocks run, and no atomics are used.
// Squares and sums are held in 64 bits: no entry of a 32-bit type overflows or vanishes when squared.
// Measured: norm of 3.1 GB in bf16 541 us, 5.8 TB/s; clipping the same into other tensors 1562 us, 6.0 TB/s with the
// second read; 3.1 GB of fp32 into bf16 1224 us, 6.3 TB/s. 28 small tensors: 8.0 us on the device.
#include <cstdlib>

#include <cuda_fp16.h>

#include "runtime.cuh"

namespace lsr {
namespace {

constexpr int GR_THREADS = 512;
constexpr int GR_CHUNK = 1 << 15;  // entries
constexpr int GR_TABLE = 1024;     // tensors per launch at most (30 bytes each of the 32764 bytes of kernel parameters)
constexpr int GR_SMALL = 96;       // a shorter list takes kernels with 3 KB of parameters instead of 30: less to copy per launch
constexpr int GR_CLUSTER = 8;      // blocks that take a short list in one launch
constexpr int GR_SHORT = 64;       // chunks of a short list
static_assert(GR_SHORT <= GR_SMALL, "a tensor has a chunk at least: only small tables hold short lists");
constexpr int GR_GRID = 592;       // blocks: 148 SMs x 4 blocks of 512 threads
enum : int { NORM_MAX = 0, NORM_ONE = 1, NORM_TWO = 2 };

template <int N>
struct GradTable {
  const void* in[N];
  void* out[N];
  long long numel[N];
  int first[N];  // first chunk of the tensor
  unsigned char tin[N], tout[N];
  int n, chunks;
};
static_assert(sizeof(GradTable<GR_TABLE>) <= 32000, "kernel parameters");

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// Running sum of |g|^p, or the largest |g| as the bits of a float: for values without a sign these
// order as integers, and a NaN is above infinity, so that it survives.
template <int KIND>
struct Acc {
  double s = 0.0;
  __device__ __forceinline__ void add(float x) {
    const double d = x;
    if (KIND == NORM_TWO) s = fma(d, d, s);
    else s += fabs(d);
  }
  __device__ __forceinline__ void join(const Acc& o) { s += o.s; }
  __device__ __forceinline__ Acc shfl(int o) const { Acc r; r.s = __shfl_xor_sync(0xffffffffu, s, o); return r; }
  __device__ __forceinline__ float norm() const { return (float)(KIND == NORM_TWO ? sqrt(s) : s); }
};
template <>
struct Acc<NORM_MAX> {
  unsigned long long s = 0;
  __device__ __forceinline__ void add(float x) {
    const unsigned long long b = __float_as_uint(x) & 0x7fffffffu;
    s = b > s ? b : s;
  }
  __device__ __forceinline__ void join(const Acc& o) { s = o.s > s ? o.s : s; }
  __device__ __forceinline__ Acc shfl(int o) const { Acc r; r.s = __shfl_xor_sync(0xffffffffu, s, o); return r; }
  __device__ __forceinline__ float norm() const { return __uint_as_float((unsigned)s); }
};

// Sum over the block, in a fixed order; every thread gets it.
template <int KIND>
__device__ __forceinline__ Acc<KIND> block_sum(Acc<KIND> a) {
  __shared__ Acc<KIND> part[GR_THREADS / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) a.join(a.shfl(o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  Acc<KIND> r = part[0];
#pragma unroll
  for (int w = 1; w < GR_THREADS / 32; ++w) r.join(part[w]);
  return r;
}

// The tensor that holds chunk c.
template <int N>
__device__ __forceinline__ int find_tensor(const GradTable<N>& t, int c) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Entries of [p, p + n) before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
  const int h = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
  return h < n ? h : n;
}

template <typename T, int KIND>
__device__ __forceinline__ void norm_chunk(const T* __restrict__ p, int n, Acc<KIND>& acc) {
  constexpr int V = 16 / sizeof(T);
  const int head = head_of(p, n), nv = (n - head) / V, done = head + nv * V;
  const int tid = threadIdx.x;
  if (tid < head) acc.add(to_f(p[tid]));
  if (tid < n - done) acc.add(to_f(p[done + tid]));
  const uint4* v = reinterpret_cast<const uint4*>(p + head);
#pragma unroll 4
  for (int i = tid; i < nv; i += GR_THREADS) {
    const uint4 x = v[i];
    const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int k = 0; k < V; ++k) acc.add(to_f(e[k]));
  }
}

// The calling thread's part of the chunks first, first + step, ...
template <int KIND, int N>
__device__ __forceinline__ Acc<KIND> norm_chunks(const GradTable<N>& t, int first, int step) {
  Acc<KIND> acc;
  for (int c = first; c < t.chunks; c += step) {
    const int k = find_tensor(t, c);
    const long long at = (long long)(c - t.first[k]) * GR_CHUNK;
    const int n = (int)min((long long)GR_CHUNK, t.numel[k] - at);
    if (t.tin[k] == LSR_DTYPE_F32) norm_chunk(static_cast<const float*>(t.in[k]) + at, n, acc);
    else if (t.tin[k] == LSR_DTYPE_BF16) norm_chunk(static_cast<const __nv_bfloat16*>(t.in[k]) + at, n, acc);
    else norm_chunk(static_cast<const __half*>(t.in[k]) + at, n, acc);
  }
  return acc;
}

template <int KIND, int N>
__global__ void __launch_bounds__(GR_THREADS) grad_norm_kernel(const __grid_constant__ GradTable<N> t,
                                                               Acc<KIND>* __restrict__ partial) {
  const Acc<KIND> acc = block_sum(norm_chunks<KIND>(t, (int)blockIdx.x, (int)gridDim.x));
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

template <int KIND>
__device__ __forceinline__ float total_norm(const Acc<KIND>* __restrict__ partial, int n) {
  Acc<KIND> acc;
  for (int i = threadIdx.x; i < n; i += GR_THREADS) acc.join(partial[i]);
  return block_sum(acc).norm();
}

template <int KIND>
__global__ void __launch_bounds__(GR_THREADS) grad_norm_finish_kernel(const Acc<KIND>* __restrict__ partial, int n,
                                                                      float* __restrict__ norm) {
  const float r = total_norm<KIND>(partial, n);
  if (threadIdx.x == 0) *norm = r;
}

// in and out may be the same tensor, so neither pointer is restrict.
template <typename TI, typename TO>
__device__ __forceinline__ void scale_chunk(const TI* p, TO* q, int n, float coef) {
  const int tid = threadIdx.x;
  // out's vectors start where its first 16-byte boundary is; in's have to start there too
  const int head = head_of(q, n);
  if ((reinterpret_cast<uintptr_t>(p + head) & 15) == 0) {
    constexpr int V = 8;
    const int nv = (n - head) / V, done = head + nv * V;
    if (tid < head) q[tid] = from_f<TO>(to_f(p[tid]) * coef);
    if (tid < n - done) q[done + tid] = from_f<TO>(to_f(p[done + tid]) * coef);
#pragma unroll 2
    for (int i = tid; i < nv; i += GR_THREADS) {
      alignas(16) TI x[V];
      alignas(16) TO y[V];
#pragma unroll
      for (int k = 0; k < (int)(V * sizeof(TI) / 16); ++k)
        reinterpret_cast<uint4*>(x)[k] = reinterpret_cast<const uint4*>(p + head + (size_t)i * V)[k];
#pragma unroll
      for (int k = 0; k < V; ++k) y[k] = from_f<TO>(to_f(x[k]) * coef);
#pragma unroll
      for (int k = 0; k < (int)(V * sizeof(TO) / 16); ++k)
        reinterpret_cast<uint4*>(q + head + (size_t)i * V)[k] = reinterpret_cast<const uint4*>(y)[k];
    }
  } else {
    for (int i = tid; i < n; i += GR_THREADS) q[i] = from_f<TO>(to_f(p[i]) * coef);
  }
}

template <typename TI>
__device__ __forceinline__ void scale_chunk_to(const TI* p, void* out, int tout, long long at, int n, float coef) {
  if (tout == LSR_DTYPE_F32) scale_chunk(p, static_cast<float*>(out) + at, n, coef);
  else if (tout == LSR_DTYPE_BF16) scale_chunk(p, static_cast<__nv_bfloat16*>(out) + at, n, coef);
  else scale_chunk(p, static_cast<__half*>(out) + at, n, coef);
}

__device__ __forceinline__ float coefficient(float total, float max_norm) {
  const float c = max_norm / (total + 1e-6f);
  return c > 1.f ? 1.f : c;  // a NaN stays
}

// The last chunks first: those are the ones that the pass before left in L2.
template <int N>
__device__ __forceinline__ void scale_chunks(const GradTable<N>& t, float coef, int first, int step) {
  for (int c = t.chunks - 1 - first; c >= 0; c -= step) {
    const int k = find_tensor(t, c);
    if (coef == 1.f && t.in[k] == t.out[k]) continue;  // nothing changes
    const long long at = (long long)(c - t.first[k]) * GR_CHUNK;
    const int n = (int)min((long long)GR_CHUNK, t.numel[k] - at);
    if (t.tin[k] == LSR_DTYPE_F32) scale_chunk_to(static_cast<const float*>(t.in[k]) + at, t.out[k], t.tout[k], at, n, coef);
    else if (t.tin[k] == LSR_DTYPE_BF16)
      scale_chunk_to(static_cast<const __nv_bfloat16*>(t.in[k]) + at, t.out[k], t.tout[k], at, n, coef);
    else scale_chunk_to(static_cast<const __half*>(t.in[k]) + at, t.out[k], t.tout[k], at, n, coef);
  }
}

// A short list in one launch: the blocks of one cluster take the chunks, read one another's sums from shared
// memory, add them in rank order, and (CLIP) scale what they have just read.
template <int KIND, bool CLIP, int N>
__global__ void __cluster_dims__(GR_CLUSTER) __launch_bounds__(GR_THREADS)
    grad_short_kernel(const __grid_constant__ GradTable<N> t, float max_norm, float* __restrict__ norm) {
  __shared__ Acc<KIND> sum;
  const int rank = (int)cluster_ctarank();
  const Acc<KIND> own = block_sum(norm_chunks<KIND>(t, rank, GR_CLUSTER));
  if (threadIdx.x == 0) sum = own;
  cluster_sync_all();
  Acc<KIND> all;
#pragma unroll
  for (int r = 0; r < GR_CLUSTER; ++r) {
    Acc<KIND> other;
    asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(*reinterpret_cast<unsigned long long*>(&other.s))
                 : "r"(mapa_shared(smem_u32(&sum), r)) : "memory");
    all.join(other);
  }
  cluster_sync_all();  // nobody leaves while its sum may be read
  const float total = all.norm();
  if (rank == 0 && threadIdx.x == 0) *norm = total;
  if (CLIP) scale_chunks(t, coefficient(total, max_norm), rank, GR_CLUSTER);
}

// GIVEN: *norm is read (a norm of more tensors than these); else it is the partials' and is written.
template <int KIND, bool GIVEN, int N>
__global__ void __launch_bounds__(GR_THREADS) grad_scale_kernel(const __grid_constant__ GradTable<N> t,
                                                                const Acc<KIND>* __restrict__ partial, int npartial,
                                                                float max_norm, float* norm, int write_norm) {
  float total;
  if (GIVEN) total = *norm;
  else total = total_norm<KIND>(partial, npartial);
  if (!GIVEN && write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  scale_chunks(t, coefficient(total, max_norm), (int)blockIdx.x, (int)gridDim.x);
}

bool dtype_ok(int d) { return d == LSR_DTYPE_F32 || d == LSR_DTYPE_BF16 || d == LSR_DTYPE_F16; }
int dtype_size(int d) { return d == LSR_DTYPE_F32 ? 4 : 2; }
bool kind_ok(int k) { return k == NORM_MAX || k == NORM_ONE || k == NORM_TWO; }

int check_list(const void* const* ptrs, const long long* numel, const int* dtypes, int n) {
  if (n < 0 || (n > 0 && (!ptrs || !numel || !dtypes))) return LSR_ERR_ARG;
  for (int i = 0; i < n; ++i) {
    if (numel[i] < 0 || !dtype_ok(dtypes[i]) || (numel[i] > 0 && !ptrs[i])) return LSR_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(ptrs[i]) % dtype_size(dtypes[i])) return LSR_ERR_SHAPE;
    if (numel[i] > (1ll << 40)) return LSR_ERR_SHAPE;
  }
  return LSR_OK;
}

struct Span {
  uintptr_t lo, hi;
};
int span_order(const void* a, const void* b) {
  const Span *x = static_cast<const Span*>(a), *y = static_cast<const Span*>(b);
  return x->lo < y->lo ? -1 : x->lo > y->lo;
}
// By address; views of one buffer, the common list, come so.
void sort_spans(Span* s, int n) {
  for (int i = 1; i < n; ++i)
    if (s[i].lo < s[i - 1].lo) {
      qsort(s, n, sizeof(Span), span_order);
      return;
    }
}

// LSR_OK unless a written range overlaps another tensor's written or read range, or its own read
// range other than exactly (in place): the blocks run in no order. The norm is one more read value (given) or
// written one.
int check_overlap(const void* const* in, void* const* out, const long long* numel, const int* tin, const int* tout,
                  int n, const float* norm, bool given) {
  Span* w = static_cast<Span*>(malloc(sizeof(Span) * 2 * ((size_t)n + 1)));
  if (!w) return LSR_ERR_WORKSPACE;
  Span* r = w + n + 1;
  int nw = 0, nr = 0;
  const Span at_norm{reinterpret_cast<uintptr_t>(norm), reinterpret_cast<uintptr_t>(norm + 1)};
  if (given) r[nr++] = at_norm;
  else w[nw++] = at_norm;
  for (int i = 0; i < n; ++i) {
    if (!numel[i]) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(in[i]), b = reinterpret_cast<uintptr_t>(out[i]);
    w[nw++] = Span{b, b + (uintptr_t)numel[i] * dtype_size(tout[i])};
    if (a != b || tin[i] != tout[i]) r[nr++] = Span{a, a + (uintptr_t)numel[i] * dtype_size(tin[i])};
  }
  sort_spans(w, nw);
  sort_spans(r, nr);
  int rc = LSR_OK;
  for (int i = 1; i < nw && rc == LSR_OK; ++i)
    if (w[i].lo < w[i - 1].hi) rc = LSR_ERR_ARG;
  // reads may overlap one another, so a written range is compared with the furthest end of those that begin before its own
  uintptr_t read_end = 0;
  for (int i = 0, k = 0; i < nw && rc == LSR_OK; ++i) {
    for (; k < nr && r[k].lo < w[i].hi; ++k) read_end = std::max(read_end, r[k].hi);
    if (read_end > w[i].lo) rc = LSR_ERR_ARG;
  }
  free(w);
  return rc;
}

// The next tensors of the list, from *i on, as one launch's table.
template <int N>
void fill_table(GradTable<N>& t, const void* const* in, void* const* out, const long long* numel, const int* tin,
                const int* tout, int n, int* i) {
  t.n = 0;
  t.chunks = 0;
  for (; *i < n; ++*i) {
    if (!numel[*i]) continue;
    if (t.n == N) break;
    const long long c = (numel[*i] + GR_CHUNK - 1) / GR_CHUNK;
    if (t.n && t.chunks + c > (1ll << 30)) break;
    t.in[t.n] = in[*i];
    t.out[t.n] = out ? out[*i] : nullptr;
    t.numel[t.n] = numel[*i];
    t.first[t.n] = t.chunks;
    t.tin[t.n] = (unsigned char)tin[*i];
    t.tout[t.n] = (unsigned char)(tout ? tout[*i] : tin[*i]);
    t.chunks += (int)c;
    ++t.n;
  }
}

size_t ws_bytes(int n) { return (size_t)(n / GR_TABLE + 2) * GR_GRID * sizeof(double); }

// Partials of every table; *count receives their number.
template <int KIND, int N>
int launch_partials(GradTable<N>& t, const void* const* in, const long long* numel, const int* tin, int n,
                    Acc<KIND>* partial, int room, int* count, cudaStream_t st) {
  *count = 0;
  for (int i = 0; i < n;) {
    fill_table(t, in, nullptr, numel, tin, nullptr, n, &i);
    if (!t.n) break;
    const int grid = std::min(t.chunks, GR_GRID);
    if (*count + grid > room) return LSR_ERR_WORKSPACE;
    ProfScope prof(PK_EW_OTHER, st);
    grad_norm_kernel<KIND, N><<<grid, GR_THREADS, 0, st>>>(t, partial + *count);
    if (cudaGetLastError() != cudaSuccess) return LSR_ERR_LAUNCH;
    *count += grid;
  }
  return LSR_OK;
}

template <int KIND, int N>
int norm_table(const void* const* in, const long long* numel, const int* tin, int n, float* norm, void* ws, size_t bytes,
              cudaStream_t st) {
  GradTable<N> t;
  int taken = 0;
  if constexpr (N == GR_SMALL) fill_table(t, in, nullptr, numel, tin, nullptr, n, &taken);
  if constexpr (N == GR_SMALL)
    if (taken == n && t.chunks <= GR_SHORT) {
      ProfScope prof(PK_EW_OTHER, st);
      grad_short_kernel<KIND, false, N><<<GR_CLUSTER, GR_THREADS, 0, st>>>(t, 0.f, norm);
      return cudaGetLastError() == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
    }
  auto* partial = static_cast<Acc<KIND>*>(ws);
  int count = 0;
  const int rc = launch_partials<KIND, N>(t, in, numel, tin, n, partial, (int)(bytes / sizeof(double)), &count, st);
  if (rc != LSR_OK) return rc;
  ProfScope prof(PK_EW_OTHER, st);
  grad_norm_finish_kernel<KIND><<<1, GR_THREADS, 0, st>>>(partial, count, norm);
  return cudaGetLastError() == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
}

template <int KIND, bool GIVEN, int N>
int clip_table(const void* const* in, void* const* out, const long long* numel, const int* tin, const int* tout, int n,
              float max_norm, float* norm, void* ws, size_t bytes, cudaStream_t st) {
  GradTable<N> t;
  auto* partial = static_cast<Acc<KIND>*>(ws);
  int count = 0;
  if (!GIVEN) {
    if constexpr (N == GR_SMALL) {
      int taken = 0;
      fill_table(t, in, out, numel, tin, tout, n, &taken);
      if (taken == n && t.chunks <= GR_SHORT) {
        ProfScope prof(PK_EW_OTHER, st);
        grad_short_kernel<KIND, true, N><<<GR_CLUSTER, GR_THREADS, 0, st>>>(t, max_norm, norm);
        return cudaGetLastError() == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
      }
    }
    const int rc = launch_partials<KIND, N>(t, in, numel, tin, n, partial, (int)(bytes / sizeof(double)), &count, st);
    if (rc != LSR_OK) return rc;
  }
  int first = 1;
  for (int i = 0; i < n || first;) {
    fill_table(t, in, out, numel, tin, tout, n, &i);
    if (!t.n && !first) break;
    ProfScope prof(PK_EW_OTHER, st);
    const int grid = std::max(1, std::min(t.chunks, GR_GRID));
    grad_scale_kernel<KIND, GIVEN, N><<<grid, GR_THREADS, 0, st>>>(t, partial, count, max_norm, norm, first);
    if (cudaGetLastError() != cudaSuccess) return LSR_ERR_LAUNCH;
    first = 0;
  }
  return LSR_OK;
}

// Whether the tensors that have entries fit a small table (with more, no list is a short one).
bool few(const long long* numel, int n) {
  int k = 0;
  for (int i = 0; i < n && k <= GR_SMALL; ++i) k += numel[i] > 0;
  return k <= GR_SMALL;
}

template <int KIND>
int norm_impl(const void* const* in, const long long* numel, const int* tin, int n, float* norm, void* ws, size_t bytes,
              cudaStream_t st) {
  return few(numel, n) ? norm_table<KIND, GR_SMALL>(in, numel, tin, n, norm, ws, bytes, st)
                       : norm_table<KIND, GR_TABLE>(in, numel, tin, n, norm, ws, bytes, st);
}

template <int KIND, bool GIVEN>
int clip_impl(const void* const* in, void* const* out, const long long* numel, const int* tin, const int* tout, int n,
              float max_norm, float* norm, void* ws, size_t bytes, cudaStream_t st) {
  return few(numel, n)
             ? clip_table<KIND, GIVEN, GR_SMALL>(in, out, numel, tin, tout, n, max_norm, norm, ws, bytes, st)
             : clip_table<KIND, GIVEN, GR_TABLE>(in, out, numel, tin, tout, n, max_norm, norm, ws, bytes, st);
}

}  // namespace
}  // namespace lsr

extern "C" {

size_t lsr_grad_workspace_bytes(int count) { return count < 0 ? 0 : lsr::ws_bytes(count); }

int lsr_grad_norm(const void* const* grads, const long long* numel, const int* dtypes, int count, int norm_kind,
                  float* norm, void* ws, size_t ws_bytes, lsr_stream_t stream) {
  using namespace lsr;
  if (!norm || !kind_ok(norm_kind)) return LSR_ERR_ARG;
  int rc = check_list(grads, numel, dtypes, count);
  if (rc != LSR_OK) return rc;
  if (!ws || ws_bytes < lsr_grad_workspace_bytes(count)) return LSR_ERR_WORKSPACE;
  if ((rc = check_device()) != LSR_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (norm_kind) {
    case NORM_MAX: return norm_impl<NORM_MAX>(grads, numel, dtypes, count, norm, ws, ws_bytes, st);
    case NORM_ONE: return norm_impl<NORM_ONE>(grads, numel, dtypes, count, norm, ws, ws_bytes, st);
    default: return norm_impl<NORM_TWO>(grads, numel, dtypes, count, norm, ws, ws_bytes, st);
  }
}

int lsr_grad_clip(const void* const* grads, void* const* outs, const long long* numel, const int* dtypes,
                  const int* out_dtypes, int count, int norm_kind, float max_norm, int norm_given, float* norm, void* ws,
                  size_t ws_bytes, lsr_stream_t stream) {
  using namespace lsr;
  if (!norm || !kind_ok(norm_kind) || !(max_norm >= 0.f)) return LSR_ERR_ARG;
  int rc = check_list(grads, numel, dtypes, count);
  if (rc != LSR_OK) return rc;
  if ((rc = check_list(reinterpret_cast<const void* const*>(outs), numel, out_dtypes, count)) != LSR_OK) return rc;
  if (count && (rc = check_overlap(grads, outs, numel, dtypes, out_dtypes, count, norm, norm_given != 0)) != LSR_OK) return rc;
  if (!norm_given && (!ws || ws_bytes < lsr_grad_workspace_bytes(count))) return LSR_ERR_WORKSPACE;
  if ((rc = check_device()) != LSR_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (norm_given)
    return clip_impl<NORM_TWO, true>(grads, outs, numel, dtypes, out_dtypes, count, max_norm, norm, ws, ws_bytes, st);
  switch (norm_kind) {
    case NORM_MAX:
      return clip_impl<NORM_MAX, false>(grads, outs, numel, dtypes, out_dtypes, count, max_norm, norm, ws, ws_bytes, st);
    case NORM_ONE:
      return clip_impl<NORM_ONE, false>(grads, outs, numel, dtypes, out_dtypes, count, max_norm, norm, ws, ws_bytes, st);
    default:
      return clip_impl<NORM_TWO, false>(grads, outs, numel, dtypes, out_dtypes, count, max_norm, norm, ws, ws_bytes, st);
  }
}

}  // extern "C"
