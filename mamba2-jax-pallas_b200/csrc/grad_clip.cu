// Global gradient norm over many tensors, and the clipped gradients.
//
//   norm = sqrt(sum_i sum_j g_ij^2);  c = min(1, max_norm / (norm + eps));  out_ij = c * g_ij
//
// Bound by HBM: the norm reads everything once, and only then is c known, so the scaled copy
// reads everything again (from L2 as far as that reaches) and writes it once.
//
// The tensors' addresses travel in the kernel's parameters (up to 32 KB), so a call copies
// nothing to the device and can be captured in a graph.  Each tensor is cut into chunks of
// CHUNK values; a CTA takes a run of consecutive chunks, whatever tensors they belong to, so
// a thousand small tensors cost as many CTAs as one large one.  Every CTA leaves one partial
// sum and the second kernel adds the partial sums in a fixed order in each CTA: no atomics,
// the same norm in every run, and two launches.
//
// Measured, 1.09e9 bf16 values into f32: 1.61 ms (5.4 TB/s of the 8.7 GB that the two kernels move);
// 218 tensors, 2.1 MB in all: norm 5 us, scaled copy 9 us.
//
// Sums are f64: squares of f32 gradients leave the range of f32 on both sides
// (1e-23 and 1e19), and a sum over 1e9 values in f32 loses its last digits.  Only groups of four
// squares are added in f32, where they stay in its range (squares()): at most 3 u of a sum, u = 2^-24, so
// 1.5 u of the norm before its own rounding.
#include <algorithm>

#include "common.cuh"
#include "ssd_kernels.h"

namespace ssd {
namespace {

constexpr int GC_THREADS = 256;
constexpr int CHUNK = 8192;             // values; 32 per thread
constexpr int MAX_TENSORS = 1000;       // 1000 x 28 bytes: inside the 32764 bytes of parameters
constexpr int CTAS_PER_SM = 4;          // resident (64 registers); a CTA's run of chunks is its share of all
constexpr int MAX_PARTIALS = 148 * CTAS_PER_SM;

template <int N>
struct Table {
  int count;                            // tensors
  int chunks;                           // chunks of all of them
  const void* g[N];
  void* out[N];
  int64_t numel[N];
  int first[N];                         // first chunk of each tensor
};

// Tensor of a chunk: the last i with first[i] <= chunk (tensors are never empty here).
template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// V values from i on (zeros past the end); one access of V * sizeof(T) bytes where `al`.
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T* p, int64_t i, int64_t n, bool al, float (&v)[V]) {
  if (al && i + V <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p + i);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
      uint32_t u[V / 2];
      if constexpr (V == 8) *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(p + i);
      else *reinterpret_cast<uint2*>(u) = *reinterpret_cast<const uint2*>(p + i);
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        v[2 * k] = __uint_as_float(u[k] << 16);
        v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = i + k < n ? ld(p + i + k) : 0.f;
}

// `align`: the output's alignment in bytes, 16, 8, 4 or 2 (pieces of one flat buffer start anywhere).
template <int V, typename T>
__device__ __forceinline__ void store_vec(T* p, int64_t i, int64_t n, int align, const float (&v)[V]) {
  if (i + V > n || align < 4) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (i + k < n) st(p + i + k, v[k]);
    return;
  }
  constexpr int W = V * sizeof(T) / 4;         // 32-bit words
  uint32_t u[W];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < W; ++k) u[k] = __float_as_uint(v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
      u[k] = *reinterpret_cast<uint32_t*>(&h);
    }
  }
  if (W == 4 && align >= 16) {
    *reinterpret_cast<uint4*>(p + i) = make_uint4(u[0], u[1], u[W - 2], u[W - 1]);
  } else if (align >= 8) {
#pragma unroll
    for (int k = 0; k < W; k += 2) reinterpret_cast<uint2*>(p + i)[k / 2] = make_uint2(u[k], u[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k) reinterpret_cast<uint32_t*>(p + i)[k] = u[k];
  }
}

// V values to an aligned address, not to be kept in L2 (the gradients are).
template <int V, typename T>
__device__ __forceinline__ void store_stream(T* p, const float (&v)[V]) {
  if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  } else {
    uint32_t u[V / 2];
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
      u[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (V == 8) __stcs(reinterpret_cast<uint4*>(p), make_uint4(u[0], u[1], u[2], u[3]));
    else __stcs(reinterpret_cast<uint2*>(p), make_uint2(u[0], u[1]));
  }
}

__device__ __forceinline__ int align_of(const void* p) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  return a % 16 == 0 ? 16 : a % 8 == 0 ? 8 : a % 4 == 0 ? 4 : 2;
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0;
  for (int i = 0; i < GC_THREADS / 32; ++i) s += sh[i];
  return s;
}

// Sum of V squares.  Four are added in f32 before they go to f64: a conversion per value would
// bound the kernel (16 per clock and SM).  Sums that may have left f32's range are taken again in f64.
template <int V>
__device__ __forceinline__ double squares(const float (&v)[V]) {
  double s = 0;
#pragma unroll
  for (int k = 0; k < V; k += 4) {
    const float q = fmaf(v[k], v[k], v[k + 1] * v[k + 1]) + fmaf(v[k + 2], v[k + 2], v[k + 3] * v[k + 3]);
    if (q > 1e-25f && q < 1e38f) {
      s += (double)q;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fma((double)v[k + j], (double)v[k + j], s);
    }
  }
  return s;
}

// A whole chunk of an aligned tensor: U accesses per thread with no condition between them, so
// that all of them are in flight.  (A load under a condition is merged with its other value at
// once, and waits there.)
template <int V, int U, typename T>
__device__ __forceinline__ void load_chunk(const T* p, float (&v)[U][V]) {
  constexpr int W = V * sizeof(T) / 4;
  uint32_t u[U][W];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const T* q = p + (j * GC_THREADS + threadIdx.x) * V;
    if constexpr (W == 4) *reinterpret_cast<uint4*>(u[j]) = *reinterpret_cast<const uint4*>(q);
    else *reinterpret_cast<uint2*>(u[j]) = *reinterpret_cast<const uint2*>(q);
  }
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int k = 0; k < W; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[j][k] = __uint_as_float(u[j][k]);
      } else {
        v[j][2 * k] = __uint_as_float(u[j][k] << 16);
        v[j][2 * k + 1] = __uint_as_float(u[j][k] & 0xffff0000u);
      }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(GC_THREADS, CTAS_PER_SM) norm_kernel(const __grid_constant__ Table<N> t, double* partial) {
  constexpr int V = 16 / sizeof(T), U = CHUNK / GC_THREADS / V;
  __shared__ double sh[GC_THREADS / 32];
  const int c0 = (int)((int64_t)t.chunks * blockIdx.x / gridDim.x), c1 = (int)((int64_t)t.chunks * (blockIdx.x + 1) / gridDim.x);
  double sum = 0;
  int i = c0 < c1 ? tensor_of(t, c0) : 0;
  for (int c = c0; c < c1; ++c) {
    if (i + 1 < t.count && t.first[i + 1] <= c) ++i;
    const T* g = static_cast<const T*>(t.g[i]);
    const int64_t n = t.numel[i], base = (int64_t)(c - t.first[i]) * CHUNK;
    const bool al = reinterpret_cast<uintptr_t>(g) % 16 == 0;
    if (al && base + CHUNK <= n) {
      float v[U][V];
      load_chunk<V, U>(g + base, v);
#pragma unroll
      for (int j = 0; j < U; ++j) sum += squares<V>(v[j]);
    } else {
      for (int64_t e = base + threadIdx.x * V; e < n; e += GC_THREADS * V) {
        if (e >= base + CHUNK) break;
        float v[V];
        load_vec<V>(g, e, n, al, v);
        sum += squares<V>(v);
      }
    }
  }
  sum = block_sum(sum, sh);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The norm and the factor, from the partial sums; the same order in every CTA.
__device__ __forceinline__ float2 norm_and_factor(const double* partial, int npartial, float max_norm, float eps,
                                                  double* sh) {
  double s = 0;
  for (int i = threadIdx.x; i < npartial; i += GC_THREADS) s += partial[i];
  const double norm = sqrt(block_sum(s, sh));
  const double f = (double)max_norm / (norm + (double)eps);
  return make_float2((float)norm, f >= 1.0 ? 1.f : (float)f);   // NaN stays NaN
}

template <typename T, typename TO, int N>
__global__ void __launch_bounds__(GC_THREADS, CTAS_PER_SM) scale_kernel(const __grid_constant__ Table<N> t, const double* partial,
                                                           int npartial, float max_norm, float eps, float* norm) {
  // 16 bytes of the wider type per access: neighbouring lanes write neighbouring 16 bytes
  constexpr int V = 16 / (sizeof(T) > sizeof(TO) ? sizeof(T) : sizeof(TO)), U = CHUNK / GC_THREADS / V;
  __shared__ double sh[GC_THREADS / 32];
  const float2 nf = norm_and_factor(partial, npartial, max_norm, eps, sh);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = nf.x;
  const float f = nf.y;
  const int c0 = (int)((int64_t)t.chunks * blockIdx.x / gridDim.x), c1 = (int)((int64_t)t.chunks * (blockIdx.x + 1) / gridDim.x);
  // backwards: the norm read the run's end last, and L2 may still hold it
  int i = c0 < c1 ? tensor_of(t, c1 - 1) : 0;
  for (int c = c1 - 1; c >= c0; --c) {
    if (t.first[i] > c) --i;
    const T* g = static_cast<const T*>(t.g[i]);
    TO* o = static_cast<TO*>(t.out[i]);
    if (f == 1.f && static_cast<const void*>(o) == static_cast<const void*>(g)) continue;   // times one, in place
    const int64_t n = t.numel[i], base = (int64_t)(c - t.first[i]) * CHUNK;
    const bool al = reinterpret_cast<uintptr_t>(g) % 16 == 0;
    const int oal = align_of(o);
    if (al && oal == 16 && base + CHUNK <= n) {
      float v[U][V];
      load_chunk<V, U>(g + base, v);
#pragma unroll
      for (int j = 0; j < U; ++j) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[j][k] *= f;
        store_stream<V>(o + base + (j * GC_THREADS + threadIdx.x) * V, v[j]);
      }
    } else {
      for (int64_t e = base + threadIdx.x * V; e < n; e += GC_THREADS * V) {
        if (e >= base + CHUNK) break;
        float v[V];
        load_vec<V>(g, e, n, al, v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] *= f;
        store_vec<V>(o, e, n, oal, v);
      }
    }
  }
}

__global__ void __launch_bounds__(GC_THREADS) norm_only_kernel(const double* partial, int npartial, float* norm) {
  __shared__ double sh[GC_THREADS / 32];
  const float2 nf = norm_and_factor(partial, npartial, 0.f, 1.f, sh);
  if (threadIdx.x == 0) *norm = nf.x;
}

int grid_of(int chunks) { return std::min(chunks, MAX_PARTIALS); }

template <int N>
void fill(Table<N>* t, const ssd_grad_tensor_t* list, const int* index, int count) {
  t->count = count;
  int64_t chunk = 0;
  for (int i = 0; i < count; ++i) {
    const ssd_grad_tensor_t& e = list[index[i]];
    t->g[i] = e.grad;
    t->out[i] = e.out;
    t->numel[i] = e.numel;
    t->first[i] = (int)chunk;
    chunk += (e.numel + CHUNK - 1) / CHUNK;
  }
  t->chunks = (int)chunk;
}

// One launch's tensors: of one type pair, at most MAX_TENSORS, at most 2^30 chunks.
struct Batch {
  int gd, od, count, chunks;
  int start;                     // into the index list
};

template <int N>
cudaError_t norm_batch(const ssd_grad_tensor_t* list, const int* index, const Batch& b, double* partial,
                       cudaStream_t stream) {
  Table<N> t;
  fill(&t, list, index, b.count);
  const int grid = grid_of(t.chunks);
  if (b.gd == SSD_DTYPE_BF16) norm_kernel<bf16, N><<<grid, GC_THREADS, 0, stream>>>(t, partial);
  else norm_kernel<float, N><<<grid, GC_THREADS, 0, stream>>>(t, partial);
  return cudaGetLastError();
}

template <int N>
cudaError_t scale_batch(const ssd_grad_tensor_t* list, const int* index, const Batch& b, const double* partial,
                        int npartial, float max_norm, float eps, float* norm, cudaStream_t stream) {
  Table<N> t;
  fill(&t, list, index, b.count);
  const int grid = grid_of(t.chunks);
  const bool gb = b.gd == SSD_DTYPE_BF16, ob = b.od == SSD_DTYPE_BF16;
  if (gb && ob) scale_kernel<bf16, bf16, N><<<grid, GC_THREADS, 0, stream>>>(t, partial, npartial, max_norm, eps, norm);
  else if (gb) scale_kernel<bf16, float, N><<<grid, GC_THREADS, 0, stream>>>(t, partial, npartial, max_norm, eps, norm);
  else if (ob) scale_kernel<float, bf16, N><<<grid, GC_THREADS, 0, stream>>>(t, partial, npartial, max_norm, eps, norm);
  else scale_kernel<float, float, N><<<grid, GC_THREADS, 0, stream>>>(t, partial, npartial, max_norm, eps, norm);
  return cudaGetLastError();
}

// Cut the list into launches.  `each(batch, index)` is called for every one.
template <typename F>
cudaError_t for_batches(const ssd_grad_tensor_t* list, int64_t count, bool by_out, F&& each) {
  int index[MAX_TENSORS];
  for (int gd = 0; gd < 2; ++gd) {
    for (int od = 0; od < (by_out ? 2 : 1); ++od) {
      Batch b{gd, od, 0, 0, 0};
      for (int64_t i = 0; i <= count; ++i) {
        const bool mine = i < count && list[i].numel > 0 && list[i].grad_dtype == gd &&
                          (!by_out || list[i].out_dtype == od);
        const int64_t chunks = mine ? (list[i].numel + CHUNK - 1) / CHUNK : 0;
        if (b.count && (i == count || b.count == MAX_TENSORS || b.chunks + chunks > (1 << 30))) {
          const cudaError_t e = each(b, index);
          if (e != cudaSuccess) return e;
          b.count = b.chunks = 0;
        }
        if (mine) {
          index[b.count++] = (int)i;
          b.chunks += (int)chunks;
        }
      }
    }
  }
  return cudaSuccess;
}

}  // namespace

// Partial sums of the norm's launches.
int64_t grad_clip_partials(const ssd_grad_tensor_t* list, int64_t count) {
  int64_t n = 0;
  for_batches(list, count, false, [&](const Batch& b, const int*) {
    n += grid_of(b.chunks);
    return cudaSuccess;
  });
  return n;
}

cudaError_t launch_grad_clip(const ssd_grad_tensor_t* list, int64_t count, float max_norm, float eps, bool scale,
                             float* norm, void* workspace, cudaStream_t stream) {
  double* partial = static_cast<double*>(workspace);
  int npartial = 0;
  cudaError_t e = for_batches(list, count, false, [&](const Batch& b, const int* index) {
    double* p = partial + npartial;
    npartial += grid_of(b.chunks);
    // the table is copied at the launch: a short list takes a short one
    return b.count <= 64    ? norm_batch<64>(list, index, b, p, stream)
           : b.count <= 256 ? norm_batch<256>(list, index, b, p, stream)
                            : norm_batch<MAX_TENSORS>(list, index, b, p, stream);
  });
  if (e != cudaSuccess) return e;
  if (!scale || npartial == 0) {
    norm_only_kernel<<<1, GC_THREADS, 0, stream>>>(partial, npartial, norm);
    return cudaGetLastError();
  }
  float* out = norm;   // the first launch writes the norm
  return for_batches(list, count, true, [&](const Batch& b, const int* index) {
    float* n = out;
    out = nullptr;
    return b.count <= 64    ? scale_batch<64>(list, index, b, partial, npartial, max_norm, eps, n, stream)
           : b.count <= 256 ? scale_batch<256>(list, index, b, partial, npartial, max_norm, eps, n, stream)
                            : scale_batch<MAX_TENSORS>(list, index, b, partial, npartial, max_norm, eps, n, stream);
  });
}

}  // namespace ssd
