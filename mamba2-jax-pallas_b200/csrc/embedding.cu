// Token embedding and its gradient: the first step of a language model around the mixer
// layers and the scatter that trains its table.
//
//   out[t,:] = scale * W[id_t,:]                      (a zero row where id_t is dropped)
//   dW[v,:]  = scale * sum_{t: id_t = v} g[t,:]       (in the order of t)
// An id is dropped when it lies outside [0, V) or equals padding_idx.
//
// Both move bytes and compute next to nothing, so both are bound by HBM: the lookup by the
// named rows in and T rows out, the gradient by T rows in and the whole table out (a dense
// gradient has V rows, most of them zero).
//
// The gradient is a sum by sorted ids, so that it is the same in every run: no atomics on
// floats.  Three launches:
//   1. one cluster sorts (id, position) pairs by a stable radix sort whose histograms live in
//      distributed shared memory, while every other CTA of the grid writes the zero rows of
//      the ids that do not occur (it marks the ids of its own rows in a shared bitmap);
//   2. the sorted order is cut into pieces of equal length, whatever the ids, so that one
//      frequent id cannot hold up a CTA; a warp sums a piece's rows over 256 columns in f32
//      and writes each id's row where the id begins and ends inside the piece; an id that
//      crosses into another piece leaves its part in the workspace;
//   3. the piece in which such an id begins adds its parts up, again in order.
#include <algorithm>

#include <cooperative_groups.h>

#include "common.cuh"
#include "ssd_kernels.h"

namespace cg = cooperative_groups;

namespace ssd {
namespace {

constexpr int VEC = 8;            // values per lane and load: 16 bytes of bf16, 32 of f32

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[VEC]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(u[k] << 16);
      v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[VEC]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      u[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// The row an id names, or -1.
__device__ __forceinline__ int64_t row_of(const void* ids, int is64, int64_t t, int64_t vocab, int64_t pad) {
  const int64_t v = is64 ? __ldg(static_cast<const long long*>(ids) + t) : (int64_t)__ldg(static_cast<const int*>(ids) + t);
  return (v < 0 || v >= vocab || v == pad) ? -1 : v;
}

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
struct LookupArgs {
  int64_t n, vocab, dim, ws, os, pad;
  int is64;
  float scale;
  const void* ids;
  const void* w;
  void* out;
};

constexpr int LK_THREADS = 256;
constexpr int LK_UNROLL = 4;      // 16-byte loads in flight per lane

// One warp per (token, run of 32 * LK_UNROLL vectors of 8).
template <typename TW, typename TO>
__global__ void __launch_bounds__(LK_THREADS) lookup_vec_kernel(const LookupArgs a, int runs) {
  const int64_t unit = (int64_t)blockIdx.x * (LK_THREADS / 32) + threadIdx.x / 32;
  const int64_t t = unit / runs;
  if (t >= a.n) return;
  const int lane = threadIdx.x & 31;
  const int64_t c0 = (unit - t * runs) * (32 * LK_UNROLL * VEC);
  const int64_t row = row_of(a.ids, a.is64, t, a.vocab, a.pad);
  TO* o = static_cast<TO*>(a.out) + t * a.os;
  const TW* w = static_cast<const TW*>(a.w) + (row < 0 ? 0 : row) * a.ws;
  float v[LK_UNROLL][VEC];
#pragma unroll
  for (int i = 0; i < LK_UNROLL; ++i) {
    const int64_t c = c0 + (int64_t)(i * 32 + lane) * VEC;
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[i][k] = 0.f;
    if (row >= 0 && c < a.dim) load8(w + c, v[i]);
  }
#pragma unroll
  for (int i = 0; i < LK_UNROLL; ++i) {
    const int64_t c = c0 + (int64_t)(i * 32 + lane) * VEC;
    if (c >= a.dim) continue;
    if (row >= 0) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[i][k] *= a.scale;
    }
    store8(o + c, v[i]);
  }
}

// Any width and alignment: one warp per token, one value per lane and step.
template <typename TW, typename TO>
__global__ void __launch_bounds__(LK_THREADS) lookup_any_kernel(const LookupArgs a) {
  const int64_t t = (int64_t)blockIdx.x * (LK_THREADS / 32) + threadIdx.x / 32;
  if (t >= a.n) return;
  const int64_t row = row_of(a.ids, a.is64, t, a.vocab, a.pad);
  TO* o = static_cast<TO*>(a.out) + t * a.os;
  const TW* w = static_cast<const TW*>(a.w) + (row < 0 ? 0 : row) * a.ws;
  for (int64_t c = threadIdx.x & 31; c < a.dim; c += 32) st(o + c, row < 0 ? 0.f : ldg(w + c) * a.scale);
}

bool rows16(const void* p, int64_t stride, int64_t dim, int dtype) {
  const int64_t es = dtype == SSD_DTYPE_BF16 ? 2 : 4;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * es) % 16 == 0 && dim % VEC == 0;
}

template <typename TW, typename TO>
cudaError_t lookup(const LookupArgs& a, bool vec, cudaStream_t stream) {
  constexpr int W = LK_THREADS / 32;
  if (vec) {
    const int64_t runs = (a.dim + 32 * LK_UNROLL * VEC - 1) / (32 * LK_UNROLL * VEC);
    lookup_vec_kernel<TW, TO><<<(unsigned)((a.n * runs + W - 1) / W), LK_THREADS, 0, stream>>>(a, (int)runs);
  } else {
    lookup_any_kernel<TW, TO><<<(unsigned)((a.n + W - 1) / W), LK_THREADS, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// gradient, launch 1: sort and zero rows
// ---------------------------------------------------------------------------
constexpr int SORT_CTAS = 8;      // the sorting cluster
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_BITS = 9;
constexpr int SORT_BINS = 1 << SORT_BITS;
constexpr int ZERO_ROWS = 8192;   // rows whose bits the bitmap holds at a time

struct GradArgs {
  int64_t n, vocab, dim, gs, os, pad, piece, npieces;
  int is64, passes, accumulate, zero_ctas;
  float scale;
  const void* ids;
  const void* g;
  void* out;
  uint32_t* key[2];               // sorted ids (V = dropped, last); result in key[0], pos[0]
  uint32_t* pos[2];
  float* part;                    // (npieces, 2, dim)
};

struct SortShared {
  uint32_t warp_bin[SORT_WARPS][SORT_BINS];   // this CTA's counts, then each warp's next slot
  uint32_t cta_bin[SORT_BINS];                // this CTA's count of each digit, read by the cluster
  uint32_t scan[SORT_WARPS];
};

// One stable pass of the radix sort over the cluster.  CTA c and its warp w own consecutive
// tokens; a warp takes 32 of them at a time and lanes with equal digits find each other by
// match_any, so equal digits keep their order.
template <bool FIRST>
__device__ void sort_pass(const GradArgs& a, SortShared* s, int shift, const uint32_t* ki, const uint32_t* pi,
                          uint32_t* ko, uint32_t* po) {
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank(), tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  for (int i = tid; i < SORT_WARPS * SORT_BINS; i += SORT_THREADS) (&s->warp_bin[0][0])[i] = 0;
  __syncthreads();
  const int64_t per = (a.n + SORT_CTAS * SORT_WARPS - 1) / (SORT_CTAS * SORT_WARPS);
  const int64_t lo = (int64_t)(cta * SORT_WARPS + w) * per, hi = min(lo + per, a.n);
  auto key_at = [&](int64_t t) -> uint32_t {
    if constexpr (FIRST) {
      const int64_t v = row_of(a.ids, a.is64, t, a.vocab, a.pad);
      return v < 0 ? (uint32_t)a.vocab : (uint32_t)v;
    } else {
      return ki[t];
    }
  };
  for (int64_t t0 = lo; t0 < hi; t0 += 32) {
    const int64_t t = t0 + lane;
    const bool in = t < hi;
    const unsigned live = __ballot_sync(0xffffffffu, in);
    if (in) {
      const uint32_t d = (key_at(t) >> shift) & (SORT_BINS - 1);
      const unsigned same = __match_any_sync(live, d);
      if (lane == __ffs(same) - 1) s->warp_bin[w][d] += __popc(same);
    }
    __syncwarp();
  }
  __syncthreads();
  // counts of each digit: exclusive over this CTA's warps, total over the CTA
  if (tid < SORT_BINS) {
    uint32_t sum = 0;
    for (int i = 0; i < SORT_WARPS; ++i) {
      const uint32_t c = s->warp_bin[i][tid];
      s->warp_bin[i][tid] = sum;
      sum += c;
    }
    s->cta_bin[tid] = sum;
  }
  cluster.sync();
  // first slot of digit d for this CTA: all smaller digits, then digit d in the CTAs before
  uint32_t before = 0, total = 0;
  if (tid < SORT_BINS) {
    for (int c = 0; c < SORT_CTAS; ++c) {
      const uint32_t v = cluster.map_shared_rank(s->cta_bin, c)[tid];
      before += c < cta ? v : 0;
      total += v;
    }
  }
  uint32_t incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s->scan[w] = incl;
  __syncthreads();
  if (tid < SORT_BINS) {
    uint32_t base = incl - total + before;
    for (int i = 0; i < w; ++i) base += s->scan[i];
    for (int i = 0; i < SORT_WARPS; ++i) s->warp_bin[i][tid] += base;
  }
  __syncthreads();
  for (int64_t t0 = lo; t0 < hi; t0 += 32) {
    const int64_t t = t0 + lane;
    const bool in = t < hi;
    const unsigned live = __ballot_sync(0xffffffffu, in);
    if (in) {
      const uint32_t k = key_at(t), d = (k >> shift) & (SORT_BINS - 1);
      const unsigned same = __match_any_sync(live, d);
      const uint32_t slot = s->warp_bin[w][d] + __popc(same & ((1u << lane) - 1));
      __syncwarp(live);
      if (lane == __ffs(same) - 1) s->warp_bin[w][d] += __popc(same);
      ko[slot] = k;
      po[slot] = FIRST ? (uint32_t)t : pi[t];
    }
    __syncwarp();
  }
  cluster.sync();   // the cluster's keys are in place; every CTA has read the others' counts
}

// Zero rows of the ids that do not occur.  A CTA owns rows [r0, r1) and marks those that
// occur in a shared bitmap, ZERO_ROWS at a time, reading all ids (L2) once for each.
template <typename TO>
__device__ void zero_rows(const GradArgs& a, uint32_t* bits, int cta) {
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int64_t per = (a.vocab + a.zero_ctas - 1) / a.zero_ctas;
  const int64_t r0 = cta * per, r1 = min(r0 + per, a.vocab);
  const bool vec = (reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.os * sizeof(TO))) % 16 == 0;
  for (int64_t b0 = r0; b0 < r1; b0 += ZERO_ROWS) {
    const int64_t b1 = min(b0 + ZERO_ROWS, r1);
    for (int i = tid; i < ZERO_ROWS / 32; i += SORT_THREADS) bits[i] = 0;
    __syncthreads();
    for (int64_t t = tid; t < a.n; t += SORT_THREADS) {
      const int64_t v = row_of(a.ids, a.is64, t, a.vocab, a.pad);
      if (v >= b0 && v < b1) atomicOr(&bits[(v - b0) >> 5], 1u << ((v - b0) & 31));
    }
    __syncthreads();
    for (int64_t r = b0 + w; r < b1; r += SORT_WARPS) {
      if ((bits[(r - b0) >> 5] >> ((r - b0) & 31)) & 1) continue;
      TO* o = static_cast<TO*>(a.out) + r * a.os;
      int64_t c = 0;
      if (vec) {
        constexpr int PER = 16 / sizeof(TO);
        for (c = lane * PER; c + PER <= a.dim; c += 32 * PER) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
        c = a.dim / PER * PER;
      }
      for (c += lane; c < a.dim; c += 32) st(o + c, 0.f);
    }
    __syncthreads();
  }
}

template <typename TO>
__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_THREADS, 1)
    grad_sort_kernel(const GradArgs a) {
  extern __shared__ uint8_t smem[];
  if (blockIdx.x >= SORT_CTAS) {
    zero_rows<TO>(a, reinterpret_cast<uint32_t*>(smem), (int)blockIdx.x - SORT_CTAS);
    return;
  }
  SortShared* s = reinterpret_cast<SortShared*>(smem);
  // the passes end in key[0] / pos[0]
  int to = (a.passes - 1) & 1;
  sort_pass<true>(a, s, 0, nullptr, nullptr, a.key[to], a.pos[to]);
  for (int p = 1; p < a.passes; ++p) {
    sort_pass<false>(a, s, p * SORT_BITS, a.key[to], a.pos[to], a.key[to ^ 1], a.pos[to ^ 1]);
    to ^= 1;
  }
}

// ---------------------------------------------------------------------------
// gradient, launches 2 and 3: sums
// ---------------------------------------------------------------------------
constexpr int SUM_THREADS = 256;
constexpr int SUM_COLS = 32 * VEC;   // columns of a warp
constexpr int SUM_UNROLL = 8;        // rows in flight

template <typename T, bool V>
__device__ __forceinline__ void load_cols(const T* row, int64_t c, int64_t dim, float (&v)[VEC]) {
  if constexpr (V) {
    if (c < dim) {
      load8(row + c, v);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = 0.f;
    }
  } else {   // columns c + 32 k: neighbouring lanes read neighbouring values
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = c + 32 * k < dim ? ldg(row + c + 32 * k) : 0.f;
  }
}

template <typename T, bool V>
__device__ __forceinline__ void store_cols(T* row, int64_t c, int64_t dim, const float (&v)[VEC]) {
  if constexpr (V) {
    if (c < dim) store8(row + c, v);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (c + 32 * k < dim) st(row + c + 32 * k, v[k]);
  }
}

template <typename TO, bool V>
__device__ __forceinline__ void put_row(const GradArgs& a, uint32_t id, int64_t c, float (&acc)[VEC]) {
  TO* o = static_cast<TO*>(a.out) + (int64_t)id * a.os;
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] *= a.scale;
  if (a.accumulate) {
    float old[VEC];
    if constexpr (V) {
      if (c < a.dim) {
        load8(o + c, old);
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += old[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (c + 32 * k < a.dim) acc[k] += ld(o + c + 32 * k);
    }
  }
  store_cols<TO, V>(o, c, a.dim, acc);
}

// Warp (piece p, columns): rows of the sorted positions [p * piece, + piece).
template <typename TG, typename TO, bool V>
__global__ void __launch_bounds__(SUM_THREADS) grad_sum_kernel(const GradArgs a, int col_warps) {
  const int64_t unit = (int64_t)blockIdx.x * (SUM_THREADS / 32) + threadIdx.x / 32;
  const int64_t p = unit / col_warps;
  if (p >= a.npieces) return;
  const int lane = threadIdx.x & 31;
  const int64_t c = (unit - p * col_warps) * SUM_COLS + (V ? lane * VEC : lane);
  const int64_t lo = p * a.piece, hi = min(lo + a.piece, a.n);
  const uint32_t* key = a.key[0];
  const uint32_t* pos = a.pos[0];
  const TG* g = static_cast<const TG*>(a.g);
  uint32_t cur = key[lo];
  bool open = lo > 0 && key[lo - 1] == cur;   // the id began in an earlier piece
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  for (int64_t i0 = lo; i0 < hi && cur != (uint32_t)a.vocab; i0 += 32) {
    const int m = (int)min((int64_t)32, hi - i0);
    const uint32_t mk = lane < m ? key[i0 + lane] : (uint32_t)a.vocab;
    const uint32_t mp = lane < m ? pos[i0 + lane] : 0;
    for (int j0 = 0; j0 < m; j0 += SUM_UNROLL) {
      float v[SUM_UNROLL][VEC];
#pragma unroll
      for (int j = 0; j < SUM_UNROLL; ++j) {
        const uint32_t kj = __shfl_sync(0xffffffffu, mk, j0 + j);
        const int64_t t = __shfl_sync(0xffffffffu, mp, j0 + j);
        if (kj != (uint32_t)a.vocab) load_cols<TG, V>(g + t * a.gs, c, a.dim, v[j]);
      }
#pragma unroll
      for (int j = 0; j < SUM_UNROLL; ++j) {
        const uint32_t kj = __shfl_sync(0xffffffffu, mk, j0 + j);
        if (j0 + j < m && cur != (uint32_t)a.vocab) {
          if (kj != cur) {
            if (open)
              store_cols<float, V>(a.part + (p * 2) * a.dim, c, a.dim, acc);
            else
              put_row<TO, V>(a, cur, c, acc);
            open = false;
            cur = kj;
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
          }
          if (kj != (uint32_t)a.vocab) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += v[j][k];
          }
        }
      }
    }
  }
  if (cur == (uint32_t)a.vocab) return;
  const bool goes_on = hi < a.n && key[hi] == cur;
  if (open)
    store_cols<float, V>(a.part + (p * 2) * a.dim, c, a.dim, acc);
  else if (goes_on)
    store_cols<float, V>(a.part + (p * 2 + 1) * a.dim, c, a.dim, acc);
  else
    put_row<TO, V>(a, cur, c, acc);
}

// CTA (piece p, 256 columns): where an id begins in piece p and goes on, the sum of its parts.
// The parts of the following pieces are shared out over the CTA's warps in runs, each summed
// in order, and the runs are added in order.
template <typename TO, bool V>
__global__ void __launch_bounds__(SUM_THREADS) grad_join_kernel(const GradArgs a) {
  __shared__ float sums[SUM_THREADS / 32][SUM_COLS];
  const int64_t p = blockIdx.y;
  const uint32_t* key = a.key[0];
  const int64_t lo = p * a.piece, hi = lo + a.piece;
  if (hi >= a.n) return;
  const uint32_t id = key[hi - 1];
  if (id == (uint32_t)a.vocab || key[hi] != id || (lo > 0 && key[lo - 1] == id && key[lo] == id)) return;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // last piece that holds the id: pieces p+1, p+2, ... whose first key is the id
  int64_t last = p + 1;
  while (true) {
    const int64_t q = last + 1 + lane;
    const bool same = q < a.npieces && key[q * a.piece] == id;
    const unsigned b = __ballot_sync(0xffffffffu, same);
    const int more = b == 0xffffffffu ? 32 : __ffs(~b) - 1;
    last += more;
    if (more < 32) break;
  }
  const int64_t count = last - p, per = (count + SUM_THREADS / 32 - 1) / (SUM_THREADS / 32);
  const int64_t q0 = p + 1 + w * per, q1 = min(q0 + per, last + 1);
  const int64_t c = (int64_t)blockIdx.x * SUM_COLS + (V ? lane * VEC : lane);
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  if (w == 0) load_cols<float, V>(a.part + (p * 2 + 1) * a.dim, c, a.dim, acc);
#pragma unroll 4
  for (int64_t q = q0; q < q1; ++q) {
    float v[VEC];
    load_cols<float, V>(a.part + (q * 2) * a.dim, c, a.dim, v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += v[k];
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) sums[w][k * 32 + lane] = acc[k];
  __syncthreads();
  if (w != 0) return;
  for (int i = 1; i < SUM_THREADS / 32; ++i) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += sums[i][k * 32 + lane];
  }
  put_row<TO, V>(a, id, c, acc);
}

template <typename TG, typename TO, bool V>
cudaError_t grad_sums(const GradArgs& a, cudaStream_t stream) {
  const int64_t col_warps = (a.dim + SUM_COLS - 1) / SUM_COLS;
  constexpr int W = SUM_THREADS / 32;
  grad_sum_kernel<TG, TO, V><<<(unsigned)((a.npieces * col_warps + W - 1) / W), SUM_THREADS, 0, stream>>>(a, (int)col_warps);
  if (a.npieces > 1)
    grad_join_kernel<TO, V><<<dim3((unsigned)col_warps, (unsigned)a.npieces), SUM_THREADS, 0, stream>>>(a);
  return cudaGetLastError();
}

int64_t piece_len(int64_t n) {
  // at least 32 rows, so that a warp's loads are worth its start, and at most 2048 pieces,
  // which bounds the parts' workspace and the join's grid
  int64_t len = 32;
  while ((n + len - 1) / len > 2048) len *= 2;
  return len;
}

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

}  // namespace

cudaError_t launch_embedding(const ssd_embedding_params_t* p, cudaStream_t stream) {
  LookupArgs a;
  a.n = p->num_tokens; a.vocab = p->vocab; a.dim = p->dim;
  a.ws = p->weight_stride_row; a.os = p->dim; a.pad = p->padding_idx;
  a.is64 = p->tokens_int64; a.scale = p->scale;
  a.ids = p->tokens; a.w = p->weight; a.out = p->out;
  const bool vec = rows16(p->weight, a.ws, a.dim, p->weight_dtype) && rows16(p->out, a.os, a.dim, p->out_dtype);
  const bool wb = p->weight_dtype == SSD_DTYPE_BF16, ob = p->out_dtype == SSD_DTYPE_BF16;
  if (wb) return ob ? lookup<bf16, bf16>(a, vec, stream) : lookup<bf16, float>(a, vec, stream);
  return ob ? lookup<float, bf16>(a, vec, stream) : lookup<float, float>(a, vec, stream);
}

size_t embedding_grad_workspace(int64_t n, int64_t dim) {
  const int64_t pieces = (n + piece_len(n) - 1) / piece_len(n);
  return 4 * up256((size_t)n * 4) + (size_t)pieces * 2 * dim * 4;
}

cudaError_t launch_embedding_grad(const ssd_embedding_grad_params_t* p, void* workspace, cudaStream_t stream) {
  GradArgs a;
  a.n = p->num_tokens; a.vocab = p->vocab; a.dim = p->dim;
  a.gs = p->grad_stride_row; a.os = p->out_stride_row; a.pad = p->padding_idx;
  a.is64 = p->tokens_int64; a.accumulate = p->accumulate; a.scale = p->scale;
  a.ids = p->tokens; a.g = p->grad; a.out = p->out;
  a.piece = piece_len(a.n);
  a.npieces = (a.n + a.piece - 1) / a.piece;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const size_t list = up256((size_t)a.n * 4);
  for (int i = 0; i < 2; ++i) {
    a.key[i] = reinterpret_cast<uint32_t*>(ws + (2 * i) * list);
    a.pos[i] = reinterpret_cast<uint32_t*>(ws + (2 * i + 1) * list);
  }
  a.part = reinterpret_cast<float*>(ws + 4 * list);
  int bits = 1;
  while (((int64_t)1 << bits) <= a.vocab) ++bits;   // the largest key is V itself (dropped)
  a.passes = (bits + SORT_BITS - 1) / SORT_BITS;
  const bool gb = p->grad_dtype == SSD_DTYPE_BF16, ob = p->out_dtype == SSD_DTYPE_BF16;
  // one CTA per SM next to the sorting cluster, in whole clusters: 8 + 17 * 8 = 144 of 148 SMs
  a.zero_ctas = a.accumulate ? 0 : 17 * SORT_CTAS;
  const size_t smem = sizeof(SortShared);
  const void* fn = ob ? (const void*)grad_sort_kernel<bf16> : (const void*)grad_sort_kernel<float>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  void* args[] = {&a};
  e = cudaLaunchKernel(fn, dim3((unsigned)(SORT_CTAS + a.zero_ctas)), dim3(SORT_THREADS), args, smem, stream);
  if (e != cudaSuccess || a.n == 0) return e;
  const bool vec = rows16(p->grad, a.gs, a.dim, p->grad_dtype) && rows16(p->out, a.os, a.dim, p->out_dtype);
  if (gb) {
    if (ob) return vec ? grad_sums<bf16, bf16, true>(a, stream) : grad_sums<bf16, bf16, false>(a, stream);
    return vec ? grad_sums<bf16, float, true>(a, stream) : grad_sums<bf16, float, false>(a, stream);
  }
  if (ob) return vec ? grad_sums<float, bf16, true>(a, stream) : grad_sums<float, bf16, false>(a, stream);
  return vec ? grad_sums<float, float, true>(a, stream) : grad_sums<float, float, false>(a, stream);
}

}  // namespace ssd
