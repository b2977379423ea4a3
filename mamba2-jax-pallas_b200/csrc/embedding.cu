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
// floats.  Launches:
//   1. one cluster of 8 CTAs sorts (id, position) pairs by a stable radix sort whose histograms
//      live in distributed shared memory; few ids are placed by counting instead;
//   2. a programmatic dependent launch that begins at once.  Its first CTAs write the zero rows of
//      the ids that do not occur, most of a dense gradient: a CTA marks the ids of its own rows
//      in a shared bitmap.  The others wait for the sort; they cut the sorted order into pieces
//      of equal length, whatever the ids, so that one frequent id cannot hold up a CTA.  A warp
//      sums a piece's rows over 256 columns in f32 and writes each id's row.  An id that goes on
//      for at most `extend` rows into the next piece is finished by the piece it began in; a
//      longer one leaves its parts in the workspace;
//   3. the parts of such ids are added up, again in order.
#include <algorithm>

#include <cooperative_groups.h>

#include "common.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "ssd_kernels.h"

namespace cg = cooperative_groups;

namespace ssd {
namespace {

constexpr int VEC = 8;            // columns per lane

// Which columns of a run of 256 a lane holds.
//   EIGHT  8 lane .. + 7: one 16-byte access of bf16
//   FOURS  4 lane .. + 3, and the same 128 further on: two 16-byte accesses of f32, each of
//          them 512 contiguous bytes per warp (8 f32 side by side would leave half sectors)
//   ONES   lane, lane + 32, ...: any width and alignment
enum Cols { EIGHT, FOURS, ONES };

template <Cols M>
__device__ __forceinline__ int col_of(int lane, int k) {
  return M == EIGHT ? lane * 8 + k : M == FOURS ? lane * 4 + (k & 3) + 128 * (k >> 2) : lane + 32 * k;
}

__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b) {
  a = __uint_as_float(u << 16);
  b = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The lane's columns of `row` (the start of a run of 256; `left` columns to the row's end).
template <typename T, Cols M>
__device__ __forceinline__ void load_cols(const T* row, int64_t left, float (&v)[VEC]) {
  const int lane = threadIdx.x & 31;
  if constexpr (M == EIGHT && sizeof(T) == 2) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (lane * 8 < left) q = *reinterpret_cast<const uint4*>(row + lane * 8);
    unpack2(q.x, v[0], v[1]); unpack2(q.y, v[2], v[3]); unpack2(q.z, v[4], v[5]); unpack2(q.w, v[6], v[7]);
  } else if constexpr (M != ONES) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int c = col_of<M>(lane, 4 * g);
      if constexpr (sizeof(T) == 4) {
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < left) q = *reinterpret_cast<const float4*>(row + c);
        v[4 * g] = q.x; v[4 * g + 1] = q.y; v[4 * g + 2] = q.z; v[4 * g + 3] = q.w;
      } else {
        uint2 q = make_uint2(0, 0);
        if (c < left) q = *reinterpret_cast<const uint2*>(row + c);
        unpack2(q.x, v[4 * g], v[4 * g + 1]); unpack2(q.y, v[4 * g + 2], v[4 * g + 3]);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = lane + 32 * k < left ? ld(row + lane + 32 * k) : 0.f;
  }
}

template <typename T, Cols M>
__device__ __forceinline__ void store_cols(T* row, int64_t left, const float (&v)[VEC]) {
  const int lane = threadIdx.x & 31;
  if constexpr (M == EIGHT && sizeof(T) == 2) {
    if (lane * 8 < left)
      *reinterpret_cast<uint4*>(row + lane * 8) =
          make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
  } else if constexpr (M != ONES) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int c = col_of<M>(lane, 4 * g);
      if (c < left) {
        if constexpr (sizeof(T) == 4)
          *reinterpret_cast<float4*>(row + c) = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        else
          *reinterpret_cast<uint2*>(row + c) = make_uint2(pack2(v[4 * g], v[4 * g + 1]), pack2(v[4 * g + 2], v[4 * g + 3]));
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (lane + 32 * k < left) st(row + lane + 32 * k, v[k]);
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
constexpr int LK_UNROLL = 4;      // runs of 256 columns in flight per warp

// One warp per (token, LK_UNROLL runs of 256 columns).  HBM-bound: 16384 rows of 2560 bf16 out of 50000
// 19.5 us (5.9 TB/s of the named rows and the result); 256 rows of 4096 2.2 us.
template <typename TW, typename TO, Cols M>
__global__ void __launch_bounds__(LK_THREADS) lookup_kernel(const LookupArgs a, int runs) {
  const int64_t unit = (int64_t)blockIdx.x * (LK_THREADS / 32) + threadIdx.x / 32;
  const int64_t t = unit / runs;
  if (t >= a.n) return;
  const int64_t c0 = (unit - t * runs) * (256 * LK_UNROLL);
  const int64_t row = row_of(a.ids, a.is64, t, a.vocab, a.pad);
  TO* o = static_cast<TO*>(a.out) + t * a.os;
  const TW* w = static_cast<const TW*>(a.w) + (row < 0 ? 0 : row) * a.ws;
  float v[LK_UNROLL][VEC];
#pragma unroll
  for (int i = 0; i < LK_UNROLL; ++i) {
    const int64_t c = c0 + 256 * i;
    load_cols<TW, M>(w + c, row < 0 ? 0 : a.dim - c, v[i]);   // a dropped token reads nothing
  }
#pragma unroll
  for (int i = 0; i < LK_UNROLL; ++i) {
    const int64_t c = c0 + 256 * i;
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[i][k] = row < 0 ? 0.f : v[i][k] * a.scale;
    store_cols<TO, M>(o + c, a.dim - c, v[i]);
  }
}

bool rows16(const void* p, int64_t stride, int64_t dim, int dtype) {
  const int64_t es = dtype == SSD_DTYPE_BF16 ? 2 : 4;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * es) % 16 == 0 && dim % VEC == 0;
}

template <typename TW, typename TO>
cudaError_t lookup(const LookupArgs& a, bool vec, cudaStream_t stream) {
  constexpr int W = LK_THREADS / 32;
  constexpr Cols M = sizeof(TW) == 2 && sizeof(TO) == 2 ? EIGHT : FOURS;
  const int64_t runs = (a.dim + 256 * LK_UNROLL - 1) / (256 * LK_UNROLL);
  const unsigned grid = (unsigned)((a.n * runs + W - 1) / W);
  if (vec) lookup_kernel<TW, TO, M><<<grid, LK_THREADS, 0, stream>>>(a, (int)runs);
  else lookup_kernel<TW, TO, ONES><<<grid, LK_THREADS, 0, stream>>>(a, (int)runs);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// gradient: sort
// ---------------------------------------------------------------------------
constexpr int SORT_CTAS = 8;      // the sorting cluster
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_AHEAD = 4;
constexpr int SORT_BITS = 9;
constexpr int SORT_BINS = 1 << SORT_BITS;
constexpr int ZERO_ROWS = 8192;   // rows whose bits the bitmap holds at a time

struct GradArgs {
  int64_t n, vocab, dim, gs, os, pad, piece, npieces;
  int is64, passes, bits, accumulate;   // `bits` of an id per pass
  int zero_ctas, zero_first;      // CTAs that write zero rows; so many of them come before the sums' CTAs
  int zero_lanes;                 // lanes of a zero row, as a power of two
  int extend;                     // rows that a piece may take from the next one, at most a piece and 32
  float scale;
  const void* ids;
  const void* g;
  void* out;
  uint2* list[2];                 // (id, position), sorted by id (V = dropped, last); result in list[0]
  float* part;                    // (npieces, 2, dim)
  int* heavy;                     // count, then the pieces in which an id with parts begins
};

struct SortShared {
  // this CTA's counts, then each warp's next slot among the CTA's; a column lies in 32 banks
  uint32_t warp_bin[SORT_WARPS][SORT_BINS + 1];
  uint32_t cta_bin[SORT_BINS];                // this CTA's count of each digit, read by the cluster
  uint32_t base[SORT_BINS];                   // first slot of each digit for this CTA
  uint32_t scan[SORT_WARPS];
};

// One stable pass of the radix sort over the cluster, by the `bits` from `shift` on.  What bounds
// it are the scattered stores, a line for every lane: id and position go in one 8-byte store
// (32768 ids: 34 -> 28 us).  CTA c and its warp w own consecutive tokens; a warp takes 32 of them
// at a time and lanes with equal digits find each other by match_any, so equal digits keep
// their order.
template <bool FIRST>
__device__ void sort_pass(const GradArgs& a, SortShared* s, int shift, int bits, const uint2* from, uint2* to) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, bins = 1 << bits;
  for (int i = tid; i < SORT_WARPS * bins; i += SORT_THREADS) s->warp_bin[i >> bits][i & (bins - 1)] = 0;
  __syncthreads();
  const int64_t per = (a.n + ctas * SORT_WARPS - 1) / (ctas * SORT_WARPS);
  const int64_t lo = (int64_t)(cta * SORT_WARPS + w) * per, hi = min(lo + per, a.n);
  auto key_at = [&](int64_t t) -> uint32_t {
    if constexpr (FIRST) {
      const int64_t v = row_of(a.ids, a.is64, t, a.vocab, a.pad);
      return v < 0 ? (uint32_t)a.vocab : (uint32_t)v;
    } else {
      return from[t].x;
    }
  };
  // SORT_AHEAD groups of 32 tokens are loaded at a time
  for (int64_t t0 = lo; t0 < hi; t0 += 32 * SORT_AHEAD) {
    uint32_t k[SORT_AHEAD];
#pragma unroll
    for (int j = 0; j < SORT_AHEAD; ++j) k[j] = key_at(min(t0 + 32 * j + lane, hi - 1));
#pragma unroll
    for (int j = 0; j < SORT_AHEAD; ++j) {
      const bool in = t0 + 32 * j + lane < hi;
      const unsigned live = __ballot_sync(0xffffffffu, in);
      if (in) {
        const uint32_t d = (k[j] >> shift) & (bins - 1);
        const unsigned same = __match_any_sync(live, d);
        if (lane == __ffs(same) - 1) s->warp_bin[w][d] += __popc(same);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  // a warp per digit: exclusive over this CTA's warps, total over the CTA
  for (int d = w; d < bins; d += SORT_WARPS) {
    const uint32_t c = s->warp_bin[lane][d];
    uint32_t incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    s->warp_bin[lane][d] = incl - c;
    if (lane == 31) s->cta_bin[d] = incl;
  }
  cluster.sync();
  // first slot of digit d for this CTA: all smaller digits, then digit d in the CTAs before
  uint32_t before = 0, total = 0;
  if (tid < bins) {
    for (int c = 0; c < ctas; ++c) {
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
  if (tid < bins) {
    uint32_t base = incl - total + before;
    for (int i = 0; i < w; ++i) base += s->scan[i];
    s->base[tid] = base;
  }
  __syncthreads();
  for (int64_t t0 = lo; t0 < hi; t0 += 32 * SORT_AHEAD) {
    uint2 e[SORT_AHEAD];
#pragma unroll
    for (int j = 0; j < SORT_AHEAD; ++j) {
      const int64_t t = min(t0 + 32 * j + lane, hi - 1);
      if constexpr (FIRST) e[j] = make_uint2(key_at(t), (uint32_t)t);
      else e[j] = from[t];
    }
#pragma unroll
    for (int j = 0; j < SORT_AHEAD; ++j) {
      const bool in = t0 + 32 * j + lane < hi;
      const unsigned live = __ballot_sync(0xffffffffu, in);
      if (in) {
        const uint32_t d = (e[j].x >> shift) & (bins - 1);
        const unsigned same = __match_any_sync(live, d);
        const uint32_t slot = s->base[d] + s->warp_bin[w][d] + __popc(same & ((1u << lane) - 1));
        __syncwarp(live);
        if (lane == __ffs(same) - 1) s->warp_bin[w][d] += __popc(same);
        to[slot] = e[j];
      }
      __syncwarp();
    }
  }
  cluster.sync();   // the cluster's keys are in place; every CTA has read the others' counts
}

__global__ void __launch_bounds__(SORT_THREADS, 1) sort_kernel(const GradArgs a) {
  extern __shared__ uint8_t smem[];
  ptx::griddep_launch_dependents();   // the zero rows need nothing from here
  SortShared* s = reinterpret_cast<SortShared*>(smem);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.heavy = 0;
  // the passes end in list[0]
  int to = (a.passes - 1) & 1;
  sort_pass<true>(a, s, 0, a.bits, nullptr, a.list[to]);
  for (int p = 1; p < a.passes; ++p) {
    sort_pass<false>(a, s, p * a.bits, a.bits, a.list[to], a.list[to ^ 1]);
    to ^= 1;
  }
}

// Few ids: a warp finds a token's place by counting the ids before it, four tokens at a time, all
// ids in the shared memory of every CTA.  An id and its position make one 32-bit number, so each pair
// takes one comparison: n^2 of them, spread over the GPU, against the radix sort's passes, which
// wait for one another.  777 ids 3.4 us, 4000 ids 9 us.
constexpr int RANK_THREADS = 512, RANK_WARPS = RANK_THREADS / 32, RANK_KEYS = 4;
constexpr int64_t RANK_MAX = 4096;
constexpr int64_t RANK_TABLE = 64 << 20;

__global__ void __launch_bounds__(RANK_THREADS) rank_kernel(const GradArgs a, int shift) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* code = reinterpret_cast<uint32_t*>(smem);
  ptx::griddep_launch_dependents();   // the zero rows need nothing from here
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, n = (int)a.n, padded = (n + 127) / 128 * 128;
  if (blockIdx.x == 0 && tid == 0) *a.heavy = 0;
#pragma unroll 4
  for (int t = tid; t < padded; t += RANK_THREADS) {
    const int64_t v = row_of(a.ids, a.is64, min(t, n - 1), a.vocab, a.pad);
    code[t] = t < n ? (uint32_t)(v < 0 ? a.vocab : v) << shift | (uint32_t)t : ~0u;
  }
  __syncthreads();
  const int warps = gridDim.x * RANK_WARPS;
  for (int t0 = blockIdx.x * RANK_WARPS + w; t0 < n; t0 += warps * RANK_KEYS) {
    uint32_t mine[RANK_KEYS], before[RANK_KEYS];
#pragma unroll
    for (int k = 0; k < RANK_KEYS; ++k) {
      mine[k] = t0 + k * warps < n ? code[t0 + k * warps] : 0;
      before[k] = 0;
    }
#pragma unroll 2
    for (int j = lane * 4; j < padded; j += 128) {
      const uint4 q = *reinterpret_cast<const uint4*>(code + j);
#pragma unroll
      for (int k = 0; k < RANK_KEYS; ++k)
        before[k] += (q.x < mine[k]) + (q.y < mine[k]) + (q.z < mine[k]) + (q.w < mine[k]);
    }
#pragma unroll
    for (int k = 0; k < RANK_KEYS; ++k) {
      const uint32_t at = __reduce_add_sync(0xffffffffu, before[k]);
      if (lane == 0 && t0 + k * warps < n) a.list[0][at] = make_uint2(mine[k] >> shift, (uint32_t)(t0 + k * warps));
    }
  }
}

// ---------------------------------------------------------------------------
// gradient: zero rows and sums
// ---------------------------------------------------------------------------
constexpr int SUM_THREADS = 256;
constexpr int SUM_COLS = 32 * VEC;   // columns of a warp

// A row's columns as they were loaded, unpacked when they are added: bf16 in flight takes half
// the registers of f32, so twice the rows fit.
template <typename T, Cols M>
struct Raw {
  static constexpr int ROWS = 4;    // in flight
  float v[VEC];
  __device__ __forceinline__ void load(const T* row, int64_t left) { load_cols<T, M>(row, left, v); }
  __device__ __forceinline__ void add(float (&acc)[VEC]) const {
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += v[k];
  }
};
template <Cols M>
struct RawPacked {
  static constexpr int ROWS = 8;
  uint32_t u[4];
  __device__ __forceinline__ void load(const bf16* row, int64_t left) {
    const int lane = threadIdx.x & 31;
    if constexpr (M == EIGHT) {
      uint4 q = make_uint4(0, 0, 0, 0);
      if (lane * 8 < left) q = *reinterpret_cast<const uint4*>(row + lane * 8);
      u[0] = q.x; u[1] = q.y; u[2] = q.z; u[3] = q.w;
    } else {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint2 q = make_uint2(0, 0);
        if (col_of<FOURS>(lane, 4 * g) < left) q = *reinterpret_cast<const uint2*>(row + col_of<FOURS>(lane, 4 * g));
        u[2 * g] = q.x; u[2 * g + 1] = q.y;
      }
    }
  }
  __device__ __forceinline__ void add(float (&acc)[VEC]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a, b;
      unpack2(u[k], a, b);
      acc[2 * k] += a;
      acc[2 * k + 1] += b;
    }
  }
};
template <>
struct Raw<bf16, EIGHT> : RawPacked<EIGHT> {};
template <>
struct Raw<bf16, FOURS> : RawPacked<FOURS> {};

template <typename TO, Cols M>
__device__ __forceinline__ void put_row(const GradArgs& a, uint32_t id, int64_t c0, float (&acc)[VEC]) {
  TO* o = static_cast<TO*>(a.out) + (int64_t)id * a.os + c0;
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] *= a.scale;
  if (a.accumulate) {
    float old[VEC];
    load_cols<TO, M>(o, a.dim - c0, old);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += old[k];
  }
  store_cols<TO, M>(o, a.dim - c0, acc);
}

// Zero rows of the ids that do not occur.  A CTA owns rows [r0, r1) and marks those that
// occur in a shared bitmap, ZERO_ROWS at a time, reading all ids (L2) once for each.  2^zero_lanes
// lanes write a row.
template <typename TO>
__device__ void zero_rows(const GradArgs& a, int cta, uint32_t* bits) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int rows_at_once = 32 >> a.zero_lanes, sub = lane & ((1 << a.zero_lanes) - 1), step = 1 << a.zero_lanes;
  const int64_t per = (a.vocab + a.zero_ctas - 1) / a.zero_ctas;
  const int64_t r0 = cta * per, r1 = min(r0 + per, a.vocab);
  // two 64-bit ids at a time where they lie so
  const int64_t pairs = a.is64 && reinterpret_cast<uintptr_t>(a.ids) % 16 == 0 ? a.n / 2 : 0;
  for (int64_t b0 = r0; b0 < r1; b0 += ZERO_ROWS) {
    const int count = (int)min((int64_t)ZERO_ROWS, r1 - b0);
    for (int i = tid; i < ZERO_ROWS / 32; i += SUM_THREADS) bits[i] = 0;
    __syncthreads();
    auto mark = [&](int64_t v) {
      if (v >= b0 && v < b0 + count && v != a.pad) atomicOr(&bits[(v - b0) >> 5], 1u << ((v - b0) & 31));
    };
#pragma unroll 8
    for (int64_t t = tid; t < pairs; t += SUM_THREADS) {
      const longlong2 q = __ldg(static_cast<const longlong2*>(a.ids) + t);
      mark(q.x);
      mark(q.y);
    }
#pragma unroll 8
    for (int64_t t = 2 * pairs + tid; t < a.n; t += SUM_THREADS) mark(row_of(a.ids, a.is64, t, a.vocab, a.pad));
    __syncthreads();
    for (int i = (tid >> 5) * rows_at_once + (lane >> a.zero_lanes); i < count; i += SUM_THREADS / 32 * rows_at_once) {
      if ((bits[i >> 5] >> (i & 31)) & 1) continue;
      TO* o = static_cast<TO*>(a.out) + (b0 + i) * a.os;
      // values before the first 16-byte boundary, whole 16 bytes, and what is left
      constexpr int PER = 16 / sizeof(TO);
      const int dim = (int)a.dim, head = min((int)((0 - reinterpret_cast<uintptr_t>(o)) % 16 / sizeof(TO)), dim);
      const int body = (dim - head) / PER;
      uint4* q = reinterpret_cast<uint4*>(o + head);
      // streaming: nothing reads them soon (plain stores: 777 x 50257 x 768 f32 34.6 us, so 32.8)
      for (int c = sub; c < body; c += step) __stcs(q + c, make_uint4(0, 0, 0, 0));
      for (int c = sub; c < head; c += step) st(o + c, 0.f);
      for (int c = head + body * PER + sub; c < dim; c += step) st(o + c, 0.f);
    }
    __syncthreads();
  }
}

// HBM-bound: 32768 tokens into 131072 x 4096 bf16 232 us (5.8 TB/s), 777 into 50257 x 768 f32 27 us.
// The first a.zero_first CTAs: zero rows.  Then a warp for each (piece p, 256 columns): rows of the
// sorted positions [p * piece, + piece).  Then the other CTAs of zero rows.
template <typename TG, typename TO, Cols M>
__global__ void __launch_bounds__(SUM_THREADS, 4) grad_rows_kernel(const __grid_constant__ GradArgs a, int col_warps) {
  __shared__ uint32_t bits[ZERO_ROWS / 32];
  const int sum_ctas = (int)gridDim.x - a.zero_ctas, at = (int)blockIdx.x - a.zero_first;
  if (at < 0 || at >= sum_ctas) {
    zero_rows<TO>(a, at < 0 ? (int)blockIdx.x : (int)blockIdx.x - sum_ctas, bits);
    ptx::griddep_wait();   // what is launched behind may take the sort as done, too
    return;
  }
  using R = Raw<TG, M>;
  ptx::griddep_wait();
  const int unit = at * (SUM_THREADS / 32) + threadIdx.x / 32;
  const int p = unit / col_warps;
  if (p >= (int)a.npieces) return;
  const int lane = threadIdx.x & 31, n = (int)a.n, top = n - 1, piece = (int)a.piece, extend = a.extend;
  const int c0 = (unit - p * col_warps) * SUM_COLS, left = (int)a.dim - c0;
  const int lo = p * piece, hi = min(lo + piece, n);
  const uint32_t none = (uint32_t)a.vocab;
  const uint2* list = a.list[0];
  // every key that decides about the piece's ends, in one round trip
  const uint32_t first = list[lo].x, last = list[hi - 1].x;
  const uint32_t k_prev = list[max(lo - 1, 0)].x, k_before = list[max(lo - piece - 1, 0)].x;
  const uint32_t k_far = list[min(lo + extend, top)].x, k_next = list[min(hi, top)].x, k_next_far = list[min(hi + extend, top)].x;
  const uint32_t k_ext = list[min(hi + lane, top)].x;
  uint2 mine = list[min(lo + lane, top)];
  if (first == none) return;
  // the first id: it may have begun in an earlier piece, and then either the piece before
  // finishes it (skip) or this piece's share of it is a part (open)
  bool open = lo > 0 && k_prev == first;
  const bool skip = open && (lo == piece || k_before != first) && (lo + extend >= n || k_far != first);
  // the last id: rows of the next piece that this one takes, or the id goes on too long
  int end = hi;
  bool goes_on = false;
  if (hi < n && last != none && k_next == last) {
    if ((lo == 0 || k_prev != last) && (hi + extend >= n || k_next_far != last))
      end += __popc(__ballot_sync(0xffffffffu, lane < extend && hi + lane < n && k_ext == last));
    else
      goes_on = true;
  }
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  uint32_t cur = first;
  auto close = [&]() {   // the rows of `cur` in this piece are added up
    if (open) {
      if (!skip) store_cols<float, M>(a.part + (int64_t)(p * 2) * a.dim + c0, left, acc);
    } else if (cur != none) {
      put_row<TO, M>(a, cur, c0, acc);
    }
    open = false;
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  };
  for (int i0 = lo; i0 < end; i0 += 32) {
    if (i0 > lo) mine = list[min(i0 + lane, top)];
    const uint32_t mk = mine.x;
    const int mp = (int)mine.y;
    const int m = min(32, end - i0);
    // rows that add something, and rows at which another id begins
    const unsigned live = __ballot_sync(0xffffffffu, lane < m && mk != none);
    uint32_t before = __shfl_up_sync(0xffffffffu, mk, 1);
    if (lane == 0) before = cur;
    unsigned turns = __ballot_sync(0xffffffffu, lane < m && mk != before);
#pragma unroll 1
    for (int j0 = 0; j0 < m; j0 += R::ROWS) {
      R v[R::ROWS];
#pragma unroll
      for (int j = 0; j < R::ROWS; ++j) {
        const int64_t t = __shfl_sync(0xffffffffu, mp, j0 + j);
        v[j].load(static_cast<const TG*>(a.g) + t * a.gs + c0, (live >> (j0 + j)) & 1 ? left : 0);
      }
#pragma unroll
      for (int j = 0; j < R::ROWS; ++j) {
        if ((turns >> (j0 + j)) & 1) {
          close();
          cur = __shfl_sync(0xffffffffu, mk, j0 + j);
        }
        v[j].add(acc);   // zeros past the end
      }
    }
  }
  if (open || !goes_on) {
    close();
  } else {
    store_cols<float, M>(a.part + (int64_t)(p * 2 + 1) * a.dim + c0, left, acc);
    if (c0 == 0 && lane == 0) a.heavy[1 + atomicAdd(a.heavy, 1)] = p;
  }
}

// CTA (64 columns, every gridDim.y-th listed piece p): the id that begins in piece p, the sum of
// its parts.  The parts of the following pieces are shared out over the CTA's warps in runs,
// each summed in order, and the runs are added in order; which CTA does it, and when, changes
// nothing.  3.5 us with few parts; 32768 tokens by Zipf's law, 4096 columns 18 us.
constexpr int JOIN_COLS = 64;
template <typename TO>
__global__ void __launch_bounds__(SUM_THREADS) grad_join_kernel(const __grid_constant__ GradArgs a) {
  constexpr int W = SUM_THREADS / 32;
  __shared__ float2 sums[W][32];
  __shared__ int pieces;
  ptx::griddep_wait();
  const uint2* list = a.list[0];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, listed = *a.heavy, npieces = (int)a.npieces;
  const int64_t c = (int64_t)blockIdx.x * JOIN_COLS + 2 * lane;
  const bool one = c < a.dim, two = c + 1 < a.dim;
  for (int h = blockIdx.y; h < listed; h += gridDim.y) {
    const int p = a.heavy[1 + h];
    const uint32_t id = list[(int64_t)(p + 1) * a.piece - 1].x;
    if (threadIdx.x == 0) pieces = 0;
    __syncthreads();
    // pieces p+1, p+2, ... whose first key is the id: they follow one another
    int mine = 0;
#pragma unroll 8
    for (int q = p + 1 + threadIdx.x; q < npieces; q += SUM_THREADS) mine += list[(int64_t)q * a.piece].x == id;
    if (mine) atomicAdd(&pieces, mine);
    __syncthreads();
    const int count = pieces, per = (count + W - 1) / W;
    const int q0 = p + 1 + w * per, q1 = min(q0 + per, p + 1 + count);
    float2 acc = make_float2(0.f, 0.f);
    if (w == 0) {
      const float* row = a.part + (int64_t)(p * 2 + 1) * a.dim + c;
      if (one) acc.x = row[0];
      if (two) acc.y = row[1];
    }
#pragma unroll 8
    for (int q = q0; q < q1; ++q) {
      const float* row = a.part + (int64_t)q * 2 * a.dim + c;
      acc.x += one ? row[0] : 0.f;
      acc.y += two ? row[1] : 0.f;
    }
    sums[w][lane] = acc;
    __syncthreads();
    if (w == 0 && one) {
      for (int i = 1; i < W; ++i) {
        acc.x += sums[i][lane].x;
        acc.y += sums[i][lane].y;
      }
      TO* o = static_cast<TO*>(a.out) + (int64_t)id * a.os + c;
      st(o, acc.x * a.scale + (a.accumulate ? ld(o) : 0.f));
      if (two) st(o + 1, acc.y * a.scale + (a.accumulate ? ld(o + 1) : 0.f));
    }
    __syncthreads();
  }
}

template <typename TG, typename TO, Cols M>
cudaError_t grad_rows(const GradArgs& a, cudaStream_t stream) {
  const int64_t col_warps = (a.dim + SUM_COLS - 1) / SUM_COLS;
  constexpr int W = SUM_THREADS / 32;
  cudaError_t e = launch_dependent(grad_rows_kernel<TG, TO, M>,
                                   dim3((unsigned)(a.zero_ctas + (a.npieces * col_warps + W - 1) / W)), SUM_THREADS, 0, 1, stream, a, (int)col_warps);
  if (e == cudaSuccess && a.n > a.piece + a.extend)   // shorter lists have no id with parts
    e = launch_dependent(grad_join_kernel<TO>,
                         dim3((unsigned)((a.dim + JOIN_COLS - 1) / JOIN_COLS), (unsigned)std::min<int64_t>(a.npieces, 64)), SUM_THREADS, 0, 1, stream, a);
  return e;
}

template <typename TG, typename TO>
cudaError_t grad_rows(const GradArgs& a, bool vec, cudaStream_t stream) {
  constexpr Cols M = sizeof(TG) == 2 && sizeof(TO) == 2 ? EIGHT : FOURS;
  return vec ? grad_rows<TG, TO, M>(a, stream) : grad_rows<TG, TO, ONES>(a, stream);
}

int64_t piece_len(int64_t n, int64_t dim) {
  // at most 2048 pieces, which bounds the parts' workspace; 32 rows, which a warp reads in a few
  // microseconds, unless that leaves most of the GPU without a warp: 777 x 768 f32 takes 20 us in
  // pieces of 32 and 6 us in pieces of 4
  const int64_t col_warps = (dim + SUM_COLS - 1) / SUM_COLS;
  int64_t len = 32;
  while ((n + len - 1) / len > 2048) len *= 2;
  while (len > 4 && len <= 32 && n / len * col_warps < 148 * 16 && (2 * n + len - 1) / len <= 2048) len /= 2;
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
  const int64_t len = piece_len(n, dim), pieces = (n + len - 1) / len;
  return 2 * up256((size_t)n * 8) + up256((size_t)(pieces + 1) * 4) + (size_t)pieces * 2 * dim * 4;
}

// (positions, pieces and columns are ints in the kernels: checked by the caller)
cudaError_t launch_embedding_grad(const ssd_embedding_grad_params_t* p, void* workspace, cudaStream_t stream) {
  GradArgs a{};
  a.n = p->num_tokens; a.vocab = p->vocab; a.dim = p->dim;
  a.gs = p->grad_stride_row; a.os = p->out_stride_row; a.pad = p->padding_idx;
  a.is64 = p->tokens_int64; a.accumulate = p->accumulate; a.scale = p->scale;
  a.ids = p->tokens; a.g = p->grad; a.out = p->out;
  a.piece = piece_len(a.n, a.dim);
  a.extend = (int)std::min<int64_t>(a.piece, 32);
  a.npieces = (a.n + a.piece - 1) / a.piece;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const size_t list = up256((size_t)a.n * 8);
  for (int i = 0; i < 2; ++i) a.list[i] = reinterpret_cast<uint2*>(ws + i * list);
  a.heavy = reinterpret_cast<int*>(ws + 2 * list);
  a.part = reinterpret_cast<float*>(ws + 2 * list + up256((size_t)(a.npieces + 1) * 4));
  int bits = 1, shift = 1;
  while (((int64_t)1 << bits) <= a.vocab) ++bits;   // the largest key is V itself (dropped)
  while (((int64_t)1 << shift) < a.n) ++shift;
  a.passes = (bits + SORT_BITS - 1) / SORT_BITS;
  a.bits = (bits + a.passes - 1) / a.passes;
  const bool gb = p->grad_dtype == SSD_DTYPE_BF16, ob = p->out_dtype == SSD_DTYPE_BF16;
  cudaError_t e;
  // (us by counting / by the cluster) 4 x 1395 x 71 6 / 12, 875 x 6111 x 128 12 / 21, 4096 x 2000 x 128 19 / 23,
  // 8192 x 2000 x 128 29 / 28.  Where zero rows take longer than the sort, the counting's CTAs on every
  // SM only hold them up: 2274 x 64120 x 223 f32 (57 MB) 24 / 27, 6000 x 50000 x 768 bf16 (77 MB) 35 / 31,
  // 777 x 50257 x 768 f32 (154 MB) 35 / 34.
  const int out_size = p->out_dtype == SSD_DTYPE_BF16 ? 2 : 4;
  if (a.n <= RANK_MAX && bits + shift <= 32 && (a.accumulate || a.vocab * a.dim <= RANK_TABLE / out_size)) {
    const int64_t ctas = std::min<int64_t>(148, std::max<int64_t>(1, (a.n + RANK_WARPS - 1) / RANK_WARPS));
    rank_kernel<<<(unsigned)ctas, RANK_THREADS, (size_t)(a.n + 127) / 128 * 512, stream>>>(a, shift);
    e = cudaGetLastError();
  } else {
    const size_t smem = sizeof(SortShared);
    static std::atomic<uint64_t> allowed{0};
    e = allow_smem((const void*)sort_kernel, smem, &allowed);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SORT_CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(SORT_CTAS);
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, sort_kernel, a);
  }
  if (e != cudaSuccess) return e;
  // Two of the four resident CTAs of an SM write zeros while the sort runs, the others wait for it;
  // all four where there are few sums.  Where the table is large against the ids (which every CTA of
  // zero rows reads), half of the zero rows or more come behind the sums, which would else leave their
  // slots empty (us without / with): 5000 ids, 100000 x 1600 f32 132 / 118; 3000 ids, 131072 x 4096 bf16 201 /
  // 185; 4000 ids, 60000 x 1216 f32 (292 MB) 61 / 58; but 777 ids, 50257 x 768 f32 (154 MB) 33 / 37; 32768 ids,
  // 131072 x 4096 bf16 254 / 267.  The two sides meet at 22000 ids for 131072 x 4096 bf16, 15500 for 100000 x
  // 1600 f32 and 12500 for 50257 x 2560 f32; the rule changes at 28339, 16891 and 13582, at most 5 % off.
  const int64_t sum_ctas = (a.npieces * ((a.dim + SUM_COLS - 1) / SUM_COLS) + SUM_THREADS / 32 - 1) / (SUM_THREADS / 32);
  if (!a.accumulate) {
    a.zero_first = 148 * 4 - (int)std::min<int64_t>(148 * 2, sum_ctas);
    const bool large = a.vocab * a.dim * out_size / (148 * 8) >= std::max<int64_t>(4 * 8 * a.n, (256 << 20) / (148 * 8));
    a.zero_ctas = large ? 148 * 8 : a.zero_first;
  }
  // a lane for every 16 bytes of a row (8192 ids, a table of 400000 x 64 bf16: 41 -> 29 us)
  while (a.zero_lanes < 5 && ((int64_t)16 << a.zero_lanes) < a.dim * out_size) ++a.zero_lanes;
  if (a.accumulate && a.n == 0) return e;
  const bool vec = rows16(p->grad, a.gs, a.dim, p->grad_dtype) && rows16(p->out, a.os, a.dim, p->out_dtype);
  if (gb) return ob ? grad_rows<bf16, bf16>(a, vec, stream) : grad_rows<bf16, float>(a, vec, stream);
  return ob ? grad_rows<float, bf16>(a, vec, stream) : grad_rows<float, float>(a, vec, stream);
}

}  // namespace ssd
