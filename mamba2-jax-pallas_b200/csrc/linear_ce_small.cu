// Linear cross entropy of a few tokens (scoring a drafted continuation, a small fine-tuning
// step): the same operator as linear_ce.cu where the weight is read for so few rows that
// nothing but its bytes counts.
//
// The products run in f32 on the CUDA cores, straight from the weight as it lies in memory: a
// tensor-core tile would be mostly padding, and f32 weights would first have to be split into
// planes (three times their bytes).  Bound by HBM: the loss reads the weight once, the gradients
// read it once more and write as much.
//   1. a warp takes four words at a time, all rows of hidden in shared memory: logits, and per row
//      the running maximum and sum over the words that the warp saw;
//   2. one CTA: losses, their sum or mean, the factors of the gradients;
//   3. gradients: a CTA takes a range of words and 1024 columns; every value of the weight that it
//      loads goes into grad_hidden's sums in registers, and the same dl times hidden is
//      grad_weight's row;
//   4. the ranges' sums of grad_hidden are added, in order.
//
// Measured: loss of 1 x 131072 x 4096 bf16 162 us (6.6 TB/s) + 4 us, 7 x 50257 x 768 f32 32 us (4.8 TB/s) + 4
// us; gradients of 2 x 50000 x 2560 bf16 190 us, 8 x 50257 x 768 f32 150 us.
#include <algorithm>

#include "common.cuh"
#include "launch.cuh"
#include "linear_ce.cuh"
#include "ptx_sm100.cuh"
#include "ssd_kernels.h"

namespace ssd {
namespace {
using namespace ce;

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_CTAS = 148;
constexpr int WORDS = 4;                     // words of a warp at a time
constexpr int MAX_ROWS = 8;                  // rows of one pass over the weight
constexpr int MAX_TOKENS = 4 * MAX_ROWS;     // of a call
constexpr size_t MAX_SMEM = 222 * 1024;      // besides the static part
constexpr int G_THREADS = 256, G_COLS = 4 * G_THREADS, G_TILE = 64;

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }
int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

struct SmallArgs {
  int tokens, vocab, dim, is64, ns;
  int64_t xs, ws, ignore, ld;
  const void* x;
  const void* w;
  const void* targets;
  unsigned* status;         // the workspace's status word: cleared (nothing here waits)
  float2* stats;            // (tokens, ns)
  float* picked;            // (tokens)
  float* logits;            // (tokens, ld) or NULL
  // finish
  int reduction;
  const float* grad_loss;
  float* loss;
  float* lse;
  RowFactors* factors;      // (tokens) or NULL
  // gradients
  float* part;              // (ranges, rows, dim): grad_hidden's sums
  int ranges, group;        // ranges of words; threads that share one
  void* gx;
  void* gw;
  int gw_bf16;
};

template <typename T>
__device__ __forceinline__ float value(const T* p, int64_t i) { return ld(p + i); }

// 16 bytes of one word's row, as a lane holds them: U accesses of K values each.  U = 1 where rows
// are aligned to 16 bytes; else the widest access that every row allows.
template <typename T, int U>
struct Piece {
  static constexpr int K = 16 / sizeof(T) / U, COLS = 32 * K * U;   // columns of a warp's piece
  // asynchronous copies of 4 bytes were slower than loads (77 against 51 us for 6 x 56640 x 1106)
  static constexpr bool ASYNC = U == 1;
  uint32_t u[4];

  // Into the lane's own 16 bytes of shared memory, asynchronously.  Columns past the end are
  // read at the last ones and cleared by cut().
  static __device__ __forceinline__ void copy(void* slot, const T* row, int c0, int dim) {
    const int lane = threadIdx.x & 31;
    const uint32_t to = ptx::smem_u32(slot);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(row + min(c0 + lane * K, dim - K)) : "memory");
  }
  __device__ __forceinline__ void take(const void* slot) {
    const uint4 q = *static_cast<const uint4*>(slot);
    u[0] = q.x; u[1] = q.y; u[2] = q.z; u[3] = q.w;
  }
  // The same straight into registers, for U = 4 and 8.
  __device__ __forceinline__ void load(const T* row, int c0, int dim) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (U == 4) {
        u[i] = *reinterpret_cast<const uint32_t*>(row + min(c0 + (i * 32 + lane) * K, dim - K));
        continue;
      }
      const int c = c0 + 2 * i * 32 + lane;
      u[i] = *reinterpret_cast<const uint16_t*>(row + min(c, dim - 1)) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(row + min(c + 32, dim - 1)) << 16;
    }
  }
  __device__ __forceinline__ void cut(int c0, int dim) {
    constexpr int V = 16 / sizeof(T), W = 4 / sizeof(T);   // values of a piece, of a 32-bit word
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c0 + col(i) >= dim) u[i / W] &= W == 1 ? 0u : i & 1 ? 0xffffu : 0xffff0000u;
  }
  // value i of the 16 / sizeof(T), and its column (from c0)
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[i]);
    return __uint_as_float(i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
  }
  static __device__ __forceinline__ int col(int i) { return (i / K * 32 + (threadIdx.x & 31)) * K + i % K; }
};

// Values v[0..N) summed over the warp; lane l ends with the sum of value l % N.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int bit = 1;
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2, bit *= 2) {
    // lanes that differ in `bit` keep the values with that bit of the index clear and set
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = lane & bit ? v[2 * i + 1] : v[2 * i], give = lane & bit ? v[2 * i] : v[2 * i + 1];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
    }
  }
  float s = v[0];
#pragma unroll
  for (int o = N; o < 32; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// blockIdx.y: rows 8 y ..; R of them are computed (those past the last token on zeros).  A lane
// copies its pieces of the weight STAGES - 1 steps ahead, across the ends of the words, into
// slots of its own: 96 KB in flight per SM, which registers could not hold.
template <typename T, int R, int U, int STAGES>
__global__ void __launch_bounds__(SM_THREADS, 1) small_logits_kernel(const __grid_constant__ SmallArgs a) {
  using P = Piece<T, U>;
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];   // ring, then hidden (R, dim rounded up to whole pieces)
  __shared__ float2 red[SM_WARPS][R * WORDS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint4* ring = reinterpret_cast<uint4*>(smem) + warp * (STAGES * WORDS * 32) + lane;   // [stage][word][lane]
  float* xs = reinterpret_cast<float*>(smem + SM_WARPS * STAGES * WORDS * 512);
  const int row0 = blockIdx.y * MAX_ROWS, rows = min(R, a.tokens - row0);
  const int steps = (a.dim + P::COLS - 1) / P::COLS, pitch = steps * P::COLS;
  const T* x = static_cast<const T*>(a.x) + row0 * a.xs;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *a.status = 0;
  const int stride = SM_CTAS * SM_WARPS * WORDS, v_first = (blockIdx.x * SM_WARPS + warp) * WORDS;
  int next_v = v_first, next_s = 0, next_slot = 0;
  auto fetch = [&]() {   // the next piece of the next words, in the order of their use
    if (next_v < a.vocab) {
#pragma unroll
      for (int j = 0; j < WORDS; ++j)
        P::copy(ring + (next_slot * WORDS + j) * 32, static_cast<const T*>(a.w) + (int64_t)min(next_v + j, a.vocab - 1) * a.ws,
                next_s * P::COLS, a.dim);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    next_slot = next_slot + 1 == STAGES ? 0 : next_slot + 1;
    if (++next_s == steps) {
      next_s = 0;
      next_v += stride;
    }
  };
  if constexpr (P::ASYNC)
    for (int i = 0; i < STAGES - 1; ++i) fetch();
  for (int i = tid; i < R * pitch; i += SM_THREADS) {
    const int r = i / pitch, c = i - r * pitch;
    xs[i] = r < rows && c < a.dim ? value(x + r * a.xs, c) : 0.f;
  }
  // lane l: row l / WORDS (if below R), word l % WORDS of the warp's four
  const int my_row = (lane / WORDS) % R, my_word = lane % WORDS;
  const int64_t y = my_row < rows ? target_at(a.targets, a.is64, row0 + my_row) : -1;
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  int slot = 0;
  for (int v0 = v_first; v0 < a.vocab; v0 += stride) {
    float acc[WORDS * R];
#pragma unroll
    for (int i = 0; i < WORDS * R; ++i) acc[i] = 0.f;
#pragma unroll (P::ASYNC ? 1 : 2)
    for (int s = 0; s < steps; ++s) {
      P q[WORDS];
      if constexpr (P::ASYNC) {
        fetch();   // into the slot that the last step emptied
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
#pragma unroll
        for (int j = 0; j < WORDS; ++j) q[j].take(ring + (slot * WORDS + j) * 32);
        slot = slot + 1 == STAGES ? 0 : slot + 1;
      } else {
#pragma unroll
        for (int j = 0; j < WORDS; ++j)
          q[j].load(static_cast<const T*>(a.w) + (int64_t)min(v0 + j, a.vocab - 1) * a.ws, s * P::COLS, a.dim);
      }
      if (s == steps - 1 && pitch > a.dim) {
#pragma unroll
        for (int j = 0; j < WORDS; ++j) q[j].cut(s * P::COLS, a.dim);
      }
      const float* xc = xs + s * P::COLS;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        constexpr int G = P::K >= 4 ? 4 : P::K;    // columns side by side in shared memory
#pragma unroll
        for (int i = 0; i < V; i += G) {
          float xv[G];
          const float* at = xc + r * pitch + P::col(i);
          if constexpr (G == 4) *reinterpret_cast<float4*>(xv) = *reinterpret_cast<const float4*>(at);
          else if constexpr (G == 2) *reinterpret_cast<float2*>(xv) = *reinterpret_cast<const float2*>(at);
          else xv[0] = *at;
#pragma unroll
          for (int k = 0; k < G; ++k)
#pragma unroll
            for (int j = 0; j < WORDS; ++j) acc[r * WORDS + j] = fmaf(q[j].at(i + k), xv[k], acc[r * WORDS + j]);
        }
      }
    }
    const float s = warp_sums(acc);
    const int v = v0 + my_word;
    if (v < a.vocab && lane < WORDS * R && my_row < rows) {
      if (a.logits) a.logits[(row0 + my_row) * a.ld + v] = s;
      if (v == y) {
        a.picked[row0 + my_row] = s;     // kept out of the sum
      } else {
        const float n = fmaxf(top, s * LOG2E), at = n == -INFINITY ? 0.f : n;
        sum = sum * exp2f(top - at) + exp2f(fmaf(s, LOG2E, -at));
        top = n;
      }
    }
  }
  if (lane < WORDS * R) red[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (tid < rows) {
    float t = -INFINITY;
    for (int i = 0; i < SM_WARPS * WORDS; ++i) t = fmaxf(t, red[i / WORDS][tid * WORDS + i % WORDS].x);
    const float at = t == -INFINITY ? 0.f : t;
    float l = 0.f;
    for (int i = 0; i < SM_WARPS * WORDS; ++i) {
      const float2 e = red[i / WORDS][tid * WORDS + i % WORDS];
      l += e.y * exp2f(e.x - at);
    }
    a.stats[(row0 + tid) * a.ns + blockIdx.x] = make_float2(t, l);
  }
}

// One CTA, a warp per token (in turns).
__global__ void __launch_bounds__(256) small_finish_kernel(const __grid_constant__ SmallArgs a) {
  __shared__ float losses[MAX_TOKENS];
  ptx::griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int count = 0;
  for (int t = 0; t < a.tokens; ++t) count += target_at(a.targets, a.is64, t) != a.ignore;
  const bool none = a.reduction == SSD_REDUCE_NONE, mean = a.reduction == SSD_REDUCE_MEAN;
  const float scale = mean ? (float)(1.0 / (double)max(count, 1)) : 1.f;
  for (int t = warp; t < a.tokens; t += 8) {
    const int64_t y64 = target_at(a.targets, a.is64, t);
    const bool counts = y64 != a.ignore;
    const RowResult r = warp_row(a.stats + t * a.ns, a.ns, a.picked + t, y64 >= 0 && y64 < a.vocab ? (int)y64 : -1);
    if (lane) continue;
    const float loss = counts ? r.loss : 0.f;
    losses[t] = loss;
    if (none) a.loss[t] = loss;
    if (a.lse) a.lse[t] = counts ? r.lse : 0.f;
    if (a.factors) {
      const float w = scale * (a.grad_loss ? a.grad_loss[none ? t : 0] : 1.f);
      RowFactors f = {0.f, 0.f, 0.f};
      if (counts) f = {r.top, w * r.inv, w * r.pm1};
      a.factors[t] = f;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && !none) {
    double s = 0;
    for (int t = 0; t < a.tokens; ++t) s += (double)losses[t];
    *a.loss = (float)(mean ? s / (double)max(count, 1) : s);
  }
}

template <typename T, bool VECTOR>
__device__ __forceinline__ void load4(const T* row, int c, int dim, int step, float (&v)[4]) {
  if constexpr (VECTOR) {
    // 4 columns side by side
    if constexpr (sizeof(T) == 4) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < dim) q = *reinterpret_cast<const float4*>(row + c);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      uint2 q = make_uint2(0, 0);
      if (c < dim) q = *reinterpret_cast<const uint2*>(row + c);
      v[0] = __uint_as_float(q.x << 16); v[1] = __uint_as_float(q.x & 0xffff0000u);
      v[2] = __uint_as_float(q.y << 16); v[3] = __uint_as_float(q.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = c + k * step < dim ? value(row, c + k * step) : 0.f;
  }
}
template <typename T, bool VECTOR>
__device__ __forceinline__ void store4(T* row, int c, int dim, int step, const float (&v)[4]) {
  if constexpr (VECTOR) {
    if (c >= dim) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
      *reinterpret_cast<uint2*>(row + c) = *reinterpret_cast<const uint2*>(h);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k * step < dim) st(row + c + k * step, v[k]);
  }
}

// CTA (ranges of words, 1024 columns); a thread holds 4 columns of every row of hidden and of
// grad_hidden's sums.  Where hidden is narrow, groups of `a.group` threads take ranges of their own.
template <typename T, typename TW, int R, bool VECTOR>
__global__ void __launch_bounds__(G_THREADS) small_grad_kernel(const __grid_constant__ SmallArgs a) {
  extern __shared__ float dl[];   // (groups * G_TILE, R)
  ptx::griddep_wait();
  const int tid = threadIdx.x, groups = G_THREADS / a.group, g = tid / a.group, t = tid - g * a.group;
  const int c = blockIdx.y * G_COLS + (VECTOR ? 4 * t : t), step = a.group;
  const int per = (a.vocab + a.ranges - 1) / a.ranges, range = blockIdx.x * groups + g;
  float x[R][4], acc[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[r][k] = acc[r][k] = 0.f;
    // an ignored row may hold anything
    if (r < a.tokens && target_at(a.targets, a.is64, r) != a.ignore)
      load4<T, VECTOR>(static_cast<const T*>(a.x) + r * a.xs, c, a.dim, step, x[r]);
  }
  for (int off = 0; off < per; off += G_TILE) {
    __syncthreads();
    for (int i = tid; i < groups * G_TILE * R; i += G_THREADS) {
      const int r = i / (groups * G_TILE), e = i - r * (groups * G_TILE);
      const int rg = blockIdx.x * groups + e / G_TILE, j = off + e % G_TILE;
      const int64_t v = (int64_t)rg * per + j;
      float d = 0.f;
      if (r < a.tokens && j < per && v < a.vocab) {
        const RowFactors f = a.factors[r];
        d = target_at(a.targets, a.is64, r) == v ? f.at_y : f.f * exp2f(fmaf(a.logits[r * a.ld + v], LOG2E, -f.top));
        if (f.f == 0.f && f.at_y == 0.f) d = 0.f;   // ignored: its logits may be NaN
      }
      dl[e * R + r] = d;
    }
    __syncthreads();
    const int64_t v0 = (int64_t)range * per + off;
    const int n = (int)min((int64_t)min(G_TILE, per - off), a.vocab - v0);
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      float w[4] = {0.f, 0.f, 0.f, 0.f}, gw[4] = {0.f, 0.f, 0.f, 0.f};
      if (a.gx) load4<T, VECTOR>(static_cast<const T*>(a.w) + (v0 + j) * a.ws, c, a.dim, step, w);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float d = dl[(g * G_TILE + j) * R + r];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          acc[r][k] = fmaf(d, w[k], acc[r][k]);
          gw[k] = fmaf(d, x[r][k], gw[k]);
        }
      }
      if (a.gw) store4<TW, VECTOR>(static_cast<TW*>(a.gw) + (v0 + j) * a.dim, c, a.dim, step, gw);
    }
  }
  if (a.gx) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= a.tokens) continue;
      if (target_at(a.targets, a.is64, r) == a.ignore) {   // zero times an infinite or NaN weight is not zero
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[r][k] = 0.f;
      }
      store4<float, VECTOR>(a.part + ((int64_t)range * a.tokens + r) * a.dim, c, a.dim, step, acc[r]);
    }
  }
}

// grad_hidden: the ranges' sums.  A CTA takes 32 values: each of its warps adds a run of ranges,
// and the runs are added in order.
constexpr int J_WARPS = 16;
template <typename T>
__global__ void __launch_bounds__(32 * J_WARPS) small_join_kernel(const __grid_constant__ SmallArgs a) {
  __shared__ float sums[J_WARPS][32];
  ptx::griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = (int64_t)a.tokens * a.dim, i = (int64_t)blockIdx.x * 32 + lane;
  const int per = (a.ranges + J_WARPS - 1) / J_WARPS, lo = warp * per, hi = min(lo + per, a.ranges);
  float s = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int j = lo; j < hi; ++j) s += a.part[j * n + i];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp || i >= n) return;
  for (int w = 1; w < J_WARPS; ++w) s += sums[w][lane];
  st(static_cast<T*>(a.gx) + i, s);
}

int row_width(int64_t tokens) { return tokens == 1 ? 1 : tokens == 2 ? 2 : tokens <= 4 ? 4 : 8; }

// hidden's rows in f32, padded to whole pieces (at most 256 columns)
size_t logits_smem(const ssd_linear_ce_params_t* p) {
  return (size_t)row_width(p->tokens) * ((p->dim + 255) / 256 * 256) * 4;
}

size_t ring_bytes(int stages) { return (size_t)SM_WARPS * stages * WORDS * 512; }

template <typename T, int R, int U, int STAGES>
cudaError_t run_logits(const SmallArgs& a, size_t smem, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  const auto kernel = small_logits_kernel<T, R, U, STAGES>;
  const cudaError_t e = allow_smem((const void*)kernel, MAX_SMEM, &allowed);
  if (e != cudaSuccess) return e;
  kernel<<<dim3(SM_CTAS, (unsigned)cdiv(a.tokens, MAX_ROWS)), SM_THREADS, smem + ring_bytes(STAGES), st>>>(a);
  return cudaGetLastError();
}
template <typename T, int R, int U>
cudaError_t run_logits(const SmallArgs& a, size_t smem, cudaStream_t st) {
  // four stages where hidden leaves the room, else two
  if (smem + ring_bytes(4) <= MAX_SMEM) return run_logits<T, R, U, 4>(a, smem, st);
  return run_logits<T, R, U, 2>(a, smem, st);
}
template <typename T, int U>
cudaError_t run_logits(const SmallArgs& a, size_t smem, cudaStream_t st) {
  switch (row_width(a.tokens)) {
    case 1: return run_logits<T, 1, U>(a, smem, st);
    case 2: return run_logits<T, 2, U>(a, smem, st);
    case 4: return run_logits<T, 4, U>(a, smem, st);
    default:   // (most_tokens)
      if constexpr (sizeof(T) == 4 || U > 1) return run_logits<T, 8, U>(a, smem, st);
      return cudaErrorInvalidValue;
  }
}
// Every row of the weight can be read in accesses of `bytes`.
bool reads_by(const ssd_linear_ce_params_t* p, int bytes) {
  const int64_t es = p->dtype == SSD_DTYPE_BF16 ? 2 : 4;
  return reinterpret_cast<uintptr_t>(p->weight) % bytes == 0 && p->weight_stride_row * es % bytes == 0 && p->dim * es % bytes == 0;
}
cudaError_t run_logits(const ssd_linear_ce_params_t* p, const SmallArgs& a, cudaStream_t st) {
  const size_t smem = logits_smem(p);
  if (p->dtype == SSD_DTYPE_F32) return reads_by(p, 16) ? run_logits<float, 1>(a, smem, st) : run_logits<float, 4>(a, smem, st);
  if (reads_by(p, 16)) return run_logits<bf16, 1>(a, smem, st);
  return reads_by(p, 4) ? run_logits<bf16, 4>(a, smem, st) : run_logits<bf16, 8>(a, smem, st);
}

template <typename T, typename TW, int R>
cudaError_t run_grad(const SmallArgs& a, bool vec, cudaStream_t st) {
  return launch_dependent(vec ? small_grad_kernel<T, TW, R, true> : small_grad_kernel<T, TW, R, false>,
                          dim3((unsigned)(a.ranges / (G_THREADS / a.group)), (unsigned)cdiv(a.dim, G_COLS)), G_THREADS,
                          (size_t)(G_THREADS / a.group) * G_TILE * R * sizeof(float), 1, st, a);
}
template <typename T, typename TW>
cudaError_t run_grad(const SmallArgs& a, bool vec, cudaStream_t st) {
  switch (row_width(a.tokens)) {
    case 1: return run_grad<T, TW, 1>(a, vec, st);
    case 2: return run_grad<T, TW, 2>(a, vec, st);
    default:   // (most_tokens)
      if constexpr (sizeof(T) == 4) return a.tokens <= 4 ? run_grad<T, TW, 4>(a, vec, st) : run_grad<T, TW, 8>(a, vec, st);
      return cudaErrorInvalidValue;
  }
}

bool aligned(const void* p, int64_t stride, int64_t dim, int dtype) {
  const int64_t es = dtype == SSD_DTYPE_BF16 ? 2 : 4;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * es % 16 == 0 && dim * es % 16 == 0;
}

struct SmallPlan {
  size_t picked, factors, stats, logits, part, total;
  int ranges, group;
  int64_t ld;
};

SmallPlan plan_of(const ssd_linear_ce_params_t* p) {
  SmallPlan q{};
  const bool grad = p->grad_hidden || p->grad_weight;
  q.ld = (p->vocab + 63) / 64 * 64;
  q.group = 32;
  while (q.group < G_THREADS && q.group * 4 < p->dim) q.group *= 2;
  // about eight CTAs per SM over the ranges and column blocks, and 16 words or more in a range
  const int groups = G_THREADS / q.group;
  q.ranges = groups * (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(SM_CTAS * 8, cdiv(p->dim, G_COLS)), cdiv(p->vocab, 16 * groups)));
  size_t at = 256;   // the status word, as in every workspace
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  q.picked = take((size_t)p->tokens * 4);
  q.factors = take((size_t)p->tokens * sizeof(RowFactors));
  q.stats = take((size_t)p->tokens * SM_CTAS * sizeof(float2));
  q.logits = take(grad ? (size_t)p->tokens * q.ld * 4 : 0);
  q.part = take(p->grad_hidden ? (size_t)q.ranges * p->tokens * p->dim * 4 : 0);
  q.total = at;
  return q;
}

// The most tokens of this form, from both forms' times (us, this one against tensor cores):
//   bf16 loss       4 x 131072 x 4096 180 / 207, 5: 301 / 205; 4 x 50257 x 768 25 / 31, 6: 37 / 31; where the
//                   weight would have to be copied for the tensor maps: 8 x 50000 x 1001 59 / 81, 16: 105 / 82
//   bf16 gradients  2 x 50257 x 768 76 / 91, 4: 119 / 91; 2 x 50000 x 2560 190 / 193, 3: 313 / 195
//   f32 loss        32 x 50257 x 768 123 / 132, 32 x 50000 x 2560 331 / 384
//   f32 gradients   8 x 50257 x 768 150 / 223, 8 x 50000 x 2560 385 / 595 (rows of one pass)
int64_t most_tokens(const ssd_linear_ce_params_t* p) {
  const bool grad = p->grad_hidden || p->grad_weight;
  if (p->dtype == SSD_DTYPE_F32) return grad ? MAX_ROWS : MAX_TOKENS;
  if (grad) return 2;
  return reinterpret_cast<uintptr_t>(p->weight) % 16 == 0 && p->weight_stride_row % 8 == 0 ? 4 : MAX_ROWS;
}

}  // namespace

bool linear_ce_is_small(const ssd_linear_ce_params_t* p) {
  return p->tokens <= most_tokens(p) && logits_smem(p) + ring_bytes(2) <= MAX_SMEM && p->vocab < (1 << 30);
}

size_t linear_ce_small_workspace(const ssd_linear_ce_params_t* p) { return plan_of(p).total; }

#define CE_CHECK(call, where)     \
  do {                            \
    const cudaError_t e_ = (call); \
    if (e_ != cudaSuccess) {      \
      *at = where;                \
      return e_;                  \
    }                             \
  } while (0)

cudaError_t launch_linear_ce_small(const ssd_linear_ce_params_t* p, void* workspace, cudaStream_t st, const char** at) {
  const SmallPlan q = plan_of(p);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool bf = p->dtype == SSD_DTYPE_BF16, grad = p->grad_hidden || p->grad_weight;
  SmallArgs a{};
  a.tokens = (int)p->tokens; a.vocab = (int)p->vocab; a.dim = (int)p->dim; a.is64 = p->targets_int64; a.ns = SM_CTAS;
  a.xs = p->hidden_stride_row; a.ws = p->weight_stride_row; a.ignore = p->ignore_index; a.ld = q.ld;
  a.x = p->hidden; a.w = p->weight; a.targets = p->targets;
  a.status = reinterpret_cast<unsigned*>(ws);
  a.stats = reinterpret_cast<float2*>(ws + q.stats);
  a.picked = reinterpret_cast<float*>(ws + q.picked);
  a.logits = grad ? reinterpret_cast<float*>(ws + q.logits) : nullptr;
  a.reduction = p->reduction; a.grad_loss = p->grad_loss; a.loss = p->loss; a.lse = p->lse;
  a.factors = grad ? reinterpret_cast<RowFactors*>(ws + q.factors) : nullptr;
  a.part = reinterpret_cast<float*>(ws + q.part);
  a.ranges = q.ranges;
  a.group = q.group;
  a.gx = p->grad_hidden; a.gw = p->grad_weight; a.gw_bf16 = p->grad_weight_dtype == SSD_DTYPE_BF16;
  CE_CHECK(run_logits(p, a, st), "logits");
  CE_CHECK(launch_dependent(small_finish_kernel, dim3(1), 256, 0, 1, st, a), "loss");
  if (!grad) return cudaSuccess;
  const bool gvec = aligned(p->weight, p->weight_stride_row, p->dim, p->dtype) && aligned(p->hidden, p->hidden_stride_row, p->dim, p->dtype) &&
                    (!p->grad_weight || aligned(p->grad_weight, p->dim, p->dim, p->grad_weight_dtype));
  if (bf) CE_CHECK((a.gw_bf16 ? run_grad<bf16, bf16>(a, gvec, st) : run_grad<bf16, float>(a, gvec, st)), "gradients");
  else CE_CHECK((a.gw_bf16 ? run_grad<float, bf16>(a, gvec, st) : run_grad<float, float>(a, gvec, st)), "gradients");
  if (p->grad_hidden)
    CE_CHECK(launch_dependent(bf ? small_join_kernel<bf16> : small_join_kernel<float>,
                              dim3((unsigned)cdiv(p->tokens * p->dim, 32)), 32 * J_WARPS, 0, 1, st, a), "grad_hidden");
  return cudaSuccess;
}

}  // namespace ssd
