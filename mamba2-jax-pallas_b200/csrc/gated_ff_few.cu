// Gated feed-forward block of a few tokens (decoding, a drafted continuation): the same operator as gated_ff.cu
// where the weights are read for so few rows that nothing but their bytes counts.
//
// The products run in f32 on the CUDA cores, straight from the weights as they lie in memory.  A warp takes
// some rows of a weight (for g and u the same row of both), or a part of their columns where a weight has few rows, against all tokens' values,
// which stay in L1.  Two launches, the second set up while the first runs; bound by HBM.
#include <algorithm>

#include "common.cuh"
#include "gated_ff.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "ssd_kernels.h"

namespace ssd {
namespace {

constexpr int WARPS = 8;
constexpr int SMS = 148;   // of a B200

struct FewArgs {
  const void* x;                   // (tokens, K) values of T
  const void* w[2];                // rows of the weight, and of the other one
  void* out;                       // (tokens, rows)
  int64_t xs, ws[2], os;           // values between rows
  int64_t rows;
  int K, tokens, act, parts;       // parts: warps that share rows, a power of two
  unsigned* status;                // cleared by the first launch (nothing here waits)
};

// 16 bytes as f32.
template <typename T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int N = 4;
  uint4 q;
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w); }
};
template <>
struct Piece<bf16> {
  static constexpr int N = 8;
  uint4 q;
  __device__ __forceinline__ float at(int i) const {
    const uint32_t u = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
  }
};

// The piece from column c of a row of K values; zeros past the end.
template <typename T, bool ALIGNED>
__device__ __forceinline__ Piece<T> load(const T* row, int c, int K) {
  Piece<T> p;
  p.q = make_uint4(0, 0, 0, 0);
  if constexpr (ALIGNED) {
    if (c < K) p.q = __ldg(reinterpret_cast<const uint4*>(row + c));
  } else {
    T* v = reinterpret_cast<T*>(&p.q);
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i)
      if (c + i < K) v[i] = row[c + i];
  }
  return p;
}

// Values v[0..N) summed over the warp; lane l ends with the sum of value l % N.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int bit = 1;
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2, bit *= 2) {
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

// R tokens; a warp's rows: ROWS of each of W weights.  W = 2: out = act(g) u, else the product itself.
template <typename T, int R, int ROWS, int W, bool ALIGNED>
__global__ void __launch_bounds__(32 * WARPS) few_kernel(const __grid_constant__ FewArgs a) {
  constexpr int N = R * ROWS * W;   // sums of a warp, at most 32
  __shared__ float sh[WARPS][N];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % a.parts, units = WARPS / a.parts;   // groups of rows of the CTA
  const int64_t r0 = ((int64_t)blockIdx.x * units + warp / a.parts) * ROWS;
  constexpr int STEP = 32 * Piece<T>::N;
  const int steps = (a.K + STEP - 1) / STEP, s0 = (int)((int64_t)steps * part / a.parts), s1 = (int)((int64_t)steps * (part + 1) / a.parts);
  const T* row[W * ROWS];
#pragma unroll
  for (int i = 0; i < W * ROWS; ++i)   // rows past the end are read as the last one
    row[i] = static_cast<const T*>(a.w[i % W]) + min(r0 + i / W, a.rows - 1) * a.ws[i % W];
  const T* x = static_cast<const T*>(a.x);
  float sum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0.f;
  // pieces of the weights on their way, always this many steps ahead
  constexpr int AHEAD = W * ROWS == 1 ? 8 : W * ROWS == 2 ? 6 : 3;
  Piece<T> w[AHEAD][W * ROWS];
  auto fetch = [&](int k, int s) {
#pragma unroll
    for (int i = 0; i < W * ROWS; ++i) w[k][i] = load<T, ALIGNED>(row[i], s < s1 ? (s * 32 + lane) * Piece<T>::N : a.K, a.K);
  };
  auto start = [&]() {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) fetch(k, s0 + k);
  };
  // The first launch waits for whatever ran before it (an optimizer may have written the weights) and lets the second
  // one be set up, which may read its weight at once: the first has waited for that.
  if constexpr (W == 2) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    start();
  } else {
    start();
    ptx::griddep_wait();
  }
  for (int s = s0; s < s1; s += AHEAD) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int c = s + k < s1 ? ((s + k) * 32 + lane) * Piece<T>::N : a.K;
#pragma unroll
      for (int t = 0; t < R; ++t) {
        const Piece<T> v = load<T, ALIGNED>(x + min(t, a.tokens - 1) * a.xs, c, a.K);
#pragma unroll
        for (int j = 0; j < Piece<T>::N; ++j)
#pragma unroll
          for (int i = 0; i < W * ROWS; ++i) sum[t * W * ROWS + i] = fmaf(v.at(j), w[k][i].at(j), sum[t * W * ROWS + i]);
      }
      fetch(k, s + k + AHEAD);
    }
  }
  const float total = warp_sums<N>(sum);
  if (lane < N) sh[warp][lane] = total;
  __syncthreads();
  // a thread per token and row: the parts in order
  constexpr int OUT = R * ROWS;
  for (int i = threadIdx.x; i < units * OUT; i += 32 * WARPS) {
    const int unit = i / OUT, t = i % OUT / ROWS, r = i % ROWS;
    const int64_t at = ((int64_t)blockIdx.x * units + unit) * ROWS + r;
    if (t >= a.tokens || at >= a.rows) continue;
    float v[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      v[k] = 0.f;
      for (int j = 0; j < a.parts; ++j) v[k] += sh[unit * a.parts + j][t * W * ROWS + r * W + k];
    }
    T* o = static_cast<T*>(a.out) + t * a.os + at;
    if constexpr (W == 2) st(o, ff::activate(a.act, v[0], nullptr) * v[1]);
    else st(o, v[0]);
  }
}

template <typename T, int R, int ROWS, int W>
cudaError_t launch_rows(FewArgs a, bool aligned, cudaStream_t st) {
  // warps of a row: as many as fill the GPU
  a.parts = 1;
  while (a.parts < WARPS && (a.rows + ROWS - 1) / ROWS * a.parts < SMS * 24 && a.K / (a.parts * 2) >= 32 * Piece<T>::N) a.parts *= 2;
  const int64_t per = WARPS / a.parts * ROWS, ctas = (a.rows + per - 1) / per;
  return aligned ? launch_dependent(few_kernel<T, R, ROWS, W, true>, dim3((unsigned)ctas), 32 * WARPS, 0, 1, st, a)
                 : launch_dependent(few_kernel<T, R, ROWS, W, false>, dim3((unsigned)ctas), 32 * WARPS, 0, 1, st, a);
}

template <typename T, int W>
cudaError_t launch_tokens(const FewArgs& a, bool aligned, cudaStream_t st) {
  if (a.tokens == 1) return launch_rows<T, 1, 1, W>(a, aligned, st);
  if (a.tokens == 2) return launch_rows<T, 2, 1, W>(a, aligned, st);
  if (a.tokens <= 4) return launch_rows<T, 4, 2, W>(a, aligned, st);
  return launch_rows<T, 8, 2, W>(a, aligned, st);
}

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

template <typename T>
bool aligned16(const void* p, int64_t stride, int64_t rows) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || stride * sizeof(T) % 16 == 0);
}

template <typename T>
cudaError_t launch_as(const ssd_gated_ff_params_t* p, uint8_t* ws, cudaStream_t st, const char** at) {
  const int64_t ldh = (p->hidden + 7) / 8 * 8;
  FewArgs a{};
  a.x = p->x; a.xs = p->x_stride_row;
  a.w[0] = p->w_gate; a.w[1] = p->w_up;
  a.ws[0] = p->w_gate_stride_row; a.ws[1] = p->w_up_stride_row;
  a.out = ws + 256; a.os = ldh;
  a.rows = p->hidden;
  a.K = (int)p->dim;
  a.tokens = (int)p->tokens;
  a.act = p->activation;
  a.status = reinterpret_cast<unsigned*>(ws);
  constexpr int N = Piece<T>::N;
  cudaError_t e = launch_tokens<T, 2>(a, p->dim % N == 0 && aligned16<T>(p->x, a.xs, p->tokens) && aligned16<T>(p->w_gate, a.ws[0], a.rows) &&
                                            aligned16<T>(p->w_up, a.ws[1], a.rows), st);
  *at = "gate and up";
  if (e != cudaSuccess) return e;
  a.x = ws + 256; a.xs = ldh;
  a.w[0] = p->w_down; a.w[1] = nullptr;
  a.ws[0] = p->w_down_stride_row;
  a.out = p->y; a.os = p->dim_out;
  a.rows = p->dim_out;
  a.K = (int)p->hidden;
  a.status = nullptr;
  *at = "down";
  return launch_tokens<T, 1>(a, p->hidden % N == 0 && aligned16<T>(p->w_down, a.ws[0], a.rows), st);
}

}  // namespace

bool gated_ff_is_few(const ssd_gated_ff_params_t* p) { return p->tokens <= 8; }

size_t gated_ff_few_workspace(const ssd_gated_ff_params_t* p) { return 256 + up256((size_t)p->tokens * ((p->hidden + 7) / 8 * 8) * 4); }

cudaError_t launch_gated_ff_few(const ssd_gated_ff_params_t* p, void* workspace, cudaStream_t st, const char** at) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return p->dtype == SSD_DTYPE_BF16 ? launch_as<bf16>(p, ws, st, at) : launch_as<float>(p, ws, st, at);
}

}  // namespace ssd
