// Gated feed-forward block of a few tokens (decoding, a drafted continuation): the same operator as gated_ff.cu
// where the weights are read for so few rows that nothing but their bytes counts.
//
// The products run in f32 on the CUDA cores, straight from the weights as they lie in memory.  A warp takes
// some rows of a weight (for g and u the same row of both), or a part of their columns, against all tokens' values, which stay in
// L1.  The hidden values between the two launches stay f32: nothing here needs bf16 operands (rounded to bf16 they would double the
// square of the result's error, 0.0024 against 0.0017).  One or two CTAs per SM walk over the rows; every lane copies its own 16
// bytes of the weights some steps ahead, across the ends of the rows, into slots of shared memory that no other lane reads: 96 KB in
// flight per SM.  Bound by HBM and the two launches' ends: 1 token of 4096 x 12288 bf16 59.5 us (5.1 TB/s), 4 tokens 72, 1 token of
// 2560 x 7680 f32 43.6 us (5.4 TB/s), of 768 x 2048 bf16 6.1 us.  Rows that start at no 16-byte boundary: 1 token of 4095 x 12287
// bf16 95 us, 4 tokens 134 (value by value 144 and 284).
#include <algorithm>

#include "common.cuh"
#include "gated_ff.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "ssd_kernels.h"

namespace ssd {
namespace {

constexpr int WARPS = 16;          // of a CTA
// CTAs of an SM (two where the sums leave room: 1 token of 4096 x 12288 in 56.5 us, with one CTA 60.1), and the ring's places for 16
// bytes of every lane of a warp (twice as many gained nothing)
template <int N>
struct Shape {
  static constexpr int CTAS = N <= 4 ? 2 : 1, SLOTS = 12 / CTAS;
};
constexpr int SMS = 148;   // of a B200

struct FewArgs {
  const void* x;                   // (tokens, K) values, of T for g and u, else f32; blockIdx.y takes R of the tokens
  const void* w[2];                // rows of the weight, and of the other one
  void* out;                       // (tokens, rows): f32 hidden values, or the results in T
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

// As many f32 values as a piece of T holds.  In memory a row is N / 4 runs of a fraction of its length each: the first four values of
// every piece, then the next four, so that neighbouring lanes read neighbouring 16 bytes.
template <int N>
struct Hidden {
  float4 q[N / 4];
  static __device__ __forceinline__ int64_t place(int64_t c, int64_t length) {
    return N == 4 ? c : (c >> 2 & 1) * (length / 2) + (c >> 3) * 4 + (c & 3);
  }
  __device__ __forceinline__ float at(int i) const {
    const float4& p = q[i / 4];
    return i % 4 == 0 ? p.x : i % 4 == 1 ? p.y : i % 4 == 2 ? p.z : p.w;
  }
};

// Those whose first four lie at p and the next `run` behind; zeros where there are none.
template <int N>
__device__ __forceinline__ Hidden<N> hidden_at(const float* p, int run, bool there) {
  Hidden<N> h = {};
  if (there) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) h.q[k] = *reinterpret_cast<const float4*>(p + k * run);
  }
  return h;
}
// All but the first `left` become zeros: rows hold whole pieces, and what lies behind their last value was not written.
template <int R, int N>
__device__ __forceinline__ void cut(Hidden<N> (&h)[R], int left) {
#pragma unroll
  for (int t = 0; t < R; ++t)
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      float4& q = h[t].q[k];
      if (left < 4 * k + 1) q.x = 0.f;
      if (left < 4 * k + 2) q.y = 0.f;
      if (left < 4 * k + 3) q.z = 0.f;
      if (left < 4 * k + 4) q.w = 0.f;
    }
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

// The sums of a CTA's warps, `parts` of them to a group of rows, to the output: a thread per token and row.
template <typename T, int R, int ROWS, int W>
__device__ __forceinline__ void finish(const FewArgs& a, const float (*sh)[R * ROWS * W], int groups, int64_t first) {
  constexpr int OUT = R * ROWS;
  const int t0 = blockIdx.y * R;
  for (int i = threadIdx.x; i < groups * OUT; i += blockDim.x) {
    const int unit = i / OUT, t = i % OUT / ROWS, r = i % ROWS;
    const int64_t at = (first + unit) * ROWS + r;
    if (t0 + t >= a.tokens || at >= a.rows) continue;
    float v[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      v[k] = 0.f;
      for (int j = 0; j < a.parts; ++j) v[k] += sh[unit * a.parts + j][t * W * ROWS + r * W + k];   // in order
    }
    if constexpr (W == 2)
      static_cast<float*>(a.out)[(t0 + t) * a.os + Hidden<Piece<T>::N>::place(at, a.os)] = ff::activate(a.act, v[0], nullptr) * v[1];
    else
      st(static_cast<T*>(a.out) + (t0 + t) * a.os + at, v[0]);
  }
}

template <typename T, int R, int NR, typename X>
__device__ __forceinline__ void accumulate(float (&sum)[R * NR], const X (&x)[R], const Piece<T> (&w)[NR]) {
#pragma unroll
  for (int j = 0; j < Piece<T>::N; ++j)
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int i = 0; i < NR; ++i) sum[t * NR + i] = fmaf(x[t].at(j), w[i].at(j), sum[t * NR + i]);
}

// The first launch (W = 2: out = act(g) u) waits for whatever ran before it (an optimizer may have written the weights) and
// lets the second one (W = 1: the product itself) be set up, which may read its weight at once: the first has waited for that.
template <int W>
__device__ __forceinline__ void before_weights(const FewArgs& a) {
  if constexpr (W == 2) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.status = 0;
  }
}

// 16 bytes that start `shift` bytes into `own`, behind which `next` lies.  (The shift is the same for the warp.)
__device__ __forceinline__ uint4 window(const uint4& own, const uint4& next, unsigned shift) {
  uint32_t w[8] = {own.x, own.y, own.z, own.w, next.x, next.y, next.z, next.w};
#pragma unroll
  for (int k = 0; k < 7; ++k) w[k] = shift & 4 ? w[k + 1] : w[k];
#pragma unroll
  for (int k = 0; k < 5; ++k) w[k] = shift & 8 ? w[k + 2] : w[k];
  const unsigned half = shift << 3 & 16;
  return make_uint4(__funnelshift_r(w[0], w[1], half), __funnelshift_r(w[1], w[2], half), __funnelshift_r(w[2], w[3], half),
                    __funnelshift_r(w[3], w[4], half));
}

// Columns of a warp's step: every lane's 16 bytes.  Rows that do not start at 16 bytes are copied from the boundary in front, and a lane's
// columns lie in its own piece and the next lane's, so that the last lane has none.
template <typename T>
constexpr int step_columns(bool aligned) { return (aligned ? 32 : 31) * Piece<T>::N; }

// R tokens; a warp's rows: ROWS of each of W weights.
template <typename T, int R, int ROWS, int W, bool ALIGNED>
__global__ void __launch_bounds__(32 * WARPS, Shape<R * ROWS * W>::CTAS) few_kernel(const __grid_constant__ FewArgs a) {
  constexpr int N = R * ROWS * W, NR = W * ROWS, SLOTS = Shape<N>::SLOTS, STAGES = SLOTS / NR, STEP = (ALIGNED ? 32 : 31) * Piece<T>::N;
  extern __shared__ __align__(16) uint4 ring[];          // [WARPS][SLOTS][32]
  __shared__ float sh[2][WARPS][N];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % a.parts, groups = WARPS / a.parts;
  const int steps = (a.K + STEP - 1) / STEP, s0 = steps * part / a.parts, s1 = steps * (part + 1) / a.parts;
  const int64_t all = (a.rows + ROWS - 1) / ROWS, stride = (int64_t)gridDim.x * groups;
  uint4* const mine = ring + warp * SLOTS * 32 + lane;
  before_weights<W>(a);
  // the next step to copy: of group `next`, step `at`, into slot `to`
  int64_t next = (int64_t)blockIdx.x * groups + warp / a.parts;
  int at = s0, to = 0;
  const T* row[NR];
  auto rows_of = [&]() {
#pragma unroll
    for (int i = 0; i < NR; ++i)   // rows past the end are read as the last one
      row[i] = static_cast<const T*>(a.w[i % W]) + min(next * ROWS + i / W, a.rows - 1) * a.ws[i % W];
  };
  rows_of();
  auto copy = [&]() {
    if (next < all) {
      const int c = at * STEP + lane * Piece<T>::N;
#pragma unroll
      for (int i = 0; i < NR; ++i) {   // columns past the end are zeros
        const uint8_t* p = reinterpret_cast<const uint8_t*>(row[i]);
        int left = min(a.K - c, 32) * (int)sizeof(T);
        if constexpr (!ALIGNED) {      // (what lies in front of the row in its first 16 bytes is in its allocation)
          const int in = (int)(reinterpret_cast<uintptr_t>(p) & 15);
          p -= in;
          left += in;
        }
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(mine + (to * NR + i) * 32)),
                     "l"(left > 0 ? p + (int64_t)c * sizeof(T) : p), "r"(max(0, min(left, 16))) : "memory");
      }
      if (++at == s1) {
        at = s0;
        next += stride;
        rows_of();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++to == STAGES) to = 0;
  };
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) copy();
  if constexpr (W == 1) ptx::griddep_wait();
  const int tokens = min(R, a.tokens - (int)blockIdx.y * R);
  typedef std::conditional_t<W == 2, T, float> X;
  const X* x = static_cast<const X*>(a.x) + (int64_t)blockIdx.y * R * a.xs;
  // one load of each 128 bytes of x, all at once: found missing step by step, they would cost the first rows a trip to L2 each
  const int length = W == 1 ? (int)a.xs : a.K;
  for (int t = 0; t < tokens; ++t)
    for (int c = threadIdx.x * (128 / (int)sizeof(X)); c < length; c += 32 * WARPS * (128 / (int)sizeof(X))) {
      if constexpr (ALIGNED || W == 1) {
        uint32_t unused;
        asm volatile("ld.global.ca.b32 %0, [%1];" : "=r"(unused) : "l"(x + t * a.xs + c));
      } else {
        unsigned short unused;
        asm volatile("ld.global.ca.b16 %0, [%1];" : "=h"(unused) : "l"(x + t * a.xs + c));
      }
    }
  int from = 0, turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * groups; first < all; first += stride, turn ^= 1) {
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.f;
    unsigned shift[NR];    // not ALIGNED: of the rows' starts
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
        shift[i] = (unsigned)reinterpret_cast<uintptr_t>(static_cast<const T*>(a.w[i % W]) + min((first + warp / a.parts) * ROWS + i / W, a.rows - 1) * a.ws[i % W]) & 15;
    }
    for (int s = s0; s < s1; ++s) {
      const int c = s * STEP + lane * Piece<T>::N;
      std::conditional_t<W == 2, Piece<T>, Hidden<Piece<T>::N>> v[R];
      Piece<T> w[NR];
#pragma unroll
      for (int t = 0; t < R; ++t) {
        const X* xt = x + min(t, tokens - 1) * a.xs + (W == 1 ? c / (Piece<T>::N / 4) : c);
        v[t] = {};
        if constexpr (W == 1) {
          v[t] = hidden_at<Piece<T>::N>(xt, (int)a.xs / 2, c < a.K);
        } else if constexpr (ALIGNED) {
          if (c < a.K) v[t].q = *reinterpret_cast<const uint4*>(xt);
        } else if (c + 2 * Piece<T>::N <= a.K) {   // by the 16 bytes that hold them, which end within the row
          const unsigned in = (unsigned)reinterpret_cast<uintptr_t>(xt) & 15;
          const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(xt) - in);
          const uint4 own = q[0];
          v[t].q = in ? window(own, q[1], in) : own;
        } else if (lane < 31) {
          alignas(16) T u[Piece<T>::N];
#pragma unroll
          for (int k = 0; k < Piece<T>::N; ++k) u[k] = c + k < a.K ? xt[k] : T(0.f);
          v[t].q = *reinterpret_cast<const uint4*>(u);
        }
      }
      if constexpr (W == 1 && !ALIGNED) {
        if (a.K - c < Piece<T>::N) cut(v, a.K - c);
      }
      if constexpr (!ALIGNED) __syncwarp();   // the lane in front has read what is copied over
      copy();
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      if constexpr (!ALIGNED) __syncwarp();
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        w[i].q = mine[(from * NR + i) * 32];
        if constexpr (!ALIGNED) w[i].q = window(w[i].q, mine[(from * NR + i) * 32 + (lane < 31)], shift[i]);
      }
      if (++from == STAGES) from = 0;
      if (ALIGNED || lane < 31) accumulate<T, R, NR>(sum, v, w);
    }
    const float total = warp_sums<N>(sum);
    if (lane < N) sh[turn][warp][lane] = total;
    __syncthreads();       // (the buffer of the turn before is read by now only)
    finish<T, R, ROWS, W>(a, sh[turn], groups, first);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, int R, int ROWS, int W, bool ALIGNED>
cudaError_t launch_rows(FewArgs a, cudaStream_t st) {
  const int64_t groups = (a.rows + ROWS - 1) / ROWS;
  const unsigned passes = (unsigned)((a.tokens + R - 1) / R);
  const int steps = (a.K + step_columns<T>(ALIGNED) - 1) / step_columns<T>(ALIGNED);
  // parts of a row: the fewest steps of a warp; a turn's sums and meeting count as half a step
  using S = Shape<R * ROWS * W>;
  const int64_t slots = (int64_t)SMS * S::CTAS * WARPS;
  int best = 1;
  double least = 1e300;
  for (int parts = 1; parts <= WARPS && parts <= steps; parts *= 2) {
    const int64_t turns = (groups * parts + slots - 1) / slots;
    const double cost = (double)turns * ((double)((steps + parts - 1) / parts) + 0.5);
    if (cost < least) {
      least = cost;
      best = parts;
    }
  }
  a.parts = best;
  static std::atomic<uint64_t> allowed{0};
  constexpr int smem = WARPS * S::SLOTS * 512;
  const cudaError_t e = allow_smem((const void*)few_kernel<T, R, ROWS, W, ALIGNED>, smem, &allowed);
  if (e != cudaSuccess) return e;
  const int64_t ctas = std::min<int64_t>(SMS * S::CTAS, (groups * best + WARPS - 1) / WARPS);
  return launch_dependent(few_kernel<T, R, ROWS, W, ALIGNED>, dim3((unsigned)ctas, passes), 32 * WARPS, smem, 1, st, a);
}

// Of 3 or 4 tokens' f32 hidden values a warp reads as many bytes as of 4 rows of bf16: 2 rows of the weight against them take 84 us
// (4096 x 12288), 4 rows 72.
template <typename T, int W, bool ALIGNED>
cudaError_t launch_tokens(const FewArgs& a, cudaStream_t st) {
  if (a.tokens == 1) return launch_rows<T, 1, 1, W, ALIGNED>(a, st);
  if (a.tokens == 2) return launch_rows<T, 2, 2, W, ALIGNED>(a, st);
  if (a.tokens <= 4) return launch_rows<T, 4, W == 1 && sizeof(T) == 2 ? 4 : 2, W, ALIGNED>(a, st);
  if constexpr (sizeof(T) == 4) return launch_rows<T, 8, 2, W, ALIGNED>(a, st);   // 8 at a time
  return cudaErrorInvalidValue;
}
template <typename T, int W>
cudaError_t launch_tokens(const FewArgs& a, bool aligned, cudaStream_t st) {
  return aligned ? launch_tokens<T, W, true>(a, st) : launch_tokens<T, W, false>(a, st);
}

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

template <typename T>
bool aligned16(const void* p, int64_t stride, int64_t rows) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || stride * sizeof(T) % 16 == 0);
}

// Whether x, the rows of w_gate and w_up, and those of w_down start at 16 bytes, the weights' rows in whole pieces.
struct Starts {
  bool x, in, down;
};
template <typename T>
Starts starts_of(const ssd_gated_ff_params_t* p) {
  constexpr int N = Piece<T>::N;
  return {aligned16<T>(p->x, p->x_stride_row, p->tokens),
          p->dim % N == 0 && aligned16<T>(p->w_gate, p->w_gate_stride_row, p->hidden) && aligned16<T>(p->w_up, p->w_up_stride_row, p->hidden),
          p->hidden % N == 0 && aligned16<T>(p->w_down, p->w_down_stride_row, p->dim_out)};
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
  const Starts s = starts_of<T>(p);
  cudaError_t e = launch_tokens<T, 2>(a, s.x && s.in, st);
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
  return launch_tokens<T, 1>(a, s.down, st);
}

}  // namespace

// bf16: up to 4 tokens (2560 x 7680: 4 tokens 36 us, by the products 42; 8 tokens 63 and 42).  f32: up to 24, 8 to a pass, where the
// passes take less than the products, whose operands have to be split first.  Both in us, fitted to 768 x 2048, 4096 x 4096, 2560 x 7680 and
// 4096 x 12288 of 8 to 25 tokens.  Rows that start off 16 bytes are shifted into place in every pass, those of x once more for every row of a
// weight.  2560 x 7680, 8, 16 and 24 tokens: 79, 145, 209, by the products 252; w_down off 16 bytes 87, 164, 236; w_gate and w_up 111, 208,
// 273; x 185, 340, 492.
bool gated_ff_is_few(const ssd_gated_ff_params_t* p) {
  if (p->dtype == SSD_DTYPE_BF16) return p->tokens <= 4;
  if (p->tokens > 24) return false;
  const Starts s = starts_of<float>(p);
  const double size = (2e-6 / 3 * (double)p->dim + 1e-6 / 3 * (double)p->dim_out) * (double)p->hidden;   // millions of values of a weight
  const double pass = (3.3 + (s.down ? 0 : 0.6) + (!s.x ? 4.3 : !s.in ? 1.3 : 0)) * size + (s.x ? 6 : 9);
  return (double)((p->tokens + 7) / 8) * pass <= 45 + 10.4 * size;
}

size_t gated_ff_few_workspace(const ssd_gated_ff_params_t* p) { return 256 + up256((size_t)p->tokens * ((p->hidden + 7) / 8 * 8) * 4); }

cudaError_t launch_gated_ff_few(const ssd_gated_ff_params_t* p, void* workspace, cudaStream_t st, const char** at) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return p->dtype == SSD_DTYPE_BF16 ? launch_as<bf16>(p, ws, st, at) : launch_as<float>(p, ws, st, at);
}

}  // namespace ssd
