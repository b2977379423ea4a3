// Output projection and softmax cross entropy of a language model, in one operator that never
// holds the logits of a whole batch, and its gradients.
//
//   s_tv = x_t . w_v;  lse_t = log sum_v exp(s_tv);  loss_t = lse_t - s_{t,y_t}
//   dl_tv = c_t (exp(s_tv - lse_t) - [v = y_t]);  dX = dl W;  dW = dl^T X
//
// The work is three products of 2 T V D operations, so it is bound by the tensor pipe; what
// lies between them is made small:
//   loss       the GEMM's epilogue keeps, per row and 128 columns, the running maximum and the
//              sum of exponentials of the accumulator in TMEM: no logit leaves the SM but the
//              target's.  The sums leave the target out, so that a token predicted with
//              confidence keeps the digits of 1 - p, which a sum with p in it would lose.
//   gradients  tokens go in chunks whose logits fit a bounded workspace.  The same epilogue also
//              stores the f32 logits; a row pass forms lse and dl (rounded once, to bf16, for
//              the tensor pipe); two GEMMs follow.  Keeping f32 logits for the chunk costs 10
//              bytes of HBM per logit; computing them again would cost 2 D operations, more
//              from D = 512 on.
// f32 inputs are split into two bf16 planes, three products per pair (tc_gemm.cuh).
#include <algorithm>

#include "common.cuh"
#include "ssd_kernels.h"
#include "ssd_tc.h"
#include "tc_gemm.cuh"

namespace ssd {
namespace {

using gemm::BM;
using gemm::BN;

#ifndef CE_PAIR
#define CE_PAIR 1
#endif
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;
constexpr int64_t LOSS_CHUNK = 16384;              // tokens whose statistics are kept at a time
constexpr int64_t GRAD_BYTES = int64_t(3) << 30;   // logits and dl of a chunk of tokens

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// ---------------------------------------------------------------------------
// the tokens that count
// ---------------------------------------------------------------------------
__device__ __forceinline__ int64_t target_at(const void* y, int is64, int64_t t) {
  return is64 ? __ldg(static_cast<const long long*>(y) + t) : (int64_t)__ldg(static_cast<const int*>(y) + t);
}

// Tokens whose target is not ignore_index, in order.  Everything behind works on these rows
// alone: an ignored token costs no products, and what its row of hidden holds (padding, NaN)
// cannot reach the others' gradients through a product with zero.
struct Selected {
  int* count;              // one value
  int* index;              // (tokens): row r is token index[r]
  int* target;             // (tokens): its target, or -1 where that is outside [0, vocab)
  float* alpha;            // the factor common to all rows: 1 or 1 / count, times a scalar grad_loss
};

// One CTA; each thread owns a run of tokens: count, one scan over the threads, write.
__global__ void __launch_bounds__(1024) select_kernel(const void* targets, int is64, int64_t n, int64_t vocab,
                                                      int64_t ignore, int mean, const float* grad_loss, Selected s,
                                                      float* loss, float* lse) {
  __shared__ int sh[32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t per = (n + 1023) / 1024, lo = min(tid * per, n), hi = min(lo + per, n);
  int mine = 0;
  for (int64_t t = lo; t < hi; ++t) mine += target_at(targets, is64, t) != ignore;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh[w] = incl;
  __syncthreads();
  int at = incl - mine, total = 0;
  for (int i = 0; i < 32; ++i) {
    at += i < w ? sh[i] : 0;
    total += sh[i];
  }
  for (int64_t t = lo; t < hi; ++t) {
    const int64_t y = target_at(targets, is64, t);
    if (y == ignore) {
      loss[t] = 0.f;
      if (lse) lse[t] = 0.f;
      continue;
    }
    s.index[at] = (int)t;
    s.target[at++] = y >= 0 && y < vocab ? (int)y : -1;
  }
  if (tid == 0) {
    *s.count = total;
    *s.alpha = (mean ? (float)(1.0 / (double)max(total, 1)) : 1.f) * (grad_loss ? *grad_loss : 1.f);
  }
}

// ---------------------------------------------------------------------------
// operands: bf16 rows whose stride is a multiple of 16 bytes
// ---------------------------------------------------------------------------
__device__ __forceinline__ void split_store(float v, bf16* hi, bf16* lo, int64_t i) {
  const bf16 h = __float2bfloat16_rn(v);
  hi[i] = h;
  // an infinite value has no rest; v - hi would make it NaN
  if (lo) lo[i] = isinf(v) ? __float2bfloat16_rn(0.f) : __float2bfloat16_rn(v - __bfloat162float(h));
}

// Planes of a whole matrix (the weight, where the tensor maps cannot read it as it is).
template <typename T>
__global__ void __launch_bounds__(256) planes_kernel(const T* src, int64_t stride, int64_t rows, int64_t dim,
                                                     int64_t ld, bf16* hi, bf16* lo) {
  const int64_t n = rows * ld;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / ld, c = i - r * ld;
    split_store(c < dim ? ldg(src + r * stride + c) : 0.f, hi, lo, i);
  }
}

// Rows of hidden that count, side by side; zero rows up to the next 64 (a K block of the
// weight's gradient).  blockIdx.y = 1: zero rows of grad_hidden for the ignored tokens.
template <typename T>
__global__ void __launch_bounds__(256) gather_kernel(const T* src, int64_t stride, int64_t tokens, int64_t dim, int64_t ld,
                                                     Selected s, const void* targets, int is64, int64_t ignore, bf16* hi,
                                                     bf16* lo, T* grad_hidden) {
  const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= tokens) return;
  if (blockIdx.y == 1) {
    if (target_at(targets, is64, r) == ignore)
      for (int64_t c = lane; c < dim; c += 32) st(grad_hidden + r * dim + c, 0.f);
    return;
  }
  const int64_t count = *s.count;
  if (r >= (count + 63) / 64 * 64) return;
  const T* x = src + (r < count ? s.index[r] : 0) * stride;
  for (int64_t c = lane; c < ld; c += 32) split_store(r < count && c < dim ? ldg(x + c) : 0.f, hi, lo, r * ld + c);
}

// A matrix as the GEMMs read it.
struct Operand {
  const void* plane[2];
  int64_t rows, dim, ld;   // ld in bf16 values
};

bool direct(const void* p, int64_t stride, int dtype) {
  return dtype == SSD_DTYPE_BF16 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0;
}

// Where the planes of an operand go.
void place_planes(Operand* o, int dtype, uint8_t* mem) {
  o->ld = (o->dim + 7) / 8 * 8;
  o->plane[0] = mem;
  o->plane[1] = dtype == SSD_DTYPE_F32 ? mem + up256((size_t)o->rows * o->ld * 2) : nullptr;
}

cudaError_t make_planes(const void* src, int dtype, int64_t stride, Operand* o, uint8_t* mem, cudaStream_t st) {
  place_planes(o, dtype, mem);
  bf16* hi = static_cast<bf16*>(const_cast<void*>(o->plane[0]));
  bf16* lo = static_cast<bf16*>(const_cast<void*>(o->plane[1]));
  const int64_t n = o->rows * o->ld;
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 8 * 4);
  if (dtype == SSD_DTYPE_F32)
    planes_kernel<float><<<grid, 256, 0, st>>>(static_cast<const float*>(src), stride, o->rows, o->dim, o->ld, hi, lo);
  else
    planes_kernel<bf16><<<grid, 256, 0, st>>>(static_cast<const bf16*>(src), stride, o->rows, o->dim, o->ld, hi, lo);
  return cudaGetLastError();
}

size_t planes_bytes(int64_t rows, int64_t dim, int dtype) {
  return (dtype == SSD_DTYPE_F32 ? 2 : 1) * up256((size_t)rows * ((dim + 7) / 8 * 8) * 2);
}

// ---------------------------------------------------------------------------
// logits and their row statistics
// ---------------------------------------------------------------------------
struct LogitArgs {
  int64_t vocab;
  const int* target;       // of this chunk's rows
  int ns;                  // statistics per row: one for each 128 columns
  float2* stats;           // (rows, ns), target left out: maximum * log2(e), sum of 2^(s log2(e) - that)
  float* picked;           // (rows): the target's logit
  float* logits;           // (rows, ld) or NULL
  int64_t ld;
};

template <int CG>
__global__ void __launch_bounds__(gemm::THREADS, 1) logits_kernel(const __grid_constant__ gemm::Problem p,
                                                                  const __grid_constant__ LogitArgs a) {
  extern __shared__ uint8_t smem[];
  __shared__ gemm::Ctl ctl;
  const int lane = threadIdx.x & 31;
  gemm::run<CG, false, false>(p, smem, &ctl, [&](const gemm::Tile& t, uint32_t acc, int quad, int half, int m0, int live) {
    const int64_t row = m0 + 32 * quad + lane;
    const int64_t n0 = (int64_t)t.n * BN + half * 128;
    const int64_t y = row < live ? a.target[row] : -1;
    float m2 = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int ch = 0; ch < 4; ++ch) {
      const int64_t c0 = n0 + 32 * ch;
      if (c0 >= a.vocab) break;
      float v[32];
      ptx::tmem_ld32(acc + half * 128 + 32 * ch, v);
      ptx::tmem_ld_wait();
      if (c0 + 32 > a.vocab) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = c0 + i < a.vocab ? v[i] : -INFINITY;
      }
      if (a.logits && row < live) {
        float4* o = reinterpret_cast<float4*>(a.logits + row * a.ld + c0);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
      if (y >= c0 && y < c0 + 32) {   // the target's logit is kept out of the sum
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s = y == c0 + i ? v[i] : s;
          v[i] = y == c0 + i ? -INFINITY : v[i];
        }
        a.picked[row] = s;
      }
      float top = v[0];
#pragma unroll
      for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
      // the anchor is the rounded product itself, so that what is stored says what was summed
      const float n2 = fmaxf(m2, top * LOG2E), at = n2 == -INFINITY ? 0.f : n2;
      float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 32; ++i) e[i & 3] += exp2f(fmaf(v[i], LOG2E, -at));
      l = l * exp2f(m2 - at) + ((e[0] + e[1]) + (e[2] + e[3]));
      m2 = n2;
    }
    if (row < live) a.stats[row * a.ns + 2 * t.n + half] = make_float2(m2, l);
  });
}

// A row's results from its statistics, by one warp; the few values behind the sum in f64.
struct RowResult {
  float loss, lse;
  float pm1;               // p - 1 of the target
  float top, inv;          // p of another column: inv * 2^(s log2(e) - top)
};

__device__ __forceinline__ RowResult warp_row(const float2* stats, int ns, const float* picked, int target) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int i = lane; i < ns; i += 32) top = fmaxf(top, stats[i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;
  double others = 0;
  for (int i = lane; i < ns; i += 32) {
    const float2 s = stats[i];
    others += (double)(s.y * exp2f(s.x - top));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) others += __shfl_xor_sync(0xffffffffu, others, o);
  const double anchor = LN2 * (double)top;
  RowResult r;
  r.top = top;
  if (target < 0) {        // an invalid target: its loss is NaN, and so is its gradient
    r.loss = r.pm1 = r.inv = NAN;
    r.lse = (float)(anchor + log(others));
    return r;
  }
  const double s = (double)*picked, d = anchor - s;
  // others / e^s: the odds against the target
  const double odds = others == 0.0 ? 0.0 : others * exp(d);
  const bool far = d > 600.0;
  double loss = far ? log(others) + d : log1p(odds);
  if (!(s < INFINITY)) loss = NAN;   // an infinite or NaN logit, as the formula has it
  r.loss = (float)loss;
  r.lse = (float)(loss + s);
  r.pm1 = (float)(!(s < INFINITY) ? NAN : far ? -1.0 : -odds / (1.0 + odds));
  r.inv = (float)(1.0 / (others + exp(-d)));
  return r;
}

__global__ void __launch_bounds__(256) loss_kernel(const float2* stats, int ns, const float* picked, Selected s, int from,
                                                   int rows, float* loss, float* lse) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows || from + row >= *s.count) return;
  const RowResult r = warp_row(stats + row * ns, ns, picked + row, s.target[from + row]);
  if ((threadIdx.x & 31) == 0) {
    const int t = s.index[from + row];
    loss[t] = r.loss;
    if (lse) lse[t] = r.lse;
  }
}

// One CTA: sum (or mean over the tokens that count) of the tokens' losses, in a fixed order.
__global__ void __launch_bounds__(1024) reduce_kernel(const float* rows, int64_t n, const int* count, int mean, float* out) {
  __shared__ double sh[32];
  double s = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += (double)rows[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 32; ++i) s += sh[i];
  *out = (float)(mean ? s / (double)max(*count, 1) : s);
}

// ---------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------
// The factor alpha common to all rows is applied in f32 in the GEMMs' epilogues: folded into
// dl, the rounding of dl's largest entries (all near -alpha) would be one common error.
struct RowArgs {
  int64_t vocab, ld;
  Selected sel;
  int from, ns;            // first of the rows that count, of this chunk
  const float2* stats;
  const float* picked;
  const float* logits;
  const float* weight;     // per-token factor or NULL
  bf16* dl[2];             // (rows, ld); [1] for f32 inputs only
  float* loss;             // (tokens)
  float* lse;              // (tokens) or NULL
};

constexpr int ROW_THREADS = 512;

// One CTA per row that counts: lse and loss, then dl over the row.  Zero rows up to the next 64.
template <bool SPLIT>
__global__ void __launch_bounds__(ROW_THREADS) row_kernel(const RowArgs a) {
  __shared__ float sh_at, sh_inv, sh_y;
  const int64_t row = blockIdx.x;
  const int64_t live = (int64_t)*a.sel.count - a.from;
  if (live <= 0 || row >= (live + 63) / 64 * 64) return;
  const bool counted = row < live;
  const int y = counted ? a.sel.target[a.from + row] : -1;
  if (threadIdx.x < 32 && counted) {
    const RowResult r = warp_row(a.stats + row * a.ns, a.ns, a.picked + row, y);
    if (threadIdx.x == 0) {
      const int token = a.sel.index[a.from + row];
      const float w = a.weight ? a.weight[token] : 1.f;
      sh_at = r.top;
      sh_inv = w * r.inv;
      sh_y = w * r.pm1;
      a.loss[token] = r.loss;
      if (a.lse) a.lse[token] = r.lse;
    }
  }
  __syncthreads();
  const float at = counted ? sh_at : 0.f, f = counted ? sh_inv : 0.f, at_y = counted ? sh_y : 0.f;
  const float* s = a.logits + row * a.ld;
  bf16* hi = a.dl[0] + row * a.ld;
  bf16* lo = SPLIT ? a.dl[1] + row * a.ld : nullptr;
  for (int64_t c = threadIdx.x * 4; c < a.vocab; c += ROW_THREADS * 4) {
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    if (counted) {
      const float4 v = *reinterpret_cast<const float4*>(s + c);
      d[0] = f * exp2f(fmaf(v.x, LOG2E, -at));
      d[1] = f * exp2f(fmaf(v.y, LOG2E, -at));
      d[2] = f * exp2f(fmaf(v.z, LOG2E, -at));
      d[3] = f * exp2f(fmaf(v.w, LOG2E, -at));
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k == y) d[k] = at_y;
    }
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(d[0], d[1]), __floats2bfloat162_rn(d[2], d[3])};
    *reinterpret_cast<uint2*>(hi + c) = *reinterpret_cast<uint2*>(h);
    if constexpr (SPLIT) {
      const float2 g0 = __bfloat1622float2(h[0]), g1 = __bfloat1622float2(h[1]);
      __nv_bfloat162 l[2] = {__floats2bfloat162_rn(d[0] - g0.x, d[1] - g0.y), __floats2bfloat162_rn(d[2] - g1.x, d[3] - g1.y)};
      *reinterpret_cast<uint2*>(lo + c) = *reinterpret_cast<uint2*>(l);
    }
  }
}

// Epilogue of the gradients' GEMMs.
struct OutArgs {
  int64_t rows, cols;
  const int* index;        // row r of the result goes to row index[r] of out (NULL: to row r)
  void* out;               // (rows, cols), the result times alpha; NULL: into `part` only
  int out_bf16;
  const float* alpha;
  float* part;             // f32: parts of a split K range (splits, rows, cols), or the running sum
  int add_part;            // add what `part` holds (the running sum over token chunks)
};

__device__ __forceinline__ void put32(const OutArgs& a, int64_t row, int64_t c0, float (&v)[32], float alpha) {
  const int64_t at = row * a.cols + c0;
  if (a.out_bf16) {
    bf16* o = static_cast<bf16*>(a.out) + at;
    if (c0 + 32 <= a.cols && reinterpret_cast<uintptr_t>(o) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * i + 2 * k] * alpha, v[8 * i + 2 * k + 1] * alpha);
          u[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
        reinterpret_cast<uint4*>(o)[i] = make_uint4(u[0], u[1], u[2], u[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (c0 + i < a.cols) o[i] = __float2bfloat16_rn(v[i] * alpha);
    }
  } else {
    float* o = static_cast<float*>(a.out) + at;
    if (c0 + 32 <= a.cols && reinterpret_cast<uintptr_t>(o) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<float4*>(o)[i] = make_float4(v[4 * i] * alpha, v[4 * i + 1] * alpha, v[4 * i + 2] * alpha, v[4 * i + 3] * alpha);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (c0 + i < a.cols) o[i] = v[i] * alpha;
    }
  }
}

template <int CG, bool A_MN>
__global__ void __launch_bounds__(gemm::THREADS, 1) grad_gemm_kernel(const __grid_constant__ gemm::Problem p,
                                                                     const __grid_constant__ OutArgs a) {
  extern __shared__ uint8_t smem[];
  __shared__ gemm::Ctl ctl;
  const int lane = threadIdx.x & 31;
  const float alpha = a.out ? *a.alpha : 1.f;
  gemm::run<CG, A_MN, true>(p, smem, &ctl, [&](const gemm::Tile& t, uint32_t acc, int quad, int half, int m0, int live) {
    const int64_t row = m0 + 32 * quad + lane;
    const int64_t n0 = (int64_t)t.n * BN + half * 128;
    const int64_t rows = p.limit_k ? a.rows : live;
    const int64_t to = a.index && row < rows ? a.index[row] : row;
#pragma unroll 1
    for (int ch = 0; ch < 4; ++ch) {
      const int64_t c0 = n0 + 32 * ch;
      if (c0 >= a.cols) break;
      float v[32];
      ptx::tmem_ld32(acc + half * 128 + 32 * ch, v);
      ptx::tmem_ld_wait();
      if (row >= rows) continue;
      if (t.k0 == t.k1) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
      }
      if (a.part) {
        float* q = a.part + ((int64_t)t.split * a.rows + row) * a.cols + c0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (c0 + i < a.cols) {
            if (a.add_part) v[i] += q[i];
            if (!a.out) q[i] = v[i];
          }
        }
      }
      if (a.out) put32(a, to, c0, v, alpha);
    }
  });
}

// Sum of the parts of a split K range, in order, times alpha.  One CTA row per row that counts.
template <typename TO>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int splits, int64_t rows, int64_t cols, Selected s,
                                                   int from, TO* out) {
  const int64_t row = blockIdx.x;
  if (from + row >= *s.count) return;
  const float f = *s.alpha;
  TO* o = out + (int64_t)s.index[from + row] * cols;
  for (int64_t c = threadIdx.x; c < cols; c += 256) {
    float v = 0.f;
    for (int j = 0; j < splits; ++j) v += part[(j * rows + row) * cols + c];
    st(o + c, v * f);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

template <int CG, typename Kernel, typename Args>
cudaError_t launch_gemm(Kernel kernel, const gemm::Problem& p, const Args& a, cudaStream_t st) {
  constexpr int smem = gemm::Shape<CG>::SMEM;
  cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)p.m_tiles * p.n_tiles * p.splits;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(CG * std::min<int64_t>(units, sm_count() / CG)));
  cfg.blockDim = dim3(gemm::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  if (CG > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, p, a);
}

// Maps of an operand's planes.  K-major: 64 values of the reduced dimension x `box` rows.
// MN-major: 64 values of the other dimension x 64 rows of the reduced one.
bool maps(CUtensorMap (&m)[2], const Operand& o, int planes, uint32_t box) {
  for (int i = 0; i < planes; ++i)
    if (!tc_map_2d(&m[i], o.plane[i], (uint64_t)o.dim, (uint64_t)o.rows, (uint64_t)o.ld * 2, box)) return false;
  return true;
}

int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

struct Plan {
  bool grad;
  int planes;
  int64_t chunk, nchunks, ns, ld;   // tokens of a chunk; statistics per row; logits' row length
  int splits;                       // of the reduction over the vocabulary (dX)
  bool pack_w, sum_w;       // sum_w: dW's running sum over chunks needs its own f32 buffer
  size_t one, index, target, rows, picked, stats, x, w, logits, dl[2], part, wsum, total;
};

int split_k(int64_t rows, int64_t dim, int64_t vocab) {
  // enough units of work to fill the GPU: the split whose last wave wastes least, no part
  // shorter than 32 K blocks
  const int64_t tiles = (int64_t)cdiv(rows, 2 * BM) * cdiv(dim, BN), sms = 74;
  const int most = (int)std::min<int64_t>(16, std::max<int64_t>(1, vocab / (32 * 64)));
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= most; ++s) {
    const double c = (double)cdiv(tiles * s, sms) / s * (1.0 + 0.01 * s);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
}

Plan plan_of(const ssd_linear_ce_params_t* p) {
  Plan q{};
  q.grad = p->grad_hidden || p->grad_weight;
  q.planes = p->dtype == SSD_DTYPE_F32 ? 2 : 1;
  q.ns = 2 * (int64_t)cdiv(p->vocab, BN);
  q.ld = (p->vocab + 63) / 64 * 64;
  if (q.grad) {
    const int64_t per = q.ld * (4 + 2 * q.planes);
    const int64_t most = std::max<int64_t>(128, GRAD_BYTES / per / 128 * 128);
    q.nchunks = cdiv(p->tokens, most);
    q.chunk = std::min<int64_t>(p->tokens, (cdiv(p->tokens, q.nchunks) + 127) / 128 * 128);
  } else {
    q.chunk = std::min<int64_t>(p->tokens, LOSS_CHUNK);
  }
  q.nchunks = cdiv(p->tokens, q.chunk);
  q.pack_w = !direct(p->weight, p->weight_stride_row, p->dtype);
  q.splits = p->grad_hidden ? split_k(q.chunk, p->dim, p->vocab) : 1;
  q.sum_w = p->grad_weight && q.nchunks > 1;
  size_t at = 256;   // the status word
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  q.one = take(8);
  q.index = take((size_t)p->tokens * 4);
  q.target = take((size_t)p->tokens * 4);
  q.rows = take(p->reduction == SSD_REDUCE_NONE ? 0 : (size_t)p->tokens * 4);
  q.picked = take((size_t)q.chunk * 4);
  q.stats = take((size_t)q.chunk * q.ns * 8);
  q.x = take(planes_bytes(p->tokens, p->dim, p->dtype));
  q.w = take(q.pack_w ? planes_bytes(p->vocab, p->dim, p->dtype) : 0);
  if (q.grad) {
    q.logits = take((size_t)q.chunk * q.ld * 4);
    for (int i = 0; i < q.planes; ++i) q.dl[i] = take((size_t)q.chunk * q.ld * 2);
    q.part = take(q.splits > 1 ? (size_t)q.splits * q.chunk * p->dim * 4 : 0);
    q.wsum = take(q.sum_w ? (size_t)p->vocab * p->dim * 4 : 0);
  }
  q.total = at;
  return q;
}

#define CE_CHECK(call, where)                                     \
  do {                                                            \
    const cudaError_t e_ = (call);                                \
    if (e_ != cudaSuccess) {                                      \
      *at = where;                                                \
      return e_;                                                  \
    }                                                             \
  } while (0)

template <int CG>
cudaError_t logits_gemm(const Operand& x, const Operand& w, int planes, const LogitArgs& a, const int* count, int from,
                        unsigned* status, cudaStream_t st) {
  gemm::Problem g{};
  g.limit = count;
  g.limit_from = from;
  g.rows = (int)x.rows;
  if (!maps(g.a, x, planes, BM) || !maps(g.b, w, planes, BN / CG)) return cudaErrorInvalidValue;
  g.m_tiles = cdiv(x.rows, BM * CG);
  g.n_tiles = cdiv(a.vocab, BN);
  g.splits = 1;
  g.k_blocks = cdiv(x.dim, gemm::BK);
  g.passes = planes == 2 ? 3 : 1;
  g.m_fastest = 1;
  g.status = status;
  return launch_gemm<CG>(logits_kernel<CG>, g, a, st);
}

template <int CG, bool A_MN>
cudaError_t grad_gemm(const Operand& a, const Operand& b, int64_t k, int planes, int splits, const OutArgs& o,
                      const int* count, int from, unsigned* status, cudaStream_t st) {
  gemm::Problem g{};
  g.limit = count;
  g.limit_from = from;
  g.rows = (int)a.rows;    // dl's rows: the result's for dX, the reduced ones for dW
  g.limit_k = A_MN;
  if (!maps(g.a, a, planes, A_MN ? 64 : BM) || !maps(g.b, b, planes, 64)) return cudaErrorInvalidValue;
  g.m_tiles = cdiv(o.rows, BM * CG);
  g.n_tiles = cdiv(o.cols, BN);
  g.splits = splits;
  g.k_blocks = cdiv(k, gemm::BK);
  g.passes = planes == 2 ? 3 : 1;
  g.m_fastest = 0;
  g.status = status;
  return launch_gemm<CG>(grad_gemm_kernel<CG, A_MN>, g, o, st);
}

}  // namespace

size_t linear_ce_workspace(const ssd_linear_ce_params_t* p) { return plan_of(p).total; }

cudaError_t launch_linear_ce(const ssd_linear_ce_params_t* p, void* workspace, cudaStream_t st, const char** at) {
  const Plan q = plan_of(p);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  unsigned* status = reinterpret_cast<unsigned*>(ws);
  CE_CHECK(cudaMemsetAsync(status, 0, 4, st), "status");
  Selected sel;
  sel.count = reinterpret_cast<int*>(ws + q.one);
  sel.alpha = reinterpret_cast<float*>(ws + q.one) + 1;
  sel.index = reinterpret_cast<int*>(ws + q.index);
  sel.target = reinterpret_cast<int*>(ws + q.target);
  float* rows = p->reduction == SSD_REDUCE_NONE ? p->loss : reinterpret_cast<float*>(ws + q.rows);
  const bool bf = p->dtype == SSD_DTYPE_BF16, mean = p->reduction == SSD_REDUCE_MEAN;
  const bool per_row = p->reduction == SSD_REDUCE_NONE && p->grad_loss;
  select_kernel<<<1, 1024, 0, st>>>(p->targets, p->targets_int64, p->tokens, p->vocab, p->ignore_index, mean,
                                    per_row ? nullptr : p->grad_loss, sel, rows, p->lse);
  CE_CHECK(cudaGetLastError(), "select");
  Operand x{}, w{};
  x.rows = p->tokens; x.dim = p->dim;
  place_planes(&x, p->dtype, ws + q.x);
  const dim3 grid((unsigned)cdiv(p->tokens, 8), p->grad_hidden ? 2 : 1);
  bf16* hi = static_cast<bf16*>(const_cast<void*>(x.plane[0]));
  bf16* lo = static_cast<bf16*>(const_cast<void*>(x.plane[1]));
  if (bf)
    gather_kernel<bf16><<<grid, 256, 0, st>>>(static_cast<const bf16*>(p->hidden), p->hidden_stride_row, p->tokens, p->dim,
                                              x.ld, sel, p->targets, p->targets_int64, p->ignore_index, hi, lo,
                                              static_cast<bf16*>(p->grad_hidden));
  else
    gather_kernel<float><<<grid, 256, 0, st>>>(static_cast<const float*>(p->hidden), p->hidden_stride_row, p->tokens,
                                               p->dim, x.ld, sel, p->targets, p->targets_int64, p->ignore_index, hi, lo,
                                               static_cast<float*>(p->grad_hidden));
  CE_CHECK(cudaGetLastError(), "gather");
  w.rows = p->vocab; w.dim = p->dim; w.ld = p->weight_stride_row; w.plane[0] = p->weight;
  if (q.pack_w) CE_CHECK(make_planes(p->weight, p->dtype, p->weight_stride_row, &w, ws + q.w, st), "weight planes");
  for (int64_t c = 0; c < q.nchunks; ++c) {
    const int64_t t0 = c * q.chunk, n = std::min(q.chunk, p->tokens - t0);
    const int from = (int)t0;
    Operand xc = x;
    xc.rows = n;
    for (int i = 0; i < 2; ++i)
      if (xc.plane[i]) xc.plane[i] = static_cast<const char*>(xc.plane[i]) + t0 * x.ld * 2;
    LogitArgs a{};
    a.vocab = p->vocab; a.target = sel.target + t0; a.ns = (int)q.ns;
    a.stats = reinterpret_cast<float2*>(ws + q.stats);
    a.picked = reinterpret_cast<float*>(ws + q.picked);
    a.logits = q.grad ? reinterpret_cast<float*>(ws + q.logits) : nullptr;
    a.ld = q.ld;
    if (n > BM) CE_CHECK(logits_gemm<CE_PAIR>(xc, w, q.planes, a, sel.count, from, status, st), "logits");
    else CE_CHECK(logits_gemm<1>(xc, w, q.planes, a, sel.count, from, status, st), "logits");
    if (!q.grad) {
      loss_kernel<<<(unsigned)cdiv(n, 8), 256, 0, st>>>(a.stats, a.ns, a.picked, sel, from, (int)n, rows, p->lse);
      CE_CHECK(cudaGetLastError(), "loss");
      continue;
    }
    RowArgs r{};
    r.vocab = p->vocab; r.ld = q.ld; r.sel = sel; r.from = from;
    r.ns = a.ns; r.stats = a.stats; r.picked = a.picked; r.logits = a.logits;
    r.weight = per_row ? p->grad_loss : nullptr;
    for (int i = 0; i < q.planes; ++i) r.dl[i] = reinterpret_cast<bf16*>(ws + q.dl[i]);
    r.loss = rows; r.lse = p->lse;
    if (q.planes == 2) row_kernel<true><<<(unsigned)n, ROW_THREADS, 0, st>>>(r);
    else row_kernel<false><<<(unsigned)n, ROW_THREADS, 0, st>>>(r);
    CE_CHECK(cudaGetLastError(), "rows");
    Operand dl{};
    dl.rows = n; dl.dim = p->vocab; dl.ld = q.ld;
    for (int i = 0; i < q.planes; ++i) dl.plane[i] = r.dl[i];
    if (p->grad_hidden) {
      OutArgs o{};
      o.rows = n; o.cols = p->dim; o.alpha = sel.alpha; o.out_bf16 = bf; o.index = sel.index + t0;
      if (q.splits > 1) o.part = reinterpret_cast<float*>(ws + q.part);
      else o.out = p->grad_hidden;
      if (n > BM) CE_CHECK((grad_gemm<CE_PAIR, false>(dl, w, p->vocab, q.planes, q.splits, o, sel.count, from, status, st)), "grad_hidden");
      else CE_CHECK((grad_gemm<1, false>(dl, w, p->vocab, q.planes, q.splits, o, sel.count, from, status, st)), "grad_hidden");
      if (q.splits > 1) {
        if (bf)
          join_kernel<bf16><<<(unsigned)n, 256, 0, st>>>(o.part, q.splits, n, p->dim, sel, from, static_cast<bf16*>(p->grad_hidden));
        else
          join_kernel<float><<<(unsigned)n, 256, 0, st>>>(o.part, q.splits, n, p->dim, sel, from, static_cast<float*>(p->grad_hidden));
        CE_CHECK(cudaGetLastError(), "grad_hidden join");
      }
    }
    if (p->grad_weight) {
      OutArgs o{};
      o.rows = p->vocab; o.cols = p->dim; o.alpha = sel.alpha; o.out_bf16 = p->grad_weight_dtype == SSD_DTYPE_BF16;
      if (q.sum_w) o.part = reinterpret_cast<float*>(ws + q.wsum);
      o.add_part = c > 0;
      o.out = c == q.nchunks - 1 ? p->grad_weight : nullptr;
      if (p->vocab > BM) CE_CHECK((grad_gemm<CE_PAIR, true>(dl, xc, n, q.planes, 1, o, sel.count, from, status, st)), "grad_weight");
      else CE_CHECK((grad_gemm<1, true>(dl, xc, n, q.planes, 1, o, sel.count, from, status, st)), "grad_weight");
    }
  }
  if (p->reduction != SSD_REDUCE_NONE) {
    reduce_kernel<<<1, 1024, 0, st>>>(rows, p->tokens, sel.count, mean, p->loss);
    CE_CHECK(cudaGetLastError(), "reduce");
  }
  return cudaSuccess;
}

}  // namespace ssd
