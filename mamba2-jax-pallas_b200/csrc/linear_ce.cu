// Output projection and softmax cross entropy of a language model, in one operator that never
// holds the logits of a whole batch, and its gradients.
//
//   s_tv = x_t . w_v;  lse_t = log sum_v exp(s_tv);  loss_t = lse_t - s_{t,y_t}
//   dl_tv = c_t (exp(s_tv - lse_t) - [v = y_t]);  dX = dl W;  dW = dl^T X
//
// The work is three products of 2 T V D operations, so it is bound by the tensor pipe; what
// lies between them is made small:
//   loss       the GEMM's epilogue keeps, per row and 64 columns, the running maximum and the
//              sum of exponentials of the accumulator in TMEM: no logit leaves the SM but the
//              target's.  The sums leave the target out, so that a token predicted with
//              confidence keeps the digits of 1 - p, which a sum with p in it would lose.
//   gradients  tokens go in chunks whose logits fit a bounded workspace.  The same epilogue also
//              stores the f32 logits; a row pass forms lse and dl (rounded once, to bf16, for
//              the tensor pipe; f32 inputs: two f16, in a pass for each product); two GEMMs follow.  Keeping
//              f32 logits for the chunk costs 10 bytes of HBM per logit; computing them again would cost 2 D
//              operations, more from D = 512 on.
// f32 inputs are split into two f16 planes, three products per pair (tc_gemm.cuh).
//
// Measured, kernels alone: loss of 4096 x 131072 x 4096, bf16, 2.79 ms (1.58 PFLOP/s; calls back to back,
// under the power limit, 3.10); gradients of 16384 x 50000 x 2560, bf16, 10.4 ms under the power limit (1.21
// PFLOP/s): logits 3.35, dX 3.00, dW 3.03, rows 0.75, parts 0.15, the rest 0.1 (calls 11.0; in a burst 9.5);
// gradients of 2048 x 50257 x 768, f32, 1.34 ms (1.06 PFLOP/s of f16 products): logits 0.39, dX 0.29, dW
// 0.31, the passes over the logits 0.26, planes 0.05, the rest 0.04.
#include <algorithm>

#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"
#include "linear_ce.cuh"
#include "ssd_kernels.h"
#include "ssd_tc.h"
#include "tc_gemm.cuh"

namespace ssd {
namespace {

using namespace ce;
using gemm::BM;
using gemm::BN;
constexpr int EC = gemm::EPI_COLS;

// K blocks summed in TMEM before the sum goes to registers (tc_gemm.cuh), measured over K = 4096:
// one segment 3.3e-6 off in the loss, 16 blocks 7.7e-7, 8 blocks 3.6e-7 at the same speed (4096 x
// 131072 in 2.67 and 2.69 ms).  f32 operands, with three products a block, take 2: gradients
// 7.6e-7 off (3 blocks 1.0e-6 and 3 % faster, 1 block 5.8e-7 and 3 % slower).
// The gradients of bf16 take 32: over 131072 words grad_hidden is 3.5e-6 too small by the adds (whole range 1.07e-4,
// a fifth of bf16's own rounding and all of one sign; 64 blocks 1.1e-5, 16 blocks 1.1e-6 and 0.6 % slower;
// 32 as fast as the whole range: 16384 x 50000 x 2560 in 11.7 ms back to back).
constexpr int SEGMENT_BF16 = 8, SEGMENT_F32 = 2, SEGMENT_GRAD = 32;
constexpr int64_t LOSS_CHUNK = 16384;              // tokens whose statistics are kept at a time
// logits and dl of a chunk of tokens (16384 x 50000 x 2560: chunks of 1 GiB 9.6 ms, 3 GiB 9.5, 6 GiB 9.6)
constexpr int64_t GRAD_BYTES = int64_t(3) << 30;

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// ---------------------------------------------------------------------------
// the tokens that count
// ---------------------------------------------------------------------------
// f32 inputs: a row of hidden or of the weight has a power of two that brings its largest finite
// magnitude (as the bits of a float, which order like it) to [2^14, 2^15): f16 ends at 65504, and two
// planes keep 22 bits down to 2^-1.  Rows have one each, so that a large row takes no digits from the
// others; the powers come out again in the logits' epilogue, and go into dl where a product runs over
// the rows.
__device__ __forceinline__ int shift_of(unsigned largest) {
  const int e = (int)(largest >> 23);                       // biased exponent; 0 also for subnormals
  return e == 0 ? 0 : min(127 + 14 - e, 126);
}
// 2^k; 0 below f32's normal numbers.
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((unsigned)min(max(k + 127, 0), 254) << 23); }
// Logits of f32 inputs stay times a power of two that belongs to their row until log2(e) multiplies them;
// 14 of the 28 that the two operands' powers have beyond their values, so that neither part leaves f32
// (a word or row below 2^-98 throughout counts as zero).
__device__ __forceinline__ float logit_scale(int x_shift) { return pow2(14 - x_shift); }
__device__ __forceinline__ float word_scale(int w_shift) { return pow2(-14 - w_shift); }
__device__ __forceinline__ unsigned finite_bits(float v) {
  const unsigned u = __float_as_uint(v) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// Tokens whose target is not ignore_index, in order.  Everything behind works on these rows
// alone: an ignored token costs no products, and what its row of hidden holds (padding, NaN)
// cannot reach the others' gradients through a product with zero.
struct Selected {
  int* count;              // one value
  int* index;              // (tokens): row r is token index[r]
  int* target;             // (tokens): its target, or -1 where that is outside [0, vocab)
  float* alpha;            // the factor common to all rows: 1 or 1 / count, times a scalar grad_loss
  unsigned* status;        // the workspace's status word
  int* ticket;
};

// One CTA; each warp owns a run of tokens and reads 32 at a time: count, one scan over the warps,
// then the same again to write.  Latency-bound: 6 us for 2048 tokens, 13 us for 16384.
__global__ void __launch_bounds__(1024) select_kernel(const void* targets, int is64, int64_t n, int64_t vocab,
                                                      int64_t ignore, int mean, const float* grad_loss,
                                                      Selected s, float* loss, float* lse) {
  __shared__ int sh[32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t per = (n + 1023) / 1024 * 32, lo = min(w * per, n), hi = min(lo + per, n);
  int mine = 0;
#pragma unroll 8
  for (int64_t t = lo + lane; t < hi; t += 32) mine += target_at(targets, is64, t) != ignore;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) sh[w] = mine;
  __syncthreads();
  int at = 0, total = 0;
  for (int i = 0; i < 32; ++i) {
    at += i < w ? sh[i] : 0;
    total += sh[i];
  }
#pragma unroll 4
  for (int64_t t0 = lo; t0 < hi; t0 += 32) {
    const int64_t t = t0 + lane;
    const int64_t y = t < hi ? target_at(targets, is64, t) : ignore;
    const unsigned b = __ballot_sync(0xffffffffu, t < hi && y != ignore);
    if (t < hi && y == ignore) {
      loss[t] = 0.f;
      if (lse) lse[t] = 0.f;
    } else if (t < hi) {
      const int r = at + __popc(b & ((1u << lane) - 1));
      s.index[r] = (int)t;
      s.target[r] = y >= 0 && y < vocab ? (int)y : -1;
    }
    at += __popc(b);
  }
  if (tid == 0) {
    *s.status = 0;
    *s.ticket = 0;
    *s.count = total;
    *s.alpha = (mean ? (float)(1.0 / (double)max(total, 1)) : 1.f) * (grad_loss ? *grad_loss : 1.f);
  }
}

// ---------------------------------------------------------------------------
// operands: 16-bit rows whose stride is a multiple of 16 bytes
// ---------------------------------------------------------------------------
// 8 values of a row from column c on (zeros past the end); one 16-byte load per 4 or 8 values
// where the row allows it.
__device__ __forceinline__ void load8(const float* row, int64_t c, int64_t dim, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= dim) {
    const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < dim ? row[c + k] : 0.f;
  }
}

// 8 values into the planes: bf16 values as they are; f32 values times the scale, as two f16.
__device__ __forceinline__ void planes8(const bf16* row, int64_t c, int64_t dim, bool vec, float, void* hi, void*, int64_t i) {
  uint4 q;
  if (vec && c + 8 <= dim) {
    q = *reinterpret_cast<const uint4*>(row + c);
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = c + 2 * k < dim ? h[c + 2 * k] : 0, b = c + 2 * k + 1 < dim ? h[c + 2 * k + 1] : 0;
      u[k] = a | b << 16;
    }
    q = make_uint4(u[0], u[1], u[2], u[3]);
  }
  *reinterpret_cast<uint4*>(static_cast<bf16*>(hi) + i) = q;
}
__device__ __forceinline__ void planes8(const float* row, int64_t c, int64_t dim, bool vec, float scale, void* hi, void* lo,
                                        int64_t i) {
  float v[8];
  load8(row, c, dim, vec, v);
  uint32_t h[4], l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = v[2 * k] * scale, b = v[2 * k + 1] * scale;
    const __half2 p = __floats2half2_rn(a, b);
    const float2 f = __half22float2(p);
    // an infinite value has no rest; v - hi would make it NaN
    const __half2 r = __floats2half2_rn(isinf(a) ? 0.f : a - f.x, isinf(b) ? 0.f : b - f.y);
    h[k] = *reinterpret_cast<const uint32_t*>(&p);
    l[k] = *reinterpret_cast<const uint32_t*>(&r);
  }
  *reinterpret_cast<uint4*>(static_cast<__half*>(hi) + i) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(static_cast<__half*>(lo) + i) = make_uint4(l[0], l[1], l[2], l[3]);
}

template <typename T>
__device__ __forceinline__ bool vec_rows(const T* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * sizeof(T) % 16 == 0;
}

// The lane's share of the largest finite magnitude of a row, for `lanes` lanes of which this is `lane`.
__device__ __forceinline__ unsigned largest_of(const float* row, int64_t dim, bool vec, int lane, int lanes) {
  unsigned m = 0;
#pragma unroll 4
  for (int64_t c = lane * 8; c < dim; c += lanes * 8) {
    float v[8];
    load8(row, c, dim, vec, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, finite_bits(v[k]));
  }
  return m;
}

// The weight where the tensor maps cannot read it as it is.  bf16: the same values, 256 columns of a row a
// warp at a time.
__global__ void __launch_bounds__(256) repack_kernel(const bf16* src, int64_t stride, int64_t rows, int64_t dim, int64_t ld,
                                                     void* out) {
  ptx::griddep_wait();
  const bool vec = vec_rows(src, stride);
  const int64_t runs = (ld + 255) / 256, n = rows * runs;
#pragma unroll 2
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < n; u += (int64_t)gridDim.x * 8) {
    const int64_t r = u / runs, c = (u - r * runs) * 256 + (threadIdx.x & 31) * 8;
    if (c < ld) planes8(src + r * stride, c, dim, vec, 1.f, out, nullptr, r * ld + c);
  }
}

// f32: two planes and a power of two per row, a warp per row, whose second reading comes from L1.
__global__ void __launch_bounds__(256) planes_kernel(const float* src, int64_t stride, int64_t rows, int64_t dim, int64_t ld,
                                                     void* hi, void* lo, float* shift, float* unscale) {
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31;
  const bool vec = vec_rows(src, stride);
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const float* row = src + r * stride;
    const int e = shift_of(__reduce_max_sync(0xffffffffu, largest_of(row, dim, vec, lane, 32)));
    if (lane == 0) {
      shift[r] = (float)e;
      unscale[r] = word_scale(e);
    }
    const float scale = pow2(e);
#pragma unroll 4
    for (int64_t c = lane * 8; c < ld; c += 256) planes8(row, c, dim, vec, scale, hi, lo, r * ld + c);
  }
}

// Rows of hidden that count, side by side; zero rows up to the next 64 (a K block of the
// weight's gradient).  f32: a power of two per row.  blockIdx.y = 1: zero rows of grad_hidden for the
// ignored tokens.  HBM-bound: bf16 16384 x 2560 35 us (4.8 TB/s).
template <typename T>
__global__ void __launch_bounds__(128) gather_kernel(const T* src, int64_t stride, int64_t dim, int64_t ld, Selected s,
                                                     const void* targets, int is64, int64_t ignore, void* hi, void* lo,
                                                     int* shift, T* grad_hidden) {
  ptx::griddep_wait();
  const int64_t r = blockIdx.x;
  if (blockIdx.y == 1) {
    if (target_at(targets, is64, r) == ignore)
      for (int64_t c = threadIdx.x; c < dim; c += 128) grad_hidden[r * dim + c] = T(0.f);
    return;
  }
  const int64_t count = *s.count;
  if (r >= (count + 63) / 64 * 64) return;
  const T* x = src + (r < count ? s.index[r] : 0) * stride;
  const bool vec = vec_rows(src, stride);
  float scale = 1.f;
  if constexpr (sizeof(T) == 4) {
    __shared__ unsigned sh[4];
    const unsigned m = __reduce_max_sync(0xffffffffu, largest_of(x, r < count ? dim : 0, vec, threadIdx.x, 128));
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
    const int e = shift_of(max(max(sh[0], sh[1]), max(sh[2], sh[3])));
    if (threadIdx.x == 0) shift[r] = e;
    scale = pow2(e);
  }
#pragma unroll 2
  for (int64_t c = threadIdx.x * 8; c < ld; c += 128 * 8)
    planes8(x, r < count ? c : dim, dim, vec, scale, hi, lo, r * ld + c);
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

size_t planes_bytes(int64_t rows, int64_t dim, int dtype) {
  return (dtype == SSD_DTYPE_F32 ? 2 : 1) * up256((size_t)rows * ((dim + 7) / 8 * 8) * 2);
}

// ---------------------------------------------------------------------------
// logits and their row statistics
// ---------------------------------------------------------------------------
struct LogitArgs {
  int64_t vocab;
  const int* target;       // of this chunk's rows
  int ns;                  // statistics per row: one for each 64 columns
  float2* stats;           // (rows, ns), target left out: maximum * log2(e), sum of 2^(s log2(e) - that)
  float* picked;           // (rows): the target's logit
  float* logits;           // (rows, ld) or NULL; f32 inputs: over logit_scale of their row
  int64_t ld;
  // f32 inputs: the rows' and the words' powers of two, the latter as numbers and as word_scale (readable up
  // to the tile's end), and with `peak` (rows, ns) the largest s log2(e) - w_shift of each 64 columns, the
  // target left out
  const int* x_shift;
  const float* w_shift;
  const float* w_scale;
  float* peak;
  CUtensorMap map;         // of the logits, 32 x 32 values a box (pairs)
};

// Four values from L1.  Volatile: a tile's 64 shifts, kept from one use to the next, would spill.
__device__ __forceinline__ float4 load_again(const float* p) {
  float4 q;
  asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(q.x), "=f"(q.y), "=f"(q.z), "=f"(q.w) : "l"(p));
  return q;
}

// Half a warp's 32 x 64 block to global memory: through its 4 KB of shared memory, in the layout
// of a swizzled box, by one bulk store (f32, 2048 x 50257 x 768, before operands had a power of two per
// row, which takes 40 us: 370 us where the warp stores values itself, 354 us so, 297 us without any store).
template <int HALF>
__device__ __forceinline__ void store_half(const CUtensorMap* map, uint4* stage, const float (&v)[EC], int n0, int row0) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) ptx::bulk_wait_read();   // the store before has left the shared memory
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float* x = v + 32 * HALF + 4 * i;
    stage[gemm::epi_at<2>(lane, i)] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  ptx::fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    ptx::tma_store_2d(map, stage, n0 + 32 * HALF, row0);
    ptx::bulk_commit();
  }
}

template <int CG, int PLANES>
__global__ void __launch_bounds__(gemm::THREADS, 1) logits_kernel(const __grid_constant__ gemm::Problem p,
                                                                  const __grid_constant__ LogitArgs a) {
  extern __shared__ uint8_t smem[];
  __shared__ gemm::Ctl ctl;
  gemm::run<CG, PLANES, false, false>(p, smem, &ctl, [] {}, [&](const gemm::Tile& t, float (&v)[EC], int row0, int n0, int live,
                                                       int, uint4* stage) {
    const int row = row0 + (threadIdx.x & 31);
    const int y = row < live ? a.target[row] : -1;
    float scale = 1.f;
    if constexpr (PLANES == 2) {
      if (row < live) scale = logit_scale(a.x_shift[row]);
#pragma unroll
      for (int i = 0; i < EC; i += 4) {
        const float4 q = load_again(a.w_scale + n0 + i);
        v[i] *= q.x; v[i + 1] *= q.y; v[i + 2] *= q.z; v[i + 3] *= q.w;
      }
    }
    const float to_log2 = PLANES == 2 ? LOG2E * scale : LOG2E;
    // the logits' rows are a multiple of 64 long
    if (CG == 2) {
      if (a.logits && row0 < live && n0 < a.vocab) {
        store_half<0>(&a.map, stage, v, n0, row0);
        store_half<1>(&a.map, stage, v, n0, row0);
      }
    } else if (a.logits) {
      float* o = a.logits + row0 * a.ld + n0;
      const int cols = (int)min((int64_t)EC, a.vocab - n0);
      gemm::by_rows<CG, float>(stage, v, true, live - row0, [&](int i, int c, uint4 q) {
        if (c < cols) *reinterpret_cast<uint4*>(o + i * a.ld + c) = q;
      }, [](int, int, float) {});
    }
    if (n0 + EC > a.vocab) {
#pragma unroll
      for (int i = 0; i < EC; ++i) v[i] = n0 + i < a.vocab ? v[i] : -INFINITY;
    }
    if (y >= n0 && y < n0 + EC) {   // the target's logit is kept out of the sum
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        s = y == n0 + i ? v[i] : s;
        v[i] = y == n0 + i ? -INFINITY : v[i];
      }
      a.picked[row] = PLANES == 2 ? s * scale : s;
    }
    if constexpr (PLANES == 2) {
      if (a.peak) {
        float k = -INFINITY;
#pragma unroll
        for (int i = 0; i < EC; i += 4) {
          const float4 q = load_again(a.w_shift + n0 + i);
          k = fmaxf(fmaxf(k, fmaf(v[i], to_log2, -q.x)), fmaf(v[i + 1], to_log2, -q.y));
          k = fmaxf(fmaxf(k, fmaf(v[i + 2], to_log2, -q.z)), fmaf(v[i + 3], to_log2, -q.w));
        }
        if (row < live) a.peak[(int64_t)row * a.ns + n0 / EC] = k;
      }
    }
    float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 4; i < EC; ++i) m[i & 3] = fmaxf(m[i & 3], v[i]);
    // the anchor is the rounded product itself, so that what is stored says what was summed
    const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * to_log2, at = top == -INFINITY ? 0.f : top;
    float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < EC; ++i) e[i & 3] += exp2f(fmaf(v[i], to_log2, -at));
    if (row < live) a.stats[(int64_t)row * a.ns + n0 / (EC)] = make_float2(top, (e[0] + e[1]) + (e[2] + e[3]));
  });
  if (CG == 2) ptx::bulk_wait_all();
}

// The sum (or mean over the tokens that count) of the tokens' losses.
struct Reduced {
  float* out;              // one value, or NULL: the tokens' losses are the result
  int64_t tokens;
  int mean;
  int* ticket;
  int ctas;                // of loss_kernel, over all chunks
};

// f32 inputs: what dl is made of.  A row's values may lie anywhere between 1e-38 and the largest
// grad_loss, and f16 has five bits of exponent, so every factor is kept as a number and a power of two.
struct SplitRow {
  float top;               // p of another column than the target's: f 2^(fe + s log2(e) - top)
  float f, y;              // 1 <= |f| < 2, or zero, or not finite; y 2^ye is dl of the target
  int fe, ye;
};

struct SplitOut {
  SplitRow* rows;          // of the chunk
  int* row_shift;          // powers of two for dX: a row's largest |dl| 2^(shift - w_shift) is in (2^12, 2^14]
  int* col_top;            // (ld): cleared here (see split_kernel)
  const float* peak;       // NULL where grad_hidden is not wanted
  const float* w_shift;
  int64_t vocab;
};

constexpr int NO_TOP = -(1 << 20);   // of a column in which dl is zero

// Powers of two that split_kernel and the products agree on.
__device__ __forceinline__ int col_shift_of(int top) { return top == NO_TOP ? 0 : min(max(14 - top, -120), 180); }

__device__ __forceinline__ float split2(double v, int* e) {
  *e = 0;
  if (v == 0.0 || !isfinite(v)) return (float)v;
  const double m = frexp(v, e);
  *e -= 1;
  return (float)(2.0 * m);   // may round up to 2: the bounds below have room for it
}

// `peak`: of the row.
__device__ __forceinline__ void put_split(const SplitOut& o, int64_t row, const RowResult& r, double w, float peak, int target) {
  SplitRow q;
  q.top = r.top;
  q.f = split2(w * (double)r.inv, &q.fe);
  q.y = split2(w * (double)r.pm1, &q.ye);
  o.rows[row] = q;
  if (!o.peak) return;
  int top = NO_TOP;        // |dl| 2^-w_shift <= 2^top
  if (q.f != 0.f && peak > -INFINITY) top = q.fe + 1 + (int)ceilf(fminf(fmaxf(peak - r.top, -1000.f), 1000.f));
  if (q.y != 0.f && target >= 0) top = max(top, q.ye + 1 - (int)o.w_shift[target]);
  // f 2^(fe + shift) has to be a normal number (it would not be where all of the weight is below 1e-33)
  o.row_shift[row] = top == NO_TOP ? 0 : min(min(max(14 - top, -240), 240), 126 - q.fe);
}

// A warp per row that counts: its loss, and with `factors` or `split` what the gradients need.  The last
// CTA of the last chunk reduces the losses, in a fixed order.  Bound by the statistics' bytes: 8192 rows of
// 784 statistics 26 us (2 TB/s, from L2), f64 sums included.
__global__ void __launch_bounds__(256) loss_kernel(const float2* stats, int ns, const float* picked, Selected s, int from,
                                                   int rows, float* loss, float* lse, const float* weight,
                                                   RowFactors* factors, const SplitOut split, const Reduced red) {
  ptx::griddep_wait();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row < rows && from + row < *s.count) {
    const int target = s.target[from + row];
    const RowResult r = warp_row(stats + row * ns, ns, picked + row, target);
    float peak = -INFINITY;
    if (split.peak) {
      for (int i = threadIdx.x & 31; i < ns; i += 32) peak = fmaxf(peak, split.peak[row * ns + i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    }
    if ((threadIdx.x & 31) == 0) {
      const int t = s.index[from + row];
      loss[t] = r.loss;
      if (lse) lse[t] = r.lse;
      const float w = weight ? weight[t] : 1.f;
      if (factors) factors[row] = {r.top, w * r.inv, w * r.pm1};
      if (split.rows) put_split(split, row, r, (double)w, peak, target);
    }
  }
  if (split.rows)
    for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < split.vocab; v += (int64_t)gridDim.x * 256) split.col_top[v] = NO_TOP;
  if (!red.out) return;
  __shared__ int last;
  __shared__ double sh[8];
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(red.ticket, 1) == red.ctas - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < red.tokens; i += 256) sum += (double)__ldcg(loss + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 8; ++i) sum += sh[i];
  *red.out = (float)(red.mean ? sum / (double)max(*s.count, 1) : sum);
}

// ---------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------
// The factor alpha common to all rows is applied in f32 in the GEMMs' epilogues: folded into
// dl, the rounding of dl's largest entries (all near -alpha) would be one common error.
struct RowArgs {
  int64_t vocab, ld;
  Selected sel;
  int from;                // first of the rows that count, of this chunk
  const RowFactors* factors;
  const float* logits;
  bf16* dl;                // (rows, ld)
};

constexpr int ROW_THREADS = 256, ROW_UNROLL = 8, ROW_COLS = ROW_THREADS * 4 * ROW_UNROLL;

// dl from the logits, ROW_COLS columns of a row per CTA, every load issued before the first use.
// Zero rows up to the next 64.  HBM-bound: 6 bytes per logit; 8192 x 50000 in 367 us (6.7 TB/s).
__global__ void __launch_bounds__(ROW_THREADS) row_kernel(const RowArgs a) {
  ptx::griddep_wait();
  const int64_t row = blockIdx.x;
  const int64_t live = (int64_t)*a.sel.count - a.from;
  if (live <= 0 || row >= (live + 63) / 64 * 64) return;
  const bool counted = row < live;
  const int64_t c0 = (int64_t)blockIdx.y * ROW_COLS + threadIdx.x * 4;
  const float* s = a.logits + row * a.ld;
  float4 x[ROW_UNROLL];
#pragma unroll
  for (int u = 0; u < ROW_UNROLL; ++u) {
    const int64_t c = c0 + u * ROW_THREADS * 4;
    x[u] = counted && c < a.vocab ? *reinterpret_cast<const float4*>(s + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int y = counted ? a.sel.target[a.from + row] : -1;
  RowFactors r = {0.f, 0.f, 0.f};
  if (counted) r = a.factors[row];
  uint2* out = reinterpret_cast<uint2*>(a.dl + row * a.ld);
#pragma unroll
  for (int u = 0; u < ROW_UNROLL; ++u) {
    const int64_t c = c0 + u * ROW_THREADS * 4;
    if (c >= a.vocab) break;
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    if (counted) {
      d[0] = r.f * exp2f(fmaf(x[u].x, LOG2E, -r.top));
      d[1] = r.f * exp2f(fmaf(x[u].y, LOG2E, -r.top));
      d[2] = r.f * exp2f(fmaf(x[u].z, LOG2E, -r.top));
      d[3] = r.f * exp2f(fmaf(x[u].w, LOG2E, -r.top));
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k == y) d[k] = r.at_y;
    }
    const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(d[0], d[1]), __floats2bfloat162_rn(d[2], d[3])};
    out[c / 4] = *reinterpret_cast<const uint2*>(h);
  }
}

// f32 inputs: dl as two f16 planes, hi + lo, times a power of two that belongs to what the product
// keeps apart: to a row for dX = dl W, where every token's gradient stands for itself, and to a
// column for dW = dl^T X, where every word's does.  (One power for all of dl lost the rows of small
// grad_loss, of confident tokens and of improbable words.)  The other operand's rows have powers of their
// own (shift_of), which a product over these rows takes from dl.  So the logits are read twice, 16 bytes per logit
// in all, HBM-bound: 2048 x 50257 in 138 + 131 us (6.1 TB/s).
//   ROWS      planes for dX; with MAX also each column's largest |dl|, as a power of two
//   MAX alone the latter, where grad_hidden is not wanted
//   COLS      planes for dW, over the ones for dX
// A column's maximum is that of integers, so the order in which CTAs add to it changes nothing.
struct SplitArgs {
  int64_t vocab, ld;
  Selected sel;
  int from, n, per;        // first of the rows that count; rows of the chunk; rows of a CTA, 64 at most
  unsigned col_blocks;
  const SplitRow* rows;
  const int* row_shift;
  int* col_top;            // (ld): |dl| 2^-x_shift <= 2^col_top in this column, NO_TOP where dl is zero
  const int* x_shift;      // of the chunk's rows of hidden
  const float* w_shift;    // (ld)
  const float* logits;
  __half* hi;
  __half* lo;
};

enum Planes { ROWS = 1, MAX = 2, COLS = 4 };
constexpr int SPLIT_THREADS = 256, SPLIT_COLS = 4 * SPLIT_THREADS, SPLIT_ROWS = 64, SPLIT_AHEAD = 8;

template <int WHAT>
__global__ void __launch_bounds__(SPLIT_THREADS) split_kernel(const SplitArgs a) {
  struct Row {
    float to_log2, top;
    float f;               // the factor as a number and a power of two, and (ff) as one number
    int k;
    float ff, mf;          // mf: what it adds to a column's maximum, as a power of two
    int target, ky;        // the same of the target's column, if it has one
    float y, my;
  };
  __shared__ Row rows[SPLIT_ROWS];
  ptx::griddep_wait();
  const unsigned rb = blockIdx.x / a.col_blocks, cb = blockIdx.x - rb * a.col_blocks;
  const int live = min(*a.sel.count - a.from, a.n), first = (int)rb * a.per;
  const int end = min(min(first + a.per, a.n), WHAT == MAX ? live : (live + 63) / 64 * 64);
  if (live <= 0 || first >= end) return;
  const int tid = threadIdx.x;
  if (tid < end - first) {
    const int row = first + tid;
    Row q = {0.f, 0.f, 0.f, 0, 0.f, -INFINITY, -1, 0, 0.f, -INFINITY};   // a row that does not count: zeros
    if (row < live) {
      const SplitRow r = a.rows[row];
      const int x_shift = a.x_shift[row], shift = (WHAT & ROWS) != 0 ? a.row_shift[row] : -x_shift;
      q.to_log2 = LOG2E * logit_scale(x_shift);
      q.top = r.top; q.f = r.f; q.y = r.y;
      q.target = a.sel.target[a.from + row];
      q.k = r.fe + shift; q.ky = r.ye + shift;
      q.ff = q.k > 127 ? r.f * INFINITY : r.f * pow2(q.k);
      if (r.f != 0.f) q.mf = (float)(r.fe + 1 - x_shift);
      if (r.y != 0.f) q.my = (float)(r.ye + 1 - x_shift);
    }
    rows[tid] = q;
  }
  __syncthreads();
  const int64_t c = (int64_t)cb * SPLIT_COLS + tid * 4;
  if (c >= a.vocab) return;      // (rows of logits and planes are ld long, a multiple of 64)
  int shift[4] = {0, 0, 0, 0};
  if constexpr ((WHAT & COLS) != 0) {
    const int4 q = *reinterpret_cast<const int4*>(a.col_top + c);
    shift[0] = col_shift_of(q.x); shift[1] = col_shift_of(q.y); shift[2] = col_shift_of(q.z); shift[3] = col_shift_of(q.w);
  } else if constexpr ((WHAT & ROWS) != 0) {
    const float4 q = *reinterpret_cast<const float4*>(a.w_shift + c);
    shift[0] = -(int)q.x; shift[1] = -(int)q.y; shift[2] = -(int)q.z; shift[3] = -(int)q.w;
  }
  // Columns whose largest |dl| (with the row's power) is above 2^-86 hold nothing below f32's normal numbers that an f16 of them
  // could keep: plain products.  For the others the exponential's argument takes 64 of the shift, which
  // is exact there, z being as far below; from a shift of 190 on p is below 1e-52.
  const bool plain = max(max(shift[0], shift[1]), max(shift[2], shift[3])) <= 100;
  const float cs[4] = {pow2(shift[0]), pow2(shift[1]), pow2(shift[2]), pow2(shift[3])};
  float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  for (int r0 = first; r0 < end; r0 += SPLIT_AHEAD) {
    float4 x[SPLIT_AHEAD];
#pragma unroll
    for (int j = 0; j < SPLIT_AHEAD; ++j)
      x[j] = r0 + j < min(end, live) ? *reinterpret_cast<const float4*>(a.logits + (int64_t)(r0 + j) * a.ld + c)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < SPLIT_AHEAD; ++j) {
      if (r0 + j >= end) break;
      const Row& r = rows[r0 + j - first];
      const int at_y = r.target - (int)c;
      float z[4] = {fmaf(x[j].x, r.to_log2, -r.top), fmaf(x[j].y, r.to_log2, -r.top), fmaf(x[j].z, r.to_log2, -r.top),
                    fmaf(x[j].w, r.to_log2, -r.top)};
      float d[4];
      if constexpr ((WHAT & (ROWS | COLS)) != 0) {
        if constexpr ((WHAT & ROWS) != 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = r.ff * exp2f(z[i]) * cs[i];
        } else if (plain) {
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = r.ff * exp2f(z[i]) * cs[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = r.k + shift[i];
            d[i] = k > 190 ? 0.f : k > 100 ? r.f * exp2f(z[i] + 64.f) * pow2(k - 64) : r.f * exp2f(z[i]) * pow2(k);
          }
        }
      }
      if constexpr ((WHAT & MAX) != 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] += r.mf;
      }
      if ((unsigned)at_y < 4u && r.target >= 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i == at_y) {
            if constexpr ((WHAT & (ROWS | COLS)) != 0) d[i] = r.y * pow2(r.ky + shift[i]);
            z[i] = r.my;
          }
      }
      if constexpr ((WHAT & MAX) != 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) most[i] = fmaxf(most[i], z[i]);
      }
      if constexpr ((WHAT & (ROWS | COLS)) != 0) {
        const int64_t at = (int64_t)(r0 + j) * a.ld + c;
        const __half2 h[2] = {__floats2half2_rn(d[0], d[1]), __floats2half2_rn(d[2], d[3])};
        const float2 g0 = __half22float2(h[0]), g1 = __half22float2(h[1]);
        const __half2 l[2] = {__floats2half2_rn(d[0] - g0.x, d[1] - g0.y), __floats2half2_rn(d[2] - g1.x, d[3] - g1.y)};
        *reinterpret_cast<uint2*>(a.hi + at) = *reinterpret_cast<const uint2*>(h);
        *reinterpret_cast<uint2*>(a.lo + at) = *reinterpret_cast<const uint2*>(l);
      }
    }
  }
  if constexpr ((WHAT & MAX) != 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c + i >= a.vocab || most[i] == -INFINITY) continue;
      const int top = (int)ceilf(fminf(fmaxf(most[i], -1000.f), 1000.f));
      // it only grows, so a look at it saves most CTAs the atomic (4000 rows of 500 columns: 23 -> 20 us)
      if (__ldcg(a.col_top + c + i) < top) atomicMax(a.col_top + c + i, top);
    }
  }
}

// Epilogue of the gradients' GEMMs.
struct OutArgs {
  int64_t rows, cols;
  const int* index;        // row r of the result goes to row index[r] of out (NULL: to row r)
  void* out;               // (rows, cols), the result times alpha; NULL: into `part` only
  const float* alpha;
  float* part;             // f32: parts of a split K range (splits, rows, cols), or the running sum
  int sum, add_part;       // `part` is the running sum over chunks of tokens; add what it holds
  // f32 inputs: the power of two to take out again of each row of the result is row_shift, or
  // col_shift_of(col_top)
  const int* row_shift;
  const int* col_top;
};

// OUT: tiles go to the output, times alpha.  PART: to f32 parts where the K range is split, or to
// the running sum over chunks of tokens; the last chunk, and a range that the device did not
// split, go to the output.
enum Mode { OUT, PART };

template <int CG, int PLANES, bool A_MN, typename TO, Mode MODE>
__global__ void __launch_bounds__(gemm::THREADS, 1) grad_gemm_kernel(const __grid_constant__ gemm::Problem p,
                                                                     const __grid_constant__ OutArgs a) {
  extern __shared__ uint8_t smem[];
  __shared__ gemm::Ctl ctl;
  float alpha = 1.f;
  auto prep = [&]() { alpha = *a.alpha; };
  gemm::run<CG, PLANES, A_MN, true>(p, smem, &ctl, prep, [&](const gemm::Tile& t, float (&v)[EC], int row0, int n0, int live,
                                                     int splits, uint4* stage) {
    const int64_t all = p.limit_k ? a.rows : live;
    const int rows = (int)min((int64_t)32, all - row0), cols = (int)min((int64_t)EC, a.cols - n0);
    if (rows <= 0 || cols <= 0) return;
    if constexpr (PLANES == 2) {
      const int row = row0 + min((int)(threadIdx.x & 31), rows - 1);
      const int e = A_MN ? col_shift_of(a.col_top[row]) : a.row_shift[row];
      // in two steps: the whole power may lie outside f32
      const float f0 = pow2(-(e / 2)), f1 = pow2(-(e - e / 2));
#pragma unroll
      for (int i = 0; i < EC; ++i) v[i] = v[i] * f0 * f1;
    }
    if constexpr (MODE == OUT) {
#pragma unroll
      for (int i = 0; i < EC; ++i) v[i] *= alpha;
    }
    TO* out = static_cast<TO*>(a.out) + n0;
    auto row_at = [&](int i) { return out + (int64_t)(a.index ? a.index[row0 + i] : row0 + i) * a.cols; };
    bool vec = vec_rows(out, a.cols) && cols % (16 / (int)sizeof(TO)) == 0;
    if constexpr (MODE == OUT) {
      gemm::by_rows<CG, TO>(stage, v, vec, rows, [&](int i, int c, uint4 q) {
        if (c < cols) *reinterpret_cast<uint4*>(row_at(i) + c) = q;
      }, [&](int i, int c, TO x) {
        if (c < cols) row_at(i)[c] = x;
      });
    } else {
      const bool done = a.sum ? a.out != nullptr : splits == 1, add = a.sum && a.add_part;
      float* part = a.part + ((int64_t)t.split * all + row0) * a.cols + n0;
      vec = vec_rows(part, a.cols) && cols % 4 == 0 && (!done || vec);
      gemm::by_rows<CG, float>(stage, v, vec, rows, [&](int i, int c, uint4 q) {
        if (c >= cols) return;
        float4 x = make_float4(__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w));
        float4* at = reinterpret_cast<float4*>(part + i * a.cols + c);
        if (add) {
          const float4 y = *at;
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        if (!done)
          *at = x;
        else if constexpr (sizeof(TO) == 4)
          *reinterpret_cast<float4*>(row_at(i) + c) = make_float4(x.x * alpha, x.y * alpha, x.z * alpha, x.w * alpha);
        else
          *reinterpret_cast<uint2*>(row_at(i) + c) =
              make_uint2(gemm::pack_bf16(x.x * alpha, x.y * alpha), gemm::pack_bf16(x.z * alpha, x.w * alpha));
      }, [&](int i, int c, float x) {
        if (c >= cols) return;
        float* at = part + i * a.cols + c;
        if (add) x += *at;
        if (done) st(row_at(i) + c, x * alpha);
        else *at = x;
      });
    }
  });
}

// Sum of the parts of a split K range, in order, times alpha; nothing where it was not split.
// CTAs take rows of the result in turns.  HBM-bound: 70 us for the parts of 8192 x 2560.
template <int CG, typename TO>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ gemm::Problem p, const __grid_constant__ OutArgs a) {
  ptx::griddep_wait();
  const int live = gemm::live_rows(p), splits = gemm::splits_of<CG>(p, live);
  if (splits == 1) return;
  const int64_t rows = p.limit_k ? a.rows : live, step = rows * a.cols;
  const float f = *a.alpha;
  const bool vec = a.cols % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;   // the parts start at 256 bytes
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    TO* o = static_cast<TO*>(a.out) + (int64_t)(a.index ? a.index[row] : row) * a.cols;
    const float* q = a.part + row * a.cols;
    if (vec) {
#pragma unroll 2
      for (int64_t c = threadIdx.x * 4; c < a.cols; c += 1024) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int j = 0; j < splits; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(q + j * step + c);
          v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        if constexpr (sizeof(TO) == 4)
          *reinterpret_cast<float4*>(o + c) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
        else
          *reinterpret_cast<uint2*>(o + c) = make_uint2(gemm::pack_bf16(v.x * f, v.y * f), gemm::pack_bf16(v.z * f, v.w * f));
      }
    } else {
      for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
        float v = 0.f;
#pragma unroll 4
        for (int j = 0; j < splits; ++j) v += q[j * step + c];
        st(o + c, v * f);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int SMS = 148;   // of a B200
constexpr int MAX_SPLITS = 32;

template <int CG, typename Kernel, typename Args>
cudaError_t launch_gemm(Kernel kernel, const gemm::Problem& p, const Args& a, std::atomic<uint64_t>* allowed, cudaStream_t st) {
  constexpr int smem = gemm::Shape<CG>::SMEM;
  const cudaError_t e = allow_smem((const void*)kernel, smem, allowed);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)p.m_tiles * p.n_tiles * std::max(1, p.max_splits);
  if (units >= (int64_t(1) << 31) || (int64_t)p.k_blocks * MAX_SPLITS >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
  return launch_dependent(kernel, dim3((unsigned)(CG * std::min<int64_t>(units, SMS / CG))), gemm::THREADS, smem, CG, st, p, a);
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
  int64_t part_x, part_w;           // values that the parts of split K ranges may take (0: no split)
  bool pack_w, sum_w;       // sum_w: dW's running sum over chunks needs its own f32 buffer
  size_t one, index, target, rows, picked, factors, row_shift, col_top, stats, peak, x, w, x_shift, w_shift, w_scale, logits, dl[2], part, wsum, total;
};

Plan plan_of(const ssd_linear_ce_params_t* p) {
  Plan q{};
  q.grad = p->grad_hidden || p->grad_weight;
  q.planes = p->dtype == SSD_DTYPE_F32 ? 2 : 1;
  q.ns = BN / EC * (int64_t)cdiv(p->vocab, BN);
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
  q.sum_w = p->grad_weight && q.nchunks > 1;
  // the reduction over the vocabulary may be split in up to 32 parts (how many, the device decides:
  // it knows how many rows count); that over tokens only where the weight is a few tiles
  const int64_t x_values = q.chunk * p->dim, w_values = p->vocab * p->dim;
  q.part_x = p->grad_hidden ? std::min<int64_t>(MAX_SPLITS * x_values, std::max<int64_t>(4 * x_values, 1 << 25)) : 0;
  q.part_w = p->grad_weight && !q.sum_w && w_values <= (1 << 24) ? std::min<int64_t>(MAX_SPLITS * w_values, 1 << 25) : 0;
  size_t at = 256;   // the status word
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  q.one = take(64);
  q.index = take((size_t)p->tokens * 4);
  q.target = take((size_t)p->tokens * 4);
  q.rows = take(p->reduction == SSD_REDUCE_NONE ? 0 : (size_t)p->tokens * 4);
  q.picked = take((size_t)q.chunk * 4);
  const bool split = q.grad && q.planes == 2;
  q.factors = take(q.grad ? (size_t)q.chunk * (split ? sizeof(SplitRow) : sizeof(RowFactors)) : 0);
  q.row_shift = take(split ? (size_t)q.chunk * 4 : 0);
  q.col_top = take(split ? (size_t)q.ld * 4 : 0);
  q.stats = take((size_t)q.chunk * q.ns * 8);
  q.peak = take(split && p->grad_hidden ? (size_t)q.chunk * q.ns * 4 : 0);
  q.x = take(planes_bytes(p->tokens, p->dim, p->dtype));
  q.w = take(q.pack_w ? planes_bytes(p->vocab, p->dim, p->dtype) : 0);
  q.x_shift = take(q.planes == 2 ? (size_t)p->tokens * 4 : 0);
  const size_t words = q.planes == 2 ? (size_t)cdiv(p->vocab, BN) * BN * 4 : 0;   // whole tiles
  q.w_shift = take(words);
  q.w_scale = take(words);
  if (q.grad) {
    q.logits = take((size_t)q.chunk * q.ld * 4);
    for (int i = 0; i < q.planes; ++i) q.dl[i] = take((size_t)q.chunk * q.ld * 2);
    q.part = take((size_t)std::max(q.part_x, q.part_w) * 4);   // one after the other
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

// Rows of a CTA: 64, and fewer where that would leave SMs without work (300 x 50257 with maxima: 64 rows 24
// us, 16 rows 21), but not so few that a column's maximum is bound by atomics to one address (4000 x 500: 500
// CTAs of 8 rows 19 us, 250 of 16 rows 11).
template <int WHAT>
cudaError_t launch_split(SplitArgs a, cudaStream_t st) {
  a.col_blocks = (unsigned)cdiv(a.vocab, SPLIT_COLS);
  a.per = SPLIT_ROWS;
  while (a.per > SPLIT_AHEAD && (int64_t)a.col_blocks * cdiv(a.n, a.per) < 4 * SMS && ((WHAT & MAX) == 0 || cdiv(a.n, a.per) < 128))
    a.per /= 2;
  const int64_t ctas = (int64_t)a.col_blocks * cdiv(a.n, a.per);
  if (ctas >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
  return launch_dependent(split_kernel<WHAT>, dim3((unsigned)ctas), SPLIT_THREADS, 0, 1, st, a);
}

template <int CG>
cudaError_t logits_gemm(const Operand& x, const Operand& w, int planes, LogitArgs a, const int* count, int from,
                        unsigned* status, cudaStream_t st) {
  gemm::Problem g{};
  g.limit = count;
  g.limit_from = from;
  g.rows = (int)x.rows;
  if (!maps(g.a, x, planes, BM) || !maps(g.b, w, planes, BN / CG)) return cudaErrorInvalidValue;
  g.m_tiles = cdiv(x.rows, BM * CG);
  g.n_tiles = cdiv(a.vocab, BN);
  g.k_blocks = cdiv(x.dim, gemm::BK);
  g.planes = planes;
  g.m_fastest = 1;
  g.segment = planes == 2 ? SEGMENT_F32 : SEGMENT_BF16;
  g.status = status;
  if (CG == 2 && a.logits && !tc_map_2d(&a.map, a.logits, (uint64_t)a.ld, (uint64_t)x.rows, (uint64_t)a.ld * 4, 32, true))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> allowed[2] = {};
  if (planes == 2) return launch_gemm<CG>(logits_kernel<CG, 2>, g, a, &allowed[1], st);
  return launch_gemm<CG>(logits_kernel<CG, 1>, g, a, &allowed[0], st);
}

// One gradient: the GEMM, and where its K range may be split the sum of the parts.
template <int CG, bool A_MN, typename TO>
cudaError_t grad_gemm(const Operand& a, const Operand& b, int64_t k, int planes, int64_t part_values,
                      const OutArgs& o, const int* count, int from, unsigned* status, cudaStream_t st) {
  gemm::Problem g{};
  g.limit = count;
  g.limit_from = from;
  g.rows = (int)a.rows;    // dl's rows: the result's for dX, the reduced ones for dW
  g.limit_k = A_MN;
  if (!maps(g.a, a, planes, A_MN ? 64 : BM) || !maps(g.b, b, planes, 64)) return cudaErrorInvalidValue;
  g.m_tiles = cdiv(o.rows, BM * CG);
  g.n_tiles = cdiv(o.cols, BN);
  g.rows_out = (int)o.rows;
  g.cols = (int)o.cols;
  g.max_splits = part_values > 0 ? MAX_SPLITS : 1;
  g.part_values = part_values;
  g.k_blocks = cdiv(k, gemm::BK);
  g.planes = planes;
  g.m_fastest = 0;
  g.segment = planes == 2 ? SEGMENT_F32 : SEGMENT_GRAD;
  g.status = status;
  static std::atomic<uint64_t> allowed[4] = {};
  const bool out = !o.sum && g.max_splits == 1;
  cudaError_t e;
  if (planes == 2)
    e = out ? launch_gemm<CG>(grad_gemm_kernel<CG, 2, A_MN, TO, OUT>, g, o, &allowed[0], st)
            : launch_gemm<CG>(grad_gemm_kernel<CG, 2, A_MN, TO, PART>, g, o, &allowed[1], st);
  else
    e = out ? launch_gemm<CG>(grad_gemm_kernel<CG, 1, A_MN, TO, OUT>, g, o, &allowed[2], st)
            : launch_gemm<CG>(grad_gemm_kernel<CG, 1, A_MN, TO, PART>, g, o, &allowed[3], st);
  if (e != cudaSuccess || g.max_splits == 1) return e;
  return launch_dependent(join_kernel<CG, TO>, dim3((unsigned)std::min<int64_t>(o.rows, SMS * 8)), 256, 0, 1, st, g, o);
}

template <bool A_MN, typename... Args>
cudaError_t grad_gemm_as(bool pair, bool bf16_out, Args&&... args) {
  if (pair) return bf16_out ? grad_gemm<2, A_MN, bf16>(args...) : grad_gemm<2, A_MN, float>(args...);
  return bf16_out ? grad_gemm<1, A_MN, bf16>(args...) : grad_gemm<1, A_MN, float>(args...);
}

}  // namespace

size_t linear_ce_workspace(const ssd_linear_ce_params_t* p) {
  return linear_ce_is_small(p) ? linear_ce_small_workspace(p) : plan_of(p).total;
}

cudaError_t launch_linear_ce(const ssd_linear_ce_params_t* p, void* workspace, cudaStream_t st, const char** at) {
  if (linear_ce_is_small(p)) return launch_linear_ce_small(p, workspace, st, at);
  const Plan q = plan_of(p);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  unsigned* status = reinterpret_cast<unsigned*>(ws);
  Selected sel;
  sel.status = status;
  sel.count = reinterpret_cast<int*>(ws + q.one);
  sel.alpha = reinterpret_cast<float*>(ws + q.one) + 1;
  sel.ticket = reinterpret_cast<int*>(ws + q.one + 32);
  sel.index = reinterpret_cast<int*>(ws + q.index);
  sel.target = reinterpret_cast<int*>(ws + q.target);
  float* rows = p->reduction == SSD_REDUCE_NONE ? p->loss : reinterpret_cast<float*>(ws + q.rows);
  const bool bf = p->dtype == SSD_DTYPE_BF16, mean = p->reduction == SSD_REDUCE_MEAN;
  const bool per_row = p->reduction == SSD_REDUCE_NONE && p->grad_loss;
  select_kernel<<<1, 1024, 0, st>>>(p->targets, p->targets_int64, p->tokens, p->vocab, p->ignore_index, mean,
                                    per_row ? nullptr : p->grad_loss, sel, rows, p->lse);
  cudaError_t err = cudaGetLastError();
  CE_CHECK(err, "select");
  Operand x{}, w{};
  x.rows = p->tokens; x.dim = p->dim;
  place_planes(&x, p->dtype, ws + q.x);
  const dim3 grid((unsigned)p->tokens, p->grad_hidden ? 2 : 1);
  void* hi = const_cast<void*>(x.plane[0]);
  void* lo = const_cast<void*>(x.plane[1]);
  const unsigned wide = 148 * 8;
  int* x_shift = reinterpret_cast<int*>(ws + q.x_shift);
  float* w_shift = reinterpret_cast<float*>(ws + q.w_shift);
  float* w_scale = reinterpret_cast<float*>(ws + q.w_scale);
  if (bf)
    err = launch_dependent(gather_kernel<bf16>, grid, 128, 0, 1, st, static_cast<const bf16*>(p->hidden), p->hidden_stride_row, p->dim,
                                              x.ld, sel, p->targets, p->targets_int64, p->ignore_index, hi, lo, nullptr,
                                              static_cast<bf16*>(p->grad_hidden));
  else
    err = launch_dependent(gather_kernel<float>, grid, 128, 0, 1, st, static_cast<const float*>(p->hidden), p->hidden_stride_row, p->dim,
                                               x.ld, sel, p->targets, p->targets_int64, p->ignore_index, hi, lo, x_shift,
                                               static_cast<float*>(p->grad_hidden));
  CE_CHECK(err, "gather");
  w.rows = p->vocab; w.dim = p->dim; w.ld = p->weight_stride_row; w.plane[0] = p->weight;
  if (q.pack_w) {
    place_planes(&w, p->dtype, ws + q.w);
    void* whi = const_cast<void*>(w.plane[0]);
    void* wlo = const_cast<void*>(w.plane[1]);
    const unsigned g = (unsigned)std::min<int64_t>((w.rows * ((w.ld + 255) / 256) + 7) / 8, wide * 2);
    if (bf)
      err = launch_dependent(repack_kernel, g, 256, 0, 1, st, static_cast<const bf16*>(p->weight), p->weight_stride_row, p->vocab, p->dim,
                                            w.ld, whi);
    else
      err = launch_dependent(planes_kernel, (unsigned)std::min<int64_t>((w.rows + 7) / 8, wide * 2), 256, 0, 1, st,
                             static_cast<const float*>(p->weight), p->weight_stride_row, p->vocab, p->dim, w.ld, whi, wlo, w_shift,
                             w_scale);
    CE_CHECK(err, "weight planes");
  }
  Reduced red{};
  if (p->reduction != SSD_REDUCE_NONE) {
    red.out = p->loss;
    red.tokens = p->tokens;
    red.mean = mean;
    red.ticket = sel.ticket;
    for (int64_t c = 0; c < q.nchunks; ++c) red.ctas += cdiv(std::min(q.chunk, p->tokens - c * q.chunk), 8);
  }
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
    a.x_shift = x_shift + t0;
    a.w_shift = w_shift;
    a.w_scale = w_scale;
    a.peak = q.planes == 2 && p->grad_hidden ? reinterpret_cast<float*>(ws + q.peak) : nullptr;
    // one SM's tiles where a pair's second half would be empty (loss of 128 x 50000 x 2560: 68 us, by pairs 70;
    // of 200 tokens, in two rows of tiles: 78, by pairs 71)
    if (n > BM) CE_CHECK(logits_gemm<2>(xc, w, q.planes, a, sel.count, from, status, st), "logits");
    else CE_CHECK(logits_gemm<1>(xc, w, q.planes, a, sel.count, from, status, st), "logits");
    RowFactors* factors = q.grad && bf ? reinterpret_cast<RowFactors*>(ws + q.factors) : nullptr;
    SplitOut split{};
    if (q.grad && !bf) {
      split.rows = reinterpret_cast<SplitRow*>(ws + q.factors);
      split.row_shift = reinterpret_cast<int*>(ws + q.row_shift);
      split.col_top = reinterpret_cast<int*>(ws + q.col_top);
      split.peak = a.peak;
      split.w_shift = w_shift;
      split.vocab = p->vocab;
    }
    err = launch_dependent(loss_kernel, (unsigned)cdiv(n, 8), 256, 0, 1, st, a.stats, a.ns, a.picked, sel, from, (int)n, rows, p->lse,
                                                     per_row ? p->grad_loss : nullptr, factors, split, red);
    CE_CHECK(err, "loss");
    if (!q.grad) continue;
    SplitArgs sp{};
    if (bf) {
      RowArgs r{};
      r.vocab = p->vocab; r.ld = q.ld; r.sel = sel; r.from = from; r.factors = factors; r.logits = a.logits;
      r.dl = reinterpret_cast<bf16*>(ws + q.dl[0]);
      CE_CHECK(launch_dependent(row_kernel, dim3((unsigned)n, (unsigned)cdiv(p->vocab, ROW_COLS)), ROW_THREADS, 0, 1, st, r), "rows");
    } else {
      sp.vocab = p->vocab; sp.ld = q.ld; sp.sel = sel; sp.from = from; sp.n = (int)n;
      sp.rows = split.rows; sp.row_shift = split.row_shift; sp.col_top = split.col_top; sp.logits = a.logits;
      sp.x_shift = a.x_shift; sp.w_shift = w_shift;
      sp.hi = reinterpret_cast<__half*>(ws + q.dl[0]);
      sp.lo = reinterpret_cast<__half*>(ws + q.dl[1]);
      CE_CHECK(p->grad_hidden ? p->grad_weight ? launch_split<ROWS | MAX>(sp, st) : launch_split<ROWS>(sp, st)
                              : launch_split<MAX>(sp, st), "rows");
    }
    Operand dl{};
    dl.rows = n; dl.dim = p->vocab; dl.ld = q.ld;
    for (int i = 0; i < q.planes; ++i) dl.plane[i] = ws + q.dl[i];
    OutArgs o{};
    o.alpha = sel.alpha;
    o.row_shift = split.row_shift;
    o.col_top = split.col_top;
    o.part = reinterpret_cast<float*>(ws + q.part);
    if (p->grad_hidden) {
      OutArgs ox = o;
      ox.rows = n; ox.cols = p->dim; ox.index = sel.index + t0; ox.out = p->grad_hidden;
      CE_CHECK(grad_gemm_as<false>(n > BM, bf, dl, w, p->vocab, q.planes, q.part_x, ox, sel.count, from, status, st),
               "grad_hidden");
    }
    if (p->grad_weight) {
      if (!bf) CE_CHECK(launch_split<COLS>(sp, st), "columns");
      OutArgs ow = o;
      ow.rows = p->vocab; ow.cols = p->dim;
      if (q.sum_w) ow.part = reinterpret_cast<float*>(ws + q.wsum);
      ow.sum = q.sum_w;
      ow.add_part = c > 0;
      ow.out = c == q.nchunks - 1 ? p->grad_weight : nullptr;
      CE_CHECK(grad_gemm_as<true>(p->vocab > BM, p->grad_weight_dtype == SSD_DTYPE_BF16, dl, xc, n, q.planes, q.part_w, ow,
                                  sel.count, from, status, st), "grad_weight");
    }
  }
  return cudaSuccess;
}

}  // namespace ssd
