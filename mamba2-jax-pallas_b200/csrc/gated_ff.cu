// Gated feed-forward block and its gradients:
//
//   g = x Wg^T, u = x Wu^T;  h = act(g) u;  y = h Wd^T
//   dh = dy Wd;  dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu
//   dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Both passes are products of 2 T D F operations each (3 forward, 6 backward and 2 for g and u again),
// bound by the tensor pipe; what lies between is kept out of memory:
//   gate/up     one product whose tile has 128 columns of g and the same 128 of u, so that an epilogue warp
//               holds both and writes h alone.  In a pair of CTAs each loads one weight's rows.
//   backward    the same product again (keeping g and u would need 8 bytes a value in f32, or round them), whose
//               epilogue reads dh and writes dg, du and h
//   dx          one product over K = 2 F: dg against Wg, then du against Wu
//   dWg, dWu    one launch, F rows of each
// The products' loop is that of tc_gemm.cuh (pairs of CTAs, 256 x 256 tiles, TMA into a ring of stages, two
// accumulators in TMEM, K segments added in registers), with operands in two parts.
//
// bf16: h, dg and du are rounded once, as operands; everything else stays f32 up to the result.  f32: every operand
// as three bf16 terms of its value (24 bits down to 2^-110; terms below 2^-126 are lost), six products per pair: those above 2^-24 of
// the value.
#include <algorithm>

#include "common.cuh"
#include "gated_ff.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "ssd_kernels.h"
#include "ssd_tc.h"
#include "tc_gemm.cuh"

namespace ssd {
namespace {

using gemm::BK;
using gemm::BM;
using gemm::BN;
using gemm::EPI_COLS;
using gemm::EPI_WARPS;
using gemm::THREADS;

// K blocks summed in TMEM before they are added in registers (the tensor core's adds truncate, tc_gemm.cuh).  Of bf16
// operands 64 where the sum is rounded to bf16 behind it: the loss, 1.1e-5 and of one sign, is a two-hundredth of that
// rounding, and the MMAs wait for an epilogue that takes longer than a segment.  32 for the weights' gradients, which may go to f32: 3.5e-6.
constexpr int SEGMENT_BF16 = 64, SEGMENT_DW = 32, SEGMENT_F32 = 1;

// ---------------------------------------------------------------------------
// the products' loop
// ---------------------------------------------------------------------------
// Operands in parts: DUAL: B is 128 rows of b[0] and the same of b[1]; TWO_K: the K range is that of (a[0], b[0]),
// then that of (a[1], b[1]); TWO_M: the rows are those of a[0], then those of a[1].
enum Parts { ONE, DUAL, TWO_K, TWO_M };

struct Product {
  CUtensorMap a[2][3], b[2][3];   // [part][plane]
  int m_tiles, n_tiles, k_blocks; // over all parts
  int half;                       // k blocks (TWO_K) or m tiles (TWO_M) of a part
  int group;                      // m tiles that are walked together, n by n: what they share stays in L2
  int full;                       // tiles computed whole; the K range of those behind is split
  int splits, segment;
  int clear;                      // the first launch of a call clears the status word
  unsigned* status;
};

struct Tile {
  int m, n, split, k0, k1;
};

__device__ __forceinline__ Tile tile_of(const Product& p, unsigned r) {
  Tile t;
  const unsigned span = (unsigned)p.group * p.n_tiles, g = r / span, first = g * p.group, q = r - g * span;
  const unsigned rows = min((unsigned)p.group, (unsigned)p.m_tiles - first);
  t.n = (int)(q / rows);
  t.m = (int)(first + q - (unsigned)t.n * rows);
  t.split = -1;
  t.k0 = 0;
  t.k1 = p.k_blocks;
  return t;
}
__device__ __forceinline__ unsigned units_of(const Product& p) {
  return (unsigned)p.full + ((unsigned)p.m_tiles * p.n_tiles - p.full) * p.splits;
}
// Unit u: a whole tile (split -1), or a part of the K range of one of the last tiles.
__device__ __forceinline__ Tile tile_at(const Product& p, unsigned u) {
  if (u < (unsigned)p.full) return tile_of(p, u);
  const unsigned tail = (unsigned)p.m_tiles * p.n_tiles - p.full, v = u - p.full, split = v / tail;
  Tile t = tile_of(p, p.full + v - split * tail);
  t.split = (int)v;                // of the parts: split * tail + tile - full
  t.k0 = (int)((unsigned)p.k_blocks * split / p.splits);
  t.k1 = (int)((unsigned)p.k_blocks * (split + 1) / p.splits);
  return t;
}

// pre(tile, row0, column group) runs on the epilogue warps before they wait for a tile, epi(tile, v, row0, column group,
// stage) behind it; v holds 64 columns of row row0 + lane: those of the group, or (DUAL) 32 of g and the same 32 of u.
template <int CG, int PLANES, bool A_MN, bool B_MN, int PARTS, typename Pre, typename Epi>
__device__ __forceinline__ void run(const Product& p, uint8_t* smem_raw, gemm::Ctl* c, Pre&& pre, Epi&& epi) {
  using S = gemm::Shape<CG>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? gemm::cluster_rank() : 0;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      ptx::mbar_init(&c->full[i], 1);
      ptx::mbar_init(&c->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&c->acc_full[i], 1);
      ptx::mbar_init(&c->acc_empty[i], EPI_WARPS * CG);
    }
    ptx::mbar_init(&c->drain, 1);
    c->abort = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) gemm::tmem_alloc_all<CG>(&c->tmem);
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) gemm::cluster_sync_all();
  ptx::tc_fence_after();
  const uint32_t tmem = c->tmem;
  ptx::griddep_wait();   // all above needs nothing from the launches before
  if (p.clear && blockIdx.x == 0 && threadIdx.x == 0) *p.status = 0;   // (a wait takes seconds to give up)
  const unsigned unit0 = blockIdx.x / CG, units = units_of(p), step = gridDim.x / CG;
  const uint32_t smem0 = ptx::smem_u32(smem);

  if (warp == 0) {
    if (gemm::elect_one()) {
      uint32_t it = 0, s = 0, phase = 1;   // stage, and the parity of its last release
      bool ok = true;
      for (unsigned u = unit0; ok && u < units; u += step) {
        const Tile t = tile_at(p, u);
        const int ma = PARTS == TWO_M && t.m >= p.half;
        const int m0 = ((t.m - (ma ? p.half : 0)) * CG + (int)rank) * BM;
        const int n0 = PARTS == DUAL ? t.n * (BN / 2) : t.n * BN + (int)rank * (BN / CG);
        for (int kb = t.k0; ok && kb < t.k1; ++kb) {
          const int ka = PARTS == TWO_K && kb >= p.half, k = (kb - (ka ? p.half : 0)) * BK;
#pragma unroll
          for (int pl = PLANES - 1; pl >= 0; --pl, ++it) {   // the lowest terms first
            if (!gemm::wait(c, &c->empty[s], phase, p.status, 1)) {
              ok = false;
              break;
            }
            const uint32_t sa = smem0 + s * S::STAGE_BYTES, sb = sa + S::A_BYTES;
            uint32_t bar = ptx::smem_u32(&c->full[s]);
            // the pair's first CTA counts the bytes of both
            if (rank == 0) ptx::mbar_arrive_expect_tx(&c->full[s], CG * S::STAGE_BYTES);
            if constexpr (CG == 2) bar = gemm::map_rank(bar, 0);
            const CUtensorMap* am = &p.a[PARTS == TWO_K ? ka : PARTS == TWO_M ? ma : 0][pl];
            if constexpr (A_MN) {
              for (int i = 0; i < BM / 64; ++i) gemm::tma_load_2d<CG>(sa + i * 8192, am, bar, m0 + 64 * i, k);
            } else {
              gemm::tma_load_2d<CG>(sa, am, bar, k, m0);
            }
            if constexpr (PARTS == DUAL) {
              if constexpr (CG == 2) {
                gemm::tma_load_2d<CG>(sb, &p.b[rank][pl], bar, k, n0);
              } else {
                gemm::tma_load_2d<CG>(sb, &p.b[0][pl], bar, k, n0);
                gemm::tma_load_2d<CG>(sb + BN / 2 * BK * 2, &p.b[1][pl], bar, k, n0);
              }
            } else {
              const CUtensorMap* bm = &p.b[PARTS == TWO_K ? ka : 0][pl];
              if constexpr (B_MN) {
                for (int i = 0; i < BN / CG / 64; ++i) gemm::tma_load_2d<CG>(sb + i * 8192, bm, bar, n0 + 64 * i, k);
              } else {
                gemm::tma_load_2d<CG>(sb, bm, bar, k, n0);
              }
            }
            if (++s == S::STAGES) {
              s = 0;
              phase ^= 1;
            }
          }
        }
      }
      // a wait gave up: let the loads that are still in flight land before the CTA ends
      if (!ok) {
        const long long t0 = clock64();
        for (uint32_t j = it > S::STAGES ? it - S::STAGES : 0; rank == 0 && j < it; ++j)
          while (!ptx::mbar_try_wait(&c->full[j % S::STAGES], (j / S::STAGES) & 1) && clock64() - t0 < gemm::WAIT_CYCLES) {
          }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && gemm::elect_one()) {
      const uint32_t ID = gemm::idesc<CG, 1, A_MN, B_MN>();   // bf16 planes
      uint32_t s = 0, phase = 0, n = 0;
      bool ok = true;
      for (unsigned u = unit0; ok && u < units; u += step) {
        const Tile t = tile_at(p, u);
        uint32_t d = 0;
        for (int kb = t.k0, left = 0; kb < t.k1 && ok; ++kb, --left) {
          const bool first = left == 0;
          if (first) {
            left = min(p.segment, t.k1 - kb);
            if (n >= 2 && !gemm::wait(c, &c->acc_empty[n & 1], ((n >> 1) - 1) & 1, p.status, 2)) {
              ok = false;
              break;
            }
            ptx::tc_fence_after();
            d = tmem + (n & 1) * BN;
          }
          // Small products first: what an add cuts off goes by the sum that is there (three planes, products in the order
          // of the planes: gradients 2.3e-6 off).  The lowest plane's stage is free first, and was loaded first.
          uint32_t at[PLANES];
          uint64_t* done[PLANES];
#pragma unroll
          for (int i = PLANES - 1; i >= 0; --i) {
            if (ok && !gemm::wait(c, &c->full[s], phase, p.status, 3)) ok = false;
            at[i] = smem0 + s * S::STAGE_BYTES;
            done[i] = &c->empty[s];
            if (++s == S::STAGES) {
              s = 0;
              phase ^= 1;
            }
          }
          if (!ok) break;
          ptx::tc_fence_after();
          auto product = [&](int i, int j, bool add) { gemm::mma_block<CG, A_MN, B_MN>(d, at[i], at[j] + S::A_BYTES, ID, add); };
          if constexpr (PLANES == 3) {
            product(1, 1, !first);
            product(0, 2, true);
            product(2, 0, true);
            gemm::commit<CG>(done[2]);
            product(0, 1, true);
            product(1, 0, true);
            gemm::commit<CG>(done[1]);
            product(0, 0, true);
          } else {
            product(0, 0, !first);
          }
          gemm::commit<CG>(done[0]);
          if (left == 1) {
            gemm::commit<CG>(&c->acc_full[n & 1]);
            ++n;
          }
        }
      }
      if (!ok) {   // let the MMAs in flight finish
        ptx::tc_fence_before();
        if constexpr (CG == 2)
          asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(ptx::smem_u32(&c->drain)) : "memory");
        else
          ptx::mma_commit(&c->drain);
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(&c->drain, 0) && clock64() - t0 < gemm::WAIT_CYCLES) {
        }
      }
    }
  } else {
    const int quad = warp & 3, group = (warp - 2) / 4;
    uint4* stage = reinterpret_cast<uint4*>(smem + S::STAGES * S::STAGE_BYTES + (warp - 2) * S::EPI_WARP_BYTES);
    uint32_t n = 0;
    bool ok = true;
    for (unsigned u = unit0; ok && u < units; u += step) {
      const Tile t = tile_at(p, u);
      const int row0 = (t.m * CG + (int)rank) * BM + 32 * quad;
      pre(t, row0, group, stage);
      float v[EPI_COLS];
#pragma unroll
      for (int i = 0; i < EPI_COLS; ++i) v[i] = 0.f;
      for (int left = t.k1 - t.k0; left > 0; left -= p.segment, ++n) {
        // one lane waits for the warp, so that the warp stays converged for its TMEM loads
        int there = 0;
        if (lane == 0) there = gemm::wait(c, &c->acc_full[n & 1], (n >> 1) & 1, p.status, 4);
        if (!__shfl_sync(0xffffffffu, there, 0)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t from = tmem + (n & 1) * BN + ((uint32_t)(32 * quad) << 16);
#pragma unroll
        for (int ch = 0; ch < EPI_COLS / 16; ++ch) {
          const int col = PARTS == DUAL ? (ch >> 1) * (BN / 2) + group * 32 + (ch & 1) * 16 : group * EPI_COLS + ch * 16;
          float x[16];
          ptx::tmem_ld16(from + col, x);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[16 * ch + i] += x[i];
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            gemm::arrive_remote(gemm::map_rank(ptx::smem_u32(&c->acc_empty[n & 1]), 0));
          else
            ptx::mbar_arrive(&c->acc_empty[n & 1]);
        }
      }
      if (ok) epi(t, v, row0, group, stage);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");   // what pre() may have under way where a wait gave up
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) gemm::cluster_sync_all();   // no CTA leaves while its peer may still signal it
  if (warp == 1) {
    ptx::tc_fence_after();
    gemm::tmem_free_all<CG>(tmem);
  }
  if constexpr (CG == 2) gemm::cluster_sync_all();
}

// ---------------------------------------------------------------------------
// f32 values as three bf16 terms
// ---------------------------------------------------------------------------
// Two values as a pair of bf16, and what is left of them.  (What is left of an infinity is NaN: a value that is not finite makes its
// products so.)  CUT: a finite value that would round to infinity is cut instead.
template <bool CUT>
__device__ __forceinline__ uint32_t term_of(float& a, float& b) {
  uint32_t w = gemm::pack_bf16(a, b);
  if (CUT && ((w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u)) w = __float_as_uint(a) >> 16 | (__float_as_uint(b) & 0xffff0000u);
  a -= __uint_as_float(w << 16);
  b -= __uint_as_float(w & 0xffff0000u);
  return w;
}

// 8 values as planes of 16 bytes each: v = t[0] + t[1] + t[2] up to 2^-25 of it.
template <int PLANES>
__device__ __forceinline__ void planes_of(const float (&x)[8], uint4 (&q)[PLANES]) {
  if constexpr (PLANES == 1) {
    q[0] = make_uint4(gemm::pack_bf16(x[0], x[1]), gemm::pack_bf16(x[2], x[3]), gemm::pack_bf16(x[4], x[5]), gemm::pack_bf16(x[6], x[7]));
  } else {
    float v[8] = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
    q[0] = make_uint4(term_of<true>(v[0], v[1]), term_of<true>(v[2], v[3]), term_of<true>(v[4], v[5]), term_of<true>(v[6], v[7]));
#pragma unroll
    for (int i = 1; i < PLANES; ++i)
      q[i] = make_uint4(term_of<false>(v[0], v[1]), term_of<false>(v[2], v[3]), term_of<false>(v[4], v[5]), term_of<false>(v[6], v[7]));
  }
}

// Inputs that the tensor maps cannot read as they are: f32, or bf16 rows that do not start at 16 bytes.
struct Pack {
  const void* src;
  int64_t stride, rows, dim, ld;
  uint8_t* dst;                    // planes of rows x ld bf16, `plane` bytes apart
  int64_t plane;
  int64_t first;                   // the matrix's first unit of 256 columns of a row
};
struct PackArgs {
  Pack m[5];
  int n;
  int64_t units;
  unsigned* status;
};

// A warp takes 256 columns of a row at a time; bound by HBM.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackArgs a) {
  constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
  const int lane = threadIdx.x & 31;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < a.units; u += (int64_t)gridDim.x * 8) {
    int k = 0;
    while (k + 1 < a.n && u >= a.m[k + 1].first) ++k;
    const Pack& m = a.m[k];
    const int64_t runs = (m.ld + 255) / 256, r = (u - m.first) / runs, c = (u - m.first - r * runs) * 256 + lane * 8;
    if (c >= m.ld) continue;
    const T* row = static_cast<const T*>(m.src) + r * m.stride;
    float v[8];
    if (sizeof(T) == 4 && reinterpret_cast<uintptr_t>(row) % 16 == 0 && c + 8 <= m.dim) {
      const float4 x = *reinterpret_cast<const float4*>(row + c), y = *reinterpret_cast<const float4*>(row + c + 4);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
      v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < m.dim ? ld(row + c + i) : 0.f;
    }
    uint4 q[PLANES];
    planes_of<PLANES>(v, q);
#pragma unroll
    for (int i = 0; i < PLANES; ++i) *reinterpret_cast<uint4*>(m.dst + i * m.plane + (r * m.ld + c) * 2) = q[i];
  }
}

// ---------------------------------------------------------------------------
// g and u, and what is made of them
// ---------------------------------------------------------------------------
struct HiddenArgs {
  int rows;                        // T
  int64_t F, ld;                   // rows of h, dg, du and dh are ld values long, a multiple of 64
  uint8_t* h;                      // planes of (T, ld) bf16, `plane` bytes apart; backward NULL where no product reads it
  uint8_t* dg;
  uint8_t* du;
  int64_t plane;
  const float* dh;                 // (T, ld)
};

// 32 rows x 8 N columns of bf16 from packed rows, by runs of 16 N bytes (neighbouring lanes at neighbouring columns).
template <int N>
__device__ __forceinline__ void store_block(uint4* stage, const uint4 (&q)[N], uint8_t* out, int64_t ld, int row0, int rows, int64_t f0, int64_t F) {
  const int lane = threadIdx.x & 31;
  auto at = [](int i, int k) { return N == 4 ? gemm::epi_at<1>(i, k) : i * 2 + (k ^ (i >> 2 & 1)); };
  __syncwarp();
#pragma unroll
  for (int i = 0; i < N; ++i) stage[at(lane, i)] = q[i];
  __syncwarp();
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = j * (32 / N) + lane / N, k = lane % N;
    if (row0 + i < rows && f0 + k * 8 < F) *reinterpret_cast<uint4*>(out + ((int64_t)(row0 + i) * ld + f0 + k * 8) * 2) = stage[at(i, k)];
  }
}

// dh of 32 rows and 4 CHUNKS columns on its way into the warp's stage.
template <int CHUNKS>
__device__ __forceinline__ void fetch_block(uint4* stage, const HiddenArgs& a, int row0, int64_t f0) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < CHUNKS; ++j) {
    const int i = j * (32 / CHUNKS) + lane / CHUNKS, k = lane % CHUNKS;
    const bool there = row0 + i < a.rows && f0 + k * 4 < a.ld;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(stage + gemm::epi_at<CHUNKS / 4>(i, k))),
                 "l"(there ? a.dh + (int64_t)(row0 + i) * a.ld + f0 + k * 4 : a.dh), "r"(there ? 16 : 0) : "memory");
  }
}

template <int CG, int PLANES, int ACT, bool BACKWARD>
__global__ void __launch_bounds__(THREADS, 1) hidden_kernel(const __grid_constant__ Product p, const __grid_constant__ HiddenArgs a) {
  extern __shared__ uint8_t smem[];
  __shared__ gemm::Ctl ctl;
  // columns that are turned into results at a time: the warp's 32, or 16 where shared memory (one SM's tiles) or registers (three
  // terms a value) are short
  constexpr int COLS = CG == 2 && PLANES == 1 ? 32 : 16, CHUNKS = COLS / 4;
  run<CG, PLANES, false, false, DUAL>(p, smem, &ctl, [&](const Tile& t, int row0, int group, uint4* stage) {
    if constexpr (BACKWARD) fetch_block<CHUNKS>(stage, a, row0, (int64_t)t.n * (BN / 2) + group * 32);   // while the tile is computed
  }, [&](const Tile& t, float (&v)[EPI_COLS], int row0, int group, uint4* stage) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c0 = 0; c0 < 32; c0 += COLS) {
      const int64_t f0 = (int64_t)t.n * (BN / 2) + group * 32 + c0;
      if constexpr (BACKWARD) {
        if (c0 > 0) fetch_block<CHUNKS>(stage, a, row0, f0);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
      }
      // results over the accumulators: dg over g, du over u (h over g forward)
      uint4 h[COLS / 8];
      float hv[8];
#pragma unroll
      for (int i = 0; i < COLS; i += 4) {
        float4 d = make_float4(0.f, 0.f, 0.f, 0.f);
        if constexpr (BACKWARD) d = *reinterpret_cast<const float4*>(stage + gemm::epi_at<CHUNKS / 4>(lane, i / 4));
        const float dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float &g = v[c0 + i + k], &u = v[32 + c0 + i + k], slope;
          const float act = ff::activate<ACT>(g, BACKWARD ? &slope : nullptr), hk = act * u;
          if constexpr (BACKWARD) {
            g = dv[k] * u * slope;
            u = dv[k] * act;
          } else {
            g = hk;
          }
          if constexpr (BACKWARD && PLANES == 1) hv[i % 8 + k] = hk;
          // (three terms: h again from what dg and du are made of would need both; it goes through shared memory)
          if constexpr (BACKWARD && PLANES == 3) reinterpret_cast<float*>(stage + gemm::epi_at<CHUNKS / 4>(lane, i / 4))[k] = hk;
        }
        if constexpr (BACKWARD && PLANES == 1) {
          if (i % 8 == 4) {
            uint4 q[1];
            planes_of<1>(hv, q);
            h[i / 8] = q[0];
          }
        }
      }
      if constexpr (PLANES == 1) {
        if constexpr (!BACKWARD) {
#pragma unroll
          for (int i = 0; i < COLS / 8; ++i)
            h[i] = make_uint4(gemm::pack_bf16(v[c0 + 8 * i], v[c0 + 8 * i + 1]), gemm::pack_bf16(v[c0 + 8 * i + 2], v[c0 + 8 * i + 3]),
                              gemm::pack_bf16(v[c0 + 8 * i + 4], v[c0 + 8 * i + 5]), gemm::pack_bf16(v[c0 + 8 * i + 6], v[c0 + 8 * i + 7]));
          store_block(stage, h, a.h, a.ld, row0, a.rows, f0, a.F);
        } else {
          if (a.h) store_block(stage, h, a.h, a.ld, row0, a.rows, f0, a.F);
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const float* x = v + 32 * which + c0;
#pragma unroll
            for (int i = 0; i < COLS / 8; ++i)
              h[i] = make_uint4(gemm::pack_bf16(x[8 * i], x[8 * i + 1]), gemm::pack_bf16(x[8 * i + 2], x[8 * i + 3]),
                                gemm::pack_bf16(x[8 * i + 4], x[8 * i + 5]), gemm::pack_bf16(x[8 * i + 6], x[8 * i + 7]));
            store_block(stage, h, which ? a.du : a.dg, a.ld, row0, a.rows, f0, a.F);
          }
        }
      } else {
        // three planes of one result after another (hidden values above 3.396e38 count as infinite)
        auto put = [&](float* x, uint8_t* out) {
#pragma unroll
          for (int k = 0; k < PLANES; ++k) {
#pragma unroll
            for (int i = 0; i < COLS / 8; ++i)
              h[i] = make_uint4(term_of<false>(x[8 * i], x[8 * i + 1]), term_of<false>(x[8 * i + 2], x[8 * i + 3]),
                                term_of<false>(x[8 * i + 4], x[8 * i + 5]), term_of<false>(x[8 * i + 6], x[8 * i + 7]));
            store_block(stage, h, out + k * a.plane, a.ld, row0, a.rows, f0, a.F);
          }
        };
        if constexpr (BACKWARD) {
          if (a.h) {
            float x[COLS];
#pragma unroll
            for (int i = 0; i < COLS; i += 4) {
              const float4 d = *reinterpret_cast<const float4*>(stage + gemm::epi_at<CHUNKS / 4>(lane, i / 4));
              x[i] = d.x; x[i + 1] = d.y; x[i + 2] = d.z; x[i + 3] = d.w;
            }
            put(x, a.h);
          }
          put(v + c0, a.dg);
          put(v + 32 + c0, a.du);
        } else {
          put(v + c0, a.h);
        }
      }
    }
  });
}

// ---------------------------------------------------------------------------
// the other products
// ---------------------------------------------------------------------------
struct OutArgs {
  int64_t rows, cols, ld;          // of a part of the result; its rows are ld values apart
  void* out[2];                    // of the parts (TWO_M), else the first
  int bf16_out;
  int64_t m_rows;                  // rows of the tiles of a part: m tiles of a part start at row 0
  float* part;                     // f32 parts of split tiles: (splits, tiles, rows, BN)
};

template <int CG, int PLANES, bool A_MN, bool B_MN, int PARTS>
__global__ void __launch_bounds__(THREADS, 1) product_kernel(const __grid_constant__ Product p, const __grid_constant__ OutArgs a) {
  extern __shared__ uint8_t smem[];
  __shared__ gemm::Ctl ctl;
  run<CG, PLANES, A_MN, B_MN, PARTS>(p, smem, &ctl, [](const Tile&, int, int, uint4*) {},
                                     [&](const Tile& t, float (&v)[EPI_COLS], int row_of, int group, uint4* stage) {
    const int second = PARTS == TWO_M && t.m >= p.half;
    const int64_t row0 = second ? row_of - a.m_rows : row_of, n0 = (int64_t)t.n * BN + group * EPI_COLS;
    const int rows = (int)min((int64_t)32, a.rows - row0), cols = (int)min((int64_t)EPI_COLS, a.cols - n0);
    if (rows <= 0 || cols <= 0) return;
    if (t.split >= 0) {
      float* o = a.part + ((int64_t)t.split * BM * CG + row_of - t.m * BM * CG) * BN + group * EPI_COLS;
      gemm::by_rows<CG, float>(stage, v, true, rows, [&](int i, int c, uint4 q) { *reinterpret_cast<uint4*>(o + i * BN + c) = q; },
                               [](int, int, float) {});
    } else if (a.bf16_out) {
      bf16* o = static_cast<bf16*>(a.out[second]) + row0 * a.ld + n0;
      const bool wide = reinterpret_cast<uintptr_t>(o) % 16 == 0 && a.ld % 8 == 0 && cols % 8 == 0;
      gemm::by_rows<CG, bf16>(stage, v, wide, rows, [&](int i, int c, uint4 q) {
        if (c < cols) *reinterpret_cast<uint4*>(o + i * a.ld + c) = q;
      }, [&](int i, int c, bf16 x) {
        if (c < cols) o[i * a.ld + c] = x;
      });
    } else {
      float* o = static_cast<float*>(a.out[second]) + row0 * a.ld + n0;
      const bool wide = reinterpret_cast<uintptr_t>(o) % 16 == 0 && a.ld % 4 == 0 && cols % 4 == 0;
      gemm::by_rows<CG, float>(stage, v, wide, rows, [&](int i, int c, uint4 q) {
        if (c < cols) *reinterpret_cast<uint4*>(o + i * a.ld + c) = q;
      }, [&](int i, int c, float x) {
        if (c < cols) o[i * a.ld + c] = x;
      });
    }
  });
}

// Sum of the parts of split tiles, in order: a warp takes a row of a tile, 4 columns a lane and half.  Bound by L2.
template <int CG>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Product p, const __grid_constant__ OutArgs a) {
  ptx::griddep_wait();
  constexpr int ROWS = BM * CG;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tail = p.m_tiles * p.n_tiles - p.full;
  const int index = blockIdx.x / (ROWS / 8), r = blockIdx.x % (ROWS / 8) * 8 + warp;
  const Tile t = tile_of(p, p.full + index);
  const int second = a.out[1] != nullptr && t.m >= p.half;
  const int64_t row = (int64_t)t.m * ROWS + r - (second ? a.m_rows : 0);
  if (row >= a.rows) return;
  const float* q = a.part + ((int64_t)index * ROWS + r) * BN;
  const int64_t step = (int64_t)tail * ROWS * BN, n0 = (int64_t)t.n * BN, at = row * a.ld + n0;
  const bool wide = a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.out[second]) % 16 == 0;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int c = half * 128 + lane * 4;
    if (n0 + c >= a.cols) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j < p.splits; ++j) {
      const float4 x = *reinterpret_cast<const float4*>(q + j * step + c);
      v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
    if (wide && n0 + c + 4 <= a.cols) {
      if (a.bf16_out) *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out[second]) + at + c) = make_uint2(gemm::pack_bf16(v.x, v.y), gemm::pack_bf16(v.z, v.w));
      else *reinterpret_cast<float4*>(static_cast<float*>(a.out[second]) + at + c) = v;
    } else {
      const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (n0 + c + k >= a.cols) break;
        if (a.bf16_out) st(static_cast<bf16*>(a.out[second]) + at + c + k, w[k]);
        else static_cast<float*>(a.out[second])[at + c + k] = w[k];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int SMS = 148;   // of a B200
constexpr int MAX_SPLITS = 32;
constexpr int GROUP = 8;   // m tiles of a walk: the 74 tiles at work are then about as many rows as columns of tiles

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }
int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

// A matrix as the products read it.
struct Operand {
  const uint8_t* p;                // planes, `plane` bytes apart
  int64_t rows, dim, ld, plane;    // ld in values
};

// Tensor maps: K-major 64 values of a row x `box` rows; MN-major 64 values x 64 rows of the reduced dimension.
bool maps(CUtensorMap (&m)[3], const Operand& o, int planes, uint32_t box) {
  for (int i = 0; i < planes; ++i)
    if (!tc_map_2d(&m[i], o.p + i * o.plane, (uint64_t)o.dim, (uint64_t)o.rows, (uint64_t)o.ld * 2, box)) return false;
  return true;
}

// Which tiles are computed whole, and into how many parts the K range of the others goes.  Whole rounds of tiles fill all CTAs;
// those left over are split so that the last round is short (2560 x 7680 over 16384 tokens, 300 tiles on 74 pairs: 620 -> 525 us under the
// power limit; 4096 x 4096 over 12288: 335 -> 313).  In K blocks of a unit (its start and epilogue count as 12), and 8 bytes a value and part written and
// read again (a K block takes 0.37 us, which is 2.2 MB at 6 TB/s).
void pick_splits(int64_t tiles, int pairs, int64_t blocks, int per, int values, int* full, int* splits) {
  *full = (int)tiles;
  *splits = 1;
  const int64_t tail = tiles % pairs;
  if (tail == 0) return;
  double least = (double)(blocks * per + 12);
  for (int s = 2; s <= MAX_SPLITS && s <= blocks; ++s) {
    const double rounds = (double)((tail * s + pairs - 1) / pairs);
    const double cost = rounds * (double)((blocks + s - 1) / s * per + 12) + (double)(tail * s) * values * 3.6e-6 + 8.0;
    if (cost < least) {
      least = cost;
      *full = (int)(tiles - tail);
      *splits = s;
    }
  }
}

enum Step { Y, DH, DX, DW_IN, DW_OUT, STEPS };

// One product of a call.
struct Plan {
  int cg, full, splits, m_tiles, n_tiles, k_blocks, half, parts;
  int64_t rows, cols;              // of a part of the result

  int64_t tail() const { return (int64_t)m_tiles * n_tiles - full; }
  int64_t part_values() const { return tail() * splits * BM * cg * BN; }
};

Plan plan_of(int step, const ssd_gated_ff_params_t* p) {
  const int64_t T = p->tokens, D = p->dim, F = p->hidden, O = p->dim_out;
  Plan q{};
  q.parts = 1;
  int64_t k = 0;
  switch (step) {
    case Y: q.rows = T; q.cols = O; k = F; break;
    case DH: q.rows = T; q.cols = F; k = O; break;
    case DX: q.rows = T; q.cols = D; k = F; break;
    case DW_IN: q.rows = F; q.cols = D; k = T; q.parts = 2; break;
    default: q.rows = O; q.cols = F; k = T; break;
  }
  // one SM's tiles where a pair's second half would be empty
  q.cg = q.rows > BM || step >= DW_IN ? 2 : 1;
  q.m_tiles = cdiv(q.rows, BM * q.cg) * q.parts;
  q.n_tiles = cdiv(q.cols, BN);
  q.k_blocks = cdiv(k, BK) * (step == DX ? 2 : 1);
  q.half = step == DX ? q.k_blocks / 2 : q.m_tiles / 2;
  const int per = p->dtype == SSD_DTYPE_F32 ? 6 : 1;   // products a K block
  pick_splits((int64_t)q.m_tiles * q.n_tiles, SMS / q.cg, q.k_blocks, per, BM * q.cg * BN, &q.full, &q.splits);
  return q;
}

bool direct(const void* p, int64_t stride, int dtype) {
  return dtype == SSD_DTYPE_BF16 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0;
}

// Where everything lies in the workspace.
struct Layout {
  int planes;
  int64_t ldf;                     // of h, dg, du and dh
  size_t plane_h;                  // bytes of a plane of them
  size_t in[5], h, dg, du, dh, part, total;   // in: x, w_gate, w_up, w_down, dy (0: read as they are)
};

struct Inputs {
  const void* p[5];
  int64_t stride[5], rows[5], dim[5];
  int n;
};

// Whether a call needs dg and du, so dh as well; the gradient of w_down alone needs h, as the forward pass makes it.
bool goes_back(const ssd_gated_ff_grads_t* g) { return g && (g->grad_x || g->grad_w_gate); }

Inputs inputs_of(const ssd_gated_ff_params_t* p, const ssd_gated_ff_grads_t* g) {
  Inputs in{};
  const void* ptr[5] = {p->x, p->w_gate, p->w_up, g && !goes_back(g) ? nullptr : p->w_down, g ? g->grad_y : nullptr};   // NULL: not read
  const int64_t stride[5] = {p->x_stride_row, p->w_gate_stride_row, p->w_up_stride_row, p->w_down_stride_row, g ? g->grad_y_stride_row : 0};
  const int64_t rows[5] = {p->tokens, p->hidden, p->hidden, p->dim_out, p->tokens};
  const int64_t dim[5] = {p->dim, p->dim, p->dim, p->hidden, p->dim_out};
  in.n = g ? 5 : 4;
  for (int i = 0; i < in.n; ++i) {
    in.p[i] = ptr[i]; in.stride[i] = stride[i]; in.rows[i] = rows[i]; in.dim[i] = dim[i];
  }
  return in;
}

Layout layout_of(const ssd_gated_ff_params_t* p, const ssd_gated_ff_grads_t* g) {
  Layout q{};
  q.planes = p->dtype == SSD_DTYPE_F32 ? 3 : 1;
  q.ldf = up64(p->hidden);
  q.plane_h = up256((size_t)p->tokens * q.ldf * 2);
  size_t at = 256;   // the status word
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  const Inputs in = inputs_of(p, g);
  for (int i = 0; i < in.n; ++i)
    if (in.p[i] && !direct(in.p[i], in.stride[i], p->dtype)) q.in[i] = take((size_t)q.planes * up256((size_t)in.rows[i] * ((in.dim[i] + 7) / 8 * 8) * 2));
  if (!g || g->grad_w_down) q.h = take(q.planes * q.plane_h);
  int64_t part = 0;
  auto parts = [&](int step) {
    const Plan s = plan_of(step, p);
    part = std::max(part, s.part_values());
  };
  if (!g) {
    parts(Y);
  } else {
    if (goes_back(g)) {
      q.dg = take(q.planes * q.plane_h);
      q.du = take(q.planes * q.plane_h);
      q.dh = take((size_t)p->tokens * q.ldf * 4);
      parts(DH);
    }
    if (g->grad_x) parts(DX);
    if (g->grad_w_gate) parts(DW_IN);
    if (g->grad_w_down) parts(DW_OUT);
  }
  q.part = take((size_t)part * 4);
  q.total = at;
  return q;
}

#define FF_CHECK(call, where)                                     \
  do {                                                            \
    const cudaError_t e_ = (call);                                \
    if (e_ != cudaSuccess) {                                      \
      *at = where;                                                \
      return e_;                                                  \
    }                                                             \
  } while (0)

template <auto KERNEL, int CG, typename A>
cudaError_t launch_tiles(const Product& p, const A& a, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int smem = gemm::Shape<CG>::SMEM;
  const cudaError_t e = allow_smem((const void*)KERNEL, smem, &allowed);
  if (e != cudaSuccess) return e;
  const int64_t units = p.full + ((int64_t)p.m_tiles * p.n_tiles - p.full) * p.splits;
  if ((int64_t)p.m_tiles * p.n_tiles >= (int64_t(1) << 31) || units >= (int64_t(1) << 31) || (int64_t)p.k_blocks * MAX_SPLITS >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
  return launch_dependent(KERNEL, dim3((unsigned)(CG * std::min<int64_t>(units, SMS / CG))), THREADS, smem, CG, st, p, a);
}

// Segments of nearly the same length, at most `most`.
int even_segment(int blocks, int most) {
  const int n = (blocks + most - 1) / most;
  return (blocks + n - 1) / n;
}

template <int CG, int PLANES, bool BACKWARD>
cudaError_t launch_hidden(int act, const Product& p, const HiddenArgs& a, cudaStream_t st) {
  switch (act) {
    case SSD_ACT_GELU: return launch_tiles<hidden_kernel<CG, PLANES, SSD_ACT_GELU, BACKWARD>, CG>(p, a, st);
    case SSD_ACT_GELU_TANH: return launch_tiles<hidden_kernel<CG, PLANES, SSD_ACT_GELU_TANH, BACKWARD>, CG>(p, a, st);
    case SSD_ACT_RELU: return launch_tiles<hidden_kernel<CG, PLANES, SSD_ACT_RELU, BACKWARD>, CG>(p, a, st);
    default: return launch_tiles<hidden_kernel<CG, PLANES, SSD_ACT_SILU, BACKWARD>, CG>(p, a, st);
  }
}

template <int CG, int PLANES>
cudaError_t hidden(const ssd_gated_ff_params_t* p, const Layout& q, const Operand& x, const Operand& wg, const Operand& wu,
                   const HiddenArgs& a, bool clear, unsigned* status, cudaStream_t st) {
  Product g{};
  if (!maps(g.a[0], x, PLANES, BM) || !maps(g.b[0], wg, PLANES, BN / 2) || !maps(g.b[1], wu, PLANES, BN / 2)) return cudaErrorInvalidValue;
  g.m_tiles = cdiv(p->tokens, BM * CG);
  g.n_tiles = cdiv(p->hidden, BN / 2);
  g.k_blocks = cdiv(p->dim, BK);
  g.group = GROUP;
  g.full = g.m_tiles * g.n_tiles;
  g.splits = 1;
  g.segment = PLANES == 3 ? SEGMENT_F32 : even_segment(g.k_blocks, SEGMENT_BF16);
  g.clear = clear;
  g.status = status;
  return a.dh ? launch_hidden<CG, PLANES, true>(p->activation, g, a, st) : launch_hidden<CG, PLANES, false>(p->activation, g, a, st);
}

template <int CG, int PLANES, bool A_MN, bool B_MN, int PARTS>
cudaError_t product_as(const Plan& s, const Operand (&a)[2], const Operand (&b)[2], void* out0, void* out1, bool bf16_out, int64_t ld,
                       float* part, bool clear, unsigned* status, cudaStream_t st) {
  Product g{};
  const int pa = PARTS == TWO_K || PARTS == TWO_M ? 2 : 1, pb = PARTS == TWO_K ? 2 : 1;
  for (int i = 0; i < pa; ++i)
    if (!maps(g.a[i], a[i], PLANES, A_MN ? 64 : BM)) return cudaErrorInvalidValue;
  for (int i = 0; i < pb; ++i)
    if (!maps(g.b[i], b[i], PLANES, B_MN ? 64 : BN / CG)) return cudaErrorInvalidValue;
  g.m_tiles = s.m_tiles;
  g.n_tiles = s.n_tiles;
  g.k_blocks = s.k_blocks;
  g.half = s.half;
  g.group = GROUP;
  g.full = s.full;
  g.splits = s.splits;
  g.segment = PLANES == 3 ? SEGMENT_F32 : even_segment(s.k_blocks, A_MN ? SEGMENT_DW : SEGMENT_BF16);
  g.clear = clear;
  g.status = status;
  OutArgs o{};
  o.rows = s.rows;
  o.cols = s.cols;
  o.ld = ld;
  o.out[0] = out0;
  o.out[1] = out1;
  o.bf16_out = bf16_out;
  o.m_rows = (int64_t)s.half * BM * CG;
  o.part = part;
  const cudaError_t e = launch_tiles<product_kernel<CG, PLANES, A_MN, B_MN, PARTS>, CG>(g, o, st);
  if (e != cudaSuccess || s.tail() == 0) return e;
  return launch_dependent(join_kernel<CG>, dim3((unsigned)(s.tail() * (BM * CG / 8))), 256, 0, 1, st, g, o);
}

template <bool A_MN, bool B_MN, int PARTS, typename... Args>
cudaError_t product(int planes, const Plan& s, Args&&... args) {
  if constexpr (A_MN) {
    return planes == 3 ? product_as<2, 3, A_MN, B_MN, PARTS>(s, args...) : product_as<2, 1, A_MN, B_MN, PARTS>(s, args...);
  } else {
    if (s.cg == 2) return planes == 3 ? product_as<2, 3, A_MN, B_MN, PARTS>(s, args...) : product_as<2, 1, A_MN, B_MN, PARTS>(s, args...);
    return planes == 3 ? product_as<1, 3, A_MN, B_MN, PARTS>(s, args...) : product_as<1, 1, A_MN, B_MN, PARTS>(s, args...);
  }
}

template <typename... Args>
cudaError_t hidden_as(int planes, int64_t tokens, Args&&... args) {
  if (tokens > BM) return planes == 3 ? hidden<2, 3>(args...) : hidden<2, 1>(args...);
  return planes == 3 ? hidden<1, 3>(args...) : hidden<1, 1>(args...);
}

}  // namespace

size_t gated_ff_workspace(const ssd_gated_ff_params_t* p, const ssd_gated_ff_grads_t* g) {
  if (!g && gated_ff_is_few(p)) return gated_ff_few_workspace(p);
  return layout_of(p, g).total;
}

cudaError_t launch_gated_ff(const ssd_gated_ff_params_t* p, const ssd_gated_ff_grads_t* g, void* workspace, cudaStream_t st, const char** at) {
  if (!g && gated_ff_is_few(p)) return launch_gated_ff_few(p, workspace, st, at);
  const Layout q = layout_of(p, g);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  unsigned* status = reinterpret_cast<unsigned*>(ws);
  if (g && !goes_back(g) && !g->grad_w_down) {   // nothing is wanted
    FF_CHECK(cudaMemsetAsync(status, 0, sizeof(*status), st), "status");
    return cudaSuccess;
  }
  const bool bf = p->dtype == SSD_DTYPE_BF16;
  const Inputs in = inputs_of(p, g);
  Operand op[5] = {};
  PackArgs pack{};
  pack.status = status;
  for (int i = 0; i < in.n; ++i) {
    op[i] = {static_cast<const uint8_t*>(in.p[i]), in.rows[i], in.dim[i], in.stride[i], 0};
    if (!in.p[i] || direct(in.p[i], in.stride[i], p->dtype)) continue;
    Pack& m = pack.m[pack.n++];
    m.src = in.p[i]; m.stride = in.stride[i]; m.rows = in.rows[i]; m.dim = in.dim[i];
    m.ld = (in.dim[i] + 7) / 8 * 8;
    m.dst = ws + q.in[i];
    m.plane = (int64_t)up256((size_t)m.rows * m.ld * 2);
    m.first = pack.units;
    pack.units += m.rows * ((m.ld + 255) / 256);
    op[i].p = m.dst;
    op[i].ld = m.ld;
    op[i].plane = m.plane;
  }
  bool clear = true;   // the next launch clears the status word
  if (pack.n) {
    const unsigned ctas = (unsigned)std::min<int64_t>((pack.units + 7) / 8, SMS * 16);
    if (bf) pack_kernel<bf16><<<ctas, 256, 0, st>>>(pack);
    else pack_kernel<float><<<ctas, 256, 0, st>>>(pack);
    FF_CHECK(cudaGetLastError(), "operands");
    clear = false;
  }
  const Operand &x = op[0], &wg = op[1], &wu = op[2], &wd = op[3];
  float* part = reinterpret_cast<float*>(ws + q.part);
  auto middle = [&](size_t o) { return Operand{ws + o, p->tokens, p->hidden, q.ldf, (int64_t)q.plane_h}; };
  const Operand h = middle(q.h);
  HiddenArgs ha{};
  ha.rows = (int)p->tokens;
  ha.F = p->hidden;
  ha.ld = q.ldf;
  ha.h = q.h ? ws + q.h : nullptr;
  ha.plane = (int64_t)q.plane_h;
  const Operand none{};
  if (!g) {
    FF_CHECK(hidden_as(q.planes, p->tokens, p, q, x, wg, wu, ha, clear, status, st), "gate and up");
    const Operand a[2] = {h, none}, b[2] = {wd, none};
    FF_CHECK((product<false, false, ONE>(q.planes, plan_of(Y, p), a, b, p->y, (void*)nullptr, bf, p->dim_out, part, false, status, st)), "down");
    return cudaSuccess;
  }
  const Operand& dy = op[4];
  const Operand dg = middle(q.dg), du = middle(q.du);
  if (goes_back(g)) {
    const Operand a[2] = {dy, none}, b[2] = {wd, none};
    FF_CHECK((product<false, true, ONE>(q.planes, plan_of(DH, p), a, b, ws + q.dh, (void*)nullptr, false, q.ldf, part, clear, status, st)), "grad_hidden");
    clear = false;
    ha.dg = ws + q.dg;
    ha.du = ws + q.du;
    ha.dh = reinterpret_cast<const float*>(ws + q.dh);
  }
  FF_CHECK(hidden_as(q.planes, p->tokens, p, q, x, wg, wu, ha, clear, status, st), "gate and up");
  if (g->grad_x) {
    const Operand a[2] = {dg, du}, b[2] = {wg, wu};
    FF_CHECK((product<false, true, TWO_K>(q.planes, plan_of(DX, p), a, b, g->grad_x, (void*)nullptr, bf, p->dim, part, false, status, st)), "grad_x");
  }
  const bool bw = g->grad_weight_dtype == SSD_DTYPE_BF16;
  if (g->grad_w_gate) {
    const Operand a[2] = {dg, du}, b[2] = {x, none};
    FF_CHECK((product<true, true, TWO_M>(q.planes, plan_of(DW_IN, p), a, b, g->grad_w_gate, g->grad_w_up, bw, p->dim, part, false, status, st)), "grad_w_gate");
  }
  if (g->grad_w_down) {
    const Operand a[2] = {dy, none}, b[2] = {h, none};
    FF_CHECK((product<true, true, ONE>(q.planes, plan_of(DW_OUT, p), a, b, g->grad_w_down, (void*)nullptr, bw, p->hidden, part, false, status, st)), "grad_w_down");
  }
  return cudaSuccess;
}

}  // namespace ssd
