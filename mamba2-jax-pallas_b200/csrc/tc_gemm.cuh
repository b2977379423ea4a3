// Tensor-core GEMM core for the language-model head: D = A B^T (+ epilogue), 16-bit operands,
// f32 accumulation.
//
// One persistent CTA per SM, or a pair of CTAs per two SMs (CG = 2: tcgen05 cta_group::2, one
// 256 x 256 tile per pair).  The pair halves what each SM fetches of B, in shared memory and
// from L2: a 128 x 256 tile per SM needs 48 KB per 64-wide K block, which at the tensor
// pipe's rate is 16 TB/s over the GPU; a pair needs 32 KB per SM.  Warps:
//   0     TMA producer: A and B boxes into a ring of shared-memory stages
//   1     MMA issuer (the pair's first CTA only issues): four K = 16 MMAs per stage
//   2..17 epilogue: warp w reads the TMEM lanes of quadrant w % 4, 64 columns at (w - 2) / 4 * 64
// (16 epilogue warps of 64 columns: with 8 of 128 the logits of 900 x 32003 x 1000 took 84 us, so 81.)
// Bound by the tensor pipe where K is long: 4096 x 131072 x 4096 without a store takes 2.68 ms, 1.64
// PFLOP/s (8192 x 50000 x 2560: the pipe active 98 % of the cycles); by what an epilogue writes where
// K is short.
// Two accumulators (2 x 256 TMEM columns) let the reading of one overlap the MMAs into the
// other.  Operands are K-major (the reduced dimension contiguous in memory) or MN-major (the
// other one contiguous), so no operand is ever transposed in memory.
//
// The tensor core's f32 adds truncate: over K = 4096 a dot product loses about 1e-5 of its
// value, always towards zero.  So a tile's K range runs in segments, each from zero in its own
// TMEM accumulator, and the epilogue warps add the segments in registers, rounding to nearest:
// 64 values per thread.
//
// f32 operands come as two f16 planes of the values times a power of two, v = hi + lo, and a K
// block takes the products hi*hi, hi*lo, lo*hi from two stages.  Two f16 hold 22 bits of a value down
// to 2^-16 of the largest, so three products carry what f32 carries; two bf16 hold 16.
//
// Every wait is bounded; one that gives up sets the status word and the CTA drains and ends.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace ssd {
namespace gemm {

constexpr int BK = 64;                    // one 128-byte swizzled row
constexpr int BN = 256;                   // columns of a tile
constexpr int BM = 128;                   // rows of a CTA's part of a tile
constexpr int EPI_WARPS = 16;
constexpr int EPI_COLS = 64;               // columns of an epilogue warp
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr long long WAIT_CYCLES = 4000000000LL;   // about 2 s at the boost clock

// Each epilogue warp turns its 32 rows through shared memory, so that what it writes to global
// memory are runs of one row and not one value of 32 rows: whole 128-byte lines in a pair's
// tiles, 64 bytes where shared memory is shorter.  A row's 16-byte chunks are permuted by its number, which keeps the accesses of a
// quarter-warp in different banks, by rows and by columns.
template <int CG>
struct Shape {
  static constexpr int STAGES = CG == 2 ? 5 : 4;
  static constexpr int EPI_ROW = CG == 2 ? 128 : 64;         // bytes of a staged row
  static constexpr int EPI_WARP_BYTES = 32 * EPI_ROW;
  static constexpr int A_BYTES = BM * BK * 2;
  static constexpr int B_BYTES = BN / CG * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * EPI_WARP_BYTES + 1024;   // + alignment
};

struct Ctl {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drain;
  uint32_t tmem;
  volatile uint32_t abort;
};

// What the kernel runs over.  Tiles are numbered m fastest or n fastest; a tile's K range is
// split into `splits` parts, each its own unit of work.
// A dimension whose size only the device knows (rows that count) is `limit`: rows from
// `limit_from` on, at most `rows`; it bounds the m tiles, or the K blocks with limit_k.
struct Problem {
  CUtensorMap a[2], b[2];                 // planes hi and lo (lo unused for bf16 operands)
  const int* limit;
  int limit_from, rows, limit_k;
  int m_tiles, n_tiles;                   // m tiles of CG * 128 rows
  int max_splits;                         // of the K range, decided on the device (pick_splits)
  int64_t part_values;                    // room for the parts
  int rows_out, cols;                     // of the result (limit_k; else its rows are the live ones)
  int k_blocks;                           // of 64
  int planes;                             // 1 (bf16), or 2 (f32 as two f16 planes, three products)
  int segment;                            // K blocks that are summed in TMEM
  int m_fastest;
  unsigned* status;
};

struct Tile {
  int m, n, split, k0, k1;
};

// Rows that count, of those that the launch was made for.
__device__ __forceinline__ int live_rows(const Problem& p) { return min(max(*p.limit - p.limit_from, 0), p.rows); }

// Parts of the K range: enough units of work to fill the GPU where there are few tiles.  Cost in
// K blocks of one wave of units (a unit's start and epilogue count as 12), plus 8 bytes per
// value and part written and read again (at 6 TB/s; a K block takes 0.37 us).  A warp tries 32.
template <int CG>
__device__ __forceinline__ int pick_splits(int tiles, int blocks, int64_t values, int max_splits, int64_t part_values) {
  if (max_splits <= 1 || tiles <= 0) return 1;
  const int s = (threadIdx.x & 31) + 1, ctas = 148 / CG;   // `blocks`: as many MMAs as a bf16 K block
  float cost = (float)((tiles * s + ctas - 1) / ctas) * (float)((blocks + s - 1) / s + 12);
  if (s > 1) cost += (float)s * (float)values * 3.6e-6f + 8.f;
  if (s > max_splits || s * values > part_values || s > blocks) cost = 3e38f;
  if (s == 1) cost = fminf(cost, 1e38f);
  // positive floats order like their bits; the lowest lane of the least cost
  const unsigned bits = __float_as_uint(cost), least = __reduce_min_sync(0xffffffffu, bits);
  return __ffs(__ballot_sync(0xffffffffu, bits == least));
}

__device__ __forceinline__ Tile tile_at(const Problem& p, unsigned m_tiles, int k_blocks, unsigned splits, unsigned u) {
  Tile t;
  const unsigned n_tiles = (unsigned)p.n_tiles, per = m_tiles * n_tiles;
  const unsigned split = splits == 1 ? 0 : u / per, r = u - split * per;
  const unsigned a = p.m_fastest ? m_tiles : n_tiles, q = r / a, rest = r - q * a;
  t.split = (int)split;
  t.n = (int)(p.m_fastest ? q : rest);
  t.m = (int)(p.m_fastest ? rest : q);
  t.k0 = splits == 1 ? 0 : (int)((unsigned)k_blocks * split / splits);   // splits <= 32
  t.k1 = splits == 1 ? k_blocks : (int)((unsigned)k_blocks * (split + 1) / splits);
  return t;
}

// A probe that lets the hardware suspend the thread for up to 20 us (20 ns to 1 ms measured
// alike): 16 waiting epilogue warps that poll cost 10 % of a power-bound GEMM.
__device__ __forceinline__ bool probe(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(ptx::smem_u32(bar)), "r"(parity), "r"(20000)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ bool wait(Ctl* c, uint64_t* bar, uint32_t parity, unsigned* status, int id) {
  if (probe(bar, parity)) return true;
  const long long t0 = clock64();
  while (!probe(bar, parity)) {
    if (c->abort) return false;
    if (clock64() - t0 > WAIT_CYCLES) {
      atomicCAS(status, 0u, (unsigned)(0x100 | id));
      c->abort = 1;
      return false;
    }
  }
  return true;
}

// The parts of a launch, given its live rows: the GEMM and what adds the parts agree on it.
template <int CG>
__device__ __forceinline__ int splits_of(const Problem& p, int live) {
  const int m_tiles = p.limit_k ? p.m_tiles : (live + BM * CG - 1) / (BM * CG);
  const int k_blocks = p.limit_k ? (live + BK - 1) / BK : p.k_blocks;
  return pick_splits<CG>(m_tiles * p.n_tiles, k_blocks * (2 * p.planes - 1), (int64_t)(p.limit_k ? p.rows_out : live) * p.cols,
                         p.max_splits, p.part_values);
}

// One thread of a converged warp.  The compiler knows that what this guards runs on one thread and
// keeps descriptors and barrier addresses in uniform registers; under `lane == 0` four MMAs and
// their commit took 335 + 66 cycles to issue, of the 512 that they take to run, and the tensor pipe
// was busy 70 % of the time (85 % so: 8192 x 50000 x 2560, 1.52 -> 1.34 ms).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// ---- the pair's forms of the PTX wrappers ------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared::cluster address of the same variable in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
// What the arrival orders are TMEM reads, by tcgen05 fences on both sides; a release at cluster
// scope would also wait for the thread's global stores (that and fewer spilled registers took the
// weight's gradient of 64 x 95131 x 1400, one K block a tile, from 153 to 82 us).
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    ptx::mma_f16(d, a, b, idesc, acc);
}

// Arrive on `bar` (of both CTAs of a pair) once this thread's MMAs have completed.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            ptx::smem_u32(bar)), "h"((uint16_t)3) : "memory");
  else
    ptx::mma_commit(bar);
}

template <int CG>
__device__ __forceinline__ void tmem_alloc_all(uint32_t* dst) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(dst)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    ptx::tmem_alloc(dst, 512);
    ptx::tmem_relinquish();
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free_all(uint32_t t) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(512) : "memory");
  else
    ptx::tmem_dealloc(t, 512);
}

// Instruction descriptor: f16 operands have format 0, bf16 format 1.
template <int CG, int PLANES, bool A_MN, bool B_MN>
__device__ __forceinline__ constexpr uint32_t idesc() {
  constexpr uint32_t ID = ptx::idesc_bf16_f32(BM * CG, BN, A_MN, B_MN);
  return PLANES == 2 ? ID & ~((1u << 7) | (1u << 10)) : ID;
}

// Where chunk `c` of a staged row lies, in 16-byte units.
template <int CG>
__device__ __forceinline__ int epi_at(int row, int c) {
  return CG == 2 ? row * 8 + (c ^ (row & 7)) : row * 4 + (c ^ ((row >> 1) & 3));
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The warp's 32 x 64 block as values of T, by rows.  With `wide`, put(i, c, q) for every 16 bytes q
// (row i, columns from c on); else put1(i, c, x) for every value, neighbouring lanes at
// neighbouring columns.
template <int CG, typename T, typename Put, typename Put1>
__device__ __forceinline__ void by_rows(uint4* stage, const float (&v)[EPI_COLS], bool wide, int rows, Put&& put,
                                        Put1&& put1) {
  constexpr int CHUNKS = Shape<CG>::EPI_ROW / 16, PER = 16 / sizeof(T), COLS = CHUNKS * PER;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int at = 0; at < EPI_COLS; at += COLS) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const float* x = v + at + i * PER;
      if constexpr (sizeof(T) == 4)
        stage[epi_at<CG>(lane, i)] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      else
        stage[epi_at<CG>(lane, i)] = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
    }
    __syncwarp();
    if (wide) {
#pragma unroll 2
      for (int j = 0; j < CHUNKS; ++j) {
        const int i = j * (32 / CHUNKS) + lane / CHUNKS, c = lane % CHUNKS;
        if (i < rows) put(i, at + c * PER, stage[epi_at<CG>(i, c)]);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < rows; ++i) {
#pragma unroll 1
        for (int c0 = 0; c0 < COLS; c0 += 32) {
          const int c = c0 + lane;
          if (c < COLS) put1(i, at + c, reinterpret_cast<const T*>(stage + epi_at<CG>(i, c / PER))[c % PER]);
        }
      }
    }
  }
}

// One K block: A at sa and B at sb in shared memory.
template <int CG, bool A_MN, bool B_MN>
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t sa, uint32_t sb, uint32_t id, bool accumulate) {
#pragma unroll
  for (int k = 0; k < BK / 16; ++k) {
    const uint64_t da = A_MN ? ptx::sdesc_sw128(sa + k * 2048, 8192, 1024) : ptx::sdesc_sw128(sa + k * 32, 16, 1024);
    const uint64_t db = B_MN ? ptx::sdesc_sw128(sb + k * 2048, 8192, 1024) : ptx::sdesc_sw128(sb + k * 32, 16, 1024);
    mma<CG>(d, da, db, id, (accumulate || k > 0) ? 1u : 0u);
  }
}

// The kernel's body.  prep() runs on every thread once the launches before are complete.  epi(tile, v, row0, first column, rows that count, splits, stage) runs on each
// epilogue thread; v holds 64 values of row row0 + lane; `splits` parts of the K range.
template <int CG, int PLANES, bool A_MN, bool B_MN, typename Prep, typename Epi>
__device__ __forceinline__ void run(const Problem& p, uint8_t* smem_raw, Ctl* c, Prep&& prep, Epi&& epi) {
  using S = Shape<CG>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
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
  if (warp == 1) tmem_alloc_all<CG>(&c->tmem);
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  ptx::tc_fence_after();
  const uint32_t tmem = c->tmem;
  ptx::griddep_wait();   // all above needs nothing from the launches before
  prep();
  const int live = live_rows(p);
  const int m_tiles = p.limit_k ? p.m_tiles : (live + BM * CG - 1) / (BM * CG);
  const int k_blocks = p.limit_k ? (live + BK - 1) / BK : p.k_blocks;
  const int splits = splits_of<CG>(p, live);
  const unsigned unit0 = blockIdx.x / CG, units = (unsigned)m_tiles * p.n_tiles * splits, step = gridDim.x / CG;   // below 2^31
  const uint32_t smem0 = ptx::smem_u32(smem);

  if (warp == 0) {
    if (elect_one()) {
      for (int i = 0; i < PLANES; ++i) {
        ptx::prefetch_tmap(&p.a[i]);
        ptx::prefetch_tmap(&p.b[i]);
      }
      uint32_t it = 0, s = 0, phase = 1;   // stage, and the parity of its last release
      bool ok = true;
      for (unsigned u = unit0; ok && u < units; u += step) {
        const Tile t = tile_at(p, m_tiles, k_blocks, splits, u);
        const int m0 = (t.m * CG + (int)rank) * BM, n0 = t.n * BN + (int)rank * (BN / CG);
        for (int kb = t.k0; ok && kb < t.k1; ++kb) {
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl, ++it) {
            // (a barrier's phase before its first counts as complete)
            if (!wait(c, &c->empty[s], phase, p.status, 1)) {
              ok = false;
              break;
            }
            const uint32_t sa = smem0 + s * S::STAGE_BYTES, sb = sa + S::A_BYTES;
            uint32_t bar = ptx::smem_u32(&c->full[s]);
            // the pair's first CTA counts the bytes of both
            if (rank == 0) ptx::mbar_arrive_expect_tx(&c->full[s], CG * S::STAGE_BYTES);
            if constexpr (CG == 2) bar = map_rank(bar, 0);
            const int k = kb * BK;
            if constexpr (A_MN) {
              for (int i = 0; i < BM / 64; ++i) tma_load_2d<CG>(sa + i * 8192, &p.a[pl], bar, m0 + 64 * i, k);
            } else {
              tma_load_2d<CG>(sa, &p.a[pl], bar, k, m0);
            }
            if constexpr (B_MN) {
              for (int i = 0; i < BN / CG / 64; ++i) tma_load_2d<CG>(sb + i * 8192, &p.b[pl], bar, n0 + 64 * i, k);
            } else {
              tma_load_2d<CG>(sb, &p.b[pl], bar, k, n0);
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
          while (!ptx::mbar_try_wait(&c->full[j % S::STAGES], (j / S::STAGES) & 1) && clock64() - t0 < WAIT_CYCLES) {
          }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t ID = idesc<CG, PLANES, A_MN, B_MN>();
      uint32_t s = 0, phase = 0, n = 0;
      bool ok = true;
      for (unsigned u = unit0; ok && u < units; u += step) {
        const Tile t = tile_at(p, m_tiles, k_blocks, splits, u);
        uint32_t d = 0;
        for (int kb = t.k0, left = 0; kb < t.k1; ++kb, --left) {
          const bool first = left == 0;
          if (first) {
            left = min(p.segment, t.k1 - kb);
            if (n >= 2 && !wait(c, &c->acc_empty[n & 1], ((n >> 1) - 1) & 1, p.status, 2)) {
              ok = false;
              break;
            }
            ptx::tc_fence_after();
            d = tmem + (n & 1) * BN;
          }
          if (!wait(c, &c->full[s], phase, p.status, 3)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t sa = smem0 + s * S::STAGE_BYTES;
          uint64_t* const done = &c->empty[s];
          mma_block<CG, A_MN, B_MN>(d, sa, sa + S::A_BYTES, ID, !first);
          if (++s == S::STAGES) {
            s = 0;
            phase ^= 1;
          }
          if constexpr (PLANES == 2) {   // the low planes lie in the next stage
            if (!wait(c, &c->full[s], phase, p.status, 3)) {
              ok = false;
              break;
            }
            ptx::tc_fence_after();
            const uint32_t sl = smem0 + s * S::STAGE_BYTES;
            mma_block<CG, A_MN, B_MN>(d, sa, sl + S::A_BYTES, ID, true);
            mma_block<CG, A_MN, B_MN>(d, sl, sa + S::A_BYTES, ID, true);
            commit<CG>(&c->empty[s]);
            if (++s == S::STAGES) {
              s = 0;
              phase ^= 1;
            }
          }
          commit<CG>(done);
          if (left == 1) {
            commit<CG>(&c->acc_full[n & 1]);
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
        while (!ptx::mbar_try_wait(&c->drain, 0) && clock64() - t0 < WAIT_CYCLES) {
        }
      }
    }
  } else {
    const int quad = warp & 3, col = (warp - 2) / 4 * EPI_COLS;
    uint4* stage = reinterpret_cast<uint4*>(smem + S::STAGES * S::STAGE_BYTES + (warp - 2) * S::EPI_WARP_BYTES);
    uint32_t n = 0;
    bool ok = true;
    for (unsigned u = unit0; ok && u < units; u += step) {
      const Tile t = tile_at(p, m_tiles, k_blocks, splits, u);
      float v[EPI_COLS];
#pragma unroll
      for (int i = 0; i < EPI_COLS; ++i) v[i] = 0.f;
      for (int left = t.k1 - t.k0; left > 0; left -= p.segment, ++n) {
        // one lane waits for the warp, so that the warp stays converged for its TMEM loads
        int there = 0;
        if (lane == 0) there = wait(c, &c->acc_full[n & 1], (n >> 1) & 1, p.status, 4);
        if (!__shfl_sync(0xffffffffu, there, 0)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t from = tmem + (n & 1) * BN + col + ((uint32_t)(32 * quad) << 16);
#pragma unroll
        for (int ch = 0; ch < EPI_COLS / 16; ++ch) {
          float x[16];
          ptx::tmem_ld16(from + 16 * ch, x);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[16 * ch + i] += x[i];
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            arrive_remote(map_rank(ptx::smem_u32(&c->acc_empty[n & 1]), 0));
          else
            ptx::mbar_arrive(&c->acc_empty[n & 1]);
        }
      }
      if (ok) epi(t, v, (t.m * CG + (int)rank) * BM + 32 * quad, t.n * BN + col, live, splits, stage);
    }
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();   // no CTA leaves while its peer may still signal it
  if (warp == 1) {
    ptx::tc_fence_after();
    tmem_free_all<CG>(tmem);
  }
  if constexpr (CG == 2) cluster_sync_all();
}

}  // namespace gemm
}  // namespace ssd
