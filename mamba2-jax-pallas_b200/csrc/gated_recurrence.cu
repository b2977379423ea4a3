// Gated linear recurrence over long sequences, its backward pass and its single-token step.
//
//   k = scale softplus(decay);  la_t = -k sigmoid(decay_gate_t);  a_t = exp(la_t)
//   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(input_gate_t) x_t;  y_t = h_t
//
// per channel; where a packed sequence starts, h_{t-1} is 0.  Backward, with w_t = sigmoid(i_t) x_t,
// b_t = sqrt(1 - a_t^2) and g_t the gradient that reaches y_t:
//
//   delta_t = g_t + c_{t+1};  c_t = a_t delta_t (0 where a sequence starts)
//   m_t = la_t a_t (h_{t-1} - a_t w_t / b_t)      (d h_t / d log la_t; its second term is 0 where b_t is)
//   dr = delta m (1 - sigmoid(r));  dx = delta b sigmoid(i);  di = delta b w (1 - sigmoid(i))
//   d decay = sigmoid(decay) / softplus(decay) sum delta m;  dh_0 = c_0
//
// Both passes are bound by HBM (8 and 14 bytes per bf16 value), and close behind it by the issue slots and the special-function
// unit: 32 and 68 instructions and 4 and 5 special functions a value, the gates' above all.  64 x 512 x 5120 bf16: forward 229 us
// (5.9 TB/s), gradients 456 us (5.2 TB/s).  With few rows and channels the sequence is the only parallelism left: 1 x 32768 x 5120
// in clusters of 5 forward 325 us (4.1 TB/s), gradients 642 us; 1 x 65536 x 256 102 and 175 us.  Packed, 16 sequences: 349 and 772.
//
// A step is the map h -> a h + b; maps compose, so a run of steps is one pair (P, H).  Warps take 16
// steps (8 backward) of 128 bytes of channels (a lane: one 32-bit word, 2 bf16 or 1 f32 channel), CTAs
// 4 such warps, and a cluster of CTAs that many tiles of one channel group side by side: every
// warp scans its steps from zero, the CTA's warps exchange their maps through shared memory, the
// cluster's CTAs theirs through distributed shared memory (st.async, which counts its bytes on the
// receiver's barrier: a cluster barrier's release would wait for the outputs' stores as well), and each warp runs its
// steps again from the state that then is known, out of registers.  The cluster walks along the
// sequence, so the inputs are read once and the carry never leaves the SMs.  Sums are made in a fixed order.
//
// A state that lives for thousands of steps has a near 1, where errors of one sign in a add up (an exponential
// that is half a unit too small on average leaves states 2e-6 off): a is 1 + expm1(la) there, rounded once,
// and 1 - a^2 comes from expm1 as well.
#include <algorithm>

#include "common.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "ssd_kernels.h"

namespace ssd {
namespace {

constexpr int FWD_STEPS = 16, BWD_STEPS = 8;   // of a warp
constexpr int POINT = 32;        // tokens between two checkpoints
constexpr int MAX_WARPS = 16;    // of an SM, by registers
constexpr int MAX_CLUSTER = 16;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESTART = -1.f;   // in a map's P: a sequence starts in it, what came before is dropped
constexpr long long WAIT_CYCLES = 4000000000LL;   // about 2 s at the boost clock

// ---- a lane's channels: one f32, or two in a packed pair --------------------------------------
typedef unsigned long long pair_t;

__device__ __forceinline__ pair_t pack(float a, float b) {
  pair_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 unpack(pair_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ pair_t mul(pair_t a, pair_t b) {
  pair_t d;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ pair_t add(pair_t a, pair_t b) {
  pair_t d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ pair_t fma(pair_t a, pair_t b, pair_t c) {
  pair_t d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }

__device__ __forceinline__ float ex2(float v) {
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float rcp(float v) {
  float d;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float rsq(float v) {
  float d;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float root(float v) {
  float d;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
  return d;
}
template <typename F>
__device__ __forceinline__ float each(float a, F&& f) { return f(a); }
template <typename F>
__device__ __forceinline__ pair_t each(pair_t a, F&& f) {
  const float2 u = unpack(a);
  return pack(f(u.x), f(u.y));
}
template <typename F>
__device__ __forceinline__ float each(float a, float b, F&& f) { return f(a, b); }
template <typename F>
__device__ __forceinline__ pair_t each(pair_t a, pair_t b, F&& f) {
  const float2 u = unpack(a), v = unpack(b);
  return pack(f(u.x, v.x), f(u.y, v.y));
}
template <typename V>
__device__ __forceinline__ V all(float v);
template <>
__device__ __forceinline__ float all<float>(float v) { return v; }
template <>
__device__ __forceinline__ pair_t all<pair_t>(float v) { return pack(v, v); }

// A lane's 32-bit word of a row, and its channels' f32 values in memory.
template <typename T>
struct Lane;
template <>
struct Lane<bf16> {
  static constexpr int CH = 2;
  typedef pair_t V;
  struct alignas(16) Map { float p0, h0, p1, h1; };
  static __device__ __forceinline__ V get(uint32_t u) { return pack(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t put(V v) {
    const float2 f = unpack(v);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ Map map(V p, V h) {
    const float2 a = unpack(p), b = unpack(h);
    return {a.x, b.x, a.y, b.y};
  }
  static __device__ __forceinline__ V load(const float* p, int64_t c, int64_t D, float none = 0.f) {
    return pack(c < D ? p[c] : none, c + 1 < D ? p[c + 1] : none);
  }
  static __device__ __forceinline__ void store(float* p, int64_t c, int64_t D, V v) {
    const float2 f = unpack(v);
    if (c < D) p[c] = f.x;
    if (c + 1 < D) p[c + 1] = f.y;
  }
};
template <>
struct Lane<float> {
  static constexpr int CH = 1;
  typedef float V;
  struct alignas(8) Map { float p0, h0; };
  static __device__ __forceinline__ V get(uint32_t u) { return __uint_as_float(u); }
  static __device__ __forceinline__ uint32_t put(V v) { return __float_as_uint(v); }
  static __device__ __forceinline__ Map map(V p, V h) { return {p, h}; }
  static __device__ __forceinline__ V load(const float* p, int64_t c, int64_t D, float none = 0.f) { return c < D ? p[c] : none; }
  static __device__ __forceinline__ void store(float* p, int64_t c, int64_t D, V v) {
    if (c < D) p[c] = v;
  }
};
__device__ __forceinline__ pair_t map_p(const Lane<bf16>::Map& m) { return pack(m.p0, m.p1); }
__device__ __forceinline__ pair_t map_h(const Lane<bf16>::Map& m) { return pack(m.h0, m.h1); }
__device__ __forceinline__ float map_p(const Lane<float>::Map& m) { return m.p0; }
__device__ __forceinline__ float map_h(const Lane<float>::Map& m) { return m.h0; }

// What a run of steps makes of the state before it.  (A restart is one of all channels: of the token.)
template <bool PACKED, typename M, typename V>
__device__ __forceinline__ V through(const M& m, V h) {
  if (PACKED && m.p0 < 0.f) return map_h(m);
  return fma(map_p(m), h, map_h(m));
}
template <bool PACKED, typename M, typename V>
__device__ __forceinline__ void compose(const M& m, V& P, V& H) {   // (P, H) then m
  const bool restart = PACKED && m.p0 < 0.f;
  H = restart ? map_h(m) : fma(map_p(m), H, map_h(m));
  if constexpr (PACKED) {
    // a P that is negative already stays so: it is RESTART, and m's is 0 at least, so keep it apart
    P = restart ? map_p(m) : each(P, map_p(m), [](float a, float b) { return a < 0.f ? a : a * b; });
  } else {
    P = mul(P, map_p(m));
  }
}

// The CTA's warps meet; whether a sequence starts in any of their steps.
template <bool PACKED>
__device__ __forceinline__ bool meet(bool mine) {
  if constexpr (PACKED) return __syncthreads_or(mine);
  __syncthreads();
  return false;
}

// ---- per-channel and per-value arithmetic --------------------------------------------------
// e^v of v up to 80, within 2 units, where the approximate instruction's 2^-22 would be one error of all of a channel's steps:
// v = n ln 2 + f in two parts (Cody and Waite), the series up to f^7 (5e-9).  0 where e^v is below 2^-126, however far: the series
// holds for what v is reduced to, so v is cut off before that.  NaN stays.
__device__ __forceinline__ float exp_near(float v) {
  v = v < -100.f ? -100.f : v;
  const float n = rintf(v * LOG2E);
  const float f = fmaf(n, -3.1946183e-5f, fmaf(n, -0.693115234375f, v));   // n times the first is exact
  const float p = fmaf(f, fmaf(f, fmaf(f, fmaf(f, fmaf(f, fmaf(f, fmaf(f, 1.f / 5040, 1.f / 720), 1.f / 120), 1.f / 24), 1.f / 6), 0.5f), 1.f), 1.f);
  return p * exp2f(n);
}
__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(exp_near(v)); }
// A channel's k.  Beyond float32 it is 2^127, not infinite: a closed gate's sigmoid is 0, and 0 times it has to be 0 (the steps behind
// the last token are closed gates, and so are gates below -88).  NaN stays.
__device__ __forceinline__ float rate_of(float scale, float decay) {
  const float k = scale * softplus(decay);
  return k > 0x1p127f ? 0x1p127f : k;
}

// 1 / (1 + e^-v); 0 where e^-v is beyond 2^126.  (Two at once by one reciprocal of the product need a second form for large
// products, whose registers cost more than the special-function unit's share: 249 -> 273 us.)
template <typename V>
__device__ __forceinline__ V sigmoid(V v) {
  const V e = each(mul(v, all<V>(-LOG2E)), [](float t) { return ex2(t); });
  return each(add(e, all<V>(1.f)), [](float t) { return rcp(t); });
}

// A channel's rate: the exponent of a is -k sigmoid(decay_gate).
template <typename V>
struct Rate {
  V nk;                    // -k log2(e)
  V scale;                 // sqrt(2 k)
};

// What a decay gate makes of a step: sigmoid, exponent l of a = 2^l, a and b = sqrt(1 - a^2).
// NEAR, l above -0.36 (a above e^-1/4): 1 - a = l M(l) and b = sqrt(-2 l ln 2) G(l), with polynomials for M = (1 - 2^l) / l and
// G^2 = (1 - 2^2l) / (-2 l ln 2) through Chebyshev points (1.2e-8 and 9.6e-9 off), so that a is off by its own rounding only; and with
// s = q^2 the root is sqrt(2 k) q, so that one reciprocal square root serves the sigmoid and b (the special-function unit
// is what binds the forward pass).  A warp takes this form where k is at most 1/4 in all its channels, so that no gate leads out of it.
// 64 x 512 x 5120 bf16: forward 229 us, gradients 456; with k of 5.5 in every channel, by the other form, 332 and 535; with one such channel
// in every warp's 64, 347 and 562 (f32 x 2560: 208 and 379; 206 and 382; 220 and 395).
constexpr float NEAR_EXPONENT = -0.25f * LOG2E;
template <bool NEAR, typename V>
__device__ __forceinline__ void decay_of(V gate, const Rate<V>& k, V* sig, V* l, V* a, V* b) {
  const V e = each(mul(gate, all<V>(-LOG2E)), [](float t) { return ex2(t); }), d = add(e, all<V>(1.f));
  if constexpr (NEAR) {
    const V q = each(d, [](float t) { return rsq(t); });
    *sig = mul(q, q);
    const V v = mul(k.nk, *sig);
    *l = v;
    V m = fma(v, all<V>(-0.0012021972797811031f), all<V>(-0.009577498771250248f));
    V g = fma(v, all<V>(0.00284821935929358f), all<V>(0.020715761929750443f));
    m = fma(v, m, all<V>(-0.05549892038106918f));
    g = fma(v, g, all<V>(0.10008183121681213f));
    m = fma(v, m, all<V>(-0.24022626876831055f));
    g = fma(v, g, all<V>(0.34657302498817444f));
    m = fma(v, m, all<V>(-0.6931471824645996f));
    g = fma(v, g, all<V>(1.f));
    *a = fma(mul(v, m), all<V>(-1.f), all<V>(1.f));
    *b = mul(mul(k.scale, q), g);
  } else {
    *sig = each(d, [](float t) { return rcp(t); });
    *l = mul(k.nk, *sig);
    // 1 - a by the series where the difference would cancel
    const V m = each(*l, [](float t) {
      const float w = t * 0.6931471805599453f;
      const float p = fmaf(w, fmaf(w, fmaf(w, fmaf(w, fmaf(w, 1.f / 720, 1.f / 120), 1.f / 24), 1.f / 6), 0.5f), 1.f) * w;
      return t < NEAR_EXPONENT ? 1.f - ex2(t) : -p;
    });
    *a = each(*l, m, [](float t, float u) { return t < NEAR_EXPONENT ? ex2(t) : 1.f - u; });
    *b = each(m, [](float u) { return root(u * (2.f - u)); });
  }
}

// ---- cluster ---------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A map to the same place in CTA `rank`'s shared memory; its bytes count on that CTA's `bar`.
__device__ __forceinline__ void put_remote(void* at, uint64_t* bar, uint32_t rank, const Lane<bf16>::Map& m) {
  asm volatile("{\n\t.reg .b32 ra, rb;\n\tmapa.shared::cluster.u32 ra, %0, %2;\n\tmapa.shared::cluster.u32 rb, %1, %2;\n\t"
               "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [ra], {%3, %4, %5, %6}, [rb];\n\t}" ::"r"(ptx::smem_u32(at)),
               "r"(ptx::smem_u32(bar)), "r"(rank), "f"(m.p0), "f"(m.h0), "f"(m.p1), "f"(m.h1) : "memory");
}
__device__ __forceinline__ void put_remote(void* at, uint64_t* bar, uint32_t rank, const Lane<float>::Map& m) {
  asm volatile("{\n\t.reg .b32 ra, rb;\n\tmapa.shared::cluster.u32 ra, %0, %2;\n\tmapa.shared::cluster.u32 rb, %1, %2;\n\t"
               "st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [ra], {%3, %4}, [rb];\n\t}" ::"r"(ptx::smem_u32(at)),
               "r"(ptx::smem_u32(bar)), "r"(rank), "f"(m.p0), "f"(m.h0) : "memory");
}
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!ptx::mbar_try_wait(bar, parity))
    if (clock64() - t0 > WAIT_CYCLES) return false;
  return true;
}

// The maps of a cluster's tiles, turn by turn, in two buffers.  A CTA may write a peer's buffer of turn n + 2 once
// it has that peer's map of turn n + 1, which the peer's warps send behind the __syncthreads() that follows their reading of turn n.
template <typename T, int WARPS>
struct Peers {
  typedef typename Lane<T>::Map Map;
  Map* maps;               // [2][cluster][32]
  uint64_t* bars;          // [2]
  int cluster, rank;
  unsigned* status;        // or NULL
  bool broken;             // a wait gave up: the CTA's results are NaN

  __device__ __forceinline__ void arm(int par) { ptx::mbar_arrive_expect_tx(&bars[par], (uint32_t)(cluster * 32 * sizeof(Map))); }
  __device__ __forceinline__ void start() {
    if (cluster == 1) return;
    if (threadIdx.x == 0) {
      ptx::mbar_init(&bars[0], 1);
      ptx::mbar_init(&bars[1], 1);
      ptx::fence_mbar_init();
      arm(0);
      arm(1);
    }
    cluster_sync();        // every CTA is there before any writes to it
  }
  __device__ __forceinline__ void send(int64_t turn, const Map& m) {
    const int par = (int)(turn & 1), lane = threadIdx.x & 31;
    for (int to = threadIdx.x >> 5; to < cluster; to += WARPS) put_remote(&maps[(par * cluster + rank) * 32 + lane], &bars[par], to, m);
  }
  __device__ __forceinline__ const Map* wait(int64_t turn) {
    const int par = (int)(turn & 1);
    const uint32_t phase = (uint32_t)(turn >> 1) & 1;
    if (!broken && !ptx::mbar_try_wait(&bars[par], phase) && !wait_long(&bars[par], phase)) {
      broken = true;
      if (status) atomicCAS(status, 0u, 0x101u);
    }
    if (threadIdx.x == 0 && !broken) arm(par);   // of turn + 2, which no peer sends before this CTA's warps have met again
    return maps + par * cluster * 32 + (threadIdx.x & 31);
  }
  __device__ __forceinline__ void end() {
    // no CTA leaves while another may send to it; nothing is released, so that the outputs' stores need not be waited for
    if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  }
};

// ---- the asynchronous loads ------------------------------------------------------------------
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

struct Input {
  const void* p;
  int64_t stride_b, stride_t;      // in values; channels are contiguous
};

struct Args {
  Input in[4];                     // x, decay_gate, input_gate, grad of y
  const float* decay;              // (D)
  const float* state_in;           // (b, D) before the first token, or NULL
  const float* grad_final;         // (b, D) or NULL
  const int* seq_idx;              // (b, L) or NULL
  float* states;                   // (b, ceil(L / 32), D): before each 32 tokens; written forward (or NULL), read backward
  void* out[3];                    // y (or NULL); dx, ddecay_gate, dinput_gate: (b, L, D)
  float* state_out;                // (b, D) after the last token, or NULL; grad of state_in, or NULL
  float* part;                     // (b * cluster, D): sums of delta m
  unsigned* status;                // or NULL: set where a wait gave up
  int64_t L, D, points, groups;
  float scale;
};

// Lanes that hold channels.  Rows that start anywhere are copied from the 16-byte boundary in front of them, so that 128 bytes
// hold 28 words at any of them (value by value, 1 x 64078 x 7927 took 4235 us in place of 1487).
constexpr int lanes_of(bool aligned) { return aligned ? 32 : 28; }

// A warp's rows of N tensors, 128 bytes each, into its part of a stage; zeros beyond the sequence and beyond the channels.
template <typename T, int N, int STEPS, int WARPS, bool ALIGNED>
struct Rows {
  static constexpr int WARP_BYTES = N * STEPS * 128, STAGE = WARPS * WARP_BYTES, LANES = ALIGNED ? 32 : 28;
  const uint8_t* at[N];            // the lane's first row of the next turn, and where ALIGNED its 16 bytes there
  uint8_t* smem;                   // the warp's part of stage 0
  int bytes;                       // ALIGNED: 16, or 0 beyond the channels; else of the group's channels
  int64_t t0;                      // of the next turn
  uint32_t low[N], step[N];        // not ALIGNED: addresses of the present turn's first row and from row to row, of which four bits count

  __device__ __forceinline__ Rows(const Args& a, uint8_t* stages, int64_t b, int64_t c0, int64_t first) {
    const int lane = threadIdx.x & 31;
    smem = stages + (threadIdx.x >> 5) * WARP_BYTES;
    t0 = first;
    const int64_t c = ALIGNED ? c0 + lane % 8 * (16 / (int)sizeof(T)) : c0;
    if constexpr (ALIGNED) bytes = c < a.D ? 16 : 0;
    else bytes = (int)(min((int64_t)(LANES * Lane<T>::CH), a.D - c0) * (int)sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const T* p = static_cast<const T*>(a.in[i].p) + b * a.in[i].stride_b + (first + lane / 8) * a.in[i].stride_t + (bytes ? c : 0);
      at[i] = reinterpret_cast<const uint8_t*>(p);
      if constexpr (!ALIGNED) {
        step[i] = (uint32_t)(a.in[i].stride_t * (int64_t)sizeof(T));
        low[i] = (uint32_t)reinterpret_cast<uintptr_t>(p) - (uint32_t)(lane / 8) * step[i];
      }
    }
  }
  __device__ __forceinline__ uint8_t* row(int stage, int i, int s) { return smem + stage * STAGE + (i * STEPS + s) * 128; }
  __device__ __forceinline__ const uint32_t* words(int stage) { return reinterpret_cast<const uint32_t*>(smem + stage * STAGE) + (threadIdx.x & 31); }
  // The lane's channels of tensor i in step s; `words` is of this turn's stage.
  __device__ __forceinline__ uint32_t word(const uint32_t* words, int i, int s) const {
    if constexpr (ALIGNED) {
      return words[(i * STEPS + s) * 32];
    } else {
      const int lane = threadIdx.x & 31;
      const uint32_t shift = low[i] + (uint32_t)s * step[i];
      const uint32_t* w = words + (i * STEPS + s) * 32 + ((int)(shift >> 2 & 3) + min(lane, LANES - 1) - lane);
      return sizeof(T) == 2 ? __funnelshift_r(w[0], w[1], shift << 3 & 16) : w[0];
    }
  }
  // The turn is over: `ahead` tokens on.
  __device__ __forceinline__ void turn(int64_t ahead) {
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < N; ++i) low[i] += (uint32_t)ahead * step[i];
    }
  }

  // `ahead`: tokens from this turn to the next
  __device__ __forceinline__ void load(const Args& a, int stage, int64_t ahead) {
    const int lane = threadIdx.x & 31;
    const uint32_t dst = ptx::smem_u32(row(stage, 0, lane / 8)) + lane % 8 * 16;
    if constexpr (ALIGNED) {
      if (t0 + STEPS <= a.L) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
          for (int j = 0; j < STEPS / 4; ++j)
            cp16(dst + (i * STEPS + 4 * j) * 128, at[i] + j * (4 * (int64_t)sizeof(T)) * a.in[i].stride_t, bytes);
          at[i] += ahead * a.in[i].stride_t * (int64_t)sizeof(T);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
          for (int j = 0; j < STEPS / 4; ++j) {
            const bool there = t0 + lane / 8 + 4 * j < a.L;
            cp16(dst + (i * STEPS + 4 * j) * 128, there ? at[i] + j * (4 * (int64_t)sizeof(T)) * a.in[i].stride_t : a.in[i].p, there ? bytes : 0);
          }
          at[i] += ahead * a.in[i].stride_t * (int64_t)sizeof(T);
        }
      }
    } else {
      // Nothing is read behind the row's channels.  In front of them up to 14 bytes are, which lie in the same 16 bytes as the
      // first channel and so in its allocation.
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int j = 0; j < STEPS / 4; ++j) {
          const uint8_t* p = at[i] + j * (4 * (int64_t)sizeof(T)) * a.in[i].stride_t;
          const int in = (int)(reinterpret_cast<uintptr_t>(p) & 15), left = in + bytes - lane % 8 * 16;
          const bool there = t0 + lane / 8 + 4 * j < a.L && left > 0;
          cp16(dst + (i * STEPS + 4 * j) * 128, there ? p - in + lane % 8 * 16 : reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(a.in[i].p) & ~uintptr_t(15)),
               there ? min(left, 16) : 0);
        }
        at[i] += ahead * a.in[i].stride_t * (int64_t)sizeof(T);
      }
    }
    t0 += ahead;
  }
  // Steps beyond the sequence leave the state as it is: their decay gates are closed.
  __device__ __forceinline__ void close(int stage, int live) {
    const uint32_t shut = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
    for (int s = live; s < STEPS; ++s) reinterpret_cast<uint32_t*>(row(stage, 1, s))[threadIdx.x & 31] = shut;
    if (!ALIGNED) __syncwarp();
  }
};

// `channels`: of the lane's, that there are.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void store_word(T* o, int channels, typename Lane<T>::V v) {
  const uint32_t u = Lane<T>::put(v);
  if constexpr (ALIGNED) {
    if (channels) *reinterpret_cast<uint32_t*>(o) = u;
  } else {
    const T* w = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int k = 0; k < Lane<T>::CH; ++k)
      if (k < channels) o[k] = w[k];
  }
}

// Which of the warp's steps start a sequence: lane i holds the id of step i - 1.
template <int STEPS>
__device__ __forceinline__ int load_ids(const int* seq, int64_t t0, int64_t L) {
  const int lane = threadIdx.x & 31;
  const int64_t t = t0 - 1 + lane;
  return lane <= STEPS && t < L ? __ldg(seq + (t < 0 ? 0 : t)) : 0;
}
__device__ __forceinline__ unsigned starts_of(int ids, int live) {
  const int next = __shfl_down_sync(0xffffffffu, ids, 1);
  return __ballot_sync(0xffffffffu, next != ids) & ((1u << live) - 1);
}

// The channels' rates; whether no step can take the state further than NEAR_EXPONENT.
template <typename T>
__device__ __forceinline__ Rate<typename Lane<T>::V> rates(const Args& a, int64_t c, bool* near) {
  typedef typename Lane<T>::V V;
  const V lam = Lane<T>::load(a.decay, c, a.D, -1000.f);   // (channels beyond the last decay by nothing)
  const V k = each(lam, [&](float v) { return rate_of(a.scale, v); });
  bool ok = true;
  each(k, [&](float v) { ok = ok && v <= 0.25f; return v; });
  *near = __all_sync(0xffffffffu, ok);
  return {mul(k, all<V>(-LOG2E)), each(k, [](float v) { return __fsqrt_rn(2.f * v); })};
}

// ---- forward -----------------------------------------------------------------------------------
template <typename T>
constexpr int peers_bytes(int cluster) { return 2 * 32 * (int)sizeof(typename Lane<T>::Map) * (cluster > 1 ? cluster : 0); }
template <typename T>
constexpr int fwd_smem(int warps, int cluster) {
  return 2 * 3 * warps * FWD_STEPS * 128 + peers_bytes<T>(cluster) + 2 * warps * 32 * (int)sizeof(typename Lane<T>::Map);
}

template <typename T, int WARPS, bool ALIGNED, bool PACKED>
__global__ void __launch_bounds__(32 * WARPS, MAX_WARPS / WARPS) forward_kernel(const __grid_constant__ Args a, const int cluster) {
  typedef typename Lane<T>::V V;
  typedef typename Lane<T>::Map Map;
  constexpr int CH = Lane<T>::CH, STEPS = FWD_STEPS, TILE = WARPS * STEPS;
  typedef Rows<T, 3, STEPS, WARPS, ALIGNED> In;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int64_t unit = blockIdx.x / (unsigned)cluster, b = unit / a.groups, c0 = (unit - b * a.groups) * (In::LANES * CH);
  const int64_t c = lane < In::LANES ? c0 + lane * CH : a.D;
  Map* const maps = reinterpret_cast<Map*>(smem + 2 * In::STAGE);   // [2][WARPS][32]
  Peers<T, WARPS> peers{maps + 2 * WARPS * 32, bars, cluster, rank, a.status, false};
  const int64_t tiles = (a.L + TILE - 1) / TILE, turns = (tiles + cluster - 1) / cluster, ahead = (int64_t)cluster * TILE;
  const int64_t first = (int64_t)rank * TILE + warp * STEPS;
  In in(a, smem, b, c0, first);
  in.load(a, 0, ahead);
  cp_commit();
  const int* seq = PACKED ? a.seq_idx + b * a.L : nullptr;
  int ids = PACKED ? load_ids<STEPS>(seq, first, a.L) : 0;
  bool near;
  const Rate<V> rate = rates<T>(a, c, &near);
  V carry = a.state_in ? Lane<T>::load(a.state_in + b * a.D, c, a.D) : all<V>(0.f);
  T* out = static_cast<T*>(a.out[0]) + (b * a.L + first) * a.D + c;
  const int channels = (int)max((int64_t)0, min((int64_t)CH, a.D - c));
  peers.start();

  int64_t t0 = first;
  for (int64_t n = 0; n < turns; ++n, t0 += ahead) {
    const int stage = (int)(n & 1);
    const int live = (int)max((int64_t)0, min((int64_t)STEPS, a.L - t0));
    if (n + 1 < turns) in.load(a, stage ^ 1, ahead);
    cp_commit();
    unsigned starts = 0;
    if constexpr (PACKED) {
      starts = starts_of(ids, live);
      ids = load_ids<STEPS>(seq, t0 + ahead, a.L);
    }
    cp_wait<1>();
    __syncwarp();
    if (live < STEPS) in.close(stage, live);
    const uint32_t* words = in.words(stage);
    V av[STEPS], bw[STEPS], P = all<V>(1.f), H = all<V>(0.f);
    auto gates = [&](auto is_near) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        V sr, l, b;
        decay_of<decltype(is_near)::value>(Lane<T>::get(in.word(words, 1, s)), rate, &sr, &l, &av[s], &b);
        bw[s] = mul(b, mul(sigmoid(Lane<T>::get(in.word(words, 2, s))), Lane<T>::get(in.word(words, 0, s))));
        P = mul(P, av[s]);
        H = fma(av[s], H, bw[s]);
      }
    };
    if (near) gates(std::true_type());
    else gates(std::false_type());
    if (PACKED && starts) {   // seldom: again, from where the last sequence starts
      P = all<V>(RESTART);
      H = all<V>(0.f);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (starts >> s & 1) H = all<V>(0.f);
        H = fma(av[s], H, bw[s]);
      }
    }
    Map* const own = maps + stage * WARPS * 32 + lane;
    own[warp * 32] = Lane<T>::map(P, H);
    const bool restarts = meet<PACKED>(starts != 0);
    V h;                   // the state before the warp's steps
    if (cluster > 1) {
      V Pt = all<V>(1.f), Ht = all<V>(0.f);
      if (restarts) {
#pragma unroll
        for (int j = 0; j < WARPS; ++j) compose<PACKED>(own[j * 32], Pt, Ht);
      } else {
#pragma unroll
        for (int j = 0; j < WARPS; ++j) compose<false>(own[j * 32], Pt, Ht);
      }
      peers.send(n, Lane<T>::map(Pt, Ht));
      const Map* q = peers.wait(n);
      h = carry;
      for (int j = 0; j < cluster; j += 4) {   // four loads at a time
        Map m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = q[min(j + k, cluster - 1) * 32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (j + k == rank) h = carry;
          if (j + k < cluster) carry = through<PACKED>(m[k], carry);
        }
      }
      if (peers.broken) h = carry = all<V>(NAN);
      if (restarts) {
#pragma unroll
        for (int j = 0; j < WARPS - 1; ++j)
          if (j < warp) h = through<PACKED>(own[j * 32], h);
      } else {
#pragma unroll
        for (int j = 0; j < WARPS - 1; ++j)
          if (j < warp) h = through<false>(own[j * 32], h);
      }
    } else {
      h = carry;
      if (restarts) {
#pragma unroll
        for (int j = 0; j < WARPS; ++j) {
          if (j == warp) h = carry;
          carry = through<PACKED>(own[j * 32], carry);
        }
      } else {
#pragma unroll
        for (int j = 0; j < WARPS; ++j) {
          if (j == warp) h = carry;
          carry = through<false>(own[j * 32], carry);
        }
      }
    }
    if (a.states && (warp * STEPS) % POINT == 0 && t0 < a.L)
      Lane<T>::store(a.states + (b * a.points + t0 / POINT) * a.D, c, a.D, h);
    if (a.out[0]) {
      T* o = out;
      auto run = [&](auto plain) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          if (!decltype(plain)::value && PACKED && (starts >> s & 1)) h = all<V>(0.f);
          h = fma(av[s], h, bw[s]);
          if (decltype(plain)::value || s < live) store_word<T, ALIGNED>(o, channels, h);
          o += a.D;
        }
      };
      // the checks of every step (and of c against D beside them) were 9 of its 60 instructions
      if (live == STEPS && !(PACKED && starts)) run(std::true_type());
      else run(std::false_type());
      out += ahead * a.D;
    }
    in.turn(ahead);
  }
  if (a.state_out && rank == 0 && warp == 0) Lane<T>::store(a.state_out + b * a.D, c, a.D, carry);
  peers.end();
}

// ---- backward ----------------------------------------------------------------------------------
template <typename T>
constexpr int bwd_smem(int warps, int cluster) {
  return 2 * 4 * warps * BWD_STEPS * 128 + peers_bytes<T>(cluster) + 2 * warps * 32 * ((int)sizeof(typename Lane<T>::Map) + Lane<T>::CH * 4);
}

// Tiles from the last to the first.  The states before each tile are known, so only the reversed
// recurrence of c crosses CTAs; a warp's maps are (P, H) forward and (P, R) backward, with one P.
template <typename T, int WARPS, bool ALIGNED, bool PACKED>
__global__ void __launch_bounds__(32 * WARPS, MAX_WARPS / WARPS) backward_kernel(const __grid_constant__ Args a, const int cluster) {
  typedef typename Lane<T>::V V;
  typedef typename Lane<T>::Map Map;
  constexpr int CH = Lane<T>::CH, STEPS = BWD_STEPS, TILE = WARPS * STEPS;
  typedef Rows<T, 4, STEPS, WARPS, ALIGNED> In;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[2];
  Map* const maps = reinterpret_cast<Map*>(smem + 2 * In::STAGE);                       // (P, R) [2][WARPS][32]
  V* const ends = reinterpret_cast<V*>(maps + 2 * 32 * (WARPS + (cluster > 1 ? cluster : 0)));   // H [2][WARPS][32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int64_t unit = blockIdx.x / (unsigned)cluster, b = unit / a.groups, c0 = (unit - b * a.groups) * (In::LANES * CH);
  const int64_t c = lane < In::LANES ? c0 + lane * CH : a.D;
  Peers<T, WARPS> peers{maps + 2 * WARPS * 32, bars, cluster, rank, a.status, false};
  const int64_t tiles = (a.L + TILE - 1) / TILE, turns = (tiles + cluster - 1) / cluster, ahead = -(int64_t)cluster * TILE;
  int64_t t0 = ((turns - 1) * cluster + rank) * TILE + warp * STEPS;
  In in(a, smem, b, c0, t0);
  in.load(a, 0, ahead);
  cp_commit();
  const int* seq = PACKED ? a.seq_idx + b * a.L : nullptr;
  int ids = PACKED ? load_ids<STEPS>(seq, t0, a.L) : 0;
  // before the 32 tokens that hold the warp's
  auto state_before = [&](int64_t t) {
    return t >= 0 && t < a.L ? Lane<T>::load(a.states + (b * a.points + t / POINT) * a.D, c, a.D) : all<V>(0.f);
  };
  V state = state_before(t0);
  bool near;
  const Rate<V> rate = rates<T>(a, c, &near);
  V carry = a.grad_final ? Lane<T>::load(a.grad_final + b * a.D, c, a.D) : all<V>(0.f);
  V sum = all<V>(0.f), total = all<V>(0.f);   // of delta m: over the turns, and of a turn with what the sum has lost so far
  int64_t at = (b * a.L + t0) * a.D + c;
  const int channels = (int)max((int64_t)0, min((int64_t)CH, a.D - c));
  peers.start();

  for (int64_t n = 0; n < turns; ++n, t0 += ahead) {
    const int stage = (int)(n & 1);
    const int live = (int)max((int64_t)0, min((int64_t)STEPS, a.L - t0));
    __syncwarp();          // the other lanes have read the stage that is loaded next
    if (n + 1 < turns) in.load(a, stage ^ 1, ahead);
    cp_commit();
    V h = state;
    state = state_before(t0 + ahead);
    unsigned starts = 0;
    if constexpr (PACKED) {
      starts = starts_of(ids, live);
      if (n + 1 < turns) ids = load_ids<STEPS>(seq, t0 + ahead, a.L);
    }
    cp_wait<1>();
    __syncwarp();
    if (live < STEPS) in.close(stage, live);
    const uint32_t* words = in.words(stage);
    V av[STEPS], bv[STEPS], sr[STEPS], si[STEPS], P = all<V>(1.f), H = all<V>(0.f), R = all<V>(0.f);
    auto gates = [&](auto is_near) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        V l;
        decay_of<decltype(is_near)::value>(Lane<T>::get(in.word(words, 1, s)), rate, &sr[s], &l, &av[s], &bv[s]);
        si[s] = sigmoid(Lane<T>::get(in.word(words, 2, s)));
        P = mul(P, av[s]);
        if (PACKED && (starts >> s & 1)) H = all<V>(0.f);
        H = fma(av[s], H, mul(bv[s], mul(si[s], Lane<T>::get(in.word(words, 0, s)))));
      }
    };
    if (near) gates(std::true_type());
    else gates(std::false_type());
#pragma unroll
    for (int s = STEPS - 1; s >= 0; --s) {
      R = mul(av[s], add(R, Lane<T>::get(in.word(words, 3, s))));
      if (PACKED && (starts >> s & 1)) R = all<V>(0.f);
    }
    Map* const own = maps + (stage * WARPS) * 32 + lane;
    V* const own_end = ends + (stage * WARPS) * 32 + lane;
    own[warp * 32] = Lane<T>::map(PACKED && starts ? all<V>(RESTART) : P, R);
    own_end[warp * 32] = H;
    __syncthreads();
    V after;               // what reaches the CTA's tile from behind, then the warp's steps
    if (cluster > 1) {
      V Pt = all<V>(1.f), Rt = all<V>(0.f);
#pragma unroll 4
      for (int j = WARPS - 1; j >= 0; --j) compose<PACKED>(own[j * 32], Pt, Rt);
      peers.send(n, Lane<T>::map(Pt, Rt));
    }
    constexpr int BEFORE = POINT / STEPS;   // warps of a checkpoint
#pragma unroll
    for (int j = 0; j < BEFORE - 1; ++j) {
      const int k = warp / BEFORE * BEFORE + j;
      if (k < warp) h = through<PACKED>(Lane<T>::map(map_p(own[k * 32]), own_end[k * 32]), h);
    }
    // m of each step, from the states before them, into the words of the gates, which are not needed again; what the other
    // CTAs send is on its way meanwhile
    uint32_t* keep = const_cast<uint32_t*>(words);
    const V nkl = mul(rate.nk, all<V>(0.6931471805599453f));
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (PACKED && (starts >> s & 1)) h = all<V>(0.f);
      const V w = mul(si[s], Lane<T>::get(in.word(words, 0, s)));
      const V inverse = each(bv[s], [](float t) { return t == 0.f ? 0.f : -rcp(t); });
      const V m = mul(mul(mul(sr[s], nkl), av[s]), fma(mul(av[s], inverse), w, h));
      if constexpr (CH == 2) {
        const float2 u = unpack(m);
        keep[(STEPS + s) * 32] = __float_as_uint(u.x);
        keep[(2 * STEPS + s) * 32] = __float_as_uint(u.y);
      } else {
        keep[(STEPS + s) * 32] = __float_as_uint(m);
      }
      if (s + 1 < STEPS) h = fma(av[s], h, mul(bv[s], w));
    }
    if (cluster > 1) {
      const Map* q = peers.wait(n);
      after = carry;
      for (int j = cluster - 1; j >= 0; j -= 4) {   // four loads at a time
        Map m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = q[max(j - k, 0) * 32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (j - k == rank) after = carry;
          if (j - k >= 0) carry = through<PACKED>(m[k], carry);
        }
      }
      if (peers.broken) after = carry = all<V>(NAN);
#pragma unroll 4
      for (int j = WARPS - 1; j > 0; --j)
        if (j > warp) after = through<PACKED>(own[j * 32], after);
    } else {
      after = carry;
#pragma unroll 4
      for (int j = WARPS - 1; j >= 0; --j) {
        if (j == warp) after = carry;
        carry = through<PACKED>(own[j * 32], carry);
      }
    }
    auto finish = [&](auto whole) {
      int64_t row = at + (STEPS - 1) * a.D;
#pragma unroll
      for (int s = STEPS - 1; s >= 0; --s) {
        const V x = Lane<T>::get(in.word(words, 0, s)), w = mul(si[s], x);
        V m;
        if constexpr (CH == 2) m = pack(__uint_as_float(words[(STEPS + s) * 32]), __uint_as_float(words[(2 * STEPS + s) * 32]));
        else m = __uint_as_float(words[(STEPS + s) * 32]);
        const V d = add(after, Lane<T>::get(in.word(words, 3, s)));
        after = mul(av[s], d);
        if (PACKED && (starts >> s & 1)) after = all<V>(0.f);
        const V dm = mul(d, m), db = mul(d, bv[s]);
        total = add(total, dm);
        if (decltype(whole)::value || s < live) {
          store_word<T, ALIGNED>(static_cast<T*>(a.out[0]) + row, channels, mul(db, si[s]));
          store_word<T, ALIGNED>(static_cast<T*>(a.out[1]) + row, channels, mul(dm, fma(sr[s], all<V>(-1.f), all<V>(1.f))));
          store_word<T, ALIGNED>(static_cast<T*>(a.out[2]) + row, channels, mul(mul(db, w), fma(si[s], all<V>(-1.f), all<V>(1.f))));
        }
        row -= a.D;
      }
    };
    if (live == STEPS) finish(std::true_type());
    else finish(std::false_type());
    // What the addition loses stays in total (Kahan): where summands are alike a plain sum rounds the same way each time, and 4096
    // tokens of a warp were 6e-5 off
    const V now = add(sum, total);
    total = fma(fma(sum, all<V>(-1.f), now), all<V>(-1.f), total);
    sum = now;
    at += ahead * a.D;
    in.turn(ahead);
  }
  // the CTA's sum for the decay, warps in order
  __syncthreads();
  ends[warp * 32 + lane] = sum;
  __syncthreads();
  if (warp == 0) {
    for (int j = 1; j < WARPS; ++j) sum = add(sum, ends[j * 32 + lane]);
    Lane<T>::store(a.part + (b * cluster + rank) * a.D, c, a.D, sum);
    if (a.state_out && rank == 0) Lane<T>::store(a.state_out + b * a.D, c, a.D, carry);
  }
  peers.end();
}

// Sum of the CTAs' parts, in order, in f64: 8 rows of threads to 32 channels.
__global__ void __launch_bounds__(256) decay_kernel(const float* part, int64_t rows, int64_t D, const float* decay, float* out) {
  __shared__ double sh[8][32];
  ptx::griddep_wait();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + x;
  double v = 0;
  if (c < D) {
#pragma unroll 4
    for (int64_t r = y; r < rows; r += 8) v += (double)part[r * D + c];
  }
  sh[y][x] = v;
  __syncthreads();
  if (y || c >= D) return;
  for (int j = 1; j < 8; ++j) v += sh[j][x];
  const double d = (double)decay[c], e = exp(-fabs(d));
  // sigmoid / softplus; 1 in the limit of far negative values, where both are e^d
  const double sig = d >= 0 ? 1.0 / (1.0 + e) : e / (1.0 + e), soft = d > 0 ? d + log1p(e) : log1p(e);
  out[c] = (float)(v * (soft > 0 ? sig / soft : 1.0));
}

// ---- one token -----------------------------------------------------------------------------------
struct StepArgs {
  const void* in[3];
  int64_t stride[3];               // between rows
  const float* decay;
  const float* state;
  float* new_state;                // may be state itself
  void* y;
  int64_t batch, D;
  float scale;
  int rows;                        // of a thread
};

// A thread takes VEC channels of `rows` rows, so that the rate of its channels is computed once.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) step_kernel(const StepArgs a) {
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC, r0 = (int64_t)blockIdx.y * a.rows;
  if (c >= a.D) return;
  float nk[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) nk[i] = -LOG2E * rate_of(a.scale, a.decay[c + i]);
  const int64_t r1 = min(r0 + a.rows, a.batch);
  const T* x = static_cast<const T*>(a.in[0]) + c;
  const T* r = static_cast<const T*>(a.in[1]) + c;
  const T* g = static_cast<const T*>(a.in[2]) + c;
#pragma unroll 2
  for (int64_t row = r0; row < r1; ++row) {
    struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };
    struct alignas(VEC * 4) State { float v[VEC]; };
    const Pack px = *reinterpret_cast<const Pack*>(x + row * a.stride[0]);
    const Pack pr = *reinterpret_cast<const Pack*>(r + row * a.stride[1]);
    const Pack pg = *reinterpret_cast<const Pack*>(g + row * a.stride[2]);
    State h = *reinterpret_cast<const State*>(a.state + row * a.D + c);
    Pack y;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float s, l, A, B;
      decay_of<false>(ld(&pr.v[i]), Rate<float>{nk[i], 0.f}, &s, &l, &A, &B);
      h.v[i] = fmaf(A, h.v[i], B * (sigmoid(ld(&pg.v[i])) * ld(&px.v[i])));
      st(&y.v[i], h.v[i]);
    }
    *reinterpret_cast<State*>(a.new_state + row * a.D + c) = h;
    *reinterpret_cast<Pack*>(static_cast<T*>(a.y) + row * a.D + c) = y;
  }
}

// ---- host side -------------------------------------------------------------------------------------
constexpr int SMS = 148;   // of a B200

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Everything that a launch needs to know of one kernel: clusters of c CTAs that the GPU holds at once.
struct Kernel {
  const void* f;
  int warps, tile;
  int (*smem)(int warps, int cluster);
  std::atomic<uint64_t>* ready;            // devices on which its attributes are set
  std::atomic<int>* capacity;              // [MAX_CLUSTER + 1], 0: not asked yet
};

cudaError_t make_ready(const Kernel& k) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (bit && (k.ready->load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(k.f, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem(k.warps, MAX_CLUSTER));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k.f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) k.ready->fetch_or(bit, std::memory_order_release);
  return e;
}

void configure(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, const Kernel& k, int64_t ctas, int cluster, cudaStream_t st) {
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = (unsigned)cluster;
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cfg->gridDim = dim3((unsigned)ctas);
  cfg->blockDim = dim3((unsigned)(32 * k.warps));
  cfg->dynamicSmemBytes = (size_t)k.smem(k.warps, cluster);
  cfg->stream = st;
  cfg->attrs = attr;
  cfg->numAttrs = cluster > 1 ? 1 : 0;
}

int capacity_of(const Kernel& k, int cluster) {
  const int known = k.capacity[cluster].load(std::memory_order_relaxed);
  if (known) return known;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  configure(&cfg, attr, k, cluster, cluster, nullptr);
  cfg.numAttrs = 1;
  int n = 0;
  if (make_ready(k) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, k.f, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = -1;                                // not to be had
  }
  k.capacity[cluster].store(n, std::memory_order_relaxed);
  return n;
}

// Microseconds of `units` clusters: a turn takes `turn`, and `warp` more for each warp that its SM holds, `wide` for each warp of a CTA
// above 4 (they meet), and in a cluster `exchange` and `peer` for each CTA; a CTA takes `start`.  Fitted to 26 shapes of both types, of
// 1 to 64 rows, 300 to 65536 tokens and 128 to 8192 channels, each with 1 to 16 CTAs of 4, 8 and 16 warps: what the rule picks is 3 %
// slower than the best on average (14 and 17 % at worst).  Both sides, forward: 64 x 512 x 5120, CTAs of 4 warps alone 228 us, of 8 266,
// pairs of CTAs 286; 1 x 65536 x 256: alone 1295, clusters of 16 CTAs of 4 warps 135, of 16 warps 102.
struct Times {
  double turn, warp, exchange, peer, start, wide;
};
constexpr Times FORWARD = {0.83, 0.167, 0.374, 0.033, 2.8, 0.068}, BACKWARD = {0.65, 0.184, 0.101, 0.141, 1.24, 0.082};

double time_of(const Kernel& k, const Times& t, int64_t units, int64_t L, int cluster) {
  const int cap = capacity_of(k, cluster);
  if (cap <= 0) return 1e30;
  const int64_t turns = cdiv(cdiv(L, k.tile), cluster), full = units / cap, rest = units - full * cap;
  const double alone = t.turn + (cluster > 1 ? t.exchange + t.peer * cluster : 0.0) + t.wide * (k.warps - 4);
  const double warps = std::min<double>(MAX_WARPS, k.warps * (double)cdiv(rest * cluster, SMS));
  return (double)full * (t.start + (double)turns * (alone + t.warp * MAX_WARPS)) +
         (rest ? t.start + (double)turns * (alone + t.warp * warps) : 0.0);
}

struct Choice {
  int kernel, cluster;
};

Choice pick(const Kernel* list, int n, const Times& times, int64_t units, int64_t L) {
  Choice best = {0, 1};
  double least = 1e300;
  for (int k = 0; k < n; ++k)
    for (int c = 1; c <= MAX_CLUSTER && (c == 1 || (int64_t)(c - 1) * list[k].tile < L); ++c) {
      const double t = time_of(list[k], times, units, L, c);
      if (t < least) {
        least = t;
        best = {k, c};
      }
    }
  return best;
}

template <auto KERNEL, int WARPS, int STEPS>
Kernel kernel_of(int (*smem)(int, int)) {
  static std::atomic<uint64_t> ready{0};
  static std::atomic<int> capacity[MAX_CLUSTER + 1] = {};
  return {(const void*)KERNEL, WARPS, WARPS * STEPS, smem, &ready, capacity};
}

// CTAs of 4, 8 and 16 warps (rows that are not aligned: of 4).
struct Kernels {
  Kernel list[3];
  int n;
};

template <typename T>
Kernels forward_kernels(bool aligned, bool packed) {
  constexpr int S = FWD_STEPS;
  if (!aligned)
    return {{packed ? kernel_of<forward_kernel<T, 4, false, true>, 4, S>(fwd_smem<T>) : kernel_of<forward_kernel<T, 4, false, false>, 4, S>(fwd_smem<T>)}, 1};
  if (packed)
    return {{kernel_of<forward_kernel<T, 4, true, true>, 4, S>(fwd_smem<T>), kernel_of<forward_kernel<T, 8, true, true>, 8, S>(fwd_smem<T>),
             kernel_of<forward_kernel<T, 16, true, true>, 16, S>(fwd_smem<T>)}, 3};
  return {{kernel_of<forward_kernel<T, 4, true, false>, 4, S>(fwd_smem<T>), kernel_of<forward_kernel<T, 8, true, false>, 8, S>(fwd_smem<T>),
           kernel_of<forward_kernel<T, 16, true, false>, 16, S>(fwd_smem<T>)}, 3};
}

template <typename T>
Kernels backward_kernels(bool aligned, bool packed) {
  constexpr int S = BWD_STEPS;
  if (!aligned)
    return {{packed ? kernel_of<backward_kernel<T, 4, false, true>, 4, S>(bwd_smem<T>) : kernel_of<backward_kernel<T, 4, false, false>, 4, S>(bwd_smem<T>)}, 1};
  if (packed)
    return {{kernel_of<backward_kernel<T, 4, true, true>, 4, S>(bwd_smem<T>), kernel_of<backward_kernel<T, 8, true, true>, 8, S>(bwd_smem<T>),
             kernel_of<backward_kernel<T, 16, true, true>, 16, S>(bwd_smem<T>)}, 3};
  return {{kernel_of<backward_kernel<T, 4, true, false>, 4, S>(bwd_smem<T>), kernel_of<backward_kernel<T, 8, true, false>, 8, S>(bwd_smem<T>),
           kernel_of<backward_kernel<T, 16, true, false>, 16, S>(bwd_smem<T>)}, 3};
}

cudaError_t launch(const Kernels& ks, Choice c, const Args& a, int64_t units, cudaStream_t st) {
  const Kernel& k = ks.list[c.kernel];
  const int64_t ctas = units * c.cluster;
  if (ctas >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  configure(&cfg, attr, k, ctas, c.cluster, st);
  Args args = a;
  int cluster = c.cluster;
  void* params[] = {&args, &cluster};
  return cudaLaunchKernelExC(&cfg, k.f, params);
}

template <typename T, int VEC>
cudaError_t launch_step(const StepArgs& a, cudaStream_t st) {
  const int64_t columns = cdiv(a.D, 256 * VEC), bands = cdiv(a.batch, a.rows);
  step_kernel<T, VEC><<<dim3((unsigned)columns, (unsigned)bands), 256, 0, st>>>(a);
  return cudaGetLastError();
}

int value_bytes(int dtype) { return dtype == SSD_DTYPE_BF16 ? 2 : 4; }

// Rows that start at 16 bytes, and hold whole 16-byte pieces.
bool rows_aligned(const void* p, int64_t stride_b, int64_t stride_t, int64_t batch, int64_t L, int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (batch == 1 || stride_b * es % 16 == 0) && (L == 1 || stride_t * es % 16 == 0);
}

Args args_of(const ssd_gated_recurrence_params_t* p) {
  Args a{};
  a.in[0] = {p->x, p->x_stride_b, p->x_stride_t};
  a.in[1] = {p->decay_gate, p->decay_gate_stride_b, p->decay_gate_stride_t};
  a.in[2] = {p->input_gate, p->input_gate_stride_b, p->input_gate_stride_t};
  a.decay = p->decay;
  a.seq_idx = p->seq_idx;
  a.L = p->seqlen;
  a.D = p->dim;
  a.points = cdiv(p->seqlen, POINT);
  a.scale = p->scale;
  a.status = p->status;
  return a;
}

bool all_aligned(const ssd_gated_recurrence_params_t* p, const Args& a, int inputs) {
  const int es = value_bytes(p->dtype);
  bool ok = p->dim * es % 16 == 0;
  for (int i = 0; i < inputs; ++i) ok = ok && rows_aligned(a.in[i].p, a.in[i].stride_b, a.in[i].stride_t, p->batch, p->seqlen, es);
  for (int i = 0; i < 3; ++i) ok = ok && reinterpret_cast<uintptr_t>(a.out[i]) % 16 == 0;
  return ok;
}

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// The kernels of a call, on the current device, and which of them; the groups that its channels make.
cudaError_t choose(const ssd_gated_recurrence_params_t* p, Args& a, bool backward, bool aligned, Kernels* ks, Choice* c) {
  a.groups = cdiv(p->dim, 4 / value_bytes(p->dtype) * lanes_of(aligned));
  const bool bf = p->dtype == SSD_DTYPE_BF16, packed = a.seq_idx != nullptr;
  if (backward) *ks = bf ? backward_kernels<bf16>(aligned, packed) : backward_kernels<float>(aligned, packed);
  else *ks = bf ? forward_kernels<bf16>(aligned, packed) : forward_kernels<float>(aligned, packed);
  // the rule's answer for the sizes of this thread's last calls, forward and backward (it takes 1 us, a third of a launch)
  struct Last {
    const void* f;
    int64_t units, L;
    Choice c;
  };
  static thread_local Last last[2] = {};
  Last& l = last[backward];
  const int64_t units = p->batch * a.groups;
  if (l.f != ks->list[0].f || l.units != units || l.L != a.L) l = {ks->list[0].f, units, a.L, pick(ks->list, ks->n, backward ? BACKWARD : FORWARD, units, a.L)};
  *c = l.c;
  return make_ready(ks->list[c->kernel]);
}

// Sums for the decay: one for each CTA of a cluster, whatever its size will be.
size_t part_bytes(const ssd_gated_recurrence_params_t* p) { return up256((size_t)p->batch * MAX_CLUSTER * p->dim * 4); }

}  // namespace

static_assert(POINT == SSD_GATED_RECURRENCE_CHECKPOINT, "the header names the distance of checkpoints");

cudaError_t launch_gated_recurrence(const ssd_gated_recurrence_params_t* p, cudaStream_t st) {
  Args a = args_of(p);
  a.state_in = p->initial_state;
  a.states = p->checkpoints;
  a.out[0] = p->y;
  a.state_out = p->final_state;
  Kernels ks;
  Choice c;
  const cudaError_t e = choose(p, a, false, all_aligned(p, a, 3), &ks, &c);
  return e != cudaSuccess ? e : launch(ks, c, a, p->batch * a.groups, st);
}

size_t gated_recurrence_grad_workspace(const ssd_gated_recurrence_params_t* p) {
  return part_bytes(p) + (p->checkpoints ? 0 : up256((size_t)p->batch * cdiv(p->seqlen, POINT) * p->dim * 4));
}

cudaError_t launch_gated_recurrence_grad(const ssd_gated_recurrence_params_t* p, const ssd_gated_recurrence_grads_t* g,
                                         void* workspace, cudaStream_t st) {
  Args a = args_of(p);
  a.part = static_cast<float*>(workspace);
  a.states = p->checkpoints;
  if (!a.states) {   // the forward pass again, for the states alone
    a.states = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + part_bytes(p));
    ssd_gated_recurrence_params_t f = *p;
    f.checkpoints = a.states;
    f.y = nullptr;
    f.final_state = nullptr;
    const cudaError_t e = launch_gated_recurrence(&f, st);
    if (e != cudaSuccess) return e;
  }
  a.in[3] = {g->grad_y, g->grad_y_stride_b, g->grad_y_stride_t};
  a.grad_final = g->grad_final_state;
  a.out[0] = g->grad_x;
  a.out[1] = g->grad_decay_gate;
  a.out[2] = g->grad_input_gate;
  a.state_out = g->grad_initial_state;
  Kernels ks;
  Choice c;
  cudaError_t e = choose(p, a, true, all_aligned(p, a, 4), &ks, &c);
  if (e == cudaSuccess) e = launch(ks, c, a, p->batch * a.groups, st);
  if (e != cudaSuccess) return e;
  return launch_dependent(decay_kernel, dim3((unsigned)cdiv(p->dim, 32)), 256, 0, 1, st, a.part, p->batch * c.cluster, p->dim,
                          p->decay, g->grad_decay);
}

cudaError_t launch_gated_recurrence_update(const ssd_gated_recurrence_update_params_t* p, cudaStream_t st) {
  StepArgs a{};
  a.in[0] = p->x; a.in[1] = p->decay_gate; a.in[2] = p->input_gate;
  a.stride[0] = p->x_stride_row; a.stride[1] = p->decay_gate_stride_row; a.stride[2] = p->input_gate_stride_row;
  a.decay = p->decay;
  a.state = p->state;
  a.new_state = p->new_state;
  a.y = p->y;
  a.batch = p->batch;
  a.D = p->dim;
  a.scale = p->scale;
  const int es = value_bytes(p->dtype);
  // Two channels a thread: the rates of four are a longer way to the first load than their wider loads save (bf16, in a graph,
  // 256 x 8192 8.9 against 8.1 us, 64 x 5120 3.4 against 3.1, 1 x 8192 2.3 against 2.0; 512 x 8192 13.4 and 13.4)
  bool wide = p->dim % 2 == 0 && (reinterpret_cast<uintptr_t>(p->state) | reinterpret_cast<uintptr_t>(p->new_state)) % 8 == 0 &&
              reinterpret_cast<uintptr_t>(p->y) % (2 * es) == 0;
  for (int i = 0; i < 3; ++i)
    wide = wide && reinterpret_cast<uintptr_t>(a.in[i]) % (2 * es) == 0 && (p->batch == 1 || a.stride[i] % 2 == 0);
  // rows of a thread: so many that the GPU holds all threads at once, and even, since two are loaded at a time (256 x 8192: 1 row
  // 10.4 us, 2 rows 9.1, 4 rows 8.1, 8 rows 9.8)
  const int64_t columns = cdiv(p->dim, 256 * (wide ? 2 : 1)), rows = std::max(cdiv(columns * p->batch, SMS * 8), cdiv(p->batch, 65535));
  a.rows = (int)(rows > 1 ? (rows + 1) / 2 * 2 : 1);
  if (p->dtype == SSD_DTYPE_BF16) return wide ? launch_step<bf16, 2>(a, st) : launch_step<bf16, 1>(a, st);
  return wide ? launch_step<float, 2>(a, st) : launch_step<float, 1>(a, st);
}

}  // namespace ssd
