// Linear layer with its epilogue fused, for sm_100a (tcgen05 kind::f16, fp32 accumulate; bf16 or fp16 operands):
//   y[m, n] = cast( act(x[m, :] . w[n, :] + bias[n]) + residual[m, n] )
// and, gated, with the weight's rows split into a gate half [0, N) and an up half [N, 2 N):
//   y[m, n] = cast( act(x . w[n] + bias[n]) * (x . w[N + n] + bias[N + n]) + residual[m, n] ).
// Everything between the accumulator and the one final rounding happens in fp32.
//
// linear_stream_kernel streams the WEIGHT through the tensor core's M side: a tile is 128 weight rows (64 gate and 64
// up rows when gated) by up to 128 rows of x, and the accumulator holds y transposed (lane = weight row, column =
// row of x).  A decode step is bound by the weight's bytes, and one SM streams about 1/148 of the HBM bandwidth, so
// the K range of a tile is split over a thread-block cluster of up to 8 CTAs until there are two CTAs for every SM
// (one, where a tile is wider than 64 rows of x).  The partial sums meet in distributed shared memory: column c of the
// tile belongs to rank c % split, every rank stores its fp32 partial of a column into the owner's shared memory, and
// after one cluster barrier the owner adds them in rank order (ascending K: the result does not depend on timing) and
// runs the epilogue.  No workspace, no counters, no atomics: calls on any streams and replays of any graphs are
// independent of each other.  Measured: one row, 8192 x 28672, 69-72 us = 6.5-6.8 TB/s; 16 rows, gated 57344 x 8192,
// 140-145 us = 6.5-6.7 TB/s (a copy runs at 6.54).
//
// linear_pair_kernel takes over where x has more rows than that form can hide behind the weight (see plan_pair).
//
// CTAs of 192 threads: warp 0 TMA producer (128-byte swizzle, no multicast), warp 1 MMA issuer, warps 2-5 move the
// accumulator out of tensor memory; all six run the epilogue.  Every wait is bounded.
#include "gemm_common.cuh"

#include <atomic>
#include <type_traits>

namespace hb200 {

__device__ int g_device_status_linear = 0;

namespace linear {

using namespace sm100;

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kGeluTanh = 4 };

struct Args {
  void* out;             // [M, N], row pitch ldo
  const void* bias;      // [weight rows] in the operand type or (bias_f32) fp32, or nullptr
  const void* residual;  // [M, N] in the output type, row pitch ldr, or nullptr
  int64_t ldo, ldr;
  int m, n, k;           // n: output columns (the weight has 2 n rows when gated)
  int activation;
  int bias_f32;
  int out_vec, res_vec;  // 16-byte accesses are possible
  int cols, m_chunks;    // rows of x per tile (a multiple of 16), tiles along M
  int num_kb;            // K blocks of 64 elements
  int split;             // stream kernel: CTAs per tile (cluster size)
  int stages, stage_bytes;
  int stash_offset;      // bytes from the ring's start to the partial sums (0: they take the ring's place)
  // pair kernel
  int m_tiles, n_tiles;
  int split_log;         // log2 of the pairs per tile
  int tile_cols;         // accumulator columns = weight rows per tile: 128, 192 or 256
  int band;              // row tiles per band of the tile order
};

// ------------------------------------------------------------------ epilogue arithmetic
// The exponential and the reciprocal are the hardware's approximations, off by two units in the last place of fp32:
// far less than what fp32 accumulation of K products leaves in v itself.  Their denormals are zero.
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float activate(float v, int activation) {
  switch (activation) {
    case kRelu: return v > 0.f ? v : (v != v ? v : 0.f);  // a NaN stays a NaN
    case kSilu: return v * reciprocal_fast(1.f + exp2_fast(-kLog2e * v));
    case kGelu: {
      // v Phi(v) = max(v, 0) - |v| Phi(-|v|), Phi(-a) = exp(-a^2 / 2) t R(t) with t = 1 / (1 + 0.44 a / sqrt 2): R is a
      // degree-7 fit of this file's own (weighted least squares on Chebyshev points), off by at most 1.8e-7 of its
      // value for every a, so the small values of the left tail keep their relative precision
      const float a = fminf(fabsf(v), 1e4f), t = reciprocal_fast(fmaf(0.31112698f, a, 1.f));
      float p = fmaf(0.03561173379421234f, t, -0.13897401094436646f);
      p = fmaf(p, t, 0.1483437418937683f);
      p = fmaf(p, t, -0.010090325959026814f);
      p = fmaf(p, t, 0.10790611058473587f);
      p = fmaf(p, t, 0.10865677893161774f);
      p = fmaf(p, t, 0.12443558871746063f);
      p = fmaf(p, t, 0.12411047518253326f);
      // (min(v, -a): -inf times a tail of 0 is NaN as in the formula, while the clamped a keeps +inf)
      return fmaf(fminf(v, -a), exp2_fast(-0.5f * kLog2e * v * v) * (t * p), fmaxf(v, 0.f));
    }
    case kGeluTanh: {
      // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (v + 0.044715 v^3)
      const float u = v * fmaf(-2.f * kLog2e * 0.79788456080286536f * 0.044715f * v, v, -2.f * kLog2e * 0.79788456080286536f);
      return v * reciprocal_fast(1.f + exp2_fast(u));
    }
    default: return v;
  }
}

// The same for an array: one branch on the (uniform) kind in front of the unrolled arithmetic.
template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int activation) {
#define HB200_ACTIVATE(kind)                                  \
  case kind: {                                                \
    _Pragma("unroll") for (int j = 0; j < N; ++j) v[j] = activate(v[j], kind); \
  } break
  switch (activation) {
    HB200_ACTIVATE(kRelu);
    HB200_ACTIVATE(kSilu);
    HB200_ACTIVATE(kGelu);
    HB200_ACTIVATE(kGeluTanh);
    default: break;
  }
#undef HB200_ACTIVATE
}

template <typename T> __device__ __forceinline__ T cast_out(float v);
template <> __device__ __forceinline__ __nv_bfloat16 cast_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half cast_out<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float cast_out<float>(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(float v) { return v; }

// Two values of a 16-byte piece, rounded, in one word (fp32: one value).
template <typename OutT> __device__ __forceinline__ uint32_t pack_word(const float* v);
template <> __device__ __forceinline__ uint32_t pack_word<__nv_bfloat16>(const float* v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack_word<__half>(const float* v) { return h2_as_u32(__floats2half2_rn(v[0], v[1])); }
template <> __device__ __forceinline__ uint32_t pack_word<float>(const float* v) { return __float_as_uint(v[0]); }

template <typename T>
__device__ __forceinline__ float load_bias(const Args& g, int64_t i) {
  return g.bias_f32 ? static_cast<const float*>(g.bias)[i] : widen(static_cast<const T*>(g.bias)[i]);
}

// Eight consecutive values of a row: one or two 16-byte accesses where alignment allows.
template <typename OutT>
__device__ __forceinline__ void load8(const OutT* p, int valid, bool vec, OutT (&v)[8]) {
  if (vec && valid >= 8) {
    constexpr int kPieces = int(sizeof(OutT)) / 2;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < valid ? p[j] : cast_out<OutT>(0.f);
  }
}

template <typename OutT>
__device__ __forceinline__ void store8(OutT* p, int valid, bool vec, const float (&v)[8]) {
  if (vec && valid >= 8) {
    __align__(16) OutT t[8];
    constexpr int kPieces = int(sizeof(OutT)) / 2;
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = cast_out<OutT>(v[j]);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) p[j] = cast_out<OutT>(v[j]);
  }
}

// ------------------------------------------------------------------ tensor core
// Shared-memory descriptors are the low word of the operand's address (with the leading offset) under one constant
// high word (stride 1024 bytes, descriptor version, 128-byte swizzle): the issue loop adds to low words only, so one
// MMA costs it a handful of instructions, fewer than the 128 clocks the MMA runs.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_addr) { return ((smem_addr & 0x3ffffu) >> 4) | (1u << 16); }

__device__ __forceinline__ void mma_f16(uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}

// kind::f16: fp32 accumulator (bits 4-5 = 1), operand format 0 = f16 / 1 = bf16 at bits 7-9 and 10-12 (both operands
// alike), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t make_idesc(int m, int n, bool bf16) {
  return (1u << 4) | (uint32_t(bf16 ? 1 : 0) << 7) | (uint32_t(bf16 ? 1 : 0) << 10) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// Programmatic dependent launch: the kernel may be resident, its barriers and tensor memory set up, before the kernel
// in front of it on the stream has finished.  Nothing of global memory, weights included, is touched before that
// kernel's completion, and the next kernel is let in only after it, so whoever follows sees what a plain order gives.
__device__ __forceinline__ void wait_for_previous_kernel() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// The bounded wait as one decision of a converged warp: what follows is executed by all of its lanes or by none.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// A kernel that gave up a wait lets its own loads land before it leaves: `issued` stages were requested in order.
__device__ __forceinline__ void drain_loads(uint64_t* full_bar, int stages, int issued) {
  const long long t0 = clock64();
  for (int it = issued > stages ? issued - stages : 0; it < issued; ++it)
    while (!mbar_try_wait(smem_u32(&full_bar[it % stages]), (it / stages) & 1) && clock64() - t0 < 20000000) {}
}

// ... and its MMAs finish: they were committed to `bar`, whose phase this waits for.
__device__ __forceinline__ void drain_mmas(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 < 20000000) {}
}

// The tensor core truncates every addition to its accumulator, so a sum drifts towards zero with the length of its
// chain: 1e-9 of the result per element of K (3.8e-6 at 3584, 3.3e-5 at 28672), twice that in a gated product.  That is
// invisible under a 16-bit rounding, but up to 200 times the error of an fp32 product.  For fp32 outputs a chain is
// this many blocks of 64 elements (3e-7 to 7e-7 of the result), and the partial sums are added outside the tensor core,
// to nearest, while the next chain runs in a second accumulator.  Short chains cost the stream kernel nothing; in the
// pair kernel a tile's epilogue hides behind two chains of the next tile only: 4096^3 takes 112 us in one chain, 118 in
// chains of 24 blocks, 125 of 12, 130 of 8.
constexpr int kStreamChain = 4;
template <bool GATED> constexpr int kPairChain = GATED ? 5 : 10;

// ------------------------------------------------------------------ streaming kernel
constexpr int kStreamThreads = 192;
constexpr int kTileRows = 128;                 // weight rows per tile
constexpr int kWBytes = kTileRows * 128;       // one stage of weights: 128 rows x 64 elements
constexpr int kMaxCols = 128;                  // rows of x per tile: 256 took 13 us where 128 takes 8 (512 x 128 x 4096)
constexpr int kMaxStages = 12;
constexpr int kMaxSplit = 8;

template <typename T, typename OutT, bool GATED>
__global__ void __launch_bounds__(kStreamThreads)
linear_stream_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Args g) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kOutRows = GATED ? 64 : 128;  // output columns per tile
  constexpr bool kSums = std::is_same<OutT, float>::value;  // sums over chains of K
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(base);
  uint64_t* empty_bar = full_bar + kMaxStages;
  uint64_t* sum_bar = empty_bar + kMaxStages;  // an accumulator's chain is complete
  uint64_t* free_bar = sum_bar + 2;            // ... and read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(free_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* ring = base + 1024;
  float* stash = reinterpret_cast<float*>(ring + g.stash_offset);  // [rank][column of mine][128] partial sums
  const bool overlay = g.stash_offset == 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = g.split, rank = int(cluster_ctarank());
  const int tile = int(blockIdx.x) / split;
  const int m0 = (tile % g.m_chunks) * g.cols, n0 = (tile / g.m_chunks) * kOutRows;
  const int kb0 = range_start(rank, g.num_kb, split), kb1 = range_start(rank + 1, g.num_kb, split);
  const int live_cols = min(g.cols, g.m - m0);     // columns past the last row of x are never stored
  const int per = (live_cols + split - 1) / split;  // a rank finishes columns rank, rank + split, ...: at most this many
  const int count = (live_cols - rank + split - 1) / split;

  // Epilogue items: eight neighbouring outputs of one column, the same eight for all of a thread's columns.  Their
  // biases and the first residuals are requested before the sums are complete.
  constexpr int kItemsPerCol = kOutRows / 8, kStep = kStreamThreads / kItemsPerCol;
  const int piece = (threadIdx.x % kItemsPerCol) * 8, first = threadIdx.x / kItemsPerCol;
  const int col = n0 + piece, valid = g.n - col;
  float bias[8], bias_up[8];
  __align__(16) OutT res[8];
  auto fetch = [&](int i, OutT (&v)[8]) {
    if (g.residual != nullptr && i < count && valid > 0)
      load8(static_cast<const OutT*>(g.residual) + int64_t(m0 + i * split + rank) * g.ldr + col, valid, g.res_vec != 0, v);
  };
  auto prefetch = [&] {
    fetch(first, res);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool some = g.bias != nullptr && j < valid;
      bias[j] = some ? load_bias<T>(g, col + j) : 0.f;
      bias_up[j] = GATED && some ? load_bias<T>(g, int64_t(g.n) + col + j) : 0.f;
    }
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&sum_bar[a]), 1);
      mbar_init(smem_u32(&free_bar[a]), 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  uint32_t tmem_cols = 32;  // of one accumulator
  while (tmem_cols < uint32_t(g.cols)) tmem_cols *= 2;
  // two accumulators that take turns, then the sums of the chains before them; or one accumulator
  const uint32_t tmem_all = kSums ? 4 * tmem_cols : tmem_cols;
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), tmem_all);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_previous_kernel();
  const int last_chain = kSums ? (kb1 - kb0 - 1) / kStreamChain : 0;
  // A CTA's shared memory may be written by its peers once it runs (or, where the partial sums take the ring's
  // place, once its MMAs have read the ring): arrive here or below, wait in front of the first remote store.
  if (!overlay) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  if (warp == 0) {
    const uint32_t bytes = uint32_t(kWBytes + g.cols * 128);
    int it = 0, s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++it) {
      if (!warp_wait(smem_u32(&empty_bar[s]), phase ^ 1, abort_flag)) break;
      if (elect_one()) {
        const uint32_t bar = smem_u32(&full_bar[s]);
        uint8_t* st = ring + s * g.stage_bytes;
        mbar_arrive_expect_tx(bar, bytes);
        tma_load_2d(smem_u32(st), &tmap_w, kb * 64, n0, bar);
        if constexpr (GATED) tma_load_2d(smem_u32(st + kWBytes / 2), &tmap_w, kb * 64, g.n + n0, bar);
        tma_load_2d(smem_u32(st + kWBytes), &tmap_x, kb * 64, m0, bar);
      }
      __syncwarp();
      if (++s == g.stages) s = 0, phase ^= 1;
    }
    if (*abort_flag) drain_loads(full_bar, g.stages, it);
    prefetch();
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc(kTileRows, g.cols, kBf16);
    const uint32_t ring_low = desc_low(smem_u32(ring)), stage_low = uint32_t(g.stage_bytes) >> 4;
    const int tail_steps = (g.k - (g.num_kb - 1) * 64 + 15) / 16;  // K tail: TMA zero-fills past K
    bool ok = true;
    int link = 0, chains = 0;  // blocks of the current chain so far, chains before it
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      uint32_t tmem_d = tmem_base;
      if constexpr (kSums) {
        tmem_d += (chains & 1) * tmem_cols;
        if (link == 0 && !warp_wait(smem_u32(&free_bar[chains & 1]), ((chains >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
      }
      if (!warp_wait(smem_u32(&full_bar[s]), phase, abort_flag)) { ok = false; break; }
      tcgen05_fence_after();
      const uint32_t w_low = ring_low + uint32_t(s) * stage_low, x_low = w_low + (kWBytes >> 4);
      const uint32_t more = link != 0 ? 1u : 0u;
      if (elect_one()) {
        if (kb != g.num_kb - 1 || tail_steps == 4) {
          mma_f16(tmem_d, w_low, x_low, idesc, more);
#pragma unroll
          for (int a = 1; a < 4; ++a) mma_f16(tmem_d, w_low + a * 2, x_low + a * 2, idesc, 1u);
        } else {
          for (int a = 0; a < tail_steps; ++a) mma_f16(tmem_d, w_low + a * 2, x_low + a * 2, idesc, more | uint32_t(a));
        }
        tcgen05_commit(smem_u32(&empty_bar[s]));
        if (kb == kb1 - 1 || (kSums && link == kStreamChain - 1)) tcgen05_commit(smem_u32(&sum_bar[chains & 1]));
      }
      __syncwarp();
      ++link;
      if (kSums && link == kStreamChain) link = 0, ++chains;
      if (++s == g.stages) s = 0, phase ^= 1;
    }
    if (!ok) {
      if (elect_one()) tcgen05_commit(smem_u32(&sum_bar[chains & 1]));
      __syncwarp();
      drain_mmas(smem_u32(&sum_bar[chains & 1]), (chains >> 1) & 1);
    }
    prefetch();
  } else {
    prefetch();
    bool ok = true;
    if constexpr (kSums) {  // all chains but the last: into the sums
      const uint32_t taddr = tmem_base + (uint32_t((warp & 3) * 32) << 16);
      for (int chain = 0; chain < last_chain && ok; ++chain) {
        ok = warp_wait(smem_u32(&sum_bar[chain & 1]), (chain >> 1) & 1, abort_flag);
        tcgen05_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < live_cols; c0 += 16) {
          uint32_t r[16], t[16];
          tmem_ld_32x32b_x16(taddr + (chain & 1) * tmem_cols + c0, r);
          if (chain > 0) {
            tmem_ld_32x32b_x16(taddr + 2 * tmem_cols + c0, t);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(t[j]));
          } else {
            tmem_ld_wait();
          }
          tmem_st_32x32b_x16(taddr + 2 * tmem_cols + c0, r);
        }
        tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&free_bar[chain & 1]));
      }
    }
    if (ok) warp_wait(smem_u32(&sum_bar[last_chain & 1]), (last_chain >> 1) & 1, abort_flag);
    tcgen05_fence_after();
  }
  __syncwarp();
  if (overlay) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  if (warp >= 2) {
    const int quarter = warp & 3;
    const int r_in = quarter * 32 + lane;  // weight row inside the tile = accumulator lane
    const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16);
    const uint32_t mine = smem_u32(stash) + uint32_t((rank * per) * 128 + r_in) * 4u;
    int owner = 0, index = 0;  // of column c: c % split and c / split (in turn: runs would send all ranks to one at a time)
#pragma unroll 1
    for (int c0 = 0; c0 < live_cols; c0 += 8) {
      uint32_t r[8];
      tmem_ld_32x32b_x8(taddr + (last_chain & 1) * tmem_cols + c0, r);
      if (kSums && last_chain > 0) {
        uint32_t t[8];
        tmem_ld_32x32b_x8(taddr + 2 * tmem_cols + c0, t);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(t[j]));
      } else {
        tmem_ld_wait();
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c0 + j < live_cols) st_cluster_f32(map_to_cta(mine + uint32_t(index) * 512u, uint32_t(owner)), __uint_as_float(r[j]));
        if (++owner == split) owner = 0, ++index;
      }
    }
    tcgen05_fence_before();
  }
  __syncwarp();
  // Orders the remote stores before the loads below; after it nobody touches another CTA's shared memory again.
  cluster_sync_all();

  // (not unrolled: a launch runs this code once, and its instructions come in at the speed of a cold cache)
#pragma unroll 1
  for (int i = first; i < count && valid > 0; i += kStep) {
    __align__(16) OutT r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = res[j];
    fetch(i + kStep, res);
    float acc[8], up[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = up[j] = 0.f;
    for (int q = 0; q < split; ++q) {
      const float4* src = reinterpret_cast<const float4*>(stash + (q * per + i) * 128 + piece);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 v = src[h];
        acc[4 * h] += v.x, acc[4 * h + 1] += v.y, acc[4 * h + 2] += v.z, acc[4 * h + 3] += v.w;
        if constexpr (GATED) {
          const float4 w = src[16 + h];
          up[4 * h] += w.x, up[4 * h + 1] += w.y, up[4 * h + 2] += w.z, up[4 * h + 3] += w.w;
        }
      }
    }
    if (g.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += bias[j], up[j] += bias_up[j];
    }
    activate_all(acc, g.activation);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (GATED) acc[j] *= up[j];
      if (g.residual != nullptr) acc[j] += widen(r[j]);
    }
    store8(static_cast<OutT*>(g.out) + int64_t(m0 + i * split + rank) * g.ldo + col, valid, g.out_vec != 0, acc);
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, tmem_all);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicMin(&g_device_status_linear, HB200_ERR_DEVICE_TIMEOUT);
}

// ------------------------------------------------------------------ pair kernel
// Many rows of x: two CTAs on neighbouring SMs own one tile of 256 rows of x by 256 weight rows (gated: 128 gate rows,
// held by the leader, and the 128 up rows of the same outputs, held by its peer, so gate and up of an output meet in
// one accumulator lane 128 columns apart).  CTA r of the pair loads its 128 rows of x and its 128 weight rows, the
// leader issues 256 x 256 x 16 MMAs (cta_group::2) that read both: per 64 elements of K every SM pulls 32 KB from L2
// for 512 clocks of tensor work.  Two accumulators in tensor memory, so a tile's epilogue runs beside the next
// tile's MMAs; the grid is persistent.  At 8192^3 the tensor pipe is 98 % active and the GPU's power limit sets the
// time: 1.30 PFLOP/s in sequence, 1.58 in a single launch.  Tiles of 512 x 256 (a quarter fewer bytes out of L2 per
// product) measured 1 to 3 % faster there and up to 15 % slower at K = 1024, where their epilogue shows: not taken.
//
// Epilogue: sixteen warps per CTA, each 32 rows by 64 accumulator columns (gated: 32 gate and 32 up columns), a lane
// per row.  Outputs leave through boxes of 32 rows x 64 bytes in shared memory, two per warp in turn, by TMA where the
// output's pitch allows, else row by row with consecutive lanes on consecutive elements; the residual comes in through
// the same boxes.  Measured at 4096 x 16384 x 1024, where the epilogue shows, SiLU and residual: 151 us; a lane reading
// and writing its own row in 32-byte sectors 167; one box per warp and a sixth stage in its place 165 (the two are level
// from K = 4096 on).
constexpr int kPairThreads = 576;              // producer, MMA issuer, sixteen epilogue warps
constexpr int kPairTile = 256;                 // rows of x per tile
constexpr int kHalfBytes = 128 * 128;          // 128 rows of x (or of the weight) x 64 elements of K
constexpr int kPairRingBytes = 10 * kHalfBytes;  // 160 KB: five or six stages
constexpr int kPairMaxStages = 6;
constexpr int kBoxBytes = 2048;                // two boxes per epilogue warp
constexpr int kEpilogueWarps = 16;
constexpr int kAcc = 2;
constexpr int kPairBand = 8;                   // row tiles per band: 8192^3 reads 1.06 GB of DRAM (4: 1.51 GB, 16: 1.23 GB)
constexpr size_t kPairSmem = size_t(kPairRingBytes) + kEpilogueWarps * 2 * kBoxBytes + (2 * kPairMaxStages + 2 * kAcc) * 8 + 16 + 1024;
static_assert(kPairSmem <= 232448, "shared memory budget exceeded");

__device__ __forceinline__ void mma_pair_f16(uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}

// Bands of `band` row tiles; inside a band the row tile runs fastest: the pairs at work at one time share a few row
// tiles of x and a few tiles of the weight, which stay in L2.
__device__ __forceinline__ void decode_tile(const Args& g, int tile, int& m_blk, int& n_blk) {
  const int per_band = g.band * g.n_tiles;
  const int b = tile / per_band, r = tile - b * per_band;
  const int rows_here = min(g.band, g.m_tiles - b * g.band);
  n_blk = r / rows_here;
  m_blk = b * g.band + (r - n_blk * rows_here);
}

// 16-byte chunk c of row r of a box: the 64-byte swizzle of the TMA store.
__device__ __forceinline__ uint32_t box_chunk(int r, int c) { return uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4)); }

// Residual rows [row0, row0 + 32) x columns [col, col + 64 / size) into a box: aligned ones asynchronously in 16-byte
// pieces (four lanes on the 64 bytes of a row; no registers wait for them), others element by element, consecutive
// lanes on consecutive elements.
template <typename OutT>
__device__ __forceinline__ void fetch_box_async(const Args& g, uint8_t* box, int row0, int col, int lane) {
  constexpr int kPer = 16 / int(sizeof(OutT));
  const OutT* src = static_cast<const OutT*>(g.residual) + col + (lane & 3) * kPer;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    if (row0 + r < g.m)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(box + box_chunk(r, lane & 3))),
                   "l"(src + int64_t(row0 + r) * g.ldr) : "memory");
  }
}

template <typename OutT>
__device__ __forceinline__ void fetch_box(const Args& g, uint8_t* box, int row0, int col, int lane) {
  constexpr int kCols = 64 / int(sizeof(OutT)), kPer = 16 / int(sizeof(OutT));
  const OutT* src = static_cast<const OutT*>(g.residual);
  constexpr int kRowsAtOnce = 32 / kCols, kLoads = 32 / kRowsAtOnce;  // 32 (16-bit) or 16 (fp32), all in flight at once
  const int c = lane % kCols;
  OutT v[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = i * kRowsAtOnce + lane / kCols;
    v[i] = cast_out<OutT>(0.f);
    if (row0 + r < g.m && col + c < g.n) v[i] = src[int64_t(row0 + r) * g.ldr + col + c];
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    *reinterpret_cast<OutT*>(box + box_chunk(i * kRowsAtOnce + lane / kCols, c / kPer) + (c % kPer) * sizeof(OutT)) = v[i];
}

// A box to the output: consecutive lanes write consecutive elements.
template <typename OutT>
__device__ __forceinline__ void flush_box(const Args& g, const uint8_t* box, int row0, int col, int lane) {
  constexpr int kCols = 64 / int(sizeof(OutT)), kPer = 16 / int(sizeof(OutT)), kRowsAtOnce = 32 / kCols;
  OutT* dst = static_cast<OutT*>(g.out);
  const int c = lane % kCols;
#pragma unroll 8
  for (int i = 0; i < 32; i += kRowsAtOnce) {
    const int r = i + lane / kCols;
    if (row0 + r < g.m && col + c < g.n)
      dst[int64_t(row0 + r) * g.ldo + col + c] =
          *reinterpret_cast<const OutT*>(box + box_chunk(r, c / kPer) + (c % kPer) * sizeof(OutT));
  }
}

// One warp polls an mbarrier for all sixteen epilogue warps; the others wait in a named barrier, which takes neither
// issue slots nor power from the tensor work (a large product runs at the power limit).  The outcome is reduced over
// the barrier, so every warp takes the same way.
__device__ __forceinline__ bool epilogue_wait(bool polls, uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t got = 1;
  if (polls) got = warp_wait(bar, parity, abort_flag) ? 1u : 0u;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred.aligned q, 1, 512, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(got)
      : "r"(got)
      : "memory");
  return got != 0;
}

__device__ __forceinline__ void st_cluster_v4(uint32_t cluster_addr, const uint32_t (&v)[32], int at) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "r"(v[at]), "r"(v[at + 1]), "r"(v[at + 2]),
               "r"(v[at + 3]) : "memory");
}
__device__ __forceinline__ void cluster_arrive_all() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait_all() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// SPLIT: fewer tiles than half the pairs of the GPU.  A cluster of two or four pairs works on one tile, each pair on a
// share of K, and the partial sums meet in distributed shared memory: of the four groups of 64 accumulator columns that
// a CTA's epilogue warps hold, pair q finishes groups [4 q / split, 4 (q + 1) / split) and receives the others' partials
// of these, of its own 128 rows, in the place of the ring that all MMAs have read.  They are added in the order of the
// pairs (own first), so the result does not depend on timing.  200 x 8192 x 8192 in a loop of this call alone: 35 us with
// two pairs per tile (whether the weight changes from call to call or not), 51 with one, 42 in the streaming form.
template <typename T, typename OutT, bool GATED, bool SPLIT>
__global__ void __launch_bounds__(kPairThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                   const __grid_constant__ CUtensorMap tmap_out, const Args g) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const int tile_cols = g.tile_cols, out_cols = GATED ? tile_cols / 2 : tile_cols;  // (accumulator, output) columns per tile
  const int w_bytes = tile_cols * 64;                   // this CTA's half of the tile's weight rows x 64 elements of K
  const int num_stages = g.stages, stage_bytes = g.stage_bytes;
  constexpr int kBoxCols = 64 / int(sizeof(OutT));      // output columns per box
  constexpr int kBoxesPer32 = 32 / kBoxCols;            // 1 (16-bit outputs) or 2 (fp32)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* boxes = smem + kPairRingBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(boxes + kEpilogueWarps * 2 * kBoxBytes);  // used in the leader only
  uint64_t* empty_bar = full_bar + kPairMaxStages;                           // one set per CTA
  uint64_t* tmem_full_bar = empty_bar + kPairMaxStages;
  uint64_t* tmem_empty_bar = tmem_full_bar + kAcc;                           // used in the leader only
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty_bar + kAcc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cluster_rank = cluster_ctarank(), rank = cluster_rank & 1u;  // rank in the pair
  const uint32_t leader_rank = cluster_rank & ~1u;
  const bool leader = rank == 0;
  const uint16_t pair_mask = uint16_t(3u << leader_rank);
  const int split_log = SPLIT ? g.split_log : 0, part = SPLIT ? int(cluster_rank >> 1) : 0;
  // a tile per cluster when split, else tiles dealt to the pairs in turn
  const int pair = blockIdx.x >> (1 + split_log), num_pairs = gridDim.x >> (1 + split_log);
  const int num_tiles = g.m_tiles * g.n_tiles;
  const int kb0 = SPLIT ? range_start(part, g.num_kb, 1 << split_log) : 0;
  const int kb1 = SPLIT ? range_start(part + 1, g.num_kb, 1 << split_log) : g.num_kb;
  constexpr bool kSums = std::is_same<OutT, float>::value;  // sums over chains of K
  constexpr int kChain = kPairChain<GATED>;

  if (threadIdx.x == 0) {
    for (int s = 0; s < num_stages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);   // the leader's producer arms it; bytes come from both CTAs
      mbar_init(smem_u32(&empty_bar[s]), 1);  // the leader's commit, sent to both CTAs
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(smem_u32(&tmem_full_bar[a]), 1);
      mbar_init(smem_u32(&tmem_empty_bar[a]), 32);  // sixteen epilogue warps in each CTA
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // barriers of both CTAs are initialised before anything remote happens
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_previous_kernel();

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    int it = 0, s = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      int m_blk, n_blk;
      decode_tile(g, tile, m_blk, n_blk);
      const int x_row = m_blk * kPairTile + int(rank) * 128;
      const int w_row = n_blk * out_cols + int(rank) * (GATED ? g.n : tile_cols / 2);
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        if (!warp_wait(smem_u32(&empty_bar[s]), phase ^ 1, abort_flag)) { ok = false; break; }
        uint8_t* st = smem + s * stage_bytes;
        const uint32_t bar = map_to_cta(smem_u32(&full_bar[s]), leader_rank);  // always the leader's barrier
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(smem_u32(&full_bar[s]), uint32_t(2 * (kHalfBytes + w_bytes)));
          tma_load_2d_pair(smem_u32(st), &tmap_x, kb * 64, x_row, bar);
          tma_load_2d_pair(smem_u32(st + kHalfBytes), &tmap_w, kb * 64, w_row, bar);
        }
        __syncwarp();
        if (++s == num_stages) s = 0, phase ^= 1;
      }
    }
    if (leader && *abort_flag) drain_loads(full_bar, num_stages, it);
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer (leader only)
    if (leader) {
      const uint32_t idesc = make_idesc(256, tile_cols, kBf16);
      const uint32_t ring_low = desc_low(smem_u32(smem));
      const int tail_steps = (g.k - (g.num_kb - 1) * 64 + 15) / 16;  // K tail: TMA zero-fills past K
      bool ok = true;
      uint32_t s = 0, phase = 0, tc = 0;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
        int link = 0;  // blocks of the current chain so far; tc counts chains
        for (int kb = kb0; kb < kb1; ++kb) {
          const uint32_t acc = tc % kAcc, tmem_d = tmem_base + acc * 256;
          if (link == 0 && !warp_wait(smem_u32(&tmem_empty_bar[acc]), ((tc / kAcc) & 1) ^ 1, abort_flag)) { ok = false; break; }
          if (!warp_wait(smem_u32(&full_bar[s]), phase, abort_flag)) { ok = false; break; }
          tcgen05_fence_after();
          const uint32_t x_low = ring_low + s * uint32_t(stage_bytes >> 4), w_low = x_low + (kHalfBytes >> 4);
          const bool last = kb == kb1 - 1 || (kSums && link == kChain - 1);
          const uint32_t more = link != 0 ? 1u : 0u;
          if (elect_one()) {
            if (kb != g.num_kb - 1 || tail_steps == 4) {
              mma_pair_f16(tmem_d, x_low, w_low, idesc, more);
#pragma unroll
              for (int a = 1; a < 4; ++a) mma_pair_f16(tmem_d, x_low + a * 2, w_low + a * 2, idesc, 1u);
            } else {
              for (int a = 0; a < tail_steps; ++a) mma_pair_f16(tmem_d, x_low + a * 2, w_low + a * 2, idesc, more | uint32_t(a));
            }
            tcgen05_commit_pair(smem_u32(&empty_bar[s]), pair_mask);  // stage free in both CTAs
            if (last) tcgen05_commit_pair(smem_u32(&tmem_full_bar[acc]), pair_mask);
          }
          __syncwarp();
          if (++s == uint32_t(num_stages)) s = 0, phase ^= 1;
          ++link;
          if (last) link = 0, ++tc;
        }
      }
      if (!ok) {
        const uint32_t bar = smem_u32(&tmem_full_bar[tc % kAcc]);
        if (elect_one()) tcgen05_commit_pair(bar, pair_mask);
        __syncwarp();
        drain_mmas(bar, (tc / kAcc) & 1);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quarter = warp & 3, cgroup = (warp - 2) >> 2;  // a warp may read lane quarter warp % 4 only
    uint8_t* my_boxes = boxes + (warp - 2) * 2 * kBoxBytes;
    constexpr int kBlocks = GATED ? 1 : 2;                // blocks of 32 output columns per warp and tile
    constexpr int kPer = 16 / int(sizeof(OutT));          // elements per 16-byte chunk
    const OutT* residual = static_cast<const OutT*>(g.residual);
    const bool tma_out = g.out_vec != 0;
    uint32_t tc = 0;
    constexpr int kSub = kBlocks * kBoxesPer32;           // boxes of outputs per warp and tile
    uint32_t boxes_used = 0;                              // the two boxes take turns
    for (int tile = pair; tile < num_tiles; tile += num_pairs) {
      int m_blk, n_blk;
      decode_tile(g, tile, m_blk, n_blk);
      const int row0 = m_blk * kPairTile + int(rank) * 128 + quarter * 32;
      const int col0 = n_blk * out_cols + cgroup * (32 * kBlocks);
      // this warp has columns to finish: the tile is that wide, and (split) they are this pair's
      const bool mine = cgroup * (32 * kBlocks) < out_cols && (!SPLIT || (cgroup >> (2 - split_log)) == part);
      // the columns' biases: lane l keeps that of column l of each of the two blocks of 32 accumulator columns
      float bias_l[2] = {0.f, 0.f};
      if (mine && g.bias != nullptr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = col0 + (GATED ? 0 : h * 32) + lane;
          if (c < g.n) bias_l[h] = load_bias<T>(g, c + (GATED && h == 1 ? g.n : 0));
        }
      }
      // Both boxes' residuals are requested before the wait for the accumulator: a load queues behind the ring's
      // 160 KB in flight and takes microseconds.
      auto async = [&](int i) { return g.res_vec != 0 && col0 + (i + 1) * kBoxCols <= g.n; };
      if (mine && residual != nullptr) {
        if (lane == 0) {  // the last stores have left the boxes that are filled now
          if constexpr (kSub == 1) bulk_wait_group_read1(); else bulk_wait_group_read0();
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < (kSub < 2 ? kSub : 2); ++i) {
          uint8_t* box = my_boxes + ((boxes_used + i) & 1) * kBoxBytes;
          if (async(i)) fetch_box_async<OutT>(g, box, row0, col0 + i * kBoxCols, lane);
          else if (col0 + i * kBoxCols < g.n) fetch_box<OutT>(g, box, row0, col0 + i * kBoxCols, lane);
        }
      }
      bool ready = epilogue_wait(warp == 2, smem_u32(&tmem_full_bar[tc % kAcc]), (tc / kAcc) & 1, abort_flag);
      if (!SPLIT && !ready) break;  // (split: the cluster's barriers are still to be met)
      tcgen05_fence_after();
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + cgroup * (32 * kBlocks);
      uint32_t r[2][32];  // two blocks of 32 columns (gated: gate and up)
      tmem_ld_32x32b_x32(taddr + (tc % kAcc) * 256, r[0]);
      tmem_ld_32x32b_x32(taddr + (tc % kAcc) * 256 + (GATED ? out_cols : 32), r[1]);
      tmem_ld_wait();
      // everything is in registers: hand the accumulator back
      auto hand_back = [&] {
        tcgen05_fence_before();
        __syncwarp();
        if ((!SPLIT || kSums) && lane == 0)
          mbar_arrive_cluster(map_to_cta(smem_u32(&tmem_empty_bar[tc % kAcc]), leader_rank));
        ++tc;
      };
      hand_back();
      if constexpr (kSums) {
#pragma unroll 1
        for (int kb = kb0 + kChain; kb < kb1 && ready; kb += kChain) {
          ready = epilogue_wait(warp == 2, smem_u32(&tmem_full_bar[tc % kAcc]), (tc / kAcc) & 1, abort_flag);
          tcgen05_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < 64; c0 += 8) {
            uint32_t t[8];
            tmem_ld_32x32b_x8(taddr + (tc % kAcc) * 256 + (c0 < 32 ? c0 : c0 - 32 + (GATED ? out_cols : 32)), t);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t& sum = r[c0 / 32][c0 % 32 + j];
              sum = __float_as_uint(__uint_as_float(sum) + __uint_as_float(t[j]));
            }
          }
          hand_back();
        }
        if (!SPLIT && !ready) break;
      }
      if constexpr (SPLIT) {
        // groups per pair; slot = [source][group of mine][quarter][block of 32 columns], 4 KB each: 32 lanes x 16 bytes x 8
        const int own_log = 2 - split_log, owner = cgroup >> own_log, split = 1 << split_log;
        auto slot = [&](int source) {
          return uint32_t(((((source << own_log) + (cgroup & ((1 << own_log) - 1))) * 4 + quarter) * 2) * 4096 + lane * 16);
        };
        cluster_arrive_all();
        cluster_wait_all();  // every pair's MMAs have read its ring
        if (owner != part) {
          const int index = part < owner ? part : part - 1;  // among the owner's sources
          const uint32_t dst = map_to_cta(smem_u32(smem) + slot(index), uint32_t(owner * 2) + rank);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; ++j) st_cluster_v4(dst + uint32_t(h * 4096 + j * 512), r[h], 4 * j);
        }
        __syncwarp();
        cluster_arrive_all();
        cluster_wait_all();  // the partial sums are here
        if (!mine) continue;
        for (int source = 0; source < split - 1; ++source) {
          const uint8_t* src = smem + slot(source);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 v = *reinterpret_cast<const float4*>(src + h * 4096 + j * 512);
              r[h][4 * j] = __float_as_uint(__uint_as_float(r[h][4 * j]) + v.x);
              r[h][4 * j + 1] = __float_as_uint(__uint_as_float(r[h][4 * j + 1]) + v.y);
              r[h][4 * j + 2] = __float_as_uint(__uint_as_float(r[h][4 * j + 2]) + v.z);
              r[h][4 * j + 3] = __float_as_uint(__uint_as_float(r[h][4 * j + 3]) + v.w);
            }
        }
      }
      if (!mine) continue;
#pragma unroll
      for (int h = 0; h < kBlocks; ++h) {
        if (col0 + h * 32 >= g.n) break;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[h][j]);
        if (g.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += __shfl_sync(0xffffffffu, bias_l[h], j);
        }
        activate_all(v, g.activation);
        if constexpr (GATED) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float up = __uint_as_float(r[1][j]);
            if (g.bias != nullptr) up += __shfl_sync(0xffffffffu, bias_l[1], j);
            v[j] *= up;
          }
        }
#pragma unroll
        for (int b = 0; b < kBoxesPer32; ++b, ++boxes_used) {
          const int i = h * kBoxesPer32 + b, col = col0 + i * kBoxCols;
          uint8_t* box = my_boxes + (boxes_used & 1) * kBoxBytes;
          if (residual == nullptr || i >= 2) {
            if (lane == 0) bulk_wait_group_read1();  // this box's last store has left it (the other's may be on its way)
            __syncwarp();
          }
          if (residual != nullptr) {
            if (i >= 2 && async(i)) fetch_box_async<OutT>(g, box, row0, col, lane);
            else if (i >= 2) fetch_box<OutT>(g, box, row0, col, lane);
            asm volatile("cp.async.wait_all;" ::: "memory");
          }
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint4* slot = reinterpret_cast<uint4*>(box + box_chunk(lane, c));
            float* e = v + b * kBoxCols + c * kPer;
            if (residual != nullptr) {
              const uint4 raw = *slot;
              const OutT* res = reinterpret_cast<const OutT*>(&raw);
#pragma unroll
              for (int j = 0; j < kPer; ++j) e[j] += widen(res[j]);
            }
            constexpr int kPerWord = kPer / 4;
            *slot = make_uint4(pack_word<OutT>(e), pack_word<OutT>(e + kPerWord), pack_word<OutT>(e + 2 * kPerWord),
                               pack_word<OutT>(e + 3 * kPerWord));
          }
          if (tma_out) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (row0 < g.m && col < g.n) tma_store_2d(&tmap_out, col, row0, smem_u32(box));  // clipped at the edges
              bulk_commit_group();  // one group per box, stored or not: the waits above count groups
            }
          } else {
            __syncwarp();
            flush_box<OutT>(g, box, row0, col, lane);
            __syncwarp();
          }
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (lane == 0) bulk_wait_group_read0();
  }

  if constexpr (SPLIT) {
    if (warp < 2) {  // the two barriers of the exchange
      __syncwarp();
      cluster_arrive_all();
      cluster_wait_all();
      cluster_arrive_all();
      cluster_wait_all();
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer is done with this CTA's shared memory, barriers and tensor memory
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicMin(&g_device_status_linear, HB200_ERR_DEVICE_TIMEOUT);
}

// ------------------------------------------------------------------ host side
// K-major 2-byte matrix [rows, K] with a row pitch of `pitch` elements; box = 64 elements (128 bytes) x box_rows.
bool make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t pitch, int box_rows, bool bf16) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cuuint64_t(k), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(pitch) * 2};
  const cuuint32_t box[2] = {64, cuuint32_t(box_rows)};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base),
            dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Output boxes of the pair kernel: 64 bytes x 32 rows, 64-byte swizzle.
bool make_out_map(CUtensorMap* map, void* base, int64_t rows, int64_t cols, int64_t pitch, bool f32, bool bf16) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const int size = f32 ? 4 : 2;
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(pitch) * size};
  const cuuint32_t box[2] = {cuuint32_t(64 / size), 32};
  const cuuint32_t elem[2] = {1, 1};
  const CUtensorMapDataType type = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : (bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
  return fn(map, type, 2, base, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a launch asks the runtime about the device and the kernel, asked once per device: together these calls cost as
// much host time as the launch itself.
int device_sms(int dev) {
  static std::atomic<int> known[64];
  if (dev < 0 || dev >= 64) return 148;
  int sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
    known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

template <auto KERNEL>
bool allow_shared_memory(int dev) {
  static std::atomic<bool> done[64];
  if (dev < 0 || dev >= 64) return false;
  if (done[dev].load(std::memory_order_acquire)) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return false;
  done[dev].store(true, std::memory_order_release);
  return true;
}

// How many clusters of `size` CTAs with `smem` bytes each the device holds at once; asked once per device and kind.
template <auto KERNEL>
int max_clusters(int dev, int kind, int size, int threads, size_t smem) {
  static std::atomic<int> known[64][2][4];
  if (dev < 0 || dev >= 64) return 0;
  const int log = size == 8 ? 3 : (size == 4 ? 2 : (size == 2 ? 1 : 0));
  int n = known[dev][kind][log].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(size) * 64, 1, 1);
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!allow_shared_memory<KERNEL>(dev) || cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();  // the launch itself will say what is wrong
      n = -1;
    }
    known[dev][kind][log].store(n, std::memory_order_relaxed);
  }
  return n > 0 ? n : 0;
}

constexpr size_t kNarrowSmem = 111 * 1024, kWideSmem = 227 * 1024;

struct StreamPlan {
  int cols, m_chunks, num_kb, split, stages, stage_bytes, stash_offset;
  int64_t tiles;
  size_t smem;
};

// Shared memory decides how many CTAs share an SM, and tensor memory must never run short while they do (a CTA that
// waits for columns could hold up its cluster peers): narrow tiles (at most 64 columns) get half an SM, wider ones a
// whole SM.  The K range is split while all CTAs run at once and every one keeps four K blocks or more.  One row, 8192 x
// 28672: 64 tiles over 4 CTAs each 72.8 us, over 2 88.7, over 8 (more CTAs than places) 76.9.
StreamPlan plan_stream(int64_t m, int64_t n, int64_t k, bool gated, int dev, int sms) {
  StreamPlan p{};
  p.m_chunks = int((m + kMaxCols - 1) / kMaxCols);
  p.cols = int(((m + p.m_chunks - 1) / p.m_chunks + 15) / 16 * 16);
  p.num_kb = int((k + 63) / 64);
  const int out_rows = gated ? 64 : 128;
  p.tiles = ((n + out_rows - 1) / out_rows) * p.m_chunks;
  const bool narrow = p.cols <= 64;
  p.smem = narrow ? kNarrowSmem : kWideSmem;
  p.split = 1;
  if (narrow) {
    const int64_t places = 2 * sms / p.tiles, shares = p.num_kb / 4;
    const int64_t split = places < shares ? places : shares;
    p.split = split < 1 ? 1 : (split > kMaxSplit ? kMaxSplit : int(split));
  } else {
    while (p.split < kMaxSplit && p.num_kb >= 8 * p.split &&
           p.tiles <= max_clusters<linear_stream_kernel<__nv_bfloat16, __nv_bfloat16, false>>(dev, 1, p.split * 2, kStreamThreads, p.smem))
      p.split *= 2;
  }
  p.stage_bytes = kWBytes + ((p.cols * 128 + 1023) / 1024) * 1024;
  const int budget = int(p.smem) - 2048;  // less barriers and alignment
  const int stash = (p.cols + p.split - 1) / p.split * p.split * 512;
  p.stages = (narrow ? budget - stash : budget) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.stash_offset = narrow ? p.stages * p.stage_bytes : 0;  // wide: the partial sums take the ring's place
  return p;
}

struct PairPlan {
  int tile_cols, split_log;
  int64_t m_tiles, n_tiles;
};

// Estimated microseconds, from single-GPU measurements of both kernels over N = 1024 .. 28672, K = 1024 .. 28672 and
// M = 48 .. 2048: they only have to put the forms in the right order (the pick is within 10 % of the best form on that
// grid, mostly the best).  A pair takes 0.27 us per 64 elements of K and 256 columns, 0.215 for 192 and 0.20 for 128
// (bound by what an SM gets out of L2, not by the MMAs), a third more when every SM is busy (the clock drops), 7 us for
// launch, first loads and last epilogue, and 2 to 3 us for an exchange of partial sums.  The stream kernel is bound by
// the weight's bytes at 4.8 TB/s or by 55 bytes per clock into an SM, and every wave of its CTAs pays for its start and its epilogue.
PairPlan plan_pair(int64_t m, int64_t weight_rows, int64_t k, int dev, int sms, double* us) {
  constexpr int kCols[3] = {256, 192, 128};
  constexpr double kPerBlock[3] = {0.27, 0.215, 0.20}, kExchange[3] = {0.0, 2.0, 3.0};
  const double num_kb = double((k + 63) / 64);
  PairPlan best{};
  *us = 1e30;
  for (int c = 0; c < 3; ++c) {
    const int64_t m_tiles = (m + kPairTile - 1) / kPairTile, n_tiles = (weight_rows + kCols[c] - 1) / kCols[c];
    const int64_t tiles = m_tiles * n_tiles;
    for (int log = 0; log < 3; ++log) {
      if (log > 0 && (num_kb < 4 << log ||
                      tiles > max_clusters<linear_pair_kernel<__nv_bfloat16, __nv_bfloat16, false, true>>(
                                  dev, 0, 2 << log, kPairThreads, kPairSmem)))
        break;
      const double pairs = sms / 2, busy = double(tiles << log) < pairs ? double(tiles << log) / pairs : 1.0;
      const double waves = log > 0 ? 1.0 : double((tiles + sms / 2 - 1) / (sms / 2));
      const double t = 7.0 + kExchange[log] + waves * num_kb / (1 << log) * kPerBlock[c] * (1.0 + 0.35 * busy);
      if (t < *us) {
        *us = t;
        best = PairPlan{kCols[c], log, m_tiles, n_tiles};
      }
    }
  }
  return best;
}

double stream_us(const StreamPlan& p, double weight_bytes, int sms) {
  const double waves = double((p.tiles * p.split + sms - 1) / sms);
  const double feed = waves * p.num_kb / p.split * (kWBytes + p.cols * 128) / (55.0 * 1900.0);
  const double memory = weight_bytes / 4.8e6;
  return waves * (2.5 + 0.03 * p.cols) + (memory > feed ? memory : feed);
}

// A cluster of `size` CTAs, launched as a programmatic dependent of whatever precedes it on the stream.
void launch_attributes(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], unsigned size) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
}

template <typename T, typename OutT, bool GATED>
int launch_stream(const CUtensorMap& tw, const CUtensorMap& tx, const Args& g, const StreamPlan& p, int dev, cudaStream_t stream) {
  auto kernel = linear_stream_kernel<T, OutT, GATED>;
  if (!allow_shared_memory<linear_stream_kernel<T, OutT, GATED>>(dev)) return HB200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.tiles * p.split), 1, 1);
  cfg.blockDim = dim3(kStreamThreads, 1, 1);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  launch_attributes(cfg, attr, unsigned(p.split));
  if (cudaLaunchKernelEx(&cfg, kernel, tw, tx, g) != cudaSuccess) return HB200_ERR_CUDA;
  return HB200_OK;
}

template <typename T>
int launch_stream_typed(const CUtensorMap& tw, const CUtensorMap& tx, const Args& g, const StreamPlan& p, bool gated,
                        bool out_f32, int dev, cudaStream_t s) {
  if (gated) return out_f32 ? launch_stream<T, float, true>(tw, tx, g, p, dev, s) : launch_stream<T, T, true>(tw, tx, g, p, dev, s);
  return out_f32 ? launch_stream<T, float, false>(tw, tx, g, p, dev, s) : launch_stream<T, T, false>(tw, tx, g, p, dev, s);
}

template <typename T, typename OutT, bool GATED, bool SPLIT>
int launch_pair(const CUtensorMap& tw, const CUtensorMap& tx, const CUtensorMap& to, const Args& g, int pairs, int dev,
                cudaStream_t stream) {
  auto kernel = linear_pair_kernel<T, OutT, GATED, SPLIT>;
  if (!allow_shared_memory<linear_pair_kernel<T, OutT, GATED, SPLIT>>(dev)) return HB200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(2 * pairs), 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  launch_attributes(cfg, attr, SPLIT ? 2u << g.split_log : 2u);
  if (cudaLaunchKernelEx(&cfg, kernel, tw, tx, to, g) != cudaSuccess) return HB200_ERR_CUDA;
  return HB200_OK;
}

template <typename T, bool SPLIT>
int launch_pair_typed(const CUtensorMap& tw, const CUtensorMap& tx, const CUtensorMap& to, const Args& g, int pairs, bool gated,
                      bool out_f32, int dev, cudaStream_t s) {
  if (gated)
    return out_f32 ? launch_pair<T, float, true, SPLIT>(tw, tx, to, g, pairs, dev, s)
                   : launch_pair<T, T, true, SPLIT>(tw, tx, to, g, pairs, dev, s);
  return out_f32 ? launch_pair<T, float, false, SPLIT>(tw, tx, to, g, pairs, dev, s)
                 : launch_pair<T, T, false, SPLIT>(tw, tx, to, g, pairs, dev, s);
}

}  // namespace linear

// Wait budget and sticky status of this translation unit (see hb200_set_wait_budget_cycles, hb200_device_status).
int linear_set_wait_budget(long long cycles) { return sm100::set_wait_budget_cycles(cycles) ? HB200_OK : HB200_ERR_CUDA; }

int linear_device_status(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_status_linear, sizeof(int)) != cudaSuccess) return HB200_ERR_CUDA;
  if (reset && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_device_status_linear, &zero, sizeof(int)) != cudaSuccess) return HB200_ERR_CUDA;
  }
  return v;
}

}  // namespace hb200

extern "C" int hb200_linear(const hb200_linear_args* args, void* stream) {
  using namespace hb200;
  using namespace hb200::linear;
  if (!args) return HB200_ERR_INVALID_ARGUMENT;
  const auto [x, weight, bias, residual, out, m, n, k, ldx, ldw, ldr, ldo, activation, gated, is_bf16, bias_f32, out_f32,
              reserved] = *args;
  if (!x || !weight || !out || m <= 0 || n <= 0 || k <= 0 || ldx < k || ldw < k || ldo < n || (residual && ldr < 0))
    return HB200_ERR_INVALID_ARGUMENT;
  if (activation < kNone || activation > kGeluTanh || reserved != 0) return HB200_ERR_INVALID_ARGUMENT;
  // TMA: 16-byte aligned bases and row pitches
  if (reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(weight) % 16 || (k % 8) != 0 || (ldx % 8) != 0 ||
      (ldw % 8) != 0)
    return HB200_ERR_UNSUPPORTED;
  if (m > 0x3fffff00 || n > 0x3fffff00 || k > 0x3fffff00 || ldx > (int64_t(1) << 38) || ldw > (int64_t(1) << 38))
    return HB200_ERR_UNSUPPORTED;
  const int out_size = out_f32 ? 4 : 2;
  const uintptr_t item = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual);
  if (item % out_size || reinterpret_cast<uintptr_t>(bias) % (bias_f32 ? 4 : 2)) return HB200_ERR_INVALID_ARGUMENT;
  const bool bf16 = is_bf16 != 0, f32 = out_f32 != 0, is_gated = gated != 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HB200_ERR_CUDA;
  const int sms = device_sms(dev);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Args g{};
  g.out = out;
  g.bias = bias;
  g.residual = residual;
  g.ldo = ldo;
  g.ldr = ldr;
  g.m = int(m);
  g.n = int(n);
  g.k = int(k);
  g.activation = activation;
  g.bias_f32 = bias_f32 != 0;
  g.out_vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (ldo * out_size) % 16 == 0;
  g.res_vec = reinterpret_cast<uintptr_t>(residual) % 16 == 0 && (ldr * out_size) % 16 == 0;
  g.num_kb = int((k + 63) / 64);
  const int64_t weight_rows = is_gated ? 2 * n : n;
  CUtensorMap tw, tx, to{};
  const StreamPlan p = plan_stream(m, n, k, is_gated, dev, sms);
  double pair_us = 0;
  // up to 64 rows of x the weight's stream is the work whatever the sizes (6.2 to 6.5 TB/s)
  const PairPlan q = m > 64 ? plan_pair(m, weight_rows, k, dev, sms, &pair_us) : PairPlan{};
  if (m > 64 && pair_us < stream_us(p, double(weight_rows) * double(k) * 2, sms)) {
    if (q.m_tiles * q.n_tiles > 0x7fffffff) return HB200_ERR_UNSUPPORTED;
    if (!make_map(&tw, weight, weight_rows, k, ldw, q.tile_cols / 2, bf16) || !make_map(&tx, x, m, k, ldx, 128, bf16))
      return HB200_ERR_CUDA;
    if ((n * out_size) % 16 != 0) g.out_vec = 0;  // a TMA store's last 16 bytes of a row are written whole
    if (g.out_vec && !make_out_map(&to, out, m, n, ldo, f32, bf16)) return HB200_ERR_CUDA;
    g.m_tiles = int(q.m_tiles);
    g.n_tiles = int(q.n_tiles);
    g.tile_cols = q.tile_cols;
    g.band = kPairBand;
    g.stage_bytes = kHalfBytes + q.tile_cols * 64;
    g.stages = kPairRingBytes / g.stage_bytes < kPairMaxStages ? kPairRingBytes / g.stage_bytes : kPairMaxStages;
    g.split_log = q.split_log;
    const int64_t tiles = q.m_tiles * q.n_tiles;
    if (q.split_log > 0) {
      const int pairs = int(tiles << q.split_log);
      return bf16 ? launch_pair_typed<__nv_bfloat16, true>(tw, tx, to, g, pairs, is_gated, f32, dev, s)
                  : launch_pair_typed<__half, true>(tw, tx, to, g, pairs, is_gated, f32, dev, s);
    }
    const int pairs = int(tiles < sms / 2 ? tiles : sms / 2);
    return bf16 ? launch_pair_typed<__nv_bfloat16, false>(tw, tx, to, g, pairs, is_gated, f32, dev, s)
                : launch_pair_typed<__half, false>(tw, tx, to, g, pairs, is_gated, f32, dev, s);
  }
  if (p.tiles * p.split > 0x7fffffff) return HB200_ERR_UNSUPPORTED;
  if (!make_map(&tw, weight, weight_rows, k, ldw, is_gated ? 64 : 128, bf16)) return HB200_ERR_CUDA;
  if (!make_map(&tx, x, m, k, ldx, p.cols, bf16)) return HB200_ERR_CUDA;
  g.cols = p.cols;
  g.m_chunks = p.m_chunks;
  g.split = p.split;
  g.stages = p.stages;
  g.stage_bytes = p.stage_bytes;
  g.stash_offset = p.stash_offset;
  return bf16 ? launch_stream_typed<__nv_bfloat16>(tw, tx, g, p, is_gated, f32, dev, s)
              : launch_stream_typed<__half>(tw, tx, g, p, is_gated, f32, dev, s);
}
