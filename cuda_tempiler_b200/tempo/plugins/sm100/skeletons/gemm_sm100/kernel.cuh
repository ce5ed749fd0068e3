// gemm_sm100: the sm_100a GEMM skeleton family (fp16 and W8A16).
//
//   D[p, q] = sum_k P[p, k] * Q[q, k]         (both operands K-major, fp32 accumulate)
//
// Non-swapped (prefill):  P = A [M,K] activations, Q = B [N,K] weights, C[p][q] = C[m][n].
// Swapped (decode, "swap-AB"): P = B [N,K] weights fill the 128-row MMA M side, Q = A [M,K]
// activations become the narrow MMA N side (BN = 16..128), C[q][p] = C[m][n].
// This is the op of the reference skeleton (C = A * B^T with B stored [N][K]; reference
// tempo/plugins/sm70/skeletons/gemm_hmma884/kernel.cuh:587-753 and the shipped
// kernels/shipped/gemm_fp16/sm_70/launch.cuh:20-26), re-designed for Blackwell:
//
//   warp 0        TMA producer: 2-D tiles of P and Q (or the raw 8-bit weight) into a
//                 STAGES-deep shared-memory ring, completion as mbarrier transaction bytes
//   warp 1        MMA issuer: allocates TMEM, one thread issues tcgen05.mma (128 x BN x 16)
//                 into a double-buffered fp32 TMEM accumulator, tcgen05.commit frees stages
//   warps 2-5     epilogue: tcgen05.ld accumulator -> fp16 -> swizzled staging -> TMA store
//                 (or direct stores when swapped, or fp32 split-K partials + last-CTA fixup)
//   warps 6-9     (W8A16 only) dequant: raw int8/uint8 weight tile -> fp16 swizzled tile,
//                 (q - z) * s for group-wise asymmetric weights; per-channel scale is
//                 applied in the epilogue.
//
// Persistent: the grid is at most one CTA per SM; CTAs stride over work units
// (tile_p, tile_q, k-split).  Every mbarrier wait is bounded (2 s) and reports through
// g_status instead of hanging the GPU.
#pragma once

#include "sm100_ptx.cuh"

namespace tempo_sm100 {

enum WeightQuant : int { kWFp16 = 0, kWInt8PerChannel = 1, kWUint8Group = 2 };

// Epilogue of the 2-CTA kernels' EPI instantiations: y = act(acc * scale[n] + bias[n]) + res[m][n], in fp32 on
// the accumulator, rounded once to fp16.  Null pointers leave their term out.  Every load is 16
// bytes of 8 columns (N % 8 == 0, 16-byte aligned), made where the accumulator already is: the
// separate pass it replaces reads and writes C once more (4 M N bytes).
enum EpiAct : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

struct EpiArgs {
  const __half* scale = nullptr;  // per output channel (weights expanded without their scale)
  const __half* bias = nullptr;   // [N]
  const __half* res = nullptr;    // [M][N], may be C itself
  long long ldr = 0;              // row stride of res in elements
  int act = kActNone;
};

struct GemmArgs {
  int rows_p, rows_q, K;
  int tiles_p, tiles_q, num_kb, splits, num_units;
  int group_m;          // raster group height (in P tiles) for L2 reuse
  __half* C;
  long long ldc;        // row stride of C in elements
  float* ws;            // split-K partials (splits > 1)
  int* counters;        // per-tile arrival counters (zero between calls)
  const __half* scale;  // per-channel [N] or group-wise [N][K/group]
  const uint8_t* zero;  // group-wise [N][K/group]
  int group_size;       // group-wise quantisation group along K
  int groups_per_row;   // K / group_size
  int weight_rows;      // N (rows of the weight operand)
  int sz_bytes;         // group-wise: scale + zero bytes one stage loads
  // k-split inside a cluster (1-CTA kernel): the cluster_split CTAs of a cluster hold the
  // k-slices of one tile and reduce through distributed shared memory (0: not used)
  int cluster_split;
  // Split tail of the 2-CTA kernel: tiles [sk_tile0, sk_tile0 + sk_tiles) each run as sk_splits
  // k-slices; tiles before sk_tile0 are whole units (sk_splits 0: no tail).
  int sk_tile0;         // first tail tile
  int sk_tiles;         // tail tiles
  int sk_splits;        // k-slices per tail tile
  EpiArgs epi;          // EPI instantiations only
};

__host__ __device__ constexpr int round_up(int x, int a) { return (x + a - 1) / a * a; }

constexpr int kMaxClusterSplitDev = 8;  // largest k-split reduced inside one cluster
__host__ __device__ constexpr int cmin(int a, int b) { return a < b ? a : b; }
__host__ __device__ constexpr int tmem_cols_for(int c) {
  return c <= 32 ? 32 : c <= 64 ? 64 : c <= 128 ? 128 : c <= 256 ? 256 : 512;
}

constexpr int kMaxDynSmem = 232448;  // 227 KB per CTA on sm_100

// SMEMDQ_ (swapped 8-bit weights only): dequantise the weight tile into shared memory (the A
// operand read by tcgen05.mma from smem, 4 dequant warps) instead of into TMEM.
template <int BN_, int WQ_, bool SWAP_, bool SMEMDQ_ = false>
struct SkelCfg {
  static constexpr int BM = 128, BN = BN_, BK = 64, WQ = WQ_;
  static constexpr bool SWAP = SWAP_;
  // Swapped 8-bit weights are dequantised straight into TMEM as the MMA's A operand
  // (tcgen05.mma A-from-TMEM); no fp16 copy of the weight tile ever lands in shared memory.
  static constexpr bool TA = WQ != 0 && SWAP && !SMEMDQ_;
  static constexpr int WROWS = WQ ? (SWAP ? BM : BN) : 0;  // rows of the raw weight tile
  static constexpr int P_BYTES = TA ? 0 : BM * BK * 2;
  // TA stages cover KS = 128 k: one 128-byte (128B-swizzled) raw row per weight row and TMA
  // request, and SUB = 2 sub-blocks of 64 k for the MMA.  Every other path: KS = BK = 64.
  static constexpr int KS = TA ? 128 : BK;
  static constexpr int SUB = KS / BK;
  static constexpr int Q_BYTES = BN * KS * 2;  // SUB swizzled atoms of BN x 64 fp16
  static constexpr int RAW_BYTES = WROWS * KS;
  static constexpr int P_OFF = 0;
  static constexpr int Q_OFF = round_up(P_BYTES, 1024);
  static constexpr int RAW_OFF = Q_OFF + round_up(Q_BYTES, 1024);
  // group-wise: this k-block's scale row (fp16) and zero row (uint8) for the tile's weight rows
  // (up to SUB group rows per stage: a stage spans KS / group_size groups, group_size >= 64)
  static constexpr int SZ_BYTES = WQ == 2 ? WROWS * 3 * SUB : 0;
  static constexpr int S_OFF = RAW_OFF + RAW_BYTES;
  static constexpr int Z_OFF = S_OFF + WROWS * 2 * SUB;
  static constexpr int STAGE_BYTES = RAW_OFF + round_up(RAW_BYTES + SZ_BYTES, 1024);
  static constexpr int EPI_BYTES = SWAP ? 0 : 4 * 2 * 2048;  // per epilogue warp: 2 x [32][32] fp16
  static constexpr int BAR_BYTES = 1024;
  // TA: a deep shared-memory ring for the raw weight + activation tiles (bytes in flight are
  // what an HBM-bound decode needs) and a separate, shallower ring of ASLOTS fp16 A slots of
  // 32 TMEM columns each next to the 2 x BN accumulator columns.  Both counts are even so each
  // of the two dequant warp groups owns every other stage and every other A slot.
  static constexpr int SMEM_STAGES = (kMaxDynSmem - 1024 - EPI_BYTES - BAR_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = TA ? cmin(SMEM_STAGES, 24) & ~1 : cmin(SMEM_STAGES, 12);
  // Independent accumulators per tile: a k-block's four 16-deep UMMAs rotate over NACC
  // accumulators so that narrow tiles (whose UMMAs are short) are not serialised on the
  // latency of accumulating into one TMEM region; the epilogue adds them up.
  static constexpr int NACC = BN <= 32 ? 4 : (BN <= 64 ? 2 : 1);
  static constexpr int ACC_COLS = NACC * BN;  // TMEM columns of one accumulator buffer
  // as many A slots as TMEM leaves, a multiple of 2 x SUB (two dequant groups, SUB per stage)
  static constexpr int ASLOTS = TA ? cmin(16, ((512 - 2 * ACC_COLS) / 32) & ~3) : 1;
  static constexpr int A_TMEM_COL = 2 * ACC_COLS;  // first TMEM column of the A slots (TA)
  static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + EPI_BYTES + BAR_BYTES;
  static constexpr int NUM_WARPS = 6 + (TA ? 8 : (WQ ? 4 : 0));
  static constexpr int THREADS = NUM_WARPS * 32;
  static constexpr int TMEM_COLS = TA ? 512 : tmem_cols_for(2 * ACC_COLS);
  // accumulator columns per tcgen05.ld (16 where NACC x 32 columns would not fit the wide
  // dequant CTAs' register budget)
  static constexpr int CW = (BN < 32 || (TA && NACC > 2)) ? 16 : 32;
  static_assert(BN % 16 == 0 && BN >= 16 && BN <= 256, "UMMA N for M=128 is 16..256 step 16");
  static_assert(SWAP || BN >= 32, "non-swapped epilogue stores 32-column boxes");
  static_assert(STAGES >= 2, "pipeline needs at least two stages");
  static_assert(!TA || 2 * ACC_COLS + 2 * 32 <= 512, "TMEM: accumulators plus two A slots");
  static_assert(2 * ACC_COLS <= 512, "TMEM: two accumulator buffers");
  // barriers: full[STAGES], empty[STAGES], deq[NDEQ] (indexed by stage, or by A slot for TA),
  // tmem full[2], tmem empty[2], done, aempty[ASLOTS]
  static constexpr int NDEQ = STAGES > ASLOTS ? STAGES : ASLOTS;
  // + 3 for the cluster k-split: operand rings idle, partial rows delivered, deliveries done
  static constexpr int NBARS = 2 * STAGES + NDEQ + 5 + ASLOTS + 3;
  static_assert(NBARS <= BAR_BYTES / 8 - 2, "barrier area too small");
  // cluster k-split: an owner's S slots of partial rows in its idle operand ring, rows of C's
  // contiguous dimension ([q][p] swapped, [p][q] otherwise) padded by 4 floats; at most
  // (rows + S) rows in all
  static constexpr int PART_ROW = (SWAP ? BM : BN) + 4;
  static_assert(((SWAP ? BN : BM) + kMaxClusterSplitDev) * PART_ROW * 4 <= STAGES * STAGE_BYTES,
                "operand ring too small for the cluster k-split partial");
  // Bulk exchange: this CTA's whole partial tile at the front of its ring and the owner slots
  // behind it, where the ring holds both (every tile but the widest); else remote stores.
  static constexpr int PART_SRC_BYTES = (SWAP ? BN : BM) * PART_ROW * 4;
  static constexpr bool BULK_SPLIT =
      PART_SRC_BYTES + ((SWAP ? BN : BM) + kMaxClusterSplitDev) * PART_ROW * 4 <=
      STAGES * STAGE_BYTES;
};

__device__ __forceinline__ void decode_unit(const GemmArgs& a, int unit, int& tile, int& tp,
                                            int& tq, int& split, int& kb0, int& kb1) {
  tile = unit / a.splits;
  split = unit - tile * a.splits;
  const int gsz = a.group_m * a.tiles_q;
  const int g = tile / gsz;
  const int first = g * a.group_m;
  const int gm = min(a.tiles_p - first, a.group_m);
  const int r = tile - g * gsz;
  tp = first + r % gm;
  tq = r / gm;
  kb0 = (int)(((long long)a.num_kb * split) / a.splits);
  kb1 = (int)(((long long)a.num_kb * (split + 1)) / a.splits);
}

__device__ __forceinline__ bool mbar_drain(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer() - t0 > limit_ns) return false;
  }
  return true;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Columns [c*CW, c*CW+CW) of this warp's 32 accumulator rows, summed over the NACC
// independent accumulators (TMEM -> registers, fp32).
template <int CW, int NACC, int BN>
__device__ __forceinline__ void acc_chunk(uint32_t t_acc, int c, float (&f)[32]) {
  uint32_t v[NACC][32];
#pragma unroll
  for (int i = 0; i < NACC; ++i) {
    if (CW == 32) {
      tmem_ld_x32(t_acc + i * BN + c * 32, v[i]);
    } else {
      uint32_t (&v16)[16] = *reinterpret_cast<uint32_t(*)[16]>(v[i]);
      tmem_ld_x16(t_acc + i * BN + c * 16, v16);
    }
  }
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < CW; ++j) {
    float a = __uint_as_float(v[0][j]);
#pragma unroll
    for (int i = 1; i < NACC; ++i) a += __uint_as_float(v[i][j]);
    f[j] = a;
  }
}

// Phi(-|x|), the normal distribution's tail: exp(-x^2 / 2) Q(t) with t = 1 / (1 + 0.3 |x|), the form
// of Hastings' approximations (Abramowitz and Stegun 7.1.26), here with Q of degree 6 fitted for the
// relative error: 2^-18.5 up to |x| = 6 in fp32 with an exact exponential, 2^-17.5 with __expf;
// beyond, x Phi(x) is less than half of fp16's smallest value.  (0.5 x (1 + erff) cancels for x < -3:
// outputs off by up to 3 roundings to fp16.  100 x 15360 x 3840 25.5 us, with erff 25.6, with erfcf
// 27.4; 4096 x 15360 x 3840 398, 382 and 517.)
__device__ __forceinline__ float normal_tail(float x) {
  const float t = __fdividef(1.f, fmaf(0.3f, fabsf(x), 1.f));
  float q = -0.08242921f;
  q = fmaf(q, t, 0.23232886f);
  q = fmaf(q, t, -0.03598287f);
  q = fmaf(q, t, 0.15476678f);
  q = fmaf(q, t, 0.11096748f);
  q = fmaf(q, t, 0.12034819f);
  return q * t * __expf(-0.5f * x * x);
}

// The activation of N values, chosen once for all of them by plain branches (a switch per value
// became an indirect jump each: 140 cycles, 25 us of a 256-row tile's epilogue).  __expf and
// __fdividef: their errors (2^-17 relative at the largest finite exponents, 2^-21 at ordinary
// ones) are far below the rounding to fp16 that follows, 2^-11; where __fdividef gives 0 for a
// quotient below 2^-100, so does that rounding.
template <int N>
__device__ __forceinline__ void epi_act(float (&f)[N], int act) {
  if (act == kActNone) return;
  if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = f[i] > 0.f || f[i] != f[i] ? f[i] : 0.f;  // NaN passes
  } else if (act == kActSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __fdividef(f[i], 1.f + __expf(-f[i]));
  } else if (act == kActGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float q = normal_tail(f[i]);
      f[i] *= f[i] < 0.f ? q : 1.f - q;
    }
  } else {  // kActGeluTanh: 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)): one exponential, one division
#pragma unroll
    for (int i = 0; i < N; ++i)
      f[i] = __fdividef(
          f[i],
          1.f + __expf(-1.5957691216057308f * (f[i] + 0.044715f * f[i] * f[i] * f[i])));
  }
}

__device__ __forceinline__ void unpack_half8(uint4 v, float (&f)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = __half22float2(h[i]);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}

// Columns [n0, n0 + 32) of the residual's row m, for one thread, loaded while an earlier chunk is
// worked on, or before the tile's MMAs are done (4096 x 3840 x 15360 with the loads where the values
// are added: 397 us, so: 378).  Plain loads: C may be the same memory, and this thread reads an
// element before anyone writes it.
struct EpiRes {
  uint4 v[4];
  __device__ __forceinline__ void load(const EpiArgs& e, int m, int m_rows, int n0, int n_cols) {
    if (!e.res || m >= m_rows) return;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (n0 + 8 * g < n_cols)
        v[g] = *reinterpret_cast<const uint4*>(e.res + (long long)m * e.ldr + n0 + 8 * g);
  }
};

// The epilogue of columns [n0, n0 + 32) of row m held by one thread.
__device__ __forceinline__ void epi_row32(const EpiArgs& e, float (&f)[32], const EpiRes& res,
                                          int m, int m_rows, int n0, int n_cols) {
  if (m >= m_rows) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int n = n0 + 8 * g;
    if (n >= n_cols) break;
    float v[8];
    if (e.scale) {
      unpack_half8(__ldg(reinterpret_cast<const uint4*>(e.scale + n)), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[8 * g + i] *= v[i];
    }
    if (e.bias) {
      unpack_half8(__ldg(reinterpret_cast<const uint4*>(e.bias + n)), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[8 * g + i] += v[i];
    }
  }
  epi_act(f, e.act);
  if (!e.res) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if (n0 + 8 * g >= n_cols) break;
    float v[8];
    unpack_half8(res.v[g], v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[8 * g + i] += v[i];
  }
}

template <int BN, int WQ, bool SWAP, bool SMEMDQ = false>
__global__ void __launch_bounds__(SkelCfg<BN, WQ, SWAP, SMEMDQ>::THREADS, 1)
    k_gemm_sm100(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ,
                 const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapC,
                 const __grid_constant__ CUtensorMap mapS, const __grid_constant__ CUtensorMap mapZ,
                 const GemmArgs args) {
  using Cfg = SkelCfg<BN, WQ, SWAP, SMEMDQ>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* epi_smem = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi_smem + Cfg::EPI_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* last_flag = abort_flag + 1;

  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_u32(bars);
  constexpr int kDeq0 = 2 * STAGES, kT0 = kDeq0 + Cfg::NDEQ;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  // deq_bar: dequantised tile of stage s ready, or (TA) A slot s written by 4 quadrant warps
  auto deq_bar = [&](int s) { return bar_base + 8u * (kDeq0 + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (kT0 + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (kT0 + 2 + b); };
  const uint32_t done_bar = bar_base + 8u * (kT0 + 4);
  // TA: aempty_bar(a) = A slot a consumed by the MMAs
  auto aempty_bar = [&](int a) { return bar_base + 8u * (kT0 + 5 + a); };
  // cluster k-split: every CTA's operand ring idle / every CTA's partial rows delivered
  const uint32_t rfree_bar = bar_base + 8u * (kT0 + 5 + Cfg::ASLOTS);
  const uint32_t pready_bar = rfree_bar + 8u;
  const uint32_t rdone_bar = rfree_bar + 16u;
  auto p_addr = [&](int s) { return smem_base + s * Cfg::STAGE_BYTES + Cfg::P_OFF; };
  auto q_addr = [&](int s) { return smem_base + s * Cfg::STAGE_BYTES + Cfg::Q_OFF; };
  auto raw_ptr = [&](int s) { return smem + s * Cfg::STAGE_BYTES + Cfg::RAW_OFF; };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < Cfg::NDEQ; ++s)
      mbar_init(deq_bar(s), Cfg::TA ? 4 : 1);  // TA: 4 quadrant warps; else 1 warp per stage
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 4);
    }
    mbar_init(done_bar, 1);
    for (int a = 0; a < Cfg::ASLOTS; ++a) mbar_init(aempty_bar(a), 1);
    const int csplit = args.cluster_split > 1 ? args.cluster_split : 1;
    mbar_init(rfree_bar, 4 * csplit);  // 4 epilogue warps of each CTA of the cluster
    // bulk exchange: the owner's own expect_tx arrival plus the slots' bytes; remote stores:
    // the 4 epilogue warps of each CTA
    mbar_init(pready_bar, Cfg::BULK_SPLIT ? 1 : 4 * csplit);
    mbar_init(rdone_bar, csplit);  // each owner, once its slots are filled
    *abort_flag = 0;
    *last_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&mapQ);
    if (WQ) tma_prefetch_desc(&mapW);
    if (WQ == kWUint8Group) {
      tma_prefetch_desc(&mapS);
      tma_prefetch_desc(&mapZ);
    }
    if (!WQ || !SWAP) tma_prefetch_desc(&mapP);
    if (!SWAP) tma_prefetch_desc(&mapC);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (args.cluster_split > 1) cluster_sync();  // peers' barriers initialised before arrivals
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Nothing above touches global memory another grid may write: overlap it with that grid.
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      // Weights streamed exactly once (swapped decode) go evict-first; the small activation
      // operand is re-read by every CTA and stays.  Prefill re-reads both: normal policy.
      const uint64_t pol_w = SWAP ? policy_evict_first() : policy_evict_normal();
      const uint64_t pol_a = SWAP ? policy_evict_last() : policy_evict_normal();
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int unit = blockIdx.x; unit < args.num_units; unit += gridDim.x) {
        int tile, tp, tq, split, kb0, kb1;
        decode_unit(args, unit, tile, tp, tq, split, kb0, kb1);
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, 1)) {
            ok = false;
            break;
          }
          const int kx = kb * Cfg::KS;
          if (WQ == kWFp16) {
            mbar_arrive_expect_tx(full_bar(stage), Cfg::P_BYTES + Cfg::Q_BYTES);
            tma_load_2d(p_addr(stage), &mapP, full_bar(stage), kx, tp * Cfg::BM, SWAP ? pol_w : pol_a);
            tma_load_2d(q_addr(stage), &mapQ, full_bar(stage), kx, tq * BN, SWAP ? pol_a : pol_w);
          } else {
            const int wrow0 = SWAP ? tp * Cfg::BM : tq * BN;
            mbar_arrive_expect_tx(full_bar(stage), Cfg::RAW_BYTES + args.sz_bytes +
                                                       (SWAP ? Cfg::Q_BYTES : Cfg::P_BYTES));
            if (SWAP) {
#pragma unroll
              for (int a = 0; a < Cfg::SUB; ++a)
                tma_load_2d(q_addr(stage) + a * BN * 128, &mapQ, full_bar(stage), kx + a * Cfg::BK,
                            tq * BN, pol_a);
            } else
              tma_load_2d(p_addr(stage), &mapP, full_bar(stage), kx, tp * Cfg::BM, pol_a);
            tma_load_2d(smem_u32(raw_ptr(stage)), &mapW, full_bar(stage), kx, wrow0, pol_w);
            if (WQ == kWUint8Group) {
              const int g = kx / args.group_size;
              const uint32_t sbase = smem_base + stage * Cfg::STAGE_BYTES;
              tma_load_2d(sbase + Cfg::S_OFF, &mapS, full_bar(stage), wrow0, g, pol_a);
              tma_load_2d(sbase + Cfg::Z_OFF, &mapZ, full_bar(stage), wrow0, g, pol_a);
            }
          }
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
      }
      // Drain: every load this thread issued must have landed before the CTA can exit
      // (normally already true; matters only after an abort).
      const int pending = issued < STAGES ? issued : STAGES;
      int s = stage;
      uint32_t ph = phase;
      for (int i = 0; i < pending; ++i) {
        if (--s < 0) {
          s = STAGES - 1;
          ph ^= 1u;
        }
        mbar_drain(full_bar(s), ph, 100000000ull);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_f16_f32(Cfg::BM, BN);
      int stage = 0;
      uint32_t phase = 0;
      int lu = 0;
      int it = 0;  // k-block sequence number (A-slot ring position for TA)
      for (int unit = blockIdx.x; unit < args.num_units; unit += gridDim.x, ++lu) {
        int tile, tp, tq, split, kb0, kb1;
        decode_unit(args, unit, tile, tp, tq, split, kb0, kb1);
        const int buf = lu & 1;
        const uint32_t uphase = (lu >> 1) & 1;
        if (!mbar_wait(tempty_bar(buf), uphase ^ 1u, abort_flag, 2)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * Cfg::ACC_COLS;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, 3)) { ok = false; break; }
          if (!Cfg::TA && WQ && !mbar_wait(deq_bar(stage), phase, abort_flag, 4)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t pa = p_addr(stage), qa = q_addr(stage);
          if (Cfg::TA) {
#pragma unroll 1
            for (int j = 0; j < Cfg::SUB; ++j) {
              const int aslot = it % Cfg::ASLOTS;
              const uint32_t aphase = (uint32_t)((it / Cfg::ASLOTS) & 1);
              ++it;
              if (!mbar_wait(deq_bar(aslot), aphase, abort_flag, 4)) { ok = false; break; }
              tc_fence_after();
              const uint32_t a_tmem = tmem_base + Cfg::A_TMEM_COL + aslot * 32;
#pragma unroll
              for (int k = 0; k < Cfg::BK / 16; ++k)
                umma_f16_ts(d_tmem + (k % Cfg::NACC) * BN, a_tmem + k * 8,
                            sdesc_k_sw128(qa + j * BN * 128 + k * 32), idesc,
                            (kb > kb0 || j > 0 || k >= Cfg::NACC) ? 1u : 0u);
              umma_commit(aempty_bar(aslot));
            }
            if (!ok) break;
          } else {
#pragma unroll
            for (int k = 0; k < Cfg::BK / 16; ++k) {
              umma_f16_ss(d_tmem + (k % Cfg::NACC) * BN, sdesc_k_sw128(pa + k * 32),
                          sdesc_k_sw128(qa + k * 32), idesc, (kb > kb0 || k >= Cfg::NACC) ? 1u : 0u);
            }
          }
          umma_commit(empty_bar(stage));
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(tfull_bar(buf));
      }
      // Wait for every MMA this thread issued before TMEM is released.
      umma_commit(done_bar);
      mbar_drain(done_bar, 0, 100000000ull);
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------------ epilogue
    const int quad = warp & 3;  // TMEM lane quadrant this warp may access
    const int row = quad * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    uint8_t* stage_buf = epi_smem + (warp - 2) * 4096;
    int sb = 0;
    int lu = 0;
    for (int unit = blockIdx.x; unit < args.num_units; unit += gridDim.x, ++lu) {
      int tile, tp, tq, split, kb0, kb1;
      decode_unit(args, unit, tile, tp, tq, split, kb0, kb1);
      const int buf = lu & 1;
      const uint32_t uphase = (lu >> 1) & 1;
      if (!mbar_wait(tfull_bar(buf), uphase, abort_flag, 5)) break;
      tc_fence_after();
      const uint32_t t_acc = t_lane + buf * Cfg::ACC_COLS;
      const int p = tp * Cfg::BM + row;
      const int q0 = tq * BN;

      if (args.cluster_split > 1) {
        // k-split inside a cluster: the S CTAs of this cluster hold the S k-slices of one tile
        // (each CTA has exactly this one unit).  The tile's partial rows (rows of C's
        // contiguous dimension) are dealt out to owners, rows [R r / S, R (r + 1) / S) to CTA
        // r.  Once every CTA's mainloop is done (all operand rings idle), each CTA delivers
        // its fp32 rows into slot (its rank) of each owner's ring -- one bulk shared-to-shared
        // copy per owner, or remote stores where the ring cannot hold the whole partial next
        // to the slots -- and each owner sums its rows over the S slots in rank order
        // (deterministic) from its own shared memory and writes C.
        const int S = args.cluster_split;
        const int rk = (int)cluster_ctarank();
        constexpr int PR = Cfg::PART_ROW;                // floats per partial row (+ pad)
        constexpr int R = SWAP ? BN : Cfg::BM;           // partial rows (C rows of the tile)
        const int rpo = (R + S - 1) / S;                 // slot height: most rows one owner has
        const uint32_t ring_s = smem_u32(smem);
        // owner slots: behind the local partial (bulk exchange), or at the front of the ring
        const uint32_t part_s = ring_s + (Cfg::BULK_SPLIT ? Cfg::PART_SRC_BYTES : 0);
        auto lo_of = [&](int o) { return R * o / S; };
        if (Cfg::BULK_SPLIT) {
          // 1. the partial tile, [row][PR], into this CTA's own (idle) ring
          float* src = reinterpret_cast<float*>(smem);
#pragma unroll 1
          for (int c = 0; c < BN / Cfg::CW; ++c) {
            float f[32];
            acc_chunk<Cfg::CW, Cfg::NACC, BN>(t_acc, c, f);
            if (SWAP) {
#pragma unroll
              for (int j = 0; j < Cfg::CW; ++j) src[(c * Cfg::CW + j) * PR + row] = f[j];
            } else {
#pragma unroll
              for (int k = 0; k < Cfg::CW / 4; ++k)
                *reinterpret_cast<float4*>(src + row * PR + c * Cfg::CW + 4 * k) =
                    make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
            }
          }
          tc_fence_before();
          fence_proxy_async_smem();  // the bulk copies read it through the async proxy
          __syncwarp();
          // 2. every ring idle and every partial written: one thread sends each owner its rows
          if (lane == 0) {
            mbar_arrive(tempty_bar(buf));
            for (int j = 0; j < S; ++j) mbar_arrive_cluster(mapa_shared(rfree_bar, j));
          }
          if (!mbar_wait_cluster(rfree_bar, 0, abort_flag, 8)) break;
          if (threadIdx.x == 64) {
            mbar_arrive_expect_tx(pready_bar,
                                  (uint32_t)(S * (lo_of(rk + 1) - lo_of(rk)) * PR * 4));
            for (int o = 0; o < S; ++o) {
              const int rows = lo_of(o + 1) - lo_of(o);
              bulk_copy_to_cluster(mapa_shared(part_s + (uint32_t)(rk * rpo * PR * 4), o),
                                   ring_s + (uint32_t)(lo_of(o) * PR * 4),
                                   (uint32_t)(rows * PR * 4), mapa_shared(pready_bar, o));
            }
          }
          if (!mbar_wait_cluster(pready_bar, 0, abort_flag, 9)) break;
        } else {
          // 1. this CTA's ring is idle: tell every CTA, then wait until every ring is
          tc_fence_before();
          __syncwarp();
          if (lane == 0)
            for (int j = 0; j < S; ++j) mbar_arrive_cluster(mapa_shared(rfree_bar, j));
          if (!mbar_wait_cluster(rfree_bar, 0, abort_flag, 8)) break;
          // 2. push: partial row pr goes to owner o(pr) = the r with lo(r) <= pr < lo(r + 1)
          auto owner = [&](int pr) { return (int)(((pr + 1) * S - 1) / R); };
#pragma unroll 1
          for (int c = 0; c < BN / Cfg::CW; ++c) {
            float f[32];
            acc_chunk<Cfg::CW, Cfg::NACC, BN>(t_acc, c, f);
            if (SWAP) {
              // lane = p (column of C), f[j] = partial row q = c * CW + j
#pragma unroll
              for (int j = 0; j < Cfg::CW; ++j) {
                const int pr = c * Cfg::CW + j;
                const int o = owner(pr);
                const int lr = pr - lo_of(o);
                st_dsmem_f32(
                    mapa_shared(part_s + (uint32_t)(((rk * rpo + lr) * PR + row) * 4), o), f[j]);
              }
            } else {
              // lane = p (row of C), f = columns c * CW ... of that row
              const int o = owner(row);
              const int lr = row - lo_of(o);
              const uint32_t dst = mapa_shared(
                  part_s + (uint32_t)(((rk * rpo + lr) * PR + c * Cfg::CW) * 4), o);
#pragma unroll
              for (int k = 0; k < Cfg::CW / 4; ++k)
                st_dsmem_f4(dst + 16 * k, make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2],
                                                      f[4 * k + 3]));
            }
          }
          tc_fence_before();
          fence_acq_rel_cluster();  // this thread's remote stores before the warp's arrival
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(tempty_bar(buf));
            for (int j = 0; j < S; ++j) mbar_arrive_cluster(mapa_shared(pready_bar, j));
          }
          if (!mbar_wait_cluster(pready_bar, 0, abort_flag, 9)) break;
        }
        // 3. owner: rows [lo, hi) of the tile, 4 columns per step, slots summed in rank order
        const int lo = R * rk / S, hi = R * (rk + 1) / S;
        constexpr int G = (SWAP ? Cfg::BM : BN) / 4;  // float4 groups per partial row
        const float* part =
            reinterpret_cast<const float*>(smem + (Cfg::BULK_SPLIT ? Cfg::PART_SRC_BYTES : 0));
        const int m_rows = SWAP ? args.rows_q : args.rows_p;
        const int n_cols = SWAP ? args.rows_p : args.rows_q;
#pragma unroll 1
        for (int i = threadIdx.x - 64; i < (hi - lo) * G; i += 128) {
          const int lr = i / G, pc = (i - lr * G) * 4;
          // all S slots' loads issued before the first add (S <= kMaxClusterSplitDev); the
          // sum runs in rank order from zero, as before
          float4 v[kMaxClusterSplitDev];
#pragma unroll
          for (int j = 0; j < kMaxClusterSplitDev; ++j)
            if (j < S) v[j] = *reinterpret_cast<const float4*>(part + (j * rpo + lr) * PR + pc);
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int j = 0; j < kMaxClusterSplitDev; ++j) {
            if (j < S) {
              acc.x += v[j].x;
              acc.y += v[j].y;
              acc.z += v[j].z;
              acc.w += v[j].w;
            }
          }
          // C row m, first of 4 C columns n: swapped [q][p] -> (q0 + pr, p0 + pc)
          const int pr = lo + lr;
          const int m = SWAP ? q0 + pr : tp * Cfg::BM + pr;
          const int n = SWAP ? tp * Cfg::BM + pc : q0 + pc;
          if (m < m_rows && n < n_cols) {
            if (WQ == kWInt8PerChannel) {
              acc.x *= __half2float(__ldg(args.scale + n));
              acc.y *= __half2float(__ldg(args.scale + n + 1));
              acc.z *= __half2float(__ldg(args.scale + n + 2));
              acc.w *= __half2float(__ldg(args.scale + n + 3));
            }
            uint2 w;
            w.x = pack_half2(acc.x, acc.y);
            w.y = pack_half2(acc.z, acc.w);
            *reinterpret_cast<uint2*>(args.C + (long long)m * args.ldc + n) = w;
          }
        }
        if (Cfg::BULK_SPLIT && threadIdx.x == 64) {
          // this CTA's slots are filled; it leaves only when every owner has filled its slots
          // (so no copy still reads this CTA's partial)
          for (int j = 0; j < S; ++j) mbar_arrive_cluster(mapa_shared(rdone_bar, j));
          if (!mbar_wait_cluster(rdone_bar, 0, abort_flag, 10)) break;
        }
        continue;
      }

      if (args.splits == 1 && !SWAP) {
        // fp16 tile through swizzled staging and TMA stores, 32 columns per box.
        // chunks that hold at least one in-range column; boxes wholly below M are skipped
        const int live_cols = args.rows_q - q0;
        const int nchunk = live_cols >= BN ? BN / 32 : (live_cols + 31) / 32;
        const bool rows_live = tp * Cfg::BM + quad * 32 < args.rows_p;
#pragma unroll 1
        for (int c = 0; c < nchunk; ++c) {
          float f[32];
          acc_chunk<32, Cfg::NACC, BN>(t_acc, c, f);
          if (c == nchunk - 1) {
            // accumulator fully read: hand the TMEM buffer back to the MMA warp early
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(buf));
          }
          if (!rows_live) continue;
          if (WQ == kWInt8PerChannel) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const int q = q0 + c * 32 + j;
              f[j] *= __half2float(q < args.weight_rows ? __ldg(args.scale + q) : __half(0.f));
            }
          }
          if (lane == 0) bulk_wait_group_read<1>();
          __syncwarp();
          uint8_t* sbuf = stage_buf + sb * 2048;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint4 w;
            w.x = pack_half2(f[8 * g + 0], f[8 * g + 1]);
            w.y = pack_half2(f[8 * g + 2], f[8 * g + 3]);
            w.z = pack_half2(f[8 * g + 4], f[8 * g + 5]);
            w.w = pack_half2(f[8 * g + 6], f[8 * g + 7]);
            const int pg = g ^ ((lane >> 1) & 3);  // 64-byte swizzle
            *reinterpret_cast<uint4*>(sbuf + lane * 64 + pg * 16) = w;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&mapC, smem_u32(sbuf), q0 + c * 32, tp * Cfg::BM + quad * 32);
            bulk_commit_group();
          }
          sb ^= 1;
        }
      } else if (args.splits == 1) {
        // swapped: C[q][p]; lanes run along p (= n), so each column store is coalesced.
        const float sc =
            (WQ == kWInt8PerChannel && p < args.rows_p) ? __half2float(__ldg(args.scale + p)) : 1.f;
#pragma unroll 1
        for (int c = 0; c < BN / Cfg::CW; ++c) {
          float f[32];
          acc_chunk<Cfg::CW, Cfg::NACC, BN>(t_acc, c, f);
          if (c == BN / Cfg::CW - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(buf));
          }
          if (p < args.rows_p) {
#pragma unroll
            for (int j = 0; j < Cfg::CW; ++j) {
              const int q = q0 + c * Cfg::CW + j;
              if (q < args.rows_q)
                args.C[(long long)q * args.ldc + p] = __float2half_rn(f[j] * sc);
            }
          }
        }
      } else {
        // split-K: fp32 partial slice, [column][row] so the warp's stores are coalesced.
        float* part = args.ws + ((long long)tile * args.splits + split) * (Cfg::BM * BN);
#pragma unroll 1
        for (int c = 0; c < BN / Cfg::CW; ++c) {
          float f[32];
          acc_chunk<Cfg::CW, Cfg::NACC, BN>(t_acc, c, f);
#pragma unroll
          for (int j = 0; j < Cfg::CW; ++j)
            __stcg(part + (c * Cfg::CW + j) * Cfg::BM + row, f[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(buf));
        __threadfence();
        named_barrier_sync(1, 128);
        if (threadIdx.x == 64) {
          const int old = atomicAdd(args.counters + tile, 1);
          const int last = (old == args.splits - 1);
          if (last) atomicExch(args.counters + tile, 0);  // ready for the next call
          *last_flag = last;
        }
        named_barrier_sync(1, 128);
        if (*last_flag) {
          __threadfence();
          // Sum the k-slices in split order (deterministic), 32 columns at a time with all 32
          // loads of a slice independent, so each slice costs one L2 round trip per chunk.
          const float* base = args.ws + (long long)tile * args.splits * (Cfg::BM * BN);
          const float sc_row = (SWAP && WQ == kWInt8PerChannel && p < args.rows_p)
                                   ? __half2float(__ldg(args.scale + p)) : 1.f;
#pragma unroll 1
          for (int c0 = 0; c0 < BN; c0 += Cfg::CW) {
            if (q0 + c0 >= args.rows_q || p >= args.rows_p) break;
            float acc[Cfg::CW];
#pragma unroll
            for (int i = 0; i < Cfg::CW; ++i) acc[i] = 0.f;
            const float* col = base + c0 * Cfg::BM + row;
            int s = 0;
#pragma unroll 1
            for (; s + 2 <= args.splits; s += 2) {
              float x[Cfg::CW], y[Cfg::CW];
#pragma unroll
              for (int i = 0; i < Cfg::CW; ++i) {
                x[i] = __ldcg(col + (long long)s * (Cfg::BM * BN) + i * Cfg::BM);
                y[i] = __ldcg(col + (long long)(s + 1) * (Cfg::BM * BN) + i * Cfg::BM);
              }
#pragma unroll
              for (int i = 0; i < Cfg::CW; ++i) acc[i] = (acc[i] + x[i]) + y[i];
            }
            if (s < args.splits) {
#pragma unroll
              for (int i = 0; i < Cfg::CW; ++i)
                acc[i] += __ldcg(col + (long long)s * (Cfg::BM * BN) + i * Cfg::BM);
            }
            if (SWAP) {
#pragma unroll
              for (int i = 0; i < Cfg::CW; ++i) {
                const int q = q0 + c0 + i;
                if (q < args.rows_q)
                  args.C[(long long)q * args.ldc + p] = __float2half_rn(acc[i] * sc_row);
              }
            } else {
#pragma unroll
              for (int i0 = 0; i0 < Cfg::CW; i0 += 8) {
                const int q = q0 + c0 + i0;
                if (q >= args.rows_q) break;
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  o[i] = acc[i0 + i] *
                         (WQ == kWInt8PerChannel ? __half2float(__ldg(args.scale + q + i)) : 1.f);
                uint4 w;
                w.x = pack_half2(o[0], o[1]);
                w.y = pack_half2(o[2], o[3]);
                w.z = pack_half2(o[4], o[5]);
                w.w = pack_half2(o[6], o[7]);
                *reinterpret_cast<uint4*>(args.C + (long long)p * args.ldc + q) = w;
              }
            }
          }
        }
      }
    }
    if (!SWAP && lane == 0) bulk_wait_group<0>();
  } else {
    // ------------------------------------------------------------------ dequant (W8A16)
    // Dequant warp d owns the stages s with s % 4 == d, so up to four stages are converted
    // concurrently.  Lane l always handles 16-byte chunk (l & 3) of rows
    // (l >> 2) + 8 j, so its swizzled destination granules are fixed.
    if (Cfg::TA) {
      // Two groups of four warps alternate stages; within a group warp (w & 3) converts the
      // 32 weight rows of its TMEM lane quadrant, one row per thread: per 64-k sub-block, 64 raw
      // bytes -> 32 packed fp16 pairs -> tcgen05.st into one A slot (32 TMEM columns).
      const int grp = (warp - 6) >> 2;
      const int quad = warp & 3;
      const int r = quad * 32 + lane;
      const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + Cfg::A_TMEM_COL;
      const int sw = r & 7;  // 128-byte swizzle: 16-byte granule g of row r lives at g ^ (r & 7)
      int sit = 0;           // stage-iteration sequence number
      for (int unit = blockIdx.x; unit < args.num_units; unit += gridDim.x) {
        int tile, tp, tq, split, kb0, kb1;
        decode_unit(args, unit, tile, tp, tq, split, kb0, kb1);
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb, ++sit) {
          // a stage always has the same owner, so no owner ever skips one of its phases
          const int stage = sit % STAGES;
          if ((stage & 1) != grp) continue;
          const uint32_t phase = (uint32_t)((sit / STAGES) & 1);
          if (!mbar_wait(full_bar(stage), phase, abort_flag, 6)) { ok = false; break; }
          const uint8_t* sb = smem + stage * Cfg::STAGE_BYTES;
          const uint8_t* raw = sb + Cfg::RAW_OFF + r * Cfg::KS;
#pragma unroll 1
          for (int j = 0; j < Cfg::SUB; ++j) {
            const int it = sit * Cfg::SUB + j;
            const int aslot = it % Cfg::ASLOTS;
            const uint32_t aphase = (uint32_t)((it / Cfg::ASLOTS) & 1);
            if (!mbar_wait(aempty_bar(aslot), aphase ^ 1u, abort_flag, 7)) { ok = false; break; }
            tc_fence_after();
            uint4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              x[u] = *reinterpret_cast<const uint4*>(raw + (((j * 4 + u) ^ sw) * 16));
            __half2 h[32];
            if (WQ == kWInt8PerChannel) {
              const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152.0
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                u8x4_to_h2x2_biased(x[u].x ^ 0x80808080u, h[8 * u + 0], h[8 * u + 1]);
                u8x4_to_h2x2_biased(x[u].y ^ 0x80808080u, h[8 * u + 2], h[8 * u + 3]);
                u8x4_to_h2x2_biased(x[u].z ^ 0x80808080u, h[8 * u + 4], h[8 * u + 5]);
                u8x4_to_h2x2_biased(x[u].w ^ 0x80808080u, h[8 * u + 6], h[8 * u + 7]);
              }
#pragma unroll
              for (int i = 0; i < 32; ++i) h[i] = __hsub2(h[i], bias);
            } else {
              // this sub-block's group row inside the stage's scale/zero rows
              const int gl = (j * Cfg::BK) / args.group_size;
              const __half2 zb = __half2half2(__ushort_as_half(
                  (unsigned short)(0x6400u | sb[Cfg::Z_OFF + gl * Cfg::WROWS + r])));
              const __half2 s2 = __half2half2(
                  reinterpret_cast<const __half*>(sb + Cfg::S_OFF)[gl * Cfg::WROWS + r]);
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                u8x4_to_h2x2_biased(x[u].x, h[8 * u + 0], h[8 * u + 1]);
                u8x4_to_h2x2_biased(x[u].y, h[8 * u + 2], h[8 * u + 3]);
                u8x4_to_h2x2_biased(x[u].z, h[8 * u + 4], h[8 * u + 5]);
                u8x4_to_h2x2_biased(x[u].w, h[8 * u + 6], h[8 * u + 7]);
              }
#pragma unroll
              for (int i = 0; i < 32; ++i) h[i] = __hmul2(__hsub2(h[i], zb), s2);
            }
            tmem_st_x32(t_row + aslot * 32, *reinterpret_cast<const uint32_t(*)[32]>(h));
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(deq_bar(aslot));
          }
          if (!ok) break;
        }
        if (!ok) break;
      }
    } else if (WQ) {
      const int dw = warp - 6;
      const int kc = lane & 3;
      const int r0 = lane >> 2;
      const int g0 = ((2 * kc) ^ (r0 & 7)) * 16;
      const int g1 = ((2 * kc + 1) ^ (r0 & 7)) * 16;
      constexpr int ROWS_PER_PASS = 8;
      constexpr int PASSES = Cfg::WROWS / ROWS_PER_PASS;
      int it = 0;
      for (int unit = blockIdx.x; unit < args.num_units; unit += gridDim.x) {
        int tile, tp, tq, split, kb0, kb1;
        decode_unit(args, unit, tile, tp, tq, split, kb0, kb1);
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          // a stage always has the same owner, so no owner ever skips one of its phases
          const int stage = it % STAGES;
          if ((stage & 3) != dw) continue;
          const uint32_t phase = (uint32_t)((it / STAGES) & 1);
          if (!mbar_wait(full_bar(stage), phase, abort_flag, 6)) { ok = false; break; }
          uint8_t* sb = smem + stage * Cfg::STAGE_BYTES;
          const uint8_t* raw = sb + Cfg::RAW_OFF;
          uint8_t* dst = sb + (SWAP ? Cfg::P_OFF : Cfg::Q_OFF);
          const __half* srow = reinterpret_cast<const __half*>(sb + Cfg::S_OFF);
          const uint8_t* zrow = sb + Cfg::Z_OFF;
#pragma unroll
          for (int j0 = 0; j0 < PASSES; j0 += 4) {
            uint4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              x[u] = *reinterpret_cast<const uint4*>(raw + (r0 + ROWS_PER_PASS * (j0 + u)) * 64 + kc * 16);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int r = r0 + ROWS_PER_PASS * (j0 + u);
              __half2 h[8];
              if (WQ == kWInt8PerChannel) {
                // signed byte b -> (b ^ 0x80) = b + 128; 1024 + (b + 128) - 1152 = b, exact
                const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152.0
                u8x4_to_h2x2_biased(x[u].x ^ 0x80808080u, h[0], h[1]);
                u8x4_to_h2x2_biased(x[u].y ^ 0x80808080u, h[2], h[3]);
                u8x4_to_h2x2_biased(x[u].z ^ 0x80808080u, h[4], h[5]);
                u8x4_to_h2x2_biased(x[u].w ^ 0x80808080u, h[6], h[7]);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = __hsub2(h[i], bias);
              } else {
                // (1024 + q) - (1024 + z) = q - z exactly; one rounding in the scale product.
                // Rows past N were filled with zeros by TMA, so s = 0 and the weight is 0.
                const __half2 zb = __half2half2(__ushort_as_half((unsigned short)(0x6400u | zrow[r])));
                const __half2 s2 = __half2half2(srow[r]);
                u8x4_to_h2x2_biased(x[u].x, h[0], h[1]);
                u8x4_to_h2x2_biased(x[u].y, h[2], h[3]);
                u8x4_to_h2x2_biased(x[u].z, h[4], h[5]);
                u8x4_to_h2x2_biased(x[u].w, h[6], h[7]);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = __hmul2(__hsub2(h[i], zb), s2);
              }
              const uint4* hv = reinterpret_cast<const uint4*>(h);
              uint8_t* drow = dst + r * 128;
              *reinterpret_cast<uint4*>(drow + g0) = hv[0];
              *reinterpret_cast<uint4*>(drow + g1) = hv[1];
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(deq_bar(stage));
        }
        if (!ok) break;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace tempo_sm100

namespace tempo_sm100 {

// ---------------------------------------------------------------------------------------------
// k_gemv_sm100: the decode-sized (M <= 16) streaming GEMV, C[m][n] = sum_k A[m][k] * W[n][k].
//
// At M <= 16 a 128 x N x 16 UMMA costs about as much as a wide one, so the tensor-core path is
// instruction-bound there; this kernel instead streams each weight row once with 16-byte
// read-only loads (kept out of L1), dequantises in registers and multiplies on the CUDA cores.
//
// Work split: CTA b (kGemvThreads threads) owns the R weight rows [b R, b R + R) and its threads
// split K: thread t reads 16-byte chunks t, t + T, ... of each of the R rows, U chunks of every
// row in flight before any of them is used.  Many small CTAs (N / R of them, thousands at the
// BASELINE shapes) let the block scheduler even out the bytes each SM streams, where one warp
// per row group left a ragged last wave (e.g. 240 CTAs of 16 rows on 148 SMs).  Products of
// one chunk are summed in packed fp16 (4 or 8 terms per half), then added to fp32
// accumulators; a warp shuffle and a fixed-order sum over the CTA's warps in shared memory
// finish each (m, row), so results do not depend on scheduling.
// ---------------------------------------------------------------------------------------------
constexpr int kGemvThreads = 128;

template <int WQ>
__device__ __forceinline__ void gemv_weights(uint4 x, __half2 (&w)[8], __half2 zb, __half2 s2) {
  if (WQ == kWInt8PerChannel) {
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152.0
    u8x4_to_h2x2_biased(x.x ^ 0x80808080u, w[0], w[1]);
    u8x4_to_h2x2_biased(x.y ^ 0x80808080u, w[2], w[3]);
    u8x4_to_h2x2_biased(x.z ^ 0x80808080u, w[4], w[5]);
    u8x4_to_h2x2_biased(x.w ^ 0x80808080u, w[6], w[7]);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __hsub2(w[i], bias);
  } else {
    u8x4_to_h2x2_biased(x.x, w[0], w[1]);
    u8x4_to_h2x2_biased(x.y, w[2], w[3]);
    u8x4_to_h2x2_biased(x.z, w[4], w[5]);
    u8x4_to_h2x2_biased(x.w, w[6], w[7]);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __hmul2(__hsub2(w[i], zb), s2);
  }
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// k_expand_w8: the 8-bit weights of a W8A16 problem expanded to fp16 (W = q * s, or
// (q - z) * s group-wise), 16 k per thread: 16 bytes in, 32 bytes out, streamed once.  For
// prefill-sized M the tensor-core kernel then runs on fp16 weights at the full 2-CTA rate;
// the pass costs 3 bytes per weight of HBM traffic, small against the GEMM at such M.
// ldsz: row stride of the group-wise scale / zero arrays [K/g][ldsz].  wait = 0 skips the
// programmatic-launch wait: the launch that expands a later slice of the weights reads only the
// weights, never the preceding GEMM's output, so it may run beside that GEMM.
template <int WQ>
__global__ void __launch_bounds__(256)
    k_expand_w8(const uint8_t* __restrict__ W, const __half* __restrict__ scale,
                const uint8_t* __restrict__ zero, __half* __restrict__ out, int N, int K,
                long long ldw, int group, int ldsz, int wait) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int per_row = K / 16;
  if (i >= (long long)N * per_row) return;
  if (wait) pdl_wait();
  pdl_launch_dependents();
  const int n = (int)(i / per_row);
  const int k0 = (int)(i - (long long)n * per_row) * 16;
  const uint4 x = ld_stream(W + (long long)n * ldw + k0);
  __half2 zb = __float2half2_rn(0.f), s2 = zb;
  if (WQ == kWUint8Group) {
    const long long gi = (long long)(k0 / group) * ldsz + n;
    zb = __half2half2(__ushort_as_half((unsigned short)(0x6400u | __ldg(zero + gi))));
    s2 = __half2half2(__ldg(scale + gi));
  }
  __half2 w[8];
  gemv_weights<WQ>(x, w, zb, s2);
  if (WQ == kWInt8PerChannel) {
    const __half2 sc = __half2half2(__ldg(scale + n));
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __hmul2(w[j], sc);
  }
  uint4* o = reinterpret_cast<uint4*>(out + (long long)n * K + k0);
  o[0] = *reinterpret_cast<const uint4*>(&w[0]);
  o[1] = *reinterpret_cast<const uint4*>(&w[4]);
}

template <int WQ, int MM, int R>
__global__ void __launch_bounds__(kGemvThreads)
    k_gemv_sm100(const __half* __restrict__ A, const uint8_t* __restrict__ W,
                 const __half* __restrict__ scale, const uint8_t* __restrict__ zero,
                 __half* __restrict__ C, int M, int N, int K, long long lda, long long ldw,
                 long long ldc, int group) {
  constexpr int T = kGemvThreads;
  constexpr int NWARP = T / 32;
  constexpr int ESZ = WQ ? 1 : 2;       // weight bytes per element
  constexpr int KC = 16 / ESZ;          // k per 16-byte chunk
  constexpr int NW = KC / 2;            // packed fp16 pairs per chunk
  // chunks of each row in flight per thread: 8 / R, halved where 4+ activation rows hold the
  // registers (keeps every instantiation free of spills)
  constexpr int UC = MM >= 4 ? 4 : 8;
  constexpr int U = R >= UC ? 1 : UC / R;
  __shared__ float red[NWARP][MM * R];
  const int tid = threadIdx.x;
  const int lane = tid & 31;
  const int warp = tid >> 5;
  const int n0 = blockIdx.x * R;
  pdl_wait();
  pdl_launch_dependents();
  const int nchunks = K / KC;           // K % KC == 0 (checked by applicability)
  const uint8_t* wrow[R];
#pragma unroll
  for (int r = 0; r < R; ++r) wrow[r] = W + (long long)min(n0 + r, N - 1) * ldw * ESZ;
  float acc[MM][R];
#pragma unroll
  for (int m = 0; m < MM; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[m][r] = 0.f;
  const int G = WQ == kWUint8Group ? group : 1;

  // one chunk (c) of the R rows, already loaded: dequantise, multiply, accumulate
  auto use_chunk = [&](int c, const uint4 (&x)[R]) {
    const int k0 = c * KC;
    __half2 w[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (WQ == kWFp16) {
        w[r][0] = *reinterpret_cast<const __half2*>(&x[r].x);
        w[r][1] = *reinterpret_cast<const __half2*>(&x[r].y);
        w[r][2] = *reinterpret_cast<const __half2*>(&x[r].z);
        w[r][3] = *reinterpret_cast<const __half2*>(&x[r].w);
      } else {
        __half2 zb = __float2half2_rn(0.f), s2 = zb;
        if (WQ == kWUint8Group) {
          // (measured: fetching these with the weight chunks instead costs this kernel 3-5 %
          // at the M <= 2 it serves -- more registers, fewer resident CTAs)
          const int n = min(n0 + r, N - 1);
          const long long gi = (long long)(k0 / G) * N + n;
          zb = __half2half2(__ushort_as_half((unsigned short)(0x6400u | __ldg(zero + gi))));
          s2 = __half2half2(__ldg(scale + gi));
        }
        gemv_weights<WQ>(x[r], w[r], zb, s2);
      }
    }
    // one activation row at a time (its chunk is reused by the R weight rows), so the
    // register footprint does not grow with MM
#pragma unroll
    for (int m = 0; m < MM; ++m) {
      if (MM > 4 && m >= M) break;
      __half2 a[NW];
      if (MM <= 4 && m >= M) {
#pragma unroll
        for (int q = 0; q < NW; ++q) a[q] = __float2half2_rn(0.f);
      } else {
        const uint4* ap = reinterpret_cast<const uint4*>(A + (long long)m * lda + k0);
#pragma unroll
        for (int q = 0; q < KC / 8; ++q) {
          const uint4 v = __ldg(ap + q);
          a[4 * q + 0] = *reinterpret_cast<const __half2*>(&v.x);
          a[4 * q + 1] = *reinterpret_cast<const __half2*>(&v.y);
          a[4 * q + 2] = *reinterpret_cast<const __half2*>(&v.z);
          a[4 * q + 3] = *reinterpret_cast<const __half2*>(&v.w);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        __half2 p = __hmul2(w[r][0], a[0]);
#pragma unroll
        for (int q = 1; q < NW; ++q) p = __hfma2(w[r][q], a[q], p);
        const float2 f = __half22float2(p);
        acc[m][r] += f.x + f.y;
      }
    }
  };

  int c = tid;
  // U chunks of every row issued before the first is used: U * R * 16 bytes in flight
  for (; c + (U - 1) * T < nchunks; c += U * T) {
    uint4 x[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) x[u][r] = ld_stream(wrow[r] + (long long)(c + u * T) * 16);
#pragma unroll
    for (int u = 0; u < U; ++u) use_chunk(c + u * T, x[u]);
  }
  for (; c < nchunks; c += T) {
    uint4 x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = ld_stream(wrow[r] + (long long)c * 16);
    use_chunk(c, x);
  }

#pragma unroll
  for (int m = 0; m < MM; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v = acc[m][r];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) red[warp][m * R + r] = v;
    }
  __syncthreads();
  for (int i = tid; i < MM * R; i += T) {
    const int m = i / R;
    const int n = n0 + (i - m * R);
    if (m >= M || n >= N) continue;
    float v = red[0][i];
#pragma unroll
    for (int w = 1; w < NWARP; ++w) v += red[w][i];
    const float sc = WQ == kWInt8PerChannel ? __half2float(__ldg(scale + n)) : 1.f;
    C[(long long)m * ldc + n] = __float2half_rn(v * sc);
  }
}


// ---------------------------------------------------------------------------------------------
// k_gemv_mma_sm100: the decode GEMV for 5..16 activation rows, with the products on the warp
// tensor-core instruction (mma.sync m16n8k16, fp16 inputs, fp32 accumulate) instead of packed
// fp16 FMAs.  The op is HBM-bound at these M; what limits the CUDA-core kernel above is
// instruction issue (8 FMA instructions per activation row per 16 weights), which one MMA per
// 16 x 8 x 16 block removes.  Operands go straight from registers (the weight chunks streamed
// from HBM and dequantised in registers, the activation chunks from L1) -- no shared-memory
// staging, so the 5th-generation tcgen05 path (which needs operands in shared memory / TMEM and
// a single-thread issue chain per CTA) buys nothing here.
//
// Work split: a CTA (4 warps) owns 16 weight rows and one of `splits` k-slices; the k-slices of
// a row group run in one cluster (splits CTAs) and reduce through distributed shared memory.
// Lane (g, t) = (lane / 4, lane % 4) of warp w streams 16-byte chunk c = c0 + 16 i + 4 w + t of
// weight rows g and g + 8; every lane with the same t holds the same k range, so mapping the
// chunk's k values onto MMA k slots (slot 2t <-> k 4j, 2t+1 <-> 4j+1, 2t+8 <-> 4j+2, 2t+9 <->
// 4j+3 of chunk j-th quarter) is the same permutation for the weight (A) and activation (B)
// fragments, and the dot products are unchanged.  The CTA's four warps sum in shared memory,
// the cluster's CTAs into rank 0, each in a fixed order (deterministic).
// ---------------------------------------------------------------------------------------------
constexpr int kGemvMmaMaxSplit = 8;

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int WQ, int MG>  // MG: groups of 8 activation rows (1: M <= 8, 2: M <= 16)
__global__ void __launch_bounds__(kGemvThreads)
    k_gemv_mma_sm100(const __half* __restrict__ A, const uint8_t* __restrict__ W,
                     const __half* __restrict__ scale, const uint8_t* __restrict__ zero,
                     __half* __restrict__ C, int M, int N, int K, long long lda, long long ldw,
                     long long ldc, int group, int splits) {
  constexpr int NWARP = kGemvThreads / 32;
  constexpr int ESZ = WQ ? 1 : 2;   // weight bytes per element
  constexpr int KC = 16 / ESZ;      // k per 16-byte chunk
  constexpr int NMMA = KC / 4;      // MMAs per chunk (4 k of each lane per MMA)
  constexpr int U = MG == 1 ? 4 : 3; // chunk steps in flight per lane (fewer where 16 rows
                                    // of activations hold registers: no spills)
  constexpr int TILE = 16 * 16;     // [16 weight rows][16 activation rows] fp32
  __shared__ float red[NWARP][TILE];
  __shared__ float slots[kGemvMmaMaxSplit][TILE];
  const int tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rgroup = blockIdx.x / splits;
  const int rank = blockIdx.x - rgroup * splits;  // == rank in the cluster (cluster dims splits)
  const int n0 = rgroup * 16;
  pdl_wait();
  pdl_launch_dependents();
  const int ra = min(n0 + g, N - 1), rb = min(n0 + g + 8, N - 1);
  const uint8_t* wa = W + (long long)ra * ldw * ESZ;
  const uint8_t* wb = W + (long long)rb * ldw * ESZ;
  const int nch = K / KC;
  const int c0 = (int)((long long)nch * rank / splits);
  const int c1 = (int)((long long)nch * (rank + 1) / splits);
  const int steps = (c1 - c0 + 15) / 16;  // warp-uniform: every lane runs every step
  const int G = WQ == kWUint8Group ? group : 1;
  float acc[MG][4];
#pragma unroll
  for (int i = 0; i < MG; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

  // group-wise scale and zero-point bytes of rows ra / rb for chunk c, fetched together with
  // the weight chunk so that their latency overlaps the HBM stream
  struct GroupQ {
    unsigned short sa, sb;
    uint8_t za, zb;
  };
  auto load_q = [&](int c, GroupQ& q) {
    if (WQ == kWUint8Group) {
      const long long gi = (long long)((c * KC) / G) * N;
      q.sa = __ldg(reinterpret_cast<const unsigned short*>(scale) + gi + ra);
      q.sb = __ldg(reinterpret_cast<const unsigned short*>(scale) + gi + rb);
      q.za = __ldg(zero + gi + ra);
      q.zb = __ldg(zero + gi + rb);
    }
  };

  auto use_chunk = [&](int c, bool valid, uint4 xa, uint4 xb, const GroupQ& q) {
    const int k0 = c * KC;
    __half2 ha[8], hb[8];
    if (WQ == kWFp16) {
      ha[0] = *reinterpret_cast<const __half2*>(&xa.x);
      ha[1] = *reinterpret_cast<const __half2*>(&xa.y);
      ha[2] = *reinterpret_cast<const __half2*>(&xa.z);
      ha[3] = *reinterpret_cast<const __half2*>(&xa.w);
      hb[0] = *reinterpret_cast<const __half2*>(&xb.x);
      hb[1] = *reinterpret_cast<const __half2*>(&xb.y);
      hb[2] = *reinterpret_cast<const __half2*>(&xb.z);
      hb[3] = *reinterpret_cast<const __half2*>(&xb.w);
    } else {
      __half2 za = __float2half2_rn(0.f), sa = za, zb2 = za, sb = za;
      if (WQ == kWUint8Group) {
        za = __half2half2(__ushort_as_half((unsigned short)(0x6400u | q.za)));
        sa = __half2half2(__ushort_as_half(q.sa));
        zb2 = __half2half2(__ushort_as_half((unsigned short)(0x6400u | q.zb)));
        sb = __half2half2(__ushort_as_half(q.sb));
      }
      gemv_weights<WQ>(xa, ha, za, sa);
      gemv_weights<WQ>(xb, hb, zb2, sb);
    }
#pragma unroll
    for (int mg = 0; mg < MG; ++mg) {
      const int m = mg * 8 + g;
      uint32_t bf[KC / 2];  // activation pairs of row m over the chunk's k range
      if (valid && m < M) {
        const uint4* ap = reinterpret_cast<const uint4*>(A + (long long)m * lda + k0);
#pragma unroll
        for (int q = 0; q < KC / 8; ++q) {
          const uint4 v = __ldg(ap + q);
          bf[4 * q + 0] = v.x;
          bf[4 * q + 1] = v.y;
          bf[4 * q + 2] = v.z;
          bf[4 * q + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int q = 0; q < KC / 2; ++q) bf[q] = 0u;  // zero activations: the chunk adds 0
      }
#pragma unroll
      for (int j = 0; j < NMMA; ++j)
        mma_16816(acc[mg], *reinterpret_cast<const uint32_t*>(&ha[2 * j]),
                  *reinterpret_cast<const uint32_t*>(&hb[2 * j]),
                  *reinterpret_cast<const uint32_t*>(&ha[2 * j + 1]),
                  *reinterpret_cast<const uint32_t*>(&hb[2 * j + 1]), bf[2 * j], bf[2 * j + 1]);
    }
  };

  const int cl = c0 + 4 * warp + t;  // this lane's chunk at step 0
  int st = 0;
  for (; st + U <= steps; st += U) {
    uint4 xa[U], xb[U];
    GroupQ q[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = cl + 16 * (st + u);
      ok[u] = c < c1;
      xa[u] = xb[u] = make_uint4(0u, 0u, 0u, 0u);
      q[u] = GroupQ{0, 0, 0, 0};
      if (ok[u]) {
        xa[u] = ld_stream(wa + (long long)c * 16);
        xb[u] = ld_stream(wb + (long long)c * 16);
        load_q(c, q[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) use_chunk(cl + 16 * (st + u), ok[u], xa[u], xb[u], q[u]);
  }
  for (; st < steps; ++st) {
    const int c = cl + 16 * st;
    const bool ok = c < c1;
    uint4 xa = make_uint4(0u, 0u, 0u, 0u), xb = xa;
    GroupQ q{0, 0, 0, 0};
    if (ok) {
      xa = ld_stream(wa + (long long)c * 16);
      xb = ld_stream(wb + (long long)c * 16);
      load_q(c, q);
    }
    use_chunk(c, ok, xa, xb, q);
  }

  // accumulator (g, 2t / 2t+1) and (g + 8, 2t / 2t+1) of each 8-row group -> [row][m]
#pragma unroll
  for (int mg = 0; mg < MG; ++mg) {
    const int m = mg * 8 + 2 * t;
    red[warp][g * 16 + m] = acc[mg][0];
    red[warp][g * 16 + m + 1] = acc[mg][1];
    red[warp][(g + 8) * 16 + m] = acc[mg][2];
    red[warp][(g + 8) * 16 + m + 1] = acc[mg][3];
  }
  __syncthreads();
  float part[TILE / kGemvThreads];
#pragma unroll
  for (int q = 0; q < TILE / kGemvThreads; ++q) {
    const int i = tid + q * kGemvThreads;
    float v = red[0][i];
#pragma unroll
    for (int w = 1; w < NWARP; ++w) v += red[w][i];
    part[q] = v;
  }
  if (splits > 1) {
    // every k-slice's CTA total into slot `rank` of the cluster's rank 0
#pragma unroll
    for (int q = 0; q < TILE / kGemvThreads; ++q) {
      const int i = tid + q * kGemvThreads;
      st_dsmem_f32(mapa_shared(smem_u32(&slots[rank][i]), 0), part[q]);
    }
    cluster_sync();
    if (rank != 0) return;
#pragma unroll
    for (int q = 0; q < TILE / kGemvThreads; ++q) {
      const int i = tid + q * kGemvThreads;
      float v = slots[0][i];
      for (int s2 = 1; s2 < splits; ++s2) v += slots[s2][i];
      part[q] = v;
    }
  }
#pragma unroll
  for (int q = 0; q < TILE / kGemvThreads; ++q) {
    const int i = tid + q * kGemvThreads;
    const int r = i >> 4, m = i & 15;
    const int n = n0 + r;
    if (m < M && n < N) {
      const float sc = WQ == kWInt8PerChannel ? __half2float(__ldg(scale + n)) : 1.f;
      C[(long long)m * ldc + n] = __float2half_rn(part[q] * sc);
    }
  }
}

}  // namespace tempo_sm100

namespace tempo_sm100 {

// ---------------------------------------------------------------------------------------------
// k_gemm_sm100_pair: fp16 prefill tiles of 256 x BN on a 2-CTA cluster (cta_group::2).
//
// CTA r of the pair holds A rows [256 t + 128 r, +128) and B rows [BN u + (BN/2) r, +BN/2) of
// every k-block, loaded by its own TMA (no multicast); the leader (rank 0) issues
// tcgen05.mma.cta_group::2 with M = 256, which reads both CTAs' shared memory and writes each
// CTA's own 128 x BN accumulator in its TMEM.  Per SM this halves the B feed of the 1-CTA
// 128 x BN tile.  Stage completion: both CTAs' TMA bytes are counted on the leader's full
// barrier; tcgen05.commit multicasts stage release and accumulator-ready to both CTAs; both
// epilogues report accumulator-consumed to the leader.  Non-swapped, no split-K.
// ---------------------------------------------------------------------------------------------
// One unit of work of the 2-CTA kernel: k-blocks [kb0, kb1) of a tile.  contrib is the number
// of k-slices the tile is cut into (1: the cluster owns the whole tile), slot this unit's
// k-slice and t the tile's place in the tail.
struct PairSeg {
  int tile, kb0, kb1, slot, contrib, t;
};

// Walks a cluster's units: its whole tiles (cluster, cluster + P, ... below sk_tile0), then
// its tail units u = cluster, cluster + P, ... below sk_tiles * sk_splits, numbered k-slice
// major (u = slice * sk_tiles + t) so that the clusters of one wave work on neighbouring
// k-slices and the tail's operand panels stay in L2.
struct PairSegIter {
  int dp_next, u, P;
  __device__ __forceinline__ PairSegIter(const GemmArgs& a, int cluster, int nclusters)
      : dp_next(cluster), u(cluster), P(nclusters) {}
  __device__ __forceinline__ bool next(const GemmArgs& a, PairSeg& s) {
    if (dp_next < a.sk_tile0) {
      s.tile = dp_next;
      s.kb0 = 0;
      s.kb1 = a.num_kb;
      s.slot = 0;
      s.contrib = 1;
      s.t = 0;
      dp_next += P;
      return true;
    }
    if (a.sk_splits == 0 || u >= a.sk_tiles * a.sk_splits) return false;
    const int slice = u / a.sk_tiles;
    s.t = u - slice * a.sk_tiles;
    s.tile = a.sk_tile0 + s.t;
    s.kb0 = (int)((long long)a.num_kb * slice / a.sk_splits);
    s.kb1 = (int)((long long)a.num_kb * (slice + 1) / a.sk_splits);
    s.slot = slice;
    s.contrib = a.sk_splits;
    u += P;
    return true;
  }
};

// Raster position (tp, tq) of a tile (group_m rows of tiles at a time, for L2 reuse).
__device__ __forceinline__ void tile_pos(const GemmArgs& a, int tile, int& tp, int& tq) {
  const int gsz = a.group_m * a.tiles_q;
  const int g = tile / gsz;
  const int first = g * a.group_m;
  const int gm = min(a.tiles_p - first, a.group_m);
  const int r = tile - g * gsz;
  tp = first + r % gm;
  tq = r / gm;
}

template <int BN_>
struct PairCfg {
  static constexpr int BM = 128, BN = BN_, BK = 64;
  static constexpr int A_BYTES = BM * BK * 2;
  static constexpr int B_BYTES = (BN / 2) * BK * 2;
  static constexpr int B_OFF = A_BYTES;
  static constexpr int STAGE_BYTES = A_BYTES + round_up(B_BYTES, 1024);
  static constexpr int EPI_BYTES = 4 * 2 * 2048;
  static constexpr int BAR_BYTES = 512;
  static constexpr int STAGES = cmin((kMaxDynSmem - 1024 - EPI_BYTES - BAR_BYTES) / STAGE_BYTES, 8);
  static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + EPI_BYTES + BAR_BYTES;
  static constexpr int THREADS = 192;
  // accumulator buffer b starts at TMEM column b * ACC_STRIDE (a power of two)
  static constexpr int ACC_STRIDE = BN <= 128 ? 128 : 256;
  static constexpr int TMEM_COLS = tmem_cols_for(2 * ACC_STRIDE);
  static_assert(BN % 32 == 0 && BN >= 128 && BN <= 256,
                "pair tiles are 256 x BN, BN in 128..256 step 32 (32-column epilogue chunks)");
  static_assert(2 * STAGES + 5 <= BAR_BYTES / 8 - 2, "barrier area too small");
};

template <int BN, bool SWIGLU, bool EPI = false>
__global__ void __launch_bounds__(PairCfg<BN>::THREADS, 1)
    k_gemm_sm100_pair(const __grid_constant__ CUtensorMap mapA,
                      const __grid_constant__ CUtensorMap mapB,
                      const __grid_constant__ CUtensorMap mapC, const GemmArgs args) {
  using Cfg = PairCfg<BN>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* epi_smem = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi_smem + Cfg::EPI_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* last_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);

  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1;
  const int nclusters = gridDim.x >> 1;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
  const uint32_t done_bar = bar_base + 8u * (2 * STAGES + 4);
  auto a_addr = [&](int s) { return smem_base + s * Cfg::STAGE_BYTES; };
  auto b_addr = [&](int s) { return smem_base + s * Cfg::STAGE_BYTES + Cfg::B_OFF; };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);   // leader: its own arrive.expect_tx + both CTAs' bytes
      mbar_init(empty_bar(s), 1);  // multicast commit from the leader's MMA thread
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 8);  // leader: 4 epilogue warps of each CTA
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&mapA);
    tma_prefetch_desc(&mapB);
    tma_prefetch_desc(&mapC);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised before any cross-CTA traffic
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Nothing above touches global memory another grid may write: overlap it with that grid.
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both)
    if (lane == 0) {
      const uint64_t pol = policy_evict_normal();
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      PairSegIter segs(args, cluster, nclusters);
      PairSeg sg;
      while (segs.next(args, sg)) {
        int tp, tq;
        tile_pos(args, sg.tile, tp, tq);
        bool ok = true;
        for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, 11)) { ok = false; break; }
          if (leader) mbar_arrive_expect_tx(full_bar(stage), 2 * (Cfg::A_BYTES + Cfg::B_BYTES));
          const uint32_t lead_full = mapa_shared(full_bar(stage), 0);
          const int kx = kb * Cfg::BK;
          tma_load_2d_pair(a_addr(stage), &mapA, lead_full, kx, tp * 256 + (int)rank * 128, pol);
          tma_load_2d_pair(b_addr(stage), &mapB, lead_full, kx, tq * BN + (int)rank * (BN / 2), pol);
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
      }
      // Drain: the leader's full barriers see every byte both CTAs requested.
      if (leader) {
        const int pending = issued < STAGES ? issued : STAGES;
        int s = stage;
        uint32_t ph = phase;
        for (int i = 0; i < pending; ++i) {
          if (--s < 0) {
            s = STAGES - 1;
            ph ^= 1u;
          }
          mbar_drain(full_bar(s), ph, 100000000ull);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader)
    if (leader && lane == 0) {
      constexpr uint32_t idesc = idesc_f16_f32(256, BN);
      int stage = 0;
      uint32_t phase = 0;
      int lu = 0;
      PairSegIter segs(args, cluster, nclusters);
      PairSeg sg;
      for (; segs.next(args, sg); ++lu) {
        const int kb0 = sg.kb0;
        const int buf = lu & 1;
        const uint32_t uphase = (lu >> 1) & 1;
        if (!mbar_wait_cluster(tempty_bar(buf), uphase ^ 1u, abort_flag, 12)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * Cfg::ACC_STRIDE;
        bool ok = true;
        for (int kb = kb0; kb < sg.kb1; ++kb) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, 13)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < Cfg::BK / 16; ++k)
            umma_f16_ss_pair(d_tmem, sdesc_k_sw128(a_addr(stage) + k * 32),
                             sdesc_k_sw128(b_addr(stage) + k * 32), idesc,
                             (kb > kb0 || k > 0) ? 1u : 0u);
          umma_commit_pair_mc(empty_bar(stage), 0x3);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair_mc(tfull_bar(buf), 0x3);
      }
      umma_commit_pair_mc(done_bar, 0x1);
      mbar_drain(done_bar, 0, 100000000ull);
    }
  } else {
    // ------------------------------------------------------------------ epilogue (both)
    const int quad = warp & 3;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    uint8_t* stage_buf = epi_smem + (warp - 2) * 4096;
    int sb = 0;
    int lu = 0;
    PairSegIter segs(args, cluster, nclusters);
    PairSeg sg;
    for (; segs.next(args, sg); ++lu) {
      int tp, tq;
      tile_pos(args, sg.tile, tp, tq);
      const int buf = lu & 1;
      const uint32_t uphase = (lu >> 1) & 1;
      const int q0 = tq * BN;
      const int row0 = tp * 256 + (int)rank * 128 + quad * 32;
      EpiRes res;
      if (EPI && sg.contrib <= 1) res.load(args.epi, row0 + lane, args.rows_p, q0, args.rows_q);
      // one lane's wait may run out where another's did not: the TMEM loads below take whole warps,
      // a tail's barriers all four, so all go on or none does
      if (!named_barrier_and(1, 128, mbar_wait(tfull_bar(buf), uphase, abort_flag, 14))) break;
      tc_fence_after();
      const uint32_t t_acc = t_lane + buf * Cfg::ACC_STRIDE;
      if (sg.contrib > 1 && (args.ws == nullptr || args.counters == nullptr)) {
        // a tail without workspace is a host-side bug: report it instead of faulting
        if (lane == 0 && atomicCAS(&g_status[0], 0, 2) == 0) {
          g_status[1] = 16;
          g_status[2] = blockIdx.x;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
        continue;
      }
      if (sg.contrib > 1) {
        // Tail k-slice: this CTA's 128 x BN fp32 partial goes to slot (slice, t), laid out
        // [32-column chunk][row][32] so each thread writes and reads its row's 128 contiguous
        // bytes per chunk as float4s.  The last of the tile's k-slices to arrive keeps its own
        // accumulator in TMEM, adds the other slots in k order (deterministic) and writes C.
        const int skt = sg.t;
        const long long slice = (long long)128 * BN;
        const long long slot_stride = 2LL * args.sk_tiles * slice;  // next k-slice, same tile
        const float* base = args.ws + ((long long)skt * 2 + rank) * slice;
        const int row = quad * 32 + lane;
        float4* part = reinterpret_cast<float4*>(const_cast<float*>(base) + sg.slot * slot_stride);
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          float f[32];
          acc_chunk<32, 1, BN>(t_acc, c, f);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            __stcg(part + (c * 128 + row) * 8 + q,
                   make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]));
        }
        __threadfence();
        named_barrier_sync(1, 128);
        if (threadIdx.x == 64) {
          int* ctr = args.counters + skt * 2 + rank;
          const int old = atomicAdd(ctr, 1);
          const int last = old == sg.contrib - 1;
          if (last) atomicExch(ctr, 0);  // ready for the next call
          *last_flag = last;
        }
        named_barrier_sync(1, 128);
        const bool last = *last_flag != 0;
        if (!last) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
          continue;
        }
        __threadfence();
        const int p = row0 + lane;
        const int S = sg.contrib;
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          if (EPI) res.load(args.epi, p, args.rows_p, q0 + c * 32, args.rows_q);
          float acc[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[i] = 0.f;
          // slots in k order, four at a time (32 float4 loads in flight per thread); this
          // CTA's own slot comes from TMEM
          for (int j0 = 0; j0 < S; j0 += 4) {
            float4 x[4][8];
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const int j = j0 + jj;
              if (j < S && j != sg.slot) {
                const float4* src = reinterpret_cast<const float4*>(base + j * slot_stride) +
                                    (c * 128 + row) * 8;
#pragma unroll
                for (int q = 0; q < 8; ++q) x[jj][q] = __ldcg(src + q);
              }
            }
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const int j = j0 + jj;
              if (j >= S) break;
              if (j == sg.slot) {
                float f[32];
                acc_chunk<32, 1, BN>(t_acc, c, f);
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[i] += f[i];
              } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                  acc[4 * q] += x[jj][q].x;
                  acc[4 * q + 1] += x[jj][q].y;
                  acc[4 * q + 2] += x[jj][q].z;
                  acc[4 * q + 3] += x[jj][q].w;
                }
              }
            }
          }
          if (c == BN / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
          }
          if (p >= args.rows_p) continue;
          if (EPI) epi_row32(args.epi, acc, res, p, args.rows_p, q0 + c * 32, args.rows_q);
#pragma unroll
          for (int i0 = 0; i0 < 32; i0 += 8) {
            const int q = q0 + c * 32 + i0;
            if (q >= args.rows_q) break;
            uint4 w;
            w.x = pack_half2(acc[i0 + 0], acc[i0 + 1]);
            w.y = pack_half2(acc[i0 + 2], acc[i0 + 3]);
            w.z = pack_half2(acc[i0 + 4], acc[i0 + 5]);
            w.w = pack_half2(acc[i0 + 6], acc[i0 + 7]);
            *reinterpret_cast<uint4*>(args.C + (long long)p * args.ldc + q) = w;
          }
        }
        continue;
      }
      const int live_cols = args.rows_q - q0;
      const bool rows_live = row0 < args.rows_p;
      if (SWIGLU) {
        // Fused SwiGLU: the weight rows are gate/up blocks of 64 interleaved, so each 128
        // accumulator columns of the tile hold 64 gate and the matching 64 up columns.  Out
        // column j of group h: silu(acc[h*128 + j]) * acc[h*128 + 64 + j]; C has N / 2
        // columns and this tile writes [q0 / 2, q0 / 2 + BN / 2).
        const int groups = (live_cols >= BN ? BN : live_cols) / 128;
#pragma unroll 1
        for (int h = 0; h < groups; ++h) {
#pragma unroll 1
          for (int cc = 0; cc < 2; ++cc) {
            float g[32], u[32];
            acc_chunk<32, 1, BN>(t_acc, h * 4 + cc, g);
            acc_chunk<32, 1, BN>(t_acc, h * 4 + 2 + cc, u);
            if (h == groups - 1 && cc == 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
            }
            if (!rows_live) continue;
#pragma unroll
            for (int j = 0; j < 32; ++j) g[j] = g[j] / (1.f + expf(-g[j])) * u[j];
            if (lane == 0) bulk_wait_group_read<1>();
            __syncwarp();
            uint8_t* sbuf = stage_buf + sb * 2048;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint4 w;
              w.x = pack_half2(g[8 * k + 0], g[8 * k + 1]);
              w.y = pack_half2(g[8 * k + 2], g[8 * k + 3]);
              w.z = pack_half2(g[8 * k + 4], g[8 * k + 5]);
              w.w = pack_half2(g[8 * k + 6], g[8 * k + 7]);
              const int pg = k ^ ((lane >> 1) & 3);  // 64-byte swizzle
              *reinterpret_cast<uint4*>(sbuf + lane * 64 + pg * 16) = w;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&mapC, smem_u32(sbuf), q0 / 2 + h * 64 + cc * 32, row0);
              bulk_commit_group();
            }
            sb ^= 1;
          }
        }
        continue;
      }
      const int nchunk = live_cols >= BN ? BN / 32 : (live_cols + 31) / 32;
#pragma unroll 1
      for (int c = 0; c < nchunk; ++c) {
        float f[32];
        acc_chunk<32, 1, BN>(t_acc, c, f);
        if (c == nchunk - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
        }
        if (!rows_live) continue;
        if (EPI) {
          const EpiRes cur = res;
          if (c + 1 < nchunk)
            res.load(args.epi, row0 + lane, args.rows_p, q0 + c * 32 + 32, args.rows_q);
          epi_row32(args.epi, f, cur, row0 + lane, args.rows_p, q0 + c * 32, args.rows_q);
        }
        if (lane == 0) bulk_wait_group_read<1>();
        __syncwarp();
        uint8_t* sbuf = stage_buf + sb * 2048;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint4 w;
          w.x = pack_half2(f[8 * g + 0], f[8 * g + 1]);
          w.y = pack_half2(f[8 * g + 2], f[8 * g + 3]);
          w.z = pack_half2(f[8 * g + 4], f[8 * g + 5]);
          w.w = pack_half2(f[8 * g + 6], f[8 * g + 7]);
          const int pg = g ^ ((lane >> 1) & 3);  // 64-byte swizzle
          *reinterpret_cast<uint4*>(sbuf + lane * 64 + pg * 16) = w;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&mapC, smem_u32(sbuf), q0 + c * 32, row0);
          bulk_commit_group();
        }
        sb ^= 1;
      }
    }
    if (lane == 0) bulk_wait_group<0>();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still touch its barriers or smem
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------
// k_gemm_sm100_pair_w8: W8A16 prefill tiles of 256 x BN on a 2-CTA cluster (cta_group::2).
//
// The fp16 pair kernel's shape (CTA r holds A rows [256 t + 128 r, +128) and weight rows
// [BN u + (BN/2) r, +BN/2); the leader issues tcgen05.mma.cta_group::2), with the weights read
// as 8 bits and dequantised to fp16 in shared memory by each CTA for its own half.  Each of the
// NS slots holds an MMA part [A 128 x 64 fp16 | B half (BN/2) x 64 fp16, 128-byte swizzle] and a
// raw part [raw B half (BN/2) x 64 bytes | group-wise scale row | zero row].  The raw part is
// released (and refilled by warp 6) as soon as its dequant warps have read it, well before the
// MMA frees the slot's MMA part, so the weights' HBM latency hides behind the conversions and
// MMAs of the other slots.  A slot's MMA part: the MMA reading it completes (commit multicast:
// empty) -> warp 0 refills its A (the leader's full barrier counts both CTAs' bytes) while the
// slot's dequant warps convert its raw part into the B half, fence the generic-proxy stores for
// the async proxy and arrive on the leader's deq barrier -> the leader's MMA waits for full and
// deq.  Measured on B200 (clock64 trace of one stage): raw TMA latency 1000-3000 cycles, one
// warp converting 8192 weights ~700-1100 cycles, the arrive with cluster-scope release
// 1000-2000 cycles: every slot has its own dequant warps, so these overlap across slots.
//
// Warps: 0 A producer, 1 MMA issuer (leader) / TMEM owner, 2-5 epilogue, 6 raw producer,
// 7 .. 6 + NS * WPG dequant (WPG warps own each slot, so every wait on a slot's barriers is
// made by its single owner group, in order, and never sees an older phase).  Per-channel scales
// are applied in the epilogue; group-wise scale and zero point in the dequant.  The tiles of a
// ragged last wave -- or all tiles, when there are fewer tiles than clusters (the narrow-N
// shapes at M = 256) -- may run as k-slices (pair_plan's split tail), their fp32 partials
// summed in k order by the last slice to arrive, which applies the per-channel scale.  No
// SwiGLU.
// ---------------------------------------------------------------------------------------------
template <int BN_>
struct PairW8Cfg {
  static constexpr int BM = 128, BN = BN_, BK = 64;
  static constexpr int A_BYTES = BM * BK * 2;
  static constexpr int B_BYTES = (BN / 2) * BK * 2;
  static constexpr int X_BYTES = A_BYTES + round_up(B_BYTES, 1024);  // a slot's MMA part
  static constexpr int RAW_BYTES = (BN / 2) * BK;
  static constexpr int S_OFF = RAW_BYTES;                   // group-wise scale row (fp16)
  static constexpr int Z_OFF = RAW_BYTES + (BN / 2) * 2;    // group-wise zero row (uint8)
  static constexpr int SZ_BYTES = (BN / 2) * 3;
  static constexpr int R_BYTES = round_up(RAW_BYTES + SZ_BYTES, 1024);  // a slot's raw part
  static constexpr int EPI_BYTES = 4 * 2 * 2048;
  static constexpr int BAR_BYTES = 512;
  static constexpr int NS = cmin((kMaxDynSmem - 1024 - EPI_BYTES - BAR_BYTES) / (X_BYTES + R_BYTES), 8);
  static constexpr int SMEM = 1024 + NS * (X_BYTES + R_BYTES) + EPI_BYTES + BAR_BYTES;
  static constexpr int WPG = BN / 128;  // dequant warps per slot: 256 raw chunks each
  static constexpr int DEQ_WARPS = NS * WPG;
  static constexpr int THREADS = 32 * (7 + DEQ_WARPS);
  static constexpr int CHUNKS_PER_WARP = RAW_BYTES / 16 / WPG;
  static constexpr int NBARS = 5 * NS + 5;
  static constexpr int ACC_STRIDE = BN <= 128 ? 128 : 256;
  static constexpr int TMEM_COLS = tmem_cols_for(2 * ACC_STRIDE);
  static_assert(BN == 128 || BN == 256, "W8A16 pair tiles are 256 x 128 or 256 x 256");
  static_assert(NS >= 2, "at least two slots");
  static_assert(NBARS <= BAR_BYTES / 8 - 2, "barrier area too small");
  static_assert(CHUNKS_PER_WARP % 128 == 0, "dequant: whole passes of 4 chunks per lane");
  static_assert(SMEM <= kMaxDynSmem, "shared memory");
};

template <int BN, int WQ>
__global__ void __launch_bounds__(PairW8Cfg<BN>::THREADS, 1)
    k_gemm_sm100_pair_w8(const __grid_constant__ CUtensorMap mapA,
                         const __grid_constant__ CUtensorMap mapW,
                         const __grid_constant__ CUtensorMap mapC,
                         const __grid_constant__ CUtensorMap mapS,
                         const __grid_constant__ CUtensorMap mapZ, const GemmArgs args) {
  using Cfg = PairW8Cfg<BN>;
  constexpr int NS = Cfg::NS;
  static_assert(WQ == kWInt8PerChannel || WQ == kWUint8Group, "8-bit weights");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* raw_smem = smem + NS * Cfg::X_BYTES;
  uint8_t* epi_smem = raw_smem + NS * Cfg::R_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi_smem + Cfg::EPI_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* last_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);

  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1;
  const int nclusters = gridDim.x >> 1;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (NS + s); };
  auto deq_bar = [&](int s) { return bar_base + 8u * (2 * NS + s); };
  auto rfull_bar = [&](int s) { return bar_base + 8u * (3 * NS + s); };
  auto rempty_bar = [&](int s) { return bar_base + 8u * (4 * NS + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (5 * NS + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (5 * NS + 2 + b); };
  const uint32_t done_bar = bar_base + 8u * (5 * NS + 4);
  auto a_addr = [&](int s) { return smem_base + s * Cfg::X_BYTES; };
  auto b_addr = [&](int s) { return smem_base + s * Cfg::X_BYTES + Cfg::A_BYTES; };
  auto r_addr = [&](int s) { return smem_u32(raw_smem) + s * Cfg::R_BYTES; };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full_bar(s), 1);              // leader: both CTAs' A bytes
      mbar_init(empty_bar(s), 1);             // multicast commit from the leader's MMA thread
      mbar_init(deq_bar(s), 2 * Cfg::WPG);    // leader: the slot's dequant warps of both CTAs
      mbar_init(rfull_bar(s), 1);             // this CTA's raw (+ scale / zero) bytes
      mbar_init(rempty_bar(s), Cfg::WPG);     // this CTA's dequant warps done reading them
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 8);            // leader: 4 epilogue warps of each CTA
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&mapA);
    tma_prefetch_desc(&mapC);
  }
  if (warp == 6 && lane == 0) {
    tma_prefetch_desc(&mapW);
    if (WQ == kWUint8Group) {
      tma_prefetch_desc(&mapS);
      tma_prefetch_desc(&mapZ);
    }
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised before any cross-CTA traffic
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------------ A producer (both)
    if (lane == 0) {
      const uint64_t pol = policy_evict_normal();
      int it = 0;
      PairSegIter segs(args, cluster, nclusters);
      PairSeg sg;
      bool ok = true;
      while (ok && segs.next(args, sg)) {
        int tp, tq;
        tile_pos(args, sg.tile, tp, tq);
        for (int kb = sg.kb0; kb < sg.kb1; ++kb, ++it) {
          const int s = it % NS;
          const uint32_t ph = (uint32_t)((it / NS) & 1);
          if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, 11)) { ok = false; break; }
          if (leader) mbar_arrive_expect_tx(full_bar(s), 2 * Cfg::A_BYTES);
          tma_load_2d_pair(a_addr(s), &mapA, mapa_shared(full_bar(s), 0), kb * Cfg::BK,
                           tp * 256 + (int)rank * 128, pol);
        }
      }
      if (leader) {  // the leader's full barriers see every A byte both CTAs requested
        const int pending = it < NS ? it : NS;
        for (int j = it - pending; j < it; ++j)
          mbar_drain(full_bar(j % NS), (uint32_t)((j / NS) & 1), 100000000ull);
      }
    }
  } else if (warp == 6) {
    // ------------------------------------------------------------------ raw producer (both)
    if (lane == 0) {
      const uint64_t pol = policy_evict_normal();
      int it = 0;
      PairSegIter segs(args, cluster, nclusters);
      PairSeg sg;
      bool ok = true;
      while (ok && segs.next(args, sg)) {
        int tp, tq;
        tile_pos(args, sg.tile, tp, tq);
        const int nrow = tq * BN + (int)rank * (BN / 2);
        for (int kb = sg.kb0; kb < sg.kb1; ++kb, ++it) {
          const int s = it % NS;
          const uint32_t ph = (uint32_t)((it / NS) & 1);
          if (!mbar_wait(rempty_bar(s), ph ^ 1u, abort_flag, 19)) { ok = false; break; }
          mbar_arrive_expect_tx(rfull_bar(s),
                                Cfg::RAW_BYTES + (WQ == kWUint8Group ? Cfg::SZ_BYTES : 0));
          const int kx = kb * Cfg::BK;
          tma_load_2d(r_addr(s), &mapW, rfull_bar(s), kx, nrow, pol);
          if (WQ == kWUint8Group) {
            const int g = kx / args.group_size;
            tma_load_2d(r_addr(s) + Cfg::S_OFF, &mapS, rfull_bar(s), nrow, g, pol);
            tma_load_2d(r_addr(s) + Cfg::Z_OFF, &mapZ, rfull_bar(s), nrow, g, pol);
          }
        }
      }
      const int pending = it < NS ? it : NS;  // every raw byte landed before the CTA exits
      for (int j = it - pending; j < it; ++j)
        mbar_drain(rfull_bar(j % NS), (uint32_t)((j / NS) & 1), 100000000ull);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader)
    if (leader && lane == 0) {
      constexpr uint32_t idesc = idesc_f16_f32(256, BN);
      int it = 0;
      int lu = 0;
      PairSegIter segs(args, cluster, nclusters);
      PairSeg sg;
      for (; segs.next(args, sg); ++lu) {
        const int buf = lu & 1;
        const uint32_t uphase = (lu >> 1) & 1;
        if (!mbar_wait_cluster(tempty_bar(buf), uphase ^ 1u, abort_flag, 12)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * Cfg::ACC_STRIDE;
        bool ok = true;
        for (int kb = sg.kb0; kb < sg.kb1; ++kb, ++it) {
          const int s = it % NS;
          const uint32_t ph = (uint32_t)((it / NS) & 1);
          if (!mbar_wait(full_bar(s), ph, abort_flag, 13)) { ok = false; break; }
          if (!mbar_test_wait_cluster(deq_bar(s), ph) &&
              !mbar_poll_cluster(deq_bar(s), ph, abort_flag, 18)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < Cfg::BK / 16; ++k)
            umma_f16_ss_pair(d_tmem, sdesc_k_sw128(a_addr(s) + k * 32),
                             sdesc_k_sw128(b_addr(s) + k * 32), idesc,
                             (kb > sg.kb0 || k > 0) ? 1u : 0u);
          umma_commit_pair_mc(empty_bar(s), 0x3);
        }
        if (!ok) break;
        umma_commit_pair_mc(tfull_bar(buf), 0x3);
      }
      umma_commit_pair_mc(done_bar, 0x1);
      mbar_drain(done_bar, 0, 100000000ull);
    }
  } else if (warp >= 7) {
    // ------------------------------------------------------------------ dequant (both)
    // Group g = (warp - 7) / WPG owns slot g, hence every iteration it with it % NS == g.
    // Warp w of the group converts raw chunks [w, w + 1) x CHUNKS_PER_WARP: chunk c is 16
    // weights of row c / 4, k-range 16 (c % 4); lane l takes c = l + 32 i, so reads are
    // consecutive 16-byte chunks, and the row's two fp16 granules 2 (c % 4), 2 (c % 4) + 1 go
    // to granule ^ (row & 7), the 128-byte swizzle of the MMA operand (each pass of stores hits
    // every granule position of its 8 rows once: no bank conflicts).
    const int dw = warp - 7;
    const int grp = dw / Cfg::WPG;
    const int c0 = (dw % Cfg::WPG) * Cfg::CHUNKS_PER_WARP;
    const uint32_t lead_deq = mapa_shared(deq_bar(grp), 0);
    const uint8_t* raw = raw_smem + grp * Cfg::R_BYTES;
    uint8_t* dst = smem + grp * Cfg::X_BYTES + Cfg::A_BYTES;
    int it = 0;
    PairSegIter segs(args, cluster, nclusters);
    PairSeg sg;
    bool ok = true;
    while (ok && segs.next(args, sg)) {
      for (int kb = sg.kb0; kb < sg.kb1; ++kb, ++it) {
        if (it % NS != grp) continue;
        const uint32_t ph = (uint32_t)((it / NS) & 1);
        if (!mbar_wait(rfull_bar(grp), ph, abort_flag, 17) ||
            !mbar_wait(empty_bar(grp), ph ^ 1u, abort_flag, 20)) {
          ok = false;
          break;
        }
#pragma unroll 1
        for (int i0 = 0; i0 < Cfg::CHUNKS_PER_WARP / 32; i0 += 4) {
          uint4 x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            x[u] = *reinterpret_cast<const uint4*>(raw + (c0 + lane + 32 * (i0 + u)) * 16);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int c = c0 + lane + 32 * (i0 + u);
            const int row = c >> 2, kq = c & 3;
            __half2 h[8];
            if (WQ == kWInt8PerChannel) {
              // signed byte b -> (b ^ 0x80) = b + 128; 1024 + (b + 128) - 1152 = b, exact
              const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152.0
              u8x4_to_h2x2_biased(x[u].x ^ 0x80808080u, h[0], h[1]);
              u8x4_to_h2x2_biased(x[u].y ^ 0x80808080u, h[2], h[3]);
              u8x4_to_h2x2_biased(x[u].z ^ 0x80808080u, h[4], h[5]);
              u8x4_to_h2x2_biased(x[u].w ^ 0x80808080u, h[6], h[7]);
#pragma unroll
              for (int j = 0; j < 8; ++j) h[j] = __hsub2(h[j], bias);
            } else {
              // (1024 + q) - (1024 + z) = q - z exactly, then one rounding in the scale
              // product; rows past N were zero-filled by TMA (s = 0), so their weights are 0
              const __half2 zb = __half2half2(
                  __ushort_as_half((unsigned short)(0x6400u | raw[Cfg::Z_OFF + row])));
              const __half2 s2 =
                  __half2half2(reinterpret_cast<const __half*>(raw + Cfg::S_OFF)[row]);
              u8x4_to_h2x2_biased(x[u].x, h[0], h[1]);
              u8x4_to_h2x2_biased(x[u].y, h[2], h[3]);
              u8x4_to_h2x2_biased(x[u].z, h[4], h[5]);
              u8x4_to_h2x2_biased(x[u].w, h[6], h[7]);
#pragma unroll
              for (int j = 0; j < 8; ++j) h[j] = __hmul2(__hsub2(h[j], zb), s2);
            }
            const uint4* hv = reinterpret_cast<const uint4*>(h);
            uint8_t* drow = dst + row * 128;
            *reinterpret_cast<uint4*>(drow + (((2 * kq) ^ (row & 7)) * 16)) = hv[0];
            *reinterpret_cast<uint4*>(drow + (((2 * kq + 1) ^ (row & 7)) * 16)) = hv[1];
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(rempty_bar(grp));  // raw part read: the producer may refill
        fence_proxy_async_smem();  // generic-proxy stores -> the MMA's async-proxy reads
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(lead_deq);  // this half of the B operand is ready
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue (both)
    const int quad = warp & 3;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    uint8_t* stage_buf = epi_smem + (warp - 2) * 4096;
    int sb = 0;
    int lu = 0;
    PairSegIter segs(args, cluster, nclusters);
    PairSeg sg;
    for (; segs.next(args, sg); ++lu) {
      int tp, tq;
      tile_pos(args, sg.tile, tp, tq);
      const int buf = lu & 1;
      const uint32_t uphase = (lu >> 1) & 1;
      if (!mbar_wait(tfull_bar(buf), uphase, abort_flag, 14)) break;
      tc_fence_after();
      const uint32_t t_acc = t_lane + buf * Cfg::ACC_STRIDE;
      const int q0 = tq * BN;
      const int row0 = tp * 256 + (int)rank * 128 + quad * 32;
      if (sg.contrib > 1 && (args.ws == nullptr || args.counters == nullptr)) {
        // a split unit without workspace is a host-side bug: report it instead of faulting
        if (lane == 0 && atomicCAS(&g_status[0], 0, 2) == 0) {
          g_status[1] = 16;
          g_status[2] = blockIdx.x;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
        continue;
      }
      if (sg.contrib > 1) {
        // Tail k-slice: this CTA's 128 x BN fp32 partial goes to slot (slice, t), laid out
        // [32-column chunk][row][32] so each thread writes and reads its row's 128 contiguous
        // bytes per chunk as float4s.  The last of the tile's k-slices to arrive keeps its own
        // accumulator in TMEM, adds the other slots in k order (deterministic) and writes C.
        const int skt = sg.t;
        const long long slice = (long long)128 * BN;
        const long long slot_stride = 2LL * args.sk_tiles * slice;  // next k-slice, same tile
        const float* base = args.ws + ((long long)skt * 2 + rank) * slice;
        const int row = quad * 32 + lane;
        float4* part = reinterpret_cast<float4*>(const_cast<float*>(base) + sg.slot * slot_stride);
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          float f[32];
          acc_chunk<32, 1, BN>(t_acc, c, f);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            __stcg(part + (c * 128 + row) * 8 + q,
                   make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]));
        }
        __threadfence();
        named_barrier_sync(1, 128);
        if (threadIdx.x == 64) {
          int* ctr = args.counters + skt * 2 + rank;
          const int old = atomicAdd(ctr, 1);
          const int last = old == sg.contrib - 1;
          if (last) atomicExch(ctr, 0);  // ready for the next call
          *last_flag = last;
        }
        named_barrier_sync(1, 128);
        const bool last = *last_flag != 0;
        if (!last) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
          continue;
        }
        __threadfence();
        const int p = row0 + lane;
        const int S = sg.contrib;
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          float acc[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[i] = 0.f;
          // slots in k order, one at a time (the wide CTA has fewer registers per thread
          // than the fp16 kernel); this CTA's own slot comes from TMEM
          for (int j = 0; j < S; ++j) {
            if (j == sg.slot) {
              float f[32];
              acc_chunk<32, 1, BN>(t_acc, c, f);
#pragma unroll
              for (int i = 0; i < 32; ++i) acc[i] += f[i];
            } else {
              const float4* src = reinterpret_cast<const float4*>(base + j * slot_stride) +
                                  (c * 128 + row) * 8;
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const float4 x = __ldcg(src + q);
                acc[4 * q] += x.x;
                acc[4 * q + 1] += x.y;
                acc[4 * q + 2] += x.z;
                acc[4 * q + 3] += x.w;
              }
            }
          }
          if (c == BN / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
          }
          if (p >= args.rows_p) continue;
#pragma unroll
          for (int i0 = 0; i0 < 32; i0 += 8) {
            const int q = q0 + c * 32 + i0;
            if (q >= args.rows_q) break;
            if (WQ == kWInt8PerChannel) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                acc[i0 + j] *= q + j < args.rows_q ? __half2float(__ldg(args.scale + q + j)) : 0.f;
            }
            uint4 w;
            w.x = pack_half2(acc[i0 + 0], acc[i0 + 1]);
            w.y = pack_half2(acc[i0 + 2], acc[i0 + 3]);
            w.z = pack_half2(acc[i0 + 4], acc[i0 + 5]);
            w.w = pack_half2(acc[i0 + 6], acc[i0 + 7]);
            *reinterpret_cast<uint4*>(args.C + (long long)p * args.ldc + q) = w;
          }
        }
        continue;
      }
      const int live_cols = args.rows_q - q0;
      const bool rows_live = row0 < args.rows_p;
      const int nchunk = live_cols >= BN ? BN / 32 : (live_cols + 31) / 32;
#pragma unroll 1
      for (int c = 0; c < nchunk; ++c) {
        float f[32];
        acc_chunk<32, 1, BN>(t_acc, c, f);
        if (WQ == kWInt8PerChannel) {
          // per-output-channel scale of columns q0 + 32 c + j: lane j loads one, all share it
          const int n = q0 + c * 32 + lane;
          const float sv = n < args.rows_q ? __half2float(__ldg(args.scale + n)) : 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] *= __shfl_sync(0xffffffffu, sv, j);
        }
        if (c == nchunk - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(buf), 0));
        }
        if (!rows_live) continue;
        if (lane == 0) bulk_wait_group_read<1>();
        __syncwarp();
        uint8_t* sbuf = stage_buf + sb * 2048;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint4 w;
          w.x = pack_half2(f[8 * g + 0], f[8 * g + 1]);
          w.y = pack_half2(f[8 * g + 2], f[8 * g + 3]);
          w.z = pack_half2(f[8 * g + 4], f[8 * g + 5]);
          w.w = pack_half2(f[8 * g + 6], f[8 * g + 7]);
          const int pg = g ^ ((lane >> 1) & 3);  // 64-byte swizzle
          *reinterpret_cast<uint4*>(sbuf + lane * 64 + pg * 16) = w;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&mapC, smem_u32(sbuf), q0 + c * 32, row0);
          bulk_commit_group();
        }
        sb ^= 1;
      }
    }
    if (lane == 0) bulk_wait_group<0>();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still touch its barriers or smem
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace tempo_sm100
