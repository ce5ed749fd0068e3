// k_epi_swap: the GEMM with a fused epilogue for 17 .. 384 rows (M), where the weights are most of
// the bytes and a 128- or 256-row tile of activations would be mostly padding.
//
//   D[n][m] = sum_k W[n][k] A[m][k]       128 weight rows are the MMA's M side, ALL activation rows
//                                         its N side: one tcgen05.mma of N <= 256 up to 256 rows,
//                                         two of N <= 192 above
//
// so every weight byte is read from HBM by exactly one CTA and used for all of M; the 128 x M fp32
// accumulator stays in TMEM.  The activations (M x 128 bytes per k-block) come from L2 by TMA once
// per weight tile.  (8-bit weights of more rows: tiles of up to 384 of them, a weight tile's one
// after the other.)
//
// What bounds it: up to 128 rows the weights from HBM and 400 (fp16) to 500 (8-bit) cycles that a
// k-block's chain of barriers and MMA issue takes; above, the activations' way from L2, 40 B per
// cycle and SM.  Measured (us, floor in brackets): fp16 17 x 15360 x 3840 21.5 (18.2),
// 100 x 15360 x 3840 23.8 (18.7), 256 x 18944 x 3840 37.6 (24.1), 333 x 18944 x 3840 47.6 (28.9);
// int8 100 x 15360 x 3840 23.5 (9.6); uint8 333 x 5120 x 17408 65.4 (35.4), the time of
// k_swap_finish behind it, about 10, included.  (A pair of CTAs per tile, cta_group::2 with half the
// activations each: the same with fp16 weights, up to twice as long with 8-bit ones.)
//
// 8-bit weights: raw tiles in a ring of their own (released as soon as they are unpacked, so that
// the HBM latency hides behind more bytes than the fp16 slots could hold); eight warps turn them
// into the slot's swizzled fp16 operand: int8 exactly (the channel's scale multiplies the sum),
// group-wise (q - z) * s rounded once to fp16, the only form the tensor core takes.  (Weights by
// plain loads into a register ring instead of TMA: 500 cycles of one warp's time per k-block for
// eight loads and their addresses, 100 x 15360 x 3840 42 us.)
//
// Work split: the k-blocks of all weight tiles are one sequence, cut into equal contiguous shares,
// one per CTA, unless whole tiles fill the GPU well enough (epi_swap_cost).  A share starts and
// ends inside a tile: the fp32 sums of such partial tiles go to the workspace and k_swap_finish,
// one launch behind, adds them in k order and applies the epilogue with every SM (the last CTA to
// arrive doing so alone took 20 us for 5 parts of a 128 x 128 tile).  No CTA waits for another.
//
// Epilogue: D's rows are output columns, so 16 output rows at a time go through shared memory
// transposed; bias, activation and residual then work on 8 consecutive columns per thread with
// 16-byte accesses, the residual of the next rows in flight meanwhile.
//
// Warps: 0 TMA, 1 MMA (and TMEM), two groups of four for the epilogue that take its chunks of 16
// rows in turn (256 x 18944 x 3840: 38.6 us with one group, 35.8 with two); 8-bit weights: one warp
// for TMA of the raw tiles, eight for unpacking.
#pragma once

namespace tempo_sm100 {

// A bounded wait of a whole warp.  It may run out, or see the abort flag, in some lanes only: the
// warp goes on or gives up as one, since what follows takes all of its lanes (elect.sync,
// __syncwarp).  The loops over k-blocks vote less often, since until they do a wait that ran out
// costs only the result, which is reported as lost (a vote per wait: int8 100 x 15360 x 3840 24.2 us,
// so 23.7; no vote 23.4).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, where));
}

// True in one lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

constexpr int kSwapMaxRows = 384;  // of a tile: two accumulators of 192 columns
constexpr int kSwapRawBytes = 128 * 64 + 1024;           // raw tile, scale row, zero row
constexpr int kSwapStageRow = 132;                       // floats of a transposed output row
constexpr int kSwapStageBytes = 16 * kSwapStageRow * 4;  // one group's
constexpr int kSwapBarBytes = 512;
constexpr int kSwapMaxSlots = 8;

struct SwapArgs {
  int M, N, num_kb;
  int tiles, mt;              // tile t: weight rows from 128 (t / mt), activations from rows (t % mt)
  int rows;                   // activation rows of a tile: n groups
  int n, groups;              // rows per MMA (multiple of 16), MMAs per k step
  int nx, nr;                 // operand slots, raw tiles
  int x_bytes;                // one operand slot: 16 KB of weights, the activations
  int bufs;                   // accumulator buffers (2 when they fit 512 columns)
  int epis;                   // groups of epilogue warps at work
  int unit;                   // shares are multiples of it (k-blocks)
  __half* C;
  long long ldc;
  float* part;                // partial tiles [2 per CTA][rows][128]
  const __half* scale;        // int8: per channel
  int group_size;
  EpiArgs epi;
};

// A CTA's share [begin(c), begin(c + 1)) of the k-blocks of all tiles, in units of `unit` (1, or a
// whole tile).
struct SwapShare {
  int q, r, unit;
  __host__ __device__ SwapShare(int total, int ctas, int unit_) : unit(unit_) {
    q = total / unit / ctas;
    r = total / unit - q * ctas;
  }
  __host__ __device__ int begin(int c) const { return (c * q + (c < r ? c : r)) * unit; }
  // the CTA whose share holds k-block x
  __host__ __device__ int owner(int x) const {
    const int u = x / unit, cut = r * (q + 1);
    return u < cut ? u / (q + 1) : r + (u - cut) / q;
  }
};

struct SwapSeg {
  int n_row, m_row, kb0, kb1;  // first weight row, first activation row, k-blocks
};

struct SwapIter {
  int pos, end, num_kb, mt, rows;
  __device__ __forceinline__ bool next(SwapSeg& s) {
    if (pos >= end) return false;
    const int tile = pos / num_kb, wt = tile / mt;
    s.n_row = wt * 128;
    s.m_row = (tile - wt * mt) * rows;
    s.kb0 = pos - tile * num_kb;
    s.kb1 = min(num_kb, s.kb0 + end - pos);
    pos += s.kb1 - s.kb0;
    return true;
  }
};

// Epilogue of 8 consecutive columns of one output row.
struct EpiCols {
  float bias[8], scale[8];
  __device__ __forceinline__ void load(const EpiArgs& e, const __half* sc, int n0, bool on) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bias[i] = 0.f;
      scale[i] = 1.f;
    }
    if (on && e.bias) unpack_half8(__ldg(reinterpret_cast<const uint4*>(e.bias + n0)), bias);
    if (on && sc) unpack_half8(__ldg(reinterpret_cast<const uint4*>(sc + n0)), scale);
  }
  __device__ __forceinline__ uint4 apply(const EpiArgs& e, float (&o)[8], uint4 res) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = fmaf(o[j], scale[j], bias[j]);
    epi_act(o, e.act);
    if (e.res) {
      float r[8];
      unpack_half8(res, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] += r[j];
    }
    uint4 w;
    w.x = pack_half2(o[0], o[1]);
    w.y = pack_half2(o[2], o[3]);
    w.z = pack_half2(o[4], o[5]);
    w.w = pack_half2(o[6], o[7]);
    return w;
  }
};

template <int WQ>
constexpr int kSwapThreads = WQ ? 19 * 32 : 10 * 32;

// LG: groups of unpacking warps.  2: four warps fill a slot, the others the next one (a slot's
// turn, its data, the fence and the arrival take a warp longer than a k-block may); a
// slot and a raw tile then always have the same group, so nx and nr are even.  1: all eight fill
// every slot.
template <int WQ, int LG>
__global__ void __launch_bounds__(kSwapThreads<WQ>, 1)
    k_epi_swap(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapA,
               const __grid_constant__ CUtensorMap mapS, const __grid_constant__ CUtensorMap mapZ,
               const SwapArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* raw = smem + a.nx * a.x_bytes;
  float* stage0 = reinterpret_cast<float*>(raw + a.nr * kSwapRawBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(stage0) +
                                               a.epis * kSwapStageBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 * kSwapMaxSlots + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t bar0 = smem_u32(bars);
  auto xfull = [&](int s) { return bar0 + 8u * s; };
  auto xempty = [&](int s) { return bar0 + 8u * (kSwapMaxSlots + s); };
  auto rfull = [&](int s) { return bar0 + 8u * (2 * kSwapMaxSlots + s); };
  auto rempty = [&](int s) { return bar0 + 8u * (3 * kSwapMaxSlots + s); };
  auto tfull = [&](int b) { return bar0 + 8u * (4 * kSwapMaxSlots + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (4 * kSwapMaxSlots + 2 + b); };
  const uint32_t done_bar = bar0 + 8u * (4 * kSwapMaxSlots + 4);
  const uint32_t x0 = smem_u32(smem), r0 = smem_u32(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.nx; ++s) {
      mbar_init(xfull(s), 1 + (WQ ? 8 / LG : 0));  // TMA's bytes, the slot's unpacking warps
      mbar_init(xempty(s), 1);                     // the MMAs that read the slot
    }
    for (int s = 0; s < a.nr; ++s) {
      mbar_init(rfull(s), 1);
      mbar_init(rempty(s), 8 / LG);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull(b), 1);
      mbar_init(tempty(b), 4 * a.epis);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&mapW);
    tma_prefetch_desc(&mapA);
    if (WQ == kWUint8Group) {
      tma_prefetch_desc(&mapS);
      tma_prefetch_desc(&mapZ);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  const SwapShare share(a.tiles * a.num_kb, gridDim.x, a.unit);
  SwapIter segs{share.begin(blockIdx.x), share.begin(blockIdx.x + 1), a.num_kb, a.mt,
                a.rows};
  const int n_its = segs.end - segs.pos;  // k-blocks of this CTA
  SwapSeg sg;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA
    if (lane == 0) {
      const uint64_t pol_w = policy_evict_first(), pol = policy_evict_last();
      const uint32_t bytes = (uint32_t)a.rows * 128 + (WQ ? 0u : 16384u);
      int s = 0, it = 0;
      uint32_t ph = 1;
      bool ok = true;
      while (ok && segs.next(sg)) {
        for (int kb = sg.kb0; kb < sg.kb1; ++kb, ++it) {
          if (!mbar_wait(xempty(s), ph, abort_flag, 31)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(xfull(s), bytes);
          if (!WQ)
            tma_load_2d(x0 + s * a.x_bytes, &mapW, xfull(s), kb * 64, sg.n_row, pol_w);
          for (int g = 0; g < a.groups; ++g)
            tma_load_2d(x0 + s * a.x_bytes + 16384 + g * a.n * 128, &mapA, xfull(s),
                        kb * 64, sg.m_row + g * a.n, pol);
          if (++s == a.nx) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // every load issued here has landed before the CTA can exit (matters after an abort)
      for (int j = it > a.nx ? it - a.nx : 0; j < it; ++j)
        mbar_drain(xfull(j % a.nx), (uint32_t)((j / a.nx) & 1), 100000000ull);
    }
  } else if (WQ && warp == 10) {
    // ------------------------------------------------------------------ TMA: raw weights
    if (lane == 0) {
      const uint64_t pol_w = policy_evict_first(), pol = policy_evict_last();
      int s = 0, it = 0;
      uint32_t ph = 1;
      bool ok = true;
      while (ok && segs.next(sg)) {
        for (int kb = sg.kb0; kb < sg.kb1; ++kb, ++it) {
          if (!mbar_wait(rempty(s), ph, abort_flag, 32)) {
            ok = false;
            break;
          }
          const int kx = kb * 64, row = sg.n_row;
          const uint32_t dst = r0 + s * kSwapRawBytes;
          mbar_arrive_expect_tx(rfull(s), 8192 + (WQ == kWUint8Group ? 384 : 0));
          tma_load_2d(dst, &mapW, rfull(s), kx, row, pol_w);
          if (WQ == kWUint8Group) {
            const int g = kx / a.group_size;
            tma_load_2d(dst + 8192, &mapS, rfull(s), row, g, pol);
            tma_load_2d(dst + 8192 + 256, &mapZ, rfull(s), row, g, pol);
          }
          if (++s == a.nr) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      for (int j = it > a.nr ? it - a.nr : 0; j < it; ++j)
        mbar_drain(rfull(j % a.nr), (uint32_t)((j / a.nr) & 1), 100000000ull);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    // The whole warp runs the loop, so that descriptors and barrier addresses stay uniform; one
    // lane issues.  (All of it in one lane: 550 cycles for a k-block's four MMAs, so 210.)
    const uint32_t idesc = idesc_f16_f32(128, a.n);
    // sdesc_k_sw128 split into its words: only the low one changes
    const uint32_t hi = (uint32_t)(sdesc_k_sw128(0) >> 32);
    auto low = [](uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); };
    auto desc = [&](uint32_t lo) { return (uint64_t)hi << 32 | lo; };
    int lu = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (; ok && segs.next(sg); ++lu) {
      const int buf = lu % a.bufs;
      if (!warp_wait(tempty(buf), (uint32_t)((lu / a.bufs) & 1) ^ 1u, abort_flag, 33)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + buf * 256;
      uint32_t add = 0;
      for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
        ok &= mbar_wait(xfull(s), ph, abort_flag, 34);
        tc_fence_after();
        const uint32_t wa = low(x0 + s * a.x_bytes);
        const uint32_t ba = wa + (16384 >> 4), bb = ba + a.n * 8;  // second group: n rows further
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ss(d, desc(wa + 2 * k), desc(ba + 2 * k), idesc, k ? 1u : add);
          if (a.groups > 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16_ss(d + a.n, desc(wa + 2 * k), desc(bb + 2 * k), idesc, k ? 1u : add);
          }
          umma_commit(xempty(s));
        }
        __syncwarp();
        add = 1;
        if (++s == a.nx) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (elect_one()) umma_commit(tfull(buf));
      ok = __all_sync(0xffffffffu, ok);
    }
    if (elect_one()) {
      umma_commit(done_bar);
      mbar_drain(done_bar, 0, 100000000ull);
    }
    __syncwarp();
  } else if (warp < 2 + 4 * a.epis) {
    // ------------------------------------------------------------------ epilogue
    const int quad = warp & 3, row = quad * 32 + lane;  // TMEM lane = weight row of the tile
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    const int grp = (warp - 2) >> 2;                    // takes the chunks grp, grp + epis, ...
    const int tid = (threadIdx.x - 64) & 127, bar = 1 + grp;
    float* stage = stage0 + grp * (kSwapStageBytes / 4);
    const int v8 = (tid & 15) * 8, trow = tid >> 4;     // columns and first output row of a chunk
    int lu = 0;
    for (; segs.next(sg); ++lu) {
      const int buf = lu % a.bufs;
      const uint32_t t_acc = t_lane + buf * 256;
      const bool whole = sg.kb0 == 0 && sg.kb1 == a.num_kb;
      const int live = min(a.rows, a.M - sg.m_row), chunks = (live + 15) / 16;
      const int n0 = sg.n_row + v8;
      const bool n_ok = n0 < a.N;  // N % 8 == 0
      uint4 res[2];
      auto load_res = [&](int c) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int m = c * 16 + trow + 8 * i;
          if (n_ok && m < live)
            res[i] = *reinterpret_cast<const uint4*>(
                a.epi.res + (long long)(sg.m_row + m) * a.epi.ldr + n0);
        }
      };
      EpiCols ec;
      if (whole) {
        ec.load(a.epi, WQ == kWInt8PerChannel ? a.scale : nullptr, n0, n_ok);
        if (a.epi.res) load_res(grp);
      }
      // one warp's wait may run out where another's did not: all four go on or none does
      if (!named_barrier_and(bar, 128, mbar_wait(tfull(buf), (uint32_t)((lu / a.bufs) & 1),
                                                 abort_flag, 36)))
        break;
      tc_fence_after();
      // a partial tile: part 0 of this CTA when the tile began in an earlier share, else part 1
      float* dst = a.part + (blockIdx.x * 2LL + (sg.kb0 > 0 ? 0 : 1)) * a.rows * 128 + row;
      if (grp >= chunks && lane == 0) mbar_arrive(tempty(buf));
#pragma unroll 1
      for (int c = grp; c < chunks; c += a.epis) {
        uint32_t v[16];
        tmem_ld_x16(t_acc + c * 16, v);
        tmem_wait_ld();
        if (c + a.epis >= chunks) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(tempty(buf));
        }
        if (!whole) {
#pragma unroll
          for (int j = 0; j < 16; ++j) __stcg(dst + (c * 16 + j) * 128, __uint_as_float(v[j]));
          continue;
        }
        named_barrier_sync(bar, 128);  // the previous chunk has been read
#pragma unroll
        for (int j = 0; j < 16; ++j) stage[j * kSwapStageRow + row] = __uint_as_float(v[j]);
        named_barrier_sync(bar, 128);
        const uint4 cur[2] = {res[0], res[1]};
        if (a.epi.res && c + a.epis < chunks) load_res(c + a.epis);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int m = c * 16 + trow + 8 * i;
          if (!n_ok || m >= live) continue;
          const float* src = stage + (trow + 8 * i) * kSwapStageRow + v8;
          const float4 lo = *reinterpret_cast<const float4*>(src);
          const float4 hi = *reinterpret_cast<const float4*>(src + 4);
          float o[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          *reinterpret_cast<uint4*>(a.C + (long long)(sg.m_row + m) * a.ldc + n0) =
              ec.apply(a.epi, o, cur[i]);
        }
      }
    }
  } else if (WQ && warp > 10) {
    // ------------------------------------------------------------------ unpacking
    // Group g takes the k-blocks g, g + LG, ...; warp d of it fills rows R d .. R d + R - 1 of the
    // slot, 4 lanes per row: 16 weights of lane (row, lc) are the fp16 granules 2 lc, 2 lc + 1, and
    // granule j of row r lives at j ^ (r % 8) (the operand's 128-byte swizzle); neither reads nor
    // stores conflict.
    constexpr int R = 16 * LG, L = R / 8;  // rows per warp, chunks per lane
    const int grp = LG == 2 ? (warp - 11) >> 2 : 0, d = LG == 2 ? (warp - 11) & 3 : warp - 11;
    const int lr = lane >> 2, lc = lane & 3;
    int s = grp, r = grp;
    uint32_t ph = 1, rph = 0;
    for (int it = grp; it < n_its; it += LG) {
      bool ok = mbar_wait(rfull(r), rph, abort_flag, 37);
      const uint8_t* src = raw + r * kSwapRawBytes;
      uint4 x[L];
      __half2 zb[L], s2[L];
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int wr = R * d + i * 8 + lr;
        x[i] = *reinterpret_cast<const uint4*>(src + wr * 64 + lc * 16);
        zb[i] = s2[i] = __half2half2(__ushort_as_half(0));
        if (WQ == kWUint8Group) {
          zb[i] = __half2half2(__ushort_as_half((unsigned short)(0x6400u | src[8192 + 256 + wr])));
          s2[i] = __half2half2(reinterpret_cast<const __half*>(src + 8192)[wr]);
        }
      }
      ok &= mbar_wait(xempty(s), ph, abort_flag, 38);
      uint8_t* dst = smem + s * a.x_bytes + R * d * 128;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int wr = i * 8 + lr;
        __half2 h[8];
        gemv_weights<WQ>(x[i], h, zb[i], s2[i]);
        const uint4* hv = reinterpret_cast<const uint4*>(h);
        *reinterpret_cast<uint4*>(dst + wr * 128 + (((2 * lc) ^ lr) * 16)) = hv[0];
        *reinterpret_cast<uint4*>(dst + wr * 128 + (((2 * lc + 1) ^ lr) * 16)) = hv[1];
      }
      fence_proxy_async_smem();
      if (!__all_sync(0xffffffffu, ok)) break;
      __syncwarp();
      // The raw tile is released behind the stores that need its values: an arrival right behind
      // the loads does not wait for them, and TMA then overwrites what they are still to read.
      if (lane == 0) {
        mbar_arrive(xfull(s));
        mbar_arrive(rempty(r));
      }
      s += LG;
      if (s >= a.nx) {
        s -= a.nx;
        ph ^= 1u;
      }
      r += LG;
      if (r >= a.nr) {
        r -= a.nr;
        rph ^= 1u;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// The tiles that k_epi_swap's shares cut: their parts added in k order, then the epilogue.  One CTA
// per tile and 16 output rows, 8 columns of a row per thread.
template <int WQ>
__global__ void __launch_bounds__(256, 3) k_swap_finish(const SwapArgs a, int ctas) {
  const int tile = blockIdx.x;
  const SwapShare share(a.tiles * a.num_kb, ctas, a.unit);
  const int first = share.owner(tile * a.num_kb), last = share.owner((tile + 1) * a.num_kb - 1);
  const int v8 = (threadIdx.x & 15) * 8, r = blockIdx.y * 16 + (threadIdx.x >> 4);
  const int wt = tile / a.mt, m = (tile - wt * a.mt) * a.rows + r;
  const int n0 = wt * 128 + v8;
  const bool on = first != last && m < a.M && n0 < a.N;
  // What k_epi_swap does not write can be read while it still runs: it started this launch only
  // after its own wait for whatever wrote these.
  uint4 res = make_uint4(0u, 0u, 0u, 0u);
  if (on && a.epi.res)
    res = *reinterpret_cast<const uint4*>(a.epi.res + (long long)m * a.epi.ldr + n0);
  EpiCols ec;
  ec.load(a.epi, WQ == kWInt8PerChannel ? a.scale : nullptr, n0, on);
  pdl_wait();
  pdl_launch_dependents();
  if (!on) return;
  float o[8] = {};
  for (int c0 = first; c0 <= last; c0 += 4) {
    float4 lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + i;
      lo[i] = hi[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c > last) continue;
      const int part = share.begin(c) > tile * a.num_kb ? 0 : 1;
      const float4* src = reinterpret_cast<const float4*>(
          a.part + ((c * 2LL + part) * a.rows + r) * 128 + v8);
      lo[i] = __ldcg(src);
      hi[i] = __ldcg(src + 1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[0] += lo[i].x;
      o[1] += lo[i].y;
      o[2] += lo[i].z;
      o[3] += lo[i].w;
      o[4] += hi[i].x;
      o[5] += hi[i].y;
      o[6] += hi[i].z;
      o[7] += hi[i].w;
    }
  }
  *reinterpret_cast<uint4*>(a.C + (long long)m * a.ldc + n0) = ec.apply(a.epi, o, res);
}

namespace {

struct SwapPlan {
  int n, groups, rows, mt, x_bytes, nx, nr, bufs, epis, tiles, num_kb, ctas, unit, smem;
  size_t ws_bytes;  // 0: whole tiles, no workspace
};

// How an M x N x K problem runs with mt tiles of activation rows, given ws_bytes of workspace, and
// its cost in cycles.  Model of one k-block on one SM: its MMAs, its activations from L2 at
// 64 B/cycle, its weights from HBM at 30 B/cycle of an SM and at 3400 of the GPU.  It ranks whole
// tiles against equal shares and is no forecast of the time: the chain of barriers and issue, 400 to
// 500 cycles a k-block, is left out on both sides.  Measured, whole / shares us (the
// one chosen):
//   fp16 100 x 15360 x 3840 24.3 / 29.7 (whole)   100 x 10240 x 5120 26.6 / 27.0 (shares)
//        100 x 3840 x 15360 63.4 / 28.0 (shares)  333 x 18944 x 3840 49.4 / 56.7 (whole)
//   int8 100 x 15360 x 3840 23.7 / 27.3 (whole)   100 x 10240 x 5120 29.5 / 25.0 (shares)
//        100 x 3840 x 15360 68.6 / 25.8 (shares)  333 x 18944 x 3840 51.3 / 58.4 (whole)
// Small problems with a long share of the fixed costs can go the wrong way: fp16 200 x 1024 x 1024
// runs whole, 10.9 / 8.8.
double epi_swap_cost(SwapPlan& p, int wkind, int M, int N, int K, int sms, size_t ws_bytes,
                     int mt) {
  const int want = (int)(((long long)M + mt - 1) / mt);
  p.groups = want > 256 ? 2 : 1;
  p.n = ((want + p.groups - 1) / p.groups + 15) / 16 * 16;
  p.rows = p.groups * p.n;
  p.mt = (M + p.rows - 1) / p.rows;
  p.tiles = (N + 127) / 128 * p.mt;
  p.num_kb = (K + 63) / 64;
  p.bufs = p.rows <= 256 ? 2 : 1;
  p.x_bytes = 16384 + p.rows * 128;
  // One group of epilogue warps where the staging of the second would cost an operand slot: 8-bit
  // weights above 320 rows, which then have 2 (333 x 5120 x 17408: 69 us against 65).
  const int room = kMaxDynSmem - 1024 - kSwapBarBytes;
  for (p.epis = 2;; --p.epis) {
    const int left = room - p.epis * kSwapStageBytes;
    p.nx = std::min(left / p.x_bytes, kSwapMaxSlots);
    p.nr = 0;
    if (wkind) {
      // up to 4 operand slots that leave at least 4 raw tiles
      p.nx = std::max(2, std::min(4, (left - 4 * kSwapRawBytes) / p.x_bytes));
      p.nr = std::min((left - p.nx * p.x_bytes) / kSwapRawBytes, kSwapMaxSlots) & ~1;
    }
    if (p.epis == 1 || p.nx > 2) break;
  }
  p.smem = 1024 + p.nx * p.x_bytes + p.nr * kSwapRawBytes + p.epis * kSwapStageBytes +
           kSwapBarBytes;
  const double wb = 128.0 * 64 * (wkind == 0 ? 2 : 1) / p.mt;
  auto kb_cycles = [&](int active) {
    return std::max({p.groups * 4.0 * std::max(45.0, p.n / 2.0), p.rows * 128.0 / 64.0, wb / 30.0,
                     wb * active / 3400.0});
  };
  // the epilogue of a CTA's last tile, which nothing hides
  const double tail = 12.0 * p.rows;
  const int waves = (p.tiles + sms - 1) / sms;
  const double whole = (double)waves * p.num_kb * kb_cycles(std::min(p.tiles, sms)) + tail;
  // equal shares of at least 4 k-blocks; the partial tiles' way through L2 and one more launch
  const long long total = (long long)p.tiles * p.num_kb;
  const int ctas = (int)std::min<long long>(sms, std::max(1LL, total / 4));
  const double share =
      (double)((total + ctas - 1) / ctas) * kb_cycles(ctas) + 5000.0 + 10.0 * p.rows + tail;
  const size_t need = kCounterBytes + 2 * (size_t)ctas * p.rows * 128 * sizeof(float);
  if (share < whole && need <= ws_bytes) {
    p.ctas = ctas;
    p.unit = 1;
    p.ws_bytes = need;
    return share;
  }
  p.ctas = std::min(p.tiles, sms);
  p.unit = p.num_kb;
  p.ws_bytes = 0;
  return whole;
}

// As few tiles of activation rows as fit: what bounds the kernel above 256 rows is the activations'
// way from L2 (1024 x 5120 x 8192 in tiles of 352 rows 97 us, in tiles of 256 rows 117).
SwapPlan epi_swap_plan(int wkind, int M, int N, int K, int sms, size_t ws_bytes) {
  SwapPlan p{};
  epi_swap_cost(p, wkind, M, N, K, sms, ws_bytes, (M + kSwapMaxRows - 1) / kSwapMaxRows);
  return p;
}

template <int WQ, int LG>
cudaError_t launch_epi_swap_lg(const SwapPlan& p, const CUtensorMap (&m)[4], const SwapArgs& a,
                               cudaStream_t st) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::once_flag once[kMaxDevices];
  static cudaError_t attr_err[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(
        k_epi_swap<WQ, LG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynSmem);
  });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  return launch_ex(k_epi_swap<WQ, LG>, dim3(p.ctas), dim3(kSwapThreads<WQ>), p.smem, st, 1, m[0],
                   m[1], m[2], m[3], a);
}

template <int WQ>
cudaError_t launch_epi_swap(const Problem& pr, cudaStream_t st) {
  const SwapPlan p =
      epi_swap_plan(WQ, pr.M, pr.N, pr.K, current_sms(), pr.ws ? pr.ws_bytes : 0);
  // positions in the sequence of k-blocks are ints
  if (p.nx < 2 || (WQ && p.nr < 2) || p.ctas < 1 ||
      (long long)((pr.N + 127) / 128) * p.mt * p.num_kb > 0x7fffffff)
    return cudaErrorInvalidConfiguration;
  SwapArgs a{};
  a.M = pr.M;
  a.N = pr.N;
  a.num_kb = p.num_kb;
  a.tiles = p.tiles;
  a.mt = p.mt;
  a.rows = p.rows;
  a.n = p.n;
  a.groups = p.groups;
  a.nx = p.nx;
  a.nr = p.nr;
  a.x_bytes = p.x_bytes;
  a.bufs = p.bufs;
  a.epis = p.epis;
  a.unit = p.unit;
  a.C = static_cast<__half*>(pr.C);
  a.ldc = pr.ldc;
  // behind the arrival counters that other users of the workspace keep at its start
  if (p.ws_bytes) a.part = reinterpret_cast<float*>(static_cast<char*>(pr.ws) + kCounterBytes);
  a.scale = static_cast<const __half*>(pr.scale);
  a.group_size = pr.group > 0 ? pr.group : 64;
  a.epi = pr.epi;
  CUtensorMap m[4];
  std::memset(m, 0, sizeof(m));
  const auto F16 = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const auto U8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const auto SW128 = CU_TENSOR_MAP_SWIZZLE_128B, PLAIN = CU_TENSOR_MAP_SWIZZLE_NONE;
  bool ok = WQ ? make_map(&m[0], pr.W, U8, 1, pr.K, pr.N, pr.ldw, 64, 128, PLAIN)
               : make_map(&m[0], pr.W, F16, 2, pr.K, pr.N, pr.ldw, 64, 128, SW128);
  ok &= make_map(&m[1], pr.A, F16, 2, pr.K, pr.M, pr.lda, 64, p.n, SW128);
  if (WQ == kWUint8Group) {
    const uint64_t ng = (uint64_t)(pr.K / pr.group);
    ok &= make_map(&m[2], pr.scale, F16, 2, pr.N, ng, pr.N, 128, 1, PLAIN);
    ok &= make_map(&m[3], pr.zero, U8, 1, pr.N, ng, pr.N, 128, 1, PLAIN);
  }
  if (!ok) return cudaErrorInvalidValue;
  const cudaError_t e = WQ && p.nx % 2 == 0 ? launch_epi_swap_lg<WQ, (WQ ? 2 : 1)>(p, m, a, st)
                                            : launch_epi_swap_lg<WQ, 1>(p, m, a, st);
  if (e != cudaSuccess || !p.ws_bytes) return e;
  return launch_ex(k_swap_finish<WQ>, dim3(p.tiles, p.rows / 16), dim3(256), 0, st, 1, a,
                   p.ctas);
}

}  // namespace
}  // namespace tempo_sm100
