// Products with few activation rows: each weight byte is read from HBM once, used by every row,
// and never staged in shared memory.
//
//   y[m][n] = act(sum_k A[m][k] W[n][k] * s + bias[n]) + res[m][n],  M <= 16
//
// What bounds it is the weight stream (N K bytes or 2 N K bytes against 2 M K + 2 M N), so the
// arithmetic has to cost nothing beside it: the products run on the warp tensor-core instruction
// (m16n8k16, fp16 inputs, fp32 accumulators) with 16 weight rows as its M side and 8 activation
// rows as its N side, operands straight from the registers the loads fill.  Sums are fp32
// throughout; 8-bit weights enter as exact integers (q, or q - z) and their scale multiplies the
// fp32 sum (per group of k, or per channel at the end), so no weight is rounded.
//
// Lane (g, t) = (lane / 4, lane % 4) holds the 16-byte chunk t of a step of 4 chunks of rows g
// and g + 8.  Lanes with equal t hold equal k ranges, so taking a chunk's k values in storage
// order as the MMA's k slots is the same permutation for both operands (slots 2t, 2t+1, 2t+8,
// 2t+9 of MMA j <-> values 4j .. 4j+3 of chunk t) and the sums are unchanged.
//
// Split: one CTA per SM; CTA b of G owns the rows [N b / G, N (b + 1) / G) -- every SM streams the
// same number of bytes to one row -- and its NW warps split K, warp w taking steps w, w + NW, ...;
// the partial sums of the warps meet in shared memory and are added in warp order (deterministic).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "stream.h"
#ifndef LIN_NW
#define LIN_NW 16
#define GU_NW 16
#define GU_RT 2
#define DN_NW 16
#define DN_NW2 8
#endif

namespace tempo_sm100 {

template <int WQ>
struct StreamStep {
  static constexpr int ESZ = WQ ? 1 : 2;   // weight bytes per element
  static constexpr int KC = 16 / ESZ;      // k of a 16-byte chunk
  static constexpr int STEP = 4 * KC;      // k a warp covers per step
  static constexpr int NMMA = KC / 4;      // MMAs per step and row tile
  static constexpr int NB = KC / 2;        // 32-bit registers of one activation chunk
};

// The exact fp16 values of a chunk in storage order: fp16 weights as they are, int8 q, or
// uint8 q - z with zb = (1024 + z) in both halves.
template <int WQ>
__device__ __forceinline__ void stream_unpack(uint4 x, __half2 zb,
                                              uint32_t (&h)[StreamStep<WQ>::NB]) {
  if constexpr (WQ == kWFp16) {
    h[0] = x.x;
    h[1] = x.y;
    h[2] = x.z;
    h[3] = x.w;
  } else {
    const uint32_t flip = WQ == kWInt8PerChannel ? 0x80808080u : 0u;
    const __half2 bias =
        WQ == kWInt8PerChannel ? __half2half2(__ushort_as_half(0x6480)) : zb;  // 1024 + 128, or z
    __half2 v[8];
    u8x4_to_h2x2_biased(x.x ^ flip, v[0], v[1]);
    u8x4_to_h2x2_biased(x.y ^ flip, v[2], v[3]);
    u8x4_to_h2x2_biased(x.z ^ flip, v[4], v[5]);
    u8x4_to_h2x2_biased(x.w ^ flip, v[6], v[7]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = __hsub2(v[i], bias);
      h[i] = *reinterpret_cast<const uint32_t*>(&v[i]);
    }
  }
}

__device__ __forceinline__ __half2 zero_bias(uint8_t z) {
  return __half2half2(__ushort_as_half((unsigned short)(0x6400u | z)));
}

// ---------------------------------------------------------------------------------------------
// A warp's FIFO of steps in shared memory, filled by 16-byte asynchronous copies.  A step holds
//   [RT][2][32 lanes][16 B]   weights: the lane's chunk of rows g and g + 8 of each row tile
//   [MG][BV blocks of 528 B]  activations: of column g of each group the 4 BV vectors of 16 bytes
//                             of the step, vector c in block c / 4 at 16 (4 g + c % 4); the lane's
//                             chunk is vectors BV t .. BV t + BV - 1
//   [RT][128 B]               group-wise weights: the tile's 16 scales and zero points
// Weights are read back by the lane that copied them.  The vectors of an activation chunk are not
// copied by one lane each -- two lanes' copies would then touch every 32-byte sector twice (int8
// M = 16: 77 MB of L2 traffic for 39) -- but four in a row by four lanes; blocks 16 bytes off a
// multiple of 128 keep the reads free of bank conflicts.  Registers hold one step, the FIFO S, so the bytes in flight do not depend on how long a
// step's arithmetic takes: with the steps in registers instead a kernel of 2 x 8 warps per SM
// had half the bytes in flight and waited for its activations in every step (o_proj M = 1, 31 MB:
// 12.9 us; one token through 4 fp16 experts: gate_up 35 us, down 48 us).
// ---------------------------------------------------------------------------------------------
template <int WQ, int MG, int RT, int BV>
struct StreamFifo {
  static constexpr int W_OFF = 0;
  static constexpr int B_OFF = RT * 1024;
  static constexpr int Z_OFF = B_OFF + (BV == 1 ? MG * 512 : MG * BV * 528);
  static constexpr int STAGE = Z_OFF + (WQ == kWUint8Group ? RT * 128 : 0);
  __host__ __device__ static constexpr int depth(int bytes_per_warp) {
    return bytes_per_warp / STAGE < 2 ? 2 : bytes_per_warp / STAGE > 8 ? 8 : bytes_per_warp / STAGE;
  }
};

// 16 bytes (zeros when off: then nothing is read at the address)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// Offset in a group's activations of vector c of column g.
template <int BV>
__device__ __forceinline__ int b_vec(int mg, int c, int g) {
  constexpr int BLK = BV == 1 ? 512 : 528;
  return (mg * BV + (c >> 2)) * BLK + (g * 4 + (c & 3)) * 16;
}

// The 16 scales and zero points of rows [r0, r0 + 16) of one group row: lanes 0-8 copy the scales
// two by two, lanes 16-20 the zero points four by four, from the aligned word below r0 on (rows of
// the group arrays are multiples of 16 long, so an aligned word that starts inside one ends there).
__device__ __forceinline__ void copy_group_row(uint32_t dst, const __half* scale,
                                               const uint8_t* zero, int r0, int n_rows, int lane,
                                               bool on) {
  if (lane < 9) {
    const int r = (r0 & ~1) + 2 * lane;
    cp_async4(dst + 4 * lane, scale + (on && r < n_rows ? r : 0), on && r < n_rows);
  } else if (lane >= 16 && lane < 21) {
    const int r = (r0 & ~3) + 4 * (lane - 16);
    cp_async4(dst + 64 + 4 * (lane - 16), zero + (on && r < n_rows ? r : 0), on && r < n_rows);
  }
}

__device__ __forceinline__ void read_group_row(uint32_t src, int r0, int row, float& s, __half2& zb) {
  unsigned short hs;
  unsigned z;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(hs) : "r"(src + 2 * ((r0 & 1) + row)) : "memory");
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(z) : "r"(src + 64 + (r0 & 3) + row) : "memory");
  s = __half2float(__ushort_as_half(hs));
  zb = zero_bias((uint8_t)z);
}

// A step's weights as MMA operands (and, group-wise, the scales of the lane's two rows).
template <int WQ, int RT>
struct StreamA {
  uint32_t a[RT][StreamStep<WQ>::NB], b[RT][StreamStep<WQ>::NB];
  float fa[WQ == kWUint8Group ? RT : 1], fb[WQ == kWUint8Group ? RT : 1];
};

template <int WQ, int RT>
__device__ __forceinline__ void stream_read_weights(StreamA<WQ, RT>& o, uint32_t stage,
                                                    uint32_t z_off, const int (&z_row)[RT],
                                                    int lane) {
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const uint4 xa = lds16(stage + rt * 1024 + lane * 16);
    const uint4 xb = lds16(stage + rt * 1024 + 512 + lane * 16);
    __half2 za = __float2half2_rn(0.f), zb = za;
    if constexpr (WQ == kWUint8Group) {
      read_group_row(stage + z_off + rt * 128, z_row[rt], lane >> 2, o.fa[rt], za);
      read_group_row(stage + z_off + rt * 128, z_row[rt], (lane >> 2) + 8, o.fb[rt], zb);
    }
    stream_unpack<WQ>(xa, za, o.a[rt]);
    stream_unpack<WQ>(xb, zb, o.b[rt]);
  }
}

// acc += weights of row tile rt x one activation chunk; group-wise the step's sum is scaled first.
// STEPS: the step's sum starts at zero and is added in fp32.  A tensor core truncates what it adds
// to a large accumulator; over a long K that shows in fp32 results (not in fp16 ones).
template <int WQ, int RT, bool STEPS = false>
__device__ __forceinline__ void stream_mma(const StreamA<WQ, RT>& w, int rt,
                                           const uint32_t (&b)[StreamStep<WQ>::NB],
                                           float (&acc)[4]) {
  using S = StreamStep<WQ>;
  if constexpr (WQ == kWUint8Group || STEPS) {
    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < S::NMMA; ++j)
      mma_16816(d, w.a[rt][2 * j], w.b[rt][2 * j], w.a[rt][2 * j + 1], w.b[rt][2 * j + 1],
                b[2 * j], b[2 * j + 1]);
    const float fa = WQ == kWUint8Group ? w.fa[WQ == kWUint8Group ? rt : 0] : 1.f;
    const float fb = WQ == kWUint8Group ? w.fb[WQ == kWUint8Group ? rt : 0] : 1.f;
    acc[0] = fmaf(d[0], fa, acc[0]);
    acc[1] = fmaf(d[1], fa, acc[1]);
    acc[2] = fmaf(d[2], fb, acc[2]);
    acc[3] = fmaf(d[3], fb, acc[3]);
  } else {
#pragma unroll
    for (int j = 0; j < S::NMMA; ++j)
      mma_16816(acc, w.a[rt][2 * j], w.b[rt][2 * j], w.a[rt][2 * j + 1], w.b[rt][2 * j + 1],
                b[2 * j], b[2 * j + 1]);
  }
}

// How many of nsteps steps warp w of NW has: w, w + NW, ...
template <int NW>
__device__ __forceinline__ int stream_count(int warp, int nsteps) {
  return nsteps > warp ? (nsteps - warp + NW - 1) / NW : 0;
}

// The work of one CTA as a sequence of pieces (RT row tiles x all of K), streamed without a pause
// between them: a warp's copies run S - 1 steps ahead of its arithmetic across piece boundaries,
// so the next piece is in flight while this one's partial sums are added.
//
// Job::ROTATE: CTA b starts at step nsteps b / G and wraps around, so that CTAs that run together
// read different k of the activations they share, not all of them the same few lines of L2 at once
// (int8 M = 16: 26 us without, 21 with).  The order of a sum then depends on its CTA.
//
// Job: Piece, first(Piece&), next(Piece&) -> whether there is (another) piece;
//      copy(piece, step, stage) issues one step; use_cols(piece) -> bit mg: the lane's column of
//      group mg exists; live(piece) -> bit mg: any column of group mg exists (warp-uniform);
//      z_rows(piece, r) the first row of each tile; finish(piece, rt, mg, float4) the whole sums
//      of (row g, columns 2t, 2t + 1) and (row g + 8, the same).
template <int WQ, int MG, int RT, int BV, int NW, int S, bool STEPS = false, class Job>
__device__ __forceinline__ void stream_run(Job& job, uint8_t* smem, float4* red, int nsteps) {
  using F = StreamFifo<WQ, MG, RT, BV>;
  using St = StreamStep<WQ>;
  static_assert(BV == St::NB / 4, "activations as they are");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t fifo = smem_u32(smem) + warp * S * F::STAGE;
  typename Job::Piece lp, up;
  const int n_mine = stream_count<NW>(warp, nsteps);
  bool more = n_mine > 0 && job.first(lp);
  const int rot = Job::ROTATE ? (int)((long long)nsteps * blockIdx.x / gridDim.x) : 0;
  int lstep = warp, lslot = 0;
  auto issue = [&]() {
    if (more) {
      const int step = lstep + rot;
      job.copy(lp, step < nsteps ? step : step - nsteps, fifo + lslot * F::STAGE);
      lstep += NW;
      if (lstep >= nsteps) {
        lstep = warp;
        more = job.next(lp);
      }
    }
    cp_async_commit();  // one group per step, empty at the end: the wait below counts groups
    lslot = lslot + 1 == S ? 0 : lslot + 1;
  };
#pragma unroll 1
  for (int i = 0; i < S - 1; ++i) issue();
  int slot = 0;
  for (bool on = job.first(up); on; on = job.next(up)) {
    float acc[RT][MG][4] = {};
    int z_row[RT];
    job.z_rows(up, z_row);
    const unsigned cols = job.use_cols(up), live = job.live(up);
#pragma unroll 1
    for (int j = 0; j < n_mine; ++j) {
      cp_async_wait<S - 2>();
      __syncwarp();  // every lane's copies of this step; every lane is done with the previous one
      issue();
      const uint32_t stage = fifo + slot * F::STAGE;
      StreamA<WQ, RT> w;
      stream_read_weights<WQ, RT>(w, stage, F::Z_OFF, z_row, lane);
#pragma unroll
      for (int mg = 0; mg < MG; ++mg) {
        if (MG > 1 && !((live >> mg) & 1u)) continue;
        uint32_t b[St::NB];
#pragma unroll
        for (int v = 0; v < BV; ++v) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if ((cols >> mg) & 1u)
            x = lds16(stage + F::B_OFF + b_vec<BV>(mg, BV * (lane & 3) + v, lane >> 2));
          b[4 * v] = x.x;
          b[4 * v + 1] = x.y;
          b[4 * v + 2] = x.z;
          b[4 * v + 3] = x.w;
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) stream_mma<WQ, RT, STEPS>(w, rt, b, acc[rt][mg]);
      }
      slot = slot + 1 == S ? 0 : slot + 1;
    }
    // the upper half of the warps hands its sums to the lower half, which adds its own
    constexpr int HALF = NW > 8 ? NW / 2 : NW;
    if (NW > 8 && warp >= HALF) {
#pragma unroll
      for (int i = 0; i < RT * MG; ++i) {
        const float(&v)[4] = acc[i / MG][i % MG];
        red[((warp - HALF) * RT * MG + i) * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    if (NW > 8) __syncthreads();
    if (warp < HALF) {
#pragma unroll
      for (int i = 0; i < RT * MG; ++i) {
        const float(&v)[4] = acc[i / MG][i % MG];
        float4& r = red[(warp * RT * MG + i) * 32 + lane];
        float4 o = make_float4(v[0], v[1], v[2], v[3]);
        if (NW > 8) {
          o.x += r.x;
          o.y += r.y;
          o.z += r.z;
          o.w += r.w;
        }
        r = o;
      }
    }
    __syncthreads();
    // whole warps take whole (rt, mg) groups
    for (int i = warp; i < RT * MG; i += NW) {
      float4 v = red[i * 32 + lane];
#pragma unroll
      for (int w = 1; w < HALF; ++w) {
        const float4 x = red[(w * RT * MG + i) * 32 + lane];
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      job.finish(up, i / MG, i % MG, v);
    }
    __syncthreads();
  }
  cp_async_wait<0>();
}

// A step's group without a division: ceil(2^31 / steps per group), then multiply and shift (exact
// while steps x steps per group < 2^31).
template <int WQ>
__device__ __forceinline__ unsigned group_magic(int group) {
  const unsigned n = WQ == kWUint8Group ? (unsigned)group / StreamStep<WQ>::STEP : 1u;
  return (0x80000000u + n - 1u) / n;
}
__device__ __forceinline__ int step_group(int step, unsigned magic) {
  return (int)(((unsigned long long)(unsigned)step * magic) >> 31);
}

template <int WQ, int MG, int RT>
struct LinearJob {
  using St = StreamStep<WQ>;
  using F = StreamFifo<WQ, MG, RT, St::NB / 4>;
  static constexpr bool ROTATE = true;
  const LinearArgs& a;
  int lo, hi, npieces, lane;
  unsigned per_group;  // group_magic
  const __half* x;     // vector lane % 4 of row lane / 4 of A
  struct Piece {
    int i, n0, n1;
    const uint8_t* w;  // this lane's chunk of row n0 + g at k = 0
  };
  __device__ __forceinline__ void bounds(Piece& p) const {
    p.n0 = lo + (hi - lo) * p.i / npieces;
    p.n1 = lo + (hi - lo) * (p.i + 1) / npieces;
    p.w = a.W + ((long long)(p.n0 + (lane >> 2)) * a.ldw + (lane & 3) * St::KC) * St::ESZ;
  }
  __device__ __forceinline__ bool first(Piece& p) const {
    p.i = 0;
    if (npieces) bounds(p);
    return npieces > 0;
  }
  __device__ __forceinline__ bool next(Piece& p) const {
    if (++p.i >= npieces) return false;
    bounds(p);
    return true;
  }
  __device__ __forceinline__ void copy(const Piece& p, int step, uint32_t stage) const {
    const int g = lane >> 2, kw = step * St::STEP;
    const bool ok = kw + (lane & 3) * St::KC < a.K;
    const uint8_t* w = p.w + (long long)kw * St::ESZ;
    const long long half = 8 * a.ldw * St::ESZ;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int ra = p.n0 + rt * 16 + g;
      const uint32_t d = stage + rt * 1024 + lane * 16;
      // rows past the piece are never stored: whatever their lanes hold stays in their own row
      if (ra < p.n1) cp_async16(d, w, ok);
      if (ra + 8 < p.n1) cp_async16(d + 512, w + half, ok);
      w += 2 * half;
      if (WQ == kWUint8Group) {
        const long long gi = (long long)step_group(step, per_group) * a.N;
        copy_group_row(stage + F::Z_OFF + rt * 128, a.scale + gi, a.zero + gi, p.n0 + rt * 16,
                       a.N, lane, true);
      }
    }
#pragma unroll
    for (int mg = 0; mg < MG; ++mg) {
      const int m = mg * 8 + g;
      if (m < a.M) {
        const __half* src = x + 8 * mg * a.lda + kw;
#pragma unroll
        for (int v = 0; v < St::NB / 4; ++v)
          cp_async16(stage + F::B_OFF + b_vec<St::NB / 4>(mg, 4 * v + (lane & 3), g), src + 32 * v,
                     kw + 32 * v + 8 * (lane & 3) < a.K);
      }
    }
  }
  __device__ __forceinline__ unsigned use_cols(const Piece&) const {
    unsigned c = 0;
#pragma unroll
    for (int mg = 0; mg < MG; ++mg) c |= (mg * 8 + (lane >> 2) < a.M ? 1u : 0u) << mg;
    return c;
  }
  __device__ __forceinline__ unsigned live(const Piece&) const { return (1u << MG) - 1u; }
  __device__ __forceinline__ void z_rows(const Piece& p, int (&r)[RT]) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) r[rt] = p.n0 + rt * 16;
  }
  __device__ __forceinline__ void finish(const Piece& p, int rt, int mg, float4 v) const {
    const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = p.n0 + rt * 16 + (lane >> 2) + (j >= 2 ? 8 : 0);
      const int m = mg * 8 + 2 * (lane & 3) + (j & 1);
      if (n >= p.n1 || m >= a.M) continue;
      const float sc = WQ == kWInt8PerChannel ? __half2float(__ldg(a.scale + n)) : 1.f;
      const float b = a.epi.bias ? __half2float(__ldg(a.epi.bias + n)) : 0.f;
      a.C[m * a.ldc + n] = __float2half_rn(epi_one(a.epi, o[j] * sc, b, m, n));
    }
  }
};

// NW warps share the shared memory left beside the partial sums.  16 of them: with 8 the unpacking
// of 8-bit weights ran at the speed of two warps per scheduler, not of the memory.
template <int WQ, int MG, int RT>
struct LinearCfg {
  static constexpr int NW = LIN_NW;
  static constexpr int BV = StreamStep<WQ>::NB / 4;
  using F = StreamFifo<WQ, MG, RT, BV>;
  static constexpr int RED = 8 * RT * MG * 512;
  static constexpr int S = F::depth((kMaxDynSmem - RED) / NW);
  static constexpr int FIFO = NW * S * F::STAGE;
  static constexpr int SMEM = FIFO + RED;
  static_assert(SMEM <= kMaxDynSmem, "shared memory");
};

template <int WQ, int MG, int RT>
__global__ void __launch_bounds__(32 * LinearCfg<WQ, MG, RT>::NW, 1)
    k_stream_linear(const LinearArgs a) {
  using C = LinearCfg<WQ, MG, RT>;
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  LinearJob<WQ, MG, RT> job{a};
  job.lo = (int)((long long)a.N * blockIdx.x / gridDim.x);
  job.hi = (int)((long long)a.N * (blockIdx.x + 1) / gridDim.x);
  job.npieces = (job.hi - job.lo + 16 * RT - 1) / (16 * RT);
  job.lane = threadIdx.x & 31;
  job.per_group = group_magic<WQ>(a.group);
  job.x = a.A + (job.lane >> 2) * a.lda + 8 * (job.lane & 3);
  stream_run<WQ, MG, RT, C::BV, C::NW, C::S>(
      job, smem, reinterpret_cast<float4*>(smem + C::FIFO),
      (a.K + StreamStep<WQ>::STEP - 1) / StreamStep<WQ>::STEP);
}

}  // namespace tempo_sm100
