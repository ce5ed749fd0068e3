// Products with few activation rows: each weight byte is read from HBM once and used by every row.
//
//   y[m][n] = act(sum_k A[m][k] W[n][k] * s + bias[n]) + res[m][n],  M <= 16
//
// What bounds it is the weight stream (N K bytes or 2 N K bytes against 2 M K + 2 M N), so the
// arithmetic has to cost nothing beside it: the products run on the warp tensor-core instruction
// (m16n8k16, fp16 inputs, fp32 accumulators) with 16 weight rows as its M side and 8 activation
// rows as its N side.  Every warp has a FIFO of its own in shared memory, filled by 16-byte
// asynchronous copies several steps ahead (bytes in flight are what HBM needs, and registers for
// them ran out), and reads its operands back as the registers of the MMA.  Sums are fp32
// throughout; 8-bit weights enter as exact integers and their scale multiplies the fp32 sum (per
// group of k, or per channel at the end), so no weight is rounded.
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

namespace tempo_sm100 {

template <int WQ>
struct StreamStep {
  static constexpr int ESZ = WQ ? 1 : 2;   // weight bytes per element
  static constexpr int KC = 16 / ESZ;      // k of a 16-byte chunk
  static constexpr int STEP = 4 * KC;      // k a warp covers per step
  static constexpr int NMMA = KC / 4;      // MMAs per step and row tile
  static constexpr int NB = KC / 2;        // 32-bit registers of one activation chunk
};

// The fp16 operands of a chunk in storage order: fp16 weights as they are; 8-bit weights as the
// integers they stand for, q or q - z (8 magnitude bits: exact in fp16).  A byte in the low half of
// 0x6400 is 1024 + u with u the unsigned byte (int8 q: u = q + 128); what has to go, `off` = 1152 or
// 1024 + z, is subtracted from every weight, two at a time.  (Left in and taken off the step's sum
// instead, by an MMA chain over the activations alone: the sum then passes through values 1152 / |q|
// times its own, of which a tensor core truncates the low bits, always in the same direction where
// the activations have one sign.  With weights of +-3 results were off by up to 25 times the bound
// that the exact operands keep, and no faster: one token through 8 int8 experts 69.9 us, so 68.9.)
template <int WQ>
__device__ __forceinline__ void stream_unpack(uint4 x, uint32_t (&h)[StreamStep<WQ>::NB],
                                              __half2 off) {
  if constexpr (WQ == kWFp16) {
    h[0] = x.x;
    h[1] = x.y;
    h[2] = x.z;
    h[3] = x.w;
  } else {
    const uint32_t flip = WQ == kWInt8PerChannel ? 0x80808080u : 0u;
    const uint32_t v[4] = {x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __byte_perm(v[i >> 1], 0x64646464u, i & 1 ? 0x5352 : 0x5150);
      const __half2 w = __hsub2(*reinterpret_cast<const __half2*>(&u), off);
      h[i] = *reinterpret_cast<const uint32_t*>(&w);
    }
  }
}

// d += a x b (not volatile: the compiler may move it)
__device__ __forceinline__ void stream_mma_16816(float (&d)[4], uint32_t a0, uint32_t a1,
                                                 uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// multiple of 128 keep the reads free of bank conflicts.  Registers hold one step, the FIFO S, so
// the bytes in flight do not depend on how long a step's arithmetic takes: with the steps in
// registers instead a kernel of 2 x 8 warps per SM had half the bytes in flight and waited for its
// activations in every step (o_proj M = 1, 31 MB: 12.9 us, so 6.6; one token through 4 fp16
// experts: gate_up 35 us, so 20, down 48, so 12).
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
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(const uint8_t* p) {
  return *reinterpret_cast<const uint4*>(p);
}

// Offset in a group's activations of vector c of column g.
template <int BV>
__device__ __forceinline__ int b_vec(int mg, int c, int g) {
  constexpr int BLK = BV == 1 ? 512 : 528;
  return (mg * BV + (c >> 2)) * BLK + (g * 4 + (c & 3)) * 16;
}

// The scales and zero points of a row tile's 16 rows in one group row, one 4-byte word per lane:
// scales two by two from lane 0, zero points four by four from lane kZeroLane, each from the aligned
// word at or below the first row on.  A lane's word of group j is at src + j * step.
constexpr int kZeroLane = 9;
struct GroupWord {
  const uint8_t* src;
  unsigned step;  // bytes from one group row to the next; 0: this lane has no word
};

// Rows [r0, r0 + 16) of arrays [groups][n_rows] (n_rows a multiple of 16, so that an aligned word
// that starts inside a group row ends there).
__device__ __forceinline__ GroupWord group_word(const __half* scale, const uint8_t* zero, int r0,
                                                int n_rows, int lane) {
  if (lane < kZeroLane) {
    const int r = (r0 & ~1) + 2 * lane;
    return {reinterpret_cast<const uint8_t*>(scale + r), r < n_rows ? 2u * n_rows : 0u};
  }
  const int r = (r0 & ~3) + 4 * (lane - kZeroLane);
  return {zero + r, lane < kZeroLane + 5 && r < n_rows ? (unsigned)n_rows : 0u};
}
__device__ __forceinline__ void copy_group_word(uint32_t dst, const GroupWord& w, int group,
                                                int lane) {
  if (w.step) cp_async4(dst + 4 * lane, w.src + (unsigned long long)w.step * (unsigned)group);
}

// Scale and 1024 + zero point of `row` of the tile.
__device__ __forceinline__ void read_group_row(const uint8_t* src, int r0, int row, float& s,
                                               __half2& off) {
  s = __half2float(*reinterpret_cast<const __half*>(src + 2 * ((r0 & 1) + row)));
  off = __half2half2(
      __ushort_as_half((unsigned short)(0x6400u | src[4 * kZeroLane + (r0 & 3) + row])));
}

// A step's weights as MMA operands (and, group-wise, the scales of the lane's two rows).
template <int WQ, int RT>
struct StreamA {
  uint32_t a[RT][StreamStep<WQ>::NB], b[RT][StreamStep<WQ>::NB];
  float fa[WQ == kWUint8Group ? RT : 1], fb[WQ == kWUint8Group ? RT : 1];
};

template <int WQ, int RT>
__device__ __forceinline__ void stream_read_weights(StreamA<WQ, RT>& o, const uint8_t* stage,
                                                    uint32_t z_off, const int (&z_row)[RT],
                                                    int lane) {
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const uint4 xa = lds16(stage + rt * 1024 + lane * 16);
    const uint4 xb = lds16(stage + rt * 1024 + 512 + lane * 16);
    __half2 za = __half2half2(__ushort_as_half(0x6480)), zb = za;  // 1152
    if constexpr (WQ == kWUint8Group) {
      read_group_row(stage + z_off + rt * 128, z_row[rt], lane >> 2, o.fa[rt], za);
      read_group_row(stage + z_off + rt * 128, z_row[rt], (lane >> 2) + 8, o.fb[rt], zb);
    }
    stream_unpack<WQ>(xa, o.a[rt], za);
    stream_unpack<WQ>(xb, o.b[rt], zb);
  }
}

// acc += weights of row tile rt x the step's activation chunks b (N of them: their values add up).
// The step's sum starts at zero and is added in fp32 (group-wise: times the scale), except (STEPS
// false) for fp16 weights: a tensor core truncates what it adds to a large accumulator, which over
// a long K shows in fp32 results, not in fp16 ones.
template <int WQ, int RT, bool STEPS, int N>
__device__ __forceinline__ void stream_mma(const StreamA<WQ, RT>& w, int rt,
                                           const uint32_t (&b)[N][StreamStep<WQ>::NB],
                                           float (&acc)[4]) {
  using S = StreamStep<WQ>;
  constexpr bool own = WQ != kWFp16 || STEPS;
  float step[4] = {};
  float(&d)[4] = own ? step : acc;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < S::NMMA; ++j)
      stream_mma_16816(d, w.a[rt][2 * j], w.b[rt][2 * j], w.a[rt][2 * j + 1], w.b[rt][2 * j + 1],
                       b[n][2 * j], b[n][2 * j + 1]);
  if constexpr (WQ == kWUint8Group) {
    acc[0] = fmaf(d[0], w.fa[rt], acc[0]);
    acc[1] = fmaf(d[1], w.fa[rt], acc[1]);
    acc[2] = fmaf(d[2], w.fb[rt], acc[2]);
    acc[3] = fmaf(d[3], w.fb[rt], acc[3]);
  } else if constexpr (own) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += d[i];
  }
}

// [lo, hi) of part `id` of n items in `count` parts of sizes that differ by at most one.
__device__ __forceinline__ void split_even(unsigned n, unsigned id, unsigned count, int& lo,
                                           int& hi) {
  const unsigned q = n / count, r = n - q * count;
  lo = (int)(id * q + min(id, r));
  hi = lo + (int)(q + (id < r ? 1u : 0u));
}

// Worker `id` of `count`: this warp is its `warp`-th of `warps`.
struct StreamWorker {
  int id, count, in_cta, warp, warps;
};
template <int NW>
__device__ __forceinline__ StreamWorker stream_worker(int ks) {
  const int w = threadIdx.x >> 5, sh = 31 - __clz(ks);  // ks divides NW, both powers of two
  const int per = NW >> sh;
  return {(int)blockIdx.x * per + (w >> sh), (int)gridDim.x * per, w >> sh, w & (ks - 1), ks};
}

// The work of one worker -- KS warps of a CTA -- as a sequence of pieces (RT row tiles x all of K),
// streamed without a pause between them: a warp's copies run S - 1 steps ahead of its arithmetic
// across piece boundaries, so the next piece is in flight while this one's partial sums are added.
// The warps of a worker split K (warp w: steps w, w + KS, ...); a CTA of NW warps has NW / KS
// workers, which share nothing and meet at barriers of their own.  Fewer warps to a worker: more
// steps to a piece, so less of its fixed cost (its sums' way through shared memory, its pointers);
// more: fewer rows needed to fill the row tiles.
//
// Job::ROTATE: worker b of G starts at step nsteps b / G and wraps around, so that workers that run
// together read different k of the activations they share, not all of them the same few lines of
// L2 at once (int8 M = 16: 26 us without, 21 with).  The order of a sum depends on its worker.
//
// Job: Piece, first(Piece&), next(Piece&) -> whether there is (another) piece;
//      copy(piece, step, stage) issues one step; live(piece) -> bit mg: any column of group mg
//      exists (warp-uniform);
//      z_rows(piece, r) the first row of each tile; finish(piece, rt, mg, float4) the whole sums
//      of (row g, columns 2t, 2t + 1) and (row g + 8, the same).
template <int WQ, int MG, int RT, int BV, int NW, int S, bool STEPS = false, class Job>
__device__ __forceinline__ void stream_run(Job& job, uint8_t* smem, float4* red_all, int nsteps,
                                           StreamWorker wk) {
  using F = StreamFifo<WQ, MG, RT, BV>;
  using St = StreamStep<WQ>;
  static_assert(BV == St::NB / 4, "activations as they are");
  const int lane = threadIdx.x & 31, warp = wk.warp, KS = wk.warps;
  const uint8_t* fifo_p = smem + (threadIdx.x >> 5) * S * F::STAGE;
  const uint32_t fifo = smem_u32(fifo_p);
  float4* red = red_all + wk.in_cta * KS * RT * MG * 32;
  typename Job::Piece lp, up;
  const int n_mine = nsteps > warp ? ((nsteps - 1 - warp) >> (31 - __clz(KS))) + 1 : 0;
  bool more = n_mine > 0 && job.first(lp);
  const int rot = Job::ROTATE ? (int)((unsigned)nsteps * (unsigned)wk.id / (unsigned)wk.count) : 0;
  int lstep = warp;
  auto issue = [&](int to) {  // the next step into slot `to`
    if (more) {
      const int step = lstep + rot;
      job.copy(lp, step < nsteps ? step : step - nsteps, fifo + to * F::STAGE);
      lstep += KS;
      if (lstep >= nsteps) {
        lstep = warp;
        more = job.next(lp);
      }
    }
    cp_async_commit();  // one group per step, empty at the end: the wait below counts groups
  };
#pragma unroll 1
  for (int i = 0; i < S - 1; ++i) issue(i);
  int slot = 0;
  for (bool on = job.first(up); on; on = job.next(up)) {
    float acc[RT][MG][4] = {};
    int z_row[RT];
    job.z_rows(up, z_row);
    const unsigned live = job.live(up);
#pragma unroll 1
    for (int j = 0; j < n_mine; ++j) {
      cp_async_wait<S - 2>();
      __syncwarp();  // every lane's copies of this step; every lane is done with the previous one
      issue(slot ? slot - 1 : S - 1);
      const uint8_t* stage = fifo_p + slot * F::STAGE;
      uint32_t b[MG][1][St::NB];
#pragma unroll
      for (int mg = 0; mg < MG; ++mg) {
        if (MG > 1 && !((live >> mg) & 1u)) continue;
#pragma unroll
        for (int v = 0; v < BV; ++v) {
          // a column that does not exist holds whatever the FIFO held: it stays in its column
          const uint4 x = lds16(stage + F::B_OFF + b_vec<BV>(mg, BV * (lane & 3) + v, lane >> 2));
          b[mg][0][4 * v] = x.x;
          b[mg][0][4 * v + 1] = x.y;
          b[mg][0][4 * v + 2] = x.z;
          b[mg][0][4 * v + 3] = x.w;
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {  // one tile's operands in registers at a time
        StreamA<WQ, 1> w;
        const int zr[1] = {z_row[rt]};
        stream_read_weights<WQ, 1>(w, stage + rt * 1024, F::Z_OFF + rt * 128 - rt * 1024, zr, lane);
#pragma unroll
        for (int mg = 0; mg < MG; ++mg)
          if (MG == 1 || ((live >> mg) & 1u)) stream_mma<WQ, 1, STEPS>(w, 0, b[mg], acc[rt][mg]);
      }
      slot = slot + 1 == S ? 0 : slot + 1;
    }
#pragma unroll
    for (int i = 0; i < RT * MG; ++i) {
      const float(&v)[4] = acc[i / MG][i % MG];
      red[(warp * RT * MG + i) * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
    }
    named_barrier_sync(1 + wk.in_cta, 32 * KS);
    // whole warps take whole (rt, mg) groups, and add the warps' sums in order
    for (int i = warp; i < RT * MG; i += KS) {
      float4 v = red[i * 32 + lane];
#pragma unroll 5
      for (int w = 1; w < KS; ++w) {
        const float4 x = red[(w * RT * MG + i) * 32 + lane];
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      job.finish(up, i / MG, i % MG, v);
    }
    named_barrier_sync(1 + wk.in_cta, 32 * KS);
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
    GroupWord z[WQ == kWUint8Group ? RT : 1];
  };
  __device__ __forceinline__ void bounds(Piece& p) const {
    split_even(hi - lo, p.i, npieces, p.n0, p.n1);
    p.n0 += lo;
    p.n1 += lo;
    p.w = a.W + ((long long)(p.n0 + (lane >> 2)) * a.ldw + (lane & 3) * St::KC) * St::ESZ;
    if (WQ == kWUint8Group) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        p.z[WQ == kWUint8Group ? rt : 0] =
            group_word(a.scale, a.zero, p.n0 + rt * 16, a.N, lane);
    }
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
      if (WQ == kWUint8Group)
        copy_group_word(stage + F::Z_OFF + rt * 128, p.z[WQ == kWUint8Group ? rt : 0],
                        step_group(step, per_group), lane);
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
  __device__ __forceinline__ unsigned live(const Piece&) const { return (1u << MG) - 1u; }
  __device__ __forceinline__ void z_rows(const Piece& p, int (&r)[RT]) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) r[rt] = p.n0 + rt * 16;
  }
  __device__ __forceinline__ void finish(const Piece& p, int rt, int mg, float4 v) const {
    const int n0 = p.n0 + rt * 16 + (lane >> 2), m0 = mg * 8 + 2 * (lane & 3);
    float f[4] = {v.x, v.y, v.z, v.w};  // (n0, m0), (n0, m0 + 1), (n0 + 8, m0), (n0 + 8, m0 + 1)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + 8 * h;
      if (n >= p.n1) continue;
      const float sc = WQ == kWInt8PerChannel ? __half2float(__ldg(a.scale + n)) : 1.f;
      const float b = a.epi.bias ? __half2float(__ldg(a.epi.bias + n)) : 0.f;
      f[2 * h] = f[2 * h] * sc + b;
      f[2 * h + 1] = f[2 * h + 1] * sc + b;
    }
    epi_act(f, a.epi.act);  // rows that do not exist too: once for all four
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 4 * (j & 2), m = m0 + (j & 1);
      if (n >= p.n1 || m >= a.M) continue;
      if (a.epi.res) f[j] += __half2float(a.epi.res[m * a.epi.ldr + n]);
      a.C[m * a.ldc + n] = __float2half_rn(f[j]);
    }
  }
};

// 16 warps share the shared memory left beside the partial sums: with 8 the unpacking of 8-bit
// weights ran at the speed of two warps per scheduler, not of the memory.
template <int WQ, int MG, int RT>
struct LinearCfg {
  static constexpr int NW = 16;
  static constexpr int BV = StreamStep<WQ>::NB / 4;
  using F = StreamFifo<WQ, MG, RT, BV>;
  static constexpr int RED = NW * RT * MG * 512;
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
  const StreamWorker wk = stream_worker<C::NW>(C::NW);
  LinearJob<WQ, MG, RT> job{a};
  split_even(a.N, wk.id, wk.count, job.lo, job.hi);
  job.npieces = (job.hi - job.lo + 16 * RT - 1) / (16 * RT);
  job.lane = threadIdx.x & 31;
  job.per_group = group_magic<WQ>(a.group);
  job.x = a.A + (job.lane >> 2) * a.lda + 8 * (job.lane & 3);
  stream_run<WQ, MG, RT, C::BV, C::NW, C::S>(
      job, smem, reinterpret_cast<float4*>(smem + C::FIFO),
      (a.K + StreamStep<WQ>::STEP - 1) / StreamStep<WQ>::STEP, wk);
}

}  // namespace tempo_sm100
