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
// Split: CTA b of G owns the rows [N b / G, N (b + 1) / G) -- every SM streams the same number
// of bytes to one row -- and its warps split K, warp w taking steps w, w + 8, ...; the partial
// sums of the 8 warps meet in shared memory and are added in warp order (deterministic).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace tempo_sm100 {

constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = 32 * kStreamWarps;
constexpr int kStreamMaxM = 16;

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
__device__ __forceinline__ void stream_unpack(uint4 x, __half2 zb, uint32_t (&h)[8]) {
  if (WQ == kWFp16) {
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

// Whether a step's activation chunks are fetched with its weights (their latency then hides under
// the steps in flight) or only when the step is used (more than 8 registers per step in flight
// would cost the weight stream more than it gains; other warps hide the L1 / L2 latency).
template <int WQ, int MG>
constexpr bool kStreamPreB = MG * StreamStep<WQ>::NB <= 8;

// One step's operands of a warp: RT row tiles of 16 weight rows and MG groups of 8 activation
// rows.
template <int WQ, int MG, int RT>
struct StreamStage {
  uint4 xa[RT], xb[RT];
  uint32_t b[kStreamPreB<WQ, MG> ? MG : 1][StreamStep<WQ>::NB];
  // group-wise scale and zero point of row (lane % 16) of each tile; the other rows' by shuffle
  unsigned short s[WQ == kWUint8Group ? RT : 1];
  uint8_t z[WQ == kWUint8Group ? RT : 1];
};

// Steps in flight per warp: what 128 registers (two CTAs of 8 warps per SM) leave beside the
// accumulators and the operands in use.
template <int WQ, int MG, int RT>
__host__ __device__ constexpr int stream_depth() {
  const int used = kStreamPreB<WQ, MG> ? 34 : 28 + RT * (WQ ? 16 : 8);
  const int stage = RT * (WQ == kWUint8Group ? 10 : 8) +
                    (kStreamPreB<WQ, MG> ? MG * StreamStep<WQ>::NB : 0);
  const int d = (128 - used - 4 * RT * MG) / stage;
  return d < 1 ? 1 : d > 4 ? 4 : d;
}

// acc += (weights of row tile) x (activation chunk b), one row tile and group
template <int WQ>
__device__ __forceinline__ void stream_mma_one(const uint32_t (&ha)[8], const uint32_t (&hb)[8],
                                               const uint32_t (&b)[StreamStep<WQ>::NB],
                                               float fa, float fb, float (&acc)[4]) {
  using S = StreamStep<WQ>;
  if (WQ == kWUint8Group) {
    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < S::NMMA; ++j)
      mma_16816(d, ha[2 * j], hb[2 * j], ha[2 * j + 1], hb[2 * j + 1], b[2 * j], b[2 * j + 1]);
    acc[0] = fmaf(d[0], fa, acc[0]);
    acc[1] = fmaf(d[1], fa, acc[1]);
    acc[2] = fmaf(d[2], fb, acc[2]);
    acc[3] = fmaf(d[3], fb, acc[3]);
  } else {
#pragma unroll
    for (int j = 0; j < S::NMMA; ++j)
      mma_16816(acc, ha[2 * j], hb[2 * j], ha[2 * j + 1], hb[2 * j + 1], b[2 * j], b[2 * j + 1]);
  }
}

// acc += W-step x A-step.  load_b(mg, regs) fetches the activation chunk of a group (only called
// where the stage does not hold it); live(mg): whether the group has any row (warp-uniform).
template <int WQ, int MG, int RT, typename LoadB, typename Live>
__device__ __forceinline__ void stream_mma(const StreamStage<WQ, MG, RT>& s,
                                           float (&acc)[RT][MG][4], LoadB load_b, Live live) {
  using S = StreamStep<WQ>;
  const int g = (threadIdx.x & 31) >> 2;
  auto unpack = [&](int rt, uint32_t (&ha)[8], uint32_t (&hb)[8], float& fa, float& fb) {
    __half2 za = __float2half2_rn(0.f), zb = za;
    if (WQ == kWUint8Group) {
      // scale and zero point of one row in one word
      const unsigned sz = (unsigned)s.s[rt] << 16 | s.z[rt];
      const unsigned a = __shfl_sync(0xffffffffu, sz, g), b = __shfl_sync(0xffffffffu, sz, g + 8);
      za = zero_bias((uint8_t)a);
      zb = zero_bias((uint8_t)b);
      fa = __half2float(__ushort_as_half((unsigned short)(a >> 16)));
      fb = __half2float(__ushort_as_half((unsigned short)(b >> 16)));
    }
    stream_unpack<WQ>(s.xa[rt], za, ha);
    stream_unpack<WQ>(s.xb[rt], zb, hb);
  };
  if constexpr (kStreamPreB<WQ, MG>) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      uint32_t ha[8], hb[8];
      float fa = 1.f, fb = 1.f;
      unpack(rt, ha, hb, fa, fb);
#pragma unroll
      for (int mg = 0; mg < MG; ++mg)
        if (live(mg))
          stream_mma_one<WQ>(ha, hb, s.b[mg], fa, fb, acc[rt][mg]);
    }
  } else {
    uint32_t ha[RT][8], hb[RT][8];
    float fa[RT], fb[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) unpack(rt, ha[rt], hb[rt], fa[rt], fb[rt]);
#pragma unroll
    for (int mg = 0; mg < MG; ++mg) {
      if (!live(mg)) continue;
      uint32_t b[S::NB];
      load_b(mg, b);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        stream_mma_one<WQ>(ha[rt], hb[rt], b, fa[rt], fb[rt], acc[rt][mg]);
    }
  }
}

template <int WQ, int MG, int RT>
__global__ void __launch_bounds__(kStreamThreads, 2)
    k_stream_linear(const __half* __restrict__ A, const uint8_t* __restrict__ W,
                    const __half* __restrict__ scale, const uint8_t* __restrict__ zero, __half* C,
                    const EpiArgs epi, int M, int N, int K, long long lda, long long ldw,
                    long long ldc, int group) {
  using S = StreamStep<WQ>;
  constexpr int U = stream_depth<WQ, MG, RT>();
  __shared__ float4 red[kStreamWarps][RT][MG][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  const int lo = (int)((long long)N * blockIdx.x / gridDim.x);
  const int hi = (int)((long long)N * (blockIdx.x + 1) / gridDim.x);
  const int nsteps = (K + S::STEP - 1) / S::STEP;
  const int npieces = (hi - lo + 16 * RT - 1) / (16 * RT);
  for (int pc = 0; pc < npieces; ++pc) {
    const int n0 = lo + (hi - lo) * pc / npieces;
    const int n1 = lo + (hi - lo) * (pc + 1) / npieces;
    float acc[RT][MG][4] = {};
    StreamStage<WQ, MG, RT> st[U];
    auto load_b = [&](int step, int mg, uint32_t (&b)[S::NB]) {
      const int k0 = step * S::STEP + t * S::KC;
      const int m = mg * 8 + g;
#pragma unroll
      for (int q = 0; q < S::KC / 8; ++q) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (k0 < K && m < M) v = __ldg(reinterpret_cast<const uint4*>(A + m * lda + k0) + q);
        b[4 * q] = v.x;
        b[4 * q + 1] = v.y;
        b[4 * q + 2] = v.z;
        b[4 * q + 3] = v.w;
      }
    };
    auto load = [&](StreamStage<WQ, MG, RT>& s, int step) {
      const int k0 = step * S::STEP + t * S::KC;
      const bool ok = step < nsteps && k0 < K;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int ra = n0 + rt * 16 + g, rb = ra + 8;
        s.xa[rt] = s.xb[rt] = make_uint4(0u, 0u, 0u, 0u);
        if (ok && ra < n1) s.xa[rt] = ld_stream(W + ((long long)ra * ldw + k0) * S::ESZ);
        if (ok && rb < n1) s.xb[rt] = ld_stream(W + ((long long)rb * ldw + k0) * S::ESZ);
        if (WQ == kWUint8Group) {  // a step's 64 k lie in one group (group % 64 == 0)
          const int r = n0 + rt * 16 + (lane & 15);
          s.s[rt] = 0;
          s.z[rt] = 0;
          if (ok && r < n1) {
            const long long gi = (long long)(k0 / group) * N + r;
            s.s[rt] = __ldg(reinterpret_cast<const unsigned short*>(scale) + gi);
            s.z[rt] = __ldg(zero + gi);
          }
        }
      }
      if constexpr (kStreamPreB<WQ, MG>) {
#pragma unroll
        for (int mg = 0; mg < MG; ++mg) load_b(step, mg, s.b[mg]);
      }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) load(st[u], warp + u * kStreamWarps);
    for (int step = warp; step < nsteps;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (step < nsteps) {
          stream_mma<WQ, MG, RT>(
              st[u], acc, [&](int mg, uint32_t(&b)[S::NB]) { load_b(step, mg, b); },
              [](int) { return true; });
          load(st[u], step + U * kStreamWarps);
        }
        step += kStreamWarps;
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int mg = 0; mg < MG; ++mg)
        red[warp][rt][mg][lane] =
            make_float4(acc[rt][mg][0], acc[rt][mg][1], acc[rt][mg][2], acc[rt][mg][3]);
    __syncthreads();
    for (int i = tid; i < RT * MG * 32; i += kStreamThreads) {
      const int l = i & 31, mg = (i >> 5) % MG, rt = (i >> 5) / MG;
      float4 v = red[0][rt][mg][l];
#pragma unroll
      for (int w = 1; w < kStreamWarps; ++w) {
        const float4 x = red[w][rt][mg][l];
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + rt * 16 + (l >> 2) + (j >= 2 ? 8 : 0);
        const int m = mg * 8 + 2 * (l & 3) + (j & 1);
        if (n >= n1 || m >= M) continue;
        const float sc = WQ == kWInt8PerChannel ? __half2float(__ldg(scale + n)) : 1.f;
        const float b = epi.bias ? __half2float(__ldg(epi.bias + n)) : 0.f;
        C[m * ldc + n] = __float2half_rn(epi_one(epi, o[j] * sc, b, m, n));
      }
    }
    __syncthreads();
  }
}

namespace {

template <int WQ, int MG, int RT>
cudaError_t launch_stream_rt(const Problem& pr, int grid, cudaStream_t st) {
  return launch_ex(k_stream_linear<WQ, MG, RT>, dim3(grid), dim3(kStreamThreads), 0, st, 1,
                   static_cast<const __half*>(pr.A), static_cast<const uint8_t*>(pr.W),
                   static_cast<const __half*>(pr.scale), static_cast<const uint8_t*>(pr.zero),
                   static_cast<__half*>(pr.C), pr.epi, pr.M, pr.N, pr.K, (long long)pr.lda,
                   (long long)pr.ldw, (long long)pr.ldc, pr.group > 0 ? pr.group : 1);
}

template <int WQ, int MG>
cudaError_t launch_stream_mg(const Problem& pr, cudaStream_t st) {
  const int sms = std::max(1, current_sms());
  // two CTAs per SM (one's reduction under the other's stream), at least 8 rows each
  const int grid = std::min(2 * sms, (pr.N + 7) / 8);
  const int rows = (pr.N + grid - 1) / grid;
  if (rows <= 16) return launch_stream_rt<WQ, MG, 1>(pr, grid, st);
  // four tiles only where the activations of a step ride with its weights (registers)
  if (rows <= 32 || !kStreamPreB<WQ, MG>) return launch_stream_rt<WQ, MG, 2>(pr, grid, st);
  return launch_stream_rt<WQ, MG, kStreamPreB<WQ, MG> ? 4 : 2>(pr, grid, st);
}

// The epilogue product for M <= kStreamMaxM.
cudaError_t run_stream(const Problem& pr, cudaStream_t st) {
  if (pr.M < 1 || pr.M > kStreamMaxM) return cudaErrorInvalidConfiguration;
  const bool one = pr.M <= 8;
  switch (pr.wkind) {
    case kWFp16: return one ? launch_stream_mg<0, 1>(pr, st) : launch_stream_mg<0, 2>(pr, st);
    case kWInt8PerChannel:
      return one ? launch_stream_mg<1, 1>(pr, st) : launch_stream_mg<1, 2>(pr, st);
    case kWUint8Group:
      return one ? launch_stream_mg<2, 1>(pr, st) : launch_stream_mg<2, 2>(pr, st);
    default: return cudaErrorInvalidConfiguration;
  }
}

}  // namespace
}  // namespace tempo_sm100
