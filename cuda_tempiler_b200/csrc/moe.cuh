// A mixture-of-experts layer for a few tokens (T <= 32), three launches on one stream:
//
//   k_moe_route    logits x Wr^T + b, top-k of each token, softmax weights, and the plan: the
//                  experts that were reached (slots), each with the set of its tokens
//   k_moe_gate_up  h[r][i] = w_r * silu(gate_i(x_t)) * up_i(x_t) for every routed row r = (t, e)
//   k_moe_down     y[t][n] = res[t][n] + sum_e sum_i down_e[n][i] h[(t, e)][i]
//
// The bytes are the weights of the reached experts, read once each whatever the number of
// tokens; everything else is small.  The products are those of stream.cuh: weights through a FIFO
// per warp into the registers of warp MMAs, fp32 sums, 8-bit weights as exact integers.
//
// A slot is an expert with at most 16 of its tokens (an expert with more has several slots; the
// second one finds the weights in L2).  The columns of its MMAs are its tokens in ascending
// order, so an expert that two tokens chose costs one MMA per 16 x 16 weights however many tokens
// the call has.  k_moe_down keeps one fp32 sum per (warp, token, row) in shared memory over all
// slots: no atomics, no partial outputs, the same order of sums on every run, and an infinite
// weight of an expert reaches only the tokens that chose it.
//
// h is kept in fp32.  The down product needs fp16 operands, so each row of h is scaled by a
// power of two (its largest value to [2^14, 2^15)) and split into fp16 high and low parts: 22
// bits, against 11 for a single fp16, for one more MMA per step.
#pragma once

#include "stream.cuh"

namespace tempo_sm100 {

constexpr int kMoeMaxT = 32;
constexpr int kMoeMaxK = 16;
constexpr int kMoeMaxE = 512;
constexpr int kMoeMaxRows = kMoeMaxT * kMoeMaxK;
constexpr int kMoeCols = 16;  // tokens of a slot
constexpr int kRouteCluster = 16;
constexpr int kPlanThreads = 256;

// What the router tells the two products (in the caller's workspace; every call writes it whole).
struct MoePlan {
  int n_slots;                      // every slot has a token, so at most T * top_k
  int pad[3];
  int meta[kMoeMaxRows];            // slot -> expert (ascending) | number of its rows << 16
  int base[kMoeMaxRows];            // slot -> its first row
  unsigned char token[kMoeMaxRows]; // row -> token, ascending within an expert
  float weight[kMoeMaxRows];        // row -> routing weight
  unsigned amax[kMoeMaxRows];       // row -> bits of max |h| (k_moe_gate_up)
};

struct MoeArgs {
  const __half* x;
  long long ldx;
  int T, E, H, I;
  const uint8_t *wgu, *wd;          // [E][2I][H], [E][H][I]
  const __half *sgu, *sd;           // int8: [E][2I], [E][H]; uint8: [E][H/g][2I], [E][I/g][H]
  const uint8_t *zgu, *zd;
  int group, gu_block;
  MoePlan* plan;
  float* h;                         // [rows][I]
  const __half* res;
  long long ldr;
  __half* y;
  long long ldy;
};

// The plan from ids [T][k] and weights [T][k] in shared memory, by one CTA.  An id outside
// [0, E) names no expert; an id that a token names twice is one row with the sum of its weights.
__device__ void moe_build_plan(MoePlan* plan, const int* ids, const float* w, int T, int k, int E,
                               unsigned* emask, int* ebase) {
  const int tid = threadIdx.x, n = T * k;
  for (int e = tid; e < E; e += blockDim.x) emask[e] = 0u;
  __syncthreads();
  for (int i = tid; i < n; i += blockDim.x) {
    const int e = ids[i];
    if (e >= 0 && e < E) atomicOr(&emask[e], 1u << (i / k));
  }
  __syncthreads();
  if (tid < 32) {
    int slot = 0, row = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + tid;
      const unsigned m = e < E ? emask[e] : 0u;
      const int c = __popc(m);
      // rows and slots of the experts before this one, in one scan (rows < 2^16)
      const int mine = c | ((c + kMoeCols - 1) / kMoeCols) << 16;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += v;
      }
      const int excl = incl - mine;
      int b = row + (excl & 0xffff), s = slot + (excl >> 16);
      if (e < E) ebase[e] = b;
      for (unsigned left = m; left; ++s, b += kMoeCols) {
        unsigned rest = left;
        for (int i = 0; i < kMoeCols && rest; ++i) rest &= rest - 1u;
        plan->meta[s] = e | __popc(left & ~rest) << 16;
        plan->base[s] = b;
        left = rest;
      }
      const int all = __shfl_sync(0xffffffffu, incl, 31);
      slot += all >> 16;
      row += all & 0xffff;
    }
    if (tid == 0) plan->n_slots = slot;
  }
  __syncthreads();
  for (int i = tid; i < n; i += blockDim.x) {
    const int t = i / k, e = ids[i];
    plan->amax[i] = 0u;
    if (e < 0 || e >= E) continue;
    float sum = 0.f;
    bool first = true;
    for (int j = t * k; j < (t + 1) * k; ++j) {
      if (ids[j] != e) continue;
      if (j < i) first = false;
      sum += w[j];
    }
    if (!first) continue;
    const int row = ebase[e] + __popc(emask[e] & ((1u << t) - 1u));
    plan->weight[row] = sum;
    plan->token[row] = (unsigned char)t;
  }
}

// Order-preserving integer key of a logit; NaN below everything, -0 equal to +0.
__device__ __forceinline__ unsigned logit_key(float x) {
  if (x != x) return 0u;
  const unsigned u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Top-k of one token's E logits by one warp: lane l holds experts l, l + 32, ...  The largest
// first, equal ones by index; out-of-range k never happens (k <= E, checked by the host).
// Weights: softmax over the chosen (normalize) or over all experts.  A NaN logit makes every
// weight of the token NaN, as the softmax over all experts is; the ids stay valid.  Lane j < k
// returns the j-th choice.
__device__ void moe_topk(const float* logits, int E, int k, bool normalize, int& id, float& w) {
  constexpr int P = kMoeMaxE / 32;
  const int lane = threadIdx.x & 31;
  unsigned key[P];
  bool nan_any = false;
  float mx = -INFINITY;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    if (32 * p >= E) break;
    const int e = lane + 32 * p;
    key[p] = 0u;
    if (e < E) {
      const float x = logits[e];
      key[p] = logit_key(x);
      nan_any |= x != x;
      mx = fmaxf(mx, x);
    }
  }
  const bool bad = __any_sync(0xffffffffu, nan_any);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float total = 0.f;
  if (!normalize) {
    for (int e = lane; e < E; e += 32) total += expf(logits[e] - mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  unsigned taken = 0u;
  int mine_id = 0;
  for (int j = 0; j < k; ++j) {
    unsigned best = 0u;
    int bp = -1;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (32 * p >= E) break;
      if (lane + 32 * p < E && !((taken >> p) & 1u) && (bp < 0 || key[p] > best)) {
        best = key[p];
        bp = p;
      }
    }
    const unsigned top = __reduce_max_sync(0xffffffffu, bp < 0 ? 0u : best);
    const unsigned cand = (bp >= 0 && best == top) ? (unsigned)(lane + 32 * bp) : 0xffffffffu;
    const unsigned e = __reduce_min_sync(0xffffffffu, cand);
    if ((e & 31u) == (unsigned)lane) taken |= 1u << (e >> 5);
    if (lane == j) mine_id = (int)e;
  }
  const float mine = lane < k ? expf(logits[mine_id] - mx) : 0.f;
  if (normalize) {
    total = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  id = mine_id;
  w = bad ? __int_as_float(0x7fffffff) : mine / total;
}

struct RouteArgs {
  const __half* x;
  long long ldx;
  const __half* wr;
  long long ldw;
  const __half* bias;
  int T, E, H, k, normalize;
  int* ids;
  float* weights;
  MoePlan* plan;
};

// The experts [lo, hi) times the nt tokens, 16 experts at a time.
template <int MG>
struct RouteJob {
  using St = StreamStep<kWFp16>;
  using F = StreamFifo<kWFp16, MG, 1, 1>;
  static constexpr bool ROTATE = false;  // equal router rows have equal logits
  const RouteArgs& a;
  int lo, hi, nt, lane;
  float* logits;  // [tokens this CTA owns][kMoeMaxE], the same place in every CTA of the cluster
  struct Piece {
    int n0;
    const __half* w;
  };
  __device__ __forceinline__ bool at(Piece& p, int n0) const {
    p.n0 = n0;
    p.w = a.wr + (n0 + (lane >> 2)) * a.ldw + 8 * (lane & 3);
    return n0 < hi;
  }
  __device__ __forceinline__ bool first(Piece& p) const { return at(p, lo); }
  __device__ __forceinline__ bool next(Piece& p) const { return at(p, p.n0 + 16); }
  __device__ __forceinline__ void copy(const Piece& p, int step, uint32_t stage) const {
    const int g = lane >> 2, kw = step * St::STEP;
    const bool ok = kw + 8 * (lane & 3) < a.H;
    if (p.n0 + g < hi) cp_async16(stage + lane * 16, p.w + kw, ok);
    if (p.n0 + g + 8 < hi) cp_async16(stage + 512 + lane * 16, p.w + 8 * a.ldw + kw, ok);
#pragma unroll
    for (int mg = 0; mg < MG; ++mg) {
      const int m = mg * 8 + g;
      if (m < nt)
        cp_async16(stage + F::B_OFF + mg * 512 + lane * 16,
                   a.x + m * a.ldx + kw + 8 * (lane & 3), ok);
    }
  }
  __device__ __forceinline__ unsigned live(const Piece&) const {
    return (1u << ((nt + 7) / 8)) - 1u;
  }
  __device__ __forceinline__ void z_rows(const Piece&, int (&r)[1]) const { r[0] = 0; }
  __device__ __forceinline__ void finish(const Piece& p, int, int mg, float4 v) const {
    const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = p.n0 + (lane >> 2) + (j >= 2 ? 8 : 0);
      const int m = mg * 8 + 2 * (lane & 3) + (j & 1);
      if (e >= hi || m >= nt) continue;
      const float z = o[j] + (a.bias ? __half2float(__ldg(a.bias + e)) : 0.f);
      // token m's logits go to the CTA that picks its experts
      st_dsmem_f32(mapa_shared(smem_u32(logits + (m / kRouteCluster) * kMoeMaxE + e),
                               m % kRouteCluster), z);
    }
  }
};

template <int MG>
struct RouteCfg {
  static constexpr int NW = 16;
  static constexpr int TOK = MG * 8;  // tokens of a cluster
  static constexpr int OWN = (TOK + kRouteCluster - 1) / kRouteCluster;
  using F = StreamFifo<kWFp16, MG, 1, 1>;
  static constexpr int RED = NW * MG * 512;
  static constexpr int REST = OWN * kMoeMaxE * 4 + 2 * kMoeMaxRows * 4 + 2 * kMoeMaxE * 4;
  static constexpr int S = F::depth((kMaxDynSmem - RED - REST) / NW);
  static constexpr int FIFO = NW * S * F::STAGE;
  static constexpr int SMEM = FIFO + RED + REST;
};

// One cluster of 16 CTAs routes up to 8 or 32 tokens: CTA r multiplies them with the experts
// [E r / 16, E (r + 1) / 16) -- its share of the router's weights is in flight at once -- hands
// each token's logits to the CTA that owns the token (t % 16) through distributed shared memory,
// and picks the top-k of its own tokens, a warp each.  With a plan wanted
// CTA 0 collects the choices and builds it.
template <int MG>
__global__ void __launch_bounds__(32 * RouteCfg<MG>::NW, 1) k_moe_route(const RouteArgs a) {
  using C = RouteCfg<MG>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* logits = reinterpret_cast<float*>(smem + C::FIFO + C::RED);
  int* s_ids = reinterpret_cast<int*>(logits + C::OWN * kMoeMaxE);  // CTA 0: everyone's choices
  float* s_w = reinterpret_cast<float*>(s_ids + kMoeMaxRows);
  unsigned* emask = reinterpret_cast<unsigned*>(s_w + kMoeMaxRows);
  int* ebase = reinterpret_cast<int*>(emask + kMoeMaxE);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = (int)cluster_ctarank();
  const int nt = a.T;
  cluster_sync();  // every CTA of the cluster runs before its shared memory is written
  pdl_wait();
  pdl_launch_dependents();
  RouteJob<MG> job{a, a.E * rank / kRouteCluster, a.E * (rank + 1) / kRouteCluster, nt, lane,
                   logits};
  stream_run<kWFp16, MG, 1, 1, C::NW, C::S, true>(
      job, smem, reinterpret_cast<float4*>(smem + C::FIFO),
      (a.H + StreamStep<kWFp16>::STEP - 1) / StreamStep<kWFp16>::STEP, stream_worker<C::NW>(C::NW));
  cluster_sync();
  for (int q = warp; q < C::OWN; q += C::NW) {
    const int m = q * kRouteCluster + rank;
    if (m >= nt) continue;
    int id;
    float w;
    moe_topk(logits + q * kMoeMaxE, a.E, a.k, a.normalize != 0, id, w);
    if (lane >= a.k) continue;
    const int i = m * a.k + lane;
    if (a.plan) {
      st_dsmem_f32(mapa_shared(smem_u32(s_ids + i), 0), __int_as_float(id));
      st_dsmem_f32(mapa_shared(smem_u32(s_w + i), 0), w);
    }
    a.ids[i] = id;
    a.weights[i] = w;
  }
  if (!a.plan) return;
  cluster_sync();
  if (rank == 0) moe_build_plan(a.plan, s_ids, s_w, a.T, a.k, a.E, emask, ebase);
}

// More than 32 tokens: a cluster of 8 CTAs routes 32 of them.  CTA r takes an eighth of k for all
// experts, 128 at a time: warp (p, q) has 32 of the experts and every other 32-wide block of the
// CTA's k range.  Its router weights go from L2 straight into the registers of the warp MMAs (no
// other warp of the CTA wants them), 16 vectors in flight per thread; the tokens' part of k is in
// shared memory.  The two sums of a logit are added, sent to the CTA that owns the token (t % 8)
// and added there in rank order.  Every expert's sum has the same order, so equal router rows have
// equal logits.  Two CTAs fit an SM for up to 200 experts.
//
// What bounds it is the chain of latencies of one cluster, not the 6.5 MB of 509 tokens, E = 128,
// H = 5120: 14.8 us (with 20 vectors in flight, some of them spilled, 16.3; E = 256, H = 7168 35 and
// 41); with 16 warps that split k in four and one CTA per SM 21.5 (the GPU then holds 13 or 14
// clusters at a time); by clusters of 16 as above, 32 tokens each, 30.
constexpr int kManyTok = 32;
constexpr int kManyCluster = 8;
constexpr int kManySplit = 2;                        // warps that share a CTA's k
constexpr int kManyThreads = 128 * kManySplit;
constexpr int kManyRound = 4;                        // blocks of k a warp holds at once (5: spills)
constexpr int kManyBlocks = 20;                      // 32-wide blocks of k in shared memory
constexpr int kManyRow = kManyBlocks * 64;           // bytes of a token's row there
constexpr int kManyOwn = kManyTok / kManyCluster;
constexpr int kManyRed = (kManySplit - 1) * 4 * 8 * 512;
__host__ __device__ constexpr int many_smem(int E) {
  return kManyTok * kManyRow + kManyRed + kManyCluster * kManyOwn * E * 4;
}

__global__ void __launch_bounds__(kManyThreads, 2) k_moe_route_many(const RouteArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  const uint8_t* xs = smem;
  float4* red = reinterpret_cast<float4*>(smem + kManyTok * kManyRow);
  // [rank][own token][expert], written by the CTAs of the cluster
  float* recv = reinterpret_cast<float*>(smem + kManyTok * kManyRow + kManyRed);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rp = warp / kManySplit, ks = warp % kManySplit;
  const int rank = (int)cluster_ctarank();
  const long long t0 = (long long)(blockIdx.x / kManyCluster) * kManyTok;
  const int nt = (int)min((long long)kManyTok, a.T - t0);
  const int n32 = (a.H + 31) / 32;
  const int b0 = n32 * rank / kManyCluster, b1 = n32 * (rank + 1) / kManyCluster;
  cluster_sync();  // every CTA of the cluster runs before its shared memory is written
  pdl_wait();
  pdl_launch_dependents();
  for (int e0 = 0; e0 < a.E; e0 += 128) {
    float acc[2][4][4] = {};
    const int rows = a.E - (e0 + rp * 32 + g);  // of this lane's, 8 apart
    const __half* wp = a.wr + (e0 + rp * 32 + g) * a.ldw;
    for (int c0 = b0; c0 < b1; c0 += kManyBlocks) {
      const int c1 = min(b1, c0 + kManyBlocks), kend = min(a.H, c1 * 32);
      constexpr int STEP = kManySplit * kManyRound;  // blocks of a round
#pragma unroll 1
      for (int r0 = 0; r0 < kManyBlocks && c0 + r0 < c1; r0 += STEP) {
        uint4 w[kManyRound][4];
#pragma unroll
        for (int i = 0; i < kManyRound; ++i) {
          const int k = (c0 + r0 + ks + kManySplit * i) * 32 + 8 * t;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            w[i][r] = make_uint4(0u, 0u, 0u, 0u);
            if (k < kend && r * 8 < rows)
              w[i][r] = __ldg(reinterpret_cast<const uint4*>(wp + r * 8 * a.ldw + k));
          }
        }
        // the tokens' blocks, unless they are there still
        if (r0 == 0 && (e0 == 0 || b1 - b0 > kManyBlocks)) {
          __syncthreads();                 // everyone has read the previous ones
          const int nv = (c1 - c0) * 4;    // vectors of a row
          for (int i = threadIdx.x; i < kManyTok * nv; i += kManyThreads) {
            const int m = i / nv, v = i - m * nv, k = c0 * 32 + 8 * v;
            const bool on = m < nt && k < a.H;
            cp_async16(smem_u32(xs + m * kManyRow + ((v ^ ((m & 1) << 2)) * 16)),
                       on ? a.x + (t0 + m) * a.ldx + k : a.x, on);
          }
          cp_async_commit();
          cp_async_wait<0>();
          __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kManyRound; ++i) {
          const int j = r0 + ks + kManySplit * i;
          if (c0 + j >= c1) break;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const uint4 x = *reinterpret_cast<const uint4*>(
                xs + (n * 8 + g) * kManyRow + (((j * 4 + t) ^ ((g & 1) << 2)) * 16));
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              stream_mma_16816(acc[q][n], w[i][2 * q].x, w[i][2 * q + 1].x, w[i][2 * q].y,
                               w[i][2 * q + 1].y, x.x, x.y);
              stream_mma_16816(acc[q][n], w[i][2 * q].z, w[i][2 * q + 1].z, w[i][2 * q].w,
                               w[i][2 * q + 1].w, x.z, x.w);
            }
          }
        }
      }
    }
    if (ks > 0) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        red[(((ks - 1) * 4 + rp) * 8 + u) * 32 + lane] =
            *reinterpret_cast<const float4*>(acc[u >> 2][u & 3]);
    }
    __syncthreads();
    if (ks == 0) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        float4 v = *reinterpret_cast<const float4*>(acc[u >> 2][u & 3]);
#pragma unroll
        for (int s = 0; s < kManySplit - 1; ++s) {
          const float4 o = red[((s * 4 + rp) * 8 + u) * 32 + lane];
          v.x += o.x;
          v.y += o.y;
          v.z += o.z;
          v.w += o.w;
        }
        const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = e0 + rp * 32 + (u >> 2) * 16 + (j >= 2 ? 8 : 0) + g;
          const int m = (u & 3) * 8 + 2 * t + (j & 1);
          if (e < a.E && m < nt)
            st_dsmem_f32(mapa_shared(smem_u32(recv + (rank * kManyOwn + m / kManyCluster) * a.E + e),
                                     m % kManyCluster), o[j]);
        }
      }
    }
    __syncthreads();  // the next experts' sums take the same place
  }
  cluster_sync();
  for (int i = threadIdx.x; i < kManyOwn * a.E; i += kManyThreads) {
    const int q = i / a.E, e = i - q * a.E;
    if (q * kManyCluster + rank >= nt) break;
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < kManyCluster; ++r) v += recv[r * kManyOwn * a.E + i];
    recv[i] = v + (a.bias ? __half2float(__ldg(a.bias + e)) : 0.f);
  }
  __syncthreads();
  const int m = warp * kManyCluster + rank;
  if (warp >= kManyOwn || m >= nt) return;
  int id;
  float w;
  moe_topk(recv + warp * a.E, a.E, a.k, a.normalize != 0, id, w);
  if (lane < a.k) {
    a.ids[(t0 + m) * a.k + lane] = id;
    a.weights[(t0 + m) * a.k + lane] = w;
  }
}

// The plan of a routing the caller brings.
__global__ void __launch_bounds__(kPlanThreads)
    k_moe_plan(const int* __restrict__ ids, const float* __restrict__ weights, int T, int k, int E,
               MoePlan* plan) {
  __shared__ int s_ids[kMoeMaxRows];
  __shared__ float s_w[kMoeMaxRows];
  __shared__ unsigned emask[kMoeMaxE];
  __shared__ int ebase[kMoeMaxE];
  pdl_wait();
  pdl_launch_dependents();
  for (int i = threadIdx.x; i < T * k; i += blockDim.x) {
    s_ids[i] = ids[i];
    s_w[i] = weights[i];
  }
  __syncthreads();
  moe_build_plan(plan, s_ids, s_w, T, k, E, emask, ebase);
}

// Row of weight matrix gate_up that holds gate column c (its up row: `up` rows later).
__device__ __forceinline__ int gate_row(int c, int block) {
  return block ? (c / block) * 2 * block + c % block : c;
}

// The plan's slots and rows in shared memory, for kernels that look them up as they go.
struct SlotTable {
  int* meta;
  int* base;
  unsigned char* token;
  static constexpr int BYTES = 9;  // per row
  __device__ __forceinline__ SlotTable(uint8_t* smem, int rows)
      : meta(reinterpret_cast<int*>(smem)), base(meta + rows),
        token(reinterpret_cast<unsigned char*>(base + rows)) {}
  // All rows' entries, whatever the number of slots: it is read at the same time.
  __device__ __forceinline__ int load(const MoePlan& p, int rows) {
    const int n_slots = p.n_slots;
    for (int i = threadIdx.x; i < rows; i += blockDim.x) {
      meta[i] = p.meta[i];
      base[i] = p.base[i];
      token[i] = p.token[i];
    }
    return n_slots;
  }
  __device__ __forceinline__ int expert(int slot) const { return meta[slot] & 0xffff; }
  __device__ __forceinline__ int cols(int slot) const { return meta[slot] >> 16; }
};

// A row tile is 8 columns of h: MMA rows 0-7 are their gate rows, rows 8-15 their up rows, so
// silu(gate) * up needs no exchange.  CTA b of G owns the quads of columns [n b / G, n (b + 1) / G)
// of the n = n_slots * I / 4 in slot order (whole tiles would be 6 or 7 for each CTA where one
// token reaches 4 experts), taken in pieces of at most RT tiles of one slot, the last one partly
// filled.
template <int WQ, int MG, int RT>
struct GateUpJob {
  using St = StreamStep<WQ>;
  using F = StreamFifo<WQ, MG, RT, St::NB / 4>;
  static constexpr bool ROTATE = true;
  const MoeArgs& a;
  const SlotTable& tab;
  int lo, hi;  // quads of columns, all slots' in one sequence
  int lane, up, per_slot;
  long long up_bytes;  // from a gate row to its up row
  unsigned per_group;  // group_magic
  struct Piece {
    int slot, q, left;    // first quad in the slot; quads of the worker from it on
    int c0, c1;           // columns
    int expert, base, n_cols;
    const uint8_t* w[RT];  // this lane's chunk of each tile's gate row at k = 0
    const __half* x[MG];   // vector lane % 4 of the token of column lane / 4
    GroupWord z[WQ == kWUint8Group ? RT : 1];
  };
  __device__ __forceinline__ void enter_slot(Piece& p) const {
    p.expert = tab.expert(p.slot);
    p.base = tab.base[p.slot];
    p.n_cols = tab.cols(p.slot);
#pragma unroll
    for (int mg = 0; mg < MG; ++mg) {
      const int c = mg * 8 + (lane >> 2);
      p.x[mg] = a.x + (c < p.n_cols ? tab.token[p.base + c] : 0) * a.ldx + 8 * (lane & 3);
    }
  }
  __device__ __forceinline__ bool enter(Piece& p) const {
    if (p.left <= 0) return false;
    const int left = min(per_slot - p.q, p.left);
    const int np = (left + 2 * RT - 1) / (2 * RT);
    const int cnt = (left + np - 1) / np;
    p.c0 = 4 * p.q;
    p.c1 = 4 * (p.q + cnt);
    const long long e = p.expert;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      // past the piece's columns the last one's row (never copied)
      const int c = min(p.c0 + rt * 8 + (lane >> 2), p.c1 - 1);
      p.w[rt] = a.wgu + ((e * 2 * a.I + gate_row(c, a.gu_block)) * a.H + (lane & 3) * St::KC) * St::ESZ;
    }
    if (WQ == kWUint8Group) {
      // a tile's scales and zero points: 8 gate rows, then 8 up rows (columns come in quads and
      // blocks of rows are multiples of 8, so every word is aligned): two scales each of lanes
      // 0-7, four zero points each of lanes kZeroLane ..+ 3
      const bool sc = lane < kZeroLane;
      const int half = sc ? lane >> 2 : (lane - kZeroLane) >> 1;
      const int at = sc ? 2 * (lane & 3) : 4 * ((lane - kZeroLane) & 1);
      const long long z0 = e * (a.H / a.group) * 2 * a.I;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int c = p.c0 + rt * 8 + at;
        const bool on = half < 2 && c < p.c1;
        const long long r = z0 + (on ? gate_row(c, a.gu_block) + half * up : 0);
        p.z[WQ == kWUint8Group ? rt : 0] = {
            sc ? reinterpret_cast<const uint8_t*>(a.sgu + r) : a.zgu + r,
            on ? (sc ? 4u : 2u) * a.I : 0u};
      }
    }
    return true;
  }
  __device__ __forceinline__ bool first(Piece& p) const {
    p.left = hi - lo;
    if (p.left <= 0) return false;
    p.slot = lo / per_slot;
    p.q = lo - p.slot * per_slot;
    enter_slot(p);
    return enter(p);
  }
  __device__ __forceinline__ bool next(Piece& p) const {
    const int cnt = (p.c1 - p.c0) >> 2;
    p.left -= cnt;
    if (p.left <= 0) return false;
    p.q += cnt;
    if (p.q == per_slot) {
      p.q = 0;
      ++p.slot;
      enter_slot(p);
    }
    return enter(p);
  }
  __device__ __forceinline__ void copy(const Piece& p, int step, uint32_t stage) const {
    const int kw = step * St::STEP;
    const bool ok = kw + (lane & 3) * St::KC < a.H;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int c = p.c0 + rt * 8;
      if (c >= p.c1) break;  // columns past the piece are never stored
      const uint8_t* src = p.w[rt] + kw * St::ESZ;
      const uint32_t d = stage + rt * 1024 + lane * 16;
      if (c + (lane >> 2) < p.c1) {
        cp_async16(d, src, ok);
        cp_async16(d + 512, src + up_bytes, ok);
      }
      if (WQ == kWUint8Group)
        copy_group_word(stage + F::Z_OFF + rt * 128, p.z[WQ == kWUint8Group ? rt : 0],
                        step_group(step, per_group), lane);
    }
#pragma unroll
    for (int mg = 0; mg < MG; ++mg) {
      if (mg * 8 + (lane >> 2) < p.n_cols) {
#pragma unroll
        for (int v = 0; v < St::NB / 4; ++v)
          cp_async16(stage + F::B_OFF + b_vec<St::NB / 4>(mg, 4 * v + (lane & 3), lane >> 2),
                     p.x[mg] + kw + 32 * v, kw + 32 * v + 8 * (lane & 3) < a.H);
      }
    }
  }
  __device__ __forceinline__ unsigned live(const Piece& p) const {
    return p.n_cols > 8 ? 3u : 1u;
  }
  __device__ __forceinline__ void z_rows(const Piece&, int (&r)[RT]) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) r[rt] = 0;
  }
  __device__ __forceinline__ void finish(const Piece& p, int rt, int mg, float4 v) const {
    const int n_cols = p.n_cols;
    if (p.c0 + rt * 8 >= p.c1 || mg * 8 >= n_cols) return;  // warp-uniform
    const int g = lane >> 2, t = lane & 3;
    const int c = p.c0 + rt * 8 + g;
    const bool in = c < p.c1;
    float sg = 1.f, su = 1.f;
    if (WQ == kWInt8PerChannel && in) {
      const __half* sc = a.sgu + (long long)p.expert * 2 * a.I + gate_row(c, a.gu_block);
      sg = __half2float(__ldg(sc));
      su = __half2float(__ldg(sc + up));
    }
    const float gt[2] = {v.x * sg, v.y * sg}, ut[2] = {v.z * su, v.w * su};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = mg * 8 + 2 * t + j;
      const bool on = col < n_cols;
      const int row = p.base + col;
      float hv = 0.f;
      if (on && in) {
        hv = gt[j] / (1.f + expf(-gt[j])) * ut[j] * a.plan->weight[row];
        a.h[(long long)row * a.I + c] = hv;
      }
      unsigned bits = __float_as_uint(fabsf(hv));
      bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 4));
      bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 8));
      bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 16));
      if (on && g == 0) atomicMax(&a.plan->amax[row], bits);  // a maximum: any order
    }
  }
};

template <int WQ, int MG, int RT>
struct GateUpCfg {
  static constexpr int NW = 16;
  static constexpr int BV = StreamStep<WQ>::NB / 4;
  using F = StreamFifo<WQ, MG, RT, BV>;
  static constexpr int RED = NW * RT * MG * 512;
  static constexpr int TABLE = kMoeMaxRows * SlotTable::BYTES;
  static constexpr int S = F::depth((kMaxDynSmem - RED - TABLE) / NW);
  static constexpr int FIFO = NW * S * F::STAGE;
  static constexpr int SMEM = FIFO + RED;  // + the slot table
  static_assert(SMEM + TABLE <= kMaxDynSmem, "shared memory");
};

template <int WQ, int MG, int RT>
__global__ void __launch_bounds__(32 * GateUpCfg<WQ, MG, RT>::NW, 1)
    k_moe_gate_up(const MoeArgs a, int rows, int ks) {
  using C = GateUpCfg<WQ, MG, RT>;
  extern __shared__ __align__(16) uint8_t smem[];
  SlotTable tab(smem + C::SMEM, rows);
  pdl_wait();
  pdl_launch_dependents();
  const int n_slots = tab.load(*a.plan, rows);
  __syncthreads();
  const StreamWorker wk = stream_worker<C::NW>(ks);
  const int per_slot = a.I / 4;
  int lo, hi;
  if (n_slots > 0 && wk.count >= 16 * n_slots) {  // no slot: every id named no expert
    // Many workers to a slot: each slot has its own, so that no worker's columns lie in two slots
    // (one piece more than the others need, and everyone waits for it: the last CTA 37.7 us after
    // the wait instead of 40.4 with 8 int8 experts, 19.3 instead of 22.4 with 13 group-wise slots).
    // With fewer the slots' numbers of workers differ by more than that.
    const int q = wk.count / n_slots, r = wk.count - q * n_slots, cut = r * (q + 1);
    const int slot = wk.id < cut ? wk.id / (q + 1) : r + (wk.id - cut) / q;
    split_even(per_slot, wk.id - (slot * q + min(slot, r)), q + (slot < r ? 1 : 0), lo, hi);
    lo += slot * per_slot;
    hi += slot * per_slot;
  } else {
    split_even(n_slots * per_slot, wk.id, wk.count, lo, hi);
  }
  GateUpJob<WQ, MG, RT> job{a, tab, lo, hi,
                            (int)(threadIdx.x & 31), a.gu_block ? a.gu_block : a.I, per_slot,
                            (long long)(a.gu_block ? a.gu_block : a.I) * a.H *
                                StreamStep<WQ>::ESZ,
                            group_magic<WQ>(a.group)};
  stream_run<WQ, MG, RT, C::BV, C::NW, C::S>(
      job, smem, reinterpret_cast<float4*>(smem + C::FIFO),
      (a.H + StreamStep<WQ>::STEP - 1) / StreamStep<WQ>::STEP, wk);
}

// s such that 2^s takes a largest value with these bits to [2^14, 2^15); 0 for zero.
constexpr int kNotFinite = 127;
__device__ __forceinline__ int pow2_shift(unsigned amax_bits) {
  const int ex = (int)(amax_bits >> 23);
  if (ex == 255) return kNotFinite;
  if (ex == 0) return 0;
  return max(-126, min(126, 127 + 14 - ex));
}
__device__ __forceinline__ float pow2f(int s) { return __int_as_float((127 + s) << 23); }

// Rows of y are split like k_stream_linear's (CTA b: [H b / G, H (b + 1) / G)).  A warp walks the
// steps of all slots as one sequence, of which it has one contiguous run, so the weight stream does
// not pause between experts; at a slot's end it adds its sums to its own fp32 sums per token in shared
// memory, which are added over the warps, in warp order, at the end.  The FIFO holds the fp32 h of
// a slot's first 8 tokens; those of tokens 9-16, which few slots have, are read when used.
template <int WQ, int MG, int RT>
struct DownCfg {
  using St = StreamStep<WQ>;
  static constexpr int NW = MG == 1 ? 16 : 8;  // the sums of 32 tokens leave room for 8 warps
  static constexpr int MAX_T = MG == 1 ? 8 : kMoeMaxT;
  static constexpr int HV = St::KC / 4;  // 16-byte vectors of an fp32 chunk
  using F = StreamFifo<WQ, 1, RT, HV>;
  static constexpr int YROW = RT * 16 + 8;  // floats per token (padded: 4 tokens, 4 bank groups)
  __host__ __device__ static constexpr int y_bytes(int T) { return NW * T * YROW * 4; }
  static constexpr int TABLE = MAX_T * kMoeMaxK * 10 + 16;
  static constexpr int S = F::depth((kMaxDynSmem - y_bytes(MAX_T) - TABLE) / NW);
  static constexpr int FIFO = NW * S * F::STAGE;
  __host__ __device__ static constexpr int smem(int T, int rows) {
    return FIFO + y_bytes(T) + rows * 10 + 16;
  }
  static_assert(FIFO + y_bytes(MAX_T) + TABLE <= kMaxDynSmem, "shared memory");
};

template <int WQ, int MG, int RT>
__global__ void __launch_bounds__(32 * DownCfg<WQ, MG, RT>::NW, 1)
    k_moe_down(const MoeArgs a, int rows) {
  using C = DownCfg<WQ, MG, RT>;
  using St = StreamStep<WQ>;
  using F = typename C::F;
  constexpr int S = C::S, HV = C::HV, NW = C::NW;
  extern __shared__ __align__(16) uint8_t smem[];
  float* y_all = reinterpret_cast<float*>(smem + C::FIFO);
  SlotTable tab(smem + C::FIFO + C::y_bytes(a.T), rows);
  signed char* shift = reinterpret_cast<signed char*>(tab.token + rows);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  // The plan may be read before the wait: k_moe_gate_up lets this grid start only after its own
  // wait, when the router (and all before it) had finished.  So the first steps' weights are
  // fetched here, under the rest of k_moe_gate_up; only h and its largest values need the wait.
  const int n_slots = tab.load(*a.plan, rows);
  __syncthreads();
  int lo, hi;
  split_even(a.H, blockIdx.x, gridDim.x, lo, hi);
  const int nsteps = (a.I + St::STEP - 1) / St::STEP;
  const int npieces = (hi - lo + 16 * RT - 1) / (16 * RT);
  float* y = y_all + warp * a.T * C::YROW;
  const uint8_t* fifo_p = smem + warp * S * F::STAGE;
  const uint32_t fifo = smem_u32(fifo_p);
  const int rot = (int)((unsigned)nsteps * blockIdx.x / gridDim.x);
  // The warp's share of the sequence of all slots' steps: one run of them, so that it meets few
  // slots and adds few sums to its tokens' (steps dealt out in turn instead: one token through 8
  // int8 experts 77 us, so 71).
  const int run = (n_slots * nsteps + NW - 1) / NW;
  struct At {
    int slot, step, left;  // left: steps of the run from here on
  };
  auto advance = [&](At& p) {  // -> whether the slot changed
    --p.left;
    if (++p.step < nsteps) return false;
    p.step = 0;
    ++p.slot;
    return true;
  };
  auto k_of = [&](int step) {  // this lane's first k of a step (rotated as in stream_run)
    const int s = step + rot;
    return (s < nsteps ? s : s - nsteps) * St::STEP;
  };
  for (int pc = 0; pc < npieces; ++pc) {
    int n0, n1;
    split_even(hi - lo, pc, npieces, n0, n1);
    n0 += lo;
    n1 += lo;
    for (int i = lane; i < a.T * C::YROW; i += 32) y[i] = 0.f;
    // rows this lane's copies belong to, and where they start in an expert's matrix
    const long long row_bytes = (long long)a.I * St::ESZ;
    const uint8_t* w0 = a.wd + (n0 + g) * row_bytes + t * 16;
    const unsigned magic = group_magic<WQ>(a.group);
    const int first = warp * run;
    At l{first / nsteps, first % nsteps, min(run, n_slots * nsteps - first)};
    At u = l;
    int lfifo = 0;
    // the slot being copied: this lane's chunks at k = 0
    const uint8_t* lw;
    const float* lh;
    GroupWord lz[WQ == kWUint8Group ? RT : 1];
    bool lon;
    auto enter = [&]() {
      if (l.left <= 0) return;
      const long long e = tab.expert(l.slot);
      lw = w0 + e * a.H * row_bytes;
      lh = a.h + (long long)(tab.base[l.slot] + g) * a.I + 4 * t;
      lon = g < tab.cols(l.slot);
      if (WQ == kWUint8Group) {
        const long long z0 = e * (a.I / a.group) * a.H;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          lz[WQ == kWUint8Group ? rt : 0] =
              group_word(a.sd + z0, a.zd + z0, n0 + rt * 16, a.H, lane);
      }
    };
    enter();
    const long long row8 = 8 * row_bytes;
    auto issue = [&](bool weights, bool hidden) {
      if (l.left > 0) {
        const int step = l.step + rot < nsteps ? l.step + rot : l.step + rot - nsteps;
        const int kw = step * St::STEP;
        const uint32_t stage = fifo + lfifo * F::STAGE;
        if (weights) {
          const bool ok = kw + t * St::KC < a.I;
          const uint8_t* src = lw + kw * St::ESZ;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const int ra = n0 + rt * 16 + g;
            const uint32_t d = stage + rt * 1024 + lane * 16;
            // rows past the piece are never stored
            if (ra < n1) cp_async16(d, src, ok);
            src += row8;
            if (ra + 8 < n1) cp_async16(d + 512, src, ok);
            src += row8;
            if (WQ == kWUint8Group)
              copy_group_word(stage + F::Z_OFF + rt * 128, lz[WQ == kWUint8Group ? rt : 0],
                              step_group(step, magic), lane);
          }
        }
        if (hidden && lon) {
          const float* h = lh + kw;
#pragma unroll
          for (int v = 0; v < HV; ++v)
            cp_async16(stage + F::B_OFF + b_vec<HV>(0, 4 * v + t, g), h + 16 * v,
                       kw + 16 * v + 4 * t < a.I);
        }
        if (advance(l)) enter();
      }
      if (hidden) cp_async_commit();
      lfifo = lfifo + 1 == S ? 0 : lfifo + 1;
    };
    if (pc == 0) {
      const At l0 = l;
#pragma unroll 1
      for (int i = 0; i < S - 1; ++i) issue(true, false);
      l = l0;
      lfifo = 0;
      enter();
      pdl_wait();
      pdl_launch_dependents();
      for (int i = tid; i < rows; i += 32 * NW)
        shift[i] = (signed char)pow2_shift(a.plan->amax[i]);
#pragma unroll 1
      for (int i = 0; i < S - 1; ++i) issue(false, true);
      __syncthreads();
    } else {
#pragma unroll 1
      for (int i = 0; i < S - 1; ++i) issue(true, true);
    }
    int ufifo = 0;
    int z_row[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) z_row[rt] = n0 + rt * 16;
    while (u.left > 0) {
      const int slot = u.slot;
      const int base = tab.base[slot], n_cols = tab.cols(slot);
      float up2[MG];  // 2^s of this lane's columns
      bool fin[MG];   // whether the row of h is finite: if not its low parts (inf - inf) are left out
#pragma unroll
      for (int mg = 0; mg < MG; ++mg) {
        const int sh = mg * 8 + g < n_cols ? shift[base + mg * 8 + g] : 0;
        fin[mg] = sh != kNotFinite;
        up2[mg] = fin[mg] ? pow2f(sh) : 1.f;
      }
      float acc[RT][MG][4] = {};
      while (u.left > 0 && u.slot == slot) {
        cp_async_wait<S - 2>();
        __syncwarp();
        issue(true, true);
        const uint8_t* stage = fifo_p + ufifo * F::STAGE;
        StreamA<WQ, RT> w;
        stream_read_weights<WQ, RT>(w, stage, F::Z_OFF, z_row, lane);
#pragma unroll
        for (int mg = 0; mg < MG; ++mg) {
          if (mg * 8 >= n_cols) continue;  // warp-uniform
          uint32_t b[2][St::NB];  // high and low parts
#pragma unroll
          for (int v = 0; v < HV; ++v) {
            float4 x;  // a column without a row holds anything: it stays in its column
            if (mg == 0) {
              x = *reinterpret_cast<const float4*>(stage + F::B_OFF + b_vec<HV>(0, HV * t + v, g));
            } else {
              const int k0 = k_of(u.step) + t * St::KC;
              x = make_float4(0.f, 0.f, 0.f, 0.f);
              if (mg * 8 + g < n_cols && k0 < a.I)
                x = *reinterpret_cast<const float4*>(
                    a.h + (long long)(base + mg * 8 + g) * a.I + k0 + 4 * v);
            }
            const float s4[4] = {x.x * up2[mg], x.y * up2[mg], x.z * up2[mg], x.w * up2[mg]};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const __half2 hi2 = __floats2half2_rn(s4[2 * i], s4[2 * i + 1]);
              const float2 back = __half22float2(hi2);
              const __half2 lo2 =
                  __floats2half2_rn(s4[2 * i] - back.x, s4[2 * i + 1] - back.y);
              b[0][2 * v + i] = *reinterpret_cast<const uint32_t*>(&hi2);
              b[1][2 * v + i] = fin[mg] ? *reinterpret_cast<const uint32_t*>(&lo2) : 0u;
            }
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) stream_mma<WQ, RT, false>(w, rt, b, acc[rt][mg]);
        }
        ufifo = ufifo + 1 == S ? 0 : ufifo + 1;
        advance(u);
      }
      // the slot's sums: undo the row's power of two, apply the channel's scale
#pragma unroll
      for (int mg = 0; mg < MG; ++mg) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int col = mg * 8 + 2 * t + j;
          if (col >= n_cols) continue;
          float* yt = y + tab.token[base + col] * C::YROW;
          const int sh = shift[base + col];
          const float f = sh != kNotFinite ? pow2f(-sh) : 1.f;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int r = rt * 16 + 8 * half + g;
              float v = acc[rt][mg][2 * half + j] * f;
              if (WQ == kWInt8PerChannel && n0 + r < n1)
                v *= __half2float(__ldg(a.sd + (long long)tab.expert(slot) * a.H + n0 + r));
              yt[r] += v;
            }
          }
        }
      }
      __syncwarp();
    }
    cp_async_wait<0>();
    __syncthreads();
    const int nr = n1 - n0;
    for (int i = tid; i < a.T * nr; i += 32 * NW) {
      const int m = i / nr, r = i - m * nr, n = n0 + r;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) v += y_all[(w * a.T + m) * C::YROW + r];
      if (a.res) v += __half2float(a.res[m * a.ldr + n]);
      a.y[m * a.ldy + n] = __float2half_rn(v);
    }
    __syncthreads();
  }
}

namespace {

size_t moe_plan_bytes() { return (sizeof(MoePlan) + 255) / 256 * 256; }

template <int MG>
cudaError_t launch_route_mg(const RouteArgs& a, cudaStream_t st) {
  using C = RouteCfg<MG>;
  static BigSmem big;
  return launch_big(k_moe_route<MG>, big, C::SMEM, kRouteCluster, 32 * C::NW, C::SMEM, st,
                    kRouteCluster, a);
}

cudaError_t launch_route(const RouteArgs& a, cudaStream_t st) {
  if (a.T > RouteCfg<4>::TOK) {
    static BigSmem big;
    const long long grid = ((long long)a.T + kManyTok - 1) / kManyTok * kManyCluster;
    return launch_big(k_moe_route_many, big, many_smem(kMoeMaxE), (int)grid, kManyThreads,
                      many_smem(a.E), st, kManyCluster, a);
  }
  return a.T <= 8 ? launch_route_mg<1>(a, st) : launch_route_mg<4>(a, st);
}

template <int WQ, int MG, int RT>
cudaError_t launch_down(const MoeArgs& a, int rows, int grid, cudaStream_t st) {
  using C = DownCfg<WQ, MG, RT>;
  static BigSmem big;
  return launch_big(k_moe_down<WQ, MG, RT>, big, C::smem(C::MAX_T, C::MAX_T * kMoeMaxK),
                    grid, 32 * C::NW, C::smem(a.T, rows), st, 1, a, rows);
}

// Warps of a k_moe_gate_up worker: with few steps to a row fewer warps share them (a piece's fixed
// cost is then spread over more of each warp's steps).  Measured with 4 / 8 / 16: 7 tokens, uint8,
// 32 steps: 42.7 / 43.2 / 47 us; one token, int8, 80 steps: 71.9 / 70.8 / 75; 32 tokens, fp16, 120
// steps: 459 / 454 / 463.
int gate_up_warps(int nsteps) { return nsteps >= 64 ? 8 : 4; }

// MG: groups of 8 columns a slot can have (1 up to 8 tokens, else 2).
template <int WQ, int MG>
cudaError_t launch_experts(const MoeArgs& a, int rows, cudaStream_t st) {
  const int sms = std::max(1, current_sms());
  {
    constexpr int RT = 2;
    using C = GateUpCfg<WQ, MG, RT>;
    static BigSmem big;
    const cudaError_t e =
        launch_big(k_moe_gate_up<WQ, MG, RT>, big, C::SMEM + kMoeMaxRows * SlotTable::BYTES, sms,
                   32 * C::NW, C::SMEM + rows * SlotTable::BYTES, st, 1, a, rows,
                   gate_up_warps((a.H + StreamStep<WQ>::STEP - 1) / StreamStep<WQ>::STEP));
    if (e != cudaSuccess) return e;
  }
  const int grid = std::min(sms, (a.H + 7) / 8);
  const int per = (a.H + grid - 1) / grid;
  if (per <= 16) return launch_down<WQ, MG, 1>(a, rows, grid, st);
  if (per <= 32) return launch_down<WQ, MG, 2>(a, rows, grid, st);
  return launch_down<WQ, MG, 3>(a, rows, grid, st);
}

template <int WQ>
cudaError_t launch_experts_t(const MoeArgs& a, int rows, cudaStream_t st) {
  return a.T <= 8 ? launch_experts<WQ, 1>(a, rows, st) : launch_experts<WQ, 2>(a, rows, st);
}

cudaError_t run_experts(const MoeArgs& a, int top_k, int kind, cudaStream_t st) {
  const int rows = a.T * top_k;
  switch (kind) {
    case kWFp16: return launch_experts_t<0>(a, rows, st);
    case kWInt8PerChannel: return launch_experts_t<1>(a, rows, st);
    case kWUint8Group: return launch_experts_t<2>(a, rows, st);
    default: return cudaErrorInvalidConfiguration;
  }
}

}  // namespace
}  // namespace tempo_sm100
