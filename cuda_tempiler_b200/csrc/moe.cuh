// A mixture-of-experts layer for a few tokens (T <= 32), three launches on one stream:
//
//   k_moe_route    logits x Wr^T + b, top-k of each token, softmax weights, and the plan: the
//                  experts that were reached (slots), each with the set of its tokens
//   k_moe_gate_up  h[r][i] = w_r * silu(gate_i(x_t)) * up_i(x_t) for every routed row r = (t, e)
//   k_moe_down     y[t][n] = res[t][n] + sum_e sum_i down_e[n][i] h[(t, e)][i]
//
// The bytes are the weights of the reached experts, read once each whatever the number of
// tokens; everything else is small.  The products are those of stream.cuh: weights straight from
// HBM into the registers of warp MMAs, fp32 sums, 8-bit weights as exact integers.
//
// The columns of every MMA are the tokens themselves (column m = token m): a token that did not
// choose the expert is a column of zeros, which costs nothing beside the weight stream, and
// k_moe_down can keep one fp32 sum per (n, token) in registers over all experts: no atomics, no
// partial outputs, the same order of sums on every run.  A column a token did not choose is left
// out of its sum (not added as zero), so an infinite weight of one expert reaches only the tokens
// that chose it.
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
constexpr int kRouteCluster = 8;

// What the router tells the two products (in the caller's workspace; every call writes it whole).
struct MoePlan {
  int n_slots;                      // experts reached by at least one token
  int pad[3];
  int expert[kMoeMaxE];             // slot -> expert, ascending
  int base[kMoeMaxE];               // slot -> its first row
  unsigned mask[kMoeMaxE];          // slot -> its tokens; row of token t: base + rank of bit t
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
      const unsigned act = __ballot_sync(0xffffffffu, m != 0u);
      const int c = __popc(m);
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += v;
      }
      const int b = row + incl - c;
      if (e < E) ebase[e] = b;
      if (m) {
        const int s = slot + __popc(act & ((1u << tid) - 1u));
        plan->expert[s] = e;
        plan->base[s] = b;
        plan->mask[s] = m;
      }
      slot += __popc(act);
      row += __shfl_sync(0xffffffffu, incl, 31);
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
    if (first) plan->weight[ebase[e] + __popc(emask[e] & ((1u << t) - 1u))] = sum;
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
// weight of the token NaN, as the softmax over all experts is; the ids stay valid.
__device__ void moe_topk(const float* logits, int E, int k, bool normalize, int* ids, float* w) {
  constexpr int P = kMoeMaxE / 32;
  const int lane = threadIdx.x & 31;
  unsigned key[P];
  unsigned long long nan_any = 0;
  float mx = -INFINITY;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int e = lane + 32 * p;
    key[p] = 0u;
    if (e < E) {
      const float x = logits[e];
      key[p] = logit_key(x);
      nan_any |= (x != x);
      mx = fmaxf(mx, x);
    }
  }
  const bool bad = __any_sync(0xffffffffu, nan_any != 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float total = 0.f;
  if (!normalize) {
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (lane + 32 * p < E) total += expf(logits[lane + 32 * p] - mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  unsigned taken = 0u;
  float mine = 0.f;  // lane j keeps the j-th choice
  int mine_id = 0;
  for (int j = 0; j < k; ++j) {
    unsigned best = 0u;
    int bp = -1;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (lane + 32 * p < E && !((taken >> p) & 1u) && (bp < 0 || key[p] > best)) {
        best = key[p];
        bp = p;
      }
    }
    const unsigned top = __reduce_max_sync(0xffffffffu, bp < 0 ? 0u : best);
    const unsigned cand = (bp >= 0 && best == top) ? (unsigned)(lane + 32 * bp) : 0xffffffffu;
    const unsigned e = __reduce_min_sync(0xffffffffu, cand);
    if ((e & 31u) == (unsigned)lane) taken |= 1u << (e >> 5);
    if (lane == j) {
      mine_id = (int)e;
      mine = expf(logits[e] - mx);
    }
  }
  if (normalize) {
    total = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane < k) {
    ids[lane] = mine_id;
    w[lane] = bad ? __int_as_float(0x7fffffff) : mine / total;
  }
}

// One cluster of 8 CTAs routes 32 tokens: CTA r multiplies them with the experts
// [E r / 8, E (r + 1) / 8) (its 8 warps split H), hands each token's logits to the CTA that owns
// the token (t % 8) through distributed shared memory, and picks the top-k of its own tokens.
// With a plan wanted (one cluster, T <= 32) CTA 0 collects the choices and builds it.
// Each step's sum starts at zero and is added in fp32: a tensor core truncates what it adds to a
// large accumulator, which over a long K is visible in fp32 weights.
template <int MG>
__global__ void __launch_bounds__(kStreamThreads)
    k_moe_route(const __half* __restrict__ x, long long ldx, const __half* __restrict__ wr,
                long long ldw, const __half* __restrict__ bias, int T, int E, int H, int k,
                int normalize, int* __restrict__ ids, float* __restrict__ weights,
                MoePlan* plan) {
  using S = StreamStep<kWFp16>;
  constexpr int U = 4;
  constexpr int TOK = MG * 8;                    // tokens of a cluster
  constexpr int OWN = (TOK + kRouteCluster - 1) / kRouteCluster;
  __shared__ float4 red[kStreamWarps][MG][32];
  __shared__ float logits[OWN][kMoeMaxE];        // of this CTA's tokens
  __shared__ int s_ids[kMoeMaxRows];             // CTA 0: every token's choices
  __shared__ float s_w[kMoeMaxRows];
  __shared__ unsigned emask[kMoeMaxE];
  __shared__ int ebase[kMoeMaxE];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rank = (int)cluster_ctarank();
  const int t0 = (blockIdx.x / kRouteCluster) * TOK;
  const int nt = min(TOK, T - t0);
  pdl_wait();
  pdl_launch_dependents();
  cluster_sync();  // every CTA of the cluster runs before its shared memory is written
  const int lo = E * rank / kRouteCluster, hi = E * (rank + 1) / kRouteCluster;
  const int nsteps = (H + S::STEP - 1) / S::STEP;
  for (int n0 = lo; n0 < hi; n0 += 16) {
    float acc[MG][4] = {};
    StreamStage<kWFp16, MG, 1> st[U];
    auto load_b = [&](int step, int mg, uint32_t (&b)[S::NB]) {
      const int k0 = step * S::STEP + t * S::KC;
      const int m = mg * 8 + g;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (k0 < H && m < nt)
        v = __ldg(reinterpret_cast<const uint4*>(x + (long long)(t0 + m) * ldx + k0));
      b[0] = v.x;
      b[1] = v.y;
      b[2] = v.z;
      b[3] = v.w;
    };
    auto load = [&](StreamStage<kWFp16, MG, 1>& s, int step) {
      const int k0 = step * S::STEP + t * S::KC;
      const bool ok = step < nsteps && k0 < H;
      const int ra = n0 + g, rb = ra + 8;
      s.xa[0] = s.xb[0] = make_uint4(0u, 0u, 0u, 0u);
      if (ok && ra < hi) s.xa[0] = __ldg(reinterpret_cast<const uint4*>(wr + ra * ldw + k0));
      if (ok && rb < hi) s.xb[0] = __ldg(reinterpret_cast<const uint4*>(wr + rb * ldw + k0));
      if constexpr (kStreamPreB<kWFp16, MG>) {
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
          float d[1][MG][4] = {};
          stream_mma<kWFp16, MG, 1>(
              st[u], d, [&](int mg, uint32_t(&b)[S::NB]) { load_b(step, mg, b); },
              [](int) { return true; });
#pragma unroll
          for (int mg = 0; mg < MG; ++mg)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[mg][j] += d[0][mg][j];
          load(st[u], step + U * kStreamWarps);
        }
        step += kStreamWarps;
      }
    }
#pragma unroll
    for (int mg = 0; mg < MG; ++mg)
      red[warp][mg][lane] = make_float4(acc[mg][0], acc[mg][1], acc[mg][2], acc[mg][3]);
    __syncthreads();
    for (int i = tid; i < MG * 32; i += kStreamThreads) {
      const int l = i & 31, mg = i >> 5;
      float4 v = red[0][mg][l];
#pragma unroll
      for (int w = 1; w < kStreamWarps; ++w) {
        const float4 a = red[w][mg][l];
        v.x += a.x;
        v.y += a.y;
        v.z += a.z;
        v.w += a.w;
      }
      const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = n0 + (l >> 2) + (j >= 2 ? 8 : 0);
        const int m = mg * 8 + 2 * (l & 3) + (j & 1);
        if (e >= hi || m >= nt) continue;
        const float z = o[j] + (bias ? __half2float(__ldg(bias + e)) : 0.f);
        st_dsmem_f32(mapa_shared(smem_u32(&logits[m / kRouteCluster][e]), m % kRouteCluster), z);
      }
    }
    __syncthreads();
  }
  cluster_sync();
  for (int q = warp; q < OWN; q += kStreamWarps) {
    const int m = q * kRouteCluster + rank;
    if (m >= nt) continue;
    int* id = ids + (long long)(t0 + m) * k;
    float* w = weights + (long long)(t0 + m) * k;
    moe_topk(logits[q], E, k, normalize != 0, id, w);
    __syncwarp();
    if (plan && lane < k) {
      // lane < k wrote these two itself
      st_dsmem_f32(mapa_shared(smem_u32(&s_ids[m * k + lane]), 0), __int_as_float(id[lane]));
      st_dsmem_f32(mapa_shared(smem_u32(&s_w[m * k + lane]), 0), w[lane]);
    }
  }
  if (!plan) return;
  cluster_sync();
  if (rank == 0) moe_build_plan(plan, s_ids, s_w, T, k, E, emask, ebase);
}

// The plan of a routing the caller brings.
__global__ void __launch_bounds__(kStreamThreads)
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

// A row tile is 8 columns of h: MMA rows 0-7 are their gate rows, rows 8-15 their up rows, so
// silu(gate) * up needs no exchange.  CTA b of G owns the tiles [n b / G, n (b + 1) / G) of the
// n = n_slots * I / 8 tiles in slot order, taken in pieces of at most RT tiles of one slot.
template <int WQ, int MG, int RT>
__global__ void __launch_bounds__(kStreamThreads, 2) k_moe_gate_up(const MoeArgs a) {
  using S = StreamStep<WQ>;
  constexpr int U = stream_depth<WQ, MG, RT>();
  __shared__ float4 red[kStreamWarps][RT][MG][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  const MoePlan& plan = *a.plan;
  const int per_slot = a.I / 8;
  const long long n_tiles = (long long)plan.n_slots * per_slot;
  const long long lo = n_tiles * blockIdx.x / gridDim.x;
  const long long hi = n_tiles * (blockIdx.x + 1) / gridDim.x;
  const int nsteps = (a.H + S::STEP - 1) / S::STEP;
  const int up = a.gu_block ? a.gu_block : a.I;
  const int groups = WQ == kWUint8Group ? a.H / a.group : 0;
  for (long long pos = lo; pos < hi;) {
    const int slot = (int)(pos / per_slot);
    const int c_tile = (int)(pos - (long long)slot * per_slot);
    const int left = (int)min((long long)(per_slot - c_tile), hi - pos);
    const int np = (left + RT - 1) / RT;
    const int cnt = (left + np - 1) / np;  // tiles of this piece (<= RT)
    pos += cnt;
    const int e = plan.expert[slot];
    const unsigned mask = plan.mask[slot];
    const int base = plan.base[slot];
    const uint8_t* W = a.wgu + (long long)e * 2 * a.I * a.H * S::ESZ;
    const __half* sc = WQ == kWFp16 ? nullptr
                       : a.sgu + (long long)e * 2 * a.I * (WQ == kWUint8Group ? groups : 1);
    const uint8_t* zp = WQ == kWUint8Group ? a.zgu + (long long)e * 2 * a.I * groups : nullptr;
    float acc[RT][MG][4] = {};
    StreamStage<WQ, MG, RT> st[U];
    auto load_b = [&](int step, int mg, uint32_t (&b)[S::NB]) {
      const int k0 = step * S::STEP + t * S::KC;
      const int m = mg * 8 + g;
#pragma unroll
      for (int q = 0; q < S::KC / 8; ++q) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (k0 < a.H && ((mask >> m) & 1u))
          v = __ldg(reinterpret_cast<const uint4*>(a.x + m * a.ldx + k0) + q);
        b[4 * q] = v.x;
        b[4 * q + 1] = v.y;
        b[4 * q + 2] = v.z;
        b[4 * q + 3] = v.w;
      }
    };
    auto load = [&](StreamStage<WQ, MG, RT>& s, int step) {
      const int k0 = step * S::STEP + t * S::KC;
      const bool ok = step < nsteps && k0 < a.H;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int ra = gate_row((c_tile + rt) * 8 + g, a.gu_block), rb = ra + up;
        const bool on = ok && rt < cnt;
        s.xa[rt] = s.xb[rt] = make_uint4(0u, 0u, 0u, 0u);
        if (on) {
          s.xa[rt] = ld_stream(W + ((long long)ra * a.H + k0) * S::ESZ);
          s.xb[rt] = ld_stream(W + ((long long)rb * a.H + k0) * S::ESZ);
        }
        if (WQ == kWUint8Group) {
          s.s[rt] = 0;
          s.z[rt] = 0;
          if (on) {  // lane % 16 < 8: a gate row, else an up row
            const int r = gate_row((c_tile + rt) * 8 + (lane & 7), a.gu_block) +
                          ((lane & 8) ? up : 0);
            const long long gi = (long long)(k0 / a.group) * 2 * a.I + r;
            s.s[rt] = __ldg(reinterpret_cast<const unsigned short*>(sc) + gi);
            s.z[rt] = __ldg(zp + gi);
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
              [&](int mg) { return ((mask >> (8 * mg)) & 0xffu) != 0u; });
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
    // RT * MG * 32 items; every warp runs whole (rt, mg) groups, so the shuffles are convergent
    for (int i = tid; i < RT * MG * 32; i += kStreamThreads) {
      const int mg = (i >> 5) % MG, rt = (i >> 5) / MG;
      if (rt >= cnt) continue;
      float4 v = red[0][rt][mg][lane];
#pragma unroll
      for (int w = 1; w < kStreamWarps; ++w) {
        const float4 q = red[w][rt][mg][lane];
        v.x += q.x;
        v.y += q.y;
        v.z += q.z;
        v.w += q.w;
      }
      const int c = (c_tile + rt) * 8 + g;
      float sg = 1.f, su = 1.f;
      if (WQ == kWInt8PerChannel) {
        const int ra = gate_row(c, a.gu_block);
        sg = __half2float(__ldg(sc + ra));
        su = __half2float(__ldg(sc + ra + up));
      }
      const float gt[2] = {v.x * sg, v.y * sg}, ut[2] = {v.z * su, v.w * su};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int m = mg * 8 + 2 * t + j;
        const bool on = (mask >> m) & 1u;
        const int row = base + __popc(mask & ((1u << m) - 1u));
        float hv = 0.f;
        if (on) {
          hv = gt[j] / (1.f + expf(-gt[j])) * ut[j] * plan.weight[row];
          a.h[(long long)row * a.I + c] = hv;
        }
        unsigned bits = __float_as_uint(fabsf(hv));
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 4));
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 8));
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 16));
        if (on && g == 0) atomicMax(&a.plan->amax[row], bits);
      }
    }
    __syncthreads();
  }
}

// 2^s that takes a largest value with these bits to [2^14, 2^15); 1 for zero, infinite and NaN.
__device__ __forceinline__ int pow2_shift(unsigned amax_bits) {
  const int ex = (int)(amax_bits >> 23);
  if (ex == 0 || ex == 255) return 0;
  return max(-126, min(126, 127 + 14 - ex));
}
__device__ __forceinline__ float pow2f(int s) { return __int_as_float((127 + s) << 23); }

// Rows of y are split like k_stream_linear's (CTA b: [H b / G, H (b + 1) / G)); a warp walks the
// steps of all slots as one sequence (warp w: steps w, w + 8, ...), so the weight stream does not
// pause between experts.
template <int WQ, int MG, int RT>
__global__ void __launch_bounds__(kStreamThreads, 2) k_moe_down(const MoeArgs a) {
  using S = StreamStep<WQ>;
  constexpr int U = RT == 1 ? (MG == 4 ? 3 : 4) : (MG == 4 && WQ ? 1 : 2);
  __shared__ float4 red[kStreamWarps][RT][MG][32];
  __shared__ int s_expert[kMoeMaxE], s_base[kMoeMaxE];
  __shared__ unsigned s_mask[kMoeMaxE];
  __shared__ signed char s_shift[kMoeMaxRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  const int n_slots = a.plan->n_slots;
  for (int i = tid; i < n_slots; i += kStreamThreads) {
    s_expert[i] = a.plan->expert[i];
    s_base[i] = a.plan->base[i];
    s_mask[i] = a.plan->mask[i];
  }
  __syncthreads();
  const int n_rows =
      n_slots ? s_base[n_slots - 1] + __popc(s_mask[n_slots - 1]) : 0;
  for (int i = tid; i < n_rows; i += kStreamThreads)
    s_shift[i] = (signed char)pow2_shift(a.plan->amax[i]);
  __syncthreads();
  const int lo = (int)((long long)a.H * blockIdx.x / gridDim.x);
  const int hi = (int)((long long)a.H * (blockIdx.x + 1) / gridDim.x);
  const int nsteps = (a.I + S::STEP - 1) / S::STEP;
  const int total = n_slots * nsteps;
  const int groups = WQ == kWUint8Group ? a.I / a.group : 1;
  const int npieces = (hi - lo + 16 * RT - 1) / (16 * RT);
  struct Stage {
    uint4 xa[RT], xb[RT];
    unsigned short s[RT];
    uint8_t z[RT];
  };
  for (int pc = 0; pc < npieces; ++pc) {
    const int n0 = lo + (hi - lo) * pc / npieces;
    const int n1 = lo + (hi - lo) * (pc + 1) / npieces;
    float acc[RT][MG][4] = {};
    Stage st[U];
    auto load = [&](Stage& s, int fs) {
      const int slot = fs / nsteps;
      const int k0 = (fs - slot * nsteps) * S::STEP + t * S::KC;
      const bool ok = fs < total && k0 < a.I;
      const int e = fs < total ? s_expert[slot] : 0;
      const uint8_t* W = a.wd + (long long)e * a.H * a.I * S::ESZ;
      const long long gi = WQ == kWUint8Group
                               ? ((long long)e * groups + k0 / a.group) * a.H
                               : (long long)e * a.H;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int ra = n0 + rt * 16 + g, rb = ra + 8;
        s.xa[rt] = s.xb[rt] = make_uint4(0u, 0u, 0u, 0u);
        if (ok && ra < n1) s.xa[rt] = ld_stream(W + ((long long)ra * a.I + k0) * S::ESZ);
        if (ok && rb < n1) s.xb[rt] = ld_stream(W + ((long long)rb * a.I + k0) * S::ESZ);
        s.s[rt] = 0;
        s.z[rt] = 0;
        if (WQ) {  // scale (and zero point) of row lane % 16; k0 >= I only in int8's last step
          const int r = n0 + rt * 16 + (lane & 15);
          if (fs < total && r < n1) {
            s.s[rt] = __ldg(reinterpret_cast<const unsigned short*>(a.sd) + gi + r);
            if (WQ == kWUint8Group) s.z[rt] = __ldg(a.zd + gi + r);
          }
        }
      }
    };
    auto use = [&](const Stage& s, int fs) {
      const int slot = fs / nsteps;
      const int k0 = (fs - slot * nsteps) * S::STEP + t * S::KC;
      const unsigned mask = s_mask[slot];
      const int base = s_base[slot];
      uint32_t ha[RT][8], hb[RT][8];
      float fa[RT], fb[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const unsigned sz = (unsigned)s.s[rt] << 16 | s.z[rt];
        const unsigned za = WQ ? __shfl_sync(0xffffffffu, sz, g) : 0u;
        const unsigned zb = WQ ? __shfl_sync(0xffffffffu, sz, g + 8) : 0u;
        fa[rt] = WQ ? __half2float(__ushort_as_half((unsigned short)(za >> 16))) : 1.f;
        fb[rt] = WQ ? __half2float(__ushort_as_half((unsigned short)(zb >> 16))) : 1.f;
        stream_unpack<WQ>(s.xa[rt], zero_bias((uint8_t)za), ha[rt]);
        stream_unpack<WQ>(s.xb[rt], zero_bias((uint8_t)zb), hb[rt]);
      }
#pragma unroll
      for (int mg = 0; mg < MG; ++mg) {
        if (((mask >> (8 * mg)) & 0xffu) == 0u) continue;  // warp-uniform
        const int m = mg * 8 + g;
        uint32_t bh[S::NB], bl[S::NB];
        if (k0 < a.I && ((mask >> m) & 1u)) {
          const int row = base + __popc(mask & ((1u << m) - 1u));
          const float f = pow2f(s_shift[row]);
          const float4* hp = reinterpret_cast<const float4*>(a.h + (long long)row * a.I + k0);
#pragma unroll
          for (int q = 0; q < S::KC / 4; ++q) {
            const float4 v = hp[q];
            const float s4[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const __half2 hi2 = __floats2half2_rn(s4[2 * i], s4[2 * i + 1]);
              const float2 back = __half22float2(hi2);
              // an infinite high part has no low part (inf - inf is NaN)
              const float l0 = isinf(back.x) ? 0.f : s4[2 * i] - back.x;
              const float l1 = isinf(back.y) ? 0.f : s4[2 * i + 1] - back.y;
              const __half2 lo2 = __floats2half2_rn(l0, l1);
              bh[2 * q + i] = *reinterpret_cast<const uint32_t*>(&hi2);
              bl[2 * q + i] = *reinterpret_cast<const uint32_t*>(&lo2);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < S::NB; ++i) bh[i] = bl[i] = 0u;
        }
        // this lane's two columns: their 2^-s, and whether the token chose the expert
        const int m0 = mg * 8 + 2 * t;
        const bool on0 = (mask >> m0) & 1u, on1 = (mask >> (m0 + 1)) & 1u;
        const int r0 = base + __popc(mask & ((1u << m0) - 1u));
        const float f0 = on0 ? pow2f(-s_shift[r0]) : 0.f;
        const float f1 = on1 ? pow2f(-s_shift[r0 + (on0 ? 1 : 0)]) : 0.f;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < S::NMMA; ++j) {
            mma_16816(d, ha[rt][2 * j], hb[rt][2 * j], ha[rt][2 * j + 1], hb[rt][2 * j + 1],
                      bh[2 * j], bh[2 * j + 1]);
            mma_16816(d, ha[rt][2 * j], hb[rt][2 * j], ha[rt][2 * j + 1], hb[rt][2 * j + 1],
                      bl[2 * j], bl[2 * j + 1]);
          }
          if (on0) {
            acc[rt][mg][0] = fmaf(d[0], fa[rt] * f0, acc[rt][mg][0]);
            acc[rt][mg][2] = fmaf(d[2], fb[rt] * f0, acc[rt][mg][2]);
          }
          if (on1) {
            acc[rt][mg][1] = fmaf(d[1], fa[rt] * f1, acc[rt][mg][1]);
            acc[rt][mg][3] = fmaf(d[3], fb[rt] * f1, acc[rt][mg][3]);
          }
        }
      }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) load(st[u], warp + u * kStreamWarps);
    for (int fs = warp; fs < total;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (fs < total) {
          use(st[u], fs);
          load(st[u], fs + U * kStreamWarps);
        }
        fs += kStreamWarps;
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
      const int mg = (i >> 5) % MG, rt = (i >> 5) / MG;
      float4 v = red[0][rt][mg][lane];
#pragma unroll
      for (int w = 1; w < kStreamWarps; ++w) {
        const float4 q = red[w][rt][mg][lane];
        v.x += q.x;
        v.y += q.y;
        v.z += q.z;
        v.w += q.w;
      }
      const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + rt * 16 + g + (j >= 2 ? 8 : 0);
        const int m = mg * 8 + 2 * t + (j & 1);
        if (n >= n1 || m >= a.T) continue;
        float r = o[j];
        if (a.res) r += __half2float(a.res[m * a.ldr + n]);
        a.y[m * a.ldy + n] = __float2half_rn(r);
      }
    }
    __syncthreads();
  }
}

namespace {

size_t moe_plan_bytes() { return (sizeof(MoePlan) + 255) / 256 * 256; }

cudaError_t launch_route(const __half* x, long long ldx, const __half* wr, long long ldw,
                         const __half* bias, int T, int E, int H, int k, int normalize, int* ids,
                         float* weights, MoePlan* plan, cudaStream_t st) {
  const int tok = T <= 8 ? 8 : 32;
  const dim3 grid((unsigned)((T + tok - 1) / tok * kRouteCluster));
  auto kern = T <= 8 ? k_moe_route<1> : k_moe_route<4>;
  return launch_ex(kern, grid, dim3(kStreamThreads), 0, st, kRouteCluster, x, ldx, wr, ldw, bias,
                   T, E, H, k, normalize, ids, weights, plan);
}

template <int WQ, int MG>
cudaError_t launch_experts(const MoeArgs& a, cudaStream_t st) {
  const int sms = std::max(1, current_sms());
  const int grid = 2 * sms;
  cudaError_t e = launch_ex(k_moe_gate_up<WQ, MG, MG == 1 ? 4 : 2>, dim3(grid),
                            dim3(kStreamThreads), 0, st, 1, a);
  if (e != cudaSuccess) return e;
  const int gd = std::min(grid, (a.H + 7) / 8);
  const int rows = (a.H + gd - 1) / gd;
  if (rows <= 16)
    return launch_ex(k_moe_down<WQ, MG, 1>, dim3(gd), dim3(kStreamThreads), 0, st, 1, a);
  return launch_ex(k_moe_down<WQ, MG, 2>, dim3(gd), dim3(kStreamThreads), 0, st, 1, a);
}

template <int WQ>
cudaError_t launch_experts_t(const MoeArgs& a, cudaStream_t st) {
  if (a.T <= 8) return launch_experts<WQ, 1>(a, st);
  if (a.T <= 16) return launch_experts<WQ, 2>(a, st);
  return launch_experts<WQ, 4>(a, st);
}

cudaError_t run_experts(const MoeArgs& a, int kind, cudaStream_t st) {
  switch (kind) {
    case kWFp16: return launch_experts_t<0>(a, st);
    case kWInt8PerChannel: return launch_experts_t<1>(a, st);
    case kWUint8Group: return launch_experts_t<2>(a, st);
    default: return cudaErrorInvalidConfiguration;
  }
}

}  // namespace
}  // namespace tempo_sm100
