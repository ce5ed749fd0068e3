// The GEMM with a fused epilogue, y = act(A W^T + bias) + residual: which kernel runs.
//
//   M <= 16    k_stream_linear (stream.cuh)
//   M > 16     the hyperform the shipped dispatcher plans for the same problem, in its EPI
//              instantiation; W8A16 at prefill sizes expands the weights to fp16 first, the
//              per-channel kind without its scale, which multiplies the fp32 accumulator instead
//              (an int8 value is exact in fp16, its product with a scale is not).
#pragma once

#include "stream.h"

namespace tempo_sm100 {

// int8 -> fp16, 16 values per thread (16 bytes in, 32 out); exact.
__global__ void __launch_bounds__(256)
    k_expand_i8(const uint8_t* __restrict__ W, __half* __restrict__ out, int N, int K,
                long long ldw) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int per_row = K / 16;
  if (i >= (long long)N * per_row) return;
  pdl_wait();
  pdl_launch_dependents();
  const int n = (int)(i / per_row);
  const int k0 = (int)(i - (long long)n * per_row) * 16;
  __half2 h[8];
  gemv_weights<kWInt8PerChannel>(ld_stream(W + (long long)n * ldw + k0), h, __half2{}, __half2{});
  uint4* o = reinterpret_cast<uint4*>(out + (long long)n * K + k0);
  o[0] = *reinterpret_cast<const uint4*>(&h[0]);
  o[1] = *reinterpret_cast<const uint4*>(&h[4]);
}

namespace {

cudaError_t run_pair_epi(const Problem& pr, const Hyper& h, cudaStream_t st) {
  if (pr.wkind == kWInt8PerChannel)
    return h.bn == 256 ? launch_pair_w8<256, 1, true>(pr, h, st)
                       : launch_pair_w8<128, 1, true>(pr, h, st);
  if (pr.wkind == kWUint8Group)
    return h.bn == 256 ? launch_pair_w8<256, 2, true>(pr, h, st)
                       : launch_pair_w8<128, 2, true>(pr, h, st);
  switch (h.bn) {
    case 256: return launch_pair<256, false, true>(pr, h, st);
    case 224: return launch_pair<224, false, true>(pr, h, st);
    case 192: return launch_pair<192, false, true>(pr, h, st);
    case 160: return launch_pair<160, false, true>(pr, h, st);
    case 128: return launch_pair<128, false, true>(pr, h, st);
    default: return cudaErrorInvalidConfiguration;
  }
}

// The EPI instantiations of the 1-CTA tiles the shipped ladders name from M = 17 on.
cudaError_t run_tile_epi(const Problem& pr, const Hyper& h, cudaStream_t st) {
  const int key = pr.wkind * 10000 + h.swap * 1000 + h.bn;
  switch (key) {
    case 1064: return launch_inst<64, 0, true, false, true>(pr, h, st);
    case 1128: return launch_inst<128, 0, true, false, true>(pr, h, st);
    case 128: return launch_inst<128, 0, false, false, true>(pr, h, st);
    case 256: return launch_inst<256, 0, false, false, true>(pr, h, st);
    case 12032: return launch_inst<32, 1, true, true, true>(pr, h, st);
    case 12064: return launch_inst<64, 1, true, true, true>(pr, h, st);
    case 11128: return launch_inst<128, 1, true, false, true>(pr, h, st);
    case 22032: return launch_inst<32, 2, true, true, true>(pr, h, st);
    case 22064: return launch_inst<64, 2, true, true, true>(pr, h, st);
    case 21128: return launch_inst<128, 2, true, false, true>(pr, h, st);
    default: return cudaErrorInvalidConfiguration;
  }
}

cudaError_t run_epilogue(const Problem& pr, cudaStream_t st) {
  if (pr.M <= kStreamMaxM)
    return run_stream({static_cast<const __half*>(pr.A), static_cast<const uint8_t*>(pr.W),
                       static_cast<const __half*>(pr.scale), static_cast<const uint8_t*>(pr.zero),
                       static_cast<__half*>(pr.C), pr.epi, pr.M, pr.N, pr.K, pr.lda, pr.ldw,
                       pr.ldc, pr.group > 0 ? pr.group : 1},
                      pr.wkind, st);
  const size_t cap = pr.ws ? pr.ws_bytes : 0;
  tempo::gen::Choice c{};
  cudaError_t e;
  if (pr.wkind == kWFp16) {
    tempo::gen::GemmParams p{};
    p.M = pr.M; p.N = pr.N; p.K = pr.K;
    p.lda = (int)pr.lda; p.ldb = (int)pr.ldw; p.ldc = (int)pr.ldc;
    p.ws_bytes = cap;
    e = tempo::gen::plan(p, &c);
  } else {
    tempo::gen::W8A16Params p{};
    p.M = pr.M; p.N = pr.N; p.K = pr.K;
    p.lda = (int)pr.lda; p.ldw = (int)pr.ldw; p.ldc = (int)pr.ldc;
    p.scale_kind = pr.wkind; p.group = pr.group;
    p.ws_bytes = cap;
    e = tempo::gen::plan(p, &c);
  }
  if (e != cudaSuccess) return e;
  Hyper h{c.bn, c.swap, c.splits, c.group_m, 0};
  h.cta_group = c.cta_group;
  if (c.expand) {
    const size_t wexp = expand_ws_bytes(pr.N, pr.K);
    char* base = static_cast<char*>(pr.ws);
    __half* wf = reinterpret_cast<__half*>(base + kExpandOffset);
    if (pr.wkind == kWInt8PerChannel) {
      const long long n = (long long)pr.N * (pr.K / 16);
      e = launch_ex(k_expand_i8, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, 1,
                    static_cast<const uint8_t*>(pr.W), wf, pr.N, pr.K, (long long)pr.ldw);
    } else {
      e = launch_expand(pr, wf, st);
    }
    if (e != cudaSuccess) return e;
    Problem q = pr;
    q.wkind = kWFp16;
    q.W = wf;
    q.ldw = pr.K;
    q.group = 0;
    q.scale = q.zero = nullptr;
    if (pr.wkind == kWInt8PerChannel) q.epi.scale = static_cast<const __half*>(pr.scale);
    q.ws_bytes = pr.ws_bytes - wexp;
    q.ws_parts = base + kExpandOffset + wexp;
    return run_pair_epi(q, h, st);
  }
  return c.cta_group == 2 ? run_pair_epi(pr, h, st) : run_tile_epi(pr, h, st);
}

}  // namespace
}  // namespace tempo_sm100
