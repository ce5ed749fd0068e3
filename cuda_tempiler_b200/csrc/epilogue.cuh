// The GEMM with a fused epilogue, y = act(A W^T + bias) + residual: which kernel runs.
//
//   M <= 16    k_stream_linear (stream.cuh) where a CTA's weight rows are few (stream_epilogue)
//   M <= 384   k_epi_swap (swap_tile.cuh); 8-bit weights up to 1279 rows
//   above      the 2-CTA tiles the shipped dispatcher plans for the fp16 problem, with the epilogue
//              on the accumulator; 8-bit weights are expanded to fp16 first, the per-channel kind
//              without its scale, which multiplies the fp32 accumulator instead (an int8 value is
//              exact in fp16, its product with a scale is not).
#pragma once

#include "stream.h"
#include "swap_tile.cuh"

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

// Up to kStreamMaxM rows: the stream while a CTA's share of the weight rows fits a piece or two
// (every further piece reads the activations again and adds up its warps' sums), above that the
// swapped tiles.  Measured, stream / swapped us at 8 and at 16 rows (N x K):
//   fp16   3840 x 4096   7.4 / 11.2   8.3 / 11.1     5120 x 8192  17.5 / 19.2  21.0 / 19.6
//          8192 x 3840  15.4 / 15.6  20.2 / 15.8    15360 x 3840  24.8 / 21.4  31.1 / 21.5
//   int8   5120 x 8192  12.8 / 17.7  13.8 / 18.5     8192 x 3840  13.1 / 15.0  15.4 / 15.7
//         10240 x 5120  17.2 / 19.6  19.0 / 20.3    15360 x 3840  20.4 / 20.3  23.3 / 20.5
// Group-wise weights always (5120 x 8192 13.3 / 20.7 and 14.6 / 21.5, 15360 x 3840 20.5 / 25.7 and
// 24.4 / 25.8): the stream takes them as they are, the tiles round each to fp16.
bool stream_epilogue(int M, int N, int wkind) {
  if (M > kStreamMaxM) return false;
  const int sms = current_sms() > 0 ? current_sms() : 1;
  const int rows = (N + sms - 1) / sms;
  switch (wkind) {
    case kWFp16: return rows <= (M <= 8 ? 48 : 32);
    case kWInt8PerChannel: return rows <= (M <= 8 ? 96 : 72);
    default: return true;
  }
}

// Above them: the swapped tiles, or the 2-CTA ones (8-bit weights expanded first).  Measured,
// swapped / 2-CTA us: fp16 15360 x 3840 at 384 rows 50 / 56 (385 rows), 5120 x 17408 72 / 96,
// 3840 x 4096 29 / 30; from 385 rows on a second tile of rows would be mostly padding.  8-bit
// 1024 x 5120 x 8192 97 / 118, 15360 x 3840 at 1280 rows 172 / 154, 1536 x 5120 x 17408 304 / 265.
bool swap_epilogue(int M, int N, int K, int wkind, size_t ws_bytes) {
  if (wkind == kWFp16) return M <= kSwapMaxRows;
  return M < 1280 || ws_bytes < kExpandOffset + expand_ws_bytes(N, K);
}

// Workspace the kernel of choice would like (0: none).
size_t epilogue_ws_bytes(int M, int N, int K, int wkind) {
  if (stream_epilogue(M, N, wkind)) return 0;
  if (swap_epilogue(M, N, K, wkind, ~(size_t)0))
    return epi_swap_plan(wkind, M, N, K, std::max(1, current_sms()), ~(size_t)0).ws_bytes;
  const size_t ws = tempo_sm100_workspace_bytes(M, N, K, 0);
  return wkind == kWFp16 ? ws : std::max(ws, (size_t)kExpandOffset) + expand_ws_bytes(N, K);
}

cudaError_t run_pair_epi(const Problem& pr, const Hyper& h, cudaStream_t st) {
  switch (h.bn) {
    case 256: return launch_pair<256, false, true>(pr, h, st);
    case 224: return launch_pair<224, false, true>(pr, h, st);
    case 192: return launch_pair<192, false, true>(pr, h, st);
    case 160: return launch_pair<160, false, true>(pr, h, st);
    case 128: return launch_pair<128, false, true>(pr, h, st);
    default: return cudaErrorInvalidConfiguration;
  }
}

cudaError_t run_epilogue(const Problem& pr, cudaStream_t st) {
  const size_t cap = pr.ws ? pr.ws_bytes : 0;
  // the stream needs no workspace; without one the swapped tiles would run whole, on few SMs
  if (stream_epilogue(pr.M, pr.N, pr.wkind) ||
      (pr.M <= kStreamMaxM && cap < epilogue_ws_bytes(pr.M, pr.N, pr.K, pr.wkind)))
    return run_stream({static_cast<const __half*>(pr.A), static_cast<const uint8_t*>(pr.W),
                       static_cast<const __half*>(pr.scale), static_cast<const uint8_t*>(pr.zero),
                       static_cast<__half*>(pr.C), pr.epi, pr.M, pr.N, pr.K, pr.lda, pr.ldw,
                       pr.ldc, pr.group > 0 ? pr.group : 1},
                      pr.wkind, st);
  if (swap_epilogue(pr.M, pr.N, pr.K, pr.wkind, cap)) {
    switch (pr.wkind) {
      case kWFp16: return launch_epi_swap<kWFp16>(pr, st);
      case kWInt8PerChannel: return launch_epi_swap<kWInt8PerChannel>(pr, st);
      default: return launch_epi_swap<kWUint8Group>(pr, st);
    }
  }
  tempo::gen::Choice c{};
  tempo::gen::GemmParams p{};
  p.M = pr.M; p.N = pr.N; p.K = pr.K;
  p.lda = (int)pr.lda; p.ldb = (int)pr.ldw; p.ldc = (int)pr.ldc;
  p.ws_bytes = pr.wkind == kWFp16 ? cap : cap - expand_ws_bytes(pr.N, pr.K);
  cudaError_t e = tempo::gen::plan(p, &c);
  if (e != cudaSuccess) return e;
  if (c.cta_group != 2) return cudaErrorInvalidConfiguration;
  Hyper h{c.bn, c.swap, c.splits, c.group_m, 0};
  h.cta_group = c.cta_group;
  if (pr.wkind != kWFp16) {
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
  return run_pair_epi(pr, h, st);
}

}  // namespace
}  // namespace tempo_sm100
