// The weight-streaming products (stream.cu) as the other translation units see them.
#pragma once

#ifndef TEMPO_SM100_KERNEL_CUH  // the shipped directories' frozen copy of the same file
#include "../tempo/plugins/sm100/skeletons/gemm_sm100/kernel.cuh"
#endif

#include <cstdint>
#include <mutex>

namespace tempo_sm100 {

// Held by an entry point while it enqueues: the launches of a call hand data on in the caller's
// workspace, which host threads that share a stream may share too, so no other call's launch may get
// between them.  One mutex per stream, up to collisions.
inline std::mutex& launch_mutex(const void* stream) {
  static std::mutex m[64];
  return m[(reinterpret_cast<uintptr_t>(stream) >> 4) % 64];
}

constexpr int kStreamMaxM = 16;

// y = act(A W^T * scale + bias) + res, M <= kStreamMaxM; layouts of the C-ABI's epilogue entries.
struct LinearArgs {
  const __half* A;
  const uint8_t* W;  // bytes of the fp16 or 8-bit weights; ldw in elements
  const __half* scale;
  const uint8_t* zero;
  __half* C;
  EpiArgs epi;
  int M, N, K;
  long long lda, ldw, ldc;
  int group;
};

cudaError_t run_stream(const LinearArgs& a, int wkind, cudaStream_t st);

}  // namespace tempo_sm100
