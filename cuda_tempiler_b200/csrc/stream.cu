// Host side of the weight-streaming kernels: the products with an epilogue for few rows (used by
// the epilogue entry points) and the mixture-of-experts entry points of include/tempo_sm100.h.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <utility>

#include "tempo_sm100.h"
#include "stream.cuh"

namespace tempo_sm100 {
namespace {

constexpr int kMaxDevices = 64;

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool aligned16(const void* p) { return aligned(p, 16); }

int current_sms() {
  static int sms[kMaxDevices];
  static std::once_flag once[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 1;
  std::call_once(once[dev], [dev] {
    cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  });
  return std::max(1, sms[dev]);
}

// Programmatic dependent launch and clusters as the GEMM kernels use them (TEMPO_SM100_PDL=0
// turns the former off).
template <typename... KArgs, typename... Args>
cudaError_t launch_ex(void (*kern)(KArgs...), int grid, int threads, int smem, cudaStream_t st,
                      int cluster, Args&&... args) {
  static const bool pdl = [] {
    const char* v = std::getenv("TEMPO_SM100_PDL");
    return !(v && v[0] == '0');
  }();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Launch of a kernel that may ask for more than 48 KB: the attribute once per device.
struct BigSmem {
  std::once_flag once[kMaxDevices];
  cudaError_t err[kMaxDevices];
};

template <typename... KArgs, typename... Args>
cudaError_t launch_big(void (*kern)(KArgs...), BigSmem& b, int max_smem, int grid, int threads,
                       int smem, cudaStream_t st, int cluster, Args&&... args) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::call_once(b.once[dev], [&] {
    b.err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem);
    if (b.err[dev] == cudaSuccess && cluster > 8)
      b.err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (b.err[dev] != cudaSuccess) return b.err[dev];
  return launch_ex(kern, grid, threads, smem, st, cluster, std::forward<Args>(args)...);
}

template <int WQ, int MG, int RT>
cudaError_t launch_stream_rt(const LinearArgs& a, int grid, cudaStream_t st) {
  using C = LinearCfg<WQ, MG, RT>;
  static BigSmem big;
  return launch_big(k_stream_linear<WQ, MG, RT>, big, C::SMEM, grid, 32 * C::NW, C::SMEM, st, 1, a);
}

template <int WQ, int MG>
cudaError_t launch_stream_mg(const LinearArgs& a, cudaStream_t st) {
  // One CTA per SM, 8 rows at least, as one worker in the fewest row tiles that hold its rows.
  // (When this was chosen: o_proj M = 1, 26 rows per CTA, 6.6 us in 2 tiles, 7.2 in 3, 8.7 as two
  // workers of 8 warps; int8 M = 16, 35 rows, 15.4 us in 3 tiles, 22 in 2 pieces of 2, 20 as two
  // workers.  Now 6.4 and 13.8.)
  const int grid = std::min(current_sms(), (a.N + 7) / 8);
  const int rows = (a.N + grid - 1) / grid;
  if (rows <= 16) return launch_stream_rt<WQ, MG, 1>(a, grid, st);
  if (rows <= 32) return launch_stream_rt<WQ, MG, 2>(a, grid, st);
  return launch_stream_rt<WQ, MG, 3>(a, grid, st);
}

template <int WQ>
cudaError_t launch_stream(const LinearArgs& a, cudaStream_t st) {
  return a.M <= 8 ? launch_stream_mg<WQ, 1>(a, st) : launch_stream_mg<WQ, 2>(a, st);
}

}  // namespace

cudaError_t run_stream(const LinearArgs& a, int wkind, cudaStream_t st) {
  if (a.M < 1 || a.M > kStreamMaxM) return cudaErrorInvalidConfiguration;
  switch (wkind) {
    case kWFp16: return launch_stream<0>(a, st);
    case kWInt8PerChannel: return launch_stream<1>(a, st);
    case kWUint8Group: return launch_stream<2>(a, st);
    default: return cudaErrorInvalidConfiguration;
  }
}

}  // namespace tempo_sm100

#include "moe.cuh"

namespace tempo_sm100 {
namespace {

int route_args(const void* x, const void* wr, const void* bias, const int* ids,
               const float* weights, int T, int E, int H, int k, int ldx, int ldw) {
  if (!x || !wr || !ids || !weights || T < 1 || E < 1 || H < 1 || k < 1 || k > E)
    return cudaErrorInvalidValue;
  if (E > kMoeMaxE || k > kMoeMaxK || H % 8 || ldx < H || ldw < H || ldx % 8 || ldw % 8 ||
      !aligned16(x) || !aligned16(wr) || !aligned(bias, 2) || !aligned(ids, 4) ||
      !aligned(weights, 4))
    return cudaErrorInvalidConfiguration;
  return 0;
}

int moe_args(MoeArgs& a, const void* x, const void* wgu, const void* wd, const void* sgu,
             const void* zgu, const void* sd, const void* zd, const void* res, void* y, int T,
             int E, int H, int I, int k, int ldx, int ldr, int ldy, int kind, int group,
             int gu_block, void* ws, size_t ws_bytes) {
  if (!x || !wgu || !wd || !y || T < 1 || E < 1 || H < 1 || I < 1 || k < 1)
    return cudaErrorInvalidValue;
  if (kind < kWFp16 || kind > kWUint8Group || (kind && (!sgu || !sd)) ||
      (kind == kWUint8Group && (!zgu || !zd)))
    return cudaErrorInvalidValue;
  if (T > kMoeMaxT || E > kMoeMaxE || k > kMoeMaxK || H % 16 || I % 16 || ldx < H || ldx % 8 ||
      ldy < H || (res && ldr < H) || !aligned16(x) || !aligned16(wgu) || !aligned16(wd) ||
      !aligned(res, 2) || !aligned(y, 2))
    return cudaErrorInvalidConfiguration;
  // group-wise scales and zero points are copied in 4-byte words (copy_group_word), a channel's
  // scale is read by itself
  const unsigned word = kind == kWUint8Group ? 4 : 2;
  if (kind && (!aligned(sgu, word) || !aligned(sd, word))) return cudaErrorInvalidConfiguration;
  if (kind == kWUint8Group && (!aligned(zgu, word) || !aligned(zd, word)))
    return cudaErrorInvalidConfiguration;
  if (kind == kWUint8Group && (group <= 0 || group % 64 || H % group || I % group))
    return cudaErrorInvalidConfiguration;
  if (gu_block < 0 || (gu_block && (gu_block % 8 || I % gu_block)))
    return cudaErrorInvalidConfiguration;
  if (!ws || !aligned16(ws) || ws_bytes < tempo_sm100_moe_workspace_bytes(T, k, I))
    return cudaErrorInvalidValue;
  a.x = static_cast<const __half*>(x);
  a.ldx = ldx;
  a.T = T;
  a.E = E;
  a.H = H;
  a.I = I;
  a.wgu = static_cast<const uint8_t*>(wgu);
  a.wd = static_cast<const uint8_t*>(wd);
  a.sgu = static_cast<const __half*>(sgu);
  a.sd = static_cast<const __half*>(sd);
  a.zgu = static_cast<const uint8_t*>(zgu);
  a.zd = static_cast<const uint8_t*>(zd);
  a.group = group > 0 ? group : 1;
  a.gu_block = gu_block;
  a.plan = static_cast<MoePlan*>(ws);
  a.h = reinterpret_cast<float*>(static_cast<char*>(ws) + moe_plan_bytes());
  a.res = static_cast<const __half*>(res);
  a.ldr = ldr;
  a.y = static_cast<__half*>(y);
  a.ldy = ldy;
  return 0;
}

}  // namespace
}  // namespace tempo_sm100

using namespace tempo_sm100;

extern "C" {

int tempo_sm100_moe_route(const void* x, const void* w_router, const void* bias, int* ids,
                          float* weights, int T, int E, int H, int top_k, int ldx, int ldw,
                          int normalize, void* stream) {
  const int rc = route_args(x, w_router, bias, ids, weights, T, E, H, top_k, ldx, ldw);
  if (rc) return rc;
  return launch_route({static_cast<const __half*>(x), ldx, static_cast<const __half*>(w_router),
                       ldw, static_cast<const __half*>(bias), T, E, H, top_k, normalize, ids,
                       weights, nullptr},
                      static_cast<cudaStream_t>(stream));
}

size_t tempo_sm100_moe_workspace_bytes(int T, int top_k, int I) {
  if (T < 1 || top_k < 1 || I < 1) return 0;
  return moe_plan_bytes() + (size_t)T * top_k * I * sizeof(float);
}

int tempo_sm100_moe_layer(const void* x, const void* w_router, const void* bias,
                          const void* w_gate_up, const void* w_down, const void* s_gate_up,
                          const void* z_gate_up, const void* s_down, const void* z_down,
                          const void* residual, void* y, int* ids, float* weights, int T, int E,
                          int H, int I, int top_k, int ldx, int ldw, int ldr, int ldy,
                          int weight_kind, int group_size, int gu_block, int normalize, void* ws,
                          size_t ws_bytes, void* stream) {
  int rc = route_args(x, w_router, bias, ids, weights, T, E, H, top_k, ldx, ldw);
  if (rc) return rc;
  MoeArgs a{};
  rc = moe_args(a, x, w_gate_up, w_down, s_gate_up, z_gate_up, s_down, z_down, residual, y, T, E,
                H, I, top_k, ldx, ldr, ldy, weight_kind, group_size, gu_block, ws, ws_bytes);
  if (rc) return rc;
  const std::lock_guard<std::mutex> lock(launch_mutex(stream));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      launch_route({a.x, ldx, static_cast<const __half*>(w_router), ldw,
                    static_cast<const __half*>(bias), T, E, H, top_k, normalize, ids, weights,
                    a.plan},
                   st);
  return e != cudaSuccess ? e : run_experts(a, top_k, weight_kind, st);
}

int tempo_sm100_moe_experts(const void* x, const int* ids, const float* weights,
                            const void* w_gate_up, const void* w_down, const void* s_gate_up,
                            const void* z_gate_up, const void* s_down, const void* z_down,
                            const void* residual, void* y, int T, int E, int H, int I, int top_k,
                            int ldx, int ldr, int ldy, int weight_kind, int group_size,
                            int gu_block, void* ws, size_t ws_bytes, void* stream) {
  if (!ids || !weights) return cudaErrorInvalidValue;
  if (!aligned(ids, 4) || !aligned(weights, 4)) return cudaErrorInvalidConfiguration;
  MoeArgs a{};
  const int rc =
      moe_args(a, x, w_gate_up, w_down, s_gate_up, z_gate_up, s_down, z_down, residual, y, T, E,
               H, I, top_k, ldx, ldr, ldy, weight_kind, group_size, gu_block, ws, ws_bytes);
  if (rc) return rc;
  const std::lock_guard<std::mutex> lock(launch_mutex(stream));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_ex(k_moe_plan, 1, kPlanThreads, 0, st, 1, ids,
                                  weights, T, top_k, E, a.plan);
  return e != cudaSuccess ? e : run_experts(a, top_k, weight_kind, st);
}

}  // extern "C"
