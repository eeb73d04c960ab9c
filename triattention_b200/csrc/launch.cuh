// Host-side helpers of the entry points: alignment and layout checks, kernel launches.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>
#include <utility>

#include "../../include/triattn_b200.h"

namespace triattn {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

inline int check_launch() { return cudaGetLastError() == cudaSuccess ? TRIATTN_OK : TRIATTN_ERR_CUDA; }

// Kernel launch, optionally as a programmatic dependent of the preceding kernel in the stream: the launch is
// processed and its CTAs become resident while that kernel drains (every kernel of this library executes griddepcontrol.wait before it
// writes anything or reads what its predecessor writes.  All but one start with it; attend_combine_kernel reads lengths and
// offsets before, which is sound because the attention kernel releases it only after its own wait).
template <typename... KArgs, typename... Args>
int launch_kernel(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...) == cudaSuccess ? TRIATTN_OK : TRIATTN_ERR_CUDA;
}

// Opt a kernel in to `smem` bytes of dynamic shared memory; the attribute call is made only when a device has
// not yet been raised to that size for this kernel.  Some kernels are sized by the call (the width of a block table), so two threads may ask
// for different sizes at once: calls that raise are made one at a time, and the attribute is never lowered.
constexpr int kMaxDevicesSmem = 64;
template <auto Kern>
bool ensure_dynamic_smem(size_t smem) {
  static std::atomic<size_t> raised[kMaxDevicesSmem];
  static std::mutex raising;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevicesSmem) return false;
  if (raised[dev].load(std::memory_order_acquire) >= smem) return true;
  std::lock_guard<std::mutex> lock(raising);
  if (raised[dev].load(std::memory_order_relaxed) >= smem) return true;
  if (cudaFuncSetAttribute(reinterpret_cast<const void*>(Kern), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return false;
  raised[dev].store(smem, std::memory_order_release);
  return true;
}

inline int validate_layout(const triattn_paged_layout* L) {
  if (L == nullptr) return TRIATTN_ERR_INVALID_ARGUMENT;
  if (L->num_layers <= 0 || L->num_reqs <= 0 || L->num_kv_heads <= 0 || L->group_size <= 0 || L->head_dim <= 0 ||
      L->block_size <= 0 || L->num_blocks <= 0 || L->max_blocks_per_req <= 0)
    return TRIATTN_ERR_INVALID_ARGUMENT;
  if (L->head_dim % 8 != 0) return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  if (L->num_reqs > 65535 || L->num_layers > 65535) return TRIATTN_ERR_UNSUPPORTED_SHAPE;
  if (L->block_stride % 8 != 0 || L->token_stride % 8 != 0 || L->head_stride % 8 != 0) return TRIATTN_ERR_MISALIGNED;
  return TRIATTN_OK;
}

}  // namespace triattn
