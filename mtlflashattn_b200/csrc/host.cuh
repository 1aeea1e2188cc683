// Host-side helpers shared by the library's translation units: fault injection, NVTX ranges,
// cached device attributes, and a kernel's shared-memory attributes.
#pragma once
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "../../include/mfa.h"

namespace mfa {

// ------------------------------------------------------------------ host fault injection
// MFA_FAULT=<site>[,<site>...] makes the named entry point fail before it launches anything,
// so callers' error handling can be tested without touching a GPU. Sites: fwd (every
// form of the forward), combine (the merges), kv4 (append, gather and attention of the 4-bit
// cache), norm_rope.
inline bool fault_injected(const char* site) {
  const char* env = std::getenv("MFA_FAULT");
  if (env == nullptr || *env == 0) return false;
  const size_t n = std::strlen(site);
  for (const char* p = env; *p;) {
    const char* e = std::strchr(p, ',');
    const size_t len = e ? (size_t)(e - p) : std::strlen(p);
    if (len == n && std::strncmp(p, site, n) == 0) return true;
    if (!e) break;
    p = e + 1;
  }
  return false;
}

// ------------------------------------------------------------------ NVTX
// Host-side range around each launching entry point, named after it, so an nsys / ncu timeline
// shows which library call queued which kernels. NVTX v3 is header-only: with no tool attached
// a push/pop is a test of a null function pointer.
struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
};

struct DevInfo {
  int major = -1, minor = -1, sms = 0;
};
inline DevInfo dev_info(int dev) {
  static std::mutex mu;
  static DevInfo cache[64];
  std::lock_guard<std::mutex> lk(mu);
  if (dev < 0 || dev >= 64) return DevInfo{};
  if (cache[dev].major < 0) {
    cudaDeviceGetAttribute(&cache[dev].major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&cache[dev].minor, cudaDevAttrComputeCapabilityMinor, dev);
    cudaDeviceGetAttribute(&cache[dev].sms, cudaDevAttrMultiProcessorCount, dev);
  }
  return cache[dev];
}

// cudaFuncSetAttribute once per (kernel, device).
template <typename K>
cudaError_t ensure_smem(K kernel, int dev, int bytes) {
  static std::mutex mu;
  static const void* seen[256];
  static int seen_dev[256];
  static int nseen = 0;
  std::lock_guard<std::mutex> lk(mu);
  for (int i = 0; i < nseen; ++i)
    if (seen[i] == (const void*)kernel && seen_dev[i] == dev) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  // all of the SM's unified L1/shared storage as shared memory (two one-tile CTAs per SM)
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && nseen < 256) {
    seen[nseen] = (const void*)kernel;
    seen_dev[nseen] = dev;
    ++nseen;
  }
  return e;
}

// mfa_fwd of dense, padded keys whose sequence b has k_lens[b] (device; at most p->Lk, which it is
// cut to) of them; a row's centre follows from that length (mfa_api.cu).
int forward_padded(const mfa_fwd_params* p, const int32_t* k_lens, cudaStream_t st);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace mfa
