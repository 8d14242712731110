// Plaintext Mamba-2 operators behind the fhe_ssm_scan, fhe_causal_conv and
// fhe_token_logprobs entry points: argument checks and launches.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/fhe_b200.h"
#include "context.h"

namespace fhe {

uint64_t ssm_scan_workspace(const fhe_ssm_scan_args& a);
void ssm_scan(const fhe_ssm_scan_args& a);
uint64_t ssm_scan_backward_workspace(const fhe_ssm_scan_grad_args& g);
void ssm_scan_backward(const fhe_ssm_scan_grad_args& g);
void causal_conv(const fhe_causal_conv_args& a);
uint64_t causal_conv_backward_workspace(const fhe_causal_conv_grad_args& g);
void causal_conv_backward(const fhe_causal_conv_grad_args& g);
void token_logprobs(const fhe_token_logprobs_args& a);
void token_logprobs_backward(const fhe_token_logprobs_grad_args& g);

// Makes `device` current and restores the caller's device on destruction.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    int count = 0;
    FHE_CUDA(cudaGetDeviceCount(&count));
    require(device >= 0 && device < count, "device ordinal out of range");
    FHE_CUDA(cudaGetDevice(&old_));
    if (device != old_) FHE_CUDA(cudaSetDevice(device));
    changed_ = device != old_;
  }
  ~DeviceGuard() {
    if (changed_) cudaSetDevice(old_);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;

 private:
  int old_ = 0;
  bool changed_ = false;
};

// Carves a caller's workspace into 256-byte aligned arrays; with a null base
// it only counts.
struct Carver {
  uint8_t* base;
  uint64_t used = 0;
  explicit Carver(void* p) : base(static_cast<uint8_t*>(p)) {}
  template <class T>
  T* take(uint64_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (count * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

inline void check_workspace(const void* ws, uint64_t have, uint64_t need) {
  if (need == 0) return;
  require(ws != nullptr && have >= need,
          "workspace too small: " + std::to_string(have) + " of " + std::to_string(need) + " bytes");
  require(reinterpret_cast<uintptr_t>(ws) % 256 == 0, "workspace must be 256-byte aligned");
}

inline uint32_t elem_size(int32_t dtype) { return dtype == FHE_F32 ? 4 : 2; }

template <class T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T from_f(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// N consecutive elements of T, loaded and stored as one word.
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// Calls f with a value of the element type `dtype` names.
template <class F>
void with_type(int32_t dtype, F&& f) {
  if (dtype == FHE_F32) f(float{});
  else if (dtype == FHE_BF16) f(__nv_bfloat16{});
  else if (dtype == FHE_F16) f(__half{});
  else require(false, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
}

}  // namespace fhe
