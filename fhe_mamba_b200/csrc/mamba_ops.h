// Plaintext Mamba-2 operators behind the fhe_ssm_scan, fhe_causal_conv,
// fhe_token_logprobs, fhe_rms_norm, fhe_embedding and fhe_beam_* entry points:
// argument checks and launches.
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
void rms_norm(const fhe_rms_norm_args& a);
uint64_t rms_norm_backward_workspace(const fhe_rms_norm_grad_args& g);
void rms_norm_backward(const fhe_rms_norm_grad_args& g);
void embedding(const fhe_embedding_args& a);
uint64_t embedding_backward_workspace(const fhe_embedding_grad_args& g);
void embedding_backward(const fhe_embedding_grad_args& g);
void beam_select(const fhe_beam_select_args& a);
void beam_reorder(const fhe_beam_reorder_args& a);

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

// Tokens of row b (lengths may be nullptr: all).
__device__ __forceinline__ int clamp_length(const int32_t* lengths, uint32_t b, uint32_t length) {
  if (!lengths) return (int)length;
  return min(max(lengths[b], 0), (int)length);
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

// Lets a kernel have up to `bytes` of dynamic shared memory.  The limit is state of the
// whole process and of every call of that kernel: `bytes` is the most that any launch of
// it asks for, never the size of one launch, so that calls from other threads, of other
// sizes, do not take it from this one.
template <class K>
void allow_shared(K kernel, uint32_t bytes) {
  FHE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
}

// Two fp32 operations per instruction (sm_100): elementwise over arrays of V,
// pairs packed when V is even.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// o = a * b + c, o = a * b, o = a + b
template <int V>
__device__ __forceinline__ void vfma(float (&o)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 2)
      unpair(fma2(pair(a[v], a[v + 1]), pair(b[v], b[v + 1]), pair(c[v], c[v + 1])), o[v], o[v + 1]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = fmaf(a[v], b[v], c[v]);
  }
}
template <int V>
__device__ __forceinline__ void vmul(float (&o)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 2) unpair(mul2(pair(a[v], a[v + 1]), pair(b[v], b[v + 1])), o[v], o[v + 1]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = a[v] * b[v];
  }
}
template <int V>
__device__ __forceinline__ void vadd(float (&o)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 2) unpair(add2(pair(a[v], a[v + 1]), pair(b[v], b[v + 1])), o[v], o[v + 1]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = a[v] + b[v];
  }
}
template <int V>
__device__ __forceinline__ void vset(float (&o)[V], float a) {
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = a;
}
template <class T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& p, float (&o)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = to_f(p.v[v]);
}
template <class T, int V>
__device__ __forceinline__ Pack<T, V> pack(const float (&o)[V]) {
  Pack<T, V> p;
  if constexpr (V % 2 == 0 && std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
    for (int v = 0; v < V; v += 2)
      *reinterpret_cast<__nv_bfloat162*>(&p.v[v]) = __floats2bfloat162_rn(o[v], o[v + 1]);
  } else if constexpr (V % 2 == 0 && std::is_same_v<T, __half>) {
#pragma unroll
    for (int v = 0; v < V; v += 2) *reinterpret_cast<__half2*>(&p.v[v]) = __floats2half2_rn(o[v], o[v + 1]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) p.v[v] = from_f<T>(o[v]);
  }
  return p;
}

// 1 / (1 + exp(-v)) with the special-function exponential and reciprocal: off by
// (6 + 3 |v|) 2^-24 relative to itself, since v log2 e is rounded before the
// exponential (0 from v = -87.3 down, where it is below 2^-126), at a quarter of
// the instructions of expf and a division, which would bound the 16-bit forms.
template <int V>
__device__ __forceinline__ void sigmoid(float (&o)[V], const float (&v)[V]) {
  float k[V], one[V];
  vset(k, -1.4426950408889634f);
  vset(one, 1.f);
  vmul(o, v, k);
#pragma unroll
  for (int i = 0; i < V; ++i) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(o[i]) : "f"(o[i]));
  vadd(o, o, one);
#pragma unroll
  for (int i = 0; i < V; ++i) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(o[i]) : "f"(o[i]));
}

// Calls f with a value of the element type `dtype` names.
template <class F>
void with_type(int32_t dtype, F&& f) {
  if (dtype == FHE_F32) f(float{});
  else if (dtype == FHE_BF16) f(__nv_bfloat16{});
  else if (dtype == FHE_F16) f(__half{});
  else require(false, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
}

}  // namespace fhe
