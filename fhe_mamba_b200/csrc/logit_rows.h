// Rows of logits in 16-byte words, and the order of their entries.
#pragma once
#include "mamba_ops.h"

namespace fhe {

// Order of two entries: larger value first, then the lower index; NaN last,
// -0 equal to 0.  The value as an unsigned key in ascending order.
__device__ __forceinline__ uint32_t order_key(float z) {
  if (isnan(z)) return 0u;
  const uint32_t u = __float_as_uint(z + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ bool before(uint32_t ka, uint32_t ia, uint32_t kb, uint32_t ib) {
  return ka > kb || (ka == kb && ia < ib);
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// What entries are raised to before they are summed: finite, and so far below
// every maximum that counts that nothing is left of it.
template <class T>
__device__ __forceinline__ float floor_of() {
  return std::is_same_v<T, __half> ? -65504.f : -1e38f;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// A 16-byte load of a row as four words, kept as words until its elements are
// needed: maxima and the floor of the 16-bit types work on two at a time.
template <class T>
struct Quad {
  static constexpr int kElems = 16 / sizeof(T), kPer = 4 / sizeof(T);  // elements, elements per word
  uint32_t w[4];
  __device__ __forceinline__ static uint32_t minus_inf() {
    if constexpr (sizeof(T) == 4) return 0xff800000u;
    else return std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
  }
  __device__ __forceinline__ void load(const T* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = minus_inf();
  }
  // Elements i * kPer + 0 (and 1) of a word.
  __device__ __forceinline__ static void floats(uint32_t x, float (&f)[kPer]) {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(x);
    } else if constexpr (std::is_same_v<T, __half>) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&x));
      f[0] = v.x, f[1] = v.y;
    } else {
      f[0] = __uint_as_float(x << 16), f[1] = __uint_as_float(x & 0xffff0000u);
    }
  }
  __device__ __forceinline__ float element(int e) const {
    float f[kPer];
    floats(w[e / kPer], f);
    return f[e % kPer];
  }
  __device__ __forceinline__ static uint32_t max_words(uint32_t a, uint32_t b) {  // NaN if either is
    uint32_t r;
    if constexpr (sizeof(T) == 4) asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (std::is_same_v<T, __half>) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ uint32_t max_word() const {
    return max_words(max_words(w[0], w[1]), max_words(w[2], w[3]));
  }
  __device__ __forceinline__ static float max_of(uint32_t x) {
    float f[kPer];
    floats(x, f);
    if constexpr (kPer == 1) return f[0];
    else return max_nan(f[0], f[1]);
  }
  // Adds the elements, all below m, to the sums in base 2; `shift` = -shift_of(m).
  __device__ __forceinline__ void add(uint64_t& s, uint64_t& u, float shift) const {
    const uint64_t k = pair(kLog2e, kLog2e), sh = pair(shift, shift);
    uint32_t low;
    if constexpr (sizeof(T) == 4) low = __float_as_uint(floor_of<T>());
    else low = std::is_same_v<T, __half> ? 0xfbfffbffu : 0xfe96fe96u;  // -65504; -1e38 rounded
#pragma unroll
    for (int i = 0; i < kElems / 2; ++i) {
      float f[2];
      if constexpr (sizeof(T) == 4) {
        f[0] = fmaxf(__uint_as_float(w[2 * i]), floor_of<T>());
        f[1] = fmaxf(__uint_as_float(w[2 * i + 1]), floor_of<T>());
      } else {
        uint32_t x;
        if constexpr (std::is_same_v<T, __half>) asm("max.f16x2 %0, %1, %2;" : "=r"(x) : "r"(w[i]), "r"(low));
        else asm("max.bf16x2 %0, %1, %2;" : "=r"(x) : "r"(w[i]), "r"(low));
        floats(x, f);
      }
      const uint64_t d = fma2(pair(f[0], f[1]), k, sh);
      float d0, d1;
      unpair(d, d0, d1);
      const uint64_t e = pair(exp2_fast(d0), exp2_fast(d1));
      s = add2(s, e);
      u = fma2(e, d, u);
    }
  }
};

}  // namespace fhe
