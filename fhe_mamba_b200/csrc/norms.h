// What the norms and their gradients share: arguments, the layout of a row over
// threads, and the choice of it.
#pragma once
#include <algorithm>

#include "mamba_ops.h"

namespace fhe {

enum { kNormPlain = 0, kNormAdd = 1, kNormAddScaled = 2, kNormGate = 3 };
constexpr uint32_t kMaxNormWidth = 16384;  // channels of a group

struct NormArgs {
  const void *x, *res, *gate;
  int64_t xs, rs, gs;
  const float *cscale, *weight;
  void *y, *h;
  float* rstd;
  const void *dy, *dh;
  void *dx, *dres, *dgate;
  float* part;  // sums of each block: [grid.x][width] for the weight, then as much for the channel scale
  uint32_t rows, width, gw, groups;
  float eps, scale;
  int stages;  // rows in the gradients' ring
};

// Eight elements as 16-byte words (or, where alignment does not allow that,
// element by element).
template <class T>
struct alignas(16) Eight {
  T v[8];
  __device__ __forceinline__ void floats(float (&o)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = to_f(v[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    const Pack<T, 8> p = pack<T, 8>(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p.v[i];
  }
};

// A row's (or group's) channels over T = blockDim.x threads: chunk c of thread t
// holds channels (c T + t) 8 .. + 8 where words are loaded, (c 8 + i) T + t
// otherwise; both read consecutive memory across a warp.
template <bool VEC>
__device__ __forceinline__ uint32_t channel(int c, int i) {
  return VEC ? (c * blockDim.x + threadIdx.x) * 8 + i : (c * 8 + i) * blockDim.x + threadIdx.x;
}
template <bool VEC, class T>
__device__ __forceinline__ void load_chunk(Eight<T>& e, const T* p, int c, uint32_t gw) {
  if constexpr (VEC) {
    const uint32_t at = channel<true>(c, 0);
    if (at < gw) {
      const uint4* s = reinterpret_cast<const uint4*>(p + at);
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(&e)[k] = s[k];
      return;
    }
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(&e)[k] = make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = channel<false>(c, i) < gw ? p[channel<false>(c, i)] : from_f<T>(0.f);
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void store_chunk(const Eight<T>& e, T* p, int c, uint32_t gw) {
  if constexpr (VEC) {
    const uint32_t at = channel<true>(c, 0);
    if (at >= gw) return;
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k)
      reinterpret_cast<uint4*>(p + at)[k] = reinterpret_cast<const uint4*>(&e)[k];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (channel<false>(c, i) < gw) p[channel<false>(c, i)] = e.v[i];
  }
}

// Sum over the threads of a row, one value for all of them: a warp, or all warps
// of the block by two sets of partial sums used in turn.
struct RowSum {
  float (*red)[16];
  int turn = 0;
  __device__ __forceinline__ float operator()(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (blockDim.x == 32) return v;
    float* r = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) v += r[w];
    return v;
  }
};

// Warps per row and chunks of eight channels per thread.  Few rows are spread over
// as many warps as have a chunk.  Else a thread takes three chunks where that fills
// every lane, else four (single elements, which need more registers: two); at most 16
// warps.  Four rows of one warp share a block, a longer row has its own.
struct NormShape {
  uint32_t warps, chunks, rows_per_block;
};
inline NormShape norm_shape(uint32_t gw, uint64_t rows, bool vec) {
  const uint32_t all = (gw + 7) / 8;
  const bool whole = vec && all % 96 == 0 && all / 96 <= 8;
  const uint32_t want = rows < 2 * 148 ? 1 : whole ? 3 : vec ? 4 : 2;
  NormShape s;
  s.warps = std::min(16u, (all + 32 * want - 1) / (32 * want));
  s.chunks = (all + 32 * s.warps - 1) / (32 * s.warps);
  if (s.chunks == 3 && (!vec || s.warps > 8)) s.chunks = 4;
  s.rows_per_block = s.warps == 1 ? 4 : 1;
  return s;
}

inline bool norm_aligned(const void* p, int64_t stride, uint32_t elem) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % (int64_t)(16 / elem) == 0;
}

void check_norm(const fhe_rms_norm_args& a);
NormArgs norm_args(const fhe_rms_norm_args& a);
inline int norm_mode(const fhe_rms_norm_args& a) {
  return a.gate ? kNormGate : !a.residual ? kNormPlain : a.channel_scale ? kNormAddScaled : kNormAdd;
}

// Calls f(mode, A{}, H{}, chunks, words) with constants: the activations' and the
// stream's type, chunks per thread, whether 16-byte words are loaded.
template <class F>
void with_norm(const fhe_rms_norm_args& a, uint32_t chunks, bool vec, F&& f) {
  auto shape = [&](auto mode, auto act, auto str) {
    if (!vec) {
      if (chunks == 1) f(mode, act, str, std::integral_constant<int, 1>{}, std::false_type{});
      else if (chunks == 2) f(mode, act, str, std::integral_constant<int, 2>{}, std::false_type{});
      else f(mode, act, str, std::integral_constant<int, 4>{}, std::false_type{});
      return;
    }
    if (chunks == 1) f(mode, act, str, std::integral_constant<int, 1>{}, std::true_type{});
    else if (chunks == 2) f(mode, act, str, std::integral_constant<int, 2>{}, std::true_type{});
    else if (chunks == 3) f(mode, act, str, std::integral_constant<int, 3>{}, std::true_type{});
    else f(mode, act, str, std::integral_constant<int, 4>{}, std::true_type{});
  };
  with_type(a.dtype, [&](auto act) {
    auto stream = [&](auto mode) {
      if (a.stream_dtype == FHE_F32) shape(mode, act, float{});
      else shape(mode, act, act);
    };
    switch (norm_mode(a)) {
      case kNormPlain: stream(std::integral_constant<int, kNormPlain>{}); break;
      case kNormAdd: stream(std::integral_constant<int, kNormAdd>{}); break;
      case kNormAddScaled: stream(std::integral_constant<int, kNormAddScaled>{}); break;
      default: shape(std::integral_constant<int, kNormGate>{}, act, act);
    }
  });
}

}  // namespace fhe
