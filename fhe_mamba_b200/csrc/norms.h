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
  int stages;       // rows in the ring
  uint32_t lanes;   // of a narrow row
};

// Eight elements as 32-bit words, in memory's order.
template <class T>
struct alignas(16) Eight {
  static constexpr int kWords = sizeof(T) * 2, kQuads = kWords / 4;  // of 4 and of 16 bytes
  uint32_t w[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void floats(float (&o)[8]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        o[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        o[2 * i] = f.x, o[2 * i + 1] = f.y;
      } else {
        o[2 * i] = __uint_as_float(w[i] << 16), o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(f[i]);
      } else if constexpr (std::is_same_v<T, __half>) {
        const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
  }
};

// How a row's (or group's) channels lie over lanes: N chunks of 256 to a warp, or in
// narrow rows (up to 128 channels) one of eight to each of `lanes` lanes and several
// rows to a warp.  Chunk c of a lane holds the channels from(): + c 256 .. + 8 where
// 16-byte words are loaded or rows are narrow, four pairs 64 apart where rows and
// widths are even, + (c 8 + i) 32 otherwise; they read consecutive memory across a
// warp, at constant distances.  (25000 rows of 1002, bfloat16 on float32: 61 us by
// pairs, 77 by single elements, gradients 64 and 86.)
enum { kSingles = 0, kWords = 1, kNarrowSingles = 2, kNarrowWords = 3, kPairs = 4 };
constexpr bool is_words(int lay) { return lay == kWords || lay == kNarrowWords; }
constexpr bool is_narrow(int lay) { return lay == kNarrowSingles || lay == kNarrowWords; }

template <int N, int LAY>
__device__ __forceinline__ uint32_t from(uint32_t lanes) {
  if constexpr (is_narrow(LAY)) return (threadIdx.x & (lanes - 1)) * 8;
  return (threadIdx.x >> 5) * (N * 256) + (threadIdx.x & 31) * (is_words(LAY) ? 8 : LAY == kPairs ? 2 : 1);
}
template <int LAY>
__host__ __device__ constexpr int away(int c, int i) {
  return LAY == kSingles ? (c * 8 + i) * 32 : LAY == kPairs ? (c * 4 + i / 2) * 64 + i % 2 : c * 256 + i;
}
// Chunk c of the lane's channels at p; `left` of them are before the row's end, the
// others stay as they are.
template <int LAY, class T>
__device__ __forceinline__ void load_chunk(Eight<T>& e, const T* p, int c, int left) {
  if constexpr (is_words(LAY)) {
    if (away<LAY>(c, 0) < left) {
#pragma unroll
      for (int k = 0; k < Eight<T>::kQuads; ++k)
        reinterpret_cast<uint4*>(e.w)[k] = reinterpret_cast<const uint4*>(p + away<LAY>(c, 0))[k];
    }
  } else if constexpr (LAY == kPairs) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (away<LAY>(c, i) >= left) continue;  // a pair lies before the row's end, or behind
      if constexpr (sizeof(T) == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p + away<LAY>(c, i));
        e.w[i] = v.x, e.w[i + 1] = v.y;
      } else {
        e.w[i / 2] = *reinterpret_cast<const uint32_t*>(p + away<LAY>(c, i));
      }
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (away<LAY>(c, i) < left) e.w[i] = reinterpret_cast<const uint32_t*>(p)[away<LAY>(c, i)];
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = away<LAY>(c, i) < left ? q[away<LAY>(c, i)] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.w[i] = v[2 * i] | v[2 * i + 1] << 16;
  }
}
template <int LAY, class T>
__device__ __forceinline__ void store_chunk(const Eight<T>& e, T* p, int c, int left) {
  if constexpr (is_words(LAY)) {
    if (away<LAY>(c, 0) < left) {
#pragma unroll
      for (int k = 0; k < Eight<T>::kQuads; ++k)
        reinterpret_cast<uint4*>(p + away<LAY>(c, 0))[k] = reinterpret_cast<const uint4*>(e.w)[k];
    }
  } else if constexpr (LAY == kPairs) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (away<LAY>(c, i) >= left) continue;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint2*>(p + away<LAY>(c, i)) = make_uint2(e.w[i], e.w[i + 1]);
      else *reinterpret_cast<uint32_t*>(p + away<LAY>(c, i)) = e.w[i / 2];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (away<LAY>(c, i) >= left) continue;
      if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[away<LAY>(c, i)] = e.w[i];
      else reinterpret_cast<uint16_t*>(p)[away<LAY>(c, i)] = (uint16_t)(e.w[i / 2] >> (i % 2 * 16));
    }
  }
}

// A warp's ring in shared memory: rows of `words` 16-byte words a lane, filled by
// asynchronous copies.  Arrays lie in it as in memory, chunk by chunk, and each
// copy of a warp takes whole lines: with float32 a lane copies words that its
// neighbours read (two of its own lie in one sector, which a second copy would fetch
// again).  So the warp meets behind its waits and before it fills a row again.
// Words past the row's end hold 0.
template <int WORDS>
struct Ring {
  uint32_t base;
  static constexpr uint32_t kRow = WORDS * 512;  // bytes of a warp's row
  __device__ __forceinline__ Ring(const void* shared, int stages) {
    const uint32_t warp = threadIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
    base = (uint32_t)__cvta_generic_to_shared(shared) + warp * stages * kRow + (threadIdx.x & 31) * 16;
  }
  // Word k of chunk c that this lane copies, from the lane's own channels on.
  template <class T>
  __device__ __forceinline__ static int word(int c, int k) {
    return away<kWords>(c, 0) + (Eight<T>::kQuads == 2 ? k * 128 - (int)(threadIdx.x & 31) * 4 : 0);
  }
  // Chunk c of an array whose words start at `first`.
  template <class T>
  __device__ __forceinline__ void copy(int stage, int first, const T* p, int c, int left) const {
    constexpr int Q = Eight<T>::kQuads;
#pragma unroll
    for (int k = 0; k < Q; ++k)
      if (word<T>(c, k) < left)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + stage * kRow + (first + c * Q + k) * 512),
                     "l"(p + word<T>(c, k)) : "memory");
  }
  template <class T>
  __device__ __forceinline__ void take(Eight<T>& e, int stage, int first, int c) const {
    constexpr int Q = Eight<T>::kQuads;
    const uint32_t at = base + stage * kRow + (first + c * Q) * 512 + (Q == 2 ? (threadIdx.x & 31) * 16 : 0);
#pragma unroll
    for (int k = 0; k < Q; ++k)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(e.w[4 * k]), "=r"(e.w[4 * k + 1]), "=r"(e.w[4 * k + 2]), "=r"(e.w[4 * k + 3])
                   : "r"(at + k * 16) : "memory");
  }
  // 0 where no copy of chunk c goes, in every row.
  template <class T>
  __device__ __forceinline__ void blank(int stages, int first, const T*, int c, int left) const {
    constexpr int Q = Eight<T>::kQuads;
#pragma unroll
    for (int k = 0; k < Q; ++k)
      if (word<T>(c, k) >= left)
        for (int stage = 0; stage < stages; ++stage)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(base + stage * kRow + (first + c * Q + k) * 512), "r"(0)
                       : "memory");
  }
};

// The sigmoid of gates of type A: the fast form, whose error of (6 + 3 |v|) 2^-24 vanishes
// behind a 16-bit gate's own rounding.  float32 gates keep 8 2^-24 whatever v is: 2^d for
// the rounded d = -v log2 e is off by the factor e^(-v - d ln 2), 1 + its exponent here
// (5000 x 1536 float32 from memory: 18.2 us, 17.6 without; from the second cache 18.5,
// 16.5, and 28 with expf and a rounded reciprocal).  Exponents are kept where all of that
// is finite; below -88.5 the reciprocal is 0 as without, and an infinite or NaN v comes
// back with the product that SiLU is.
template <class A, int V>
__device__ __forceinline__ void gate_sigmoid(float (&o)[V], const float (&v)[V]) {
  if constexpr (sizeof(A) == 4) {
    float log2e[V], ln2[V], low[V], one[V], t[V], d[V];
    vset(log2e, 1.4426950408889634f);
    vset(ln2, -0.6931471805599453f);
    vset(low, 1.9046543e-9f);  // that float less -ln 2
    vset(one, 1.f);
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = fminf(fmaxf(-v[i], -128.f), 88.5f);
    vmul(d, t, log2e);
#pragma unroll
    for (int i = 0; i < V; ++i) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(o[i]) : "f"(d[i]));
    vfma(t, d, ln2, t);
    vfma(t, d, low, t);
    vfma(o, o, t, o);
    vadd(o, o, one);
#pragma unroll
    for (int i = 0; i < V; ++i) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(o[i]) : "f"(o[i]));
  } else {
    sigmoid(o, v);
  }
}

// Waits until all but the last `stages` - 1 (0 or 1) groups of the warp's copies are there.
__device__ __forceinline__ void wait_copies(int stages) {
  if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
}

// Sum over the threads of a row, one value for all of them: some lanes, a warp, or
// all warps of the block by two sets of partial sums used in turn.
template <bool NARROW>
struct RowSum {
  float (*red)[16];
  uint32_t lanes;
  int turn = 0;
  __device__ __forceinline__ float operator()(float v) {
    if constexpr (NARROW) {
      for (uint32_t o = lanes / 2; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
    } else {
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
      if (blockDim.x == 32) return v;
      float* r = red[turn];
      turn ^= 1;
      if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
      __syncthreads();
      v = 0.f;
      for (uint32_t w = 0; w < blockDim.x / 32; ++w) v += r[w];
    }
    return v;
  }
};

// Warps per row and chunks of eight channels per thread.  Few rows are spread over
// as many warps as have a chunk.  Else a thread takes three chunks where that fills
// every lane, else four (single elements and gradients through a gate, which need more
// registers: two; 40000 x 1024 bfloat16 gradients 79 us, 104); at most 16 warps.
// Four rows of one warp share a block, a longer row has its own.  Narrow rows share a
// warp (5938332 rows of one channel with a gate and gradients: 0.3 ms, 4.2 with a warp
// each).
struct NormShape {
  uint32_t warps, chunks, rows_per_block, lanes;
  int layout(uint32_t together) const {  // elements that may be loaded together: 8, 2 or 1
    if (lanes < 32) return together == 8 ? kNarrowWords : kNarrowSingles;
    return together == 8 ? kWords : together == 2 ? kPairs : kSingles;
  }
};
inline NormShape norm_shape(uint32_t gw, uint64_t rows, uint32_t together, bool heavy = false) {
  const bool vec = together == 8;
  const uint32_t all = (gw + 7) / 8;
  if (all <= 16) {
    uint32_t lanes = 1;
    while (lanes < all) lanes *= 2;
    return {1, 1, 4 * 32 / lanes, lanes};
  }
  const bool whole = vec && all % 96 == 0 && all / 96 <= 8;
  const uint32_t want = rows < 2 * 148 ? 1 : whole ? 3 : vec && !heavy ? 4 : 2;
  NormShape s;
  s.warps = std::min(16u, (all + 32 * want - 1) / (32 * want));
  s.chunks = (all + 32 * s.warps - 1) / (32 * s.warps);
  if (s.chunks == 3 && (!vec || s.warps > 8)) s.chunks = 4;
  s.rows_per_block = s.warps == 1 ? 4 : 1;
  s.lanes = 32;
  return s;
}

constexpr uint32_t kSmShared = 227 * 1024, kBlockShared = 1024 + 256;  // of an SM; of a block beside its ring, which has the rest at most

// Rows in the ring and blocks an SM for blocks of `warps` warps whose row takes `row`
// bytes: two rows, and as many blocks as bring the rings to about `target` bytes but 8
// warps at least.  More traffic in flight is slower, not faster: 32768 x 1536 bfloat16
// with a gate, gradients, two rows: 93 us with 8 warps (74 KB), 80 with 12 (110 KB), 88
// with 16, 102 with 20; forward 62, 53, 50 and 53 us.
struct RingPlan {
  uint32_t stages, blocks;
};
inline RingPlan ring_plan(uint32_t row, uint32_t warps, uint32_t target) {
  RingPlan p{2, 1};
  if (2 * row + kBlockShared > kSmShared) p.stages = 1;
  const uint32_t block = p.stages * row, most = std::max(1u, kSmShared / (block + kBlockShared));
  p.blocks = std::min(most, std::max(target / block, (8 + warps - 1) / warps));
  return p;
}

// Elements that may be loaded together from every one of these arrays: 8 (16-byte
// words), 2 or 1.
struct Together {
  uint32_t n;
  explicit Together(uint32_t gw) : n(gw % 8 == 0 ? 8 : gw % 2 == 0 ? 2 : 1) {}
  void with(const void* p, int64_t stride, uint32_t elem) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    if (n == 8 && (at % 16 || stride % (int64_t)(16 / elem))) n = 2;
    if (n == 2 && (at % (2 * elem) || stride % 2)) n = 1;
  }
};

void check_norm(const fhe_rms_norm_args& a);
NormArgs norm_args(const fhe_rms_norm_args& a);
inline int norm_mode(const fhe_rms_norm_args& a) {
  return a.gate ? kNormGate : !a.residual ? kNormPlain : a.channel_scale ? kNormAddScaled : kNormAdd;
}

// Calls f(mode, A{}, H{}, chunks, layout) with constants: the activations' and the
// stream's type, chunks per thread, the layout.
template <class F>
void with_norm(const fhe_rms_norm_args& a, uint32_t chunks, int layout, F&& f) {
  auto shape = [&](auto mode, auto act, auto str) {
    auto with = [&](auto n, auto lay) { f(mode, act, str, n, lay); };
    using std::integral_constant;
    if (layout == kNarrowSingles) with(integral_constant<int, 1>{}, integral_constant<int, kNarrowSingles>{});
    else if (layout == kNarrowWords) with(integral_constant<int, 1>{}, integral_constant<int, kNarrowWords>{});
    else if (layout == kPairs && chunks == 1) with(integral_constant<int, 1>{}, integral_constant<int, kPairs>{});
    else if (layout == kPairs && chunks == 2) with(integral_constant<int, 2>{}, integral_constant<int, kPairs>{});
    else if (layout == kPairs) with(integral_constant<int, 4>{}, integral_constant<int, kPairs>{});
    else if (layout == kSingles && chunks == 1) with(integral_constant<int, 1>{}, integral_constant<int, kSingles>{});
    else if (layout == kSingles && chunks == 2) with(integral_constant<int, 2>{}, integral_constant<int, kSingles>{});
    else if (layout == kSingles) with(integral_constant<int, 4>{}, integral_constant<int, kSingles>{});
    else if (chunks == 1) with(integral_constant<int, 1>{}, integral_constant<int, kWords>{});
    else if (chunks == 2) with(integral_constant<int, 2>{}, integral_constant<int, kWords>{});
    else if (chunks == 3) with(integral_constant<int, 3>{}, integral_constant<int, kWords>{});
    else with(integral_constant<int, 4>{}, integral_constant<int, kWords>{});
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
