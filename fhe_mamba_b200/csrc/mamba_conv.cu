// Causal depthwise convolution of the Mamba-2 layer (fhe_causal_conv) and its
// gradients, channels innermost.
//
// y_t = act(bias + sum_i w_i row_(t+i)) with row = [initial_state; x]: a few
// multiplies per element read and written, so memory bounds it.  A thread
// keeps the last taps - 1 elements of a few neighbouring channels in
// registers and walks a run of tokens, so each element is loaded once (and
// taps - 1 of them once more at each run's start, from the cache).
#include <algorithm>

#include "launch_count.h"
#include "mamba_ops.h"

namespace fhe {
namespace {

constexpr int kThreads = 128;

struct ConvArgs {
  const void* x;
  int64_t sb, sl;
  const void *weight, *bias, *initial;
  const int32_t* lengths;
  void *y, *final_state;
  uint32_t batch, length, channels, run, runs;
  uint64_t walkers;  // threads that walk tokens; later ones copy the final state
};

// Row element: t < 0 is the initial state's entry t + K - 1.
template <class T, int V, int K>
__device__ __forceinline__ void load_row(const T* x, const T* init, int64_t sl, uint32_t channels, int t,
                                         float (&o)[V]) {
  const T* p = t >= 0 ? x + (int64_t)t * sl : init ? init + (int64_t)(t + K - 1) * channels : nullptr;
  if (p) unpack(*reinterpret_cast<const Pack<T, V>*>(p), o);
  else vset(o, 0.f);
}

// w[i]: tap i of V channels; the taps of V channels lie together.
template <class T, int V, int K>
__device__ __forceinline__ void load_taps(const void* weight, uint32_t c, float (&w)[K][V]) {
  const T* p = static_cast<const T*>(weight) + (int64_t)c * K;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p + j * V);
#pragma unroll
    for (int v = 0; v < V; ++v) w[(j * V + v) % K][(j * V + v) / K] = to_f(k.v[v]);
  }
}
template <class T, int V>
__device__ __forceinline__ void load_bias(const void* bias, uint32_t c, float (&o)[V]) {
  if (bias) unpack(*reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(bias) + c), o);
  else vset(o, 0.f);
}

// A thread's own tokens on their way to it: batches of kAhead packs go to its
// slots of a ring in shared memory by asynchronous copies, so that RING - 1
// batches are in flight without holding registers.  No thread reads another's
// slots, so no barrier is needed.  8 x 4096 tokens of 1792 bfloat16 channels, 4
// taps: 45 us, 5.2 TB/s (60 us with the batches in registers, half of them in
// flight).
constexpr int kAhead = 4;
template <class T, int V>
__device__ __forceinline__ void copy_pack(Pack<T, V>* to, const T* from) {
  constexpr int kBytes = V * sizeof(T);
  const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
template <class T, int V>
constexpr bool kCopies = V * sizeof(T) >= 4;  // the smallest asynchronous copy

// Thread = V channels x one run of tokens, channels fastest.  `STEP` (one
// token): the same thread also writes the window behind it, so the state may
// be updated in place.
template <class T, int V, int K, bool SILU, bool STEP>
__global__ void __launch_bounds__(kThreads) k_conv(const ConvArgs g) {
  uint64_t id = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  const uint32_t groups = g.channels / V;
  if (id >= g.walkers) {
    if constexpr (!STEP && K > 1) {
      id -= g.walkers;
      if (id >= (uint64_t)g.batch * (K - 1) * g.channels) return;
      const uint32_t c = id % g.channels, j = id / g.channels % (K - 1), b = id / g.channels / (K - 1);
      const int t = clamp_length(g.lengths, b, g.length) + (int)j - (K - 1);
      T v = from_f<T>(0.f);
      if (t >= 0) v = static_cast<const T*>(g.x)[(int64_t)b * g.sb + (int64_t)t * g.sl + c];
      else if (g.initial) v = static_cast<const T*>(g.initial)[((int64_t)b * (K - 1) + t + K - 1) * g.channels + c];
      static_cast<T*>(g.final_state)[id] = v;
    }
    return;
  }
  const uint32_t c = id % groups * V;
  id /= groups;
  const uint32_t run = id % g.runs, b = id / g.runs;
  const int len = clamp_length(g.lengths, b, g.length);
  const int t0 = run * g.run, t1 = min(t0 + g.run, g.length);
  const T* x = static_cast<const T*>(g.x) + (int64_t)b * g.sb + c;
  const T* init = g.initial ? static_cast<const T*>(g.initial) + (int64_t)b * (K - 1) * g.channels + c : nullptr;
  float w[K][V], bias[V], win[K][V];
#pragma unroll
  for (int i = 0; i < K - 1; ++i) {
    const int t = t0 + i - (K - 1);
    if (t < len) load_row<T, V, K>(x, init, g.sl, g.channels, t, win[i + 1]);
  }
  load_taps<T, V, K>(g.weight, c, w);
  load_bias<T, V>(g.bias, c, bias);
  T* y = static_cast<T*>(g.y) + ((int64_t)b * g.length + t0) * g.channels + c;
  auto token = [&](const Pack<T, V>& in) {  // win moves on by one token
    float o[V];
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) win[i][v] = win[i + 1][v];
    unpack(in, win[K - 1]);
    vfma(o, w[0], win[0], bias);
#pragma unroll
    for (int i = 1; i < K; ++i) vfma(o, w[i], win[i], o);
    if constexpr (SILU) {
      float e[V];
      sigmoid(e, o);
      vmul(o, o, e);
    }
    *reinterpret_cast<Pack<T, V>*>(y) = pack<T>(o);
    y += g.channels;
  };
  int t = t0;
  const int t_live = min(t1, len);
  const T* xt = x + (int64_t)t * g.sl;
  if constexpr (!STEP) {
    if constexpr (kCopies<T, V>) {
      constexpr int kRing = 4;
      __shared__ Pack<T, V> ring[kRing][kAhead][kThreads];
      const int batches = t_live > t ? (t_live - t) / kAhead : 0;
      auto fetch = [&](int i) {
        if (i < batches) {
#pragma unroll
          for (int j = 0; j < kAhead; ++j, xt += g.sl) copy_pack(&ring[i % kRing][j][threadIdx.x], xt);
        }
        copies_done();
      };
#pragma unroll
      for (int i = 0; i < kRing - 1; ++i) fetch(i);
      for (int i = 0; i < batches; ++i) {
        wait_copies<kRing - 2>();
        Pack<T, V> in[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) in[j] = ring[i % kRing][j][threadIdx.x];
        fetch(i + kRing - 1);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) token(in[j]);
      }
      t += batches * kAhead;
    }
  }
  for (; t < t_live; ++t, xt += g.sl) token(*reinterpret_cast<const Pack<T, V>*>(xt));
  float zero[V];
  vset(zero, 0.f);
  for (; t < t1; ++t, y += g.channels) *reinterpret_cast<Pack<T, V>*>(y) = pack<T>(zero);
  if constexpr (STEP && K > 1) {
    // an empty sequence keeps its window (win[1..K-1]), else it moved by one (also win[1..K-1] after the shift)
    T* f = static_cast<T*>(g.final_state) + (int64_t)b * (K - 1) * g.channels + c;
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      Pack<T, V> o;
#pragma unroll
      for (int v = 0; v < V; ++v) o.v[v] = from_f<T>(win[i + 1][v]);
      *reinterpret_cast<Pack<T, V>*>(f + (int64_t)i * g.channels) = o;
    }
  }
}

struct ConvGradArgs {
  ConvArgs f;
  const void *dy, *dfinal;
  void *dx, *dinitial;
  float* part;  // [batch * runs][K + 1][channels]: taps, then bias
};

// Thread = V channels x one run of tokens.  It walks the run and taps - 1
// tokens more: dpre_t = dy_t act'(pre_t) enters a window of taps values, and
// drow_u = sum_i w_i dpre_(u-i) (u a row index, u - (K - 1) a token) leaves
// it.  The taps' and bias's gradients of the run's own tokens go to `part`.
// 8 x 1001 tokens of 1792 float32 channels: 44 us, 3.9 TB/s (and 5 for the sums
// of the parts); registers (two windows and the taps' sums) keep it to 20 warps
// an SM.
template <class T, int V, int K, bool SILU>
__global__ void __launch_bounds__(kThreads) k_conv_grad(const ConvGradArgs a) {
  const ConvArgs& g = a.f;
  uint64_t id = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (id >= g.walkers) return;
  const uint32_t groups = g.channels / V;
  const uint32_t c = id % groups * V;
  id /= groups;
  const uint32_t run = id % g.runs, b = id / g.runs;
  const int len = clamp_length(g.lengths, b, g.length);
  const int t0 = run * g.run, t1 = min(t0 + g.run, g.length);
  const T* x = static_cast<const T*>(g.x) + (int64_t)b * g.sb + c;
  const T* init = g.initial ? static_cast<const T*>(g.initial) + (int64_t)b * (K - 1) * g.channels + c : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + (int64_t)b * g.length * g.channels + c;
  const T* dfinal = a.dfinal ? static_cast<const T*>(a.dfinal) + (int64_t)b * (K - 1) * g.channels + c : nullptr;
  T* dx = static_cast<T*>(a.dx) + (int64_t)b * g.length * g.channels + c;
  T* dinit = a.dinitial ? static_cast<T*>(a.dinitial) + (int64_t)b * (K - 1) * g.channels + c : nullptr;
  float w[K][V], bias[V], win[K][V], dp[K][V], dw[K][V], db[V];
  load_taps<T, V, K>(g.weight, c, w);
  load_bias<T, V>(g.bias, c, bias);
  vset(db, 0.f);
#pragma unroll
  for (int i = 0; i < K; ++i) {
    vset(dw[i], 0.f);
    vset(dp[i], 0.f);
    vset(win[i], 0.f);
  }
#pragma unroll
  for (int i = 0; i < K - 1; ++i) {
    const int t = t0 + i - (K - 1);
    if (t < len) load_row<T, V, K>(x, init, g.sl, g.channels, t, win[i + 1]);
  }
  // A token's dpre enters the window; its own tokens also add to the taps'
  // gradients; the row element taps - 1 before it leaves.
  auto slope = [&](const Pack<T, V>& xin, const Pack<T, V>& din) {
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) win[i][v] = win[i + 1][v];
    unpack(xin, win[K - 1]);
    unpack(din, dp[K - 1]);
    if constexpr (SILU) {  // slope e (1 + p (1 - e)) of p e, e = sigmoid(p)
      float p[V], e[V], one[V], f[V];
      vset(one, 1.f);
      vfma(p, w[0], win[0], bias);
#pragma unroll
      for (int i = 1; i < K; ++i) vfma(p, w[i], win[i], p);
      sigmoid(e, p);
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = -p[v];
      vfma(f, f, e, p);  // p - p e
      vadd(f, f, one);
      vmul(f, f, e);
      vmul(dp[K - 1], dp[K - 1], f);
    }
  };
  auto shift = [&] {
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) dp[i][v] = dp[i + 1][v];
  };
  auto taps = [&] {
    vadd(db, db, dp[K - 1]);
#pragma unroll
    for (int i = 0; i < K; ++i) vfma(dw[i], dp[K - 1], win[i], dw[i]);
  };
  // dp[j] holds dpre of token u + j; the gradient of row element u (a token, or below 0 of the initial state)
  auto leave = [&](int u) {
    float o[V];
    const int j = u + (K - 1) - len;
    if (dfinal && j >= 0 && j < K - 1) unpack(*reinterpret_cast<const Pack<T, V>*>(dfinal + (int64_t)j * g.channels), o);
    else vset(o, 0.f);
#pragma unroll
    for (int i = 0; i < K; ++i) vfma(o, w[i], dp[K - 1 - i], o);
    T* out = u >= 0 ? dx + (int64_t)u * g.channels : dinit + (int64_t)(u + K - 1) * g.channels;
    *reinterpret_cast<Pack<T, V>*>(out) = pack<T>(o);
  };
  const int t2 = t1 + K - 1, t_live = min(t2, len);
  const T *xt = x + (int64_t)t0 * g.sl, *dt = dy + (int64_t)t0 * g.channels;
  auto one = [&](int t) {  // any token
    shift();
    if (t < t_live) {
      slope(*reinterpret_cast<const Pack<T, V>*>(xt), *reinterpret_cast<const Pack<T, V>*>(dt));
      if (t < t1) taps();
    } else {
      vset(dp[K - 1], 0.f);
    }
    xt += g.sl;
    dt += g.channels;
    const int u = t - (K - 1);
    if (u >= t0 || (t0 == 0 && dinit)) leave(u);
  };
  int t = t0;
  for (; t < min(t0 + K - 1, t2); ++t) one(t);
  // whole batches of the run's own live tokens, none of whose row elements takes a final state's gradient
  const int t_main = min(t1, len);
  if constexpr (kCopies<T, V>) {
    constexpr int kRing = 3;
    __shared__ Pack<T, V> ring[2][kRing][kAhead][kThreads];
    const int batches = t_main > t ? (t_main - t) / kAhead : 0;
    auto fetch = [&](int i) {
      if (i < batches) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j, xt += g.sl, dt += g.channels) {
          copy_pack(&ring[0][i % kRing][j][threadIdx.x], xt);
          copy_pack(&ring[1][i % kRing][j][threadIdx.x], dt);
        }
      }
      copies_done();
    };
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) fetch(i);
    T* out = dx + (int64_t)(t - (K - 1)) * g.channels;
    for (int i = 0; i < batches; ++i) {
      wait_copies<kRing - 2>();
      Pack<T, V> xin[kAhead], din[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        xin[j] = ring[0][i % kRing][j][threadIdx.x];
        din[j] = ring[1][i % kRing][j][threadIdx.x];
      }
      fetch(i + kRing - 1);
#pragma unroll
      for (int j = 0; j < kAhead; ++j, out += g.channels) {
        shift();
        slope(xin[j], din[j]);
        taps();
        float o[V];
        vmul(o, w[0], dp[K - 1]);
#pragma unroll
        for (int i = 1; i < K; ++i) vfma(o, w[i], dp[K - 1 - i], o);
        *reinterpret_cast<Pack<T, V>*>(out) = pack<T>(o);
      }
    }
    t += batches * kAhead;
  }
  for (; t < t2; ++t) one(t);
  float* part = a.part + ((int64_t)b * g.runs + run) * (K + 1) * g.channels + c;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int i = 0; i < K; ++i) part[(int64_t)i * g.channels + v] = dw[i][v];
    part[(int64_t)K * g.channels + v] = db[v];
  }
}

// Sums the runs' parts in a fixed order: 32 channels x 8 strands of runs.
template <class T>
__global__ void k_conv_grad_sum(const float* part, void* dweight, void* dbias, uint32_t channels, uint32_t taps,
                                uint32_t parts) {
  __shared__ float s[8][33];
  const uint32_t c = blockIdx.x * 32 + threadIdx.x, i = blockIdx.y;
  float v = 0.f;
  if (c < channels)
    for (uint32_t r = threadIdx.y; r < parts; r += 8) v += part[((int64_t)r * (taps + 1) + i) * channels + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < channels) {
    for (int r = 1; r < 8; ++r) v += s[r][threadIdx.x];
    if (i < taps) static_cast<T*>(dweight)[(int64_t)c * taps + i] = from_f<T>(v);
    else if (dbias) static_cast<T*>(dbias)[c] = from_f<T>(v);
  }
}

void check_conv(const fhe_causal_conv_args& a) {
  require(a.dtype == FHE_F32 || a.dtype == FHE_BF16 || a.dtype == FHE_F16, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
  require(a.taps >= 1 && a.taps <= 8, "taps must be in [1, 8]");
  require(a.channels >= 1, "channels must be positive");
  require(a.length <= (1u << 30) && (uint64_t)a.batch * a.length < (1ull << 31) && a.channels < (1u << 24),
          "sizes too large");
}

template <class F>
void with_taps(uint32_t taps, F&& f) {
  switch (taps) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 5: f(std::integral_constant<int, 5>{}); break;
    case 6: f(std::integral_constant<int, 6>{}); break;
    case 7: f(std::integral_constant<int, 7>{}); break;
    default: f(std::integral_constant<int, 8>{}); break;
  }
}

bool aligned(const void* p, uint32_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

ConvArgs conv_args(const fhe_causal_conv_args& a, uint32_t vec, uint32_t least_run) {
  ConvArgs g{};
  g.x = a.x;
  g.sb = a.x_stride[0];
  g.sl = a.x_stride[1];
  g.weight = a.weight;
  g.bias = a.bias;
  g.initial = a.initial_state;
  g.lengths = a.lengths;
  g.y = a.y;
  g.final_state = a.final_state;
  g.batch = a.batch;
  g.length = a.length;
  g.channels = a.channels;
  // runs as long as still leave about 1024 threads per SM
  const uint64_t per_token = (uint64_t)a.batch * (a.channels / vec);
  uint32_t run = 64;
  while (run > least_run && per_token * ((a.length + run - 1) / run) < 148ull * 1024) run /= 2;
  g.run = run;
  g.runs = (a.length + run - 1) / run;
  g.walkers = per_token * g.runs;
  return g;
}

// Channels per thread: 4 (8 or 16 bytes a load: with 8 channels the window and
// taps leave three warps to a scheduler, 71 against 61 us at 8 x 4096 tokens of
// 1792 bfloat16 channels), 1 where channels or alignment do not divide.
uint32_t conv_vec(const fhe_causal_conv_args& a, uint32_t want, const void* p0, const void* p1, const void* p2) {
  const uint32_t e = elem_size(a.dtype);
  const bool ok = a.channels % want == 0 && a.x_stride[0] % want == 0 && a.x_stride[1] % want == 0 &&
                  aligned(a.x, want * e) && aligned(a.initial_state, want * e) && aligned(a.weight, want * e) &&
                  aligned(a.bias, want * e) && aligned(p0, want * e) &&
                  aligned(p1, want * e) && aligned(p2, want * e);
  return ok ? want : 1;
}

uint32_t grad_runs(const fhe_causal_conv_args& a, uint32_t vec) { return conv_args(a, vec, 16).runs; }

}  // namespace

void causal_conv(const fhe_causal_conv_args& a) {
  check_conv(a);
  if (a.batch == 0) return;
  require(a.weight != nullptr, "null weight");
  require(a.length == 0 || (a.x && a.y), "null input or output");
  require(a.taps == 1 || a.final_state, "null final_state");
  require(a.length <= 1 || a.taps == 1 || a.final_state != a.initial_state,
          "final_state may be initial_state's memory only for one token");
  DeviceGuard dev(a.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  with_type(a.dtype, [&](auto tv) {
    using T = decltype(tv);
    constexpr int kVec = 4;
    const uint32_t vec = conv_vec(a, kVec, a.y, a.length == 1 ? a.final_state : nullptr, nullptr);
    ConvArgs g = conv_args(a, vec, 4);
    const bool step = a.length == 1;
    if (a.length == 0 && a.final_state == a.initial_state) return;
    const uint64_t threads = g.walkers + (step ? 0 : (uint64_t)a.batch * (a.taps - 1) * a.channels);
    const uint64_t blocks = (threads + kThreads - 1) / kThreads;
    if (blocks == 0) return;
    require(blocks < (1ull << 31), "too many blocks");
    with_taps(a.taps, [&](auto kv) {
      constexpr int K = decltype(kv)::value;
      auto go = [&](auto vv, auto silu, auto one) {
        k_conv<T, decltype(vv)::value, K, decltype(silu)::value, decltype(one)::value>
            <<<(uint32_t)blocks, kThreads, 0, st>>>(g);
      };
      auto with_vec = [&](auto silu, auto one) {
        if (vec == 1) go(std::integral_constant<int, 1>{}, silu, one);
        else go(std::integral_constant<int, kVec>{}, silu, one);
      };
      auto with_silu = [&](auto one) {
        if (a.silu) with_vec(std::true_type{}, one);
        else with_vec(std::false_type{}, one);
      };
      if (step) with_silu(std::true_type{});
      else with_silu(std::false_type{});
    });
    note_launch();
    FHE_CUDA(cudaGetLastError());
  });
}

uint64_t causal_conv_backward_workspace(const fhe_causal_conv_grad_args& g) {
  check_conv(g.f);
  // more channels to a thread, fewer threads, shorter runs: 4 has the most of them
  const uint64_t runs = std::max(grad_runs(g.f, 1), grad_runs(g.f, 4));
  return g.f.batch * runs * (g.f.taps + 1) * g.f.channels * sizeof(float);
}

void causal_conv_backward(const fhe_causal_conv_grad_args& a) {
  check_conv(a.f);
  require(a.f.weight != nullptr && a.dweight != nullptr, "null weight");
  require(a.f.batch == 0 || a.f.length == 0 || (a.f.x && a.dy && a.dx), "null input or output");
  check_workspace(a.workspace, a.workspace_bytes, causal_conv_backward_workspace(a));
  DeviceGuard dev(a.f.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  const uint32_t e = elem_size(a.f.dtype);
  const size_t state_bytes = (size_t)a.f.batch * (a.f.taps - 1) * a.f.channels * e;
  if (a.f.batch == 0 || a.f.length == 0) {
    FHE_CUDA(cudaMemsetAsync(a.dweight, 0, (size_t)a.f.channels * a.f.taps * e, st));
    if (a.dbias) FHE_CUDA(cudaMemsetAsync(a.dbias, 0, (size_t)a.f.channels * e, st));
    if (a.dinitial && state_bytes) {
      if (a.dfinal) FHE_CUDA(cudaMemcpyAsync(a.dinitial, a.dfinal, state_bytes, cudaMemcpyDeviceToDevice, st));
      else FHE_CUDA(cudaMemsetAsync(a.dinitial, 0, state_bytes, st));
    }
    return;
  }
  with_type(a.f.dtype, [&](auto tv) {
    using T = decltype(tv);
    // 8 bytes a load: the gradients hold twice the registers (8 x 1001 tokens of 1792
    // float32 channels, sums of the parts included: 49 us with 2 channels, 58 with 4)
    constexpr int kVec = sizeof(T) == 4 ? 2 : 4;
    uint32_t vec = conv_vec(a.f, kVec, a.dy, a.dx, a.dfinal);
    if (!aligned(a.dinitial, vec * e)) vec = 1;
    ConvGradArgs g{};
    g.f = conv_args(a.f, vec, 16);
    g.dy = a.dy;
    g.dfinal = a.dfinal;
    g.dx = a.dx;
    g.dinitial = a.dinitial;
    g.part = static_cast<float*>(a.workspace);
    const uint64_t blocks = (g.f.walkers + kThreads - 1) / kThreads;
    require(blocks < (1ull << 31), "too many blocks");
    with_taps(a.f.taps, [&](auto kv) {
      constexpr int K = decltype(kv)::value;
      auto go = [&](auto vv, auto silu) {
        k_conv_grad<T, decltype(vv)::value, K, decltype(silu)::value><<<(uint32_t)blocks, kThreads, 0, st>>>(g);
      };
      if (vec == 1) {
        if (a.f.silu) go(std::integral_constant<int, 1>{}, std::true_type{});
        else go(std::integral_constant<int, 1>{}, std::false_type{});
      } else {
        if (a.f.silu) go(std::integral_constant<int, kVec>{}, std::true_type{});
        else go(std::integral_constant<int, kVec>{}, std::false_type{});
      }
    });
    note_launch();
    const dim3 grid((a.f.channels + 31) / 32, a.f.taps + 1);
    k_conv_grad_sum<T><<<grid, dim3(32, 8), 0, st>>>(g.part, a.dweight, a.dbias, a.f.channels, a.f.taps,
                                                     a.f.batch * g.f.runs);
    note_launch();
    FHE_CUDA(cudaGetLastError());
  });
}

}  // namespace fhe
