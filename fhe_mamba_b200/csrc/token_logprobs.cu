// Log-probabilities of given tokens with the row's entropy and its top
// entries (fhe_token_logprobs), and their gradient.
//
// One read of the row: every thread keeps a running maximum m, s = sum of
// exp(z - m) and u = sum of exp(z - m) (z - m) over its elements, so that
// lse = m + log s and the entropy is log s - u / s.
// The top entries come out of the same read.  The first elements give a lower
// bound on the k-th largest (the k-th largest of 64 disjoint groups' maxima);
// from then on only elements at or above it enter a list in shared memory,
// whose members are ranked by counting.  A row with more candidates than the
// list holds (many equal entries) is searched again, one rank per pass.
#include <algorithm>

#include "launch_count.h"
#include "mamba_ops.h"

namespace fhe {
namespace {

constexpr int kThreads = 512;
constexpr int kGroups = 64;             // groups of 8 threads
constexpr int kSample = 4;              // loads per thread before the bound is taken
constexpr int kCap = 2048;              // candidates held
constexpr int kMaxTop = 64;
static_assert(kThreads / 8 == kGroups && kMaxTop <= kGroups, "bound");

// Order of two entries: larger value first, then the lower index; NaN last,
// -0 equal to 0.  The value as an unsigned key in ascending order.
__device__ __forceinline__ uint32_t order_key(float z) {
  if (isnan(z)) return 0u;
  const uint32_t u = __float_as_uint(z + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ bool before(uint32_t ka, uint32_t ia, uint32_t kb, uint32_t ib) {
  return ka > kb || (ka == kb && ia < ib);
}

struct Stats {
  float m = -INFINITY, s = 0.f, u = 0.f;
  __device__ __forceinline__ void raise(float mx) {
    if (mx > m) {
      if (s != 0.f) {
        const float d = m - mx, c = __expf(d);
        u = c * fmaf(d, s, u);
        s *= c;
      }
      m = mx;
    }
  }
  __device__ __forceinline__ void add(float z) {  // after raise(a maximum that covers z)
    const float d = z - m, e = __expf(d);
    if (z != -INFINITY) {
      s += e;
      u = fmaf(e, d, u);
    }
  }
  __device__ __forceinline__ void merge(float m2, float s2, float u2) {
    raise(m2);
    if (s2 != 0.f) {  // a NaN sum is not 0
      const float d = m2 - m, c = __expf(d);
      u += c * fmaf(d, s2, u2);
      s = fmaf(s2, c, s);
    }
  }
};

__device__ __forceinline__ Stats warp_merge(Stats a) {
  for (int o = 16; o; o >>= 1) {
    const float m = __shfl_xor_sync(~0u, a.m, o), s = __shfl_xor_sync(~0u, a.s, o), u = __shfl_xor_sync(~0u, a.u, o);
    a.merge(m, s, u);
  }
  return a;
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads) k_logprobs(const fhe_token_logprobs_args g) {
  __shared__ float red[3][kThreads / 32];
  __shared__ uint32_t gmax[kGroups];
  __shared__ uint32_t ckey[kCap], cidx[kCap];
  __shared__ uint32_t bound, count;
  __shared__ float score[2];
  const uint32_t row = blockIdx.x, tid = threadIdx.x;
  const T* z = static_cast<const T*>(g.logits) + (int64_t)row * g.logits_stride;
  const uint32_t vocab = g.vocab, packs = (vocab + V - 1) / V, k = g.top_k;
  if (tid == 0) count = 0;
  Stats st;
  auto fetch = [&](uint32_t i) {
    Pack<T, V> p;
    if ((i + 1) * V <= vocab) return *reinterpret_cast<const Pack<T, V>*>(z + (uint64_t)i * V);
#pragma unroll
    for (int v = 0; v < V; ++v) p.v[v] = i * V + v < vocab ? z[(uint64_t)i * V + v] : from_f<T>(-INFINITY);
    return p;
  };
  auto use = [&](const Pack<T, V>& p) {
    float f[V], mx = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f[v] = to_f(p.v[v]);
      mx = fmaxf(mx, f[v]);
    }
    st.raise(mx);
#pragma unroll
    for (int v = 0; v < V; ++v) st.add(f[v]);
    return mx;
  };
  auto offer = [&](const Pack<T, V>& p, uint32_t i, uint32_t bnd) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t key = order_key(to_f(p.v[v])), idx = i * V + v;
      if (key >= bnd && idx < vocab) {
        const uint32_t at = atomicAdd(&count, 1u);
        if (at < kCap) {
          ckey[at] = key;
          cidx[at] = idx;
        }
      }
    }
  };
  uint32_t i = tid;
  if (k) {
    Pack<T, V> p[kSample];
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < kSample; ++j)
      if (i + j * kThreads < packs) p[j] = fetch(i + j * kThreads);
#pragma unroll
    for (int j = 0; j < kSample; ++j)
      if (i + j * kThreads < packs) {
        use(p[j]);
#pragma unroll
        for (int v = 0; v < V; ++v)
          if ((i + j * kThreads) * V + v < vocab) mx = max(mx, order_key(to_f(p[j].v[v])));
      }
    // a group without elements leaves key 0, below everything
    for (int o = 4; o; o >>= 1) mx = max(mx, __shfl_xor_sync(~0u, mx, o));
    if ((tid & 7) == 0) gmax[tid / 8] = mx;
    __syncthreads();
    if (tid < kGroups) {
      const uint32_t own = gmax[tid];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < kGroups; ++j) rank += before(gmax[j], j, own, tid);
      if (rank == k - 1) bound = own;
    }
    __syncthreads();
    const uint32_t bnd = bound;
#pragma unroll
    for (int j = 0; j < kSample; ++j)
      if (i + j * kThreads < packs) offer(p[j], i + j * kThreads, bnd);
    i += kSample * kThreads;
    for (; i < packs; i += kSample * kThreads) {
#pragma unroll
      for (int j = 0; j < kSample; ++j)
        if (i + j * kThreads < packs) p[j] = fetch(i + j * kThreads);
#pragma unroll
      for (int j = 0; j < kSample; ++j)
        if (i + j * kThreads < packs) {
          use(p[j]);
          offer(p[j], i + j * kThreads, bnd);
        }
    }
  } else {
    for (; i < packs; i += kSample * kThreads) {
      Pack<T, V> p[kSample];
#pragma unroll
      for (int j = 0; j < kSample; ++j)
        if (i + j * kThreads < packs) p[j] = fetch(i + j * kThreads);
#pragma unroll
      for (int j = 0; j < kSample; ++j)
        if (i + j * kThreads < packs) use(p[j]);
    }
  }
  st = warp_merge(st);
  if ((tid & 31) == 0) {
    red[0][tid >> 5] = st.m;
    red[1][tid >> 5] = st.s;
    red[2][tid >> 5] = st.u;
  }
  __syncthreads();
  if (tid < 32) {
    Stats a;
    if (tid < kThreads / 32) {
      a.m = red[0][tid];
      a.s = red[1][tid];
      a.u = red[2][tid];
    }
    a = warp_merge(a);
    if (tid == 0) {
      const bool empty = a.s == 0.f;  // every entry is -inf
      const float ls = empty ? 0.f : logf(a.s);
      const float lse = empty ? -INFINITY : a.m + ls;
      const int64_t t = g.targets[row];
      float lp = 0.f;
      // (z - m) - log s keeps the small digits that m + log s would round away
      if (t >= (int64_t)vocab) lp = NAN;
      else if (t >= 0) lp = empty ? -INFINITY : (to_f(z[t]) - a.m) - ls;
      g.logprob[row] = lp;
      g.entropy[row] = empty ? 0.f : ls - a.u / a.s;
      g.lse[row] = lse;
      score[0] = a.m;
      score[1] = empty ? INFINITY : ls;
    }
  }
  if (!k) return;
  __syncthreads();
  const float m = score[0], ls = score[1];
  auto write = [&](uint32_t rank, uint32_t idx) {
    const float v = to_f(z[idx]);
    g.top_ids[(int64_t)row * k + rank] = idx;
    g.top_logprobs[(int64_t)row * k + rank] = ls == INFINITY ? -INFINITY : (v - m) - ls;
  };
  if (count <= kCap) {
    const uint32_t n = count;
    for (uint32_t c = tid; c < n; c += kThreads) {
      const uint32_t key = ckey[c], idx = cidx[c];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n && rank < k; ++j) rank += before(ckey[j], cidx[j], key, idx);
      if (rank < k) write(rank, idx);
    }
    return;
  }
  // too many candidates: the next entry after the last, k times
  uint32_t lk = ~0u, li = 0;
  bool any = false;
  for (uint32_t r = 0; r < k; ++r) {
    uint32_t bk = 0, bi = ~0u;
    for (uint32_t e = tid; e < vocab; e += kThreads) {
      const uint32_t key = order_key(to_f(z[e]));
      if (any && !before(lk, li, key, e)) continue;
      if (before(key, e, bk, bi)) {
        bk = key;
        bi = e;
      }
    }
    for (int o = 16; o; o >>= 1) {
      const uint32_t ok = __shfl_xor_sync(~0u, bk, o), oi = __shfl_xor_sync(~0u, bi, o);
      if (before(ok, oi, bk, bi)) {
        bk = ok;
        bi = oi;
      }
    }
    __syncthreads();
    if ((tid & 31) == 0) {
      ckey[tid >> 5] = bk;
      cidx[tid >> 5] = bi;
    }
    __syncthreads();
    bk = ckey[0];
    bi = cidx[0];
    for (int w = 1; w < kThreads / 32; ++w)
      if (before(ckey[w], cidx[w], bk, bi)) {
        bk = ckey[w];
        bi = cidx[w];
      }
    if (tid == 0) write(r, bi);
    lk = bk;
    li = bi;
    any = true;
  }
}

// dlogits = p (-G - g_e (log p + H)) plus, at the target and the top entries,
// their own gradients; G is the sum of those.  One read, one write.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) k_logprobs_grad(const fhe_token_logprobs_grad_args a, uint32_t parts) {
  const fhe_token_logprobs_args& g = a.f;
  const uint32_t row = blockIdx.x / parts, part = blockIdx.x % parts, tid = threadIdx.x;
  const uint32_t vocab = g.vocab, k = a.dtop_logprobs ? g.top_k : 0;
  const T* z = static_cast<const T*>(g.logits) + (int64_t)row * g.logits_stride;
  T* dz = static_cast<T*>(a.dlogits) + (int64_t)row * vocab;
  const float lse = g.lse[row];
  const int64_t t = g.targets[row];
  const bool used = t >= 0 && t < (int64_t)vocab;
  const float gl = used && a.dlogprob ? a.dlogprob[row] : 0.f;
  const float ge = a.dentropy ? a.dentropy[row] : 0.f, H = a.dentropy ? g.entropy[row] : 0.f;
  float G = gl;
  for (uint32_t i = 0; i < k; ++i) G += a.dtop_logprobs[(int64_t)row * k + i];
  auto base = [&](float v) {
    const float lp = v - lse;
    const float d = __expf(lp) * (-G - ge * (lp + H));
    return v == -INFINITY ? 0.f : d;
  };
  const uint32_t packs = (vocab + V - 1) / V, each = (packs + parts - 1) / parts;
  const uint32_t p0 = part * each, p1 = min(p0 + each, packs);
  for (uint32_t i = p0 + tid; i < p1; i += kThreads) {
    if ((i + 1) * V <= vocab) {
      const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(z + (uint64_t)i * V);
      Pack<T, V> o;
#pragma unroll
      for (int v = 0; v < V; ++v) o.v[v] = from_f<T>(base(to_f(p.v[v])));
      *reinterpret_cast<Pack<T, V>*>(dz + (uint64_t)i * V) = o;
    } else {
      for (uint32_t e = i * V; e < vocab; ++e) dz[e] = from_f<T>(base(to_f(z[e])));
    }
  }
  if (lse == -INFINITY) return;
  __syncthreads();
  // the target and the top entries of this part, each written once more whole
  if (tid <= k) {
    int64_t at = t;
    float add = gl;
    bool mine = used;
    const int64_t* ids = g.top_ids + (int64_t)row * k;
    if (tid < k) {
      at = ids[tid];
      add = a.dtop_logprobs[(int64_t)row * k + tid] + (used && at == t ? gl : 0.f);
      mine = at >= 0 && at < (int64_t)vocab;
    } else {
      for (uint32_t i = 0; i < k; ++i) mine = mine && ids[i] != t;
    }
    if (mine && at >= (int64_t)p0 * V && at < (int64_t)p1 * V) dz[at] = from_f<T>(base(to_f(z[at])) + add);
  }
}

void check_logprobs(const fhe_token_logprobs_args& a) {
  require(a.dtype == FHE_F32 || a.dtype == FHE_BF16 || a.dtype == FHE_F16, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
  require(a.vocab >= 1 && a.vocab <= (1u << 30), "vocab must be in [1, 2^30]");
  require(a.rows < (1u << 31), "rows must be below 2^31");
  require(a.top_k <= kMaxTop && a.top_k <= a.vocab, "top_k must be at most 64 and at most vocab");
}

bool row_aligned(const void* p, int64_t stride, uint32_t vec, uint32_t elem) {
  return reinterpret_cast<uintptr_t>(p) % (vec * elem) == 0 && stride % vec == 0;
}

}  // namespace

void token_logprobs(const fhe_token_logprobs_args& a) {
  check_logprobs(a);
  if (a.rows == 0) return;
  require(a.logits && a.targets && a.logprob && a.entropy && a.lse, "null input or output");
  require(a.top_k == 0 || (a.top_logprobs && a.top_ids), "null top outputs");
  DeviceGuard dev(a.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  with_type(a.dtype, [&](auto tv) {
    using T = decltype(tv);
    constexpr int V = 16 / sizeof(T);
    if (row_aligned(a.logits, a.logits_stride, V, sizeof(T))) k_logprobs<T, V><<<a.rows, kThreads, 0, st>>>(a);
    else k_logprobs<T, 1><<<a.rows, kThreads, 0, st>>>(a);
    note_launch();
    FHE_CUDA(cudaGetLastError());
  });
}

void token_logprobs_backward(const fhe_token_logprobs_grad_args& a) {
  check_logprobs(a.f);
  if (a.f.rows == 0) return;
  require(a.f.logits && a.f.targets && a.f.lse && a.dlogits, "null input or output");
  require(!a.dentropy || a.f.entropy, "null entropy");
  require(!a.dtop_logprobs || a.f.top_k == 0 || a.f.top_ids, "null top_ids");
  DeviceGuard dev(a.f.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  with_type(a.f.dtype, [&](auto tv) {
    using T = decltype(tv);
    constexpr int V = 16 / sizeof(T);
    const bool vec = row_aligned(a.f.logits, a.f.logits_stride, V, sizeof(T)) &&
                     row_aligned(a.dlogits, a.f.vocab, V, sizeof(T));
    const uint64_t packs = (a.f.vocab + (vec ? V : 1) - 1) / (vec ? V : 1);
    // about four loads per thread
    const uint32_t parts = (uint32_t)std::max<uint64_t>(1, packs / (kThreads * 4));
    require((uint64_t)a.f.rows * parts < (1ull << 31), "too many blocks");
    if (vec) k_logprobs_grad<T, V><<<a.f.rows * parts, kThreads, 0, st>>>(a, parts);
    else k_logprobs_grad<T, 1><<<a.f.rows * parts, kThreads, 0, st>>>(a, parts);
    note_launch();
    FHE_CUDA(cudaGetLastError());
  });
}

}  // namespace fhe
