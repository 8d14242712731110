// Log-probabilities of given tokens with the row's entropy and its top
// entries (fhe_token_logprobs), and their gradient.
//
// One read of the row: every thread keeps a running maximum m, s = sum of
// exp(z - m) and u = sum of exp(z - m) (z - m) over its elements, so that
// lse = m + log s and the entropy is log s - u / s (in base 2, see Stats).
// The top entries come out of the same read.  The first elements give a lower
// bound on the k-th largest (the k-th largest of 64 disjoint groups' maxima);
// from then on only loads that reach it are noted, and at the end their
// elements at or above it are listed in shared memory and ranked by counting.
// A row with more candidates than the lists hold (many equal entries) is
// searched again, one rank per pass.
#include <algorithm>
#include <cooperative_groups.h>

#include "launch_count.h"
#include "logit_rows.h"

namespace fhe {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kGroups = 64;   // groups of 4 threads
constexpr int kAhead = 4;     // 16-byte loads in flight per thread
constexpr int kCap = 1024;    // candidates held
constexpr int kHits = 512;    // turns of a thread that hold candidates
constexpr int kMaxTop = 64;
static_assert(kMaxTop <= kGroups && 8 * kMaxTop <= kCap && kThreads / 32 >= 8, "bounds and parts");

// The running sums are kept in base 2 around a shift derived from the running
// maximum m: d = log2(e) z - shift, s = sum of 2^d, u = sum of 2^d d.  The
// shift cancels from every score, so its rounding does not matter as long as
// 2^d survives it: it follows m between -2^20 and 2^20, where it is off by at
// most 1/16, and stays at either end beyond (below, all d lie far below 0 and
// the sums stay 0 until an entry within the range comes).  Entries are raised
// to the type's floor first, which makes d finite.  Rows whose own maximum
// lies outside, and rows with a NaN or infinite maximum, are summed again entry
// by entry (exact_stats).
constexpr float kFar = 1048576.f;  // 2^20
template <class T>
__device__ __forceinline__ float least_max() {  // for float16 far enough above its floor
  return std::is_same_v<T, __half> ? -60000.f : -kFar;
}
template <class T>
__device__ __forceinline__ bool plain_max(float m) {
  return m > least_max<T>() && m < kFar;
}
// Rounded on its own (never contracted into an fma): equal maxima, equal shifts.
template <class T>
__device__ __forceinline__ float shift_of(float m) {
  return __fmul_rn(kLog2e, fminf(fmaxf(m, least_max<T>()), kFar));
}

template <class T>
struct Stats {
  float m = -INFINITY, s = 0.f, u = 0.f;
  __device__ __forceinline__ void raise(float mx) {  // to a maximum that covers mx
    const float to = max_nan(m, mx), d = fmaxf(shift_of<T>(m) - shift_of<T>(to), -1e30f), c = exp2_fast(d);
    u = c * fmaf(d, s, u);
    s *= c;
    m = to;
  }
  __device__ __forceinline__ void merge(float m2, float s2, float u2) {
    raise(m2);
    const float d = fmaxf(shift_of<T>(m2) - shift_of<T>(m), -1e30f), c = exp2_fast(d);
    u += c * fmaf(d, s2, u2);
    s = fmaf(s2, c, s);
  }
};

template <class T>
__device__ __forceinline__ Stats<T> warp_merge(Stats<T> a) {
  for (int o = 16; o; o >>= 1) {
    const float m = __shfl_xor_sync(~0u, a.m, o), s = __shfl_xor_sync(~0u, a.s, o), u = __shfl_xor_sync(~0u, a.u, o);
    a.merge(m, s, u);
  }
  return a;
}

// The sums of a row whose maximum m is not plain, by the whole CTA in natural
// units: sum of exp(z - m) and of exp(z - m) (z - m); every thread gets them.
template <class T>
__device__ void exact_stats(const T* z, uint32_t vocab, float m, float (&red)[3][kThreads / 32], float& s, float& u) {
  s = u = 0.f;
  for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
    const float v = to_f(z[i]);
    if (v == -INFINITY) continue;
    const float d = v - m, e = expf(d);  // +inf - +inf and NaN: NaN
    s += e;
    if (e != 0.f) u = fmaf(e, d, u);
  }
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(~0u, s, o);
    u += __shfl_xor_sync(~0u, u, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    red[0][threadIdx.x >> 5] = s;
    red[1][threadIdx.x >> 5] = u;
  }
  __syncthreads();
  s = u = 0.f;
  for (int i = 0; i < kThreads / 32; ++i) {
    s += red[0][i];
    u += red[1][i];
  }
}

// Shared memory of one CTA that others of its cluster read.
struct Part {
  float m, s, u;
  uint32_t count;
  uint32_t key[kMaxTop], idx[kMaxTop];  // its top entries in order
};

// A row is one CTA's, or a cluster's of `split` CTAs when rows are few: each
// CTA takes a share of the row, and the first puts the shares together over
// distributed shared memory.  Elements before the row's first 16-byte boundary
// and after its last go to threads of the first CTA one by one.
// 2048 bfloat16 rows of 50304: 51 us, 4.0 TB/s; 4095 rows of 50280 with the 8 top
// entries: 118 us, 3.5 TB/s (126 with four CTAs to an SM, 151 with six and half the
// loads in flight).  Issue slots (60% busy) and the latency between a
// row's turns bound it: 9 instructions an element, 4.5 of them the conversion,
// exponential and sums.
template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads, 5) k_logprobs(const fhe_token_logprobs_args g, uint32_t split) {
  using Q = Quad<T>;
  constexpr uint32_t V = Q::kElems;
  __shared__ float red[3][kThreads / 32];
  __shared__ __align__(16) uint32_t gmax[kGroups];
  __shared__ uint32_t ckey[TOP ? kCap : kThreads / 32], cidx[TOP ? kCap : kThreads / 32];
  __shared__ uint32_t hit[TOP ? kHits : 1], hits, bound, count;
  __shared__ Part mine;
  const uint32_t row = blockIdx.x / split, rank = blockIdx.x % split, tid = threadIdx.x;
  const T* z = static_cast<const T*>(g.logits) + (int64_t)row * g.logits_stride;
  const uint32_t vocab = g.vocab, k = g.top_k;
  const uint32_t head = min(vocab, (uint32_t)((0 - reinterpret_cast<uintptr_t>(z)) % 16 / sizeof(T)));
  const T* body = z + head;
  const uint32_t all = (vocab - head) / V, loose = vocab - all * V;
  const uint32_t each = (all + split - 1) / split, first = min(rank * each, all), packs = min(first + each, all);
  if (tid == 0) hits = count = 0;
  if constexpr (TOP) __syncthreads();
  Stats<T> st;
  uint64_t s2 = 0, u2 = 0;  // st's sums in two strands
  float shift = -shift_of<T>(st.m);
  auto collect = [&] {
    float a, b;
    unpair(s2, a, b);
    st.s = a + b;
    unpair(u2, a, b);
    st.u = a + b;
  };
  auto raise = [&](float top) {  // rare: the sums so far move to a new maximum
    collect();
    st.raise(top);
    s2 = pair(st.s, 0.f);
    u2 = pair(st.u, 0.f);
    shift = -shift_of<T>(st.m);
  };
  float fbnd = -INFINITY;
  Q p[kAhead], next[kAhead];
  auto fetch = [&](uint32_t turn) {
    const T* at = body + (uint64_t)(turn + tid) * V;
    if (turn + kAhead * kThreads <= packs) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) next[j].load(at + j * kThreads * V);
    } else {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        next[j].clear();
        if (turn + tid + j * kThreads < packs) next[j].load(at + j * kThreads * V);
      }
    }
  };
  bool sampled = false;
  fetch(first);
  for (uint32_t turn = first; turn < packs; turn += kAhead * kThreads) {  // the whole CTA takes each turn
#pragma unroll
    for (int j = 0; j < kAhead; ++j) p[j] = next[j];
    if (turn + kAhead * kThreads < packs) fetch(turn + kAhead * kThreads);
    uint32_t top_word = p[0].max_word();
#pragma unroll
    for (int j = 1; j < kAhead; ++j) top_word = Q::max_words(top_word, p[j].max_word());
    const float top = Q::max_of(top_word);
    if (!(top <= st.m)) raise(top);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) p[j].add(s2, u2, shift);
    if constexpr (TOP) {
      if (!sampled) {  // the first turn's maxima bound the k-th largest from below
        sampled = true;
        float most = isnan(top) ? -INFINITY : top;
        for (int o = kThreads / kGroups / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
        if (tid % (kThreads / kGroups) == 0) gmax[tid / (kThreads / kGroups)] = order_key(most);
        __syncthreads();
        if (tid < kGroups) {
          const uint32_t own = gmax[tid];
          uint32_t above = 0;
#pragma unroll
          for (uint32_t j = 0; j < kGroups; j += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(&gmax[j]);
            above += before(o.x, j, own, tid) + before(o.y, j + 1, own, tid) + before(o.z, j + 2, own, tid) +
                     before(o.w, j + 3, own, tid);
          }
          if (above == k - 1) bound = own;
        }
        __syncthreads();
        // at or below -inf (few numbers in the sample) it lets all in, NaN too
        if (bound > order_key(-INFINITY)) fbnd = key_value(bound);
      }
      if (!(top < fbnd)) {  // this thread's loads of the turn hold a candidate
        const uint32_t at = atomicAdd(&hits, 1u);
        if (at < kHits) hit[at] = turn + tid;
      }
    }
  }
  if (rank == 0 && tid < loose) {
    const uint32_t e = tid < head ? tid : all * V + tid;
    const float f = to_f(z[e]);
    if (!(f <= st.m)) raise(f);
    const float d = fmaf(fmaxf(f, floor_of<T>()), kLog2e, shift), x = exp2_fast(d);
    s2 = add2(s2, pair(x, 0.f));
    u2 = fma2(pair(x, 0.f), pair(d, 0.f), u2);
  }
  if constexpr (TOP) {
    // the candidates' loads once more, from the cache, spread over the threads
    __syncthreads();
    const uint32_t bnd = fbnd > -INFINITY ? order_key(fbnd) : 0u;
    auto offer = [&](float f, uint32_t idx) {
      if (f < fbnd) return;
      const uint32_t key = order_key(f);
      if (key < bnd) return;  // a NaN
      const uint32_t at = atomicAdd(&count, 1u);
      if (at < kCap) {
        ckey[at] = key;
        cidx[at] = idx;
      }
    };
    if (hits <= kHits) {
      for (uint32_t c = tid; c < hits * kAhead; c += kThreads) {
        const uint32_t i = hit[c / kAhead] + c % kAhead * kThreads;
        if (i >= packs) continue;
        Q q;
        q.load(body + (uint64_t)i * V);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) offer(q.element(v), head + i * V + v);
      }
      if (rank == 0 && tid < loose) {
        const uint32_t e = tid < head ? tid : all * V + tid;
        offer(to_f(z[e]), e);
      }
    } else if (tid == 0) {
      count = kCap + 1;
    }
  }
  collect();
  st = warp_merge(st);
  if ((tid & 31) == 0) {
    red[0][tid >> 5] = st.m;
    red[1][tid >> 5] = st.s;
    red[2][tid >> 5] = st.u;
  }
  __syncthreads();
  if (tid < 32) {
    Stats<T> a;
    if (tid < kThreads / 32) {
      a.m = red[0][tid];
      a.s = red[1][tid];
      a.u = red[2][tid];
    }
    a = warp_merge(a);
    if (tid == 0) {
      mine.m = a.m;
      mine.s = a.s;
      mine.u = a.u;
    }
  }
  if constexpr (TOP) {
    const uint32_t n = count;
    if (n <= kCap) {
      if (tid == 0) mine.count = min(n, k);
      for (uint32_t c = tid; c < n; c += kThreads) {
        const uint32_t key = ckey[c], idx = cidx[c];
        uint32_t above = 0;
        for (uint32_t j = 0; j < n && above < k; ++j) above += before(ckey[j], cidx[j], key, idx);
        if (above < k) {
          mine.key[above] = key;
          mine.idx[above] = idx;
        }
      }
    } else {
      // too many candidates: the next entry after the last, one rank at a time
      const uint32_t mine_n = (packs - first) * V + (rank == 0 ? loose : 0u);
      uint32_t lk = ~0u, li = 0;
      for (uint32_t r = 0; r < k; ++r) {  // n > kCap: more than k entries
        uint32_t bk = 0, bi = ~0u;
        for (uint32_t c = tid; c < mine_n; c += kThreads) {
          uint32_t e = head + first * V + c;  // the share's packs, then the loose elements
          if (c >= (packs - first) * V) {
            e = c - (packs - first) * V;
            if (e >= head) e += all * V;
          }
          const uint32_t key = order_key(to_f(z[e]));
          if ((r == 0 || before(lk, li, key, e)) && before(key, e, bk, bi)) {
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
        if (tid == 0) {
          mine.key[r] = lk = bk;
          mine.idx[r] = li = bi;
        }
        lk = bk;
        li = bi;
      }
      if (tid == 0) mine.count = k;
    }
  }
  auto part = [&](uint32_t r) { return split == 1 ? &mine : cg::this_cluster().map_shared_rank(&mine, r); };
  if (split > 1) cg::this_cluster().sync();
  else __syncthreads();
  if (rank == 0) {
    // the parts come over in one go: sums into red, top entries into ckey, cidx
    // (whose own entries have been ranked), key 0 and index ~0 past a part's end
    if (tid < split) {
      const Part* o = part(tid);
      red[0][tid] = o->m;
      red[1][tid] = o->s;
      red[2][tid] = o->u;
    }
    if constexpr (TOP) {
      for (uint32_t c = tid; c < split * kMaxTop; c += kThreads) {
        const Part* o = part(c / kMaxTop);
        const bool in = c % kMaxTop < o->count;
        ckey[c] = in ? o->key[c % kMaxTop] : 0u;
        cidx[c] = in ? o->idx[c % kMaxTop] : ~0u;
      }
    }
    __syncthreads();
    Stats<T> a;
    for (uint32_t r = 0; r < split; ++r) a.merge(red[0][r], red[1][r], red[2][r]);
    const bool empty = a.m == -INFINITY;
    float ls, shift_a = shift_of<T>(a.m);  // log of s, and the shift, in base 2
    const bool plain = plain_max<T>(a.m);
    if (!plain && !empty) exact_stats(z, vocab, a.m, red, a.s, a.u);
    ls = plain ? log2f(a.s) : logf(a.s);
    auto score = [&](float v) {  // log-probability of an entry
      if (empty || v == -INFINITY) return isnan(ls) ? ls : -INFINITY;
      if (plain && v < -1e30f) return v - a.m;  // the logarithm is lost in it
      return plain ? kLn2 * (fmaf(v, kLog2e, -shift_a) - ls) : v - a.m - ls;
    };
    if (tid == 0) {
      const int64_t t = g.targets[row];
      float lp = 0.f;
      if (t >= (int64_t)vocab) lp = NAN;
      else if (t >= 0) lp = score(to_f(z[t]));
      const float h = ls - a.u / a.s;
      g.logprob[row] = lp;
      g.entropy[row] = empty ? 0.f : plain ? kLn2 * h : h;
      // the shift's own rounding, left out of m, goes back into the sum
      g.norm[2 * (int64_t)row] = a.m;
      g.norm[2 * (int64_t)row + 1] = empty ? 0.f : plain ? kLn2 * (ls + fmaf(-a.m, kLog2e, shift_a)) : ls;
    }
    if constexpr (TOP) {
      for (uint32_t c = tid; c < split * kMaxTop; c += kThreads) {
        const uint32_t key = ckey[c], idx = cidx[c], pos = c % kMaxTop;
        if (idx == ~0u) continue;
        uint32_t above = pos;
        for (uint32_t r = 0; r < split && above < k; ++r) {
          if (r == c / kMaxTop) continue;
          for (uint32_t j = r * kMaxTop; j < (r + 1) * kMaxTop && before(ckey[j], cidx[j], key, idx); ++j) ++above;
        }
        if (above < k) {
          g.top_ids[(int64_t)row * k + above] = idx;
          g.top_logprobs[(int64_t)row * k + above] = score(to_f(z[idx]));
        }
      }
    }
  }
  if (split > 1) cg::this_cluster().sync();  // the first CTA has read the others' shared memory
}

// dlogits = p (-G - g_e (log p + H)) plus, at the target and the top entries,
// their own gradients; G is the sum of those.  One read, one write, in 16-byte
// words where logits and dlogits reach a 16-byte boundary at the same element.
// 2048 bfloat16 rows of 50304: 64 us, 6.4 TB/s, a measured copy's rate.
template <class T>
__global__ void __launch_bounds__(kThreads) k_logprobs_grad(const fhe_token_logprobs_grad_args a, uint32_t parts) {
  using Q = Quad<T>;
  constexpr uint32_t V = Q::kElems;
  const fhe_token_logprobs_args& g = a.f;
  const uint32_t row = blockIdx.x / parts, part = blockIdx.x % parts, tid = threadIdx.x;
  const uint32_t vocab = g.vocab, k = a.dtop_logprobs ? g.top_k : 0;
  const T* z = static_cast<const T*>(g.logits) + (int64_t)row * g.logits_stride;
  T* dz = static_cast<T*>(a.dlogits) + (int64_t)row * vocab;
  const uint32_t each = (vocab + parts - 1) / parts;  // elements of this part
  const uint32_t e0 = min(part * each, vocab), e1 = min(e0 + each, vocab);
  // log p = (z - m) - log s: neither loses the other's digits at large |m|
  const float m = g.norm[2 * (int64_t)row], ls = g.norm[2 * (int64_t)row + 1];
  if (m == -INFINITY) {  // nothing is possible: no gradient
    for (uint32_t e = e0 + tid; e < e1; e += kThreads) dz[e] = from_f<T>(0.f);
    return;
  }
  const int64_t t = g.targets[row];
  const bool used = t >= 0 && t < (int64_t)vocab;
  const float gl = used && a.dlogprob ? a.dlogprob[row] : 0.f;
  const float ge = a.dentropy ? a.dentropy[row] : 0.f, H = a.dentropy ? g.entropy[row] : 0.f;
  float G = gl;
  for (uint32_t i = 0; i < k; ++i) G += a.dtop_logprobs[(int64_t)row * k + i];
  const float c = isnan(ls) ? ls : -G - ge * H;  // a row without scores has no gradient either
  // Entries this far below the maximum have p = 0 and are held there, so that no
  // multiple of their log p overflows into 0 times infinity.
  constexpr float kGone = -1e4f;
  auto base = [&](float v) {
    const float lp = fmaxf((v - m) - ls, kGone), d = exp2_fast(lp * kLog2e) * fmaf(-ge, lp, c);
    return isnan(v) ? v : v == -INFINITY && !isnan(ls) ? 0.f : d;
  };
  auto scalar = [&](uint32_t lo, uint32_t hi) {
    for (uint32_t e = lo + tid; e < hi; e += kThreads) dz[e] = from_f<T>(base(to_f(z[e])));
  };
  const uint32_t head = min(e1 - e0, (uint32_t)((0 - reinterpret_cast<uintptr_t>(dz + e0)) % 16 / sizeof(T)));
  if (plain_max<T>(m) && isfinite(ls) && reinterpret_cast<uintptr_t>(z + e0 + head) % 16 == 0) {
    const uint32_t packs = (e1 - e0 - head) / V;
    const T* zb = z + e0 + head;
    T* db = dz + e0 + head;
    const uint64_t sub = pair(-m, -m), sub2 = pair(-ls, -ls), l2 = pair(kLog2e, kLog2e), nge = pair(-ge, -ge), cc = pair(c, c);
    const float low = m + kGone;
    for (uint32_t i = tid; i < packs; i += kAhead * kThreads) {
      Q p[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i + j * kThreads < packs) p[j].load(zb + (uint64_t)(i + j * kThreads) * V);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (i + j * kThreads >= packs) break;
        float o[V];
#pragma unroll
        for (uint32_t v = 0; v < V; v += 2) {
          const uint64_t lp = add2(
              add2(pair(fmaxf(p[j].element(v), low), fmaxf(p[j].element(v + 1), low)), sub), sub2);
          float x0, x1;
          unpair(mul2(lp, l2), x0, x1);
          unpair(mul2(pair(exp2_fast(x0), exp2_fast(x1)), fma2(nge, lp, cc)), o[v], o[v + 1]);
        }
        *reinterpret_cast<Pack<T, V>*>(db + (uint64_t)(i + j * kThreads) * V) = pack<T>(o);
      }
    }
    scalar(e0, e0 + head);
    scalar(e0 + head + packs * V, e1);
  } else {
    scalar(e0, e1);
  }
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
    if (mine && at >= (int64_t)e0 && at < (int64_t)e1) dz[at] = from_f<T>(base(to_f(z[at])) + add);
  }
}

void check_logprobs(const fhe_token_logprobs_args& a) {
  require(a.dtype == FHE_F32 || a.dtype == FHE_BF16 || a.dtype == FHE_F16, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
  require(a.vocab >= 1 && a.vocab <= (1u << 30), "vocab must be in [1, 2^30]");
  require(a.rows < (1u << 31), "rows must be below 2^31");
  require(a.top_k <= kMaxTop && a.top_k <= a.vocab, "top_k must be at most 64 and at most vocab");
}

}  // namespace

void token_logprobs(const fhe_token_logprobs_args& a) {
  check_logprobs(a);
  if (a.rows == 0) return;
  require(a.logits && a.targets && a.logprob && a.entropy && a.norm, "null input or output");
  require(a.top_k == 0 || (a.top_logprobs && a.top_ids), "null top outputs");
  DeviceGuard dev(a.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  with_type(a.dtype, [&](auto tv) {
    using T = decltype(tv);
    // Few rows leave SMs idle: a cluster of up to 8 CTAs per row then, as long
    // as each has a turn of loads.
    const uint32_t packs = a.vocab / Quad<T>::kElems;
    uint32_t split = 1;
    while (split < 8 && (uint64_t)a.rows * split * 2 <= 2 * 148 && packs >= split * 2 * kAhead * kThreads) split *= 2;
    require((uint64_t)a.rows * split < (1ull << 31), "too many blocks");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.rows * split);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = split;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = split > 1 ? 1 : 0;
    if (a.top_k) FHE_CUDA(cudaLaunchKernelEx(&cfg, k_logprobs<T, true>, a, split));
    else FHE_CUDA(cudaLaunchKernelEx(&cfg, k_logprobs<T, false>, a, split));
    note_launch();
    FHE_CUDA(cudaGetLastError());
  });
}

void token_logprobs_backward(const fhe_token_logprobs_grad_args& a) {
  check_logprobs(a.f);
  if (a.f.rows == 0) return;
  require(a.f.logits && a.f.targets && a.f.norm && a.dlogits, "null input or output");
  require(!a.dentropy || a.f.entropy, "null entropy");
  require(!a.dtop_logprobs || a.f.top_k == 0 || a.f.top_ids, "null top_ids");
  DeviceGuard dev(a.f.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  with_type(a.f.dtype, [&](auto tv) {
    using T = decltype(tv);
    // about two turns of loads per thread
    const uint32_t parts = std::max(1u, a.f.vocab / (kThreads * kAhead * 2 * Quad<T>::kElems));
    require((uint64_t)a.f.rows * parts < (1ull << 31), "too many blocks");
    k_logprobs_grad<T><<<a.f.rows * parts, kThreads, 0, st>>>(a, parts);
    note_launch();
    FHE_CUDA(cudaGetLastError());
  });
}

}  // namespace fhe
