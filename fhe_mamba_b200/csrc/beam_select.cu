// Beam search's selection (fhe_beam_select): the `width` best of score_i + z_iv -
// log sum exp z_i over the beams i and tokens v of each batch item.
//
// A cluster of up to sixteen CTAs takes a batch item, a row or a share of a row to a
// CTA at a time, in one read: sums of exp(z - m) around a running shift m, and the
// largest entry of each thread.  The `width`-th largest of 64 groups' maxima is a lower
// bound on the share's best entries; the loads of the threads that reach it come once
// more, from the cache, and what reaches it is ranked by counting.  Shares go to the
// first CTA over distributed shared memory, which ranks them together.  Within a beam
// the order is that of the logits; between beams it hangs on the beams' sums, which
// fp32 knows to a few 2^-20.  Where a beam's entry lies closer than that to one of the
// best of another, the cluster sums those beams again in 64 bits, so that the choice
// is always that of the formula.
//
// 64 items of 8 bfloat16 beams of 50304, 15% of them finished: 24 us.  The reads come at
// 5.8 TB/s (7.5 us, all 512 CTAs at once); then bound, candidates and ranks of each share
// (2.7 us), the meeting, and the ranking of the item's entries while others still read.
// One item of 4 float32 beams: 10.5 us, of which the reads 3.4.  Rows in which fewer
// groups of threads hold a possible token than are wanted (a mask that leaves one to five
// tokens, or thirty neighbours; rows of one value alike) have no bound above the
// impossible ones and read their share again for each rank: 490 us and 68 us.
#include <algorithm>
#include <cfloat>
#include <cooperative_groups.h>

#include "launch_count.h"
#include "logit_rows.h"

namespace fhe {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kGroups = 64;   // groups of 4 threads
constexpr uint32_t kFineWidth = 32;    // more best entries than this are bounded by every thread's maximum
constexpr uint32_t kAllRanked = 512;   // entries of an item up to which none is left out before ranking
constexpr int kAhead = 4;     // 16-byte loads in flight per thread
constexpr int kCap = 1024;    // candidates held
constexpr uint32_t kMaxBeams = 64, kMaxWidth = 64, kMaxCluster = 16;
static_assert(kMaxWidth <= kGroups, "the bound is the width-th of the groups' maxima");

// What a row's logits and its log sum exp are counted from.  Rows below zero are counted
// from their largest: where the mask leaves nothing but numbers like -1e30 or the type's
// lowest, score and log of the sum would be lost beside them and the total come out as 0,
// the best of all.  Others from 0: logits past 2^30 are no mask, and their totals are
// good to 2^-52 of them.
__device__ __forceinline__ double origin(double largest) { return fmin(largest, 0.); }

// One share of a row: sum of exp(z - m), and its best entries in order.
struct Share {
  double s;
  float m;
  uint32_t raises, count, pad;
};

// Dynamic shared memory, of the first CTA: every share with its entries.
struct Layout {
  Share* share;
  double* total;
  uint32_t *key, *idx;
  uint32_t bytes;
  __host__ __device__ Layout(uint8_t* p, uint32_t lists, uint32_t kk) {
    uint8_t* at = p;
    auto take = [&](uint32_t n) {
      uint8_t* r = at;
      at += (n + 15) / 16 * 16;
      return r;
    };
    share = reinterpret_cast<Share*>(take(lists * sizeof(Share)));
    total = reinterpret_cast<double*>(take(lists * kk * 8));
    key = reinterpret_cast<uint32_t*>(take(lists * kk * 4));
    idx = reinterpret_cast<uint32_t*>(take(lists * kk * 4));
    bytes = (uint32_t)(at - p);
  }
};

struct SelectArgs {
  fhe_beam_select_args a;
  uint32_t cluster, kk;  // CTAs per item; entries of a row that count
};

// exp(z - m) summed over the elements of a load, m finite.
template <class T>
__device__ __forceinline__ uint64_t add_exps(const Quad<T>& q, uint64_t acc, uint64_t minus_m) {
  using Q = Quad<T>;
  const uint64_t k = pair(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < Q::kElems / 2; ++i) {
    float f[2];
    if constexpr (Q::kPer == 2) {
      Q::floats(q.w[i], f);
    } else {
      f[0] = __uint_as_float(q.w[2 * i]);
      f[1] = __uint_as_float(q.w[2 * i + 1]);
    }
    float d0, d1;
    unpair(mul2(add2(pair(f[0], f[1]), minus_m), k), d0, d1);
    acc = add2(acc, pair(exp2_fast(d0), exp2_fast(d1)));
  }
  return acc;
}

struct Scratch {
  float fred[kWarps];
  double dred[kWarps];
  __align__(16) uint32_t gmax[kThreads];
  uint32_t ckey[kCap], cidx[kCap], hit[kThreads];
  uint32_t hits, bound, count, raises;
};

// A number as an unsigned integer of the same order, and back.
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double number(uint64_t o) {
  return __longlong_as_double((int64_t)(o >> 63 ? o & ~(1ull << 63) : ~o));
}

__device__ __forceinline__ double block_sum(double v, double (&red)[kWarps]) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.;
  for (int i = 0; i < kWarps; ++i) v += red[i];
  return v;
}

// Share `part` of `parts` of the row z: 16-byte words between the row's first and
// last 16-byte boundaries; the elements before and after go with the first share.
template <class T>
__device__ void scan_share(const T* z, uint32_t vocab, uint32_t part, uint32_t parts, uint32_t k, Scratch& sm, Share* out,
                           uint32_t* key_out, uint32_t* idx_out) {
  using Q = Quad<T>;
  constexpr uint32_t V = Q::kElems;
  const uint32_t tid = threadIdx.x;
  const uint32_t head = min(vocab, (uint32_t)((0 - reinterpret_cast<uintptr_t>(z)) % 16 / sizeof(T)));
  const T* body = z + head;
  const uint32_t all = (vocab - head) / V, loose = part == 0 ? vocab - all * V : 0;
  const uint32_t each = (all + parts - 1) / parts, first = min(part * each, all), packs = min(first + each, all);
  const uint32_t mine = (packs - first) * V + loose;  // elements of this share
  __syncthreads();
  if (tid == 0) sm.hits = sm.count = sm.raises = 0;
  __syncthreads();
  float m = -INFINITY;
  double s = 0.;
  uint32_t raises = 0;
  auto raise = [&](float top) {  // rare: the sum so far moves to a new shift
    s *= m == -INFINITY ? 0.f : exp2_fast((m - top) * kLog2e);
    m = top;
    ++raises;
  };
  auto shift = [&] {
    const float v = -fmaxf(m, -FLT_MAX);
    return pair(v, v);
  };
  constexpr float kSlack = 4.f;  // a sum may hold terms up to e^4 before its shift moves
  float best = -INFINITY;  // NaN left out
  Q p[kAhead], next[kAhead];
  auto fetch = [&](uint32_t turn) {
    const T* at = body + (uint64_t)(turn + tid) * V;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      next[j].clear();
      if (turn + tid + j * kThreads < packs) next[j].load(at + j * kThreads * V);
    }
  };
  fetch(first);
  for (uint32_t turn = first; turn < packs; turn += kAhead * kThreads) {  // the whole CTA takes each turn
#pragma unroll
    for (int j = 0; j < kAhead; ++j) p[j] = next[j];
    if (turn + kAhead * kThreads < packs) fetch(turn + kAhead * kThreads);
    uint32_t top_word = p[0].max_word();
#pragma unroll
    for (int j = 1; j < kAhead; ++j) top_word = Q::max_words(top_word, p[j].max_word());
    const float top = Q::max_of(top_word);
    if (!(top <= m + kSlack)) raise(top);
    uint64_t acc = 0;
    const uint64_t minus_m = shift();
#pragma unroll
    for (int j = 0; j < kAhead; ++j) acc = add_exps<T>(p[j], acc, minus_m);
    float a, b;
    unpair(acc, a, b);
    s += (double)(a + b);
    best = fmaxf(best, top);
  }
  if (tid < loose) {
    const float f = to_f(z[tid < head ? tid : all * V + tid]);
    if (!(f <= m + kSlack)) raise(f);
    s += (double)exp2_fast((f - fmaxf(m, -FLT_MAX)) * kLog2e);
    best = fmaxf(best, f);
  }
  // a lower bound on the k-th largest: that of the maxima of groups of threads, or of
  // all threads where there are many to find or fewer groups have loads than there are
  // to find; and the threads that reach it
  const bool fine = k > kFineWidth || packs - first < 4 * k;
  float group = best;
  if (!fine)
    for (int o = kThreads / kGroups / 2; o; o >>= 1) group = fmaxf(group, __shfl_xor_sync(~0u, group, o));
  float most = m;
  for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
  const uint32_t groups = fine ? kThreads : kGroups, per = kThreads / groups;
  if (tid % per == 0) sm.gmax[tid / per] = order_key(group);
  if ((tid & 31) == 0) sm.fred[tid >> 5] = most;
  if (raises > 1) atomicMax(&sm.raises, raises);
  __syncthreads();
  if (tid < groups) {
    const uint32_t own = sm.gmax[tid];
    uint32_t above = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < groups; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&sm.gmax[j]);
      above += before(o.x, j, own, tid) + before(o.y, j + 1, own, tid) + before(o.z, j + 2, own, tid) +
               before(o.w, j + 3, own, tid);
    }
    if (above == k - 1) sm.bound = own;
  }
  // meanwhile the sums of the threads, each moved to the largest shift
  most = sm.fred[0];
  for (int i = 1; i < kWarps; ++i) most = fmaxf(most, sm.fred[i]);
  if (m != most && s != 0.) s *= exp2_fast((m - most) * kLog2e);
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if ((tid & 31) == 0) sm.dred[tid >> 5] = s;
  __syncthreads();
  const uint32_t bnd = sm.bound;
  if (order_key(best) >= bnd) sm.hit[atomicAdd(&sm.hits, 1u)] = tid;
  __syncthreads();
  auto offer = [&](float f, uint32_t i) {
    const uint32_t key = order_key(f);
    if (key < bnd) return;
    const uint32_t at = atomicAdd(&sm.count, 1u);
    if (at < kCap) {
      sm.ckey[at] = key;
      sm.cidx[at] = i;
    }
  };
  const uint32_t loads = (packs - first + kThreads - 1) / kThreads;  // of a thread
  for (uint32_t c = tid; c < sm.hits * loads; c += kThreads) {
    const uint32_t i = first + c % loads * kThreads + sm.hit[c / loads];
    if (i >= packs) continue;
    Q q;
    q.load(body + (uint64_t)i * V);
    if (order_key(Q::max_of(q.max_word())) < bnd) continue;
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) offer(q.element(v), head + i * V + v);
  }
  if (tid < loose) {
    const uint32_t e = tid < head ? tid : all * V + tid;
    offer(to_f(z[e]), e);
  }
  __syncthreads();
  const uint32_t n = sm.count, want = min(k, mine);
  if (tid == 0) {
    double sum = 0.;
    for (int i = 0; i < kWarps; ++i) sum += sm.dred[i];
    *out = Share{sum, most, sm.raises, want, 0};
  }
  if (n <= kCap) {
    for (uint32_t c = tid; c < n; c += kThreads) {
      const uint32_t key = sm.ckey[c], i = sm.cidx[c];
      uint32_t above = 0;
      for (uint32_t j = 0; j < n && above < k; ++j) above += before(sm.ckey[j], sm.cidx[j], key, i);
      if (above < k) {
        key_out[above] = key;
        idx_out[above] = i;
      }
    }
  } else {
    // too many candidates (many equal entries): the next entry after the last, one rank at a time
    uint32_t lk = ~0u, li = 0;
    for (uint32_t r = 0; r < want; ++r) {
      uint32_t bk = 0, bi = ~0u;
      for (uint32_t c = tid; c < mine; c += kThreads) {
        uint32_t e = head + first * V + c;  // the share's words, then the loose elements
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
        sm.ckey[tid >> 5] = bk;
        sm.cidx[tid >> 5] = bi;
      }
      __syncthreads();
      bk = sm.ckey[0];
      bi = sm.cidx[0];
      for (int w = 1; w < kWarps; ++w)
        if (before(sm.ckey[w], sm.cidx[w], bk, bi)) {
          bk = sm.ckey[w];
          bi = sm.cidx[w];
        }
      lk = bk;
      li = bi;
      if (tid == 0) {
        key_out[r] = bk;
        idx_out[r] = bi;
      }
    }
  }
  __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_select(const SelectArgs g) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Scratch sm;
  __shared__ float score[kMaxBeams];
  __shared__ uint32_t live[kMaxBeams], ended[kMaxBeams], alive[2];
  __shared__ double lse[kMaxBeams], err[kMaxBeams], top[kMaxBeams], again[kMaxBeams];
  __shared__ uint32_t lcount[kMaxBeams + kMaxCluster], lbeam[kMaxBeams + kMaxCluster];
  __shared__ double rtotal[kMaxWidth];
  __shared__ uint32_t rbeam[kMaxWidth], rtok[kMaxWidth];
  __shared__ uint32_t votes[kMaxBeams + kMaxCluster];
  __shared__ uint64_t unsure, agreed;  // beams to sum again: the first CTA's, all CTAs'
  const fhe_beam_select_args& a = g.a;
  const uint32_t tid = threadIdx.x, C = g.cluster, rank = blockIdx.x % C, item = blockIdx.x / C;
  const uint32_t B = a.beams, k = a.width, kk = g.kk;
  cg::cluster_group cluster = cg::this_cluster();
  if (C > 1) cluster.barrier_arrive();  // every CTA has to run before another's memory is written
  if (tid < 64) {  // the live beams, in order
    const bool mine = tid < B;
    const float v = mine ? a.scores[(int64_t)item * B + tid] : 0.f;
    const bool end = mine && a.finished && a.finished[(int64_t)item * B + tid];
    const uint32_t on = __ballot_sync(~0u, mine && !end && isfinite(v));
    if (mine) {
      score[tid] = v;
      ended[tid] = end;
    }
    if (tid % 32 == 0) alive[tid / 32] = on;
  }
  __syncthreads();
  if (tid < 64) {
    const uint32_t w = tid / 32, on = alive[w], skip = w ? __popc(alive[0]) : 0;
    if (on >> tid % 32 & 1) live[skip + __popc(on & ((1u << tid % 32) - 1))] = tid;
  }
  const uint32_t lives = __popc(alive[0]) + __popc(alive[1]);
  __syncthreads();
  const uint32_t parts = lives ? max(1u, C / lives) : 1, units = lives * parts;
  const Layout l(dynamic, B + C, kk);
  auto row_of = [&](uint32_t beam) {
    return static_cast<const T*>(a.logits) + ((int64_t)item * B + beam) * a.logits_stride;
  };
  auto of = [&](auto* p, uint32_t r) { return C == 1 ? p : cluster.map_shared_rank(p, r); };
  auto meet = [&] {
    if (C > 1) cluster.sync();
    else __syncthreads();
  };
  if (C > 1) cluster.barrier_wait();
  for (uint32_t u = rank; u < units; u += C)
    scan_share<T>(row_of(live[u / parts]), a.vocab, u % parts, parts, kk, sm, of(l.share, 0) + u, of(l.key, 0) + u * kk,
                  of(l.idx, 0) + u * kk);
  meet();
  uint32_t lists = 0;
  if (rank == 0) {
    // sums of the live beams
    if (tid < lives) {
      float m = -INFINITY;
      uint32_t raises = 0, most = 0;
      bool bad = false;
      const Share* s = l.share + tid * parts;
      for (uint32_t p = 0; p < parts; ++p) {
        m = fmaxf(m, s[p].m);
        if (s[p].count) most = max(most, l.key[(tid * parts + p) * kk]);
        raises = max(raises, s[p].raises);
        bad = bad || !isfinite(s[p].s);
      }
      double sum = s[0].s;
      if (parts > 1 && !bad && m > -INFINITY) {
        sum = 0.;
        for (uint32_t p = 0; p < parts; ++p)
          if (s[p].s != 0.) sum += s[p].s * exp((double)s[p].m - (double)m);
      }
      const uint32_t i = live[tid];
      const bool fine = !bad && isfinite(m) && sum > 0.;
      top[i] = key_value(most);  // the row's largest: a shift that, unlike m, is the same at any alignment
      lse[i] = fine ? (double)m - origin(top[i]) + log(sum) : -INFINITY;
      // Roundings of u = 2^-24: three of an exponent d = (z - m) log2 e, whose mean over
      // the sum is at most log2(vocab / sum) and twice the slack, the exponential's four,
      // at most 17 additions, 6 for moving the threads' sums to one shift; 8 u for each
      // time that a thread's shift moved
      err[i] = fine ? 0x1p-24 * (2.2 * (log2((double)a.vocab) - log2(sum) + 12.) + 32. + 8. * raises) : 0.;
    }
    __syncthreads();
    if (tid < units) {
      const uint32_t i = live[tid / parts];
      const bool fine = isfinite(lse[i]);
      lbeam[tid] = i;
      lcount[tid] = fine ? l.share[tid].count : tid % parts == 0 ? kk : 0;  // its impossible tokens, once
    }
    lists = units + B - lives;
    if (tid < B && !(alive[tid / 32] >> tid % 32 & 1)) {  // the others offer what is impossible, or their end
      const uint32_t at = units + tid - (tid >= 32 ? __popc(alive[0]) : 0) - __popc(alive[tid / 32] & ((1u << tid % 32) - 1));
      lbeam[at] = tid;
      lcount[at] = kk;
      lse[tid] = -INFINITY;
      err[tid] = 0.;
    }
    __syncthreads();
  }
  for (;;) {
    if (rank == 0) {
      if (tid == 0) unsure = 0;
      for (uint32_t c = tid; c < lists * kk; c += kThreads) {
        const uint32_t u = c / kk, j = c % kk, i = lbeam[u];
        if (j >= lcount[u]) continue;
        if (isfinite(lse[i])) {
          l.total[c] = (double)score[i] + ((double)key_value(l.key[c]) - origin(top[i])) - lse[i];
        } else {
          // a finished beam: its end, then the impossible tokens; others impossible alone
          const bool end = ended[i] && isfinite(score[i]);
          const uint32_t eos = (uint32_t)a.eos;
          l.key[c] = 0;
          l.idx[c] = !end ? j : j == 0 ? eos : j - 1 < eos ? j - 1 : j;
          l.total[c] = end && j == 0 ? (double)score[i] : -INFINITY;
        }
      }
      __syncthreads();
      // Many entries: the lists, which are in order, are cut behind what lies within reach
      // of the k-th largest total, whose upper word is found bit by bit.
      if (lists * kk > kAllRanked) {
        auto upper = [&](double v) { return (uint32_t)(ordered(v) >> 32); };
        auto at_least = [&](auto&& in) {  // entries of this thread's list up to the first that is not in
          uint32_t lo = 0;
          for (uint32_t len = tid < lists ? lcount[tid] : 0; len;) {
            const uint32_t half = len / 2;
            const bool f = in(l.total[tid * kk + lo + half]);
            lo = f ? lo + half + 1 : lo;
            len = f ? len - half - 1 : half;
          }
          return lo;
        };
        uint32_t kth = 0;
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
          if (tid < lists) votes[tid] = at_least([&](double v) { return upper(v) >= (kth | bit); });
          __syncthreads();
          uint32_t all = 0;
          for (uint32_t u = tid & 31; u < lists; u += 32) all += votes[u];
          all = __reduce_add_sync(~0u, all);
          if (all >= k) kth |= bit;
          __syncthreads();
        }
        double reach = 0.;
        for (uint32_t i = 0; i < B; ++i) reach = fmax(reach, 2. * err[i]);
        // (the word of -inf with zeros behind it is no number)
        const double least = kth <= upper(-INFINITY) ? -INFINITY : number((uint64_t)kth << 32) - reach;
        const uint32_t keep = at_least([&](double v) { return v >= least; });
        __syncthreads();
        if (tid < lists) lcount[tid] = keep;
        __syncthreads();
      }
      // Ranks: larger total, lower beam, larger logit, lower token.  An entry of another
      // beam may belong before one of the best if the next of its list is too close to
      // that one.
      uint32_t lanes = 1;  // that share an entry, a list each at a time
      while (lanes < 32 && lanes < lists && lanes * lists * kk < kThreads * 2) lanes *= 2;
      const uint32_t turns = (lists * kk * lanes + kThreads - 1) / kThreads;
      for (uint32_t n = 0; n < turns; ++n) {
        const uint32_t c = (n * kThreads + tid) / lanes, lane = tid % lanes;
        const uint32_t u = c / kk, j = c % kk;
        uint32_t above = k;
        uint64_t close = 0;
        if (u < lists && j < lcount[u]) {
          const uint32_t i = lbeam[u], key = l.key[c], id = l.idx[c];
          const double t = l.total[c];
          above = lane == 0 ? j : 0;
          for (uint32_t v = lane; v < lists && above < k; v += lanes) {
            if (v == u) continue;
            const uint32_t w = lbeam[v], end = lcount[v];
            uint32_t lo = 0, len = end;
            while (len) {
              const uint32_t half = len / 2, e = v * kk + lo + half;
              const double o = l.total[e];
              const bool first = o > t || (o == t && (w < i || (w == i && before(l.key[e], l.idx[e], key, id))));
              lo = first ? lo + half + 1 : lo;
              len = first ? len - half - 1 : half;
            }
            above += lo;
            const double e = err[i] + err[w];
            if (w != i && e > 0. && lo < end && t - l.total[v * kk + lo] <= e)  // false for impossible entries
              close |= (err[i] > 0. ? 1ull << i : 0ull) | (err[w] > 0. ? 1ull << w : 0ull);
          }
        }
        for (uint32_t o = lanes / 2; o; o /= 2) {
          above += __shfl_xor_sync(~0u, above, o);
          close |= __shfl_xor_sync(~0u, close, o);
        }
        if (lane == 0 && above < k) {
          rtotal[above] = l.total[c];
          rbeam[above] = lbeam[u];
          rtok[above] = l.idx[c];
          if (close) atomicOr(reinterpret_cast<unsigned long long*>(&unsure), (unsigned long long)close);
        }
      }
      __syncthreads();
      if (tid < C) *of(&agreed, tid) = unsure;
    }
    meet();
    const uint64_t todo = agreed;
    if (todo == 0) break;
    // those beams' sums in 64 bits, from a shift and in an order that do not hang on alignment: equal rows
    // give equal sums
    for (uint32_t i = 0; i < B; ++i) {
      if (!(todo >> i & 1)) continue;
      const T* z = row_of(i);
      const double m = *of(&top[i], 0);
      double s = 0.;
      for (uint32_t e = rank * kThreads + tid; e < a.vocab; e += C * kThreads) s += exp((double)to_f(z[e]) - m);
      s = block_sum(s, sm.dred);
      if (tid == 0) again[i] = s;
    }
    meet();
    if (rank == 0 && tid < B && (todo >> tid & 1)) {
      double s = 0.;
      for (uint32_t r = 0; r < C; ++r) s += of(again, r)[tid];
      lse[tid] = top[tid] - origin(top[tid]) + log(s);
      err[tid] = 0.;
    }
    __syncthreads();
  }
  if (rank != 0) return;
  // the best child of a beam takes its place, the others the free places in turn
  uint32_t place = tid;
  if (a.keep_slots && tid < k) {
    uint64_t seen = 0, before_me = 0;
    uint32_t later = 0;  // children before this one that do not take their beam's place
    for (uint32_t r = 0; r < k; ++r) {
      const uint64_t bit = 1ull << rbeam[r];
      if (r == tid) before_me = seen;
      later += r < tid && (seen & bit) != 0;
      seen |= bit;
    }
    place = rbeam[tid];
    if (before_me >> place & 1) {
      uint64_t open = ~seen;
      for (uint32_t n = 0; n < later; ++n) open &= open - 1;
      place = __ffsll((long long)open) - 1;
    }
  }
  if (tid < k) {
    const uint32_t i = rbeam[tid], t = rtok[tid];
    const int64_t at = (int64_t)item * k + place;
    a.out_scores[at] = (float)rtotal[tid];
    a.parents[at] = i;
    a.tokens[at] = t;
    if (a.out_finished) a.out_finished[at] = ended[i] || (a.eos >= 0 && t == (uint64_t)a.eos);
  }
}

}  // namespace

void beam_select(const fhe_beam_select_args& a) {
  require(a.dtype == FHE_F32 || a.dtype == FHE_BF16 || a.dtype == FHE_F16, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
  require(a.beams >= 1 && a.beams <= kMaxBeams, "beams must be in [1, 64]");
  require(a.vocab >= 1 && a.vocab <= (1u << 30), "vocab must be in [1, 2^30]");
  require(a.width >= 1 && a.width <= kMaxWidth && (uint64_t)a.width <= (uint64_t)a.beams * a.vocab,
          "width must be in [1, 64] and at most beams * vocab");
  require(a.batch < (1u << 24), "batch must be below 2^24");
  require(a.eos < (int64_t)a.vocab, "eos past the vocabulary");
  require(!a.finished || a.eos >= 0, "finished beams need an eos token");
  require(!a.keep_slots || a.width == a.beams, "keep_slots needs a width of beams");
  if (a.batch == 0) return;
  require(a.logits && a.scores && a.out_scores && a.parents && a.tokens, "null input or output");
  DeviceGuard dev(a.device);
  with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    // As many CTAs to an item as the device takes at once, a beam or a turn of loads for each;
    // nine an SM while a CTA has two beams, up to where one round of larger shares takes as
    // long as those and their last, part-filled round (300 x 8 bfloat16 beams: 87 us with four,
    // 105 with one; 333 x 8: 87 with four, 94 with two; but 360 x 8 float32: 141 with four, 112
    // with two, and 128 x 4 bfloat16: 22 with four, 32 with eight); sixteen where
    // eight would take several beams each (1 x 10 beams of 50280 bfloat16: 17 us, 23 with
    // eight; 1 x 4: 11 us with either).
    const uint64_t packs = (uint64_t)a.beams * (a.vocab / Quad<T>::kElems);
    SelectArgs g{a, 1, std::min(a.width, a.vocab)};
    while (g.cluster < (a.beams > 8 ? kMaxCluster : 8) &&
           (uint64_t)a.batch * g.cluster * 2 <= (g.cluster * 4 <= a.beams ? 148 * 9 : 148 * 4) &&
           (g.cluster < a.beams || packs >= (uint64_t)g.cluster * 2 * kAhead * kThreads))
      g.cluster *= 2;
    const uint32_t shared = Layout(nullptr, a.beams + g.cluster, g.kk).bytes;
    if (shared > 32768) allow_shared(k_select<T>, Layout(nullptr, kMaxBeams + kMaxCluster, kMaxWidth).bytes);
    if (g.cluster > 8) FHE_CUDA(cudaFuncSetAttribute(k_select<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.batch * g.cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = static_cast<cudaStream_t>(a.stream);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = g.cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    FHE_CUDA(cudaLaunchKernelEx(&cfg, k_select<T>, g));
  });
  note_launch();
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
