// Mamba-2 state recurrence (fhe_ssm_scan) and its gradients.
//
//   S_t = a_t S_(t-1) + w_t x_t (x) b_t,  a_t = exp(log_decay_t),  y_t = S_t c_t + d x_t
//
// The kernel below walks tokens with a tile of S in registers.  It is written
// for "rows" (the axis of the output) and "columns" (the summed axis): a row
// input r, a key k and a query q give S += r (x) k and o = S q.  With
// dS_t = a_(t+1) dS_(t+1) + dy_t (x) c_t the gradients are the same walk:
//   dx   rows p, reversed:  r = dy, k = c, q = b   (times w, plus d dy)
//   U    rows n, reversed:  r = c, k = dy, q = x   db = sum over heads of w U, dw = <b, U>
//   dC_h rows n, forward:   r = b, k = x, q = dy   dc = sum over heads of dC_h
// and, with alpha = <c, dC_h> and beta = w dw, the gradient of log_decay is
//   g_t = <a_t dS_t, S_(t-1)> = g_(t+1) + alpha_t - beta_t,
// a running sum that each segment starts anew from <dS, S> at its end, so
// that its rounding does not add up over a long row.
//
// Long rows are cut into segments: one pass leaves each segment's state from
// zero, a join carries the states across segments, a second pass walks every
// segment from its own start.
#include <algorithm>
#include <cmath>

#include "launch_count.h"
#include "mamba_ops.h"
#include "mamba_scan.h"

namespace fhe {
namespace {

constexpr int kThreads = 128;
constexpr int kTok = 16;      // tokens staged per step
constexpr uint32_t kTcTokens = 64;  // shortest rows the tensor-core form takes

// Four consecutive elements of a row of `width` at column col, zeros outside.
template <class T>
__device__ __forceinline__ Pack<T, 4> load4(const T* row, int col, int width, bool vec, bool live) {
  Pack<T, 4> v;
  if (live && vec && col + 4 <= width) return *reinterpret_cast<const Pack<T, 4>*>(row + col);
#pragma unroll
  for (int i = 0; i < 4; ++i) v.v[i] = (live && col + i < width) ? row[col + i] : from_f<T>(0.f);
  return v;
}

template <class T>
__device__ __forceinline__ float4 unpack4(const Pack<T, 4>& v) {
  return make_float4(to_f(v.v[0]), to_f(v.v[1]), to_f(v.v[2]), to_f(v.v[3]));
}

// One block walks one segment of one (batch, head) for a tile of 16 R rows.
// A thread holds R rows x CW columns: lane bits 0-2 choose the columns
// 4 (lane & 7) + 32 i, lane bits 3-4 and the warp the rows.  S q of 16 / R
// tokens is left in 16 partial sums per lane, which the 8 lanes of a row then
// add with 14 shuffles for all of them (one token's alone would take three,
// each waited for: 113 instructions a token against 80, and the latency).
// The next tokens are fetched into registers while the present ones are used.
// 8 x 509 float32 tokens of 24 heads x 64, state 128: 166 us, 67 at the FMA
// pipe's rate (three operations an element); the shared-memory loads of k and q
// and 10 warps an SM bound it.
template <class T, int CW, int R, bool REV, int OUT>
__global__ void __launch_bounds__(kThreads) k_rec(const RecArgs g) {
  constexpr int kRowTile = 16 * R, kGroup = 16 / R;  // rows per block, tokens per round of sums
  constexpr int W = CW * 8;
  constexpr int kFetch = kTok * W / 4 / kThreads;  // 4-element loads per thread, k and q each
  static_assert(kFetch >= 1 && kTok * W / 4 % kThreads == 0, "tile");
  __shared__ __align__(16) float ks[kTok][W];
  __shared__ __align__(16) float qs[OUT == kOutNone ? 1 : kTok][W];
  __shared__ __align__(16) float rs[kTok][kRowTile];
  __shared__ __align__(16) float os[OUT == kOutNone ? 1 : kTok][kRowTile + 2];
  __shared__ float as[kTok], wsm[kTok];

  if (g.only_if && *g.only_if == 0) return;
  const uint32_t tiles = (g.rows + kRowTile - 1) / kRowTile;
  uint32_t id = blockIdx.x;
  const uint32_t tile = id % tiles;
  id /= tiles;
  const uint32_t seg = id % g.nseg;
  id /= g.nseg;
  const uint32_t h = id % g.heads, b = id / g.heads;
  const int row0 = tile * kRowTile;
  const int len = clamp_length(g.lengths, b, g.length);
  const int t_lo = seg * g.seglen, t_hi = min((int)((seg + 1) * g.seglen), (int)g.length);
  const int steps = (t_hi - t_lo + kTok - 1) / kTok;

  const int tid = threadIdx.x, lane = tid & 31;
  const int c0 = 4 * (lane & 7);
  const int rp = R * ((tid >> 5) * 4 + (lane >> 3));  // first row within the tile
  const T* rbase = g.r.at<T>(b, h) + row0;
  const T* kbase = g.k.at<T>(b, h);
  const T* qbase = g.q.at<T>(b, h);
  const float* wbase = g.write.p ? g.write.p + (int64_t)b * g.write.sb + (int64_t)h * g.write.sh : nullptr;
  const float* abase = g.log_decay.p + (int64_t)b * g.log_decay.sb + (int64_t)h * g.log_decay.sh;

  uint64_t s[R][CW / 2];  // two columns each
  const int64_t bh = (int64_t)b * g.heads + h;
#pragma unroll
  for (int j = 0; j < R; ++j)
#pragma unroll
    for (int i = 0; i < CW; i += 2) {
      float v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = row0 + rp + j, col = c0 + (i / 4) * 32 + (i & 3) + u;
        v[u] = (OUT != kOutNone && g.state_in && row < (int)g.rows && col < (int)g.cols)
                   ? g.state_in[bh * g.in_bh + seg * g.in_seg + row * g.st_row + col * g.st_col]
                   : 0.f;
      }
      s[j][i / 2] = pair(v[0], v[1]);
    }
  float decay = 1.f;  // thread 0 of a STATE pass

  constexpr int kFetchR = kTok * kRowTile / 4 / kThreads;
  Pack<T, 4> pk[kFetch], pq[kFetch], pr[kFetchR];
  float pa = 1.f, pw = 0.f;
  auto first = [&](int step) { return REV ? t_hi - kTok * (step + 1) : t_lo + kTok * step; };
  auto fetch = [&](int step) {
    const int t0 = first(step);
    auto live = [&](int t) { return t >= t_lo && t < t_hi && t < len; };
#pragma unroll
    for (int i = 0; i < kFetch; ++i) {
      const int e = tid + i * kThreads, t = t0 + e / (W / 4), col = 4 * (e % (W / 4));
      pk[i] = load4(kbase + (int64_t)t * g.k.sl, col, g.cols, g.vec, live(t));
      if constexpr (OUT != kOutNone) pq[i] = load4(qbase + (int64_t)t * g.q.sl, col, g.cols, g.vec, live(t));
    }
#pragma unroll
    for (int i = 0; i < kFetchR; ++i) {
      const int e = tid + i * kThreads, t = t0 + e / (kRowTile / 4), col = 4 * (e % (kRowTile / 4));
      pr[i] = load4(rbase + (int64_t)t * g.r.sl, col, (int)g.rows - row0, g.vec, live(t));
    }
    if (tid < kTok) {
      const int t = t0 + tid;
      const bool l = live(t);
      pa = l ? expf(abase[(int64_t)t * g.log_decay.sl]) : 1.f;
      pw = l ? (wbase ? wbase[(int64_t)t * g.write.sl] : 1.f) : 0.f;
    }
  };
  fetch(0);
  for (int step = 0; step < steps; ++step) {
    __syncthreads();  // the previous tile's reads are done
#pragma unroll
    for (int i = 0; i < kFetch; ++i) {
      const int e = tid + i * kThreads, t = e / (W / 4), col = 4 * (e % (W / 4));
      *reinterpret_cast<float4*>(&ks[t][col]) = unpack4(pk[i]);
      if constexpr (OUT != kOutNone) *reinterpret_cast<float4*>(&qs[t][col]) = unpack4(pq[i]);
    }
#pragma unroll
    for (int i = 0; i < kFetchR; ++i) {
      const int e = tid + i * kThreads;
      *reinterpret_cast<float4*>(&rs[e / (kRowTile / 4)][4 * (e % (kRowTile / 4))]) = unpack4(pr[i]);
    }
    if (tid < kTok) {
      as[tid] = pa;
      wsm[tid] = pw;
    }
    __syncthreads();
    if (step + 1 < steps) fetch(step + 1);
#pragma unroll 1
    for (int i0 = 0; i0 < kTok; i0 += kGroup) {
      float part[16];  // [token of the group][row]
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        const int t = REV ? kTok - 1 - i0 - j : i0 + j;
        const float a = as[t], w = wsm[t];
        const uint64_t aa = pair(a, a);
        uint64_t rr[R], o[R];  // two columns at a time (f32x2)
#pragma unroll
        for (int r = 0; r < R; r += 2) {
          const float2 r2 = *reinterpret_cast<const float2*>(&rs[t][rp + r]);
          rr[r] = pair(r2.x * w, r2.x * w);
          rr[r + 1] = pair(r2.y * w, r2.y * w);
          o[r] = o[r + 1] = 0;
        }
#pragma unroll
        for (int v = 0; v < CW / 4; ++v) {
          const ulonglong2 k4 = *reinterpret_cast<const ulonglong2*>(&ks[t][c0 + 32 * v]);
          ulonglong2 q4 = make_ulonglong2(0, 0);
          if constexpr (OUT != kOutNone) q4 = *reinterpret_cast<const ulonglong2*>(&qs[t][c0 + 32 * v]);
          const uint64_t kk[2] = {k4.x, k4.y}, qq[2] = {q4.x, q4.y};
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
              uint64_t& x = s[r][2 * v + u];
              x = fma2(rr[r], kk[u], REV ? x : mul2(x, aa));
              if constexpr (OUT != kOutNone) o[r] = fma2(x, qq[u], o[r]);
              if constexpr (REV) x = mul2(x, aa);
            }
        }
        if constexpr (OUT == kOutNone) decay *= a;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float even, odd;
          unpair(o[r], even, odd);
          part[j * R + r] = even + odd;
        }
      }
      if constexpr (OUT != kOutNone) {
        // lane bits 2, 1, 0 end with entries 8, 4, 2 x those bits, and the next one
#pragma unroll
        for (int n = 8, bit = 4; n >= 2; n /= 2, bit /= 2) {
          const bool up = lane & bit;
#pragma unroll
          for (int e = 0; e < n; ++e) {
            const float keep = up ? part[e + n] : part[e], give = up ? part[e] : part[e + n];
            part[e] = keep + __shfl_xor_sync(~0u, give, bit);
          }
        }
        const int e = 2 * (lane & 7), j = e / R, t = REV ? kTok - 1 - i0 - j : i0 + j;
        *reinterpret_cast<float2*>(&os[t][rp + e % R]) = make_float2(part[0], part[1]);
      }
    }
    if constexpr (OUT != kOutNone) {
      __syncthreads();
      const int t0 = first(step);
#pragma unroll
      for (int i = 0; i < kTok * kRowTile / kThreads; ++i) {
        const int e = tid + i * kThreads, tt = e / kRowTile, rr = e % kRowTile;
        const int t = t0 + tt, row = row0 + rr;
        if (t < t_lo || t >= t_hi || row >= (int)g.rows) continue;
        const int64_t at = (((int64_t)b * g.length + t) * g.heads + h) * g.rows + row;
        float v = 0.f;
        if (t < len) {
          v = os[tt][rr];
          if constexpr (OUT == kOutDx) v *= g.out_scale.p[b * g.out_scale.sb + t * g.out_scale.sl + h * g.out_scale.sh];
          if constexpr (OUT == kOutY || OUT == kOutDx)
            if (g.d) v = fmaf(g.d[h], rs[tt][rr], v);
        }
        if constexpr (OUT == kOutRaw) static_cast<float*>(g.out)[at] = v;
        else static_cast<T*>(g.out)[at] = from_f<T>(v);
      }
    }
  }
  if (g.state_out) {
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < CW; i += 2) {
        float v[2];
        unpair(s[j][i / 2], v[0], v[1]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = row0 + rp + j, col = c0 + (i / 4) * 32 + (i & 3) + u;
          if (row < (int)g.rows && col < (int)g.cols)
            g.state_out[bh * g.out_bh + seg * g.out_seg + row * g.st_row + col * g.st_col] = v[u];
        }
      }
  }
  if (OUT == kOutNone && tile == 0 && tid == 0) g.seg_decay[bh * g.nseg + seg] = decay;
}

// One token: S' = a S + w x (x) b and y = S' c + d x.  The state is read and
// written once, which is nearly all there is to move, so memory bounds it.
// A row of S lies across G lanes in 16-byte words (NV words per lane); a warp
// takes kStepRows x 32 / G rows and has all their loads in flight at once.
// Each element is read and written by one thread: the state may be updated
// in place.  192 sequences of 24 heads x 64 x 128: 55 us, 5.5 TB/s (85% of a
// measured copy's rate).
struct StepArgs {
  Src x, b, c;
  Gate write, log_decay;
  const int32_t* lengths;
  uint32_t batch, heads, head_dim, d_state;
  const float* d;
  const float* state_in;
  float* state_out;
  void* y;
};
constexpr int kStepRows = 4;
template <class T, int G, int NV>
__global__ void __launch_bounds__(kThreads) k_step(const StepArgs g) {
  constexpr uint32_t kRows = kStepRows * 32 / G;  // per warp
  const uint32_t warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t per = (g.head_dim + kRows - 1) / kRows;  // warps per head
  const uint32_t bh = warp / per;
  if (bh >= g.batch * g.heads) return;
  const uint32_t h = bh % g.heads, b = bh / g.heads, N = g.d_state, nv = N / 4;
  const uint32_t li = lane % G, row0 = warp % per * kRows + lane / G;
  const float4* in = reinterpret_cast<const float4*>(g.state_in ? g.state_in + (int64_t)bh * g.head_dim * N : nullptr);
  float4* out = reinterpret_cast<float4*>(g.state_out + (int64_t)bh * g.head_dim * N);
  float4 s[kStepRows][NV];
#pragma unroll
  for (int r = 0; r < kStepRows; ++r)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const uint32_t row = row0 + r * (32 / G), at = li + v * G;
      s[r][v] = in && row < g.head_dim && at < nv ? in[row * nv + at] : make_float4(0, 0, 0, 0);
    }
  const bool live = clamp_length(g.lengths, b, 1) > 0;
  float a = 1.f, w = 0.f, d = 0.f;
  float4 kb[NV], kc[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) kb[v] = kc[v] = make_float4(0, 0, 0, 0);
  const T* xp = g.x.at<T>(b, h);
  if (live) {
    a = expf(g.log_decay.p[b * g.log_decay.sb + h * g.log_decay.sh]);
    w = g.write.p[b * g.write.sb + h * g.write.sh];
    d = g.d ? g.d[h] : 0.f;
    const T *bp = g.b.at<T>(b, h), *cp = g.c.at<T>(b, h);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int at = li + v * G;
      kb[v] = unpack4(load4(bp, 4 * at, N, true, true));
      kc[v] = unpack4(load4(cp, 4 * at, N, true, true));
    }
  }
#pragma unroll
  for (int r = 0; r < kStepRows; ++r) {
    const uint32_t row = row0 + r * (32 / G);
    const bool mine = row < g.head_dim;
    const float x = live && mine ? to_f(xp[row]) : 0.f, wx = w * x;
    float o = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float4& q = s[r][v];
      q.x = fmaf(wx, kb[v].x, a * q.x);
      q.y = fmaf(wx, kb[v].y, a * q.y);
      q.z = fmaf(wx, kb[v].z, a * q.z);
      q.w = fmaf(wx, kb[v].w, a * q.w);
      o = fmaf(q.x, kc[v].x, fmaf(q.y, kc[v].y, fmaf(q.z, kc[v].z, fmaf(q.w, kc[v].w, o))));
      const uint32_t at = li + v * G;
      if (mine && at < nv) out[row * nv + at] = q;
    }
#pragma unroll
    for (int e = G / 2; e; e >>= 1) o += __shfl_xor_sync(~0u, o, e);
    if (mine && li == 0) static_cast<T*>(g.y)[(int64_t)bh * g.head_dim + row] = from_f<T>(live ? fmaf(d, x, o) : 0.f);
  }
}

// Carries the segments' states across a row.  slots [bh][nseg + 1][size]:
// forward, slot s + 1 holds segment s's state from zero and becomes the state
// at its end, slot 0 the initial state; reversed, slot s holds what segment s
// passes back from zero and becomes the gradient of the state before it,
// slot nseg the final state's gradient.  `end` receives the last slot written;
// `bad` (or nullptr) is cleared for the walks to come.
template <bool REV>
__global__ void k_join(float* slots, const float* seg_decay, const float* start, float* end, uint32_t nseg,
                       uint32_t size, int* bad) {
  if (bad && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *bad = 0;
  const uint32_t e = blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t bh = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (e >= size) return;
  float* at = slots + bh * (nseg + 1) * (int64_t)size + e;
  float v = start ? start[bh * size + e] : 0.f;
  at[REV ? (int64_t)nseg * size : 0] = v;
  for (uint32_t i = 0; i < nseg; ++i) {
    const uint32_t s = REV ? nseg - 1 - i : i;
    float* p = at + (int64_t)(REV ? s : s + 1) * size;
    v = fmaf(seg_decay[bh * nseg + s], v, *p);
    *p = v;
  }
  if (end) end[bh * size + e] = v;
}

// gamma[bh][s] = <gradient, state> at the end of segment s.
__global__ void __launch_bounds__(256) k_anchor(const float* s_slots, const float* d_slots, float* gamma, uint32_t nseg,
                                                uint32_t size) {
  const int64_t bh = blockIdx.x / nseg;
  const uint32_t seg = blockIdx.x % nseg;
  const int64_t at = (bh * (nseg + 1) + seg + 1) * (int64_t)size;
  float v = 0.f;
  if (size % 4 == 0) {  // the slots start 256-byte aligned
    const float4 *s = reinterpret_cast<const float4*>(s_slots + at), *d = reinterpret_cast<const float4*>(d_slots + at);
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < size / 4; i += 256) {
      const float4 x = s[i], y = d[i];
      v = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, v))));
    }
  } else {
    for (uint32_t i = threadIdx.x; i < size; i += 256) v = fmaf(s_slots[at + i], d_slots[at + i], v);
  }
  __shared__ float part[8];
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) v += part[i];
    gamma[bh * nseg + seg] = v;
  }
}

struct SumArgs {
  Src x, b, c;
  Gate write;
  const void* dy;
  const int32_t* lengths;
  uint32_t length, heads, head_dim, d_state, groups;
  const float *u, *dch;  // [b][length][heads][d_state]
  void *db, *dc;
  float* dwrite;
  float* diff;  // [b][length][heads]: alpha - beta
  float* skip;  // [b][length][heads]: <dy, x>, or nullptr
};

// Sums COUNT values of every lane over the warp; lane i ends with the sum of
// value i % COUNT (a power of two): each step halves the values a lane holds.
template <int COUNT>
__device__ __forceinline__ float sum_each(float (&v)[COUNT], uint32_t lane) {
#pragma unroll
  for (int n = COUNT / 2; n >= 1; n /= 2) {
    const bool up = lane & n;
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = (up ? v[i + n] : v[i]) + __shfl_xor_sync(~0u, up ? v[i] : v[i + n], n);
  }
  float r = v[0];
#pragma unroll
  for (int o = COUNT; o < 32; o <<= 1) r += __shfl_xor_sync(~0u, r, o);
  return r;
}

// One warp per token: sums U and dC_h over the heads of each group in order
// and forms the per-head products.  Memory-bound: it reads the two per-head
// arrays once, H heads at a time with all their loads in flight.  A lane holds
// V neighbouring columns of every 32 V, NP of those.  4 x 2048 bfloat16 tokens of
// 24 heads: 94 us, 2.7 TB/s (a block of 8 warps per token: 180 us).
template <class T, int V, int NP, int H>
__global__ void __launch_bounds__(128) k_sum(const SumArgs g, uint32_t tokens) {
  const uint32_t id = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;  // threads may pass 2^32
  if (id >= tokens) return;
  const uint32_t t = id % g.length, b = id / g.length;
  const bool live = (int)t < clamp_length(g.lengths, b, g.length);
  const uint32_t each = g.heads / g.groups, N = g.d_state, P = g.head_dim;
  const int64_t tok = id;
  for (uint32_t grp = 0; grp < g.groups; ++grp) {
    const T* bp = g.b.at<T>(b, grp * each) + (int64_t)t * g.b.sl;
    const T* cp = g.c.at<T>(b, grp * each) + (int64_t)t * g.c.sl;
    float bv[NP][V], cv[NP][V], sb[NP][V], sc[NP][V];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const uint32_t n = (i * 32 + lane) * V + v;
        bv[i][v] = live && n < N ? to_f(bp[n]) : 0.f;
        cv[i][v] = live && n < N ? to_f(cp[n]) : 0.f;
        sb[i][v] = sc[i][v] = 0.f;
      }
    for (uint32_t h0 = 0; h0 < each; h0 += H) {
      Pack<float, V> u[H][NP], dc[H][NP];
      // lane j < H: write of head h0 + j
      const uint32_t mine = grp * each + h0 + lane % H;
      const bool has = live && h0 + lane % H < each;
      const float wl = has ? g.write.p[b * g.write.sb + t * g.write.sl + mine * g.write.sh] : 0.f;
#pragma unroll
      for (int j = 0; j < H; ++j)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const uint32_t n = (i * 32 + lane) * V;
          const int64_t at = (tok * g.heads + grp * each + h0 + j) * N + n;
#pragma unroll
          for (int v = 0; v < V; ++v) u[j][i].v[v] = dc[j][i].v[v] = 0.f;
          if (live && h0 + j < each && n < N) {  // N is a multiple of V
            u[j][i] = *reinterpret_cast<const Pack<float, V>*>(g.u + at);
            dc[j][i] = *reinterpret_cast<const Pack<float, V>*>(g.dch + at);
          }
        }
      float dot[2 * H], skip[H];  // <b, U>, then <c, dC_h>; <x, dy>
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const float w = __shfl_sync(~0u, wl, j);
        dot[j] = dot[j + H] = skip[j] = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            dot[j] = fmaf(bv[i][v], u[j][i].v[v], dot[j]);
            dot[j + H] = fmaf(cv[i][v], dc[j][i].v[v], dot[j + H]);
            sb[i][v] = fmaf(w, u[j][i].v[v], sb[i][v]);
            sc[i][v] += dc[j][i].v[v];
          }
        if (g.skip && live && h0 + j < each) {
          const uint32_t h = grp * each + h0 + j;
          const T* xp = g.x.at<T>(b, h) + (int64_t)t * g.x.sl;
          const T* dyp = static_cast<const T*>(g.dy) + (tok * g.heads + h) * P;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t p = lane + 32 * i;
            if (p < P) skip[j] = fmaf(to_f(xp[p]), to_f(dyp[p]), skip[j]);
          }
        }
      }
      const float d = sum_each(dot, lane);  // lane j: <b, U> of head j, lane j + H: alpha
      const float alpha = __shfl_down_sync(~0u, d, H);
      const float sk = g.skip ? sum_each(skip, lane) : 0.f;
      if (lane < H && h0 + lane < each) {
        const int64_t at = tok * g.heads + mine;
        g.dwrite[at] = d;
        g.diff[at] = alpha - wl * d;
        if (g.skip) g.skip[at] = sk;
      }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t n = (i * 32 + lane) * V;
      if (n < N) {
        const int64_t at = (tok * g.groups + grp) * N + n;
        *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(g.db) + at) = pack<T>(sb[i]);
        *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(g.dc) + at) = pack<T>(sc[i]);
      }
    }
  }
}

// One warp per (batch, head, segment): the running sum of alpha - beta from
// the segment's end (fp64: it is a difference of sums), which starts anew from
// an exact 0 at a token that clears the state, and the segment's share of dd.
__global__ void __launch_bounds__(128)
    k_log_decay_grad(const float* diff, const float* skip, const float* gamma, Gate log_decay, const int32_t* lengths,
                     float* out, float* dd_part, uint32_t length, uint32_t heads, uint32_t seglen, uint32_t nseg,
                     uint32_t count) {
  const uint32_t id = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;  // blocks of 128 threads
  if (id >= count) return;
  const uint32_t seg = id % nseg, h = id / nseg % heads, b = id / nseg / heads;
  const int len = clamp_length(lengths, b, length);
  const int t_lo = seg * seglen, t_hi = min(t_lo + seglen, length);
  double carry = gamma[id];
  float dd = 0.f;
  for (int hi = t_hi; hi > t_lo; hi -= 32) {
    const int t = hi - 1 - (int)lane;
    const bool in = t >= t_lo;
    const int64_t at = ((int64_t)b * length + (in ? t : t_lo)) * heads + h;
    const bool live = in && t < len;
    const float la = live ? log_decay.p[b * log_decay.sb + t * log_decay.sl + h * log_decay.sh] : 0.f;
    bool cut = expf(la) == 0.f;  // the sum before this lane's token owes nothing to later ones
    double v = in && !cut ? diff[at] : 0.0;
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(~0u, v, o);
      const bool c = __shfl_up_sync(~0u, cut, o);
      if ((int)lane >= o && !cut) {
        v += u;
        cut = c;
      }
    }
    if (!cut) v += carry;
    if (in) {
      out[at] = live ? (float)v : 0.f;
      if (skip && live) dd += skip[at];
    }
    carry = __shfl_sync(~0u, v, 31);
  }
  if (skip) {
    for (int o = 16; o; o >>= 1) dd += __shfl_xor_sync(~0u, dd, o);
    if (lane == 0) dd_part[id] = dd;
  }
}

__global__ void k_dd(const float* part, float* dd, uint32_t batch, uint32_t heads, uint32_t nseg) {
  const uint32_t h = blockIdx.x, lane = threadIdx.x;
  float v = 0.f;
  for (uint32_t i = lane; i < batch * nseg; i += 32) v += part[((int64_t)(i / nseg) * heads + h) * nseg + i % nseg];
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (lane == 0) dd[h] = v;
}

// ---- host -----------------------------------------------------------------

void check_scan(const fhe_ssm_scan_args& a) {
  require(a.dtype == FHE_F32 || a.dtype == FHE_BF16 || a.dtype == FHE_F16, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
  require(a.heads >= 1 && a.groups >= 1 && a.heads % a.groups == 0, "heads must be a positive multiple of groups");
  require(a.head_dim >= 1 && a.head_dim <= 128, "head_dim must be in [1, 128]");
  require(a.d_state >= 1 && a.d_state <= 256, "d_state must be in [1, 256]");
  require(a.length <= (1u << 30) && a.batch <= (1u << 20) && a.heads <= (1u << 16), "sizes too large");
  require((uint64_t)a.batch * a.length < (1ull << 31), "batch x length must be below 2^31");
  require((uint64_t)a.batch * a.heads < (1ull << 24), "batch x heads must be below 2^24");
  require((uint64_t)a.batch * a.heads * (a.length / 16 + 1) < (1ull << 31), "batch x heads x length must be below 2^35");
}

void check_scan_pointers(const fhe_ssm_scan_args& a) {
  if (a.batch == 0) return;
  if (a.length > 0) require(a.x && a.write && a.log_decay && a.b && a.c, "null input");
}

Src src_of(const void* p, const int64_t* st, uint32_t share) { return Src{p, st[0], st[1], st[2], share}; }
Gate gate_of(const float* p, const int64_t* st) { return Gate{p, st[0], st[1], st[2]}; }

bool vec4_ok(const Src& s, uint32_t elem) {
  return reinterpret_cast<uintptr_t>(s.p) % (4 * elem) == 0 && s.sb % 4 == 0 && s.sl % 4 == 0 && s.sh % 4 == 0;
}

// Whether one token can take k_step: rows of S in 16-byte words.
bool step_ok(const fhe_ssm_scan_args& a, const StepArgs& g) {
  return a.d_state % 4 == 0 && vec4_ok(g.b, elem_size(a.dtype)) && vec4_ok(g.c, elem_size(a.dtype)) &&
         reinterpret_cast<uintptr_t>(a.initial_state) % 16 == 0 && reinterpret_cast<uintptr_t>(a.final_state) % 16 == 0;
}

template <class T>
void launch_step(const StepArgs& g, cudaStream_t st) {
  auto go = [&](auto gv, auto nv) {
    constexpr int G = decltype(gv)::value, NV = decltype(nv)::value;
    constexpr uint32_t rows = kStepRows * 32 / G;
    const uint64_t warps = (uint64_t)g.batch * g.heads * ((g.head_dim + rows - 1) / rows);
    const uint64_t blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
    require(blocks < (1ull << 25), "too many blocks");
    k_step<T, G, NV><<<(uint32_t)blocks, kThreads, 0, st>>>(g);
  };
  const uint32_t words = g.d_state / 4;
  using One = std::integral_constant<int, 1>;
  if (words <= 4) go(std::integral_constant<int, 4>{}, One{});
  else if (words <= 8) go(std::integral_constant<int, 8>{}, One{});
  else if (words <= 16) go(std::integral_constant<int, 16>{}, One{});
  else if (words <= 32) go(std::integral_constant<int, 32>{}, One{});
  else go(std::integral_constant<int, 32>{}, std::integral_constant<int, 2>{});
  note_launch();
  FHE_CUDA(cudaGetLastError());
}

// One walk; whether the tensor-core form took it.  `fp32` keeps to the fp32 form.
template <class T, bool REV, int OUT>
bool launch_rec(RecArgs g, uint32_t batch, cudaStream_t st, bool fp32) {
  if constexpr (sizeof(T) == 2)
    if (!fp32 && g.length >= kTcTokens && launch_scan_tc<T>(g, REV, OUT, batch, st)) return true;
  g.vec = vec4_ok(g.r, sizeof(T)) && vec4_ok(g.k, sizeof(T)) && (OUT == kOutNone || vec4_ok(g.q, sizeof(T)));
  auto go = [&](auto cw, auto rv) {
    constexpr int CW = decltype(cw)::value, R = decltype(rv)::value;
    const uint64_t blocks = (uint64_t)((g.rows + 16 * R - 1) / (16 * R)) * g.nseg * g.heads * batch;
    require(blocks < (1ull << 31), "too many blocks");
    k_rec<T, CW, R, REV, OUT><<<(uint32_t)blocks, kThreads, 0, st>>>(g);
  };
  using std::integral_constant;
  // narrow states: four rows to a thread, so that a token's fixed work serves as many elements
  if (g.cols <= 32 && g.rows > 32) go(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (g.cols <= 32) go(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  else if (g.cols <= 64 && g.rows > 32) go(integral_constant<int, 8>{}, integral_constant<int, 4>{});
  else if (g.cols <= 64) go(integral_constant<int, 8>{}, integral_constant<int, 2>{});
  else if (g.cols <= 128) go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  else go(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  note_launch();
  FHE_CUDA(cudaGetLastError());
  return false;
}

void launch_join(bool rev, float* slots, const float* dec, const float* start, float* end, uint32_t nseg,
                 uint32_t size, uint32_t bh, int* bad, cudaStream_t st) {
  const uint32_t y = std::min(bh, 32768u);
  // bh < 2^24; whole rows of y blocks, then the rest
  for (uint32_t at = 0; at < bh; at += y) {
    const uint32_t n = std::min(y, bh - at);
    const dim3 grid((size + 255) / 256, n, 1);
    float* sl = slots + (int64_t)at * (nseg + 1) * size;
    const float* de = dec + (int64_t)at * nseg;
    const float* b0 = start ? start + (int64_t)at * size : nullptr;
    float* e0 = end ? end + (int64_t)at * size : nullptr;
    if (rev) k_join<true><<<grid, 256, 0, st>>>(sl, de, b0, e0, nseg, size, bad);
    else k_join<false><<<grid, 256, 0, st>>>(sl, de, b0, e0, nseg, size, bad);
    note_launch();
  }
  FHE_CUDA(cudaGetLastError());
}

struct Cut {
  uint32_t seglen, nseg;
};

bool tc_type(const fhe_ssm_scan_args& a) { return a.dtype != FHE_F32 && a.length >= kTcTokens; }

// Rows are cut when the (batch, head, row tile) blocks alone leave SMs idle.
Cut forward_cut(const fhe_ssm_scan_args& a) {
  if (tc_type(a)) {
    // two CTAs of 64 rows to an SM; segments of whole chunks of 128 tokens
    const uint64_t blocks = (uint64_t)a.batch * a.heads * ((a.head_dim + 63) / 64);
    const uint32_t chunks = (a.length + 127) / 128;
    uint32_t nseg = 1;
    if (blocks < 148) nseg = (uint32_t)std::min<uint64_t>(296 / std::max<uint64_t>(blocks, 1), std::max(1u, chunks / 2));
    nseg = std::max(1u, nseg);
    const uint32_t seglen = (chunks + nseg - 1) / nseg * 128;
    return {seglen, std::max(1u, (a.length + seglen - 1) / seglen)};
  }
  const uint64_t blocks = (uint64_t)a.batch * a.heads * ((a.head_dim + 31) / 32);
  uint32_t nseg = 1;
  if (blocks < 148 * 2) nseg = (uint32_t)(148 * 4 / std::max<uint64_t>(blocks, 1));
  nseg = std::max(1u, std::min(nseg, a.length / 64));
  uint32_t seglen = (a.length + nseg - 1) / nseg;
  seglen = std::max(1u, (seglen + kTok - 1) / kTok * kTok);
  return {seglen, std::max(1u, (a.length + seglen - 1) / seglen)};
}

// The backward pass cuts rows into segments of at most 128 tokens: its running
// sums start anew at each, and its walks, which read every segment's start,
// have that many more blocks (8 x 509 fp32: 0.91 ms, 0.99 with 256).
Cut backward_cut(const fhe_ssm_scan_args& a) {
  Cut c = forward_cut(a);
  c.seglen = tc_type(a) ? 128u : std::min(c.seglen, 128u);
  c.nseg = std::max(1u, (a.length + c.seglen - 1) / c.seglen);
  return c;
}

RecArgs rec_args(const fhe_ssm_scan_args& a, const Cut& cut) {
  RecArgs g{};
  g.log_decay = gate_of(a.log_decay, a.log_decay_stride);
  g.lengths = a.lengths;
  g.length = a.length;
  g.heads = a.heads;
  g.seglen = cut.seglen;
  g.nseg = cut.nseg;
  return g;
}

}  // namespace

namespace {
struct ForwardSpace {
  int* bad;
  float *slots, *dec, *start;
  uint64_t bytes;
};
ForwardSpace forward_space(const fhe_ssm_scan_args& a, const Cut& cut, void* base) {
  const uint64_t bh = (uint64_t)a.batch * a.heads;
  Carver w(base);
  ForwardSpace s{};
  if (tc_type(a)) s.bad = w.take<int>(1);
  if (cut.nseg > 1) {
    s.slots = w.take<float>(bh * (cut.nseg + 1) * a.head_dim * a.d_state);
    s.dec = w.take<float>(bh * cut.nseg);
  } else if (tc_type(a) && a.initial_state && a.initial_state == a.final_state) {
    s.start = w.take<float>(bh * a.head_dim * a.d_state);  // a second walk must not start from the first one's end
  }
  s.bytes = w.used;
  return s;
}
}  // namespace

uint64_t ssm_scan_workspace(const fhe_ssm_scan_args& a) {
  check_scan(a);
  if (a.batch == 0 || a.length == 0) return 0;
  return forward_space(a, forward_cut(a), nullptr).bytes;
}

void ssm_scan(const fhe_ssm_scan_args& a) {
  check_scan(a);
  check_scan_pointers(a);
  if (a.batch == 0) return;
  require(a.final_state != nullptr && (a.y != nullptr || a.length == 0), "null output");
  check_workspace(a.workspace, a.workspace_bytes, ssm_scan_workspace(a));
  DeviceGuard dev(a.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  const uint32_t size = a.head_dim * a.d_state, bh = a.batch * a.heads;
  if (a.length == 0) {
    if (a.initial_state == a.final_state) return;
    const size_t n = (size_t)bh * size * 4;
    if (a.initial_state) FHE_CUDA(cudaMemcpyAsync(a.final_state, a.initial_state, n, cudaMemcpyDeviceToDevice, st));
    else FHE_CUDA(cudaMemsetAsync(a.final_state, 0, n, st));
    return;
  }
  const Cut cut = forward_cut(a);
  RecArgs g = rec_args(a, cut);
  const uint32_t each = a.heads / a.groups;
  g.r = src_of(a.x, a.x_stride, 1);
  g.k = src_of(a.b, a.b_stride, each);
  g.q = src_of(a.c, a.c_stride, each);
  g.write = gate_of(a.write, a.write_stride);
  g.rows = a.head_dim;
  g.cols = a.d_state;
  g.d = a.d;
  g.st_row = a.d_state;
  g.st_col = 1;
  g.out = a.y;
  const StepArgs one{g.r, g.k, g.q, g.write, g.log_decay, a.lengths, a.batch, a.heads, a.head_dim, a.d_state,
                     a.d, a.initial_state, a.final_state, a.y};
  with_type(a.dtype, [&](auto v) {
    using T = decltype(v);
    if (a.length == 1 && step_ok(a, one)) return launch_step<T>(one, st);
    const ForwardSpace sp = forward_space(a, cut, a.workspace);
    const float* start = a.initial_state;
    if (sp.start) {
      FHE_CUDA(cudaMemcpyAsync(sp.start, start, (size_t)bh * size * 4, cudaMemcpyDeviceToDevice, st));
      start = sp.start;
    }
    RecArgs r = g;
    r.bad = sp.bad;
    if (cut.nseg > 1) {
      r.seg_decay = sp.dec;
      r.out_bh = (int64_t)(cut.nseg + 1) * size;
      r.out_seg = size;
      r.state_out = sp.slots + size;
      launch_rec<T, false, kOutNone>(r, a.batch, st, false);
      launch_join(false, sp.slots, sp.dec, start, a.final_state, cut.nseg, size, bh, sp.bad, st);
      r.state_in = sp.slots;
      r.in_bh = r.out_bh;
      r.in_seg = size;
      r.state_out = nullptr;
    } else {
      if (sp.bad) FHE_CUDA(cudaMemsetAsync(sp.bad, 0, sizeof(int), st));
      r.state_in = start;
      r.state_out = a.final_state;
      r.in_bh = r.out_bh = size;
    }
    if (launch_rec<T, false, kOutY>(r, a.batch, st, false)) {
      r.only_if = sp.bad;
      launch_rec<T, false, kOutY>(r, a.batch, st, true);
    }
  });
}

namespace {
struct BackwardSpace {
  int* bad;
  float *s_slots, *d_slots, *dec_f, *dec_r, *gamma, *u, *dch, *diff, *skip, *dd_part;
  uint64_t bytes;
};
BackwardSpace backward_space(const fhe_ssm_scan_grad_args& g, const Cut& cut, void* base) {
  const fhe_ssm_scan_args& a = g.f;
  const uint64_t bh = (uint64_t)a.batch * a.heads, tok = (uint64_t)a.batch * a.length * a.heads;
  const uint64_t slots = bh * (cut.nseg + 1) * a.head_dim * a.d_state;
  Carver w(base);
  BackwardSpace s{};
  s.s_slots = w.take<float>(slots);
  s.d_slots = w.take<float>(slots);
  s.dec_f = w.take<float>(bh * cut.nseg);
  s.dec_r = w.take<float>(bh * cut.nseg);
  s.gamma = w.take<float>(bh * cut.nseg);
  s.u = w.take<float>(tok * a.d_state);
  s.dch = w.take<float>(tok * a.d_state);
  s.diff = w.take<float>(tok);
  s.skip = w.take<float>(tok);
  s.dd_part = w.take<float>(bh * cut.nseg);
  if (tc_type(a)) s.bad = w.take<int>(1);
  s.bytes = w.used;
  return s;
}
}  // namespace

uint64_t ssm_scan_backward_workspace(const fhe_ssm_scan_grad_args& g) {
  check_scan(g.f);
  if (g.f.batch == 0 || g.f.length == 0) return 0;
  return backward_space(g, backward_cut(g.f), nullptr).bytes;
}

void ssm_scan_backward(const fhe_ssm_scan_grad_args& g) {
  const fhe_ssm_scan_args& a = g.f;
  check_scan(a);
  check_scan_pointers(a);
  check_workspace(g.workspace, g.workspace_bytes, ssm_scan_backward_workspace(g));
  DeviceGuard dev(a.device);
  cudaStream_t st = static_cast<cudaStream_t>(g.stream);
  const uint32_t size = a.head_dim * a.d_state, bh = a.batch * a.heads;
  if (bh == 0 || a.length == 0) {
    if (g.dd) FHE_CUDA(cudaMemsetAsync(g.dd, 0, a.heads * 4, st));
    if (g.dinitial && bh) {
      if (g.dfinal) FHE_CUDA(cudaMemcpyAsync(g.dinitial, g.dfinal, (size_t)bh * size * 4, cudaMemcpyDeviceToDevice, st));
      else FHE_CUDA(cudaMemsetAsync(g.dinitial, 0, (size_t)bh * size * 4, st));
    }
    return;
  }
  require(g.dy && g.dx && g.dwrite && g.dlog_decay && g.db && g.dc, "null gradient");
  const Cut cut = backward_cut(a);
  const BackwardSpace s = backward_space(g, cut, g.workspace);
  const uint32_t each = a.heads / a.groups;
  const Src x = src_of(a.x, a.x_stride, 1), b = src_of(a.b, a.b_stride, each), c = src_of(a.c, a.c_stride, each);
  const Src dy{g.dy, (int64_t)a.length * a.heads * a.head_dim, (int64_t)a.heads * a.head_dim, a.head_dim, 1};
  const Gate write = gate_of(a.write, a.write_stride);
  const int64_t slot_bh = (int64_t)(cut.nseg + 1) * size;
  with_type(a.dtype, [&](auto v) {
    using T = decltype(v);
    RecArgs base = rec_args(a, cut);
    base.bad = s.bad;
    base.in_bh = base.out_bh = slot_bh;
    base.in_seg = base.out_seg = size;
    base.rows = a.head_dim;
    base.cols = a.d_state;
    base.st_row = a.d_state;
    base.st_col = 1;
    {  // states at the segments' ends
      RecArgs r = base;
      r.r = x; r.k = b; r.q = c;
      r.write = write;
      r.state_out = s.s_slots + size;
      r.seg_decay = s.dec_f;
      launch_rec<T, false, kOutNone>(r, a.batch, st, false);
      launch_join(false, s.s_slots, s.dec_f, a.initial_state, nullptr, cut.nseg, size, bh, s.bad, st);
    }
    {  // gradients of the states before the segments
      RecArgs r = base;
      r.r = dy; r.k = c; r.q = b;
      r.state_out = s.d_slots;
      r.seg_decay = s.dec_r;
      launch_rec<T, true, kOutNone>(r, a.batch, st, false);
      launch_join(true, s.d_slots, s.dec_r, g.dfinal, g.dinitial, cut.nseg, size, bh, nullptr, st);
    }
    auto walks = [&](bool fp32, const int* only_if) {
      bool tc = false;
      RecArgs r = base;
      r.only_if = only_if;
      r.r = dy; r.k = c; r.q = b;
      r.state_in = s.d_slots + size;
      r.out_scale = write;
      r.d = a.d;
      r.out = g.dx;
      tc |= launch_rec<T, true, kOutDx>(r, a.batch, st, fp32);
      r.d = nullptr;
      r.rows = a.d_state;
      r.cols = a.head_dim;
      r.st_row = 1;
      r.st_col = a.d_state;
      r.r = c; r.k = dy; r.q = x;  // out_scale: for the tensor-core form's roundings alone
      r.out = s.u;
      tc |= launch_rec<T, true, kOutRaw>(r, a.batch, st, fp32);
      r.r = b; r.k = x; r.q = dy;
      r.out_scale = Gate{};
      r.write = write;
      r.state_in = s.s_slots;
      r.out = s.dch;
      tc |= launch_rec<T, false, kOutRaw>(r, a.batch, st, fp32);
      return tc;
    };
    if (walks(false, nullptr)) walks(true, s.bad);
    k_anchor<<<bh * cut.nseg, 256, 0, st>>>(s.s_slots, s.d_slots, s.gamma, cut.nseg, size);
    note_launch();
    SumArgs u{x, b, c, write, g.dy, a.lengths, a.length, a.heads, a.head_dim, a.d_state, a.groups,
              s.u, s.dch, g.db, g.dc, g.dwrite, s.diff, g.dd ? s.skip : nullptr};
    const uint32_t tokens = a.batch * a.length, grid = (tokens + 3) / 4;
    const bool wide = a.d_state % 4 == 0 && reinterpret_cast<uintptr_t>(g.db) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(g.dc) % 16 == 0;
    if (wide && a.d_state <= 128) k_sum<T, 4, 1, 8><<<grid, 128, 0, st>>>(u, tokens);
    else if (wide) k_sum<T, 4, 2, 4><<<grid, 128, 0, st>>>(u, tokens);
    else k_sum<T, 1, 8, 4><<<grid, 128, 0, st>>>(u, tokens);
    note_launch();
  });
  const uint32_t count = bh * cut.nseg;
  k_log_decay_grad<<<(count + 3) / 4, 128, 0, st>>>(s.diff, g.dd ? s.skip : nullptr, s.gamma,
                                                    gate_of(a.log_decay, a.log_decay_stride), a.lengths,
                                                    g.dlog_decay, s.dd_part, a.length, a.heads, cut.seglen, cut.nseg,
                                                    count);
  note_launch();
  if (g.dd) {
    k_dd<<<a.heads, 32, 0, st>>>(s.dd_part, g.dd, a.batch, a.heads, cut.nseg);
    note_launch();
  }
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
