// Token embedding and its gradient (fhe_embedding).
//
// The lookup moves rows: a warp a row, 16 bytes a lane.  The gradient of a table
// row is the sum over the positions that hold its token, so positions are sorted
// by token: runs of 256 by counting, then groups of 32 runs put together by rank
// (an element's place is its own index plus, for every other run, how many of its
// elements come before, found by halving), which waits for nothing and keeps equal
// tokens in the order of their positions.  Blocks of equally many sorted positions
// then sum the rows; a token that reaches past its block leaves partial sums, which a
// last launch adds in order.  No atomics: the same call gives the same bits.  Rows
// without a position are cleared by blocks beside those that sort.
//
// 32768 tokens of natural text's frequencies, 50280 x 768 bfloat16, float32 outputs:
// lookup 22 us (5.2 TB/s); gradient 68 us, of which sorting and clearing (77 MB) 32, the
// sums (115 MB) 25, at 4.6 TB/s by the loads of scattered rows, and the joins 11, a chain
// of dependent loads (the first token has 2100 positions).
#include <algorithm>

#include "launch_count.h"
#include "mamba_ops.h"

namespace fhe {
namespace {

constexpr uint32_t kRun = 256, kMerge = 32, kMergeWarps = 8;
constexpr uint32_t kNone = ~0u;  // sorts behind every token
constexpr int kAhead = 8;        // rows in flight

template <class I>
__device__ __forceinline__ uint32_t token_at(const void* ids, uint32_t i, uint32_t vocab) {
  const I t = static_cast<const I*>(ids)[i];
  return t < 0 || (uint64_t)t >= vocab ? kNone : (uint32_t)t;
}
__device__ __forceinline__ uint32_t token_of(const void* ids, bool wide, uint32_t i, uint32_t vocab) {
  return wide ? token_at<int64_t>(ids, i, vocab) : token_at<int32_t>(ids, i, vocab);
}

// A warp takes R positions at a time, all their loads before the first store.  V
// elements a lane: as many as make 16 bytes of the output, so that a warp's stores
// are whole lines; 1 where alignment does not allow that.
template <class T, class Y, int V, int R>
__global__ void __launch_bounds__(128) k_embed(const fhe_embedding_args g) {
  constexpr int kCols = V > 1 ? 2 : 4;  // loads of a lane and position in a turn
  const uint32_t lane = threadIdx.x % 32, i0 = (blockIdx.x * 4 + threadIdx.x / 32) * R;
  uint32_t t[R];
#pragma unroll
  for (int r = 0; r < R; ++r) t[r] = i0 + r < g.count ? token_of(g.ids, g.wide_ids, i0 + r, g.vocab) : kNone;
  const T* table = static_cast<const T*>(g.table);
  Y* out = static_cast<Y*>(g.out) + (int64_t)i0 * g.width;
  for (uint32_t c0 = lane * V; c0 < g.width; c0 += kCols * 32 * V) {
    Pack<T, V> p[R][kCols];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < kCols; ++j)
        if (t[r] != kNone && c0 + j * 32 * V < g.width)
          p[r][j] = *reinterpret_cast<const Pack<T, V>*>(table + (int64_t)t[r] * g.table_stride + c0 + j * 32 * V);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (i0 + r >= g.count) break;
      float none = 0.f;
      if (t[r] == kNone)
        none = (g.wide_ids ? static_cast<const int64_t*>(g.ids)[i0 + r] >= 0
                           : static_cast<const int32_t*>(g.ids)[i0 + r] >= 0) ? NAN : 0.f;
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        if (c0 + j * 32 * V >= g.width) break;
        float f[V];
        unpack(p[r][j], f);
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = t[r] == kNone ? none : f[k] * g.scale;
        *reinterpret_cast<Pack<Y, V>*>(out + (int64_t)r * g.width + c0 + j * 32 * V) = pack<Y, V>(f);
      }
    }
  }
}

// The part `b` of `blocks` of the table's gradient, cleared by a block.
__device__ __forceinline__ void clear(uint8_t* p, uint64_t bytes, uint64_t b, uint64_t blocks) {
  const uint64_t head = min(bytes, (uint64_t)((0 - reinterpret_cast<uintptr_t>(p)) % 16)), words = (bytes - head) / 16;
  const uint64_t each = (words + blocks - 1) / blocks, first = min(words, b * each), last = min(words, first + each);
  uint4* w = reinterpret_cast<uint4*>(p + head);
#pragma unroll 8
  for (uint64_t i = first + threadIdx.x; i < last; i += blockDim.x) w[i] = make_uint4(0, 0, 0, 0);
  if (b == 0) {
    for (uint64_t i = threadIdx.x; i < head; i += blockDim.x) p[i] = 0;
    for (uint64_t i = head + words * 16 + threadIdx.x; i < bytes; i += blockDim.x) p[i] = 0;
  }
}

struct Sorted {
  uint32_t *token, *pos;
};
struct Fill {
  uint8_t* p;
  uint64_t bytes;
  uint32_t blocks;  // before the launch's own, so that they write while those wait
};

// The blocks behind those that clear sort a run of positions by (token, position), a
// thread a position whose place is the number of those before it.
__global__ void __launch_bounds__(kRun) k_sort(const void* ids, bool wide, uint32_t count, uint32_t vocab, Sorted out,
                                               Fill fill) {
  __shared__ __align__(16) uint32_t token[kRun];
  if (blockIdx.x < fill.blocks) return clear(fill.p, fill.bytes, blockIdx.x, fill.blocks);
  const uint32_t first = (blockIdx.x - fill.blocks) * kRun, i = threadIdx.x, n = min(kRun, count - first);
  const uint32_t t = i < n ? token_of(ids, wide, first + i, vocab) : kNone;
  token[i] = t;
  __syncthreads();
  uint32_t at = 0;
#pragma unroll 16
  for (uint32_t j = 0; j < kRun; j += 4) {
    const uint4 o = *reinterpret_cast<const uint4*>(&token[j]);
    at += (o.x < t) + (o.y < t) + (o.z < t) + (o.w < t);
    at += (o.x == t && j < i) + (o.y == t && j + 1 < i) + (o.z == t && j + 2 < i) + (o.w == t && j + 3 < i);
  }
  if (i < n) {
    out.token[first + at] = t;
    out.pos[first + at] = first + i;
  }
}

// Puts groups of kMerge sorted runs of `run` (a power of two) elements together, 32
// elements to a block: its warps share the other runs, four searches of a lane at a
// time.  The first blocks clear.
__global__ void __launch_bounds__(32 * kMergeWarps) k_merge(Sorted in, Sorted out, uint32_t count, uint32_t run_log,
                                                            Fill fill) {
  __shared__ uint32_t places[kMergeWarps][32];
  if (blockIdx.x < fill.blocks) return clear(fill.p, fill.bytes, blockIdx.x, fill.blocks);
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint64_t at0 = (uint64_t)(blockIdx.x - fill.blocks) * 32;
  const uint32_t e = (uint32_t)at0 + lane;
  const bool live = e < count;
  const uint32_t t = live ? in.token[e] : 0;
  const uint64_t group = (uint64_t)kMerge << run_log, base = at0 / group * group;
  const uint32_t mine = (uint32_t)((at0 - base) >> run_log);  // the block's elements lie in one run
  const uint32_t runs = (uint32_t)min((uint64_t)kMerge, ((uint64_t)count - base + ((uint64_t)1 << run_log) - 1) >> run_log);
  uint32_t before_me = 0;
  for (uint32_t r0 = warp; r0 < runs; r0 += 4 * kMergeWarps) {
    const uint32_t* p[4];
    uint32_t n[4], lo[4], top[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t r = r0 + k * kMergeWarps;
      const uint64_t first = base + ((uint64_t)r << run_log);
      const bool other = r < runs && r != mine;
      p[k] = in.token + (other ? first : 0);
      n[k] = other ? (uint32_t)min((uint64_t)1 << run_log, (uint64_t)count - first) : 0;
      lo[k] = 0;
      top[k] = t + (r < mine);  // equal tokens of earlier runs come before (kNone wraps: see below)
    }
    for (uint32_t step = 1u << run_log; step; step >>= 1) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t at = lo[k] + step;
        if (at <= n[k] && p[k][at - 1] < top[k]) lo[k] = at;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) before_me += t == kNone && top[k] == 0 ? n[k] : lo[k];  // nothing is past kNone
  }
  places[warp][lane] = before_me;
  __syncthreads();
  if (warp == 0 && live) {
    uint64_t at = base + (e - base - ((uint64_t)mine << run_log));
    for (uint32_t w = 0; w < kMergeWarps; ++w) at += places[w][lane];
    out.token[at] = t;
    out.pos[at] = in.pos[e];
  }
}

// blockDim.y blocks of `chunk` sorted positions, V columns to a thread.  A token
// whose positions lie in one block is written whole; else its sums go to
// part[block][0] (began earlier) or part[block][1] (begins here).
template <class T, class Y, int V>
__global__ void __launch_bounds__(256) k_sum(const fhe_embedding_grad_args a, Sorted s, uint32_t chunk, uint32_t chunks,
                                             float* part) {
  const uint32_t c = blockIdx.x * blockDim.y + threadIdx.y, col = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const uint32_t count = a.f.count, width = a.f.width;
  if (c >= chunks || col >= width) return;
  const uint32_t first = c * chunk, last = min(count, first + chunk);
  const Y* dy = static_cast<const Y*>(a.dout) + col;
  uint32_t now = s.token[first];
  if (now == kNone) return;
  bool begins = first == 0 || s.token[first - 1] != now;
  float acc[V];
  vset(acc, 0.f);
  auto put = [&](bool ends) {
    if (begins && ends) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = acc[v] * a.f.scale;
      *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.dtable) + (int64_t)now * width + col) = pack<T, V>(o);
    } else {
      float* to = part + ((int64_t)c * 2 + begins) * width + col;
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = acc[v];
    }
  };
  for (uint32_t i = first; i < last; i += kAhead) {
    uint32_t token[kAhead];
    Pack<Y, V> row[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      token[j] = i + j < last ? s.token[i + j] : kNone;
      if (token[j] != kNone) row[j] = *reinterpret_cast<const Pack<Y, V>*>(dy + (int64_t)s.pos[i + j] * width);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (token[j] != now) {  // the same for the whole block
        if (token[j] == kNone) {
          put(i + j < last || last == count || s.token[last] != now);
          return;
        }
        put(true);
        now = token[j];
        begins = true;
        vset(acc, 0.f);
      }
      float f[V];
      unpack(row[j], f);
      vadd(acc, acc, f);
    }
  }
  put(last == count || s.token[last] != now);
}

// Adds the partial sums of the tokens that begin in one of kJoin blocks of positions
// and reach past it: each warp looks at one of the blocks.  Up to kFew shares are
// added in order by a warp, four columns a lane, a token a warp; more by the whole
// CTA, strand y every eighth share, the strands in order.
constexpr uint32_t kJoin = 8, kFew = 16;
template <class T, bool VEC>
__global__ void __launch_bounds__(32 * kJoin) k_join(const fhe_embedding_grad_args a, Sorted s, uint32_t chunk,
                                                     uint32_t chunks, const float* part) {
  __shared__ float4 sums[kJoin][32];
  __shared__ uint32_t tokens[kJoin], stops[kJoin];
  const uint32_t count = a.f.count, width = a.f.width;
  {
    const uint32_t c = blockIdx.x * kJoin + threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t first = c * chunk, next = first + chunk;
    uint32_t t = kNone, stop = c + 1;  // the last block with a share: its first position has the token
    if (c < chunks && next < count) {
      t = s.token[next - 1];
      const uint32_t after = s.token[next], begin = s.token[first], prior = first ? s.token[first - 1] : kNone;
      if (after != t || (begin == t && prior == t)) t = kNone;  // ends here, or began earlier
    }
    while (t != kNone) {  // the same for the whole warp
      bool same[4];  // four blocks a lane, in order over the lanes
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t b = stop + 1 + k * 32 + lane;
        same[k] = b < chunks && s.token[b * chunk] == t;
      }
      uint32_t run = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t some = __ballot_sync(~0u, same[k]);
        if (run == k * 32u) run += some == ~0u ? 32 : __ffs((int)~some) - 1;
      }
      stop += run;
      if (run < 128) break;
    }
    if (lane == 0) {
      tokens[threadIdx.x / 32] = t;
      stops[threadIdx.x / 32] = stop;
    }
  }
  __syncthreads();
  const uint32_t x = threadIdx.x % 32, y = threadIdx.x / 32;
  auto add = [&](float (&v)[4], uint32_t c, uint32_t b, uint32_t stop, uint32_t step, uint32_t col) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = 0.f;
#pragma unroll 8
    for (; b <= stop; b += step) {
      const float* p = part + ((int64_t)b * 2 + (b == c)) * width + col;
      if constexpr (VEC) {
        if (col < width) {
          const float4 q = *reinterpret_cast<const float4*>(p);
          v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col + k < width) v[k] += p[k];
      }
    }
  };
  auto put = [&](const float (&v)[4], uint32_t t, uint32_t col) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < width) static_cast<T*>(a.dtable)[(int64_t)t * width + col + k] = from_f<T>(v[k] * a.f.scale);
  };
  bool more = false;
  for (uint32_t i = 0; i < kJoin; ++i) more = more || (tokens[i] != kNone && stops[i] - (blockIdx.x * kJoin + i) >= kFew);
  if (tokens[y] != kNone && stops[y] - (blockIdx.x * kJoin + y) < kFew) {
    const uint32_t t = tokens[y], c = blockIdx.x * kJoin + y;
    for (uint32_t base = blockIdx.y * 128; base < width; base += gridDim.y * 128) {
      float v[4];
      add(v, c, c, stops[y], 1, base + x * 4);
      put(v, t, base + x * 4);
    }
  }
  if (!more) return;
  for (uint32_t i = 0; i < kJoin; ++i) {
    const uint32_t t = tokens[i], c = blockIdx.x * kJoin + i;
    if (t == kNone || stops[i] - c < kFew) continue;
    for (uint32_t base = blockIdx.y * 128; base < width; base += gridDim.y * 128) {
      float v[4];
      add(v, c, c + y, stops[i], kJoin, base + x * 4);
      __syncthreads();
      sums[y][x] = make_float4(v[0], v[1], v[2], v[3]);
      __syncthreads();
      if (y == 0) {
        for (int k = 1; k < (int)kJoin; ++k) {
          const float4 q = sums[k][x];
          v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
        }
        put(v, t, base + x * 4);
      }
    }
  }
}

void check_embedding(const fhe_embedding_args& a) {
  require(a.dtype == FHE_F32 || a.dtype == FHE_BF16 || a.dtype == FHE_F16, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
  require(a.out_dtype == a.dtype || a.out_dtype == FHE_F32, "out_dtype must be dtype or FHE_F32");
  require(a.count < (1u << 31) && a.vocab < (1u << 31), "count and vocab must be below 2^31");
  require(a.width >= 1 && a.width <= (1u << 20), "width must be in [1, 2^20]");
  require(a.scale - a.scale == 0.f, "scale must be finite");
}

// Calls f(T{}, Y{}) with the table's and the outputs' type.
template <class F>
void with_types(const fhe_embedding_args& a, F&& f) {
  with_type(a.dtype, [&](auto t) {
    if (a.out_dtype == FHE_F32) f(t, float{});
    else f(t, t);
  });
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Sorted positions to a block: fewer when there are few, so that every SM has some.
uint32_t chunk_of(uint32_t count) { return count >= 16384 ? 16 : 8; }

struct GradPlan {
  Sorted a, b;
  float* part;
  uint32_t chunk, chunks;
  uint64_t bytes;
};
GradPlan plan_of(const fhe_embedding_args& f, void* ws) {
  GradPlan p{};
  Carver c(ws);
  p.chunk = chunk_of(f.count);
  p.chunks = (f.count + p.chunk - 1) / p.chunk;
  p.a = {c.take<uint32_t>(f.count), c.take<uint32_t>(f.count)};
  if (f.count > kRun) p.b = {c.take<uint32_t>(f.count), c.take<uint32_t>(f.count)};
  p.part = c.take<float>((uint64_t)p.chunks * 2 * f.width);
  p.bytes = c.used;
  return p;
}

}  // namespace

void embedding(const fhe_embedding_args& a) {
  check_embedding(a);
  if (a.count == 0) return;
  require(a.ids && a.out && (a.table || a.vocab == 0), "null input or output");
  DeviceGuard dev(a.device);
  with_types(a, [&](auto t, auto y) {
    using T = decltype(t);
    using Y = decltype(y);
    constexpr int V = 16 / sizeof(Y);
    cudaStream_t st = static_cast<cudaStream_t>(a.stream);
    const bool vec = a.width % V == 0 && reinterpret_cast<uintptr_t>(a.table) % (V * sizeof(T)) == 0 && aligned16(a.out) &&
                     a.table_stride % V == 0;
    // four positions a warp once every SM has 32 warps
    const bool many = a.count >= 148 * 32 * 4;
    const uint32_t blocks = many ? (a.count + 15) / 16 : (a.count + 3) / 4;
    if (vec && many) k_embed<T, Y, V, 4><<<blocks, 128, 0, st>>>(a);
    else if (vec) k_embed<T, Y, V, 1><<<blocks, 128, 0, st>>>(a);
    else if (many) k_embed<T, Y, 1, 4><<<blocks, 128, 0, st>>>(a);
    else k_embed<T, Y, 1, 1><<<blocks, 128, 0, st>>>(a);
  });
  note_launch();
  FHE_CUDA(cudaGetLastError());
}

uint64_t embedding_backward_workspace(const fhe_embedding_grad_args& a) {
  check_embedding(a.f);
  return a.f.count ? plan_of(a.f, nullptr).bytes : 0;
}

void embedding_backward(const fhe_embedding_grad_args& a) {
  const fhe_embedding_args& f = a.f;
  check_embedding(f);
  require(f.count == 0 || (f.ids && a.dout), "null input");
  if (f.vocab == 0) return;
  require(a.dtable != nullptr, "null output");
  check_workspace(a.workspace, a.workspace_bytes, embedding_backward_workspace(a));
  DeviceGuard dev(f.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  const uint64_t bytes = (uint64_t)f.vocab * f.width * elem_size(f.dtype);
  if (f.count == 0) {
    FHE_CUDA(cudaMemsetAsync(a.dtable, 0, bytes, st));
    return;
  }
  GradPlan p = plan_of(f, a.workspace);
  const uint32_t runs = (f.count + kRun - 1) / kRun;
  // the table is cleared beside the launches that sort, a share each
  uint8_t* table = static_cast<uint8_t*>(a.dtable);
  uint32_t sorts = 1, share = 0;
  for (uint64_t run = kRun; run < f.count; run *= kMerge) ++sorts;
  auto fill = [&] {
    const uint64_t each = bytes / sorts / 16 * 16, from = each * share++, to = share == sorts ? bytes : each * share;
    return Fill{table + from, to - from, (uint32_t)std::min<uint64_t>(148 * 2, (to - from + 65535) / 65536)};
  };
  const Fill one = fill();
  k_sort<<<runs + one.blocks, kRun, 0, st>>>(f.ids, f.wide_ids, f.count, f.vocab, p.a, one);
  note_launch();
  Sorted s = p.a, other = p.b;
  const uint32_t own = (f.count + 31) / 32;
  static_assert(kRun == 1u << 8 && kMerge == 1u << 5, "powers of two");
  for (uint32_t log = 8; (1ull << log) < f.count; log += 5) {
    const Fill more = fill();
    k_merge<<<own + more.blocks, 32 * kMergeWarps, 0, st>>>(s, other, f.count, log, more);
    note_launch();
    std::swap(s, other);
  }
  with_types(f, [&](auto t, auto y) {
    using T = decltype(t);
    using Y = decltype(y);
    constexpr int V = 16 / sizeof(Y);
    const bool vec = f.width % V == 0 && aligned16(a.dout) && aligned16(a.dtable);
    const uint32_t per = vec ? V : 1, lanes = (f.width + per - 1) / per;
    const uint32_t tx = lanes <= 256 ? lanes : 256, ty = std::max(1u, 128 / tx);
    const dim3 grid((p.chunks + ty - 1) / ty, (lanes + tx - 1) / tx), block(tx, ty);
    if (vec) k_sum<T, Y, V><<<grid, block, 0, st>>>(a, s, p.chunk, p.chunks, p.part);
    else k_sum<T, Y, 1><<<grid, block, 0, st>>>(a, s, p.chunk, p.chunks, p.part);
    note_launch();
    if (p.chunks > 1) {
      const dim3 cover((p.chunks + kJoin - 1) / kJoin, std::min(8u, (f.width + 127) / 128));
      if (f.width % 4 == 0) k_join<T, true><<<cover, 256, 0, st>>>(a, s, p.chunk, p.chunks, p.part);
      else k_join<T, false><<<cover, 256, 0, st>>>(a, s, p.chunk, p.chunks, p.part);
      note_launch();
    }
  });
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
