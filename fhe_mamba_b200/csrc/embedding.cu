// Token embedding and its gradient (fhe_embedding).
//
// The lookup moves rows: a warp a row, 16 bytes a lane.  The gradient of a table
// row is the sum over the positions that hold its token, so positions are sorted
// by token: runs of 2048 in shared memory, then groups of 32 runs put together by
// rank (an element's place is its own index plus, for every other run, how many of
// its elements come before, found by halving), which waits for nothing and keeps
// equal tokens in the order of their positions.  Blocks of equally many sorted
// positions then sum the rows; a token that reaches past its block leaves partial
// sums, which a last launch adds in order.  No atomics: the same call gives the same
// bits.  Rows without a position are cleared by blocks beside those that sort.
#include <algorithm>

#include "launch_count.h"
#include "mamba_ops.h"

namespace fhe {
namespace {

constexpr uint32_t kRun = 2048, kMerge = 32, kSortThreads = 1024;
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

// One warp a position.  VEC: eight elements a lane and turn.
template <class T, class Y, bool VEC>
__global__ void __launch_bounds__(128) k_embed(const fhe_embedding_args g) {
  const uint32_t i = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (i >= g.count) return;
  const uint32_t t = token_of(g.ids, g.wide_ids, i, g.vocab);
  Y* out = static_cast<Y*>(g.out) + (int64_t)i * g.width;
  if (t == kNone) {
    const bool past = g.wide_ids ? static_cast<const int64_t*>(g.ids)[i] >= 0 : static_cast<const int32_t*>(g.ids)[i] >= 0;
    for (uint32_t c = lane; c < g.width; c += 32) out[c] = from_f<Y>(past ? NAN : 0.f);
    return;
  }
  const T* row = static_cast<const T*>(g.table) + (int64_t)t * g.table_stride;
  if constexpr (VEC) {
#pragma unroll 4
    for (uint32_t c = lane * 8; c < g.width; c += 256) {
      float f[8];
      Pack<T, 8> p;
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k)
        reinterpret_cast<uint4*>(&p)[k] = reinterpret_cast<const uint4*>(row + c)[k];
      unpack(p, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= g.scale;
      const Pack<Y, 8> q = pack<Y, 8>(f);
#pragma unroll
      for (int k = 0; k < (int)sizeof(Y) / 2; ++k)
        reinterpret_cast<uint4*>(out + c)[k] = reinterpret_cast<const uint4*>(&q)[k];
    }
  } else {
#pragma unroll 4
    for (uint32_t c = lane; c < g.width; c += 32) out[c] = from_f<Y>(to_f(row[c]) * g.scale);
  }
}

// The part `b` of `blocks` of the table's gradient, cleared by a block.
__device__ __forceinline__ void clear(uint8_t* p, uint64_t bytes, uint64_t b, uint64_t blocks) {
  const uint64_t head = min(bytes, (uint64_t)((0 - reinterpret_cast<uintptr_t>(p)) % 16)), words = (bytes - head) / 16;
  const uint64_t each = (words + blocks - 1) / blocks, first = min(words, b * each), last = min(words, first + each);
  uint4* w = reinterpret_cast<uint4*>(p + head);
#pragma unroll 4
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
  uint32_t blocks;  // behind the launch's own
};

// Blocks [0, runs) sort a run of positions by (token, position), the others clear.
__global__ void __launch_bounds__(kSortThreads) k_sort(const void* ids, bool wide, uint32_t count, uint32_t vocab,
                                                       uint32_t runs, Sorted out, Fill fill) {
  __shared__ uint64_t key[kRun];
  if (blockIdx.x >= runs) return clear(fill.p, fill.bytes, blockIdx.x - runs, fill.blocks);
  const uint32_t first = blockIdx.x * kRun, n = min(kRun, count - first);
  uint32_t size = 2;
  while (size < n) size *= 2;
  for (uint32_t i = threadIdx.x; i < size; i += kSortThreads)
    key[i] = i < n ? (uint64_t)token_of(ids, wide, first + i, vocab) << 32 | (first + i) : ~0ull;
  for (uint32_t span = 2; span <= size; span *= 2) {
    for (uint32_t step = span / 2; step; step /= 2) {
      __syncthreads();
      const uint32_t t = threadIdx.x;
      if (t >= size / 2) continue;
      const uint32_t a = 2 * t - (t & (step - 1)), b = a + step;
      const uint64_t x = key[a], y = key[b];
      if ((x > y) == ((a & span) == 0)) {
        key[a] = y;
        key[b] = x;
      }
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n; i += kSortThreads) {
    out.token[first + i] = (uint32_t)(key[i] >> 32);
    out.pos[first + i] = (uint32_t)key[i];
  }
}

// Tokens of p[0, n) below t, or not above it.
__device__ __forceinline__ uint32_t below(const uint32_t* p, uint32_t n, uint32_t t, bool or_equal) {
  uint32_t lo = 0;
  while (n) {
    const uint32_t half = n / 2, v = p[lo + half];
    const bool in = v < t || (or_equal && v == t);
    lo = in ? lo + half + 1 : lo;
    n = in ? n - half - 1 : half;
  }
  return lo;
}

// Puts groups of kMerge sorted runs of `run` elements together; blocks past `own` clear.
__global__ void __launch_bounds__(256) k_merge(Sorted in, Sorted out, uint32_t count, uint64_t run, uint32_t own, Fill fill) {
  if (blockIdx.x >= own) return clear(fill.p, fill.bytes, blockIdx.x - own, fill.blocks);
  const uint32_t e = blockIdx.x * 256 + threadIdx.x;
  if (e >= count) return;
  const uint64_t base = e / (run * kMerge) * (run * kMerge);
  const uint32_t mine = (uint32_t)((e - base) / run), t = in.token[e];
  uint64_t at = e - mine * run;
#pragma unroll 4
  for (uint32_t r = 0; r < kMerge; ++r) {
    const uint64_t first = base + r * run;
    if (first >= count) break;
    if (r != mine) at += below(in.token + first, (uint32_t)min(run, count - first), t, r < mine);
  }
  out.token[at] = t;
  out.pos[at] = in.pos[e];
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

// Adds the partial sums of the token that begins in a block of positions and
// reaches past it: strand y takes every eighth block, the strands follow in order.
template <class T>
__global__ void __launch_bounds__(256) k_join(const fhe_embedding_grad_args a, Sorted s, uint32_t chunk, uint32_t chunks,
                                              const float* part) {
  __shared__ float sums[8][33];
  const uint32_t c = blockIdx.x, count = a.f.count, width = a.f.width;
  const uint32_t first = c * chunk, next = first + chunk;
  if (next >= count) return;
  const uint32_t t = s.token[next - 1];
  if (t == kNone || s.token[next] != t) return;
  if (s.token[first] == t && first && s.token[first - 1] == t) return;  // began earlier
  const uint32_t end = next + below(s.token + next, count - next, t, true);
  const uint32_t stop = (end - 1) / chunk;  // the last block with a share
  for (uint32_t base = blockIdx.y * 32; base < width; base += gridDim.y * 32) {
    const uint32_t col = base + threadIdx.x;
    float v = 0.f;
    if (col < width) {
#pragma unroll 8
      for (uint32_t b = c + threadIdx.y; b <= stop; b += 8) v += part[((int64_t)b * 2 + (b == c)) * width + col];
    }
    __syncthreads();
    sums[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && col < width) {
      for (int i = 1; i < 8; ++i) v += sums[i][threadIdx.x];
      static_cast<T*>(a.dtable)[(int64_t)t * width + col] = from_f<T>(v * a.f.scale);
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
uint32_t chunk_of(uint32_t count) { return count >= 16384 ? 32 : 8; }

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
    const bool vec = a.width % 8 == 0 && aligned16(a.table) && aligned16(a.out) && a.table_stride % (16 / sizeof(T)) == 0;
    const uint32_t blocks = (a.count + 3) / 4;
    if (vec) k_embed<T, Y, true><<<blocks, 128, 0, static_cast<cudaStream_t>(a.stream)>>>(a);
    else k_embed<T, Y, false><<<blocks, 128, 0, static_cast<cudaStream_t>(a.stream)>>>(a);
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
  // half of the table is cleared beside each of the first two launches
  uint8_t* table = static_cast<uint8_t*>(a.dtable);
  const uint64_t here = runs == 1 ? bytes : bytes / 2 / 16 * 16;
  auto fill = [&](uint8_t* at, uint64_t n) {
    return Fill{at, n, (uint32_t)std::min<uint64_t>(148 * 2, (n + 65535) / 65536)};
  };
  const Fill one = fill(table, here), two = fill(table + here, bytes - here);
  k_sort<<<runs + one.blocks, kSortThreads, 0, st>>>(f.ids, f.wide_ids, f.count, f.vocab, runs, p.a, one);
  note_launch();
  Sorted s = p.a, other = p.b;
  const uint32_t own = (f.count + 255) / 256;
  for (uint64_t run = kRun; run < f.count; run *= kMerge) {
    const Fill more = run == kRun ? two : Fill{};
    k_merge<<<own + more.blocks, 256, 0, st>>>(s, other, f.count, run, own, more);
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
      k_join<T><<<dim3(p.chunks, std::min(8u, (f.width + 31) / 32)), dim3(32, 8), 0, st>>>(a, s, p.chunk, p.chunks, p.part);
      note_launch();
    }
  });
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
