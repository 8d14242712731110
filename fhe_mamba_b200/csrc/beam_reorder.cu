// Reordering of states after a selection (fhe_beam_reorder): row i of each batch
// item's beams becomes its row parents[i], in place, for every tensor at once.
//
// A thread owns the same 16 bytes of all of an item's rows: it brings the rows that
// others take into its own part of shared memory by asynchronous copies, waits for
// them, and then writes the rows that change.  So no thread reads what another
// writes, nothing waits for another thread, and only rows that change are written,
// only their parents read.  Memory bounds it.
#include <algorithm>

#include "launch_count.h"
#include "mamba_ops.h"

namespace fhe {
namespace {

constexpr uint32_t kMaxBeams = 64, kTable = 64;

struct State {
  uint8_t* p;
  uint64_t row;    // bytes
  uint32_t first;  // block of the grid
  uint32_t word;   // bytes that rows and base are multiples of, up to 16
};
struct ReorderArgs {
  State state[kTable];
  uint32_t n, beams;
  const int64_t* parents;
};

template <class W>
__device__ __forceinline__ void bring(W* to, const W* from) {
  if constexpr (sizeof(W) >= 4) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(sizeof(W)) : "memory");
  } else {
    *to = *from;
  }
}

// The block's 16 bytes a thread of each row, as words of type W.
template <class W>
__device__ __forceinline__ void move(uint8_t* base, uint64_t row, uint64_t at, uint32_t beams, const uint8_t* parent,
                                     uint64_t wanted, uint64_t changed, uint8_t* shared) {
  constexpr int N = 16 / sizeof(W);
  const uint32_t threads = blockDim.x, tid = threadIdx.x;
  auto each = [&](uint64_t rows, auto&& f) {
    for (; rows; rows &= rows - 1) f((uint32_t)__ffsll((long long)rows) - 1);
  };
  auto here = [&](uint32_t slot, int i) { return reinterpret_cast<W*>(shared) + ((uint64_t)slot * N + i) * threads + tid; };
  auto there = [&](int i) { return at + ((uint64_t)i * threads + tid) * sizeof(W); };
  uint32_t slot = 0;
  each(wanted, [&](uint32_t r) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (there(i) < row) bring(here(slot, i), reinterpret_cast<const W*>(base + r * row + there(i)));
    ++slot;
  });
  asm volatile("cp.async.wait_all;" ::: "memory");
  each(changed, [&](uint32_t r) {
    const uint32_t from = __popcll(wanted & ((1ull << parent[r]) - 1));
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (there(i) < row) *reinterpret_cast<W*>(base + r * row + there(i)) = *here(from, i);
  });
}

__global__ void __launch_bounds__(256) k_reorder(const __grid_constant__ ReorderArgs g) {
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ uint8_t parent[kMaxBeams];
  __shared__ uint64_t wanted, changed;
  const uint32_t tid = threadIdx.x, item = blockIdx.y, K = g.beams;
  if (tid == 0) wanted = changed = 0;
  __syncthreads();
  if (tid < K) {
    const int64_t p = g.parents[(int64_t)item * K + tid];
    if (p >= 0 && p < (int64_t)K && p != tid) {  // a row without a parent among the beams stays
      parent[tid] = (uint8_t)p;
      atomicOr(reinterpret_cast<unsigned long long*>(&wanted), 1ull << p);
      atomicOr(reinterpret_cast<unsigned long long*>(&changed), 1ull << tid);
    }
  }
  __syncthreads();
  if (changed == 0) return;
  uint32_t lo = 0, hi = g.n;  // the tensor of this block
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (blockIdx.x >= g.state[mid].first) lo = mid;
    else hi = mid;
  }
  const State& s = g.state[lo];
  const uint64_t at = (uint64_t)(blockIdx.x - s.first) * blockDim.x * 16;
  uint8_t* base = s.p + (uint64_t)item * K * s.row;
  if (s.word == 16) move<uint4>(base, s.row, at, K, parent, wanted, changed, shared);
  else if (s.word == 8) move<uint2>(base, s.row, at, K, parent, wanted, changed, shared);
  else if (s.word == 4) move<uint32_t>(base, s.row, at, K, parent, wanted, changed, shared);
  else if (s.word == 2) move<uint16_t>(base, s.row, at, K, parent, wanted, changed, shared);
  else move<uint8_t>(base, s.row, at, K, parent, wanted, changed, shared);
}

}  // namespace

void beam_reorder(const fhe_beam_reorder_args& a) {
  require(a.beams >= 1 && a.beams <= kMaxBeams, "beams must be in [1, 64]");
  require(a.batch <= 65535, "batch must be at most 65535");
  if (a.batch == 0 || a.count == 0 || a.beams == 1) return;
  require(a.states && a.row_bytes && a.parents, "null argument");
  for (uint32_t i = 0; i < a.count; ++i) {
    require(a.states[i] != nullptr || a.row_bytes[i] == 0, "null state");
    require(a.row_bytes[i] < (1ull << 36), "row too large");
  }
  DeviceGuard dev(a.device);
  // 16 bytes a thread and beam: 32 to 64 KB of shared memory to a block
  const uint32_t threads = a.beams <= 8 ? 256 : a.beams <= 16 ? 128 : 64;
  const uint32_t shared = threads * 16 * a.beams;
  if (shared > 32768)
    FHE_CUDA(cudaFuncSetAttribute(k_reorder, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared));
  for (uint32_t i = 0; i < a.count;) {
    ReorderArgs g{};
    g.beams = a.beams;
    g.parents = a.parents;
    uint64_t blocks = 0;
    for (; i < a.count && g.n < kTable; ++i) {
      const uint64_t row = a.row_bytes[i];
      if (row == 0) continue;
      const uint64_t more = (row + threads * 16 - 1) / (threads * 16);
      if (blocks + more >= (1ull << 31)) break;
      const uint64_t bits = row | reinterpret_cast<uintptr_t>(a.states[i]) | 16;
      g.state[g.n++] = State{static_cast<uint8_t*>(a.states[i]), row, (uint32_t)blocks, (uint32_t)(bits & (0 - bits))};
      blocks += more;
    }
    if (g.n == 0) continue;
    k_reorder<<<dim3((uint32_t)blocks, a.batch), threads, shared, static_cast<cudaStream_t>(a.stream)>>>(g);
    note_launch();
    FHE_CUDA(cudaGetLastError());
  }
}

}  // namespace fhe
